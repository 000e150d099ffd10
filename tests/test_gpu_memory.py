"""GPU checks of the memory operators (bluesky_gym.memory, csrc/bsg_delta.hip and
csrc/bsg_attention.hip) against their definitions in float64 (memory_ref), from the same rounded
inputs.

Error bounds, from the number of roundings on each path (u = half a step of the type: bf16 2^-8,
fp32 2^-24; e = 2^-24 for what is held in fp32):
 - attention: a score's dot product of D terms, its scaling, cap and bias are off by at most
   (D + 16) e of their magnitude, and p = e^s by twice that relatively (its own and the sum's), plus
   the sum over T keys; p (and ds) are rounded once to the operands' type.  With A = sum_j p_ij |v_j|
   and r = 2 max_j err(s_ij) + (T + 16) e:  |out - ref| <= u |ref| + (u + r) A.
   dv is the same sum over queries.  ds = p (dp - delta) c: its parts' magnitude is
   B = p (|do|.|v| + 2 |do|.A); delta takes out as it was rounded (u), c = 1 - y^2 the cap's
   derivative (its error is at most twice the score's): |ds err| <= (2 u + 3 r + (D + 16) e) B, and dq,
   dk are sums of it.  A p under 2^-126 is 0 in fp32: at most 2^9 such terms in a sum, each with
   factors |dp| + |delta| <= 2^10 and |k|, |q| <= 2^6, so 2^-100 in all (UNDER).
 - delta rule: fp32 chains of sums; a value passes at most 8 products (that of a boundary of
   segments among them), each a sum of up to 192 terms
   (a chunk's 64 and dim_k), so 8 * 192 e of the path's magnitude, taken as the largest
   entry of the output for that env and head, plus the growth along the rollout bounded by
   the same (unit keys, beta < 1: S does not grow).  With bf16 operands the values split into two
   parts are off by 2^-17 each: 8 * 2^-17.  Outputs are rounded once: u |ref|.  The returned states
   are fp32 sums of parts that hold 24 bits: the fp32 bound for both types.
   Gradients along the rollout pass both chains: twice the bound."""
import math

import pytest
import torch

from bluesky_gym import _native as nat
from bluesky_gym import config, core, memory
from memory_ref import U, attention_parts, attention_ref, d64, delta_ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
E24 = 2.0 ** -24
UNDER = 2.0 ** -100


def gen(seed):
    return torch.Generator().manual_seed(seed)


def flags(E, T, kind, g):
    if kind is None:
        return None
    if kind == "all":
        return torch.ones(E, T, dtype=torch.bool)
    if kind == "none":
        return torch.zeros(E, T, dtype=torch.bool)
    if kind == "edges":                    # at the borders of tiles and chunks
        f = torch.zeros(E, T, dtype=torch.bool)
        f[:, [t for t in (0, 15, 16, 63, 64, 127, 128) if t < T]] = True
        return f
    return torch.rand(E, T, generator=g) < float(kind)


def ends(E, T, kind, g):
    if kind is None:
        return None
    n = torch.randint(0, T + 1, (E,), generator=g, dtype=torch.int32)
    n[0] = 0
    if E > 1:
        n[1] = T
    return n


def rollout(x, order):
    """x [E, T, ...] on the GPU, stored env by env ("et"), step by step ("te"), or with gaps."""
    if order == "te":
        return x.transpose(0, 1).contiguous().to(DEV).transpose(0, 1)
    if order == "gap":
        E, T, H, D = x.shape
        y = torch.full((E, T + 1, H + 2, D + 16), float("nan"), dtype=x.dtype, device=DEV)
        y[:, :T, 1:H + 1, :D] = x.to(DEV)
        return y[:, :T, 1:H + 1, :D]
    if order == "odd":                     # rows that start at 4-byte places: copied by the function
        y = torch.empty(x.numel() + 1, dtype=x.dtype, device=DEV)
        y[1:] = x.to(DEV).reshape(-1)
        return y[1:].reshape(x.shape)
    return x.to(DEV)


def close(got, ref, tol, what):
    got = got.detach().double().cpu()
    assert got.shape == ref.shape, what
    assert torch.isfinite(got).all(), f"{what}: non-finite values"
    over = ((got - ref).abs() - tol - UNDER).max().item() if ref.numel() else 0.0
    assert over <= 0, f"{what}: {(got - ref).abs().max().item():.3g} off, {over:.3g} over the bound"


# ---- the gated delta rule -------------------------------------------------------------------

def delta_data(E, T, Hk, H, Dk, Dv, dtype, seed, gates=None):
    g = gen(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    q, k = r(E, T, Hk, Dk), r(E, T, Hk, Dk)
    gd = dtype if gates is None else gates
    return dict(q=(q / q.norm(dim=-1, keepdim=True)).to(dtype), k=(k / k.norm(dim=-1, keepdim=True)).to(dtype),
                v=r(E, T, H, Dv).to(dtype), g=(-torch.nn.functional.softplus(r(E, T, H) - 2)).to(gd),
                beta=torch.sigmoid(r(E, T, H)).to(gd)), r(E, T, H, Dv).to(dtype), 0.3 * r(E, H, Dk, Dv), g


def delta_tol(ref, dtype, lead, twice=False, state=False):
    """u |ref| + the path's bound times the largest entry, by env and head (`lead` leading axes kept)."""
    path = 8 * 192 * E24 + (0.0 if dtype == torch.float32 or state else 8 * 2.0 ** -17)
    dims = [d for d in range(ref.dim()) if d not in lead]
    top = ref.abs().amax(dims, keepdim=True) if ref.numel() else ref.abs()
    return (E24 if state else U[dtype]) * ref.abs() + (2 if twice else 1) * path * (top + 1e-3)


DELTA = [  # E, T, Hk, H, Dk, Dv, dtype, first, lengths, order, state, gates
    (1, 1, 1, 1, 32, 32, "fp32", None, None, "et", True, None),
    (2, 2, 1, 2, 64, 32, "bf16", None, None, "et", False, None),
    (3, 16, 2, 2, 64, 64, "fp32", "none", None, "te", True, None),
    (2, 17, 1, 3, 32, 64, "bf16", "0.2", None, "te", True, "fp32"),
    (2, 63, 1, 1, 128, 32, "fp32", "edges", None, "gap", True, None),
    (3, 64, 2, 4, 64, 64, "bf16", "all", None, "et", True, None),
    (3, 65, 1, 2, 32, 128, "fp32", "edges", "ragged", "te", True, None),
    (4, 130, 2, 2, 64, 64, "bf16", "0.03", "ragged", "gap", True, "fp32"),
    (2, 130, 1, 2, 128, 128, "bf16", "0.01", None, "te", True, None),
    (2, 129, 2, 4, 128, 64, "fp32", "0.05", "ragged", "odd", False, None),
    (2, 200, 1, 1, 128, 128, "fp32", None, None, "te", True, None),
    (1, 321, 1, 1, 64, 128, "bf16", "0.004", None, "odd", True, None),
    (5, 70, 4, 4, 32, 32, "bf16", None, "ragged", "et", True, None),
    # rows enough for every CU: chunks are solved in place
    (64, 70, 2, 4, 32, 64, "bf16", "0.03", "ragged", "te", True, None),
    (64, 66, 4, 4, 64, 64, "fp32", "0.05", None, "te", True, None),
    (86, 66, 1, 3, 32, 128, "bf16", None, None, "et", False, "fp32"),
    (65, 129, 4, 4, 32, 128, "fp32", "0.01", "ragged", "te", True, None),
    (129, 65, 1, 2, 128, 32, "bf16", "edges", None, "te", True, None),
    (260, 65, 1, 1, 128, 64, "bf16", None, "ragged", "te", True, None),
    (256, 65, 1, 1, 128, 128, "fp32", "0.1", None, "te", True, None),
    # few rows and many chunks: the rollout is cut into segments
    (1, 700, 2, 4, 128, 128, "bf16", None, None, "te", True, None),
    (3, 641, 1, 2, 32, 64, "fp32", "0.004", "ragged", "gap", True, "fp32"),
    (2, 1025, 1, 1, 64, 64, "bf16", "0.002", "ragged", "te", False, None),
    (2, 520, 1, 1, 128, 64, "fp32", None, None, "te", True, None),
    (4, 577, 2, 2, 32, 128, "bf16", "0.01", "ragged", "te", True, "fp32"),
    (2, 899, 1, 2, 64, 128, "fp32", "edges", None, "et", True, None),
]
DT = {"fp32": torch.float32, "bf16": torch.bfloat16}


@pytest.mark.parametrize("case", DELTA, ids=lambda c: "-".join(map(str, c)))
def test_gated_delta_rule(case):
    E, T, Hk, H, Dk, Dv, dt, fk, lk, order, with_state, gates = case
    dtype = DT[dt]
    x, dout, state, g = delta_data(E, T, Hk, H, Dk, Dv, dtype, 1000 + T, DT[gates] if gates else None)
    first, lengths = flags(E, T, fk, g), ends(E, T, lk, g)
    dfinal = torch.randn(E, H, Dk, Dv, generator=g)
    ref_in = {n: d64(v).requires_grad_(True) for n, v in x.items()}
    ref_state = d64(state).requires_grad_(True) if with_state else None
    out_r, fin_r = delta_ref(**ref_in, state=ref_state, first=first, lengths=lengths)
    leaves_r = list(ref_in.values()) + ([ref_state] if with_state else [])
    grads_r = torch.autograd.grad([out_r, fin_r], leaves_r, [d64(dout), d64(dfinal)])

    if lengths is not None:                # padding may hold anything
        pad = torch.arange(T)[None] >= lengths[:, None]
        for n in x:
            x[n] = x[n].masked_fill(pad.reshape(E, T, *[1] * (x[n].dim() - 2)), float("nan"))
        dout = dout.masked_fill(pad[:, :, None, None], float("inf"))
    dev = {n: (rollout(v, order) if v.dim() == 4 else rollout(v, "te")).requires_grad_(True) for n, v in x.items()}
    st = state.to(DEV).requires_grad_(True) if with_state else None
    f = None if first is None else first.transpose(0, 1).contiguous().to(DEV).transpose(0, 1)
    n = None if lengths is None else lengths.to(DEV)
    out, fin = memory.gated_delta_rule(**dev, state=st, first=f, lengths=n)
    assert out.dtype == dtype and fin.dtype == torch.float32
    close(out, out_r.detach(), delta_tol(out_r.detach(), dtype, (0, 2)), "out")
    close(fin, fin_r.detach(), delta_tol(fin_r.detach(), dtype, (0, 1), state=True), "final")
    grads = torch.autograd.grad([out, fin], list(dev.values()) + ([st] if with_state else []),
                                [rollout(dout, order), dfinal.to(DEV)])
    for name, got, ref in zip(list(x) + ["state"], grads, grads_r):
        own = got.dtype
        tol = delta_tol(ref, dtype, (0,) if name in ("q", "k") else (0, 1) if name == "state" else (0, 2), True,
                        state=name == "state")
        if own != dtype:                   # fp32 gates next to bf16 rows: the path's bound, not the type's
            assert own == torch.float32
        close(got, ref, tol, "d" + name)
    with torch.no_grad():                  # nothing is kept, the same values come out
        out2, fin2 = memory.gated_delta_rule(**dev, state=st, first=f, lengths=n)
    assert torch.equal(out2, out) and torch.equal(fin2, fin)


def test_gated_delta_rule_strong_decay_and_edge_gates():
    """Decays that leave nothing (-inf, -1e30), none (0), beta 0 and 1: the differences of far-run
    sums keep their precision, nothing overflows."""
    E, T = 2, 130
    x, dout, state, g = delta_data(E, T, 1, 1, 32, 32, torch.float32, 5)
    x["g"][0, 3::7] = -30.0
    x["g"][0, 20] = -math.inf
    x["g"][0, 90] = -1e30
    x["g"][1] = 0.0
    x["beta"][1, ::3] = 0.0
    x["beta"][1, 1::3] = 1.0
    ref = {n: d64(v).requires_grad_(True) for n, v in x.items()}
    out_r, fin_r = delta_ref(**ref, state=d64(state))
    dev = {n: v.to(DEV).requires_grad_(True) for n, v in x.items()}
    out, fin = memory.gated_delta_rule(**dev, state=state.to(DEV))
    close(out, out_r.detach(), delta_tol(out_r.detach(), torch.float32, (0, 2)), "out")
    close(fin, fin_r.detach(), delta_tol(fin_r.detach(), torch.float32, (0, 1), state=True), "final")
    got = torch.autograd.grad(out, list(dev.values()), dout.to(DEV))
    want = torch.autograd.grad(out_r, list(ref.values()), d64(dout))
    for name, a, b in zip(x, got, want):
        b = torch.nan_to_num(b)            # exp(-inf) 's own derivative is 0
        close(a, b, delta_tol(b, torch.float32, (0,), True), "d" + name)


def test_gated_delta_rule_gradients_match_differences():
    E, T = 2, 70
    x, dout, state, g = delta_data(E, T, 1, 2, 32, 32, torch.float32, 6)
    first = flags(E, T, "0.05", g)
    dev = {n: v.to(DEV).requires_grad_(True) for n, v in x.items()}
    out, _ = memory.gated_delta_rule(**dev, state=state.to(DEV), first=first.to(DEV))
    grads = torch.autograd.grad(out, list(dev.values()), dout.to(DEV))
    for name, gr in zip(x, grads):
        d = torch.randn(x[name].shape, generator=g, dtype=torch.float64)
        h, ref = 1e-5, {n: d64(v) for n, v in x.items()}
        f = [(delta_ref(**{**ref, name: ref[name] + s * h * d}, state=d64(state), first=first)[0] * d64(dout)).sum().item()
             for s in (1, -1)]
        want, got = (f[0] - f[1]) / (2 * h), (gr.double().cpu() * d).sum().item()
        # h^2 of the third derivative, and the gradient's bound times |d|_1 spread like a random walk
        assert abs(got - want) <= 2e-4 * (gr.double().norm().item() * d.norm().item()) + 1e-6, (name, got, want)


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("E,Hk,H,Dk,Dv", [(1, 1, 1, 32, 32), (5, 1, 3, 32, 128), (3, 2, 4, 64, 64), (2, 2, 2, 64, 32), (2, 1, 2, 128, 128), (3, 1, 1, 128, 64), (2, 1, 1, 32, 64), (2, 1, 1, 128, 32), (2, 1, 1, 64, 128)])
def test_gated_delta_step_is_the_rule(E, Hk, H, Dk, Dv, dt):
    """T acting steps give the rollout's outputs and state; a first step forgets a NaN state."""
    T, dtype = 9, DT[dt]
    x, _, state, g = delta_data(E, T, Hk, H, Dk, Dv, dtype, 7 + Dk)
    first = flags(E, T, "0.2", g)
    first[0, 0] = True
    out_r, fin_r = delta_ref(**{n: d64(v) for n, v in x.items()}, state=d64(state), first=first)
    dev, st = {n: v.to(DEV) for n, v in x.items()}, state.to(DEV)
    st[0] = float("nan")
    outs = []
    for t in range(T):
        outs.append(memory.gated_delta_step(**{n: v[:, t] for n, v in dev.items()}, state=st, first=first[:, t].to(DEV)))
    close(torch.stack(outs, 1), out_r, delta_tol(out_r, dtype, (0, 2)), "out")
    close(st, fin_r, delta_tol(fin_r, dtype, (0, 1), state=True), "state")


# ---- attention ------------------------------------------------------------------------------

def attention_data(E, T, H, Hk, D, dtype, seed, spread=1.0):
    g = gen(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    return dict(q=(spread * r(E, T, H, D)).to(dtype), k=(spread * r(E, T, Hk, D)).to(dtype), v=r(E, T, Hk, D).to(dtype)), \
        r(E, T, H, D).to(dtype), g


def attention_tols(x, dout, dtype, **kw):
    """Reference outputs and gradients with their bounds (the module's docstring)."""
    ref = {n: d64(v).requires_grad_(True) for n, v in x.items()}
    out, p, mag, (qh, kh, vh) = attention_parts(**ref, **kw)
    grads = torch.autograd.grad(out, list(ref.values()), dout)
    E, T, H, D = out.shape
    r_, u = H // ref["k"].shape[2], U[dtype]
    scale = D ** -0.5 if kw.get("scale") is None else kw["scale"]
    p, out = p.detach(), out.detach()
    kh, vh, qh = kh.detach(), vh.detach(), qh.detach()
    r = 2 * (D + 16) * E24 * mag.amax(-1, keepdim=True) + (T + 16) * E24            # [E, H, T, 1]
    A = (p @ vh.abs()).transpose(1, 2)
    tol_o = u * out.abs() + (u + r.transpose(1, 2)) * A
    do = dout.transpose(1, 2).abs()
    Bm = p * (do @ vh.abs().transpose(-1, -2) + 2 * (do * A.transpose(1, 2)).sum(-1, keepdim=True))
    ds = (2 * u + 3 * r + (D + 16) * E24) * Bm * abs(scale)
    share = lambda y: y.transpose(1, 2).reshape(E, T, H // r_, r_, D).sum(3)  # noqa: E731
    tol_q = u * grads[0].abs() + (ds @ kh.abs()).transpose(1, 2)
    tol_k = u * grads[1].abs() + share(ds.transpose(-1, -2) @ qh.abs())
    tol_v = u * grads[2].abs() + share(((u + r) * p).transpose(-1, -2) @ do)
    return (out, tol_o), [(g, t) for g, t in zip(grads, (tol_q, tol_k, tol_v))]


ATTEND = [  # E, T, H, Hk, D, dtype, first, lengths, order, softcap, bias, window, spread
    (1, 1, 1, 1, 32, "fp32", None, None, "et", 0.0, False, 0, 1.0),
    (2, 2, 2, 1, 64, "bf16", None, None, "te", 5.0, True, 0, 1.0),
    (3, 16, 4, 4, 64, "fp32", "none", None, "te", 0.0, True, 0, 1.0),
    (2, 17, 6, 2, 32, "bf16", "0.2", None, "te", 0.0, True, 5, 1.0),
    (2, 63, 3, 1, 128, "fp32", "edges", None, "gap", 2.0, True, 0, 1.0),
    (3, 64, 4, 2, 64, "bf16", "all", None, "et", 0.0, False, 0, 1.0),
    (3, 65, 8, 1, 64, "fp32", "edges", "ragged", "te", 0.0, True, 0, 1.0),
    (4, 130, 4, 2, 64, "bf16", "0.03", "ragged", "gap", 20.0, True, 64, 1.0),
    (2, 130, 2, 1, 128, "bf16", "0.01", None, "te", 0.0, False, 1, 1.0),
    (2, 129, 2, 2, 128, "fp32", "0.05", "ragged", "odd", 1.0, True, 65, 2.0),
    (1, 321, 4, 1, 128, "bf16", None, None, "odd", 0.0, True, 0, 3.0),
    (1, 300, 2, 2, 64, "fp32", "0.004", None, "te", 30.0, True, 200, 4.0),
    (5, 70, 5, 5, 32, "bf16", None, "ragged", "et", 0.0, False, 0, 8.0),
    # long rollouts; one key head of many envs, without partial sums
    (1, 600, 2, 1, 64, "bf16", "0.005", None, "te", 15.0, True, 0, 2.0),
    (2, 577, 2, 2, 128, "bf16", None, "ragged", "te", 0.0, False, 0, 2.0),
    (2, 530, 3, 1, 32, "bf16", "0.02", "ragged", "gap", 0.0, True, 100, 1.0),
    (350, 130, 2, 1, 32, "bf16", "0.05", "ragged", "te", 0.0, True, 0, 1.0),
    (350, 130, 2, 1, 32, "fp32", None, None, "te", 4.0, False, 0, 1.0),
]


@pytest.mark.parametrize("case", ATTEND, ids=lambda c: "-".join(map(str, c)))
def test_episode_attention(case):
    E, T, H, Hk, D, dt, fk, lk, order, cap, bias, window, spread = case
    dtype = DT[dt]
    x, dout, g = attention_data(E, T, H, Hk, D, dtype, 2000 + T, spread)
    first, lengths = flags(E, T, fk, g), ends(E, T, lk, g)
    slopes = 2.0 ** -torch.arange(1, H + 1).float() if bias else None
    kw = dict(first=first, lengths=lengths, softcap=cap, slopes=slopes, window=window)
    (out_r, tol_o), grads_r = attention_tols(x, d64(dout), dtype, **kw)
    if lengths is not None:
        pad = (torch.arange(T)[None] >= lengths[:, None])[:, :, None, None]
        x = {n: v.masked_fill(pad, float("nan")) for n, v in x.items()}
        dout = dout.masked_fill(pad, float("inf"))
    dev = {n: rollout(v, order).requires_grad_(True) for n, v in x.items()}
    on = {n: v.to(DEV) if torch.is_tensor(v) else v for n, v in kw.items()}
    if first is not None:
        on["first"] = first.transpose(0, 1).contiguous().to(DEV).transpose(0, 1)
    out = memory.episode_attention(**dev, **on)
    assert out.dtype == dtype
    close(out, out_r, tol_o, "out")
    for name, got, (ref, tol) in zip(x, torch.autograd.grad(out, list(dev.values()), rollout(dout, order)), grads_r):
        close(got, ref, tol, "d" + name)
    with torch.no_grad():
        assert torch.equal(memory.episode_attention(**dev, **on), out)


def test_episode_attention_gradients_match_differences():
    E, T, H = 2, 70, 2
    x, dout, g = attention_data(E, T, H, 1, 32, torch.float32, 8)
    kw = dict(first=flags(E, T, "0.05", g), softcap=3.0, slopes=torch.tensor([0.2, 0.05]), window=40)
    dev = {n: v.to(DEV).requires_grad_(True) for n, v in x.items()}
    out = memory.episode_attention(**dev, **{n: v.to(DEV) if torch.is_tensor(v) else v for n, v in kw.items()})
    for name, gr in zip(x, torch.autograd.grad(out, list(dev.values()), dout.to(DEV))):
        d = torch.randn(x[name].shape, generator=g, dtype=torch.float64)
        h, ref = 1e-5, {n: d64(v) for n, v in x.items()}
        f = [(attention_ref(**{**ref, name: ref[name] + s * h * d}, **kw) * d64(dout)).sum().item() for s in (1, -1)]
        want, got = (f[0] - f[1]) / (2 * h), (gr.double().cpu() * d).sum().item()
        assert abs(got - want) <= 2e-4 * (gr.double().norm().item() * d.norm().item()) + 1e-6, (name, got, want)


def test_broadcast_and_shared_inputs_get_summed_gradients():
    """One key/value head expanded over envs and steps: the gradient is the sum over what it served."""
    E, T, D = 3, 20, 32
    x, dout, g = attention_data(E, T, 2, 1, D, torch.float32, 9)
    k1, v1 = x["k"][:1, :1], x["v"][:1, :1]
    ref = [d64(k1).requires_grad_(True), d64(v1).requires_grad_(True)]
    out_r = attention_ref(d64(x["q"]), ref[0].expand(E, T, 1, D), ref[1].expand(E, T, 1, D))
    want = torch.autograd.grad(out_r, ref, d64(dout))
    dev = [k1.to(DEV).requires_grad_(True), v1.to(DEV).requires_grad_(True)]
    out = memory.episode_attention(x["q"].to(DEV), dev[0].expand(E, T, 1, D), dev[1].expand(E, T, 1, D))
    got = torch.autograd.grad(out, dev, dout.to(DEV))
    tol = E * T * 2 * (T + D + 32) * E24       # every summand's bound; |do|, |v| of a few
    for a, b in zip(got, want):
        close(a, b, torch.full_like(b, 8 * tol), "shared")


ACT = [  # E, S, H, Hk, D, dtype, softcap, bias
    (1, 1, 1, 1, 32, "fp32", 0.0, False), (3, 2, 2, 1, 64, "bf16", 4.0, True), (2, 7, 3, 3, 64, "fp32", 0.0, True),
    (3, 5, 6, 2, 128, "bf16", 0.0, True), (2, 9, 5, 1, 32, "fp32", 3.0, True), (2, 4, 8, 1, 128, "fp32", 0.0, False),
    (1, 6, 7, 7, 32, "bf16", 0.0, False)]


@pytest.mark.parametrize("case", ACT, ids=lambda c: "-".join(map(str, c)))
def test_episode_attention_step_is_the_rollout(case):
    """Acting steps over a ring that wraps give the rollout's outputs with window = slots; unheld
    slots hold NaN throughout."""
    E, S, H, Hk, D, dt, cap, bias = case
    T, dtype = 2 * S + 5, DT[dt]
    x, _, g = attention_data(E, T, H, Hk, D, dtype, 3000 + S)
    first = flags(E, T, "0.1", g)
    slopes = 2.0 ** -torch.arange(1, H + 1).float() if bias else None
    (out_r, tol), _ = attention_tols(x, torch.zeros(E, T, H, D, dtype=torch.float64), dtype, first=first, softcap=cap, slopes=slopes, window=S)
    kc = torch.full((E, Hk, S, D), float("nan"), dtype=dtype, device=DEV)
    vc = torch.full((E, Hk, S, D), float("inf"), dtype=dtype, device=DEV)
    steps = torch.zeros(E, dtype=torch.int32, device=DEV)
    outs, n = [], torch.zeros(E, dtype=torch.int32)
    for t in range(T):
        outs.append(memory.episode_attention_step(*(x[i][:, t].to(DEV) for i in "qkv"), kc, vc, steps, first[:, t].to(DEV),
                                                  softcap=cap, slopes=None if slopes is None else slopes.to(DEV)))
        n = torch.where(first[:, t], 0, n)
        for e in range(E):
            assert torch.equal(kc[e, :, n[e] % S].cpu(), x["k"][e, t]) and torch.equal(vc[e, :, n[e] % S].cpu(), x["v"][e, t])
        n += 1
        assert torch.equal(steps.cpu(), n)
    close(torch.stack(outs, 1), out_r, tol, "out")


@pytest.mark.parametrize("E,S,H,Hk,D,dt", [(1, 5000, 8, 2, 128, "bf16"), (2, 4097, 3, 1, 64, "fp32"), (3, 2048, 2, 2, 32, "bf16"), (40, 700, 2, 2, 64, "bf16")])
def test_episode_attention_step_long_ring(E, S, H, Hk, D, dt):
    """Rings long enough to be split over workgroups: full, part full, one short and one empty."""
    dtype, g = DT[dt], gen(S)
    q, k, v = (torch.randn(E, h, D, generator=g).to(dtype) for h in (H, Hk, Hk))
    kc, vc = (torch.randn(E, Hk, S, D, generator=g).to(dtype) for _ in range(2))
    steps = torch.tensor([S + 123, S // 2, 3][:E] + [S - 1] * (E - 3), dtype=torch.int32)
    first = torch.zeros(E, dtype=torch.bool)
    first[-1] = E > 1
    slopes = 2.0 ** -torch.arange(3, H + 3).float()
    n = torch.where(first, 0, steps)
    T = S
    # the held steps in order, as one rollout per env whose last row is this step
    want, tol = [], []
    for e in range(E):
        m = min(int(n[e]), S - 1)
        at = [(int(n[e]) - m + i) % S for i in range(m)]
        ks, vs = torch.cat([kc[e][:, at], k[e][:, None]], 1), torch.cat([vc[e][:, at], v[e][:, None]], 1)
        kh, vh = (d64(y).repeat_interleave(H // Hk, 0) for y in (ks, vs))
        s = (d64(q[e])[:, None] * kh).sum(-1) * D ** -0.5
        mag = (d64(q[e])[:, None].abs() * kh.abs()).sum(-1) * D ** -0.5
        bias = slopes.double()[:, None] * torch.arange(m, -1, -1)
        p = torch.softmax(s - bias, -1)
        want.append((p[..., None] * vh).sum(1))
        r = 2 * (D + 16) * E24 * (mag + bias).amax(-1, keepdim=True) + (T + 16) * E24
        tol.append(U[dtype] * want[-1].abs() + r * (p[..., None] * vh.abs()).sum(1))
    st = steps.to(DEV)
    kd, vd = kc.to(DEV), vc.to(DEV)
    for e in range(E):                     # what is not held may be anything
        kd[e, :, int(n[e]):] = float("nan")
        vd[e, :, int(n[e]):] = float("nan")
    out = memory.episode_attention_step(q.to(DEV), k.to(DEV), v.to(DEV), kd, vd, st, first.to(DEV), slopes=slopes.to(DEV))
    close(out, torch.stack(want), torch.stack(tol), "out")
    assert torch.equal(st.cpu(), n + 1)


def test_episode_attention_step_count_stays_at_its_largest():
    x = torch.randn(2, 1, 32, device=DEV)
    c = torch.randn(2, 1, 4, 32, device=DEV)
    steps = torch.tensor([2 ** 31 - 1, -5], dtype=torch.int32, device=DEV)
    memory.episode_attention_step(x, x, x, c, c.clone(), steps)
    assert steps.tolist() == [2 ** 31 - 1, 1]


# ---- as they are used -----------------------------------------------------------------------

def test_empty_batches():
    for dt in (torch.float32, torch.bfloat16):
        for E, T in ((0, 5), (3, 0)):
            q = torch.zeros(E, T, 2, 32, dtype=dt, device=DEV, requires_grad=True)
            gb = torch.zeros(E, T, 2, dtype=dt, device=DEV)
            st = torch.randn(E, 2, 32, 32, device=DEV, requires_grad=True)
            out, fin = memory.gated_delta_rule(q, q, q, gb, gb, st)
            assert out.shape == q.shape and torch.equal(fin, st)
            torch.autograd.grad([out.sum() + fin.sum()], [q, st])
            assert memory.episode_attention(q, q, q).shape == q.shape
        z = torch.zeros(0, 2, 32, dtype=dt, device=DEV)
        memory.gated_delta_step(z, z, z, z[..., 0], z[..., 0], torch.zeros(0, 2, 32, 32, device=DEV))
        c = torch.zeros(0, 2, 4, 32, dtype=dt, device=DEV)
        memory.episode_attention_step(z, z, z, c, c.clone(), torch.zeros(0, dtype=torch.int32, device=DEV))


def test_refusals_on_the_device():
    x = torch.zeros(2, 3, 2, 32, device=DEV)
    gb = torch.zeros(2, 3, 2, device=DEV)
    with pytest.raises(ValueError):
        memory.gated_delta_rule(x, x, x.cpu(), gb, gb)
    with pytest.raises(ValueError):
        memory.episode_attention(x, x, x, softcap=-1.0)
    with pytest.raises(ValueError):
        memory.episode_attention(x, x, x, softcap=float("inf"))
    with pytest.raises(ValueError):
        memory.episode_attention(x, x, x, window=-1)
    with pytest.raises(ValueError):
        memory.episode_attention(x, x, x, slopes=torch.zeros(2, device=DEV, requires_grad=True))
    with pytest.raises(ValueError):
        memory.episode_attention(x, x, x, slopes=torch.zeros(3, device=DEV))
    s = torch.zeros(2, 2, 32, 64, device=DEV)
    one = x[:, 0]
    with pytest.raises(ValueError):        # a view with gaps cannot be updated in place
        memory.gated_delta_step(one, one, one, gb[:, 0], gb[:, 0], s[..., :32])
    with pytest.raises(ValueError):
        memory.gated_delta_step(one.clone().requires_grad_(True), one, one, gb[:, 0], gb[:, 0], s[..., :32].contiguous())
    c = torch.zeros(2, 2, 4, 32, device=DEV)
    n = torch.zeros(2, dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError):
        memory.episode_attention_step(one, one, one, c.transpose(1, 2).contiguous().transpose(1, 2), c, n)
    with pytest.raises(ValueError):
        memory.episode_attention_step(one, one, one, c, c.clone(), n, out=torch.zeros(2, 2, 33, device=DEV)[..., :32])
    q = x.clone().requires_grad_(True)
    with pytest.raises(RuntimeError):      # differentiable once
        g1, = torch.autograd.grad(memory.episode_attention(q, x, x).square().sum(), q, create_graph=True)
        torch.autograd.grad(g1.sum(), q)


def layers(dtype, seed=11, O=40, H=4, D=64):
    """A small policy with memory over MergeEnv's 40-value observation rows: both layers, then the heads."""
    g = gen(seed)
    r = lambda *s: (torch.randn(*s, generator=g) / s[-1] ** 0.5).to(dtype).to(DEV)  # noqa: E731
    return {"emb": r(H * D, O), "qkv": r(3 * H * D, H * D), "gb": r(2 * H, H * D), "qkv2": r(3 * H * D, H * D), "mu": r(2, H * D)}


def project(p, x):
    H, D = 4, 64
    h = torch.tanh(x @ p["emb"].T)
    q, k, v = (h @ p["qkv"].T).reshape(*h.shape[:-1], 3, H, D).unbind(-3)
    q, k = torch.nn.functional.normalize(q, dim=-1), torch.nn.functional.normalize(k, dim=-1)
    g, b = (h @ p["gb"].T).chunk(2, -1)
    return h, q, k, v, -torch.nn.functional.softplus(g - 2), torch.sigmoid(b)


def project2(p, h):
    return (h @ p["qkv2"].T).reshape(*h.shape[:-1], 3, 4, 64).unbind(-3)


SLOPES = [0.5, 0.25, 0.125, 0.0625]


def learn(p, obs, first, state, window):
    h, q, k, v, g, b = project(p, obs)
    o, state = memory.gated_delta_rule(q, k, v, g, b, state, first)
    h = h + o.flatten(-2)
    a = memory.episode_attention(*project2(p, h), first, softcap=20.0, slopes=torch.tensor(SLOPES, device=DEV), window=window)
    return (h + a.flatten(-2)) @ p["mu"].T, state


def test_policy_with_memory_acts_as_it_learns():
    """Both layers in a policy that steps a MergeEnv batch: what it answered while acting (one RL
    step at a time, memories updated in place, episodes ending in between) is what the learner
    computes from the stored rollout, and the learner's gradients are those of the definitions."""
    E, T, S = 24, 70, 16                   # TimeLimit 50: every env starts at least one episode in between
    b = core.DeviceBatch(config.merge_config(num_ac=16), E, autoreset=nat.AUTORESET_SAME_STEP, compute_cd=False, seed=3)
    b.reset()
    p = layers(torch.float32)
    state = torch.zeros(E, 4, 64, 64, device=DEV)
    kc, vc = torch.zeros(E, 4, S, 64, device=DEV), torch.zeros(E, 4, S, 64, device=DEV)
    steps = torch.zeros(E, dtype=torch.int32, device=DEV)
    first = torch.ones(E, dtype=torch.uint8, device=DEV)
    slopes = torch.tensor(SLOPES, device=DEV)
    obs, firsts, acted = [], [], []
    with torch.no_grad():
        for _ in range(T):
            x = b.obs[:, :40].clone()
            h, q, k, v, g, bt = project(p, x)
            h = h + memory.gated_delta_step(q, k, v, g, bt, state, first).flatten(-2)
            h = h + memory.episode_attention_step(*project2(p, h), kc, vc, steps, first, softcap=20.0, slopes=slopes).flatten(-2)
            a = h @ p["mu"].T
            obs.append(x)
            firsts.append(first.clone())
            acted.append(a)
            b.step(torch.tanh(a).double())
            first = ((b.terminated != 0) | (b.truncated != 0)).to(torch.uint8)
    obs, firsts, acted = torch.stack(obs), torch.stack(firsts), torch.stack(acted)
    assert firsts[1:].any() and torch.isfinite(acted).all()
    for x in p.values():
        x.requires_grad_(True)
    out, fin = learn(p, obs.transpose(0, 1), firsts.transpose(0, 1), torch.zeros_like(state), S)
    # two fp32 computations of one function through ~6 layers of sums of up to 256 terms
    tol = 6 * 256 * E24 * max(1.0, acted.abs().max().item())
    assert (out.transpose(0, 1) - acted).abs().max().item() <= tol
    assert (fin - state).abs().max().item() <= 8 * 192 * E24 * max(1.0, state.abs().max().item())
    w = torch.randn(E, T, 2, generator=gen(4)).to(DEV)
    grads = torch.autograd.grad((out * w).sum(), list(p.values()))
    p64 = {n: d64(x).requires_grad_(True) for n, x in p.items()}
    f = firsts.transpose(0, 1).cpu().bool()
    h, q, k, v, g, bt = project(p64, d64(obs.transpose(0, 1)))
    o, _ = delta_ref(q, k, v, g, bt, None, f)
    h = h + o.flatten(-2)
    a = attention_ref(*project2(p64, h), first=f, softcap=20.0, slopes=torch.tensor(SLOPES), window=S)
    ref = torch.autograd.grad((((h + a.flatten(-2)) @ p64["mu"].T) * d64(w)).sum(), list(p64.values()))
    for n, x, y in zip(p, grads, ref):     # sums over E T = 1680 rows of values with the chain's bound
        assert (x.double().cpu() - y).norm() <= 2 * 6 * 256 * E24 * y.norm() * 10, n


def test_graph_capture_and_replay():
    """An acting step of both layers and a learner's pass with gradients, each captured into a graph
    and replayed three times with eager work in between: every replay equals the eager result."""
    E, T, H, D = 6, 80, 2, 64
    x, dout, g = attention_data(E, T, H, 1, D, torch.bfloat16, 21)
    dd, _, state, _ = delta_data(E, T, 1, H, D, D, torch.bfloat16, 22)
    first = flags(E, T, "0.05", g).to(DEV)
    lengths = torch.full((E,), T, dtype=torch.int32, device=DEV)
    att = {n: v.to(DEV).requires_grad_(True) for n, v in x.items()}
    dlt = {n: v.to(DEV).requires_grad_(True) for n, v in dd.items()}
    dout = dout.to(DEV)
    S = 600
    kc = torch.randn(2, 1, S, D, device=DEV).to(torch.bfloat16)
    vc = torch.randn(2, 1, S, D, device=DEV).to(torch.bfloat16)
    steps = torch.full((2,), 590, dtype=torch.int32, device=DEV)
    st0 = state.to(DEV)
    st = st0.clone()

    def learner():
        o1 = memory.episode_attention(**att, first=first, lengths=lengths, window=50)
        o2, fin = memory.gated_delta_rule(**dlt, first=first, lengths=lengths)
        return [o1.detach(), o2.detach(), fin.detach(),
                *torch.autograd.grad([o1, o2], list(att.values()) + list(dlt.values()), [dout, dout])]

    def actor():
        with torch.no_grad():
            a = memory.gated_delta_step(*(dlt[n].detach()[:, 0] for n in ("q", "k", "v", "g", "beta")), state=st)
            b = memory.episode_attention_step(att["q"].detach()[:2, 0], att["k"].detach()[:2, 0], att["v"].detach()[:2, 0], kc, vc, steps)
        return [a, b]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        learner(), actor()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = learner() + actor()
    for i in range(3):
        with torch.no_grad():
            for v in list(att.values()) + [dlt["v"]]:
                v.copy_(torch.randn(v.shape, generator=gen(50 + i)).to(v.dtype))
            first.copy_(torch.rand(E, T, generator=gen(60 + i)) < 0.05)
            lengths.copy_(torch.randint(1, T + 1, (E,), generator=gen(70 + i)))
            st.copy_(st0)
            kc0, vc0, n0 = kc.clone(), vc.clone(), steps.clone()
        want = learner() + actor()
        kc.copy_(kc0), vc.copy_(vc0), steps.copy_(n0), st.copy_(st0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, w in zip(captured, want):
            assert torch.equal(a, w)
        assert torch.equal(steps, n0 + 1)


def test_backward_twice_and_again_is_the_same():
    """A kept graph's second backward pass, and a second forward and backward, repeat bit for bit."""
    x, dout, g = attention_data(3, 200, 4, 2, 64, torch.bfloat16, 61)
    d, do2, state, _ = delta_data(3, 200, 2, 4, 64, 64, torch.bfloat16, 62)
    first = flags(3, 200, "0.02", g).to(DEV)
    a = {n: v.to(DEV).requires_grad_(True) for n, v in x.items()}
    b = {n: v.to(DEV).requires_grad_(True) for n, v in d.items()}
    runs = []
    for _ in range(2):
        o1 = memory.episode_attention(**a, first=first)
        o2, f = memory.gated_delta_rule(**b, state=state.to(DEV), first=first)
        for keep in (True, False):
            runs.append([o1.detach(), o2.detach(), f.detach(), *torch.autograd.grad(
                [o1, o2], list(a.values()) + list(b.values()), [dout.to(DEV), do2.to(DEV)], retain_graph=keep)])
    for r in runs[1:]:
        assert all(torch.equal(x, y) for x, y in zip(r, runs[0]))


def test_only_some_inputs_and_the_state_alone_need_gradients():
    d, dout, state, _ = delta_data(2, 70, 1, 2, 32, 32, torch.float32, 63)
    dev = {n: v.to(DEV) for n, v in d.items()}
    st = state.to(DEV).requires_grad_(True)
    out, fin = memory.gated_delta_rule(**dev, state=st)
    got, = torch.autograd.grad(fin.sum(), st)          # out takes no part: its gradient is None
    ref = {n: d64(v) for n, v in d.items()}
    sr = d64(state).requires_grad_(True)
    want, = torch.autograd.grad(delta_ref(**ref, state=sr)[1].sum(), sr)
    close(got, want, delta_tol(want, torch.float32, (0, 1), True, state=True), "dstate")
    x, do, _ = attention_data(2, 70, 2, 1, 32, torch.float32, 64)
    q, k, v = (x[n].to(DEV) for n in "qkv")
    v.requires_grad_(True)
    got, = torch.autograd.grad(memory.episode_attention(q, k, v), v, do.to(DEV))
    (_, _), grads = attention_tols(x, d64(do), torch.float32)
    close(got, *grads[2], "dv")


def test_nan_gate_is_not_hidden():
    d, _, state, _ = delta_data(2, 70, 1, 1, 32, 32, torch.float32, 65)
    d["g"][0, 40] = float("nan")
    dev = {n: v.to(DEV) for n, v in d.items()}
    out, fin = memory.gated_delta_rule(**dev, state=state.to(DEV))
    assert out[0, 40:].isnan().all() and fin[0].isnan().all()
    assert out[1].isfinite().all() and fin[1].isfinite().all()      # no other env's
    st = state.to(DEV)
    memory.gated_delta_step(*(dev[n][:, 40] for n in ("q", "k", "v", "g", "beta")), state=st)
    assert st[0].isnan().all() and st[1].isfinite().all()


def test_ring_whose_offsets_pass_32_bits():
    """More than 2^31 values to a ring: the last slots are found, the step goes where it belongs."""
    S, D = 34_000_000, 64
    kc = torch.zeros(1, 1, S, D, dtype=torch.bfloat16, device=DEV)
    vc = torch.zeros(1, 1, S, D, dtype=torch.bfloat16, device=DEV)
    q = torch.ones(1, 1, D, dtype=torch.bfloat16, device=DEV)
    kc[0, 0, S - 2] = 40 * D ** 0.5 / D                # score 40: e^40 against S e^0
    vc[0, 0, S - 2] = 3.0
    steps = torch.tensor([S - 1], dtype=torch.int32, device=DEV)
    out = memory.episode_attention_step(q, torch.zeros_like(q), torch.full_like(q, 5.0), kc, vc, steps)
    assert (out.float() - 3.0).abs().max().item() <= 3 * 2.0 ** -8 and steps.item() == S
    assert (vc[0, 0, S - 1] == 5).all() and (vc[0, 0, S - 2] == 3).all() and not vc[0, 0, :4].any()


def test_side_stream_and_two_calls_in_flight():
    """Two learners on two streams at once, each with its own workspaces."""
    E, T = 64, 128
    sets, want = [], []
    for i in range(2):
        x, _, g = attention_data(E, T, 4, 2, 64, torch.bfloat16, 31 + i)
        d, _, _, _ = delta_data(E, T, 2, 4, 64, 64, torch.bfloat16, 41 + i)
        sets.append(({n: v.to(DEV).requires_grad_(True) for n, v in x.items()}, {n: v.to(DEV).requires_grad_(True) for n, v in d.items()}))

    def go(a, d):
        o1 = memory.episode_attention(**a, window=30)
        o2, f = memory.gated_delta_rule(**d)
        return [o1.detach(), o2.detach(), f.detach(), *torch.autograd.grad([o1, o2], list(a.values()) + list(d.values()), [torch.ones_like(o1), torch.ones_like(o2)])]

    want = [go(*s) for s in sets]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in sets], []
    for s, st in zip(sets, streams):
        with torch.cuda.stream(st):
            got.append(go(*s))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_out_tensors_are_written_in_place():
    x, _, g = attention_data(3, 2, 2, 1, 64, torch.float32, 51)
    big = torch.full((3, 4, 64), -7.0, device=DEV)
    c = torch.zeros(3, 1, 4, 64, device=DEV)
    got = memory.episode_attention_step(x["q"][:, 0].to(DEV), x["k"][:, 0].to(DEV), x["v"][:, 0].to(DEV), c, c.clone(),
                                        torch.zeros(3, dtype=torch.int32, device=DEV), out=big[:, 1:3])
    assert got.data_ptr() == big[:, 1:3].data_ptr()
    assert (big[:, 0] == -7).all() and (big[:, 3] == -7).all()
    assert torch.equal(big[:, 1:3].cpu(), x["v"][:, 0].expand(3, 2, 64))


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
def test_acting_calls_look_at_every_address_and_number(dt):
    """What is known of a call's layouts from the one before says nothing of its addresses, scale or cap."""
    dtype, g = DT[dt], gen(77)
    r = lambda *s: torch.randn(*s, generator=g).to(dtype).to(DEV)  # noqa: E731
    shift = lambda x: torch.cat([x.new_zeros(1), x.reshape(-1)])[1:].view(x.shape)  # noqa: E731  (one element further)
    q, k, v = r(3, 2, 64), r(3, 2, 64), r(3, 2, 64)
    gates = -torch.rand(3, 2, generator=g).to(DEV), torch.rand(3, 2, generator=g).to(DEV)
    S, caches = torch.randn(3, 2, 64, 64, generator=g).to(DEV), (r(3, 2, 7, 64), r(3, 2, 7, 64))

    def delta(q, k, v, state=None, **kw):
        state = S.clone() if state is None else state
        return memory.gated_delta_step(q, k, v, *gates, state, **kw), state

    def attend(q, k, v, kc=None, **kw):
        kc, vc = caches[0].clone() if kc is None else kc, caches[1].clone()
        steps = torch.full((3,), 5, dtype=torch.int32, device=DEV)
        return memory.episode_attention_step(q, k, v, kc, vc, steps, **kw), kc, vc, steps

    for act, kw in ((delta, dict(scale=0.3)), (attend, dict(scale=0.3)), (attend, dict(softcap=0.5))):
        plain, other = act(q, k, v), act(q, k, v, **kw)
        assert not torch.equal(plain[0], other[0])
        for args in ((shift(q), k, v), (q, shift(k), v), (q, k, shift(v)), (q, k, v)):
            assert all(torch.equal(a, b) for a, b in zip(act(*args), plain))
            assert all(torch.equal(a, b) for a, b in zip(act(*args, **kw), other))
        assert torch.equal(act(q, k, v, out=torch.empty_like(q))[0], plain[0])
        gap = torch.zeros(3, 4, 64, dtype=dtype, device=DEV)[:, ::2]
        assert torch.equal(act(q, k, v, out=gap)[0], plain[0]) and gap.stride() == (256, 128, 1)
        turned = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v)]
        assert all(torch.equal(a, b) for a, b in zip(act(*turned), plain))
        with pytest.raises(ValueError):
            act(q, k, v, out=shift(torch.empty_like(q)))
    with pytest.raises(ValueError):
        delta(q, k, v, state=shift(S))
    with pytest.raises(ValueError):
        attend(q, k, v, kc=shift(caches[0]))


def test_saved_tensors_in_another_order():
    """A hook on saved tensors may give them back with other strides: the gradients stay the same."""
    x, dout, g = attention_data(2, 70, 2, 1, 64, torch.bfloat16, 5)
    d, ddout, state, g = delta_data(2, 70, 1, 2, 64, 64, torch.float32, 6)
    first = flags(2, 70, "0.05", g).to(DEV)
    turn = lambda t: t.transpose(0, 1).contiguous().transpose(0, 1) if t.dim() in (2, 3, 4) and t.shape[1] == 70 else t  # noqa: E731
    dev = lambda y: {n: t.to(DEV).requires_grad_(True) for n, t in y.items()}  # noqa: E731
    for call, y, go in ((lambda y: memory.episode_attention(**y, first=first, window=40), x, dout),
                        (lambda y: memory.gated_delta_rule(**y, state=state.to(DEV), first=first)[0], d, ddout)):
        y = dev(y)
        want = torch.autograd.grad(call(y), list(y.values()), go.to(DEV))
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, turn):
            out = call(y)
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, list(y.values()), go.to(DEV)), want))


def test_segments_replay_with_lengths_that_end_at_their_boundaries():
    """A long rollout's learning call captured once and replayed for other lengths, two graphs in turn."""
    E, T = 3, 700
    d, dout, state, g = delta_data(E, T, 1, 2, 64, 64, torch.bfloat16, 91)
    first = flags(E, T, "0.003", g).to(DEV)
    lengths = torch.full((E,), T, dtype=torch.int32, device=DEV)
    x, dout, state = {n: v.to(DEV).requires_grad_(True) for n, v in d.items()}, dout.to(DEV), state.to(DEV).requires_grad_(True)

    def learner():
        o, fin = memory.gated_delta_rule(**x, state=state, first=first, lengths=lengths)
        return [o.detach(), fin.detach(), *torch.autograd.grad([o, fin], [*x.values(), state], [dout, state.detach()])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        learner()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    captured = []
    for graph in graphs:
        with torch.cuda.graph(graph):
            captured.append(learner())
    for n in ((T, 0, 1), (256, 257, 255), (512, 640, 699), (64, 192, 384)):
        lengths.copy_(torch.tensor(n, dtype=torch.int32))
        want = learner()
        torch.cuda.synchronize()
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for got in captured:
            assert all(torch.equal(a, w) for a, w in zip(got, want))
        for e in range(E):
            assert not want[0][e, n[e]:].any() and (n[e] > 0 or torch.equal(want[1][e], state[e]))
