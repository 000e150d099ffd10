"""The memory operators without a GPU: struct layouts of the ctypes mirror, what the C entry points
and the Python functions refuse, and the 64-bit references against each other (the gated delta
rule in its chunked form, both gradients against differences)."""
import ctypes as C
import os
import subprocess

import pytest
import torch

from bluesky_gym import _native as nat
from bluesky_gym import memory
from memory_ref import attention_ref, delta_ref

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_struct_layouts_match_c(tmp_path):
    structs = {"bsg_rows": nat.BsgRows, "bsg_delta": nat.BsgDelta, "bsg_delta_act": nat.BsgDeltaAct, "bsg_attention": nat.BsgAttention,
               "bsg_attention_act": nat.BsgAttentionAct}
    lines = []
    for name, cls in structs.items():
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        lines += [f'printf("%zu\\n", offsetof({name}, {f[0]}));' for f in cls._fields_]
    prog = tmp_path / "layout.c"
    prog.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "bsg.h"\nint main(void) {\n'
                    + "\n".join(lines) + "\nreturn 0; }\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", os.path.join(REPO, "include"), "-o", str(exe), str(prog)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    want = []
    for cls in structs.values():
        want.append(C.sizeof(cls))
        want += [getattr(cls, f[0]).offset for f in cls._fields_]
    assert got == want


P = 1 << 20        # a pointer that is never followed: every call below is refused before a launch


def rows(p=P, env=64, step=64, head=64):
    return nat.BsgRows(p, env, step, head)


def delta_args(**kw):
    a = nat.BsgDelta(num_envs=2, steps=3, heads_k=1, heads_v=1, dim_k=64, dim_v=64, scale=1.0,
                     q=rows(), k=rows(), v=rows(), g=rows(), beta=rows(), out=rows(), dout=rows(), dq=rows(),
                     dk=rows(), dv=rows(), dg=rows(), dbeta=rows(), kept_states=P, kept_w=P, work_states=P, work_w=P)
    for n, x in kw.items():
        setattr(a, n, x)
    return a


def step_args(**kw):
    a = nat.BsgDeltaAct(num_envs=2, heads_k=1, heads_v=1, dim_k=64, dim_v=64, scale=1.0, q=rows(), k=rows(), v=rows(), g=rows(),
                        beta=rows(), out=rows(), state=P)
    for n, x in kw.items():
        setattr(a, n, x)
    return a


def attention_args(**kw):
    a = nat.BsgAttention(num_envs=2, steps=3, heads_q=2, heads_k=1, dim=64, scale=1.0, q=rows(), k=rows(), v=rows(),
                         out=rows(), dout=rows(), dq=rows(), dk=rows(), dv=rows(), lse=P, delta=P)
    for n, x in kw.items():
        setattr(a, n, x)
    return a


def act_args(**kw):
    a = nat.BsgAttentionAct(num_envs=1, slots=4096, heads_q=2, heads_k=1, dim=64, scale=1.0, q=rows(), k=rows(), v=rows(),
                            out=rows(), steps=P, k_cache=P, v_cache=P, work=P, work_bytes=1 << 40)
    for n, x in kw.items():
        setattr(a, n, x)
    return a


INVALID = -1
BAD_DELTA = [dict(num_envs=-1), dict(steps=-1), dict(heads_k=0), dict(heads_k=2, heads_v=3), dict(dim_k=48), dict(dim_v=256),
             dict(dtype=2), dict(gate_dtype=1), dict(dtype=1, gate_dtype=2), dict(num_envs=1 << 23), dict(q=rows(0)),
             dict(k=rows(P + 4)), dict(v=rows(env=3)), dict(g=rows(0)), dict(beta=rows(0))]


@pytest.mark.parametrize("kw", BAD_DELTA, ids=str)
def test_delta_entry_points_refuse(kw):
    lib = nat.load_library()
    assert lib.bsg_delta_forward(C.byref(delta_args(**kw)), None) == INVALID
    assert lib.bsg_delta_backward(C.byref(delta_args(**kw)), None) == INVALID
    if "steps" not in kw:
        assert lib.bsg_delta_step(C.byref(step_args(**kw)), None) == INVALID
    assert lib.bsg_last_error()


@pytest.mark.parametrize("fn,kw", [
    ("bsg_delta_forward", dict(out=rows(P + 8))), ("bsg_delta_forward", dict(kept_w=None)),
    ("bsg_delta_backward", dict(dq=rows(0))), ("bsg_delta_backward", dict(dv=rows(step=1))),
    ("bsg_delta_backward", dict(dbeta=rows(0))), ("bsg_delta_backward", dict(work_states=None)),
    ("bsg_delta_backward", dict(kept_w=P + 4)),
    ("bsg_delta_forward", dict(kept_states=P + 4)), ("bsg_delta_step", dict(state=None)), ("bsg_delta_step", dict(state=P + 4)),
    ("bsg_delta_step", dict(out=rows(P + 2)))], ids=str)
def test_delta_calls_refuse(fn, kw):
    args = step_args if fn == "bsg_delta_step" else delta_args
    assert getattr(nat.load_library(), fn)(C.byref(args(**kw)), None) == INVALID


@pytest.mark.parametrize("kw", [
    dict(num_envs=-1), dict(steps=-1), dict(window=-1), dict(heads_q=0), dict(heads_q=3, heads_k=2), dict(dim=16), dict(dtype=7),
    dict(softcap=-1.0), dict(softcap=float("nan")), dict(num_envs=1 << 23), dict(num_envs=1 << 20, steps=1000), dict(q=rows(0)), dict(k=rows(P + 2)), dict(out=rows(head=2)),
    dict(window=4), dict(first=P)], ids=str)
def test_attention_entry_points_refuse(kw):
    lib = nat.load_library()
    assert lib.bsg_attention_forward(C.byref(attention_args(**kw)), None) == INVALID
    assert lib.bsg_attention_backward(C.byref(attention_args(**kw)), None) == INVALID


@pytest.mark.parametrize("kw", [dict(lse=None), dict(delta=None), dict(dout=rows(0)), dict(dk=rows(P + 4)), dict(parts=P),
                                dict(steps=300), dict(steps=300, parts=P + 4), dict(steps=300, parts=P, dtype=1),
                                dict(out_rest=P + 2)], ids=str)
def test_attention_backward_refuses(kw):
    assert nat.load_library().bsg_attention_backward(C.byref(attention_args(**kw)), None) == INVALID


@pytest.mark.parametrize("kw", [
    dict(num_envs=-1), dict(slots=0), dict(slots=-5), dict(slots=(1 << 30) + 1), dict(heads_q=3, heads_k=2), dict(dim=65), dict(dtype=-1),
    dict(softcap=-1.0), dict(num_envs=1 << 23), dict(q=rows(0)), dict(out=rows(P + 8)), dict(steps=None), dict(k_cache=None), dict(v_cache=P + 2), dict(work=None),
    dict(work_bytes=16)], ids=str)
def test_attention_step_refuses(kw):
    assert nat.load_library().bsg_attention_step(C.byref(act_args(**kw)), None) == INVALID


def test_packed_blocks_are_the_structures():
    """The byte blocks that bluesky_gym.memory passes are the ctypes structures."""
    for cls in (nat.BsgDelta, nat.BsgDeltaAct, nat.BsgAttention, nat.BsgAttentionAct):
        flat = []
        for n, t in cls._fields_:
            flat += [len(flat) + i + 1 for i in range(4)] if t is nat.BsgRows else [len(flat) + 1]
        a = cls.from_buffer_copy(nat.packer(cls)(*flat))
        i = 0
        for n, t in cls._fields_:
            x = getattr(a, n)
            got = [x.p, x.env, x.step, x.head] if t is nat.BsgRows else [x]
            assert got == flat[i:i + len(got)], (cls.__name__, n)
            i += len(got)


def test_delta_work_is_wanted_where_rows_are_few():
    """Scratch for chunks solved beforehand: few envs x heads, more than one chunk."""
    lib = nat.load_library()
    need = lambda back=0, **kw: lib.bsg_delta_work_bytes(C.byref(delta_args(**kw)), back)  # noqa: E731
    assert need() == 0 and need(steps=64) == 0 and need(steps=65, dim_v=32) == 0 and need(steps=65, num_envs=4096) == 0
    assert need(steps=65) == 2 * 2 * (need(steps=65, num_envs=1) // 2) > 0 and need(steps=-1) == INVALID
    # and for the sums over value heads that share a key head, backward
    assert need(1, steps=64, heads_v=3) == 2 * 64 * 64 * 2 * 4 and need(0, steps=64, heads_v=3) == 0 and need(1, steps=64) == 0
    assert lib.bsg_delta_backward(C.byref(delta_args(steps=64, heads_v=3)), None) == INVALID
    for fn in ("bsg_delta_forward", "bsg_delta_backward"):
        assert getattr(lib, fn)(C.byref(delta_args(steps=65)), None) == INVALID
        assert getattr(lib, fn)(C.byref(delta_args(steps=65, work=P + 4)), None) == INVALID


def test_delta_work_holds_the_segments_of_long_rollouts():
    """From nine chunks on, few rows: a transition [dim_k][dim_k + dim_v] of fp32 per row and boundary."""
    lib = nat.load_library()
    need = lambda back=0, **kw: lib.bsg_delta_work_bytes(C.byref(delta_args(**kw)), back)  # noqa: E731
    chunk = need(steps=128) // 4                                       # two rows of two chunks
    for back in (0, 1):
        assert need(back, steps=512) == 2 * 8 * chunk
        assert need(back, steps=513) == 2 * 9 * chunk + 2 * 2 * 64 * 128 * 4
        assert need(back, steps=64 * 64, num_envs=255) == 255 * 64 * chunk      # rows for every CU: one segment


def test_parts_are_wanted_where_key_tiles_are_few():
    """By query head where shared key heads leave CUs idle, from bsg_attention_parts_bytes alone."""
    lib = nat.load_library()
    need = lambda **kw: lib.bsg_attention_parts_bytes(C.byref(attention_args(**kw)))  # noqa: E731
    assert need() == 0 and need(steps=64) == 0 and need(steps=65, heads_q=1) == 0
    assert need(steps=65) == 2 * 2 * 65 * 2 * 64 * 4
    assert need(steps=65, num_envs=4096) == 0
    assert need(steps=-1) == INVALID


def test_empty_calls_do_nothing_and_null_arguments_are_refused():
    lib = nat.load_library()
    assert lib.bsg_delta_forward(C.byref(delta_args(num_envs=0)), None) == 0
    assert lib.bsg_delta_backward(C.byref(delta_args(steps=0)), None) == 0
    assert lib.bsg_attention_forward(C.byref(attention_args(steps=0)), None) == 0
    assert lib.bsg_attention_step(C.byref(act_args(num_envs=0)), None) == 0
    for fn in ("bsg_delta_forward", "bsg_delta_backward", "bsg_delta_step", "bsg_attention_forward",
               "bsg_attention_backward", "bsg_attention_step"):
        assert getattr(lib, fn)(None, None) == INVALID


# ---- the Python functions -------------------------------------------------------------------

def delta_inputs(E=2, T=3, Hk=2, H=4, Dk=32, Dv=64, lead=None):
    lead = (E, T) if lead is None else lead
    z = lambda *s: torch.zeros(*lead, *s)  # noqa: E731
    return dict(q=z(Hk, Dk), k=z(Hk, Dk), v=z(H, Dv), g=z(H), beta=z(H))


BAD_RULE = [
    ("q", torch.zeros(2, 3, 2, 48)), ("q", torch.zeros(2, 3, 2, 32, dtype=torch.float16)), ("k", torch.zeros(2, 3, 1, 32)),
    ("v", torch.zeros(2, 3, 3, 64)), ("v", torch.zeros(2, 4, 4, 64)), ("v", torch.zeros(2, 3, 4, 48)), ("v", torch.zeros(2, 3, 0, 64)),
    ("g", torch.zeros(2, 3, 2)), ("g", torch.zeros(2, 3, 4, dtype=torch.bfloat16)), ("beta", torch.zeros(2, 3, 4, dtype=torch.float64)),
    ("state", torch.zeros(2, 4, 32, 32)), ("state", torch.zeros(2, 4, 32, 64, dtype=torch.bfloat16)),
    ("first", torch.zeros(2, 3)), ("first", torch.zeros(3, 2, dtype=torch.bool)),
    ("lengths", torch.zeros(2, dtype=torch.int64)), ("lengths", torch.zeros(3, dtype=torch.int32))]


@pytest.mark.parametrize("name,x", BAD_RULE, ids=lambda x: str(tuple(x.shape)) if torch.is_tensor(x) else x)
def test_gated_delta_rule_refuses(name, x):
    with pytest.raises(ValueError):
        memory.gated_delta_rule(**{**delta_inputs(), name: x})


def test_operators_need_a_hip_device():
    with pytest.raises(nat.BsgError):
        memory.gated_delta_rule(**delta_inputs())
    with pytest.raises(nat.BsgError):
        memory.gated_delta_step(**delta_inputs(lead=(2,)), state=torch.zeros(2, 4, 32, 64))
    x = torch.zeros(2, 3, 2, 32)
    with pytest.raises(nat.BsgError):
        memory.episode_attention(x, x, x)
    c = torch.zeros(2, 2, 5, 32)
    with pytest.raises(nat.BsgError):
        memory.episode_attention_step(x[:, 0], x[:, 0], x[:, 0], c, c.clone(), torch.zeros(2, dtype=torch.int32))


def test_gated_delta_step_refuses():
    good = delta_inputs(lead=(2,))
    for kw in (dict(state=None), dict(state=torch.zeros(2, 4, 64, 32)), dict(state=torch.zeros(2, 4, 32, 64, dtype=torch.float64)),
               dict(state=torch.zeros(2, 4, 32, 64), first=torch.zeros(2)),
               dict(state=torch.zeros(2, 4, 32, 64), q=torch.zeros(2, 3, 2, 32))):
        with pytest.raises(ValueError):
            memory.gated_delta_step(**{**good, **kw})


@pytest.mark.parametrize("kw", [
    dict(q=torch.zeros(2, 3, 3, 32)), dict(q=torch.zeros(2, 3, 4, 16)), dict(k=torch.zeros(2, 2, 2, 32)), dict(v=torch.zeros(2, 3, 2, 64)),
    dict(v=torch.zeros(2, 3, 2, 32, dtype=torch.bfloat16)), dict(first=torch.zeros(2, 3, dtype=torch.int32)),
    dict(lengths=torch.zeros(2))], ids=lambda k: next(iter(k)))
def test_episode_attention_refuses(kw):
    good = dict(q=torch.zeros(2, 3, 4, 32), k=torch.zeros(2, 3, 2, 32), v=torch.zeros(2, 3, 2, 32))
    with pytest.raises(ValueError):
        memory.episode_attention(**{**good, **kw})


@pytest.mark.parametrize("kw", [
    dict(k_cache=torch.zeros(2, 2, 0, 32)), dict(k_cache=torch.zeros(2, 5, 2, 32)), dict(v_cache=torch.zeros(2, 2, 6, 32)),
    dict(steps=torch.zeros(2, dtype=torch.int64)), dict(first=torch.zeros(3, dtype=torch.bool)), dict(k=torch.zeros(2, 1, 32))],
    ids=lambda k: next(iter(k)))
def test_episode_attention_step_refuses(kw):
    c = torch.zeros(2, 2, 5, 32)
    good = dict(q=torch.zeros(2, 4, 32), k=torch.zeros(2, 2, 32), v=torch.zeros(2, 2, 32), k_cache=c, v_cache=c.clone(),
                steps=torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError):
        memory.episode_attention_step(**{**good, **kw})


# ---- the references -------------------------------------------------------------------------

def make_delta(E, T, Hk, H, Dk, Dv, seed):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64)  # noqa: E731
    q, k = r(E, T, Hk, Dk), r(E, T, Hk, Dk)
    return (q / q.norm(dim=-1, keepdim=True), k / k.norm(dim=-1, keepdim=True), r(E, T, H, Dv),
            -torch.nn.functional.softplus(r(E, T, H) - 2), torch.sigmoid(r(E, T, H)), 0.3 * r(E, H, Dk, Dv))


def test_chunked_formula_is_the_recurrence():
    """The formulas in csrc/bsg_delta.hip's header for one chunk, against the recurrence."""
    T = 64
    q, k, v, g, beta, state = make_delta(1, T, 1, 1, 32, 32, 0)
    first = torch.zeros(1, T, dtype=torch.bool)
    first[0, [17, 40]] = True
    out, final = delta_ref(q, k, v, g, beta, state, first)
    q, k, v, g, b, S = q[0, :, 0], k[0, :, 0], v[0, :, 0], g[0, :, 0], beta[0, :, 0], state[0, 0]
    c, ep = g.cumsum(0), first[0].long().cumsum(0)
    G = torch.where((ep[:, None] == ep[None]) & (torch.arange(T)[:, None] >= torch.arange(T)[None]),
                    (c[:, None] - c[None]).exp(), torch.zeros((), dtype=torch.float64))
    N, P = (G * (k @ k.T)).tril(-1), G * (q @ k.T) * 32 ** -0.5
    enter, leave = c.exp() * (ep == 0), (c[-1] - c).exp() * (ep == ep[-1])
    W = torch.linalg.solve(torch.eye(T, dtype=torch.float64) + N * b[None], v - enter[:, None] * (k @ S))
    O = 32 ** -0.5 * enter[:, None] * (q @ S) + P @ (b[:, None] * W)
    assert torch.allclose(O, out[0, :, 0], atol=1e-12)
    S1 = (c[-1].exp() if ep[-1] == 0 else 0) * S + k.T @ (leave[:, None] * b[:, None] * W)
    assert torch.allclose(S1, final[0, 0], atol=1e-12)


def test_reference_gradients_match_differences():
    first = torch.zeros(2, 9, dtype=torch.bool)
    first[0, 4] = first[1, 0] = True
    lengths = torch.tensor([9, 6], dtype=torch.int32)
    xs = [x.requires_grad_(True) for x in make_delta(2, 9, 1, 2, 3, 2, 1)]
    assert torch.autograd.gradcheck(lambda *a: delta_ref(*a[:5], a[5], first, lengths), xs, atol=1e-6)
    gen = torch.Generator().manual_seed(2)
    qkv = [torch.randn(2, 9, h, 4, generator=gen, dtype=torch.float64).requires_grad_(True) for h in (2, 1, 1)]
    assert torch.autograd.gradcheck(
        lambda *a: attention_ref(*a, first, lengths, softcap=2.0, slopes=torch.tensor([0.3, 0.1]), window=4), qkv, atol=1e-6)
