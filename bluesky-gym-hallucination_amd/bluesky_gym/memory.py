"""Operators of a policy with memory, as fused HIP kernels (``bsg_delta_*`` and
``bsg_attention_*``, include/bsg.h; csrc/bsg_delta.hip, csrc/bsg_attention.hip): the sequence
layers a policy needs where one observation does not tell the state (the wind and uncertainty
wrappers, bluesky_gym/wrappers).  The reference's actors are feed-forward; these stand beside
``policy.SACPolicy``.

Two layers, each in two forms that compute the same function:

===========================  ======================================  ==========================
layer                        learns from rollouts (with gradients)   acts for one RL step
===========================  ======================================  ==========================
gated delta rule             :func:`gated_delta_rule`                :func:`gated_delta_step`
attention over the episode   :func:`episode_attention`               :func:`episode_attention_step`
===========================  ======================================  ==========================

Rollout tensors are ``[E, T, heads, dim]``: ``E`` envs, ``T`` steps.  Any strides serve; rollouts
collected step by step as ``[T, E, ...]`` are passed as ``x.transpose(0, 1)`` and read in place
(rows that are not contiguous, or not 16-byte aligned, are copied first).  fp32 or bf16, head
dims 32, 64 or 128, everything on one HIP device; sums, softmax statistics and states are fp32.

``first[e, t]`` (bool or uint8) says that step ``t`` is the first of an episode: nothing from
before it is seen.  ``lengths[e]`` (int32, in ``[0, T]``) ends the rollout of env ``e`` early: the
steps behind it are padding, never read, and their outputs and gradients are zero.  A non-finite
value may reach every output of its env's rollout, but no other env's.

Work is enqueued on the current stream of the tensors' device; all calls can be captured into a
HIP graph (a backward pass, as any in torch, once no eager graph of the same leaves is alive:
their gradients would be accumulated on that graph's stream).  ``first`` and ``lengths`` are read
again by the backward pass: they may not change in between.  Sums have a fixed order, so results
repeat bit for bit.  ``out=`` tensors may not overlap inputs.  No CPU fallback.
"""
from __future__ import annotations

from functools import lru_cache
from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from . import _native as nat

HEAD_DIMS = (32, 64, 128)
_DTYPES = {torch.float32: nat.F32, torch.bfloat16: nat.BF16}

__all__ = ["gated_delta_rule", "gated_delta_step", "episode_attention", "episode_attention_step"]


# ---- checks and views -----------------------------------------------------------------------

class _Layout(NamedTuple):
    """What of a tensor its checks look at, its address aside."""
    dtype: torch.dtype
    shape: torch.Size
    strides: tuple
    device: int                            # -1: not a HIP device

    def dim(self):
        return len(self.shape)


def _layout(x):
    return None if x is None else (x.dtype, x.shape, x.stride(), x.get_device())


def _layouts(who, **named):
    """Of several tensors, all on one HIP device; its index first."""
    ls = {n: None if x is None else _Layout(*x) for n, x in named.items()}
    at = ls["q"].device
    if at < 0:
        raise nat.BsgError(f"{who} runs on a HIP device (no CPU fallback)")
    for n, x in ls.items():
        if x is not None and x.device != at:
            raise ValueError(f"{who}: {n} is on device {x.device}, q is on {at}")
    return at


def _shape(who, name, x, shape, dtypes=None):
    if x.shape != shape:
        raise ValueError(f"{who}: {name} has shape {tuple(x.shape)}, expected {shape}")
    if dtypes is not None and x.dtype not in dtypes:
        raise ValueError(f"{who}: {name} has dtype {x.dtype}, expected one of {dtypes}")


_FP32, _INT32, _FLAGS = (torch.float32,), (torch.int32,), (torch.bool, torch.uint8)


def _heads(who, q, k, v, rank, **dims):
    """Type and shape of q, k, v; returns the dtype code."""
    if q.dim() != rank or k.dim() != rank or v.dim() != rank:
        raise ValueError(f"{who}: q, k and v must have {rank} axes")
    t = q.dtype
    if t not in _DTYPES or k.dtype != t or v.dtype != t:
        raise ValueError(f"{who}: q, k and v must share one dtype, float32 or bfloat16 "
                         f"(got {t}, {k.dtype}, {v.dtype})")
    for n, d in dims.items():
        if d not in HEAD_DIMS:
            raise ValueError(f"{who}: {n} must be 32, 64 or 128 (got {d})")
    return _DTYPES[t]


def _vector_strides(shape, s, size):
    """Whether rows of elements of `size` bytes keep to 16-byte vectors once the first one does."""
    m = 16 // size - 1
    if s[-1] != 1:
        return False
    either = 0
    for y in s[:-1]:
        either |= y
    # the strides of axes of one are not looked at
    return not either & m or all(n == 1 or not y & m for n, y in zip(shape[:-1], s[:-1]))


def _aligned(x):
    """Whether the kernels can read or write x's rows in 16-byte vectors."""
    return not x.data_ptr() & 15 and _vector_strides(x.shape, x.stride(), x.element_size())


def _vectors(x):
    return x if _aligned(x) else x.clone(memory_format=torch.contiguous_format)


def _row_strides(shape, s):
    """The strides of a bsg_rows: a rollout's [E, T, H, D], a gate's [E, T, H]."""
    return (s[0] if shape[0] > 1 else 0, s[1] if shape[1] > 1 else 0, s[2] if shape[2] > 1 else 0)


def _rows(x):
    return (x.data_ptr(), *_row_strides(x.shape, x.stride()))


def _new_strides(x):
    """The strides of a tensor made like one of this layout (the same where it is dense and its rows
    can be written, else contiguous), and a bsg_rows' of them."""
    size, strides = 1, x.strides
    for y, n in sorted((y, n) for y, n in zip(strides, x.shape) if n > 1):
        if y != size:                      # a gap or an overlap
            break
        size *= n
    if size != x.shape.numel() or not _vector_strides(x.shape, strides, x.dtype.itemsize):
        _, T, H, D = x.shape
        strides = (T * H * D, H * D, D, 1)
    return strides, _row_strides(x.shape, strides)


def _new(x, strides):
    return torch.empty_strided(x.shape, strides, dtype=x.dtype, device=x.device)


def _step_strides(x):
    """The strides of a bsg_rows of one step: a layout of [E, H, D], or a gate's [E, H]."""
    s, n = x.strides, x.shape
    return (s[0] if n[0] > 1 else 0, 0, s[1] if n[1] > 1 else 0)


_NO_ROWS = (0, 0, 0, 0)


def _ptr(x):
    return 0 if x is None else x.data_ptr()


def _numbers(who, scale, dim, softcap=0.0, window=0):
    if not 0.0 <= softcap < float("inf"):
        raise ValueError(f"{who}: softcap must be finite and >= 0 (0 = none), got {softcap}")
    if window < 0:
        raise ValueError(f"{who}: window must be >= 0 (0 = the whole episode), got {window}")
    return dim ** -0.5 if scale is None else float(scale)


def _slopes(who, slopes, heads):
    if slopes is None:
        return None
    _shape(who, "slopes", slopes, (heads,), _FP32)
    if slopes.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{who}: slopes are constants; they get no gradient")
    return slopes.contiguous()


def _no_grad(who, *xs):
    if torch.is_grad_enabled() and any(x.requires_grad for x in xs):
        raise ValueError(f"{who} has no gradient: act under torch.no_grad()")


# A call on a few envs is host time, so what follows from the layouts alone (checks, strides, sizes) is
# worked out once per combination of them (an acting step of 4 envs: attention 14.5 -> 9.8 us, delta rule
# 14.8 -> 8.9 us).  Addresses are looked at in every call.

_ROWS_OUT = "out must have contiguous, 16-byte aligned rows"


def _plan_out(who, out, like):
    """Strides of the output, or None: a contiguous one is made, and q, k and v are brought into order."""
    if out is not None:
        _shape(who, "out", out, like.shape, (like.dtype,))
        if not _vector_strides(*out[1:3], out.dtype.itemsize):
            raise ValueError(f"{who}: {_ROWS_OUT}")
        return _step_strides(out)
    row, head = like.shape[1] * like.shape[2], like.shape[2]
    return (row, 0, head) if like.strides == (row, head, 1) else None


def _make_out(who, out, like, strides):
    if out is None:
        out = torch.empty_like(like) if strides else torch.empty(like.shape, dtype=like.dtype, device=like.device)
    elif out.data_ptr() & 15:
        raise ValueError(f"{who}: {_ROWS_OUT}")
    return out


_raw_stream = torch._C._cuda_getCurrentRawStream   # current_stream(i).cuda_stream without the object


def _call(fn, block, i):
    """The launch goes to the tensors' device, on its current stream."""
    call = getattr(nat.load_library(), fn)
    if torch.cuda.current_device() == i:
        rc = call(block, _raw_stream(i))
    else:
        with torch.cuda.device(i):
            rc = call(block, _raw_stream(i))
    if rc:
        nat.check(rc, fn)


# ---- the gated delta rule -------------------------------------------------------------------

_pack_delta, _pack_delta_act = nat.packer(nat.BsgDelta), nat.packer(nat.BsgDeltaAct)


def _delta_check(who, q, k, v, g, beta, state, first, lead):
    Hk, Dk = q.shape[-2:]
    H, Dv = v.shape[-2:]
    _shape(who, "q", q, (*lead, Hk, Dk))
    _shape(who, "k", k, (*lead, Hk, Dk))
    if Hk < 1 or H < 1 or H % Hk:
        raise ValueError(f"{who}: {H} value heads do not share {Hk} key heads evenly")
    _shape(who, "g", g, (*lead, H), (torch.float32, q.dtype))
    _shape(who, "beta", beta, (*lead, H), (g.dtype,))
    if state is not None:
        _shape(who, "state", state, (lead[0], H, Dk, Dv), _FP32)
    if first is not None:
        _shape(who, "first", first, lead, _FLAGS)


@lru_cache(maxsize=256)
def _delta_sizes(E, T, Hk, H, Dk, Dv, dtype):
    """From the sizes alone: floats of kept_states and of kept_w, bytes of work forward and backward."""
    block = _pack_delta(E, T, Hk, H, Dk, Dv, dtype, dtype, 1.0, 0, *_NO_ROWS * 6, 0, 0, 0, 0, 0, 0, 0, 0, 0, *_NO_ROWS * 6, 0, 0, 0, 0)
    work = [nat.load_library().bsg_delta_work_bytes(block, back) for back in (0, 1)]
    for n in work:
        if n < 0:
            nat.check(n, "bsg_delta_work_bytes")
    rows = E * H * -(-T // nat.DELTA_CHUNK) * Dv
    return rows * Dk, rows * nat.DELTA_CHUNK, *work


class _Plan(NamedTuple):
    """What a learning call takes from its layouts."""
    head: tuple                            # the leading fields of its block
    device: int
    strides: tuple                         # of the tensors that the backward pass reads again
    vectors: bool                          # whether q, k and v are read as they are
    rows: list                             # their bsg_rows strides, and the gates'
    like: tuple                            # strides of what is made like q, k and v (_new),
    to: tuple                              # ... as bsg_rows has them (delta rule: and of the gates' gradients)
    first: tuple                           # strides
    sizes: tuple                           # of scratch
    key: tuple                             # the numbers the plan was made with


def _dense(*xs):
    return [None if x is None else x.contiguous() for x in xs]


def _strides(*xs):
    return tuple([None if x is None else x.stride() for x in xs])


@lru_cache(maxsize=256)
def _delta_plan(q, k, v, g, beta, state, first, lengths, scale):
    who = "gated_delta_rule"
    named = dict(q=q, k=k, v=v, g=g, beta=beta, state=state, first=first, lengths=lengths)
    q, k, v, g, beta, state, first, lengths = (None if x is None else _Layout(*x) for x in named.values())
    dtype = _heads(who, q, k, v, 4, Dk=q.shape[-1], Dv=v.shape[-1])
    E, T, H, Dv = v.shape
    _delta_check(who, q, k, v, g, beta, state, first, (E, T))
    if lengths is not None:
        _shape(who, "lengths", lengths, (E,), _INT32)
    device, Hk, Dk = _layouts(who, **named), q.shape[2], q.shape[3]
    like, to = zip(*(_new_strides(x) for x in (q, k, v)))
    return _Plan((E, T, Hk, H, Dk, Dv, dtype, _DTYPES[g.dtype], _numbers(who, scale, Dk), 0), device,
                 tuple([None if x is None else x.strides for x in (q, k, v, g, beta, first)]),
                 all(_vector_strides(x.shape, x.strides, x.dtype.itemsize) for x in (q, k, v)),
                 [_row_strides(x.shape, x.strides) for x in (q, k, v, g, beta)], like,
                 (*to, _row_strides(g.shape, (T * H, H, 1))), (0, 0) if first is None else first.strides,
                 _delta_sizes(E, T, Hk, H, Dk, Dv, dtype) if E and T else (), (scale,))


def _plan_again(plan, numbers, *xs):
    return plan(*[_layout(x) for x in xs], *numbers)


def _delta_inputs(p, q, k, v, g, beta, out, first, lengths):
    """The leading fields of bsg_delta, up to lengths."""
    r = p.rows
    return (*p.head, q.data_ptr(), *r[0], k.data_ptr(), *r[1], v.data_ptr(), *r[2], g.data_ptr(), *r[3],
            beta.data_ptr(), *r[4], *out, _ptr(first), *p.first, _ptr(lengths))


class _DeltaRule(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, g, beta, state, first, lengths, p, keep):
        if not p.vectors or (q.data_ptr() | k.data_ptr() | v.data_ptr()) & 15:
            q, k, v = _vectors(q), _vectors(k), _vectors(v)
            p = _plan_again(_delta_plan, p.key, q, k, v, g, beta, state, first, lengths)
        state = None if state is None else state.contiguous()
        E, T, Hk, H, Dk, Dv = p.head[:6]
        dev = v.device
        ns, nw, work, _ = p.sizes
        out = _new(v, p.like[2])
        final = torch.empty((E, H, Dk, Dv), dtype=torch.float32, device=dev)
        scratch = torch.empty(work, dtype=torch.uint8, device=dev) if work else None
        kept, at = None, (0, 0)
        if keep:                               # the states, then w
            kept = torch.empty(ns + nw, dtype=torch.float32, device=dev)
            at = kept.data_ptr(), kept.data_ptr() + 4 * ns
        _call("bsg_delta_forward", _pack_delta(
            *_delta_inputs(p, q, k, v, g, beta, (out.data_ptr(), *p.to[2]), first, lengths), _ptr(state),
            final.data_ptr(), *at, _ptr(scratch), *_NO_ROWS * 6, 0, 0, 0, 0), p.device)
        if keep:
            ctx.save_for_backward(q, k, v, g, beta, first, lengths, kept)
            ctx.plan = p
            ctx.set_materialize_grads(False)
        return out, final

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, dfinal):
        q, k, v, g, beta, first, *rest = ctx.saved_tensors
        lengths, kept = _dense(*rest)
        p = ctx.plan
        if _strides(q, k, v, g, beta, first) != p.strides:     # a saved tensor that came back in another order
            q, k, v = _vectors(q), _vectors(k), _vectors(v)
            p = _plan_again(_delta_plan, p.key, q, k, v, g, beta, None, first, lengths)
        E, T, Hk, H, Dk, Dv = p.head[:6]
        dev = v.device
        ns, nw, _, work = p.sizes
        dout = torch.zeros_like(v, memory_format=torch.contiguous_format) if dout is None else _vectors(dout)
        dfinal = None if dfinal is None else dfinal.contiguous()
        dq, dk, dv = _new(q, p.like[0]), _new(k, p.like[1]), _new(v, p.like[2])
        dg = torch.empty(g.shape, dtype=g.dtype, device=dev)
        db = torch.empty(beta.shape, dtype=beta.dtype, device=dev)
        dstate = torch.empty((E, H, Dk, Dv), dtype=torch.float32, device=dev) if ctx.needs_input_grad[5] else None
        scratch = torch.empty(4 * (ns + nw) + work, dtype=torch.uint8, device=dev)
        at, s, to = kept.data_ptr(), scratch.data_ptr(), p.to
        _call("bsg_delta_backward", _pack_delta(
            *_delta_inputs(p, q, k, v, g, beta, _NO_ROWS, first, lengths), 0, 0, at, at + 4 * ns, s + 4 * (ns + nw),
            *_rows(dout), dq.data_ptr(), *to[0], dk.data_ptr(), *to[1], dv.data_ptr(), *to[2], dg.data_ptr(), *to[3],
            db.data_ptr(), *to[3], _ptr(dfinal), _ptr(dstate), s, s + 4 * ns), p.device)
        return dq, dk, dv, dg, db, dstate, None, None, None, None


def gated_delta_rule(q, k, v, g, beta, state=None, first=None, lengths=None, *, scale=None):
    """The gated delta rule over a rollout: per env and value head, with a state ``S`` [Dk, Dv],

        S <- exp(g) S  (0 at a first step);  S <- S + beta k (v - S^T k)^T;  out = scale S^T q

    q, k [E, T, Hk, Dk]; v [E, T, Hv, Dv], Hv a multiple of Hk (key head h serves value heads
    h r .. h r + r - 1); g (log decay, <= 0) and beta [E, T, Hv], both in q's dtype or fp32;
    ``state`` fp32 [E, Hv, Dk, Dv] before the first step (None = 0).  Keys are used as given: make
    them unit vectors (beta in [0, 2] then keeps S from growing).  scale: Dk ** -0.5 by default.

    Returns ``out`` [E, T, Hv, Dv] and the state after the last step, fp32.  Differentiable once in
    q, k, v, g, beta and state."""
    if lengths is not None:
        lengths = lengths.contiguous()
    p = _delta_plan(_layout(q), _layout(k), _layout(v), _layout(g), _layout(beta), _layout(state), _layout(first),
                    _layout(lengths), None if scale is None else float(scale))
    E, T, Hk, H, Dk, Dv = p.head[:6]
    if E == 0 or T == 0:
        zero = torch.zeros((E, H, Dk, Dv), dtype=torch.float32, device=v.device)
        return v.clone(), zero if state is None else zero + state
    keep = torch.is_grad_enabled() and any(
        x is not None and x.requires_grad for x in (q, k, v, g, beta, state))
    return _DeltaRule.apply(q, k, v, g, beta, state, first, lengths, p, keep)


def gated_delta_step(q, k, v, g, beta, state, first=None, *, scale=None, out=None):
    """One RL step of the gated delta rule for a batch of envs, ``state`` updated in place.

    q, k [E, Hk, Dk]; v [E, Hv, Dv]; g, beta [E, Hv]; state fp32 [E, Hv, Dk, Dv], contiguous;
    ``first`` [E]: envs whose episode begins with this step (their state is forgotten, whatever it
    holds).  Returns out [E, Hv, Dv] (``out=`` to write into a given tensor).  No gradient: a
    learner replays the steps through :func:`gated_delta_rule`."""
    who = "gated_delta_step"
    if state is None:
        raise ValueError(f"{who}: state is updated in place and must be given")
    head, device, vectors, rows, to, first_env = _delta_step_plan(
        _layout(q), _layout(k), _layout(v), _layout(g), _layout(beta), _layout(state), _layout(first), _layout(out),
        None if scale is None else float(scale))
    _no_grad(who, q, k, v, g, beta, state)
    s = state.data_ptr()
    if s & 15:
        raise ValueError(f"{who}: {_STATE}")
    out = _make_out(who, out, v, to)
    if head[0] == 0:
        return out
    pq, pk, pv = q.data_ptr(), k.data_ptr(), v.data_ptr()
    if not vectors or (pq | pk | pv) & 15:
        return gated_delta_step(_vectors(q), _vectors(k), _vectors(v), g, beta, state, first, scale=scale, out=out)
    _call("bsg_delta_step", _pack_delta_act(
        *head, pq, *rows[0], pk, *rows[1], pv, *rows[2], g.data_ptr(), *rows[3], beta.data_ptr(), *rows[4],
        out.data_ptr(), *to, _ptr(first), first_env, s), device)
    return out


_STATE = "state must be contiguous and 16-byte aligned"


@lru_cache(maxsize=256)
def _delta_step_plan(q, k, v, g, beta, state, first, out, scale):
    who = "gated_delta_step"
    named = dict(q=q, k=k, v=v, g=g, beta=beta, state=state, first=first, out=out)
    q, k, v, g, beta, state, first, out = (None if x is None else _Layout(*x) for x in named.values())
    dtype = _heads(who, q, k, v, 3, Dk=q.shape[-1], Dv=v.shape[-1])
    E, H, Dv = v.shape
    _delta_check(who, q, k, v, g, beta, state, first, (E,))
    device = _layouts(who, **named)
    Dk = q.shape[2]
    if any(n > 1 and y != x for n, y, x in zip(state.shape, state.strides, (H * Dk * Dv, Dk * Dv, Dv, 1))):
        raise ValueError(f"{who}: {_STATE}")
    to = _plan_out(who, out, v)
    vectors = to is not None and all(_vector_strides(x.shape, x.strides, x.dtype.itemsize) for x in (q, k, v))
    return ((E, q.shape[1], H, Dk, Dv, dtype, _DTYPES[g.dtype], _numbers(who, scale, Dk)), device, vectors,
            [_step_strides(x) for x in (q, k, v, g, beta)], to, 0 if first is None else first.strides[0])


# ---- attention over the episode -------------------------------------------------------------

_pack_attention, _pack_attention_act = nat.packer(nat.BsgAttention), nat.packer(nat.BsgAttentionAct)


def _attention_block(p, q, k, v, slopes, first, lengths, begins, lse, rest, out, out_rows, grads=_NO_ROWS * 4, delta=0, parts=0):
    r = p.rows
    return _pack_attention(*p.head, q.data_ptr(), *r[0], k.data_ptr(), *r[1], v.data_ptr(), *r[2], out.data_ptr(), *out_rows,
                           _ptr(slopes), _ptr(first), *p.first, _ptr(lengths), _ptr(begins), _ptr(lse), _ptr(rest), *grads,
                           delta, parts)


@lru_cache(maxsize=256)
def _attention_parts(E, T, H, Hk, D, dtype):
    """Bytes of bsg_attention.parts, from the sizes alone."""
    r = (16, 0, 0, 0)                          # an address that is checked and never followed
    n = nat.load_library().bsg_attention_parts_bytes(
        _pack_attention(E, T, H, Hk, D, dtype, 0, 1.0, 0.0, 0, *r * 4, *[0] * 8, *_NO_ROWS * 4, 0, 0))
    if n < 0:
        nat.check(n, "bsg_attention_parts_bytes")
    return n


@lru_cache(maxsize=256)
def _attention_step_work(E, S, H, Hk, D, dtype):
    n = nat.load_library().bsg_attention_step_bytes(
        _pack_attention_act(E, S, H, Hk, D, dtype, 1.0, 0.0, *_NO_ROWS * 4, *[0] * 8))
    if n < 0:
        nat.check(n, "bsg_attention_step_bytes")
    return n


@lru_cache(maxsize=256)
def _attention_plan(q, k, v, first, lengths, slopes, scale, softcap, window):
    who = "episode_attention"
    named = dict(q=q, k=k, v=v, first=first, lengths=lengths, slopes=slopes)
    q, k, v, first, lengths, slopes = (None if x is None else _Layout(*x) for x in named.values())
    dtype = _heads(who, q, k, v, 4, D=q.shape[-1])
    E, T, H, D = q.shape
    Hk = k.shape[2]
    _shape(who, "k", k, (E, T, Hk, D))
    _shape(who, "v", v, (E, T, Hk, D))
    if Hk < 1 or H < 1 or H % Hk:
        raise ValueError(f"{who}: {H} query heads do not share {Hk} key heads evenly")
    if first is not None:
        _shape(who, "first", first, (E, T), _FLAGS)
    if lengths is not None:
        _shape(who, "lengths", lengths, (E,), _INT32)
    if slopes is not None:
        _shape(who, "slopes", slopes, (H,), _FP32)
    device = _layouts(who, **named)
    like, to = zip(*(_new_strides(x) for x in (q, k, v)))
    return _Plan((E, T, H, Hk, D, dtype, min(window, T), _numbers(who, scale, D, softcap, window), softcap, 0), device,
                 tuple([None if x is None else x.strides for x in (q, k, v, first)]),
                 all(_vector_strides(x.shape, x.strides, x.dtype.itemsize) for x in (q, k, v)),
                 [_row_strides(x.shape, x.strides) for x in (q, k, v)], like, to, (0, 0) if first is None else first.strides,
                 (_attention_parts(E, T, H, Hk, D, dtype) if E and T else 0,), (scale, softcap, window))


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, first, lengths, slopes, p, keep):
        if not p.vectors or (q.data_ptr() | k.data_ptr() | v.data_ptr()) & 15:
            q, k, v = _vectors(q), _vectors(k), _vectors(v)
            p = _plan_again(_attention_plan, p.key, q, k, v, first, lengths, slopes)
        E, T, H, Hk, D, dtype, window = p.head[:7]
        dev = q.device
        out = _new(q, p.like[0])
        begins = lse = rest = None
        if first is not None or window > 0:
            begins = torch.empty((E, T), dtype=torch.int32, device=dev)
        if keep:
            lse = torch.empty((E, H, T), dtype=torch.float32, device=dev)
            if dtype == nat.BF16 and T > nat.ATTENTION_TILE:
                rest = torch.empty((E, H, T, D), dtype=q.dtype, device=dev)
        _call("bsg_attention_forward",
              _attention_block(p, q, k, v, slopes, first, lengths, begins, lse, rest, out, p.to[0]), p.device)
        if keep:
            ctx.save_for_backward(q, k, v, slopes, first, lengths, begins, lse, rest, out)   # as _attention_block takes them
            ctx.plan = p
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, slopes, first, *more, out = ctx.saved_tensors
        slopes, lengths, begins, lse, rest = _dense(slopes, *more)
        p = ctx.plan
        if _strides(q, k, v, first) != p.strides:      # a saved tensor that came back in another order
            q, k, v = _vectors(q), _vectors(k), _vectors(v)
            p = _plan_again(_attention_plan, p.key, q, k, v, first, lengths, slopes)
        dout, out = _vectors(dout), _vectors(out)
        dq, dk, dv, delta = _new(q, p.like[0]), _new(k, p.like[1]), _new(v, p.like[2]), torch.empty_like(lse)
        need, to = p.sizes[0], p.to
        parts = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
        _call("bsg_attention_backward", _attention_block(
            p, q, k, v, slopes, first, lengths, begins, lse, rest, out, _row_strides(out.shape, out.stride()),
            (*_rows(dout), dq.data_ptr(), *to[0], dk.data_ptr(), *to[1], dv.data_ptr(), *to[2]), delta.data_ptr(),
            _ptr(parts)), p.device)
        return dq, dk, dv, None, None, None, None, None


def episode_attention(q, k, v, first=None, lengths=None, *, scale=None, softcap=0.0, slopes=None, window=0):
    """Attention of each step of a rollout to the steps of its episode so far, itself included:

        s_ij = scale q_i.k_j;  softcap tanh(s_ij / softcap) if softcap > 0;  - slopes[h] (i - j)
        out_i = sum_j softmax_j(s_ij) v_j

    q [E, T, Hq, D]; k, v [E, T, Hkv, D], Hq a multiple of Hkv (key head h serves query heads
    h r .. h r + r - 1).  ``slopes`` fp32 [Hq] (>= 0: older steps count less) or None.  ``window``:
    the number of last steps that are seen (0 = all of the episode).  scale: D ** -0.5 by default.
    Returns out [E, T, Hq, D].  Differentiable once in q, k and v."""
    who = "episode_attention"
    if lengths is not None:
        lengths = lengths.contiguous()
    p = _attention_plan(_layout(q), _layout(k), _layout(v), _layout(first), _layout(lengths), _layout(slopes),
                        None if scale is None else float(scale), float(softcap), int(window))
    slopes = _slopes(who, slopes, p.head[2])
    if q.numel() == 0:
        return q.clone()
    keep = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)
    return _Attention.apply(q, k, v, first, lengths, slopes, p, keep)


def episode_attention_step(q, k, v, k_cache, v_cache, steps, first=None, *, scale=None, softcap=0.0,
                           slopes=None, out=None):
    """One RL step of :func:`episode_attention` for a batch of envs, over a ring of the last
    steps' keys and values that the caller keeps: what ``episode_attention`` with
    ``window=slots`` gives for that step.

    q [E, Hq, D]; k, v [E, Hkv, D]; k_cache, v_cache [E, Hkv, slots, D], contiguous; ``steps``
    int32 [E]: the steps of the running episode before this one (zeros at the start).  ``first``
    [E]: envs whose episode begins with this step.  The step's key and value go into slot
    ``n % slots`` (n = steps, 0 at a first step) and ``steps`` becomes n + 1, in place; a slot that
    holds no step of the episode is not looked at, whatever it holds.  Returns out [E, Hq, D]
    (``out=`` to write into a given tensor).  No gradient."""
    who = "episode_attention_step"
    head, device, vectors, rows, to, first_env, need = _attention_step_plan(
        _layout(q), _layout(k), _layout(v), _layout(k_cache), _layout(v_cache), _layout(steps), _layout(first),
        _layout(slopes), _layout(out), None if scale is None else float(scale), float(softcap))
    _no_grad(who, q, k, v, k_cache, v_cache)
    pk, pv = k_cache.data_ptr(), v_cache.data_ptr()
    if (pk | pv) & 15:
        raise ValueError(f"{who}: k_cache and v_cache {_CACHE}")
    slopes = _slopes(who, slopes, head[2])
    out = _make_out(who, out, q, to)
    if head[0] == 0:
        return out
    at = q.data_ptr(), k.data_ptr(), v.data_ptr()
    if not vectors or (at[0] | at[1] | at[2]) & 15:
        return episode_attention_step(_vectors(q), _vectors(k), _vectors(v), k_cache, v_cache, steps, first,
                                      scale=scale, softcap=softcap, slopes=slopes, out=out)
    work = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
    _call("bsg_attention_step", _pack_attention_act(
        *head, at[0], *rows[0], at[1], *rows[1], at[2], *rows[2], out.data_ptr(), *to, _ptr(slopes), _ptr(first),
        first_env, steps.data_ptr(), pk, pv, _ptr(work), need), device)
    return out


_CACHE = "must be contiguous and 16-byte aligned"


@lru_cache(maxsize=256)
def _attention_step_plan(q, k, v, k_cache, v_cache, steps, first, slopes, out, scale, softcap):
    who = "episode_attention_step"
    named = dict(q=q, k=k, v=v, k_cache=k_cache, v_cache=v_cache, steps=steps, first=first, slopes=slopes, out=out)
    q, k, v, k_cache, v_cache, steps, first, slopes, out = (None if x is None else _Layout(*x) for x in named.values())
    dtype = _heads(who, q, k, v, 3, D=q.shape[-1])
    E, H, D = q.shape
    Hk = k.shape[1]
    _shape(who, "k", k, (E, Hk, D))
    _shape(who, "v", v, (E, Hk, D))
    if Hk < 1 or H < 1 or H % Hk:
        raise ValueError(f"{who}: {H} query heads do not share {Hk} key heads evenly")
    if k_cache.dim() != 4 or k_cache.shape[2] < 1:
        raise ValueError(f"{who}: k_cache must be [E, Hkv, slots, D] with at least one slot")
    S = k_cache.shape[2]
    _shape(who, "k_cache", k_cache, (E, Hk, S, D), (q.dtype,))
    _shape(who, "v_cache", v_cache, (E, Hk, S, D), (q.dtype,))
    _shape(who, "steps", steps, (E,), _INT32)
    if first is not None:
        _shape(who, "first", first, (E,), _FLAGS)
    if slopes is not None:
        _shape(who, "slopes", slopes, (H,), _FP32)
    device = _layouts(who, **named)
    for n, x, want in (("k_cache", k_cache, (Hk * S * D, S * D, D, 1)), ("v_cache", v_cache, (Hk * S * D, S * D, D, 1)),
                       ("steps", steps, (1,))):
        if any(i > 1 and y != z for i, y, z in zip(x.shape, x.strides, want)):
            raise ValueError(f"{who}: {n} {_CACHE}")
    to = _plan_out(who, out, q)
    vectors = to is not None and all(_vector_strides(x.shape, x.strides, x.dtype.itemsize) for x in (q, k, v))
    return ((E, S, H, Hk, D, dtype, _numbers(who, scale, D, softcap), softcap), device, vectors,
            [_step_strides(x) for x in (q, k, v)], to, 0 if first is None else first.strides[0],
            _attention_step_work(E, S, H, Hk, D, dtype))
