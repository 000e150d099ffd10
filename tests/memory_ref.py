"""The memory operators from their definitions, in float64 on the CPU: the gated delta rule step
by step, attention as a masked softmax.  Gradients come from autograd over these."""
import math

import torch

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}     # half a step of the type


def d64(x):
    return None if x is None else x.detach().cpu().double()


def delta_ref(q, k, v, g, beta, state=None, first=None, lengths=None, scale=None):
    E, T, Hk, Dk = q.shape
    H, Dv = v.shape[2], v.shape[3]
    r = H // Hk
    scale = Dk ** -0.5 if scale is None else scale
    S = torch.zeros(E, H, Dk, Dv, dtype=torch.float64) if state is None else state
    outs = []
    for t in range(T):
        on = torch.ones(E, dtype=torch.bool) if lengths is None else t < lengths.cpu()
        new = torch.zeros(E, dtype=torch.bool) if first is None else first[:, t].cpu().bool()
        # padding may hold anything: nothing is computed from it
        pick = lambda x: torch.where(on.reshape(-1, *[1] * (x.dim() - 2)), x[:, t], torch.zeros((), dtype=torch.float64))  # noqa: E731
        qt, kt = pick(q).repeat_interleave(r, 1), pick(k).repeat_interleave(r, 1)
        D = torch.where(new[:, None, None, None], torch.zeros((), dtype=torch.float64), S) * pick(g).exp()[..., None, None]
        w = pick(v) - torch.einsum("ehkv,ehk->ehv", D, kt)
        D = D + kt[..., :, None] * (pick(beta)[..., None] * w)[..., None, :]
        o = scale * torch.einsum("ehkv,ehk->ehv", D, qt)
        outs.append(torch.where(on[:, None, None], o, torch.zeros((), dtype=torch.float64)))
        S = torch.where(on[:, None, None, None], D, S)
    return torch.stack(outs, 1), S


def seen_ref(E, T, first, lengths, window):
    t = torch.arange(T)
    ago = t[:, None] - t[None, :]
    ep = torch.zeros(E, T) if first is None else first.cpu().long().cumsum(1)
    n = torch.full((E,), T) if lengths is None else lengths.cpu().long()
    see = (ago >= 0) & (ep[:, :, None] == ep[:, None, :]) & (t[None, :, None] < n[:, None, None])
    return (see & (ago < window)) if window else see


def attention_parts(q, k, v, first=None, lengths=None, scale=None, softcap=0.0, slopes=None, window=0):
    """out, the probabilities [E, Hq, T, T] and the scores' magnitudes (for the error bounds)."""
    E, T, H, D = q.shape
    r = H // k.shape[2]
    scale = D ** -0.5 if scale is None else scale
    n = torch.full((E,), T) if lengths is None else lengths.cpu().long()
    ok = (torch.arange(T)[None] < n[:, None])[:, :, None, None]
    zero = torch.zeros((), dtype=torch.float64)
    q, k, v = (torch.where(ok, x, zero) for x in (q, k, v))
    kh, vh = k.repeat_interleave(r, 2).transpose(1, 2), v.repeat_interleave(r, 2).transpose(1, 2)
    qh = q.transpose(1, 2)
    s = scale * qh @ kh.transpose(-1, -2)
    mag = abs(scale) * qh.detach().abs() @ kh.detach().abs().transpose(-1, -2)
    if softcap:
        s = softcap * torch.tanh(s / softcap)
    if slopes is not None:
        t = torch.arange(T, dtype=torch.float64)
        bias = slopes.cpu().double()[None, :, None, None] * (t[:, None] - t[None, :])
        s, mag = s - bias, mag + bias.abs()
    see = seen_ref(E, T, first, lengths, window)[:, None]
    some = see.any(-1, keepdim=True)
    p = torch.softmax(torch.where(see | ~some, s, torch.full((), -math.inf, dtype=torch.float64)), -1)
    p = torch.where(see, p, zero)
    return (p @ vh).transpose(1, 2), p, torch.where(see, mag, zero), (qh, kh, vh)


def attention_ref(*a, **kw):
    return attention_parts(*a, **kw)[0]
