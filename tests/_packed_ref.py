"""64-bit definitions of the packed-row operators, on the CPU (test infrastructure).  Documents are given as host lengths; each function
takes the tensors as the kernel gets them and returns float64."""
import math

import torch


def documents(lengths, start=0):
    """row slices of consecutive documents"""
    out, row = [], start
    for n in lengths:
        out.append(slice(row, row + n))
        row += n
    return out


def rotary(x, docs, firsts, turns, mag, layout, inverse=False):
    x = x.detach().double().cpu()
    y = torch.zeros_like(x)
    R = 2 * turns.numel()
    for sl, first in zip(docs, firsts):
        y[sl] = x[sl]
        pos = torch.arange(sl.stop - sl.start, dtype=torch.float64) + first
        angle = 2.0 * math.pi * torch.remainder(pos[:, None] * turns.double().cpu()[None], 1.0)[:, None]
        c, s = mag * angle.cos(), mag * angle.sin() * (-1.0 if inverse else 1.0)
        ia, ib = (slice(0, R // 2), slice(R // 2, R)) if layout == "half" else (slice(0, R, 2), slice(1, R, 2))
        a, b = x[sl][..., ia], x[sl][..., ib]
        y[sl, :, ia], y[sl, :, ib] = a * c - b * s, a * s + b * c
    return y


def act(z, name):
    if name == "relu":
        return z.clamp_min(0.0)
    if name == "gelu":
        return 0.5 * z * torch.erfc(-z * math.sqrt(0.5))
    return z * torch.sigmoid(z) if name == "silu" else z


def group_norm(x, w, b, docs, groups, eps, name):
    """-> y (differentiable in x, w, b when they are float64 leaves)"""
    M, C = x.shape
    parts, row = [], 0
    for sl in docs:
        if sl.start > row:
            parts.append(torch.zeros((sl.start - row, C), dtype=torch.float64))
        row = sl.stop
        n = sl.stop - sl.start
        if not n:
            continue
        xg = x[sl].reshape(n, groups, C // groups)
        m = xg.mean((0, 2), keepdim=True)
        v = ((xg - m) ** 2).mean((0, 2), keepdim=True)
        parts.append(act(((xg - m) / torch.sqrt(v + eps)).reshape(n, C) * w + b, name))
    if row < M:
        parts.append(torch.zeros((M - row, C), dtype=torch.float64))
    return torch.cat(parts)


def attention(q, k, v, qdocs, kdocs, scale, causal=False, prefix=None, softcap=0.0, slopes=None):
    """-> o (differentiable in q, k, v when they are float64 leaves).  Query i of a document stands at position keys - queries + i."""
    M, H, D = q.shape
    S = k.shape[1]
    out, row = [], 0
    for b, (qs, ks) in enumerate(zip(qdocs, kdocs)):
        nq, nk = qs.stop - qs.start, ks.stop - ks.start
        if qs.start > row:
            out.append(torch.zeros((qs.start - row, H, D), dtype=torch.float64))
        row = qs.stop
        if not nq:
            continue
        if not nk:
            out.append(torch.zeros((nq, H, D), dtype=torch.float64))
            continue
        qh = q[qs].transpose(0, 1)
        kh = k[ks].transpose(0, 1).repeat_interleave(H // S, 0)
        vh = v[ks].transpose(0, 1).repeat_interleave(H // S, 0)
        s = scale * (qh @ kh.transpose(1, 2))
        if softcap:
            s = softcap * torch.tanh(s / softcap)
        at = torch.arange(nk - nq, nk)[:, None]
        j = torch.arange(nk)[None]
        if slopes is not None:
            s = s - slopes.double().cpu()[:, None, None] * (at - j).abs().double()
        seen = torch.ones((nq, nk), dtype=torch.bool)
        if causal:
            seen = (j <= at) | (j < (0 if prefix is None else int(prefix[b])))
        s = s.masked_fill(~seen, float("-inf"))
        m = s.detach().amax(-1, keepdim=True).clamp_min(-1e300)
        p = (s - m).exp()
        total = p.sum(-1, keepdim=True)
        p = torch.where(total > 0, p / total.clamp_min(1e-300), torch.zeros_like(p))
        out.append((p @ vh).transpose(0, 1))
    if row < M:
        out.append(torch.zeros((M - row, H, D), dtype=torch.float64))
    return torch.cat(out)
