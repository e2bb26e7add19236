"""Operators on packed rows: a batch of ragged utterances as one table of rows, without padding.

``PackedRows`` says which rows of a table (M, ...) form which document; rotary positions restart in every document, group norm takes its
statistics over a document's rows, attention stays inside a document.  A padded batch (B, T, ...) flattened to (B * T, ...) is the same thing
with gaps.  Rows of no document -- a padded tail, the rows behind the last offset -- come out as zeros, in gradients too, whatever
they hold on the way in.

The handle is built once per batch from device offsets or lengths (no copy to the host) and used by every layer and direction.
Like the rest of the package: kernels go to torch's current stream on the current device, parameter gradients are accumulated into
``param.grad`` by the kernels, activations flow through autograd.

A captured graph reads the handle's tensors at every replay: build the handle inside the capture, or keep it as long as the graph.  As for any
torch operator, a backward pass is captured while no eager graph of the same leaf activations is alive.
"""
import ctypes
import functools
import math

import torch
from torch.autograd import forward_ad

from . import _lib
from . import precision as _precision
from ._lib import OspError, call, lib
from .ops import _want

ACTS = {None: 0, "none": 0, "relu": 1, "gelu": 2, "silu": 3}


@functools.lru_cache(maxsize=4096)
def _size(name, *args):
    """a size query of the library: a pure function of its sizes"""
    f = getattr(lib().cdll, name)
    f.restype = ctypes.c_int64
    return f(*(ctypes.c_int64(int(a)) for a in args))


def _wants_grad(*ts):
    """True where autograd records: elsewhere the kernels are called without an autograd node around them"""
    return torch.is_grad_enabled() and not torch.is_inference_mode_enabled() and any(t.requires_grad for t in ts)


def _first_order():
    if torch.is_grad_enabled():                                   # create_graph: the gradients below would enter the graph as constants
        raise OspError("the packed operators have no second derivatives (create_graph=True)")


def _no_tangents(*ts):
    """a dual tensor has requires_grad false and an ordinary address: it would be taken as a constant"""
    if forward_ad._current_level < 0:                             # (outside of every dual level there is none)
        return
    for t in ts:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise OspError("the packed operators have no forward-mode derivatives")


class PackedRows:
    """Documents of a table of ``rows`` rows: ``begin`` / ``length`` (docs,) int64 on the device, the tile list of the kernels, and the
    host's upper bound ``longest`` on a document's length."""

    def __init__(self, src, padded, docs, rows, longest):
        if src.dtype != torch.int64 or src.dim() != 1 or not src.is_contiguous():
            raise OspError("offsets / lengths must be a contiguous 1-D int64 tensor")
        if not src.is_cuda:
            raise OspError("offsets / lengths must live on the GPU")
        if docs < 1 or rows < 0 or longest < 0:
            raise OspError(f"a batch needs at least one document (docs {docs}, rows {rows}, longest {longest})")
        # (a bound chooses kernels and splits, never results: one of 0 counts as 1, the documents may have rows all the same)
        self.docs, self.rows, self.longest, self.device = docs, rows, min(max(longest, 1), rows), src.device
        self.cap = _size("osp_packed_rows_tiles", docs, rows)
        long = torch.empty((2, docs), device=src.device, dtype=torch.int64)
        self._buffers, self._stream = [long], _lib._raw_stream(src.device.index)
        ints = torch.empty((4 * self.cap + docs + 2,), device=src.device, dtype=torch.int32)
        self._buffers.append(ints)
        self.begin, self.length = long[0], long[1]
        self.tiles, self.base, self.ntiles = ints[:4 * self.cap], ints[4 * self.cap:4 * self.cap + docs], ints[4 * self.cap + docs:]
        call("osp_packed_rows_plan", src, int(padded), docs, rows, rows // docs if padded else 0, self.begin, self.length, self.base, self.tiles,
             self.ntiles, self.cap)

    @classmethod
    def from_offsets(cls, offsets, rows, longest=None):
        """Document b owns the rows [offsets[b], offsets[b + 1]) of a table of ``rows`` rows.  offsets (docs + 1,) int64 on the GPU, ascending
        (clamped to the table; one below its predecessor counts as its predecessor).  ``longest``: the host's bound on a document's
        length; without it the table's rows, which is always right and costs launches sized for one document that long."""
        return cls(offsets, False, offsets.numel() - 1, int(rows), int(rows if longest is None else longest))

    @classmethod
    def from_padded(cls, lengths, T):
        """Document b owns the first lengths[b] (clamped to 0 .. T) of its T rows in a (docs * T, ...) table."""
        return cls(lengths, True, lengths.numel(), lengths.numel() * int(T), int(T))

    def _check(self, t, name):
        if t.shape[0] != self.rows:
            raise OspError(f"{name} has {t.shape[0]} rows, the documents were laid out for {self.rows}")
        if t.device != self.device:
            raise OspError(f"{name} is on {t.device}, the documents on {self.device}")
        if _lib._raw_stream(self.device.index) != self._stream:
            # used on another stream than it was built on (the caller orders the two): its memory must outlive that stream's work
            for b in self._buffers:
                b.record_stream(torch.cuda.current_stream(self.device))


# ------------------------------------------------------------------------------------------------------------------ rotary positions
class Rotary:
    """Frequencies of rotary positions, f_i = base^(-2 i / channels), and their scaling for contexts longer than ``original_length``:

    ``none``; ``linear``: f_i / factor; ``base``: the base grows to base * factor^(channels / (channels - 2)), so that the slowest pair is
    slowed by the factor and the fastest is left; ``parts``: a pair that makes at least ``fast`` turns within the original length keeps f_i, one
    that makes at most ``slow`` turns gets f_i / factor, those between a blend, linear in the turns; results are scaled by
    1 + 0.1 ln factor."""

    def __init__(self, channels, base=10000.0, layout="half", scaling="none", factor=1.0, original_length=None, slow=1.0, fast=32.0,
                 device="cuda"):
        if channels < 2 or channels % 2:
            raise OspError(f"an even number of channels turns, not {channels}")
        if layout not in ("half", "interleaved"):
            raise OspError(f"layout {layout!r}: 'half' or 'interleaved'")
        if scaling not in ("none", "linear", "base", "parts"):
            raise OspError(f"scaling {scaling!r}: 'none', 'linear', 'base' or 'parts'")
        if scaling != "none" and not factor >= 1.0:
            raise OspError(f"a context is stretched by a factor >= 1, not {factor}")
        if scaling == "base" and channels == 2:
            raise OspError("a single pair has no slower one for the base to act on")
        if scaling == "parts" and (original_length is None or not fast > slow):
            raise OspError("scaling 'parts' needs original_length and fast > slow")
        if not base > 0.0:
            raise OspError(f"base {base}")
        self.channels, self.layout, self.magnitude = int(channels), layout, 1.0
        if scaling == "base":
            base = base * factor ** (channels / (channels - 2))
        f = [base ** (-2.0 * i / channels) for i in range(channels // 2)]
        if scaling == "linear":
            f = [x / factor for x in f]
        elif scaling == "parts":
            def blend(x):
                keep = min(1.0, max(0.0, (original_length * x / (2.0 * math.pi) - slow) / (fast - slow)))
                return x * keep + x / factor * (1.0 - keep)
            f = [blend(x) for x in f]
            self.magnitude = 1.0 + 0.1 * math.log(factor)
        #: turns per position, 64 bits: the kernel forms angles from it (csrc/rotary.hip)
        self.turns = torch.tensor([x / (2.0 * math.pi) for x in f], dtype=torch.float64, device=device)


def _copy(t):
    """a dense copy on memory of its own.  (`contiguous()` hands back a contiguous tensor as it is: off 16 bytes in a larger buffer, or with a dimension of one
    element whose stride says nothing)"""
    return t.clone(memory_format=torch.contiguous_format)


def _heads(t, name):
    """(M, heads, width) with contiguous channels; any row and head stride."""
    if t.dim() != 3:
        raise OspError(f"{name} must be (rows, heads, width), not {tuple(t.shape)}")
    if t.dtype not in (torch.float32, torch.bfloat16):
        raise OspError(f"{name}: float32 or bfloat16, not {t.dtype}")
    if not t.is_cuda:
        raise OspError(f"{name} must live on the GPU")
    return t if t.stride(2) == 1 or t.shape[2] == 1 else _copy(t)


def _rotate(q, k, rope, rows, first, out_dtype, inverse):
    q, k = _heads(q, "q"), _heads(k, "k")
    qo = torch.empty(q.shape, device=q.device, dtype=out_dtype)
    ko = torch.empty(k.shape, device=k.device, dtype=out_dtype)
    if q.shape[0]:
        call("osp_rotary", q, q.stride(0), q.stride(1), k, k.stride(0), k.stride(1), int(q.dtype == torch.bfloat16), qo, ko,
             int(out_dtype == torch.bfloat16), rope.turns, rows.tiles, rows.ntiles, rows.cap, first, q.shape[1], k.shape[1], q.shape[2],
             rope.channels, int(rope.layout == "interleaved"), float(rope.magnitude), int(inverse))
    return qo, ko


class RotaryFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, rope, rows, first, out_dtype):
        ctx.save_for_backward(first)                               # (its values at this call: a counter advanced in place is noticed)
        ctx.cfg = (rope, rows, q.dtype)
        ctx.shapes = (q.shape, k.shape, out_dtype, q.device)
        return _rotate(q, k, rope, rows, first, out_dtype, False)

    @staticmethod
    def backward(ctx, dq, dk):
        _first_order()
        (first,), (rope, rows, dtype) = ctx.saved_tensors, ctx.cfg
        qs, ks, od, dev = ctx.shapes
        dq = torch.zeros(qs, device=dev, dtype=od) if dq is None else dq.to(od)
        dk = torch.zeros(ks, device=dev, dtype=od) if dk is None else dk.to(od)
        gq, gk = _rotate(dq, dk, rope, rows, first, dtype, True)
        return gq, gk, None, None, None, None


def rotary(q, k, rope, rows, first=None, out_dtype=None):
    """Turn the first ``rope.channels`` channels of every head of q (M, heads, width) and k (M, shared, width) by the row's position: its index in
    its document plus ``first`` (docs,) int64 (the frames already in a cache).  One launch; results are contiguous, in ``out_dtype`` (float32
    or bfloat16; the inputs' type without it).  The gradient is the inverse turn, in the inputs' type."""
    _no_tangents(q, k)
    if q.dim() != 3 or k.dim() != 3 or q.shape[0] != k.shape[0] or q.shape[2] != k.shape[2] or q.shape[1] < 1 or k.shape[1] < 1:
        raise OspError(f"q {tuple(q.shape)} and k {tuple(k.shape)} must be (rows, heads, width) with the same rows and width")
    if q.dtype != k.dtype:
        raise OspError(f"q is {q.dtype}, k {k.dtype}")
    out_dtype = q.dtype if out_dtype is None else out_dtype
    if out_dtype not in (torch.float32, torch.bfloat16):
        raise OspError(f"out_dtype: float32 or bfloat16, not {out_dtype}")
    if rope.channels > q.shape[2]:
        raise OspError(f"{rope.channels} turned channels in heads of {q.shape[2]}")
    if rope.turns.device != q.device:
        raise OspError(f"the frequencies are on {rope.turns.device}, q on {q.device}")
    rows._check(q, "q")
    rows._check(k, "k")
    if first is not None:
        if first.dtype != torch.int64 or first.shape != (rows.docs,) or not first.is_contiguous() or first.device != q.device:
            raise OspError("first must be a contiguous (docs,) int64 tensor on q's device")
    if not _wants_grad(q, k):
        return _rotate(q, k, rope, rows, first, out_dtype, False)
    return RotaryFn.apply(q, k, rope, rows, first, out_dtype)


# ------------------------------------------------------------------------------------------------------------------ group norm
def _matrix(t, name):
    if t.dim() != 2:
        raise OspError(f"{name} must be (rows, channels), not {tuple(t.shape)}")
    if t.dtype not in (torch.float32, torch.bfloat16):
        raise OspError(f"{name}: float32 or bfloat16, not {t.dtype}")
    return t if (t.stride(1) == 1 or t.shape[1] == 1) and t.stride(0) >= t.shape[1] else _copy(t)


def _workspace(nbytes, device):
    # one per call, from the caching allocator: two captured graphs never share one
    return torch.empty((nbytes,), device=device, dtype=torch.uint8)


def _normalise(x, w, b, groups, rows, eps, act):
    """-> (x as the kernel read it, y, mean, rstd and the mean's part below 32 bits)"""
    x = _matrix(x, "x")
    M, C = x.shape
    y = torch.empty((M, C), device=x.device, dtype=x.dtype)
    stats = torch.empty((3, rows.docs, groups), device=x.device, dtype=torch.float32)
    if M:
        ws = _workspace(_size("osp_group_norm_workspace_bytes", rows.docs, M, C, groups, 0), x.device)
        call("osp_group_norm_fwd", x, x.stride(0), int(x.dtype == torch.bfloat16), w, b, y, stats, ws, rows.begin, rows.length, rows.base, rows.tiles,
             rows.ntiles, rows.cap, rows.docs, M, rows.longest, C, groups, eps, act)
    return x, y, stats


def _grad_target(p):
    """(tensor the kernel writes, 1 where it adds to what is there): param.grad, made here where there is none, or a tensor of its own beside a strided one
    (the kernels take contiguous channels), which the caller adds"""
    if not _want(p):
        return None, 0
    if p.grad is None:
        p.grad = torch.empty_like(p)
        return p.grad, 0
    return (p.grad, 1) if p.grad.is_contiguous() else (torch.empty_like(p), 0)


def _version(p):
    return None if p is None or p.is_inference() else p._version


class GroupNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, anchor, wc, bc, params, groups, rows, eps, act):
        """wc, bc: a weight or bias that was computed (its gradient goes back to what it was computed from); params: those that are leaves"""
        w, b = params[0] if wc is None else wc, params[1] if bc is None else bc
        x, y, stats = _normalise(x, w, b, groups, rows, eps, act)
        ctx.save_for_backward(x, stats, wc, bc)
        ctx.params, ctx.cfg = params, (groups, rows, act)
        ctx.versions = [_version(p) for p in params]
        return y

    @staticmethod
    def backward(ctx, dy):
        _first_order()
        x, stats, wc, bc = ctx.saved_tensors
        (w, b), (groups, rows, act) = ctx.params, ctx.cfg
        if ctx.versions != [_version(w), _version(b)]:             # as autograd does for the tensors it keeps itself
            raise OspError("a weight or bias of group_norm has been modified by an inplace operation between its forward and backward")
        M, C = x.shape
        dy = _matrix(dy, "dy")
        dx = torch.empty((M, C), device=x.device, dtype=x.dtype) if ctx.needs_input_grad[0] else None
        # (the kernels write db first, then dw: one tensor may be both)
        db, add_b = _grad_target(b) if bc is None else (torch.empty_like(bc), 0)
        dw, add_w = _grad_target(w) if wc is None else (torch.empty_like(wc), 0)
        strided = [(p, g) for p, g in ((b, db), (w, dw)) if _want(p) and not p.grad.is_contiguous()]
        w, b = w if wc is None else wc, b if bc is None else bc
        if M:
            ws = _workspace(_size("osp_group_norm_workspace_bytes", rows.docs, M, C, groups, 1), x.device)
            call("osp_group_norm_bwd", dy, dy.stride(0), x, x.stride(0), int(x.dtype == torch.bfloat16), w, b, stats, dx, dw, add_w, db, add_b, ws,
                 rows.begin, rows.length, rows.base, rows.tiles, rows.ntiles, rows.cap, rows.docs, M, rows.longest, C, groups, act)
        else:
            for t, add in ((dx, 0), (dw, add_w), (db, add_b)):
                if t is not None and not add:
                    t.zero_()
        for p, g in strided:
            p.grad.add_(g)
        return dx, None, None if wc is None else dw, None if bc is None else db, None, None, None, None, None


def group_norm(x, weight, bias, groups, rows, eps=1e-5, act=None):
    """act(weight * (x - mean) / sqrt(var + eps) + bias), mean and variance over a document's rows and a group's channels.  x (M, C) float32
    or bfloat16 (any row stride), weight / bias (C,) float32, act None, "relu", "gelu" (with erf) or "silu"; C <= 2048.  The gradients of weights that are
    leaves are added to their ``.grad``; those of computed weights (1 + gamma) go through autograd."""
    _no_tangents(x, weight, bias)
    if x.dim() != 2 or not x.is_cuda:
        raise OspError("x must be a (rows, channels) tensor on the GPU")
    if x.dtype not in (torch.float32, torch.bfloat16):
        raise OspError(f"x: float32 or bfloat16, not {x.dtype}")
    C = x.shape[1]
    if groups < 1 or C < 1 or C % groups or C > 2048:
        raise OspError(f"{C} channels (at most 2048) do not divide into {groups} groups")
    if act not in ACTS:
        raise OspError(f"act {act!r}: one of {sorted(a for a in ACTS if a)} or None")
    if not eps > 0.0:
        raise OspError(f"eps {eps}")
    for name, t in (("weight", weight), ("bias", bias)):
        if t.shape != (C,) or t.dtype != torch.float32 or not t.is_contiguous() or t.device != x.device:
            raise OspError(f"{name} must be a contiguous ({C},) float32 tensor on x's device")
    rows._check(x, "x")
    if not _wants_grad(x, weight, bias):
        return _normalise(x, weight, bias, int(groups), rows, float(eps), ACTS[act])[1]
    # The parameters stay out of the autograd graph (the kernels write their gradients), so a captured backward meets no node of an eager graph;
    # where nothing else has a gradient a leaf of the call's own keeps the backward reachable.
    wc, bc = (t if t.requires_grad and not t.is_leaf else None for t in (weight, bias))
    anchor = None if x.requires_grad or wc is not None or bc is not None else x.new_empty(0, dtype=torch.float32).requires_grad_()
    params = (weight if wc is None else None, bias if bc is None else None)
    return GroupNormFn.apply(x, anchor, wc, bc, params, int(groups), rows, float(eps), ACTS[act])


# ------------------------------------------------------------------------------------------------------------------ attention over documents
def _aligned(t, name):
    """(M, heads, width) whose rows and heads start on 16 bytes and whose rows do not overlap (the kernels' access): a copy where they do not."""
    t = _heads(t, name)
    e = 16 // t.element_size()
    r, h = t.stride(0), t.stride(1)
    return t if r % e == 0 and h % e == 0 and t.data_ptr() % 16 == 0 and t.shape[2] <= r < 1 << 22 else _copy(t)


def _attend(q, k, v, rows, keys, causal, prefix, softcap, slopes, scale, save):
    """-> (q, k, v as the kernels read them, o, what o's rounding took off (bf16) and the log2-sum-exp where a backward wants them)"""
    q, k, v = _aligned(q, "q"), _aligned(k, "k"), _aligned(v, "v")
    (M, H, D), S, bf16 = q.shape, k.shape[1], int(q.dtype == torch.bfloat16)
    o = torch.empty((M, H, D), device=q.device, dtype=q.dtype)
    lse = torch.empty((H, M), device=q.device, dtype=torch.float32) if save else None
    rest = torch.empty_like(o) if save and bf16 else None
    # new tokens over a cache: the queries that share a key head fit the 32 columns of one score tile (csrc/attention_packed_token.hip).  Its workspace
    # holds every row of the table per split: where the rows are the documents', at most 128 (width + 2) bytes x (2048 + documents x key heads).  It may take as
    # much memory as the keys and values that the call reads, or 256 MB; a table whose rows outgrow both takes the other form (8192 documents of 512 keys, 64 / 8
    # heads of 128, 260 MB beside 17 GB: 3.9 and 18.3 ms).
    few = M and not save and rows.longest * (H // S) <= 32 and keys.longest and rows.docs < 65536 and H < 65536
    nbytes = _size("osp_packed_attention_token_workspace_bytes", rows.docs, M, keys.longest, H, S, D) if few else 0
    if not k.shape[0]:                                            # no keys at all: nothing is seen
        o.zero_()
    elif few and nbytes <= max(1 << 28, 2 * k.numel() * k.element_size()):
        ws = _workspace(nbytes, q.device)
        call("osp_packed_attention_token", q, q.stride(0), q.stride(1), k, k.stride(0), k.stride(1), v, v.stride(0), v.stride(1), bf16, o, ws,
             rows.begin, rows.length, rows.tiles, rows.ntiles, rows.cap, keys.begin, keys.length, keys.longest, prefix, slopes, rows.docs, M, H, S,
             D, scale, softcap, causal)
    elif M:
        call("osp_packed_attention_fwd", q, q.stride(0), q.stride(1), k, k.stride(0), k.stride(1), v, v.stride(0), v.stride(1), bf16, o, rest,
             lse, rows.length, rows.tiles, rows.ntiles, rows.cap, keys.begin, keys.length, prefix, slopes, rows.docs, keys.longest,
             M, H, S, D, scale, softcap, causal)
    return q, k, v, o, rest, lse


class PackedAttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, rows, keys, causal, prefix, softcap, slopes, scale):
        q, k, v, o, rest, lse = _attend(q, k, v, rows, keys, causal, prefix, softcap, slopes, scale, True)
        ctx.save_for_backward(q, k, v, o, rest, lse, prefix, slopes)
        ctx.cfg = (rows, keys, causal, softcap, scale)
        return o

    @staticmethod
    def backward(ctx, do):
        _first_order()
        q, k, v, o, rest, lse, prefix, slopes = ctx.saved_tensors
        rows, keys, causal, softcap, scale = ctx.cfg
        (M, H, D), (Mk, S, _) = q.shape, k.shape
        do = _aligned(do, "the gradient of o")
        dq = torch.empty((M, H, D), device=q.device, dtype=q.dtype)
        dk, dv = (torch.empty((Mk, S, D), device=q.device, dtype=q.dtype) for _ in range(2))
        if M and Mk:
            delta = torch.empty_like(lse)
            nbytes = _size("osp_packed_attention_bwd_workspace_bytes", rows.docs, rows.longest, Mk, H, S, D, int(q.dtype == torch.bfloat16))
            ws = _workspace(nbytes, q.device) if nbytes else None
            call("osp_packed_attention_bwd", q, q.stride(0), q.stride(1), k, k.stride(0), k.stride(1), v, v.stride(0), v.stride(1), o, rest, lse, do,
                 do.stride(0), do.stride(1), int(q.dtype == torch.bfloat16), dq, dk, dv, delta, ws, rows.begin, rows.length, rows.tiles, rows.ntiles,
                 rows.cap, keys.begin, keys.length, keys.tiles, keys.ntiles, keys.cap, prefix, slopes, rows.docs, rows.longest, keys.longest, M, Mk, H, S, D,
                 scale, softcap, causal)
        else:
            dq.zero_(), dk.zero_(), dv.zero_()
        return dq, dk, dv, None, None, None, None, None, None, None


def attention(q, k, v, rows, keys=None, causal=False, prefix=None, softcap=0.0, slopes=None, scale=None):
    """softmax(score) v inside each document.  q (M, heads, width), k and v (keys, shared, width) float32 or bfloat16, any row and head strides;
    width a multiple of 8 up to 128; query head h reads key head h // (heads / shared).

    ``rows`` (PackedRows) lays out the queries; ``keys`` the keys where they differ (a cache: ``PackedRows.from_padded(lengths, capacity)``), with the
    same number of documents.  Query i of a document stands at position  keys - queries + i : the last query is at the last key.

    score = c(scale q . k) - slopes[head] |position - j|, with c(x) = softcap tanh(x / softcap) where softcap > 0 (it and scale / softcap between 1e-36 and 1e36);
    scale (positive) 1 / sqrt(width) unless given;
    slopes (heads,) float32 (no gradient).  ``causal``: key j is seen from position j on; ``prefix`` (docs,) int64 with it: the first prefix keys of
    a document are seen by all its queries.  A query that sees nothing gives zeros, and so do rows of no document; gradients likewise.
    Keys and values must be finite where any query sees them; what lies behind a document is never read into a product.

    float32 tensors are computed in exact 32-bit products, unless the package runs in its bf16 mode: then the operands are rounded to bf16, as in
    its other attention paths, and the result is float32.  Gradients for q, k and v; no attention dropout."""
    _no_tangents(q, k, v, slopes)
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3 or k.shape != v.shape or q.shape[2] != k.shape[2]:
        raise OspError(f"q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)} must be (rows, heads, width), k and v alike")
    H, S, D = q.shape[1], k.shape[1], q.shape[2]
    if S < 1 or H < 1 or H % S or H > 65536:
        raise OspError(f"{H} query heads do not share {S} key heads evenly")
    if D < 8 or D > 128 or D % 8:
        raise OspError(f"head width {D}: a multiple of 8 up to 128")
    if not (q.dtype == k.dtype == v.dtype) or q.dtype not in (torch.float32, torch.bfloat16):
        raise OspError(f"q, k, v must be all float32 or all bfloat16, not {q.dtype}, {k.dtype}, {v.dtype}")
    if not q.is_cuda or k.device != q.device or v.device != q.device:
        raise OspError("q, k, v must live on one GPU")
    if prefix is not None and not causal:
        raise OspError("a prefix extends a causal mask: pass causal=True with it")
    if not softcap >= 0.0 or math.isinf(softcap):
        raise OspError(f"softcap {softcap}: positive, or 0 for none")
    scale = D ** -0.5 if scale is None else float(scale)
    if not (scale > 0.0 and math.isfinite(scale)):
        raise OspError(f"scale {scale}: positive")
    if softcap and not (1e-36 <= softcap <= 1e36 and 1e-36 <= scale / softcap <= 1e36):
        raise OspError(f"softcap {softcap} with scale {scale}: the cap and their quotient must lie between 1e-36 and 1e36")
    keys = rows if keys is None else keys
    rows._check(q, "q")
    keys._check(k, "k")
    if keys.docs != rows.docs:
        raise OspError(f"{rows.docs} documents of queries, {keys.docs} of keys")
    if prefix is not None:
        if prefix.dtype != torch.int64 or prefix.shape != (rows.docs,) or not prefix.is_contiguous() or prefix.device != q.device:
            raise OspError("prefix must be a contiguous (docs,) int64 tensor on q's device")
    if slopes is not None:
        if slopes.dtype != torch.float32 or slopes.shape != (H,) or not slopes.is_contiguous() or slopes.device != q.device:
            raise OspError("slopes must be a contiguous (heads,) float32 tensor on q's device")
        if slopes.requires_grad:
            raise OspError("slopes get no gradient: detach them")
    rounded = q.dtype == torch.float32 and _precision.is_bf16()
    if rounded:
        q, k, v = q.to(torch.bfloat16), k.to(torch.bfloat16), v.to(torch.bfloat16)
    args = (q, k, v, rows, keys, int(bool(causal)), prefix, float(softcap), slopes, scale)
    o = PackedAttentionFn.apply(*args) if _wants_grad(q, k, v) else _attend(*args, False)[3]
    return o.to(torch.float32) if rounded else o
