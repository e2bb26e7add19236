"""Self-attention and group norm of the Transformer / Conformer backbones on packed rows (optispeech_amd/packed_ops.py).

``Transformer(..., selfattention_layer_type="packed")`` and ``Conformer(..., selfattention_layer_type="packed")`` take these in place of the
reference's attention (_transformer/attention.py:13-125, :208-313) and BatchNorm (_conformer/convolution.py:61-70): rotary positions instead of
sinusoids or relative-position products, capped scores, penalties on distance, causal attention and shared key heads, statistics over an
utterance's own frames.  Parameter names are the reference's (linear_q, linear_k, linear_v, linear_out; norm.weight, norm.bias).
"""
import torch
from torch import nn

from .. import packed_ops as P
from .. import precision
from .base import RefSchemaModule
from .transformer import _Linear


class PackedSelfAttention(nn.Module):
    """Attention inside each document of ``rows``.  ``rotary`` = keyword arguments of packed_ops.Rotary (channels: all of a head's unless given), or None
    for no positions; ``distance_slopes``: score penalties 2^(-8 (h + 1) / heads) per frame of distance."""

    def __init__(self, n_head, n_feat, shared_heads=None, rotary=None, softcap=0.0, distance_slopes=False, causal=False):
        super().__init__()
        shared_heads = n_head if shared_heads is None else shared_heads
        assert n_feat % n_head == 0 and n_head % shared_heads == 0
        self.d_k, self.h, self.s, self.softcap, self.causal = n_feat // n_head, n_head, shared_heads, float(softcap), bool(causal)
        self.linear_q, self.linear_k = _Linear(n_feat, n_feat), _Linear(n_feat, self.d_k * shared_heads)
        self.linear_v, self.linear_out = _Linear(n_feat, self.d_k * shared_heads), _Linear(n_feat, n_feat)
        self._rotary = None if rotary is None else dict({"channels": self.d_k}, **rotary)
        self._ropes = {}
        slopes = torch.tensor([2.0 ** (-8.0 * (i + 1) / n_head) for i in range(n_head)]) if distance_slopes else None
        self.register_buffer("_slopes", slopes, persistent=False)

    def _rope(self, device):
        rope = self._ropes.get(device)
        if rope is None:
            rope = self._ropes[device] = P.Rotary(device=device, **self._rotary)
        return rope

    def forward(self, x, rows, cache=None, layer=0):
        """x (B, T, C) holding the table's rows in order; with ``cache`` (FrameCache) the rows are new frames behind the cached ones."""
        B, T, C = x.shape
        q = self.linear_q(x).view(B * T, self.h, self.d_k)
        k = self.linear_k(x).view(B * T, self.s, self.d_k)
        v = self.linear_v(x).view(B * T, self.s, self.d_k)
        dtype = torch.bfloat16 if precision.is_bf16() else torch.float32              # the mode's operand type, rounded once on the way in
        if self._rotary is not None:
            q, k = P.rotary(q, k, self._rope(x.device), rows, first=None if cache is None else cache.length, out_dtype=dtype)
        q, k, v = q.to(dtype), k.to(dtype), v.to(dtype)
        keys = None
        if cache is not None:
            k, v, keys = cache.append(layer, k, v, T)
        o = P.attention(q, k, v, rows, keys=keys, causal=self.causal, softcap=self.softcap, slopes=self._slopes)
        return self.linear_out(o.to(x.dtype).view(B, T, C))


class FrameCache:
    """Keys and values of ``streams`` streams for the layers of a causal backbone, ``capacity`` frames each."""

    def __init__(self, layers, streams, capacity, shared_heads, width, device, dtype):
        self.streams, self.capacity, self.used = streams, capacity, 0
        self.k = torch.zeros((layers, streams * capacity, shared_heads, width), device=device, dtype=dtype)
        self.v = torch.zeros_like(self.k)
        self.length = torch.zeros(streams, device=device, dtype=torch.int64)
        self._rows, self._keys, self._index = None, None, None

    def begin(self, frames):
        """rows of the next ``frames`` frames of every stream"""
        if frames < 1:
            raise P.OspError(f"{frames} new frames")
        if self.used + frames > self.capacity:
            raise P.OspError(f"{self.used} + {frames} frames in a cache of {self.capacity}")
        if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():      # replays would pass the capacity unseen
            raise P.OspError("a stream's step counts its frames on the host: it cannot be captured into a graph")
        dev = self.length.device
        self._rows = P.PackedRows.from_offsets(torch.arange(0, (self.streams + 1) * frames, frames, device=dev), self.streams * frames, longest=frames)
        self._keys = P.PackedRows.from_padded(self.length + frames, self.capacity)
        self._index = (torch.arange(self.streams, device=dev)[:, None] * self.capacity + self.length[:, None] + torch.arange(frames, device=dev)).flatten()
        return self._rows

    def append(self, layer, k, v, frames):
        self.k[layer].index_copy_(0, self._index, k)
        self.v[layer].index_copy_(0, self._index, v)
        return self.k[layer], self.v[layer], self._keys

    def end(self, frames):
        self.length += frames
        self.used += frames


class PackedGroupNorm(RefSchemaModule):
    """Group norm with a fused activation over the frames of each utterance"""

    def __init__(self, groups, c, eps=1e-5, act=None):
        super().__init__()
        self.groups, self.eps, self.act = groups, eps, act
        self.weight, self.bias = nn.Parameter(torch.ones(c)), nn.Parameter(torch.zeros(c))

    def forward(self, x, rows):
        return P.group_norm(x.reshape(-1, x.shape[-1]), self.weight, self.bias, self.groups, rows, eps=self.eps, act=self.act).view(x.shape)
