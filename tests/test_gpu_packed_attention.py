"""Attention over documents against its definition in 64 bits.

The bounds, per document and head (u = 2^-24; ua: rounding of the matrix operands made from f32 values, 2^-8 for bf16 tensors, 0 for f32; uo: rounding
of the result; n keys, D channels; everything below is a sum of absolute values in 64 bits):
  score error  e = u ((D + 8) scale sum |q k| + 16 softcap + 8 slope distance + 4 |lse| + 8)      (natural units; the cap's slope is at most 1)
  probability  relative error  r = e + max over the row of e + (n + 8) u                          (its normaliser carries the row's errors)
  o            P (r + ua + n u) |V|  + uo |o|
  dV           (P (r + ua + n u))^T |dO| + uo |dV|
  dS           with t = |dP| + |delta|:  P g (t (r + (D + 8) u) + uo sum |dO o|) + 16 u P t (the cap's slope) + (ua + n u) |dS|   =: w
  dQ, dK       scale w |K| + uo |dQ|,   scale w^T |Q| + uo |dK|   (summed over the query heads of a key head)
n counts queries in dV and dK: the larger of both is used throughout."""
import pytest
import torch

from . import _packed_ref as ref

DEV = "cuda"
U = 2.0 ** -24
gpu = pytest.mark.gpu


def offsets(lengths, start=0):
    return torch.tensor([start + sum(lengths[:i]) for i in range(len(lengths) + 1)], dtype=torch.int64, device=DEV)


def randn(*shape, seed, dtype=torch.float32, std=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype).to(DEV)


def bounds(q, k, v, do, qdocs, kdocs, scale, causal, prefix, softcap, slopes, dtype):
    """want and tolerance of (o, dq, dk, dv), float64"""
    q, k, v, do = (t.detach().double().cpu() for t in (q, k, v, do))
    ua = 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
    uo = torch.finfo(dtype).eps / 2
    H, D, S = q.shape[1], q.shape[2], k.shape[1]
    want = [torch.zeros_like(t) for t in (q, q, k, v)]
    tol = [torch.zeros_like(t) for t in (q, q, k, v)]
    for b, (qs, ks) in enumerate(zip(qdocs, kdocs)):
        nq, nk = qs.stop - qs.start, ks.stop - ks.start
        if not nq or not nk:
            continue
        dist = (torch.arange(nk - nq, nk)[:, None] - torch.arange(nk)[None]).double()
        seen = torch.ones((nq, nk), dtype=torch.bool)
        if causal:
            seen = (dist >= 0) | (torch.arange(nk)[None] < (0 if prefix is None else int(prefix[b])))
        n = max(nq, nk)
        for h in range(H):
            g = h * S // H
            Q, K, V, G = q[qs, h], k[ks, g], v[ks, g], do[qs, h]
            x = scale * (Q @ K.T)
            slope = torch.ones_like(x)
            s = x
            if softcap:
                t = torch.tanh(x / softcap)
                s, slope = softcap * t, 1 - t * t
            sl = 0.0 if slopes is None else float(slopes[h])
            s = torch.where(seen, s - sl * dist.abs(), float("-inf"))
            lse = torch.logsumexp(s, -1, keepdim=True)
            P = torch.where(torch.isfinite(lse), (s - lse).exp(), torch.zeros_like(s)).nan_to_num(0.0)
            e = U * ((D + 8) * abs(scale) * (Q.abs() @ K.abs().T) + 16 * softcap + 8 * abs(sl) * dist.abs() + 4 * lse.nan_to_num(0, 0, 0).abs() + 8)
            e = torch.where(seen, e, torch.zeros_like(e))
            r = e + e.amax(-1, keepdim=True) + (n + 8) * U
            o = P @ V
            dP = G @ V.T
            delta = (G * o).sum(-1, keepdim=True)
            dS = P * (dP - delta) * slope
            t = dP.abs() + delta.abs()
            w = P * slope * (t * (r + (D + 8) * U) + uo * (G * o).abs().sum(-1, keepdim=True)) + 16 * U * P * t + (ua + n * U) * dS.abs()
            pr = P * (r + ua + n * U)
            want[0][qs, h] = o
            tol[0][qs, h] = pr @ V.abs()
            want[1][qs, h] = scale * (dS @ K)
            tol[1][qs, h] = abs(scale) * (w @ K.abs())
            want[2][ks, g] += scale * (dS.T @ Q)
            tol[2][ks, g] += abs(scale) * (w.T @ Q.abs())
            want[3][ks, g] += P.T @ G
            tol[3][ks, g] += pr.T @ G.abs()
    return want, [t + uo * (w.abs() + t) for w, t in zip(want, tol)]


def close(got, want, tol, names=("o", "dq", "dk", "dv")):
    for name, a, w, t in zip(names, got, want, tol):
        err = (a.detach().double().cpu() - w).abs()
        assert torch.isfinite(err).all(), name
        assert bool((err <= t).all()), (name, (err - t).max().item(), err.max().item())


def grads(q, k, v, do, rows, **kw):
    from optispeech_amd import packed_ops as P
    q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    o = P.attention(q, k, v, rows, **kw)
    return (o,) + torch.autograd.grad(o, (q, k, v), do)


MASKS = ["full", "causal", "prefix"]
SHAPES = [  # lengths, tail, query heads, key heads, width
    ([1], 0, 1, 1, 8), ([5, 0, 33], 3, 2, 2, 32), ([127, 1, 64], 0, 4, 2, 40), ([128, 129], 5, 3, 1, 64), ([2, 31, 32, 65], 0, 4, 4, 80),
    ([300], 1, 2, 1, 96), ([257, 1, 1], 0, 8, 2, 128), ([40] * 9, 2, 2, 2, 16)]


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("mask", MASKS)
@pytest.mark.parametrize("cap,slope", [(0.0, False), (5.0, False), (0.0, True), (20.0, True)])
@pytest.mark.parametrize("lengths,tail,H,S,D", SHAPES)
def test_attention_forward_and_gradients(dtype, mask, cap, slope, lengths, tail, H, S, D):
    from optispeech_amd import packed_ops as P
    M = sum(lengths) + tail
    q, do = randn(M, H, D, seed=1, dtype=dtype, std=3.0 if cap else 1.0), randn(M, H, D, seed=4, dtype=dtype)
    k, v = randn(M, S, D, seed=2, dtype=dtype), randn(M, S, D, seed=3, dtype=dtype)
    prefix = torch.tensor([(7 * i + 3) % (n + 2) for i, n in enumerate(lengths)], dtype=torch.int64, device=DEV) if mask == "prefix" else None
    slopes = torch.tensor([0.5 ** (h + 1) for h in range(H)], device=DEV) if slope else None
    rows = P.PackedRows.from_offsets(offsets(lengths), M, longest=max(lengths))
    got = grads(q, k, v, do, rows, causal=mask != "full", prefix=prefix, softcap=cap, slopes=slopes)
    docs = ref.documents(lengths)
    want, tol = bounds(q, k, v, do, docs, docs, D ** -0.5, mask != "full", prefix, cap, slopes, dtype)
    close(got, want, tol)


MANY = [5, 0, 33, 127, 128, 129, 1, 64, 31, 65] * 6


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("mask,cap,slope", [("full", 0.0, False), ("full", 0.0, True), ("causal", 5.0, False), ("prefix", 20.0, True), ("causal", 0.0, True)])
@pytest.mark.parametrize("H,S,D", [(8, 8, 128), (8, 4, 64), (10, 5, 40), (16, 4, 96), (12, 4, 32)])
def test_attention_over_many_documents(dtype, mask, cap, slope, H, S, D):
    """enough tiles for the kernels whose waves own 32 rows each, and for key heads whose query heads are cut into parts; forward and gradients"""
    from optispeech_amd import packed_ops as P
    M = sum(MANY) + 6
    q, do = randn(M, H, D, seed=1, dtype=dtype, std=3.0 if cap else 1.0), randn(M, H, D, seed=4, dtype=dtype)
    k, v = randn(M, S, D, seed=2, dtype=dtype), randn(M, S, D, seed=3, dtype=dtype)
    prefix = torch.tensor([(7 * i + 3) % (n + 2) for i, n in enumerate(MANY)], dtype=torch.int64, device=DEV) if mask == "prefix" else None
    slopes = torch.tensor([0.5 ** (h + 1) for h in range(H)], device=DEV) if slope else None
    rows = P.PackedRows.from_offsets(offsets(MANY), M, longest=max(MANY))
    got = grads(q, k, v, do, rows, causal=mask != "full", prefix=prefix, softcap=cap, slopes=slopes)
    docs = ref.documents(MANY)
    want, tol = bounds(q, k, v, do, docs, docs, D ** -0.5, mask != "full", prefix, cap, slopes, dtype)
    close(got, want, tol)
    for t in got:
        assert float(t.detach()[sum(MANY):].abs().sum()) == 0.0


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_long_documents(dtype):
    """documents of many tiles, queries and keys of different numbers, in both arrangements of the waves"""
    from optispeech_amd import packed_ops as P
    for qlens, klens, H, S, D in (([1500, 700], [1500, 900], 2, 1, 64), ([900] * 6, [1100, 900, 130, 900, 901, 1000], 12, 6, 128)):
        M, Mk = sum(qlens), sum(klens)
        q, do = randn(M, H, D, seed=1, dtype=dtype), randn(M, H, D, seed=4, dtype=dtype)
        k, v = randn(Mk, S, D, seed=2, dtype=dtype), randn(Mk, S, D, seed=3, dtype=dtype)
        prefix = torch.tensor([300 * i for i in range(len(qlens))], dtype=torch.int64, device=DEV)
        rows = P.PackedRows.from_offsets(offsets(qlens), M, longest=max(qlens))
        keys = P.PackedRows.from_offsets(offsets(klens), Mk, longest=max(klens))
        got = grads(q, k, v, do, rows, keys=keys, causal=True, prefix=prefix)
        want, tol = bounds(q, k, v, do, ref.documents(qlens), ref.documents(klens), D ** -0.5, True, prefix, 0.0, None, dtype)
        close(got, want, tol)


@gpu
def test_the_bounds_reference_agrees_with_autograd():
    """the gradient formulas above against autograd of the plain definition (float64, CPU)"""
    lengths, H, S, D = [9, 0, 14], 4, 2, 8
    q, k, v, do = (randn(23, h, D, seed=i).double().cpu() for i, h in enumerate((H, S, S, H)))
    slopes, prefix = torch.tensor([0.1, 0.2, 0.3, 0.4]), torch.tensor([3, 0, 30])
    docs = ref.documents(lengths)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    o = ref.attention(*leaves, docs, docs, 0.3, True, prefix, 2.0, slopes)
    auto = (o,) + torch.autograd.grad(o, leaves, do)
    want, _ = bounds(q, k, v, do, docs, docs, 0.3, True, prefix, 2.0, slopes, torch.float32)
    for a, w in zip(auto, want):
        assert torch.allclose(a.detach(), w, rtol=1e-10, atol=1e-12)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("mask", MASKS)
def test_queries_and_keys_of_different_numbers(dtype, mask):
    """keys in a padded cache, queries packed; more queries than keys under a causal mask (the first ones see nothing), no keys, no queries; the
    cache's unused rows hold NaN and infinities"""
    from optispeech_amd import packed_ops as P
    qlens, klens, T, H, S, D = [1, 5, 140, 70, 0, 33, 3], [260, 5, 150, 30, 17, 0, 300], 300, 4, 2, 64
    M, B = sum(qlens) + 2, len(klens)
    q, do = randn(M, H, D, seed=1, dtype=dtype), randn(M, H, D, seed=4, dtype=dtype)
    k, v = randn(B * T, S, D, seed=2, dtype=dtype), randn(B * T, S, D, seed=3, dtype=dtype)
    kc, vc = k.clone(), v.clone()
    for b, n in enumerate(klens):
        k[b * T + n:(b + 1) * T], v[b * T + n:(b + 1) * T] = float("nan"), float("inf")
    q[-2:], do[-2:] = float("nan"), float("-inf")
    prefix = torch.tensor([0, 2, 100, 31, 5, 0, 500], dtype=torch.int64, device=DEV) if mask == "prefix" else None
    rows = P.PackedRows.from_offsets(offsets(qlens), M)
    keys = P.PackedRows.from_padded(torch.tensor(klens, dtype=torch.int64, device=DEV), T)
    got = grads(q, k, v, do, rows, keys=keys, causal=mask != "full", prefix=prefix)
    qdocs, kdocs = ref.documents(qlens), [slice(b * T, b * T + n) for b, n in enumerate(klens)]
    want, tol = bounds(q.nan_to_num(0, 0, 0), kc, vc, do.nan_to_num(0, 0, 0), qdocs, kdocs, D ** -0.5, mask != "full", prefix, 0.0, None, dtype)
    close(got, want, tol)
    assert float(got[0].detach()[-2:].abs().sum()) == 0.0


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("mask,cap,slope", [("causal", 0.0, False), ("full", 6.0, False), ("prefix", 0.0, True), ("causal", 9.0, True)])
@pytest.mark.parametrize("H,S,D", [(2, 2, 128), (16, 2, 64), (8, 1, 40), (3, 3, 32), (4, 2, 96)])
@pytest.mark.parametrize("qlens,klens,T", [([1] * 5, [700, 1, 129, 0, 256], 700), ([1, 0, 2, 4], [3, 50, 1, 5000], 5000), ([3], [2], 2)])
def test_new_tokens_over_a_cache(dtype, mask, cap, slope, H, S, D, qlens, klens, T):
    """the split kernel (no gradient wanted, few queries) against the definition, and against the tiled kernel's bound; the cache's unused rows
    hold NaN; a document without queries and one without keys; more queries than keys"""
    from optispeech_amd import packed_ops as P
    M, B = sum(qlens) + 1, len(klens)
    q = randn(M, H, D, seed=1, dtype=dtype, std=2.0 if cap else 1.0)
    k, v = randn(B * T, S, D, seed=2, dtype=dtype), randn(B * T, S, D, seed=3, dtype=dtype)
    kc, vc = k.clone(), v.clone()
    for b, n in enumerate(klens):
        k[b * T + n:(b + 1) * T], v[b * T + n:(b + 1) * T] = float("nan"), float("nan")
    prefix = torch.tensor([(3 * i) % 7 for i in range(B)], dtype=torch.int64, device=DEV) if mask == "prefix" else None
    slopes = torch.tensor([0.5 ** (h + 2) for h in range(H)], device=DEV) if slope else None
    rows = P.PackedRows.from_offsets(offsets(qlens), M, longest=max(qlens))
    keys = P.PackedRows.from_padded(torch.tensor(klens, dtype=torch.int64, device=DEV), T)
    kw = dict(keys=keys, causal=mask != "full", prefix=prefix, softcap=cap, slopes=slopes)
    o = P.attention(q, k, v, rows, **kw)
    qdocs, kdocs = ref.documents(qlens), [slice(b * T, b * T + n) for b, n in enumerate(klens)]
    want, tol = bounds(q, kc, vc, q, qdocs, kdocs, D ** -0.5, mask != "full", prefix, cap, slopes, dtype)
    close((o,), want[:1], tol[:1])
    assert float(o[sum(qlens):].abs().sum()) == 0.0


@gpu
def test_new_tokens_beyond_the_hosts_bounds():
    """bounds on the host that are too small cost time, not results: more queries and more keys than ``longest`` says"""
    from optispeech_amd import packed_ops as P
    H, S, D = 4, 1, 64
    q, k, v = randn(50, H, D, seed=1), randn(3000, S, D, seed=2), randn(3000, S, D, seed=3)
    rows = P.PackedRows.from_offsets(offsets([50]), 50, longest=1)
    keys = P.PackedRows.from_offsets(offsets([3000]), 3000, longest=100)
    o = P.attention(q, k, v, rows, keys=keys, causal=True)
    want, tol = bounds(q, k, v, q, ref.documents([50]), ref.documents([3000]), D ** -0.5, True, None, 0.0, None, torch.float32)
    close((o,), want[:1], tol[:1])


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_views_of_one_projection_and_odd_addresses(dtype):
    """q, k, v as views into one (rows, 3 heads width) projection, and the same shifted by one element (rows that do not start on 16 bytes); a
    head-major gradient; results equal those of contiguous tensors bit for bit"""
    from optispeech_amd import packed_ops as P
    lengths, H, D = [70, 33], 2, 32
    M = sum(lengths)
    rows = P.PackedRows.from_offsets(offsets(lengths), M)
    do = randn(H, M, D, seed=9, dtype=dtype).transpose(0, 1)
    for shift in (0, 1):
        w = randn(M, 3 * H * D + 8, seed=8, dtype=dtype)
        q, k, v = (w[:, shift + i * H * D:shift + (i + 1) * H * D].unflatten(1, (H, D)) for i in range(3))
        got = grads(q, k, v, do, rows, causal=True)
        same = grads(q.contiguous(), k.contiguous(), v.contiguous(), do.contiguous(), rows, causal=True)
        for a, b in zip(got, same):
            assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_padded_batch_equals_packed_batch(dtype):
    """the same documents as a padded batch: the same values, bit for bit"""
    from optispeech_amd import packed_ops as P
    lengths, T, H, D = [50, 0, 131, 7], 140, 2, 64
    B, M = len(lengths), sum(lengths)
    pads = [randn(B * T, H, D, seed=i, dtype=dtype) for i in range(4)]
    idx = torch.cat([torch.arange(b * T, b * T + n) for b, n in enumerate(lengths)]).to(DEV)
    a = grads(*pads, P.PackedRows.from_padded(torch.tensor(lengths, dtype=torch.int64, device=DEV), T), causal=True, softcap=10.0)
    b = grads(*(t[idx] for t in pads), P.PackedRows.from_offsets(offsets(lengths), M), causal=True, softcap=10.0)
    for x, y in zip(a, b):
        assert torch.equal(x[idx], y)
        x[idx] = 0
        assert float(x.abs().sum()) == 0.0


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_large_scores_and_falling_maxima(dtype):
    """scores in the hundreds, rising and falling along the keys: the running maximum moves late, early and not at all"""
    from optispeech_amd import packed_ops as P
    M, D = 400, 32
    q, v, do = randn(M, 2, D, seed=1, dtype=dtype), randn(M, 2, D, seed=3, dtype=dtype), randn(M, 2, D, seed=4, dtype=dtype)
    ramp = torch.linspace(-6, 6, M, device=DEV)[:, None]
    k = torch.stack([randn(M, D, seed=2) + ramp, randn(M, D, seed=5) - ramp], 1).to(dtype)
    rows = P.PackedRows.from_offsets(offsets([M]), M)
    got = grads(q, k, v, do, rows, scale=1.5)
    docs = ref.documents([M])
    want, tol = bounds(q, k, v, do, docs, docs, 1.5, False, None, 0.0, None, dtype)
    close(got, want, tol)


@gpu
def test_offsets_beyond_32_bits():
    """keys whose element offset passes 2^31 (bf16 cache of 2.2 G elements per tensor): the last document's values against the definition"""
    from optispeech_amd import packed_ops as P
    S, D, T, B = 8, 128, 30000, 72
    assert B * T * S * D > 1 << 31
    k = torch.zeros((B * T, S, D), device=DEV, dtype=torch.bfloat16)
    v = torch.zeros((B * T, S, D), device=DEV, dtype=torch.bfloat16)
    lens = [3] * (B - 1) + [200]
    last = slice((B - 1) * T, (B - 1) * T + 200)
    k[last], v[last] = randn(200, S, D, seed=2, dtype=torch.bfloat16), randn(200, S, D, seed=3, dtype=torch.bfloat16)
    q, do = randn(B + 39, S, D, seed=1, dtype=torch.bfloat16), randn(B + 39, S, D, seed=4, dtype=torch.bfloat16)
    qlens = [1] * (B - 1) + [40]
    rows = P.PackedRows.from_offsets(offsets(qlens), B + 39)
    keys = P.PackedRows.from_padded(torch.tensor(lens, dtype=torch.int64, device=DEV), T)
    a = grads(q, k, v, do, rows, keys=keys, causal=True)
    want, tol = bounds(q[B - 1:], k[last], v[last], do[B - 1:], [slice(0, 40)], [slice(0, 200)], D ** -0.5, True, None, 0.0, None, torch.bfloat16)
    close((a[0][B - 1:], a[1][B - 1:], a[2][last], a[3][last]), want, tol)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_same_call_same_bits_and_other_streams(dtype):
    from optispeech_amd import packed_ops as P
    lengths, H, S, D = [300, 17, 200], 4, 2, 64
    M = sum(lengths)
    t = [randn(M, h, D, seed=i, dtype=dtype) for i, h in enumerate((H, S, S, H))]
    rows = P.PackedRows.from_offsets(offsets(lengths), M)
    a = grads(*t, rows, causal=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = grads(*t, P.PackedRows.from_offsets(offsets(lengths), M), causal=True)
    torch.cuda.current_stream().wait_stream(side)
    for x, y in zip(a, b):
        assert torch.equal(x, y)


@gpu
def test_captured_forward_replayed_with_other_lengths():
    """offsets, rows, rotary, attention and norm recorded into one graph: replays follow the lengths and values in the recorded tensors, with eager work
    between the replays"""
    from optispeech_amd import packed_ops as P
    M, H, D = 300, 2, 64
    off = offsets([100, 150])
    x = randn(M, 3 * H * D, seed=1)
    w, b = randn(H * D, seed=2), randn(H * D, seed=3)
    rope = P.Rotary(D)

    def step():
        rows = P.PackedRows.from_offsets(off, M)
        q, k, v = (x[:, i * H * D:(i + 1) * H * D].unflatten(1, (H, D)) for i in range(3))
        q, k = P.rotary(q, k, rope, rows)
        o = P.attention(q, k, v, rows, causal=True, softcap=9.0)
        return P.group_norm(o.flatten(1), w, b, 4, rows, 1e-5, "silu")
    with torch.no_grad():
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        for i, lens in enumerate(([100, 150], [300, 0], [1, 299], [5, 6])):
            off.copy_(offsets(lens))
            x.copy_(randn(M, 3 * H * D, seed=10 + i))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, step()), lens


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_captured_training_step_replayed(dtype):
    """rows, rotary, attention, group norm and their backward in one graph; every replay, with eager work in between, equals the eager step bit for bit"""
    from optispeech_amd import packed_ops as P
    M, H, S, D = 260, 4, 2, 32
    off = offsets([100, 130])
    x, g = randn(M, (H + 2 * S) * D, seed=1, dtype=dtype).requires_grad_(), randn(M, H * D, seed=5, dtype=dtype)
    w, b = torch.nn.Parameter(randn(H * D, seed=2)), torch.nn.Parameter(randn(H * D, seed=3))
    w.grad, b.grad = torch.zeros_like(w), torch.zeros_like(b)
    rope = P.Rotary(D, layout="interleaved")

    def step():
        w.grad.zero_(), b.grad.zero_()
        rows = P.PackedRows.from_offsets(off, M)
        q, k, v = (t.unflatten(1, (-1, D)) for t in x.split([H * D, S * D, S * D], 1))
        q, k = P.rotary(q, k, rope, rows)
        o = P.attention(q, k, v, rows, causal=True, softcap=9.0)
        y = P.group_norm(o.flatten(1), w, b, 4, rows, 1e-5, "gelu")
        return (y.detach(),) + torch.autograd.grad(y, (x,), g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i, lens in enumerate(([100, 130], [260, 0], [1, 259], [5, 6])):
        off.copy_(offsets(lens))
        with torch.no_grad():
            x.copy_(randn(M, (H + 2 * S) * D, seed=10 + i, dtype=dtype))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out] + [w.grad.clone(), b.grad.clone()]
        want = list(step()) + [w.grad, b.grad]
        for a, e in zip(got, want):
            assert torch.equal(a, e), lens


@gpu
def test_rows_built_on_one_stream_and_used_on_another():
    """the handle is dropped while the other stream still works: its memory is not handed out before that work is done"""
    from optispeech_amd import packed_ops as P
    lengths, H, D = [400, 300], 4, 64
    M = sum(lengths)
    q, k, v = (randn(M, H, D, seed=i, dtype=torch.bfloat16) for i in range(3))
    want = P.attention(q, k, v, P.PackedRows.from_offsets(offsets(lengths), M), causal=True)
    side = torch.cuda.Stream()
    outs = []
    for _ in range(5):
        rows = P.PackedRows.from_offsets(offsets(lengths), M)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            outs.append(P.attention(q, k, v, rows, causal=True))
        del rows
        torch.full((4096,), -1, dtype=torch.int32, device=DEV)      # would take the freed blocks
    torch.cuda.current_stream().wait_stream(side)
    for o in outs:
        assert torch.equal(o, want)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_broadcast_heads_and_rows(dtype):
    """one key head expanded over the query heads, one row expanded over the table: results of the contiguous tensors, bit for bit, and the gradient
    summed over the copies"""
    from optispeech_amd import packed_ops as P
    lengths, H, D = [50, 33], 4, 32
    M = sum(lengths)
    rows = P.PackedRows.from_offsets(offsets(lengths), M)
    q, v, do = randn(M, H, D, seed=1, dtype=dtype), randn(M, H, D, seed=3, dtype=dtype), randn(M, H, D, seed=4, dtype=dtype)
    for shape in ((M, 1, D), (1, H, D), (1, 1, D)):
        k = randn(*shape, seed=2, dtype=dtype)
        a, b = k.clone().requires_grad_(), k.clone().requires_grad_()
        oa, ob = P.attention(q, a.expand(M, H, D), v, rows, causal=True), P.attention(q, b.expand(M, H, D).contiguous(), v, rows, causal=True)
        assert torch.equal(oa, ob)
        assert torch.equal(torch.autograd.grad(oa, (a,), do)[0], torch.autograd.grad(ob, (b,), do)[0])
        with torch.no_grad():
            assert torch.equal(P.attention(a.expand(M, H, D), v, v, rows), P.attention(a.expand(M, H, D).contiguous(), v, v, rows))


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_two_streams_share_a_handle(dtype):
    """training and token calls issued on two streams at once, nothing shared but the handles and the inputs"""
    from optispeech_amd import packed_ops as P
    lengths, H, D = [200, 133, 1], 4, 64
    M = sum(lengths)
    rows = P.PackedRows.from_offsets(offsets(lengths), M)
    tokens = P.PackedRows.from_offsets(offsets([1, 1, 1]), 3, longest=1)
    sets = [[randn(M, H, D, seed=10 * j + i, dtype=dtype) for i in range(4)] for j in range(2)]
    run = lambda t: list(grads(*t, rows, causal=True)) + [P.attention(t[0][:3], t[1], t[2], tokens, keys=rows, causal=True)]      # noqa: E731
    want = [run(t) for t in sets]
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(4):
        for j, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[j].append(run(sets[j]))
    torch.cuda.synchronize()
    for j in range(2):
        for result in got[j]:
            for a, e in zip(result, want[j]):
                assert torch.equal(a, e)


@gpu
def test_new_tokens_in_a_large_table():
    """three tokens in a table of a million rows: right, zeros behind them, and no workspace that grows with rows times splits"""
    from optispeech_amd import packed_ops as P
    M, H, D, klens = 1000000, 2, 8, [9000, 1, 4000]
    q = randn(M, H, D, seed=1, dtype=torch.bfloat16)
    k, v = (randn(sum(klens), H, D, seed=i, dtype=torch.bfloat16) for i in (2, 3))
    rows = P.PackedRows.from_offsets(offsets([1, 1, 1]), M, longest=1)
    keys = P.PackedRows.from_offsets(offsets(klens), sum(klens))
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    o = P.attention(q, k, v, rows, keys=keys, causal=True)
    assert torch.cuda.max_memory_allocated() - before < 1 << 29
    want, tol = bounds(q[:3], k, v, q[:3], ref.documents([1, 1, 1]), ref.documents(klens), D ** -0.5, True, None, 0.0, None, torch.bfloat16)
    close((o[:3],), want[:1], tol[:1])
    assert float(o[3:].abs().max()) == 0.0


@gpu
def test_empty_tables_and_second_derivatives():
    """no rows, no keys: zeros of the right shapes; a second derivative is refused, not taken as zero"""
    from optispeech_amd import packed_ops as P
    none = P.PackedRows.from_offsets(offsets([0, 0]), 0)
    some = P.PackedRows.from_offsets(offsets([2, 3]), 5)
    q0, q5 = torch.zeros(0, 2, 8, device=DEV), randn(5, 2, 8, seed=1)
    o, dq, dk, dv = grads(q0, q0, q0, q0, none)
    assert o.shape == dq.shape == dk.shape == dv.shape == (0, 2, 8)
    o, dq, dk, dv = grads(q5, q0, q0, q5, some, keys=none, causal=True)
    assert float(o.detach().abs().sum()) == 0.0 and float(dq.abs().sum()) == 0.0 and dk.shape == (0, 2, 8)
    o, dq, dk, dv = grads(q0, q5, q5, q0, none, keys=some)
    assert float(dk.abs().sum()) == 0.0 and float(dv.abs().sum()) == 0.0
    with torch.no_grad():
        assert float(P.attention(q5, q0, q0, some, keys=none).abs().sum()) == 0.0
    yq, yk = P.rotary(q0, q0, P.Rotary(8), none)
    assert yq.shape == (0, 2, 8)
    assert P.group_norm(q0.flatten(1), torch.ones(16, device=DEV), torch.ones(16, device=DEV), 2, none).shape == (0, 16)
    q = q5.clone().requires_grad_()
    w = torch.nn.Parameter(torch.ones(16, device=DEV))
    from optispeech_amd._lib import OspError
    for y in (P.attention(q, q, q, some), P.rotary(q, q, P.Rotary(8), some)[0], P.group_norm(q.flatten(1), w, w, 2, some)):
        with pytest.raises(OspError, match="second"):
            torch.autograd.grad(y.sum(), (q,), create_graph=True)


@gpu
def test_gradient_against_differences():
    """<dx, u> against central differences of L = sum o do in f32, h = 1/64: truncation h^2 / 6 |L'''| and rounding 2 u sum |o do| / (2 h) both below
    1e-3 |dx| |u| at these sizes"""
    from optispeech_amd import packed_ops as P
    lengths, H, S, D = [40, 23], 2, 1, 16
    M = sum(lengths)
    q, k, v, do = (randn(M, h, D, seed=i) for i, h in enumerate((H, S, S, H)))
    slopes = torch.tensor([0.05, 0.01], device=DEV)
    rows = P.PackedRows.from_offsets(offsets(lengths), M)
    kw = dict(causal=True, softcap=4.0, slopes=slopes)
    _, *g = grads(q, k, v, do, rows, **kw)
    h = 1.0 / 64
    for i, name in enumerate("qkv"):
        u = randn(*(q, k, v)[i].shape, seed=20 + i)

        def loss(sign):
            t = [q, k, v]
            t[i] = t[i] + sign * h * u
            return float((P.attention(*t, rows, **kw).double() * do.double()).sum())
        with torch.no_grad():
            num = (loss(1) - loss(-1)) / (2 * h)
        assert abs(float((g[i].double() * u.double()).sum()) - num) <= 1e-3 * float(g[i].double().norm() * u.double().norm()), name


@gpu
def test_bf16_mode_rounds_float32_operands():
    """in the package's bf16 mode float32 tensors give the bf16 kernels' result on rounded operands, in float32, with float32 gradients"""
    from optispeech_amd import packed_ops as P, precision
    t = [randn(90, 2, 32, seed=i) for i in range(4)]
    rows = P.PackedRows.from_offsets(offsets([60, 30]), 90)
    want = grads(*(x.bfloat16() for x in t), rows, causal=True)
    precision.set_precision("bf16")
    try:
        got = grads(*t, rows, causal=True)
    finally:
        precision.set_precision("f32")
    for a, b in zip(got, want):
        assert a.dtype == torch.float32 and torch.equal(a, b.float())


# ------------------------------------------------------------------------------------------------------------------ refusals
def test_refusals():
    from optispeech_amd import packed_ops as P
    from optispeech_amd._lib import OspError
    h = torch.zeros(4, 4, 8)
    for q, k, v in ((h, h[:, :3], h[:, :3]), (h, h, h[:3]), (h, h, h.double()), (h[..., :4], h[..., :4], h[..., :4]), (h[0], h, h),
                    (torch.zeros(4, 4, 136),) * 3, (h.half(),) * 3, (torch.zeros(4, 4, 20),) * 3):
        with pytest.raises(OspError):
            P.attention(q, k, v, None)
    with pytest.raises(OspError, match="GPU"):
        P.attention(h, h, h, None)


@gpu
def test_refusals_on_the_device():
    from optispeech_amd import packed_ops as P
    from optispeech_amd._lib import OspError
    h = torch.zeros(4, 4, 8, device=DEV)
    rows = P.PackedRows.from_offsets(offsets([4]), 4)
    one = torch.ones(1, dtype=torch.int64, device=DEV)
    for kw in (dict(prefix=one), dict(causal=True, prefix=one.int()), dict(causal=True, prefix=one.cpu()), dict(causal=True, prefix=torch.cat([one, one])),
               dict(softcap=-1.0), dict(softcap=float("nan")), dict(scale=float("inf")), dict(slopes=torch.ones(3, device=DEV)),
               dict(slopes=torch.ones(4)), dict(slopes=torch.ones(4, device=DEV, requires_grad=True)),
               dict(keys=P.PackedRows.from_offsets(offsets([2, 2]), 4)), dict(keys=P.PackedRows.from_offsets(offsets([5]), 5))):
        with pytest.raises(OspError):
            P.attention(h, h, h, rows, **kw)
    with pytest.raises(OspError, match="rows"):
        P.attention(h[:3], h[:3], h[:3], rows)
