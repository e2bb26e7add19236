"""Rotary positions and group norm on packed rows against their definitions in 64 bits.

A rounding to type t is off by at most eps(t) / 2 of the value (bf16 2^-8, f32 2^-24); u = 2^-24 below."""
import pytest
import torch

from . import _packed_ref as ref

DEV = "cuda"
U = 2.0 ** -24
gpu = pytest.mark.gpu


def half_eps(t):
    return torch.finfo(t).eps / 2


def offsets(lengths, start=0):
    return torch.tensor([start + sum(lengths[:i]) for i in range(len(lengths) + 1)], dtype=torch.int64, device=DEV)


def randn(*shape, seed, dtype=torch.float32, std=1.0, mean=0.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * std + mean).to(dtype).to(DEV)


# ------------------------------------------------------------------------------------------------------------------ the rows
@gpu
@pytest.mark.parametrize("off,rows", [([0, 5, 5, 133, 400], 400), ([3, 3, 131, 132], 200), ([0, 0], 7), ([0, 10, 4, 12], 12),
                                      ([-5, 3, 900], 300), ([0, 1] + [129 * i for i in range(1, 1500)], 129 * 1500)])
def test_rows_from_offsets_cover_the_table(off, rows):
    """begin / length are the clamped running maxima, and the tiles cover every row of the table exactly once"""
    from optispeech_amd.packed_ops import PackedRows
    r = PackedRows.from_offsets(torch.tensor(off, dtype=torch.int64, device=DEV), rows)
    run, want = 0, []
    for o in off:
        run = max(run, min(max(o, 0), rows))
        want.append(run)
    assert r.begin.tolist() == want[:-1]
    assert r.length.tolist() == [b - a for a, b in zip(want[:-1], want[1:])]
    ndoc, nall = r.ntiles.tolist()
    tiles = r.tiles.view(-1, 4)[:nall].tolist()
    seen = [0] * rows
    base, per_doc = r.base.tolist(), {}
    for i, (doc, row0, n, i0) in enumerate(tiles):
        assert (doc >= 0) == (i < ndoc) and 1 <= n <= 128
        if doc >= 0:
            assert row0 == want[doc] + i0 and i0 % 128 == 0 and row0 + n <= want[doc + 1] and (n == 128 or row0 + n == want[doc + 1])
            per_doc.setdefault(doc, set()).add(base[doc] + i0 // 128)
        for x in range(row0, row0 + n):
            seen[x] += 1
    assert all(s == 1 for s in seen)
    slots = sorted(s for v in per_doc.values() for s in v)
    assert slots == list(range(ndoc))


@gpu
def test_rows_from_padded_lengths():
    from optispeech_amd.packed_ops import PackedRows
    r = PackedRows.from_padded(torch.tensor([3, 0, 300, 999, -4], dtype=torch.int64, device=DEV), 300)
    assert r.begin.tolist() == [0, 300, 600, 900, 1200] and r.length.tolist() == [3, 0, 300, 300, 0]
    seen = [0] * 1500
    for doc, row0, n, i0 in r.tiles.view(-1, 4)[:int(r.ntiles[1])].tolist():
        for x in range(row0, row0 + n):
            seen[x] += 1
            assert (x % 300 < r.length.tolist()[x // 300]) == (doc >= 0)
    assert all(s == 1 for s in seen)


# ------------------------------------------------------------------------------------------------------------------ rotary
def rotary_close(got, x, docs, firsts, rope, inverse=False):
    """angle: |a| <= pi / 4 rounded (0.79 u) + series 2e-9 + evaluation of sin / cos (2 u) + magnitude (u) + product and fma (2 u) <= 6 u of
    mag (|a| + |b|) for a pair; then the rounding to the result's type.  Untouched channels are exact up to that rounding."""
    want = ref.rotary(x, docs, firsts, rope.turns, rope.magnitude, rope.layout, inverse)
    xa = x.detach().double().cpu().abs()
    R = rope.channels
    pair = torch.zeros_like(xa)
    ia, ib = (slice(0, R // 2), slice(R // 2, R)) if rope.layout == "half" else (slice(0, R, 2), slice(1, R, 2))
    pair[..., ia] = pair[..., ib] = xa[..., ia] + xa[..., ib]
    tol = half_eps(got.dtype) * (want.abs() + 6 * U * rope.magnitude * pair) + 6 * U * rope.magnitude * pair
    err = (got.detach().double().cpu() - want).abs()
    assert bool((err <= tol).all()), (err - tol).max().item()


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("lengths,tail,H,S,D,R,first,scaling", [
    ([1], 0, 2, 2, 128, 128, 1000003, "base"), ([5, 0, 131, 64], 7, 4, 2, 64, 32, 0, "linear"), ([700, 3], 0, 3, 1, 40, 24, 12345, "none"),
    ([17, 1, 1], 2, 1, 1, 2, 2, 5, "none"), ([200], 1, 6, 3, 30, 10, 1 << 40, "parts"), ([129, 300], 0, 8, 2, 96, 96, 0, "parts")])
def test_rotary_forward_and_gradient(dtype, layout, lengths, tail, H, S, D, R, first, scaling):
    from optispeech_amd import packed_ops as P
    M = sum(lengths) + tail
    rope = P.Rotary(R, layout=layout, scaling=scaling, factor=4.0, original_length=2000)
    rows = P.PackedRows.from_offsets(offsets(lengths), M, longest=max(lengths))
    q, k = randn(M, H, D, seed=1, dtype=dtype).requires_grad_(), randn(M, S, D, seed=2, dtype=dtype).requires_grad_()
    firsts = [first + 3 * i for i in range(len(lengths))]
    fd = torch.tensor(firsts, dtype=torch.int64, device=DEV) if first else None
    firsts = firsts if first else [0] * len(lengths)
    yq, yk = P.rotary(q, k, rope, rows, first=fd)
    docs = ref.documents(lengths)
    rotary_close(yq, q, docs, firsts, rope)
    rotary_close(yk, k, docs, firsts, rope)
    gq, gk = randn(M, H, D, seed=3, dtype=dtype), randn(M, S, D, seed=4, dtype=dtype)
    dq, dk = torch.autograd.grad((yq, yk), (q, k), (gq, gk))
    rotary_close(dq, gq, docs, firsts, rope, inverse=True)
    rotary_close(dk, gk, docs, firsts, rope, inverse=True)
    assert float(yq[sum(lengths):].abs().sum()) == 0.0 and float(dk[sum(lengths):].abs().sum()) == 0.0


@gpu
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("cast", [(torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32)])
def test_rotary_reads_views_of_one_projection_and_casts(layout, cast):
    """q and k as views into one (rows, 3 * heads * width + 1) projection: row strides, an odd base address, another result type;
    rows of a padded batch; NaN in the rows of no document"""
    from optispeech_amd import packed_ops as P
    B, T, H, D = 3, 50, 2, 32
    lens = [50, 0, 13]
    rope = P.Rotary(D, layout=layout)
    for shift in (0, 1):
        w = randn(B * T, 3 * H * D + shift, seed=5, dtype=cast[0])
        for b, n in enumerate(lens):
            w[b * T + n:(b + 1) * T] = float("nan")
        q, k = w[:, shift:shift + H * D].unflatten(1, (H, D)), w[:, shift + H * D:shift + 2 * H * D].unflatten(1, (H, D))
        rows = P.PackedRows.from_padded(torch.tensor(lens, dtype=torch.int64, device=DEV), T)
        yq, yk = P.rotary(q, k, rope, rows, out_dtype=cast[1])
        assert yq.dtype == cast[1]
        docs = [slice(b * T, b * T + n) for b, n in enumerate(lens)]
        clean = torch.nan_to_num(q), torch.nan_to_num(k)
        rotary_close(yq, clean[0], docs, [0] * B, rope)
        rotary_close(yk, clean[1], docs, [0] * B, rope)


@gpu
def test_rotary_scalings():
    """each frequency rule against its formula"""
    import math
    from optispeech_amd import packed_ops as P
    two_pi = 2 * math.pi
    plain = P.Rotary(64).turns.cpu() * two_pi
    assert torch.allclose(plain, 10000.0 ** (-torch.arange(32, dtype=torch.float64) / 32), rtol=1e-12)
    assert torch.allclose(P.Rotary(64, scaling="linear", factor=4.0).turns.cpu() * two_pi, plain / 4, rtol=1e-12)
    based = P.Rotary(64, scaling="base", factor=8.0).turns.cpu() * two_pi
    assert based[0] == plain[0] and torch.allclose(based[-1], plain[-1] / 8, rtol=1e-12)
    rope = P.Rotary(64, scaling="parts", factor=8.0, original_length=2000)
    parts = rope.turns.cpu() * two_pi
    turns = 2000 * plain / two_pi
    assert torch.allclose(parts[turns >= 32], plain[turns >= 32], rtol=1e-12) and torch.allclose(parts[turns <= 1], plain[turns <= 1] / 8, rtol=1e-12)
    assert bool((parts <= plain * (1 + 1e-12)).all() and (parts >= plain / 8 * (1 - 1e-12)).all()) and rope.magnitude == 1 + 0.1 * math.log(8.0)


# ------------------------------------------------------------------------------------------------------------------ group norm
CASES = [([1], 0, 8, 2), ([37, 17], 0, 64, 4), ([5, 0, 131, 64], 7, 100, 4), ([700, 3, 129], 1, 384, 8), ([1, 1, 2], 3, 10, 5), ([513], 0, 2048, 32),
         ([260, 255], 9, 36, 1), ([64], 0, 40, 40), ([800, 5, 450], 2, 128, 2), ([400, 130], 0, 256, 2), ([1100], 0, 32, 2)]


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("act", [None, "relu", "gelu", "silu"])
@pytest.mark.parametrize("lengths,tail,C,G", CASES)
def test_group_norm_forward_and_gradients(dtype, act, lengths, tail, C, G):
    """Forward, with a = |mean| rstd |w|, h = |xhat w|: the mean's rounding (u a), the difference (u h), the product with the rounded rstd (2 u h),
    the fma (u |z|), the activation (slope <= 1.13; its own evaluation 4 u |z|, the bf16 form 1.5e-7 |z| = 2.6 u |z|): 1.2 u (a + 3 h + 6 |z| ),
    then the rounding to the result's type.
    Gradients: the same relative errors enter act' (|act''| <= 1) and xhat; with e = u (a + 3 h + 6 |z| + 4) for the error of act', the terms of
    dx carry 8 u of their own size + e |dy w| each, their means the same averaged, and the sums over a workgroup's rows (at most 128 in a chain)
    128 u of the sum of absolute values.  dw, db: the same bound summed over rows."""
    from optispeech_amd import packed_ops as P
    M, eps = sum(lengths) + tail, 1e-5
    centre, spread = randn(C, seed=11, std=2.0), randn(C, seed=12).abs() + 0.25
    x = (randn(M, C, seed=13) * spread + centre).to(dtype).requires_grad_()
    w = torch.nn.Parameter(randn(C, seed=14, std=0.2, mean=1.0))
    b = torch.nn.Parameter(randn(C, seed=15, std=0.2))
    g = randn(M, C, seed=16, dtype=dtype)
    rows = P.PackedRows.from_offsets(offsets(lengths), M, longest=max(lengths))
    y = P.group_norm(x, w, b, G, rows, eps, act)
    (dx,) = torch.autograd.grad(y, (x,), g)
    docs = ref.documents(lengths)
    X, W, Bb = (t.detach().double().cpu().requires_grad_() for t in (x, w, b))
    want = ref.group_norm(X, W, Bb, docs, G, eps, act)
    wx, ww, wb = torch.autograd.grad(want, (X, W, Bb), g.double().cpu())
    want = want.detach()
    # the pieces of the bounds
    A, Hh, Z, RS, CNT = (torch.zeros((M, C), dtype=torch.float64) for _ in range(5))
    Xd, Wd, Bd = X.detach(), W.detach(), Bb.detach()
    for sl in docs:
        n = sl.stop - sl.start
        if not n:
            continue
        xg = Xd[sl].reshape(n, G, C // G)
        m = xg.mean((0, 2), keepdim=True)
        rs = 1 / torch.sqrt(((xg - m) ** 2).mean((0, 2), keepdim=True) + eps)
        full = lambda t: t.expand(n, G, C // G).reshape(n, C)                                     # noqa: E731
        A[sl], Hh[sl], RS[sl] = full(m.abs() * rs) * Wd.abs(), full((xg - m) * rs).abs() * Wd.abs(), full(rs)
        Z[sl] = full((xg - m) * rs) * Wd + Bd
    base = 1.2 * U * (A + 3 * Hh + 6 * Z.abs())
    err = (y.detach().double().cpu() - want).abs()
    tol = half_eps(dtype) * (want.abs() + base) + base
    assert bool((err <= tol).all()), (err - tol).max().item()
    if act == "relu":                                                # the slope jumps at 0: values inside the forward's error of 0 are left out
        if bool((Z.abs() <= 2 * base)[:sum(lengths)].any()):
            return
    G64 = g.double().cpu()
    e = U * (A + 3 * Hh + 6 * Z.abs() + 4)
    t1 = (G64 * Wd).abs() * 1.13                                     # |gw|
    hat = Hh / Wd.abs().clamp_min(1e-30)
    dtol, wtol, btol = torch.zeros((M, C), dtype=torch.float64), torch.zeros(C, dtype=torch.float64), torch.zeros(C, dtype=torch.float64)
    ehat = U * (A / Wd.abs().clamp_min(1e-30) + 3 * hat)             # error of xhat
    for sl in docs:
        n = sl.stop - sl.start
        if not n:
            continue
        mean = lambda t: t.reshape(n, G, C // G).mean((0, 2), keepdim=True).expand(n, G, C // G).reshape(n, C)   # noqa: E731
        e1 = 140 * U * t1[sl] + e[sl] * (G64 * Wd)[sl].abs()
        e2 = e1 * hat[sl] + t1[sl] * ehat[sl]
        m2 = mean(t1[sl] * hat[sl])
        dtol[sl] = RS[sl] * (e1 + mean(e1) + 8 * U * (mean(t1[sl]) + hat[sl] * m2) + hat[sl] * mean(e2) + ehat[sl] * m2)
        e1w = 140 * U * 1.13 * G64[sl].abs() + e[sl] * G64[sl].abs()
        btol += e1w.sum(0)
        wtol += (e1w * hat[sl] + 1.13 * G64[sl].abs() * ehat[sl]).sum(0)
    err = (dx.detach().double().cpu() - wx).abs()
    tol = half_eps(dtype) * (wx.abs() + dtol) + dtol
    assert bool((err <= tol).all()), (err - tol).max().item()
    assert bool(((w.grad.double().cpu() - ww).abs() <= wtol + U * ww.abs()).all())
    assert bool(((b.grad.double().cpu() - wb).abs() <= btol + U * wb.abs()).all())
    n = sum(lengths)
    assert float(y[n:].abs().sum()) == 0.0 and float(dx[n:].abs().sum()) == 0.0


@gpu
def test_group_norm_mean_far_above_the_deviation():
    """x = 4096 + noise of 0.01: sums of squares in 32 bits would leave nothing of the variance; what remains is the rounding of x itself
    (taken as given) and of the mean (u 4096 rstd)"""
    from optispeech_amd import packed_ops as P
    x = randn(300, 64, seed=21, std=0.01, mean=4096.0)
    w, b = torch.ones(64, device=DEV), torch.zeros(64, device=DEV)
    rows = P.PackedRows.from_offsets(offsets([300]), 300)
    y = P.group_norm(x, w, b, 4, rows, 1e-8, None)
    want = ref.group_norm(x.double().cpu(), w.double().cpu(), b.double().cpu(), ref.documents([300]), 4, 1e-8, None)
    rstd = 1.0 / x.double().std().item()
    assert (y.double().cpu() - want).abs().max().item() <= 2 * U * 4096 * rstd + 8 * U * want.abs().max().item()


@gpu
def test_group_norm_many_partials_take_the_separate_finish():
    """a document of 30 000 rows and 32 groups: its partials are added by a launch of their own"""
    from optispeech_amd import packed_ops as P
    M, C, G = 30100, 64, 32
    lengths = [30000, 3, 0, 97]
    x = randn(M, C, seed=31, mean=0.5)
    w, b = randn(C, seed=32), randn(C, seed=33)
    rows = P.PackedRows.from_offsets(offsets(lengths), M)
    y = P.group_norm(x, w, b, G, rows, 1e-5, "silu")
    want = ref.group_norm(x.double().cpu(), w.double().cpu(), b.double().cpu(), ref.documents(lengths), G, 1e-5, "silu")
    z = 1.2 * U * (2 + 9 * 6 * w.double().cpu().abs().max().item() + 6)          # |xhat| <= 6 here
    assert ((y.double().cpu() - want).abs() <= z + U * want.abs()).all()


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_group_norm_beyond_the_hosts_bound(dtype):
    """documents longer than ``longest`` says: the rows a workgroup does not keep are read again, results agree with the right bound's
    (the same sums in another order: 64-bit in the forward, chains of at most 900 rows in the backward)"""
    from optispeech_amd import packed_ops as P
    lengths, C, G = [900, 3, 400], 64, 4
    M = sum(lengths)
    x, g = randn(M, C, seed=1, dtype=dtype).requires_grad_(), randn(M, C, seed=2, dtype=dtype)
    out = []
    for longest in (900, 7):
        w, b = torch.nn.Parameter(randn(C, seed=3)), torch.nn.Parameter(randn(C, seed=4))
        rows = P.PackedRows.from_offsets(offsets(lengths), M, longest=longest)
        y = P.group_norm(x, w, b, G, rows, 1e-5, "gelu")
        out.append((y.detach(),) + torch.autograd.grad(y, (x,), g) + (w.grad, b.grad))
    for i, (a, b) in enumerate(zip(*out)):
        scale = a.double().abs().max().item()
        assert float((a.double() - b.double()).abs().max()) <= (2 * half_eps(a.dtype) + 900 * U * (30 if i >= 2 else 1)) * scale


@gpu
def test_group_norm_strided_input_padded_rows_with_nan_and_frozen_weights():
    """x as a column slice of a wider tensor at an odd element, rows of no document hold NaN, weights want no gradient; parameter gradients of
    a second call add to the first one's"""
    from optispeech_amd import packed_ops as P
    B, T, C = 3, 40, 24
    lens = [40, 0, 11]
    big = randn(B * T, C + 3, seed=41)
    for i, n in enumerate(lens):
        big[i * T + n:(i + 1) * T] = float("nan")
    rows = P.PackedRows.from_padded(torch.tensor(lens, dtype=torch.int64, device=DEV), T)
    docs = [slice(i * T, i * T + n) for i, n in enumerate(lens)]
    g = randn(B * T, C, seed=42)
    for i, n in enumerate(lens):
        g[i * T + n:(i + 1) * T] = float("nan")
    w, b = torch.nn.Parameter(torch.ones(C, device=DEV)), torch.nn.Parameter(torch.zeros(C, device=DEV), requires_grad=False)
    x = big.detach().requires_grad_()
    grads = []
    for _ in range(2):
        y = P.group_norm(x[:, 1:1 + C], w, b, 3, rows, 1e-5, "silu")
        (dx,) = torch.autograd.grad(y, (x,), g)
        grads.append(w.grad.clone())
    assert b.grad is None and torch.equal(grads[1], grads[0] + grads[0])
    xs = torch.nan_to_num(big)[:, 1:1 + C].double().cpu().requires_grad_()
    want = ref.group_norm(xs, w.detach().double().cpu(), b.double().cpu(), docs, 3, 1e-5, "silu")
    (wx,) = torch.autograd.grad(want, (xs,), torch.nan_to_num(g).double().cpu())
    scale = 40 * U
    assert ((y.detach().double().cpu() - want.detach()).abs() <= scale * (1 + want.detach().abs())).all()
    assert ((dx[:, 1:1 + C].double().cpu() - wx).abs() <= 200 * U * wx.abs().max()).all()


@gpu
def test_group_norm_weights_alone_want_a_gradient():
    """x without a gradient (the first layer, or a frozen one below): the weights' gradients are those of the full backward"""
    from optispeech_amd import packed_ops as P
    for lengths, C in (([50, 31], 32), ([50, 31], 10), ([3000], 512)):
        M = sum(lengths) + 2
        rows = P.PackedRows.from_offsets(offsets(lengths), M)
        x, g, got = randn(M, C, seed=1), randn(M, C, seed=2), []
        for needs in (True, False):
            w, b = torch.nn.Parameter(randn(C, seed=3)), torch.nn.Parameter(randn(C, seed=4))
            P.group_norm(x.clone().requires_grad_(needs), w, b, 2, rows, 1e-5, "silu").backward(g)
            got.append((w.grad, b.grad))
        assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])


@gpu
def test_group_norm_backward_captured_beside_a_living_eager_graph():
    """the parameters have no autograd node: an eager result that still holds its graph does not reach into the capture"""
    from optispeech_amd import packed_ops as P
    lengths, C = [60, 41], 64
    rows = P.PackedRows.from_offsets(offsets(lengths), 101)
    x, g = randn(101, C, seed=1), randn(101, C, seed=2)
    w, b = torch.nn.Parameter(randn(C, seed=3)), torch.nn.Parameter(randn(C, seed=4))
    w.grad, b.grad = torch.zeros_like(w), torch.zeros_like(b)
    alive = P.group_norm(x, w, b, 4, rows, 1e-5, "silu")

    def step():
        w.grad.zero_(), b.grad.zero_()
        y = P.group_norm(x, w, b, 4, rows, 1e-5, "silu")
        y.backward(g)
        return y.detach()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = step()
    for i in range(3):
        x.copy_(randn(101, C, seed=10 + i))
        graph.replay()
        torch.cuda.synchronize()
        got = [y.clone(), w.grad.clone(), b.grad.clone()]
        for a, e in zip(got, (step(), w.grad, b.grad)):
            assert torch.equal(a, e)
    assert alive.grad_fn is not None


@gpu
@pytest.mark.parametrize("started", [False, True])
def test_group_norm_one_parameter_as_weight_and_bias(started):
    """its gradient is the sum of both; ``started``: a gradient is there already.  Each gradient is rounded once and so is every sum: the same
    operations as with two parameters, in the same order"""
    from optispeech_amd import packed_ops as P
    for lengths, C in (([50, 31], 32), ([50, 31], 10)):
        M = sum(lengths)
        rows = P.PackedRows.from_offsets(offsets(lengths), M)
        x, g = randn(M, C, seed=1).requires_grad_(), randn(M, C, seed=2)
        p, w, b = (torch.nn.Parameter(randn(C, seed=3)) for _ in range(3))
        had = randn(C, seed=5) if started else torch.zeros(C, device=DEV)
        if started:
            p.grad = had.clone()
        P.group_norm(x, p, p, 2, rows).backward(g)
        P.group_norm(x, w, b, 2, rows).backward(g)
        assert torch.equal(p.grad, w.grad + (b.grad + had))


@gpu
def test_rotary_of_broadcast_heads_and_rows():
    """heads and rows of stride 0 are read in place; their gradient is the sum over the copies, as autograd forms it"""
    from optispeech_amd import packed_ops as P
    lengths, D = [9, 4], 16
    M = sum(lengths)
    rows, rope = P.PackedRows.from_offsets(offsets(lengths), M), P.Rotary(D)
    for shape, size in (((M, 1, D), (M, 3, D)), ((1, 3, D), (M, 3, D)), ((1, 1, D), (M, 3, D))):
        t, g = randn(*shape, seed=1), randn(M, 3, D, seed=2)
        a, b = t.clone().requires_grad_(), t.clone().requires_grad_()
        ya, yb = P.rotary(a.expand(size), g, rope, rows)[0], P.rotary(b.expand(size).contiguous(), g, rope, rows)[0]
        assert torch.equal(ya, yb)
        assert torch.equal(torch.autograd.grad(ya, (a,), g)[0], torch.autograd.grad(yb, (b,), g)[0])


@gpu
def test_refused_sizes():
    from optispeech_amd import packed_ops as P
    from optispeech_amd._lib import OspError
    with pytest.raises(OspError, match="rows"):
        P.PackedRows.from_offsets(offsets([1]), 2 ** 31 - 65535)
    wide = torch.zeros(1, 1, 1, device=DEV, dtype=torch.bfloat16).expand(1, 65536, 2048)       # 2^27 channels in a row
    with pytest.raises(OspError, match="channels"):
        P.rotary(wide, wide[:, :1], P.Rotary(8), P.PackedRows.from_offsets(offsets([1]), 1))


@gpu
def test_group_norm_gradient_against_differences():
    """<dx, u> against the central difference of L = sum y g along u, h = 1/32: truncation h^2 / 6 |L'''| and rounding 2 u sum |y g| / (2 h); both
    below 1e-3 of |u| |dx| at these sizes"""
    from optispeech_amd import packed_ops as P
    lengths, C = [33, 20], 16
    x, u, g = (randn(53, C, seed=s) for s in (51, 52, 53))
    w, b = torch.nn.Parameter(randn(C, seed=54, std=0.2, mean=1.0)), torch.nn.Parameter(randn(C, seed=55))
    rows = P.PackedRows.from_offsets(offsets(lengths), 53)
    loss = lambda t: float((P.group_norm(t, w, b, 4, rows, 1e-5, "silu").double() * g.double()).sum())       # noqa: E731
    h = 1.0 / 32
    with torch.no_grad():
        num = (loss(x + h * u) - loss(x - h * u)) / (2 * h)
    xr = x.clone().requires_grad_()
    (dx,) = torch.autograd.grad(P.group_norm(xr, w, b, 4, rows, 1e-5, "silu"), (xr,), g)
    got = float((dx.double() * u.double()).sum())
    assert abs(got - num) <= 1e-3 * float(dx.double().norm() * u.double().norm())


# ------------------------------------------------------------------------------------------------------------------ refusals (no GPU work)
def test_refusals():
    from optispeech_amd import packed_ops as P
    from optispeech_amd._lib import OspError
    x = torch.zeros(4, 8)
    with pytest.raises(OspError, match="int64"):
        P.PackedRows.from_offsets(torch.zeros(3, dtype=torch.int32), 4)
    with pytest.raises(OspError, match="GPU"):
        P.PackedRows.from_offsets(torch.zeros(3, dtype=torch.int64), 4)
    for bad in (dict(channels=3), dict(channels=4, layout="other"), dict(channels=4, scaling="x"), dict(channels=4, scaling="linear", factor=0.5),
                dict(channels=2, scaling="base", factor=2.0), dict(channels=4, scaling="parts", factor=2.0), dict(channels=4, base=0.0),
                dict(channels=4, scaling="parts", factor=2.0, original_length=10, slow=3.0, fast=3.0)):
        with pytest.raises(OspError):
            P.Rotary(device="cpu", **bad)
    rope = P.Rotary(8, device="cpu")
    h = torch.zeros(4, 2, 8)
    for q, k in ((h, h[:3]), (h[0], h[0]), (h, torch.zeros(4, 2, 16)), (h, h.bfloat16()), (h[..., :4], h[..., :4])):
        with pytest.raises(OspError):
            P.rotary(q, k, rope, None)
    with pytest.raises(OspError, match="out_dtype"):
        P.rotary(h, h, rope, None, out_dtype=torch.float16)
    with pytest.raises(OspError, match="GPU"):
        P.group_norm(x, torch.ones(8), torch.zeros(8), 2, None)


@gpu
def test_refusals_on_the_device():
    from optispeech_amd import packed_ops as P
    from optispeech_amd._lib import OspError
    rows = P.PackedRows.from_offsets(offsets([4]), 4)
    x, w = torch.zeros(4, 8, device=DEV), torch.ones(8, device=DEV)
    for bad in (dict(groups=3), dict(groups=0), dict(act="tanh"), dict(eps=0.0), dict(weight=w[:7]), dict(weight=w.double()), dict(bias=w.cpu()),
                dict(x=x[:3]), dict(x=x.half()), dict(x=torch.zeros(4, 4096, device=DEV))):
        kw = dict(x=x, weight=w, bias=w, groups=2, rows=rows)
        kw.update(bad)
        with pytest.raises(OspError):
            P.group_norm(**kw)
    h = torch.zeros(4, 2, 8, device=DEV)
    with pytest.raises(OspError, match="first"):
        P.rotary(h, h, P.Rotary(8), rows, first=torch.zeros(2, dtype=torch.int64, device=DEV))
    with pytest.raises(OspError, match="rows"):
        P.rotary(h[:3], h[:3], P.Rotary(8), rows)
