"""Edges of the packed-row operators: what a call may hold beyond the ordinary tables of the other packed tests.  u = 2^-24."""
import pytest
import torch

from . import _packed_ref as ref
from .test_gpu_packed_attention import bounds, close, grads, offsets, randn

DEV = "cuda"
U = 2.0 ** -24
gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_bound_of_no_rows_costs_time_and_not_results(dtype):
    """longest = 0 over documents that have rows: every operator and direction gives what the right bound gives.  The same kernels with other tiles and
    splits: group norm's sums in another order (chains of at most 150 rows), attention's results within the definition's bounds"""
    from optispeech_amd import packed_ops as P
    lengths, H, D = [150, 3], 2, 32
    M, C = sum(lengths), 64
    x, g = randn(M, C, seed=1, dtype=dtype).requires_grad_(), randn(M, C, seed=2, dtype=dtype)
    q, k, v, do = (randn(M, H, D, seed=3 + i, dtype=dtype) for i in range(4))
    docs = ref.documents(lengths)
    want, tol = bounds(q, k, v, do, docs, docs, D ** -0.5, True, None, 0.0, None, dtype)
    norms, turned = [], []
    for longest in (150, 0):
        rows = P.PackedRows.from_offsets(offsets(lengths), M, longest=longest)
        w, b = torch.nn.Parameter(randn(C, seed=8)), torch.nn.Parameter(randn(C, seed=9))
        y = P.group_norm(x, w, b, 4, rows, 1e-5, "silu")
        norms.append((y.detach(),) + torch.autograd.grad(y, (x,), g) + (w.grad, b.grad))
        turned.append(P.rotary(q, k, P.Rotary(D), rows))
        close(grads(q, k, v, do, rows, causal=True), want, tol)
        with torch.no_grad():
            close((P.attention(q, k, v, rows, causal=True),), want[:1], tol[:1])
    for i, (a, b) in enumerate(zip(*norms)):
        scale = a.double().abs().max().item()
        assert scale > 0.1 and float((a.double() - b.double()).abs().max()) <= (torch.finfo(a.dtype).eps + 150 * U * (30 if i >= 2 else 1)) * scale
    assert all(torch.equal(a, b) for a, b in zip(*turned))


@gpu
def test_rotary_positions_advanced_before_the_backward_are_refused():
    """`first` belongs to the call: a counter advanced in place between forward and backward raises, as for any tensor that autograd keeps"""
    from optispeech_amd import packed_ops as P
    rows = P.PackedRows.from_offsets(offsets([3, 2]), 5)
    q, k, g = (randn(5, 2, 16, seed=i).requires_grad_() for i in range(3))
    first = torch.tensor([7, 100], dtype=torch.int64, device=DEV)
    rope = P.Rotary(16)
    yq, yk = P.rotary(q, k, rope, rows, first=first)
    first += 1
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad((yq, yk), (q, k), (g, g))
    yq, yk = P.rotary(q, k, rope, rows, first=first)
    torch.autograd.grad((yq, yk), (q, k), (g, g))


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("cap", [512.0, 600.0, 1e5, 1e7, 1e12, 1e30])
@pytest.mark.parametrize("slope", [False, True])
@pytest.mark.parametrize("lengths,H,S,D", [([300, 40], 4, 2, 64), ([129] * 40, 8, 4, 128), ([33, 5], 2, 2, 32)])
def test_caps_far_above_the_scores(dtype, cap, slope, lengths, H, S, D):
    """A cap far above the scores leaves them as they are, and with the accuracy of uncapped ones.  The bound is the uncapped one: the tanh's form adds to a score s
    at most 8 u |s| above 512 (scale / cap, its product, tanhf 2 ulp = 4 u, the product with cap log2 e and its rounding) and 16 u 512 = 8192 u up to there
    (stated separately); (D + 8) u sum |q k| grows to (D + 16) u: a factor of at most 1.2 for D >= 32."""
    from optispeech_amd import packed_ops as P
    M = sum(lengths)
    q, do = randn(M, H, D, seed=1, dtype=dtype), randn(M, H, D, seed=4, dtype=dtype)
    k, v = randn(M, S, D, seed=2, dtype=dtype), randn(M, S, D, seed=3, dtype=dtype)
    slopes = torch.tensor([0.5 ** (h + 1) for h in range(H)], device=DEV) if slope else None
    rows = P.PackedRows.from_offsets(offsets(lengths), M, longest=max(lengths))
    docs = ref.documents(lengths)
    want, tol = bounds(q, k, v, do, docs, docs, D ** -0.5, True, None, cap, slopes, dtype)
    if cap > 512 or dtype == torch.float32:
        tol = [1.25 * t for t in bounds(q, k, v, do, docs, docs, D ** -0.5, True, None, 0.0, slopes, dtype)[1]]
    close(grads(q, k, v, do, rows, causal=True, softcap=cap, slopes=slopes), want, tol)
    # a new token over the same keys
    B = len(lengths)
    last = torch.tensor([sum(lengths[:i + 1]) - 1 for i in range(B)], device=DEV)
    o = P.attention(q[last], k, v, P.PackedRows.from_offsets(offsets([1] * B), B, longest=1), keys=rows, causal=True, softcap=cap, slopes=slopes)
    close((o,), (want[0][last.cpu()],), (tol[0][last.cpu()],))


@gpu
def test_caps_out_of_range_are_refused():
    """the cap and scale / cap have to be ordinary f32 numbers: beyond that one of them is 0, infinite or a few bits"""
    from optispeech_amd import packed_ops as P
    from optispeech_amd._lib import OspError
    h = torch.zeros(4, 4, 8, device=DEV)
    rows = P.PackedRows.from_offsets(offsets([4]), 4)
    for cap, scale in ((1e-40, 1.0), (1e-37, 1.0), (1e37, 1.0), (1e38, 1.0), (1e300, 1.0), (1e-46, 1e-12), (1e46, 1e12), (1e30, 1e-7), (1e-30, 1e7)):
        with pytest.raises(OspError, match="softcap"):
            P.attention(h, h, h, rows, softcap=cap, scale=scale)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("cap,slope", [(0.0, False), (9.0, True)])
@pytest.mark.parametrize("pairs,H,S,D", [([(40, 10), (5, 5)], 2, 1, 64), ([(140, 70), (200, 129), (33, 0), (12, 12)] * 15, 12, 4, 128)])
def test_queries_that_see_nothing_may_hold_nan(dtype, cap, slope, pairs, H, S, D):
    """causal, more queries than keys: the first queries see nothing.  Whatever they and their incoming gradient hold, they get zeros and the others get
    what they get without them, bit for bit"""
    from optispeech_amd import packed_ops as P
    qlens, klens = zip(*pairs)
    M, Mk = sum(qlens), sum(klens)
    q, do = randn(M, H, D, seed=1, dtype=dtype), randn(M, H, D, seed=4, dtype=dtype)
    k, v = randn(Mk, S, D, seed=2, dtype=dtype), randn(Mk, S, D, seed=3, dtype=dtype)
    rows = P.PackedRows.from_offsets(offsets(qlens), M, longest=max(qlens))
    keys = P.PackedRows.from_offsets(offsets(klens), Mk, longest=max(klens))
    blind = torch.cat([torch.arange(nq) < nq - nk for nq, nk in pairs]).to(DEV)
    slopes = torch.tensor([0.5 ** (h + 1) for h in range(H)], device=DEV) if slope else None
    out = []
    for fill in (0.0, float("nan")):
        q[blind], do[blind] = fill, fill
        out.append(grads(q, k, v, do, rows, keys=keys, causal=True, softcap=cap, slopes=slopes))
    for a, b in zip(*out):
        assert torch.isfinite(a).all() and torch.equal(a, b)
    assert float(out[1][0][blind].detach().abs().max()) == 0.0 and float(out[1][1][blind].abs().max()) == 0.0


@gpu
@pytest.mark.parametrize("lengths,C,G", [([300], 64, 4), ([90, 7], 30, 3), ([3000, 400], 64, 4), ([40], 2048, 32)])
def test_group_norm_resolves_values_far_from_zero(lengths, C, G):
    """f32 x = 4096 + noise of 0.1, values taken as given: the mean is kept with more than 32 bits, so xhat is not shifted by its rounding (u 4096 / 0.1 =
    2.4e-3).  What remains: sums in 64 bits (at most 512 additions in one chain, each 2^-53 of a sum whose squares are (mean / deviation)^2 times the
    variance) make rstd uncertain by r = 256 2^-53 (mean / deviation)^2, and 3 u for the difference, its product and rstd's rounding: e = r + 3 u relative
    to xhat, and for the mean 512 2^-53 |mean| rstd.  Gradients (act None: dz = dy): chains of at most 128 rows in 32 bits as in the other group norm tests,
    140 u of the sums of absolute values."""
    from optispeech_amd import packed_ops as P
    M = sum(lengths)
    x, g = randn(M, C, seed=21, std=0.1) + 4096.0, randn(M, C, seed=22)
    w, b = torch.nn.Parameter(randn(C, seed=23) * 0.2 + 1), torch.nn.Parameter(randn(C, seed=24))
    xr = x.clone().requires_grad_()
    rows = P.PackedRows.from_offsets(offsets(lengths), M)
    y = P.group_norm(xr, w, b, G, rows, 1e-8)
    (dx,) = torch.autograd.grad(y, (xr,), g)
    docs = ref.documents(lengths)
    X, W, B = (t.detach().double().cpu().requires_grad_() for t in (x, w, b))
    want = ref.group_norm(X, W, B, docs, G, 1e-8, None)
    wx, ww, wb = torch.autograd.grad(want, (X, W, B), g.double().cpu())
    X, W, B, g = X.detach(), W.detach(), B.detach(), g.double().cpu()
    ytol, xtol, wtol, btol = torch.zeros_like(X), torch.zeros_like(X), torch.zeros(C).double(), torch.zeros(C).double()
    for sl in docs:
        n = sl.stop - sl.start
        xg = X[sl].reshape(n, G, C // G)
        m = xg.mean((0, 2), keepdim=True)
        var = ((xg - m) ** 2).mean((0, 2), keepdim=True)
        full = lambda t: t.expand(n, G, C // G).reshape(n, C)                                     # noqa: E731
        mean = lambda t: full(t.reshape(n, G, C // G).mean((0, 2), keepdim=True))                # noqa: E731
        rs = full(1 / torch.sqrt(var + 1e-8))
        hat = full((xg - m)) * rs
        e = (full(256 * 2.0 ** -53 * m * m / var) + 3 * U) * hat.abs() + 512 * 2.0 ** -53 * full(m.abs()) * rs
        ytol[sl] = e * W.abs() + 3 * U * ((hat * W).abs() + B.abs())
        gw = (g[sl] * W).abs()
        m2 = mean(gw * hat.abs())
        xtol[sl] = rs * (150 * U * (gw + mean(gw) + hat.abs() * m2) + e * m2 + hat.abs() * mean(gw * e)) + (256 * 2.0 ** -53 * full(m * m / var)) * wx[sl].abs()
        wtol += (g[sl].abs() * (e + 140 * U * hat.abs())).sum(0)
        btol += 140 * U * g[sl].abs().sum(0)
    for name, a, t, tol in (("y", y, want, ytol), ("dx", dx, wx, xtol), ("dw", w.grad, ww, wtol), ("db", b.grad, wb, btol)):
        err = (a.detach().double().cpu() - t.detach()).abs()
        assert bool((err <= tol + U * t.detach().abs()).all()), (name, (err - tol).max().item(), err.max().item())


@gpu
@pytest.mark.parametrize("needs_x", [True, False])
@pytest.mark.parametrize("lengths,C", [([50, 31], 32), ([50, 31], 10), ([1500], 512)])
def test_group_norm_weights_computed_from_parameters(needs_x, lengths, C):
    """a weight or bias that is itself a result (1 + gamma, a scaled table) hands its gradient on: bit for bit what a parameter of its value is given, and
    nothing is written beside it"""
    from optispeech_amd import packed_ops as P
    M = sum(lengths)
    rows = P.PackedRows.from_offsets(offsets(lengths), M)
    x, g = randn(M, C, seed=1).requires_grad_(needs_x), randn(M, C, seed=2)
    gamma, beta = torch.nn.Parameter(randn(C, seed=3)), torch.nn.Parameter(randn(C, seed=4))
    w, b = torch.nn.Parameter(1 + gamma.detach()), torch.nn.Parameter(beta.detach() * 2)
    y0 = P.group_norm(x, w, b, 2, rows, act="silu")
    y0.backward(g)
    for wt, bt in ((1 + gamma, beta * 2), (1 + gamma, b), (w, beta * 2)):
        for p in (gamma, beta, w, b, x):
            if p is not w and p is not b:
                p.grad = None
        dw, db = w.grad.clone(), b.grad.clone()
        w.grad = b.grad = None
        y = P.group_norm(x, wt, bt, 2, rows, act="silu")
        assert torch.equal(y, y0)
        y.backward(g)
        assert torch.equal(gamma.grad if wt is not w else w.grad, dw)
        assert torch.equal(beta.grad / 2 if bt is not b else b.grad, db)
        w.grad, b.grad = dw, db
    both = 1 + gamma                                                # one result as weight and bias: autograd adds the two gradients
    gamma.grad = w.grad = b.grad = None
    P.group_norm(x, both, both, 2, rows, act="silu").backward(g)
    one, two = torch.nn.Parameter(both.detach().clone()), torch.nn.Parameter(both.detach().clone())
    P.group_norm(x, one, two, 2, rows, act="silu").backward(g)
    assert torch.equal(gamma.grad, one.grad + two.grad)
    y = P.group_norm(x, both, one, 2, rows)
    with torch.no_grad():
        both += 1                                                    # a kept result changed in place
    with pytest.raises(RuntimeError, match="inplace"):
        y.backward(g)


@gpu
def test_group_norm_adds_to_strided_gradients():
    """param.grad as every second element of a buffer: its elements receive the gradient, their neighbours stay"""
    from optispeech_amd import packed_ops as P
    lengths, C = [50, 31], 32
    M = sum(lengths)
    rows = P.PackedRows.from_offsets(offsets(lengths), M)
    x, g = randn(M, C, seed=1).requires_grad_(), randn(M, C, seed=2)
    w, b, p, s = (torch.nn.Parameter(randn(C, seed=3)) for _ in range(4))
    bufs = [randn(2 * C, seed=5 + i) for i in range(3)]
    kept = [t.clone() for t in bufs]
    P.group_norm(x, w, b, 2, rows).backward(g)
    dw, db = w.grad.clone(), b.grad.clone()
    w.grad, b.grad, s.grad = (t[::2] for t in bufs)
    P.group_norm(x, w, b, 2, rows).backward(g)
    assert torch.equal(bufs[0][::2], kept[0][::2] + dw) and torch.equal(bufs[1][::2], kept[1][::2] + db)
    P.group_norm(x, s, s, 2, rows).backward(g)
    assert torch.equal(bufs[2][::2], kept[2][::2] + db + dw)
    for t, k in zip(bufs, kept):
        assert torch.equal(t[1::2], k[1::2])


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=gpu)])
def test_forward_mode_derivatives_are_refused(dev):
    """a dual tensor is not taken as a constant, in whichever place it stands"""
    import torch.autograd.forward_ad as fwd
    from optispeech_amd import packed_ops as P
    from optispeech_amd._lib import OspError
    rows = P.PackedRows.from_offsets(offsets([4]), 4) if dev == "cuda" else None
    rope = P.Rotary(8, device=dev)
    h, x, c = torch.randn(4, 2, 8, device=dev), torch.randn(4, 8, device=dev), torch.ones(8, device=dev)
    s = torch.ones(2, device=dev)
    with fwd.dual_level():
        hd, xd, cd, sd = (fwd.make_dual(t, torch.ones_like(t)) for t in (h, x, c, s))
        for f, args in ((P.rotary, (hd, h, rope, rows)), (P.rotary, (h, hd, rope, rows)), (P.group_norm, (xd, c, c, 2, rows)), (P.group_norm, (x, cd, c, 2, rows)),
                        (P.group_norm, (x, c, cd, 2, rows)), (P.attention, (hd, h, h, rows)), (P.attention, (h, hd, h, rows)), (P.attention, (h, h, hd, rows))):
            with pytest.raises(OspError, match="forward-mode"):
                f(*args)
        with pytest.raises(OspError, match="forward-mode"):
            P.attention(h, h, h, rows, slopes=sd)
        if dev == "cuda":                                            # plain tensors inside the level are computed as outside
            assert torch.isfinite(P.attention(h, h, h, rows)).all()


def _shifted(t):
    """the same values, contiguous, one element behind a 16-byte border"""
    return torch.cat([t.new_zeros(1), t.flatten()])[1:].view(t.shape)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lengths", [[70, 33], [1]])
def test_contiguous_tensors_at_odd_addresses(dtype, lengths):
    """contiguous inputs and gradients that do not start on 16 bytes, tables of one row: results of the aligned tensors, bit for bit"""
    from optispeech_amd import packed_ops as P
    H, D = 2, 32
    M = sum(lengths)
    rows = P.PackedRows.from_offsets(offsets(lengths), M)
    t = [randn(M, H, D, seed=i, dtype=dtype) for i in range(4)]
    odd = [_shifted(x) for x in t]
    assert all(x.is_contiguous() and x.data_ptr() % 16 for x in odd)
    want = grads(*t, rows, causal=True)
    for args in (odd, odd[:3] + t[3:], t[:3] + odd[3:]):
        for a, b in zip(grads(*args, rows, causal=True), want):
            assert torch.equal(a, b)
    with torch.no_grad():
        for n in (M, 1):
            r = P.PackedRows.from_offsets(offsets([n]), n, longest=n)
            assert torch.equal(P.attention(odd[0][:n], odd[1], odd[2], r, keys=P.PackedRows.from_offsets(offsets([M]), M)),
                               P.attention(t[0][:n], t[1], t[2], r, keys=P.PackedRows.from_offsets(offsets([M]), M)))
        rope = P.Rotary(D)
        for a, b in zip(P.rotary(odd[0], odd[1], rope, rows), P.rotary(t[0], t[1], rope, rows)):
            assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_one_row_and_one_head_of_any_stride(dtype):
    """dimensions of one element carry strides that say nothing; a projection's slice of one row, shifted by one element"""
    from optispeech_amd import packed_ops as P
    D = 16
    rows = P.PackedRows.from_offsets(offsets([1]), 1)
    flat = randn(3 * D + 1, seed=1, dtype=dtype)
    views = [flat.as_strided((1, 1, D), s, o) for s in ((1, 1, 1), (3, 5, 1), (D, D, 1)) for o in (0, 1)]
    for v in views:
        c = v.clone(memory_format=torch.contiguous_format)
        for a, b in zip(grads(v, v, v, v, rows), grads(c, c, c, c, rows)):
            assert torch.equal(a, b)
    w = randn(1, 3 * 2 * D + 1, seed=2, dtype=dtype)[:, 1:]
    q, k, v = (w[:, i * 2 * D:(i + 1) * 2 * D].unflatten(1, (2, D)) for i in range(3))
    for a, b in zip(grads(q, k, v, q, rows), grads(q.clone(), k.clone(), v.clone(), q.clone(), rows)):
        assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_group_norm_of_one_row_of_any_stride(dtype):
    from optispeech_amd import packed_ops as P
    C = 24
    rows = P.PackedRows.from_offsets(offsets([1]), 1)
    w, b = randn(C, seed=3), randn(C, seed=4)
    x, g = randn(C, 1, seed=1, dtype=dtype).t(), randn(C, 1, seed=2, dtype=dtype).t()
    assert x.stride() == (1, 1)
    out = []
    for copy in (False, True):
        xr, gr = ((t.clone(memory_format=torch.contiguous_format) if copy else t.detach()) for t in (x, g))
        xr.requires_grad_()
        y = P.group_norm(xr, w, b, 3, rows, act="silu")
        out.append((y.detach(),) + torch.autograd.grad(y, (xr,), gr))
    assert all(torch.equal(p, q) for p, q in zip(*out))


@gpu
def test_rotary_transformer_keeps_its_positional_dropout():
    """positional_dropout_rate acts on the frames that enter the first layer, in training only"""
    from optispeech_amd import rng
    from optispeech_amd.model.transformer import Transformer
    x, pad = randn(2, 40, 64, seed=1), torch.zeros(2, 40, dtype=torch.bool, device=DEV)
    out = {}
    for rate in (0.0, 0.5):
        torch.manual_seed(3)
        m = Transformer(dim=64, attention_heads=4, linear_units=96, num_blocks=0, dropout_rate=0.0, positional_dropout_rate=rate, attention_dropout_rate=0.0,
                        selfattention_layer_type="packed", packed=dict(rotary={})).to(DEV)
        for training in (False, True):
            rng.manual_seed(11, 0)
            with torch.no_grad():
                out[rate, training] = m.train(training)(x, pad)
    assert torch.equal(out[0.0, True], out[0.0, False]) and torch.equal(out[0.5, False], out[0.0, False])
    # no blocks: the final norm of the dropped frames.  Dropped channels share one value per row (before weight and bias): about half of them
    y = out[0.5, True]
    low = (y - y.median(-1, keepdim=True).values).abs() < 1e-6
    assert not torch.equal(y, out[0.0, True]) and 0.4 < low.float().mean().item() < 0.6


@gpu
def test_taped_segments_with_the_packed_attention_equal_eager():
    """The Transformer backbone with packed attention, f32: the recorded acoustic model replayed on ANOTHER ragged batch of the same padded shape (other lengths, so
    other documents).  Steps: batch 0 twice (the second records), 1, 1, 0 without an optimizer update; gradients of both networks, taped against
    eager, to the tolerance of two eager runs (f32 atomics of the weight-gradient kernels)."""
    from oracle import schema as S
    from optispeech_amd import precision, rng, tape
    from optispeech_amd.config import ModelConfig, make_optispeech, synthetic_batch
    precision.set_precision("f32")
    keep = tape.ENABLED

    def run(tapes):
        tape.ENABLED = tapes
        c = S.SMALL
        cfg = ModelConfig(dim=c.dim, enc_inter=c.enc_inter, dec_inter=c.dec_inter, dur=c.dur + (0.0,), pitch=c.pitch + (0.0,),
                          energy=c.energy + (0.0,), voc_dim=c.voc_dim, voc_inter=c.voc_inter, voc_layers=c.voc_layers,
                          backbone="transformer", packed_attention=dict(rotary={}, softcap=30.0, distance_slopes=True)).no_dropout()
        torch.manual_seed(7)
        rng.manual_seed(7, 0)
        m = make_optispeech(cfg, batch_size=2, pretraining_steps=0).to(DEV).train()
        m.tape_segments = True
        got = {}
        for name, o in zip(("g", "d"), m.optimizers()):
            o.step = (lambda n, oo: (lambda *a, **k: got.__setitem__(n, oo.arena.grad.detach().clone())))(name, o)
        out = []
        for r in (0, 0, 1, 1, 0):
            b = synthetic_batch(2, 24, 96, cfg, seed=50 + r, ragged=True, device=DEV)
            m.generator.segment_rand01 = torch.tensor([0.25 + 0.5 * r, 0.6 - 0.3 * r], device=DEV)
            m.training_step(b, 0)
            torch.cuda.synchronize()
            out.append((got["g"].clone(), got["d"].clone()))
        names = [r[0].meta["names"] for r in m._tape_am.cache.values() if r is not tape.EAGER] if tapes else []
        return out, names

    try:
        s0 = tape.stats()
        (a, _), (b, names) = run(False), run(True)
        s1 = tape.stats()
    finally:
        tape.ENABLED = keep
    assert s1["replayed"] - s0["replayed"] >= 6 and s1["poisoned"] == s0["poisoned"], (s0, s1)
    assert names and any("osp_packed_attention_fwd" in n for n in names)
    for i, ((ga, da), (gb, db)) in enumerate(zip(a, b)):
        assert ((ga - gb).norm() / ga.norm()).item() < 1e-5, (i, "generator")
        assert ((da - db).norm() / da.norm()).item() < 1e-5, (i, "discriminator")


@gpu
def test_new_tokens_for_many_documents(monkeypatch):
    """40 000 documents: the split kernel's workspace passes 256 MB but not the cache, and the call stays with it; documents all over the batch against the
    definition, rows of no document zero"""
    from optispeech_amd import packed_ops as P
    B, T, H, S, D = 40000, 64, 32, 4, 64
    g = torch.Generator(device=DEV).manual_seed(1)
    q = torch.randn(B + 3, H, D, generator=g, device=DEV).bfloat16()
    k, v = (torch.randn(B * T, S, D, generator=g, device=DEV).bfloat16() for _ in range(2))
    klens = torch.arange(B, device=DEV) % (T + 1)
    rows = P.PackedRows.from_offsets(torch.arange(B + 1, device=DEV), B + 3, longest=1)
    names, call = [], P.call
    monkeypatch.setattr(P, "call", lambda name, *a: (names.append(name), call(name, *a)))
    o = P.attention(q, k, v, rows, keys=P.PackedRows.from_padded(klens, T), causal=True)
    assert "osp_packed_attention_token" in names
    assert P._size("osp_packed_attention_token_workspace_bytes", B, B + 3, T, H, S, D) > 1 << 28
    for b in (0, 1, 63, 64, 65, 20001, 33333, B - 1):
        n = int(klens[b])
        want, tol = bounds(q[b:b + 1], k[b * T:b * T + n], v[b * T:b * T + n], q[b:b + 1], [slice(0, 1)], [slice(0, n)], D ** -0.5, True, None, 0.0, None,
                           torch.bfloat16)
        close((o[b:b + 1],), want[:1], tol[:1])
    assert float(o[B:].abs().max()) == 0.0


@gpu
def test_group_norm_parameters_changed_before_the_backward_are_refused():
    """the gradients would be those of other weights: in-place steps in between raise, frozen weights and those of inference mode are used as they are"""
    from optispeech_amd import packed_ops as P
    rows = P.PackedRows.from_offsets(offsets([30, 11]), 41)
    x, g = randn(41, 32, seed=1).requires_grad_(), randn(41, 32, seed=2)
    for which in (0, 1):
        p = [torch.nn.Parameter(randn(32, seed=3)), torch.nn.Parameter(randn(32, seed=4))]
        y = P.group_norm(x, *p, 4, rows, act="silu")
        with torch.no_grad():
            p[which] += 0.1
        with pytest.raises(RuntimeError, match="inplace"):
            y.backward(g)
        assert p[0].grad is None and p[1].grad is None
        P.group_norm(x, *p, 4, rows, act="silu").backward(g)
    with torch.inference_mode():
        w, b = randn(32, seed=3), randn(32, seed=4)
    (a,) = torch.autograd.grad(P.group_norm(x, w, b, 4, rows, act="silu"), (x,), g)
    (c,) = torch.autograd.grad(P.group_norm(x, w.clone(), b.clone(), 4, rows, act="silu"), (x,), g)
    assert torch.equal(a, c)
