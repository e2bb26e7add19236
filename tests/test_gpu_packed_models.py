"""The packed attention and group norm inside the Transformer and Conformer backbones: rotary positions, capped scores, shared key heads, causal streams,
utterances packed behind each other.  Whole backbones are held to the package's model tolerances: 1e-3 of the tensor's scale in the f32 mode,
3e-2 in the bf16 mode."""
import numpy as np
import pytest
import torch

from . import _packed_ref as ref

DEV = "cuda"
gpu = pytest.mark.gpu


def relerr(a, b):
    a, b = a.detach().double().cpu(), b.detach().double().cpu()
    return ((a - b).abs().max() / b.abs().max().clamp_min(1e-30)).item()


def _lin(P, x, name):
    w = P[name + ".weight"]
    return x @ (w[:, 0] if w.dim() == 3 and w.shape[1] == 1 else w[..., 0] if w.dim() == 3 else w).T + P[name + ".bias"]


def _ln(P, x, name):
    m = x.mean(-1, keepdim=True)
    return (x - m) / torch.sqrt(((x - m) ** 2).mean(-1, keepdim=True) + 1e-12) * P[name + ".weight"] + P[name + ".bias"]


def _attend(P, x, name, att):
    """one utterance (n, C), float64"""
    n, C = x.shape
    d, docs = att.d_k, [slice(0, x.shape[0])]
    q, k, v = (_lin(P, x, f"{name}.linear_{c}").view(n, -1, d) for c in "qkv")
    if att._rotary is not None:
        turns = 10000.0 ** (-2.0 * torch.arange(d // 2, dtype=torch.float64) / d) / (2 * np.pi)

        def turn(t):                                              # the half layout, differentiable
            a = 2 * np.pi * torch.arange(n, dtype=torch.float64)[:, None, None] * turns
            c, s, u, w = a.cos(), a.sin(), t[..., :d // 2], t[..., d // 2:]
            return torch.cat([u * c - w * s, u * s + w * c], -1)
        q, k = turn(q), turn(k)
    slopes = None if att._slopes is None else att._slopes.cpu()
    o = ref.attention(q, k, v, docs, docs, d ** -0.5, att.causal, None, att.softcap, slopes)
    return _lin(P, o.reshape(n, C), name + ".linear_out")


def transformer_ref(P, x, m):
    for i, layer in enumerate(m.transformer.encoders):
        pre = f"transformer.encoders.{i}."
        x = x + _attend(P, _ln(P, x, pre + "norm1"), pre + "self_attn", layer.self_attn)
        x = x + _lin(P, _lin(P, _ln(P, x, pre + "norm2"), pre + "feed_forward.w_1").clamp_min(0), pre + "feed_forward.w_2")
    return _ln(P, x, "transformer.after_norm")


def make_transformer(**packed):
    from optispeech_amd.model.transformer import Transformer
    torch.manual_seed(3)
    m = Transformer(dim=64, attention_heads=4, linear_units=96, num_blocks=2, attention_dropout_rate=0.0, selfattention_layer_type="packed",
                    packed=dict(rotary={}, **packed)).to(DEV).eval()
    with torch.no_grad():
        for p in m.parameters():
            if p.dim() == 1:
                p.add_(torch.randn_like(p) * 0.1)
    return m


@gpu
@pytest.mark.parametrize("mode,tol", [("f32", 1e-3), ("bf16", 3e-2)])
@pytest.mark.parametrize("packed", [dict(), dict(softcap=5.0, shared_heads=2, causal=True), dict(distance_slopes=True, shared_heads=1)])
def test_transformer_padded_and_packed_utterances(mode, tol, packed):
    """a padded batch, the same utterances packed, and each alone in 64 bits; gradients of the packed call (f32 mode) against autograd in 64 bits"""
    from optispeech_amd import precision
    from optispeech_amd.packed_ops import PackedRows
    precision.set_precision(mode)
    try:
        m = make_transformer(**packed)
        lens, T = [37, 1, 150, 64], 150
        x = torch.randn(4, T, 64, generator=torch.Generator().manual_seed(1))
        pad = torch.arange(T)[None] >= torch.tensor(lens)[:, None]
        P = {k: v.detach().double().cpu().requires_grad_() for k, v in m.state_dict().items()}
        want = torch.cat([transformer_ref(P, x[b, :n].double(), m) for b, n in enumerate(lens)])
        y = m(x.to(DEV), pad.to(DEV))
        got = torch.cat([y[b, :n] for b, n in enumerate(lens)])
        assert relerr(got, want) < tol
        table = torch.cat([x[b, :n] for b, n in enumerate(lens)] + [torch.full((3, 64), 7.0)]).to(DEV)
        off = torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int64, device=DEV)
        rows = PackedRows.from_offsets(off, table.shape[0], longest=T)
        z = m.forward_packed(table, rows)
        assert relerr(z[:sum(lens)], want) < tol
        if mode == "f32":
            g = torch.randn(sum(lens), 64, generator=torch.Generator().manual_seed(2))
            (want * g.double()).sum().backward()
            (z[:sum(lens)] * g.to(DEV)).sum().backward()
            for k, p in m.named_parameters():
                w = P[k].grad.view(p.grad.shape) if k in P else None
                # linear_k.bias has a mathematically zero gradient without rotation or caps: an absolute floor for round-off
                err = (p.grad.double().cpu() - w).abs().max().item()
                assert err <= 2e-3 * w.abs().max().item() + 5e-6, (k, err)
    finally:
        precision.set_precision("f32")


@gpu
@pytest.mark.parametrize("mode,tol", [("f32", 1e-3), ("bf16", 3e-2)])
@pytest.mark.parametrize("chunks", [[1] * 9, [5, 1, 3], [40, 1, 1, 20]])
def test_transformer_stream_equals_the_causal_forward(mode, tol, chunks):
    """frames arriving one by one, a few at a time, and behind a long first piece: the same outputs as the causal forward over everything"""
    from optispeech_amd import precision
    precision.set_precision(mode)
    try:
        m = make_transformer(causal=True, softcap=8.0, shared_heads=2)
        T = sum(chunks)
        x = torch.randn(3, T, 64, generator=torch.Generator().manual_seed(5)).to(DEV)
        with torch.no_grad():
            want = m(x, torch.zeros(3, T, dtype=torch.bool, device=DEV))
        cache = m.start_stream(3, T)
        out, at = [], 0
        for n in chunks:
            out.append(m.stream(x[:, at:at + n], cache))
            at += n
        assert relerr(torch.cat(out, 1), want) < tol
        from optispeech_amd._lib import OspError
        with pytest.raises(OspError, match="cache"):
            m.stream(x[:, :1], cache)
    finally:
        precision.set_precision("f32")


def conformer_ref(P, x, m):
    """one utterance (n, C), float64"""
    def ff(z, name):
        return _lin(P, _lin(P, z, name + ".w_1").clamp_min(0), name + ".w_2")
    x = x * 8.0                                                    # sqrt(64)
    for i, layer in enumerate(m.conformer.encoders):
        pre = f"conformer.encoders.{i}."
        x = x + 0.5 * ff(_ln(P, x, pre + "norm_ff_macaron"), pre + "feed_forward_macaron")
        x = x + _attend(P, _ln(P, x, pre + "norm_mha"), pre + "self_attn", layer.self_attn)
        u = _lin(P, _ln(P, x, pre + "norm_conv"), pre + "conv_module.pointwise_conv1")
        u = u[:, :64] * torch.sigmoid(u[:, 64:])
        w = P[pre + "conv_module.depthwise_conv.weight"]
        u = torch.nn.functional.conv1d(u.T[None], w, P[pre + "conv_module.depthwise_conv.bias"], padding=w.shape[-1] // 2, groups=64)[0].T
        u = ref.group_norm(u, P[pre + "conv_module.norm.weight"], P[pre + "conv_module.norm.bias"], [slice(0, u.shape[0])], layer.conv_module.norm_groups,
                           1e-5, "silu")
        x = x + _lin(P, u, pre + "conv_module.pointwise_conv2")
        x = x + 0.5 * ff(_ln(P, x, pre + "norm_ff"), pre + "feed_forward")
        x = _ln(P, x, pre + "norm_final")
    return _ln(P, x, "conformer.after_norm")


@gpu
@pytest.mark.parametrize("mode,tol", [("f32", 1e-3), ("bf16", 3e-2)])
def test_conformer_utterances_do_not_see_their_padding(mode, tol):
    """rotary attention and group norm: every utterance of a padded batch equals the 64-bit result of the utterance alone, whatever the padding holds;
    gradients (f32 mode) against autograd in 64 bits"""
    from optispeech_amd import precision
    from optispeech_amd.model.conformer import Conformer
    precision.set_precision(mode)
    try:
        torch.manual_seed(4)
        m = Conformer(dim=64, attention_heads=2, linear_units=96, num_blocks=2, attention_dropout_rate=0.0, selfattention_layer_type="packed",
                      packed=dict(softcap=20.0), cnn_module_norm_groups=4, cnn_module_kernel=7).to(DEV).eval()
        lens, T = [90, 3, 41], 90
        x = torch.randn(3, T, 64, generator=torch.Generator().manual_seed(6))
        pad = torch.arange(T)[None] >= torch.tensor(lens)[:, None]
        x[pad] = 50.0
        P = {k: v.detach().double().cpu().requires_grad_() for k, v in m.state_dict().items()}
        want = torch.cat([conformer_ref(P, x[b, :n].double(), m) for b, n in enumerate(lens)])
        y = m(x.to(DEV), pad.to(DEV))
        got = torch.cat([y[b, :n] for b, n in enumerate(lens)])
        assert relerr(got, want) < tol
        if mode == "f32":
            g = torch.randn(sum(lens), 64, generator=torch.Generator().manual_seed(7))
            (want * g.double()).sum().backward()
            (got * g.to(DEV)).sum().backward()
            sd = {k: p.grad for k, p in m.named_parameters()}
            for k, p in P.items():
                if k not in sd or p.grad is None:
                    continue
                a, w = sd[k].double().cpu(), p.grad
                if a.shape != w.shape:                             # native layouts: (taps, C) and (Cout, 1, Cin)
                    a = a.T[:, None, :] if "depthwise" in k else a.permute(0, 2, 1)
                err = (a - w).abs().max().item()
                assert err <= 2e-3 * w.abs().max().item() + 1e-5, (k, err, w.abs().max().item())
    finally:
        precision.set_precision("f32")


@gpu
@pytest.mark.parametrize("mode", ["f32", "bf16"])
def test_padding_may_hold_nan(mode):
    """valid frames do not depend on what the padding holds, NaN included"""
    from optispeech_amd import precision
    from optispeech_amd.model.conformer import Conformer
    precision.set_precision(mode)
    try:
        torch.manual_seed(4)
        conformer = Conformer(dim=64, attention_heads=2, linear_units=96, num_blocks=2, attention_dropout_rate=0.0, selfattention_layer_type="packed",
                              cnn_module_norm_groups=4).to(DEV).eval()
        lens, T = [33, 1, 20], 33
        x = torch.randn(3, T, 64, generator=torch.Generator().manual_seed(6)).to(DEV)
        pad = (torch.arange(T)[None] >= torch.tensor(lens)[:, None]).to(DEV)
        for m in (conformer, make_transformer(causal=True)):
            got = []
            for fill in (0.0, float("nan")):
                x[pad] = fill
                with torch.no_grad():
                    got.append(m(x, pad)[~pad])
            assert torch.isfinite(got[0]).all() and torch.equal(got[0], got[1])
    finally:
        precision.set_precision("f32")


@gpu
@pytest.mark.parametrize("backbone", ["transformer", "conformer"])
@pytest.mark.parametrize("mode", ["bf16", "f32"])
def test_training_step_with_the_packed_attention(backbone, mode):
    """the options through ModelConfig: two GAN steps, finite losses, gradients reach the attention and the norm"""
    from optispeech_amd import precision, rng
    from optispeech_amd.config import ModelConfig, make_optispeech, synthetic_batch
    precision.set_precision(mode)
    try:
        torch.manual_seed(2)
        rng.manual_seed(2, 0)
        cfg = ModelConfig(backbone=backbone, packed_attention=dict(rotary={}, softcap=30.0, distance_slopes=True))
        m = make_optispeech(cfg, batch_size=2, pretraining_steps=0).to(DEV).train()
        batch = synthetic_batch(2, 24, 96, cfg, seed=5, ragged=True, device=DEV)
        m.optimizers()
        for step in range(2):
            m.training_step(batch, step)
        logs = m.fetch_logs()
        assert all(np.isfinite(v) for v in logs.values()), logs
        layer = getattr(m.generator.encoder, backbone).encoders[0]
        checked = [layer.self_attn.linear_q.weight, layer.self_attn.linear_k.weight]
        if backbone == "conformer":
            checked += [layer.conv_module.norm.weight, layer.conv_module.norm.bias]
        for p in checked:
            assert p.grad is not None and torch.isfinite(p.grad).all() and p.grad.abs().sum().item() > 0
    finally:
        precision.set_precision("f32")


# ------------------------------------------------------------------------------------------------------------------ refusals (no GPU work)
def test_refusals():
    from optispeech_amd.model.conformer import Conformer
    from optispeech_amd.model.packed import FrameCache
    from optispeech_amd.model.transformer import Transformer
    from optispeech_amd._lib import OspError
    with pytest.raises(AssertionError, match="packed"):
        Transformer(dim=64, packed=dict(causal=True))
    with pytest.raises(AssertionError, match="dropout"):
        Transformer(dim=64, selfattention_layer_type="packed")
    with pytest.raises(AssertionError, match="dropout"):
        Conformer(dim=64, selfattention_layer_type="packed")
    m = Transformer(dim=64, attention_dropout_rate=0.0, selfattention_layer_type="packed", packed=dict(rotary={}))
    with pytest.raises(AssertionError, match="causal"):
        m.start_stream(1, 4)
    with pytest.raises(AssertionError, match="rotary"):
        Transformer(dim=64, attention_dropout_rate=0.0, selfattention_layer_type="packed").forward_packed(torch.zeros(4, 64), None)
    cache = FrameCache(1, 2, 4, 1, 8, "cpu", torch.float32)
    with pytest.raises(OspError, match="cache"):
        cache.begin(5)


def test_stream_refusals(monkeypatch):
    """steps of no frames, and steps inside a capture, whose replays would not be counted"""
    from optispeech_amd.model.packed import FrameCache
    from optispeech_amd._lib import OspError
    cache = FrameCache(1, 2, 4, 1, 8, "cpu", torch.float32)
    with pytest.raises(OspError, match="0 new frames"):
        cache.begin(0)
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(OspError, match="captured"):
        cache.begin(1)
    assert cache.used == 0
