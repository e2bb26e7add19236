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
