"""``dr.dropout`` against the restated generator on the CPU: masks exactly, values within one
rounding (the kernel multiplies by the float32 scale and adds the residual in float32: two
roundings of 2^-24, then one of the type, half a unit in its last place)."""

import pytest
import torch

import diffrast_b200 as dr
from feature_reference import U, keep_mask, keep_scale

pytestmark = pytest.mark.gpu
CUDA = "cuda"
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def rounding(dtype):
    return 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2


def check(got, want, dtype, magnitude):
    """|got - want| within the type's rounding of want plus 3 float32 roundings of the terms; a
    float16 below its normal range is rounded to a multiple of 2^-24, half of it off."""
    bound = rounding(dtype) * want.abs() * (1 + 4 * U) + 3 * U * magnitude + 2.0**-25
    assert (got.double().cpu() - want).abs().le(bound).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("count", [1, 7, 8, 9, 2047, 2049, 5003])
@pytest.mark.parametrize("residual", [False, True])
def test_matches_the_restated_mask(dtype, count, residual):
    gen = torch.Generator().manual_seed(count)
    x = torch.randn(count, generator=gen).to(dtype)
    r = torch.randn(count, generator=gen).to(dtype) if residual else None
    g = torch.randn(count, generator=gen).to(dtype)
    seed, layer, p = 0x123456789ABCDEF, 7, 0.3
    keep = keep_mask(count, p, seed, layer)
    xd = x.to(CUDA).requires_grad_(True)
    rd = r.to(CUDA).requires_grad_(True) if residual else None
    y = dr.dropout(xd, p, seed, layer=layer, residual=rd)
    assert y.dtype == dtype
    kept = torch.where(keep, x.double() * keep_scale(p), 0.0)
    want = kept + r.double() if residual else kept
    check(y.detach(), want, dtype, kept.abs() + (r.double().abs() if residual else 0))
    if not residual:
        assert torch.equal(y.detach().cpu() != 0, keep & (x != 0))
    grads = torch.autograd.grad(y, [xd] + ([rd] if residual else []), g.to(CUDA))
    dx = torch.where(keep, g.double() * keep_scale(p), 0.0)
    check(grads[0], dx, dtype, dx.abs())
    if residual:
        assert torch.equal(grads[1].cpu(), g)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("offset", [1, 2, 3, 4])
def test_unaligned_and_strided_inputs(dtype, offset):
    """A storage offset that breaks 16-byte alignment, and a transposed input, give the same
    values as an aligned copy."""
    base = torch.randn(4104, device=CUDA).to(dtype)
    x = base[offset:offset + 4001]
    r = base[4:4005]
    assert torch.equal(dr.dropout(x, 0.5, 3), dr.dropout(x.clone(), 0.5, 3))
    assert torch.equal(dr.dropout(x, 0.5, 3, residual=r),
                       dr.dropout(x.clone(), 0.5, 3, residual=r.clone()))
    t = base[:4096].view(64, 64).t()
    assert torch.equal(dr.dropout(t, 0.5, 3), dr.dropout(t.contiguous(), 0.5, 3))


def test_dropped_values_are_zero_whatever_they_are():
    x = torch.tensor([float("nan"), float("inf"), -float("inf"), 1.0] * 64, device=CUDA)
    keep = keep_mask(256, 0.5, 11)
    y = dr.dropout(x, 0.5, 11).cpu()
    assert (y[~keep] == 0).all()
    kept = y[keep]
    torch.testing.assert_close(kept, 2 * x.cpu()[keep], rtol=0, atol=0, equal_nan=True)


def test_probabilities_at_the_ends():
    x = torch.randn(1001, device=CUDA, dtype=torch.float16)
    for p in (0.0, 2.0**-18):  # rounds to nothing dropped
        assert torch.equal(dr.dropout(x, p, 5), x)
    y = dr.dropout(torch.ones(1 << 16, device=CUDA), 1 - 2.0**-20, 5)
    assert set(y.unique().tolist()) <= {0.0, 65536.0} and (y == 0).sum() > 65000


def test_seed_tensor_layers_and_rate():
    x = torch.ones(1 << 20, device=CUDA)
    seed = torch.tensor([42], device=CUDA)
    a = dr.dropout(x, 0.25, 42)
    assert torch.equal(a, dr.dropout(x, 0.25, seed)) and torch.equal(a, dr.dropout(x, 0.25, seed[0]))
    others = [dr.dropout(x, 0.25, 43), dr.dropout(x, 0.25, 42, layer=1),
              dr.dropout(x, 0.25, 42 + (1 << 40))]
    # A share of kept elements is within 6 standard deviations, sqrt(p (1 - p) / n) = 4.2e-4; two
    # independent masks agree in 1 - 2 p (1 - p) = 0.625 of the elements, within 6 * 4.8e-4.
    for y in [a, *others]:
        assert abs(float((y != 0).float().mean()) - 0.75) < 2.6e-3
    for y in others:
        assert abs(float(((y != 0) == (a != 0)).float().mean()) - 0.625) < 2.9e-3
    negative = torch.tensor([-5], device=CUDA)
    keep = keep_mask(64, 0.5, -5)
    assert torch.equal(dr.dropout(x[:64], 0.5, negative).cpu() != 0, keep)


def test_element_indices_pass_32_bits():
    """The last elements of a tensor of 2^32 + 24 elements take counters above 2^29 - 1, and their
    addresses pass 4 G elements."""
    count = (1 << 32) + 24
    x = torch.ones(count, device=CUDA, dtype=torch.float16)
    y = dr.dropout(x, 0.5, 9)
    tail = 64
    assert torch.equal(y[-tail:].cpu() != 0, keep_mask(tail, 0.5, 9, first=count - tail))
    assert torch.equal(y[:tail].cpu() != 0, keep_mask(tail, 0.5, 9))
    del x, y
    torch.cuda.empty_cache()


def test_changed_seed_is_reported_and_empty_inputs_pass():
    x = torch.ones(16, device=CUDA, requires_grad=True)
    seed = torch.tensor([1], device=CUDA)
    y = dr.dropout(x, 0.5, seed)
    seed += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    e = torch.zeros(0, 4, device=CUDA, requires_grad=True)
    out = dr.dropout(e, 0.5, 1)
    out.sum().backward()
    assert out.shape == (0, 4) and e.grad.shape == (0, 4)
    s = dr.dropout(torch.tensor(3.0, device=CUDA), 0.5, 1)
    assert s.shape == () and s.item() in (0.0, 6.0)


def test_second_order_is_refused():
    x = torch.ones(16, device=CUDA, requires_grad=True)
    y = dr.dropout(x, 0.5, 1)
    with pytest.raises(RuntimeError, match="no second-order gradients"):
        torch.autograd.grad(y.sum(), x, create_graph=True)


def test_other_stream_and_captured_replays_with_new_seeds():
    x = torch.randn(10007, device=CUDA)
    seed = torch.tensor([1], device=CUDA)
    want = [dr.dropout(x, 0.3, s) for s in (1, 2, 3)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(dr.dropout(x, 0.3, seed), want[0])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = dr.dropout(x, 0.3, seed)
        seed += 1
    seed.fill_(1)
    for w in want:
        graph.replay()
        assert torch.equal(y, w)
