"""``dr.group_norm`` against a plain restatement in 64 bits (``feature_reference``), forward and
backward.

Bounds, with u = 2^-24 and everything per group, in units that the reference supplies:

- a mean is off by at most 64 u max|x| and a reciprocal standard deviation by 512 u relative: a
  thread sums at most 256 values about one of them, which multiplies rounding by at most their
  number, and the joins add a few dozen roundings; so h = (x - m) r is off by
  e_h = u (64 r max|x| + 520 max|h|), and z = h w + b by |w| e_h + 2 u (|z| + |b|);
- activations have slopes of at most 1.1 and their own error of 8 u |z|; silu's derivative has a
  slope of at most 0.5 and its own error of 16 u;
- a sum of n terms t in float32 (at most 256 in a row, then trees of at most 64 levels) is off by
  320 u sum|t|, plus the sum of the terms' own errors;
- the result is rounded once: half a unit in the last place of its type.
"""

import concurrent.futures

import pytest
import torch

import diffrast_b200 as dr
import feature_reference as ref
from feature_reference import U

pytestmark = pytest.mark.gpu
CUDA = "cuda"
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def features(shape, dtype, seed, offset=0.5):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=gen) * (torch.rand(shape[-1], generator=gen) + 0.5)
    x = x + offset * torch.randn(shape[0], *([1] * (len(shape) - 2)), shape[-1], generator=gen)
    x.view(-1, shape[-1])[:: 5] = 0.0  # background pixels
    return x.to(dtype)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half the spacing of a type's subnormal numbers."""
    return {torch.float32: 2.0**-150, torch.float16: 2.0**-25, torch.bfloat16: 2.0**-134}[dtype]


class Bounds:
    """The errors allowed for one case (see the top of the file), from 64-bit values."""

    def __init__(self, x, groups, weight, bias, eps, activation, factor, grad):
        batch, channels = x.shape[0], x.shape[-1]
        v = x.double().reshape(batch, -1, groups, channels // groups)
        d = v - v.mean((1, 3), keepdim=True)
        r = (d.square().mean((1, 3), keepdim=True) + eps).rsqrt()
        h = d * r
        e_h = U * (64 * r * v.abs().amax((1, 3), keepdim=True) + 520 * h.abs().amax((1, 3), keepdim=True))
        e_h = e_h.expand_as(h).reshape(batch, -1, channels)
        h, rc = h.reshape(batch, -1, channels), r.expand_as(d).reshape(batch, -1, channels)
        one = torch.ones(1, 1, channels, dtype=torch.float64)
        w = one if weight is None else weight.double().reshape(-1, 1, channels)
        b = 0 * one if bias is None else bias.double().reshape(-1, 1, channels)
        z = h * w + b
        e_z = w.abs() * e_h + 2 * U * (z.abs() + b.abs())
        f = torch.ones_like(z) if factor is None else factor.double().reshape(z.shape)
        self.y = (f * (1.1 * e_z + 8 * U * z.abs())).reshape(x.shape)
        if grad is None:
            return
        zz = z.clone().requires_grad_(True)
        slope = torch.autograd.grad(ref.activate(zz, activation).sum(), zz)[0]
        q = grad.double().reshape(z.shape) * f
        e_s = (0.5 * e_z + 16 * U) if activation == "silu" else 0 * e_z
        t, e_t = q * slope, q.abs() * e_s + 4 * U * (q * slope).abs()
        self.bias = 320 * U * t.abs().sum(1) + e_t.sum(1)
        self.weight = 320 * U * (t * h).abs().sum(1) + (e_t * h.abs() + t.abs() * e_h).sum(1)
        count = v.shape[1] * v.shape[3]

        def mean(per_channel):  # of a sum per view and channel, over each group, per channel
            g = per_channel.reshape(batch, groups, -1).sum(2, keepdim=True) / count
            return g.expand(batch, groups, channels // groups).reshape(batch, 1, channels)

        a, bb = mean((t * w).sum(1)), mean((t * h * w).sum(1))
        e_a, e_b = mean(w.abs()[:, 0] * self.bias), mean(w.abs()[:, 0] * self.weight)
        terms = (t * w).abs() + a.abs() + (h * bb).abs()
        self.x = (rc * (w.abs() * e_t + e_a + h.abs() * e_b + e_h * bb.abs() + 600 * U * terms)).reshape(x.shape)


def within(got, want, bound, dtype):
    limit = bound * (1 + half_step(dtype)) + half_step(dtype) * want.abs() + tiny(dtype)
    off = (got.detach().double().cpu() - want).abs()
    assert got.dtype == dtype and off.shape == want.shape
    assert off.le(limit).all(), f"{(off / limit).max().item():.3g} of the bound"


def compare(x, groups, weight=None, bias=None, eps=1e-5, activation="none", dropout=0.0, seed=None,
            layer=0, grad=None, on_gpu=None):
    """Run and check forward and backward; ``on_gpu`` maps a CPU tensor to the CUDA input."""
    on_gpu = on_gpu or (lambda t: t.to(CUDA))
    factor = None
    if dropout:
        factor = ref.keep_mask(x.numel(), dropout, seed, layer).view(x.shape) * ref.keep_scale(dropout)
    if grad is None:
        grad = torch.randn(x.shape, generator=torch.Generator().manual_seed(99)).to(x.dtype)
    leaves = [t.detach().clone().requires_grad_(True) for t in (x, weight, bias) if t is not None]
    it = iter(leaves)
    lx, lw, lb = (next(it) if t is not None else None for t in (x, weight, bias))
    want = ref.group_norm(lx, groups, lw, lb, eps, activation, factor)
    want_grads = torch.autograd.grad(want, leaves, grad.double())
    gx = on_gpu(x).detach().requires_grad_(True)
    gw, gb = (None if t is None else t.to(CUDA).requires_grad_(True) for t in (weight, bias))
    y = dr.group_norm(gx, groups, gw, gb, eps=eps, activation=activation, dropout=dropout, seed=seed,
                      layer=layer)
    grads = torch.autograd.grad(y, [t for t in (gx, gw, gb) if t is not None], on_gpu(grad))
    bounds = Bounds(x, groups, weight, bias, eps, activation, factor, grad)
    assert y.is_contiguous() and y.shape == x.shape
    within(y, want.detach(), bounds.y, x.dtype)
    # The reference's leaves are of the inputs' types, so its gradients come rounded to them.
    exact = [g.double() for g in want_grads]
    within(grads[0], exact[0], bounds.x + half_step(x.dtype) * exact[0].abs(), x.dtype)
    for t, g, e, b in zip([t for t in (weight, bias) if t is not None], grads[1:], exact[1:],
                          [b for b, t in ((bounds.weight, weight), (bounds.bias, bias)) if t is not None]):
        b = b if t.ndim == 2 else b.sum(0) + 32 * U * e.abs()
        within(g, e, b.reshape(e.shape) + half_step(t.dtype) * e.abs(), t.dtype)
    return y, grads


def params(channels, seed, batch=None, dtype=torch.float32):
    gen = torch.Generator().manual_seed(seed)
    shape = (channels,) if batch is None else (batch, channels)
    return ((1 + 0.3 * torch.randn(shape, generator=gen)).to(dtype),
            (0.3 * torch.randn(shape, generator=gen)).to(dtype))


SHAPES = [
    ((1, 1, 1, 2), 1), ((1, 1, 1, 8), 2), ((2, 1, 3, 5), 1), ((1, 16, 16, 64), 16), ((3, 7, 9, 30), 5),
    ((2, 13, 17, 7), 1), ((2, 8, 8, 12), 3), ((4, 3, 600), 2), ((1, 3, 3, 2100), 1),
    ((2, 4, 4, 4096), 2), ((1, 5, 5, 4098), 2), ((1, 33, 65, 257), 257), ((700, 3, 8), 2), ((2, 24, 24, 48), 6),
    ((1, 300, 300, 1), 1), ((1, 60000, 3), 1), ((2, 96, 96, 32), 32), ((2, 40, 40, 64), 2), ((5, 24), 4),
    ((2, 31, 20, 9), 3), ((1, 120, 121, 20), 10),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape, groups", SHAPES)
def test_matches_64_bits(shape, groups, dtype):
    w, b = params(shape[-1], 3)
    compare(features(shape, dtype, 1), groups, w, b, activation="silu")


# Above one megabyte images are taken in two passes: whole vectors, folded pixels, rows that start
# anywhere, groups wider than 32 channels, more views than processors.
LARGE = [
    ((2, 90, 100, 64), 32), ((1, 300, 400, 5), 5), ((3, 97, 101, 30), 5), ((2, 301, 303, 7), 1),
    ((2, 63, 65, 100), 5), ((1, 61, 47, 512), 2), ((2, 40, 41, 520), 1), ((5, 75, 75, 33), 33),
    ((150, 33, 37, 4), 1), ((2, 33, 35, 260), 4), ((1, 3, 3, 60000), 3),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape, groups", LARGE)
def test_two_passes_match_64_bits(shape, groups, dtype):
    w, b = params(shape[-1], 60)
    compare(features(shape, dtype, 61), groups, w, b, activation="silu")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape, groups", [((2, 90, 100, 64), 8), ((3, 97, 101, 30), 5), ((2, 301, 303, 7), 1)])
def test_two_passes_with_dropout_and_parameters_of_each_view(shape, groups, dtype):
    w, b = params(shape[-1], 62, batch=shape[0])
    compare(features(shape, dtype, 63), groups, w, b, activation="silu", dropout=0.2, seed=9, layer=1)
    compare(features(shape, dtype, 64), groups)


@pytest.mark.parametrize("shape, groups, dropout", [
    ((70001, 5, 6), 2, 0.0), ((131077, 7, 7), 1, 0.3), ((66000, 1, 8), 2, 0.3), ((66000, 1, 258), 1, 0.3),
    ((300, 32, 32, 32), 4, 0.0), ((90, 40, 50, 64), 2, 0.3), ((1000, 4, 4, 256), 32, 0.0)])
def test_many_views(shape, groups, dropout):
    """A launch takes 65535 views (of 258 channels in one group, too wide for clusters of blocks);
    gradients of shared parameters are sums over all views."""
    x = features(shape, torch.float16, 5)
    compare(x, groups, *params(shape[-1], 6), activation="silu", dropout=dropout, seed=4)


@pytest.mark.parametrize("dtype, pixels, channels, copies, groups, views, long", [
    (torch.float16, 1 << 16, 64, 1025, 8, True, 1), (torch.bfloat16, 100003, 33, 1310, 11, False, 70)])
def test_element_indices_pass_32_bits(dtype, pixels, channels, copies, groups, views, long):
    """Copies of one image, as views or as the pixels of one view, have the image's statistics and
    gradients. In the long view a thread of the join takes 1030 chunks in a row, each with up to
    four roundings: 64 u + 4 * 1030 u are at most 70 times the 64 u and more of the bounds."""
    image = features((1, pixels, channels), dtype, 8)
    grad = torch.randn(1, pixels, channels, generator=torch.Generator().manual_seed(9)).to(dtype)
    weight, bias = params(channels, 10)
    shape = (copies, pixels, channels) if views else (1, copies * pixels, channels)
    x, dy = (t.to(CUDA).expand(copies, -1, -1).reshape(shape) for t in (image, grad))
    x.requires_grad_(True)
    y = dr.group_norm(x, groups, weight.to(CUDA), bias.to(CUDA), activation="silu")
    grad_x, = torch.autograd.grad(y, x, dy)
    leaf = image.double().requires_grad_(True)
    want = ref.group_norm(leaf, groups, weight, bias, activation="silu")
    want_x, = torch.autograd.grad(want, leaf, grad.double())
    bounds = Bounds(image, groups, weight, bias, 1e-5, "silu", None, grad)
    for at in (0, copies - 1):
        part = slice(at, at + 1)
        within(y.view(copies, pixels, channels)[part], want.detach(), long * bounds.y, dtype)
        within(grad_x.view(copies, pixels, channels)[part], want_x, long * bounds.x, dtype)
    del x, dy, y, grad_x
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("extra", [1, 2, 4, 8])
def test_two_passes_over_channel_slices(extra, dtype):
    shape = (2, 120, 130, 32)

    def in_wide(t):
        wide = torch.full((*shape[:-1], 32 + extra), float("nan"), dtype=t.dtype, device=CUDA)
        wide[..., extra:] = t.to(CUDA)
        return wide[..., extra:]

    compare(features(shape, dtype, 65), 4, *params(32, 66), activation="silu", on_gpu=in_wide)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("activation", ["none", "relu", "silu"])
@pytest.mark.parametrize("shape, groups", [((2, 9, 11, 24), 4), ((2, 10, 12, 6), 2), ((1, 7, 5, 3), 1)])
def test_activations_and_dropout(shape, groups, activation, dtype):
    x = features(shape, dtype, 2)
    w, b = params(shape[-1], 4)
    if activation == "relu":
        # No z so near zero that rounding could choose the other slope.
        z = ref.group_norm(x, groups, w, b)
        assert z.abs().min() > 1e-5
    compare(x, groups, w, b, activation=activation, dropout=0.3, seed=77, layer=3)


@pytest.mark.parametrize("which", ["none", "weight", "bias", "views", "mixed", "type", "views type"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_weight_and_bias_forms(which, dtype):
    shape = (3, 12, 10, 24)
    x = features(shape, dtype, 5)
    w, b = params(24, 6)
    wv, bv = params(24, 7, batch=3)
    forms = {"none": (None, None), "weight": (w, None), "bias": (None, b), "views": (wv, bv),
             "mixed": (w, bv), "type": (w.to(dtype), b.to(dtype)),
             "views type": (wv.to(dtype), bv.to(dtype))}
    compare(x, 6, *forms[which], activation="silu")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("first, extra", [(0, 8), (8, 8), (2, 4), (1, 1), (3, 5)])
def test_channel_slices_are_read_in_place(first, extra, dtype):
    """Slices at aligned and odd channels: the same values as of a copy, within the bounds."""
    shape = (2, 11, 13, 16)

    def in_wide(t):
        wide = torch.full((*t.shape[:-1], t.shape[-1] + extra), float("nan"), dtype=t.dtype, device=CUDA)
        wide[..., min(first, extra):min(first, extra) + 16] = t.to(CUDA)
        return wide[..., min(first, extra):min(first, extra) + 16]

    w, b = params(16, 8)
    compare(features(shape, dtype, 9), 4, w, b, activation="silu", on_gpu=in_wide)


@pytest.mark.parametrize("dtype", TYPES)
def test_unaligned_storage_and_expanded_gradients(dtype):
    shape = (2, 8, 8, 16)

    def shifted(t):
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=CUDA)
        flat[1:] = t.reshape(-1).to(CUDA)
        return flat[1:].view(t.shape)

    x = features(shape, dtype, 10)
    compare(x, 4, *params(16, 11), on_gpu=shifted)
    xg = x.to(CUDA).requires_grad_(True)
    g1 = torch.autograd.grad(dr.group_norm(xg, 4, activation="silu").sum(), xg)[0]
    g2 = torch.autograd.grad(dr.group_norm(xg, 4, activation="silu"), xg, torch.ones_like(xg))[0]
    assert torch.equal(g1, g2)
    perm = x.to(CUDA).permute(0, 3, 1, 2).contiguous().permute(0, 2, 3, 1)  # planar storage
    assert torch.equal(dr.group_norm(perm, 4), dr.group_norm(x.to(CUDA), 4))


def test_offset_far_above_the_spread():
    """float32 data around 1000 with a spread of 0.1: deviations from the mean keep their digits.
    With whole numbers / 1024 the inputs are exact; the bounds carry the offset's share of the
    mean's error, and one far background pixel does not spoil the rest."""
    gen = torch.Generator().manual_seed(12)
    x = 1000 + torch.randint(-200, 200, (2, 40, 40, 16), generator=gen) / 1024.0
    compare(x, 2, *params(16, 13), activation="silu")
    x[:, 0, 0] = 0.0
    compare(x, 2, *params(16, 13), activation="silu")
    x = 1000 + torch.randint(-200, 200, (1, 150, 151, 16), generator=gen) / 1024.0
    x[:, 0, 0] = 0.0
    compare(x, 2, *params(16, 13), activation="silu")


def test_constant_groups_and_large_values():
    x = torch.full((2, 6, 6, 8), 3.0)
    x[1] = -7.25
    w, b = params(8, 14)
    y, grads = compare(x, 2, w, b)
    assert torch.equal(y.detach().cpu(), b.expand(2, 6, 6, 8))
    compare(features((1, 9, 9, 8), torch.float32, 15) * 1e15, 2, w, b, eps=0.0)
    compare(features((1, 9, 9, 8), torch.float32, 15) * 1e-12, 2, w, b, eps=0.0)


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape, groups", [((2, 8, 8, 16), 4), ((2, 80, 80, 12), 3), ((2, 203, 207, 12), 3)])
def test_non_finite_values_stay_in_their_group(value, dtype, shape, groups):
    x = features(shape, dtype, 16).to(CUDA)
    w, b = (t.to(CUDA) for t in params(shape[-1], 17))
    clean = dr.group_norm(x, groups, w, b, activation="silu")
    d = shape[-1] // groups
    x[1, 3, 4, d] = value  # view 1, group 1
    bad = x.clone().requires_grad_(True)
    y = dr.group_norm(bad, groups, w, b, activation="silu")
    hit = torch.zeros(shape, dtype=torch.bool, device=CUDA)
    hit[1, :, :, d:2 * d] = True
    assert y[hit].isnan().all() and torch.equal(y[~hit], clean[~hit])
    g = torch.autograd.grad(y, bad, torch.ones_like(y))[0]
    assert g[hit].isnan().all() and g[~hit].isfinite().all()


def test_fused_dropout_is_dropout_of_the_result():
    x = features((2, 20, 20, 24), torch.float32, 18).to(CUDA)
    seed = torch.tensor([5], device=CUDA)
    plain = dr.group_norm(x, 3, activation="silu")
    fused = dr.group_norm(x, 3, activation="silu", dropout=0.4, seed=seed, layer=2)
    torch.testing.assert_close(fused, dr.dropout(plain, 0.4, 5, layer=2), rtol=2 * U, atol=0)


def test_gradients_against_differences():
    """Central differences of the 64-bit form in random directions, against the kernel's gradients:
    for step s the difference is off by s^2 / 6 times the third derivative, far below the bound of
    1e-3 of the gradient's size at s = 1e-4."""
    x = features((2, 6, 5, 12), torch.float32, 19)
    w, b = params(12, 20, batch=2)
    gen = torch.Generator().manual_seed(21)
    g = torch.randn(x.shape, generator=gen)
    leaves = [t.to(CUDA).requires_grad_(True) for t in (x, w, b)]
    y = dr.group_norm(leaves[0], 3, leaves[1], leaves[2], activation="silu", dropout=0.2, seed=3)
    grads = torch.autograd.grad(y, leaves, g.to(CUDA))
    factor = ref.keep_mask(x.numel(), 0.2, 3).view(x.shape) * ref.keep_scale(0.2)

    def loss(tensors):
        return (ref.group_norm(tensors[0], 3, tensors[1], tensors[2], activation="silu",
                               factor=factor) * g).sum()

    for k in range(3):
        direction = torch.randn(leaves[k].shape, generator=gen).double()
        ends = []
        for sign in (1, -1):
            moved = [t.double() for t in (x, w, b)]
            moved[k] = moved[k] + sign * 1e-4 * direction
            ends.append(loss(moved))
        slope = float(ends[0] - ends[1]) / 2e-4
        got = float((grads[k].double().cpu() * direction).sum())
        assert abs(got - slope) < 1e-3 * float(grads[k].double().norm()) * float(direction.norm())


@pytest.mark.parametrize("shape", [(3, 20, 30, 40), (3, 100, 90, 40), (3, 101, 103, 42)])
def test_runs_agree_bit_for_bit(shape):
    x = features(shape, torch.bfloat16, 22).to(CUDA).requires_grad_(True)
    w, b = (t.to(CUDA).requires_grad_(True) for t in params(shape[-1], 23))

    def run():
        y = dr.group_norm(x, 2, w, b, activation="silu", dropout=0.1, seed=1)
        return [y, *torch.autograd.grad(y, (x, w, b), torch.ones_like(y))]

    first = run()
    for _ in range(3):
        assert all(torch.equal(p, q) for p, q in zip(run(), first))


@pytest.mark.parametrize("side", [9, 151])
def test_only_the_gradients_asked_for(side):
    x = features((2, side, side, 16), torch.float32, 24).to(CUDA)
    w, b = (t.to(CUDA) for t in params(16, 25))
    g = torch.randn_like(x)

    def grads(which):
        leaves = [t.clone().requires_grad_(k in which) for k, t in enumerate((x, w, b))]
        y = dr.group_norm(leaves[0], 4, leaves[1], leaves[2], activation="silu")
        return dict(zip(which, torch.autograd.grad(y, [leaves[k] for k in which], g)))

    full = grads((0, 1, 2))
    for which in ((0,), (1,), (2,), (0, 2), (1, 2)):
        got = grads(which)
        assert all(torch.equal(got[k], full[k]) for k in which)


def test_empty_images():
    w, b = (t.to(CUDA).requires_grad_(True) for t in params(8, 26))
    for shape in ((0, 4, 4, 8), (2, 0, 4, 8)):
        x = torch.zeros(shape, device=CUDA, requires_grad=True)
        y = dr.group_norm(x, 2, w, b, activation="silu")
        grads = torch.autograd.grad(y.sum(), (x, w, b))
        assert y.shape == shape and grads[0].shape == shape
        assert (grads[1] == 0).all() and (grads[2] == 0).all()


def test_second_order_is_refused():
    x = features((1, 4, 4, 8), torch.float32, 27).to(CUDA).requires_grad_(True)
    y = dr.group_norm(x, 2)
    with pytest.raises(RuntimeError, match="no second-order gradients"):
        torch.autograd.grad(y.sum(), x, create_graph=True)


def test_inference_tensors_pass_and_give_the_same():
    with torch.inference_mode():
        x = features((1, 8, 8, 16), torch.float32, 28).to(CUDA)
        y = dr.group_norm(x, 4, activation="silu")
    w = torch.ones(16, device=CUDA, requires_grad=True)
    torch.testing.assert_close(dr.group_norm(x, 4, w, activation="silu"), y, rtol=0, atol=0)
    dr.group_norm(x, 4, w, activation="silu").sum().backward()


def training_step(x, w, b, seed, g):
    y = dr.group_norm(x, 4, w, b, activation="silu", dropout=0.2, seed=seed)
    return [y.detach(), *torch.autograd.grad(y, (x, w, b), g)]


@pytest.mark.parametrize("dtype, width", [(torch.float32, 16), (torch.float32, 17), (torch.bfloat16, 32),
                                          (torch.bfloat16, 33)])
def test_views_at_the_size_where_the_passes_change(dtype, width):
    """Views of 256 KB and just above."""
    x = features((5, 64, width, 64), dtype, 31)
    compare(x, 8, *params(64, 32), activation="silu", dropout=0.2, seed=33)


def test_one_tensor_in_two_places():
    x = features((2, 9, 11, 16), torch.float32, 41)
    p = params(16, 42)[0]
    gx, gp = x.to(CUDA).requires_grad_(True), p.to(CUDA).requires_grad_(True)
    y = dr.group_norm(gx, 4, gp, gp, activation="relu")
    grads = torch.autograd.grad(y.square().sum(), (gx, gp))
    two = [p.to(CUDA).requires_grad_(True) for _ in range(2)]
    want = dr.group_norm(gx, 4, *two, activation="relu")
    apart = torch.autograd.grad(want.square().sum(), (gx, *two))
    assert torch.equal(y, want) and torch.equal(grads[0], apart[0])
    assert torch.equal(grads[1], apart[1] + apart[2])
    z = dr.dropout(gx, 0.5, 7, residual=gx)
    keep = ref.keep_mask(x.numel(), 0.5, 7).view(x.shape).to(CUDA)
    assert torch.equal(z, gx + 2 * gx * keep)
    assert torch.equal(torch.autograd.grad(z.sum(), gx)[0], 1 + 2.0 * keep)


def test_threads_with_streams_of_their_own():
    """Calls of four threads at once, in clusters and in passes, give what one thread gets."""
    inputs = [features(shape, torch.bfloat16, i).to(CUDA) for i, shape in
              enumerate([(2, 16, 16, 64), (2, 130, 100, 64), (3, 101, 103, 36), (40, 32, 32, 24)])]
    grads = [torch.randn_like(x) for x in inputs]

    def step(x, grad):
        leaf = x.clone().requires_grad_(True)
        y = dr.group_norm(leaf, 4, activation="silu", dropout=0.1, seed=5)
        return y.detach(), torch.autograd.grad(y, leaf, grad)[0]

    want = [step(x, g) for x, g in zip(inputs, grads)]
    torch.cuda.synchronize()

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            got = [step(inputs[i], grads[i]) for _ in range(10)]
        stream.synchronize()
        return all(torch.equal(a, b) for pair in got for a, b in zip(pair, want[i]))

    with concurrent.futures.ThreadPoolExecutor(4) as pool:
        assert all(pool.map(work, range(4)))


@pytest.mark.parametrize("shape", [(2, 9, 9, 32), (2, 200, 180, 32), (3, 101, 103, 36)])
def test_two_streams_and_two_graphs_at_once(shape):
    """Steps on two streams, and two captured steps replayed on two streams, do not share state."""
    sets, want = [], []
    for k in range(2):
        x = features(shape, torch.bfloat16, 30 + k).to(CUDA).requires_grad_(True)
        w, b = (t.to(CUDA).requires_grad_(True) for t in params(shape[-1], 32 + k))
        g = torch.randn(shape, device=CUDA).bfloat16()
        sets.append((x, w, b, torch.tensor([k], device=CUDA), g))
        want.append(training_step(*sets[k]))
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                got[k].append(training_step(*sets[k]))
    torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(p, q) for run in got[k] for p, q in zip(run, want[k]))
    graphs, outs = [], []
    for k in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=streams[k]):
            outs.append(training_step(*sets[k]))
        graphs.append(graph)
    for _ in range(4):
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                graphs[k].replay()
    torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(p, q) for p, q in zip(outs[k], want[k]))


def test_captured_step_draws_new_masks_from_its_seed():
    x = features((1, 16, 16, 32), torch.float32, 40).to(CUDA).requires_grad_(True)
    w, b = (t.to(CUDA).requires_grad_(True) for t in params(32, 41))
    g = torch.randn_like(x)
    want = [training_step(x, w, b, torch.tensor([k], device=CUDA), g) for k in (1, 2, 3)]
    seed = torch.zeros(1, dtype=torch.int64, device=CUDA)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        seed += 1
        out = training_step(x, w, b, seed, g)
    for expected in want:
        graph.replay()
        assert all(torch.equal(p, q) for p, q in zip(out, expected))


def test_residual_block_between_texture_and_antialias():
    """The operators as a learned shader uses them: texture features, a residual block (norm,
    activation and dropout, a product, dropout with the skip connection), antialias; the gradient
    reaches the texture and the block's parameters and matches the same block in float64 within
    the float32 rounding of its products (1e-4 of each gradient's largest value)."""
    import scenes

    sc = scenes.config5_small(views=2)
    ctx = dr.RasterizeContext(CUDA)
    pos, tri = sc["pos"].to(CUDA), sc["tri"].to(CUDA)
    gen = torch.Generator().manual_seed(50)
    tex = torch.randn(1, 32, 32, 16, generator=gen).to(CUDA).requires_grad_(True)
    w, b = (t.to(CUDA).requires_grad_(True) for t in params(16, 51))
    mix = (torch.randn(16, 16, generator=gen) / 4).to(CUDA).requires_grad_(True)
    out_mix = (torch.randn(16, 3, generator=gen) / 4).to(CUDA).requires_grad_(True)
    leaves = (tex, w, b, mix, out_mix)
    rast, rast_db = dr.rasterize(ctx, pos, tri, sc["resolution"])
    uv, _ = dr.interpolate(sc["attr"].to(CUDA), rast, tri)
    lookup = uv[..., 0:2].contiguous()
    target = torch.rand(*rast.shape[:3], 3, generator=gen).to(CUDA)

    def block(f, ours):
        if ours:
            h = dr.group_norm(f, 4, w, b, activation="silu", dropout=0.1, seed=7, layer=0)
            return dr.dropout(h @ mix, 0.2, 7, layer=1, residual=f) @ out_mix
        masks = [ref.keep_mask(f.numel(), p, 7, layer).view(f.shape).to(CUDA) * ref.keep_scale(p)
                 for layer, p in ((0, 0.1), (1, 0.2))]
        h = ref.group_norm(f, 4, w, b, activation="silu", factor=masks[0])
        return ((f.double() + (h @ mix.double()) * masks[1]) @ out_mix.double()).float()

    results = []
    for ours in (True, False):
        f = dr.texture(tex, lookup, filter_mode="linear")
        image, loss = dr.antialias_mse(block(f, ours), rast, pos, tri, target)
        results.append((image.detach(), torch.autograd.grad(loss, leaves)))
    torch.testing.assert_close(results[0][0], results[1][0], rtol=1e-4, atol=1e-4)
    for got, want in zip(results[0][1], results[1][1]):
        torch.testing.assert_close(got, want, rtol=1e-4, atol=1e-4 * float(want.abs().max()))
