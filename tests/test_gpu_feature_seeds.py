"""Seeds as numbers and as device words give the same masks in every kernel that draws them: in
clusters, in passes over whole vectors, folded pixels and single elements (with elements left over),
forward and backward, and in ``dr.dropout`` with and without a residual."""

import pytest
import torch

import diffrast_b200 as dr

pytestmark = pytest.mark.gpu
CUDA = "cuda"
SEED = (1 << 62) + 12345678901


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape, extra", [((2, 9, 9, 32), 0), ((2, 120, 130, 32), 0), ((3, 101, 103, 30), 0),
                                          ((2, 9, 9, 32), 1), ((2, 120, 130, 32), 1)])
@pytest.mark.parametrize("activation", ["none", "silu"])
def test_norm_masks_do_not_depend_on_the_seeds_form(shape, extra, activation, dtype):
    gen = torch.Generator(device=CUDA).manual_seed(1)
    x = torch.randn(*shape[:-1], shape[-1] + extra, generator=gen, device=CUDA).to(dtype)[..., extra:]
    grad = torch.randn(shape, generator=gen, device=CUDA).to(dtype)
    results = []
    for seed in (SEED, torch.tensor([SEED], device=CUDA)):
        leaf = x.detach().requires_grad_(True)
        y = dr.group_norm(leaf, 2, activation=activation, dropout=0.3, seed=seed, layer=2)
        results.append((y.detach(), torch.autograd.grad(y, leaf, grad)[0]))
    assert all(torch.equal(a, b) for a, b in zip(*results))
    dropped = results[0][0] == 0
    assert 0.25 < dropped.float().mean() < 0.35


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("count", [1, 4099, 1 << 20])
@pytest.mark.parametrize("residual", [False, True])
def test_dropout_masks_do_not_depend_on_the_seeds_form(count, residual, dtype):
    gen = torch.Generator(device=CUDA).manual_seed(2)
    x = torch.randn(count, generator=gen, device=CUDA).to(dtype)
    skip = torch.randn(count, generator=gen, device=CUDA).to(dtype) if residual else None
    a, b = (dr.dropout(x, 0.3, seed, layer=3, residual=skip) for seed in (SEED, torch.tensor([SEED], device=CUDA)))
    assert torch.equal(a, b)
