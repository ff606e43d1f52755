"""``dr.group_norm`` where the layouts of its images differ from one another, and two-pass calls of
more views than processors, against 64 bits with the bounds of ``test_gpu_group_norm``."""

import pytest
import torch

from test_gpu_group_norm import CUDA, TYPES, compare, features, params

pytestmark = pytest.mark.gpu


# Views above the 256 KB that clusters take: rows of folded pixels that start anywhere, of folded
# pixels that fill views, and of whole vectors.
@pytest.mark.parametrize("dtype, shape, groups, dropout", [
    (torch.float32, (150, 101, 103, 7), 7, 0.0), (torch.bfloat16, (150, 151, 129, 7), 1, 0.2),
    (torch.float16, (151, 180, 185, 4), 2, 0.0), (torch.float16, (149, 65, 67, 32), 8, 0.2),
])
def test_two_passes_over_more_views_than_processors(dtype, shape, groups, dropout):
    assert shape[1] * shape[2] * shape[3] * dtype.itemsize > 1 << 18
    compare(features(shape, dtype, 70), groups, *params(shape[-1], 71), activation="silu", dropout=dropout,
            seed=72)


def layouts(order, extra):
    """Maps the CPU image, and then its gradient, to a channel slice of a wider buffer or to a
    contiguous image, as ``order`` says for each."""
    order = iter(order)

    def on_gpu(t):
        if next(order) == "contiguous":
            return t.to(CUDA)
        wide = torch.full((*t.shape[:-1], t.shape[-1] + extra), float("nan"), dtype=t.dtype, device=CUDA)
        wide[..., extra:] = t.to(CUDA)
        return wide[..., extra:]

    return on_gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("extra", [1, 2, 4, 8])
@pytest.mark.parametrize("order", [("slice", "contiguous"), ("contiguous", "slice")], ids=["image", "gradient"])
@pytest.mark.parametrize("shape, groups", [((2, 11, 13, 16), 4), ((2, 120, 130, 32), 4), ((3, 90, 91, 30), 5)])
def test_one_of_image_and_gradient_is_a_slice(shape, groups, order, extra, dtype):
    compare(features(shape, dtype, 73), groups, *params(shape[-1], 74), activation="silu", dropout=0.1, seed=75,
            on_gpu=layouts(order, extra))
