"""CPU checks of the feature-image operators: the restated generator against published vectors,
argument checks and messages of ``dr.group_norm`` and ``dr.dropout``, and refusals of the C ABI
(made before any CUDA call)."""

import pytest
import torch

import diffrast_b200 as dr
from diffrast_b200 import _kernels as K
from diffrast_b200 import _native
from feature_reference import keep_mask, keep_scale, philox4x32_10, threshold


def test_generator_known_answers():
    """The zero and all-ones vectors published with Philox4x32-10."""
    assert philox4x32_10((0, 0, 0, 0), (0, 0)) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    ones = 0xFFFFFFFF
    assert philox4x32_10((ones,) * 4, (ones,) * 2) == [
        0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]


def test_masks_are_made_of_the_generators_words():
    seed, layer = 0xFEDCBA9876543210, 5
    for block in (0, 1, 77, (1 << 32) + 3):
        words = philox4x32_10((block & 0xFFFFFFFF, block >> 32, layer, 0), (seed & 0xFFFFFFFF, seed >> 32))
        want = [half >= threshold(0.3) for w in words for half in (w & 0xFFFF, w >> 16)]
        assert keep_mask(8, 0.3, seed, layer, first=8 * block).tolist() == want


def test_mask_of_a_range_is_a_range_of_the_mask():
    whole = keep_mask(64, 0.5, 12345, layer=2)
    assert torch.equal(keep_mask(21, 0.5, 12345, layer=2, first=13), whole[13:34])
    assert 16 < int(whole.sum()) < 48
    assert threshold(0.1) == 6554 and threshold(0.9999999) == 65535
    assert keep_scale(0.5) == 2.0


X = torch.zeros(2, 4, 4, 6)


@pytest.mark.parametrize("call, error, pattern", [
    (lambda: dr.group_norm([1.0], 1), TypeError, "x must be a torch.Tensor"),
    (lambda: dr.group_norm(X.double(), 1), TypeError, "float32, float16 or bfloat16"),
    (lambda: dr.group_norm(X.int(), 1), TypeError, "float32, float16 or bfloat16"),
    (lambda: dr.group_norm(X[0, 0, 0], 1), ValueError, r"\[batch, ..., channels\]"),
    (lambda: dr.group_norm(X[..., :0], 1), ValueError, "must have channels"),
    (lambda: dr.group_norm(X, 4), ValueError, "must divide the 6 channels"),
    (lambda: dr.group_norm(X, 0), ValueError, "must divide the 6 channels"),
    (lambda: dr.group_norm(X, 2.0), TypeError, "groups must be an int"),
    (lambda: dr.group_norm(X, True), TypeError, "groups must be an int"),
    (lambda: dr.group_norm(torch.zeros(1, 1 << 17), 1), ValueError, "at most 65536 channels"),
    (lambda: dr.group_norm(X, 2, torch.ones(5)), ValueError, r"weight must have shape"),
    (lambda: dr.group_norm(X, 2, torch.ones(3, 6)), ValueError, r"weight must have shape"),
    (lambda: dr.group_norm(X, 2, None, torch.ones(6, 2)), ValueError, r"bias must have shape"),
    (lambda: dr.group_norm(X, 2, torch.ones(6).half()), TypeError, "weight must be torch.float32"),
    (lambda: dr.group_norm(X, 2, 1.0), TypeError, "weight must be a torch.Tensor"),
    (lambda: dr.group_norm(X, 2, torch.ones(6, device="meta")), ValueError, "same device"),
    (lambda: dr.group_norm(X, 2, eps=-1e-5), ValueError, "eps must be"),
    (lambda: dr.group_norm(X, 2, eps=float("nan")), ValueError, "eps must be"),
    (lambda: dr.group_norm(X, 2, activation="gelu"), ValueError, "Unknown activation 'gelu'"),
    (lambda: dr.group_norm(X, 2, dropout=0.5), ValueError, "seed is required"),
    (lambda: dr.group_norm(X, 2, dropout=1.0, seed=1), ValueError, r"in \[0, 1\)"),
    (lambda: dr.group_norm(X, 2, dropout=0.5, seed=-1), ValueError, "seed must be in"),
    (lambda: dr.group_norm(X, 2, dropout=0.5, seed=1.5), TypeError, "seed must be an int"),
    (lambda: dr.group_norm(X, 2, dropout=0.5, seed=torch.zeros(2).long()), TypeError, "one element"),
    (lambda: dr.group_norm(X, 2, dropout=0.5, seed=torch.zeros(1)), TypeError, "one element"),
    (lambda: dr.group_norm(X, 2, dropout=0.5, seed=1, layer=-1), ValueError, "layer must be"),
    (lambda: dr.group_norm(X, 2, dropout=0.5, seed=1, layer=1 << 32), ValueError, "layer must be"),
    (lambda: dr.dropout(X, float("nan"), 1), ValueError, r"p must be a probability"),
    (lambda: dr.dropout(X, -0.1, 1), ValueError, r"p must be a probability"),
    (lambda: dr.dropout(X, True, 1), ValueError, r"p must be a probability"),
    (lambda: dr.dropout(X, 0.5, None), TypeError, "seed must be"),
    (lambda: dr.dropout(X.long(), 0.5, 1), TypeError, "float32, float16 or bfloat16"),
    (lambda: dr.dropout(X, 0.5, 1, residual=X[0]), ValueError, "residual must match x"),
    (lambda: dr.dropout(X, 0.5, 1, residual=X.half()), TypeError, "residual must be torch.float32"),
    (lambda: dr.dropout(X, 0.5, 1, residual=1.0), TypeError, "residual must be a torch.Tensor"),
    (lambda: dr.dropout(X, 0.5, 1), RuntimeError, "CUDA devices only"),
    (lambda: dr.group_norm(X, 2), RuntimeError, "CUDA devices only"),
    (lambda: dr.group_norm(X[:0], 2), RuntimeError, "CUDA devices only"),
])
def test_arguments_are_checked(call, error, pattern):
    with pytest.raises(error, match=pattern):
        call()


def test_rows_of_feature_tensors():
    """Uniform pixel strides are used in place; anything else is copied."""
    wide = torch.arange(2 * 3 * 4 * 10.0).view(2, 3, 4, 10)
    for view, stride in ((wide, 10), (wide[..., 2:7], 10), (wide[..., 3:4], 10), (wide[:, :1, :1], 120),
                         (wide[:1, :1, :1, 2:5], 3), (wide[:, :, ::2], 20)):
        rows, got = K.feature_rows(view)
        assert rows.data_ptr() == view.data_ptr() and got == stride
    for view in (wide[:, 1:], wide[..., ::2], wide.transpose(1, 2),
                 wide[:, :, :1].expand(2, 3, 4, 10), wide[..., :1].expand(2, 3, 4, 5)):
        rows, got = K.feature_rows(view)
        assert rows.is_contiguous() and got == view.shape[-1] and torch.equal(rows, view)


def fwd(lib, **change):
    a = dict(x=16, x_stride=8, dtype=0, batch=2, pixels=9, channels=8, groups=2, w=16, wd=0, wb=1,
             b=16, bd=0, bb=1, eps=1e-5, act=0, drop=0, seed=None, value=0, layer=0, y=16, state=16,
             ws=16, ws_bytes=1 << 20, stream=None)
    a.update(change)
    return lib.dr_group_norm_fwd(*a.values())


def bwd(lib, **change):
    a = dict(x=16, x_stride=8, gy=16, gy_stride=8, dtype=0, batch=2, pixels=9, channels=8, groups=2,
             state=16, act=0, drop=0, seed=None, value=0, layer=0, gx=16, w=16, wd=0, wb=1, b=16,
             bd=0, bb=1, ws=16, ws_bytes=1 << 20, stream=None)
    a.update(change)
    return lib.dr_group_norm_bwd(*a.values())


def test_c_abi_refuses_before_any_cuda_call():
    lib = _native.lib()
    bad, small = 10001, 10002
    common = [dict(dtype=3), dict(dtype=-1), dict(batch=-1), dict(pixels=-1), dict(channels=0),
              dict(groups=0), dict(groups=3), dict(x_stride=7), dict(act=3), dict(act=-1),
              dict(drop=-1), dict(drop=65536), dict(layer=-1), dict(layer=1 << 32), dict(w=16, wb=3), dict(b=16, bd=4), dict(x=None),
              dict(x=18), dict(dtype=1, x=17), dict(w=18), dict(w=17, wd=1), dict(b=18), dict(ws=24), dict(seed=20),
              dict(state=None), dict(state=8), dict(channels=1 << 17, x_stride=1 << 17, gy_stride=1 << 17)]
    for change in common + [dict(y=None), dict(y=18)]:
        change.pop("gy_stride", None)
        assert fwd(lib, **change) == bad, change
    for change in common + [dict(gy=None), dict(gy_stride=7), dict(gy=18), dict(gx=18)]:
        assert bwd(lib, **change) == bad, change
    for call in (fwd, bwd):
        # An image too large for shared memory needs scratch in both directions.
        assert call(lib, pixels=1 << 24, ws_bytes=0) == small
        assert call(lib, pixels=1 << 24, ws=None) == small
        assert call(lib, batch=0) == 0 and call(lib, pixels=0) == 0
        assert call(lib, batch=1 << 31) == 10003 and call(lib, pixels=1 << 31) == 10003
        # Sizes whose products would pass 64 bits.
        assert call(lib, batch=(1 << 31) - 1, pixels=(1 << 31) - 1) == 10003
        assert call(lib, x_stride=1 << 62) == 10003
    assert bwd(lib, gy_stride=1 << 62) == 10003
    assert lib.dr_group_norm_workspace_bytes((1 << 31) - 1, (1 << 31) - 1, 1 << 16, 2, 0, 1) == 0
    assert lib.dr_group_norm_workspace_bytes(2, 9, 8, 3, 0, 0) == 0
    assert lib.dr_group_norm_state_floats(2, 8, 4) == 2 * (3 * 8 + 4)
    for backward in (0, 1):
        assert lib.dr_group_norm_workspace_bytes(2, 1 << 24, 8, 2, 0, backward) > 0
    assert lib.dr_group_norm_workspace_bytes(2, 9, 8, 2, 0, 0) == 0

    def drop(x=16, res=None, count=8, dtype=0, thr=1, seed=None, y=16):
        return lib.dr_dropout(x, res, count, dtype, thr, seed, 0, 0, y, None)

    for change in (dict(count=-1), dict(dtype=3), dict(thr=-1), dict(thr=65536), dict(x=None),
                   dict(y=None), dict(x=18), dict(y=18), dict(res=18), dict(dtype=2, x=17), dict(seed=20)):
        assert drop(**change) == bad, change
    assert drop(count=1 << 44) == 10003
    assert drop(count=0) == 0
