"""Sizes of the row operators that do not fit 32 bits: refused before anything is copied, never cut to their lower half.  The tensors are
one element, expanded."""
import pytest
import torch

from test_gpu_native_path import _python

pytestmark = pytest.mark.gpu
DEV = "cuda"
BOTH = pytest.mark.parametrize("native", [True, False], ids=["native", "python"])
HUGE = 2 ** 32 + 4


def one(*shape, dtype=torch.bfloat16):
    return torch.ones(1, dtype=dtype, device=DEV).expand(shape)


def group(native, x, G, w, b):
    from dfa3d_b200.group_norm_ops import GroupNormFunction
    fn = GroupNormFunction if native else _python(GroupNormFunction)
    return fn.apply(x, w, b, None, None, G, 1e-5, None)


@pytest.fixture(autouse=True)
def nothing_is_allocated(lib_built):
    seed = torch.zeros(1, dtype=torch.int64, device=DEV)
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    yield seed
    assert torch.cuda.max_memory_allocated() - before < 1 << 20


@BOTH
@pytest.mark.parametrize("shape", [(HUGE, 1, 4), (2, HUGE, 4), (2 ** 31, 2, 4), (1, 2 ** 31 + 1, 4)])
def test_images_and_rows_of_a_group_norm(native, shape):
    w = torch.ones(4, device=DEV)
    with pytest.raises(RuntimeError, match="32 bits|too many"):
        group(native, one(*shape), 2, w, w)


@BOTH
def test_groups_of_a_group_norm(native):
    w = torch.ones(4, device=DEV)
    for G in (HUGE, 2 ** 31, -HUGE):
        with pytest.raises(RuntimeError, match="32 bits"):
            group(native, torch.ones(2, 3, 4, device=DEV), G, w, w)


@BOTH
def test_channels_of_a_group_norm(native):
    w = one(HUGE, dtype=torch.float32)
    with pytest.raises(RuntimeError, match="32 bits"):
        group(native, one(1, 1, HUGE), 4, w, w)


@BOTH
def test_columns_of_a_norm(native, nothing_is_allocated):
    from dfa3d_b200.dropout_ops import DropoutAddLayerNormFunction
    fn = DropoutAddLayerNormFunction if native else _python(DropoutAddLayerNormFunction)
    w = one(HUGE, dtype=torch.float32)
    with pytest.raises(RuntimeError, match="32 bits"):
        fn.apply(one(2, HUGE), one(2, HUGE), w, w, nothing_is_allocated, 0.5, 0, 1e-5)
