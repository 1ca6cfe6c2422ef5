"""The gated block in one kernel with several tiles of rows a pair of SMs, where few hidden columns make every item, or every other one, begin
new rows: x's slots, the ring, hidden rows and the result's accumulator come round again with each."""
import pytest
import torch

from test_gpu_gated_feed_forward import check, make

pytestmark = pytest.mark.gpu
ROWS = 60001          # 235 tiles of 256 rows over 74 pairs: three or four each, the last one ragged


@pytest.mark.parametrize("E,F,N", [(64, 128, 64), (8, 8, 8), (256, 100, 256), (136, 40, 200), (256, 129, 256), (72, 256, 130), (72, 256, 132)])
@pytest.mark.parametrize("residual", [None, "same", "wide"])
def test_few_hidden_columns(lib_built, E, F, N, residual):
    from dfa3d_b200 import _lib
    pairs = torch.cuda.get_device_properties(0).multi_processor_count // 2
    assert (ROWS + 255) // 256 >= 3 * pairs
    out = _lib.DTYPE_F32 if residual == "wide" else _lib.DTYPE_BF16
    one = _lib.load().dfa3d_gated_block_supported(out, ROWS, E, F, N)
    # rows of 260, 520 and 264 bytes are off the 16-byte grid: two kernels
    assert bool(one) == (N != 130 and not (N == 132 and out == _lib.DTYPE_BF16))
    check(make(ROWS, E, F, N, torch.bfloat16, residual=residual, seed=F), "silu")


def test_the_residual_that_is_x(lib_built):
    check(make(ROWS, 256, 128, 256, torch.float16, residual="x", seed=1), "gelu")
