"""Weight gradients of more tiles than pairs of SMs: one share of the rows each, and CTAs that begin when others have ended, on the tensor
memory that these gave back."""
import ctypes

import pytest
import torch

from test_gpu_linear_act import check, make, run

pytestmark = pytest.mark.gpu


def shares(rows, K, N):
    """Of the rows, and tiles of 256 x 256, from the size of the workspace: 2 x 257 x 128 fp32 sums for each of both."""
    from dfa3d_b200 import _lib
    t = (_lib.WeightGradient * 1)()
    t[0].in_features, t[0].out_features = K, N
    tiles = -(-N // 256) * -(-K // 256)
    each = tiles * 2 * 257 * 128 * 4
    need = _lib.size("dfa3d_weight_gradients_workspace", ctypes.byref(t), 1, rows)
    assert need % each == 0
    return need // each, tiles


# rows: two and eight steps of 64 for each CTA, the ring of six goes round
@pytest.mark.parametrize("rows", [70, 450])
@pytest.mark.parametrize("K,N", [(4100, 1300), (1290, 4111)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_more_tiles_than_pairs_of_sms(lib_built, rows, K, N, dtype):
    assert shares(rows, K, N) == (1, 102) and torch.cuda.get_device_properties(0).multi_processor_count // 2 < 102
    check(make(rows, K, N, dtype, seed=rows), None)


def test_same_bits_and_streams_with_several_waves(lib_built):
    """Two streams, each with CTAs of several waves that wait for an SM of their own."""
    jobs = [make(450, 4100, 1300, torch.bfloat16, seed=s) for s in (1, 2)]
    want = [run(d, "silu") for d in jobs]
    streams = [torch.cuda.Stream() for _ in jobs]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(run(jobs[i], "silu"))
    torch.cuda.synchronize()
    for i, (y, grads) in enumerate(want):
        for y2, grads2 in got[i]:
            assert torch.equal(y, y2) and all(torch.equal(grads[k], grads2[k]) for k in grads)
