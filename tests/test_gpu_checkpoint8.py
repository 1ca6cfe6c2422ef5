"""compress8 and decompress8 against the definition in 64 bits: equal, not near."""
import pytest
import torch

import ffn_reference as ref

pytestmark = pytest.mark.gpu
TYPES = (torch.float32, torch.bfloat16, torch.float16)
LARGEST = {t: torch.finfo(t).max for t in TYPES}


def expected(x, fmt):
    v = ref.stands_for(x, fmt)
    big = LARGEST[x.dtype]
    return torch.where(torch.isnan(v), v, v.clamp(-big, big)).to(x.dtype)


def same(a, b):
    return torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(torch.nan_to_num(a, 0.0), torch.nan_to_num(b, 0.0))


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 31), (3, 32), (5, 33), (64, 40), (100, 59), (1000, 256), (77, 1000), (4097, 96)])
def test_values(rows, cols, dtype, fmt):
    import dfa3d_b200 as M
    g = torch.Generator(device="cuda").manual_seed(rows * 1000 + cols)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda")
    x = (n(rows, cols) * torch.exp(2 * n(cols)) * torch.exp(2 * n(rows, 1))).to(dtype)
    c = M.compress8(x, fmt)
    assert c.codes.shape == (rows, cols) and c.scales.shape == (rows, (cols + 31) // 32)
    y = M.decompress8(c)
    assert y.dtype == dtype and y.shape == x.shape and same(y, expected(x, fmt))


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", TYPES)
def test_ends_of_the_range(dtype, fmt):
    """Largest and smallest numbers of the type, the borders of the factor, zeros, ties."""
    import dfa3d_b200 as M
    fi = torch.finfo(dtype)
    smallest = fi.smallest_normal * fi.eps
    tops = [fi.max, fi.max / 2, fi.smallest_normal, smallest, 0.0, 1.0, 127.0, 127.5, 128.0, 448.0, 449.0, 464.0, 512.0, 1.984375, 1.9921875, 1.75, 1.76]
    rows = []
    for t in tops:
        r = torch.linspace(-1, 1, 32, dtype=torch.float64) * t
        r[0] = t
        rows.append(r)
    half = torch.arange(32, dtype=torch.float64) + 0.5          # ties of int8, exact in every type
    half[0] = 127
    rows.append(half)
    x = torch.stack(rows).to(dtype).cuda()
    assert same(M.decompress8(M.compress8(x, fmt)), expected(x, fmt))


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_blocks_that_hold_no_numbers(fmt):
    import dfa3d_b200 as M
    for bad in (float("nan"), float("inf"), -float("inf")):
        for dtype in TYPES:
            x = torch.randn(4, 100, device="cuda").to(dtype)
            x[1, 40] = bad
            x[3, 99] = bad
            y = M.decompress8(M.compress8(x, fmt))
            assert torch.isnan(y[1, 32:64]).all() and torch.isnan(y[3, 96:]).all() and int(torch.isnan(y).sum()) == 36


def test_shapes_strides_and_storage_off_the_grid():
    import dfa3d_b200 as M
    x = torch.randn(6, 5, 64, device="cuda").bfloat16()
    want = M.decompress8(M.compress8(x))
    assert torch.equal(M.decompress8(M.compress8(x.transpose(0, 1).contiguous().transpose(0, 1))), want)
    off = torch.empty(x.numel() + 1, dtype=x.dtype, device="cuda")[1:].view_as(x).copy_(x)
    assert torch.equal(M.decompress8(M.compress8(off)), want)
    assert torch.equal(M.decompress8(M.compress8(x[2, 3])), want[2, 3])
    for shape in ((0, 8), (3, 0), (0,)):
        e = torch.empty(shape, device="cuda")
        assert M.decompress8(M.compress8(e)).shape == e.shape


def test_no_gradient_and_other_streams():
    import dfa3d_b200 as M
    x = torch.randn(500, 96, device="cuda", requires_grad=True)
    c = M.compress8(x)
    assert not M.decompress8(c).requires_grad
    want = M.decompress8(c)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = M.decompress8(M.compress8(x))
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)


def test_past_two_to_the_31_elements():
    import dfa3d_b200 as M
    rows, cols = (1 << 25) + 3, 96              # 3.2e9 elements, 6.4 GB
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda")
    x[-2:] = torch.randn(2, cols, device="cuda").bfloat16()
    x[0, :5] = 3.0
    y = M.decompress8(M.compress8(x, "int8"))
    assert torch.equal(y[-2:], expected(x[-2:], "int8")) and torch.equal(y[0], expected(x[:1], "int8")[0])
    assert not y[1:-2].any()
