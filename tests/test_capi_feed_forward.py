"""The C entry points of the feed-forward products and of the 8-bit checkpoints answer bad arguments with error codes before any pointer
is used (no GPU needed); so do the Python functions."""
import ctypes

import pytest
import torch

OK = 64          # an address that is aligned and never looked at


@pytest.fixture(scope="module")
def lib(lib_built):
    from dfa3d_b200 import _lib
    return _lib.load()


def refused(lib, rc, text, code=-1):
    assert rc == code and text in lib.dfa3d_last_error(), (rc, lib.dfa3d_last_error())


LINEAR = dict(x=OK, x_pitch=16, weight=OK, weight_pitch=16, bias=OK, residual=OK, dtype=1, out_dtype=1, rows=4, cols_in=16, out=24,
              activation=0, y=OK, stream=None)
SLOPE = dict(x=OK, x_pitch=16, weight=OK, weight_pitch=16, bias=OK, grad_y=OK, grad_pitch=24, dtype=1, grad_dtype=1, rows=4, cols_in=16,
             out=24, activation=2, grad_z=OK, grad_z_pitch=24, stream=None)
INPUT = dict(grad=OK, grad2=OK, grad_pitch=24, weight=OK, weight2=OK, weight_pitch=16, add=OK, add_pitch=16, dtype=1, rows=4, cols_in=16,
             out=24, grad_x=OK, stream=None)
HIDDEN = dict(x=OK, x_pitch=16, weight_gate=OK, weight_up=OK, weight_pitch=16, bias_gate=OK, bias_up=OK, dtype=1, rows=4, cols_in=16,
              hidden=24, activation=2, h=OK, hidden_pitch=24, stream=None)
HIDDEN_BACK = dict(x=OK, x_pitch=16, weight_gate=OK, weight_up=OK, weight_pitch=16, bias_gate=OK, bias_up=OK, grad_y=OK, grad_pitch=32,
                   weight_down=OK, down_pitch=24, dtype=1, rows=4, cols_in=16, hidden=24, out=32, activation=2, grad_gate=OK, grad_up=OK,
                   h=OK, hidden_pitch=24, stream=None)
BLOCK = dict(x=OK, x_pitch=16, weight_gate=OK, weight_up=OK, weight_pitch=16, bias_gate=OK, bias_up=OK, weight_down=OK, down_pitch=24,
             bias_down=OK, residual=OK, dtype=1, out_dtype=1, rows=40000, cols_in=16, hidden=24, out=32, activation=2, y=OK, stream=None)
PACK = dict(x=OK, dtype=1, rows=4, cols=16, format=0, codes=OK, scales=OK, stream=None)
UNPACK = dict(codes=OK, scales=OK, format=0, rows=4, cols=16, dtype=1, x=OK, pitch=16, stream=None)
ENTRIES = {"dfa3d_linear_act_forward": LINEAR, "dfa3d_linear_act_slope": SLOPE, "dfa3d_linear_input_gradient": INPUT,
           "dfa3d_gated_hidden_forward": HIDDEN, "dfa3d_gated_hidden_backward": HIDDEN_BACK, "dfa3d_gated_block_forward": BLOCK, "dfa3d_compress8": PACK,
           "dfa3d_decompress8": UNPACK}
PRODUCTS = list(ENTRIES)[:6]


def call(lib, name, **changed):
    args = dict(ENTRIES[name])
    assert set(changed) <= set(args)
    return getattr(lib, name)(*dict(args, **changed).values())


@pytest.mark.parametrize("name", PRODUCTS)
def test_types_widths_and_activations(lib, name):
    for dtype in (0, 2, 4, -1):
        refused(lib, call(lib, name, dtype=dtype), b"dtype")
    for width in [k for k in ENTRIES[name] if k in ("cols_in", "out", "hidden")]:
        for bad in (0, -1):
            refused(lib, call(lib, name, **{width: bad}), b"widths must be positive")
        refused(lib, call(lib, name, **{width: (1 << 24) + 1}), b"too large", -2)
    refused(lib, call(lib, name, rows=-1), b"rows must be >= 0")
    refused(lib, call(lib, name, rows=2 ** 31 - 128), b"2^31 - 128", -2)
    refused(lib, call(lib, name, rows=2 ** 31 - 129, **{k: 1 << 24 for k in ENTRIES[name] if k == "out"} or {"hidden": 1 << 24}),
            b"too large", -2)
    if "activation" in ENTRIES[name]:
        for act in (-1, 4):
            refused(lib, call(lib, name, activation=act), b"activation")


@pytest.mark.parametrize("name", PRODUCTS)
def test_operands(lib, name):
    """Null, off the 16-byte grid, pitches that are too short or no multiple of eight."""
    args = ENTRIES[name]
    direct = {"bias", "grad_x", "bias_gate", "bias_up", "bias_down", "stream"} | (set() if "weight_down" in args else {"residual", "y"})
    optional = {"bias", "residual", "bias_gate", "bias_up", "bias_down", "stream", "add"}
    for k in [k for k, v in args.items() if v == OK]:
        if k in ("grad2", "weight2"):
            refused(lib, call(lib, name, **{k: None}), b"together")
        elif k not in optional:
            refused(lib, call(lib, name, **{k: None}), b"is null")
        if k not in direct:
            refused(lib, call(lib, name, **{k: OK + 8}), b"16-byte aligned")
        else:
            refused(lib, call(lib, name, **{k: OK + 1}), b"aligned to its elements")
    for k in [k for k in args if k.endswith("pitch")]:
        refused(lib, call(lib, name, **{k: args[k] - 8}), b"pitch")
        refused(lib, call(lib, name, **{k: args[k] + 4}), b"pitch")


@pytest.mark.parametrize("name", PRODUCTS + ["dfa3d_compress8", "dfa3d_decompress8"])
def test_no_rows_need_no_addresses(lib, name):
    empty = {k: None for k, v in ENTRIES[name].items() if v == OK}
    assert call(lib, name, rows=0, **empty) == 0


def test_mixed_types(lib):
    refused(lib, call(lib, "dfa3d_linear_act_forward", out_dtype=3), b"out_dtype")
    refused(lib, call(lib, "dfa3d_linear_act_slope", grad_dtype=3), b"grad_dtype")
    refused(lib, call(lib, "dfa3d_linear_act_forward", out_dtype=0, residual=OK + 2), b"aligned to its elements")


def test_the_block_with_one_kernel(lib):
    yes = lib.dfa3d_gated_block_supported
    assert yes(1, 40000, 256, 512, 256) and yes(0, 40000, 8, 1, 4) and yes(3, 40000, 256, 1 << 20, 8)
    for no in ((1, 900, 256, 512, 256), (1, 40000, 257, 512, 256), (1, 40000, 256, 512, 257), (1, 40000, 256, 512, 36), (0, 40000, 256, 512, 34),
               (2, 40000, 256, 512, 256), (1, -1, 256, 512, 256), (1, 40000, 0, 512, 256), (1, 40000, 256, 0, 256), (1, 40000, 256, 512, 0)):
        assert not yes(*no), no
    refused(lib, call(lib, "dfa3d_gated_block_forward", rows=100), b"not for one kernel", -2)
    refused(lib, call(lib, "dfa3d_gated_block_forward", out_dtype=3), b"out_dtype")


def test_compressed(lib):
    for name in ("dfa3d_compress8", "dfa3d_decompress8"):
        for fmt in (-1, 2):
            refused(lib, call(lib, name, format=fmt), b"format")
        refused(lib, call(lib, name, dtype=2), b"dtype")
        refused(lib, call(lib, name, rows=-1), b"must be >= 0")
        refused(lib, call(lib, name, cols=-1), b"must be >= 0")
        for k in ("x", "codes", "scales"):
            refused(lib, call(lib, name, **{k: None}), b"is null")
        refused(lib, call(lib, name, x=OK + 1), b"aligned to its elements")
    refused(lib, call(lib, "dfa3d_decompress8", pitch=15), b"pitch")


def table(**changed):
    from dfa3d_b200 import _lib
    t = (_lib.WeightGradient * 1)()
    values = dict(grad=OK, x=OK, grad_pitch=24, x_pitch=16, grad_weight=OK, grad_bias=OK, in_features=16, out_features=24)
    for k, v in dict(values, **changed).items():
        setattr(t[0], k, v)
    return t


def weight(lib, t, count=1, dtype=1, rows=4, workspace=OK, size=1 << 30):
    return lib.dfa3d_weight_gradients(ctypes.byref(t), count, dtype, rows, workspace, size, None)


def test_weight_gradients(lib):
    t = table()
    need = lib.dfa3d_weight_gradients_workspace(ctypes.byref(t), 1, 4)
    assert need > 0
    for count in (0, 4, -1):
        refused(lib, weight(lib, t, count=count), b"count")
        refused(lib, lib.dfa3d_weight_gradients_workspace(ctypes.byref(t), count, 4), b"count")
    refused(lib, lib.dfa3d_weight_gradients(None, 1, 1, 4, OK, need, None), b"is null")
    refused(lib, weight(lib, t, dtype=0), b"dtype")
    refused(lib, weight(lib, t, rows=-1), b"rows")
    refused(lib, weight(lib, t, workspace=None), b"is null")
    refused(lib, weight(lib, t, workspace=OK + 8), b"16-byte aligned")
    refused(lib, weight(lib, t, size=need - 1), b"smaller than")
    refused(lib, weight(lib, table(grad_weight=None)), b"is null")
    refused(lib, weight(lib, table(grad_weight=OK + 1)), b"aligned to its elements")
    refused(lib, weight(lib, table(grad_bias=OK + 1)), b"aligned to its elements")
    for k in ("grad", "x"):
        refused(lib, weight(lib, table(**{k: None})), b"is null")
        refused(lib, weight(lib, table(**{k: OK + 8})), b"16-byte aligned")
    for k, v in (("grad_pitch", 16), ("grad_pitch", 28), ("x_pitch", 8)):
        refused(lib, weight(lib, table(**{k: v})), b"pitch")
    for k in ("in_features", "out_features"):
        refused(lib, weight(lib, table(**{k: 0})), b"widths must be positive")
    wide = table(in_features=1 << 24, out_features=1 << 24)
    refused(lib, lib.dfa3d_weight_gradients_workspace(ctypes.byref(wide), 1, 4), b"too large", -2)


def test_copies(lib):
    from dfa3d_b200 import _lib
    copy = lambda **kw: (_lib.RowCopy * 1)(_lib.RowCopy(*dict(dict(src=OK, dst=OK, rows=2, cols=8, src_pitch=8, dst_pitch=8, wide=0), **kw).values()))
    go = lambda t, count=1, dtype=1: lib.dfa3d_copy_rows(ctypes.byref(t), count, dtype, None)
    refused(lib, go(copy(), count=0), b"count")
    refused(lib, go(copy(), count=9), b"count")
    refused(lib, go(copy(), dtype=0), b"dtype")
    for bad in (dict(rows=-1), dict(cols=-1), dict(src_pitch=7), dict(dst_pitch=7), dict(rows=2 ** 31)):
        refused(lib, go(copy(**bad)), b"copy 0")
    refused(lib, go(copy(src=None)), b"is null")
    refused(lib, go(copy(dst=None)), b"is null")
    refused(lib, go(copy(src=OK + 2, wide=1)), b"aligned to its elements")
    assert go(copy(src=None, dst=None, rows=0)) == 0


def test_python_refuses_other_tensors(lib_built):
    """No tensor of the CPU, of another type or size reaches a kernel."""
    import dfa3d_b200 as M
    x, w, b = torch.randn(4, 16).bfloat16(), torch.randn(24, 16).bfloat16(), torch.randn(24).bfloat16()
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        M.linear_act(x, w, b)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        M.gated_feed_forward(x, w, w, w.t())
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        M.compress8(x)
    with pytest.raises(ValueError, match="format"):
        M.compress8(x, "int4")
    with pytest.raises(RuntimeError, match="on one CUDA device"):
        from dfa3d_b200.checkpoint_ops import Compressed8
        M.decompress8(Compressed8(torch.zeros(4, 16, dtype=torch.uint8), torch.zeros(4, 1, dtype=torch.uint8), x.shape, x.dtype, "int8"))


def test_one_kernel_where_its_rows_divide_evenly(lib):
    """Tiles of 256 rows over pairs of SMs; without a device as many as this GPU has."""
    yes = lib.dfa3d_gated_block_supported
    for hidden in (512, 513):
        for rows in (9473, 18944, 30000, 40000, 80000):
            assert yes(1, rows, 256, hidden, 256), (rows, hidden)
        assert not yes(1, 9000, 256, hidden, 256)
    assert yes(1, 18945, 256, 512, 256) and not yes(1, 18945, 256, 513, 256) and not yes(1, 22000, 256, 513, 256)
