"""ctypes binding of libdfa3d_b200.so (the C ABI declared in include/dfa3d_b200.h).

There is no CPU or pure-PyTorch fallback: if the shared library is missing or a call fails, an
exception is raised.
"""
import ctypes
import operator
import os

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.environ.get("DFA3D_B200_LIB") or os.path.join(_HERE, "libdfa3d_b200.so")

ABI_VERSION = 2
DTYPE_F32 = 0
DTYPE_BF16 = 1
DTYPE_F64 = 2
DTYPE_F16 = 3
MAX_LEVELS = 32
MAX_CHANNELS = 1024

ERROR_NAMES = {-1: "invalid argument", -2: "unsupported", -3: "CUDA error"}


class Problem(ctypes.Structure):
    """struct dfa3d_problem."""
    _fields_ = [(n, ctypes.c_int32) for n in
                ("B", "N", "H", "C", "D", "L", "Q", "P", "value_dtype", "dist_dtype")] + \
               [("dist_head_stride", ctypes.c_int64), ("dist_map_h", ctypes.c_int32),
                ("dist_map_w", ctypes.c_int32)]

    def __init__(self, *args, **kw):
        # the two dist-map fields default to 0 (dist laid out like value)
        super().__init__(*args, **kw)


class WeightGradient(ctypes.Structure):
    """struct dfa3d_weight_gradient."""
    _fields_ = [("grad", ctypes.c_void_p), ("x", ctypes.c_void_p), ("grad_pitch", ctypes.c_int64), ("x_pitch", ctypes.c_int64),
                ("grad_weight", ctypes.c_void_p), ("grad_bias", ctypes.c_void_p), ("in_features", ctypes.c_int32),
                ("out_features", ctypes.c_int32)]


class RowCopy(ctypes.Structure):
    """struct dfa3d_row_copy."""
    _fields_ = [("src", ctypes.c_void_p), ("dst", ctypes.c_void_p)] + \
               [(n, ctypes.c_int64) for n in ("rows", "cols", "src_pitch", "dst_pitch")] + [("wide", ctypes.c_int32)]


class _I32:
    """An int32 argument.  ctypes.c_int32 would pass the lower half of a number that does not fit."""

    @staticmethod
    def from_param(v):
        v = operator.index(v)
        if not -2 ** 31 <= v < 2 ** 31:
            raise OverflowError(f"{v} does not fit 32 bits")
        return v                       # ctypes passes a Python integer as a C int


_P = ctypes.POINTER(Problem)
_V = ctypes.c_void_p
_I64 = ctypes.c_int64

# name -> number of pointer arguments after the problem descriptor (the stream included)
ENTRY_POINTS = {
    "dfa3d_depth_score_forward": 6,
    "dfa3d_depth_score_backward": 8,
    "dfa3d_wms_attn_forward": 8,
    "dfa3d_wms_attn_backward": 12,
    "dfa3d_fused_forward": 9,
    "dfa3d_fused_backward": 12,
    "dfa3d_msda_forward": 7,
    "dfa3d_msda_backward": 10,
    # double-precision instantiations (same argument lists)
    "dfa3d_depth_score_forward_f64": 6,
    "dfa3d_depth_score_backward_f64": 8,
    "dfa3d_wms_attn_forward_f64": 8,
    "dfa3d_wms_attn_backward_f64": 12,
    "dfa3d_fused_forward_f64": 9,
    "dfa3d_fused_backward_f64": 12,
    # ragged variants: the query-offset table is one more pointer, right after the descriptor
    "dfa3d_fused_forward_ragged": 10,
    "dfa3d_fused_backward_ragged": 13,
}
# entry points that take `int32_t num_anchors` right after the descriptor
ENTRY_POINTS_WITH_ANCHORS = {
    "dfa3d_attn3d_forward": 10,
    "dfa3d_attn3d_backward": 15,
    "dfa3d_attn3d_forward_ragged": 11,
    "dfa3d_attn3d_backward_ragged": 16,
}
# entry points without a problem descriptor: explicit argument types
PLAIN_ENTRY_POINTS = {
    "dfa3d_attn2d_supported": [_P, _I32],
    "dfa3d_attn2d_forward": [_P, _I32, _I64, _I64] + [_V] * 8,
    "dfa3d_attn2d_backward": [_P, _I32, _I64, _I64] + [_V] * 11,
    "dfa3d_attn3d_forward_rows": [_P, _I32, _I32, _I64, _I64] + [_V] * 12,
    "dfa3d_attn3d_backward_rows": [_P, _I32, _I32, _I64, _I64] + [_V] * 16,
    "dfa3d_rebatch_plan": [ctypes.c_void_p, _I32, _I32, _I32, _I32] + [ctypes.c_void_p] * 8,
    "dfa3d_rebatch_gather": [ctypes.c_void_p] * 4 + [_I32] * 4 + [_I64, _I64] + [ctypes.c_void_p] * 2
                            + [_I64, ctypes.c_void_p],
    "dfa3d_rebatch_combine": [ctypes.c_void_p] * 3 + [_I32] * 4 + [ctypes.c_void_p] * 3,
    "dfa3d_dist_from_logits": [ctypes.c_void_p] + [_I32] * 4 + [ctypes.c_void_p, _I32, ctypes.c_void_p]
                              + [_I32] * 4 + [ctypes.c_void_p] * 2,
    "dfa3d_dist_from_logits_backward": [ctypes.c_void_p] + [_I32] * 4 + [ctypes.c_void_p, _I32, ctypes.c_void_p]
                                       + [_I32] * 3 + [ctypes.c_void_p] * 3,
    "dfa3d_dist_from_logits_backward_typed": [ctypes.c_void_p] + [_I32] * 4
                                             + [ctypes.c_void_p, _I32, ctypes.c_void_p] + [_I32] * 4
                                             + [ctypes.c_void_p] * 3,
    "dfa3d_add_layer_norm_forward": [ctypes.c_void_p] * 4 + [_I64, _I32, ctypes.c_float] + [ctypes.c_void_p] * 5,
    "dfa3d_layer_norm_backward": [ctypes.c_void_p] * 5 + [_I64, _I32] + [ctypes.c_void_p] * 4,
    "dfa3d_column_sum": [ctypes.c_void_p, _I64, _I32, ctypes.c_void_p, ctypes.c_void_p],
    "dfa3d_add_layer_norm_infer": [ctypes.c_void_p] * 4 + [_I64, _I32, ctypes.c_float] + [ctypes.c_void_p] * 2,
    "dfa3d_relu_backward_column_sum": [ctypes.c_void_p] * 2 + [_I64, _I32] + [ctypes.c_void_p] * 3,
    "dfa3d_relu_dropout_backward_column_sum": [ctypes.c_void_p] * 2 + [_I64, _I32, ctypes.c_double] + [ctypes.c_void_p] * 3,
    "dfa3d_slice_sum": [ctypes.c_void_p] + [_I32] * 3 + [ctypes.c_void_p] * 2 + [_I32] + [ctypes.c_void_p] * 3,
    "dfa3d_copy_segments": [ctypes.c_void_p] * 3 + [_I32, ctypes.c_void_p],
    "dfa3d_convert_two": [_I32, _I32, _V, _V, _I64, _V, _V, _I64, _V],
    "dfa3d_dropout_forward": [_V, _V, _I32, _I64, _I32, ctypes.c_double, _V, _I32, _V, _V],
    "dfa3d_dropout_backward": [_V, _V, _I32, _I32, _I64, ctypes.c_double, _V, _I32, _V, _V],
    "dfa3d_dropout_add_layer_norm_forward": [_V] * 4 + [_I32, _I64, _I32, ctypes.c_double, _V, _I32, ctypes.c_float] + [_V] * 4,
    "dfa3d_dropout_add_layer_norm_backward": [_V] * 6 + [_I32, _I64, _I32, ctypes.c_double, _V, _I32] + [_V] * 5 + [_I64, _V],
    "dfa3d_group_norm_forward": [_V] + [_I32] * 5 + [_V, _I32, _V, _I32, _V, _V, _I32, ctypes.c_float, _I32] + [_V] * 4
                                + [_I64, _V],
    "dfa3d_group_norm_backward": [_V, _V] + [_I32] * 5 + [_V, _I32, _V, _I32, _V, _V, _I32, _I32] + [_V] * 6 + [_I64, _V],
    "dfa3d_dropout_add_layer_norm_workspace": [_I64, _I32],
    "dfa3d_group_norm_workspace": [_I32] * 6,
    "dfa3d_linear_act_forward": [_V, _I64, _V, _I64, _V, _V, _I32, _I32, _I64, _I32, _I32, _I32, _V, _V],
    "dfa3d_linear_act_slope": [_V, _I64, _V, _I64, _V, _V, _I64, _I32, _I32, _I64, _I32, _I32, _I32, _V, _I64, _V],
    "dfa3d_linear_input_gradient": [_V, _V, _I64, _V, _V, _I64, _V, _I64, _I32, _I64, _I32, _I32, _V, _V],
    "dfa3d_gated_hidden_forward": [_V, _I64, _V, _V, _I64, _V, _V, _I32, _I64, _I32, _I32, _I32, _V, _I64, _V],
    "dfa3d_gated_block_supported": [_I32, _I64, _I32, _I32, _I32],
    "dfa3d_gated_block_forward": [_V, _I64, _V, _V, _I64, _V, _V, _V, _I64, _V, _V, _I32, _I32, _I64] + [_I32] * 4 + [_V, _V],
    "dfa3d_gated_hidden_backward": [_V, _I64, _V, _V, _I64, _V, _V, _V, _I64, _V, _I64, _I32, _I64] + [_I32] * 4
                                   + [_V, _V, _V, _I64, _V],
    "dfa3d_weight_gradients_workspace": [_V, _I32, _I64],
    "dfa3d_weight_gradients": [_V, _I32, _I32, _I64, _V, _I64, _V],
    "dfa3d_copy_rows": [_V, _I32, _I32, _V],
    "dfa3d_compress8": [_V, _I32, _I64, _I32, _I32, _V, _V, _V],
    "dfa3d_decompress8": [_V, _V, _I32, _I64, _I32, _I32, _V, _I64, _V],
    "dfa3d_zero_two": [ctypes.c_void_p, _I64, ctypes.c_void_p, _I64, ctypes.c_void_p],
}
# of these the ones that answer with a number of bytes (or a negative error code)
SIZE_ENTRY_POINTS = ("dfa3d_dropout_add_layer_norm_workspace", "dfa3d_group_norm_workspace",
                     "dfa3d_weight_gradients_workspace")
ACT_SOFTMAX, ACT_SIGMOID = 0, 1
ROW_NONE, ROW_RELU, ROW_SILU, ROW_GELU = 0, 1, 2, 3
FORMAT_INT8, FORMAT_E4M3 = 0, 1

_lib = None
_native = None
_calls = 0      # successful entry-point calls made from Python so far


def __getattr__(name):
    # `calls`: successful entry-point calls so far, from Python and from the native host path (each launches
    # at least one kernel)
    if name == "calls":
        return _calls + (_native.calls() if _native is not None else 0)
    raise AttributeError(name)


def load():
    """Load the library once; raise with build instructions if it is absent."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise ImportError(
            f"{LIB_PATH} not found: build it with `python 3d-deformable-attention_b200/build.py` "
            "(needs nvcc; targets sm_100a). dfa3d_b200 has no fallback implementation.")
    lib = ctypes.CDLL(LIB_PATH)
    lib.dfa3d_abi_version.restype = ctypes.c_int
    lib.dfa3d_abi_version.argtypes = []
    lib.dfa3d_last_error.restype = ctypes.c_char_p
    lib.dfa3d_last_error.argtypes = []
    for name, nptr in ENTRY_POINTS.items():
        fn = getattr(lib, name)
        fn.restype = ctypes.c_int
        fn.argtypes = [_P] + [_V] * nptr
    for name, nptr in ENTRY_POINTS_WITH_ANCHORS.items():
        fn = getattr(lib, name)
        fn.restype = ctypes.c_int
        fn.argtypes = [_P, _I32] + [_V] * nptr
    for name, argtypes in PLAIN_ENTRY_POINTS.items():
        fn = getattr(lib, name)
        fn.restype = ctypes.c_int
        fn.argtypes = argtypes
    for name in SIZE_ENTRY_POINTS:
        getattr(lib, name).restype = _I64
    got = lib.dfa3d_abi_version()
    if got != ABI_VERSION:
        raise ImportError(f"libdfa3d_b200.so has ABI version {got}, this package expects {ABI_VERSION}")
    _lib = lib
    return lib


def native():
    """The native host path (csrc/binding): built beside the library, bound to the library's entry points."""
    global _native
    if _native is None:
        import torch
        lib = load()
        how = "build it with `python 3d-deformable-attention_b200/build.py`. dfa3d_b200 has no fallback implementation."
        try:
            from . import _native as mod
        except ImportError as e:
            raise ImportError(f"{e}: {how}") from e
        if mod.built_for.split()[1] != str(torch.__version__):
            raise ImportError(f"{mod.__file__} was built for {mod.built_for}, this is torch {torch.__version__}: {how}")
        mod.bind({n: ctypes.cast(getattr(lib, n), ctypes.c_void_p).value for n in mod.entries()})
        _native = mod
    return _native


def native_apply(name):
    """Class decorator: ``apply`` first offers the call to the native host path (csrc/binding),
    which takes the plain case -- CUDA tensors of the usual types and layouts, no autocast, functorch or tracing -- and
    answers NotImplemented to anything else; the Python Function then runs, with its checks and messages.
    Measured on 512 queries, forward + backward: 190 us a pass through the Python Function, of which 34 us are
    kernels."""

    def wrap(cls):
        python_apply = cls.apply.__func__
        fast = None

        def apply(c, *args):
            nonlocal fast
            if c is cls:                        # a subclass may have overridden forward or backward
                if fast is None:
                    fast = getattr(native(), name)
                out = fast(*args)
                if out is not NotImplemented:
                    return out
            return python_apply(c, *args)

        cls.apply = classmethod(apply)
        return cls

    return wrap


def _invoke(name, *args):
    """What an entry point answers; arguments that cannot be passed on raise like those that it refuses."""
    try:
        return getattr(load(), name)(*args)
    except ctypes.ArgumentError as e:
        raise RuntimeError(f"{name} failed ({ERROR_NAMES[-1]}): {e}") from None


def size(name, *args):
    """Bytes of workspace that an entry point asks for."""
    n = _invoke(name, *args)
    if n < 0:
        msg = load().dfa3d_last_error().decode("utf-8", "replace")
        raise RuntimeError(f"{name} failed ({ERROR_NAMES.get(n, n)}): {msg}")
    return n


def call_plain(name, *args):
    """Invoke an entry point that takes no problem descriptor."""
    rc = _invoke(name, *args)
    if rc != 0:
        msg = load().dfa3d_last_error().decode("utf-8", "replace")
        raise RuntimeError(f"{name} failed ({ERROR_NAMES.get(rc, rc)}): {msg}")
    global _calls
    _calls += 1


def call(name, problem, *ptrs):
    """Invoke an entry point; raise RuntimeError carrying dfa3d_last_error() on failure."""
    rc = _invoke(name, ctypes.byref(problem), *ptrs)
    if rc != 0:
        msg = load().dfa3d_last_error().decode("utf-8", "replace")
        raise RuntimeError(f"{name} failed ({ERROR_NAMES.get(rc, rc)}): {msg}")
    global _calls
    _calls += 1
