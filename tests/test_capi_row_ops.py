"""The C entry points of dropout and group norm answer bad arguments with error codes before any pointer is used (no GPU needed)."""
import pytest

OK = 16          # an address that is aligned and never looked at


@pytest.fixture(scope="module")
def lib(lib_built):
    from dfa3d_b200 import _lib
    return _lib.load()


def refused(lib, rc, text, code=-1):
    assert rc == code and text in lib.dfa3d_last_error(), (rc, lib.dfa3d_last_error())


DROP = dict(x=OK, residual=None, dtype=0, n=8, activation=0, p=0.1, seed=OK, site=0, y=OK, stream=None)
DROP_BACK = dict(grad_y=OK, ref=None, by_result=0, dtype=0, n=8, p=0.1, seed=OK, site=0, grad_x=OK, stream=None)
NORM = dict(x=OK, residual=OK, gamma=OK, beta=OK, dtype=0, rows=4, E=8, p=0.1, seed=OK, site=0, eps=1e-5, y=OK, mean=OK, rstd=OK,
            stream=None)
NORM_BACK = dict(grad_y=OK, x=OK, residual=OK, gamma=OK, mean=OK, rstd=OK, dtype=0, rows=4, E=8, p=0.1, seed=OK, site=0, grad_x=OK,
                 grad_residual=OK, grad_gamma=OK, grad_beta=OK, workspace=OK, bytes=1 << 20, stream=None)
GROUP = dict(x=OK, dtype=0, B=2, N=40000, C=8, G=2, shapes=OK, stride=2, start=OK, L=2, weight=OK, bias=OK, weight_rows=1, eps=1e-5,
             activation=0, y=OK, mean=OK, rstd=OK, workspace=OK, bytes=1 << 20, stream=None)
GROUP_BACK = dict(grad_y=OK, x=OK, dtype=0, B=2, N=10, C=8, G=2, shapes=OK, stride=2, start=OK, L=2, weight=OK, bias=OK,
                  weight_rows=1, activation=0, mean=OK, rstd=OK, grad_x=OK, grad_weight=OK, grad_bias=OK, workspace=OK,
                  bytes=1 << 20, stream=None)
ENTRIES = {"dfa3d_dropout_forward": DROP, "dfa3d_dropout_backward": DROP_BACK, "dfa3d_dropout_add_layer_norm_forward": NORM,
           "dfa3d_dropout_add_layer_norm_backward": NORM_BACK, "dfa3d_group_norm_forward": GROUP,
           "dfa3d_group_norm_backward": GROUP_BACK}


def call(lib, name, **changed):
    args = dict(ENTRIES[name])
    assert set(changed) <= set(args)
    return getattr(lib, name)(*dict(args, **changed).values())


@pytest.mark.parametrize("name", list(ENTRIES)[:4])
def test_dropout_rule_is_checked(lib, name):
    for p in (-0.1, 1.1, float("nan"), float("inf")):
        refused(lib, call(lib, name, p=p), b"p must be in [0, 1]")
    refused(lib, call(lib, name, site=-1), b"site")
    refused(lib, call(lib, name, seed=None), b"`seed` is null")
    refused(lib, call(lib, name, seed=20), b"seed must be 8-byte aligned")


@pytest.mark.parametrize("name", list(ENTRIES))
def test_types_and_element_alignment_are_checked(lib, name):
    for dtype in (2, 4, -1):
        refused(lib, call(lib, name, dtype=dtype), b"dtype")
    first = next(k for k in ENTRIES[name] if k in ("x", "grad_y"))
    refused(lib, call(lib, name, **{first: 18}), b"aligned to its elements")
    refused(lib, call(lib, name, **{first: 17, "dtype": 1}), b"aligned to its elements")


@pytest.mark.parametrize("name", list(ENTRIES))
def test_null_tensors_are_refused(lib, name):
    optional = {"residual"} if name.startswith("dfa3d_dropout_forward") else set()
    optional |= {"ref", "stream", "grad_x", "grad_residual", "mean", "rstd"} if name != "dfa3d_dropout_backward" else \
        {"ref", "stream"}
    if name.endswith("norm_backward"):
        optional -= {"mean", "rstd"}
    for k, v in ENTRIES[name].items():
        if v == OK and k not in optional:
            rc = call(lib, name, **{k: None})
            assert rc == -1, (k, rc)


def test_statistics_and_parameter_gradients_come_in_pairs(lib):
    refused(lib, call(lib, "dfa3d_dropout_add_layer_norm_forward", mean=None), b"together")
    refused(lib, call(lib, "dfa3d_group_norm_forward", rstd=None), b"together")
    refused(lib, call(lib, "dfa3d_dropout_add_layer_norm_backward", grad_beta=None), b"together")
    refused(lib, call(lib, "dfa3d_group_norm_backward", grad_bias=None), b"together")


def test_sizes_are_checked(lib):
    for name in ("dfa3d_dropout_add_layer_norm_forward", "dfa3d_dropout_add_layer_norm_backward"):
        refused(lib, call(lib, name, E=1025), b"1024", -2)
        refused(lib, call(lib, name, E=0), b"E must be positive")
        refused(lib, call(lib, name, rows=-1), b"rows")
    refused(lib, call(lib, "dfa3d_dropout_forward", n=-1), b"n must be")
    refused(lib, call(lib, "dfa3d_dropout_forward", activation=2), b"activation")
    refused(lib, call(lib, "dfa3d_dropout_backward", by_result=1), b"ref_is_result")
    for name in ("dfa3d_group_norm_forward", "dfa3d_group_norm_backward"):
        refused(lib, call(lib, name, C=8, G=3), b"groups")
        refused(lib, call(lib, name, G=0), b"groups")
        refused(lib, call(lib, name, C=1032, G=1), b"exceeds", -2)
        refused(lib, call(lib, name, L=33), b"DFA3D_MAX_LEVELS", -2)
        refused(lib, call(lib, name, L=0), b"L must be positive")
        refused(lib, call(lib, name, B=-1), b"B and N")
        refused(lib, call(lib, name, N=1 << 30), b"too many", -2)
        refused(lib, call(lib, name, N=3000, B=1 << 21), b"too many", -2)
        refused(lib, call(lib, name, N=1, B=1 << 28), b"too many", -2)
        refused(lib, call(lib, name, N=40000, B=1 << 19, workspace=None), b"workspace")
        refused(lib, call(lib, name, weight_rows=3), b"weight_rows")
        refused(lib, call(lib, name, stride=1), b"shape_stride")
        refused(lib, call(lib, name, start=None), b"together")
        refused(lib, call(lib, name, start=None, shapes=None), b"without a level table")
        refused(lib, call(lib, name, activation=3), b"activation")
    refused(lib, call(lib, "dfa3d_group_norm_forward", eps=-1.0), b"eps")
    refused(lib, call(lib, "dfa3d_dropout_add_layer_norm_forward", eps=float("nan")), b"eps")


def test_workspaces_are_asked_for_and_checked(lib):
    need = lib.dfa3d_dropout_add_layer_norm_workspace(1000, 256)
    assert need > 0
    refused(lib, call(lib, "dfa3d_dropout_add_layer_norm_backward", rows=1000, E=256, bytes=need - 1), b"workspace")
    refused(lib, call(lib, "dfa3d_dropout_add_layer_norm_backward", workspace=24), b"workspace")
    assert lib.dfa3d_dropout_add_layer_norm_workspace(0, 256) == 0
    assert lib.dfa3d_dropout_add_layer_norm_workspace(5, 2000) == -2
    for backward, name in ((0, "dfa3d_group_norm_forward"), (1, "dfa3d_group_norm_backward")):
        need = lib.dfa3d_group_norm_workspace(2, 9000, 64, 4, 2, backward)
        assert need > 0
        refused(lib, call(lib, name, N=9000, C=64, G=4, bytes=need - 1), b"workspace")
        refused(lib, call(lib, name, workspace=24), b"workspace")
    assert lib.dfa3d_group_norm_workspace(2, 1000, 64, 4, 2, 0) == 0            # one launch
    assert lib.dfa3d_group_norm_workspace(2, 0, 64, 4, 2, 1) == 0
    assert lib.dfa3d_group_norm_workspace(2, 10, 64, 5, 2, 1) == -1


def test_empty_calls_are_fine_without_tensors(lib):
    assert call(lib, "dfa3d_dropout_forward", n=0, x=None, y=None, seed=None) == 0
    assert call(lib, "dfa3d_dropout_backward", n=0, grad_y=None, grad_x=None, seed=None) == 0
    assert call(lib, "dfa3d_dropout_add_layer_norm_forward", rows=0, x=None, residual=None, y=None, seed=None) == 0
    assert call(lib, "dfa3d_dropout_add_layer_norm_backward", rows=0, grad_y=None, grad_gamma=None, grad_beta=None) == 0
    assert call(lib, "dfa3d_group_norm_forward", N=0, x=None, y=None, workspace=None, bytes=0) == 0
    assert call(lib, "dfa3d_group_norm_backward", B=0, grad_y=None, grad_weight=None, grad_bias=None) == 0
