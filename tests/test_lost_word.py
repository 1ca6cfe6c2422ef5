"""What the feed-forward kernels store where a wait inside them has run out, on the CPU: NaN in every storage type.  (That a kernel gets there
is not brought about on a GPU.)"""
import ctypes
import os
import subprocess

import pytest
import torch

from conftest import PKG_DIR

SOURCE = """
#include "dfa3d_lost.h"
extern "C" uint32_t lost() { return dfa3d::kLost; }
"""


@pytest.fixture(scope="module")
def word(tmp_path_factory):
    d = tmp_path_factory.mktemp("lost")
    (d / "lost.cpp").write_text(SOURCE)
    subprocess.run([os.environ.get("CXX", "g++"), "-O1", "-std=c++17", "-shared", "-fPIC", "-I", os.path.join(PKG_DIR, "csrc"),
                    str(d / "lost.cpp"), "-o", str(d / "lost.so")], check=True)
    lib = ctypes.CDLL(str(d / "lost.so"))
    lib.lost.restype = ctypes.c_uint32
    return lib.lost()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_no_column_can_be_taken_for_a_result(word, dtype):
    row = torch.tensor([word] * 16, dtype=torch.uint32).view(dtype)
    assert row.numel() == 64 // row.element_size() and torch.isnan(row).all()
    # nor can what a later product makes of it
    assert torch.isnan(row.float() @ torch.zeros(row.numel()))
