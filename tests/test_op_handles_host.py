"""Handles of ops with one signature (csrc/aten/fused_common.h): each place that
names an op gets that op, whatever was looked up before it."""

import ctypes
import os
import subprocess

import torch
from torch.utils import cpp_extension

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "pytorch-plugin-fl_b200", "csrc")
SOURCE = """
#include "aten/fused_common.h"
using Unary = at::Tensor(const at::Tensor&);
extern "C" int names() {
  const auto name = [](const c10::TypedOperatorHandle<Unary>& op) { return op.operator_name().name; };
  for (int turn = 0; turn < 2; ++turn)
    if (name(FLB_OP(Unary, "aten::neg")) != "aten::neg" || name(FLB_OP(Unary, "aten::abs")) != "aten::abs") return 1;
  return 0;
}
"""


def test_ops_of_one_signature_do_not_share_a_handle(tmp_path):
    src, so = tmp_path / "names.cc", tmp_path / "names.so"
    src.write_text(SOURCE)
    lib = os.path.join(os.path.dirname(torch.__file__), "lib")
    paths = [CSRC, os.path.dirname(os.path.dirname(CSRC)), *cpp_extension.include_paths(), "/usr/local/cuda/include"]
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", *[f"-I{p}" for p in paths], str(src), f"-L{lib}", "-lc10",
                    "-ltorch_cpu", "-o", str(so)], check=True)
    assert ctypes.CDLL(str(so)).names() == 0
