"""The rules of csrc/product_rules.h, compiled for the CPU: which kernel takes a product."""
import ctypes
import os
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "h2o4gpu_amd", "csrc")
WAYS = ("few rows", "kept", "any rows", "128", "256")
KINDS = ("forward", "drows", "dweights")
SIZE = {"float32": 4, "bfloat16": 2, "float16": 2}

SOURCE = r"""
#include "product_rules.h"
using namespace kmhip;
extern "C" int part(int size, size_t rows, int experts, size_t out, size_t cols) {
  return rows_of_part(size, rows, experts, out, cols);
}
extern "C" int way(int kind, int size, size_t x, size_t x_stride, size_t w, size_t w_stride, size_t w_expert, int experts,
                   int rows, int n, int k, int part) {
  return way_of(ProductSizes{(Kind)kind, size, (const void *)x, (const void *)w, x_stride, w_stride, w_expert, experts, rows,
                             n, k, part});
}
extern "C" int way_four(int rows, int experts, int out, size_t cols, int gather, size_t x_rows) {
  return way_of_four(rows, experts, out, cols, (cols + 255) / 256 * 128, gather, x_rows);
}
"""


class Rules:
    def __init__(self, where):
        src, so = os.path.join(where, "rules.cpp"), os.path.join(where, "rules.so")
        with open(src, "w") as f:
            f.write(SOURCE)
        subprocess.check_call(["g++", "-std=c++17", "-Wall", "-shared", "-fPIC", "-I" + CSRC, "-o", so, src])
        self.lib = ctypes.CDLL(so)
        t = ctypes.c_size_t
        self.lib.part.argtypes = [ctypes.c_int, t, ctypes.c_int, t, t]
        self.lib.way.argtypes = [ctypes.c_int, ctypes.c_int, t, t, t, t, t] + [ctypes.c_int] * 5
        self.lib.way_four.argtypes = [ctypes.c_int, ctypes.c_int, ctypes.c_int, t, ctypes.c_int, t]

    def part(self, dtype, rows, experts, out, cols):
        return self.lib.part(SIZE[dtype], rows, experts, out, cols)

    def way(self, kind, dtype, rows, experts, out, cols, at=0, apart=None):
        """Of contiguous operands that begin at the address `at`, the matrices `apart` elements apart."""
        size, apart = SIZE[dtype], out * cols if apart is None else apart
        x, n, k, w, apart, part = {"forward": (cols, out, cols, cols, apart, 0), "drows": (out, cols, out, cols, apart, 0),
                                   "dweights": (out, cols, out, cols, 0, self.part(dtype, rows, experts, out, cols))}[kind]
        return WAYS[self.lib.way(KINDS.index(kind), size, at, x, at, w, apart, experts, rows, n, k, part)]

    def way_four(self, rows, out, cols, experts=0, gathered=0):
        """gathered: x's rows, where y's are gathered out of these."""
        return WAYS[self.lib.way_four(rows, experts, out, cols, bool(gathered), gathered or rows)]
