"""Which 16-byte words the span softmax's gradient reads of a row of y and dy:
none that holds nothing of the row, since that one may lie outside its memory.
The kernels' own arithmetic (csrc/b200/span_place.cuh), compiled for the host."""

import ctypes
import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "pytorch-plugin-fl_b200", "csrc",
                    "b200")
SOURCE = """
#include "span_place.cuh"
// The first element of each word that a row's lanes read, relative to the row.
template <int N>
int words(int vw, int shift, int lo, int hi, int cols, int* out) {
  const flb200::Packs<N> p(lo, hi, shift, cols);
  int n = 0;
  for (int v = 0; v < p.count; ++v)
    for (int k = 0; k < N / vw; ++k)
      if (N == vw || p.meets((p.p0 + v) * N + k * vw, vw)) out[n++] = (p.p0 + v) * N + k * vw - p.first;
  return n;
}
extern "C" int words_of(int n, int vw, int shift, int lo, int hi, int cols, int* out) {
  return n == 4 ? words<4>(vw, shift, lo, hi, cols, out) : words<8>(vw, shift, lo, hi, cols, out);
}
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("place")
    src, so = d / "words.cc", d / "words.so"
    src.write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-I", CSRC, "-x", "c++", str(src), "-o", str(so)], check=True)
    return ctypes.CDLL(str(so))


@pytest.mark.parametrize("pack,word", [(8, 4), (8, 8), (4, 4)])
def test_words_read_hold_something_of_the_span(lib, pack, word):
    """Every span of rows of 0 to 21 elements that begin anywhere in a pack:
    each word read holds an element of the span, and they hold all of it."""
    out = (ctypes.c_int * 64)()
    for shift in range(pack):
        for cols in range(22):
            for lo in range(cols + 1):
                for hi in range(lo, cols + 1):
                    n = lib.words_of(pack, word, shift, lo, hi, cols, out)
                    got = [e for o in out[:n] for e in range(o, o + word)]
                    assert all((o + shift) % word == 0 for o in out[:n])
                    assert all(any(lo <= e < hi for e in range(o, o + word)) for o in out[:n]), (shift, cols, lo, hi)
                    assert len(got) == len(set(got)) and set(range(lo, hi)) <= set(got)
