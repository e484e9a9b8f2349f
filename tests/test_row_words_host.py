"""Which words the RMS norm's shifted-word rows touch: the address arithmetic
of rownorm.cu's Words::fetch run on the host, over sizes, strides and
alignments, with the rule of row_words.cuh.  Every word that an inner row reads
lies wholly inside its matrix."""
import ctypes
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SOURCE = r"""
#include "row_words.cuh"
// words outside a [rows, cols] matrix, `ld` elements of `es` bytes apart, that
// starts `base` bytes after a 16-byte boundary; edge 0: edge_rows(ld)
extern "C" int64_t outside(uint64_t rows, uint32_t cols, uint64_t ld, uint32_t es, uint32_t base,
                           uint32_t edge) {
  const int64_t lo = 1024 + base, hi = lo + (int64_t)(((rows - 1) * ld + cols) * es);
  int64_t bad = 0;
  if (edge == 0) edge = edge_rows(ld);
  for (uint64_t row = 0; row < rows; row++) {
    if (!inner_row(row, rows, edge)) continue;
    for (uint32_t c = 0; c < cols; c += 8) {
      const int64_t p = lo + (int64_t)((row * ld + c) * es);
      const int64_t first = p - p % 16;
      for (uint32_t k = 0; k < 8 * es / 16 + 1; k++)
        bad += first + 16 * k < lo || first + 16 * k + 16 > hi;
    }
  }
  return bad;
}
extern "C" uint64_t inner_rows(uint64_t rows, uint64_t ld) {
  uint64_t n = 0;
  for (uint64_t row = 0; row < rows; row++) n += inner_row(row, rows, edge_rows(ld));
  return n;
}
"""


@pytest.fixture(scope="module")
def words(tmp_path_factory):
    d = tmp_path_factory.mktemp("words")
    (d / "words.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-O2", "-shared", "-fPIC", "-std=c++17", "-I",
                    os.path.join(ROOT, "browsergnn_b200", "csrc"), "-o", str(d / "words.so"),
                    str(d / "words.cpp")], check=True)
    lib = ctypes.CDLL(str(d / "words.so"))
    lib.outside.restype = ctypes.c_int64
    lib.outside.argtypes = [ctypes.c_uint64, ctypes.c_uint32, ctypes.c_uint64] + \
        [ctypes.c_uint32] * 3
    lib.inner_rows.restype = ctypes.c_uint64
    lib.inner_rows.argtypes = [ctypes.c_uint64, ctypes.c_uint64]
    return lib


@pytest.mark.parametrize("es", [2, 4])
def test_no_word_of_an_inner_row_leaves_the_matrix(words, es):
    for cols in list(range(1, 34)) + [47, 63, 100, 1433]:
        for ld in {cols, cols + 1, cols + 3, cols + 7, cols + 8, 2 * cols}:
            for rows in list(range(1, 36)) + [1000]:
                for base in range(0, 16, es):
                    assert words.outside(rows, cols, ld, es, base, 0) == 0, (rows, cols, ld, base)


def test_one_row_at_either_end_is_too_few_for_narrow_rows(words):
    # f32 [1000, 4]: the third word of row 998 begins where the matrix ends
    assert words.outside(1000, 4, 4, 4, 0, 1) > 0
    assert words.outside(1000, 1, 1, 2, 0, 1) > 0


def test_wide_rows_keep_their_fast_path(words):
    for ld in (15, 16, 47, 1433):
        assert words.inner_rows(1000, ld) == 998
    assert words.inner_rows(1000, 1) == 970 and words.inner_rows(20, 1) == 0
