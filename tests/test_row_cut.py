"""How rows of any width fall to vectors (csrc/row_cut.hpp), compiled for the host: of every row that the 8-bit integer cast sends to its kernel by
vectors, the whole vectors and the single elements are the row's own, each once."""
import ctypes as C
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent

SOURCE = r"""
#include <vector>
#include "row_cut.hpp"
// The elements that the lanes of a row touch.  Returns 0, or 1 a number of vectors that is none, 2 an element in front of the row or behind it, 3 one left
// out or taken twice.
template <int kV, bool EDGES>
static int row(int64_t r, int64_t cols) {
  const dt::RowCut<kV, EDGES> cut(r, cols);
  if (cut.nvec < 0 || cut.nvec > cols / kV) return 1;
  std::vector<int> taken(cols, 0);
  auto take = [&](int64_t element) {
    if (element < r * cols || element >= (r + 1) * cols) return false;
    ++taken[element - r * cols];
    return true;
  };
  for (int j = 0; j < cut.nvec; ++j)
    for (int i = 0; i < kV; ++i)
      if (!take((cut.vec0 + j) * kV + i)) return 2;
  for (int lane = 0; EDGES && lane < 64; ++lane)
    if (const int edge = cut.edge(lane); edge >= 0 && !take(cut.from * kV + edge)) return 2;
  for (int n : taken)
    if (n != 1) return 3;
  return 0;
}
extern "C" int check(int kV, long cols, long r) {
  if (kV == 4) return cols % 4 ? row<4, true>(r, cols) : row<4, false>(r, cols);
  return cols % 8 ? row<8, true>(r, cols) : row<8, false>(r, cols);
}
extern "C" int in_registers(int base_ok, long cols, int kV) { return dt::int8_rows_in_registers(base_ok != 0, cols, kV); }
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    where = tmp_path_factory.mktemp("row_cut")
    (where / "cut.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-fPIC", "-shared", "-D__HIP_PLATFORM_AMD__=1", "-I/opt/rocm/include", f"-I{ROOT / 'driss_torch_amd' / 'csrc'}",
                    str(where / "cut.cpp"), "-o", str(where / "cut.so")], check=True)
    so = C.CDLL(str(where / "cut.so"))
    so.check.argtypes, so.in_registers.argtypes = [C.c_int, C.c_long, C.c_long], [C.c_int, C.c_long, C.c_int]
    return so


@pytest.mark.parametrize("vec", [4, 8])
def test_rows_by_vectors_are_whole(lib, vec):
    widths = [*range(1, 70), 127, 129, 1001, 8190, 16 * 1024 * vec - 1, 16 * 1024 * vec]
    for cols in widths:
        if lib.in_registers(1, cols, vec):
            for row in (*range(2 * vec + 1), 1 << 20, 2**31 - 2):
                assert lib.check(vec, cols, row) == 0, (cols, row)


@pytest.mark.parametrize("vec", [4, 8])
def test_which_rows_they_are(lib, vec):
    """down to one vector, up to what a workgroup holds, and never off the alignment"""
    assert [cols for cols in range(1, 40) if lib.in_registers(1, cols, vec)] == list(range(vec, 40))
    assert lib.in_registers(1, 16 * 1024 * vec, vec) and not lib.in_registers(1, 16 * 1024 * vec + 1, vec)
    assert not any(lib.in_registers(0, cols, vec) for cols in (1, vec, 1000))


@pytest.mark.parametrize("vec", [4, 8])
def test_shorter_rows_cannot_be_cut(lib, vec):
    """the arithmetic does not hold for them, so they are never sent there"""
    assert any(lib.check(vec, cols, row) for cols in range(1, vec) for row in range(vec))
