"""What the products' entry points write into their workspace, compiled for the host with launches that only record their arguments: all of it lies inside
the length that was checked, also where the knobs mm.tiles and mm.splits change between any two times that a call reads them."""
import ctypes as C
import itertools
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent

SOURCE = r"""
#include <map>
#include <string>
#include <vector>
#include "dt_host.hpp"
namespace dt {
std::atomic<int> g_knob_values[(int)Knob::count];
const DeviceFacts& device_facts() {
  static const DeviceFacts facts{256};
  return facts;
}
static std::vector<int> g_splits;  // what the reads of mm.splits give, one after the other, the last again and again
static size_t g_read;
static int read_knob(Knob k) {
  if (k == Knob::mm_tiles) return 3;  // 64 x 128
  return g_splits[g_read < g_splits.size() ? g_read++ : g_splits.size() - 1];
}
}  // namespace dt
#define tuning(k) read_knob(k)
#include "gated_linear.hip"
#include "int8_bf16.hip"

static std::map<const void*, std::string> g_names;
static uintptr_t g_end;
static int g_outside, g_launches, g_too_large;
extern "C" {
void** __hipRegisterFatBinary(const void*) { static void* handle; return &handle; }
void __hipUnregisterFatBinary(void**) {}
void __hipRegisterFunction(void**, const void* host, char*, const char* name, unsigned, void*, void*, void*, void*, int*) { g_names[host] = name; }
hipError_t __hipPopCallConfiguration(dim3*, dim3*, size_t*, hipStream_t*) { return hipSuccess; }
hipError_t hipFuncSetAttribute(const void*, hipFuncAttribute, int) { return hipSuccess; }
hipError_t hipGetDevice(int* device) { *device = 0; return hipSuccess; }
hipError_t hipGetLastError() { return hipSuccess; }
hipError_t hipLaunchKernel(const void* kernel, dim3 grid, dim3 block, void** args, size_t, hipStream_t) {
  ++g_launches;
  g_too_large += (uint64_t)grid.x * block.x > 0xFFFFFFFFull;
  const std::string& name = g_names[kernel];
  auto ends = [](uintptr_t end) { g_outside += end > g_end; };
  if (name.find("mm_small_kernel") != std::string::npos || name.find("mm_join_kernel") != std::string::npos) {
    const auto& a = *static_cast<const dt::MmSmallArgs*>(args[0]);
    if (a.splits > 1) ends((uintptr_t)a.sums + (size_t)a.splits * a.t.tiles_m * a.t.tiles_n * 64 * 128 * 4);
  } else if (name.find("mm_pack_kernel") != std::string::npos) {
    for (const dt::MmPackJob& j : static_cast<const dt::MmPackJobs*>(args[0])->job) ends((uintptr_t)j.to + j.rows * ((j.bytes + 15) / 16 * 16));
  }
  return hipSuccess;
}
// -1: a launch wrote past `bytes`, -3: one had more threads than the runtime takes; otherwise the call's status.  what: 0 gated_linear, 1 its gradients, 2 int8_bf16
int call(int what, const int* splits, int n, long T, long D, long F, size_t bytes) {
  dt::g_splits.assign(splits, splits + n);
  dt::g_read = 0;
  g_outside = g_launches = g_too_large = 0;
  uint8_t* const p = reinterpret_cast<uint8_t*>((uintptr_t)1 << 40);
  void* const ws = reinterpret_cast<void*>((uintptr_t)1 << 44);
  g_end = ((uintptr_t)1 << 44) + bytes;
  int status;
  if (what == 0) status = dt_gated_linear(p, p, p, T, D, F, D, D, D, 0, p, nullptr, nullptr, ws, bytes, nullptr);
  else if (what == 1) status = dt_gated_linear_backward(p, p, p, p, p, p, T, D, F, D, D, D, 0, p, p, p, ws, bytes, nullptr);
  else status = dt_int8_bf16(p, p, (const float*)p, (const float*)p, T, F, D, D, D, p, F, ws, bytes, nullptr);
  if (g_outside) return -1;
  if (g_too_large) return -3;
  return status == 0 && g_launches == 0 ? -2 : status;
}
size_t bytes(int what, int splits, long T, long D, long F) {
  dt::g_splits = {splits};
  dt::g_read = 0;
  const void* const p = reinterpret_cast<const void*>((uintptr_t)1 << 40);
  if (what == 0) return dt_gated_linear_workspace_bytes(p, p, p, T, D, F, D, D, D);
  if (what == 1) return dt_gated_linear_backward_workspace_bytes(p, p, p, T, D, F, D, D, D);
  return dt_int8_bf16_workspace_bytes(p, p, T, F, D, D, D);
}
}
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    where = tmp_path_factory.mktemp("mm_workspace")
    (where / "calls.hip").write_text(SOURCE)
    includes = [f"-I{ROOT / 'include'}", f"-I{ROOT / 'driss_torch_amd' / 'csrc'}"]
    subprocess.run(["/opt/rocm/bin/hipcc", "--offload-host-only", "--offload-arch=gfx950", "-O0", "-std=c++17", "-fPIC", "-w", *includes, "-c", str(where / "calls.hip"), "-o",
                    str(where / "calls.o")], check=True)
    # (the device code that there is none of)
    undefined = subprocess.run(["nm", "-u", str(where / "calls.o")], check=True, capture_output=True, text=True).stdout.split()
    (where / "none.c").write_text("".join(f"const char {name}[64];\n" for name in undefined if name.startswith("__hip_fatbin")))
    subprocess.run(["gcc", "-fPIC", "-c", str(where / "none.c"), "-o", str(where / "none.o")], check=True)
    subprocess.run(["g++", "-shared", "-Wl,-Bsymbolic", str(where / "calls.o"), str(where / "none.o"), "-o", str(where / "calls.so")], check=True)
    so = C.CDLL(str(where / "calls.so"))
    so.bytes.argtypes, so.bytes.restype = [C.c_int, C.c_int, C.c_long, C.c_long, C.c_long], C.c_size_t
    so.call.argtypes = [C.c_int, C.POINTER(C.c_int), C.c_int, C.c_long, C.c_long, C.c_long, C.c_size_t]
    return so


@pytest.mark.parametrize("size", [(100, 1024, 256), (70, 1001, 301)], ids=["words", "copies"])
@pytest.mark.parametrize("what", [0, 1, 2], ids=["gated_linear", "gradients", "int8_bf16"])
def test_all_writes_are_inside(lib, what, size):
    few, many = lib.bytes(what, 1, *size), lib.bytes(what, 4, *size)
    assert many > few
    for given in (few, many - 1, many):
        for reads in itertools.product([1, 4], repeat=6):
            status = lib.call(what, (C.c_int * 6)(*reads), 6, *size, given)
            assert status in (0, 5), (given, reads, status)  # done, or the workspace refused
            if len(set(reads)) == 1:
                assert status == (0 if reads[0] == 1 or given == many else 5)


def test_more_threads_than_a_launch_has(lib):
    """2^24 tiles of 64 rows, 2^32 threads, which the runtime would cut short: an error of the call, and the next call is not affected"""
    splits = (C.c_int * 1)(1)
    assert lib.call(2, splits, 1, (1 << 30) - 1, 4, 1, 1 << 62) == 7
    assert lib.call(2, splits, 1, (1 << 30) - 64, 4, 1, 1 << 62) == 0
    assert lib.call(0, splits, 1, (1 << 30) - 1, 2, 2, 1 << 62) == 7
    assert lib.call(0, splits, 1, 100, 64, 64, 1 << 62) == 0
