"""Layer norms of several row lengths called by several threads at once, from C so that no interpreter lock orders them."""
import ctypes
import shutil
import subprocess

import pytest
import torch

pytestmark = pytest.mark.gpu

SOURCE = r"""
#include <atomic>
#include <cstdint>
#include <thread>
#include <vector>

typedef int (*layer_norm)(int64_t, int64_t, int, int, float, const void*, int64_t, const void*, const void*, void*, int64_t, float*, float*, void*);
struct call { int64_t rows, d; const void* x; void* y; void* stream; };

extern "C" int64_t run(layer_norm f, int dtype, const call* calls, int n, int times) {
  std::atomic<int64_t> failed{0};
  std::vector<std::thread> threads;
  for (int i = 0; i < n; ++i)
    threads.emplace_back([=, &failed] {
      const call c = calls[i];
      for (int k = 0; k < times; ++k)
        failed += f(c.rows, c.d, dtype, dtype, 1e-5f, c.x, c.d, nullptr, nullptr, c.y, c.d, nullptr, nullptr, c.stream) != 0;
    });
  for (auto& t : threads) t.join();
  return failed;
}
"""


class Call(ctypes.Structure):
    _fields_ = [("rows", ctypes.c_int64), ("d", ctypes.c_int64), ("x", ctypes.c_void_p), ("y", ctypes.c_void_p),
                ("stream", ctypes.c_void_p)]


def test_threads_with_rows_of_several_lengths(built_library, tmp_path):
    """Rows of 3200 and 4096 16-bit elements run in the same kernel with rings of 51 and 66 KB of shared memory: no
    call may set a limit below what another one is about to launch with."""
    if not torch.cuda.is_available():
        pytest.fail("this test needs a CUDA device")
    if shutil.which("g++") is None:
        pytest.skip("needs g++")
    from strassen_triton_b200 import _lib, layer_norm

    (tmp_path / "run.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-O2", "-shared", "-fPIC", "-pthread", "-o", str(tmp_path / "run.so"), str(tmp_path / "run.cpp")],
                   check=True)
    helper = ctypes.CDLL(str(tmp_path / "run.so"))
    helper.run.restype = ctypes.c_int64
    f = ctypes.cast(_lib.load().b200s_layer_norm, ctypes.c_void_p)
    widths = (3200, 4096, 3200, 4096)
    xs = [torch.randn(500, d, device="cuda", dtype=torch.float16) for d in widths]
    want = [layer_norm(x) for x in xs]
    ys = [torch.zeros_like(x) for x in xs]
    streams = [torch.cuda.Stream() for _ in widths]
    torch.cuda.synchronize()
    calls = (Call * len(widths))(*[Call(500, d, x.data_ptr(), y.data_ptr(), s.cuda_stream)
                                   for d, x, y, s in zip(widths, xs, ys, streams)])
    failed = helper.run(f, ctypes.c_int(_lib.FP16), calls, ctypes.c_int(len(widths)), ctypes.c_int(4000))
    torch.cuda.synchronize()
    assert failed == 0, f"{failed} of 16000 launches failed"
    assert all(torch.equal(y, w) for y, w in zip(ys, want))
