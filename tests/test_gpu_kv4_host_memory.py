"""Host memory that runs out inside a cache operator comes back as a status: a C++ program with an
operator new that fails on demand makes the calls. Nothing reaches the GPU from a failing call."""
import os
import shutil
import subprocess

import pytest

import busfill_b200 as bf

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SOURCE = r"""
#include <cstdio>
#include <cstdlib>
#include <new>
#include <vector>
#include <cuda_runtime.h>
#include "busfill.h"

static bool fail = false;
void* operator new(std::size_t n) {
  if (fail) throw std::bad_alloc();
  if (void* p = std::malloc(n ? n : 1)) return p;
  throw std::bad_alloc();
}
void operator delete(void* p) noexcept { std::free(p); }
void operator delete(void* p, std::size_t) noexcept { std::free(p); }

int main() {
  const int D = 64;
  void* mem = nullptr;
  if (cudaMalloc(&mem, 1 << 20) != cudaSuccess || cudaMemset(mem, 0, 1 << 20) != cudaSuccess) return 2;
  char* at = static_cast<char*>(mem);
  const int one = 1;   // cached token
  if (cudaMemcpy(at + 66048, &one, sizeof(one), cudaMemcpyHostToDevice) != cudaSuccess) return 2;
  busfill_kv4 c{};
  c.pages = reinterpret_cast<uint8_t*>(at), c.table = reinterpret_cast<int32_t*>(at + 65536);
  c.kv_len = reinterpret_cast<int32_t*>(at + 66048);
  c.num_pages = 1, c.table_cols = 1, c.batch = 1, c.heads = 1, c.head_dim = D;
  busfill_kv4_rows r{};
  r.k = at + 131072, r.v = at + 131072, r.k_token = r.v_token = D, r.tokens = 1, r.dtype = BUSFILL_TYPE_F16;
  busfill_attn a{};
  a.q = at + 131072, a.out = at + 262144, a.q_token = a.out_token = D, a.q_head = a.out_head = D;
  a.scale = 1.0f, a.tokens = 1, a.q_heads = 1, a.max_q = 1, a.causal = 1, a.dtype = BUSFILL_TYPE_F16;
  cudaStream_t s;
  if (cudaStreamCreateWithFlags(&s, cudaStreamNonBlocking) != cudaSuccess) return 2;
  int st[6];
  // a stream's first call makes its error words
  fail = true;
  st[0] = busfill_kv4_append(&c, &r, s);
  fail = false;
  st[1] = busfill_kv4_append(&c, &r, s);
  // its first attention makes the workspace
  fail = true;
  st[2] = busfill_attn_kv4(&c, &a, s);
  fail = false;
  st[3] = busfill_attn_kv4(&c, &a, s);
  // a capture makes one of its own
  cudaGraph_t graph = nullptr;
  if (cudaStreamBeginCapture(s, cudaStreamCaptureModeGlobal) != cudaSuccess) return 2;
  fail = true;
  st[4] = busfill_attn_kv4(&c, &a, s);
  fail = false;
  st[5] = busfill_attn_kv4(&c, &a, s);
  if (cudaStreamEndCapture(s, &graph) != cudaSuccess) return 3;
  std::printf("%d %d %d %d %d %d %d\n", st[0], st[1], st[2], st[3], st[4], st[5], busfill_stream_status(s));
  return 0;
}
"""


def test_host_memory_that_runs_out_is_a_status(tmp_path):
    cxx = shutil.which("g++")
    cuda = os.path.dirname(os.path.dirname(shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"))
    if cxx is None or not os.path.isdir(cuda):
        pytest.skip("no host C++ compiler or CUDA headers")
    src, exe = tmp_path / "calls.cpp", tmp_path / "calls"
    src.write_text(SOURCE)
    lib = os.path.abspath(bf.library_path())
    subprocess.run([cxx, "-std=c++17", "-I", os.path.join(ROOT, "include"), "-I", os.path.join(cuda, "include"), str(src),
                    "-o", str(exe), lib, "-L", os.path.join(cuda, "lib64"), "-lcudart",
                    f"-Wl,-rpath,{os.path.dirname(lib)}"], check=True)
    res = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert res.returncode == 0, (res.returncode, res.stderr)
    assert res.stdout.split() == ["-6", "0", "-6", "0", "-6", "0", "0"]
