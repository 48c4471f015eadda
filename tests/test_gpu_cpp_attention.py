"""turq::rope_table, qk_norm_rope and KvCache (include/turq.hpp): a C++ program of its own gives the bits that the Python calls give."""
import os
import subprocess

import numpy as np
import pytest
import torch

import tur_b200 as tq
from tur_b200.build import OUT

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CUDA = "/usr/local/cuda"
PROGRAM = r"""
#include <cuda_runtime.h>
#include <cstdio>
#include <vector>
#include "turq.hpp"
static FILE *in, *out;
template <class T> T* from_file(size_t n) {
  std::vector<T> h(n);
  if (std::fread(h.data(), sizeof(T), n, in) != n) throw std::runtime_error("short input");
  T* d = nullptr;
  cudaMalloc(&d, n * sizeof(T));
  cudaMemcpy(d, h.data(), n * sizeof(T), cudaMemcpyHostToDevice);
  return d;
}
template <class T> T* room(size_t n) {
  T* d = nullptr;
  cudaMalloc(&d, n * sizeof(T));
  return d;
}
template <class T> void to_file(const T* d, size_t n) {
  std::vector<T> h(n);
  cudaMemcpy(h.data(), d, n * sizeof(T), cudaMemcpyDeviceToHost);
  std::fwrite(h.data(), sizeof(T), n, out);
}
int main(int, char** argv) {
  in = std::fopen(argv[1], "rb");
  out = std::fopen(argv[2], "wb");
  const int n = 150, hq = 8, hkv = 2, d = 64, pages = 12, page = 16;
  try {
    auto ctx = std::make_shared<turq::Context>(0);
    const float *q = from_file<float>(n * hq * d), *k = from_file<float>(n * hkv * d), *v = from_file<float>(n * hkv * d);
    const float *wq = from_file<float>(d), *wk = from_file<float>(d);
    const int32_t *pos = from_file<int32_t>(n), *starts = from_file<int32_t>(2), *contexts = from_file<int32_t>(1), *table = from_file<int32_t>(10);
    const int64_t* slots = from_file<int64_t>(n);
    std::vector<double> freqs(d / 2);
    if (std::fread(freqs.data(), 8, freqs.size(), in) != freqs.size()) return 3;
    float* angles = room<float>(n * d);
    turq::rope_table(*ctx, freqs, n, angles);
    turq::Rotary rotary;
    rotary.dev_table = angles; rotary.n_positions = n; rotary.rotary_dim = d;
    const turq::HeadRows rq{q, hq * d}, rk{k, hkv * d}, rv{v, hkv * d};
    float *qo = room<float>(n * hq * d), *ko = room<float>(n * hkv * d), *kr = room<float>(n * hkv * d), *vr = room<float>(n * hkv * d);
    turq::qk_norm_rope(*ctx, rq, rk, turq::GgmlDType::F32, n, hq, hkv, d, wq, wk, 1e-6f, rotary, pos, turq::GgmlDType::F32, qo, ko);
    to_file(qo, n * hq * d);
    to_file(ko, n * hkv * d);
    turq::KvCache a(ctx, turq::GgmlDType::Q8_0, pages, page, hkv, d), b(ctx, turq::GgmlDType::Q8_0, pages, page, hkv, d);
    uint16_t *qh = room<uint16_t>(n * hq * d), *y = room<uint16_t>(n * hq * d);
    a.append(rq, rk, rv, turq::GgmlDType::F32, n, hq, wq, wk, 1e-6f, rotary, pos, slots, turq::GgmlDType::F16, qh);
    b.write(turq::HeadRows{ko, hkv * d}, rv, turq::GgmlDType::F32, n, slots);
    for (auto* c : {&a, &b}) {
      c->read(slots, n, turq::GgmlDType::F32, kr, vr);
      to_file(kr, n * hkv * d);
      to_file(vr, n * hkv * d);
    }
    turq::KvCache::Batch batch;
    batch.dev_starts = starts; batch.dev_contexts = contexts; batch.dev_page_table = table;
    batch.table_stride = 10; batch.n_seqs = 1; batch.n_tokens = n; batch.max_new = n; batch.max_context = n;
    const size_t bytes = a.workspace(batch, hq);
    void* ws = bytes ? room<uint8_t>(bytes) : nullptr;
    a.attend(turq::HeadRows{qh, hq * d}, turq::GgmlDType::F16, hq, batch, 0.125f, true, turq::GgmlDType::F16, y, ws, bytes);
    to_file(y, n * hq * d);
    try {
      turq::KvCache bad(ctx, turq::GgmlDType::Q8_0, pages, 17, hkv, d);
      return 4;
    } catch (const turq::Error& e) {
      if (e.status != TURQ_E_SHAPE) return 5;
    }
  } catch (const std::exception& e) {
    std::printf("%s\n", e.what());
    return 2;
  }
  std::fclose(out);
  return cudaDeviceSynchronize() == cudaSuccess ? 0 : 6;
}
"""


def test_the_cpp_classes_give_the_same_bits(tmp_path):
    src, exe = str(tmp_path / "t.cpp"), str(tmp_path / "t")
    with open(src, "w") as f:
        f.write(PROGRAM)
    libdir = os.path.dirname(OUT)
    subprocess.run(["g++", "-std=c++17", "-I", os.path.join(ROOT, "include"), "-I", f"{CUDA}/include", src, "-o", exe, "-L", libdir, "-lturq",
                    f"-Wl,-rpath,{libdir}", "-L", f"{CUDA}/lib64", f"-Wl,-rpath,{CUDA}/lib64", "-lcudart"], check=True)
    n, hq, hkv, d, page = 150, 8, 2, 64, 16
    g = torch.Generator(device="cuda").manual_seed(3)
    q, k, v = (torch.randn(n, h, d, device="cuda", generator=g) for h in (hq, hkv, hkv))
    wq, wk = (1 + 0.2 * torch.randn(d, device="cuda", generator=g) for _ in range(2))
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    starts, contexts = (torch.tensor(t, dtype=torch.int32, device="cuda") for t in ([0, n], [n]))
    table = torch.randperm(12, device="cuda", generator=g)[:10].to(torch.int32)
    slots = table.long()[pos.long() // page] * page + pos.long() % page
    freqs = np.array([1e4 ** (-2.0 * i / d) for i in range(d // 2)])
    path, result = tmp_path / "in", tmp_path / "out"
    path.write_bytes(b"".join(t.cpu().numpy().tobytes() for t in (q, k, v, wq, wk, pos, starts, contexts, table, slots)) + freqs.tobytes())
    run = subprocess.run([exe, str(path), str(result)], capture_output=True, text=True, timeout=120)
    assert run.returncode == 0, (run.returncode, run.stdout, run.stderr)
    rotary = tq.RotaryTable.from_frequencies(freqs.tolist(), n)
    want = list(tq.qk_norm_rope(q, k, pos, rotary, q_weight=wq, k_weight=wk))
    cache = tq.KvCache.new(tq.GgmlDType.Q8_0, 12, page, hkv, d)
    qh = cache.append(q, k, v, pos, rotary, slots, q_weight=wq, k_weight=wk, out_dtype=torch.float16)
    want += 2 * list(cache.read(slots)) + [cache.attend(qh, starts, contexts, table[None], max_new=n, max_context=n, scale=0.125)]
    assert result.read_bytes() == b"".join(t.cpu().numpy().tobytes() for t in want)
    tq.context().poll_status()
