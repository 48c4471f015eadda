// The pages of a cache as the kernels see them, and what the entries on them share.
#pragma once
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "handles.h"

namespace turq {

struct KvPages {
  uint8_t *k = nullptr, *v = nullptr;  // [n_pages, n_heads, page_size, head_dim]
  __half *ks = nullptr, *vs = nullptr; // Q8_0: [n_pages, n_heads, page_size, head_dim / 32]
  int64_t n_pages = 0;
  int n_heads = 0, page_size = 0, page_shift = 0, dtype = 0;
  // Row of the planes that holds one head of a slot; 64 bits, since a long cache has more elements than 32.
  __host__ __device__ int64_t row(int64_t slot, int head) const {
    return (((slot >> page_shift) * n_heads + head) << page_shift) + (slot & (page_size - 1));
  }
};

inline KvPages pages_of(const turq_kv_cache* c) {
  KvPages p;
  p.k = c->mem;
  p.v = c->mem + c->off_v;
  if (c->off_vs != c->off_ks) {
    p.ks = reinterpret_cast<__half*>(c->mem + c->off_ks);
    p.vs = reinterpret_cast<__half*>(c->mem + c->off_vs);
  }
  p.n_pages = c->n_pages;
  p.n_heads = c->n_kv_heads;
  p.page_size = c->page_size;
  while ((1 << p.page_shift) < c->page_size) p.page_shift++;
  p.dtype = c->dtype;
  return p;
}

// The context's device for the length of a call; the caller's current device afterwards.
struct DeviceScope {
  int before = -1;
  cudaError_t status;
  explicit DeviceScope(int device) {
    status = cudaGetDevice(&before);
    if (status == cudaSuccess && before != device) status = cudaSetDevice(device);
    else before = -1;
  }
  ~DeviceScope() {
    if (before >= 0) cudaSetDevice(before);
  }
  DeviceScope(const DeviceScope&) = delete;
  DeviceScope& operator=(const DeviceScope&) = delete;
};

}  // namespace turq
