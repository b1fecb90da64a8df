// Shared parts of the paged-cache operators: the device view of a cache, the
// place of a slot, division by a run-time constant, element conversions.
#pragma once

#include <cuda_runtime.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include <initializer_list>
#include <string>

#include "../../include/si_paged.h"
#include "common.cuh"
#include "ctx.h"

namespace si {

// n / d for n below 2^31 by a multiply and a shift (Granlund and Montgomery,
// "Division by invariant integers using multiplication", 1994).
struct FastDiv {
  uint32_t d, mul, shift;
};
inline FastDiv fast_div(uint32_t d) {
  FastDiv f;
  f.d = d;
  f.shift = 0;
  while ((uint64_t(1) << f.shift) < d) ++f.shift;
  f.mul = uint32_t((((uint64_t(1) << f.shift) - d) << 32) / d + 1);
  return f;
}
__host__ __device__ __forceinline__ uint32_t div_of(uint32_t n, const FastDiv& f) {
  const uint32_t hi = uint32_t((uint64_t(n) * f.mul) >> 32);
  return (hi + n) >> f.shift;
}

constexpr uint64_t kNoCell = ~uint64_t(0);

// si_paged_kv as the kernels read it.
struct PagedView {
  const uint16_t* k;
  const uint16_t* v;
  const int32_t* pages;
  uint64_t page_stride, head_stride, token_stride, pages_stride;
  uint32_t num_pages, kv_heads, hd, sequences, max_tokens;
  FastDiv page;  // by page_tokens
};

inline PagedView paged_view(const si_paged_kv& kv) {
  PagedView p;
  p.k = static_cast<const uint16_t*>(kv.k);
  p.v = static_cast<const uint16_t*>(kv.v);
  p.pages = kv.pages;
  p.page_stride = kv.page_stride;
  p.head_stride = kv.head_stride;
  p.token_stride = kv.token_stride;
  p.pages_stride = kv.pages_stride;
  p.num_pages = uint32_t(kv.num_pages);
  p.kv_heads = kv.kv_heads;
  p.hd = kv.head_dim;
  p.sequences = kv.sequences;
  p.max_tokens = kv.max_pages * kv.page_tokens;
  p.page = fast_div(kv.page_tokens);
  return p;
}

// Element offset of (page, token of the page, head) in a pool; kNoCell for a
// page outside it. 64-bit: a pool passes 2^32 elements on this card.
__host__ __device__ __forceinline__ uint64_t paged_cell(const PagedView& kv, int32_t page, uint32_t in_page,
                                                        uint32_t head) {
  if (uint32_t(page) >= kv.num_pages) return kNoCell;  // negative pages too
  return uint64_t(uint32_t(page)) * kv.page_stride + uint64_t(in_page) * kv.token_stride +
         uint64_t(head) * kv.head_stride;
}

// Offset of slot t (below max_tokens) of the sequence whose page-table row is `row`.
__device__ __forceinline__ uint64_t paged_slot(const PagedView& kv, const int32_t* row, uint32_t t, uint32_t head) {
  const uint32_t p = div_of(t, kv.page);
  return paged_cell(kv, __ldg(row + p), t - p * kv.page.d, head);
}

// Cached tokens of a sequence: a length outside [0, most] is reported and clamped.
__device__ __forceinline__ uint32_t checked_length(int32_t n, uint32_t most, int* err) {
  if (n < 0 || uint32_t(n) > most) {
    atomicOr(err, KERR_BAD_INDEX);
    return n < 0 ? 0u : most;
  }
  return uint32_t(n);
}

__host__ __device__ constexpr uint32_t elem_bytes(uint32_t elem) { return elem == SI_ELEM_F32 ? 4u : 2u; }

__device__ __forceinline__ float elem_to_f(uint16_t bits, uint32_t elem) {
  return elem == SI_ELEM_BF16 ? __uint_as_float(uint32_t(bits) << 16) : __half2float(__ushort_as_half(bits));
}
__device__ __forceinline__ uint16_t f_to_elem(float x, uint32_t elem) {
  return elem == SI_ELEM_BF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(x)) : __half_as_ushort(__float2half_rn(x));
}
__device__ __forceinline__ uint32_t pack2_elem(float lo, float hi, uint32_t elem) {
  if (elem == SI_ELEM_BF16) {
    const __nv_bfloat162 r = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  const __half2 r = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&r);
}

// 8 elements from / to element index i of p; `wide`: 16-byte accesses are aligned.
__device__ __forceinline__ void load8(const void* p, uint64_t i, uint32_t elem, bool wide, float x[8]) {
  if (elem == SI_ELEM_F32) {
    const float* f = static_cast<const float*>(p) + i;
    if (wide) {
      const float4 a = *reinterpret_cast<const float4*>(f), b = *reinterpret_cast<const float4*>(f + 4);
      x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = f[j];
    }
    return;
  }
  const uint16_t* h = static_cast<const uint16_t*>(p) + i;
  if (wide) {
    const uint4 a = *reinterpret_cast<const uint4*>(h);
    const uint32_t r[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = elem_to_f(uint16_t(r[j / 2] >> (j % 2 * 16)), elem);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = elem_to_f(h[j], elem);
  }
}
__device__ __forceinline__ void store8(void* p, uint64_t i, uint32_t elem, bool wide, const float x[8]) {
  if (elem == SI_ELEM_F32) {
    float* f = static_cast<float*>(p) + i;
    if (wide) {
      *reinterpret_cast<float4*>(f) = make_float4(x[0], x[1], x[2], x[3]);
      *reinterpret_cast<float4*>(f + 4) = make_float4(x[4], x[5], x[6], x[7]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = x[j];
    }
    return;
  }
  uint16_t* h = static_cast<uint16_t*>(p) + i;
  if (wide) {
    *reinterpret_cast<uint4*>(h) = make_uint4(pack2_elem(x[0], x[1], elem), pack2_elem(x[2], x[3], elem),
                                              pack2_elem(x[4], x[5], elem), pack2_elem(x[6], x[7], elem));
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) h[j] = f_to_elem(x[j], elem);
  }
}

// ---- host side ----
// Checks of a cache description; SI_OK or the status with the text in *msg.
int check_paged_kv(const si_paged_kv* kv, std::string* msg);

// Whether 8 elements starting at any (row, head) of a buffer can be moved with
// 16-byte accesses.
inline bool wide_ok(const void* p, uint32_t elem, uint64_t s0, uint64_t s1) {
  const uint64_t unit = 16 / elem_bytes(elem);
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && s0 % unit == 0 && s1 % unit == 0;
}
inline bool elem_aligned(const void* p, uint32_t elem) { return reinterpret_cast<uintptr_t>(p) % elem_bytes(elem) == 0; }
// Arrays of 32-bit numbers (null ones count as aligned).
inline bool words_aligned(std::initializer_list<const void*> arrays) {
  for (const void* p : arrays)
    if (reinterpret_cast<uintptr_t>(p) % 4) return false;
  return true;
}
// Rows of a call's buffer: [n0][n1][dims], strides and dims in elements.
struct BufferRows {
  const void* p;
  uint64_t n0, s0, n1, s1;
  uint32_t dims, elem;
};
// Whether no element belongs to two rows: every axis steps over all that the
// axes of smaller strides span. (Rows that interleave in no such order count as
// shared; views of one allocation do not.)
bool rows_distinct(const BufferRows& r);
// The same of a cache's pools.
bool pools_distinct(const si_paged_kv& kv);
// Whether any element is in both buffers, of one element type. Exact where the
// strides are the same (parts of one buffer); otherwise buffers whose ranges
// overlap count as sharing.
bool rows_meet(const BufferRows& a, const BufferRows& b);
inline bool elem_known(uint32_t elem) { return elem <= SI_ELEM_F16; }

// Makes the context's device current for the launches of one call.
struct DeviceGuard {
  int before = -1;
  bool moved = false;
  cudaError_t e;
  explicit DeviceGuard(int device) {
    e = cudaGetDevice(&before);
    if (e == cudaSuccess && before != device) {
      e = cudaSetDevice(device);
      moved = e == cudaSuccess;
    }
  }
  ~DeviceGuard() {
    if (moved) cudaSetDevice(before);
  }
};

// Launch configuration with programmatic dependent launch: the kernel's
// prologue overlaps the end of the one before it in the stream, and it waits
// (griddepcontrol.wait) before it reads anything.
struct PdlLaunch {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  PdlLaunch(dim3 grid, dim3 block, size_t smem, cudaStream_t s) {
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
  }
  void cluster(uint32_t n) {
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = n;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.numAttrs = 2;
  }
};

}  // namespace si
