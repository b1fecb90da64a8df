// Verification of drafted tokens by probabilities, with given random numbers.
//
// Draft x of place i is accepted while u_i q_i(x) < p_i(x); the next token is
// the lowest j whose cumulative weight passes u times the total, the weights
// being max(p - q, 0) of the first rejected place or the last row of p. Only
// one row of p and q a sequence is read whole, so the work is bound by its bytes
// (8 a token of the vocabulary) at large batches and by latency at small ones.
//
// The choice among 250,000 neighbouring borders has to be that of exact
// arithmetic: an f32 sum would move a border now and then. Differences are
// formed and summed in f64; two sums of different order differ by 1e-16, so
// they choose differently about once in 10^10 draws.
//
// Two kernels: every CTA of the first decides the sequence's accepted count for
// itself (a few loads) and sums one chunk of the row; one CTA a sequence of the second
// scans the chunk sums, finds the chunk that the draw falls in, and scans
// that chunk. The row is read once, one chunk of it twice.
#include <cuda_runtime.h>

#include <algorithm>

#include "paged.cuh"

namespace si {
namespace {

constexpr uint32_t kThreads = 256, kEach = 16, kChunk = kThreads * kEach;  // tokens of a chunk
constexpr uint32_t kPickThreads = 1024;

struct VerifyArgs {
  const float *p, *q;
  uint64_t p_ss, p_rs, q_ss, q_rs;
  const int32_t *tokens, *counts;
  const float *u, *u_last;
  int32_t *accepted, *next;
  uint32_t drafts, vocab, chunks;
  double2* sums;  // [sequence][chunk]: of the difference, of the target's row
  int* err;
};

__device__ __forceinline__ double weight_of(float x) {
  return x > 0.f && x < INFINITY ? double(x) : 0.0;  // NaN compares false
}

// The row that the next token is drawn from.
struct Rest {
  const float* p;
  const float* q;     // null: nothing is taken away
  uint32_t without;   // this token's weight is taken away; >= vocab: none
  __device__ __forceinline__ double at(uint32_t j, double* plain) const {
    const double x = weight_of(p[j]);
    *plain = x;
    if (q) return fmax(x - weight_of(q[j]), 0.0);
    return j == without ? 0.0 : x;
  }
};

// Drafts of sequence b, within bounds.
__device__ __forceinline__ uint32_t drafts_of(const VerifyArgs& a, uint32_t b) {
  if (!a.counts) return a.drafts;
  const int32_t n = a.counts[b];
  if (n < 0 || uint32_t(n) > a.drafts) {
    atomicOr(a.err, KERR_BAD_INDEX);
    return n < 0 ? 0u : a.drafts;
  }
  return uint32_t(n);
}

// Accepted drafts of sequence b, by one warp: a lane a draft.
__device__ __forceinline__ uint32_t accepted_of(const VerifyArgs& a, uint32_t b, uint32_t lane) {
  const uint32_t n = drafts_of(a, b);
  bool ok = false;
  if (lane < n) {
    const int32_t x = a.tokens[uint64_t(b) * a.drafts + lane];
    if (uint32_t(x) < a.vocab) {
      const double p = weight_of(a.p[b * a.p_ss + lane * a.p_rs + uint32_t(x)]);
      const double q = a.q ? weight_of(a.q[b * a.q_ss + lane * a.q_rs + uint32_t(x)]) : 1.0;
      ok = double(a.u[uint64_t(b) * a.drafts + lane]) * q < p;  // exact: 24 + 24 bits
    } else {
      atomicOr(a.err, KERR_BAD_INDEX);
    }
  }
  return __ffs(~__ballot_sync(0xffffffffu, ok)) == 0 ? 32u : uint32_t(__ffs(~__ballot_sync(0xffffffffu, ok)) - 1);
}

__device__ __forceinline__ Rest rest_of(const VerifyArgs& a, uint32_t b, uint32_t taken) {
  Rest r;
  r.p = a.p + b * a.p_ss + taken * a.p_rs;
  r.q = nullptr;
  r.without = 0xffffffffu;
  const int32_t n = a.counts ? a.counts[b] : int32_t(a.drafts);
  const uint32_t drafts = n < 0 ? 0u : min(uint32_t(n), a.drafts);
  if (taken < drafts) {
    if (a.q) r.q = a.q + b * a.q_ss + taken * a.q_rs;
    else r.without = uint32_t(a.tokens[uint64_t(b) * a.drafts + taken]);
  }
  return r;
}

__global__ void __launch_bounds__(kThreads) verify_sum_kernel(const __grid_constant__ VerifyArgs a) {
  __shared__ uint32_t s_taken;
  __shared__ double2 s_sum[kThreads / 32];
  const uint32_t b = blockIdx.y, lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  pdl_launch_dependents();
  pdl_wait();
  if (w == 0) {
    const uint32_t taken = accepted_of(a, b, lane);
    if (lane == 0) {
      s_taken = taken;
      if (blockIdx.x == 0) a.accepted[b] = int32_t(taken);
    }
  }
  __syncthreads();
  const Rest r = rest_of(a, b, s_taken);
  for (uint32_t c = blockIdx.x; c < a.chunks; c += gridDim.x) {
    const uint32_t j0 = c * kChunk + threadIdx.x;
    float x[kEach], y[kEach];
#pragma unroll
    for (uint32_t i = 0; i < kEach; ++i) {
      const uint32_t j = j0 + i * kThreads;
      x[i] = j < a.vocab ? __ldg(r.p + j) : 0.f;
      y[i] = r.q && j < a.vocab ? __ldg(r.q + j) : 0.f;
    }
    double2 s = {0.0, 0.0};
#pragma unroll
    for (uint32_t i = 0; i < kEach; ++i) {
      const double p = weight_of(x[i]);
      s.y += p;
      s.x += j0 + i * kThreads == r.without ? 0.0 : fmax(p - weight_of(y[i]), 0.0);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      s.x += __shfl_xor_sync(0xffffffffu, s.x, o);
      s.y += __shfl_xor_sync(0xffffffffu, s.y, o);
    }
    if (lane == 0) s_sum[w] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (uint32_t i = 1; i < kThreads / 32; ++i) {
        s.x += s_sum[i].x;
        s.y += s_sum[i].y;
      }
      a.sums[uint64_t(b) * a.chunks + c] = s;
    }
    __syncthreads();
  }
}

// Inclusive prefix of one value a thread over kPickThreads threads.
__device__ __forceinline__ double pick_prefix(double v, double* s_w, double* total) {
  const uint32_t lane = threadIdx.x & 31, w = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= uint32_t(o)) v += y;
  }
  __syncthreads();
  if (lane == 31) s_w[w] = v;
  __syncthreads();
  double y = s_w[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double z = __shfl_up_sync(0xffffffffu, y, o);
    if (lane >= uint32_t(o)) y += z;
  }
  *total = __shfl_sync(0xffffffffu, y, 31);
  const double before = __shfl_sync(0xffffffffu, y, w ? w - 1 : 0);
  return w ? before + v : v;
}

__global__ void __launch_bounds__(kPickThreads) verify_pick_kernel(const __grid_constant__ VerifyArgs a) {
  __shared__ double s_w[32], s_base;
  __shared__ uint32_t s_pick, s_last;
  const uint32_t b = blockIdx.x, tid = threadIdx.x;
  if (tid == 0) s_pick = 0xffffffffu, s_last = 0xffffffffu, s_base = 0.0;
  pdl_launch_dependents();
  pdl_wait();
  const uint32_t taken = uint32_t(a.accepted[b]);
  Rest r = rest_of(a, b, taken);
  const double2* sums = a.sums + uint64_t(b) * a.chunks;
  // totals; where the difference is nothing, the target's row itself
  double total = 0.0, plain = 0.0, t;
  for (uint32_t c0 = 0; c0 < a.chunks; c0 += kPickThreads) {
    const double2 s = c0 + tid < a.chunks ? sums[c0 + tid] : make_double2(0.0, 0.0);
    pick_prefix(s.x, s_w, &t);
    total += t;
    pick_prefix(s.y, s_w, &t);
    plain += t;
  }
  const bool whole = !(total > 0.0);
  if (whole) {
    total = plain;
    r.q = nullptr;
    r.without = 0xffffffffu;
  }
  if (!(total > 0.0)) {
    if (tid == 0) a.next[b] = -1;
    return;
  }
  const double goal = double(a.u_last[b]) * total;
  // the first chunk whose end passes the goal; rounding may leave none: the last one with any weight
  double run = 0.0;
  for (uint32_t c0 = 0; c0 < a.chunks; c0 += kPickThreads) {
    const double2 s = c0 + tid < a.chunks ? sums[c0 + tid] : make_double2(0.0, 0.0);
    const double v = whole ? s.y : s.x, end = run + pick_prefix(v, s_w, &t);
    if (v > 0.0) {
      if (end > goal) atomicMin(&s_pick, c0 + tid);
      atomicMax(reinterpret_cast<int*>(&s_last), int(c0 + tid));
    }
    __syncthreads();
    if (s_pick == c0 + tid || (s_pick == 0xffffffffu && s_last == c0 + tid)) s_base = end - v;
    run += t;
    if (s_pick != 0xffffffffu) break;  // the same for all threads
  }
  __syncthreads();
  const uint32_t c = s_pick != 0xffffffffu ? s_pick : s_last;
  const double base = s_base;
  __syncthreads();
  if (tid == 0) s_pick = 0xffffffffu, s_last = 0xffffffffu;
  __syncthreads();
  constexpr uint32_t kMine = kChunk / kPickThreads;  // neighbouring tokens of a thread
  double x[kMine], sum = 0.0, unused;
#pragma unroll
  for (uint32_t i = 0; i < kMine; ++i) {
    const uint32_t j = c * kChunk + tid * kMine + i;
    x[i] = j < a.vocab ? r.at(j, &unused) : 0.0;
    sum += x[i];
  }
  double end = base + (pick_prefix(sum, s_w, &t) - sum);
#pragma unroll
  for (uint32_t i = 0; i < kMine; ++i) {
    end += x[i];
    if (x[i] > 0.0) {
      if (end > goal) atomicMin(&s_pick, c * kChunk + tid * kMine + i);
      atomicMax(reinterpret_cast<int*>(&s_last), int(c * kChunk + tid * kMine + i));
    }
  }
  __syncthreads();
  if (tid == 0) a.next[b] = int32_t(s_pick != 0xffffffffu ? s_pick : s_last);
}

uint64_t verify_bytes(uint32_t sequences, uint32_t vocab) {
  return uint64_t(sequences) * ((uint64_t(vocab) + kChunk - 1) / kChunk) * sizeof(double2);
}

int check_sizes(uint32_t sequences, uint32_t vocab, std::string* msg) {
  if (sequences == 0 || sequences > 65535 || vocab == 0 || vocab > 0x7fffffffu) {
    *msg = "draft verification takes 1 to 65535 sequences and a vocabulary below 2^31";
    return SI_E_INVALID;
  }
  return SI_OK;
}

int check_verify(const si_verify_drafts* a, std::string* msg) {
  auto bad = [&](int rc, const std::string& text) {
    *msg = text;
    return rc;
  };
  if (!a) return bad(SI_E_INVALID, "null draft verification description");
  if (int rc = check_sizes(a->sequences, a->vocab, msg)) return rc;
  if (a->drafts > 32) return bad(SI_E_UNSUPPORTED, "draft verification takes at most 32 drafts a sequence");
  if (!a->target || !a->last_uniform || !a->accepted || !a->next)
    return bad(SI_E_INVALID, "draft verification buffers are null");
  if (a->drafts && (!a->tokens || !a->uniform)) return bad(SI_E_INVALID, "draft verification has no drafts or random numbers");
  for (uint64_t s : {a->target_seq_stride, a->target_row_stride, a->draft_seq_stride, a->draft_row_stride})
    if (s >> 44) return bad(SI_E_INVALID, "draft verification strides are out of range");
  const uint64_t need = verify_bytes(a->sequences, a->vocab);
  if (!a->work || reinterpret_cast<uintptr_t>(a->work) % 16 || a->work_bytes < need)
    return bad(SI_E_INVALID, "draft verification needs " + std::to_string(need) + " bytes of 16-byte aligned workspace");
  return SI_OK;
}

}  // namespace
}  // namespace si

using namespace si;

extern "C" int si_verify_drafts_workspace(uint32_t sequences, uint32_t vocab, uint64_t* bytes) {
  std::string msg;
  if (int rc = check_sizes(sequences, vocab, &msg)) return fail(nullptr, rc, msg);
  if (!bytes) return fail(nullptr, SI_E_INVALID, "null workspace size");
  *bytes = verify_bytes(sequences, vocab);
  return SI_OK;
}

extern "C" int si_verify_drafts_dev(si_ctx* ctx, const si_verify_drafts* a, void* stream) {
  std::string msg;
  if (int rc = check_verify(a, &msg)) return fail(ctx, rc, msg);
  if (!ctx) return fail(nullptr, SI_E_INVALID, "null context");
  DeviceGuard dev(ctx->device);
  if (dev.e != cudaSuccess) return cuda_fail(ctx, dev.e, "draft verification device");
  VerifyArgs p = {};
  p.p = a->target, p.q = a->drafts ? a->draft : nullptr;
  p.p_ss = a->target_seq_stride, p.p_rs = a->target_row_stride;
  p.q_ss = a->draft_seq_stride, p.q_rs = a->draft_row_stride;
  p.tokens = a->tokens, p.counts = a->drafts ? a->counts : nullptr;
  p.u = a->uniform, p.u_last = a->last_uniform;
  p.accepted = a->accepted, p.next = a->next;
  p.drafts = a->drafts, p.vocab = a->vocab;
  p.chunks = uint32_t((uint64_t(a->vocab) + kChunk - 1) / kChunk);
  p.sums = static_cast<double2*>(a->work);
  p.err = ctx->d_err;
  const cudaStream_t s = stream ? static_cast<cudaStream_t>(stream) : ctx->stream;
  PdlLaunch l(dim3(std::min(p.chunks, 65535u), a->sequences), dim3(kThreads), 0, s);
  if (cudaError_t e = cudaLaunchKernelEx(&l.cfg, verify_sum_kernel, p)) return cuda_fail(ctx, e, "draft verification launch");
  PdlLaunch k(dim3(a->sequences), dim3(kPickThreads), 0, s);
  if (cudaError_t e = cudaLaunchKernelEx(&k.cfg, verify_pick_kernel, p)) return cuda_fail(ctx, e, "draft verification launch");
  note_async_submission(ctx);
  return SI_OK;
}
