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
// Two kernels. Every warp of the first decides the sequence's accepted count
// for itself (a few loads) and sums chunks of 512 tokens of the row, no barrier;
// one CTA a sequence of the second scans the chunk sums, finds the chunk that
// the draw falls in, and scans that chunk. The row is read once, one chunk of
// it twice. A difference is max(p - q, 0) = p - min(p, q), so that the minimum is
// taken in f32 and only the subtraction and the sum in f64: conversions have an eighth
// of the f32 rate and were what bound the sums at first.
#include <cuda_runtime.h>

#include <algorithm>

#include "paged.cuh"

namespace si {
namespace {

constexpr uint32_t kThreads = 256, kEach = 16, kChunk = 32 * kEach;  // tokens of a chunk
constexpr uint32_t kPickThreads = 1024;

struct VerifyArgs {
  const float *p, *q;
  uint64_t p_ss, p_rs, q_ss, q_rs;
  const int32_t *tokens, *counts;
  const float *u, *u_last;
  int32_t *accepted, *next;
  uint32_t drafts, vocab, chunks;
  double* sums;  // [sequence][chunk]
  int* err;
};

// Negative, infinite and NaN entries count as 0 (NaN compares false).
__device__ __forceinline__ float weight_of(float x) { return x > 0.f && x < INFINITY ? x : 0.f; }

// The row that the next token is drawn from.
struct Rest {
  const float* p;
  const float* q;     // null: nothing is taken away
  uint32_t without;   // this token's weight is taken away; >= vocab: none
  __device__ __forceinline__ double at(uint32_t j) const {
    const float x = weight_of(p[j]);
    if (q) return double(x) - double(fminf(x, weight_of(q[j])));
    return j == without ? 0.0 : double(x);
  }
};

__device__ __forceinline__ float load_stream(const float* p) {
  float x;
  asm volatile("ld.global.nc.L1::no_allocate.f32 %0, [%1];" : "=f"(x) : "l"(p));
  return x;
}

// Sum of chunk c by one warp, the same in all lanes. All loads are on their way
// before the first value is used.
__device__ __forceinline__ double chunk_sum(const Rest& r, uint32_t c, uint32_t vocab, uint32_t lane) {
  const uint32_t j0 = c * kChunk + lane;
  double s = 0.0;
  float x[kEach], y[kEach];
  if (c * kChunk + kChunk <= vocab) {
#pragma unroll
    for (uint32_t i = 0; i < kEach; ++i) x[i] = load_stream(r.p + j0 + i * 32);
    if (r.q) {
#pragma unroll
      for (uint32_t i = 0; i < kEach; ++i) y[i] = load_stream(r.q + j0 + i * 32);
#pragma unroll
      for (uint32_t i = 0; i < kEach; ++i) {
        const float w = weight_of(x[i]);
        s += double(w) - double(fminf(w, weight_of(y[i])));
      }
    } else {
#pragma unroll
      for (uint32_t i = 0; i < kEach; ++i) s += j0 + i * 32 == r.without ? 0.0 : double(weight_of(x[i]));
    }
  } else {
    for (uint32_t j = j0; j < vocab; j += 32) s += r.at(j);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}

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
      const float p = weight_of(a.p[b * a.p_ss + lane * a.p_rs + uint32_t(x)]);
      const float q = a.q ? weight_of(a.q[b * a.q_ss + lane * a.q_rs + uint32_t(x)]) : 1.f;
      ok = double(a.u[uint64_t(b) * a.drafts + lane]) * double(q) < double(p);  // exact: 24 + 24 bits
    } else {
      atomicOr(a.err, KERR_BAD_INDEX);
    }
  }
  const uint32_t first = __ffs(~__ballot_sync(0xffffffffu, ok));  // 1 + the first that was not accepted
  return first ? first - 1 : 32u;
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
  const uint32_t b = blockIdx.y, lane = threadIdx.x & 31, w = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  pdl_launch_dependents();
  pdl_wait();
  if (w >= a.chunks && w) return;
  const uint32_t taken = accepted_of(a, b, lane);
  if (w == 0 && lane == 0) a.accepted[b] = int32_t(taken);
  const Rest r = rest_of(a, b, taken);
  for (uint32_t c = w; c < a.chunks; c += gridDim.x * (kThreads / 32)) {
    const double s = chunk_sum(r, c, a.vocab, lane);
    if (lane == 0) a.sums[uint64_t(b) * a.chunks + c] = s;
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

// The lowest index with weight whose end passes the goal, and the highest with
// weight at all; index rises with the lane, one atomic a warp.
__device__ __forceinline__ void note_borders(bool weight, bool passes, uint32_t index, uint32_t* pick, uint32_t* last) {
  const uint32_t lane = threadIdx.x & 31, any = __ballot_sync(0xffffffffu, weight);
  const uint32_t hit = __ballot_sync(0xffffffffu, weight && passes);
  if (hit && lane == uint32_t(__ffs(hit) - 1)) atomicMin(pick, index);
  if (any && lane == uint32_t(31 - __clz(any))) atomicMax(reinterpret_cast<int*>(last), int(index));
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
  double* sums = a.sums + uint64_t(b) * a.chunks;
  // up to kPickThreads chunks (524,288 tokens) one scan gives total and borders
  double first_total, t;
  const double first = tid < a.chunks ? sums[tid] : 0.0, first_end = pick_prefix(first, s_w, &first_total);
  double total = first_total;
  for (uint32_t c0 = kPickThreads; c0 < a.chunks; c0 += kPickThreads) {
    pick_prefix(c0 + tid < a.chunks ? sums[c0 + tid] : 0.0, s_w, &t);
    total += t;
  }
  const bool again = !(total > 0.0);
  if (again) {  // seldom: the difference is nothing; the target's row itself
    r.q = nullptr;
    r.without = 0xffffffffu;
    for (uint32_t c = tid >> 5; c < a.chunks; c += kPickThreads / 32) {
      const double s = chunk_sum(r, c, a.vocab, tid & 31);
      if ((tid & 31) == 0) sums[c] = s;
    }
    __syncthreads();
    for (uint32_t c0 = 0; c0 < a.chunks; c0 += kPickThreads) {
      pick_prefix(c0 + tid < a.chunks ? sums[c0 + tid] : 0.0, s_w, &t);
      total += t;
    }
  }
  if (!(total > 0.0)) {
    if (tid == 0) a.next[b] = -1;
    return;
  }
  const double goal = double(a.u_last[b]) * total;
  // the first chunk whose end passes the goal; rounding may leave none: the last one with any weight
  double run = 0.0;
  for (uint32_t c0 = 0; c0 < a.chunks; c0 += kPickThreads) {
    double v = first, end = first_end;
    t = first_total;
    if (c0 || again) {
      v = c0 + tid < a.chunks ? sums[c0 + tid] : 0.0;
      end = run + pick_prefix(v, s_w, &t);
    }
    note_borders(v > 0.0, end > goal, c0 + tid, &s_pick, &s_last);
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
  static_assert(kChunk <= kPickThreads, "a thread a token");
  const uint32_t j = c * kChunk + tid;
  const double x = tid < kChunk && j < a.vocab ? r.at(j) : 0.0, end = base + pick_prefix(x, s_w, &t);
  note_borders(x > 0.0, end > goal, j, &s_pick, &s_last);
  __syncthreads();
  if (tid == 0) a.next[b] = int32_t(s_pick != 0xffffffffu ? s_pick : s_last);
}

uint64_t verify_bytes(uint32_t sequences, uint32_t vocab) {
  return uint64_t(sequences) * ((uint64_t(vocab) + kChunk - 1) / kChunk) * sizeof(double);
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
  p.sums = static_cast<double*>(a->work);
  p.err = ctx->d_err;
  const cudaStream_t s = stream ? static_cast<cudaStream_t>(stream) : ctx->stream;
  // CTAs for every chunk at small batches; at large ones a few a sequence, which
  // then share the beginning (three dependent loads) among several chunks
  const uint32_t all = (p.chunks + kThreads / 32 - 1) / (kThreads / 32);
  const uint32_t few = std::max(1u, uint32_t(ctx->sm_count) * 16 / a->sequences);
  PdlLaunch l(dim3(std::min(all, few), a->sequences), dim3(kThreads), 0, s);
  if (cudaError_t e = cudaLaunchKernelEx(&l.cfg, verify_sum_kernel, p)) return cuda_fail(ctx, e, "draft verification launch");
  PdlLaunch k(dim3(a->sequences), dim3(kPickThreads), 0, s);
  if (cudaError_t e = cudaLaunchKernelEx(&k.cfg, verify_pick_kernel, p)) return cuda_fail(ctx, e, "draft verification launch");
  note_async_submission(ctx);
  return SI_OK;
}
