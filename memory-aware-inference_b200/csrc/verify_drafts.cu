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
// One kernel: a cluster of 1 to 8 CTAs a sequence. Every warp decides the
// accepted count for itself (a few loads, no barrier) and sums its own run of
// the row's tokens; the CTAs' totals meet over distributed shared memory, every CTA
// finds whose run the draw falls in, and that CTA scans that warp's run
// again. A difference is max(p - q, 0) = p - min(p, q), so that the minimum is
// taken in f32 and only the subtraction and the sum in f64. 64 windows over
// 248,320 tokens take 25 us (107 MB, 4.3 TB/s), one takes 9.5 us.
#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>

#include "paged.cuh"

namespace si {
namespace {

constexpr uint32_t kEach = 16, kTurn = 32 * kEach;  // tokens of a warp and turn
constexpr uint32_t kMaxCluster = 8;

struct VerifyArgs {
  const float *p, *q;
  uint64_t p_ss, p_rs, q_ss, q_rs;
  const int32_t *tokens, *counts;
  const float *u, *u_last;
  int32_t *accepted, *next;
  uint32_t drafts, vocab;
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

// A lane's tokens of a turn, from the turn's start: 16 bytes at a time where the
// row is aligned for that (64 windows over 248,320 tokens 28.4 us, 30.6 a token at a time).
template <bool WIDE>
__device__ __forceinline__ uint32_t token_of(uint32_t i, uint32_t lane) {
  return WIDE ? i / 4 * 128 + lane * 4 + i % 4 : i * 32 + lane;
}
template <bool WIDE>
__device__ __forceinline__ void load_turn(float x[kEach], const float* p, uint32_t lane) {
#pragma unroll
  for (uint32_t i = 0; i < kEach; i += WIDE ? 4 : 1) {
    const float* at = p + token_of<WIDE>(i, lane);
    if constexpr (WIDE)
      asm volatile("ld.global.nc.L1::no_allocate.L2::256B.v4.f32 {%0, %1, %2, %3}, [%4];"
                   : "=f"(x[i]), "=f"(x[i + 1]), "=f"(x[i + 2]), "=f"(x[i + 3])
                   : "l"(at));
    else
      asm volatile("ld.global.nc.L1::no_allocate.f32 %0, [%1];" : "=f"(x[i]) : "l"(at));
  }
}

// Sum of tokens [j0, j1) by one warp, the same in all lanes. All loads of a turn
// are on their way before the first value is used.
template <bool WIDE>
__device__ __forceinline__ double run_sum(const Rest& r, uint32_t j0, uint32_t j1, uint32_t lane) {
  double s = 0.0;
  uint32_t j = j0;
  for (; j + kTurn <= j1; j += kTurn) {
    float x[kEach], y[kEach];
    load_turn<WIDE>(x, r.p + j, lane);
    if (r.q) {
      load_turn<WIDE>(y, r.q + j, lane);
      // weight_of, but for infinities, which a turn is looked through for at once: one
      // window of 248,320 tokens 9.5 us, 10.5 with weight_of for each
      float most = 0.f;
      double turn = 0.0;
#pragma unroll
      for (uint32_t i = 0; i < kEach; ++i) {
        const float w = fmaxf(x[i], 0.f), v = fmaxf(y[i], 0.f);
        most = fmaxf(most, fmaxf(w, v));
        turn += double(w) - double(fminf(w, v));
      }
      if (most == INFINITY) {
        turn = 0.0;
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i) {
          const float w = weight_of(x[i]);
          turn += double(w) - double(fminf(w, weight_of(y[i])));
        }
      }
      s += turn;
    } else {
#pragma unroll
      for (uint32_t i = 0; i < kEach; ++i) s += j + token_of<WIDE>(i, lane) == r.without ? 0.0 : double(weight_of(x[i]));
    }
  }
#pragma unroll 4
  for (j += lane; j < j1; j += 32) s += r.at(j);
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

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ double peer_f64(const double* p, uint32_t rank) {
  uint32_t at;
  double v;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(at) : "memory");
  return v;
}

// Inclusive prefix over the lanes.
__device__ __forceinline__ double lane_prefix(double v, uint32_t lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= uint32_t(o)) v += y;
  }
  return v;
}
// Of lanes in order, each with a weight and the end of its share of the line:
// the first with weight whose end passes the goal; rounding may leave none:
// the last one with any weight. 32: no weight at all.
__device__ __forceinline__ uint32_t pick_lane(double weight, double end, double goal) {
  const uint32_t any = __ballot_sync(0xffffffffu, weight > 0.0);
  const uint32_t hit = __ballot_sync(0xffffffffu, weight > 0.0 && end > goal);
  return hit ? __ffs(hit) - 1 : any ? 31 - __clz(any) : 32;
}

// The lowest index that passes the goal, and the highest with weight at all;
// indexes rise with the lane, one atomic a warp.
__device__ __forceinline__ void note_borders(bool passes, uint32_t passing, bool weight, uint32_t index, uint32_t* pick,
                                             uint32_t* last) {
  const uint32_t lane = threadIdx.x & 31, any = __ballot_sync(0xffffffffu, weight);
  const uint32_t hit = __ballot_sync(0xffffffffu, passes);
  if (hit && lane == uint32_t(__ffs(hit) - 1)) atomicMin(pick, passing);
  if (any && lane == uint32_t(31 - __clz(any))) atomicMax(reinterpret_cast<int*>(last), int(index));
}

template <uint32_t THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) verify_kernel(const __grid_constant__ VerifyArgs a) {
  constexpr uint32_t kWarps = THREADS / 32;
  __shared__ double s_run[kWarps], s_total, s_scan[kWarps];
  __shared__ uint32_t s_pick, s_last;
  const uint32_t rank = cluster_rank(), size = cluster_size(), b = blockIdx.x / size;
  const uint32_t lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  pdl_launch_dependents();
  pdl_wait();
  const uint32_t taken = accepted_of(a, b, lane);
  Rest r = rest_of(a, b, taken);
  // runs of whole turns, but for the row's end
  const uint32_t turns = (a.vocab + kTurn - 1) / kTurn, runs = size * kWarps;
  auto border = [&](uint32_t i) { return uint32_t(min(uint64_t(a.vocab), uint64_t(turns) * i / runs * kTurn)); };
  double total = 0.0, mine = 0.0, before = 0.0;  // cluster's sum, this warp's, those of the CTAs before
  uint32_t owner = size;                           // the CTA that the draw falls in
  double goal = 0.0;
  for (int attempt = 0; attempt < 2; ++attempt) {
    if (attempt) {  // seldom: the difference is nothing; the target's row itself
      r.q = nullptr;
      r.without = 0xffffffffu;
    }
    const uint32_t i = rank * kWarps + w;
    const bool wide = ((reinterpret_cast<uintptr_t>(r.p) | reinterpret_cast<uintptr_t>(r.q)) & 15) == 0;
    mine = wide ? run_sum<true>(r, border(i), border(i + 1), lane) : run_sum<false>(r, border(i), border(i + 1), lane);
    if (lane == 0) s_run[w] = mine;
    __syncthreads();
    if (w == 0) {
      const double t = lane_prefix(lane < kWarps ? s_run[lane] : 0.0, lane);
      if (lane == 31) s_total = t;
    }
    cluster_arrive();
    cluster_wait();
    const double share = lane < size ? peer_f64(&s_total, lane) : 0.0;
    const double end = lane_prefix(share, lane);
    total = __shfl_sync(0xffffffffu, end, 31);
    goal = double(a.u_last[b]) * total;
    owner = pick_lane(share, end, goal);
    before = __shfl_sync(0xffffffffu, end - share, owner & 31);
    cluster_arrive();  // this CTA has read the totals
    if (total > 0.0 || attempt) break;  // the same decision in all CTAs
    cluster_wait();
  }
  // all CTAs of the cluster have read the count by now: `accepted` may lie over `counts`
  if (rank == 0 && threadIdx.x == 0) a.accepted[b] = int32_t(taken);
  // A CTA may not leave, nor its totals change, before all have read them.
  if (!(total > 0.0) || rank != owner) {
    if (!(total > 0.0) && rank == 0 && threadIdx.x == 0) a.next[b] = -1;
    cluster_wait();
    return;
  }
  // the warp's run within the CTA, found by every warp alike
  const double run = lane < kWarps ? s_run[lane] : 0.0, run_end = before + lane_prefix(run, lane);
  const uint32_t at = pick_lane(run, run_end, goal);
  double base = __shfl_sync(0xffffffffu, run_end - run, at & 31);
  const uint32_t j0 = border(rank * kWarps + at), j1 = border(rank * kWarps + at + 1);
  if (threadIdx.x == 0) s_pick = 0xffffffffu, s_last = 0xffffffffu;
  // A step is a chain of scans: long runs take four neighbouring tokens a thread and
  // step (64 windows over 248,320 tokens 25.7 us, 28.4 a token at a time), short ones
  // need one step either way (32,003 tokens 8.2 us, 8.7 with four).
  auto scan = [&](auto tokens) {
    constexpr uint32_t kScan = decltype(tokens)::value;
    for (uint32_t j = j0; j < j1; j += kScan * THREADS) {
      const uint32_t t = j + kScan * threadIdx.x;
      double x[kScan], sum = 0.0;
#pragma unroll
      for (uint32_t i = 0; i < kScan; ++i) x[i] = t + i < j1 ? r.at(t + i) : 0.0;
#pragma unroll
      for (uint32_t i = 0; i < kScan; ++i) sum += x[i];
      const double in_warp = lane_prefix(sum, lane);
      __syncthreads();
      if (lane == 31) s_scan[w] = in_warp;
      __syncthreads();
      const double ends = lane_prefix(lane < kWarps ? s_scan[lane] : 0.0, lane);
      const double near = __shfl_up_sync(0xffffffffu, in_warp, 1), far = __shfl_sync(0xffffffffu, ends, (w + 31) & 31);
      double end = base + (w ? far : 0.0) + (lane ? near : 0.0);
      uint32_t passing = kScan, last = kScan;  // the first that passes the goal, the last with any weight
#pragma unroll
      for (uint32_t i = 0; i < kScan; ++i) {
        end += x[i];
        if (x[i] > 0.0) last = i;
        if (x[i] > 0.0 && end > goal && passing == kScan) passing = i;
      }
      note_borders(passing < kScan, t + passing, last < kScan, t + last, &s_pick, &s_last);
      base += __shfl_sync(0xffffffffu, ends, 31);
      __syncthreads();
      if (s_pick != 0xffffffffu) break;  // the same for all threads
    }
  };
  if (j1 - j0 <= THREADS)
    scan(std::integral_constant<uint32_t, 1>());
  else
    scan(std::integral_constant<uint32_t, 4>());
  if (threadIdx.x == 0) a.next[b] = int32_t(s_pick != 0xffffffffu ? s_pick : s_last);
  cluster_wait();
}

// Nothing is kept between CTAs in memory; the smallest workspace that a caller can hold.
uint64_t verify_bytes() { return 16; }

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
  if (!words_aligned({a->target, a->draft, a->tokens, a->counts, a->uniform, a->last_uniform, a->accepted, a->next}))
    return bad(SI_E_INVALID, "draft verification buffers are not aligned to their elements");
  for (uint64_t s : {a->target_seq_stride, a->target_row_stride, a->draft_seq_stride, a->draft_row_stride})
    if (s >> 44) return bad(SI_E_INVALID, "draft verification strides are out of range");
  const uint64_t need = verify_bytes();
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
  *bytes = verify_bytes();
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
  p.err = ctx->d_err;
  const cudaStream_t s = stream ? static_cast<cudaStream_t>(stream) : ctx->stream;
  // A CTA of 1024 threads a multiprocessor, or two of 512 where the sequences fill
  // those: as many a sequence as run at once, and as the row has runs for.
  const uint32_t sms = uint32_t(ctx->sm_count);
  const bool large = a->sequences * 2 > sms;
  const uint32_t turns = (a->vocab + kTurn - 1) / kTurn, warps = large ? 16 : 32;
  uint32_t cluster = 1;
  while (cluster < kMaxCluster && a->sequences * cluster * 2 <= (large ? 2 * sms : sms) && turns > cluster * warps)
    cluster *= 2;
  PdlLaunch l(dim3(a->sequences * cluster), dim3(warps * 32), 0, s);
  l.cluster(cluster);
  if (cudaError_t e = large ? cudaLaunchKernelEx(&l.cfg, verify_kernel<512>, p) : cudaLaunchKernelEx(&l.cfg, verify_kernel<1024>, p))
    return cuda_fail(ctx, e, "draft verification launch");
  note_async_submission(ctx);
  return SI_OK;
}
