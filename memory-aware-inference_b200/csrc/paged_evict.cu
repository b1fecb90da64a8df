// Eviction from a paged cache by accumulated attention weight.
//
// Of n slots the e = n - budget with the smallest weights leave (protected
// ones last), of equal weights the lowest slots. A float becomes an unsigned
// key of the same order, so the e-th smallest key is found digit by digit
// (11, 11 and 10 bits, most significant first): a histogram of the digit over
// the slots that share the digits found so far, a scan over its bins. Then one
// ordered walk numbers the equal keys, marks who leaves, and numbers the holes
// below the new length and the kept slots behind it; pair i moves from the
// i-th kept slot to the i-th hole.
//
// Selection: one CTA a (sequence, kv head), or a cluster of up to 8 for long
// sequences; every key is read from global memory once and stays in shared
// memory for the three digits and the walk; histograms and counts meet over
// distributed shared memory. Small CTAs where the keys are few: the time is that of a
// chain of small scans, so as many rows as possible run beside each other.
// Moves: a second kernel over all pairs of all heads, because a cut of a long
// prompt moves megabytes where the selection is a few scans. Selection is bound by
// latency, moves by bandwidth: 16 rows of 131,072 slots cut to 8,192 take 77 us, of
// which the moves are 42 (252 MB, 6 TB/s).
#include <cuda_runtime.h>

#include <algorithm>

#include "paged.cuh"

namespace si {
namespace {

constexpr uint32_t kBins = 2048;
constexpr uint32_t kCtaSlots = 49152;  // keys in a CTA's shared memory
constexpr uint32_t kMaxCluster = 8;
constexpr uint32_t kKeep = 0xffffffffu;  // protected: behind every weight, +inf too

struct EvictArgs {
  PagedView kv;
  const int32_t* len_in;
  int32_t* len_out;
  const float* w_in;
  float* w_out;
  const int32_t* p_in;
  int32_t* p_out;
  const int32_t* next;
  uint64_t stride;
  uint32_t budget, sink, recent;
  uint32_t most;  // longest length that the page table and the weights' rows have room for
  uint32_t room;  // entries of a move list
  bool at_once;   // the selecting CTA moves the pairs itself
  uint32_t* moves;   // [sequence * kv_heads + head][2][room]: from, to
  uint32_t* counts;  // [sequence * kv_heads + head]
  int* err;
};

// Order of floats as unsigned numbers; -0 is 0, NaN comes first.
__device__ __forceinline__ uint32_t key_of(float w) {
  if (w != w) return 0;
  const uint32_t u = __float_as_uint(w + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
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
template <bool CLUSTER>
__device__ __forceinline__ void group_sync() {
  if constexpr (CLUSTER)
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  else
    __syncthreads();
}
__device__ __forceinline__ uint32_t peer_address(const uint32_t* p, uint32_t rank) {
  uint32_t at;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
  return at;
}
__device__ __forceinline__ uint32_t peer_u32(const uint32_t* p, uint32_t rank) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(peer_address(p, rank)) : "memory");
  return v;
}
// N neighbouring words of another CTA, zeros if not `on`.
template <uint32_t N>
__device__ __forceinline__ void peer_bins(uint32_t* v, const uint32_t* p, uint32_t rank, bool on) {
  static_assert(N == 2 || N == 4, "bins of a thread");
#pragma unroll
  for (uint32_t i = 0; i < N; ++i) v[i] = 0;
  if (!on) return;
  if constexpr (N == 2)
    asm volatile("ld.shared::cluster.v2.u32 {%0, %1}, [%2];" : "=r"(v[0]), "=r"(v[1]) : "r"(peer_address(p, rank)) : "memory");
  else
    asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
                 : "r"(peer_address(p, rank))
                 : "memory");
}

// Exclusive prefix of one value a thread over the CTA; *total gets the sum.
template <int THREADS>
__device__ __forceinline__ uint32_t cta_prefix(uint32_t v, uint32_t* s_w, uint32_t* total) {
  const uint32_t lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  uint32_t x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= uint32_t(o)) x += y;
  }
  __syncthreads();
  if (lane == 31) s_w[w] = x;
  __syncthreads();
  uint32_t y = lane < THREADS / 32 ? s_w[lane] : 0;
  const uint32_t mine = y;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t z = __shfl_up_sync(0xffffffffu, y, o);
    if (lane >= uint32_t(o)) y += z;
  }
  *total = __shfl_sync(0xffffffffu, y, 31);
  return __shfl_sync(0xffffffffu, y - mine, w) + x - v;
}

// Kept slots from behind the new length into the holes below it: sources and
// destinations do not meet, so the order is free. Eight lanes move a pair, each
// up to four 16-byte pieces of its key and of its value, all in flight at once.
// Thread `thread` of `threads` (a multiple of 8).
constexpr uint32_t kLanes = 8;
__device__ __forceinline__ void move_pairs(const EvictArgs& a, uint32_t row, uint32_t b, uint32_t h, uint32_t pairs,
                                           uint32_t thread, uint32_t threads) {
  const uint32_t chunks = a.kv.hd / 8, l = thread % kLanes;
  const uint64_t base = uint64_t(row) * a.stride;
  const uint32_t *froms = a.moves + uint64_t(row) * 2 * a.room, *tos = froms + a.room;
  const int32_t* pages = a.kv.pages + b * a.kv.pages_stride;
  uint16_t *k_pool = const_cast<uint16_t*>(a.kv.k), *v_pool = const_cast<uint16_t*>(a.kv.v);
  for (uint32_t i = thread / kLanes; i < pairs; i += threads / kLanes) {
    const uint2 mv = make_uint2(froms[i], tos[i]);
    const uint64_t from = paged_slot(a.kv, pages, mv.x, h), to = paged_slot(a.kv, pages, mv.y, h);
    float w = 0.f;
    int32_t p = 0;
    if (l == 0) {
      w = a.w_in[base + mv.x];
      p = a.p_in ? a.p_in[base + mv.x] : int32_t(mv.x);
    }
    if (from != kNoCell && to != kNoCell) {
      uint4 k[4], v[4];
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j) {
        const uint32_t ch = l + j * kLanes;
        if (ch < chunks) {
          k[j] = *reinterpret_cast<const uint4*>(k_pool + from + ch * 8);
          v[j] = *reinterpret_cast<const uint4*>(v_pool + from + ch * 8);
        }
      }
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j) {
        const uint32_t ch = l + j * kLanes;
        if (ch < chunks) {
          *reinterpret_cast<uint4*>(k_pool + to + ch * 8) = k[j];
          *reinterpret_cast<uint4*>(v_pool + to + ch * 8) = v[j];
        }
      }
    } else if (l == 0) {
      atomicOr(a.err, KERR_BAD_INDEX);
    }
    if (l == 0) {
      a.w_out[base + mv.y] = w;
      if (a.p_out) a.p_out[base + mv.y] = p;
    }
  }
}

template <int THREADS, bool CLUSTER>
__global__ void __launch_bounds__(THREADS, THREADS == 1024 ? 1 : 2) evict_select_kernel(const __grid_constant__ EvictArgs a) {
  constexpr uint32_t kWarps = THREADS / 32, kMine = kBins / THREADS;  // bins of a thread
  extern __shared__ uint32_t s_key[];
  __shared__ __align__(16) uint32_t s_bin[kBins];
  __shared__ uint32_t s_w[32], s_found[3], s_ties, s_moves[2];
  const uint32_t rank = CLUSTER ? cluster_rank() : 0, size = CLUSTER ? cluster_size() : 1;
  const uint32_t row = blockIdx.x / size, b = row / a.kv.kv_heads;
  const uint32_t tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  pdl_launch_dependents();
  pdl_wait();
  const uint32_t n = checked_length(a.len_in[b], a.most, a.err), m = min(n, a.budget);
  const uint32_t leave = n - m;
  const uint64_t base = uint64_t(row) * a.stride;
  if (row == b * a.kv.kv_heads && rank == 0 && tid == 0) {
    // other CTAs of this launch read len_in[b] too: where it is len_out itself
    // the new length is written by the second kernel
    if (a.len_out != a.len_in) a.len_out[b] = int32_t(m);
  }
  // a CTA's slots, a multiple of its threads so that every warp has whole rows of 32
  const uint32_t chunk = ((n + size - 1) / size + THREADS - 1) / THREADS * THREADS;
  const uint32_t lo = min(n, rank * chunk), hi = min(n, lo + chunk);
  // Keys; and the weights and positions below the new length go out as they
  // are (the second kernel writes over those of the holes).
  const int64_t next = a.next ? int64_t(a.next[b]) : int64_t(n);
  // positions below `low` or from `high` on are protected (none reaches a `high` past 31 bits)
  const int32_t low = int32_t(min(a.sink, 0x7fffffffu));
  const int64_t from = next - int64_t(a.recent);
  const int32_t high = int32_t(max(int64_t(INT32_MIN), min(from, int64_t(INT32_MAX))));
  const bool any_high = from <= INT32_MAX;
  const bool w_copy = a.w_out != a.w_in, p_copy = a.p_out && a.p_out != a.p_in;
  const uint32_t stop = leave ? hi : min(hi, w_copy || p_copy ? m : 0);
  for (uint32_t i = tid; i < kBins; i += THREADS) s_bin[i] = 0;
  __syncthreads();
  for (uint32_t t0 = lo + tid; t0 < stop; t0 += 4 * THREADS) {
    float wt[4];
    int32_t pos[4];
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
      const uint32_t t = t0 + i * THREADS;
      wt[i] = t < stop ? a.w_in[base + t] : 0.f;
      pos[i] = a.p_in ? (t < stop ? a.p_in[base + t] : 0) : int32_t(t);
    }
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
      const uint32_t t = t0 + i * THREADS;
      if (t >= stop) break;
      const bool held = pos[i] < low || (any_high && pos[i] >= high);
      const uint32_t k = held ? kKeep : key_of(wt[i]);
      s_key[t - lo] = k;
      atomicAdd(&s_bin[k >> 21], 1u);
      if (t < m && w_copy) a.w_out[base + t] = wt[i];
      if (t < m && p_copy) a.p_out[base + t] = pos[i];
    }
  }
  if (leave == 0) {  // the same for the whole cluster
    if (rank == 0 && tid == 0) a.counts[row] = 0;
    return;
  }
  // The leave-th smallest key, digit by digit; `want` counts within the keys
  // that share the digits so far. Once all of them leave, their lower digits do not matter.
  uint32_t found = 0, mask = 0, want = leave, same = 0;
  for (int digit = 0; digit < 3; ++digit) {
    const int shift = digit == 0 ? 21 : digit == 1 ? 10 : 0;
    const uint32_t bins = digit == 2 ? 1024 : kBins;
    if (digit) {
      for (uint32_t i = tid; i < kBins; i += THREADS) s_bin[i] = 0;
      __syncthreads();
#pragma unroll 4
      for (uint32_t t = tid; t < hi - lo; t += THREADS) {
        const uint32_t k = s_key[t];
        if ((k & mask) == found) atomicAdd(&s_bin[(k >> shift) & (bins - 1)], 1u);
      }
    }
    group_sync<CLUSTER>();
    // neighbouring bins a thread, summed over the cluster
    uint32_t c[kMine] = {}, sum = 0;
    if constexpr (CLUSTER) {
      uint32_t far[kMaxCluster][kMine];  // all on their way at once
#pragma unroll
      for (uint32_t r = 0; r < kMaxCluster; ++r) peer_bins<kMine>(far[r], &s_bin[kMine * tid], r, r < size);
#pragma unroll
      for (uint32_t r = 0; r < kMaxCluster; ++r)
#pragma unroll
        for (uint32_t i = 0; i < kMine; ++i) c[i] += far[r][i];
    } else {
#pragma unroll
      for (uint32_t i = 0; i < kMine; ++i) c[i] = s_bin[kMine * tid + i];
    }
#pragma unroll
    for (uint32_t i = 0; i < kMine; ++i) sum += c[i];
    uint32_t total;
    uint32_t before = cta_prefix<THREADS>(sum, s_w, &total);
    if (before < want && want <= before + sum) {
#pragma unroll
      for (uint32_t i = 0; i < kMine; ++i) {
        if (before < want && want <= before + c[i]) {
          s_found[0] = kMine * tid + i;
          s_found[1] = before;
          s_found[2] = c[i];
        }
        before += c[i];
      }
    }
    group_sync<CLUSTER>();  // also: every CTA has read this one's bins
    found |= s_found[0] << shift;
    mask |= (bins - 1) << shift;
    want -= s_found[1];
    same = s_found[2];
    if (same == want) break;  // the same in all threads of the cluster
  }
  // `want` of the keys equal to `found` leave, lowest slots first. A warp walks
  // its own run of consecutive slots, 32 a step.
  const uint32_t run = chunk / kWarps, w0 = min(hi, lo + w * run), w1 = min(hi, w0 + run);
  // v summed over the warps before this one, cluster-wide
  auto before_warp = [&](uint32_t v, uint32_t* s_total, uint32_t* cluster_total) {
    uint32_t total;
    const uint32_t mine = cta_prefix<THREADS>(lane == 0 ? v : 0u, s_w, &total);
    uint32_t before = 0, all = total;
    if constexpr (CLUSTER) {
      if (tid == 0) *s_total = total;
      group_sync<CLUSTER>();
      all = 0;
#pragma unroll
      for (uint32_t r = 0; r < kMaxCluster; ++r) {
        const uint32_t x = r < size ? peer_u32(s_total, r) : 0;
        if (r < rank) before += x;
        all += x;
      }
    }
    *cluster_total = all;
    return before + __shfl_sync(0xffffffffu, mine, 0);
  };
  const bool all_same = want == same;
  const uint32_t below = (1u << lane) - 1, limit = found | ~mask;  // all_same: everything up to `limit` leaves
  uint32_t seen = 0, all;
  if (!all_same) {
    uint32_t ties = 0;
#pragma unroll 4
    for (uint32_t t = w0 + lane; t - lane < w1; t += 32)
      ties += __popc(__ballot_sync(0xffffffffu, t < w1 && s_key[t - lo] == found));
    seen = before_warp(ties, &s_ties, &all);  // equal keys before the warp's run
  }
  // Bit l of word i of the run: slot 32 i + l leaves. The words go over the run's
  // first keys, which the warp has read by then (a run has a word for 32 keys).
  uint32_t* word = s_key + (w0 - lo);
#pragma unroll 4
  for (uint32_t t = w0 + lane; t - lane < w1; t += 32) {
    const bool in = t < w1;
    const uint32_t k = in ? s_key[t - lo] : kKeep;
    uint32_t gone;
    if (all_same) {
      gone = __ballot_sync(0xffffffffu, in && k <= limit);
    } else {
      const uint32_t eq = __ballot_sync(0xffffffffu, in && k == found);
      gone = __ballot_sync(0xffffffffu, in && (k < found || (k == found && seen + __popc(eq & below) < want)));
      seen += __popc(eq);
    }
    if (lane == 0) word[(t - lane - w0) / 32] = gone;
  }
  __syncwarp();
  // The words' holes below the new length, and kept slots behind it: a lane a word.
  const uint32_t words = (w1 - w0 + 31) / 32;
  auto bits_of = [&](uint32_t i, uint32_t& hole, uint32_t& stay) {
    hole = stay = 0;
    if (i >= words) return;
    const uint32_t t = w0 + 32 * i, left = w1 - t;
    const uint32_t in = left >= 32 ? 0xffffffffu : (1u << left) - 1;
    const uint32_t kept_side = m <= t ? 0u : m - t >= 32 ? 0xffffffffu : (1u << (m - t)) - 1;
    hole = word[i] & kept_side;
    stay = ~word[i] & in & ~kept_side;
  };
  uint32_t holes = 0, kept = 0;
  for (uint32_t i = lane; i < words; i += 32) {
    uint32_t hole, stay;
    bits_of(i, hole, stay);
    holes += __popc(hole);
    kept += __popc(stay);
  }
  holes = __reduce_add_sync(0xffffffffu, holes);
  kept = __reduce_add_sync(0xffffffffu, kept);
  uint32_t moved;
  uint32_t hole0 = before_warp(holes, &s_moves[0], &moved);
  uint32_t kept0 = before_warp(kept, &s_moves[1], &all);
  uint32_t *from_list = a.moves + uint64_t(row) * 2 * a.room, *to_list = from_list + a.room;
  if (holes | kept) {
    for (uint32_t i = 0; i < words; ++i) {
      uint32_t hole, stay;
      bits_of(i, hole, stay);
      const uint32_t t = w0 + 32 * i + lane;
      if (hole >> lane & 1) to_list[hole0 + __popc(hole & below)] = t;
      if (stay >> lane & 1) from_list[kept0 + __popc(stay & below)] = t;
      hole0 += __popc(hole);
      kept0 += __popc(stay);
    }
  }
  if (rank == 0 && tid == 0) a.counts[row] = moved;
  if (!CLUSTER && a.at_once) {
    __syncthreads();  // the lists, and the weights and positions that went out as they were
    move_pairs(a, row, b, row - b * a.kv.kv_heads, moved, tid, THREADS);
  }
  if constexpr (CLUSTER) group_sync<CLUSTER>();  // no CTA leaves while another may still read its counts
}

__global__ void __launch_bounds__(256) evict_move_kernel(const __grid_constant__ EvictArgs a) {
  const uint32_t row = blockIdx.y, b = row / a.kv.kv_heads, h = row - b * a.kv.kv_heads;
  pdl_launch_dependents();
  pdl_wait();
  if (a.len_out == a.len_in && blockIdx.x == 0 && h == 0 && threadIdx.x == 0) {
    const int32_t n = a.len_in[b];  // read and written by this thread alone
    a.len_out[b] = int32_t(min(n < 0 ? 0u : min(uint32_t(n), a.most), a.budget));
  }
  move_pairs(a, row, b, h, a.counts[row], blockIdx.x * 256 + threadIdx.x, gridDim.x * 256);
}

uint64_t rows_of(const si_paged_kv& kv) { return uint64_t(kv.sequences) * kv.kv_heads; }
// A list holds at most half of the slots: one of a pair is below the budget, one behind it.
uint64_t room_of(const si_paged_kv& kv) { return uint64_t(kv.max_pages) * kv.page_tokens / 2 + 1; }
uint64_t evict_bytes(const si_paged_kv& kv) {
  return ((rows_of(kv) * 4 + 15) & ~uint64_t(15)) + rows_of(kv) * room_of(kv) * 8;
}

template <int THREADS, bool CLUSTER>
cudaError_t select(const EvictArgs& p, uint32_t rows, uint32_t cluster, uint32_t each, cudaStream_t s) {
  static RaisedLimit limits[kMaxDevices];
  const uint32_t bytes = (each + THREADS - 1) / THREADS * THREADS * 4;
  if (cudaError_t e = raise_smem_limit(evict_select_kernel<THREADS, CLUSTER>, bytes, limits)) return e;
  PdlLaunch l(dim3(rows * cluster), dim3(THREADS), bytes, s);
  if (CLUSTER) l.cluster(cluster);
  return cudaLaunchKernelEx(&l.cfg, evict_select_kernel<THREADS, CLUSTER>, p);
}

int check_size(const si_paged_kv* kv, std::string* msg) {
  if (int rc = check_paged_kv(kv, msg)) return rc;
  if (uint64_t(kv->max_pages) * kv->page_tokens > uint64_t(kCtaSlots) * kMaxCluster) {
    *msg = "paged eviction takes at most " + std::to_string(kCtaSlots * kMaxCluster) + " slots a sequence";
    return SI_E_UNSUPPORTED;
  }
  if (rows_of(*kv) > 65535) {
    *msg = "paged eviction takes at most 65535 sequences times kv heads";
    return SI_E_UNSUPPORTED;
  }
  return SI_OK;
}

int check_evict(const si_paged_kv* kv, const si_paged_evict* a, std::string* msg) {
  auto bad = [&](int rc, const std::string& text) {
    *msg = text;
    return rc;
  };
  if (!a) return bad(SI_E_INVALID, "null paged eviction description");
  if (int rc = check_size(kv, msg)) return rc;
  if (!pools_distinct(*kv)) return bad(SI_E_INVALID, "paged eviction needs pools whose rows do not overlap");
  if (!a->lengths_in || !a->lengths_out || !a->weights_in || !a->weights_out)
    return bad(SI_E_INVALID, "paged eviction buffers are null");
  if (!words_aligned({a->lengths_in, a->lengths_out, a->weights_in, a->weights_out, a->positions_in, a->positions_out,
                      a->next_position}))
    return bad(SI_E_INVALID, "paged eviction buffers are not aligned to their elements");
  if (a->positions_in && !a->positions_out)
    return bad(SI_E_INVALID, "paged eviction has positions in and none out");
  if (a->next_position && a->next_position == a->lengths_out && a->lengths_in != a->lengths_out)
    return bad(SI_E_INVALID, "paged eviction would write the new lengths over the next positions");
  if (a->budget == 0 || uint64_t(a->sink) + a->recent > a->budget)
    return bad(SI_E_INVALID, "paged eviction needs a budget of at least sink + recent tokens, and of one");
  if (a->weights_stride == 0 || a->weights_stride >> 44) return bad(SI_E_INVALID, "paged eviction stride is out of range");
  const uint64_t need = evict_bytes(*kv);
  if (!a->work || reinterpret_cast<uintptr_t>(a->work) % 16 || a->work_bytes < need)
    return bad(SI_E_INVALID, "paged eviction needs " + std::to_string(need) + " bytes of 16-byte aligned workspace");
  return SI_OK;
}

}  // namespace
}  // namespace si

using namespace si;

extern "C" int si_paged_evict_workspace(const si_paged_kv* kv, uint64_t* bytes) {
  std::string msg;
  if (int rc = check_size(kv, &msg)) return fail(nullptr, rc, msg);
  if (!bytes) return fail(nullptr, SI_E_INVALID, "null workspace size");
  *bytes = evict_bytes(*kv);
  return SI_OK;
}

extern "C" int si_paged_evict_dev(si_ctx* ctx, const si_paged_kv* kv, const si_paged_evict* a, void* stream) {
  std::string msg;
  if (int rc = check_evict(kv, a, &msg)) return fail(ctx, rc, msg);
  if (!ctx) return fail(nullptr, SI_E_INVALID, "null context");
  DeviceGuard dev(ctx->device);
  if (dev.e != cudaSuccess) return cuda_fail(ctx, dev.e, "paged eviction device");
  EvictArgs p = {};
  p.kv = paged_view(*kv);
  p.len_in = a->lengths_in, p.len_out = a->lengths_out;
  p.w_in = a->weights_in, p.w_out = a->weights_out;
  p.p_in = a->positions_in, p.p_out = a->positions_out;
  p.next = a->next_position;
  p.stride = a->weights_stride;
  p.budget = a->budget, p.sink = a->sink, p.recent = a->recent;
  p.most = uint32_t(std::min<uint64_t>(p.kv.max_tokens, a->weights_stride));
  p.room = uint32_t(room_of(*kv));
  p.counts = static_cast<uint32_t*>(a->work);
  p.moves = reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(a->work) + ((rows_of(*kv) * 4 + 15) & ~uint64_t(15)));
  p.err = ctx->d_err;
  const cudaStream_t s = stream ? static_cast<cudaStream_t>(stream) : ctx->stream;
  const uint32_t rows = uint32_t(rows_of(*kv)), most = p.most;
  // A CTA for 8192 keys, as long as the clusters find room beside each other: a
  // graphics processing cluster has 14 multiprocessors or more, so 8 of them hold
  // 8 (14 / c) clusters of c CTAs for sure. Multiprocessors come in pairs, and odd
  // sizes were slower than the even ones on both sides (16 rows of 131,072 slots:
  // clusters of 8, in two waves, 92 us; 7, 95; 6, 77; 5, 78; 4, 86).
  uint32_t cluster = std::min(kMaxCluster, (most + 8191) / 8192);
  if (cluster > 1) cluster += cluster % 2;
  while (cluster > 1 && rows > 8 * (14 / cluster) && most <= (cluster > 2 ? cluster - 2 : 1) * kCtaSlots)
    cluster = cluster > 2 ? cluster - 2 : 1;
  const uint32_t each = (most + cluster - 1) / cluster;
  // Moves of one row are at most the smaller of both sides of the budget. A few
  // (a page's worth leaves in steady state) the selecting CTA makes itself, which saves a
  // launch: 32 x 8 rows of 4,160 slots that lose 64 take 16.0 us, and 18.6 us with a second
  // kernel. Not where the new lengths go over the old ones: other heads' CTAs
  // still read those.
  const uint64_t most_moves = std::min<uint64_t>(most > a->budget ? most - a->budget : 0, a->budget);
  p.at_once = cluster == 1 && most_moves <= 256 && p.len_in != p.len_out;
  // 256, 512 or 1024 threads for up to 8 or 16 keys a thread; a cluster's CTAs have their multiprocessors to themselves
  const cudaError_t e = cluster > 1   ? select<1024, true>(p, rows, cluster, each, s)
                        : each > 8192 ? select<1024, false>(p, rows, 1, each, s)
                        : each > 2048 ? select<512, false>(p, rows, 1, each, s)
                                      : select<256, false>(p, rows, 1, each, s);
  if (e != cudaSuccess) return cuda_fail(ctx, e, "paged eviction launch");
  if (!p.at_once) {
    const uint64_t lanes = most_moves * kLanes;
    const uint32_t wide = std::max(1u, uint32_t(ctx->sm_count) * 16 / rows);
    PdlLaunch v(dim3(uint32_t(std::max<uint64_t>(1, std::min<uint64_t>((lanes + 255) / 256, wide))), rows), dim3(256), 0, s);
    if (cudaError_t e = cudaLaunchKernelEx(&v.cfg, evict_move_kernel, p)) return cuda_fail(ctx, e, "paged eviction launch");
  }
  note_async_submission(ctx);
  return SI_OK;
}
