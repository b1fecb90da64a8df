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
// Selection: a cluster of 1 to 8 CTAs a (sequence, kv head); every key is read
// from global memory once and stays in shared memory for the three digits and
// the walk; histograms and counts meet over distributed shared memory. Moves: a second
// kernel over all pairs of all heads, because a cut of a long prompt
// moves megabytes where the selection is a few small scans; 16 bytes a thread
// and access. The selection is bound by latency (about five cluster barriers), the
// moves by bandwidth.
#include <cuda_runtime.h>

#include <algorithm>

#include "paged.cuh"

namespace si {
namespace {

constexpr int kThreads = 1024, kWarps = kThreads / 32;
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
  uint2* moves;      // [sequence * kv_heads + head][room] (from, to)
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
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t peer_u32(const uint32_t* p, uint32_t rank) {
  uint32_t at, v;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
  return v;
}

// Exclusive prefix of one value a thread over the CTA; *total gets the sum.
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
  uint32_t y = s_w[lane];  // kWarps == 32
  const uint32_t mine = y;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t z = __shfl_up_sync(0xffffffffu, y, o);
    if (lane >= uint32_t(o)) y += z;
  }
  *total = __shfl_sync(0xffffffffu, y, 31);
  return __shfl_sync(0xffffffffu, y - mine, w) + x - v;
}

__global__ void __launch_bounds__(kThreads, 1) evict_select_kernel(const __grid_constant__ EvictArgs a) {
  extern __shared__ uint32_t s_key[];
  __shared__ uint32_t s_bin[kBins], s_w[32], s_found[2], s_ties, s_moves[2];
  const uint32_t rank = cluster_rank(), size = cluster_size();
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
  // a CTA's slots, a multiple of 1024 so that every warp has whole rows of 32
  const uint32_t chunk = ((n + size - 1) / size + kThreads - 1) / kThreads * kThreads;
  const uint32_t lo = min(n, rank * chunk), hi = min(n, lo + chunk);
  if (leave == 0) {  // the same for the whole cluster
    if (rank == 0 && tid == 0) a.counts[row] = 0;
    for (uint32_t t = lo + tid; t < hi; t += kThreads) {
      if (a.w_out != a.w_in) a.w_out[base + t] = a.w_in[base + t];
      if (a.p_out && a.p_out != a.p_in) a.p_out[base + t] = a.p_in ? a.p_in[base + t] : int32_t(t);
    }
    return;
  }
  const int64_t next = a.next ? int64_t(a.next[b]) : int64_t(n);
  for (uint32_t t = lo + tid; t < hi; t += kThreads) {
    const int64_t pos = a.p_in ? int64_t(a.p_in[base + t]) : int64_t(t);
    const bool held = pos < int64_t(a.sink) || pos >= next - int64_t(a.recent);
    s_key[t - lo] = held ? kKeep : key_of(a.w_in[base + t]);
  }
  // the leave-th smallest key, digit by digit; `want` counts within the keys that share the digits so far
  uint32_t found = 0, mask = 0, want = leave;
  for (int digit = 0; digit < 3; ++digit) {
    const int shift = digit == 0 ? 21 : digit == 1 ? 10 : 0;
    const uint32_t bins = digit == 2 ? 1024 : kBins;
    for (uint32_t i = tid; i < bins; i += kThreads) s_bin[i] = 0;
    __syncthreads();
    for (uint32_t t = tid; t < hi - lo; t += kThreads) {
      const uint32_t k = s_key[t];
      if ((k & mask) == found) atomicAdd(&s_bin[(k >> shift) & (bins - 1)], 1u);
    }
    cluster_sync();
    // two neighbouring bins a thread, summed over the cluster
    uint32_t c0 = 0, c1 = 0;
    if (2 * tid < bins)
      for (uint32_t r = 0; r < size; ++r) {
        c0 += peer_u32(&s_bin[2 * tid], r);
        c1 += peer_u32(&s_bin[2 * tid + 1], r);
      }
    uint32_t total;
    const uint32_t before = cta_prefix(c0 + c1, s_w, &total);
    if (before < want && want <= before + c0) {
      s_found[0] = 2 * tid;
      s_found[1] = before;
    } else if (before + c0 < want && want <= before + c0 + c1) {
      s_found[0] = 2 * tid + 1;
      s_found[1] = before + c0;
    }
    cluster_sync();  // also: every CTA has read this one's bins
    found |= s_found[0] << shift;
    mask |= (bins - 1) << shift;
    want -= s_found[1];
  }
  // `want` of the keys equal to `found` leave, lowest slots first. A warp walks
  // its own run of consecutive slots.
  const uint32_t run = chunk / kWarps, w0 = min(hi, lo + w * run), w1 = min(hi, w0 + run);
  auto walk = [&](auto&& body) {
    for (uint32_t t = w0; t < w1; t += 32) body(t + lane, t + lane < w1 ? s_key[t + lane - lo] : 0u, t + lane < w1);
  };
  // number of v over the slots before this warp's, cluster-wide
  auto before_warp = [&](uint32_t v, uint32_t* s_total, uint32_t* cluster_total) {
    uint32_t total;
    const uint32_t mine = cta_prefix(lane == 0 ? v : 0u, s_w, &total);
    if (tid == 0) *s_total = total;
    cluster_sync();
    uint32_t before = 0, all = 0;
    for (uint32_t r = 0; r < size; ++r) {
      const uint32_t x = peer_u32(s_total, r);
      if (r < rank) before += x;
      all += x;
    }
    *cluster_total = all;
    return before + __shfl_sync(0xffffffffu, mine, 0);
  };
  uint32_t ties = 0, all;
  walk([&](uint32_t, uint32_t k, bool in) { ties += __popc(__ballot_sync(0xffffffffu, in && k == found)); });
  const uint32_t tie0 = before_warp(ties, &s_ties, &all);
  const uint32_t below = (1u << lane) - 1;
  uint32_t holes = 0, kept = 0, seen = tie0;
  walk([&](uint32_t t, uint32_t k, bool in) {
    const uint32_t eq = __ballot_sync(0xffffffffu, in && k == found);
    const bool gone = in && (k < found || (k == found && seen + __popc(eq & below) < want));
    seen += __popc(eq);
    holes += __popc(__ballot_sync(0xffffffffu, gone && t < m));
    kept += __popc(__ballot_sync(0xffffffffu, in && !gone && t >= m));
  });
  uint32_t moved;
  uint32_t hole0 = before_warp(holes, &s_moves[0], &moved);
  uint32_t kept0 = before_warp(kept, &s_moves[1], &all);
  seen = tie0;
  uint2* list = a.moves + uint64_t(row) * a.room;
  walk([&](uint32_t t, uint32_t k, bool in) {
    const uint32_t eq = __ballot_sync(0xffffffffu, in && k == found);
    const bool gone = in && (k < found || (k == found && seen + __popc(eq & below) < want));
    seen += __popc(eq);
    const bool hole = gone && t < m, mover = in && !gone && t >= m;
    const uint32_t hb = __ballot_sync(0xffffffffu, hole), mb = __ballot_sync(0xffffffffu, mover);
    if (hole) list[hole0 + __popc(hb & below)].y = t;
    if (mover) list[kept0 + __popc(mb & below)].x = t;
    hole0 += __popc(hb);
    kept0 += __popc(mb);
    if (in && !gone && t < m) {
      if (a.w_out != a.w_in) a.w_out[base + t] = a.w_in[base + t];
      if (a.p_out && a.p_out != a.p_in) a.p_out[base + t] = a.p_in ? a.p_in[base + t] : int32_t(t);
    }
  });
  if (rank == 0 && tid == 0) a.counts[row] = moved;
  cluster_sync();  // no CTA leaves while another may still read its counts
}

// Kept slots from behind the new length into the holes below it: sources and
// destinations do not meet, so the order is free. A thread moves 16 bytes of a
// key or a value; `parts` of them make a slot.
__global__ void __launch_bounds__(256) evict_move_kernel(const __grid_constant__ EvictArgs a, FastDiv parts) {
  const uint32_t row = blockIdx.y, b = row / a.kv.kv_heads, h = row - b * a.kv.kv_heads;
  pdl_launch_dependents();
  pdl_wait();
  if (a.len_out == a.len_in && blockIdx.x == 0 && h == 0 && threadIdx.x == 0) {
    const int32_t n = a.len_in[b];  // read and written by this thread alone
    a.len_out[b] = int32_t(min(n < 0 ? 0u : min(uint32_t(n), a.most), a.budget));
  }
  const uint32_t moved = a.counts[row];
  const uint64_t base = uint64_t(row) * a.stride;
  const uint2* list = a.moves + uint64_t(row) * a.room;
  const int32_t* pages = a.kv.pages + b * a.kv.pages_stride;
  const uint32_t chunks = a.kv.hd / 8;
  const uint64_t items = uint64_t(moved) * parts.d;
  for (uint64_t i = uint64_t(blockIdx.x) * 256 + threadIdx.x; i < items; i += uint64_t(gridDim.x) * 256) {
    const uint32_t pair = uint32_t(i / parts.d), part = uint32_t(i - uint64_t(pair) * parts.d);
    const uint2 mv = list[pair];
    const uint64_t from = paged_slot(a.kv, pages, mv.x, h), to = paged_slot(a.kv, pages, mv.y, h);
    if (from == kNoCell || to == kNoCell) {
      atomicOr(a.err, KERR_BAD_INDEX);
    } else {
      const bool is_v = part >= chunks;
      const uint16_t* src = is_v ? a.kv.v : a.kv.k;
      const uint32_t at = (is_v ? part - chunks : part) * 8;
      *reinterpret_cast<uint4*>(const_cast<uint16_t*>(src) + to + at) = *reinterpret_cast<const uint4*>(src + from + at);
    }
    if (part == 0) {
      a.w_out[base + mv.y] = a.w_in[base + mv.x];
      if (a.p_out) a.p_out[base + mv.y] = a.p_in ? a.p_in[base + mv.x] : int32_t(mv.x);
    }
  }
}

uint64_t rows_of(const si_paged_kv& kv) { return uint64_t(kv.sequences) * kv.kv_heads; }
// A list holds at most half of the slots: one of a pair is below the budget, one behind it.
uint64_t room_of(const si_paged_kv& kv) { return uint64_t(kv.max_pages) * kv.page_tokens / 2 + 1; }
uint64_t evict_bytes(const si_paged_kv& kv) {
  return ((rows_of(kv) * 4 + 15) & ~uint64_t(15)) + rows_of(kv) * room_of(kv) * sizeof(uint2);
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
  if (!a->lengths_in || !a->lengths_out || !a->weights_in || !a->weights_out)
    return bad(SI_E_INVALID, "paged eviction buffers are null");
  if (a->positions_in && !a->positions_out)
    return bad(SI_E_INVALID, "paged eviction has positions in and none out");
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
  p.moves = reinterpret_cast<uint2*>(static_cast<uint8_t*>(a->work) + ((rows_of(*kv) * 4 + 15) & ~uint64_t(15)));
  p.err = ctx->d_err;
  const cudaStream_t s = stream ? static_cast<cudaStream_t>(stream) : ctx->stream;
  const uint32_t rows = uint32_t(rows_of(*kv)), most = p.most;
  uint32_t cluster = 1;
  while (cluster < kMaxCluster && most > cluster * 8192) cluster *= 2;
  const uint32_t slots = ((most + cluster - 1) / cluster + kThreads - 1) / kThreads * kThreads;
  static std::atomic<uint32_t> cache[kMaxDevices];
  if (cudaError_t e = raise_smem_limit(evict_select_kernel, slots * 4, cache)) return cuda_fail(ctx, e, "paged eviction");
  PdlLaunch l(dim3(rows * cluster), dim3(kThreads), slots * 4, s);
  l.cluster(cluster);
  if (cudaError_t e = cudaLaunchKernelEx(&l.cfg, evict_select_kernel, p)) return cuda_fail(ctx, e, "paged eviction launch");
  const FastDiv parts = fast_div(2 * (kv->head_dim / 8));
  // moves of one row are at most the smaller of both sides of the budget
  const uint64_t items = std::min<uint64_t>(most > a->budget ? most - a->budget : 0, a->budget) * parts.d;
  const uint32_t wide = std::max(1u, uint32_t(ctx->sm_count) * 8 / rows);
  PdlLaunch v(dim3(uint32_t(std::max<uint64_t>(1, std::min<uint64_t>((items + 255) / 256, wide))), rows), dim3(256), 0, s);
  if (cudaError_t e = cudaLaunchKernelEx(&v.cfg, evict_move_kernel, p, parts)) return cuda_fail(ctx, e, "paged eviction launch");
  note_async_submission(ctx);
  return SI_OK;
}
