// Attention of one new token a sequence over a paged key-value cache.
//
// o = sum_t p_t v_t / sum_t p_t, p_t = exp(s_t - max s), s_t = scale q.k_t, for
// the query heads that share a kv head. Up to 8 query heads a kv head read every
// key and value once, so the work is bound by HBM (2 flop a byte and query head)
// once a few thousand tokens are in the batch, and by latency below that. Larger
// groups are several blocks of 8 heads, each of which reads all of them.
//
// Split. The unit of work is 16 consecutive slots of one (sequence, kv head,
// block of 8 query heads), a pair. All units of the batch, in that order, are
// shared out evenly over the workers of one resident CTA a multiprocessor,
// whatever the lengths: the counts come from lengths on the device, so a call needs no
// host copy of them and a captured call follows later lengths. A worker's share covers
// the end of one pair, some whole ones, and the beginning of another; whole
// ones are written at once, the partial ones (at most two a worker) meet in
// shared memory at the end, those that cross the CTA's borders (at most two a
// CTA) in the workspace, which a second kernel joins. Every join sums in a fixed order.
// A worker is a warp; for head_dim above 192 two warps, each with half of the
// dims, that exchange their halves of the scores once a unit (one call of 517
// slots of 256 dims 13.0 us where one warp a unit takes 14.5, 65,536 slots with bf16
// queries 53 and 56; long rows with f32 queries are 2 % slower, 131,071 slots
// 115.6 and 113, 8 rows of 8,192 with weights 62.7 and 61.3).
//
// A unit. Keys and values go from global memory straight into the registers
// in which the tensor cores (mma.m16n8k16) want them; there is no shared-memory
// stage:
//   S^T = K Q^T: the order of dims in the contraction is free as long as both
//     operands share it, so a lane's 16-byte load of 8 dims of a key is the A
//     operand of two steps. Lane (n, c) = (lane / 4, lane % 4) loads dims
//     32 s + 8 c .. + 7 of slots n and n + 8.
//   O^T = V^T P^T: the order of output rows (dims) is free too. The lane loads
//     dims 64 d + 8 n .. + 7 of slots 2c, 2c + 1, 2c + 8, 2c + 9; byte
//     permutes pair the slots, and output row r of step (d, j) is dim
//     64 d + 8 n + 2j (+ 1 for rows 8..15), so a lane ends with 8 neighbouring
//     dims of its two query heads.
//   P leaves the first product transposed; movmatrix turns it into the second
//     one's B operand.
// The keys of the next unit are requested when this unit's scores are done,
// its values step by step as this unit's are used, so loads are in flight
// throughout. What bounds it: HBM for 16-bit queries (64 ragged sequences, 0.69 GB
// in 116 us, 6.0 TB/s), the latency of a unit for f32 ones (0.54 GB in 113 us).
//
// Precision: queries are split into TQ 16-bit terms and probabilities into TP,
// each multiplied separately into f32 sums. 16-bit queries of the cache's own
// type are exact in one term, and probabilities then take 2 (16 bits in bf16, 22
// in f16: the output keeps 8 or 11). All other queries (f32, or the other 16-bit
// type) take 3 bf16 terms (24 bits) or 2 f16 terms (22 bits, after scaling each
// query by a power of two to a maximum near 2^15), and probabilities as many. In
// f16, probabilities are scaled up so that small ones keep their bits; the sum is
// taken of the same scaled values.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>

#include "paged.cuh"

namespace si {
namespace {

constexpr uint32_t kUnit = 16;  // slots of a unit
constexpr uint32_t kCols = 8;   // query heads of a block
// Beginning a pair (its queries, its first pages) and ending it costs a warp
// about as much time as this many units; shares are even in that measure.
constexpr uint32_t kPairCost = 3;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// Probabilities are 2^(score - reference + shift), below 2^(shift + slack): in
// f16 as high as its range allows.
constexpr float kSlack = 4.f;
constexpr float shift_of(bool bf16) { return bf16 ? 0.f : 11.f; }

template <int HD>
struct Shape {
  static constexpr int kSplit = HD > 192 ? 2 : 1;      // warps of a worker, a share of the dims each
  static constexpr int kDims = HD / kSplit;
  static constexpr int kWarps = kDims <= 128 ? 12 : 8;   // registers: 168 or 255 a thread
  static constexpr int kWorkers = kWarps / kSplit;
  static constexpr int kK = kDims / 32, kV = kDims / 64; // 16-byte loads a slot and lane
};

// Join records and partials in the workspace (one CTA: two partial slots).
struct Join {
  int32_t last;    // last CTA of the pair that crosses this CTA's first border; -1: none whose first border it is
  uint32_t slot0;  // partial slot of the CTA before
  uint32_t b, head;  // sequence; kv head * blocks + block
};

struct AttArgs {
  PagedView kv;
  const void* q;
  void* out;
  uint64_t q_ss, q_hs, o_ss, o_hs;
  const int32_t* lengths;
  float scale;  // times log2 e
  uint32_t elem, qh, group, blocks;
  bool q_wide, o_wide;
  float* lse;      // natural log; may be null
  float* lse2;     // log2, workspace of the weights pass; null without weights
  float* scores;   // log2 scores [b * kvh + h][slot][gpad]; null without weights
  uint32_t gpad;
  float* part;     // [ctas][2][kCols][HD + 2]
  Join* join;      // [ctas]
  int* err;
};

// 16 bytes into r if index < count, else r stays: predicated, so that loads
// stay in one run without branches between them.
__device__ __forceinline__ void ldg_if(uint4& r, const void* p, uint32_t index, uint32_t count) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.lt.u32 p, %5, %6;\n\t"
      "@p ld.global.nc.L1::no_allocate.L2::256B.v4.u32 {%0, %1, %2, %3}, [%4];\n\t}"
      : "+r"(r.x), "+r"(r.y), "+r"(r.z), "+r"(r.w)
      : "l"(p), "r"(index), "r"(count));
}
// 16 bytes to shared memory, zeros if not `on`.
__device__ __forceinline__ void cp_async16(void* dst, const void* src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(on ? 16u : 0u) : "memory");
}
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }

template <bool BF16>
__device__ __forceinline__ void mma16(float d[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
  if constexpr (BF16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The first product of a sum: nothing to add to.
template <bool BF16>
__device__ __forceinline__ void mma16_first(float d[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
  if constexpr (BF16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
// (x0, x1) += (y0, y1), rounded to nearest, in one instruction.
__device__ __forceinline__ void add2(float& x0, float& x1, float y0, float y1) {
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%0, %1};\n\tmov.b64 y, {%2, %3};\n\tadd.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "+f"(x0), "+f"(x1)
      : "f"(y0), "f"(y1));
}

// Pair (x, y) rounded to 16 bits, and what the rounding left.
template <bool BF16>
__device__ __forceinline__ uint32_t take_term(float& x, float& y) {
  if constexpr (BF16) {
    const __nv_bfloat162 r = __floats2bfloat162_rn(x, y);
    const uint32_t u = *reinterpret_cast<const uint32_t*>(&r);
    x -= __uint_as_float(u << 16);
    y -= __uint_as_float(u & 0xffff0000u);
    return u;
  } else {
    const __half2 r = __floats2half2_rn(x, y);
    const float2 f = __half22float2(r);
    x -= f.x;
    y -= f.y;
    return *reinterpret_cast<const uint32_t*>(&r);
  }
}

// 2^x, zero far below; two units in the last place.
__device__ __forceinline__ float pow2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint32_t transpose8(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

__device__ __forceinline__ uint64_t shfl64(uint64_t v, int src) {
  return __shfl_sync(0xffffffffu, v, src);
}

// The line that is shared out: the pairs (sequence, kv head, block) in order,
// each kPairCost steps and then a step for every unit. prefix[b] counts the
// steps of one head of the sequences before b; an empty sequence has none.
struct Place {
  uint32_t b, head;  // kv head * blocks + block
  uint32_t begin;    // the pair's first step
  uint32_t tiles;    // its units: steps begin + kPairCost ...
};
__device__ __forceinline__ Place place_of(uint32_t u, const uint32_t* prefix, uint32_t sequences, uint32_t heads) {
  const uint32_t t = u / heads;
  uint32_t lo = 0, hi = sequences;  // prefix[lo] <= t < prefix[hi]
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) / 2;
    if (prefix[mid] <= t) lo = mid;
    else hi = mid;
  }
  Place p;
  p.b = lo;
  const uint32_t steps = prefix[lo + 1] - prefix[lo], first = prefix[lo] * heads;
  p.head = (u - first) / steps;
  p.begin = first + p.head * steps;
  p.tiles = steps - kPairCost;
  return p;
}
__device__ __forceinline__ void next_place(Place& p, const uint32_t* prefix, uint32_t heads) {
  p.begin += p.tiles + kPairCost;
  if (++p.head < heads) return;
  p.head = 0;
  do ++p.b;
  while (prefix[p.b + 1] == prefix[p.b]);
  p.tiles = prefix[p.b + 1] - prefix[p.b] - kPairCost;
}

// prefix[0..sequences], by the whole CTA.
__device__ __forceinline__ void step_prefix(const AttArgs& a, uint32_t* prefix, uint32_t* s_warp) {
  const uint32_t lane = threadIdx.x & 31, w = threadIdx.x >> 5, nw = blockDim.x >> 5;
  uint32_t run = 0;
  if (threadIdx.x == 0) prefix[0] = 0;
  for (uint32_t base = 0; base < a.kv.sequences; base += blockDim.x) {
    const uint32_t i = base + threadIdx.x;
    uint32_t n = 0;
    if (i < a.kv.sequences) n = checked_length(a.lengths[i], a.kv.max_tokens, a.err);
    n = n ? (n + kUnit - 1) / kUnit + kPairCost : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t v = __shfl_up_sync(0xffffffffu, n, o);
      if (lane >= uint32_t(o)) n += v;
    }
    if (lane == 31) s_warp[w] = n;
    __syncthreads();
    uint32_t before = run;
    for (uint32_t j = 0; j < nw; ++j) {
      if (j < w) before += s_warp[j];
      run += s_warp[j];
    }
    if (i < a.kv.sequences) prefix[i + 1] = before + n;
    __syncthreads();
  }
}

// Even shares of `steps` for n takers: share i begins at i * steps / n.
struct Shares {
  uint32_t each, rest, n;
  __device__ __forceinline__ Shares(uint32_t steps, uint32_t takers) : each(steps / takers), rest(steps % takers), n(takers) {}
  __device__ __forceinline__ uint32_t begin(uint32_t i) const { return i * each + i * rest / n; }  // i, rest < 2^12
};

// 8 dims of a query head whose sums are complete: max (base 2), sum, values.
template <int HD>
__device__ __forceinline__ void finish(const AttArgs& a, const Place& at, uint32_t head, uint32_t chunk, float m, float l,
                                       const float* v) {
  const float inv = l == 0.f ? 0.f : 1.f / l;  // nothing left: zeros
  float o[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) o[j] = v[j] * inv;
  store8(a.out, at.b * a.o_ss + head * a.o_hs + chunk * 8, a.elem, a.o_wide, o);
  if (chunk == 0) {
    const float z = l == 0.f ? -INFINITY : m + log2f(l);
    const uint64_t i = uint64_t(at.b) * a.qh + head;
    if (a.lse) a.lse[i] = z * kLn2;
    if (a.lse2) a.lse2[i] = z;
  }
}

template <int HD, bool BF16, int TQ, int TP>
__global__ void __launch_bounds__(Shape<HD>::kWarps * 32, 1) paged_attention_kernel(const __grid_constant__ AttArgs a) {
  using Sh = Shape<HD>;
  constexpr int NW = Sh::kWarps, WK = Sh::kWorkers, KK = Sh::kK, KV = Sh::kV;
  constexpr float kShift = shift_of(BF16);
  constexpr uint32_t kPart = kCols * (HD + 2);                   // floats of a partial: values, then max and sum
  constexpr uint32_t kQ = uint32_t(TQ * KK) * 32 * 4;            // floats of a warp's query terms
  constexpr uint32_t kRegion = (kQ * Sh::kSplit > kPart ? kQ * Sh::kSplit : kPart) + kPart;
  extern __shared__ __align__(16) float smem[];
  // per worker: [query terms, later the partial of the last pair][partial of the first pair]
  __shared__ uint32_t s_warp[NW];
  __shared__ Place s_part[2 * WK];  // pairs of the workers' partials; tiles 0: no partial
  __shared__ float4 s_half[Sh::kSplit > 1 ? WK : 1][2][Sh::kSplit][32];  // scores over a share of the dims
  __shared__ uint8_t s_list[32], s_lead[32];
  __shared__ uint32_t s_leads;
  uint32_t* prefix = reinterpret_cast<uint32_t*>(smem + WK * kRegion);
  const uint32_t lane = threadIdx.x & 31, w = threadIdx.x >> 5, n8 = lane >> 2, c4 = lane & 3;
  const uint32_t heads = a.kv.kv_heads * a.blocks;
  if (threadIdx.x < 2 * WK) s_part[threadIdx.x].tiles = 0;
  pdl_launch_dependents();
  pdl_wait();
  step_prefix(a, prefix, s_warp);
  const uint32_t steps = prefix[a.kv.sequences] * heads;
  // rows of empty sequences
  for (uint32_t b = blockIdx.x; b < a.kv.sequences; b += gridDim.x) {
    if (prefix[b + 1] != prefix[b]) continue;
    const float zero[8] = {};
    for (uint32_t i = threadIdx.x; i < a.qh * (a.kv.hd / 8); i += NW * 32) {
      const uint32_t h = i / (a.kv.hd / 8), ch = i - h * (a.kv.hd / 8);
      store8(a.out, b * a.o_ss + h * a.o_hs + ch * 8, a.elem, a.o_wide, zero);
    }
    if (a.lse)
      for (uint32_t h = threadIdx.x; h < a.qh; h += NW * 32) a.lse[uint64_t(b) * a.qh + h] = -INFINITY;
  }
  // little work: fewer CTAs, so that most workers still have a unit
  const uint32_t ctas = min(gridDim.x, steps / WK + (steps % WK != 0)), cta = blockIdx.x;
  if (cta >= ctas) {
    if (threadIdx.x == 0) a.join[cta].last = -1;
    return;
  }
  const Shares cta_share(steps, ctas), worker_share(steps, ctas * WK);
  const uint32_t cu0 = cta_share.begin(cta), cu1 = cta_share.begin(cta + 1);
  const uint32_t worker = w / Sh::kSplit, half = w % Sh::kSplit, dim0 = half * Sh::kDims;
  const uint32_t u0 = worker_share.begin(cta * WK + worker), u1 = worker_share.begin(cta * WK + worker + 1);
  float* region = smem + worker * kRegion;
  uint4* s_q = reinterpret_cast<uint4*>(region + half * kQ) + lane;  // [step][term][lane]: a lane reads what it wrote
  const uint32_t chunks = a.kv.hd / 8, mine = min(uint32_t(Sh::kDims / 8), chunks - dim0 / 8);
  // steps in which the lane has dims below head_dim
  const uint32_t k_steps = (mine + 3 - c4) / 4, v_steps = (mine + 7 - n8) / 8;
  auto worker_sync = [&] {
    if constexpr (Sh::kSplit == 1)
      __syncwarp();
    else
      asm volatile("bar.sync %0, %1;" ::"r"(1 + worker), "n"(Sh::kSplit * 32) : "memory");
  };
  uint32_t flip = 0;  // which half of s_half the next unit uses

  Place at;
  if (u0 < u1) at = place_of(u0, prefix, a.kv.sequences, heads);
  uint4 kr[2][KK] = {}, vr[4][KV] = {};  // places that no load fills (dims past head_dim) stay zero
  for (uint32_t u = u0; u < u1; u = at.begin + at.tiles + kPairCost, u < u1 ? next_place(at, prefix, heads) : void()) {
    const uint32_t first = at.begin + kPairCost;
    const uint32_t t_begin = u > first ? u - first : 0, t_end = min(u1, first + at.tiles) - first;
    if (u1 <= first || t_begin >= t_end) continue;  // the share ends before the pair's units
    const uint32_t kvh = at.head / a.blocks, col0 = (at.head - kvh * a.blocks) * kCols;
    const uint32_t cols = min(kCols, a.group - col0), qhead0 = kvh * a.group + col0;
    const int32_t* row = a.kv.pages + at.b * a.kv.pages_stride;

    // The page of slot (unit, lane % 16), asked for two units ahead of its use.
    auto page_of = [&](uint32_t tile) -> int32_t {
      const uint32_t t = tile * kUnit + (lane & 15);
      return tile < t_end && t < a.kv.max_tokens ? __ldg(row + div_of(t, a.kv.page)) : -1;
    };
    int32_t page_next = page_of(t_begin + 1);
    const int32_t page_first = page_of(t_begin);
    const uint32_t len = checked_length(a.lengths[at.b], a.kv.max_tokens, a.err);
    // Queries as they are, each lane's own into its places of shared memory;
    // rolled loops here and at the pair's end: code that runs once a pair costs
    // its instruction fetches.
    const uint64_t q0 = at.b * a.q_ss + uint64_t(qhead0 + n8) * a.q_hs + dim0;
    if (a.q_wide) {
      const uint8_t* from = static_cast<const uint8_t*>(a.q) + q0 * elem_bytes(a.elem);
#pragma unroll 1
      for (uint32_t s = 0; s < KK; ++s) {
        const uint32_t ch = 4 * s + c4;
        const bool on = n8 < cols && ch < mine;
        const uint8_t* x = on ? from + ch * 8 * elem_bytes(a.elem) : static_cast<const uint8_t*>(a.q);
        cp_async16(s_q + s * TQ * 32, x, on);
        if (TQ > 1 && a.elem == SI_ELEM_F32) cp_async16(s_q + (s * TQ + 1) * 32, on ? x + 16 : x, on);
      }
    }
    auto cell_of = [&](uint32_t tile, int32_t page) -> uint64_t {
      const uint32_t t = tile * kUnit + (lane & 15);
      const bool on = tile < t_end && t < len;
      const uint64_t cell = on ? paged_cell(a.kv, page, t - div_of(t, a.kv.page) * a.kv.page.d, kvh) : kNoCell;
      if (on && cell == kNoCell) atomicOr(a.err, KERR_BAD_INDEX);
      return cell;
    };
    auto load_k = [&](uint64_t cell, bool& lo, bool& hi) {
      const uint64_t c0 = shfl64(cell, n8), c1 = shfl64(cell, n8 + 8);
      lo = c0 != kNoCell;
      hi = c1 != kNoCell;
      const uint16_t *p0 = a.kv.k + c0 + dim0 + c4 * 8, *p1 = a.kv.k + c1 + dim0 + c4 * 8;
      const uint32_t n0 = lo ? k_steps : 0, n1 = hi ? k_steps : 0;
#pragma unroll
      for (uint32_t s = 0; s < KK; ++s) {
        ldg_if(kr[0][s], p0 + s * 32, s, n0);
        ldg_if(kr[1][s], p1 + s * 32, s, n1);
      }
    };
    // A step's registers of the values are asked for again as soon as the step has used them.
    const uint16_t* vp[4];
    uint32_t vn[4];
    bool v_gap = false;
    auto rows_v = [&](uint64_t cell) {
      v_gap = __any_sync(0xffffffffu, cell == kNoCell);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint64_t c = shfl64(cell, 2 * c4 + (i & 1) + (i >> 1) * 8);
        vp[i] = a.kv.v + c + dim0 + n8 * 8;
        vn[i] = c != kNoCell ? v_steps : 0;
      }
    };
    auto load_v = [&](uint32_t d) {
      // slots that do not exist meet probability 0, and need a finite value
      if (v_gap) {
#pragma unroll
        for (int i = 0; i < 4; ++i) vr[i][d] = make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) ldg_if(vr[i][d], vp[i] + d * 64, d, vn[i]);
    };
    bool lo, hi;
    uint64_t cell = cell_of(t_begin, page_first);
    load_k(cell, lo, hi);
    rows_v(cell);
#pragma unroll
    for (uint32_t d = 0; d < KV; ++d) load_v(d);
    // queries into 16-bit terms, in place; columns past the group are zero
    auto raw = [&](uint32_t s, float x[8]) {
      const uint32_t ch = 4 * s + c4;
      if (a.q_wide) {
        const uint4 r = s_q[s * TQ * 32];
        if (TQ > 1 && a.elem == SI_ELEM_F32) {
          const uint4 z = s_q[(s * TQ + 1) * 32];
          x[0] = as_f(r.x), x[1] = as_f(r.y), x[2] = as_f(r.z), x[3] = as_f(r.w);
          x[4] = as_f(z.x), x[5] = as_f(z.y), x[6] = as_f(z.z), x[7] = as_f(z.w);
        } else {
          const uint32_t h[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
          for (int j = 0; j < 8; ++j) x[j] = elem_to_f(uint16_t(h[j / 2] >> (j % 2 * 16)), a.elem);
        }
      } else if (n8 < cols && ch < mine) {
        load8(a.q, q0 + ch * 8, a.elem, false, x);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = 0.f;
      }
    };
    cp_async_wait();
    float col_scale = a.scale, down = 1.f;
    if constexpr (!BF16) {  // to a maximum in [2^14, 2^15): small elements beside large ones keep their bits
      float big = 0.f;
#pragma unroll 1
      for (uint32_t s = 0; s < KK; ++s) {
        float x[8];
        raw(s, x);
#pragma unroll
        for (int j = 0; j < 8; ++j) big = fmaxf(big, fabsf(x[j]));
      }
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
      int e = 0;
      if (big > 0.f && big < INFINITY) e = max(-100, ilogbf(big)) - 14;
      down = ldexpf(1.f, -e);
      col_scale *= ldexpf(1.f, e);
    }
#pragma unroll 1
    for (uint32_t s = 0; s < KK; ++s) {
      float x[8];
      raw(s, x);
      if constexpr (!BF16) {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] *= down;
      }
#pragma unroll
      for (int t = 0; t < TQ; ++t) {
        uint4 r;
        r.x = take_term<BF16>(x[0], x[1]);
        r.y = take_term<BF16>(x[2], x[3]);
        r.z = take_term<BF16>(x[4], x[5]);
        r.w = take_term<BF16>(x[6], x[7]);
        s_q[(s * TQ + t) * 32] = r;
      }
    }
    // scale of the lane's two columns of S^T
    const float sc0 = __shfl_sync(0xffffffffu, col_scale, c4 * 8), sc1 = __shfl_sync(0xffffffffu, col_scale, c4 * 8 + 4);

    float acc[KV * 4][4] = {};
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
    for (uint32_t tile = t_begin; tile < t_end; ++tile) {
      const int32_t page_after = page_of(tile + 2);
      // Several chains of dependent products, two a term: shorter ones, fewer
      // roundings of a large sum, and small terms are not lost in large ones.
      float s[4], chain[2 * TQ - 1][4];
#pragma unroll
      for (int st = 0; st < KK; ++st) {
        const uint4 x = kr[0][st], y = kr[1][st];
        const uint32_t a0[4] = {x.x, y.x, x.y, y.y}, a1[4] = {x.z, y.z, x.w, y.w};
#pragma unroll
        for (int t = 0; t < TQ; ++t) {
          const uint4 qv = s_q[(st * TQ + t) * 32];
          if (st == 0) {
            mma16_first<BF16>(t ? chain[2 * t - 1] : s, a0, qv.x, qv.y);
            mma16_first<BF16>(chain[2 * t], a1, qv.z, qv.w);
          } else {
            mma16<BF16>(t ? chain[2 * t - 1] : s, a0, qv.x, qv.y);
            mma16<BF16>(chain[2 * t], a1, qv.z, qv.w);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float low = 0.f;
#pragma unroll
        for (int t = TQ - 1; t > 0; --t) low += chain[2 * t - 1][i] + chain[2 * t][i];
        s[i] += chain[0][i] + low;
      }
      // base-2 scores; over half of the dims, the other half's are added
      s[0] *= sc0, s[1] *= sc1, s[2] *= sc0, s[3] *= sc1;
      if constexpr (Sh::kSplit > 1) s_half[worker][flip][half][lane] = make_float4(s[0], s[1], s[2], s[3]);
      const bool lo_now = lo, hi_now = hi;
      cell = cell_of(tile + 1, page_next);
      page_next = page_after;
      load_k(cell, lo, hi);
      if constexpr (Sh::kSplit > 1) {
        worker_sync();  // the only one a unit: the other half of s_half is used next
        const float4 x = s_half[worker][flip][0][lane], y = s_half[worker][flip][1][lane];
        s[0] = x.x + y.x, s[1] = x.y + y.y, s[2] = x.z + y.z, s[3] = x.w + y.w;
        flip ^= 1;
      }
      // slots that do not exist leave nothing
      if (!lo_now) s[0] = s[1] = -INFINITY;
      if (!hi_now) s[2] = s[3] = -INFINITY;
      if (a.scores && half == 0) {
        float* to = a.scores + (uint64_t(at.b * a.kv.kv_heads + kvh) * a.kv.max_tokens + tile * kUnit) * a.gpad + col0 + 2 * c4;
        if (2 * c4 < cols) {  // gpad is even: the pair's second place exists
          if (tile * kUnit + n8 < len) *reinterpret_cast<float2*>(to + uint64_t(n8) * a.gpad) = make_float2(s[0], s[1]);
          if (tile * kUnit + n8 + 8 < len)
            *reinterpret_cast<float2*>(to + uint64_t(n8 + 8) * a.gpad) = make_float2(s[2], s[3]);
        }
      }
      // The reference point of the exponents follows the maximum only when a score
      // passes it by more than kSlack: that is seldom after the first units, and
      // a vote is cheaper than the maximum over the lanes.
      float x0 = fmaxf(s[0], s[2]), x1 = fmaxf(s[1], s[3]);
      if (__any_sync(0xffffffffu, x0 > m0 + kSlack || x1 > m1 + kSlack)) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
          x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, o));
          x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, o));
        }
        const float g0 = fmaxf(m0, x0), g1 = fmaxf(m1, x1);
        const float f0 = m0 == -INFINITY ? 0.f : exp2f(m0 - g0), f1 = m1 == -INFINITY ? 0.f : exp2f(m1 - g1);
        m0 = g0;
        m1 = g1;
        l0 *= f0;
        l1 *= f1;
#pragma unroll
        for (int i = 0; i < KV * 4; ++i) {
          acc[i][0] *= f0;
          acc[i][1] *= f1;
          acc[i][2] *= f0;
          acc[i][3] *= f1;
        }
      }
      const float b0 = m0 == -INFINITY ? 0.f : m0 - kShift, b1 = m1 == -INFINITY ? 0.f : m1 - kShift;
      float p[4] = {pow2(s[0] - b0), pow2(s[1] - b1), pow2(s[2] - b0), pow2(s[3] - b1)};
      l0 += p[0] + p[2];
      l1 += p[1] + p[3];
      uint32_t pb[TP][2];
#pragma unroll
      for (int t = 0; t < TP; ++t) {
        pb[t][0] = transpose8(take_term<BF16>(p[0], p[1]));
        pb[t][1] = transpose8(take_term<BF16>(p[2], p[3]));
      }
      rows_v(cell);
#pragma unroll
      for (int d = 0; d < KV; ++d) {
        const uint32_t v0[4] = {vr[0][d].x, vr[0][d].y, vr[0][d].z, vr[0][d].w};
        const uint32_t v1[4] = {vr[1][d].x, vr[1][d].y, vr[1][d].z, vr[1][d].w};
        const uint32_t v2[4] = {vr[2][d].x, vr[2][d].y, vr[2][d].z, vr[2][d].w};
        const uint32_t v3[4] = {vr[3][d].x, vr[3][d].y, vr[3][d].z, vr[3][d].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t av[4] = {__byte_perm(v0[j], v1[j], 0x5410), __byte_perm(v0[j], v1[j], 0x7632),
                                  __byte_perm(v2[j], v3[j], 0x5410), __byte_perm(v2[j], v3[j], 0x7632)};
          // The tensor core cuts its sums off: the unit's products are summed by
          // themselves and added, rounded, to the running sum. Left in the tensor
          // core, a row of 131,072 slots fell short by 9e-4, more than f16 rounds
          // off; this costs 0.7 us of 115 (64 ragged sequences).
          float o[4];
          mma16_first<BF16>(o, av, pb[TP - 1][0], pb[TP - 1][1]);
#pragma unroll
          for (int t = TP - 2; t >= 0; --t) mma16<BF16>(o, av, pb[t][0], pb[t][1]);
          add2(acc[d * 4 + j][0], acc[d * 4 + j][1], o[0], o[1]);
          add2(acc[d * 4 + j][2], acc[d * 4 + j][3], o[2], o[3]);
        }
        load_v(d);
      }
    }
    // sums of the lane's two columns over the slots
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) {
      l0 += __shfl_xor_sync(0xffffffffu, l0, o);
      l1 += __shfl_xor_sync(0xffffffffu, l1, o);
    }
    // The first pair's partial lies beside the queries; another one's lies over
    // them, as does a whole pair on its way out.
    const bool whole = t_begin == 0 && t_end == at.tiles;
    const uint32_t slot = u == u0 && !whole ? 0 : 1;
    float* part = slot ? region : region + (kRegion - kPart);
    worker_sync();  // all have read their queries
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const uint32_t col = 2 * c4 + c;
#pragma unroll
      for (int d = 0; d < KV; ++d) {
        float* to = part + col * HD + dim0 + (8 * d + n8) * 8;
        *reinterpret_cast<float4*>(to) =
            make_float4(acc[d * 4][c], acc[d * 4][2 + c], acc[d * 4 + 1][c], acc[d * 4 + 1][2 + c]);
        *reinterpret_cast<float4*>(to + 4) =
            make_float4(acc[d * 4 + 2][c], acc[d * 4 + 2][2 + c], acc[d * 4 + 3][c], acc[d * 4 + 3][2 + c]);
      }
      if (n8 == 0 && half == 0)
        *reinterpret_cast<float2*>(part + kCols * HD + 2 * col) = make_float2(c ? m1 : m0, c ? l1 : l0);
    }
    if (!whole) {
      if (half == 0 && lane == 0) s_part[2 * worker + slot] = at;
      continue;
    }
    worker_sync();
#pragma unroll 1
    for (uint32_t i = half * 32 + lane; i < cols * chunks; i += Sh::kSplit * 32) {
      const uint32_t col = i / chunks, ch = i - col * chunks;
      const float2 ml = *reinterpret_cast<const float2*>(part + kCols * HD + 2 * col);
      finish<HD>(a, at, qhead0 + col, ch, ml.x - kShift, ml.y, part + col * HD + ch * 8);
    }
    worker_sync();
  }
  if (threadIdx.x == 0) {
    Join j = {-1, 0, 0, 0};
    if (cta > 0) {
      const Place p = place_of(cu0, prefix, a.kv.sequences, heads);
      const uint32_t first = p.begin + kPairCost, end = first + p.tiles, before = cta_share.begin(cta - 1);
      if (first < cu0 && (before <= first)) {  // the first border among this pair's units
        j.slot0 = p.begin <= before ? 0 : 1;
        uint32_t last = cta;
        for (uint32_t step = 128; step; step >>= 1)  // whose share holds step end - 1
          if (last + step < ctas && cta_share.begin(last + step) < end) last += step;
        j.last = int32_t(last);
        j.b = p.b;
        j.head = p.head;
      }
    }
    a.join[cta] = j;
  }
  __syncthreads();
  // Join the workers' partials in the order of their units. Warp 0 lists them:
  // s_list[k] is the k-th partial, s_lead[i] the first one of the i-th pair.
  if (w == 0) {
    const Place p = s_part[lane < 2 * WK ? lane : 0];
    const bool on = lane < 2 * WK && p.tiles != 0;
    const uint32_t all = __ballot_sync(0xffffffffu, on), below = all & ((1u << lane) - 1);
    const uint32_t before = __shfl_sync(0xffffffffu, p.begin, below ? 31 - __clz(below) : 0);
    const uint32_t leads = __ballot_sync(0xffffffffu, on && (!below || before != p.begin));
    if (on) s_list[__popc(below)] = uint8_t(lane);
    if (leads >> lane & 1) s_lead[__popc(leads & ((1u << lane) - 1))] = uint8_t(__popc(below));
    if (lane == 0) {
      s_leads = __popc(leads);
      s_lead[__popc(leads)] = uint8_t(__popc(all));
    }
  }
  __syncthreads();
  constexpr uint32_t kItems = kCols * (HD / 8);
  auto part_of = [&](uint32_t k) {
    const uint32_t x = s_list[k];
    return smem + (x / 2) * kRegion + (x % 2 ? 0 : kRegion - kPart);
  };
  for (uint32_t i = threadIdx.x; i < s_leads * kItems; i += NW * 32) {
    const uint32_t g = i / kItems, col = i % kItems / (HD / 8), ch = i % (HD / 8);
    const uint32_t k0 = s_lead[g], k1 = s_lead[g + 1];
    const Place at = s_part[s_list[k0]];
    const uint32_t kvh = at.head / a.blocks, col0 = (at.head - kvh * a.blocks) * kCols;
    const uint32_t cols = min(kCols, a.group - col0), qhead0 = kvh * a.group + col0;
    if (col >= cols) continue;
    float m = -INFINITY, l = 0.f, o[8] = {};
    for (uint32_t k = k0; k < k1; ++k) m = fmaxf(m, part_of(k)[kCols * HD + 2 * col]);
#pragma unroll 4
    for (uint32_t k = k0; k < k1; ++k) {
      const float* from = part_of(k);
      const float2 ml = *reinterpret_cast<const float2*>(from + kCols * HD + 2 * col);
      const float f = ml.x == -INFINITY ? 0.f : exp2f(ml.x - m);
      l += ml.y * f;
      const float4 v0 = *reinterpret_cast<const float4*>(from + col * HD + ch * 8);
      const float4 v1 = *reinterpret_cast<const float4*>(from + col * HD + ch * 8 + 4);
      const float v[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] += v[j] * f;
    }
    const uint32_t first = at.begin + kPairCost;
    if (first >= cu0 && first + at.tiles <= cu1) {
      if (ch < chunks) finish<HD>(a, at, qhead0 + col, ch, m - kShift, l, o);
    } else {
      float* part = a.part + (uint64_t(cta) * 2 + (at.begin <= cu0 ? 0 : 1)) * kPart;
      *reinterpret_cast<float4*>(part + col * HD + ch * 8) = make_float4(o[0], o[1], o[2], o[3]);
      *reinterpret_cast<float4*>(part + col * HD + ch * 8 + 4) = make_float4(o[4], o[5], o[6], o[7]);
      if (ch == 0) {
        part[kCols * HD + 2 * col] = m;
        part[kCols * HD + 2 * col + 1] = l;
      }
    }
  }
}

// Joins the partials of the pairs that cross CTA borders. Block (i, column):
// the pair whose first border is the one before CTA i + 1, one query head of
// it. A pair may lie in as many partials as there are CTAs: a batch's loads are
// all in flight. Most blocks find nothing to join, so the blocks are small and
// all resident at once (1024 threads a block took 3 us longer at 147 x 6 blocks).
constexpr int kJoinBatch = 16;
template <int HD>
__global__ void __launch_bounds__(HD >= 192 ? HD : 256) paged_join_kernel(const __grid_constant__ AttArgs a, float shift) {
  constexpr int kJoinGroups = HD >= 192 ? 1 : 256 / HD;
  constexpr uint32_t kPart = kCols * (HD + 2);
  __shared__ float s_o[kJoinGroups][HD], s_m[kJoinGroups], s_l[kJoinGroups];
  pdl_launch_dependents();
  pdl_wait();
  const Join j = a.join[blockIdx.x + 1];
  if (j.last < 0) return;
  const uint32_t kvh = j.head / a.blocks, col0 = (j.head - kvh * a.blocks) * kCols, col = blockIdx.y;
  if (col >= min(kCols, a.group - col0)) return;
  const uint32_t first = blockIdx.x, d = threadIdx.x % HD, grp = threadIdx.x / HD;  // first: the CTA before the border
  float m = -INFINITY, l = 0.f, o = 0.f;
  for (uint32_t c = first + grp; c <= uint32_t(j.last); c += kJoinGroups * kJoinBatch) {
    float mx[kJoinBatch], lx[kJoinBatch], vx[kJoinBatch];
#pragma unroll
    for (int i = 0; i < kJoinBatch; ++i) {
      const uint32_t x = c + i * kJoinGroups;
      mx[i] = -INFINITY, lx[i] = 0.f, vx[i] = 0.f;
      if (x <= uint32_t(j.last)) {
        const float* p = a.part + (uint64_t(x) * 2 + (x == first ? j.slot0 : 0)) * kPart;
        const float2 ml = *reinterpret_cast<const float2*>(p + kCols * HD + 2 * col);
        mx[i] = ml.x;
        lx[i] = ml.y;
        vx[i] = p[col * HD + d];
      }
    }
    float g = m;
#pragma unroll
    for (int i = 0; i < kJoinBatch; ++i) g = fmaxf(g, mx[i]);
    if (g == -INFINITY) continue;
    const float f = exp2f(m - g);
    l *= f;
    o *= f;
    m = g;
#pragma unroll
    for (int i = 0; i < kJoinBatch; ++i) {
      const float f = exp2f(mx[i] - g);
      l += f * lx[i];
      o += f * vx[i];
    }
  }
  s_o[grp][d] = o;
  if (d == 0) s_m[grp] = m, s_l[grp] = l;
  __syncthreads();
  if (grp) return;
#pragma unroll
  for (int i = 1; i < kJoinGroups; ++i) {
    const float mi = s_m[i];
    if (mi == -INFINITY) continue;
    const float g = fmaxf(m, mi), f0 = exp2f(m - g), f1 = exp2f(mi - g);
    m = g;
    l = l * f0 + s_l[i] * f1;
    o = o * f0 + s_o[i][d] * f1;
  }
  const uint32_t head = kvh * a.group + col0 + col;
  if (d < a.kv.hd) {
    const uint64_t at = j.b * a.o_ss + head * a.o_hs + d;
    const float v = l == 0.f ? 0.f : o / l;
    if (a.elem == SI_ELEM_F32) static_cast<float*>(a.out)[at] = v;
    else static_cast<uint16_t*>(a.out)[at] = f_to_elem(v, a.elem);
  }
  if (d == 0) {
    const float z = l == 0.f ? -INFINITY : m - shift + log2f(l);
    const uint64_t y = uint64_t(j.b) * a.qh + head;
    if (a.lse) a.lse[y] = z * kLn2;
    if (a.lse2) a.lse2[y] = z;
  }
}

// weights_out = weights_in + the group's probabilities, from the stored scores.
__global__ void __launch_bounds__(256) paged_weights_kernel(const __grid_constant__ AttArgs a, const float* w_in,
                                                            float* w_out, uint64_t stride) {
  pdl_launch_dependents();
  pdl_wait();
  const uint32_t row = blockIdx.y, b = row / a.kv.kv_heads, h = row - b * a.kv.kv_heads;
  const uint32_t len = checked_length(a.lengths[b], uint32_t(min(uint64_t(a.kv.max_tokens), stride)), a.err);
  const float* z = a.lse2 + uint64_t(b) * a.qh + h * a.group;
  for (uint32_t t = blockIdx.x * 256 + threadIdx.x; t < len; t += gridDim.x * 256) {
    const float* s = a.scores + (uint64_t(row) * a.kv.max_tokens + t) * a.gpad;
    float sum = 0.f;
    for (uint32_t g = 0; g < a.group; g += 2) {
      const float2 x = *reinterpret_cast<const float2*>(s + g);
      // a score of -inf is a slot that was left out: it has no weight
      sum += x.x == -INFINITY ? 0.f : exp2f(x.x - z[g]);
      if (g + 1 < a.group) sum += x.y == -INFINITY ? 0.f : exp2f(x.y - z[g + 1]);
    }
    const uint64_t i = uint64_t(row) * stride + t;
    w_out[i] = (w_in ? w_in[i] : 0.f) + sum;
  }
}

uint32_t padded_dim(uint32_t hd) { return (hd + 63) / 64 * 64; }
uint32_t workers_of(uint32_t hd) { return padded_dim(hd) <= 128 ? 12 : padded_dim(hd) <= 192 ? 8 : 6; }

// Workspace: join records, partials, then lse and scores of the weights pass.
// The grid is one CTA a multiprocessor, so kMaxCtas bounds both.
constexpr uint32_t kMaxCtas = 256;
uint64_t part_bytes(uint32_t hd) { return uint64_t(kMaxCtas) * 2 * kCols * (padded_dim(hd) + 2) * 4; }
uint64_t round16(uint64_t n) { return (n + 15) & ~uint64_t(15); }
uint64_t work_bytes(const si_paged_kv& kv, uint32_t qh, bool weights) {
  uint64_t n = kMaxCtas * sizeof(Join) + part_bytes(kv.head_dim);
  if (weights) {
    const uint32_t group = qh / kv.kv_heads, gpad = (group + 1) & ~1u;
    n += round16(uint64_t(kv.sequences) * qh * 4);
    n += uint64_t(kv.sequences) * kv.kv_heads * kv.max_pages * kv.page_tokens * gpad * 4;
  }
  return n;
}

// Steps of the line that is shared out, if every sequence fills its pages.
uint64_t most_steps(const si_paged_kv& kv, uint32_t qh) {
  const uint64_t blocks = (qh / kv.kv_heads + kCols - 1) / kCols;
  const uint64_t tiles = (uint64_t(kv.max_pages) * kv.page_tokens + kUnit - 1) / kUnit + kPairCost;
  const unsigned __int128 n = (unsigned __int128)tiles * kv.sequences * kv.kv_heads * blocks;
  return n >> 64 ? ~uint64_t(0) : uint64_t(n);
}

int check_heads(const si_paged_kv* kv, uint32_t qh, std::string* msg) {
  if (int rc = check_paged_kv(kv, msg)) return rc;
  if (qh == 0 || qh % kv->kv_heads || qh > 65535) {
    *msg = "paged attention query heads must be a multiple of the kv heads";
    return SI_E_INVALID;
  }
  if (most_steps(*kv, qh) > 0xffffffffull) {
    *msg = "paged attention takes page tables of less than 2^32 units of 16 slots, over all sequences and heads";
    return SI_E_UNSUPPORTED;
  }
  return SI_OK;
}

int check_attention(const si_paged_kv* kv, const si_paged_attention* a, std::string* msg) {
  auto bad = [&](int rc, const std::string& text) {
    *msg = text;
    return rc;
  };
  if (!a) return bad(SI_E_INVALID, "null paged attention description");
  if (int rc = check_heads(kv, a->query_heads, msg)) return rc;
  if (!elem_known(a->elem)) return bad(SI_E_UNSUPPORTED, "paged attention elements must be f32, bf16 or f16");
  if (!a->q || !a->out || !a->lengths) return bad(SI_E_INVALID, "paged attention buffers are null");
  if (!elem_aligned(a->q, a->elem) || !elem_aligned(a->out, a->elem) ||
      !words_aligned({a->lengths, a->lse, a->weights_in, a->weights_out}))
    return bad(SI_E_INVALID, "paged attention buffers are not aligned to their elements");
  if (!(a->scale >= 0.f) || a->scale > 3e38f) return bad(SI_E_INVALID, "paged attention scale must be finite and not negative");
  if (a->weights_in && !a->weights_out) return bad(SI_E_INVALID, "paged attention has weights in and none out");
  for (uint64_t s : {a->q_seq_stride, a->q_head_stride, a->out_seq_stride, a->out_head_stride, a->weights_stride})
    if (s >> 44) return bad(SI_E_INVALID, "paged attention strides are out of range");
  const BufferRows q = {a->q, kv->sequences, a->q_seq_stride, a->query_heads, a->q_head_stride, kv->head_dim, a->elem};
  const BufferRows out = {a->out, kv->sequences, a->out_seq_stride, a->query_heads, a->out_head_stride, kv->head_dim, a->elem};
  if (!rows_distinct(out)) return bad(SI_E_INVALID, "paged attention output rows overlap");
  if (rows_meet(q, out)) return bad(SI_E_INVALID, "paged attention cannot write its output over the queries");
  if (a->weights_out && a->weights_stride == 0) return bad(SI_E_INVALID, "paged attention weights have no stride");
  if (a->weights_out && uint64_t(kv->sequences) * kv->kv_heads > 65535)
    return bad(SI_E_UNSUPPORTED, "paged attention weights take at most 65535 sequences times kv heads");
  const uint64_t need = work_bytes(*kv, a->query_heads, a->weights_out != nullptr);
  if (!a->work || reinterpret_cast<uintptr_t>(a->work) % 16 || a->work_bytes < need)
    return bad(SI_E_INVALID, "paged attention needs " + std::to_string(need) + " bytes of 16-byte aligned workspace");
  return SI_OK;
}

template <int HD, bool BF16, int TQ, int TP>
cudaError_t launch(const AttArgs& p, uint32_t grid, cudaStream_t s) {
  using Sh = Shape<HD>;
  constexpr uint32_t kPart = kCols * (HD + 2), kQ = uint32_t(TQ * Sh::kK) * 32 * 4 * Sh::kSplit;
  constexpr uint32_t kRegion = (kQ > kPart ? kQ : kPart) + kPart;
  const uint32_t smem = Sh::kWorkers * kRegion * 4 + (p.kv.sequences + 1) * 4;
  static RaisedLimit limits[kMaxDevices];
  auto kernel = paged_attention_kernel<HD, BF16, TQ, TP>;
  if (cudaError_t e = raise_smem_limit(kernel, smem, limits)) return e;
  PdlLaunch l(dim3(grid), dim3(Shape<HD>::kWarps * 32), smem, s);
  if (cudaError_t e = cudaLaunchKernelEx(&l.cfg, kernel, p)) return e;
  if (grid == 1) return cudaSuccess;
  PdlLaunch j(dim3(grid - 1, std::min(kCols, p.group)), dim3(HD >= 192 ? HD : 256), 0, s);
  return cudaLaunchKernelEx(&j.cfg, paged_join_kernel<HD>, p, shift_of(BF16));
}

template <int HD>
cudaError_t launch_hd(const AttArgs& p, bool bf16, uint32_t grid, cudaStream_t s) {
  if (bf16) {
    if (p.elem == SI_ELEM_BF16) return launch<HD, true, 1, 2>(p, grid, s);
    return launch<HD, true, 3, 3>(p, grid, s);
  }
  if (p.elem == SI_ELEM_F16) return launch<HD, false, 1, 2>(p, grid, s);
  return launch<HD, false, 2, 2>(p, grid, s);
}

}  // namespace
}  // namespace si

using namespace si;

extern "C" int si_paged_attention_workspace(const si_paged_kv* kv, uint32_t query_heads, int weights, uint64_t* bytes) {
  std::string msg;
  if (int rc = check_heads(kv, query_heads, &msg)) return fail(nullptr, rc, msg);
  if (!bytes) return fail(nullptr, SI_E_INVALID, "null workspace size");
  *bytes = work_bytes(*kv, query_heads, weights != 0);
  return SI_OK;
}

extern "C" int si_paged_attention_dev(si_ctx* ctx, const si_paged_kv* kv, const si_paged_attention* a, void* stream) {
  std::string msg;
  if (int rc = check_attention(kv, a, &msg)) return fail(ctx, rc, msg);
  if (!ctx) return fail(nullptr, SI_E_INVALID, "null context");
  DeviceGuard dev(ctx->device);
  if (dev.e != cudaSuccess) return cuda_fail(ctx, dev.e, "paged attention device");
  AttArgs p = {};
  p.kv = paged_view(*kv);
  p.q = a->q, p.out = a->out;
  p.q_ss = a->q_seq_stride, p.q_hs = a->q_head_stride, p.o_ss = a->out_seq_stride, p.o_hs = a->out_head_stride;
  p.lengths = a->lengths;
  p.scale = (a->scale > 0.f ? a->scale : 1.f / std::sqrt(float(kv->head_dim))) * kLog2e;
  p.elem = a->elem;
  p.qh = a->query_heads;
  p.group = a->query_heads / kv->kv_heads;
  p.blocks = (p.group + kCols - 1) / kCols;
  p.q_wide = wide_ok(a->q, a->elem, p.q_ss, p.q_hs);
  p.o_wide = wide_ok(a->out, a->elem, p.o_ss, p.o_hs);
  p.lse = a->lse;
  p.gpad = (p.group + 1) & ~1u;
  p.err = ctx->d_err;
  uint8_t* work = static_cast<uint8_t*>(a->work);
  p.join = reinterpret_cast<Join*>(work);
  p.part = reinterpret_cast<float*>(work + kMaxCtas * sizeof(Join));
  if (a->weights_out) {
    uint8_t* more = work + kMaxCtas * sizeof(Join) + part_bytes(kv->head_dim);
    p.lse2 = reinterpret_cast<float*>(more);
    p.scores = reinterpret_cast<float*>(more + round16(uint64_t(kv->sequences) * p.qh * 4));
  }
  const cudaStream_t s = stream ? static_cast<cudaStream_t>(stream) : ctx->stream;
  const uint64_t most = most_steps(*kv, p.qh);
  const uint32_t nw = workers_of(kv->head_dim);
  const uint32_t grid = uint32_t(std::min<uint64_t>(std::min<uint32_t>(ctx->sm_count, kMaxCtas), (most + nw - 1) / nw));
  const bool bf16 = kv->elem == SI_ELEM_BF16;
  cudaError_t e;
  switch (padded_dim(kv->head_dim)) {
    case 64: e = launch_hd<64>(p, bf16, grid, s); break;
    case 128: e = launch_hd<128>(p, bf16, grid, s); break;
    case 192: e = launch_hd<192>(p, bf16, grid, s); break;
    default: e = launch_hd<256>(p, bf16, grid, s); break;
  }
  if (e != cudaSuccess) return cuda_fail(ctx, e, "paged attention launch");
  if (a->weights_out) {
    const uint32_t rows = kv->sequences * kv->kv_heads;
    const uint32_t blocks = std::min<uint32_t>((p.kv.max_tokens + 255) / 256, std::max(1u, uint32_t(ctx->sm_count) * 8 / rows));
    PdlLaunch l(dim3(blocks, rows), dim3(256), 0, s);
    e = cudaLaunchKernelEx(&l.cfg, paged_weights_kernel, p, a->weights_in, a->weights_out, a->weights_stride);
    if (e != cudaSuccess) return cuda_fail(ctx, e, "paged attention weights launch");
  }
  note_async_submission(ctx);
  return SI_OK;
}
