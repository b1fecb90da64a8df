// Rotary positions of new queries and keys, and the append of keys and values
// into cache pages.
//
// A pair (x, y) at position p turns by p f: (x c - y s, x s + y c). The
// frequency is held as turns in units of 2^-64 (host table), so the 64-bit
// product p * turn drops whole turns by its own overflow. What is left is off by
// |p| 2^-65 turns (the table's rounding, 2^-34 at the last 32-bit position), by
// less than 2^-32 turns for the low 32 bits that are dropped, and by 2^-25 of a
// half turn where the rest becomes an f32 fraction of it for sincospif: about
// 1e-7 rad at any position, where p * f in f32 is off by 0.03 rad at 500,000.
#include <type_traits>

#include "paged.cuh"

namespace si {
namespace {

constexpr int kThreads = 256;
constexpr uint32_t kMaxTokens = 8;  // of a CTA

struct AppendArgs {
  PagedView kv;
  const void *q, *k, *v;
  void* q_out;
  uint64_t q_ts, q_hs, qo_ts, qo_hs, k_ts, k_hs, v_ts, v_hs;
  const int32_t *sequence, *slot, *position;
  const uint64_t* rope;
  float rope_scale;
  uint32_t tokens, kvh, half, interleaved;
  uint32_t per_cta;      // tokens of a CTA
  uint32_t rot_parts;    // parts of a head that rotate
  FastDiv parts;         // parts of a head, a thread each
  FastDiv q_heads, kv_heads;
  float* weights;        // accumulated weights and positions that appended slots start anew in; may be null
  int32_t* positions;
  uint64_t weights_stride;
  int* err;
};

// One thread's part of a head: VEC pairs (two runs of VEC elements in the half
// layout, one run of 2 VEC neighbouring elements in the interleaved one) or,
// past the rotated dims, a run to copy.
//
// Bandwidth bound: every element is read once and written once, and what there
// is to gain is few instructions in between. A CTA takes a few tokens and makes
// their sines and their places in the cache once in shared memory. A thread
// keeps its part of a head and walks the rows (token, head) of the queries,
// then of the keys, then of the values, in batches whose loads are all on their way
// before the first is used. Sines lie so that neighbouring parts read
// neighbouring banks. 8,192 tokens of 32 + 8 + 8 heads of 128 take 37 us (201 MB,
// 5.5 TB/s).
template <int VEC, uint32_t ELEM>
struct Run {  // VEC elements as they lie in memory
  static constexpr int kRegs = VEC == 8 ? (ELEM == SI_ELEM_F32 ? 8 : 4) : 1;
  uint32_t r[kRegs];
  __device__ __forceinline__ void load(const void* p, uint64_t i) {
    if constexpr (VEC == 8) {
      const uint4* q = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(p) + i * elem_bytes(ELEM));
#pragma unroll
      for (int j = 0; j < kRegs / 4; ++j) {
        const uint4 v = q[j];
        r[4 * j] = v.x, r[4 * j + 1] = v.y, r[4 * j + 2] = v.z, r[4 * j + 3] = v.w;
      }
    } else if constexpr (ELEM == SI_ELEM_F32) {
      r[0] = static_cast<const uint32_t*>(p)[i];
    } else {
      r[0] = static_cast<const uint16_t*>(p)[i];
    }
  }
  __device__ __forceinline__ float at(int j) const {
    if constexpr (ELEM == SI_ELEM_F32) return __uint_as_float(r[j]);
    return elem_to_f(uint16_t(r[j / 2] >> (j % 2 * 16)), ELEM);
  }
};
template <int VEC, uint32_t ELEM>
__device__ __forceinline__ void store_run(void* p, uint64_t i, const float x[VEC]) {
  if constexpr (VEC == 8) {
    store8(p, i, ELEM, true, x);
  } else if constexpr (ELEM == SI_ELEM_F32) {
    static_cast<float*>(p)[i] = x[0];
  } else {
    static_cast<uint16_t*>(p)[i] = f_to_elem(x[0], ELEM);
  }
}

enum Kind { kQuery, kKey, kValue };

template <int VEC, uint32_t ELEM, uint32_t CACHE>
__global__ void __launch_bounds__(kThreads, 4) append_kernel(const __grid_constant__ AppendArgs a) {
  constexpr int kBatch = 2;  // more would spill: 4 rows at once took 47 us where 2 take 37 (8192 tokens, 32 + 8 + 8 heads of 128)
  extern __shared__ float2 s_turn[];  // [per_cta][VEC][rotating parts] (cos, sin)
  __shared__ uint64_t s_cell[kMaxTokens];
  __shared__ int32_t s_slot[kMaxTokens];
  __shared__ uint32_t s_seq[kMaxTokens];
  pdl_launch_dependents();
  pdl_wait();
  const uint32_t t0 = blockIdx.x * a.per_cta, nt = min(a.per_cta, a.tokens - t0);
  if (threadIdx.x < nt) {
    const uint32_t tok = t0 + threadIdx.x;
    int32_t slot = a.slot[tok];
    uint64_t cell = kNoCell;
    if (slot >= 0 && a.kvh) {
      const uint32_t b = a.sequence ? uint32_t(a.sequence[tok]) : tok;
      s_seq[threadIdx.x] = b;
      if (b < a.kv.sequences && uint32_t(slot) < a.kv.max_tokens && uint32_t(slot) < a.weights_stride)
        cell = paged_slot(a.kv, a.kv.pages + b * a.kv.pages_stride, uint32_t(slot), 0);
      if (cell == kNoCell) {  // reported, and left out like padding
        atomicOr(a.err, KERR_BAD_INDEX);
        slot = -1;
      }
    }
    s_slot[threadIdx.x] = slot;
    s_cell[threadIdx.x] = cell;
  }
  for (uint32_t i = threadIdx.x; i < nt * a.half; i += kThreads) {
    const uint32_t t = i / a.half, j = i - t * a.half;
    const int32_t pos = a.position ? a.position[t0 + t] : a.slot[t0 + t];
    // two's complement: a negative position turns the other way
    const uint64_t turn = uint64_t(int64_t(pos)) * a.rope[j];
    const float half_turns = float(int32_t(uint32_t(turn >> 32))) * 0x1p-31f;  // in [-1, 1]
    float s, c;
    sincospif(half_turns, &s, &c);
    s_turn[t * a.half + j % VEC * a.rot_parts + j / VEC] = make_float2(c * a.rope_scale, s * a.rope_scale);
  }
  __syncthreads();
  if (a.weights || a.positions) {
    for (uint32_t i = threadIdx.x; i < nt * a.kvh; i += kThreads) {
      const uint32_t t = div_of(i, a.kv_heads), h = i - t * a.kvh;
      if (s_cell[t] == kNoCell) continue;
      const uint64_t at = (uint64_t(s_seq[t]) * a.kvh + h) * a.weights_stride + uint32_t(s_slot[t]);
      if (a.weights) a.weights[at] = 0.f;
      if (a.positions) a.positions[at] = a.position ? a.position[t0 + t] : s_slot[t];
    }
  }
  const uint32_t row0 = div_of(threadIdx.x, a.parts), part = threadIdx.x - row0 * a.parts.d, rows_at_once = kThreads / a.parts.d;
  if (row0 >= rows_at_once) return;
  const bool rotates = part < a.rot_parts;
  // dims of the two runs; the second may be missing in the last copied part
  uint32_t d0, d1;
  if (rotates) {
    d0 = a.interleaved ? part * 2 * VEC : part * VEC;
    d1 = a.interleaved ? d0 + VEC : d0 + a.half;
  } else {
    d0 = 2 * a.half + (part - a.rot_parts) * 2 * VEC;
    d1 = d0 + VEC;
  }
  const bool second = d1 < a.kv.hd;

  auto walk = [&](auto kind, const void* src, uint64_t ts, uint64_t hs, const FastDiv& heads) {
    constexpr Kind K = decltype(kind)::value;
    const uint32_t rows = nt * heads.d;
    for (uint32_t r0 = row0; r0 < rows; r0 += kBatch * rows_at_once) {
      Run<VEC, ELEM> x[kBatch], y[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const uint32_t r = r0 + j * rows_at_once, t = div_of(r, heads), h = r - t * heads.d;
        if (r >= rows) continue;
        const uint64_t from = uint64_t(t0 + t) * ts + h * hs;
        x[j].load(src, from + d0);
        if (second) y[j].load(src, from + d1);
      }
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const uint32_t r = r0 + j * rows_at_once, t = div_of(r, heads), h = r - t * heads.d;
        if (r >= rows || s_slot[t] < 0) continue;  // past the end, or padding
        float u[VEC], w[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) u[e] = x[j].at(e), w[e] = y[j].at(e);
        if (K != kValue && rotates) {
          float2 f[VEC];
#pragma unroll
          for (int e = 0; e < VEC; ++e) f[e] = s_turn[t * a.half + e * a.rot_parts + part];
          if (VEC == 8 && a.interleaved) {  // pairs side by side: the first four in u, the others in w
#pragma unroll
            for (int e = 0; e < VEC / 2; ++e) {
              const float u0 = u[2 * e], u1 = u[2 * e + 1], w0 = w[2 * e], w1 = w[2 * e + 1];
              const float2 g = f[e], k = f[VEC / 2 + e];
              u[2 * e] = u0 * g.x - u1 * g.y;
              u[2 * e + 1] = u0 * g.y + u1 * g.x;
              w[2 * e] = w0 * k.x - w1 * k.y;
              w[2 * e + 1] = w0 * k.y + w1 * k.x;
            }
          } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
              const float u0 = u[e], w0 = w[e];
              u[e] = u0 * f[e].x - w0 * f[e].y;
              w[e] = u0 * f[e].y + w0 * f[e].x;
            }
          }
        }
        if constexpr (K == kQuery) {
          const uint64_t to = uint64_t(t0 + t) * a.qo_ts + h * a.qo_hs;
          store_run<VEC, ELEM>(a.q_out, to + d0, u);
          if (second) store_run<VEC, ELEM>(a.q_out, to + d1, w);
        } else if (s_cell[t] != kNoCell) {
          uint16_t* dst = const_cast<uint16_t*>(K == kKey ? a.kv.k : a.kv.v);
          const uint64_t to = s_cell[t] + uint64_t(h) * a.kv.head_stride;
          store_run<VEC, CACHE>(dst, to + d0, u);
          if (second) store_run<VEC, CACHE>(dst, to + d1, w);
        }
      }
    }
  };
  if (a.q_heads.d) walk(std::integral_constant<Kind, kQuery>(), a.q, a.q_ts, a.q_hs, a.q_heads);
  if (a.kvh) {
    walk(std::integral_constant<Kind, kKey>(), a.k, a.k_ts, a.k_hs, a.kv_heads);
    walk(std::integral_constant<Kind, kValue>(), a.v, a.v_ts, a.v_hs, a.kv_heads);
  }
}

template <int VEC, uint32_t ELEM>
cudaError_t launch(const cudaLaunchConfig_t* cfg, const AppendArgs& p, uint32_t cache) {
  return cache == SI_ELEM_BF16 ? cudaLaunchKernelEx(cfg, append_kernel<VEC, ELEM, SI_ELEM_BF16>, p)
                               : cudaLaunchKernelEx(cfg, append_kernel<VEC, ELEM, SI_ELEM_F16>, p);
}
template <int VEC>
cudaError_t launch(const cudaLaunchConfig_t* cfg, const AppendArgs& p, uint32_t elem, uint32_t cache) {
  return elem == SI_ELEM_F32    ? launch<VEC, SI_ELEM_F32>(cfg, p, cache)
         : elem == SI_ELEM_BF16 ? launch<VEC, SI_ELEM_BF16>(cfg, p, cache)
                                : launch<VEC, SI_ELEM_F16>(cfg, p, cache);
}

int check_append(const si_paged_kv* kv, const si_paged_append* a, std::string* msg) {
  if (int rc = check_paged_kv(kv, msg)) return rc;
  auto bad = [&](int rc, const char* text) {
    *msg = text;
    return rc;
  };
  if (!a) return bad(SI_E_INVALID, "null paged append description");
  if (!elem_known(a->elem)) return bad(SI_E_UNSUPPORTED, "paged append elements must be f32, bf16 or f16");
  if (a->tokens > 0x7fffffu) return bad(SI_E_UNSUPPORTED, "paged append takes at most 8388607 tokens a call");
  if (!a->q != !a->q_out) return bad(SI_E_INVALID, "paged append needs q and q_out together");
  if (!a->k != !a->v) return bad(SI_E_INVALID, "paged append needs k and v together");
  if (a->q && (a->query_heads == 0 || a->query_heads > 65535))
    return bad(SI_E_INVALID, "paged append query heads are invalid");
  if (a->rotary_dim % 2 || a->rotary_dim > kv->head_dim)
    return bad(SI_E_INVALID, "paged append rotary width is invalid");
  if (a->rope_layout != SI_ROPE_INTERLEAVED && a->rope_layout != SI_ROPE_HALF)
    return bad(SI_E_INVALID, "paged append rotary layout is unknown");
  if (a->rotary_dim && (!a->rope || reinterpret_cast<uintptr_t>(a->rope) % 8))
    return bad(SI_E_INVALID, "paged append needs a rotary table, 8-byte aligned");
  if (a->tokens && !a->slot) return bad(SI_E_INVALID, "paged append slots are null");
  if (!a->sequence && a->tokens > kv->sequences)
    return bad(SI_E_INVALID, "paged append has more tokens than sequences and no sequence numbers");
  for (const void* p : {a->q, static_cast<const void*>(a->q_out), a->k, a->v})
    if (!elem_aligned(p, a->elem)) return bad(SI_E_INVALID, "paged append buffers are not aligned to their elements");
  if (!words_aligned({a->sequence, a->slot, a->position, a->weights, a->positions}))
    return bad(SI_E_INVALID, "paged append arrays of 32-bit numbers are not aligned");
  if (a->weights || a->positions) {
    if (a->tokens && !a->k) return bad(SI_E_INVALID, "paged append starts weights and positions of appended keys only");
    if (a->weights_stride == 0 || a->weights_stride >> 44)
      return bad(SI_E_INVALID, "paged append stride of weights and positions is out of range");
  }
  const uint64_t strides[] = {a->q_token_stride,     a->q_head_stride, a->q_out_token_stride, a->q_out_head_stride,
                              a->k_token_stride,     a->k_head_stride, a->v_token_stride,     a->v_head_stride};
  for (uint64_t s : strides)
    if (s >> 36) return bad(SI_E_INVALID, "paged append strides are out of range");
  if (a->tokens && a->q) {
    const BufferRows q = {a->q, a->tokens, a->q_token_stride, a->query_heads, a->q_head_stride, kv->head_dim, a->elem};
    const BufferRows out = {a->q_out,          a->tokens,    a->q_out_token_stride, a->query_heads,
                            a->q_out_head_stride, kv->head_dim, a->elem};
    if (!rows_distinct(out)) return bad(SI_E_INVALID, "paged append output rows overlap");
    const bool in_place = q.p == out.p && (q.n0 == 1 || q.s0 == out.s0) && (q.n1 == 1 || q.s1 == out.s1);
    if (!in_place && rows_meet(q, out))
      return bad(SI_E_INVALID, "paged append writes its queries in place or apart from those it reads");
    if (a->k)
      for (const BufferRows& in : {BufferRows{a->k, a->tokens, a->k_token_stride, kv->kv_heads, a->k_head_stride, kv->head_dim, a->elem},
                                   BufferRows{a->v, a->tokens, a->v_token_stride, kv->kv_heads, a->v_head_stride, kv->head_dim, a->elem}})
        if (rows_meet(in, out)) return bad(SI_E_INVALID, "paged append would write queries over new keys or values");
  }
  if (a->tokens && a->k && (!pools_distinct(*kv) || kv->k == kv->v))
    return bad(SI_E_INVALID, "paged append needs pools whose rows do not overlap");
  return SI_OK;
}

}  // namespace
}  // namespace si

using namespace si;

extern "C" int si_paged_append_dev(si_ctx* ctx, const si_paged_kv* kv, const si_paged_append* a, void* stream) {
  std::string msg;
  if (int rc = check_append(kv, a, &msg)) return fail(ctx, rc, msg);
  if (!ctx) return fail(nullptr, SI_E_INVALID, "null context");
  if (a->tokens == 0 || (!a->q && !a->k)) return SI_OK;
  DeviceGuard dev(ctx->device);
  if (dev.e != cudaSuccess) return cuda_fail(ctx, dev.e, "paged append device");
  AppendArgs p = {};
  p.kv = paged_view(*kv);
  p.q = a->q, p.k = a->k, p.v = a->v, p.q_out = a->q_out;
  p.q_ts = a->q_token_stride, p.q_hs = a->q_head_stride;
  p.qo_ts = a->q_out_token_stride, p.qo_hs = a->q_out_head_stride;
  p.k_ts = a->k_token_stride, p.k_hs = a->k_head_stride, p.v_ts = a->v_token_stride, p.v_hs = a->v_head_stride;
  p.sequence = a->sequence, p.slot = a->slot, p.position = a->position;
  p.rope = a->rope;
  p.rope_scale = a->rope_scale;
  p.tokens = a->tokens;
  if (a->q) p.q_heads = fast_div(a->query_heads);
  if (a->k) p.kv_heads = fast_div(kv->kv_heads);
  p.kvh = a->k ? kv->kv_heads : 0;
  p.half = a->rotary_dim / 2;
  p.interleaved = a->rope_layout == SI_ROPE_INTERLEAVED;
  p.weights = a->weights, p.positions = a->positions;
  p.weights_stride = a->weights || a->positions ? a->weights_stride : ~uint64_t(0);
  p.err = ctx->d_err;
  // 16-byte accesses where every run starts on a 16-byte boundary
  bool wide = p.interleaved ? a->rotary_dim % 16 == 0 : p.half % 8 == 0;
  if (a->q)
    wide = wide && wide_ok(a->q, a->elem, p.q_ts, p.q_hs) && wide_ok(a->q_out, a->elem, p.qo_ts, p.qo_hs);
  if (a->k) wide = wide && wide_ok(a->k, a->elem, p.k_ts, p.k_hs) && wide_ok(a->v, a->elem, p.v_ts, p.v_hs);
  const uint32_t vec = wide ? 8 : 1;
  p.rot_parts = p.half / vec;
  const uint32_t rest = kv->head_dim - a->rotary_dim;
  p.parts = fast_div(p.rot_parts + (rest + 2 * vec - 1) / (2 * vec));
  // a CTA takes up to 8 tokens, fewer while that leaves multiprocessors without work
  p.per_cta = 1;
  while (p.per_cta < kMaxTokens && p.tokens / (2 * p.per_cta) >= uint32_t(ctx->sm_count) * 4) p.per_cta *= 2;
  const cudaStream_t s = stream ? static_cast<cudaStream_t>(stream) : ctx->stream;
  PdlLaunch l(dim3((p.tokens + p.per_cta - 1) / p.per_cta), dim3(kThreads), size_t(p.per_cta) * p.half * sizeof(float2), s);
  const cudaError_t e = wide ? launch<8>(&l.cfg, p, a->elem, kv->elem) : launch<1>(&l.cfg, p, a->elem, kv->elem);
  if (e != cudaSuccess) return cuda_fail(ctx, e, "paged append launch");
  note_async_submission(ctx);
  return SI_OK;
}
