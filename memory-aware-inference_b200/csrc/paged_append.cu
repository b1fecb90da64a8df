// Rotary positions of new queries and keys, and the append of keys and values
// into cache pages.
//
// A pair (x, y) at position p turns by p f: (x c - y s, x s + y c). The
// frequency is held as turns in units of 2^-64 (host table), so the 64-bit
// product p * turn drops whole turns by its own overflow: the angle modulo one
// turn is exact to 2^-33 turns for any 32-bit position, where p * f in f32 is
// off by 0.03 rad at position 500,000. sincospif of the top 32 bits as a
// fraction of a half turn finishes it.
#include "paged.cuh"

namespace si {
namespace {

constexpr int kThreads = 256;

struct AppendArgs {
  PagedView kv;
  const void *q, *k, *v;
  void* q_out;
  uint64_t q_ts, q_hs, qo_ts, qo_hs, k_ts, k_hs, v_ts, v_hs;
  const int32_t *sequence, *slot, *position;
  const uint64_t* rope;
  float rope_scale;
  uint32_t elem, cache_elem, tokens, qh, kvh, half, interleaved;
  uint32_t per_cta;      // tokens of a CTA
  uint32_t rot_slots;    // threads of a head that rotate
  FastDiv slots, heads;  // threads of a head; heads of a token (q, k, v)
  int* err;
};

// One thread's part of a head: VEC pairs (two runs of VEC elements in the half
// layout, one run of 2 VEC neighbouring elements in the interleaved one) or, past the rotated
// dims, a run to copy.
//
// Bandwidth bound: every element is read once and written once. A CTA takes a
// few tokens, makes their sines once in shared memory, and walks the (token,
// head, run) items of all three inputs, so that heads share the sines and the
// accesses of a warp are contiguous.
template <int VEC>
__global__ void __launch_bounds__(kThreads) append_kernel(const __grid_constant__ AppendArgs a) {
  extern __shared__ float2 s_turn[];  // [per_cta][half] (cos, sin)
  pdl_launch_dependents();
  pdl_wait();
  const uint32_t t0 = blockIdx.x * a.per_cta, nt = min(a.per_cta, a.tokens - t0);
  for (uint32_t i = threadIdx.x; i < nt * a.half; i += kThreads) {
    const uint32_t t = i / a.half, j = i - t * a.half;
    const int32_t pos = a.position ? a.position[t0 + t] : a.slot[t0 + t];
    // two's complement: a negative position turns the other way
    const uint64_t turn = uint64_t(int64_t(pos)) * a.rope[j];
    const float x = float(int32_t(uint32_t(turn >> 32))) * 0x1p-31f;  // half turns, in [-1, 1]
    float s, c;
    sincospif(x, &s, &c);
    s_turn[i] = make_float2(c * a.rope_scale, s * a.rope_scale);
  }
  __syncthreads();
  const uint32_t rows = nt * a.heads.d, items = rows * a.slots.d;
  for (uint32_t i = threadIdx.x; i < items; i += kThreads) {
    const uint32_t row = div_of(i, a.slots), part = i - row * a.slots.d;
    const uint32_t t = div_of(row, a.heads), head = row - t * a.heads.d, tok = t0 + t;
    const int32_t slot = a.slot[tok];
    if (slot < 0) continue;  // padding
    const bool is_q = head < a.qh, is_k = !is_q && head < a.qh + a.kvh;
    const uint32_t h = is_q ? head : is_k ? head - a.qh : head - a.qh - a.kvh;
    const void* src = is_q ? a.q : is_k ? a.k : a.v;
    const uint64_t from = is_q ? tok * a.q_ts + h * a.q_hs : is_k ? tok * a.k_ts + h * a.k_hs : tok * a.v_ts + h * a.v_hs;
    uint64_t to;
    void* dst;
    uint32_t elem;
    if (is_q) {
      to = tok * a.qo_ts + h * a.qo_hs;
      dst = a.q_out;
      elem = a.elem;
    } else {
      const uint32_t b = a.sequence ? uint32_t(a.sequence[tok]) : tok;
      to = kNoCell;
      if (b < a.kv.sequences && uint32_t(slot) < a.kv.max_tokens)
        to = paged_slot(a.kv, a.kv.pages + b * a.kv.pages_stride, uint32_t(slot), h);
      if (to == kNoCell) {
        atomicOr(a.err, KERR_BAD_INDEX);
        continue;
      }
      dst = const_cast<uint16_t*>(is_k ? a.kv.k : a.kv.v);
      elem = a.cache_elem;
    }
    // dims of the two runs; a value head copies all of its runs
    uint32_t d0, d1;
    bool turn = part < a.rot_slots;
    if (turn) {
      d0 = a.interleaved ? part * 2 * VEC : part * VEC;
      d1 = a.interleaved ? d0 + VEC : d0 + a.half;
    } else {
      d0 = 2 * a.half + (part - a.rot_slots) * 2 * VEC;
      d1 = d0 + VEC;
    }
    const bool second = d1 < a.kv.hd;  // the last copied run may be single
    float x[VEC], y[VEC];
    if constexpr (VEC == 8) {
      load8(src, from + d0, a.elem, true, x);
      if (second) load8(src, from + d1, a.elem, true, y);
    } else {
      if (a.elem == SI_ELEM_F32) {
        x[0] = static_cast<const float*>(src)[from + d0];
        y[0] = second ? static_cast<const float*>(src)[from + d1] : 0.f;
      } else {
        x[0] = elem_to_f(static_cast<const uint16_t*>(src)[from + d0], a.elem);
        y[0] = second ? elem_to_f(static_cast<const uint16_t*>(src)[from + d1], a.elem) : 0.f;
      }
    }
    if (turn && (is_q || is_k)) {
      const float2* cs = s_turn + t * a.half;
      if (VEC == 8 && a.interleaved) {
#pragma unroll
        for (int j = 0; j < VEC; j += 2) {
          const float2 u = cs[(d0 + j) / 2], w = cs[(d1 + j) / 2];
          const float x0 = x[j], x1 = x[j + 1 < VEC ? j + 1 : j], y0 = y[j], y1 = y[j + 1 < VEC ? j + 1 : j];
          x[j] = x0 * u.x - x1 * u.y;
          x[j + 1 < VEC ? j + 1 : j] = x0 * u.y + x1 * u.x;
          y[j] = y0 * w.x - y1 * w.y;
          y[j + 1 < VEC ? j + 1 : j] = y0 * w.y + y1 * w.x;
        }
      } else {
        const uint32_t p0 = a.interleaved ? d0 / 2 : d0;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float2 u = cs[p0 + j];
          const float x0 = x[j], y0 = y[j];
          x[j] = x0 * u.x - y0 * u.y;
          y[j] = x0 * u.y + y0 * u.x;
        }
      }
    }
    if constexpr (VEC == 8) {
      store8(dst, to + d0, elem, true, x);
      if (second) store8(dst, to + d1, elem, true, y);
    } else {
      if (elem == SI_ELEM_F32) {
        static_cast<float*>(dst)[to + d0] = x[0];
        if (second) static_cast<float*>(dst)[to + d1] = y[0];
      } else {
        static_cast<uint16_t*>(dst)[to + d0] = f_to_elem(x[0], elem);
        if (second) static_cast<uint16_t*>(dst)[to + d1] = f_to_elem(y[0], elem);
      }
    }
  }
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
  const uint64_t strides[] = {a->q_token_stride,     a->q_head_stride, a->q_out_token_stride, a->q_out_head_stride,
                              a->k_token_stride,     a->k_head_stride, a->v_token_stride,     a->v_head_stride};
  for (uint64_t s : strides)
    if (s >> 36) return bad(SI_E_INVALID, "paged append strides are out of range");
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
  p.elem = a->elem, p.cache_elem = kv->elem;
  p.tokens = a->tokens;
  p.qh = a->q ? a->query_heads : 0;
  p.kvh = a->k ? kv->kv_heads : 0;
  p.half = a->rotary_dim / 2;
  p.interleaved = a->rope_layout == SI_ROPE_INTERLEAVED;
  p.err = ctx->d_err;
  // 16-byte accesses where every run starts on a 16-byte boundary
  bool wide = p.interleaved ? a->rotary_dim % 16 == 0 : p.half % 8 == 0;
  if (a->q)
    wide = wide && wide_ok(a->q, a->elem, p.q_ts, p.q_hs) && wide_ok(a->q_out, a->elem, p.qo_ts, p.qo_hs);
  if (a->k) wide = wide && wide_ok(a->k, a->elem, p.k_ts, p.k_hs) && wide_ok(a->v, a->elem, p.v_ts, p.v_hs);
  const uint32_t vec = wide ? 8 : 1;
  p.rot_slots = p.half / vec;
  const uint32_t rest = kv->head_dim - a->rotary_dim;
  p.slots = fast_div(p.rot_slots + (rest + 2 * vec - 1) / (2 * vec));
  p.heads = fast_div(p.qh + 2 * p.kvh);
  // a CTA takes up to 8 tokens, fewer while that leaves multiprocessors without work
  p.per_cta = 1;
  while (p.per_cta < 8 && p.tokens / (2 * p.per_cta) >= uint32_t(ctx->sm_count) * 4) p.per_cta *= 2;
  const cudaStream_t s = stream ? static_cast<cudaStream_t>(stream) : ctx->stream;
  PdlLaunch l(dim3((p.tokens + p.per_cta - 1) / p.per_cta), dim3(kThreads), size_t(p.per_cta) * p.half * sizeof(float2), s);
  const cudaError_t e = wide ? cudaLaunchKernelEx(&l.cfg, append_kernel<8>, p) : cudaLaunchKernelEx(&l.cfg, append_kernel<1>, p);
  if (e != cudaSuccess) return cuda_fail(ctx, e, "paged append launch");
  note_async_submission(ctx);
  return SI_OK;
}
