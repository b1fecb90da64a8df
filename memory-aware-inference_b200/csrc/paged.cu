// Host side of the paged cache: checks of its description, the place of a
// slot, and the table of rotary frequencies (include/si_paged.h).
#include <algorithm>
#include <cmath>

#include "paged.cuh"

namespace si {

int check_paged_kv(const si_paged_kv* kv, std::string* msg) {
  auto bad = [&](int rc, const char* text) {
    *msg = text;
    return rc;
  };
  if (!kv) return bad(SI_E_INVALID, "null paged cache description");
  if (kv->elem != SI_ELEM_BF16 && kv->elem != SI_ELEM_F16)
    return bad(SI_E_UNSUPPORTED, "paged cache elements must be bf16 or f16");
  if (kv->kv_heads == 0 || kv->kv_heads > 65535 || kv->head_dim == 0)
    return bad(SI_E_INVALID, "paged cache head dimensions are invalid");
  if (kv->head_dim % 8 || kv->head_dim > 256)
    return bad(SI_E_UNSUPPORTED, "paged cache head_dim must be a multiple of 8, at most 256");
  if (kv->page_tokens == 0 || kv->max_pages == 0 || kv->sequences == 0 || kv->num_pages == 0)
    return bad(SI_E_INVALID, "paged cache sizes must be positive");
  if (kv->num_pages > 0x7fffffffull || uint64_t(kv->page_tokens) * kv->max_pages > 0x7fffffffull)
    return bad(SI_E_UNSUPPORTED, "paged cache pages and slots must be below 2^31");
  if (kv->sequences > 4096) return bad(SI_E_UNSUPPORTED, "a paged cache call takes at most 4096 sequences");
  if (uint64_t(kv->sequences) * ((uint64_t(kv->page_tokens) * kv->max_pages + 15) / 16) > 0xffffffffull)
    return bad(SI_E_UNSUPPORTED, "paged cache page table spans too many slots");
  if (kv->pages_stride < kv->max_pages)
    return bad(SI_E_INVALID, "paged cache page-table rows overlap");
  if ((kv->page_stride | kv->head_stride | kv->token_stride) % 8)
    return bad(SI_E_INVALID, "paged cache strides must be multiples of 8 elements");
  // the largest offset has to stay inside 63 bits (in bytes)
  const unsigned __int128 last = (unsigned __int128)(kv->num_pages - 1) * kv->page_stride +
                                 (unsigned __int128)(kv->kv_heads - 1) * kv->head_stride +
                                 (unsigned __int128)(kv->page_tokens - 1) * kv->token_stride + kv->head_dim;
  if (last >> 61) return bad(SI_E_INVALID, "paged cache strides are out of range");
  if (!kv->k || !kv->v || !kv->pages) return bad(SI_E_INVALID, "paged cache pointers are null");
  if ((reinterpret_cast<uintptr_t>(kv->k) | reinterpret_cast<uintptr_t>(kv->v)) % 16 ||
      reinterpret_cast<uintptr_t>(kv->pages) % 4)
    return bad(SI_E_INVALID, "paged cache pools must be 16-byte aligned");
  return SI_OK;
}

// Overlaps, in elements. Checked descriptions keep every span below 2^61, so
// 64-bit sums of three of them do not overflow. Calls are bound by their host
// time, so what is usual is found out in a few operations.
namespace {
struct Axis {
  uint64_t n, stride;
};
bool distinct(Axis a, Axis b, Axis c, uint32_t dims) {
  if (a.stride > b.stride) std::swap(a, b);
  if (b.stride > c.stride) std::swap(b, c);
  if (a.stride > b.stride) std::swap(a, b);
  uint64_t span = dims;
  for (const Axis& x : {a, b, c}) {
    if (x.n <= 1) continue;
    if (x.stride < span) return false;
    span += (x.n - 1) * x.stride;
  }
  return true;
}
// From the first element to behind the last.
int64_t span_of(const BufferRows& r) { return int64_t((r.n0 - 1) * r.s0 + (r.n1 - 1) * r.s1 + r.dims); }
}  // namespace

bool rows_distinct(const BufferRows& r) { return distinct({r.n0, r.s0}, {r.n1, r.s1}, {1, 0}, r.dims); }
bool pools_distinct(const si_paged_kv& kv) {
  return distinct({kv.num_pages, kv.page_stride}, {kv.kv_heads, kv.head_stride}, {kv.page_tokens, kv.token_stride},
                  kv.head_dim);
}

bool rows_meet(const BufferRows& a, const BufferRows& b) {
  // both are aligned to their elements
  const int64_t apart = (static_cast<const char*>(b.p) - static_cast<const char*>(a.p)) / int64_t(elem_bytes(a.elem));
  if (apart >= span_of(a) || -apart >= span_of(b)) return false;
  // an axis of one row has no stride of its own
  if ((a.n0 > 1 && b.n0 > 1 && a.s0 != b.s0) || (a.n1 > 1 && b.n1 > 1 && a.s1 != b.s1)) return true;
  const int64_t s0 = int64_t(a.n0 > 1 ? a.s0 : b.s0), s1 = int64_t(a.n1 > 1 ? a.s1 : b.s1), dims = a.dims;
  // Parts of one buffer mostly: every step of one axis holds all of a's other axis, then all of b's.
  auto beside = [&](int64_t outer, int64_t inner, uint64_t in_a, uint64_t in_b) {
    if (outer == 0) return false;
    const int64_t at = (apart % outer + outer) % outer;
    return at >= int64_t(in_a - 1) * inner + dims && at + int64_t(in_b - 1) * inner + dims <= outer;
  };
  if (beside(s0, s1, a.n1, b.n1) || beside(s1, s0, a.n0, b.n0)) return false;
  // Rows (i0, i1) of a and (j0, j1) of b share an element if |apart - (i0 - j0) s0 -
  // (i1 - j1) s1| < dims. The shorter axis is walked, the nearest steps of the other computed.
  struct Steps {
    int64_t lo, hi, stride;
  } x = {1 - int64_t(b.n0), int64_t(a.n0) - 1, s0}, y = {1 - int64_t(b.n1), int64_t(a.n1) - 1, s1};
  if (x.hi - x.lo < y.hi - y.lo) std::swap(x, y);
  for (int64_t i = y.lo; i <= y.hi; ++i) {
    const int64_t rest = apart - i * y.stride;
    const int64_t near = std::min(std::max(x.stride ? rest / x.stride : 0, x.lo), x.hi);
    for (int64_t k = std::max(near - 1, x.lo); k <= std::min(near + 1, x.hi); ++k) {
      const int64_t left = rest - k * x.stride;
      if (left > -dims && left < dims) return true;
    }
  }
  return false;
}

}  // namespace si

extern "C" int si_paged_kv_offset(const si_paged_kv* kv, int64_t page, uint64_t slot, uint32_t head,
                                  uint64_t* offset) {
  std::string msg;
  if (int rc = si::check_paged_kv(kv, &msg)) return si::fail(nullptr, rc, msg);
  if (!offset) return si::fail(nullptr, SI_E_INVALID, "null offset");
  const si::PagedView p = si::paged_view(*kv);
  if (slot >= p.max_tokens || head >= kv->kv_heads || page < INT32_MIN || page > INT32_MAX)
    return si::fail(nullptr, SI_E_INVALID, "page, slot or head is outside the paged cache");
  const uint32_t t = uint32_t(slot);
  const uint64_t at = si::paged_cell(p, int32_t(page), t - si::div_of(t, p.page) * p.page.d, head);
  if (at == si::kNoCell) return si::fail(nullptr, SI_E_INVALID, "page, slot or head is outside the paged cache");
  *offset = at;
  return SI_OK;
}

extern "C" int si_rope_table(double theta, uint32_t rotary_dim, const si_rope_scaling* sc, uint64_t* turns,
                             float* scale) {
  auto bad = [](int rc, const char* text) { return si::fail(nullptr, rc, text); };
  const si_rope_scaling none = {};
  if (!sc) sc = &none;
  if (!(theta > 1.0) || !std::isfinite(theta)) return bad(SI_E_INVALID, "rotary theta must be above 1");
  if (rotary_dim % 2 || rotary_dim > 256) return bad(SI_E_INVALID, "rotary width must be even, at most 256");
  if (sc->kind > SI_ROPE_SCALE_BANDED) return bad(SI_E_INVALID, "unknown rotary scaling");
  if (sc->kind != SI_ROPE_SCALE_NONE && (!(sc->factor >= 1.0) || !std::isfinite(sc->factor)))
    return bad(SI_E_INVALID, "rotary scaling factor must be at least 1");
  if (sc->kind >= SI_ROPE_SCALE_YARN && (!(sc->original >= 1.0) || !std::isfinite(sc->original)))
    return bad(SI_E_INVALID, "rotary scaling needs the trained context length");
  if (sc->kind == SI_ROPE_SCALE_YARN && !(sc->beta_slow > 0.0 && sc->beta_fast > sc->beta_slow && std::isfinite(sc->beta_fast)))
    return bad(SI_E_INVALID, "rotary scaling needs beta_fast > beta_slow > 0");
  if (sc->kind == SI_ROPE_SCALE_BANDED && !(sc->low > 0.0 && sc->high > sc->low && std::isfinite(sc->high)))
    return bad(SI_E_INVALID, "rotary scaling needs high > low > 0");
  if (!turns || !scale) return bad(SI_E_INVALID, "rotary table is null");
  // long double: the 64-bit fraction of a turn wants 64 bits of mantissa
  const long double two_pi = 6.283185307179586476925286766559005768L, d = rotary_dim, factor = sc->factor;
  long double base = theta, lo = 0, hi = 0;
  if (sc->kind == SI_ROPE_SCALE_NTK && rotary_dim > 2) base *= powl(factor, d / (d - 2));
  if (sc->kind == SI_ROPE_SCALE_YARN) {
    auto pair_of = [&](long double turns_over) { return d * logl(sc->original / (turns_over * two_pi)) / (2 * logl(theta)); };
    lo = std::fmax(floorl(pair_of(sc->beta_fast)), 0.0L);
    hi = std::fmin(ceill(pair_of(sc->beta_slow)), d - 1);
  }
  for (uint32_t i = 0; i < rotary_dim / 2; ++i) {
    long double f = powl(base, -2.0L * i / d);
    if (sc->kind == SI_ROPE_SCALE_LINEAR) f /= factor;
    if (sc->kind == SI_ROPE_SCALE_YARN) {
      const long double far = std::fmin(std::fmax((i - lo) / std::fmax(hi - lo, 0.001L), 0.0L), 1.0L);
      f = f / factor * far + f * (1 - far);
    }
    if (sc->kind == SI_ROPE_SCALE_BANDED) {
      const long double over = sc->original * f / two_pi;  // turns over the trained context
      const long double near = std::fmin(std::fmax((over - sc->low) / (sc->high - sc->low), 0.0L), 1.0L);
      f = f / factor * (1 - near) + f * near;
    }
    turns[i] = uint64_t(roundl(f / two_pi * 18446744073709551616.0L));  // f <= 1 rad: below 2^62
  }
  *scale = sc->kind == SI_ROPE_SCALE_YARN ? float(0.1 * std::log(sc->factor) + 1.0) : 1.0f;
  return SI_OK;
}
