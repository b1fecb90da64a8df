"""Binding of the paged-cache operators (include/si_paged.h): descriptions of a
cache and of each call, built once from torch tensors on the GPU and reused as
long as the tensors live. The calls are methods of `CudaContext`."""
from __future__ import annotations

import ctypes as C

import numpy as np

ELEM_F32, ELEM_BF16, ELEM_F16 = 0, 1, 2
ROPE_INTERLEAVED, ROPE_HALF = 0, 1
ROPE_SCALE_NONE, ROPE_SCALE_LINEAR, ROPE_SCALE_NTK, ROPE_SCALE_YARN, ROPE_SCALE_BANDED = range(5)
_KINDS = {"none": ROPE_SCALE_NONE, "linear": ROPE_SCALE_LINEAR, "ntk": ROPE_SCALE_NTK, "yarn": ROPE_SCALE_YARN,
          "banded": ROPE_SCALE_BANDED}
_LAYOUTS = {"interleaved": ROPE_INTERLEAVED, "half": ROPE_HALF}

_vp, _u64, _u32, _f32, _f64, _i32 = C.c_void_p, C.c_uint64, C.c_uint32, C.c_float, C.c_double, C.c_int


class _Described(C.Structure):
    """A structure that keeps the tensors alive whose addresses it holds."""

    _fits = ()  # (field, value) of the caches that its tensors have the sizes for

    def _hold(self, *tensors):
        self._tensors = [t for t in tensors if t is not None]
        at = self._tensors[0].device
        self._device = at.index if at.type == "cuda" else -1
        return self

    def _for(self, kv, *fields):
        self._fits = tuple((f, getattr(kv, f)) for f in fields)
        return self

    def check_cache(self, kv):
        """Refuses a cache that the call's tensors are not made for: another
        layer's pools of the same shape are fine, other sizes would be read past the end."""
        for field, n in self._fits:
            if getattr(kv, field) != n:
                _fail(f"the call was described for a cache of {field} {n}, not {getattr(kv, field)}")


class SiPagedKv(_Described):
    _fields_ = [("k", _vp), ("v", _vp), ("pages", _vp), ("num_pages", _u64), ("page_stride", _u64), ("head_stride", _u64),
                ("token_stride", _u64), ("pages_stride", _u64), ("elem", _u32), ("kv_heads", _u32), ("head_dim", _u32),
                ("page_tokens", _u32), ("sequences", _u32), ("max_pages", _u32)]


class SiRopeScaling(C.Structure):
    _fields_ = [("kind", _u32), ("factor", _f64), ("original", _f64), ("beta_fast", _f64), ("beta_slow", _f64),
                ("low", _f64), ("high", _f64)]


class SiPagedAppend(_Described):
    _fields_ = [("q", _vp), ("q_out", _vp), ("k", _vp), ("v", _vp), ("q_token_stride", _u64), ("q_head_stride", _u64),
                ("q_out_token_stride", _u64), ("q_out_head_stride", _u64), ("k_token_stride", _u64),
                ("k_head_stride", _u64), ("v_token_stride", _u64), ("v_head_stride", _u64), ("sequence", _vp),
                ("slot", _vp), ("position", _vp), ("rope", _vp), ("rope_scale", _f32), ("elem", _u32), ("tokens", _u32),
                ("query_heads", _u32), ("rotary_dim", _u32), ("rope_layout", _u32), ("weights", _vp),
                ("positions", _vp), ("weights_stride", _u64)]


class SiPagedAttention(_Described):
    _fields_ = [("q", _vp), ("out", _vp), ("q_seq_stride", _u64), ("q_head_stride", _u64), ("out_seq_stride", _u64),
                ("out_head_stride", _u64), ("lengths", _vp), ("scale", _f32), ("elem", _u32), ("query_heads", _u32),
                ("lse", _vp), ("weights_in", _vp), ("weights_out", _vp), ("weights_stride", _u64), ("work", _vp),
                ("work_bytes", _u64)]


class SiPagedEvict(_Described):
    _fields_ = [("lengths_in", _vp), ("lengths_out", _vp), ("weights_in", _vp), ("weights_out", _vp),
                ("positions_in", _vp), ("positions_out", _vp), ("next_position", _vp), ("weights_stride", _u64),
                ("budget", _u32), ("sink", _u32), ("recent", _u32), ("work", _vp), ("work_bytes", _u64)]


class SiVerifyDrafts(_Described):
    _fields_ = [("target", _vp), ("draft", _vp), ("target_seq_stride", _u64), ("target_row_stride", _u64),
                ("draft_seq_stride", _u64), ("draft_row_stride", _u64), ("tokens", _vp), ("counts", _vp),
                ("uniform", _vp), ("last_uniform", _vp), ("accepted", _vp), ("next", _vp), ("sequences", _u32),
                ("drafts", _u32), ("vocab", _u32), ("work", _vp), ("work_bytes", _u64)]


SIGNATURES = {
    "si_paged_kv_offset": ([_vp, C.c_int64, _u64, _u32, _vp], _i32),
    "si_rope_table": ([_f64, _u32, _vp, _vp, _vp], _i32),
    "si_paged_append_dev": ([_vp, _vp, _vp, _vp], _i32),
    "si_paged_attention_workspace": ([_vp, _u32, _i32, _vp], _i32),
    "si_paged_attention_dev": ([_vp, _vp, _vp, _vp], _i32),
    "si_paged_evict_workspace": ([_vp, _vp], _i32),
    "si_paged_evict_dev": ([_vp, _vp, _vp, _vp], _i32),
    "si_verify_drafts_workspace": ([_u32, _u32, _vp], _i32),
    "si_verify_drafts_dev": ([_vp, _vp, _vp], _i32),
}


def _fail(text):
    from . import SI_E_INVALID, SiError
    raise SiError(SI_E_INVALID, text)


def _call(name, *args):
    from . import SiError, lib
    rc = getattr(lib(), name)(*args)
    if rc != 0:
        raise SiError(rc, lib().si_global_last_error().decode())


def _elem(t):
    name = str(t.dtype)
    if name not in ("torch.float32", "torch.bfloat16", "torch.float16"):
        _fail(f"elements must be float32, bfloat16 or float16, not {name}")
    return {"torch.float32": ELEM_F32, "torch.bfloat16": ELEM_BF16, "torch.float16": ELEM_F16}[name]


def _rows(t, shape, what):
    """Checks the shape of a tensor with contiguous dims; its two outer strides."""
    if t.dim() != 3 or tuple(t.shape) != tuple(shape):
        _fail(f"{what} must be {list(shape)}, not {list(t.shape)}")
    if t.stride(2) != 1 and t.shape[2] != 1:
        _fail(f"{what} must have contiguous dims")
    return t.stride(0), t.stride(1)


def _plain(t, dtype, shape, what):
    """The address of a contiguous tensor of this type and shape (None: NULL)."""
    if t is None:
        return None
    if str(t.dtype) != "torch." + dtype or not t.is_contiguous() or tuple(t.shape) != tuple(shape):
        _fail(f"{what} must be a contiguous {dtype} tensor {list(shape)}, not {t.dtype} {list(t.shape)}")
    return t.data_ptr()


def _same_device(*tensors):
    devices = {t.device for t in tensors if t is not None}
    if len(devices) > 1:
        _fail("tensors are on different devices: " + ", ".join(sorted(map(str, devices))))


def _work(t):
    return (None, 0) if t is None else (t.data_ptr(), t.numel() * t.element_size())


def paged_kv(k, v, pages) -> SiPagedKv:
    """si_paged_kv: pools [pages][kv_heads][page_tokens][head_dim] (any strides,
    so other orders are transposed views) and the page table [sequences][max_pages]."""
    if k.dim() != 4 or k.shape != v.shape or k.stride() != v.stride() or k.dtype != v.dtype:
        _fail("key and value pools must have the same four dimensions, strides and type")
    if k.stride(3) != 1 and k.shape[3] != 1:
        _fail("cache pools must have contiguous dims")
    if pages.dim() != 2 or str(pages.dtype) != "torch.int32" or (pages.stride(1) != 1 and pages.shape[1] != 1):
        _fail("the page table must be an int32 tensor [sequences][max_pages] with contiguous rows")
    _same_device(k, v, pages)
    kv = SiPagedKv(k.data_ptr(), v.data_ptr(), pages.data_ptr(), k.shape[0], k.stride(0), k.stride(1), k.stride(2),
                   max(pages.stride(0), pages.shape[1]) if pages.shape[0] == 1 else pages.stride(0),
                   _elem(k), k.shape[1], k.shape[3], k.shape[2], pages.shape[0], pages.shape[1])
    return kv._hold(k, v, pages)


def paged_kv_offset(kv: SiPagedKv, page: int, slot: int, head: int) -> int:
    """si_paged_kv_offset: where a slot lies in a pool (elements)."""
    at = C.c_uint64()
    _call("si_paged_kv_offset", C.byref(kv), page, slot, head, C.byref(at))
    return at.value


def rope_table(theta: float, rotary_dim: int, kind: str = "none", factor: float = 1.0, original: float = 0.0,
               beta_fast: float = 32.0, beta_slow: float = 1.0, low: float = 1.0, high: float = 4.0):
    """si_rope_table: (turns a position as uint64 [rotary_dim / 2], factor on rotated values)."""
    if kind not in _KINDS:
        _fail(f"unknown rotary scaling {kind!r}")
    turns, scale = np.zeros(max(rotary_dim // 2, 1), np.uint64), C.c_float()
    s = SiRopeScaling(_KINDS[kind], factor, original, beta_fast, beta_slow, low, high)
    _call("si_rope_table", theta, rotary_dim, C.byref(s), turns.ctypes.data, C.byref(scale))
    return turns[:rotary_dim // 2], scale.value


def paged_append(kv: SiPagedKv, q, k, v, q_out, slot, sequence=None, position=None, rope=None, rotary_dim: int = 0,
                 layout: str = "interleaved", rope_scale: float = 1.0, weights=None, positions=None) -> SiPagedAppend:
    """si_paged_append: q [tokens][query_heads][head_dim] with q_out, k and v
    [tokens][kv_heads][head_dim] (either pair may be None), slot, sequence and
    position int32 [tokens], rope the device copy of `rope_table`'s turns
    (int64 [rotary_dim / 2]); weights float32 and positions int32
    [sequences][kv_heads][slots], where appended slots start anew."""
    if layout not in _LAYOUTS:
        _fail(f"unknown rotary layout {layout!r}")
    if slot.dim() != 1:
        _fail("slots must be [tokens]")
    n = slot.shape[0]
    a = SiPagedAppend(rope_scale=rope_scale, tokens=n, rotary_dim=rotary_dim, rope_layout=_LAYOUTS[layout])
    given = [t for t in (q, q_out, k, v) if t is not None]
    if (q is None) != (q_out is None) or (k is None) != (v is None) or not given:
        _fail("paged append needs q and q_out together, k and v together, and one of both")
    if len({t.dtype for t in given}) > 1:
        _fail("q, k, v and q_out must have the same type")
    a.elem = _elem(given[0])
    if q is not None:
        shape = (n, q.shape[1] if q.dim() == 3 else 0, kv.head_dim)
        a.q, a.q_out, a.query_heads = q.data_ptr(), q_out.data_ptr(), shape[1]
        a.q_token_stride, a.q_head_stride = _rows(q, shape, "q")
        a.q_out_token_stride, a.q_out_head_stride = _rows(q_out, shape, "q_out")
    if k is not None:
        shape = (n, kv.kv_heads, kv.head_dim)
        a.k, a.v = k.data_ptr(), v.data_ptr()
        a.k_token_stride, a.k_head_stride = _rows(k, shape, "k")
        a.v_token_stride, a.v_head_stride = _rows(v, shape, "v")
    a.slot = _plain(slot, "int32", (n,), "slot")
    a.sequence = _plain(sequence, "int32", (n,), "sequence")
    a.position = _plain(position, "int32", (n,), "position")
    a.rope = _plain(rope, "int64", (rotary_dim // 2,), "rope") if rotary_dim else None
    started = [t for t in (weights, positions) if t is not None]
    if started:
        shape = (kv.sequences, kv.kv_heads, started[0].shape[-1])
        a.weights = _plain(weights, "float32", shape, "weights")
        a.positions = _plain(positions, "int32", shape, "positions")
        a.weights_stride = shape[2]
    _same_device(*given, slot, sequence, position, rope, *started, kv._tensors[0])
    a._for(kv, "kv_heads", "head_dim", *(("sequences",) if started else ()))
    return a._hold(*given, slot, sequence, position, rope, *started)


def paged_attention_workspace_bytes(kv: SiPagedKv, query_heads: int, weights: bool = False) -> int:
    n = C.c_uint64()
    _call("si_paged_attention_workspace", C.byref(kv), query_heads, int(weights), C.byref(n))
    return n.value


def paged_attention(kv: SiPagedKv, q, out, lengths, work, scale: float = 0.0, lse=None, weights_in=None,
                    weights_out=None) -> SiPagedAttention:
    """si_paged_attention: q and out [sequences][query_heads][head_dim], lengths
    int32 [sequences], lse float32 [sequences][query_heads], weights float32
    [sequences][kv_heads][slots]; work a byte tensor of paged_attention_workspace_bytes."""
    n, heads = kv.sequences, q.shape[1] if q.dim() == 3 else 0
    a = SiPagedAttention(q=q.data_ptr(), out=out.data_ptr(), scale=scale, elem=_elem(q), query_heads=heads)
    if out.dtype != q.dtype:
        _fail("out must have the type of q")
    a.q_seq_stride, a.q_head_stride = _rows(q, (n, heads, kv.head_dim), "q")
    a.out_seq_stride, a.out_head_stride = _rows(out, (n, heads, kv.head_dim), "out")
    a.lengths = _plain(lengths, "int32", (n,), "lengths")
    a.lse = _plain(lse, "float32", (n, heads), "lse")
    if weights_out is not None:
        shape = (n, kv.kv_heads, weights_out.shape[-1])
        a.weights_out = _plain(weights_out, "float32", shape, "weights_out")
        a.weights_stride = shape[2]
        a.weights_in = _plain(weights_in, "float32", shape, "weights_in")
    elif weights_in is not None:
        _fail("paged attention has weights in and none out")
    a.work, a.work_bytes = _work(work)
    _same_device(q, out, lengths, work, lse, weights_in, weights_out, kv._tensors[0])
    a._for(kv, "sequences", "kv_heads", "head_dim")
    return a._hold(q, out, lengths, work, lse, weights_in, weights_out)


def paged_evict_workspace_bytes(kv: SiPagedKv) -> int:
    n = C.c_uint64()
    _call("si_paged_evict_workspace", C.byref(kv), C.byref(n))
    return n.value


def paged_evict(kv: SiPagedKv, lengths_in, lengths_out, weights_in, weights_out, budget: int, work, sink: int = 0,
                recent: int = 0, positions_in=None, positions_out=None, next_position=None) -> SiPagedEvict:
    """si_paged_evict: lengths int32 [sequences], weights float32 and positions
    int32 [sequences][kv_heads][slots]; each `_in` may be its `_out`."""
    n = kv.sequences
    shape = (n, kv.kv_heads, weights_in.shape[-1])
    a = SiPagedEvict(weights_stride=shape[2], budget=budget, sink=sink, recent=recent)
    a.lengths_in = _plain(lengths_in, "int32", (n,), "lengths_in")
    a.lengths_out = _plain(lengths_out, "int32", (n,), "lengths_out")
    a.weights_in = _plain(weights_in, "float32", shape, "weights_in")
    a.weights_out = _plain(weights_out, "float32", shape, "weights_out")
    a.positions_in = _plain(positions_in, "int32", shape, "positions_in")
    a.positions_out = _plain(positions_out, "int32", shape, "positions_out")
    a.next_position = _plain(next_position, "int32", (n,), "next_position")
    a.work, a.work_bytes = _work(work)
    a._for(kv, "sequences", "kv_heads")
    held = (lengths_in, lengths_out, weights_in, weights_out, positions_in, positions_out, next_position, work)
    _same_device(*held, kv._tensors[0])
    return a._hold(*held)


def verify_drafts_workspace_bytes(sequences: int, vocab: int) -> int:
    n = C.c_uint64()
    _call("si_verify_drafts_workspace", sequences, vocab, C.byref(n))
    return n.value


def verify_drafts(target, tokens, uniform, last_uniform, accepted, next_token, work, draft_probs=None,
                  counts=None) -> SiVerifyDrafts:
    """si_verify_drafts: target float32 [sequences][drafts + 1][vocab], draft_probs
    [sequences][drafts][vocab] or None, tokens int32 and uniform float32
    [sequences][drafts], counts int32 and last_uniform float32 [sequences];
    accepted and next_token int32 [sequences] are written."""
    if target.dim() != 3 or target.shape[1] < 1 or str(target.dtype) != "torch.float32":
        _fail("target must be float32 [sequences][drafts + 1][vocab]")
    n, k, vocab = target.shape[0], target.shape[1] - 1, target.shape[2]
    a = SiVerifyDrafts(sequences=n, drafts=k, vocab=vocab, target=target.data_ptr())
    a.target_seq_stride, a.target_row_stride = _rows(target, (n, k + 1, vocab), "target")
    if draft_probs is not None and k:
        if str(draft_probs.dtype) != "torch.float32":
            _fail("draft_probs must be float32")
        a.draft_seq_stride, a.draft_row_stride = _rows(draft_probs, (n, k, vocab), "draft_probs")
        a.draft = draft_probs.data_ptr()
    if k:
        a.tokens = _plain(tokens, "int32", (n, k), "tokens")
        a.uniform = _plain(uniform, "float32", (n, k), "uniform")
    a.counts = _plain(counts, "int32", (n,), "counts")
    a.last_uniform = _plain(last_uniform, "float32", (n,), "last_uniform")
    a.accepted = _plain(accepted, "int32", (n,), "accepted")
    a.next = _plain(next_token, "int32", (n,), "next_token")
    a.work, a.work_bytes = _work(work)
    held = (target, tokens, uniform, last_uniform, accepted, next_token, work, draft_probs, counts)
    _same_device(*held)
    return a._hold(*held)
