"""CPU checks of the paged-cache operators (include/si_paged.h): the ABI's
surface, the place of a slot, the rotary tables, and every refusal of an
argument (checked before a device is touched)."""
import ctypes as C
import math
import os
import re

import numpy as np
import pytest
import torch

from conftest import REPO, load_package

mai = load_package()
L = mai.lib()
INVALID, UNSUPPORTED = mai.SI_E_INVALID, mai.SI_E_UNSUPPORTED

ABI_ENTRY_POINTS = [
    "si_paged_append_dev", "si_paged_attention_dev", "si_paged_attention_workspace", "si_paged_evict_dev",
    "si_paged_evict_workspace", "si_paged_kv_offset", "si_rope_table", "si_verify_drafts_dev",
    "si_verify_drafts_workspace",
]


def test_header_declares_exactly_the_abi_surface():
    h = open(os.path.join(REPO, "include", "si_paged.h")).read()
    h = re.sub(r"/\*.*?\*/", "", h, flags=re.S)
    assert sorted(set(re.findall(r"\b(si_[a-z0-9_]+)\s*\(", h))) == ABI_ENTRY_POINTS
    assert sorted(mai.paged.SIGNATURES) == ABI_ENTRY_POINTS
    for name in ABI_ENTRY_POINTS:
        assert hasattr(L, name)


def test_structures_match_the_header(tmp_path):
    """A C99 program prints the size and the field offsets of every structure."""
    import subprocess
    pairs = [("si_paged_kv", mai.SiPagedKv), ("si_rope_scaling", mai.paged.SiRopeScaling),
             ("si_paged_append", mai.SiPagedAppend), ("si_paged_attention", mai.SiPagedAttention),
             ("si_paged_evict", mai.SiPagedEvict), ("si_verify_drafts", mai.SiVerifyDrafts)]
    lines = []
    for name, cls in pairs:
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        lines += [f'printf("%zu\\n", offsetof({name}, {f}));' for f, _ in cls._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include "si_paged.h"\nint main(void) {\n' + "\n".join(lines) + "\nreturn 0;\n}\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Wextra", "-pedantic", "-Werror", "-I", os.path.join(REPO, "include"),
                    str(src), "-o", str(exe)], check=True)
    got = list(map(int, subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()))
    want = []
    for _, cls in pairs:
        want.append(C.sizeof(cls))
        want += [getattr(cls, f).offset for f, _ in cls._fields_]
    assert got == want


def pools(pages=6, kv_heads=2, page=4, hd=16, dtype=torch.bfloat16, seqs=3, cols=2):
    k = torch.zeros(pages, kv_heads, page, hd, dtype=dtype)
    return k, torch.zeros_like(k), torch.zeros(seqs, cols, dtype=torch.int32)


# ---- the place of a slot ----------------------------------------------------
@pytest.mark.parametrize("order", ["heads_first", "tokens_first"])
@pytest.mark.parametrize("page", [1, 3, 4, 16, 24, 256])
def test_offset_follows_the_strides(order, page):
    k = torch.zeros(7, 5, page, 24, dtype=torch.float16)
    if order == "tokens_first":
        k = torch.zeros(7, page, 5, 24, dtype=torch.float16).transpose(1, 2)
    kv = mai.paged_kv(k, k, torch.zeros(2, 9, dtype=torch.int32))
    for slot in {0, 1, page - 1, page, 2 * page + 1, 9 * page - 1} & set(range(9 * page)):
        for p in (0, 6):
            for h in (0, 4):
                assert mai.paged_kv_offset(kv, p, slot, h) == p * k.stride(0) + h * k.stride(1) + slot % page * k.stride(2)


def test_offset_passes_32_bits():
    k, v, pages = pools(pages=1, kv_heads=1, page=16, hd=128)
    kv = mai.paged_kv(k, v, pages)
    kv.num_pages, kv.page_stride = 1 << 30, 1 << 20
    assert mai.paged_kv_offset(kv, (1 << 30) - 1, 17, 0) == ((1 << 30) - 1) * (1 << 20) + 128


@pytest.mark.parametrize("page, slot, head", [(-1, 0, 0), (6, 0, 0), (1 << 40, 0, 0), (-(1 << 40), 0, 0), (0, 8, 0), (0, 0, 2)])
def test_offset_refuses_what_is_outside(page, slot, head):
    kv = mai.paged_kv(*pools())
    with pytest.raises(mai.SiError):
        mai.paged_kv_offset(kv, page, slot, head)


def test_division_of_slots_is_exact():
    """Every page size up to 600 and some large ones, at multiples and their neighbours."""
    k, v, pages = pools(page=1, hd=8)
    for page in list(range(1, 601)) + [1023, 4097, 65535, 1 << 20, (1 << 20) + 7, 1 << 28]:
        kv = mai.paged_kv(k, v, pages)
        kv.page_tokens, kv.max_pages, kv.sequences = page, (2 ** 31 - 1) // page, 1
        kv.pages_stride = kv.max_pages
        kv.token_stride, kv.page_stride, kv.head_stride = 8, 0, 0
        last = page * kv.max_pages - 1
        for t in {0, page - 1, page, last, last - page, last // 2, last // 2 // page * page, last // 2 // page * page - 1}:
            if 0 <= t <= last:
                assert mai.paged_kv_offset(kv, 0, t, 0) == t % page * 8, (page, t)


# ---- rotary tables ------------------------------------------------------------
def frequencies(theta, d, kind, factor=1.0, original=0.0, beta_fast=32.0, beta_slow=1.0, low=1.0, high=4.0):
    got = []
    for i in range(d // 2):
        base = theta * factor ** (d / (d - 2)) if kind == "ntk" and d > 2 else theta
        f = base ** (-2 * i / d)
        if kind == "linear":
            f /= factor
        if kind == "yarn":
            at = [d * math.log(original / (2 * math.pi * b)) / (2 * math.log(theta)) for b in (beta_fast, beta_slow)]
            lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), d - 1)
            far = min(max((i - lo) / max(hi - lo, 0.001), 0), 1)
            f = f / factor * far + f * (1 - far)
        if kind == "banded":
            over = original * f / (2 * math.pi)
            near = min(max((over - low) / (high - low), 0), 1)
            f = f / factor * (1 - near) + f * near
        got.append(f)
    return np.array(got)


@pytest.mark.parametrize("d", [2, 6, 20, 64, 128, 256])
@pytest.mark.parametrize("kind, more", [("none", {}), ("linear", {"factor": 4.0}), ("ntk", {"factor": 8.0}),
                                        ("yarn", {"factor": 16.0, "original": 4096}),
                                        ("yarn", {"factor": 1.0, "original": 4}),
                                        ("banded", {"factor": 8.0, "original": 8192})])
@pytest.mark.parametrize("theta", [1.5, 1e4, 1e7])
def test_rope_table(theta, kind, more, d):
    turns, scale = mai.rope_table(theta, d, kind, **more)
    want = frequencies(theta, d, kind, **more) / (2 * math.pi)
    # the table rounds to 2^-65 turns; the double formula here is off by some 2^-50 relative
    assert np.all(np.abs(turns.astype(np.float64) / 2.0 ** 64 - want) <= 2.0 ** -64 + want * 2.0 ** -46)
    assert scale == pytest.approx(0.1 * math.log(more["factor"]) + 1 if kind == "yarn" else 1.0, rel=2 ** -23)


@pytest.mark.parametrize("args, kw", [((1.0, 8), {}), ((math.nan, 8), {}), ((math.inf, 8), {}), ((1e4, 7), {}), ((1e4, 258), {}),
                                      ((1e4, 8, "linear"), {"factor": 0.5}), ((1e4, 8, "ntk"), {"factor": math.nan}),
                                      ((1e4, 8, "yarn"), {"factor": 2.0}),
                                      ((1e4, 8, "yarn"), {"factor": 2.0, "original": 8, "beta_fast": 1.0, "beta_slow": 1.0}),
                                      ((1e4, 8, "banded"), {"factor": 2.0, "original": 8, "low": 4.0, "high": 4.0}),
                                      ((1e4, 8, "sideways"), {})])
def test_rope_table_refuses(args, kw):
    with pytest.raises(mai.SiError):
        mai.rope_table(*args, **kw)


# ---- refusals -------------------------------------------------------------------
def refused(fn, *args, status=INVALID):
    """The call without a context refuses the arguments themselves."""
    rc = fn(None, *[C.byref(a) if a is not None else None for a in args], None)
    text = L.si_global_last_error().decode()
    assert rc == status, (rc, text)
    assert text and "null context" not in text, text


def accepted(fn, *args):
    """Arguments that pass the checks: only the context is missing."""
    assert fn(None, *[C.byref(a) for a in args], None) == INVALID
    assert L.si_global_last_error().decode() == "null context"


KV_FAULTS = [("elem", 0, UNSUPPORTED), ("elem", 3, UNSUPPORTED), ("kv_heads", 0, INVALID), ("kv_heads", 65536, INVALID),
             ("head_dim", 0, INVALID), ("head_dim", 12, UNSUPPORTED), ("head_dim", 264, UNSUPPORTED),
             ("page_tokens", 0, INVALID), ("page_tokens", 1 << 30, UNSUPPORTED), ("num_pages", 0, INVALID),
             ("num_pages", 1 << 31, UNSUPPORTED), ("max_pages", 0, INVALID), ("sequences", 0, INVALID),
             ("sequences", 4097, UNSUPPORTED), ("pages_stride", 1, INVALID), ("page_stride", 9, INVALID),
             ("head_stride", 4, INVALID), ("token_stride", 12, INVALID), ("page_stride", 1 << 62, INVALID),
             ("k", None, INVALID), ("v", None, INVALID), ("pages", None, INVALID)]


def attention_call(weights=False):
    kv = mai.paged_kv(*pools())
    q = torch.zeros(3, 4, 16)
    work = torch.zeros(mai.paged_attention_workspace_bytes(kv, 4, weights) // 8 + 2, dtype=torch.float64)
    w = torch.zeros(3, 2, 8) if weights else None
    return kv, mai.paged_attention(kv, q, torch.zeros_like(q), torch.zeros(3, dtype=torch.int32), work, weights_in=w,
                                   weights_out=w)


def append_call():
    kv = mai.paged_kv(*pools())
    q, k = torch.zeros(3, 4, 16), torch.zeros(3, 2, 16)
    return kv, mai.paged_append(kv, q, k, k, q, torch.zeros(3, dtype=torch.int32),
                                rope=torch.zeros(4, dtype=torch.int64), rotary_dim=8)


def evict_call():
    kv = mai.paged_kv(*pools())
    n, w, p = torch.zeros(3, dtype=torch.int32), torch.zeros(3, 2, 8), torch.zeros(3, 2, 8, dtype=torch.int32)
    work = torch.zeros(mai.paged_evict_workspace_bytes(kv) // 8 + 2, dtype=torch.float64)
    return kv, mai.paged_evict(kv, n, n, w, w, 4, work, sink=1, recent=3, positions_in=p, positions_out=p)


def verify_call():
    n = torch.zeros(3, dtype=torch.int32)
    work = torch.zeros(mai.verify_drafts_workspace_bytes(3, 50) // 8 + 2, dtype=torch.float64)
    return (mai.verify_drafts(torch.zeros(3, 5, 50), torch.zeros(3, 4, dtype=torch.int32), torch.zeros(3, 4), torch.zeros(3),
                              n, n, work, draft_probs=torch.zeros(3, 4, 50)),)


CALLS = {"append": (append_call, L.si_paged_append_dev), "attention": (attention_call, L.si_paged_attention_dev),
         "evict": (evict_call, L.si_paged_evict_dev), "verify": (verify_call, L.si_verify_drafts_dev)}


@pytest.mark.parametrize("name", CALLS)
def test_whole_descriptions_are_accepted_and_missing_ones_refused(name):
    make, fn = CALLS[name]
    args = make()
    accepted(fn, *args)
    for i in range(len(args)):
        refused(fn, *[None if j == i else a for j, a in enumerate(args)])


@pytest.mark.parametrize("name", ["append", "attention", "evict"])
@pytest.mark.parametrize("field, value, status", KV_FAULTS)
def test_cache_faults_are_refused(name, field, value, status):
    make, fn = CALLS[name]
    kv, a = make()
    setattr(kv, field, value)
    refused(fn, kv, a, status=status)


def test_misaligned_pools_are_refused():
    for field in ("k", "v"):
        kv, a = attention_call()
        setattr(kv, field, getattr(kv, field) + 2)
        refused(L.si_paged_attention_dev, kv, a)


FAULTS = [
    ("append", "elem", 3, UNSUPPORTED), ("append", "tokens", 1 << 23, UNSUPPORTED), ("append", "tokens", 4, INVALID),
    ("append", "q", None, INVALID), ("append", "q_out", None, INVALID), ("append", "k", None, INVALID),
    ("append", "query_heads", 0, INVALID), ("append", "query_heads", 65536, INVALID), ("append", "rotary_dim", 7, INVALID),
    ("append", "rotary_dim", 18, INVALID), ("append", "rope_layout", 2, INVALID), ("append", "rope", None, INVALID),
    ("append", "slot", None, INVALID), ("append", "k_token_stride", 1 << 40, INVALID),
    ("attention", "elem", 7, UNSUPPORTED), ("attention", "q", None, INVALID), ("attention", "out", None, INVALID),
    ("attention", "lengths", None, INVALID), ("attention", "query_heads", 0, INVALID),
    ("attention", "query_heads", 3, INVALID), ("attention", "scale", -1.0, INVALID), ("attention", "scale", math.inf, INVALID),
    ("attention", "scale", math.nan, INVALID), ("attention", "work", None, INVALID), ("attention", "work_bytes", 64, INVALID),
    ("attention", "q_seq_stride", 1 << 50, INVALID),
    ("evict", "lengths_in", None, INVALID), ("evict", "lengths_out", None, INVALID), ("evict", "weights_in", None, INVALID),
    ("evict", "weights_out", None, INVALID), ("evict", "positions_out", None, INVALID), ("evict", "budget", 0, INVALID),
    ("evict", "budget", 3, INVALID), ("evict", "sink", 0xffffffff, INVALID), ("evict", "weights_stride", 0, INVALID),
    ("evict", "work", None, INVALID), ("evict", "work_bytes", 8, INVALID),
    ("verify", "sequences", 0, INVALID), ("verify", "sequences", 65536, INVALID), ("verify", "vocab", 0, INVALID),
    ("verify", "vocab", 1 << 31, INVALID), ("verify", "drafts", 33, UNSUPPORTED), ("verify", "target", None, INVALID),
    ("verify", "tokens", None, INVALID), ("verify", "uniform", None, INVALID), ("verify", "last_uniform", None, INVALID),
    ("verify", "accepted", None, INVALID), ("verify", "next", None, INVALID), ("verify", "work_bytes", 0, INVALID),
    ("verify", "target_seq_stride", 1 << 60, INVALID),
]


@pytest.mark.parametrize("name, field, value, status", FAULTS)
def test_faults_of_a_call_are_refused(name, field, value, status):
    make, fn = CALLS[name]
    args = make()
    setattr(args[-1], field, value)
    refused(fn, *args, status=status)


def test_more_refusals():
    kv, a = attention_call()
    a.work += 8
    refused(L.si_paged_attention_dev, kv, a)
    kv, a = attention_call()
    a.weights_in = a.q
    refused(L.si_paged_attention_dev, kv, a)
    kv, a = attention_call(weights=True)
    a.weights_stride = 0
    refused(L.si_paged_attention_dev, kv, a)
    kv, a = attention_call(weights=True)
    a.work_bytes = mai.paged_attention_workspace_bytes(kv, 4) // 16 * 16  # room for the call without weights
    refused(L.si_paged_attention_dev, kv, a)
    kv, a = evict_call()
    kv.page_tokens, kv.max_pages = 393217, 1
    refused(L.si_paged_evict_dev, kv, a, status=UNSUPPORTED)
    with pytest.raises(mai.SiError):
        mai.paged_evict_workspace_bytes(kv)
    kv, a = attention_call()
    kv.sequences, kv.kv_heads, kv.page_tokens, kv.max_pages, kv.pages_stride = 256, 2, 1 << 20, 1 << 10, 1 << 10
    a.query_heads = 1 << 15  # 2^24 units of 256 sequences, 2 kv heads and 2048 blocks of query heads
    refused(L.si_paged_attention_dev, kv, a, status=UNSUPPORTED)
    kv, a = append_call()
    a.q += 2
    refused(L.si_paged_append_dev, kv, a)


def test_bindings_refuse_tensors_that_do_not_fit():
    k, v, pages = pools()
    bad = [lambda: mai.paged_kv(k, v[:, :1], pages), lambda: mai.paged_kv(k, v.float(), pages),
           lambda: mai.paged_kv(k[..., ::2], v[..., ::2], pages), lambda: mai.paged_kv(k, v, pages.long()),
           lambda: mai.paged_kv(k, v, pages[0])]
    kv = mai.paged_kv(k, v, pages)
    n, q, w = torch.zeros(3, dtype=torch.int32), torch.zeros(3, 4, 16), torch.zeros(1024, dtype=torch.uint8)
    att = lambda **x: mai.paged_attention(**{**dict(kv=kv, q=q, out=q, lengths=n, work=w), **x})  # noqa: E731
    bad += [lambda: att(lengths=n.long()), lambda: att(lengths=n[:2]), lambda: att(out=q.half()), lambda: att(q=q[:, :, :8]),
            lambda: att(q=q[:2]), lambda: att(weights_in=q), lambda: att(weights_out=torch.zeros(3, 4, 8)),
            lambda: att(q=q.double())]
    app = lambda **x: mai.paged_append(**{**dict(kv=kv, q=q, k=q[:, :2], v=q[:, :2], q_out=q, slot=n), **x})  # noqa: E731
    bad += [lambda: app(q_out=None), lambda: app(k=None), lambda: app(q=None, q_out=None, k=None, v=None),
            lambda: app(k=q[:, :2].half(), v=q[:, :2].half()), lambda: app(slot=n.long()), lambda: app(slot=n[:2]),
            lambda: app(layout="spiral"), lambda: app(rotary_dim=8, rope=torch.zeros(3, dtype=torch.int64))]
    p = torch.zeros(3, 5, 50)
    ver = lambda **x: mai.verify_drafts(**{**dict(target=p, tokens=torch.zeros(3, 4, dtype=torch.int32), uniform=p[:, :4, 0].contiguous(),  # noqa: E731
                                                  last_uniform=p[:, 0, 0].contiguous(), accepted=n, next_token=n, work=w), **x})
    bad += [lambda: ver(target=p.double()), lambda: ver(draft_probs=p), lambda: ver(draft_probs=p[:, :4].double()),
            lambda: ver(uniform=p[:, :4, 0]), lambda: ver(counts=n.long())]
    for i, f in enumerate(bad):
        with pytest.raises(mai.SiError):
            f()
            pytest.fail(f"case {i} was taken")


WORDS = {"append": ["sequence", "slot", "position"], "attention": ["lengths", "lse", "weights_in", "weights_out"],
         "evict": ["lengths_in", "lengths_out", "weights_in", "weights_out", "positions_in", "positions_out", "next_position"],
         "verify": ["target", "draft", "tokens", "counts", "uniform", "last_uniform", "accepted", "next"]}


@pytest.mark.parametrize("name, field", [(n, f) for n, fields in WORDS.items() for f in fields])
def test_misaligned_arrays_are_refused(name, field):
    make, fn = CALLS[name]
    args = make(True) if name == "attention" else make()
    setattr(args[-1], field, (getattr(args[-1], field) or 4096) + 2)
    refused(fn, *args)


@pytest.mark.parametrize("name, other, fits", [
    ("append", dict(seqs=5), True), ("append", dict(kv_heads=3), False), ("append", dict(hd=24), False),
    ("attention", dict(), True), ("attention", dict(pages=9, page=16), True), ("attention", dict(seqs=4), False),
    ("attention", dict(kv_heads=1), False), ("attention", dict(hd=8), False),
    ("evict", dict(hd=32), True), ("evict", dict(seqs=2), False), ("evict", dict(kv_heads=4), False)])
def test_a_call_refuses_a_cache_of_other_sizes(name, other, fits):
    """Another layer's pools of the same shape are the ordinary use."""
    _, a = CALLS[name][0]()
    ctx = object.__new__(mai.CudaContext)
    ctx.device, ctx.h = -1, None  # where tensors on the CPU are; the C call then lacks a context
    kv = mai.paged_kv(*pools(**other))
    call = {"append": ctx.paged_append_dev, "attention": ctx.paged_attention_dev, "evict": ctx.paged_evict_dev}[name]
    if name == "evict":
        a.work_bytes = 1 << 20  # not read: nothing is launched
    with pytest.raises(mai.SiError, match="described for a cache" if not fits else "null context"):
        call(kv, a)


def test_outputs_over_inputs_that_others_read_are_refused():
    kv, a = attention_call()
    a.out = a.q
    refused(L.si_paged_attention_dev, kv, a)
    kv, a = evict_call()
    other = torch.zeros(3, dtype=torch.int32)
    a.next_position = a.lengths_out
    accepted(L.si_paged_evict_dev, kv, a)  # lengths_in too: one array for all three
    a.lengths_in = other.data_ptr()
    refused(L.si_paged_evict_dev, kv, a)


# ---- host state that threads share -----------------------------------------------
LIMIT_PROGRAM = r"""
#include "raised_limit.h"

#include <chrono>
#include <cstdio>
#include <thread>

static std::atomic<uint32_t> real{0};
static std::atomic<bool> small_asks{false}, large_set{false}, small_done{false};

static void wait_for(std::atomic<bool>& flag) {  // a fifth of a second at most
  for (int i = 0; i < 200 && !flag; ++i) std::this_thread::sleep_for(std::chrono::milliseconds(1));
}

int main() {
  si::RaisedLimit limit;
  int calls = 0;
  // the smaller size asks first, and its attribute call ends after the larger one's if it may
  std::thread small([&] {
    limit.raise(100, [&](uint32_t n) { small_asks = true; wait_for(large_set); real = n; return 0; });
    small_done = true;
  });
  std::thread large([&] {
    wait_for(small_asks);
    limit.raise(200, [&](uint32_t n) { real = n; large_set = true; wait_for(small_done); return 0; });
  });
  small.join();
  large.join();
  const auto count = [&](uint32_t n) { ++calls; real = n; return 0; };
  limit.raise(200, count);
  if (real < 200 || calls != 0) return std::printf("noted 200, set %u, %d calls\n", real.load(), calls), 1;
  limit.raise(150, count);
  if (real != 200 || calls != 0) return std::printf("lowered\n"), 2;
  // a refused size is not noted
  if (limit.raise(300, [&](uint32_t) { return 7; }) != 7) return 3;
  limit.raise(300, count);
  return real == 300 && calls == 1 ? 0 : 4;
}
"""


def test_a_raised_limit_is_never_lowered_by_another_thread(tmp_path):
    """Two threads raise one kernel's limit to different sizes at once."""
    import subprocess
    src, exe = tmp_path / "limit.cpp", tmp_path / "limit"
    src.write_text(LIMIT_PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", "-pthread", "-I",
                    os.path.join(REPO, "memory-aware-inference_b200", "csrc"), str(src), "-o", str(exe)], check=True)
    got = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert got.returncode == 0, (got.returncode, got.stdout)


@pytest.mark.parametrize("field", ["weights", "positions"])
def test_started_arrays_of_an_append(field):
    """Weights and positions that an append starts anew: with keys, a stride and whole words only."""
    def call():
        kv, a = append_call()
        setattr(a, field, 4096)
        a.weights_stride = 8
        return kv, a
    kv, a = call()
    accepted(L.si_paged_append_dev, kv, a)
    for change in (dict(k=None, v=None), dict(weights_stride=0), dict(weights_stride=1 << 44), {field: 4098}):
        kv, a = call()
        for name, value in change.items():
            setattr(a, name, value)
        refused(L.si_paged_append_dev, kv, a)
    kv = mai.paged_kv(*pools())
    n, k = torch.zeros(3, dtype=torch.int32), torch.zeros(3, 2, 16)
    made = mai.paged_append(kv, None, k, k, None, n, weights=torch.zeros(3, 2, 8), positions=torch.zeros(3, 2, 8, dtype=torch.int32))
    assert made.weights_stride == 8 and made.weights and made.positions
    for wrong in (dict(weights=torch.zeros(3, 2, 8).double()), dict(weights=torch.zeros(2, 2, 8)), dict(positions=torch.zeros(3, 2, 8)),
                  dict(weights=torch.zeros(3, 2, 8), positions=torch.zeros(3, 2, 9, dtype=torch.int32))):
        with pytest.raises(mai.SiError):
            mai.paged_append(kv, None, k, k, None, n, **wrong)
    ctx = object.__new__(mai.CudaContext)
    ctx.device, ctx.h = -1, None
    with pytest.raises(mai.SiError, match="described for a cache"):
        ctx.paged_append_dev(mai.paged_kv(*pools(seqs=5)), made)


# ---- buffers that overlap ------------------------------------------------------------
def elements(at, n0, s0, n1, s1, dims):
    """Elements of each row of a buffer, by enumeration."""
    return [set(range(at + i * s0 + j * s1, at + i * s0 + j * s1 + dims)) for i in range(n0) for j in range(n1)]


def taken(fn, *args):
    """Whether the arguments pass; a refusal must name an overlap."""
    assert fn(None, *[C.byref(a) for a in args], None) == INVALID
    text = L.si_global_last_error().decode()
    assert text == "null context" or "over" in text or "apart" in text, text
    return text == "null context"


BASE = 1 << 20  # never read: the calls have no context


@pytest.mark.parametrize("seed", range(4))
def test_outputs_over_parts_of_the_inputs_are_refused(seed):
    """Random places and strides of two buffers against their elements, enumerated: with equal strides the answer
    is exact, with others a call is taken only if the buffers share nothing."""
    rng = np.random.default_rng(seed)
    seen = set()
    for turn in range(1500):
        hd, n0, n1 = 8 * int(rng.integers(1, 3)), int(rng.integers(1, 5)), 2 * int(rng.integers(1, 4))
        strides = sorted((int(rng.choice([hd, hd + 1, hd + 8, 2 * hd, 3 * hd])), int(rng.choice([1, 2, 4, 6, 8]) * (2 * hd + rng.integers(0, 9)))))
        s1, s0 = strides if rng.random() < 0.7 else strides[::-1]
        t0, t1 = (s0, s1) if rng.random() < 0.7 else (s0 + 8 * int(rng.integers(0, 3)), s1 + int(rng.integers(0, 2)))
        at = int(rng.choice([0, 1, hd - 1, hd, 2 * hd, s1, s0, n1 * s1, n0 * s0, int(rng.integers(0, 300))]))
        swap = rng.random() < 0.5
        q, out = elements(0, n0, s0, n1, s1, hd), elements(at, n0, t0, n1, t1, hd)
        alone = sum(map(len, out)) == len(set().union(*out))
        meet = bool(set().union(*q) & set().union(*out))
        kv, a = attention_call()
        kv.sequences, kv.kv_heads, kv.head_dim, a.query_heads, a.work_bytes = n0, n1 // 2, hd, n1, 1 << 40
        a.q, a.out = (BASE, BASE + 4 * at)
        a.q_seq_stride, a.q_head_stride, a.out_seq_stride, a.out_head_stride = s0, s1, t0, t1
        if swap and alone and sum(map(len, q)) == len(set().union(*q)):
            a.q, a.out = a.out, a.q
            a.q_seq_stride, a.q_head_stride, a.out_seq_stride, a.out_head_stride = t0, t1, s0, s1
        ok = taken(L.si_paged_attention_dev, kv, a)
        same = (n0 == 1 or s0 == t0) and (n1 == 1 or s1 == t1)
        seen.add((ok, same, alone, meet))
        assert not ok or (alone and not meet), (turn, hd, n0, n1, s0, s1, t0, t1, at)
        nested = (s1 >= hd and (n0 == 1 or s0 >= (n1 - 1) * s1 + hd)) or (s0 >= hd and s1 >= (n0 - 1) * s0 + hd)
        if same and nested and not meet:
            assert ok, (turn, hd, n0, n1, s0, s1, t0, t1, at)
    assert {(True, True, True, False), (False, True, True, True), (True, False, True, False), (False, False, True, True)} <= seen


def test_queries_are_written_in_place_or_apart():
    """One projection's output [tokens][q, k, v heads]: in place, into free heads, over the keys, shifted by a token."""
    heads, hd, row = 4, 16, (4 + 2 + 2 + 4) * 16  # queries, keys, values, and as many free heads
    wide = torch.zeros(3, 12, 16)
    kv, _ = append_call()
    n = torch.zeros(3, dtype=torch.int32)
    q, k, v, free = wide.split([4, 2, 2, 4], 1)

    def call(out):
        return mai.paged_append(kv, q, k, v, out, n)
    for out in (q, free, torch.zeros(3, 4, 16)):
        accepted(L.si_paged_append_dev, kv, call(out))
    late = torch.as_strided(wide, (3, 4, 16), (row, hd, 1), hd)             # a head further: over the queries and keys
    over = torch.as_strided(wide, (3, 4, 16), (row, hd, 1), heads * hd)     # over the keys and values
    turned = torch.as_strided(wide, (3, 4, 16), (hd, 3 * hd, 1), 0)         # the same place in another order
    flat = torch.zeros(3, 1, 16).expand(3, 4, 16)                           # all heads in one row
    for out in (late, over, turned, flat):
        refused(L.si_paged_append_dev, kv, call(out))
    a = call(free)
    a.v = a.q_out  # values that the queries would go over
    refused(L.si_paged_append_dev, kv, a)
    one = mai.paged_append(kv, q[:1], None, None, q[:1], n[:1])
    one.q_out_token_stride = 5 * row  # one token has no token stride
    accepted(L.si_paged_append_dev, kv, one)
    none = call(late)
    none.tokens = 0
    accepted(L.si_paged_append_dev, kv, none)


@pytest.mark.parametrize("name", ["append", "evict"])
def test_pools_with_shared_rows_are_not_written(name):
    """Pools expanded over heads or pages can be attended and not written."""
    make, fn = CALLS[name]
    flat = torch.zeros(7, 1, 4, 16, dtype=torch.bfloat16)[:6]
    for k in (flat.expand(6, 2, 4, 16), flat[:1].expand(6, 1, 4, 16), torch.as_strided(flat, (6, 2, 4, 16), (64, 8, 16, 1))):
        v = torch.as_strided(torch.zeros(7, 1, 4, 16, dtype=torch.bfloat16), k.shape, k.stride())
        refused(fn, mai.paged_kv(k, v, torch.zeros(3, 2, dtype=torch.int32)), make()[1])
        assert "overlap" in L.si_global_last_error().decode()
    kv, a = make()
    kv.num_pages, kv.page_stride = 1, 0  # one page has no stride
    accepted(fn, kv, a)
    q = torch.zeros(3, 4, 16)
    shared = mai.paged_kv(flat.expand(6, 2, 4, 16), flat.expand(6, 2, 4, 16), torch.zeros(3, 2, dtype=torch.int32))
    work = torch.zeros(mai.paged_attention_workspace_bytes(shared, 4) // 8 + 2, dtype=torch.float64)
    accepted(L.si_paged_attention_dev, shared, mai.paged_attention(shared, q, torch.zeros_like(q), torch.zeros(3, dtype=torch.int32), work))
    if name == "append":
        kv, a = make()
        kv.v = kv.k
        refused(fn, kv, a)


@pytest.mark.parametrize("seed", range(3))
def test_queries_over_keys_of_any_strides(seed):
    """Random keys (heads and tokens that may share rows: inputs may be expanded) beside the rotated queries, against
    their elements: a call is taken only if they share nothing, and always if their strides agree and they do not."""
    rng = np.random.default_rng(seed)
    seen = set()
    for turn in range(1500):
        hd, tokens, qh, kvh = 8 * int(rng.integers(1, 3)), int(rng.integers(1, 5)), int(rng.integers(1, 5)), int(rng.integers(1, 4))
        s1 = int(rng.choice([hd, hd + 8, 2 * hd]))
        s0 = int(rng.choice([1, 2])) * (qh + kvh) * s1 + int(rng.integers(0, 2)) * 8
        if rng.random() < 0.3:  # tokens inside, heads outside
            s0, s1 = s1, s0 * tokens
        t0, t1 = (s0, s1) if rng.random() < 0.6 else (int(rng.choice([0, 1, 8, s0])), int(rng.choice([0, 1, 8, s1])))
        at = int(rng.choice([0, hd, qh * s1, kvh * s1, s0, tokens * s0, int(rng.integers(0, 400))])) * int(rng.choice([1, -1]))
        out, k = elements(0, tokens, s0, qh, s1, hd), elements(at, tokens, t0, kvh, t1, hd)
        meet = bool(set().union(*k) & set().union(*out))
        kv, a = append_call()
        kv.kv_heads, kv.head_dim, kv.page_stride, kv.head_stride, kv.token_stride = kvh, hd, 4 * kvh * hd, 4 * hd, hd
        a.tokens, a.query_heads, a.rotary_dim, a.sequence = tokens, qh, 0, BASE
        a.q, a.q_out, a.k, a.v = 2 * BASE, 64 * BASE, 64 * BASE + 4 * at, BASE
        a.q_token_stride, a.q_head_stride, a.q_out_token_stride, a.q_out_head_stride = qh * hd, hd, s0, s1
        a.k_token_stride, a.k_head_stride, a.v_token_stride, a.v_head_stride = t0, t1, kvh * hd, hd
        ok = taken(L.si_paged_append_dev, kv, a)
        same = (tokens == 1 or t0 == s0) and (qh == 1 or kvh == 1 or t1 == s1)
        seen.add((ok, same, meet))
        assert not (ok and meet), (turn, hd, tokens, qh, kvh, s0, s1, t0, t1, at)
        if same and not meet:
            assert ok, (turn, hd, tokens, qh, kvh, s0, s1, t0, t1, at)
    assert {(True, True, False), (False, True, True), (True, False, False), (False, False, True)} <= seen
