"""Paged-cache operators on the GPU against plain 64-bit implementations.

Tolerances. f32 outputs: the parity bound of this library's f32 operators, 1e-5
relative L2. 16-bit outputs: the rounding of each value, at most half a step
(eps / 2 relative), on top of that. Moves, counts and tokens are exact."""
import math

import numpy as np
import pytest
import torch

from conftest import load_package

pytestmark = pytest.mark.gpu
mai = load_package()

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
LEGACY = 1  # handle of torch's default stream


def half_step(t):
    return 0.0 if t == F32 else torch.finfo(t).eps / 2


def close(got, want, dtype, f32_bound=1e-5):
    got, want = got.double().cpu(), want.double().cpu()
    assert torch.isfinite(got).all()
    norm = want.norm()
    assert (got - want).norm() <= (f32_bound + half_step(dtype)) * norm, ((got - want).norm() / norm).item()


class Cache:
    """Pools in any order of pages, heads and tokens; what no slot in use needs holds NaN."""

    def __init__(self, lengths, kv_heads, page, hd, dtype=BF16, order="heads_first", spare=2, cols=None, seed=0, room=0):
        gen = torch.Generator().manual_seed(seed)
        need = [-(-max(n, 0) // page) + (room if n >= 0 else 0) for n in lengths]
        self.cols = cols or max(1, max(need))
        total = sum(need) + spare
        shape = (total, kv_heads, page, hd) if order == "heads_first" else (total, page, kv_heads, hd)
        self.k = torch.full(shape, math.nan, dtype=dtype, device="cuda")
        self.v = torch.full(shape, math.nan, dtype=dtype, device="cuda")
        if order != "heads_first":
            self.k, self.v = self.k.transpose(1, 2), self.v.transpose(1, 2)
        ids = torch.randperm(total, generator=gen)[:sum(need)].tolist()
        self.pages = torch.full((len(lengths), self.cols), -7, dtype=torch.int32)
        for b, n in enumerate(need):
            for j in range(n):
                self.pages[b, j] = ids.pop()
        self.lengths = list(lengths)
        self.page = page
        for b, n in enumerate(lengths):
            if n > 0:
                pg, at = self.cells(b, n)
                self.k[pg, :, at] = torch.randn(n, kv_heads, hd, generator=gen).to(dtype).cuda()
                self.v[pg, :, at] = torch.randn(n, kv_heads, hd, generator=gen).to(dtype).cuda()
        self.pages_dev = self.pages.cuda()
        self.len_dev = torch.tensor(self.lengths, dtype=torch.int32, device="cuda")
        self.desc = mai.paged_kv(self.k, self.v, self.pages_dev)

    def cells(self, b, n):
        t = torch.arange(n)
        return self.pages[b].long()[t // self.page].cuda(), (t % self.page).cuda()

    def rows(self, b, n, pool):
        pg, at = self.cells(b, n)
        return pool[pg, :, at].double()  # [n][kv_heads][hd]


def reference(cache, q, scale=None, lengths=None):
    """Attention, log-sum-exp and the group's probabilities in 64 bits."""
    b_n, qh, hd = q.shape
    kvh = cache.k.shape[1]
    g = qh // kvh
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    lse = torch.full((b_n, qh), -math.inf, dtype=torch.float64, device="cuda")
    weights = []
    for b, n in enumerate(lengths or cache.lengths):
        if n <= 0:
            weights.append(None)
            continue
        k, v = cache.rows(b, n, cache.k), cache.rows(b, n, cache.v)
        s = torch.einsum("hgd,nhd->hgn", q[b].double().view(kvh, g, hd), k) * (scale or hd ** -0.5)
        p = torch.softmax(s, -1)
        out[b] = torch.einsum("hgn,nhd->hgd", p, v).reshape(qh, hd)
        lse[b] = torch.logsumexp(s, -1).view(-1)
        weights.append(p.sum(1))
    return out, lse, weights


def work_for(cache, qh, weights=False):
    return torch.empty(mai.paged_attention_workspace_bytes(cache.desc, qh, weights), dtype=torch.uint8, device="cuda")


def attend(ctx, cache, q, out=None, stream=LEGACY, **kw):
    out = torch.full_like(q, math.nan) if out is None else out
    work = work_for(cache, q.shape[1], kw.get("weights_out") is not None).fill_(255)
    args = mai.paged_attention(cache.desc, q, out, cache.len_dev, work, **kw)
    ctx.paged_attention_dev(cache.desc, args, stream)
    return out


ATTENTION = [
    # lengths, kv_heads, group, head_dim, page
    ([1], 1, 1, 64, 1),
    ([0], 1, 1, 64, 16),
    ([15, 16, 17, 0, 31, 32, 33], 2, 1, 64, 16),
    ([1, 2, 3, 0, 5], 4, 6, 256, 16),
    ([517], 4, 6, 256, 16),
    ([100, 0, 0, 7], 1, 8, 128, 5),
    ([129, 63, 1], 2, 3, 80, 24),
    ([300, 299], 5, 12, 96, 7),
    ([64], 1, 17, 192, 64),
    ([1000] * 3, 2, 2, 8, 32),
    ([777, 12], 3, 5, 40, 1),
    ([4096, 1, 2048], 2, 4, 128, 256),
    ([20000], 1, 7, 256, 48),
    (list(range(0, 400, 3)), 2, 4, 128, 16),
    ([40] * 700, 1, 1, 64, 16),
]


@pytest.mark.parametrize("io, cache_type", [(F32, BF16), (BF16, BF16), (F32, F16), (F16, F16), (BF16, F16), (F16, BF16)])
@pytest.mark.parametrize("case", range(len(ATTENTION)))
def test_attention(ctx, case, io, cache_type):
    lengths, kvh, g, hd, page = ATTENTION[case]
    cache = Cache(lengths, kvh, page, hd, cache_type, order="heads_first" if case % 2 else "tokens_first", seed=case)
    q = torch.randn(len(lengths), kvh * g, hd, device="cuda").to(io)
    lse = torch.full((len(lengths), kvh * g), math.nan, device="cuda")
    out = attend(ctx, cache, q, lse=lse)
    want, want_lse, _ = reference(cache, q)
    ctx.synchronize()
    close(out, want, io)
    empty = want_lse == -math.inf
    assert (lse[empty] == -math.inf).all() and (out[empty] == 0).all()
    if not empty.all():
        # log-sum-exp: absolute, as scores of size |q||k| round; 2^-16 covers 256 products of size 16 at 2^-24
        assert (lse.double() - want_lse)[~empty].abs().max() <= 2 ** -16


@pytest.mark.parametrize("scale", [0.0, 0.02, 1.7])
@pytest.mark.parametrize("size", [1e-4, 1.0, 300.0])
def test_attention_scales_and_ranges(ctx, scale, size):
    """Small and large queries (one-hot softmax at 300), and f16 values that bf16 terms could not hold."""
    for dtype in (BF16, F16):
        cache = Cache([333, 48], 2, 16, 128, dtype, seed=3)
        q = torch.randn(2, 8, 128, device="cuda") * size
        out = attend(ctx, cache, q, scale=scale)
        # a score of size S carries S * 2^-24 of absolute rounding into the softmax: S is up to 300 * 11 * 3 * 1.7
        worst = (scale or 128 ** -0.5) * size * 11.3 * 5
        close(out, reference(cache, q, scale or None)[0], F32, 1e-5 + worst * 2 ** -22)


def test_attention_outliers(ctx):
    """A few very large queries and keys beside small ones keep the small ones' precision."""
    for dtype in (BF16, F16):
        cache = Cache([200], 1, 8, 64, dtype, seed=5)
        q = torch.randn(1, 4, 64, device="cuda")
        q[0, 0, 3] = 1e4
        q[0, 1] = 0
        q[0, 2] *= 1e-30
        pg, at = cache.cells(0, 200)
        k = cache.k[pg, :, at]
        k[:, :, 3] *= 1e-3
        cache.k[pg, :, at] = k
        close(attend(ctx, cache, q), reference(cache, q)[0], F32)


@pytest.mark.parametrize("io", [F32, BF16])
def test_attention_strides_and_alignment(ctx, io):
    """Queries and outputs inside wider rows, off 16-byte boundaries; what lies between is left as it was."""
    cache = Cache([90, 0, 33], 2, 16, 72, BF16, seed=6)
    wide = torch.randn(3, 7, 75, device="cuda").to(io)
    room = torch.full((3, 9, 81), 5.0, device="cuda").to(io)
    q, out = wide[:, 1:5, 3:], room[:, 2:6, 1:73]
    attend(ctx, cache, q, out)
    close(out, reference(cache, q)[0], io)
    room[:, 2:6, 1:73] = 5
    assert (room == 5).all()
    turned = torch.randn(4, 3, 72, device="cuda").to(io).transpose(0, 1)
    close(attend(ctx, cache, turned, torch.empty_like(turned)), reference(cache, turned)[0], io)


def test_attention_rows_that_share_pages(ctx):
    """A window of candidates of one sequence: rows with the same pages and growing lengths."""
    cache = Cache([100], 2, 16, 128, BF16, seed=7)
    pages = cache.pages_dev.expand(5, -1).contiguous()
    kv = mai.paged_kv(cache.k, cache.v, pages)
    lengths = [96, 97, 98, 99, 100]
    q = torch.randn(5, 8, 128, device="cuda")
    out, n = torch.empty_like(q), torch.tensor(lengths, dtype=torch.int32, device="cuda")
    work = torch.empty(mai.paged_attention_workspace_bytes(kv, 8), dtype=torch.uint8, device="cuda")
    ctx.paged_attention_dev(kv, mai.paged_attention(kv, q, out, n, work), LEGACY)
    for i, m in enumerate(lengths):
        cache.lengths = [m]
        close(out[i:i + 1], reference(cache, q[i:i + 1])[0], F32)


@pytest.mark.parametrize("g", [1, 4, 5, 11])
@pytest.mark.parametrize("in_place", [True, False, None])
def test_attention_weights(ctx, g, in_place):
    """in_place None: no weights come in."""
    lengths = [500, 0, 1, 17, 2000]
    cache = Cache(lengths, 3, 16, 64, F16, seed=g, cols=150)
    q = torch.randn(5, 3 * g, 64, device="cuda")
    before = torch.rand(5, 3, 2048, device="cuda")
    w_out = before.clone() if in_place else torch.full_like(before, 7.0)
    w_in = w_out if in_place else None if in_place is None else before
    out = attend(ctx, cache, q, weights_in=w_in, weights_out=w_out)
    want, _, weights = reference(cache, q)
    close(out, want, F32)
    for b, n in enumerate(lengths):
        rest = before if in_place else torch.full_like(before, 7.0)
        assert torch.equal(w_out[b, :, n:], rest[b, :, n:])
        if n:
            start = before[b, :, :n].double() if in_place is not None else 0.0
            close(w_out[b, :, :n], weights[b] + start, F32)
    # the same call again gives the same bits
    if in_place is False:
        again = torch.full_like(before, 7.0)
        assert torch.equal(attend(ctx, cache, q, weights_in=before, weights_out=again), out) and torch.equal(again, w_out)


def test_attention_bad_pages_and_lengths(ctx):
    """A page outside the pool is left out and reported, other rows stay right; so is a length beyond the table."""
    cache = Cache([64, 64, 40], 2, 16, 64, BF16, seed=9)
    q = torch.randn(3, 4, 64, device="cuda")
    good = attend(ctx, cache, q)
    ctx.synchronize()
    for bad in (-1, cache.k.shape[0], 2 ** 31 - 1):
        cache.pages_dev[1, 2] = bad
        out = attend(ctx, cache, q)
        torch.cuda.synchronize()
        with pytest.raises(mai.SiError) as e:
            ctx.synchronize()
        assert e.value.status == mai.SI_E_INVALID
        assert torch.equal(out[[0, 2]], good[[0, 2]]) and torch.isfinite(out).all()
        left = torch.cat([torch.arange(32), torch.arange(48, 64)]).cuda()
        k, v = (cache.rows(1, 64, p)[left] for p in (cache.k, cache.v))
        p = torch.softmax(torch.einsum("hgd,nhd->hgn", q[1].double().view(2, 2, 64), k) / 8, -1)
        close(out[1], torch.einsum("hgn,nhd->hgd", p, v).reshape(4, 64), F32)
    cache.pages_dev.copy_(cache.pages)
    for bad in (-5, 65, 2 ** 31 - 1):
        cache.len_dev[1] = bad
        out = attend(ctx, cache, q)
        torch.cuda.synchronize()
        with pytest.raises(mai.SiError):
            ctx.synchronize()
        # another length shares the units out differently, so sums of the same terms group differently: 64 terms
        # of 2^-24 each stay within 2^-18 of the largest value, inside the f32 bound
        close(out[[0, 2]], good[[0, 2]], F32)
        assert torch.equal(out[1], torch.zeros_like(out[1]) if bad < 0 else good[1])
    ctx.synchronize()  # the report is given once


def test_attention_far_offsets(ctx):
    """Pools whose last page lies past 2^32 elements."""
    stride = (1 << 31) + 1024
    flat = [torch.empty(2 * stride + 4096, dtype=BF16, device="cuda") for _ in range(2)]
    k, v = (f.as_strided((3, 1, 16, 64), (stride, 1024, 64, 1)) for f in flat)
    k[...] = torch.randn(3, 1, 16, 64, device="cuda").to(BF16)
    v[...] = torch.randn(3, 1, 16, 64, device="cuda").to(BF16)
    pages = torch.tensor([[2, 0, 1]], dtype=torch.int32, device="cuda")
    kv = mai.paged_kv(k, v, pages)
    q = torch.randn(1, 2, 64, device="cuda")
    out, n = torch.empty_like(q), torch.tensor([45], dtype=torch.int32, device="cuda")
    work = torch.empty(mai.paged_attention_workspace_bytes(kv, 2), dtype=torch.uint8, device="cuda")
    ctx.paged_attention_dev(kv, mai.paged_attention(kv, q, out, n, work), LEGACY)
    keys, values = (x[[2, 0, 1], 0].reshape(48, 64)[:45].double() for x in (k, v))
    close(out[0], torch.softmax(q[0].double() @ keys.T / 8, -1) @ values, F32)
    # the append writes there too
    new = torch.randn(1, 1, 64, device="cuda").to(BF16)
    slot = torch.tensor([5], dtype=torch.int32, device="cuda")
    ctx.paged_append_dev(kv, mai.paged_append(kv, None, new, new, None, slot), LEGACY)
    assert torch.equal(k[2, 0, 5], new[0, 0]) and torch.equal(v[2, 0, 5], new[0, 0])


def test_attention_captured_follows_lengths(ctx):
    """A captured call replays with other lengths, pages and queries."""
    cache = Cache([400, 3, 90], 2, 16, 128, BF16, seed=11)
    q, s = torch.randn(3, 8, 128, device="cuda"), torch.cuda.Stream()
    out, work = torch.empty_like(q), work_for(cache, 8)
    args = mai.paged_attention(cache.desc, q, out, cache.len_dev, work)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        ctx.paged_attention_dev(cache.desc, args, s.cuda_stream)
    for lengths in ([400, 3, 90], [1, 0, 17], [0, 0, 0], [399, 2, 80]):
        cache.len_dev.copy_(torch.tensor(lengths))
        q.normal_()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        close(out, reference(cache, q, lengths=lengths)[0], F32)


def test_attention_on_two_streams(ctx):
    caches = [Cache([5000, 70], 4, 16, 128, BF16, seed=i) for i in (1, 2)]
    qs = [torch.randn(2, 16, 128, device="cuda") for _ in caches]
    outs, streams = [torch.empty_like(q) for q in qs], [torch.cuda.Stream() for _ in caches]
    args = [mai.paged_attention(c.desc, q, o, c.len_dev, work_for(c, 16)) for c, q, o in zip(caches, qs, outs)]
    torch.cuda.synchronize()
    for _ in range(20):
        for c, a, s in zip(caches, args, streams):
            ctx.paged_attention_dev(c.desc, a, s.cuda_stream)
    torch.cuda.synchronize()
    for c, q, o in zip(caches, qs, outs):
        close(o, reference(c, q)[0], F32)


# ---- rotary positions and append ------------------------------------------------
def rotated(x, angle, layout, scale):
    half = angle.shape[1]
    y = x.double().clone()
    c, s = (f(angle)[:, None] * scale for f in (torch.cos, torch.sin))
    if layout == "half":
        a, b = x[..., :half].double(), x[..., half:2 * half].double()
        y[..., :half], y[..., half:2 * half] = a * c - b * s, a * s + b * c
    else:
        a, b = x[..., :2 * half:2].double(), x[..., 1:2 * half:2].double()
        y[..., :2 * half:2], y[..., 1:2 * half:2] = a * c - b * s, a * s + b * c
    return y


APPEND = [
    # tokens, sequences, query heads, kv heads, head_dim, rotary, page
    (1, 1, 4, 4, 64, 64, 1),
    (5, 5, 24, 4, 256, 64, 16),
    (77, 3, 6, 2, 128, 128, 24),
    (40, 2, 3, 1, 80, 20, 7),
    (33, 4, 2, 2, 72, 2, 16),
    (6, 6, 8, 8, 96, 0, 8),
    (2000, 7, 4, 2, 64, 48, 32),
    (5000, 2, 5, 1, 8, 8, 5),
]


@pytest.mark.parametrize("io, cache_type", [(F32, BF16), (BF16, BF16), (F16, F16), (F32, F16), (BF16, F16)])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("case", range(len(APPEND)))
def test_append(ctx, case, layout, io, cache_type):
    tokens, seqs, qh, kvh, hd, rotary, page = APPEND[case]
    gen = torch.Generator().manual_seed(case)
    per = -(-tokens // seqs)
    cache = Cache([per + 3] * seqs, kvh, page, hd, cache_type, seed=case)
    order = torch.randperm(tokens, generator=gen)
    sequence, slot = (order // per).to(torch.int32), (order % per + 2).to(torch.int32)
    position = torch.randint(-1000, 1 << 20, (tokens,), generator=gen, dtype=torch.int32)
    position[0] = 2 ** 31 - 1
    pad = torch.rand(tokens, generator=gen) < 0.1
    slot[pad] = -1
    qkv = torch.randn(tokens, qh + 2 * kvh, hd, generator=gen).to(io).cuda()
    q, k, v = qkv.split([qh, kvh, kvh], 1)
    kind = ["none", "linear", "ntk", "yarn", "banded"][case % 5]
    table, scale = mai.rope_table(1e6, rotary, kind, factor=4.0, original=4096)
    rope = torch.from_numpy(table.view(np.int64)).cuda()
    q_out = torch.full_like(q.contiguous(), 9.0)
    want_k, want_v = cache.k.clone(), cache.v.clone()
    args = mai.paged_append(cache.desc, q, k, v, q_out, slot.cuda(), sequence=sequence.cuda(), position=position.cuda(),
                            rope=rope, rotary_dim=rotary, layout=layout, rope_scale=scale)
    ctx.paged_append_dev(cache.desc, args, LEGACY)
    torch.cuda.synchronize()
    ctx.synchronize()
    # exact angles: integer turns modulo 2^64, from the table itself
    turns = [[(int(p) * int(t)) % 2 ** 64 / 2.0 ** 64 * 2 * math.pi for t in table] for p in position]
    angle = torch.tensor(turns, dtype=torch.float64).view(tokens, rotary // 2).cuda()
    live = ~pad.cuda()

    def check(got, x, dtype):
        """2^-24 for each of three roundings, 2^-22 for the sines and the angle, of |x| + |y| <= 1.5 max"""
        want = rotated(x, angle, layout, scale)
        room = x.double().abs().amax(-1, keepdim=True) * 2 * scale * 2 ** -21 + want.abs() * half_step(dtype)
        if dtype == F16:
            room = room + 2 ** -25  # half a step of the subnormal range
        assert ((got.double() - want).abs() <= room)[live].all()

    check(q_out, q, io)
    assert (q_out[~live] == 9).all()
    pg = cache.pages_dev.long()[sequence.long().cuda(), (slot.long().clamp(min=0) // page).cuda()]
    at = (slot.long().clamp(min=0) % page).cuda()
    check(cache.k[pg, :, at], k, cache_type)
    new_v = v.to(F32).to(cache_type)
    assert torch.equal(cache.v[pg, :, at][live], new_v[live])
    # nothing else changed
    cache.k[pg[live], :, at[live]] = 0
    cache.v[pg[live], :, at[live]] = 0
    want_k[pg[live], :, at[live]] = 0
    want_v[pg[live], :, at[live]] = 0
    assert torch.equal(cache.k.view(torch.int16), want_k.view(torch.int16))
    assert torch.equal(cache.v.view(torch.int16), want_v.view(torch.int16))


def test_append_in_place_defaults_and_parts(ctx):
    """Queries in place, token t of sequence t, position = slot; queries only; keys only; off 16-byte boundaries."""
    cache = Cache([20, 20, 20], 2, 8, 64, BF16, seed=1)
    table, _ = mai.rope_table(1e4, 64)
    rope = torch.from_numpy(table.view(np.int64)).cuda()
    slot = torch.tensor([19, -1, 4], dtype=torch.int32, device="cuda")
    angle = torch.tensor([[int(p) * int(t) / 2.0 ** 64 * 2 * math.pi for t in table] for p in slot], dtype=torch.float64).cuda()
    big = torch.randn(3, 5, 67, device="cuda")
    q = big[:, :, 2:66]
    before = q.clone()
    ctx.paged_append_dev(cache.desc, mai.paged_append(cache.desc, q, None, None, q, slot, rope=rope, rotary_dim=64), LEGACY)
    want = rotated(before, angle, "interleaved", 1.0)
    want[1] = before[1]
    close(q, want, F32)
    kept = cache.k.clone()
    new = torch.randn(3, 2, 64, device="cuda").to(BF16)
    ctx.paged_append_dev(cache.desc, mai.paged_append(cache.desc, None, new, new, None, slot, rope=rope, rotary_dim=64, layout="half"),
                         LEGACY)
    for b, t in ((0, 19), (2, 4)):
        got = cache.k[cache.pages[b, t // 8].item(), :, t % 8]
        close(got, rotated(new[b:b + 1], angle[b:b + 1], "half", 1.0)[0], BF16)
        assert torch.equal(cache.v[cache.pages[b, t // 8].item(), :, t % 8], new[b])
        cache.k[cache.pages[b, t // 8].item(), :, t % 8] = kept[cache.pages[b, t // 8].item(), :, t % 8]
    assert torch.equal(cache.k.view(torch.int16), kept.view(torch.int16))
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    empty = torch.zeros(0, 2, 64, device="cuda")
    ctx.paged_append_dev(cache.desc, mai.paged_append(cache.desc, None, empty, empty, None, none), LEGACY)
    ctx.synchronize()


def test_append_bad_places_are_left_out(ctx):
    cache = Cache([16, 16], 1, 8, 64, BF16, seed=2)
    cache.pages_dev[1, 1] = cache.k.shape[0]
    k0, v0 = cache.k.clone(), cache.v.clone()
    new = torch.randn(4, 1, 64, device="cuda").to(BF16)
    slot = torch.tensor([16, 9, 3, 0], dtype=torch.int32, device="cuda")      # beyond the table, a bad page, good,
    sequence = torch.tensor([0, 1, 0, 2], dtype=torch.int32, device="cuda")   # no such sequence
    ctx.paged_append_dev(cache.desc, mai.paged_append(cache.desc, None, new, new, None, slot, sequence=sequence), LEGACY)
    torch.cuda.synchronize()
    with pytest.raises(mai.SiError) as e:
        ctx.synchronize()
    assert e.value.status == mai.SI_E_INVALID
    pg = cache.pages[0, 0].item()
    assert torch.equal(cache.k[pg, :, 3], new[2])
    cache.k[pg, :, 3], cache.v[pg, :, 3] = k0[pg, :, 3], v0[pg, :, 3]
    assert torch.equal(cache.k.view(torch.int16), k0.view(torch.int16))
    assert torch.equal(cache.v.view(torch.int16), v0.view(torch.int16))


# ---- eviction -----------------------------------------------------------------------
def evicted(w, pos, n, budget, sink, recent, nxt):
    """(holes, kept slots behind the budget) of one row: the definition, by sorting."""
    m = min(n, budget)
    key = []
    for t in range(n):
        held = pos[t] < sink or pos[t] >= nxt - recent
        x = float(w[t])
        key.append((1 if held else 0, 0.0 if held else (-math.inf if x != x else x), 0 if x != x or held else 1, t))
    gone = {k[-1] for k in sorted(key)[:n - m]}
    return [t for t in range(m) if t in gone], [t for t in range(m, n) if t not in gone]


EVICT = [
    # lengths, kv_heads, head_dim, page, budget, sink, recent
    ([1], 1, 64, 1, 1, 0, 0),
    ([2, 0, 1], 2, 8, 4, 1, 0, 1),
    ([100, 20, 0, 21, 300], 2, 64, 16, 20, 2, 5),
    ([500], 3, 256, 24, 499, 4, 100),
    ([1023, 1024, 1025], 2, 128, 64, 512, 0, 512),
    ([5000, 40], 1, 72, 7, 33, 3, 30),
    ([9000, 17000], 2, 64, 32, 4000, 4, 64),
    ([40000], 1, 8, 256, 20001, 1, 1),
    ([70001, 3], 1, 8, 128, 100, 50, 50),
    ([200], 2, 64, 16, 1000, 0, 0),
]


@pytest.mark.parametrize("kind", ["spread", "ties", "equal", "strange"])
@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("case", range(len(EVICT)))
def test_evict(ctx, case, in_place, kind):
    lengths, kvh, hd, page, budget, sink, recent = EVICT[case]
    rng = np.random.default_rng(case)
    cache = Cache(lengths, kvh, page, hd, F16 if case % 2 else BF16, order="tokens_first" if case % 3 else "heads_first", seed=case)
    width = max(lengths) + 5
    shape = (len(lengths), kvh, width)
    w = np.exp(3 * rng.normal(size=shape)).astype(np.float32)
    if kind == "ties":
        w = np.floor(w * 4) / 4
    elif kind == "equal":
        w[:] = 0.5
    elif kind == "strange":
        odd = rng.random(shape)
        w[odd < 0.1] = np.nan
        w[(odd >= 0.1) & (odd < 0.2)] = np.inf
        w[(odd >= 0.2) & (odd < 0.3)] = -np.inf
        w[(odd >= 0.3) & (odd < 0.5)] *= -1
        w[(odd >= 0.5) & (odd < 0.6)] = 0.0
        w[(odd >= 0.6) & (odd < 0.7)] = -0.0
    w = w.astype(np.float32)
    pos = np.stack([np.stack([rng.permutation(width * 2)[:width] for _ in range(kvh)]) for _ in lengths]).astype(np.int32)
    nxt = np.array([2 * width] * len(lengths), np.int32)
    w_in, p_in = torch.from_numpy(w).cuda(), torch.from_numpy(pos).cuda()
    w_out = w_in.clone() if in_place else torch.full_like(w_in, 3.5)
    p_out = p_in.clone() if in_place else torch.full_like(p_in, -9)
    n_out = cache.len_dev.clone() if in_place else torch.full_like(cache.len_dev, -1)
    work = torch.empty(mai.paged_evict_workspace_bytes(cache.desc), dtype=torch.uint8, device="cuda").fill_(255)
    k0, v0 = cache.k.clone(), cache.v.clone()
    args = mai.paged_evict(cache.desc, n_out if in_place else cache.len_dev, n_out, w_out if in_place else w_in, w_out,
                           budget, work, sink=sink, recent=recent, positions_in=p_out if in_place else p_in,
                           positions_out=p_out, next_position=torch.from_numpy(nxt).cuda())
    ctx.paged_evict_dev(cache.desc, args, LEGACY)
    torch.cuda.synchronize()
    ctx.synchronize()
    assert n_out.tolist() == [min(n, budget) for n in lengths]
    want_w = w.copy() if in_place else np.full_like(w, 3.5)
    want_p = pos.copy() if in_place else np.full_like(pos, -9)
    for b, n in enumerate(lengths):
        m = min(n, budget)
        for h in range(kvh):
            holes, movers = evicted(w[b, h], pos[b, h], n, budget, sink, recent, nxt[b])
            keep = [t for t in range(m) if t not in set(holes)]
            want_w[b, h, keep], want_p[b, h, keep] = w[b, h, keep], pos[b, h, keep]
            want_w[b, h, holes], want_p[b, h, holes] = w[b, h, movers], pos[b, h, movers]
            if holes:
                pg, at = cache.cells(b, n)
                to, of = torch.tensor(holes).cuda(), torch.tensor(movers).cuda()
                for pool, start in ((cache.k, k0), (cache.v, v0)):
                    assert torch.equal(pool[pg[to], h, at[to]], start[pg[of], h, at[of]])
                    pool[pg[to], h, at[to]] = start[pg[to], h, at[to]]
    if not in_place:  # holes of the output are written, slots behind the new length are not
        for b, n in enumerate(lengths):
            assert (w_out[b, :, min(n, budget):] == 3.5).all()
    np.testing.assert_array_equal(w_out.cpu().numpy().view(np.uint32), want_w.view(np.uint32))
    np.testing.assert_array_equal(p_out.cpu().numpy(), want_p)
    assert torch.equal(cache.k.view(torch.int16), k0.view(torch.int16))
    assert torch.equal(cache.v.view(torch.int16), v0.view(torch.int16))


def test_evict_without_positions(ctx):
    """Slots are positions: the first `sink` and the last `recent` slots stay, and the positions come out."""
    cache = Cache([50, 9], 1, 8, 64, BF16, seed=3)
    w = torch.rand(2, 1, 64, device="cuda")
    w[0, 0, 10] = w[0, 0, 3] = 0.0
    p_out = torch.full((2, 1, 64), -1, dtype=torch.int32, device="cuda")
    n_out, w_out = torch.empty_like(cache.len_dev), w.clone()
    work = torch.empty(mai.paged_evict_workspace_bytes(cache.desc), dtype=torch.uint8, device="cuda")
    args = mai.paged_evict(cache.desc, cache.len_dev, n_out, w_out, w_out, 48, work, sink=2, recent=5, positions_out=p_out)
    ctx.paged_evict_dev(cache.desc, args, LEGACY)
    assert n_out.tolist() == [48, 9]
    want = list(range(48))
    want[3], want[10] = 48, 49
    assert p_out[0, 0, :48].tolist() == want and p_out[1, 0, :9].tolist() == list(range(9))
    assert (p_out[0, 0, 48:] == -1).all() and (p_out[1, 0, 9:] == -1).all()


def test_evict_bad_pages_lengths_and_too_many_protected(ctx):
    cache = Cache([64, 64], 1, 16, 64, BF16, seed=4)
    w = torch.rand(2, 1, 64, device="cuda")
    w[:, :, :8] = 0
    work = torch.empty(mai.paged_evict_workspace_bytes(cache.desc), dtype=torch.uint8, device="cuda")
    k0 = cache.k.clone()
    cache.pages_dev[0, 3] = -3  # where the kept slots lie
    n_out = torch.empty_like(cache.len_dev)
    ctx.paged_evict_dev(cache.desc, mai.paged_evict(cache.desc, cache.len_dev, n_out, w, w.clone(), 56, work, recent=8), LEGACY)
    torch.cuda.synchronize()
    with pytest.raises(mai.SiError) as e:
        ctx.synchronize()
    assert e.value.status == mai.SI_E_INVALID
    pg = cache.pages[1].long().cuda()
    assert torch.equal(cache.k[pg[0], 0, :8], k0[pg[3], 0, 8:])  # the other sequence moved
    assert torch.equal(cache.k[cache.pages[0, 0].item()].view(torch.int16), k0[cache.pages[0, 0].item()].view(torch.int16))
    cache.pages_dev.copy_(cache.pages)
    for bad in (65, -1):
        cache.len_dev[0] = bad
        ctx.paged_evict_dev(cache.desc, mai.paged_evict(cache.desc, cache.len_dev, n_out, w, w.clone(), 56, work, recent=8), LEGACY)
        torch.cuda.synchronize()
        with pytest.raises(mai.SiError):
            ctx.synchronize()
        assert n_out.tolist() == [56 if bad > 0 else 0, 56]
    # all positions are protected: the lowest slots leave
    cache = Cache([20], 1, 16, 64, BF16, seed=4)
    p = torch.zeros(1, 1, 32, dtype=torch.int32, device="cuda")
    p_out, n_out = torch.empty_like(p), torch.empty_like(cache.len_dev)
    p[0, 0, 16:20] = torch.arange(-4, 0)
    w = torch.rand(1, 1, 32, device="cuda")
    ctx.paged_evict_dev(cache.desc, mai.paged_evict(cache.desc, cache.len_dev, n_out, w, w, 16, work, sink=16, positions_in=p,
                                                    positions_out=p_out), LEGACY)
    assert p_out[0, 0, :16].tolist() == [-4, -3, -2, -1] + [0] * 12


# ---- verification ------------------------------------------------------------------------
def verified(p, q, tokens, u, last, n):
    """The definition, in exact rational arithmetic up to the 64-bit sums."""
    good = lambda x: x if 0 < x < math.inf else 0.0  # noqa: E731
    i = 0
    while i < n:
        x = int(tokens[i])
        if not 0 <= x < p.shape[1]:
            break
        if not float(u[i]) * (good(float(q[i, x])) if q is not None else 1.0) < good(float(p[i, x])):
            break
        i += 1
    clean = lambda a: np.where((a > 0) & np.isfinite(a), a, 0).astype(np.float64)  # noqa: E731
    row = clean(p[i])
    rest = row.copy()
    if i < n:
        if q is not None:
            rest = np.maximum(row - clean(q[i]), 0)
        elif 0 <= int(tokens[i]) < len(row):
            rest[int(tokens[i])] = 0
    if not rest.sum() > 0:
        rest = row
    if not rest.sum() > 0:
        return i, -1
    cdf = np.cumsum(rest)
    hit = np.flatnonzero((cdf > float(last) * cdf[-1]) & (rest > 0))
    return i, int(hit[0] if len(hit) else np.flatnonzero(rest)[-1])


def run_verify(ctx, p, q, tokens, u, last, counts=None, stream=LEGACY):
    n = p.shape[0]
    accepted, following = (torch.full((n,), -5, dtype=torch.int32, device="cuda") for _ in range(2))
    work = torch.empty(mai.verify_drafts_workspace_bytes(n, p.shape[2]), dtype=torch.uint8, device="cuda").fill_(255)
    args = mai.verify_drafts(p, tokens, u, last, accepted, following, work, draft_probs=q, counts=counts)
    ctx.verify_drafts_dev(args, stream)
    return accepted, following


@pytest.mark.parametrize("probs", [True, False])
@pytest.mark.parametrize("n, k, vocab", [(1, 0, 1), (1, 1, 1), (5, 3, 2), (7, 8, 257), (3, 32, 4096), (4, 4, 4097), (9, 2, 32003),
                                         (2, 7, 248320), (300, 1, 100)])
def test_verify(ctx, n, k, vocab, probs):
    gen = torch.Generator(device="cuda").manual_seed(n * k + vocab)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    logits = 2 * rnd(n, k + 1, vocab)
    p = torch.softmax(logits, -1)
    q = torch.softmax(logits[:, :k] + 0.5 * rnd(n, k, vocab), -1) if probs else None
    tokens = torch.randint(0, vocab, (n, k), device="cuda", generator=gen, dtype=torch.int32)
    if k:
        tokens = torch.where(torch.rand(n, k, device="cuda", generator=gen) < 0.8, p[:, :k].argmax(-1).to(torch.int32), tokens)
    u, last = torch.rand(n, k, device="cuda", generator=gen), torch.rand(n, device="cuda", generator=gen)
    last[0] = 0.0
    if n > 2:
        last[1] = 1 - 2 ** -24
    counts = torch.randint(0, k + 1, (n,), device="cuda", generator=gen, dtype=torch.int32)
    for c in (None, counts):
        accepted, following = run_verify(ctx, p, q, tokens, u, last, c)
        ctx.synchronize()
        for b in range(n):
            want = verified(p[b].cpu().numpy(), q[b].cpu().numpy() if probs else None, tokens[b].tolist(), u[b].tolist(),
                            last[b].item(), k if c is None else int(c[b]))
            assert (accepted[b].item(), following[b].item()) == want, b


def test_verify_edges(ctx):
    """Equal rows, empty rows, values on the border, entries that are no probabilities, drafts outside the vocabulary."""
    p = torch.zeros(9, 2, 6, device="cuda")
    q = torch.zeros(9, 1, 6, device="cuda")
    tokens, u, last = torch.zeros(9, 1, dtype=torch.int32, device="cuda"), torch.zeros(9, 1, device="cuda"), torch.full((9,), 0.5, device="cuda")
    p[0, 0], q[0, 0], tokens[0] = torch.tensor([0, .5, .5, 0, 0, 0]), torch.tensor([0, .5, .5, 0, 0, 0]), 0  # 0 < 0: rejected; p - q is 0: p itself
    p[1, 0, 2], q[1, 0, 2], tokens[1], u[1] = 0.25, 0.5, 2, 0.5        # u q == p: rejected
    p[2, 0, 2], q[2, 0, 2], tokens[2], u[2] = 0.25, 0.5, 2, 0.49999997  # below: accepted
    p[2, 1, 5] = 1.0
    p[3, 0] = math.nan                                                  # nothing to draw: -1
    p[4, 0], tokens[4] = torch.tensor([math.nan, -1, math.inf, 0, .5, .5]), 0
    p[5, 0], tokens[5], u[5] = torch.tensor([.2, .2, .2, .2, .2, 0]), 4, 0.9
    q[5, 0] = torch.tensor([.1, .2, .3, .1, .3, 0])                     # left: .1 at 0 and 3
    p[6, 0, 1], p[6, 0, 3], tokens[6] = .5, .5, -1                      # outside: rejected, reported
    p[7, 0, 1], p[7, 0, 3], tokens[7] = .5, .5, 6
    p[8, 0, 0], q[8, 0, 0], p[8, 1, 3] = 1.0, 1.0, 1e-45                # accepted; a subnormal row
    accepted, following = run_verify(ctx, p, q, tokens, u, last)
    torch.cuda.synchronize()
    with pytest.raises(mai.SiError) as e:
        ctx.synchronize()
    assert e.value.status == mai.SI_E_INVALID
    assert accepted.tolist() == [0, 0, 1, 0, 0, 0, 0, 0, 1]
    # half of equal halves: the lowest whose sum passes 0.5 is the second
    assert following.tolist() == [2, 2, 5, -1, 5, 3, 3, 3, 3]
    last[0] = 0.0
    assert run_verify(ctx, p, q, tokens, u, last)[1][0].item() == 1
    torch.cuda.synchronize()
    with pytest.raises(mai.SiError):
        ctx.synchronize()


def test_verify_strides_capture_and_shared_rows(ctx):
    """Rows inside wider ones (a logits buffer with padding), captured and replayed on a stream of its own."""
    wide_p, wide_q = torch.rand(3, 4, 1003, device="cuda"), torch.rand(3, 3, 1010, device="cuda")
    p, q = wide_p[:, :, 1:1001], wide_q[:, :, 5:1005]
    tokens = torch.randint(0, 1000, (3, 3), device="cuda", dtype=torch.int32)
    u, last = torch.rand(3, 3, device="cuda"), torch.rand(3, device="cuda")
    s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    accepted, following = torch.empty(3, dtype=torch.int32, device="cuda"), torch.empty(3, dtype=torch.int32, device="cuda")
    work = torch.empty(mai.verify_drafts_workspace_bytes(3, 1000), dtype=torch.uint8, device="cuda")
    args = mai.verify_drafts(p, tokens, u, last, accepted, following, work, draft_probs=q)
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=s):
        ctx.verify_drafts_dev(args, s.cuda_stream)
    for _ in range(4):
        wide_p.uniform_(), u.uniform_(), last.uniform_()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        for b in range(3):
            assert (accepted[b].item(), following[b].item()) == verified(p[b].cpu().numpy(), q[b].cpu().numpy(), tokens[b].tolist(),
                                                                         u[b].tolist(), last[b].item(), 3)


# ---- the operators together ----------------------------------------------------------------
def test_a_bounded_cache_from_prompt_to_eviction(ctx):
    """Two sequences: prompts appended in chunks, then steps that append, attend with weights, and evict to a
    budget, all enqueued without a wait; a plain 64-bit cache that never moves anything follows along."""
    kvh, g, hd, page, budget, sink, recent = 2, 3, 64, 8, 40, 2, 8
    prompts, steps = [45, 13], 30
    cache = Cache([56, 56], kvh, page, hd, BF16, seed=8)
    table, scale = mai.rope_table(1e4, 32, "yarn", factor=4.0, original=64)
    rope = torch.from_numpy(table.view(np.int64)).cuda()
    weights = torch.zeros(2, kvh, 56, device="cuda")
    positions = torch.zeros(2, kvh, 56, dtype=torch.int32, device="cuda")
    length = torch.tensor(prompts, dtype=torch.int32, device="cuda")
    evict_work = torch.empty(mai.paged_evict_workspace_bytes(cache.desc), dtype=torch.uint8, device="cuda")
    kept = [[{} for _ in range(kvh)] for _ in range(2)]  # position -> (key, value, weight)
    # prompt
    rows = [(b, t) for b, n in enumerate(prompts) for t in range(n)]
    seq, slot = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in zip(*rows))
    k, v = (torch.randn(len(rows), kvh, hd, device="cuda") for _ in range(2))
    for lo in range(0, len(rows), 25):
        part = slice(lo, lo + 25)
        ctx.paged_append_dev(cache.desc, mai.paged_append(cache.desc, None, k[part], v[part], None, slot[part].contiguous(),
                                                          sequence=seq[part].contiguous(), rope=rope, rotary_dim=32, layout="half",
                                                          rope_scale=scale), LEGACY)
    positions[:] = torch.arange(56, dtype=torch.int32, device="cuda")
    turned = rotated(k, slot.double()[:, None] * torch.tensor(table.astype(np.float64) / 2.0 ** 64 * 2 * math.pi).cuda(), "half", scale)
    for i, (b, t) in enumerate(rows):
        for h in range(kvh):
            kept[b][h][t] = [turned[i, h].to(BF16).double(), v[i, h].to(BF16).double(), 0.0]
    seen = list(prompts)
    for step in range(steps):
        q = torch.randn(2, kvh * g, hd, device="cuda")
        k, v = (torch.randn(2, kvh, hd, device="cuda") for _ in range(2))
        position = torch.tensor(seen, dtype=torch.int32, device="cuda")
        slot = length.clone()
        q_rot, out = torch.empty_like(q), torch.empty_like(q)
        ctx.paged_append_dev(cache.desc, mai.paged_append(cache.desc, q, k, v, q_rot, slot, position=position, rope=rope,
                                                          rotary_dim=32, layout="half", rope_scale=scale), LEGACY)
        at = slot.long()[:, None].expand(2, kvh)[..., None]
        positions.scatter_(2, at, position[:, None, None].expand(2, kvh, 1).contiguous())
        weights.scatter_(2, at, 0.0)
        length += 1
        work = work_for(cache, kvh * g, True)
        ctx.paged_attention_dev(cache.desc, mai.paged_attention(cache.desc, q_rot, out, length, work, weights_in=weights,
                                                                weights_out=weights), LEGACY)
        nxt = position + 1
        ctx.paged_evict_dev(cache.desc, mai.paged_evict(cache.desc, length, length, weights, weights, budget, evict_work, sink=sink,
                                                        recent=recent, positions_in=positions, positions_out=positions,
                                                        next_position=nxt), LEGACY)
        angle = position.double()[:, None] * torch.tensor(table.astype(np.float64) / 2.0 ** 64 * 2 * math.pi).cuda()
        kr, qr = rotated(k, angle, "half", scale), rotated(q, angle, "half", scale)
        for b in range(2):
            want = torch.zeros(kvh * g, hd, dtype=torch.float64, device="cuda")
            for h in range(kvh):
                kept[b][h][seen[b]] = [kr[b, h].to(BF16).double(), v[b, h].to(BF16).double(), 0.0]
                order = sorted(kept[b][h])
                keys, values = (torch.stack([kept[b][h][p][i] for p in order]) for i in (0, 1))
                prob = torch.softmax(qr[b, h * g:(h + 1) * g] @ keys.T / 8, -1)
                want[h * g:(h + 1) * g] = prob @ values
                for p, x in zip(order, prob.sum(0).tolist()):
                    kept[b][h][p][2] += x
                free = sorted((p for p in order if sink <= p < seen[b] + 1 - recent), key=lambda p: kept[b][h][p][2])
                for p in free[:max(0, len(order) - budget)]:
                    del kept[b][h][p]
            # keys rounded from f32 and from f64 rotations differ by a bf16 step now and then: 2^-8 of one product
            close(out[b], want, F32, 1e-3)
            seen[b] += 1
    ctx.synchronize()
    assert length.tolist() == [min(n + steps, budget) for n in prompts]
    for b in range(2):
        n = length[b].item()
        for h in range(kvh):
            got = positions[b, h, :n].tolist()
            assert len(set(got)) == n and set(got) == set(kept[b][h])
            assert all(abs(weights[b, h, i].item() - kept[b][h][p][2]) < 1e-2 for i, p in enumerate(got))


def test_drafts_over_the_paged_cache(ctx):
    """A window of drafts as rows that share pages: probabilities from attention rows, verification, and the cache
    kept to the accepted tokens by the length alone."""
    kvh, g, hd, page, k_drafts, vocab = 2, 2, 64, 8, 3, 97
    cache = Cache([30], kvh, page, hd, BF16, seed=12, room=2)
    pages = cache.pages_dev.expand(k_drafts + 1, -1).contiguous()
    kv = mai.paged_kv(cache.k, cache.v, pages)
    new_k, new_v = (torch.randn(k_drafts + 1, kvh, hd, device="cuda") for _ in range(2))
    slot = torch.arange(30, 31 + k_drafts, dtype=torch.int32, device="cuda")
    ctx.paged_append_dev(kv, mai.paged_append(kv, None, new_k, new_v, None, slot), LEGACY)
    q = torch.randn(k_drafts + 1, kvh * g, hd, device="cuda")
    out, n = torch.empty_like(q), slot + 1
    work = torch.empty(mai.paged_attention_workspace_bytes(kv, kvh * g), dtype=torch.uint8, device="cuda")
    ctx.paged_attention_dev(kv, mai.paged_attention(kv, q, out, n, work), LEGACY)
    for i in range(k_drafts + 1):
        cache.lengths = [31 + i]
        close(out[i:i + 1], reference(cache, q[i:i + 1])[0], F32)
    head = torch.randn(kvh * g * hd, vocab, device="cuda") / 8
    p = torch.softmax(out.reshape(k_drafts + 1, -1) @ head, -1)[None]
    tokens = p[:, :k_drafts].argmax(-1).to(torch.int32)
    u, last = torch.tensor([[0.0, 0.9999999, 0.0]], device="cuda"), torch.tensor([0.3], device="cuda")
    accepted, following = run_verify(ctx, p, None, tokens, u, last)
    want = verified(p[0].cpu().numpy(), None, tokens[0].tolist(), u[0].tolist(), 0.3, k_drafts)
    assert (accepted.item(), following.item()) == (want[0], verified(p[0].cpu().numpy(), None, tokens[0].tolist(), u[0].tolist(),
                                                                     last.item(), k_drafts)[1])
    ctx.synchronize()


# ---- calls that the documentation allows and that come up seldom ------------------------------
@pytest.mark.parametrize("hd", [136, 184, 200, 248])
@pytest.mark.parametrize("io, cache_type", [(F32, BF16), (BF16, BF16), (F32, F16)])
def test_attention_odd_heads(ctx, hd, io, cache_type):
    """Heads that leave part of the last steps empty, long and short rows, whole pairs and split ones."""
    cache = Cache([700, 0, 1, 33, 16, 5000], 2, 16, hd, cache_type, seed=hd, order="tokens_first")
    q = torch.randn(6, 14, hd, device="cuda").to(io)
    close(attend(ctx, cache, q), reference(cache, q)[0], io)


def test_attention_many_short_sequences(ctx):
    """The most sequences that a call takes, most of them empty or of one token."""
    lengths = [(0, 1, 0, 2, 17)[i % 5] for i in range(4096)]
    cache = Cache(lengths, 1, 16, 64, BF16, seed=1)
    q = torch.randn(4096, 2, 64, device="cuda")
    out = attend(ctx, cache, q)
    want, _, _ = reference(cache, q)
    close(out, want, F32)
    assert (out[::5] == 0).all()


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_attention_keeps_rows_apart(ctx, hd, bad):
    """A sequence whose cache or query holds NaN or infinity leaves the others alone, in the same warp or not."""
    lengths = [20, 7, 300, 5, 1, 0, 40, 33]
    for io, cache_type in ((F32, BF16), (F16, F16)):
        cache = Cache(lengths, 2, 16, hd, cache_type, seed=hd)
        q = torch.randn(8, 4, hd, device="cuda").to(io)
        want, _, _ = reference(cache, q)
        for b, pool in ((1, cache.k), (3, cache.v), (6, cache.k)):
            pg, at = cache.cells(b, lengths[b])
            pool[pg, :, at] = bad
        q[4] = bad
        out = attend(ctx, cache, q)
        good = [0, 2, 5, 7]
        close(out[good], want[good], io)
        assert not torch.isfinite(out[[3, 4]]).any()


def test_operators_on_streams_of_their_own(ctx):
    """All four operators on four streams at once, twenty times, with workspaces of their own."""
    streams = [torch.cuda.Stream() for _ in range(4)]
    att = Cache([900, 33, 0], 2, 16, 128, BF16, seed=1)
    q = torch.randn(3, 8, 128, device="cuda")
    out = torch.empty_like(q)
    attention = mai.paged_attention(att.desc, q, out, att.len_dev, work_for(att, 8))
    app = Cache([40] * 4, 2, 8, 64, BF16, seed=2)
    new, slot = torch.randn(4, 2, 64, device="cuda").to(BF16), torch.tensor([3, 39, 0, 17], dtype=torch.int32, device="cuda")
    append = mai.paged_append(app.desc, None, new, new, None, slot)
    ev = Cache([600, 20], 2, 16, 64, F16, seed=3)
    w = torch.rand(2, 2, 640, device="cuda")
    w_out, n_out = torch.zeros_like(w), torch.zeros_like(ev.len_dev)
    evict = mai.paged_evict(ev.desc, ev.len_dev, n_out, w, w_out, 500,
                            torch.empty(mai.paged_evict_workspace_bytes(ev.desc), dtype=torch.uint8, device="cuda"), recent=50)
    p = torch.rand(5, 4, 3001, device="cuda")
    tokens, u, last = torch.zeros(5, 3, dtype=torch.int32, device="cuda"), torch.rand(5, 3, device="cuda"), torch.rand(5, device="cuda")
    accepted, following = (torch.zeros(5, dtype=torch.int32, device="cuda") for _ in range(2))
    verify = mai.verify_drafts(p, tokens, u, last, accepted, following, torch.empty(16, dtype=torch.uint8, device="cuda"))
    torch.cuda.synchronize()
    for _ in range(20):
        ctx.paged_attention_dev(att.desc, attention, streams[0].cuda_stream)
        ctx.paged_append_dev(app.desc, append, streams[1].cuda_stream)
        ctx.paged_evict_dev(ev.desc, evict, streams[2].cuda_stream)
        ctx.verify_drafts_dev(verify, streams[3].cuda_stream)
    torch.cuda.synchronize()
    ctx.synchronize()
    close(out, reference(att, q)[0], F32)
    for b, t in enumerate(slot.tolist()):
        assert torch.equal(app.k[app.pages[b, t // 8].item(), :, t % 8], new[b])
    assert n_out.tolist() == [500, 20]
    for h in range(2):
        holes, movers = evicted(w[0, h].tolist(), list(range(640)), 600, 500, 0, 50, 600)
        got = w[0, h, :500].clone()
        got[holes] = w[0, h, movers]
        assert torch.equal(w_out[0, h, :500], got)
    for b in range(5):
        assert (accepted[b].item(), following[b].item()) == verified(p[b].cpu().numpy(), None, tokens[b].tolist(), u[b].tolist(),
                                                                     last[b].item(), 3)


@pytest.mark.parametrize("leave", [30, 700])
def test_evict_captured_in_place(ctx, leave):
    """A captured call over its own lengths: the first replay cuts, the next ones find nothing to do."""
    n, budget = 2000, 2000 - leave
    cache = Cache([n, 100], 2, 16, 64, BF16, seed=leave)
    w = torch.rand(2, 2, n, device="cuda")
    pos = torch.arange(n, dtype=torch.int32, device="cuda").expand(2, 2, n).contiguous()
    length, before = cache.len_dev, w.clone()
    work = torch.empty(mai.paged_evict_workspace_bytes(cache.desc), dtype=torch.uint8, device="cuda")
    args = mai.paged_evict(cache.desc, length, length, w, w, budget, work, sink=4, recent=16, positions_in=pos, positions_out=pos)
    s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=s):
        ctx.paged_evict_dev(cache.desc, args, s.cuda_stream)
    k0 = cache.k.clone()
    for turn in range(3):
        g.replay()
        torch.cuda.synchronize()
        assert length.tolist() == [budget, 100]
        for h in range(2):
            holes, movers = evicted(before[0, h].tolist(), list(range(n)), n, budget, 4, 16, n)
            want = list(range(budget))
            for a, b in zip(holes, movers):
                want[a] = b
            assert pos[0, h, :budget].tolist() == want
            assert torch.equal(w[0, h, :budget], before[0, h, want])
            pg, at = cache.cells(0, n)
            assert torch.equal(cache.k[pg[:budget], h, at[:budget]], k0[pg[want], h, at[want]])
        assert torch.equal(w[1], before[1])


def test_append_captured_follows_positions(ctx):
    cache = Cache([64, 64], 2, 8, 64, BF16, seed=5)
    table, _ = mai.rope_table(1e5, 64)
    rope = torch.from_numpy(table.view(np.int64)).cuda()
    q, k = torch.randn(2, 4, 64, device="cuda"), torch.randn(2, 2, 64, device="cuda")
    out, slot = torch.empty_like(q), torch.zeros(2, dtype=torch.int32, device="cuda")
    args = mai.paged_append(cache.desc, q, k, k, out, slot, rope=rope, rotary_dim=64, layout="half")
    s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=s):
        ctx.paged_append_dev(cache.desc, args, s.cuda_stream)
    for slots in ([0, 63], [5, -1], [17, 40]):
        slot.copy_(torch.tensor(slots))
        out.fill_(7.0)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        angle = torch.tensor([[max(t, 0) * int(f) / 2.0 ** 64 * 2 * math.pi for f in table] for t in slots], dtype=torch.float64).cuda()
        want, keys = rotated(q, angle, "half", 1.0), rotated(k, angle, "half", 1.0)
        for b, t in enumerate(slots):
            if t < 0:
                assert (out[b] == 7).all()
                continue
            close(out[b], want[b], F32)
            close(cache.k[cache.pages[b, t // 8].item(), :, t % 8], keys[b], BF16)


@pytest.mark.parametrize("vocab", [300, 9000, 100003])
def test_verify_draws_from_the_target_when_nothing_is_left(ctx, vocab):
    """The drafter's row is the target's: a token of no weight is rejected, and the row itself is drawn from."""
    gen = torch.Generator(device="cuda").manual_seed(vocab)
    p = torch.softmax(torch.randn(7, 3, vocab, device="cuda", generator=gen), -1)
    p[:, :, 11] = 0
    q = p[:, :2].clone()
    tokens = torch.full((7, 2), 11, dtype=torch.int32, device="cuda")
    u, last = torch.rand(7, 2, device="cuda", generator=gen), torch.linspace(0, 0.999, 7, device="cuda")
    accepted, following = run_verify(ctx, p, q, tokens, u, last)
    for b in range(7):
        assert (accepted[b].item(), following[b].item()) == verified(p[b].cpu().numpy(), q[b].cpu().numpy(), tokens[b].tolist(),
                                                                     u[b].tolist(), last[b].item(), 2)


def test_tensors_of_another_device_are_refused(ctx):
    cache = Cache([4], 1, 4, 64)
    host = mai.paged_kv(cache.k.cpu(), cache.v.cpu(), cache.pages)
    q, n = torch.zeros(1, 1, 64), torch.zeros(1, dtype=torch.int32)
    args = mai.paged_attention(host, q, q, n, torch.empty(1 << 22, dtype=torch.uint8))
    with pytest.raises(mai.SiError):
        ctx.paged_attention_dev(host, args, LEGACY)
    with pytest.raises(mai.SiError):
        mai.paged_attention(cache.desc, q, q, n, torch.empty(1 << 22, dtype=torch.uint8))


@pytest.mark.parametrize("n, vocab", [(1, 248320), (9, 32003), (200, 700)])
def test_accepted_counts_over_the_counts(ctx, n, vocab):
    """One array for the drafts' counts and the accepted ones, many times: the
    blocks of a sequence all read the count before it is written over."""
    gen = torch.Generator(device="cuda").manual_seed(n)
    p = torch.softmax(torch.randn(n, 5, vocab, device="cuda", generator=gen), -1)
    tokens = p[:, :4].argmax(-1).to(torch.int32)
    u, last = torch.rand(n, 4, device="cuda", generator=gen) * 2e-4, torch.rand(n, device="cuda", generator=gen)
    counts = torch.randint(0, 5, (n,), device="cuda", generator=gen, dtype=torch.int32)
    work = torch.empty(16, dtype=torch.uint8, device="cuda")
    want = run_verify(ctx, p, None, tokens, u, last, counts)
    following = torch.empty_like(counts)
    for _ in range(50):
        both = counts.clone()
        torch.cuda.synchronize()
        ctx.verify_drafts_dev(mai.verify_drafts(p, tokens, u, last, both, following, work, counts=both), LEGACY)
        torch.cuda.synchronize()
        assert torch.equal(both, want[0]) and torch.equal(following, want[1])
    for b in range(min(n, 9)):
        assert (want[0][b].item(), want[1][b].item()) == verified(p[b].cpu().numpy(), None, tokens[b].tolist(), u[b].tolist(),
                                                                  last[b].item(), int(counts[b]))


@pytest.mark.parametrize("probs", [True, False])
@pytest.mark.parametrize("n, vocab", [(70, 100000), (90, 100003), (160, 65537)])
def test_verify_long_runs(ctx, n, vocab, probs):
    """Enough sequences that a warp's run is longer than its block has threads;
    rows on and off 16-byte boundaries, most tokens without weight."""
    gen = torch.Generator(device="cuda").manual_seed(n)
    rnd = lambda *s: torch.rand(*s, device="cuda", generator=gen)  # noqa: E731
    p = torch.where(rnd(n, 2, vocab) < 1e-3, rnd(n, 2, vocab), torch.zeros((), device="cuda"))
    p /= p.sum(-1, keepdim=True)
    q = torch.where(rnd(n, 1, vocab) < 0.5, p[:, :1], torch.zeros((), device="cuda")) if probs else None
    tokens = p[:, :1].argmax(-1).to(torch.int32)
    u, last = rnd(n, 1), rnd(n)
    u[::2] = 0.99999
    last[0], last[1], last[2], last[3] = 0.0, 1 - 2 ** -24, 0.0, 1 - 2 ** -24
    accepted, following = run_verify(ctx, p, q, tokens, u, last)
    for b in range(n):
        want = verified(p[b].cpu().numpy(), q[b].cpu().numpy() if probs else None, tokens[b].tolist(), u[b].tolist(), last[b].item(), 1)
        assert (accepted[b].item(), following[b].item()) == want, b


@pytest.mark.parametrize("probs", [True, False])
@pytest.mark.parametrize("n, vocab", [(3, 50000), (3, 50001), (70, 60000)])
def test_verify_leaves_out_odd_entries_of_long_rows(ctx, n, vocab, probs):
    """Infinite, NaN and negative entries anywhere in a row, of either side, count as 0."""
    gen = torch.Generator(device="cuda").manual_seed(vocab + n)
    p = torch.softmax(torch.randn(n, 2, vocab, device="cuda", generator=gen), -1)
    q = torch.softmax(torch.randn(n, 1, vocab, device="cuda", generator=gen), -1) if probs else None
    for side in (p, q):
        if side is not None:
            for odd in (math.inf, -math.inf, math.nan, -1.0):
                at = torch.randint(0, vocab, (n, side.shape[1], 5), device="cuda", generator=gen)
                side.scatter_(2, at, odd)
    tokens = torch.randint(0, vocab, (n, 1), device="cuda", generator=gen, dtype=torch.int32)
    u, last = torch.full((n, 1), 0.999, device="cuda"), torch.linspace(0, 0.999, n, device="cuda")
    accepted, following = run_verify(ctx, p, q, tokens, u, last)
    for b in range(n):
        want = verified(p[b].cpu().numpy(), q[b].cpu().numpy() if probs else None, tokens[b].tolist(), u[b].tolist(), last[b].item(), 1)
        assert (accepted[b].item(), following[b].item()) == want, b


def test_a_report_on_another_stream_is_not_lost(ctx):
    """The context's stream and the legacy one each hold a call with a bad slot, the legacy one's behind some
    work. Reporting the first must not clear the second, which is not there yet."""
    cache = Cache([16], 1, 8, 64, BF16, seed=2)
    new = torch.zeros(1, 1, 64, dtype=BF16, device="cuda")
    slot = torch.tensor([16], dtype=torch.int32, device="cuda")  # beyond the table
    bad = mai.paged_append(cache.desc, None, new, new, None, slot)
    for stream in (None, LEGACY):  # both kinds of launch once, so that nothing is loaded below
        ctx.paged_append_dev(cache.desc, bad, stream)
        torch.cuda.synchronize()
        with pytest.raises(mai.SiError):
            ctx.synchronize()
    ctx.synchronize()
    torch.cuda._sleep(200_000_000)  # about a tenth of a second
    ctx.paged_append_dev(cache.desc, bad, LEGACY)
    ctx.paged_append_dev(cache.desc, bad, None)
    with pytest.raises(mai.SiError) as e:
        ctx.synchronize()
    assert e.value.status == mai.SI_E_INVALID
    assert not torch.cuda.default_stream().query()  # the other call is still to come
    torch.cuda.synchronize()
    with pytest.raises(mai.SiError) as e:
        ctx.synchronize()
    assert e.value.status == mai.SI_E_INVALID
    ctx.synchronize()


def test_slots_behind_a_cut_start_anew(ctx):
    """The serving loop over arrays that hold other tokens' weights and positions at every slot not in use:
    whatever lies there, a new token's weight counts from 0 and its position is its own."""
    kvh, g, hd, budget, sink, recent, seqs = 2, 2, 64, 20, 2, 4, 3
    gen = torch.Generator().manual_seed(5)
    cache = Cache([0] * seqs, kvh, 8, hd, BF16, seed=6, room=4)
    weights = torch.full((seqs, kvh, 32), 7e3, device="cuda")  # would outweigh every real one
    positions = torch.full((seqs, kvh, 32), -5, dtype=torch.int32, device="cuda")  # would be protected
    length, seen = torch.zeros(seqs, dtype=torch.int32, device="cuda"), [0] * seqs
    attention_work, evict_work = work_for(cache, kvh * g, True), torch.empty(mai.paged_evict_workspace_bytes(cache.desc),
                                                                             dtype=torch.uint8, device="cuda")
    want_w, want_p = [[{} for _ in range(kvh)] for _ in range(seqs)], [[{} for _ in range(kvh)] for _ in range(seqs)]
    for step in range(12):
        rows = [(b, length[b].item() + i, seen[b] + i) for b in range(seqs) for i in range((4, 1, 3)[(b + step) % 3])]
        sequence, slot, position = (torch.tensor(x, dtype=torch.int32).cuda() for x in zip(*rows))
        k, v = (torch.randn(len(rows), kvh, hd, generator=gen).to(BF16).cuda() for _ in range(2))
        ctx.paged_append_dev(cache.desc, mai.paged_append(cache.desc, None, k, v, None, slot, sequence=sequence, position=position,
                                                          weights=weights, positions=positions), LEGACY)
        for b, t, p in rows:
            seen[b] = p + 1
            length[b] = t + 1
            for h in range(kvh):
                want_w[b][h][t], want_p[b][h][t] = 0.0, p
        q = torch.randn(seqs, kvh * g, hd, generator=gen).cuda()
        out = torch.empty_like(q)
        ctx.paged_attention_dev(cache.desc, mai.paged_attention(cache.desc, q, out, length, attention_work, weights_in=weights,
                                                                weights_out=weights), LEGACY)
        want, _, probs = reference(cache, q, lengths=length.tolist())
        close(out, want, F32)
        before = weights.clone()
        for b in range(seqs):
            for h in range(kvh):
                for t in range(length[b].item()):
                    want_w[b][h][t] += probs[b][h, t].item()
                    assert before[b, h, t].item() == pytest.approx(want_w[b][h][t], rel=1e-5, abs=1e-6)
        nxt = torch.tensor(seen, dtype=torch.int32, device="cuda")
        n = length.tolist()
        ctx.paged_evict_dev(cache.desc, mai.paged_evict(cache.desc, length, length, weights, weights, budget, evict_work, sink=sink,
                                                        recent=recent, positions_in=positions, positions_out=positions,
                                                        next_position=nxt), LEGACY)
        assert length.tolist() == [min(x, budget) for x in n]
        for b in range(seqs):
            for h in range(kvh):
                of = [want_p[b][h][t] for t in range(n[b])]
                holes, movers = evicted(before[b, h].tolist(), of, n[b], budget, sink, recent, seen[b])
                for a, c in zip(holes, movers):
                    want_w[b][h][a], want_p[b][h][a] = want_w[b][h][c], want_p[b][h][c]
                assert positions[b, h, :length[b]].tolist() == [want_p[b][h][t] for t in range(length[b].item())]
    ctx.synchronize()


def test_append_leaves_out_slots_beyond_the_started_arrays(ctx):
    """Slots that the weights have no entry for are reported, and nothing of the token is written."""
    cache = Cache([32, 32], 2, 8, 64, BF16, seed=3)
    k0 = cache.k.clone()
    weights = torch.full((2, 2, 20), 3.0, device="cuda")
    positions = torch.full((2, 2, 20), 9, dtype=torch.int32, device="cuda")
    new = torch.randn(4, 2, 64, device="cuda").to(BF16)
    slot = torch.tensor([20, 19, -1, 31], dtype=torch.int32, device="cuda")
    sequence = torch.tensor([0, 1, 1, 1], dtype=torch.int32, device="cuda")
    ctx.paged_append_dev(cache.desc, mai.paged_append(cache.desc, None, new, new, None, slot, sequence=sequence, weights=weights,
                                                      positions=positions), LEGACY)
    torch.cuda.synchronize()
    with pytest.raises(mai.SiError) as e:
        ctx.synchronize()
    assert e.value.status == mai.SI_E_INVALID
    assert (weights[1, :, 19] == 0).all() and (positions[1, :, 19] == 19).all()
    weights[1, :, 19], positions[1, :, 19] = 3.0, 9
    assert (weights == 3).all() and (positions == 9).all()
    pg = cache.pages[1, 2].item()
    assert torch.equal(cache.k[pg, :, 3], new[1])
    cache.k[pg, :, 3] = k0[pg, :, 3]
    assert torch.equal(cache.k.view(torch.int16), k0.view(torch.int16))


def test_attention_long_rows_are_not_biased(ctx):
    """Positive values over rows of 131,072 slots that one worker walks whole: sums that are cut off, not rounded,
    fall short by half a unit in the last place an addition, a few 1e-4 here. Roundings of either sign leave the
    mean error of all outputs far below one output's: half a step / sqrt(3 N) with N outputs, were they independent;
    a sixteenth of half a step (3e-5) leaves room for outputs of a dim that lie close together."""
    n, hd, page = 131072, 64, 256
    rows = min(4096, 24 * torch.cuda.get_device_properties(0).multi_processor_count)  # two for each worker of 12 a multiprocessor
    gen = torch.Generator(device="cuda").manual_seed(7)
    k = torch.randn(n // page, 1, page, hd, device="cuda", generator=gen).to(F16)
    v = ((0.5 + torch.rand(n // page, 1, page, hd, device="cuda", generator=gen)) *
         (1 + torch.rand(hd, device="cuda", generator=gen))).to(F16)
    pages = torch.arange(n // page, dtype=torch.int32, device="cuda").expand(rows, -1).contiguous()
    kv = mai.paged_kv(k, v, pages)
    q = torch.randn(rows, 1, hd, device="cuda", generator=gen).to(F16)
    out, length = torch.empty_like(q), torch.full((rows,), n, dtype=torch.int32, device="cuda")
    work = torch.empty(mai.paged_attention_workspace_bytes(kv, 1), dtype=torch.uint8, device="cuda")
    ctx.paged_attention_dev(kv, mai.paged_attention(kv, q, out, length, work), LEGACY)
    keys, values = (x.reshape(n, hd).double() for x in (k, v))
    want = torch.cat([torch.softmax(x.double() @ keys.T / hd ** 0.5, -1) @ values for x in q[:, 0].split(256)])
    error = (out[:, 0].double() - want) / want
    assert error.abs().max() <= half_step(F16) * 1.02  # the rounding itself, and 2e-2 of it for all sums
    assert abs(error.mean().item()) <= half_step(F16) / 16


def test_append_leaves_out_the_queries_of_bad_tokens(ctx):
    """A token whose slot, sequence or page does not exist is left out whole: its queries are not written either."""
    cache = Cache([16, 16], 2, 8, 64, BF16, seed=4)
    cache.pages_dev[1, 1] = -3
    slot = torch.tensor([3, 16, 9, 2, 5], dtype=torch.int32, device="cuda")
    sequence = torch.tensor([0, 0, 1, -1, 1], dtype=torch.int32, device="cuda")
    q, k = torch.randn(5, 4, 64, device="cuda"), torch.randn(5, 2, 64, device="cuda")
    out = torch.full_like(q, 7.0)
    ctx.paged_append_dev(cache.desc, mai.paged_append(cache.desc, q, k, k, out, slot, sequence=sequence), LEGACY)
    torch.cuda.synchronize()
    with pytest.raises(mai.SiError):
        ctx.synchronize()
    assert torch.equal(out[[0, 4]], q[[0, 4]]) and (out[1:4] == 7).all()


def evicted_rows(w, pos, n, budget, sink, recent, nxt):
    """`evicted` by numpy: (holes, kept slots behind the budget) of one row of finite weights."""
    held = (pos[:n] < sink) | (pos[:n] >= nxt - recent)
    order = np.lexsort((np.arange(n), np.where(held, 0, w[:n]), held))  # protected last, by weight, by slot
    gone = np.zeros(n, bool)
    gone[order[:max(0, n - budget)]] = True
    m = min(n, budget)
    return np.flatnonzero(gone[:m]), m + np.flatnonzero(~gone[m:])


EVICT_MANY = [
    # sequences, kv_heads, longest, budget: rows that outnumber the clusters' places, and the largest row
    (64, 1, 8193, 8100),     # 1024 threads, no cluster, moves in the same kernel (not over its own lengths)
    (19, 3, 20000, 9000),    # the same, moves in a second kernel
    (57, 1, 49152, 49100),   # the most keys of one CTA
    (5, 2, 70000, 4000),     # clusters of 8 cut to 6
    (10, 2, 60000, 30000),   # to 4
    (15, 2, 90000, 89990),   # to 2, 45,000 keys a CTA
    (1, 1, 393216, 200000),  # the longest row, the most keys in each CTA of a cluster of 8
    (1, 1, 393216, 393215),
]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("case", range(len(EVICT_MANY)))
def test_evict_many_and_long_rows(ctx, case, in_place):
    seqs, kvh, longest, budget = EVICT_MANY[case]
    rng = np.random.default_rng(case)
    lengths = [longest] + [int(x) for x in rng.integers(budget // 2, longest + 1, seqs - 1)]
    if seqs > 4:
        lengths[3], lengths[-1] = 0, longest
    hd, sink, recent, page = 8, 3, 40, 4096
    cache = Cache(lengths, kvh, page, hd, BF16, seed=case, cols=-(-longest // page))
    cache.k.nan_to_num_(0.0), cache.v.nan_to_num_(0.0)
    shape = (seqs, kvh, longest)
    w = (np.floor(np.exp(2 * rng.normal(size=shape)) * 64) / 64).astype(np.float32)  # many ties among the small ones
    pos = np.broadcast_to(np.arange(longest, dtype=np.int32), shape).copy()
    w_in, p_in = torch.from_numpy(w).cuda(), torch.from_numpy(pos).cuda()
    w_out = w_in if in_place else torch.full_like(w_in, 3.5)
    p_out = p_in if in_place else torch.full_like(p_in, -9)
    n_out = cache.len_dev if in_place else torch.full_like(cache.len_dev, -1)
    work = torch.empty(mai.paged_evict_workspace_bytes(cache.desc), dtype=torch.uint8, device="cuda").fill_(255)
    k0, v0 = cache.k.clone(), cache.v.clone()
    ctx.paged_evict_dev(cache.desc, mai.paged_evict(cache.desc, cache.len_dev, n_out, w_in, w_out, budget, work, sink=sink, recent=recent,
                                                    positions_in=p_in, positions_out=p_out), LEGACY)
    torch.cuda.synchronize()
    ctx.synchronize()
    assert n_out.tolist() == [min(n, budget) for n in lengths]
    want_w = w.copy() if in_place else np.full_like(w, 3.5)
    want_p = pos.copy() if in_place else np.full_like(pos, -9)
    for b, n in enumerate(lengths):
        m = min(n, budget)
        pg, at = cache.cells(b, n)
        for h in range(kvh):
            holes, movers = evicted_rows(w[b, h], pos[b, h], n, budget, sink, recent, n)
            assert len(holes) == len(movers)
            want_w[b, h, :m], want_p[b, h, :m] = w[b, h, :m], pos[b, h, :m]
            want_w[b, h, holes], want_p[b, h, holes] = w[b, h, movers], pos[b, h, movers]
            to, of = torch.from_numpy(holes).cuda(), torch.from_numpy(movers).cuda()
            for pool, start in ((cache.k, k0), (cache.v, v0)):
                moved = start[pg[of], h, at[of]].clone()
                assert torch.equal(pool[pg[to], h, at[to]], moved)
                pool[pg[to], h, at[to]] = start[pg[to], h, at[to]]
    np.testing.assert_array_equal(w_out.cpu().numpy().view(np.uint32), want_w.view(np.uint32))
    np.testing.assert_array_equal(p_out.cpu().numpy(), want_p)
    assert torch.equal(cache.k, k0) and torch.equal(cache.v, v0)


def test_evicted_rows_agree_with_the_definition():
    rng = np.random.default_rng(1)
    for n in (1, 7, 60):
        for budget in (1, 5, 30, 60):
            w = np.floor(rng.random(n) * 4).astype(np.float32)
            pos = rng.permutation(2 * n)[:n].astype(np.int32)
            holes, movers = evicted_rows(w, pos, n, budget, 1, min(3, budget - 1), 2 * n)
            assert (holes.tolist(), movers.tolist()) == evicted(w, pos, n, budget, 1, min(3, budget - 1), 2 * n)


def test_two_contexts_in_two_threads(ctx):
    """Two host threads with contexts of their own launch the same kernels with different sizes, and so different
    shared-memory needs, at once."""
    import threading
    failures = []

    def work(lengths, rows, seed):
        try:
            own, stream = mai.CudaContext(0), torch.cuda.Stream()
            with torch.cuda.stream(stream):
                cache = Cache(lengths, 1, 16, 64, BF16, seed=seed)
                q = torch.randn(len(lengths), 2, 64, device="cuda")
                out, scratch = torch.empty_like(q), work_for(cache, 2)
                attention = mai.paged_attention(cache.desc, q, out, cache.len_dev, scratch)
                long = Cache([rows], 1, 256, 8, F16, seed=seed)
                w, n_out = torch.rand(1, 1, rows, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
                w_out = torch.empty_like(w)
                evict = mai.paged_evict(long.desc, long.len_dev, n_out, w, w_out, rows - 1,
                                        torch.empty(mai.paged_evict_workspace_bytes(long.desc), dtype=torch.uint8, device="cuda"))
                for _ in range(30):
                    own.paged_attention_dev(cache.desc, attention, stream.cuda_stream)
                    own.paged_evict_dev(long.desc, evict, stream.cuda_stream)
                stream.synchronize()
                own.synchronize()
                close(out, reference(cache, q)[0], F32)
                assert n_out.item() == rows - 1
                least = w[0, 0].argmin().item()
                assert least >= rows - 1 or w_out[0, 0, least] == w[0, 0, rows - 1]
            own.close()
        except BaseException as e:  # noqa: BLE001 - reported by the test's own thread
            failures.append(e)
    threads = [threading.Thread(target=work, args=x) for x in (([5, 900], 1900, 1), ([3] * 4000, 1000, 2), ([17] * 700, 2040, 3))]
    for t in threads:
        t.start()
    for t in threads:
        t.join(120)
    assert not failures and not any(t.is_alive() for t in threads), failures


def test_a_captured_step_with_forks_and_copies(ctx):
    """One graph: inputs copied in, the append, then attention and verification on two branches that meet again,
    the eviction, a copy out. Replayed with other inputs."""
    kvh, g, hd, vocab = 2, 2, 64, 501
    cache = Cache([40, 17], kvh, 8, hd, BF16, seed=21, room=1)
    start_k, start_v = cache.k.clone(), cache.v.clone()
    host_q = torch.randn(2, kvh * g, hd, device="cuda")
    q, out = torch.empty_like(host_q), torch.empty_like(host_q)
    k = torch.randn(2, kvh, hd, device="cuda").to(BF16)
    length0 = torch.tensor([40, 17], dtype=torch.int32, device="cuda")
    slot, length = length0.clone(), length0 + 1
    weights, positions = torch.zeros(2, kvh, 48, device="cuda"), torch.zeros(2, kvh, 48, dtype=torch.int32, device="cuda")
    w_out, n_out = torch.empty_like(weights), torch.empty_like(length)
    p = torch.rand(2, 2, vocab, device="cuda")
    tokens, u, last = torch.zeros(2, 1, dtype=torch.int32, device="cuda"), torch.rand(2, 1, device="cuda"), torch.rand(2, device="cuda")
    accepted, following, copied = (torch.empty(2, dtype=torch.int32, device="cuda") for _ in range(3))
    append = mai.paged_append(cache.desc, None, k, k, None, slot, weights=weights, positions=positions)
    attention = mai.paged_attention(cache.desc, q, out, length, work_for(cache, kvh * g, True), weights_in=weights, weights_out=weights)
    verify = mai.verify_drafts(p, tokens, u, last, accepted, following, torch.empty(16, dtype=torch.uint8, device="cuda"))
    evict = mai.paged_evict(cache.desc, length, n_out, weights, w_out, 30,
                            torch.empty(mai.paged_evict_workspace_bytes(cache.desc), dtype=torch.uint8, device="cuda"))
    main, side, graph = torch.cuda.Stream(), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=main):
        q.copy_(host_q)
        ctx.paged_append_dev(cache.desc, append, main.cuda_stream)
        side.wait_stream(main)
        ctx.verify_drafts_dev(verify, side.cuda_stream)
        ctx.paged_attention_dev(cache.desc, attention, main.cuda_stream)
        main.wait_stream(side)
        ctx.paged_evict_dev(cache.desc, evict, main.cuda_stream)
        copied.copy_(n_out)
    for turn in range(3):
        host_q.normal_(), k.normal_(), u.uniform_(), last.uniform_(), p.uniform_()
        cache.k.copy_(start_k), cache.v.copy_(start_v)
        weights.uniform_(), positions.fill_(-1)
        before = weights.clone()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        ctx.synchronize()
        assert copied.tolist() == [30, 18]
        for b, n in enumerate((41, 18)):
            keys = torch.cat([start_k[cache.cells(b, n - 1)[0], :, cache.cells(b, n - 1)[1]], k[b:b + 1]]).double()
            values = torch.cat([start_v[cache.cells(b, n - 1)[0], :, cache.cells(b, n - 1)[1]], k[b:b + 1]]).double()
            prob = torch.softmax(torch.einsum("hgd,nhd->hgn", host_q[b].double().view(kvh, g, hd), keys) / 8, -1)
            close(out[b], torch.einsum("hgn,nhd->hgd", prob, values).reshape(kvh * g, hd), F32)
            before[b, :, n - 1] = 0
            close(weights[b, :, :n], before[b, :, :n].double() + prob.sum(1), F32)
            assert (positions[b, :, n - 1] == n - 1).all() and (positions[b, :, :n - 1] == -1).all()
            for h in range(kvh):
                holes, movers = evicted(weights[b, h].tolist(), list(range(48)), n, 30, 0, 0, n)
                got = weights[b, h, :min(n, 30)].clone()
                got[holes] = weights[b, h, movers]
                assert torch.equal(w_out[b, h, :min(n, 30)], got)
            assert (accepted[b].item(), following[b].item()) == verified(p[b].cpu().numpy(), None, tokens[b].tolist(), u[b].tolist(),
                                                                         last[b].item(), 1)


def test_evict_with_one_array_of_lengths(ctx):
    """Lengths in, lengths out and next positions in one array: the last `recent` slots of each row are protected."""
    cache = Cache([50, 12, 33], 2, 8, 64, BF16, seed=9)
    n = cache.len_dev.clone()
    w = torch.rand(3, 2, 64, device="cuda")
    w[:, :, 25:] = 0  # the last ones would leave first
    before = w.clone()
    work = torch.empty(mai.paged_evict_workspace_bytes(cache.desc), dtype=torch.uint8, device="cuda")
    ctx.paged_evict_dev(cache.desc, mai.paged_evict(cache.desc, n, n, w, w, 20, work, recent=10, next_position=n), LEGACY)
    assert n.tolist() == [20, 12, 20]
    for b, m in enumerate((50, 12, 33)):
        for h in range(2):
            holes, movers = evicted(before[b, h].tolist(), list(range(64)), m, 20, 0, 10, m)
            want = before[b, h].clone()
            want[holes] = before[b, h, movers]
            assert torch.equal(w[b, h, :min(m, 20)], want[:min(m, 20)])
    ctx.synchronize()
