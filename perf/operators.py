"""Cases and plain forms of the paged-cache operators: rotary positions with the
append into pages, attention of one new token a sequence over pages (with or
without accumulated attention weights), eviction by accumulated weight, and the
verification of drafted tokens by probabilities.

`run` computes an operator in its plain form (elementary torch operations) where
`own` is false, and calls the framework where it is true."""
import importlib.util
import math
import os
import random
import sys

import numpy as np
import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2}


# ---- the framework ---------------------------------------------------------
_framework = None


def _mai():
    """The package (its folder's name is no identifier) and one context."""
    global _framework
    if _framework is None:
        if "mai_b200" not in sys.modules:
            at = os.path.join(os.getcwd(), "memory-aware-inference_b200")
            spec = importlib.util.spec_from_file_location("mai_b200", os.path.join(at, "__init__.py"),
                                                          submodule_search_locations=[at])
            sys.modules["mai_b200"] = importlib.util.module_from_spec(spec)
            spec.loader.exec_module(sys.modules["mai_b200"])
        _framework = sys.modules["mai_b200"], sys.modules["mai_b200"].CudaContext(0)
    return _framework


def _stream():
    return torch.cuda.current_stream().cuda_stream or 1  # 1: the legacy default stream's own handle


# ---- cases -----------------------------------------------------------------
def _attention(name, **k):
    return {"name": name, "op": "attention", **k}


def listed():
    return [
        # one chat turn of a short conversation on the 27B shape: latency
        _attention("attention_b1_517", batch=1, kv_heads=4, group=6, head_dim=256, page=16, tokens=517, ragged=False,
                   cache="bf16", elem="f32", weights=False, shape=1),
        # the same shape over a very long document: one sequence has to fill the card
        _attention("attention_b1_131071", batch=1, kv_heads=4, group=6, head_dim=256, page=64, tokens=131071,
                   ragged=False, cache="bf16", elem="f32", weights=False, shape=2),
        # a serving batch of mixed lengths, an empty row among them
        _attention("attention_b64_ragged", batch=64, kv_heads=8, group=4, head_dim=128, page=64, tokens=16384,
                   ragged=True, cache="bf16", elem="bf16", weights=False, shape=3),
        # a cache that is later evicted from: the weights are accumulated too
        _attention("attention_b8_8192_weights", batch=8, kv_heads=4, group=6, head_dim=256, page=32, tokens=8192,
                   ragged=False, cache="f16", elem="f32", weights=True, shape=4),
        # one key head for each query head, an odd head, an odd page, an odd batch
        _attention("attention_b33_mha96", batch=33, kv_heads=16, group=1, head_dim=96, page=24, tokens=2047,
                   ragged=True, cache="f16", elem="f16", weights=False, shape=5),
        # one decode step of 32 sequences: rotary on a quarter of the head, neighbouring pairs
        {"name": "append_t32", "op": "append", "tokens": 32, "sequences": 32, "kv_heads": 4, "group": 6, "head_dim": 256,
         "rotary": 64, "layout": "interleaved", "scaling": "none", "theta": 1e7, "page": 16, "first": 8191,
         "cache": "bf16", "elem": "f32"},
        # a prefill chunk far into a scaled context, whole head, half layout
        {"name": "append_t8192", "op": "append", "tokens": 8192, "sequences": 3, "kv_heads": 8, "group": 4,
         "head_dim": 128, "rotary": 128, "layout": "half", "scaling": "yarn", "theta": 1e6, "page": 64, "first": 100003,
         "cache": "bf16", "elem": "bf16"},
        # serving in steady state: a page's worth of tokens leaves each sequence's cache
        {"name": "evict_b32_4160", "op": "evict", "batch": 32, "kv_heads": 8, "head_dim": 128, "page": 64, "tokens": 4160,
         "ragged": False, "budget": 4096, "sink": 4, "recent": 128, "cache": "bf16", "shape": 1},
        # a long prompt cut to a sixteenth
        {"name": "evict_b4_131072", "op": "evict", "batch": 4, "kv_heads": 4, "head_dim": 256, "page": 64,
         "tokens": 131072, "ragged": False, "budget": 8192, "sink": 4, "recent": 512, "cache": "bf16", "shape": 2},
        # one sequence's window of 7 drafts over the 27B vocabulary
        {"name": "verify_b1_k7", "op": "verify", "batch": 1, "drafts": 7, "vocab": 248320, "draft_probs": True},
        # a serving batch of the same
        {"name": "verify_b64_k4", "op": "verify", "batch": 64, "drafts": 4, "vocab": 248320, "draft_probs": True},
        # drafts that were looked up, not drawn: the drafter has no probabilities; an odd vocabulary
        {"name": "verify_b16_k3_lookup", "op": "verify", "batch": 16, "drafts": 3, "vocab": 32003, "draft_probs": False},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "append", "evict", "verify"])
    page = rng.choice([1, 8, 16, 24, 32, 64, 128, 256])
    kv_heads, head_dim = rng.choice([1, 2, 4, 5, 8, 16]), rng.choice([64, 80, 96, 128, 192, 256])
    cache = rng.choice(["bf16", "f16"])
    if op == "attention":
        tokens = _log_int(rng, 1, 131071)
        most = max(1, min(128, (1 << 27) // (tokens * kv_heads * head_dim)))
        return {"op": op, "batch": _log_int(rng, 1, most), "kv_heads": kv_heads, "group": rng.choice([1, 2, 3, 4, 6, 8, 12]),
                "head_dim": head_dim, "page": page, "tokens": min(tokens, (1 << 27) // (kv_heads * head_dim)),
                "ragged": rng.random() < 0.5, "cache": cache, "elem": rng.choice(["f32", cache]),
                "weights": rng.random() < 0.3, "shape": rng.randrange(1 << 20)}
    if op == "append":
        rotary = rng.choice([head_dim, head_dim // 2, head_dim // 4 // 2 * 2])
        group, tokens = rng.choice([1, 3, 4, 6, 8]), _log_int(rng, 1, 8192)
        tokens = min(tokens, max(1, 8192 * 40 * 128 // ((group + 2) * kv_heads * head_dim * 2)))
        return {"op": op, "tokens": tokens, "sequences": rng.randint(1, min(tokens, 64)), "kv_heads": kv_heads,
                "group": group, "head_dim": head_dim, "rotary": rotary,
                "layout": rng.choice(["interleaved", "half"]), "scaling": rng.choice(["none", "linear", "ntk", "yarn", "banded"]),
                "theta": rng.choice([1e4, 1e6, 1e7]), "page": page, "first": _log_int(rng, 1, 500000), "cache": cache,
                "elem": rng.choice(["f32", cache])}
    if op == "evict":
        tokens = _log_int(rng, 16, 131072)
        most = max(1, min(64, (1 << 28) // (tokens * kv_heads * head_dim)))
        budget = max(8, int(tokens * rng.uniform(0.05, 1.0)))
        return {"op": op, "batch": _log_int(rng, 1, most), "kv_heads": kv_heads, "head_dim": head_dim, "page": page,
                "tokens": min(tokens, (1 << 28) // (kv_heads * head_dim)), "ragged": rng.random() < 0.5, "budget": budget,
                "sink": rng.randint(0, 4), "recent": rng.randint(0, budget // 2), "cache": cache, "shape": rng.randrange(1 << 20)}
    vocab = _log_int(rng, 257, 248320)
    return {"op": op, "batch": _log_int(rng, 1, 64), "drafts": rng.randint(1, 8) if vocab < 100000 else rng.randint(1, 4),
            "vocab": vocab, "draft_probs": rng.random() < 0.7}


def _lengths(case):
    """Cached tokens of each sequence: part of the case, not of the seed."""
    rng = random.Random(case["shape"])
    n, top = case["batch"], case["tokens"]
    if not case["ragged"]:
        return [top] * n
    got = [_log_int(rng, 1, top) for _ in range(n)]
    got[rng.randrange(n)] = top
    if n >= 4:
        got[n - 1] = 0  # a row of the batch that no sequence uses
        got[n - 2] = top
    return got


def _append_rows(case):
    """(sequence, slot) of each token: the tokens shared out over the sequences in runs."""
    t = torch.arange(case["tokens"])
    s = case["sequences"]
    sequence = t * s // case["tokens"]
    start = (sequence * case["tokens"] + s - 1) // s
    return sequence, t - start + case["first"] % 61


# ---- work ------------------------------------------------------------------
def work(case):
    if case["op"] == "attention":
        n, kv, hd = sum(_lengths(case)), case["kv_heads"], case["head_dim"]
        qh = kv * case["group"]
        e = 2 * case["batch"] * qh * hd * _BYTES[case["elem"]]
        pages = sum(-(-x // case["page"]) for x in _lengths(case)) * 4
        return {"bytes": n * kv * hd * 4 + e + pages + (8 * n * kv if case["weights"] else 0), "flops": 4 * n * qh * hd}
    if case["op"] == "append":
        t, kv, hd, b = case["tokens"], case["kv_heads"], case["head_dim"], _BYTES[case["elem"]]
        qh = kv * case["group"]
        return {"bytes": t * hd * (2 * qh * b + 2 * kv * (b + 2)) + 12 * t, "flops": 3 * t * (qh + kv) * case["rotary"]}
    if case["op"] == "evict":
        total, row = 0.0, case["head_dim"] * 2
        for n in _lengths(case):
            m = min(n, case["budget"])
            kept = min(n, case["sink"] + case["recent"])
            leave = n - m
            moved = min(case["recent"], leave) + max(0, leave - case["recent"]) * (m - kept) / max(1, n - kept)
            total += case["kv_heads"] * (8 * n + 8 * m + (4 * row * moved if leave else 0))
        return {"bytes": total, "flops": total / 8}
    rows = 2 - 0.75 ** case["drafts"] if case["draft_probs"] else 1
    return {"bytes": case["batch"] * (rows * case["vocab"] * 4 + 16 * case["drafts"] + 12),
            "flops": case["batch"] * 3 * case["vocab"]}


# ---- inputs ----------------------------------------------------------------
def _pool(case, lengths, gen, extra=3):
    """Key and value pools [pages][kv_heads][page][head_dim] and a page table in no order."""
    page, cols = case["page"], max(1, max(-(-n // case["page"]) for n in lengths))
    need = [-(-n // page) for n in lengths]
    total = sum(need) + extra
    shape = (total, case["kv_heads"], page, case["head_dim"])
    k = torch.empty(shape, dtype=_TYPES[case["cache"]], device="cuda")
    v = torch.empty_like(k)
    k.normal_(generator=gen)
    v.normal_(generator=gen)
    order = torch.randperm(total, device="cuda", generator=gen, dtype=torch.int32)[: sum(need)]
    per = torch.tensor(need, device="cuda")
    col = torch.arange(cols, device="cuda")
    used = col[None, :] < per[:, None]
    pages = torch.full((len(lengths), cols), -1, dtype=torch.int32, device="cuda")
    pages[used] = order
    return k, v, pages


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    s = {"case": case}
    if case["op"] == "attention":
        lengths = _lengths(case)
        s["k"], s["v"], s["pages"] = _pool(case, lengths, gen)
        s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        s["q"] = rnd(case["batch"], case["kv_heads"] * case["group"], case["head_dim"]).to(_TYPES[case["elem"]])
        s["out"] = torch.zeros_like(s["q"])
        if case["weights"]:
            s["weights_in"] = torch.rand(case["batch"], case["kv_heads"], case["tokens"], device="cuda", generator=gen)
            s["weights_out"] = s["weights_in"].clone()
    elif case["op"] == "append":
        sequence, slot = _append_rows(case)
        reach = [int(slot[sequence == i].max()) + 1 for i in range(case["sequences"])]
        s["k"], s["v"], s["pages"] = _pool(case, reach, gen)
        s["sequence"] = sequence.to(torch.int32).cuda()
        s["slot"] = slot.to(torch.int32).cuda()
        jump = torch.randint(0, 1000, (1,), device="cuda", generator=gen, dtype=torch.int32)
        s["position"] = s["slot"] + case["first"] + jump
        t, kv, hd = case["tokens"], case["kv_heads"], case["head_dim"]
        # the three parts of one projection's output, as a fused product leaves them
        qkv = rnd(t, kv * (case["group"] + 2), hd).to(_TYPES[case["elem"]])
        s["q"], s["new_k"], s["new_v"] = qkv.split([kv * case["group"], kv, kv], dim=1)
        s["q_out"] = torch.zeros(t, kv * case["group"], hd, dtype=qkv.dtype, device="cuda")
    elif case["op"] == "evict":
        lengths = _lengths(case)
        s["k"], s["v"], s["pages"] = _pool(case, lengths, gen)
        s["lengths_in"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        s["lengths_out"] = torch.zeros_like(s["lengths_in"])
        shape = (case["batch"], case["kv_heads"], case["tokens"])
        # accumulated attention is spread over many powers of ten, with equal values among the smallest
        s["weights_in"] = (2.0 * rnd(*shape)).exp_().mul_(4096).floor_().div_(4096)
        s["weights_out"] = torch.zeros(shape, device="cuda")
        s["positions_in"] = torch.arange(case["tokens"], dtype=torch.int32, device="cuda").expand(shape).contiguous()
        s["positions_out"] = torch.zeros(shape, dtype=torch.int32, device="cuda")
    else:
        b, k, v = case["batch"], case["drafts"], case["vocab"]
        logits = 3.0 * rnd(b, k + 1, v)
        s["target"] = torch.softmax(logits, -1)
        s["draft"] = torch.softmax(logits[:, :k] + 0.7 * rnd(b, k, v), -1) if case["draft_probs"] else None
        near = s["draft"] if case["draft_probs"] else s["target"][:, :k]
        cdf = near.double().cumsum(-1)
        at = torch.rand(b, k, 1, device="cuda", generator=gen, dtype=torch.float64) * cdf[..., -1:]
        s["tokens"] = torch.searchsorted(cdf, at, right=True).clamp_(max=v - 1).squeeze(-1).to(torch.int32)
        del logits, cdf
        if not case["draft_probs"]:  # a looked-up draft is often the likeliest token
            s["tokens"] = torch.where(torch.rand(b, k, device="cuda", generator=gen) < 0.7,
                                      s["target"][:, :k].argmax(-1).to(torch.int32), s["tokens"])
        s["uniform"] = torch.rand(b, k, device="cuda", generator=gen)
        s["last_uniform"] = torch.rand(b, device="cuda", generator=gen)
        s["accepted"] = torch.zeros(b, dtype=torch.int32, device="cuda")
        s["next"] = torch.zeros(b, dtype=torch.int32, device="cuda")
    if own:
        _plan(s)
    return s


def _scaling(case):
    """The scaled positions' parameters, as a model's configuration holds them."""
    return {"none": {}, "linear": {"factor": 4.0}, "ntk": {"factor": 8.0},
            "yarn": {"factor": 16.0, "original": 8192, "beta_fast": 32.0, "beta_slow": 1.0},
            "banded": {"factor": 8.0, "original": 8192, "low": 1.0, "high": 4.0}}[case["scaling"]]


def _plan(s):
    """What a program of the framework keeps between calls: descriptions of its buffers, tables, workspaces."""
    mai, ctx = _mai()
    case = s["case"]
    if case["op"] != "verify":
        s["kv"] = mai.paged_kv(s["k"], s["v"], s["pages"])
    if case["op"] == "attention":
        size = mai.paged_attention_workspace_bytes(s["kv"], s["q"].shape[1], weights=case["weights"])
        s["work"] = torch.empty(max(size, 16), dtype=torch.uint8, device="cuda")
        s["args"] = mai.paged_attention(s["kv"], s["q"], s["out"], s["lengths"], work=s["work"],
                                        weights_in=s.get("weights_in"), weights_out=s.get("weights_out"))
    elif case["op"] == "append":
        table, scale = mai.rope_table(case["theta"], case["rotary"], case["scaling"], **_scaling(case))
        s["table"] = torch.from_numpy(table.view(np.int64)).cuda()
        s["args"] = mai.paged_append(s["kv"], s["q"], s["new_k"], s["new_v"], s["q_out"], s["slot"],
                                     sequence=s["sequence"], position=s["position"], rope=s["table"],
                                     rotary_dim=case["rotary"], layout=case["layout"], rope_scale=scale)
    elif case["op"] == "evict":
        size = mai.paged_evict_workspace_bytes(s["kv"])
        s["work"] = torch.empty(max(size, 16), dtype=torch.uint8, device="cuda")
        s["args"] = mai.paged_evict(s["kv"], s["lengths_in"], s["lengths_out"], s["weights_in"], s["weights_out"],
                                    case["budget"], sink=case["sink"], recent=case["recent"], work=s["work"],
                                    positions_in=s["positions_in"], positions_out=s["positions_out"])
    else:
        size = mai.verify_drafts_workspace_bytes(case["batch"], case["vocab"])
        s["work"] = torch.empty(max(size, 16), dtype=torch.uint8, device="cuda")
        s["args"] = mai.verify_drafts(s["target"], s["tokens"], s["uniform"], s["last_uniform"], s["accepted"], s["next"],
                                      draft_probs=s["draft"], work=s["work"])


# ---- plain forms -----------------------------------------------------------
def _rows(s, slots):
    """Page and place within it of slots [sequence][n]; unused ones point at page 0."""
    page = s["case"]["page"]
    at = (slots // page).clamp(max=s["pages"].shape[1] - 1)
    return s["pages"].long().gather(1, at).clamp(min=0), slots % page


def _attend(s):
    case = s["case"]
    b, kv, g, hd, n = case["batch"], case["kv_heads"], case["group"], case["head_dim"], case["tokens"]
    slot = torch.arange(n, device="cuda").expand(b, n)
    pg, at = _rows(s, slot)
    keys = s["k"][pg, :, at].float().transpose(1, 2)      # [b][kv][n][hd]
    scores = torch.matmul(s["q"].float().view(b, kv, g, hd), keys.transpose(2, 3)) * hd ** -0.5
    del keys
    live = (slot < s["lengths"][:, None])[:, None, None, :]
    scores = scores.masked_fill(~live, -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=-3e38)  # an empty row has no maximum
    p = (scores - top).exp_()
    total = p.sum(-1, keepdim=True)
    p = torch.where(total > 0, p / total, 0.0)
    values = s["v"][pg, :, at].float().transpose(1, 2)
    s["out"].copy_(torch.matmul(p, values).reshape(b, kv * g, hd))
    if not case["weights"]:
        return {"out": s["out"]}
    more = p.sum(2)
    s["weights_out"].copy_(torch.where(live[:, :, 0], s["weights_in"] + more, s["weights_in"]))
    return {"out": s["out"], "weights": s["weights_out"]}


def _frequencies(case, theta, rotary):
    """Scaled angular frequencies in 64 bits [rotary / 2] and the factor on the rotated values."""
    i = torch.arange(rotary // 2, dtype=torch.float64, device="cuda")
    k = _scaling(case)
    base, scale = theta, 1.0
    if case["scaling"] == "ntk":
        base = theta * k["factor"] ** (rotary / (rotary - 2)) if rotary > 2 else theta
    f = base ** (-2.0 * i / rotary)
    if case["scaling"] == "linear":
        f = f / k["factor"]
    elif case["scaling"] == "yarn":
        turn = lambda r: rotary * math.log(k["original"] / (r * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
        lo, hi = max(math.floor(turn(k["beta_fast"])), 0), min(math.ceil(turn(k["beta_slow"])), rotary - 1)
        keep = 1 - ((i - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        f = f / k["factor"] * (1 - keep) + f * keep
        scale = 0.1 * math.log(k["factor"]) + 1.0
    elif case["scaling"] == "banded":
        wave = 2 * math.pi / f
        mix = ((k["original"] / wave - k["low"]) / (k["high"] - k["low"])).clamp(0, 1)
        f = f / k["factor"] * (1 - mix) + f * mix
    return f, scale


def _rotate(x, cos, sin, case):
    r = case["rotary"]
    y = x.clone()
    a, b = (slice(0, r, 2), slice(1, r, 2)) if case["layout"] == "interleaved" else (slice(0, r // 2), slice(r // 2, r))
    y[..., a] = x[..., a] * cos - x[..., b] * sin
    y[..., b] = x[..., a] * sin + x[..., b] * cos
    return y


def _append(s):
    case = s["case"]
    f, scale = _frequencies(case, case["theta"], case["rotary"])
    angle = s["position"].double()[:, None, None] * f     # 64 bits: far positions
    cos, sin = (angle.cos() * scale).float(), (angle.sin() * scale).float()
    s["q_out"].copy_(_rotate(s["q"].float(), cos, sin, case))
    seq, slot = s["sequence"].long(), s["slot"].long()
    pg, at = s["pages"].long()[seq, slot // case["page"]], slot % case["page"]
    s["k"][pg, :, at] = _rotate(s["new_k"].float(), cos, sin, case).to(s["k"].dtype)
    s["v"][pg, :, at] = s["new_v"].to(s["v"].dtype)
    return {"q": s["q_out"], "k": s["k"], "v": s["v"]}


def _evict(s):
    case = s["case"]
    n = s["lengths_in"].long()[:, None, None]
    m = n.clamp(max=case["budget"])
    slot = torch.arange(case["tokens"], device="cuda")
    live, pos = slot < n, s["positions_in"]
    held = (pos < case["sink"]) | (pos >= n - case["recent"])
    rank = torch.where(live & ~held, s["weights_in"], math.inf).sort(dim=-1, stable=True).indices
    gone = torch.zeros(rank.shape, dtype=torch.bool, device="cuda")
    gone.scatter_(2, rank, (slot < n - m).expand(rank.shape))  # the smallest, of equal ones the lowest slot
    hole, mover = gone & (slot < m), ~gone & live & (slot >= m)
    b, h, dst = hole.nonzero(as_tuple=True)              # both in order of sequence, head, slot
    src = mover.nonzero(as_tuple=True)[2]
    pages = s["pages"].long()
    to, of = (pages[b, dst // case["page"]], h, dst % case["page"]), (pages[b, src // case["page"]], h, src % case["page"])
    s["k"][to] = s["k"][of]
    s["v"][to] = s["v"][of]
    for name in ("weights", "positions"):
        got = torch.where(slot < m, s[name + "_in"], s[name + "_out"])
        got[b, h, dst] = s[name + "_in"][b, h, src]
        s[name + "_out"].copy_(got)
    s["lengths_out"].copy_(m.view(-1))
    return {"lengths": s["lengths_out"], "weights": s["weights_out"], "positions": s["positions_out"], "k": s["k"], "v": s["v"]}


def _verify(s):
    case = s["case"]
    k, b = case["drafts"], case["batch"]
    t = s["tokens"].long()[..., None]
    p = s["target"][:, :k].gather(2, t).squeeze(-1).double()
    q = s["draft"].gather(2, t).squeeze(-1).double() if case["draft_probs"] else torch.ones_like(p)
    ok = s["uniform"].double() * q < p                    # 64 bits: values next to a border
    taken = ok.long().cumprod(-1).sum(-1)
    row = torch.arange(b, device="cuda")
    rest = s["target"][row, taken].double()
    last = taken.clamp(max=k - 1)
    if case["draft_probs"]:
        minus = s["draft"][row, last].double()
    else:
        minus = torch.zeros_like(rest).scatter_(1, t[row, last], math.inf)
    plain = rest
    rest = torch.where((taken < k)[:, None], (rest - minus).clamp(min=0), rest)
    rest = torch.where(rest.sum(-1, keepdim=True) > 0, rest, plain)
    cdf = rest.cumsum(-1)
    at = s["last_uniform"].double()[:, None] * cdf[:, -1:]
    s["next"].copy_(torch.searchsorted(cdf, at, right=True).view(-1).clamp(max=case["vocab"] - 1))
    s["accepted"].copy_(taken)
    return {"accepted": s["accepted"], "next": s["next"]}


def run(state):
    op = state["case"]["op"]
    if own:
        _, ctx = _mai()
        if op == "attention":
            ctx.paged_attention_dev(state["kv"], state["args"], _stream())
            return {"out": state["out"], "weights": state["weights_out"]} if state["case"]["weights"] else {"out": state["out"]}
        if op == "append":
            ctx.paged_append_dev(state["kv"], state["args"], _stream())
            return {"q": state["q_out"], "k": state["k"], "v": state["v"]}
        if op == "evict":
            ctx.paged_evict_dev(state["kv"], state["args"], _stream())
            return {"lengths": state["lengths_out"], "weights": state["weights_out"], "positions": state["positions_out"],
                    "k": state["k"], "v": state["v"]}
        ctx.verify_drafts_dev(state["args"], _stream())
        return {"accepted": state["accepted"], "next": state["next"]}
    return {"attention": _attend, "append": _append, "evict": _evict, "verify": _verify}[op](state)


# ---- the definitions in 64 bits --------------------------------------------
def _cells(pages_row, n, page):
    """(page, place) of slots 0..n-1 of one sequence."""
    slot = torch.arange(n, device=pages_row.device)
    return pages_row.long()[slot // page], slot % page


def _exact_attention(case, s):
    kv, g = case["kv_heads"], case["group"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    weights = s["weights_in"].double() if case["weights"] else None
    for b, n in enumerate(_lengths(case)):
        if not n:
            continue
        pg, at = _cells(s["pages"][b], n, case["page"])
        for h in range(kv):
            q = s["q"][b, h * g:(h + 1) * g].double()
            p = torch.softmax(q @ s["k"][pg, h, at].double().T / math.sqrt(case["head_dim"]), -1)
            out[b, h * g:(h + 1) * g] = p @ s["v"][pg, h, at].double()
            if weights is not None:
                weights[b, h, :n] += p.sum(0)
    return {"out": out} if weights is None else {"out": out, "weights": weights}


def _exact_turns(case):
    """Radians a position of each rotated pair, one at a time, and the factor on them."""
    r, theta, k = case["rotary"], case["theta"], _scaling(case)
    got = []
    for i in range(0, r, 2):
        f = math.exp(-i / r * math.log(theta))
        if case["scaling"] == "linear":
            f /= k["factor"]
        elif case["scaling"] == "ntk" and r > 2:
            f = math.exp(-i / r * (math.log(theta) + r / (r - 2) * math.log(k["factor"])))
        elif case["scaling"] == "yarn":
            # pairs that turn more than beta_fast times over the original context stay, those under beta_slow stretch
            edge = [r / 2 * math.log(k["original"] / (2 * math.pi * b)) / math.log(theta) for b in (k["beta_fast"], k["beta_slow"])]
            lo, hi = max(0, math.floor(edge[0])), min(r - 1, math.ceil(edge[1]))
            ramp = min(1.0, max(0.0, (i / 2 - lo) / max(hi - lo, 0.001)))
            f = f * (1 - ramp) + f / k["factor"] * ramp
        elif case["scaling"] == "banded":
            turns = k["original"] * f / (2 * math.pi)
            if turns <= k["low"]:
                f /= k["factor"]
            elif turns < k["high"]:
                share = (turns - k["low"]) / (k["high"] - k["low"])
                f = share * f + (1 - share) * f / k["factor"]
        got.append(f)
    scale = 1 + math.log(k["factor"]) / 10 if case["scaling"] == "yarn" else 1.0
    return torch.tensor(got, dtype=torch.float64, device="cuda"), scale


def _exact_append(case, s):
    r, half = case["rotary"], case["rotary"] // 2
    f, scale = _exact_turns(case)
    turn = torch.polar(torch.full((case["tokens"], half), scale, dtype=torch.float64, device="cuda"),
                       s["position"].double()[:, None] * f)[:, None]

    def rotated(x):
        y = x.double().clone()
        if case["layout"] == "half":
            z = torch.complex(y[..., :half].clone(), y[..., half:r].clone()) * turn
            y[..., :r] = torch.cat([z.real, z.imag], -1)
        else:
            z = torch.view_as_complex(y[..., :r].reshape(*y.shape[:-1], half, 2).contiguous()) * turn
            y[..., :r] = torch.view_as_real(z).flatten(-2)
        return y

    k, v = s["k"].double(), s["v"].double()
    seq, slot = s["sequence"].long(), s["slot"].long()
    pg, at = s["pages"][seq, slot // case["page"]].long(), slot % case["page"]
    k[pg, :, at] = rotated(s["new_k"])
    v[pg, :, at] = s["new_v"].double()
    return {"q": rotated(s["q"]), "k": k, "v": v}


def _exact_evict(case, s):
    k, v = s["k"].clone(), s["v"].clone()
    w_in, p_in = s["weights_in"].cpu().numpy(), s["positions_in"].cpu().numpy()
    w_out, p_out = np.zeros_like(w_in, dtype=np.float64), np.zeros_like(p_in)
    kept = []
    for b, n in enumerate(_lengths(case)):
        m = min(n, case["budget"])
        kept.append(m)
        for h in range(case["kv_heads"]):
            w, p = w_in[b, h, :n].astype(np.float64), p_in[b, h, :n]
            free = np.flatnonzero((p >= case["sink"]) & (p < n - case["recent"]))
            gone = set(free[np.lexsort((free, w[free]))][:n - m].tolist())
            holes = sorted(i for i in gone if i < m)
            movers = [i for i in range(m, n) if i not in gone]
            w[holes], p[holes] = w[movers], p[movers]
            w_out[b, h, :m], p_out[b, h, :m] = w[:m], p[:m]
            if holes:
                pg, at = _cells(s["pages"][b], n, case["page"])
                a, c = torch.tensor(holes, device="cuda"), torch.tensor(movers, device="cuda")
                k[pg[a], h, at[a]] = s["k"][pg[c], h, at[c]]
                v[pg[a], h, at[a]] = s["v"][pg[c], h, at[c]]
    return {"lengths": torch.tensor(kept, dtype=torch.int32), "weights": torch.from_numpy(w_out),
            "positions": torch.from_numpy(p_out), "k": k.double(), "v": v.double()}


def _exact_verify(case, s):
    accepted, following = [], []
    for b in range(case["batch"]):
        n = 0
        while n < case["drafts"]:
            x = int(s["tokens"][b, n])
            q = float(s["draft"][b, n, x]) if case["draft_probs"] else 1.0
            if not float(s["uniform"][b, n]) * q < float(s["target"][b, n, x]):
                break
            n += 1
        p = s["target"][b, n].cpu().numpy().astype(np.float64)
        rest = p.copy()
        if n < case["drafts"]:
            if case["draft_probs"]:
                rest = np.maximum(p - s["draft"][b, n].cpu().numpy().astype(np.float64), 0)
            else:
                rest[int(s["tokens"][b, n])] = 0
        cdf = np.cumsum(rest if rest.sum() > 0 else p)
        following.append(min(int(np.searchsorted(cdf, float(s["last_uniform"][b]) * cdf[-1], side="right")), len(p) - 1))
        accepted.append(n)
    return {"accepted": torch.tensor(accepted, dtype=torch.int32), "next": torch.tensor(following, dtype=torch.int32)}


def exact(case, seed):
    s = prepare(case, seed)
    return {"attention": _exact_attention, "append": _exact_append, "evict": _exact_evict, "verify": _exact_verify}[case["op"]](case, s)
