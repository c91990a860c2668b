"""What the operators on a caller's paged cache are measured on: rotary positions (alone, and with the write of new keys and values to the cache), the
pages of a cache (forking, freeing and compacting, with the copies that follow) and decode attention of a batch whose sequences share prompts.

A cache is [planes, pages, key/value heads, 64 tokens, head size] in bf16, planes = K and V of every layer.  Sizes are those of the configurations in
csrc/config.hpp (heads 32 / 8 of 64 and 128, 40 / 8 and 64 / 8 of 128), of the batches in bench.py (128 conversations on a system prompt of about 1536
tokens, contexts up to 17 thousand) and ones beside them.  The plain forms are elementary torch operations in 32 bits (angles in 64)."""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

PAGE = 64
HALVES, INTERLEAVED = 1, 0
PLAIN, LINEAR, LLAMA3, YARN = 0, 1, 2, 3
# (base, factor, first, second, original length) of each scaling: llama3 takes the low and high frequency factors, YaRN the fast and slow turns
SCALINGS = {PLAIN: (10000.0, 1.0, 0.0, 0.0, 0), LINEAR: (10000.0, 4.0, 0.0, 0.0, 0), LLAMA3: (500000.0, 32.0, 1.0, 4.0, 8192), YARN: (1000000.0, 4.0, 32.0, 1.0, 32768)}


def listed() -> list[dict]:
    return [
        # one new token of six conversations (heads of 64), rotated and written to its pages: a call's latency
        {"name": "append_6", "kind": "append", "tokens": 6, "heads": 32, "kv_heads": 8, "dim": 64, "rot": 64, "layout": HALVES, "scaling": LLAMA3},
        # a full prefill step of 8192 tokens of a model with 32 / 8 heads of 128
        {"name": "append_prefill", "kind": "append", "tokens": 8192, "heads": 32, "kv_heads": 8, "dim": 128, "rot": 128, "layout": HALVES, "scaling": LLAMA3},
        # one agent's prompt through interleaved pairs of half of each head, 40 / 8 heads, scaled for long contexts
        {"name": "append_partial", "kind": "append", "tokens": 1337, "heads": 40, "kv_heads": 8, "dim": 128, "rot": 64, "layout": INTERLEAVED, "scaling": YARN},
        # the gradient of a rotated fp32 projection: the transposed rotation, an odd number of rows
        {"name": "rotary_grad", "kind": "rotary", "tokens": 2049, "heads": 32, "dim": 128, "rot": 96, "layout": HALVES, "scaling": LINEAR, "transpose": True, "f32": True},
        # four branches of one conversation, 16 layers with heads of 64: a table change and four tails of 20 tokens
        {"name": "fork_4", "kind": "fork", "length": 1556, "children": 4, "planes": 32, "kv_heads": 8, "dim": 64},
        # 64 conversations from one that holds the system prompt, 32 layers of a model with 8 heads of 128
        {"name": "fork_64", "kind": "fork", "length": 1585, "children": 64, "planes": 64, "kv_heads": 8, "dim": 128},
        # a third of the conversations has ended: their pages are freed and the others' moved together (eight layers)
        {"name": "compact", "kind": "compact", "rows": 48, "len_min": 300, "len_max": 1100, "planes": 16, "kv_heads": 8, "dim": 128},
        # four conversations early in their first answer, heads of 64: latency counts
        {"name": "prefix_4", "kind": "prefix", "groups": 1, "seqs": 4, "prefix_min": 700, "prefix_max": 700, "own_min": 1, "own_max": 90, "heads": 32, "kv_heads": 8, "dim": 64},
        # 128 conversations on one system prompt of 1536 tokens, each with its own history
        {"name": "prefix_128", "kind": "prefix", "groups": 1, "seqs": 128, "prefix_min": 1536, "prefix_max": 1536, "own_min": 64, "own_max": 512, "heads": 32, "kv_heads": 8, "dim": 128},
        # three system prompts of unequal length in one batch of 101, 40 / 8 heads: five heads a group, ragged everywhere
        {"name": "prefix_mix", "kind": "prefix", "groups": 3, "seqs": 101, "prefix_min": 900, "prefix_max": 2500, "own_min": 1, "own_max": 700, "heads": 40, "kv_heads": 8, "dim": 128},
        # 64 questions to one document of 16 thousand tokens, 64 / 8 heads
        {"name": "prefix_long", "kind": "prefix", "groups": 1, "seqs": 64, "prefix_min": 16384, "prefix_max": 16384, "own_min": 20, "own_max": 600, "heads": 64, "kv_heads": 8, "dim": 128},
        # eight conversations that have grown long beyond their common prompt
        {"name": "prefix_far", "kind": "prefix", "groups": 1, "seqs": 8, "prefix_min": 1000, "prefix_max": 1000, "own_min": 4000, "own_max": 9000, "heads": 32, "kv_heads": 8, "dim": 128},
    ]


def _log(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))))


def draw(rng) -> dict:
    kind = rng.choice(["append", "rotary", "fork", "compact", "prefix", "prefix", "prefix"])
    heads, kv_heads, dim = rng.choice([(32, 8, 64), (32, 8, 128), (40, 8, 128), (64, 8, 128), (24, 8, 64), (12, 12, 64), (28, 4, 128), (8, 1, 64)])
    rotation = {"rot": rng.choice([dim, dim, dim // 2, dim // 4, dim - 32]), "layout": rng.choice([HALVES, INTERLEAVED]), "scaling": rng.choice(list(SCALINGS))}
    if kind == "append":
        return {"kind": kind, "tokens": _log(rng, 1, 8192 * 32 * 128 // (max(32, heads) * 128)), "heads": heads, "kv_heads": kv_heads, "dim": dim, **rotation}
    if kind == "rotary":
        f32 = rng.random() < 0.5
        return {"kind": kind, "tokens": _log(rng, 1, 4000), "heads": heads, "dim": dim, **rotation, "transpose": rng.random() < 0.5, "f32": f32}
    if kind == "fork":
        return {"kind": kind, "length": _log(rng, 1, 2500), "children": _log(rng, 1, 64), "planes": 2 * rng.randint(1, 32), "kv_heads": min(8, kv_heads), "dim": dim}
    if kind == "compact":
        top = _log(rng, 40, 1100)
        return {"kind": kind, "rows": _log(rng, 2, 48), "len_min": max(1, top // rng.choice([1, 3, 8])), "len_max": top, "planes": 2 * rng.randint(1, 8), "kv_heads": min(8, kv_heads), "dim": dim}
    seqs = _log(rng, 1, 160)
    groups = min(seqs, rng.choice([1, 1, 1, 2, 3, 7]))
    prefix = _log(rng, 1, min(16384, 64 * 64 * 16384 // (seqs * heads * groups)))
    ours = _log(rng, 1, max(1, min(9000, 60000 // seqs)))
    return {"kind": kind, "groups": groups, "seqs": seqs, "prefix_min": max(1, prefix // rng.choice([1, 1, 3])), "prefix_max": prefix,
            "own_min": max(1, ours // rng.choice([1, 4, 30])), "own_max": ours, "heads": heads, "kv_heads": kv_heads, "dim": dim}


# ---- inputs ------------------------------------------------------------------------------------------------------------------------------

def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, shape, dtype=torch.bfloat16):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _cache(g, planes, pages, kv_heads, dim):
    """Pages of a cache in use: nothing in it is zero, places behind a sequence's end hold what an earlier one left."""
    out = torch.empty((planes, pages, kv_heads, PAGE, dim), dtype=torch.bfloat16, device="cuda")
    for part in out.view(planes * pages, -1).split(4096):
        part.copy_(torch.randn(part.shape, generator=g, device="cuda"))
    return out


def _spread(case, lo, hi, n, seed) -> np.ndarray:
    """Ragged lengths: the same ones for every seed, in another order, so that outputs have one shape and calls one size."""
    return np.random.default_rng(seed).permutation(np.random.default_rng(n).integers(case[lo], case[hi] + 1, n)).astype(np.int32)


def _rotary_inputs(case, seed):
    g, rng, t, dim = _gen(seed), np.random.default_rng(seed), case["tokens"], case["dim"]
    start = int(rng.integers(0, 16000))
    positions = torch.from_numpy((start + np.arange(t)).astype(np.int32)).cuda()
    if case["kind"] == "rotary":
        x = _normal(g, (t, case["heads"], dim), torch.float32 if case["f32"] else torch.bfloat16)
        return {"x": x, "positions": positions}
    width = (case["heads"] + 2 * case["kv_heads"]) * dim
    pages = (t + PAGE - 1) // PAGE + 3
    order = rng.permutation(pages)
    at = int(rng.integers(0, PAGE)) + np.arange(t)                       # the first new token lies anywhere in its page
    slots = (order[at // PAGE] * PAGE + at % PAGE).astype(np.int32)
    return {"qkv": _normal(g, (t, width)), "positions": positions, "slots": torch.from_numpy(slots).cuda(), "cache": _cache(g, 2, pages, case["kv_heads"], dim)}


def _pages_of(length):
    return (int(length) + PAGE - 1) // PAGE


def _fork_inputs(case, seed):
    rng, n = np.random.default_rng(seed), _pages_of(case["length"])
    pages = n + case["children"] + 5
    tables = np.full((case["children"] + 1, n + 4), -1, np.int32)
    refs = np.zeros(pages, np.int32)
    held = rng.permutation(pages)[:n].astype(np.int32)
    tables[0, :n], refs[held] = held, 1
    lens = np.zeros(case["children"] + 1, np.int32)
    lens[0] = case["length"]
    return {"tables": tables, "lens": lens, "refs": refs, "pages": pages, "cache": _cache(_gen(seed), case["planes"], pages, case["kv_heads"], case["dim"])}


def _compact_inputs(case, seed):
    rng = np.random.default_rng(seed)
    lens = _spread(case, "len_min", "len_max", case["rows"], seed)
    need = (lens + PAGE - 1) // PAGE
    pages, width = int(need.sum()) + 3, int(need.max()) + 1
    order = rng.permutation(pages).astype(np.int32)
    tables = np.full((case["rows"], width), -1, np.int32)
    inside = np.arange(width)[None, :] < need[:, None]
    tables[inside] = order[: int(need.sum())]
    refs = np.zeros(pages, np.int32)
    refs[tables[inside]] = 1
    ended = np.sort(rng.permutation(case["rows"])[: (case["rows"] + 2) // 3]).astype(np.int32)
    return {"tables": tables, "lens": lens, "refs": refs, "pages": pages, "ended": ended, "cache": _cache(_gen(seed), case["planes"], pages, case["kv_heads"], case["dim"])}


def _group_rows(case) -> np.ndarray:
    """Where each prefix's rows begin: 40 %, 30 %, ... as the mix of requests has them, each at least one row."""
    weights = 1.0 / np.arange(1, case["groups"] + 1)
    cuts = np.round(np.cumsum(weights) / weights.sum() * (case["seqs"] - case["groups"])).astype(np.int64)
    return np.concatenate([[0], cuts + np.arange(1, case["groups"] + 1)]).astype(np.int32)


def _prefix_inputs(case, seed):
    g, rng, n = _gen(seed), np.random.default_rng(seed), case["groups"]
    prefix, ours = _spread(case, "prefix_min", "prefix_max", n, seed), _spread(case, "own_min", "own_max", case["seqs"], seed)
    need = np.concatenate([(prefix + PAGE - 1) // PAGE, (ours + PAGE - 1) // PAGE])
    pages = int(need.sum()) + 2
    order = rng.permutation(pages).astype(np.int32)                      # pages of a cache in use lie anywhere
    first = np.concatenate([[0], np.cumsum(need)])[:-1]
    widest = [int(need[:n].max()), int(need[n:].max()) + 1]
    tables = [np.zeros((n, widest[0]), np.int32), np.zeros((case["seqs"], widest[1]), np.int32)]
    for i, (at, k) in enumerate(zip(first, need)):
        tables[i >= n][i - (n if i >= n else 0), :k] = order[at:at + k]
    cache = _cache(g, 2, pages, case["kv_heads"], case["dim"])
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    q = _normal(g, (case["seqs"], case["heads"], case["dim"]))
    heads = torch.zeros((n, case["kv_heads"], case["dim"]), device="cuda").normal_(generator=g)
    cache[0, dev(tables[0][:, 0]).long(), :, 0] = (2.0 * heads).bfloat16()    # a prompt's first token, which rows look at more than at others
    q += 0.25 * heads[0].bfloat16().repeat_interleave(case["heads"] // case["kv_heads"], 0)[None]
    return {"q": q, "cache": cache, "pages": pages, "prefix_tables": dev(tables[0]), "prefix_lens": dev(prefix), "prefix_rows": dev(_group_rows(case)),
            "own_tables": dev(tables[1]), "own_lens": dev(ours)}


def prepare(case: dict, seed: int) -> dict:
    kind = case["kind"]
    make = {"append": _rotary_inputs, "rotary": _rotary_inputs, "fork": _fork_inputs, "compact": _compact_inputs, "prefix": _prefix_inputs}[kind]
    s = {"case": case, **make(case, seed)}
    if kind in ("append", "rotary"):                                     # frequencies are a model's: made once, in 64 bits
        s["freqs"], s["amplitude"] = _frequencies(case["rot"], case["scaling"])
        s["freqs_gpu"] = torch.from_numpy(s["freqs"]).cuda()
    if kind == "append":
        s["q_out"] = torch.empty((case["tokens"], case["heads"], case["dim"]), dtype=torch.bfloat16, device="cuda")
    if kind == "rotary":
        s["out"] = torch.empty_like(s["x"])
    if kind == "prefix":
        s["out"] = torch.empty_like(s["q"])
    return s


def _frequencies(dims, scaling):
    base, factor, first, second, original = SCALINGS[scaling]
    i = np.arange(dims // 2, dtype=np.float64)
    f = base ** (-2.0 * i / dims)
    if scaling == LINEAR:
        return f / factor, 1.0
    if scaling == LLAMA3:
        share = np.clip((original * f / (2 * np.pi) - first) / (second - first), 0.0, 1.0)
        return f * (share + (1 - share) / factor), 1.0
    if scaling == YARN:
        where = lambda t: dims * math.log(original / (2 * math.pi * t)) / (2 * math.log(base))  # noqa: E731
        lo, hi = max(math.floor(where(first)), 0), min(math.ceil(where(second)), dims - 1)
        ramp = np.clip((i - lo) / max(hi - lo, 0.001), 0.0, 1.0)
        return f / factor * ramp + f * (1 - ramp), 0.1 * math.log(factor) + 1.0
    return f, 1.0


# ---- one pass ----------------------------------------------------------------------------------------------------------------------------

def _rotate(x, positions, freqs, amplitude, layout, transpose=False):
    """x [tokens, heads, dim], the first 2 len(freqs) channels of each head rotated; in 32 bits, angles in 64."""
    half = freqs.numel()
    angle = positions.double()[:, None] * freqs
    cos, sin = (angle.cos() * amplitude).float()[:, None], (angle.sin() * amplitude).float()[:, None]
    sin = -sin if transpose else sin
    y = x.float()
    a, b = (y[..., :half], y[..., half:2 * half]) if layout == HALVES else (y[..., 0:2 * half:2], y[..., 1:2 * half:2])
    a, b = a * cos - b * sin, a * sin + b * cos
    turned = torch.cat([a, b], -1) if layout == HALVES else torch.stack([a, b], -1).flatten(-2)
    return torch.cat([turned, y[..., 2 * half:]], -1).to(x.dtype)


def _plain_append(s):
    case, slots = s["case"], s["slots"].long()
    q, k, v = s["qkv"].view(case["tokens"], -1, case["dim"]).split([case["heads"], case["kv_heads"], case["kv_heads"]], 1)
    s["q_out"].copy_(_rotate(q, s["positions"], s["freqs_gpu"], s["amplitude"], case["layout"]))
    page, place = slots // PAGE, slots % PAGE
    s["cache"][0][page, :, place] = _rotate(k, s["positions"], s["freqs_gpu"], s["amplitude"], case["layout"])
    s["cache"][1][page, :, place] = v
    return {"q": s["q_out"], "cache": s["cache"]}


def _plain_fork(s):
    length, children = s["case"]["length"], s["case"]["children"]
    tables, lens, refs = s["tables"].copy(), s["lens"].copy(), s["refs"].copy()
    full, tail = length // PAGE, length % PAGE
    tables[1:, :full] = tables[0, :full]
    refs[tables[0, :full]] += children
    lens[1:] = length
    if tail:
        fresh = np.flatnonzero(refs == 0)[:children].astype(np.int32)
        tables[1:, full], refs[fresh] = fresh, 1
        s["cache"][:, torch.from_numpy(fresh).long().cuda(), :, :tail] = s["cache"][:, int(tables[0, full]), :, :tail].unsqueeze(1)
    return {"cache": s["cache"], "tables": tables, "lens": lens, "refs": refs}


def _plain_compact(s):
    tables, lens, refs = s["tables"].copy(), s["lens"].copy(), s["refs"].copy()
    gone = tables[s["ended"]]
    np.subtract.at(refs, gone[gone >= 0], 1)
    tables[s["ended"]], lens[s["ended"]] = -1, 0
    used = np.flatnonzero(refs > 0)
    high = used[used >= used.size]
    low = np.flatnonzero(refs[: used.size] == 0)
    s["cache"][:, torch.from_numpy(low).cuda()] = s["cache"][:, torch.from_numpy(high).cuda()]
    to = np.arange(refs.size + 1, dtype=np.int32)
    to[-1], to[high] = -1, low                                           # the last entry stands for places without a page
    refs[low], refs[high] = refs[high], 0
    return {"cache": s["cache"], "tables": to[tables], "lens": lens, "refs": refs}


def _plain_prefix(s):
    case = s["case"]
    t, nkv, dim, group = case["seqs"], case["kv_heads"], case["dim"], case["heads"] // case["kv_heads"]
    q = s["q"].float().view(t, nkv, group, dim) / math.sqrt(dim)
    which = (torch.arange(t, device="cuda")[:, None] >= s["prefix_rows"][None, 1:]).sum(1)            # a row's prefix
    place = torch.arange(t, device="cuda") - s["prefix_rows"].long()[which]
    padded = torch.zeros((case["groups"], t, nkv, group, dim), device="cuda")
    padded[which, place] = q
    take = lambda plane, tables: s["cache"][plane][tables.long()].transpose(2, 3).flatten(1, 2).float()  # noqa: E731
    inside = lambda tables, lens: torch.arange(tables.shape[1] * PAGE, device="cuda")[None] < lens[:, None]  # noqa: E731
    far = torch.einsum("gtkhd,gpkd->gtkhp", padded, take(0, s["prefix_tables"]))
    far = far.masked_fill(~inside(s["prefix_tables"], s["prefix_lens"])[:, None, None, None], -math.inf)[which, place]
    near = torch.einsum("tkhd,tpkd->tkhp", q, take(0, s["own_tables"]))
    near = near.masked_fill(~inside(s["own_tables"], s["own_lens"])[:, None, None], -math.inf)
    top = torch.maximum(far.amax(-1, keepdim=True), near.amax(-1, keepdim=True))
    far, near = (far - top).exp(), (near - top).exp()
    total = far.sum(-1, keepdim=True) + near.sum(-1, keepdim=True)
    padded = torch.zeros((case["groups"], t, nkv, group, far.shape[-1]), device="cuda")
    padded[which, place] = far
    out = torch.einsum("gtkhp,gpkd->gtkhd", padded, take(1, s["prefix_tables"]))[which, place]
    out = (out + torch.einsum("tkhp,tpkd->tkhd", near, take(1, s["own_tables"]))) / total
    s["out"].copy_(out.view(t, -1, dim))
    return {"out": s["out"]}


def _ok(rc):
    if rc != 0:
        raise RuntimeError(f"call failed ({rc})")


def _own_append(s, lib, stream):
    case, row = s["case"], s["qkv"].shape[1]
    q = s["qkv"].data_ptr()
    k = q + 2 * case["heads"] * case["dim"]
    _ok(lib.oa_k_rotary_cache(q, row, k, k + 2 * case["kv_heads"] * case["dim"], row, s["q_out"].data_ptr(), case["heads"] * case["dim"], s["cache"].data_ptr(), s["cache"].shape[1],
                              s["positions"].data_ptr(), s["slots"].data_ptr(), case["tokens"], case["heads"], case["kv_heads"], case["dim"], case["rot"], case["layout"],
                              s["freqs"].ctypes.data, s["amplitude"], None, stream))
    return {"q": s["q_out"], "cache": s["cache"]}


def _own_pages(s, lib, stream):
    from opsagent_b200 import _lib
    case = s["case"]
    tables, lens, refs = s["tables"].copy(), s["lens"].copy(), s["refs"].copy()
    table = _lib.OaPageTable(tables.ctypes.data, lens.ctypes.data, refs.ctypes.data, tables.shape[0], tables.shape[1], s["pages"])
    moves = (_lib.OaPageMove * s["pages"])()
    n = _lib.C.c_int32()
    if case["kind"] == "fork":
        children = np.arange(1, case["children"] + 1, dtype=np.int32)
        _ok(lib.oa_host_cache_fork(table, 0, children.ctypes.data, children.size, moves, s["pages"], n))
    else:
        _ok(lib.oa_host_cache_free(table, s["ended"].ctypes.data, s["ended"].size))
        _ok(lib.oa_host_cache_compact(table, moves, s["pages"], n))
    _ok(lib.oa_k_cache_copy(s["cache"].data_ptr(), case["planes"], s["pages"], case["kv_heads"], case["dim"], 2, moves, n.value, stream))
    return {"cache": s["cache"], "tables": tables, "lens": lens, "refs": refs}


def _own_prefix(s, lib, stream):
    case = s["case"]
    width = case["heads"] * case["dim"]
    _ok(lib.oa_k_prefix_attention(s["q"].data_ptr(), width, s["out"].data_ptr(), width, s["cache"].data_ptr(), s["pages"], s["prefix_tables"].data_ptr(), s["prefix_tables"].shape[1],
                                  s["prefix_lens"].data_ptr(), s["prefix_rows"].data_ptr(), case["groups"], s["own_tables"].data_ptr(), s["own_tables"].shape[1],
                                  s["own_lens"].data_ptr(), case["seqs"], case["heads"], case["kv_heads"], case["dim"], 0.0, None, stream))
    return {"out": s["out"]}


def run(state: dict):
    case = state["case"]
    kind = case["kind"]
    if own:
        from opsagent_b200 import _lib
        lib, stream = _lib.load(), torch.cuda.current_stream().cuda_stream
        if kind == "append":
            return _own_append(state, lib, stream)
        if kind == "rotary":
            width = case["heads"] * case["dim"]
            _ok(lib.oa_k_rotary(state["x"].data_ptr(), width, state["out"].data_ptr(), width, state["positions"].data_ptr(), case["tokens"], case["heads"], case["dim"], case["rot"],
                                case["layout"], state["freqs"].ctypes.data, state["amplitude"], case["transpose"], case["f32"], stream))
            return {"out": state["out"]}
        return _own_prefix(state, lib, stream) if kind == "prefix" else _own_pages(state, lib, stream)
    if kind == "rotary":
        state["out"].copy_(_rotate(state["x"], state["positions"], state["freqs_gpu"], state["amplitude"], case["layout"], case["transpose"]))
        return {"out": state["out"]}
    return {"append": _plain_append, "fork": _plain_fork, "compact": _plain_compact, "prefix": _plain_prefix}[kind](state)


# ---- what a pass cannot do without -------------------------------------------------------------------------------------------------------

def work(case: dict) -> dict:
    kind, dim = case["kind"], case["dim"]
    if kind == "append":
        t, nh, nkv = case["tokens"], case["heads"], case["kv_heads"]
        return {"bytes": 4 * t * (nh + 2 * nkv) * dim + 8 * t, "flops": 3 * t * (nh + nkv) * case["rot"]}
    if kind == "rotary":
        t, nh = case["tokens"], case["heads"]
        return {"bytes": (8 if case["f32"] else 4) * t * nh * dim + 4 * t, "flops": 3 * t * nh * case["rot"]}
    row = 2 * case["kv_heads"] * dim                                     # bytes of a token's keys or values
    if kind == "fork":                                                   # the parent's tail once, and a copy of it for every child; the children's rows of the table
        tail = case["length"] % PAGE
        return {"bytes": (1 + case["children"]) * (case["planes"] * tail * row + 4 * _pages_of(case["length"])), "flops": 0}
    if kind == "compact":
        lens = _spread(case, "len_min", "len_max", case["rows"], 0)
        need = (lens + PAGE - 1) // PAGE
        kept = need.sum() * 2 / 3                                        # on average: which rows have ended differs by seed
        return {"bytes": int(2 * case["planes"] * PAGE * row * kept / 3 + 8 * need.sum()), "flops": 0}
    prefix, ours = _spread(case, "prefix_min", "prefix_max", case["groups"], 0), _spread(case, "own_min", "own_max", case["seqs"], 0)
    keys = int(ours.sum()) + int((np.diff(_group_rows(case)) * prefix.mean()).sum())
    return {"bytes": 2 * row * (int(prefix.sum()) + int(ours.sum())) + 4 * case["seqs"] * case["heads"] * dim, "flops": 4 * case["heads"] * dim * keys}


# ---- the same in 64 bits -----------------------------------------------------------------------------------------------------------------

def _turned(x, positions, case, transpose):
    """Each pair of channels as a complex number, times amplitude e^(i angle)."""
    f, amplitude = _frequencies(case["rot"], case["scaling"])
    angle = positions.double()[:, None] * torch.from_numpy(f).cuda() * (-1.0 if transpose else 1.0)
    r, y = case["rot"], x.double().clone()
    pairs = y[..., :r].unflatten(-1, (2, r // 2)).transpose(-1, -2) if case["layout"] == HALVES else y[..., :r].unflatten(-1, (r // 2, 2))
    z = torch.view_as_complex(pairs.contiguous()) * torch.polar(torch.full_like(angle, amplitude), angle)[:, None]
    z = torch.view_as_real(z)
    y[..., :r] = (z.transpose(-1, -2) if case["layout"] == HALVES else z).flatten(-2)
    return y


def exact(case: dict, seed: int):
    kind = case["kind"]
    if kind in ("fork", "compact"):                                      # copies: their bits are held to the plain form's
        return None
    if kind == "rotary":
        t = _rotary_inputs(case, seed)
        return {"out": _turned(t["x"], t["positions"], case, case["transpose"])}
    if kind == "append":
        t = _rotary_inputs(case, seed)
        x = t["qkv"].view(case["tokens"], -1, case["dim"])
        nh, nkv = case["heads"], case["kv_heads"]
        cache = t["cache"].double()
        rows = cache.transpose(2, 3).reshape(2, -1, nkv, case["dim"])    # [plane, page and place, head, channel]
        rows[0, t["slots"].long()] = _turned(x[:, nh:nh + nkv], t["positions"], case, False)
        rows[1, t["slots"].long()] = x[:, nh + nkv:].double()
        return {"q": _turned(x[:, :nh], t["positions"], case, False), "cache": rows.view(2, -1, PAGE, nkv, case["dim"]).transpose(2, 3).contiguous()}
    t = _prefix_inputs(case, seed)
    rows, out = t["prefix_rows"].tolist(), torch.empty(t["q"].shape, dtype=torch.float64, device="cuda")
    lens, prefix, nkv, dim = t["own_lens"].tolist(), t["prefix_lens"].tolist(), case["kv_heads"], case["dim"]
    flat = lambda plane, pages, n: t["cache"][plane, pages.long()].double().transpose(1, 2).reshape(-1, nkv, dim)[:n]  # noqa: E731
    for g in range(case["groups"]):
        k0, v0 = (flat(i, t["prefix_tables"][g], prefix[g]) for i in (0, 1))
        for i in range(rows[g], rows[g + 1]):
            k, v = (torch.cat([x, flat(j, t["own_tables"][i], lens[i])]) for j, x in ((0, k0), (1, v0)))
            q = t["q"][i].double().view(nkv, -1, dim)
            p = torch.softmax(torch.einsum("khd,pkd->khp", q, k) / math.sqrt(dim), -1)
            out[i] = torch.einsum("khp,pkd->khd", p, v).reshape(-1, dim)
    return {"out": out}
