"""What the operators on 8-bit caches and on drafted tokens are measured on: keys and values stored in 8 bits as they are written, read back, their pages
copied, and attention of several new tokens of each sequence (one, a chain, a tree of drafts) over a cache of bf16 or 8 bits, with or without a sliding window.

An 8-bit cache is [planes, pages, key/value heads] blocks of 64 tokens: 64 x head size values of one byte (e4m3 or int8), then the 64 tokens' scales in fp32; planes
are K and V of every layer.  A value stands for itself times its token's scale, and a scale is the largest magnitude of the token's head over 448 (e4m3) or 127 (int8).
Sizes are those of the configurations in csrc/config.hpp (heads 32 / 8 of 64 and 128, 40 / 8 and 64 / 8 of 128), of the batches in bench.py (128 conversations, contexts up to 17
thousand) and ones beside them.  The plain forms are elementary torch operations in 32 bits."""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

PAGE = 64
BF16, E4M3, INT8 = 0, 1, 2
LIMIT = {E4M3: 448.0, INT8: 127.0}


def listed() -> list[dict]:
    return [
        # one new token of six conversations, heads of 64: a call's latency
        {"name": "write_6", "kind": "write", "tokens": 6, "kv_heads": 8, "dim": 64, "format": INT8},
        # a full prefill step of 8192 tokens, 8 heads of 128
        {"name": "write_prefill", "kind": "write", "tokens": 8192, "kv_heads": 8, "dim": 128, "format": E4M3},
        # one agent's prompt, read back for a layer that works on bf16 rows
        {"name": "read_prompt", "kind": "read", "tokens": 1337, "kv_heads": 8, "dim": 64, "format": E4M3},
        # a long document read back whole
        {"name": "read_document", "kind": "read", "tokens": 50001, "kv_heads": 8, "dim": 128, "format": INT8},
        # four branches of one conversation, 16 layers with heads of 64: four tails of 20 tokens
        {"name": "copy_fork", "kind": "copy", "moves": 4, "tokens": 20, "sources": 1, "planes": 32, "kv_heads": 8, "dim": 64},
        # whole pages moved together in 32 layers of 8 heads of 128
        {"name": "copy_pages", "kind": "copy", "moves": 100, "tokens": 64, "sources": 100, "planes": 64, "kv_heads": 8, "dim": 128},
        # six conversations whose next three tokens are guessed, heads of 64: latency counts
        {"name": "draft_6", "kind": "tree", "seqs": 6, "new_min": 4, "new_max": 4, "ctx_min": 300, "ctx_max": 1556, "heads": 32, "kv_heads": 8, "dim": 64, "format": INT8,
         "chain": True, "window": 0, "sinks": 0},
        # an ordinary decoding step of 128 conversations, one new token each, over a cache of 8 bits
        {"name": "decode_128", "kind": "tree", "seqs": 128, "new_min": 1, "new_max": 1, "ctx_min": 600, "ctx_max": 2500, "heads": 32, "kv_heads": 8, "dim": 128, "format": E4M3,
         "chain": True, "window": 0, "sinks": 0},
        # trees of 64 drafted tokens behind eight conversations
        {"name": "tree_64", "kind": "tree", "seqs": 8, "new_min": 64, "new_max": 64, "ctx_min": 2000, "ctx_max": 8000, "heads": 32, "kv_heads": 8, "dim": 128, "format": BF16,
         "chain": False, "window": 0, "sinks": 0},
        # unequal trees in one batch, 40 / 8 heads: five heads a group, ragged everywhere
        {"name": "tree_mix", "kind": "tree", "seqs": 21, "new_min": 3, "new_max": 40, "ctx_min": 100, "ctx_max": 6000, "heads": 40, "kv_heads": 8, "dim": 128, "format": E4M3,
         "chain": False, "window": 0, "sinks": 0},
        # a tree of 25 behind one document of a hundred thousand tokens, 64 / 8 heads
        {"name": "tree_long", "kind": "tree", "seqs": 1, "new_min": 25, "new_max": 25, "ctx_min": 100001, "ctx_max": 100001, "heads": 64, "kv_heads": 8, "dim": 128, "format": INT8,
         "chain": False, "window": 0, "sinks": 0},
        # a layer with a window of 4096 tokens and four first ones that stay visible, chains of 8 far into 16 conversations
        {"name": "window_far", "kind": "tree", "seqs": 16, "new_min": 8, "new_max": 8, "ctx_min": 9000, "ctx_max": 30000, "heads": 32, "kv_heads": 8, "dim": 128, "format": BF16,
         "chain": True, "window": 4096, "sinks": 4},
    ]


def _log(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))))


def draw(rng) -> dict:
    kind = rng.choice(["write", "read", "copy", "tree", "tree", "tree", "tree"])
    heads, kv_heads, dim = rng.choice([(32, 8, 64), (32, 8, 128), (40, 8, 128), (64, 8, 128), (12, 12, 64), (28, 4, 128), (8, 1, 64), (32, 2, 128)])
    fmt = rng.choice([E4M3, INT8])
    if kind in ("write", "read"):
        most = (8192 if kind == "write" else 50001) * 8 * 128 // (max(8, kv_heads) * 128)
        return {"kind": kind, "tokens": _log(rng, 1, most), "kv_heads": kv_heads, "dim": dim, "format": fmt}
    if kind == "copy":
        moves = _log(rng, 1, 100)
        return {"kind": kind, "moves": moves, "tokens": rng.choice([64, rng.randint(1, 64)]), "sources": rng.choice([1, moves]), "planes": 2 * rng.randint(1, 32), "kv_heads": min(8, kv_heads), "dim": dim}
    seqs = _log(rng, 1, 128)
    new = _log(rng, 1, min(64, max(1, 512 * 32 // (seqs * heads))))
    ctx = _log(rng, 1, min(100001, 128 * 1550 // seqs, 8 * 64 * 32 * 5000 // (seqs * new * heads)))
    window = rng.choice([0, 0, 0, _log(rng, 64, 4096)])
    return {"kind": kind, "seqs": seqs, "new_min": max(1, new // rng.choice([1, 1, 4])), "new_max": new, "ctx_min": max(1, ctx // rng.choice([1, 3, 30])), "ctx_max": ctx,
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "format": rng.choice([BF16, E4M3, INT8]), "chain": rng.random() < 0.4, "window": window,
            "sinks": rng.choice([0, 4, 70]) if window else 0}


# ---- inputs ------------------------------------------------------------------------------------------------------------------------------

def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, shape, dtype=torch.bfloat16):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _quantised(x, fmt):
    """x [..., head size] -> its bytes, and the scales of its rows in fp32.  A row with an infinity or a NaN keeps nothing: scale NaN."""
    x = x.float()
    top = x.abs().amax(-1)
    scale = top / torch.full((), LIMIT[fmt], device=x.device)           # a tensor: a division, not a product with a reciprocal
    bad = ~torch.isfinite(top)
    y = torch.where((scale > 0).logical_and(~bad)[..., None], x / scale[..., None], torch.zeros((), device=x.device)).clamp(-LIMIT[fmt], LIMIT[fmt])
    y = y.to(torch.float8_e4m3fn).view(torch.uint8) if fmt == E4M3 else y.round().to(torch.int8).view(torch.uint8)
    return y, scale.masked_fill(bad, math.nan)


def _bytes_of(cache, dim):
    return cache[..., : PAGE * dim].unflatten(-1, (PAGE, dim))


def _values_of(cache, dim, fmt):
    return _bytes_of(cache, dim).view(torch.float8_e4m3fn if fmt == E4M3 else torch.int8)


def _scales_of(cache, dim):
    return cache[..., PAGE * dim:].view(torch.float32)


def _cache(g, planes, pages, kv_heads, dim, fmt):
    """Pages of a cache in use: nothing in it is zero, places behind a sequence's end hold what an earlier one left."""
    if fmt == BF16:
        out = torch.empty((planes, pages, kv_heads, PAGE, dim), dtype=torch.bfloat16, device="cuda")
        for part in out.view(planes * pages, -1).split(2048):
            part.copy_(torch.randn(part.shape, generator=g, device="cuda"))
        return out
    out = torch.empty((planes, pages, kv_heads, PAGE * (dim + 4)), dtype=torch.uint8, device="cuda")
    for part in out.view(planes * pages, kv_heads, -1).split(2048):
        y, scale = _quantised(torch.randn((part.shape[0], kv_heads, PAGE, dim), generator=g, device="cuda"), fmt)
        _bytes_of(part, dim).copy_(y)
        _scales_of(part, dim).copy_(scale)
    return out


def _spread(case, lo, hi, n, seed) -> np.ndarray:
    """Ragged lengths: the same ones for every seed, in another order, so that outputs have one shape and calls one size."""
    return np.random.default_rng(seed).permutation(np.random.default_rng(n + case[hi]).integers(case[lo], case[hi] + 1, n)).astype(np.int32)


def _dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _row_inputs(case, seed):
    g, rng, t = _gen(seed), np.random.default_rng(seed), case["tokens"]
    pages = (t + PAGE - 1) // PAGE + 3
    at = int(rng.integers(0, PAGE)) + np.arange(t)                       # the first token lies anywhere in its page
    slots = (rng.permutation(pages)[at // PAGE] * PAGE + at % PAGE).astype(np.int32)
    return {"kv": _normal(g, (t, 2, case["kv_heads"], case["dim"])), "slots": _dev(slots), "cache": _cache(g, 2, pages, case["kv_heads"], case["dim"], case["format"])}


def _copy_inputs(case, seed):
    rng = np.random.default_rng(seed)
    pages = case["moves"] + case["sources"] + 3
    order = rng.permutation(pages).astype(np.int32)
    moves = np.empty((case["moves"], 3), np.int32)
    moves[:, 0], moves[:, 1], moves[:, 2] = order[np.arange(case["moves"]) % case["sources"]], order[case["sources"]:case["sources"] + case["moves"]], case["tokens"]
    return {"moves": moves, "pages": pages, "cache": _cache(_gen(seed), case["planes"], pages, case["kv_heads"], case["dim"], INT8)}


def _trees(case, new, rng):
    """Who sees whom among a sequence's new tokens: bit u of a token's number is set where it sees token u, its ancestors and itself."""
    seen = []
    for n in new:
        rows = []
        for t in range(int(n)):
            parent = t - 1 if case["chain"] or t < 2 else int(rng.integers(max(0, t - 9), t))
            rows.append((rows[parent] if t else 0) | 1 << t)
        seen += rows
    return np.array(seen, np.uint64).view(np.int64)


def _tree_inputs(case, seed):
    g, rng, n = _gen(seed), np.random.default_rng(seed), case["seqs"]
    new, ctx = _spread(case, "new_min", "new_max", n, seed), _spread(case, "ctx_min", "ctx_max", n, seed + 1)
    need = (ctx + new + PAGE - 1) // PAGE
    pages, width = int(need.sum()) + 2, int(_spread(case, "ctx_min", "ctx_max", n, 0).max() + case["new_max"] + PAGE - 1) // PAGE
    order = rng.permutation(pages).astype(np.int32)                      # pages of a cache in use lie anywhere
    tables = np.zeros((n, width), np.int32)
    inside = np.arange(width)[None, :] < need[:, None]
    tables[inside] = order[: int(need.sum())]
    q = _normal(g, (int(new.sum()), case["heads"], case["dim"]))
    q += _normal(g, (1, case["heads"], case["dim"])) / 4                 # rows look at some of the same tokens
    return {"q": q, "cache": _cache(g, 2, pages, case["kv_heads"], case["dim"], case["format"]), "pages": pages, "tables": _dev(tables), "ctx": _dev(ctx),
            "starts": _dev(np.concatenate([[0], np.cumsum(new)]).astype(np.int32)), "seen": _dev(_trees(case, new, rng))}


def prepare(case: dict, seed: int) -> dict:
    s = {"case": case, **{"write": _row_inputs, "read": _row_inputs, "copy": _copy_inputs, "tree": _tree_inputs}[case["kind"]](case, seed)}
    if case["kind"] == "read":
        s["out"] = torch.empty_like(s["kv"])
    if case["kind"] == "tree":
        s["out"] = torch.empty_like(s["q"])
    return s


# ---- one pass ----------------------------------------------------------------------------------------------------------------------------

def _plain_write(s):
    dim, slots = s["case"]["dim"], s["slots"].long()
    y, scale = _quantised(s["kv"].transpose(0, 1), s["case"]["format"])
    page, place = slots // PAGE, slots % PAGE
    for plane in (0, 1):
        _bytes_of(s["cache"], dim)[plane][page, :, place] = y[plane]
        _scales_of(s["cache"], dim)[plane][page, :, place] = scale[plane]


def _plain_read(s):
    case, slots = s["case"], s["slots"].long()
    page, place = slots // PAGE, slots % PAGE
    for plane in (0, 1):
        y = _bytes_of(s["cache"], case["dim"])[plane][page, :, place].view(torch.float8_e4m3fn if case["format"] == E4M3 else torch.int8).float()
        s["out"][:, plane] = y * _scales_of(s["cache"], case["dim"])[plane][page, :, place][..., None]


def _plain_copy(s):
    case, moves = s["case"], torch.from_numpy(s["moves"].astype(np.int64)).cuda()
    for part in (_bytes_of(s["cache"], case["dim"]), _scales_of(s["cache"], case["dim"])):
        part[:, moves[:, 1], :, : case["tokens"]] = part[:, moves[:, 0], :, : case["tokens"]]


def _visible(case, ctx, seen, token, width):
    """[rows, places]: whether a row, token `token` of its sequence of ctx cached ones, sees a place."""
    places = torch.arange(width, device="cuda")[None]
    bits = torch.arange(63, device="cuda")[None]
    depth = (((seen[:, None] >> bits) & 1) * (bits < token[:, None])).sum(1)  # a token lies behind its ancestors
    near = places > (ctx + depth)[:, None] - case["window"] if case["window"] else torch.ones_like(places, dtype=torch.bool)
    u = places - ctx[:, None]
    return torch.where(u < 0, near | (places < case["sinks"]), (u < 64) & (seen[:, None] >> u.clamp(0, 63) & 1).bool())


def _plain_tree(s):
    case = s["case"]
    n, kv_heads, dim, starts, rows = case["seqs"], case["kv_heads"], case["dim"], s["starts"].long(), s["q"].shape[0]
    which = (torch.arange(rows, device="cuda")[:, None] >= starts[None, 1:]).sum(1)                    # a row's sequence
    token = torch.arange(rows, device="cuda") - starts[which]

    def take(plane):
        if case["format"] == BF16:
            x = s["cache"][plane][s["tables"].long()].float()
        else:
            x = _values_of(s["cache"][plane], dim, case["format"]).view(torch.uint8)[s["tables"].long()].view(torch.float8_e4m3fn if case["format"] == E4M3 else torch.int8).float()
            x = x * _scales_of(s["cache"][plane], dim)[s["tables"].long()][..., None]
        return x.transpose(1, 2).flatten(2, 3)                                                          # [sequence, head, place, channel]

    q = torch.zeros((n, kv_heads, case["new_max"], case["heads"] // kv_heads, dim), device="cuda")
    q[which, :, token] = s["q"].float().view(rows, kv_heads, -1, dim) / math.sqrt(dim)
    mask = torch.zeros((n, case["new_max"], s["tables"].shape[1] * PAGE), dtype=torch.bool, device="cuda")
    mask[which, token] = _visible(case, s["ctx"].long()[which], s["seen"], token, mask.shape[2])
    p = torch.matmul(q.flatten(2, 3), take(0).transpose(2, 3)).unflatten(2, (case["new_max"], -1))
    p = p.masked_fill(~mask[:, None, :, None], -math.inf)
    top = p.amax(-1, keepdim=True)
    p = (p - torch.where(top == -math.inf, torch.zeros_like(top), top)).exp()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.flatten(2, 3), take(1)).unflatten(2, (case["new_max"], -1)) / torch.where(total > 0, total, torch.ones_like(total))
    s["out"].copy_(o[which, :, token].reshape(rows, -1, dim))


def _ok(rc):
    if rc != 0:
        raise RuntimeError(f"call failed ({rc})")


def _own(s, lib, stream):
    case, kind, cache = s["case"], s["case"]["kind"], s["cache"].data_ptr()
    if kind == "copy":
        from opsagent_b200 import _lib
        moves = _lib.C.cast(s["moves"].ctypes.data, _lib.C.POINTER(_lib.OaPageMove))
        _ok(lib.oa_k_cache8_copy(cache, case["planes"], s["pages"], case["kv_heads"], case["dim"], moves, case["moves"], stream))
    elif kind == "tree":
        width = case["heads"] * case["dim"]
        _ok(lib.oa_k_tree_attention(s["q"].data_ptr(), width, s["out"].data_ptr(), width, cache, case["format"], s["pages"], s["tables"].data_ptr(), s["tables"].shape[1], s["ctx"].data_ptr(),
                                    s["starts"].data_ptr(), None if case["chain"] else s["seen"].data_ptr(), case["seqs"], s["q"].shape[0], case["heads"], case["kv_heads"], case["dim"],
                                    case["window"], case["sinks"], 0.0, None, stream))
    else:
        rows = s["kv"] if kind == "write" else s["out"]
        k, wide = rows.data_ptr(), case["kv_heads"] * case["dim"]
        if kind == "write":
            _ok(lib.oa_k_cache8_write(k, k + 2 * wide, 2 * wide, cache, s["cache"].shape[1], s["slots"].data_ptr(), case["tokens"], case["kv_heads"], case["dim"],
                                      case["format"], None, stream))
        else:
            _ok(lib.oa_k_cache8_read(cache, s["cache"].shape[1], s["slots"].data_ptr(), case["tokens"], case["kv_heads"], case["dim"], case["format"], k, k + 2 * wide, 2 * wide, None, stream))


def run(state: dict):
    case = state["case"]
    if own:
        from opsagent_b200 import _lib
        _own(state, _lib.load(), torch.cuda.current_stream().cuda_stream)
    else:
        {"write": _plain_write, "read": _plain_read, "copy": _plain_copy, "tree": _plain_tree}[case["kind"]](state)
    if case["kind"] in ("read", "tree"):
        return {"out": state["out"]}
    return {"values": _values_of(state["cache"], case["dim"], case.get("format", INT8)), "scales": _scales_of(state["cache"], case["dim"])}


# ---- what a pass cannot do without -------------------------------------------------------------------------------------------------------

def work(case: dict) -> dict:
    kind, dim, kv_heads = case["kind"], case["dim"], case["kv_heads"]
    stored = 2 * dim if case.get("format") == BF16 else dim + 4          # bytes of a head of a token
    if kind in ("write", "read"):
        return {"bytes": case["tokens"] * (2 * kv_heads * (2 * dim + stored) + 4), "flops": 2 * case["tokens"] * 2 * kv_heads * dim}
    if kind == "copy":
        return {"bytes": (case["sources"] + case["moves"]) * case["planes"] * kv_heads * case["tokens"] * (dim + 4), "flops": 0}
    new, ctx = (_spread(case, f"{x}_min", f"{x}_max", case["seqs"], i).astype(np.int64) for i, x in enumerate(("new", "ctx")))
    if case["window"]:
        ctx = np.minimum(ctx, case["window"] - 1 + case["sinks"])
    rows = int(new.sum())
    pairs = int(new.mean() * ctx.sum()) + rows                           # on average: which sequence has how many new tokens differs by seed
    return {"bytes": 2 * kv_heads * stored * (int(ctx.sum()) + rows) + 4 * rows * case["heads"] * dim, "flops": 4 * case["heads"] * dim * pairs}


# ---- the same in 64 bits -----------------------------------------------------------------------------------------------------------------

def exact(case: dict, seed: int):
    kind, dim = case["kind"], case["dim"]
    if kind == "copy":                                                   # copies: their bits are held to the plain form's
        return None
    if kind in ("write", "read"):
        t = _row_inputs(case, seed)
        flat = lambda x: x.transpose(2, 3).flatten(1, 2)                 # noqa: E731  [plane, page and place, head, ...]
        scales, slots = _scales_of(t["cache"], dim).double(), t["slots"].long()
        if kind == "read":
            y = _values_of(t["cache"], dim, case["format"]).double()
            return {"out": (flat(y)[:, slots] * flat(scales)[:, slots][..., None]).transpose(0, 1)}
        rows = flat(scales).contiguous()
        rows[:, slots] = t["kv"].double().abs().amax(-1).transpose(0, 1) / LIMIT[case["format"]]
        return {"values": None, "scales": rows.unflatten(1, (-1, PAGE)).transpose(2, 3).contiguous()}
    t = _tree_inputs(case, seed)
    out, starts, ctx, kv_heads = torch.empty(t["q"].shape, dtype=torch.float64, device="cuda"), t["starts"].tolist(), t["ctx"].tolist(), case["kv_heads"]
    group = case["heads"] // kv_heads
    for i in range(case["seqs"]):
        n, length, near = starts[i + 1] - starts[i], ctx[i], case["window"] or 1 << 40
        pages = t["tables"][i, : (length + n + PAGE - 1) // PAGE].long()
        if case["format"] == BF16:
            k, v = (t["cache"][j, pages].double().transpose(0, 1).flatten(1, 2) for j in (0, 1))
        else:
            k, v = ((_values_of(t["cache"][j], dim, case["format"]).view(torch.uint8)[pages].view(torch.float8_e4m3fn if case["format"] == E4M3 else torch.int8).double() *
                     _scales_of(t["cache"][j], dim)[pages].double()[..., None]).transpose(0, 1).flatten(1, 2) for j in (0, 1))
        for r in range(n):
            bits = int(t["seen"][starts[i] + r]) & (1 << 64) - 1
            at = length + bin(bits & (1 << r) - 1).count("1")
            old = torch.arange(length, device="cuda")
            see = torch.cat([old[(old < case["sinks"]) | (at - old < near)], torch.tensor([length + u for u in range(n) if bits >> u & 1], device="cuda", dtype=torch.long)])
            w = torch.einsum("khd,kpd->khp", t["q"][starts[i] + r].double().view(kv_heads, group, dim), k[:, see]) / math.sqrt(dim)
            out[starts[i] + r] = torch.einsum("khp,kpd->khd", torch.softmax(w, -1), v[:, see]).reshape(-1, dim)
    return {"out": out}
