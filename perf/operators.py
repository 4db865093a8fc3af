"""The paged 4-bit key/value cache and the attention that reads it: the cases
that are measured, the operators in plain form, and their definitions in 64 bits.

Operators (C entry points in include/ks_b200.h, Python ones in kernelsmith_b200):

  append     quantises the keys and values of new tokens into the cache (ks_b200_kv4_append_async)
             and reads them back as the values that the codes stand for (ks_b200_kv4_read_async)
  attention  softmax(scale q k^T) v over the cached tokens, grouped query heads, one new token or
             several per sequence (causal among them); optionally adds each cached token's
             attention weight to the cache's accumulated weights (ks_b200_kv4_attention_async)
  evict      keeps the newest tokens and those with the largest accumulated weight, packed in order
             into other pages (ks_b200_kv4_evict_async)

The cache.  A pool of pages; a page holds page_size tokens of every key/value head, as
[head][block][bytes]: a block is 16 tokens,
  key codes 16 x head_dim/2 bytes, key scales 16 x head_dim/group f16, value codes, value scales.
Codes are signed 4-bit numbers, the even element of a pair in a byte's low half.  A group of
`group` elements v of one token and head has scale = max(max(v, 0) / 7, -min(v, 0) / 8) rounded to
f16 (within the positive finite f16 values; 1 if all elements are 0) and codes
round_half_even(v / scale) within [-8, 7].  The pair with element d (even) is byte
  keys    ((d % 32) / 8) * (head_dim / 8) + (d / 32) * 4 + (d % 8) / 2
  values  ((d % 16) / 2) * (head_dim / 16) + d / 16
of the token's row.  Accumulated weights: f32 [page][head][slot].  Token p of sequence s is slot
p % page_size of page page_table[s][p / page_size].
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

_ROOT = Path(__file__).resolve().parent.parent
_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def _kernels():
    """This repository's package (the built library), for the framework's own calls."""
    at = str(_ROOT / "ulir-kernels_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import kernelsmith_b200

    return kernelsmith_b200


# ----------------------------------------------------------------------- cases
def _case(op, seqs, kv_heads, group_heads, head_dim, group, page, max_len, new, dtype, ragged, weights=False,
          budget=0, recent=0, name=None):
    c = {"op": op, "seqs": seqs, "kv_heads": kv_heads, "group_heads": group_heads, "head_dim": head_dim,
         "group": group, "page": page, "max_len": max_len, "new": new, "dtype": dtype, "ragged": ragged,
         "weights": weights, "budget": budget, "recent": recent}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one request with a short context, 4096 = 32 heads x 128, one key head to four: latency of a decode step
        _case("attention", 1, 8, 4, 128, 32, 64, 257, 1, "f32", False, name="attn_one_short_f32"),
        # a batch of requests of unequal lengths, f32 activations as this library's GEMMs write them
        _case("attention", 16, 8, 4, 128, 32, 64, 4096, 1, "f32", True, name="attn_batch_f32"),
        # every query head with keys of its own (the 4096-wide decode layers), 32 heads
        _case("attention", 8, 32, 1, 128, 64, 32, 2047, 1, "f16", True, name="attn_mha_f16"),
        # a single request with a very long context (8192 = 64 heads x 128)
        _case("attention", 1, 8, 8, 128, 128, 256, 131071, 1, "bf16", False, name="attn_one_long_bf16"),
        # serving at its largest: 64 requests, eight query heads to a key head
        _case("attention", 64, 8, 8, 128, 64, 128, 8192, 1, "bf16", True, name="attn_serving_bf16"),
        # checking several drafted tokens at once, seven query heads to a key head, heads of 64
        _case("attention", 8, 4, 7, 64, 32, 16, 3001, 8, "f16", True, name="attn_drafts_f16"),
        # a piece of a prompt against what is cached: 64 tokens, the batch that this library's W4A8 GEMM takes
        _case("attention", 1, 8, 4, 128, 32, 64, 8192, 64, "f32", False, name="attn_chunk_f32"),
        # a decode step that also keeps the weights that an eviction goes by
        _case("attention", 16, 8, 4, 128, 64, 64, 4096, 1, "f32", True, weights=True, name="attn_weights_f32"),
        # the new tokens of a decode step
        _case("append", 64, 8, 1, 128, 32, 64, 2000, 1, "f32", True, name="append_step_f32"),
        # prompts of unequal lengths
        _case("append", 4, 8, 1, 128, 64, 128, 8192, 8192, "bf16", True, name="append_prompts_bf16"),
        # one request trimmed back to its budget
        _case("evict", 1, 8, 1, 128, 32, 64, 1100, 0, "f16", False, budget=1000, recent=100, name="evict_one_f16"),
        # a batch of long requests cut to a quarter
        _case("evict", 32, 8, 1, 128, 64, 128, 8192, 0, "f16", True, budget=2048, recent=256, name="evict_batch_f16"),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "append", "evict"])
    head_dim = rng.choice([64, 128, 128])
    group = rng.choice([g for g in (32, 64, 128) if g <= head_dim])
    page = rng.choice([16, 32, 64, 128, 256])
    dtype = rng.choice(["f32", "f16", "bf16"])
    seqs = _spread(rng, 1, 64)
    kv_heads = rng.choice([1, 2, 3, 4, 5, 8, 8, 16, 32])
    # at most a quarter of the largest listed case's tokens times heads
    most = max(64, min(131072, (64 * 8192 * 8 // 4) // (seqs * kv_heads)))
    if op == "append":
        new = rng.choice([1, 1, 2, 5, 0])
        new = new or _spread(rng, 8, max(8, min(8192, most // 8)))
        return _case(op, seqs, kv_heads, 1, head_dim, group, page, new + rng.randrange(0, 3 * page), new, dtype,
                     rng.random() < 0.5)
    max_len = _spread(rng, 8, most)
    if op == "evict":
        max_len = min(max_len // 2, 32768)  # what is kept is written twice
        budget = max(1, int(max_len * rng.uniform(0.1, 0.9)))
        return _case(op, seqs, kv_heads, 1, head_dim, group, page, max_len, 0, dtype, rng.random() < 0.7,
                     budget=budget, recent=rng.randrange(0, budget + 1))
    group_heads = rng.choice([1, 2, 3, 4, 4, 5, 6, 7, 8, 8, 12, 16])
    new = min(max_len, rng.choice([1, 1, 1, 2, 4, 7, 16, 33, 64]))
    # nor more products than the largest does
    while seqs * kv_heads * group_heads * new * max_len * head_dim > 64 * 8 * 8 * 8192 * 128 // 2:
        new, max_len = max(1, new // 2), max_len if new > 1 else max_len // 2
    return _case(op, seqs, kv_heads, group_heads, head_dim, group, page, max_len, new, dtype, rng.random() < 0.7,
                 weights=rng.random() < 0.3)


def _lengths(case):
    """Cached tokens of each sequence (the new ones among them), and new tokens of each: the case's alone."""
    n, most, new = case["seqs"], case["max_len"], case["new"]
    if not case["ragged"]:
        return [most] * n, [new] * n
    part = [(i * 0.6180339887498949 + 1.0) % 1.0 if i else 1.0 for i in range(n)]  # the first is the longest
    lens = [max(1, int(most * f)) for f in part]
    news = [min(max(1, int(new * (1.0 - f * 0.5)) if i else new), ln) if new else 0
            for i, (f, ln) in enumerate(zip(part, lens))]
    return lens, news


def _pages(tokens, page):
    return -(-tokens // page)


def _kept(case):
    return [min(x, case["budget"]) for x in _lengths(case)[0]]


def work(case):
    h, d, g, item = case["kv_heads"], case["head_dim"], case["group"], _BYTES[case["dtype"]]
    lens, news = _lengths(case)
    row = 2 * (d // 2 + 2 * (d // g))  # a token's keys and values of one head
    if case["op"] == "attention":
        heads = h * case["group_heads"]
        seen = sum(n * ln - n * (n - 1) // 2 for ln, n in zip(lens, news))  # pairs of a new token and one it sees
        size = sum(lens) * h * (row + (8 if case["weights"] else 0)) + sum(news) * heads * (2 * d * item + 4)
        return {"bytes": size, "flops": 4 * d * heads * seen}
    if case["op"] == "append":
        tokens = sum(news)
        return {"bytes": tokens * h * (4 * d * item + row), "flops": tokens * h * 2 * d * 4}
    kept = sum(_kept(case))
    return {"bytes": h * (sum(lens) * 4 + kept * (2 * row + 4 + 4 + 2 * d * item)),
            "flops": h * (sum(lens) * 4 + kept * 2 * d)}


# ---------------------------------------------------------------------- inputs
def _quantize(x, group):
    """Codes (float) and f16 scales of x [..., head_dim]; in 64 bits, where a quotient lies next to a border."""
    v = x.double().unflatten(-1, (-1, group))
    hi, lo = v.amax(-1).clamp(min=0), v.amin(-1).clamp(max=0)
    scale = torch.maximum(hi / torch.full_like(hi, 7.0), -lo / 8)
    scale = torch.where(scale == 0, 1.0, scale.clamp(2.0**-24, 65504.0)).half()
    codes = (v / scale.double().unsqueeze(-1)).round().clamp(-8, 7)
    return codes.flatten(-2).float(), scale


def _pack(codes, order):
    """Codes [..., head_dim] as bytes [..., head_dim / 2] in the order of a row of keys ("k") or values ("v")."""
    q = codes.to(torch.int16) & 15
    if order == "k":  # d = 32 w + 8 t + 2 b + half, byte (t, w, b)
        q = q.unflatten(-1, (-1, 4, 4, 2)).transpose(-4, -3)
    else:  # d = 16 i + 2 g + half, byte (g, i)
        q = q.unflatten(-1, (-1, 8, 2)).transpose(-3, -2)
    return (q[..., 0] | (q[..., 1] << 4)).to(torch.uint8).reshape(*codes.shape[:-1], -1)


def _block_bytes(case):
    return 16 * 2 * (case["head_dim"] // 2 + 2 * (case["head_dim"] // case["group"]))


def _fill(part, x, group, order):
    """Quantises x [pages, heads, blocks, 16, head_dim] into `part` [pages, heads, blocks, bytes]."""
    codes, scale = _quantize(x, group)
    rows = _pack(codes, order).flatten(-2)
    part[..., : rows.shape[-1]] = rows
    part[..., rows.shape[-1]:] = scale.flatten(-2).contiguous().view(torch.uint8)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    h, d, page, dtype = case["kv_heads"], case["head_dim"], case["page"], _TYPES[case["dtype"]]
    lens, news = _lengths(case)
    each = [_pages(x, page) for x in lens]
    used, spare = sum(each), 3
    # an eviction's pages for what is kept stand at the end of the pool, one sequence after the other
    kept = _kept(case) if case["op"] == "evict" else [0] * len(lens)
    to_each = [_pages(x, page) for x in kept]
    n_pages = used + spare + sum(to_each)
    pool = torch.zeros(n_pages, h, page // 16, _block_bytes(case), dtype=torch.uint8, device=dev)
    if case["op"] != "append":
        # a few channels of the keys are larger than the others, as those of trained models are, and tokens
        # differ in the size of their values
        channel = 1.0 + 3.0 * (torch.rand(h, 1, 1, d, generator=gen, device=dev) < 0.06)
        half, step = _block_bytes(case) // 2, max(1, (1 << 27) // (h * page * d))
        for at in range(0, used + spare, step):  # some pages at a time: the values before they are codes are large
            some = min(step, used + spare - at)
            shape = (some, h, page // 16, 16, d)
            x = torch.randn(shape, generator=gen, device=dev) * channel
            _fill(pool[at:at + some, ..., :half], x, case["group"], "k")
            x = torch.randn(shape, generator=gen, device=dev)
            x *= torch.exp(0.5 * torch.randn(shape[:-1] + (1,), generator=gen, device=dev))
            _fill(pool[at:at + some, ..., half:], x, case["group"], "v")
            del x
    ids = torch.randperm(used + spare, generator=gen, device=dev).cpu()
    table = torch.full((len(lens), max(each)), -1, dtype=torch.int32)
    at = 0
    for s, k in enumerate(each):
        table[s, :k] = ids[at:at + k].int()
        at += k
    s = {"case": case, "pool": pool, "table": table.to(dev), "n_pages": n_pages,
         "lens": torch.tensor(lens, dtype=torch.int32, device=dev)}
    tokens = sum(news)
    s["offsets"] = torch.tensor([sum(news[:i]) for i in range(len(news) + 1)], dtype=torch.int32, device=dev)
    s["tokens"] = tokens
    if case["op"] == "attention":
        heads = h * case["group_heads"]
        s["q"] = (1.5 * torch.randn(tokens, heads, d, generator=gen, device=dev)).to(dtype)
        s["scale"] = d**-0.5
        s["out"] = torch.zeros(tokens, heads, d, dtype=dtype, device=dev)
        s["lse"] = torch.zeros(tokens, heads, device=dev)
    elif case["op"] == "append":
        x = torch.randn(2, tokens, h, d, generator=gen, device=dev)
        s["k"], s["v"] = x[0].to(dtype), x[1].to(dtype)
        s["k_out"], s["v_out"] = torch.zeros_like(s["k"]), torch.zeros_like(s["v"])
    if case["weights"] or case["op"] == "evict":
        # accumulated weights: a few tokens hold most of it, and some that were never looked at tie at 0
        w = torch.exp(2.0 * torch.randn(n_pages, h, page, generator=gen, device=dev) - 4.0)
        w *= torch.rand(w.shape, generator=gen, device=dev) > 0.05
        s["weights_before"] = w
        s["weights"] = w.clone()
    if case["op"] == "evict":
        to = torch.full((len(lens), max(to_each)), -1, dtype=torch.int32)
        at = used + spare
        for i, k in enumerate(to_each):
            to[i, :k] = torch.arange(at, at + k, dtype=torch.int32)
            at += k
        s["weights"][used + spare:] = 0
        s["first_to"], s["to_table"] = used + spare, to.to(dev)
        s["to_lens"] = torch.zeros(len(lens), dtype=torch.int32, device=dev)
        s["to_offsets"] = torch.tensor([sum(kept[:i]) for i in range(len(kept) + 1)], dtype=torch.int32, device=dev)
        s["kept"] = torch.full((len(lens), h, case["budget"]), -1, dtype=torch.int32, device=dev)
        s["k_out"] = torch.zeros(sum(kept), h, d, dtype=dtype, device=dev)
        s["v_out"] = torch.zeros_like(s["k_out"])
    if own:  # the handle of the pool and the workspace, which a program keeps for as long as the pool
        kernels = _kernels()
        s["cache"] = kernels.Kv4Cache(pool, n_pages, page, h, d, case["group"], weights=s.get("weights"))
        size = 0
        if case["op"] == "attention":
            size = kernels.kv4_attention_workspace(s["cache"], heads, len(lens), tokens, case["new"], case["max_len"])
        elif case["op"] == "evict":
            size = kernels.kv4_evict_workspace(s["cache"], len(lens), case["max_len"], case["budget"])
        s["workspace"] = torch.zeros(max(size, 16), dtype=torch.uint8, device=dev)
    return s


# ------------------------------------------------------------------ plain form
def _values(rows, case, order):
    """The numbers [..., 16, head_dim] that a half of a block, bytes [...], stands for, in f32."""
    d, size = case["head_dim"], 8 * case["head_dim"]
    b = rows[..., :size].unflatten(-1, (16, -1))
    q = torch.stack((b & 15, b >> 4), -1)
    if order == "k":
        q = q.unflatten(-2, (4, d // 32, 4)).transpose(-4, -3)
    else:
        q = q.unflatten(-2, (8, d // 16)).transpose(-3, -2)
    q = q.reshape(*q.shape[: rows.dim()], d)
    scale = rows[..., size:].contiguous().view(torch.float16).unflatten(-1, (16, -1)).float()
    codes = ((q ^ 8).float() - 8.0).unflatten(-1, (-1, case["group"]))
    return (codes * scale.unsqueeze(-1)).flatten(-2)


def _cached(s, order):
    """Keys or values of every sequence, [sequences, heads, tokens of the table, head_dim] in f32."""
    case = s["case"]
    rows = s["pool"][s["table"].clamp(min=0).long()]
    half = rows.shape[-1] // 2
    rows = (rows[..., :half] if order == "k" else rows[..., half:]).transpose(1, 2).flatten(2, 3)
    return _values(rows, case, order).flatten(2, 3)


def _attention(s):
    case = s["case"]
    n, h, g, d, new = case["seqs"], case["kv_heads"], case["group_heads"], case["head_dim"], case["new"]
    dev = s["pool"].device
    first, count = s["offsets"][:-1].long(), s["offsets"][1:].long() - s["offsets"][:-1].long()
    j = torch.arange(new, device=dev)
    there = j < count[:, None]  # [sequences, new]
    token = (first[:, None] + j).clamp(max=max(s["tokens"] - 1, 0))
    q = s["q"].float()[token].unflatten(2, (h, g)).permute(0, 2, 1, 3, 4).reshape(n, h, new * g, d)
    score = torch.matmul(q, _cached(s, "k").transpose(-1, -2)) * s["scale"]
    at = torch.arange(score.shape[-1], device=dev)
    last = s["lens"].long()[:, None] - count[:, None] + j  # the position of each new token
    seen = (at <= last[..., None]) & there[..., None]
    score = score.unflatten(2, (new, g)).masked_fill(~seen[:, None, :, None], float("-inf")).flatten(2, 3)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == float("-inf"), 0.0, top)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    lse = (top + torch.log(total)).unflatten(2, (new, g)).permute(0, 2, 1, 3, 4)
    out = torch.matmul(p, _cached(s, "v")).unflatten(2, (new, g)).permute(0, 2, 1, 3, 4)
    out, lse = out.reshape(n, new, h * g, d)[there], lse.reshape(n, new, h * g)[there]
    got = {"out": out.to(s["q"].dtype), "lse": lse}
    if case["weights"]:
        add = p.sum(2).unflatten(-1, (-1, case["page"])).transpose(1, 2)  # [sequences, pages, heads, slots]
        got["weights"] = s["weights_before"].index_add(0, s["table"].clamp(min=0).long().flatten(), add.flatten(0, 1))
    return got


def _append(s):
    group, got = s["case"]["group"], {}
    for name in ("k", "v"):
        codes, scale = _quantize(s[name], group)
        x = codes.unflatten(-1, (-1, group)) * scale.float().unsqueeze(-1)
        got[name] = x.flatten(-2).to(s[name].dtype)
    return got


def _evict(s):
    case = s["case"]
    n, h, budget, recent = case["seqs"], case["kv_heads"], case["budget"], case["recent"]
    table, lens = s["table"].clamp(min=0).long(), s["lens"].long()
    w = s["weights_before"][table].transpose(1, 2).flatten(2)  # [sequences, heads, tokens]
    at = torch.arange(w.shape[-1], device=w.device)
    key = torch.where(at >= lens[:, None] - recent, float("inf"), w.transpose(0, 1)).transpose(0, 1)
    key = torch.where((at >= lens[:, None])[:, None], float("-inf"), key)
    count = lens.clamp(max=budget)
    best = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :budget]
    slot = torch.arange(best.shape[-1], device=w.device)
    live = (slot < count[:, None])[:, None]
    best = torch.sort(torch.where(live, best, w.shape[-1]), dim=-1).values
    live = live.expand_as(best)
    kept = torch.full((n, h, budget), -1, dtype=torch.int32, device=w.device)
    kept[..., : best.shape[-1]] = torch.where(live, best, -1).int()
    got = {"kept": kept, "lens": count.int()}
    at = best.clamp(max=w.shape[-1] - 1)
    rows, row = live.transpose(1, 2)[:, :, 0], at[..., None]
    for order in ("k", "v"):
        x = _cached(s, order).gather(2, row.expand(-1, -1, -1, case["head_dim"]))
        got[order] = x.transpose(1, 2)[rows].to(_TYPES[case["dtype"]])
    to = torch.zeros_like(s["weights_before"][s["first_to"]:]).transpose(0, 1).flatten(1)  # [heads, slots of the pages]
    place = (s["to_table"].long() - s["first_to"]).clamp(min=0) * case["page"]
    place = place.repeat_interleave(case["page"], 1)[:, : best.shape[-1]] + slot % case["page"]
    to.scatter_add_(1, place[rows].expand(h, -1), w.gather(2, at).transpose(1, 2)[rows].T.contiguous())
    got["weights"] = to.unflatten(1, (-1, case["page"])).transpose(0, 1)
    return got


def run(s):
    case = s["case"]
    if not own:
        return {"attention": _attention, "append": _append, "evict": _evict}[case["op"]](s)
    kernels = _kernels()
    cache = s["cache"]
    if case["op"] == "attention":
        if case["weights"]:
            s["weights"].copy_(s["weights_before"])  # a pass starts from the same weights each time
        kernels.kv4_attention_async(cache, s["table"], s["lens"], s["q"], s["out"], s["scale"], s["workspace"],
                                    token_offsets=s["offsets"], max_new=case["new"], max_len=case["max_len"],
                                    lse=s["lse"], accumulate=case["weights"])
        got = {"out": s["out"], "lse": s["lse"]}
        return dict(got, weights=s["weights"]) if case["weights"] else got
    if case["op"] == "append":
        kernels.kv4_append_async(cache, s["table"], s["lens"], s["k"], s["v"], token_offsets=s["offsets"])
        kernels.kv4_read_async(cache, s["table"], s["lens"], s["k_out"], s["v_out"], token_offsets=s["offsets"])
        return {"k": s["k_out"], "v": s["v_out"]}
    kernels.kv4_evict_async(cache, s["table"], s["lens"], s["to_table"], s["to_lens"], case["max_len"],
                            case["budget"], case["recent"], s["workspace"], kept=s["kept"])
    kernels.kv4_read_async(cache, s["to_table"], s["to_lens"], s["k_out"], s["v_out"], token_offsets=s["to_offsets"])
    return {"kept": s["kept"], "lens": s["to_lens"], "k": s["k_out"], "v": s["v_out"],
            "weights": s["weights"][s["first_to"]:]}


# ------------------------------------------------------------------ in 64 bits
def _places(case, order, dev):
    """For each element of a token's row: its byte, and how far its code stands from the byte's low end."""
    e, d = torch.arange(case["head_dim"], device=dev), case["head_dim"]
    if order == "k":
        byte = ((e % 32) // 8) * (d // 8) + (e // 32) * 4 + (e % 8) // 2
    else:
        byte = ((e % 16) // 2) * (d // 16) + e // 16
    return byte, 4 * (e % 2)


def _exact_rows(s, i, positions, order):
    """Keys or values [heads, positions, head_dim] of sequence i at the given positions [heads, positions]."""
    case, dev = s["case"], s["pool"].device
    d, page, per = case["head_dim"], case["page"], case["head_dim"] // case["group"]
    flat = s["pool"].flatten(1)  # a page's bytes
    size = _block_bytes(case)
    head = torch.arange(case["kv_heads"], device=dev)[:, None]
    pages = s["table"][i].long()[positions // page]
    slot = positions % page
    start = (head * (page // 16) + slot // 16) * size + (size // 2 if order == "v" else 0)
    byte, shift = _places(case, order, dev)
    raw = flat[pages[..., None], (start + (slot % 16) * (d // 2))[..., None] + byte].int()
    code = (raw >> shift.int()) % 16
    code = torch.where(code > 7, code - 16, code).double()
    where = (start + 8 * d + (slot % 16) * 2 * per)[..., None] + 2 * torch.arange(per, device=dev)
    bits = flat[pages[..., None], where].int() + 256 * flat[pages[..., None], where + 1].int()
    sign, power, part = bits >> 15, (bits >> 10) % 32, (bits % 1024).double()
    scale = torch.where(power == 0, part * 2.0**-24, (1 + part / 1024) * torch.exp2((power - 15).double()))
    scale = torch.where(sign == 1, -scale, scale)
    return code * scale[..., torch.arange(d, device=dev) // case["group"]]


def _exact_attention(s):
    case = s["case"]
    h, g, dev = case["kv_heads"], case["group_heads"], s["pool"].device
    lens, news = _lengths(case)
    out, lse, at = [], [], 0
    weights = s["weights_before"].double() if case["weights"] else None
    for i, (ln, n) in enumerate(zip(lens, news)):
        every = torch.arange(ln, device=dev)
        k, v = (_exact_rows(s, i, every.expand(h, ln), o) for o in ("k", "v"))
        q = s["q"][at:at + n].double().reshape(n, h, g, -1)
        x = torch.einsum("nhgd,htd->nhgt", q, k) * s["scale"]
        x[(every > (ln - n + torch.arange(n, device=dev))[:, None])[:, None, None].expand_as(x)] = -math.inf
        z = torch.logsumexp(x, -1)
        p = torch.exp(x - z[..., None])
        out.append(torch.einsum("nhgt,htd->nhgd", p, v).flatten(1, 2))
        lse.append(z.flatten(1))
        if weights is not None:
            weights[s["table"][i].long()[every // case["page"]], :, every % case["page"]] += p.sum((0, 2)).T
        at += n
    got = {"out": torch.cat(out), "lse": torch.cat(lse)}
    return dict(got, weights=weights) if weights is not None else got


def _exact_append(s):
    case, got = s["case"], {}
    for name in ("k", "v"):
        v = s[name].double().reshape(*s[name].shape[:2], -1, case["group"])
        scale = torch.maximum(v.amax(-1, keepdim=True) / torch.tensor(7.0, device=v.device, dtype=v.dtype),
                              -v.amin(-1, keepdim=True) / 8)
        scale = torch.where((v == 0).all(-1, keepdim=True), 1.0, scale.clamp(2.0**-24, 65504.0)).half().double()
        low = torch.floor(v / scale)  # the nearer neighbour, the even one where both are as near
        rest = v - low * scale
        up = (rest * 2 > scale) | ((rest * 2 == scale) & (low % 2 == 1))
        got[name] = ((low + up).clamp(-8, 7) * scale).reshape(s[name].shape)
    return got


def _exact_evict(s):
    case = s["case"]
    h, page, dev = case["kv_heads"], case["page"], s["pool"].device
    lens, _ = _lengths(case)
    kept = torch.full((len(lens), h, case["budget"]), -1, dtype=torch.int32, device=dev)
    weights = torch.zeros(s["weights_before"][s["first_to"]:].shape, dtype=torch.float64, device=dev)
    k, v = [], []
    for i, ln in enumerate(lens):
        n = min(ln, case["budget"])
        at = torch.arange(ln, device=dev)
        w = s["weights_before"][s["table"][i].long()[at // page], :, at % page].double().T  # [heads, tokens]
        old = max(ln - case["recent"], 0)
        if n < ln:  # the n - recent largest of the older tokens, the lower position first among equals
            order = torch.sort(-w[:, :old], dim=1, stable=True).indices[:, : n - (ln - old)]
            best = torch.cat((order, at[old:].expand(h, -1)), 1).sort(1).values
        else:
            best = at.expand(h, ln)
        kept[i, :, :n] = best.int()
        k.append(_exact_rows(s, i, best, "k").transpose(0, 1))
        v.append(_exact_rows(s, i, best, "v").transpose(0, 1))
        to = torch.arange(n, device=dev)
        weights[s["to_table"][i].long()[to // page] - s["first_to"], :, to % page] = w.gather(1, best).T
    return {"kept": kept, "lens": torch.tensor([min(x, case["budget"]) for x in lens], dtype=torch.int32, device=dev),
            "k": torch.cat(k), "v": torch.cat(v), "weights": weights}


def exact(case, seed):
    s = prepare(case, seed)
    return {"attention": _exact_attention, "append": _exact_append, "evict": _exact_evict}[case["op"]](s)
