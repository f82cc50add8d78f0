"""The operators of a batched serving step over a paged 8-bit KV cache, as cases that can be timed and compared.

Four operators that follow one another in such a step: the plan of the step (which page and slot every new token
gets), the store of its K and V into 8-bit pages, the attention that reads them, and the sampling of the next
tokens from the logits.  listed() names the cases, draw() gives more of the same ranges, prepare() makes what a
program holds before the call, run() is one pass (in plain torch, or through the framework's entry points where
`own` is true), work() the bytes and operations that one pass cannot do without, exact() the same outputs from the
definition in 64 bits.

The definitions:

plan     A batch has `lens` cached tokens per sequence and `new` tokens this step (negative: the sequence has ended
         and its pages go back on the free stack before any are taken).  A sequence is admitted if its new length
         fits its row of the block table and its tokens end within max_tokens, and either it needs no new page or
         the pages needed up to and including it, in batch order, are free.  Pages come off the top of the stack.
store    slots[t] = page * page_size + offset of token t.  The tokens of one page come one after the other.  One
         scale per page and head, for K and for V: scale = max(old, fp32(max|new| / 127)) (448 for e4m3), where
         old counts as 0 if the tokens begin at offset 0; if it grew, the codes before them are rounded again to
         the new scale, to nearest, ties to even.
attend   Softmax attention with grouped heads over the dequantised pages of each sequence; query i of a sequence
         sees the positions up to kv_len - q_len + i.  A query that sees none gets zeros.
sample   Logits in descending order, the lowest index first among equals, weights exp((x - max) / T).  Kept: the
         first top_k; of these the shortest beginning that holds top_p of their weight; of these the ones whose
         weight is at least min_p.  The answer is the first whose running sum passes u times the kept weight.
"""
import glob
import math
import os
import random
import sys

import numpy as np
import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _fence():
    """The framework's binding."""
    pkg = glob.glob(os.path.join(glob.escape(ROOT), "*_amd"))[0]
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import fence_ops

    return fence_ops


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # A decode step of 64 running sequences: one new token each, few of them on a new page.
        {"name": "plan_decode_64", "kind": "plan", "batch": 64, "new": 1, "ctx": 4096, "page": 16, "ended": 2},
        # A step that admits many prompts at once (odd lengths), while some sequences end.
        {"name": "plan_prompts_384", "kind": "plan", "batch": 384, "new": 700, "ctx": 8192, "page": 32, "ended": 37},
        # The K and V of one decode step of 64 sequences, appended to pages that are partly full (Qwen3-4B heads).
        {"name": "store_decode_64", "kind": "store", "batch": 64, "new": 1, "kv_heads": 8, "head_dim": 128, "page": 32,
         "cache": "int8", "dtype": "f32", "fused_rows": False},
        # The K and V of a prefill step, 9 prompts of odd lengths, out of the rows of a fused q/k/v product.
        {"name": "store_prefill_8001", "kind": "store", "batch": 9, "new": 889, "kv_heads": 8, "head_dim": 128, "page": 64,
         "cache": "e4m3", "dtype": "f16", "fused_rows": True},
        # Decode of a single sequence at a long context (Qwen3-4B): where latency counts.
        {"name": "attend_decode_1x2916", "kind": "attend", "batch": 1, "new": 1, "ctx": 2916, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "page": 16, "cache": "int8", "dtype": "f32"},
        # Decode of a large ragged batch at contexts up to 32k: the cache's bytes are all there is.
        {"name": "attend_decode_64x32k", "kind": "attend", "batch": 64, "new": 1, "ctx": 32768, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "page": 64, "cache": "int8", "dtype": "f16"},
        # A few drafted tokens per sequence to verify, small heads in a group of seven.
        {"name": "attend_verify_24x5", "kind": "attend", "batch": 24, "new": 5, "ctx": 4001, "heads": 14, "kv_heads": 2,
         "head_dim": 64, "page": 32, "cache": "e4m3", "dtype": "f32"},
        # Prefill of one long prompt (Qwen3-4B and Llama-3-8B heads): the matrix products are all there is.
        {"name": "attend_prefill_8192", "kind": "attend", "batch": 1, "new": 8192, "ctx": 8192, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "page": 64, "cache": "int8", "dtype": "f16"},
        # A step of prompt chunks of odd lengths behind contexts of their own, in binary32.
        {"name": "attend_chunks_6x500", "kind": "attend", "batch": 6, "new": 500, "ctx": 4001, "heads": 16, "kv_heads": 8,
         "head_dim": 128, "page": 128, "cache": "e4m3", "dtype": "f32"},
        # One sequence's next token, at the settings that a chat model is served with.
        {"name": "sample_1", "kind": "sample", "rows": 1, "vocab": 151936, "which": "chat"},
        # A batch that is sampled with top-p alone, over rows from peaked to flat.
        {"name": "sample_top_p_32", "kind": "sample", "rows": 32, "vocab": 128256, "which": "top_p"},
        # A large batch in which every request has settings of its own, greedy and unfiltered ones among them.
        {"name": "sample_mixed_256", "kind": "sample", "rows": 256, "vocab": 151936, "which": "mixed"},
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(["plan", "store", "store", "attend", "attend", "attend", "sample", "sample"])
    page = rng.choice([16, 32, 64, 128])
    heads, kv_heads = rng.choice([(32, 8), (32, 8), (16, 8), (14, 2), (16, 16), (40, 8), (64, 8), (6, 2), (8, 1)])
    head_dim = rng.choice([128, 128, 128, 64, 64, 96, 256])
    cache, dtype = rng.choice(["int8", "e4m3"]), rng.choice(["f32", "f16"])
    if kind == "plan":
        batch = _log(rng, 1, 384)
        return {"kind": kind, "batch": batch, "new": rng.choice([1, 1, _log(rng, 1, 700)]), "ctx": _log(rng, 1024, 8192),
                "page": page, "ended": rng.randrange(0, batch // 8 + 1)}
    if kind == "store":
        new = rng.choice([1, 1, _log(rng, 2, 4000)])
        return {"kind": kind, "batch": _log(rng, 1, max(1, 5000 // max(new, page))), "new": new,
                "kv_heads": min(kv_heads, 8), "head_dim": min(head_dim, 128), "page": page, "cache": cache, "dtype": dtype,
                "fused_rows": rng.random() < 0.5}
    if kind == "attend":
        which = rng.choice(["decode", "decode", "verify", "prefill"])
        new = 1 if which == "decode" else rng.randrange(2, 9) if which == "verify" else _log(rng, 9, 4000)
        ctx = _log(rng, max(16, new), 32768 if new == 1 else 8192 if new < 9 else max(4000, new))
        most = int(2e8 / (heads * new * ctx)) if new > 1 else int(4e8 / (kv_heads * head_dim * ctx))
        return {"kind": kind, "batch": _log(rng, 1, max(1, min(64, most))), "new": new, "ctx": ctx, "heads": heads,
                "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "cache": cache, "dtype": dtype}
    return {"kind": kind, "rows": _log(rng, 1, 256), "vocab": rng.choice([151936, 128256, _log(rng, 1000, 151936)]),
            "which": rng.choice(["chat", "top_p", "top_k", "mixed", "mixed"])}


def _spread(case):
    """(cached tokens, new tokens) of each sequence, odd ones among them; the same for every seed."""
    r = random.Random("%s %d %d" % (case["kind"], case["batch"], case["new"]))
    n, ctx, lens, news = case["batch"], case.get("ctx", case["new"] + 4 * case["page"]), [], []
    for b in range(n):
        new = case["new"] if case["new"] < 9 or n == 1 else r.randint(max(1, case["new"] // 2), case["new"] * 3 // 2)
        new = min(new, ctx)
        total = ctx if b == 0 else max(new, int(ctx * math.exp(-r.random() * 2.5)))
        lens.append(total - new)
        news.append(new)
    return lens, news


# ------------------------------------------------------------------ inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 11)


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _codes(shape, cache, g):
    """8-bit codes as a store leaves them: the largest of a page near the end of the range."""
    x = torch.randn(shape, generator=g, device="cuda", dtype=torch.float16)
    if cache == "int8":
        return x.mul_(36).round_().clamp_(-127, 127).to(torch.int8)
    return x.mul_(128).clamp_(-448, 448).to(torch.float8_e4m3fn)


def _table(blocks, max_blocks, pages, g):
    """A block table: every page in use by one sequence, in no order; the entries behind a sequence's pages are 0."""
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    used = torch.arange(max_blocks, device="cuda") < _int(blocks)[:, None]
    at = (torch.cumsum(_int(blocks), 0) - _int(blocks))[:, None] + torch.arange(max_blocks, device="cuda")
    return torch.where(used, order[at.clamp(max=pages - 1)], 0).to(torch.int32).contiguous(), order


def prepare(case, seed):
    return {"plan": _prepare_plan, "store": _prepare_store, "attend": _prepare_attend, "sample": _prepare_sample}[
        case["kind"]](case, _gen(seed), seed)


def _prepare_plan(case, g, seed):
    lens, news = _spread(case)
    page, n = case["page"], case["batch"]
    held = [-(-length // page) for length in lens]
    max_blocks = -(-(case["ctx"] + 2 * case["new"]) // page) + 1
    # enough pages for most of the batch: the last few prompts wait
    need = sum(-(-(length + new) // page) - h for length, new, h in zip(lens, news, held))
    pages = sum(held) + max(1, need - need // 16 - sum(held) * case["ended"] // n)
    max_tokens = sum(news)
    max_tokens += -max_tokens % 64
    for b in random.Random(int(seed)).sample(range(n), case["ended"]):
        news[b] = -1
    table, order = _table(held, max_blocks, pages, g)
    free = torch.zeros(pages, dtype=torch.int32, device="cuda")
    free[: pages - sum(held)] = order[sum(held):]
    e = lambda *s: torch.empty(s, dtype=torch.int32, device="cuda")  # noqa: E731
    return {"case": case, "lens": _int(lens), "new": _int(news), "table": table, "free": free,
            "free_count": _int([pages - sum(held)]), "lens_out": e(n), "free_count_out": e(1), "q_start": e(n + 1),
            "positions": e(max_tokens), "slots": e(max_tokens), "admitted": e(n)}


def _prepare_store(case, g, seed):
    lens, news = _spread(case)
    page, h, d = case["page"], case["kv_heads"], case["head_dim"]
    lens = [length % page for length in lens]  # the pages before the last one are not touched: the pool holds the others
    blocks = [-(-(length + new) // page) for length, new in zip(lens, news)]
    table, _ = _table(blocks, max(blocks), sum(blocks), g)
    tokens = sum(news)
    seq = torch.repeat_interleave(torch.arange(len(news), device="cuda"), _int(news), output_size=tokens)
    at = torch.arange(tokens, device="cuda") - (torch.cumsum(_int(news), 0) - _int(news))[seq] + _int(lens)[seq]
    slots = table[seq, at // page] * page + (at % page).to(torch.int32)
    dtype = torch.float32 if case["dtype"] == "f32" else torch.float16
    row = 3 * h * d if case["fused_rows"] else h * d
    # K has a few channels far larger than the others, as trained models do
    size = torch.ones(row, device="cuda")
    size[::37] = 6.0
    k = (torch.randn(tokens, row, generator=g, device="cuda") * size).to(dtype)
    v = k[:, h * d:] if case["fused_rows"] else torch.randn(tokens, row, generator=g, device="cuda").to(dtype)
    codes = torch.stack([_codes((sum(blocks), h, page, d), case["cache"], g).view(torch.uint8) for _ in range(2)])
    scale = torch.rand((2, sum(blocks), h), generator=g, device="cuda") * (0.02 if case["cache"] == "int8" else 0.006) + 0.005
    return {"case": case, "k": k[:, : h * d], "v": v[:, : h * d], "ld": row, "slots": slots.contiguous(), "codes": codes,
            "scale": scale}


def _prepare_attend(case, g, seed):
    lens, news = _spread(case)
    total = [length + new for length, new in zip(lens, news)]
    page, h, d = case["page"], case["kv_heads"], case["head_dim"]
    blocks = [-(-t // page) for t in total]
    pages = sum(blocks)
    table, _ = _table(blocks, max(blocks), pages, g)
    codes = torch.empty((2, pages, h, page, d), dtype=torch.uint8, device="cuda")
    for c in codes:
        c.copy_(_codes((pages, h, page, d), case["cache"], g).view(torch.uint8))
    scale = (0.5 + torch.rand((2, pages, h), generator=g, device="cuda")) / (36 if case["cache"] == "int8" else 128)
    dtype = torch.float32 if case["dtype"] == "f32" else torch.float16
    q = (torch.randn(sum(news), case["heads"] * d, generator=g, device="cuda") * 2).to(dtype)
    start = [0]
    for new in news:
        start.append(start[-1] + new)
    return {"case": case, "q": q, "out": torch.zeros_like(q), "codes": codes, "scale": scale, "table": table,
            "kv_lens": _int(total), "q_start": _int(start), "max_q": max(news), "max_kv": max(total)}


def _prepare_sample(case, g, seed):
    rows, vocab, which = case["rows"], case["vocab"], case["which"]
    u = lambda lo, hi: lo + (hi - lo) * torch.rand(rows, generator=g, device="cuda")  # noqa: E731
    # a bulk of logits and a few words that the model thinks likely; some rows are flatter than others
    x = torch.randn(rows, vocab, generator=g, device="cuda") * u(0.5, 3.0)[:, None]
    likely = torch.randint(0, vocab, (rows, 64), generator=g, device="cuda")
    x.scatter_add_(1, likely, torch.randn(rows, 64, generator=g, device="cuda") * 4 + 4)
    pick = torch.randint(0, 4, (4, rows), generator=g, device="cuda")
    temperature, top_k, top_p, min_p = u(0.6, 1.2), torch.zeros(rows), u(0.85, 0.98), torch.zeros(rows, device="cuda")
    if which == "chat":
        top_k = torch.full((rows,), 20)
    elif which == "top_k":
        top_k = 1 + (u(0, 1) ** 3 * min(1000, vocab - 1))
    elif which == "mixed":
        temperature = torch.where(pick[0] == 0, torch.zeros(rows, device="cuda"), temperature)
        top_k = torch.where(pick[1] < 2, torch.zeros(rows, device="cuda"), 1 + u(0, 100))
        top_p = torch.where(pick[2] == 0, torch.ones(rows, device="cuda"), top_p)
        min_p = torch.where(pick[3] == 0, u(0.01, 0.1), min_p)
    return {"case": case, "x": x, "temperature": temperature.cuda(), "top_k": top_k.to("cuda", torch.int32),
            "top_p": top_p, "min_p": min_p, "u": u(0, 1), "out": torch.empty(rows, dtype=torch.int32, device="cuda")}


# ------------------------------------------------------------------ one pass

def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"plan": _own_plan, "store": _own_store, "attend": _own_attend, "sample": _own_sample}[kind](state)
    return {"plan": _plain_plan, "store": _plain_store, "attend": _plain_attend, "sample": _plain_sample}[kind](state)


def _planned(s, **outputs):
    return {"table": s["table"], "free": s["free"], **outputs}


def _plain_plan(s):
    page, lens, new, table, free = s["case"]["page"], s["lens"].long(), s["new"].long(), s["table"], s["free"]
    batch, max_blocks, max_tokens = lens.numel(), table.shape[1], s["slots"].numel()
    ended, add = new < 0, new.clamp(min=0)
    held = (lens + page - 1) // page
    block = torch.arange(max_blocks, device="cuda")
    # the pages of ended sequences, in batch and block order, onto the stack
    back = torch.where(ended, held, 0)
    count = s["free_count"].long()
    put = (torch.cumsum(back, 0) - back)[:, None] + block + count
    put = torch.where(block < back[:, None], put, free.numel())
    stack = torch.cat([free, free[:1]])  # the entry behind the stack takes what is not put back
    stack = stack.scatter(0, put.flatten().clamp(max=free.numel()), table.flatten())[:-1]
    count = count + back.sum()
    # the pages that the others need
    q_end = torch.cumsum(add, 0)
    after = (lens + add + page - 1) // page
    fits = ~ended & (after <= max_blocks) & (q_end <= max_tokens)
    need = torch.where(fits, after - held, 0)
    upto = torch.cumsum(need, 0)
    admitted = fits & ((need == 0) | (upto <= count))
    taken = torch.where(admitted, need, 0)
    nth = (upto - need)[:, None] + block - held[:, None]
    fresh = (block >= held[:, None]) & (block < (held + taken)[:, None])
    table.copy_(torch.where(fresh, stack[(count - 1 - nth).clamp(0, free.numel() - 1)], table))
    free.copy_(stack)
    # every token's sequence, position and slot
    t = torch.arange(max_tokens, device="cuda")
    seq = torch.searchsorted(q_end, t, right=True).clamp(max=batch - 1)
    inside = t < q_end[-1]
    position = torch.where(inside, lens[seq] + t - (q_end - add)[seq], 0)
    at = table[seq, (position // page).clamp(max=max_blocks - 1)].long() * page + position % page
    return _planned(
        s, lens=torch.where(ended, 0, torch.where(admitted, lens + add, lens)).int(),
        free_count=(count - taken.sum()).int(), q_start=torch.cat([torch.zeros_like(q_end[:1]), q_end]).int(),
        positions=position.int(), slots=torch.where(inside & admitted[seq], at, -1).int(), admitted=(admitted | ended).int())


def _own_plan(s):
    F = _fence()
    p = {k: v.data_ptr() for k, v in s.items() if k != "case"}
    F.kv_plan(p["lens_out"], p["lens"], p["new"], s["lens"].numel(), p["table"], s["table"].shape[1], s["case"]["page"],
              p["free"], p["free_count_out"], p["free_count"], s["free"].numel(), p["q_start"], p["positions"],
              p["slots"], s["slots"].numel(), p["admitted"], torch.cuda.current_stream().cuda_stream)
    return _planned(s, lens=s["lens_out"], free_count=s["free_count_out"], q_start=s["q_start"], positions=s["positions"],
                    slots=s["slots"], admitted=s["admitted"])


def _values(s):
    """What a cache of codes and scales stands for, beside the scales."""
    codes = s["codes"].view(torch.int8 if s["case"]["cache"] == "int8" else torch.float8_e4m3fn)
    if s["case"]["cache"] != "int8":
        codes = codes.to(torch.float32)
    return {"values": codes * s["scale"][..., None, None], "scale": s["scale"]}


def _nearest(y, cache):
    """y, in 64 bits, rounded to the values that a code can hold."""
    if cache == "int8":
        return y.round()
    step = torch.exp2(torch.frexp(y)[1].clamp(min=-5).double() - 4)  # 3 bits behind the first; 2^-9 at the least
    return (y / step).round() * step


def _plain_store(s):
    c = s["case"]
    page, h, d, top = c["page"], c["kv_heads"], c["head_dim"], 127.0 if c["cache"] == "int8" else 448.0
    pages, slots = s["scale"].shape[1], s["slots"].long()
    x = torch.stack([s["k"].unflatten(1, (h, d)), s["v"].unflatten(1, (h, d))]).float()  # [2][tokens][h][d]
    at, where = slots // page, slots % page
    first = torch.full((pages,), page, device="cuda").scatter_reduce(0, at, where, "amin")  # where the new tokens begin
    most = torch.zeros((2, pages, h), device="cuda")
    most.scatter_reduce_(1, at[None, :, None].expand(2, -1, h), x.abs().amax(3), "amax")
    old = torch.where((first > 0)[None, :, None], s["scale"], torch.zeros_like(s["scale"]))
    touched = (first < page)[None, :, None]
    scale = torch.where(touched, torch.maximum(old, (most.double() / top).float()), s["scale"])
    codes = s["codes"].view(torch.int8 if c["cache"] == "int8" else torch.float8_e4m3fn)
    # what the touched pages held before the new tokens, at the new scale
    held = torch.arange(page, device="cuda")[None, :] < first[:, None]
    grown = (touched & (scale > old))[..., None, None] & held[None, :, None, :, None]
    ratio = (old.double() / scale.double()).nan_to_num(0.0)
    again = codes.double() * old.double()[..., None, None] / scale.double()[..., None, None]
    again = _nearest(torch.where((ratio > 0)[..., None, None], again, 0.0), c["cache"])
    new = torch.where(grown, again, codes.double())
    # the new tokens
    over = scale.double()[:, at][..., None]
    y = _nearest(torch.where(over > 0, x.double() / over, 0.0).clamp(-top, top), c["cache"])
    new[:, at, :, where] = y.transpose(0, 1)
    s["codes"].copy_(new.float().to(codes.dtype).view(torch.uint8))
    s["scale"].copy_(scale)
    return _values(s)


def _pages(F, s):
    c, pages = s["case"], s["scale"].shape[1]
    k, v = s["codes"][0].data_ptr(), s["codes"][1].data_ptr()
    return F.kv_pages(k, v, s["scale"][0].data_ptr(), s["scale"][1].data_ptr(), pages, c["page"], c["kv_heads"], c["head_dim"],
                      F.KV_INT8 if c["cache"] == "int8" else F.KV_E4M3)


def _own_store(s):
    F = _fence()
    F.store_kv_q8(_pages(F, s), s["k"].data_ptr(), s["v"].data_ptr(), F.F32 if s["case"]["dtype"] == "f32" else F.F16,
                  s["ld"], s["slots"].data_ptr(), s["slots"].numel(), torch.cuda.current_stream().cuda_stream)
    return _values(s)


def _plain_attend(s):
    c = s["case"]
    page, h, d, group = c["page"], c["kv_heads"], c["head_dim"], c["heads"] // c["kv_heads"]
    batch, lq, blocks = s["table"].shape[0], s["max_q"], s["table"].shape[1]
    codes = s["codes"].view(torch.int8 if c["cache"] == "int8" else torch.float8_e4m3fn)
    table = s["table"].long()

    def dense(i):  # [batch][h][blocks * page][d]
        x = codes[i].view(torch.uint8)[table].view(codes.dtype).float() * s["scale"][i][table][..., None, None]
        return x.transpose(1, 2).reshape(batch, h, blocks * page, d)

    start, q_len = s["q_start"][:-1].long(), s["q_start"].long().diff()
    i = torch.arange(lq, device="cuda")
    rows = (start[:, None] + i).clamp(max=s["q"].shape[0] - 1)
    q = s["q"][rows].float().reshape(batch, lq, h, group, d).permute(0, 2, 1, 3, 4).reshape(batch, h, lq * group, d)
    scores = torch.matmul(q * (1.0 / math.sqrt(d)), dense(0).transpose(2, 3).contiguous())
    see = s["kv_lens"].long()[:, None] - q_len[:, None] + i + 1  # positions that query i sees
    hidden = torch.arange(blocks * page, device="cuda") >= torch.minimum(see, s["kv_lens"].long()[:, None])[..., None]
    hidden = hidden[:, None, :, None, :].expand(-1, 1, -1, group, -1).reshape(batch, 1, lq * group, blocks * page)
    scores.masked_fill_(hidden, -math.inf)
    most = scores.amax(3, keepdim=True).clamp(min=-1e30)
    scores.sub_(most).exp_()
    total = scores.sum(3, keepdim=True)
    o = torch.matmul(scores, dense(1)) / torch.where(total > 0, total, 1.0)
    o = o.reshape(batch, h, lq, group, d).permute(0, 2, 1, 3, 4).reshape(batch, lq, h * group * d)
    here = i < q_len[:, None]
    # rows that are no query of any sequence go to a row behind the last
    to = torch.where(here, start[:, None] + i, s["q"].shape[0])
    out = torch.empty(s["q"].shape[0] + 1, h * group * d, device="cuda", dtype=s["q"].dtype)
    out[to.flatten()] = o.flatten(0, 1).to(out.dtype)
    return out[:-1]


def _own_attend(s):
    F, c = _fence(), s["case"]
    if "workspace" not in s:
        size = F.gqa_attention_q8_workspace(s["table"].shape[0], s["max_q"], c["heads"], c["kv_heads"], c["head_dim"])
        s["workspace"] = torch.empty(size, dtype=torch.uint8, device="cuda")
    F.gqa_attention_q8(s["out"].data_ptr(), s["q"].data_ptr(), F.F32 if c["dtype"] == "f32" else F.F16, s["q"].shape[1],
                       s["out"].shape[1], _pages(F, s), s["table"].data_ptr(), s["table"].shape[1], s["kv_lens"].data_ptr(),
                       s["q_start"].data_ptr(), s["table"].shape[0], s["max_q"], c["heads"], s["workspace"].data_ptr(),
                       s["workspace"].numel(), torch.cuda.current_stream().cuda_stream)
    return s["out"]


def _plain_sample(s):
    # in 64 bits: a sum of 150,000 weights is compared with borders that lie close together
    x, at = torch.sort(s["x"], dim=1, descending=True, stable=True)
    greedy = s["temperature"] <= 0
    t = torch.where(greedy, 1.0, s["temperature"]).double()[:, None]
    w = ((x.double() - x[:, :1].double()) / t).exp()
    rank = torch.arange(x.shape[1], device="cuda")
    k = torch.where((s["top_k"] <= 0) | (s["top_k"] > x.shape[1]), x.shape[1], s["top_k"])[:, None]
    k = torch.where(greedy[:, None], 1, k)
    w = torch.where(rank < k, w, 0.0)
    run_ = w.cumsum(1)
    total = run_[:, -1:]
    # the sum before a token is under top_p: the token belongs to the shortest beginning that reaches it
    inside = ((run_ - w) < s["top_p"].double()[:, None] * total) | (s["top_p"] >= 1)[:, None] | (rank == 0)
    kept = torch.where(inside & (w >= s["min_p"].double()[:, None]), w, 0.0)
    run_ = kept.cumsum(1)
    passed = run_ > s["u"].double()[:, None] * run_[:, -1:]
    return at.gather(1, passed.int().argmax(1, keepdim=True))[:, 0].int()


def _own_sample(s):
    F, (rows, vocab) = _fence(), s["x"].shape
    if "workspace" not in s:
        s["workspace"] = torch.empty(F.sample_workspace(rows, vocab), dtype=torch.uint8, device="cuda")
    F.sample(s["out"].data_ptr(), s["x"].data_ptr(), rows, vocab, vocab, s["temperature"].data_ptr(), s["top_k"].data_ptr(),
             s["top_p"].data_ptr(), s["min_p"].data_ptr(), s["u"].data_ptr(), s["workspace"].data_ptr(), s["workspace"].numel(),
             torch.cuda.current_stream().cuda_stream)
    return s["out"]


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    kind = case["kind"]
    if kind == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": 4 * n + 24 * case["rows"], "flops": 4 * n}
    lens, news = _spread(case)
    page, tokens = case["page"], sum(news)
    if kind == "plan":
        # lengths in and out, the pages taken off the stack and into the table, three words a token
        taken = sum(-(-(n + m) // page) - -(-n // page) for n, m in zip(lens, news))
        return {"bytes": 4 * (5 * case["batch"] + 3 * taken + 2 * tokens), "flops": 0}
    h, d, size = case["kv_heads"], case["head_dim"], 4 if case["dtype"] == "f32" else 2
    if kind == "store":
        # K and V in, their codes and scales out, and the codes and scales read again as the values they stand for
        held = sum(-(-(n % page + m) // page) for n, m in zip(lens, news)) * page
        return {"bytes": 2 * h * d * (tokens * (size + 1) + held * 5) + 8 * tokens, "flops": 0}
    cached = sum(n + m for n, m in zip(lens, news))
    pairs = sum(m * n + m * (m + 1) // 2 for n, m in zip(lens, news))
    return {"bytes": 2 * h * d * cached + 2 * size * tokens * case["heads"] * d, "flops": 4 * case["heads"] * d * pairs}


# ------------------------------------------------------------------ the definitions in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return {"plan": _exact_plan, "store": _exact_store, "attend": _exact_attend, "sample": _exact_sample}[case["kind"]](case, s)


def _exact_plan(case, s):
    """Sequence by sequence, on lists."""
    page, lens, new = case["page"], s["lens"].tolist(), s["new"].tolist()
    table, free, count = s["table"].tolist(), s["free"].tolist(), int(s["free_count"])
    size, max_tokens = len(table[0]), s["slots"].numel()
    for b, n in enumerate(lens):
        if new[b] < 0:
            for j in range(-(-n // page)):
                free[count] = table[b][j]
                count += 1
    q_start, positions, slots, admitted, upto, left = [0], [], [], [], 0, count
    for b, n in enumerate(list(lens)):
        m = max(0, new[b])
        q_start.append(q_start[-1] + m)
        held, after = -(-n // page), -(-(n + m) // page)
        ok = new[b] >= 0 and after <= size and q_start[-1] <= max_tokens
        if ok:
            upto += after - held
            ok = after == held or upto <= count
        if ok:
            for j in range(held, after):
                table[b][j] = free[count - 1 - (upto - (after - held)) - (j - held)]
                left -= 1
        admitted.append(int(ok or new[b] < 0))
        positions += [n + i for i in range(m)]
        slots += [table[b][(n + i) // page] * page + (n + i) % page if ok else -1 for i in range(m)]
        lens[b] = 0 if new[b] < 0 else n + m if ok else n
    pad = max_tokens - len(slots)
    return {"table": _int(table), "free": _int(free), "lens": _int(lens), "free_count": _int([left]), "q_start": _int(q_start),
            "positions": _int(positions + [0] * pad), "slots": _int(slots + [-1] * pad), "admitted": _int(admitted)}


def _exact_store(case, s):
    """Page by page."""
    page, int8 = case["page"], case["cache"] == "int8"
    h, d, top = case["kv_heads"], case["head_dim"], 127.0 if int8 else 448.0
    values = np.array(sorted({m * 2.0 ** (e - 3) for e in range(-6, 9) for m in range(8, 16)} | {m * 2.0 ** -9 for m in range(8)}))
    values = torch.from_numpy(values[values <= 448]).cuda()
    between = (values[1:] + values[:-1]) / 2

    def nearest(y):
        if int8:
            return torch.round(y)
        a = y.abs()
        i = torch.bucketize(a, between)  # a tie comes to the lower one
        tie = (a == between[i.clamp(max=between.numel() - 1)]) & (i % 2 == 1) & (i < between.numel())
        return values[i + tie.long()] * torch.sign(y)

    slots = s["slots"].tolist()
    codes = s["codes"].view(torch.int8 if int8 else torch.float8_e4m3fn).double()
    scale, given = s["scale"].double(), s["scale"].clone()
    t = 0
    while t < len(slots):
        p, off = divmod(slots[t], page)
        n = 1
        while t + n < len(slots) and slots[t + n] == slots[t] + n and off + n < page:
            n += 1
        for i, name in enumerate("kv"):
            x = s[name][t: t + n].double().reshape(n, h, d).transpose(0, 1)
            old = given[i, p].double() if off else torch.zeros(h, dtype=torch.float64, device="cuda")
            new = torch.maximum(old, (x.abs().amax((1, 2)) / top).float().double())
            scale[i, p] = new
            over = torch.where(new > 0, new, 1.0)[:, None, None]
            before = codes[i, p, :, :off]
            codes[i, p, :, :off] = torch.where((new > old)[:, None, None], nearest(before * old[:, None, None] / over), before)
            codes[i, p, :, off: off + n] = nearest((x / over).clamp(-top, top))
        t += n
    return {"values": codes * scale[..., None, None], "scale": scale}


def _exact_attend(case, s):
    """Sequence by sequence and head by head, a few thousand queries' products at a time."""
    page, d, group = case["page"], case["head_dim"], case["heads"] // case["kv_heads"]
    if work(case)["flops"] > 2e12:
        return None
    codes = s["codes"].view(torch.int8 if case["cache"] == "int8" else torch.float8_e4m3fn)
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    start, kv_lens = s["q_start"].tolist(), s["kv_lens"].tolist()
    for b, n in enumerate(kv_lens):
        pages = s["table"][b, : -(-n // page)].long()
        m = start[b + 1] - start[b]
        for j in range(case["kv_heads"]):
            k, v = ((codes[i].view(torch.uint8)[pages, j].view(codes.dtype).double() * s["scale"][i][pages, j].double()[:, None, None])
                    .reshape(-1, d)[:n] for i in range(2))
            for q0 in range(0, m, 1024):
                rows = slice(start[b] + q0, min(start[b] + q0 + 1024, start[b + 1]))
                q = s["q"][rows].double().reshape(-1, case["heads"], d)[:, j * group: (j + 1) * group]
                i = torch.arange(q0, q0 + q.shape[0], device="cuda")
                score = (q.reshape(-1, d) @ k.T / math.sqrt(d)).reshape(q.shape[0], group, n)
                score.masked_fill_((torch.arange(n, device="cuda") > (n - m + i)[:, None])[:, None], -math.inf)
                p = torch.softmax(score, 2)
                out[rows].view(-1, case["heads"], d)[:, j * group: (j + 1) * group] = (p.reshape(-1, n) @ v).reshape(q.shape)
    return out


def _exact_sample(case, s):
    """Row by row, on the host."""
    x, got = s["x"].cpu().numpy().astype(np.float64), []
    par = {k: s[k].cpu().numpy().astype(np.float64) for k in ("temperature", "top_k", "top_p", "min_p", "u")}
    for r in range(x.shape[0]):
        t, k = par["temperature"][r], int(par["top_k"][r])
        if t <= 0:
            got.append(int(np.argmax(x[r])))
            continue
        order = np.argsort(-x[r], kind="stable")
        order = order[:k] if k > 0 else order
        w = np.exp((x[r][order] - x[r][order[0]]) / t)
        if par["top_p"][r] < 1:
            order = order[: 1 + int(np.searchsorted(np.cumsum(w), par["top_p"][r] * w.sum(), side="left"))]
        w = w[: len(order)]
        w = w[w >= par["min_p"][r]]
        got.append(int(order[int(np.searchsorted(np.cumsum(w), par["u"][r] * w.sum(), side="right"))]))
    return torch.tensor(got, dtype=torch.int32)
