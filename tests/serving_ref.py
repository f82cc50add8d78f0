"""The operators of a batched step over a paged 8-bit cache, in numpy and 64
bits: fence_kv_plan, fence_store_kv_q8, fence_gqa_attention_q8, fence_sample."""
from __future__ import annotations

import numpy as np

INT8, E4M3 = 0, 1
TOP = (127.0, 448.0)

# the values of e4m3 codes 0..127 (127 is NaN)
E4M3_VALUES = np.array([m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10) for e in range(16) for m in range(8)])
E4M3_VALUES[127] = np.nan


def decode(codes, cache):
    """uint8 codes -> float64."""
    if cache == INT8:
        return codes.view(np.int8).astype(np.float64)
    return np.where(codes & 128, -1.0, 1.0) * E4M3_VALUES[codes & 127]


def encode(y, cache):
    """float64 -> uint8 codes, nearest, ties to even."""
    if cache == INT8:
        return np.clip(np.rint(y), -127, 127).astype(np.int8).view(np.uint8)
    a = np.minimum(np.abs(y), 448.0)
    hi = np.searchsorted(E4M3_VALUES[:127], a, side="left").clip(0, 126)  # the first value not below a
    lo = np.maximum(hi - 1, 0)
    up, down = E4M3_VALUES[hi] - a, a - E4M3_VALUES[lo]
    code = np.where(up < down, hi, np.where(up > down, lo, np.where(hi % 2 == 0, hi, lo)))
    code = np.where(E4M3_VALUES[hi] == a, hi, code)
    return (code | np.where(np.signbit(y), 128, 0)).astype(np.uint8)


def plan(lens, new, table, page, free, count, max_tokens):
    """Sequence by sequence; table and free are changed in place."""
    lens, out = list(lens), {}
    n_pages, blocks = len(free), table.shape[1]
    count = min(max(count, 0), n_pages)
    for b, n in enumerate(lens):
        if new[b] < 0:
            for j in range(min(-(-max(n, 0) // page), blocks)):
                if count < n_pages:
                    free[count] = table[b, j]
                    count += 1
    q_start, pos, slots, admitted, upto, left = [0], [], [], [], 0, count
    for b, n in enumerate(list(lens)):
        n = max(n, 0)
        m = max(int(new[b]), 0)
        q_start.append(q_start[-1] + m)
        held, after = -(-n // page), -(-(n + m) // page)
        ok = new[b] >= 0 and after <= blocks and q_start[-1] <= max_tokens
        if ok:
            upto += after - held
            ok = after == held or upto <= count
        if ok:
            for j in range(held, after):
                left -= 1
                table[b, j] = free[left]
        admitted.append(int(ok or new[b] < 0))
        for i in range(m):
            pos.append(n + i)
            slots.append(table[b, (n + i) // page] * page + (n + i) % page if ok else -1)
        lens[b] = 0 if new[b] < 0 else n + m if ok else n
    pos, slots = pos[:max_tokens], slots[:max_tokens]
    pad = max_tokens - len(pos)
    return {"lens": lens, "count": left, "q_start": q_start, "positions": pos + [0] * pad, "slots": slots + [-1] * pad,
            "admitted": admitted}


def store(codes, scale, x, slots, cache):
    """codes [pages][heads][page][d] uint8 and scale [pages][heads] float32 of K or V, changed in place; x
    [tokens][heads][d], slots [tokens]."""
    pages, heads, page, d = codes.shape
    t = 0
    while t < len(slots):
        s = int(slots[t])
        if s < 0 or s >= pages * page:
            t += 1
            continue
        p, off = divmod(s, page)
        n = 1
        while t + n < len(slots) and off + n < page and slots[t + n] == s + n:
            n += 1
        for h in range(heads):
            v = x[t:t + n, h].astype(np.float64)
            with np.errstate(invalid="ignore"):
                mine = np.float32(np.max(np.abs(v)) / TOP[cache])  # NaN if any is
            old = np.float32(scale[p, h]) if off else np.float32(0)
            new = np.float32(np.nan) if np.isnan(old) or np.isnan(mine) else max(old, mine)
            if off and new > old:
                was = decode(codes[p, h, :off], cache) * np.float64(old)
                codes[p, h, :off] = encode(was / np.float64(new) if np.isfinite(new) else was * 0, cache)
            ok = np.isfinite(new) and new > 0
            codes[p, h, off:off + n] = encode(v / np.float64(new), cache) if ok else 0
            scale[p, h] = new
        t += n


def attention(q, codes, scale, table, kv_lens, q_start, cache, max_q=None):
    """q [rows][heads][d]; codes (k, v), scale (k, v).  Returns the output (NaN in rows of no sequence) and what a
    tolerance is made of: sum_j p_j |v_j| per output and max_j sum_i |q_i k_ji| * scale per row and head."""
    rows, heads, d = q.shape
    pages, kvh, page, _ = codes[0].shape
    group, out = heads // kvh, np.full((rows, heads, d), np.nan)
    spread, big = np.zeros((rows, heads, d)), np.zeros((rows, heads, 1))
    for b in range(len(kv_lens)):
        m = max(q_start[b + 1] - q_start[b], 0)
        n = min(max(int(kv_lens[b]), 0), table.shape[1] * page)
        ids = table[b, : -(-n // page)]
        there = np.repeat((ids >= 0) & (ids < pages), page)[:n]
        ids = np.where((ids >= 0) & (ids < pages), ids, 0)
        for h in range(kvh):
            with np.errstate(invalid="ignore"):
                k, v = ((decode(codes[i][ids, h], cache) * scale[i][ids, h].astype(np.float64)[:, None, None])
                        .reshape(-1, d)[:n] for i in range(2))
            for i in range(min(m, max_q) if max_q is not None else m):
                r, see = q_start[b] + i, there & (np.arange(n) < n - m + i + 1)
                if not see.any():
                    out[r, h * group:(h + 1) * group] = 0.0
                    continue
                qq = q[r, h * group:(h + 1) * group].astype(np.float64)
                with np.errstate(invalid="ignore", over="ignore"):
                    s = qq @ k[see].T / np.sqrt(d)
                    p = np.exp(s - s.max(1, keepdims=True))
                    p /= p.sum(1, keepdims=True)
                    out[r, h * group:(h + 1) * group] = p @ v[see]
                    spread[r, h * group:(h + 1) * group] = p @ np.abs(v[see])
                    big[r, h * group:(h + 1) * group, 0] = (np.abs(qq) @ np.abs(k[see]).T).max(1) / np.sqrt(d)
    return out, spread, big


def sample(x, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, u=0.0):
    """One row of float32 logits."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    f = lambda v: float(np.float32(v))  # noqa: E731
    temperature, top_p, min_p, u = f(temperature), f(top_p), f(min_p), f(u)
    if x.max() == -np.inf:
        return 0
    if not temperature > 0:
        return int(np.argmax(x))
    order = np.argsort(-x, kind="stable")
    if 0 < top_k < len(x):
        order = order[:top_k]
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.exp((x[order] - x[order[0]]) / temperature)
    if x[order[0]] == np.inf:
        w = np.where(x[order] == np.inf, 1.0, 0.0)
    if top_p < 1:
        w = w[: 1 + int(np.searchsorted(np.cumsum(w), max(top_p, 0.0) * np.cumsum(w)[-1], side="left"))]
    if min_p > 0:
        w = w[w >= min(min_p, 1.0)]
    at = int(np.searchsorted(np.cumsum(w), min(max(u, 0.0), 1.0) * np.cumsum(w)[-1], side="right"))
    return int(order[min(at, int(np.flatnonzero(w)[-1]))])
