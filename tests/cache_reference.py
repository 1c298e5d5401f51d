"""The cache operators in 64 bits, from their definitions (include/pmkl_cache.h): plain loops over requests, runs and
heads on the CPU, and the bounds of the device results against them."""
from __future__ import annotations

import numpy as np

HALF_STEP = {"fp32": 2.0 ** -24, "fp16": 2.0 ** -11, "bf16": 2.0 ** -8}


def _table():
    codes = np.arange(256)
    sign = np.where(codes & 0x80, -1.0, 1.0)
    exponent, mantissa = (codes >> 3) & 15, codes & 7
    value = np.where(exponent > 0, (1 + mantissa / 8) * 2.0 ** (exponent - 7), mantissa * 2.0 ** -9)
    return np.where((codes & 0x7f) == 0x7f, np.nan, sign * value)


E4M3 = _table()
_FINITE = E4M3[:127]   # codes 0 .. 0x7e, ascending


def encode(x):
    """e4m3 codes of float64 values of magnitude 448 at most: the nearest, ties to the even code; NaN as 0x7f."""
    x = np.asarray(x, dtype=np.float64)
    a = np.abs(np.where(np.isnan(x), 0.0, x))
    assert (a <= 448).all()
    hi = np.searchsorted(_FINITE, a).clip(0, 126)
    lo = np.maximum(hi - 1, 0)
    low, high = a - _FINITE[lo], _FINITE[hi] - a
    code = np.where(low < high, lo, np.where(high < low, hi, np.where(lo % 2 == 0, lo, hi)))
    code = np.where(_FINITE[hi] == a, hi, code)
    return np.where(np.isnan(x), 0x7f, code | np.where(np.signbit(x), 0x80, 0)).astype(np.uint8)


def need(largest):
    """The least power of two from 2^-126 on under which `largest` is at most 448."""
    e = -126
    while largest > 448 * 2.0 ** e:
        e += 1
    return 2.0 ** e


def slots(cached, new, table, free, head, page_size, tokens):
    """seq_lens, query_start, slots, free_head and the table after the call (a copy)."""
    table = table.copy()
    width = table.shape[1]
    rows = []
    starts = [0]
    seq_lens = []
    for b, (c, n) in enumerate(zip(cached, new)):
        c, n = max(int(c), 0), max(int(n), 0)
        for w in range(min(-(-c // page_size), width), min(-(-(c + n) // page_size), width)):
            table[b, w] = free[head] if 0 <= head < len(free) else -1
            head += 1
        for at in range(c, c + n):
            w = at // page_size
            page = int(table[b, w]) if w < width else -1
            rows.append(-1 if page < 0 else page * page_size + at % page_size)
        starts.append(starts[-1] + n)
        seq_lens.append(c + n)
    rows = (rows + [-1] * tokens)[:tokens]
    return np.array(seq_lens), np.array(starts), np.array(rows), head, table


def append(k, v, slot, k_codes, v_codes, k_scale, v_scale):
    """The four arrays of the cache after the call (copies).  k, v: float64 [N, H, D]; codes uint8.  Quotients and products
    are single fp32 operations, as the definition has them (by a power of two they are exact)."""
    page_size = k_codes.shape[2]
    caches = [(k, k_codes.copy(), k_scale.astype(np.float64)), (v, v_codes.copy().swapaxes(2, 3), v_scale.astype(np.float64))]
    t = 0
    while t < len(slot):
        if not 0 <= slot[t] < k_codes.shape[0] * page_size:
            t += 1
            continue
        page, first = divmod(int(slot[t]), page_size)
        n = 1
        while t + n < len(slot) and slot[t + n] == slot[t] + n and first + n < page_size:
            n += 1
        for x, codes, scale in caches:
            for h in range(x.shape[1]):
                run = x[t:t + n, h]
                largest = np.abs(run[np.isfinite(run)]).max(initial=0.0)
                was, now = scale[page, h], need(largest)
                if first and was > 0 and np.isfinite(was):
                    now = max(was, now)
                    if now != was:
                        codes[page, h, :first] = encode(
                            E4M3[codes[page, h, :first]].astype(np.float32) * (np.float32(was) / np.float32(now)))
                codes[page, h, first:first + n] = encode(
                    np.where(np.isfinite(run), run, np.nan).astype(np.float32) / np.float32(now))
                scale[page, h] = now
        t += n
    return caches[0][1], caches[1][1].swapaxes(2, 3), caches[0][2], caches[1][2]


def attend(q, k_codes, v_codes, k_scale, v_scale, table, seq_lens, query_start, causal, scale, dtype):
    """out, m, l in float64 and the bounds of their errors, all [N, heads(, D)]; rows of no request are NaN with a bound of
    -1.

    Bounds.  A score is a sum of D products in fp32, of terms that hold q and k exactly, times three fp32 factors: off by at
    most ds = (D + 8) 2^-24 scale sum_d |q_d k_d| (its largest over the row's keys).  A weight exp(s - m) is off by 2 ds
    (s and m) and by 2^-21 (the exponent's rounding for |s - m| < 8, larger differences weigh less; exp2; the factor of the
    values' scale), and by the rounding of its f16 terms.  A term has 11 significant bits, so it is off by at most half of
    its last one, 2^-11 of itself: under bf16 queries, with one term, each w_j v_j is off by 2^-11 |w_j v_j|, and the
    ratio by 2^-11 sum w |v| / sum w (an eighth of a bf16 output's own half step, 2^-8); with two terms by 2^-22.  Sums over L keys are made of at
    most L / 32 + 64 additions to one accumulator, each off by 2^-24 of the sum of magnitudes.  The output is a ratio of two
    such sums, rounded once: by half a step of its type, which for numbers below fp16's least normal one, 2^-14, is
    half of its least step of 2^-24 (bf16's and fp32's are below 1e-30, which stands for them)."""
    n_tokens, heads, D = q.shape
    page_size, kv_heads = k_codes.shape[2], k_codes.shape[1]
    group = heads // kv_heads
    out = np.full(q.shape, np.nan)
    m, l = np.full(q.shape[:2], np.nan), np.full(q.shape[:2], np.nan)
    out_bound, m_bound, l_bound = np.full(q.shape, -1.0), np.full(m.shape, -1.0), np.full(m.shape, -1.0)
    terms = 2.0 ** -11 if dtype == "bf16" else 2.0 ** -22
    for b in range(len(seq_lens)):
        lo, hi = int(query_start[b]), int(query_start[b + 1])
        keys = min(int(seq_lens[b]), table.shape[1] * page_size)
        at = np.arange(keys)
        page = table[b, at // page_size]
        held = (page >= 0) & (page < k_codes.shape[0])
        page = np.where(held, page, 0)
        if lo == hi:
            continue
        position = int(seq_lens[b]) - (hi - lo) + np.arange(hi - lo)
        seen = held & ((at <= position[:, None]) if causal else np.ones((hi - lo, keys), bool))
        some = seen.any(1)
        for h in range(heads):
            g = h // group
            kk = E4M3[k_codes[page, g, at % page_size]] * k_scale[page, g][:, None].astype(np.float64)
            vv = E4M3[v_codes[page, g, :, at % page_size]] * v_scale[page, g][:, None].astype(np.float64)
            rows = slice(lo, hi)
            s = np.where(seen, scale * (q[rows, h] @ kk.T), -np.inf)
            mx = s.max(1, initial=-np.inf)
            p = np.exp(s - np.where(some, mx, 0.0)[:, None])
            total = p.sum(1)
            # a NaN value reaches the rows that see its token, hidden ones (p = 0) none
            bad = (seen.astype(float) @ np.isnan(vv)) > 0
            vv = np.nan_to_num(vv, nan=0.0)
            safe = np.where(some, total, 1.0)[:, None]
            out[rows, h] = np.where(bad, np.nan, p @ vv / safe)
            m[rows, h], l[rows, h] = mx, total
            size = scale * (np.abs(q[rows, h]) @ np.abs(kk).T)
            ds = (D + 8) * 2.0 ** -24 * np.where(seen, size, 0.0).max(1, initial=0.0)
            sums = (seen.sum(1) / 32 + 64) * 2.0 ** -24
            m_bound[rows, h] = np.where(some, ds + 2.0 ** -23 * np.abs(np.where(some, mx, 0.0)), 0.0)
            l_bound[rows, h] = total * (2 * ds + 2.0 ** -21 + sums)
            mean = p @ np.abs(vv) / safe
            out_bound[rows, h] = HALF_STEP[dtype] * np.abs(out[rows, h]) * 1.01 + \
                mean * (2 * (2 * ds + 2.0 ** -21 + sums) + terms)[:, None] + some[:, None] * (2.0 ** -25 if dtype == "fp16" else 1e-30)
    return (out, m, l), (out_bound, m_bound, l_bound)
