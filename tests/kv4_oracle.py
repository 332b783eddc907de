"""Plain 64-bit implementations of the 4-bit cache's format and attention, and of the page stack, for the tests.

Written from the definitions in include/sa_hip.h with element-by-element index formulas; numpy only."""
from __future__ import annotations

import numpy as np

PAGE = 32
LIMIT = 32000.0


# ---- the format ---------------------------------------------------------------

def places(d):
    """Byte and nibble of the codes and byte of the halves of token t, channel c: dict of [32][d] arrays."""
    ng, nc = d // 32, d // 16
    t, c = np.arange(PAGE)[:, None], np.arange(d)[None]
    T, j, i = t // 16, t // 4 % 4, t % 4
    g, n = c // 32, c % 8
    J = c % 32 // 8
    r, m = c // nc, c % nc
    full = lambda x: np.broadcast_to(x, (PAGE, d))
    return {"k": full(t * (d // 2) + (J * ng + g) * 4 + n // 2), "kn": full(n % 2),
            "v": full(16 * d + ((T * 4 + j) * 16 + r) * 2 * nc + i * (nc // 2) + m // 2), "vn": full(m % 2),
            "ks": full(32 * d + 2 * (((T * 4 + j) * ng + g) * 4 + i)), "km": full(34 * d + 2 * (t * ng + g)),
            "vs": full(36 * d + 2 * ((g * 4 + j) * 8 + 4 * T + i)), "vm": full(38 * d + 2 * ((g * 4 + j) * 8 + 4 * T + i))}


def quantise(x):
    """x [..., d] -> codes (int), scale and minimum [..., d] as float64, by the stated roundings."""
    with np.errstate(all="ignore"):
        x = np.asarray(x, np.float32)
        shape = x.shape
        x = np.clip(x, -LIMIT, LIMIT).astype(np.float32).reshape(*shape[:-1], shape[-1] // 32, 32)
        m = x.min(-1, keepdims=True).astype(np.float16).astype(np.float32) + np.float32(0)
        raw = (np.maximum(x.max(-1, keepdims=True) - m, np.float32(0)) / np.float32(15)).astype(np.float32)
        mant, e = np.frexp(raw.astype(np.float64))
        unit = np.exp2(np.maximum(e - 7, -24).astype(np.float64))
        s = np.where(raw > 0, np.ceil(raw.astype(np.float64) / unit) * unit, 0.0)
        q = ((x - m).astype(np.float32) / s.astype(np.float32)).astype(np.float32)
        code = np.clip(np.rint(q), 0, 15)
        nan = np.isnan(m)
        code = np.where((s > 0) & ~nan, code, 0.0)
        s = np.where(nan, 0.0, s)
    spread = lambda a: np.broadcast_to(a, x.shape).reshape(shape)
    return code.reshape(shape).astype(np.int64), spread(s).astype(np.float64), spread(m).astype(np.float64)


def values(x):
    code, s, m = quantise(x)
    return code * s + m


def put(pool, slot, k, v):
    """Writes a token's k, v [heads][d] into pool uint8 [pages][heads][40 d]."""
    d = k.shape[-1]
    at, t = places(d), slot % PAGE
    for h in range(k.shape[0]):
        rec = pool[slot // PAGE, h]
        for x, name in ((k[h], "k"), (v[h], "v")):
            code, s, m = quantise(x)
            for c in range(d):
                b, nib = at[name][t, c], at[name + "n"][t, c]
                rec[b] = (rec[b] & (0xF0 if nib == 0 else 0x0F)) | (int(code[c]) << (4 * nib))
            for c in range(0, d, 32):
                for half, name2 in ((s[c], "s"), (m[c], "m")):
                    b = at[name + name2][t, c]
                    rec[b:b + 2] = np.array([half], np.float16).view(np.uint8)


def read(pool):
    """Keys and values [pages][heads][32][d] float64 of pool uint8 [pages][heads][40 d]."""
    d = pool.shape[-1] // 40
    at = places(d)
    half = lambda b: (pool[..., b].astype(np.uint16) | (pool[..., b + 1].astype(np.uint16) << 8)).view(np.float16) \
        .astype(np.float64)
    code = lambda b, n: ((pool[..., b] >> (4 * n)) & 15).astype(np.float64)
    with np.errstate(all="ignore"):
        k = code(at["k"], at["kn"]) * half(at["ks"]) + half(at["km"])
        v = code(at["v"], at["vn"]) * half(at["vs"]) + half(at["vm"])
    return k, v


# ---- attention ------------------------------------------------------------------

def attend(q, k, v, scale):
    """q [rows][d], k, v [tokens][d] float64; no tokens: zeros.  Returns out and the largest |value| seen."""
    if k.shape[0] == 0:
        return np.zeros_like(q), 0.0
    with np.errstate(all="ignore"):
        s = q @ k.T * scale
        p = np.exp(s - s.max(-1, keepdims=True))
        return p @ v / p.sum(-1, keepdims=True), float(np.abs(v).max())


def error_bound(q, k, v, scale, dtype, eps, rounded=False):
    """How far a row's output may be off, absolute, for q [rows][d] on k, v [tokens][d] (eps: half a step of the
    output's type, relative).

    Scores: a group's 32 products of q and codes are exact and summed in 32 bits (33 roundings), multiplied by the
    scale and added to the other groups' and the minima's (at most 16 more); with |k| <= kmax a scaled code is at most
    2 kmax and a minimum kmax, so that is at most 49 * 2^-24 * 3 kmax sum|q|.  Queries and their groups' sums enter in
    two FP16 parts: 2^-22 of the row's largest for each channel, for rows whose mean magnitude is at least 1/128 of
    their largest at most 2^-15 * 3 kmax sum|q|.  Both together are below 2^-17 * 12 kmax sum|q|, times the scale in the
    exponent, and as much in a probability, relative.
    Probabilities rounded to FP16 (16-bit types) are off by 2^-11, in two FP16 parts by 2^-22; numerator and denominator
    both.  Sums of up to 2^17 terms in 32 bits on the matrix cores, in chunks: 2^-18.

    rounded: several tokens a sequence in 16-bit types, whose keys and values may be rounded to FP16: 2^-11 of every
    key's element in the exponent, and 2^-11 of the values."""
    if k.shape[0] == 0:
        return np.zeros((q.shape[0], 1))
    kmax, vmax = np.abs(k).max(), np.abs(v).max()
    rounded = rounded and dtype != "fp32"
    delta = (2.0 ** -17 * 12 + (2.0 ** -11 if rounded else 0)) * scale * np.abs(q).sum(-1, keepdims=True) * kmax
    prob = 2.0 ** -22 if dtype == "fp32" else 2.0 ** -11
    out = (2 * np.expm1(delta) + 2 * prob + 2.0 ** -18 + (2.0 ** -11 if rounded else 0)) * vmax
    return out + eps * vmax


# ---- the page stack ---------------------------------------------------------------

def reserve(table, seq_len, new, free_pages, free_count, max_tokens, num_pages):
    """(ok, table, seq_len, free_count, query_start, slots, positions) after reserve_tokens."""
    table, seq_len = table.copy(), seq_len.astype(np.int64).copy()
    B, stride = table.shape
    blocks = lambda n: -(-int(n) // PAGE)
    need = [blocks(seq_len[b] + new[b]) - blocks(seq_len[b]) for b in range(B)]
    bad = any(seq_len[b] < 0 or new[b] < 0 or seq_len[b] + new[b] > 2 ** 31 - 1 or
              (new[b] > 0 and blocks(seq_len[b] + new[b]) > stride) for b in range(B))
    slots, positions = np.full(max_tokens, -1, np.int64), np.full(max_tokens, -1, np.int64)
    start = np.zeros(B + 1, np.int64)
    if bad or sum(need) > free_count or sum(int(n) for n in new) > max_tokens:
        return False, table, seq_len, free_count, start, slots, positions
    taken, at = 0, 0
    for b in range(B):
        start[b] = at
        for i in range(need[b]):
            table[b, blocks(seq_len[b]) + i] = free_pages[free_count - 1 - taken]
            taken += 1
        for i in range(int(new[b])):
            pos = int(seq_len[b]) + i
            page = int(table[b, pos // PAGE])
            positions[at] = pos
            slots[at] = page * PAGE + pos % PAGE if 0 <= page < num_pages else -1
            at += 1
        seq_len[b] += int(new[b])
    start[B] = at
    return True, table, seq_len, free_count - taken, start, slots, positions


def release(table, seq_len, finished, free_pages, free_count, num_pages):
    """(ok, seq_len, free_pages, free_count) after release_sequences."""
    seq_len, free_pages = seq_len.copy(), free_pages.copy()
    blocks = lambda n: -(-int(n) // PAGE)
    gone = [b for b in range(table.shape[0]) if finished[b]]
    if any(seq_len[b] < 0 or blocks(seq_len[b]) > table.shape[1] for b in gone) or \
            free_count + sum(blocks(seq_len[b]) for b in gone) > num_pages:
        return False, seq_len, free_pages, free_count
    for b in gone:
        for i in range(blocks(seq_len[b])):
            free_pages[free_count] = table[b, i]
            free_count += 1
        seq_len[b] = 0
    return True, seq_len, free_pages, free_count
