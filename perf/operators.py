"""Performance cases of the serving operators around a KV cache held in 4 bits: what is timed, on which inputs.

Operators, by the kind of a case:
  reserve  the pages, slots and positions of the next tokens of a batch, from the requests' lengths; with finished
           requests, their pages go back to the free list first
  store    a prompt's keys and values into the 4-bit pages at their slots, and those slots read back as values
  append   one decode token a sequence into the 4-bit pages, and the seal of the blocks it fills
  decode   attention of one token a sequence over the 4-bit pages, all of them or selected blocks and the tail
  prompt   attention of several tokens a sequence (a prompt's chunk, or drafted tokens to verify), causal

A page holds 32 tokens.  A page's record of one KV head, for head_dim D (64, 128 or 256) and groups of 32 channels
(NG = D / 32, NC = D / 16), has 40 D bytes.  Token t = 16 T + 4 j + i (T < 2, j < 4, i < 4):
  key codes      byte t D/2 + (J NG + g) 4 + n/2, nibble n % 2: channel 32 g + 8 J + n  (J < 4, n < 8)
  value codes    from 16 D: byte ((T 4 + j) 16 + r) 2 NC + i NC/2 + n/2, nibble n % 2: channel r NC + n  (r < 16)
  key scales     from 32 D: half ((T 4 + j) NG + g) 4 + i
  key minima     from 34 D: half t NG + g
  value scales   from 36 D: half (g 4 + j) 8 + 4 T + i
  value minima   from 38 D: half (g 4 + j) 8 + 4 T + i
The value is scale * code + minimum.  A group is quantised as: x limited to +-32000, minimum = fp16(min x), scale =
fp32((max x - minimum) / 15) rounded up to 7 significant bits and to a multiple of 2^-24, code =
round_half_even(fp32(fp32(x - minimum) / scale)) within 0..15.  A NaN makes its group's minimum NaN.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False  # True: run() calls the framework's operators

PAGE = 32
LIMIT = 32000.0
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
BANK = 512  # distinct pages that a cache is filled from


def _package():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    path = os.path.join(root, "solidattention-repro_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import solidattention_amd
    return solidattention_amd


# ---- the cases --------------------------------------------------------------

def listed():
    return [
        # the next token of every request of a running batch: launches and latency count
        _reserve("reserve-64", 64, 16384, 1, False),
        # a scheduler's turn on many requests: a third finish, the others take their next chunk of a prompt
        _reserve("reserve-turnover-512", 512, 8192, 127, True),
        # the keys and values of a 16K prompt, parts of the projection's fused output
        _store("store-16k", 1, 16384, 16, 8, 128, "bf16", True),
        # the prompts of several short requests, an odd number of tokens, a small head dimension
        _store("store-ragged-hd64", 37, 5003, 16, 8, 64, "fp16", False),
        # a decode token of 64 requests; a few of them fill a block
        _append("append-64", 64, 16384, 16, 8, 128, "fp32"),
        # one user, a short context: the latency of a decode step's attention
        _decode("decode-1x2k", 1, 2048, 16, 8, 128, "bf16", 0, False),
        # the selected blocks of 64 sequences of 16K tokens, fp32 queries as the decode step has them
        _decode("decode-64x16k-selected", 64, 16384, 16, 8, 128, "fp32", 64, False),
        # whole contexts of different lengths, a small head dimension
        _decode("decode-32x10k-hd64", 32, 10000, 16, 8, 64, "fp16", 0, True),
        # whole contexts, long: 4 query heads on a KV head
        _decode("decode-8x128k-gqa4", 8, 131072, 32, 8, 128, "bf16", 0, True),
        # a prompt of 4K tokens that attends to itself
        _prompt("prompt-1x4k", 1, 4096, 4096, 16, 8, 128, "bf16", False),
        # drafted tokens verified at an ordinary context: few rows on long caches
        _prompt("verify-16x5-at-8k", 16, 5, 8192, 32, 8, 128, "bf16", True),
        # chunks of prompts at long contexts, ragged
        _prompt("prompt-8x1k-at-16k-gqa4", 8, 1024, 16384, 32, 8, 128, "fp16", True),
    ]


def _reserve(name, batch, context, new, turnover):
    return {"name": name, "kind": "reserve", "batch": batch, "context": context, "new": new, "turnover": turnover}


def _store(name, batch, tokens, query_heads, kv_heads, head_dim, dtype, fused):
    return {"name": name, "kind": "store", "batch": batch, "tokens": tokens, "query_heads": query_heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype, "fused": fused}


def _append(name, batch, context, query_heads, kv_heads, head_dim, dtype):
    return {"name": name, "kind": "append", "batch": batch, "context": context, "query_heads": query_heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype}


def _decode(name, batch, context, query_heads, kv_heads, head_dim, dtype, budget, ragged):
    return {"name": name, "kind": "decode", "batch": batch, "context": context, "query_heads": query_heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype, "budget": budget, "ragged": ragged}


def _prompt(name, batch, new, context, query_heads, kv_heads, head_dim, dtype, ragged):
    """`new` tokens a sequence (fewer for some where ragged), the last of a context of `context` tokens."""
    return {"name": name, "kind": "prompt", "batch": batch, "new": new, "context": context,
            "query_heads": query_heads, "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype, "ragged": ragged}


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: a kind, then its sizes over their ranges (log-uniform where they span more than a factor of ten)."""
    kind = rng.choice(["reserve", "store", "append", "decode", "decode", "decode", "prompt", "prompt", "prompt"])
    if kind == "reserve":
        batch = _log(rng, 1, 1024)
        new = 1 if rng.random() < 0.5 else _log(rng, 1, max(1, 65536 // batch))
        c = _reserve("", batch, _log(rng, 32, min(131072, 2 ** 23 // batch)), new, rng.random() < 0.5)
    else:
        kv_heads = rng.choice([1, 4, 8])
        query_heads = kv_heads * rng.choice([1, 2, 4, 8])
        head_dim = rng.choice([64, 128, 128, 128, 256])
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        batch = _log(rng, 1, 64)
        if kind == "store":
            tokens = _log(rng, 1, 16384 * 128 // max(head_dim, 128))
            c = _store("", min(batch, tokens), tokens, query_heads, kv_heads, head_dim, dtype, rng.random() < 0.5)
        elif kind == "append":
            c = _append("", batch, _log(rng, 33, 16384), query_heads, kv_heads, head_dim, dtype)
        elif kind == "decode":
            context = _log(rng, 1, min(131072, 2 ** 19 * 128 // (batch * max(head_dim, 128))))
            budget = rng.choice([0, 0, 16, 64, 128])
            c = _decode("", batch, context, query_heads, kv_heads, head_dim, dtype, budget, rng.random() < 0.7)
        else:
            context = _log(rng, 1, 16384)
            # at most half of the largest listed case's products, an eighth in fp32, which costs more for each
            pairs = (2 ** 37 if dtype == "fp32" else 2 ** 39) // (4 * query_heads * head_dim)
            new = min(context, _log(rng, 1, 4096), pairs // context)
            batch = max(1, min(batch, pairs // (new * context), 2 ** 19 // context))
            c = _prompt("", batch, new, context, query_heads, kv_heads, head_dim, dtype, rng.random() < 0.7)
    del c["name"]
    return c


# ---- the format -------------------------------------------------------------

_PLACES = {}


def _places(d, device):
    """[32][5 d/4] byte of a record that holds each byte of a token: key codes, value codes, then the halves of key
    scales, key minima, value scales and value minima."""
    if (d, device) not in _PLACES:
        ng, nc = d // 32, d // 16
        rows = []
        for t in range(PAGE):
            T, j, i = t // 16, t // 4 % 4, t % 4
            row = [t * d // 2 + b for b in range(d // 2)]
            row += [16 * d + ((T * 4 + j) * 16 + r) * 2 * nc + i * nc // 2 + b for r in range(16) for b in range(nc // 2)]
            row += [32 * d + 2 * (((T * 4 + j) * ng + g) * 4 + i) + b for g in range(ng) for b in (0, 1)]
            row += [34 * d + 2 * (t * ng + g) + b for g in range(ng) for b in (0, 1)]
            row += [36 * d + 2 * ((g * 4 + j) * 8 + 4 * T + i) + b for g in range(ng) for b in (0, 1)]
            row += [38 * d + 2 * ((g * 4 + j) * 8 + 4 * T + i) + b for g in range(ng) for b in (0, 1)]
            rows.append(row)
        _PLACES[(d, device)] = torch.tensor(rows, dtype=torch.int64, device=device)
    return _PLACES[(d, device)]


def _round_scale(raw):
    up = ((raw.view(torch.int32) + 0x1FFFF) & ~0x1FFFF).view(torch.float32)
    fine = torch.ceil(raw * 2.0 ** 24) * 2.0 ** -24
    return torch.where(up < 2.0 ** -18, fine, up)


def _quantise(x):
    """x [..., d] -> codes [..., d] uint8, scales and minima [..., d / 32] fp16."""
    x = x.float().unflatten(-1, (-1, 32)).clamp(-LIMIT, LIMIT)
    low = x.amin(-1).to(torch.float16) + 0.0  # (NaN stays)
    span = (x.amax(-1) - low.float()).clamp(min=0.0).nan_to_num(0.0)
    scale = _round_scale((span.double() / 15.0).float())
    # the two fp32 roundings, each of a 64-bit result: next to a border they decide the code
    off = (x.double() - low.double()[..., None]).float()
    code = torch.round((off.double() / scale.double()[..., None]).float())
    code = torch.where(scale[..., None] > 0, code, torch.zeros_like(code)).nan_to_num(0.0).clamp(0, 15)
    return code.to(torch.uint8).flatten(-2), scale.to(torch.float16), low


def _halves(x):
    return x.contiguous().view(torch.uint8)


def _token_bytes(k, v):
    """k, v [..., d] -> [..., 5 d/4] bytes in _places order."""
    kc, ks, km = _quantise(k)
    vc, vs, vm = _quantise(v)
    kc = kc.unflatten(-1, (-1, 4, 8)).transpose(-3, -2).reshape(kc.shape)
    pack = lambda c: c[..., 0::2] | (c[..., 1::2] << 4)
    return torch.cat([pack(kc), pack(vc), _halves(ks), _halves(km), _halves(vs), _halves(vm)], dim=-1)


def _values(raw, d):
    """[..., 5 d/4] bytes in _places order -> keys and values [..., d] fp32."""
    ng = d // 32
    kc, vc, ks, km, vs, vm = raw.split([d // 2, d // 2] + [2 * ng] * 4, dim=-1)
    nibbles = lambda c: torch.stack([c & 15, c >> 4], dim=-1).flatten(-2).float()
    half = lambda b: b.contiguous().view(torch.float16).float()[..., None]
    k = nibbles(kc).unflatten(-1, (4, ng, 8)).transpose(-3, -2).flatten(-2)
    v = nibbles(vc).unflatten(-1, (ng, 32))
    return (k * half(ks) + half(km)).flatten(-2), (v * half(vs) + half(vm)).flatten(-2)


def _write_tokens(pool, slots, raw, d):
    """raw [n][heads][5 d/4] to the slots (page * 32 + offset) of pool [pages][heads][40 d]."""
    heads = torch.arange(pool.shape[1], device=pool.device)
    pool[(slots // PAGE).long()[:, None, None], heads[None, :, None], _places(d, pool.device)[slots.long() % PAGE][:, None]] = raw


def _read_tokens(pool, slots, d):
    heads = torch.arange(pool.shape[1], device=pool.device)
    raw = pool[(slots // PAGE).long()[:, None, None], heads[None, :, None],
               _places(d, pool.device)[slots.long() % PAGE][:, None]]
    return _values(raw, d)


def _read_records(pool, records, d):
    """Keys and values [n][32][d] fp32 of the records numbered page * heads + head."""
    raw = pool.view(-1, 40 * d)[records]
    return _values(raw[:, _places(d, pool.device).flatten()].unflatten(-1, (PAGE, 5 * d // 4)), d)


# ---- inputs -----------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, shape, dtype=torch.float32):
    return torch.empty(shape, dtype=torch.float32, device="cuda").normal_(generator=g).to(dtype)


def _spread(n, lo, hi):
    return [hi if n == 1 else int(lo + (hi - lo) * i / (n - 1)) for i in range(n)]


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _deal(values, g):
    """The values in an order that the seed gives."""
    order = torch.randperm(len(values), generator=g, device="cuda").tolist()
    return [values[i] for i in order]


def _lengths(c):
    """The multiset of the batch's lengths (prepare() deals them out by the seed)."""
    n, context = c["batch"], c["context"]
    return _spread(n, max(1, context // 2), context) if c["ragged"] else [context] * n


def _new_tokens(c):
    """prompt: tokens of each sequence in the order of _lengths."""
    lengths = _lengths(c)
    new = _spread(c["batch"], max(1, c["new"] // 2), c["new"]) if c["ragged"] else [c["new"]] * c["batch"]
    return [min(a, b) for a, b in zip(new, lengths)]


def _table(g, blocks, stride, pages):
    """A block table of `blocks` blocks a sequence out of shuffled pages."""
    need = _int32(blocks)
    perm = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    first = torch.cumsum(need, 0) - need
    col = torch.arange(stride, device="cuda")
    at = (first[:, None] + col[None]).clamp(max=pages - 1)
    return torch.where(col[None] < need[:, None], perm[at], torch.zeros_like(perm[at])).contiguous()


def _cache(g, lengths, kv_heads, d):
    """A filled 4-bit pool and its table.  Keys have a few large channels, as post-RoPE keys do; the pages are copies
    of a bank of quantised ones.  The slots behind a sequence's last token hold bytes that decode to NaN."""
    blocks = [(n + PAGE - 1) // PAGE for n in lengths]
    stride, pages = max(blocks) + 1, sum(blocks) + 8
    table = _table(g, blocks, stride, pages)
    n = min(BANK, pages)
    k, v = _normal(g, (n, PAGE, kv_heads, d)), _normal(g, (n, PAGE, kv_heads, d))
    k[..., :4] *= 3.0
    bank = torch.empty((n, kv_heads, 40 * d), dtype=torch.uint8, device="cuda")
    bank[:, :, _places(d, bank.device).flatten()] = _token_bytes(k, v).transpose(1, 2).flatten(-2)
    pool = bank[torch.randint(n, (pages,), generator=g, device="cuda")]
    for b, length in enumerate(lengths):
        if length % PAGE:
            pool[table[b, length // PAGE].long(), :, _places(d, pool.device)[length % PAGE:].flatten()] = 255
    return pool, table, stride


def _reserve_inputs(c, g):
    B, context = c["batch"], c["context"]
    lengths = _deal(_spread(B, max(1, context // 2), context), g)
    finished = [int(c["turnover"] and b % 3 == 1) for b in range(B)]
    new = [0 if finished[b] else (1 + (c["new"] - 1) * (b % 7) // 6 if c["turnover"] else c["new"]) for b in range(B)]
    blocks = [(n + PAGE - 1) // PAGE for n in lengths]
    more = [max(n, (lengths[b] * (1 - finished[b]) + new[b] + PAGE - 1) // PAGE) for b, n in enumerate(blocks)]
    pages, stride = sum(more) + 8, (context + max(new)) // PAGE + 2
    held = sum(blocks)
    perm = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    need, col = _int32(blocks), torch.arange(stride, device="cuda")
    at = (torch.cumsum(need, 0) - need)[:, None] + col[None]
    table = torch.where(col[None] < need[:, None], perm[at.clamp(max=pages - 1)], torch.full_like(perm[:1], -1))
    free = torch.zeros(pages, dtype=torch.int32, device="cuda")
    free[:pages - held] = perm[held:]
    total = sum(new)
    slots = torch.empty(total + (total // 8 if c["turnover"] else 0) + 1, dtype=torch.int32, device="cuda")
    s = {"table": table.contiguous(), "seq_len": _int32(lengths), "new": _int32(new), "finished": _int32(finished),
         "free_pages": free, "free_count": _int32([pages - held]), "stride": stride, "pages": pages,
         "slots": slots, "positions": torch.empty_like(slots), "query_start": _int32([0] * (B + 1)),
         "mid_len": _int32([0] * B), "mid_free": _int32([0]), "out_len": _int32([0] * B), "out_free": _int32([0])}
    return s


def _store_inputs(c, g):
    B, n, hq, h, d = c["batch"], c["tokens"], c["query_heads"], c["kv_heads"], c["head_dim"]
    dtype = TYPES[c["dtype"]]
    shares = [n // B + (b < n % B) for b in range(B)]
    starts = [(7 * b) % PAGE for b in range(B)]  # where a request's new tokens begin in its first page
    blocks = [(a + m + PAGE - 1) // PAGE for a, m in zip(starts, shares)]
    pages = sum(blocks) + 8
    perm = torch.randperm(pages, generator=g, device="cuda").tolist()
    slots, first = [], 0
    for a, m, k in zip(starts, shares, blocks):
        slots += [perm[first + p // PAGE] * PAGE + p % PAGE for p in range(a, a + m)]
        first += k
    slots += [-1] * (n // 16)  # the rows behind the last sequence of a padded batch
    rows = len(slots)
    x = _normal(g, (rows, hq + 2 * h if c["fused"] else 2 * h, d), dtype)
    x[:, -2 * h:-h, :4] *= 3.0
    k, v = x[:, -2 * h:-h], x[:, -h:]
    if not c["fused"]:
        k, v = k.contiguous(), v.contiguous()
    return {"k": k, "v": v, "slots": _int32(slots), "tokens": n, "pages": pages,
            "pool": torch.zeros((pages, h, 40 * d), dtype=torch.uint8, device="cuda"),
            "k_out": torch.zeros((rows, h, d), dtype=dtype, device="cuda"),
            "v_out": torch.zeros((rows, h, d), dtype=dtype, device="cuda")}


def _append_inputs(c, g):
    B, h, d, dtype = c["batch"], c["kv_heads"], c["head_dim"], TYPES[c["dtype"]]
    lengths = _deal([max(0, n - (n % PAGE) + (b * 5) % PAGE) for b, n in enumerate(_spread(B, c["context"] // 2, c["context"]))], g)
    stride = max(lengths) // PAGE + 2
    last = [n // PAGE for n in lengths]
    # the pages of earlier blocks are not touched: they share one page of the pool
    table = torch.zeros((B, stride), dtype=torch.int32, device="cuda")
    table[torch.arange(B, device="cuda"), torch.tensor(last, device="cuda")] = \
        1 + torch.randperm(B, generator=g, device="cuda").to(torch.int32)
    k, v = _normal(g, (B + 1, PAGE, h, d)), _normal(g, (B + 1, PAGE, h, d))
    pool = torch.empty((B + 1, h, 40 * d), dtype=torch.uint8, device="cuda")
    pool[:, :, _places(d, pool.device).flatten()] = _token_bytes(k, v).transpose(1, 2).flatten(-2)
    slots = [n % PAGE for n in lengths]
    base = _int32([lengths, last, last])
    return {"pool": pool, "table": table, "stride": stride, "base": base, "live": base.clone(), "lengths": lengths,
            "slots": table[torch.arange(B, device="cuda"), torch.tensor(last, device="cuda")] * PAGE + _int32(slots),
            "full": [b for b in range(B) if slots[b] == PAGE - 1],
            "reps": torch.zeros((B, h, d, (stride + 31) // 32 * 32), dtype=torch.float32, device="cuda"),
            "k": _normal(g, (B, h, d), dtype), "v": _normal(g, (B, h, d), dtype),
            "k_out": torch.empty((B, h, d), dtype=torch.float32, device="cuda"),
            "v_out": torch.empty((B, h, d), dtype=torch.float32, device="cuda"), "pages": B + 1}


def _decode_inputs(c, g):
    B, hq, h, d = c["batch"], c["query_heads"], c["kv_heads"], c["head_dim"]
    lengths = _deal(_lengths(c), g)
    pool, table, stride = _cache(g, lengths, h, d)
    s = {"pool": pool, "table": table, "stride": stride, "lengths": lengths, "pages": pool.shape[0],
         "seq_len": _int32(lengths), "sealed": _int32([n // PAGE for n in lengths]),
         "q": _normal(g, (B, hq, d), TYPES[c["dtype"]]), "selected": None, "counts": None}
    if c["budget"]:  # ids ascending, as the selection writes them; a short context takes every block
        selected = torch.full((B, h, c["budget"]), -1, dtype=torch.int32, device="cuda")
        for b, n in enumerate(lengths):
            m = min(c["budget"], n // PAGE)
            ids = torch.rand((h, n // PAGE), generator=g, device="cuda").argsort(dim=-1)[:, :m].sort(dim=-1).values
            selected[b, :, :m] = ids.to(torch.int32)
        s["selected"] = selected
        s["taken"] = [min(c["budget"], n // PAGE) for n in lengths]
        s["counts"] = _int32(s["taken"])[:, None].expand(B, h).contiguous()
    return s


def _prompt_inputs(c, g):
    B, hq, h, d = c["batch"], c["query_heads"], c["kv_heads"], c["head_dim"]
    both = _deal(list(zip(_lengths(c), _new_tokens(c))), g)
    lengths, new = [a for a, _ in both], [b for _, b in both]
    pool, table, stride = _cache(g, lengths, h, d)
    starts = [sum(new[:b]) for b in range(B + 1)]
    return {"pool": pool, "table": table, "stride": stride, "lengths": lengths, "new": new, "starts": starts,
            "pages": pool.shape[0], "seq_len": _int32(lengths), "sealed": _int32([n // PAGE for n in lengths]),
            "query_start": _int32(starts), "q": _normal(g, (starts[-1], hq, d), TYPES[c["dtype"]])}


_INPUTS = {"reserve": _reserve_inputs, "store": _store_inputs, "append": _append_inputs, "decode": _decode_inputs,
           "prompt": _prompt_inputs}


def prepare(case, seed):
    s = _INPUTS[case["kind"]](case, _gen(seed))
    s["case"] = case
    if own:
        _attach(s)
    return s


def _attach(s):
    """The handles that a user's program keeps: the cache's view, its workspace, the output."""
    sa = _package()
    c = s["case"]
    s["sa"] = sa
    if c["kind"] == "reserve":
        kv = sa.PagedKV4(c["batch"], 1, 1, s["stride"], num_pages=s["pages"], rep_stride=1,
                         pool=torch.empty((s["pages"], 1, 40 * 128), dtype=torch.uint8, device="cuda"))
        kv.block_table, kv.seq_len = s["table"], s["seq_len"]
        s["kv"] = kv
        if c["turnover"]:
            after = sa.PagedKV4(c["batch"], 1, 1, s["stride"], num_pages=s["pages"], rep_stride=1, pool=kv.pool)
            after.block_table, after.seq_len = s["table"], s["mid_len"]
            s["after"] = after
        return
    hq, h, d = c["query_heads"], c["kv_heads"], c["head_dim"]
    kv = sa.PagedKV4(c["batch"], hq, h, s.get("stride", 1), num_pages=s["pages"], head_dim=d, pool=s["pool"],
                     rep_stride=None if c["kind"] == "append" else 1)
    s["kv"] = kv
    if c["kind"] == "append":
        kv.block_table, kv.reps = s["table"], s["reps"]
        kv.seq_len, kv.sealed, kv.generation = s["live"][0], s["live"][1], s["live"][2]
    elif c["kind"] != "store":
        kv.block_table, kv.seq_len, kv.sealed = s["table"], s["seq_len"], s["sealed"]
        s["ws"] = sa.kv4_attention_workspace(kv, s["q"].shape[0])
        s["out"] = torch.empty_like(s["q"])


# ---- one pass ---------------------------------------------------------------

def run(state):
    return _PASSES[own][state["case"]["kind"]](state)


def _own_reserve(s):
    sa, kv, free_count = s["sa"], s["kv"], s["free_count"]
    if s["case"]["turnover"]:
        sa.release_sequences(kv, s["finished"], s["free_pages"], free_count, seq_len_out=s["mid_len"],
                             free_count_out=s["mid_free"])
        kv, free_count = s["after"], s["mid_free"]
    sa.reserve_tokens(kv, s["new"], s["free_pages"], free_count, s["query_start"], s["slots"], s["positions"],
                      seq_len_out=s["out_len"], free_count_out=s["out_free"])
    return {k: s[k] for k in ("table", "out_len", "out_free", "query_start", "slots", "positions")}


def _own_store(s):
    sa = s["sa"]
    sa.kv4_store(s["kv"], s["k"], s["v"], s["slots"])
    sa.kv4_load(s["kv"], s["slots"], s["k_out"], s["v_out"])
    return {"k": s["k_out"], "v": s["v_out"]}


def _own_append(s):
    sa = s["sa"]
    s["live"].copy_(s["base"])
    sa.kv4_append_seal(s["kv"], s["k"], s["v"], 0)
    sa.kv4_load(s["kv"], s["slots"], s["k_out"], s["v_out"])
    return {"k": s["k_out"], "v": s["v_out"], "reps": s["reps"], "live": s["live"]}


def _own_decode(s):
    d = s["case"]["head_dim"]
    return s["sa"].kv4_decode_attention(s["kv"], s["q"], d ** -0.5, s["selected"], s["counts"], out=s["out"],
                                        workspace=s["ws"])


def _own_prompt(s):
    d = s["case"]["head_dim"]
    return s["sa"].kv4_prompt_attention(s["kv"], s["q"], s["query_start"], d ** -0.5, out=s["out"], workspace=s["ws"])


def _plain_reserve(s):
    table, length, free_count, free = s["table"], s["seq_len"], s["free_count"], s["free_pages"]
    stride, rows = s["stride"], s["slots"].shape[0]
    col = torch.arange(stride, device="cuda", dtype=torch.int32)
    if s["case"]["turnover"]:
        gone = s["finished"] != 0
        count = torch.where(gone, (length + PAGE - 1) // PAGE, torch.zeros_like(length))
        at = free_count + torch.cumsum(count, 0, dtype=torch.int32) - count
        dest = torch.where(col[None] < count[:, None], at[:, None] + col[None], free.shape[0])
        longer = torch.cat([free, free[:1]])  # one more place takes what is not written
        longer.scatter_(0, dest.flatten().long().clamp(max=free.shape[0]), table.flatten())
        free.copy_(longer[:-1])
        free_count = free_count + count.sum(dtype=torch.int32)
        length = torch.where(gone, torch.zeros_like(length), length)
    new = s["new"]
    old_blocks, blocks = (length + PAGE - 1) // PAGE, (length + new + PAGE - 1) // PAGE
    need = blocks - old_blocks
    first = torch.cumsum(need, 0, dtype=torch.int32) - need
    order = free_count - 1 - (first[:, None] + col[None] - old_blocks[:, None])
    fresh = (col[None] >= old_blocks[:, None]) & (col[None] < blocks[:, None])
    table.copy_(torch.where(fresh, free[order.clamp(0, free.shape[0] - 1).long()], table))
    ends = torch.cumsum(new, 0, dtype=torch.int32)
    start = torch.cat([torch.zeros_like(ends[:1]), ends])
    token = torch.arange(rows, device="cuda", dtype=torch.int32)
    b = torch.searchsorted(ends, token, right=True).clamp(max=length.shape[0] - 1)
    position = length[b] + token - start[b]
    page = table[b, (position // PAGE).clamp(0, stride - 1).long()]
    live = token < ends[-1]
    none = torch.full_like(token, -1)
    return {"table": table, "out_len": length + new, "out_free": free_count - need.sum(dtype=torch.int32),
            "query_start": start, "slots": torch.where(live, page * PAGE + position % PAGE, none),
            "positions": torch.where(live, position, none)}


def _plain_store(s):
    d, n = s["case"]["head_dim"], s["tokens"]
    slots = s["slots"][:n]
    for i in range(0, n, 4096):
        _write_tokens(s["pool"], slots[i:i + 4096], _token_bytes(s["k"][i:min(i + 4096, n)], s["v"][i:min(i + 4096, n)]), d)
    for i in range(0, n, 4096):
        k, v = _read_tokens(s["pool"], slots[i:i + 4096], d)
        s["k_out"][i:min(i + 4096, n)], s["v_out"][i:min(i + 4096, n)] = k, v
    return {"k": s["k_out"], "v": s["v_out"]}


def _plain_append(s):
    d, h = s["case"]["head_dim"], s["case"]["kv_heads"]
    s["live"].copy_(s["base"])
    _write_tokens(s["pool"], s["slots"], _token_bytes(s["k"], s["v"]), d)
    s["live"][0] += 1
    full = s["live"][0] - PAGE * s["live"][1] >= PAGE
    s["live"][1:] += full.to(torch.int32)
    if s["full"]:
        rows = torch.tensor(s["full"], device="cuda")
        block = s["base"][1][rows].long()
        record = s["table"][rows, block].long()[:, None] * h + torch.arange(h, device="cuda")[None]
        k, _ = _read_records(s["pool"], record.flatten(), d)
        s["reps"][rows[:, None], torch.arange(h, device="cuda")[None], :, block[:, None]] = \
            (k.sum(1) / PAGE).view(len(s["full"]), h, d)
    k, v = _read_tokens(s["pool"], s["slots"], d)
    return {"k": k, "v": v, "reps": s["reps"], "live": s["live"]}


def _attend(q, k, v, scale, hidden):
    """q [n][rows][d], k and v [n][tokens][d], hidden: True where a row does not see a token."""
    score = torch.matmul(k, q.transpose(1, 2).contiguous()).transpose(1, 2) * scale
    score = score.masked_fill(hidden, -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    return torch.matmul(p, v) / p.sum(-1, keepdim=True)


def _plain_decode(s):
    c = s["case"]
    B, hq, h, d = c["batch"], c["query_heads"], c["kv_heads"], c["head_dim"]
    out = torch.empty_like(s["q"])
    heads = torch.arange(h, device="cuda")
    full = [s["taken"][b] if c["budget"] else n // PAGE for b, n in enumerate(s["lengths"])]
    blocks = [m + (n % PAGE > 0) for m, n in zip(full, s["lengths"])]
    step = max(1, 2 ** 28 // (max(blocks) * PAGE * h * d))
    for b0 in range(0, B, step):
        some = range(b0, min(b0 + step, B))
        width = max(blocks[b] for b in some)
        col = torch.arange(width, device="cuda")
        logical = col[None, None].expand(len(some), h, width)
        taken = torch.tensor([full[b] for b in some], device="cuda")[:, None, None]
        length = s["seq_len"][b0:b0 + step].long()[:, None, None]
        if c["budget"]:
            ids = s["selected"][b0:b0 + step].long()
            ids = torch.cat([ids, ids[..., :1].expand(-1, -1, max(0, width - ids.shape[-1]))], dim=-1)[..., :width]
            logical = torch.where(logical < taken, ids, length // PAGE)
        page = torch.gather(s["table"][b0:b0 + step].long()[:, None].expand(-1, h, -1), 2,
                            logical.clamp(0, s["stride"] - 1))
        k, v = _read_records(s["pool"], (page * h + heads[:, None]).flatten(), d)
        valid = torch.where(col[None, None] < taken, PAGE, torch.where(col[None, None] == taken, length % PAGE, 0))
        valid = valid.expand(-1, h, -1)[..., None]
        hidden = (torch.arange(PAGE, device="cuda") >= valid).reshape(len(some) * h, -1)
        k = k.view(len(some) * h, -1, d)
        v = v.view(len(some) * h, -1, d).masked_fill(hidden[..., None], 0.0)
        q = s["q"][b0:b0 + step].float().view(len(some) * h, hq // h, d)
        out[b0:b0 + step] = _attend(q, k, v, d ** -0.5, hidden[:, None]).view(len(some), hq, d)
    return out


def _plain_prompt(s):
    c = s["case"]
    hq, h, d = c["query_heads"], c["kv_heads"], c["head_dim"]
    out = torch.empty_like(s["q"])
    for b, (n, m) in enumerate(zip(s["lengths"], s["new"])):
        rows = slice(s["starts"][b], s["starts"][b] + m)
        pages = s["table"][b, :(n + PAGE - 1) // PAGE].long()
        seen = n - m + torch.arange(m, device="cuda")
        hidden = (torch.arange(n, device="cuda")[None] > seen[:, None]).repeat_interleave(hq // h, 0)[None]
        step = max(1, min(h, 2 ** 27 // (n * (m * hq // h + d))))
        for g0 in range(0, h, step):
            some = torch.arange(g0, min(g0 + step, h), device="cuda")
            k, v = (x.view(some.shape[0], -1, d)[:, :n]
                    for x in _read_records(s["pool"], (pages[None] * h + some[:, None]).flatten(), d))
            heads = slice(g0 * (hq // h), (g0 + some.shape[0]) * (hq // h))
            q = s["q"][rows, heads].float().view(m, -1, hq // h, d).transpose(0, 1).reshape(-1, m * hq // h, d)
            got = _attend(q, k, v, d ** -0.5, hidden).view(-1, m, hq // h, d).transpose(0, 1)
            out[rows, heads] = got.reshape(m, -1, d).to(out.dtype)
    return out


_PASSES = {True: {"reserve": _own_reserve, "store": _own_store, "append": _own_append, "decode": _own_decode,
                  "prompt": _own_prompt},
           False: {"reserve": _plain_reserve, "store": _plain_store, "append": _plain_append, "decode": _plain_decode,
                   "prompt": _plain_prompt}}


# ---- work -------------------------------------------------------------------

def work(case):
    c, kind = case, case["kind"]
    if kind == "reserve":
        B, context = c["batch"], c["context"]
        lengths = _spread(B, max(1, context // 2), context)
        gone = [c["turnover"] and b % 3 == 1 for b in range(B)]
        new = [0 if gone[b] else (1 + (c["new"] - 1) * (b % 7) // 6 if c["turnover"] else c["new"]) for b in range(B)]
        total = sum(new)
        # lengths, counts and starts; the slots and positions; the pages handed out and back
        pages = sum(n // PAGE + 1 for n in new if n) + sum(n // PAGE + 1 for n, f in zip(lengths, gone) if f)
        return {"bytes": 4 * (4 * B + 2 * total + 2 * pages), "flops": 2 * total}
    hq, h, d = c["query_heads"], c["kv_heads"], c["head_dim"]
    token = h * 5 * d // 4  # K and V of a token in 4 bits, with scales and minima
    size = 4 if c["dtype"] == "fp32" else 2
    if kind == "store":  # read k and v, write records; read records, write values
        return {"bytes": c["tokens"] * (4 * h * d * size + 2 * token), "flops": 8 * c["tokens"] * 2 * h * d}
    if kind == "append":
        full = sum((b * 5) % PAGE == PAGE - 1 for b in range(c["batch"]))
        return {"bytes": c["batch"] * (2 * h * d * (size + 4) + 2 * token) + full * h * d * (PAGE * 5 // 8 + 4),
                "flops": 8 * c["batch"] * 2 * h * d + full * PAGE * h * d}
    if kind == "decode":
        seen = [min(c["budget"], n // PAGE) * PAGE + n % PAGE if c["budget"] else n for n in _lengths(c)]
        return {"bytes": sum(seen) * token + 2 * c["batch"] * hq * d * size, "flops": 4 * sum(seen) * hq * d}
    new, lengths = _new_tokens(c), _lengths(c)
    pairs = sum(m * n - m * (m - 1) // 2 for m, n in zip(new, lengths))
    return {"bytes": sum(lengths) * token + 2 * sum(new) * hq * d * size, "flops": 4 * pairs * hq * d}


# ---- 64-bit results ---------------------------------------------------------

def _exact_values(record, d):
    """Keys and values [n][32][d] in 64 bits of records [n][40 d], element by element from the layout's formulas."""
    dev = record.device
    t, ch = torch.arange(PAGE, device=dev)[:, None], torch.arange(d, device=dev)[None]
    ng, nc = d // 32, d // 16
    T, j, i, g = t // 16, t // 4 % 4, t % 4, ch // 32
    k_at = t * (d // 2) + ((ch % 32 // 8) * ng + g) * 4 + ch % 8 // 2
    v_at = 16 * d + ((T * 4 + j) * 16 + ch // nc) * 2 * nc + i * (nc // 2) + ch % nc // 2

    def code(at, nibble):
        byte = record[:, at.flatten()].view(-1, PAGE, d).to(torch.int32)
        return (torch.bitwise_right_shift(byte, 4 * (nibble % 2).to(torch.int32)) & 15).double()

    def half(at):
        at = at.expand(PAGE, d).flatten()
        bits = record[:, at].to(torch.int32) | (record[:, at + 1].to(torch.int32) << 8)
        return bits.to(torch.int16).view(torch.float16).double().view(-1, PAGE, d)

    k_at, v_at = k_at.expand(PAGE, d), v_at.expand(PAGE, d)
    k = code(k_at, ch) * half(32 * d + 2 * (((T * 4 + j) * ng + g) * 4 + i)) + half(34 * d + 2 * (t * ng + g))
    v_half = 2 * ((g * 4 + j) * 8 + 4 * T + i)
    v = code(v_at, ch) * half(36 * d + v_half) + half(38 * d + v_half)
    return k, v


def _exact_rounded(x):
    """What a cache in 4 bits holds for x [..., d], in 64 bits; the steps that the format rounds are rounded."""
    x = x.double().clamp(-LIMIT, LIMIT)
    x = x.reshape(*x.shape[:-1], -1, 32)
    low = x.min(-1, keepdim=True).values.half().double()
    step = (((x.max(-1, keepdim=True).values - low).float().double()) / 15).float().double().clamp(min=0)
    _, e = torch.frexp(step)
    unit = torch.exp2(torch.maximum(e - 7, torch.full_like(e, -24)).double())
    step = torch.ceil(step / unit) * unit
    code = torch.round(((x - low).float().double() / step).float().double())
    code = torch.where(step > 0, code, torch.zeros_like(code)).clamp(0, 15)
    return (code * step + low).flatten(-2)


def _exact_attend(q, k, v, scale, hidden):
    s = torch.matmul(q, k.t().contiguous()) * scale
    s = s.masked_fill(hidden, -math.inf)
    return torch.matmul(torch.softmax(s, dim=-1), v)


def exact(case, seed):
    c, kind = case, case["kind"]
    if kind == "reserve":
        return None  # whole numbers
    s = _INPUTS[kind](c, _gen(seed))
    hq, h, d = c["query_heads"], c["kv_heads"], c["head_dim"]
    if kind == "store":
        n = s["tokens"]
        k, v = torch.zeros(s["k_out"].shape, dtype=torch.float64, device="cuda"), \
            torch.zeros(s["k_out"].shape, dtype=torch.float64, device="cuda")
        k[:n], v[:n] = _exact_rounded(s["k"][:n]), _exact_rounded(s["v"][:n])
        return {"k": k, "v": v}
    if kind == "append":
        k, v = _exact_rounded(s["k"]), _exact_rounded(s["v"])
        reps = torch.zeros(s["reps"].shape, dtype=torch.float64, device="cuda")
        for b in s["full"]:
            page, block = int(s["slots"][b]) // PAGE, s["lengths"][b] // PAGE
            keys, _ = _exact_values(s["pool"][page], d)
            keys[:, PAGE - 1] = k[b]
            reps[b, :, :, block] = keys.mean(1)
        return {"k": k, "v": v, "reps": reps, "live": None}
    G = hq // h
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(s["lengths"]):
        row = s["table"][b].long()
        for g in range(h):
            ids = torch.arange((n + PAGE - 1) // PAGE, device="cuda")
            if kind == "decode" and c["budget"]:
                ids = s["selected"][b, g, :s["taken"][b]].long()
                if n % PAGE:
                    ids = torch.cat([ids, torch.tensor([n // PAGE], device="cuda")])
            at = (ids[:, None] * PAGE + torch.arange(PAGE, device="cuda")).flatten()
            k, v = _exact_values(s["pool"][row[ids], g], d)
            k, v = k.view(-1, d)[at < n], v.view(-1, d)[at < n]
            heads = slice(g * G, (g + 1) * G)
            if kind == "decode":
                out[b, heads] = _exact_attend(s["q"][b, heads].double(), k, v, d ** -0.5, torch.zeros((), dtype=torch.bool, device="cuda"))
                continue
            m, first = s["new"][b], s["starts"][b]
            seen = n - m + torch.arange(m, device="cuda")
            hidden = torch.arange(n, device="cuda")[None] > seen[:, None]
            for j in range(G):
                out[first:first + m, g * G + j] = _exact_attend(s["q"][first:first + m, g * G + j].double(), k, v,
                                                                d ** -0.5, hidden)
    return out
