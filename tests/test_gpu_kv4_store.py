"""Tokens into 4-bit pages and back, appends and seals, against the format's definition in 64 bits.  The format's
roundings are stated, so the bytes are equal; representatives are fp32 sums."""
import numpy as np
import pytest
import torch

import kv4_oracle as K

pytestmark = pytest.mark.gpu
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def ints(a):
    return torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()


def cache(sa, pages, heads, d, batch=1, stride=1, rep_heads=None, rep_stride=None):
    kv = sa.PagedKV4(batch, 2 * heads, heads, stride, num_pages=pages, head_dim=d, rep_heads=rep_heads,
                     rep_stride=rep_stride)
    kv.pool.copy_(torch.randint(0, 256, kv.pool.shape, generator=torch.Generator().manual_seed(pages),
                                dtype=torch.uint8))
    return kv


def f64(x):
    return x.detach().cpu().to(torch.float64).numpy()


def tokens(seed, n, heads, d, dtype):
    """Rows of very different sizes: ordinary, tiny (FP16 subnormal scales), large, constant and zero groups, infinities."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((n, heads, d), generator=g)
    kind = torch.arange(n) % 8
    x[kind == 1] *= 1e-5
    x[kind == 2] *= 1e4
    x[kind == 3, :, :32] = 0.7
    x[kind == 4] = 0.0
    x[kind == 5, 0, 5] = float("inf")
    x[kind == 5, 0, 40] = float("-inf")
    x[kind == 6] = x[kind == 6] * 2e-7 + 1.0
    x[kind == 7, :, 3] = 300.0
    return x.to(TYPES[dtype])


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("n,heads,strided", [(1, 1, False), (2, 8, True), (33, 3, True), (70, 2, False)])
def test_store_bytes_and_load(hip, n, heads, d, dtype, strided):
    rng = np.random.default_rng(n)
    pages = (n + 31) // 32 + 2
    kv = cache(hip, pages, heads, d)
    before = kv.pool.cpu().numpy().copy()
    slots = rng.permutation(pages * 32)[:n]
    slots[n // 2:n // 2 + 1] = -1 if n > 2 else slots[n // 2:n // 2 + 1]
    k, v = tokens(1, n, heads, d, dtype), tokens(2, n, heads, d, dtype)
    if strided:  # parts of one fused row
        x = torch.cat([torch.randn(n, heads, d).to(k.dtype), k, v], dim=1).cuda()
        kd, vd = x[:, heads:2 * heads], x[:, 2 * heads:]
    else:
        kd, vd = k.cuda(), v.cuda()
    status = ints([0])
    hip.kv4_store(kv, kd, vd, ints(slots), status=status)
    expect = before.copy()
    for i, s in enumerate(slots):
        if s >= 0:
            K.put(expect, int(s), f64(k[i]), f64(v[i]))
    got = kv.pool.cpu().numpy()
    assert int(status) == 0
    np.testing.assert_array_equal(got, expect)

    out = torch.full((n, 2 * heads, d), -5.0, dtype=k.dtype, device="cuda")
    hip.kv4_load(kv, ints(slots), out[:, :heads], out[:, heads:], status=status)
    for i, s in enumerate(slots):
        want = np.full((2 * heads, d), -5.0) if s < 0 else np.concatenate([K.values(f64(k[i])), K.values(f64(v[i]))])
        want = torch.from_numpy(want).to(torch.float32).to(k.dtype)
        assert torch.equal(out[i].cpu(), want), (i, s)


def test_values_are_within_half_a_step(hip):
    """The error of a stored value is at most half a scale plus the minimum's rounding."""
    x = tokens(3, 64, 4, 128, "fp32")
    x[x.abs() > 1e30] = 1.0
    kv = cache(hip, 2, 4, 128)
    hip.kv4_store(kv, x.cuda(), (-x).cuda(), ints(np.arange(64)))
    k, v = torch.empty_like(x).cuda(), torch.empty_like(x).cuda()
    hip.kv4_load(kv, ints(np.arange(64)), k, v)
    for got, want in ((k, x), (v, -x)):
        _, s, m = K.quantise(f64(want))
        want = np.clip(f64(want), -K.LIMIT, K.LIMIT)
        bound = 0.5 * s * (1 + 2.0 ** -20) + np.abs(m) * 2.0 ** -10 + 2.0 ** -24
        assert (np.abs(f64(got) - want) <= bound).all()


def test_nan_spoils_its_group_only(hip):
    x = tokens(4, 8, 2, 128, "fp32")
    x[6, 1, 70] = float("nan")
    kv = cache(hip, 1, 2, 128)
    hip.kv4_store(kv, x.cuda(), x.cuda(), ints(np.arange(8)))
    k, v = torch.empty_like(x).cuda(), torch.empty_like(x).cuda()
    hip.kv4_load(kv, ints(np.arange(8)), k, v)
    want = torch.zeros(8, 2, 128, dtype=torch.bool)
    want[6, 1, 64:96] = True
    assert torch.equal(k.cpu().isnan(), want) and torch.equal(v.cpu().isnan(), want)


def test_slots_past_the_pool(hip):
    kv = cache(hip, 2, 1, 64)
    before = kv.pool.clone()
    x = tokens(5, 3, 1, 64, "fp16").cuda()
    status = ints([0])
    hip.kv4_store(kv, x, x, ints([64, 2 ** 31 - 1, -2 ** 31]), status=status)
    assert int(status) == 1 and torch.equal(kv.pool, before)
    out = torch.full_like(x, 3.0)
    hip.kv4_load(kv, ints([64, -1, 2 ** 30]), out, out, status=status)
    assert (out == 3.0).all()


def sequences(sa, lengths, heads, d, group=2, per_query_head=False, local=0):
    """A cache of sequences whose tokens are stored; returns kv and the keys as held, [b][tokens][heads][d]."""
    B = len(lengths)
    stride = max(lengths) // 32 + 2
    rng = np.random.default_rng(sum(lengths))
    table = rng.permutation(B * stride).astype(np.int32).reshape(B, stride)
    kv = sa.PagedKV4(B, heads * group, heads, stride, num_pages=B * stride, head_dim=d,
                     rep_heads=heads * group if per_query_head else None)
    kv.block_table.copy_(ints(table))
    kv.seq_len.copy_(ints(lengths))
    slots = np.concatenate([[table[b, t // 32] * 32 + t % 32 for t in range(n)] for b, n in enumerate(lengths)])
    g = torch.Generator().manual_seed(B)
    k, v = (torch.randn((len(slots), heads, d), generator=g).to(torch.bfloat16) for _ in range(2))
    sa.kv4_store(kv, k.cuda(), v.cuda(), ints(slots))
    held, at = [], 0
    for n in lengths:
        held.append(K.values(f64(k[at:at + n])))
        at += n
    return kv, held, table


def check_reps(kv, held, sealed, group):
    reps = kv.reps.cpu().numpy().astype(np.float64)
    heads = kv.kv_heads
    for b, n in enumerate(sealed):
        for s in range(n):
            want = held[b][32 * s:32 * s + 32].mean(0)  # [heads][d]
            for r in range(kv.rep_heads):
                got = reps[b, r, :, s]
                # a sum of 32 in fp32, each value rounded once: (32 + 1) / 2 steps of the sum of magnitudes
                bound = 2.0 ** -24 * 34 * np.abs(held[b][32 * s:32 * s + 32]).mean(0)[r * heads // kv.rep_heads]
                assert (np.abs(got - want[r * heads // kv.rep_heads]) <= bound).all(), (b, s, r)
        assert not reps[b, :, :, n:].any()


@pytest.mark.parametrize("d,per_query_head,local", [(64, False, 0), (128, True, 0), (128, False, 40), (256, False, 0)])
def test_seal(hip, d, per_query_head, local):
    lengths = [0, 31, 32, 64, 1200, 33, 1057]
    kv, held, _ = sequences(hip, lengths, 3, d, per_query_head=per_query_head)
    status = ints([0])
    kv.sealed[4] = 2  # two blocks are sealed already; their representatives stay as they are
    kv.generation[4] = 7
    hip.kv4_seal(kv, local, status=status)
    sealed = [max(0, (n - local) // 32) for n in lengths]
    assert int(status) == 0
    assert kv.sealed.tolist() == sealed
    assert kv.generation.tolist() == [s - 2 + 7 if i == 4 else s for i, s in enumerate(sealed)]
    assert not kv.reps[4, :, :, :2].any()
    kv.sealed[4] = 0
    hip.kv4_seal(kv, local)
    check_reps(kv, held, sealed, 2)


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("d,heads,local", [(64, 8, 0), (128, 1, 0), (128, 8, 33), (256, 5, 0)])
def test_append_seal(hip, d, heads, local, dtype):
    lengths = [0, 1, 30, 31, 63, 64, 95, 500]
    kv, held, table = sequences(hip, lengths, heads, d)
    hip.kv4_seal(kv, local)
    sealed = [max(0, (n - local) // 32) for n in lengths]
    kv.reps.zero_()
    status = ints([0])
    for step in range(3):
        k, v = tokens(step, len(lengths), heads, d, "fp32"), tokens(9 + step, len(lengths), heads, d, "fp32")
        k[5, 0], v[5, 0] = 1.0, 2.0  # (no infinities in what is averaged)
        k, v = k.to(TYPES[dtype]), v.to(TYPES[dtype])
        before = kv.pool.cpu().numpy().copy()
        hip.kv4_append_seal(kv, k.cuda(), v.cuda(), local, status=status)
        for b, n in enumerate(lengths):
            K.put(before, int(table[b, n // 32]) * 32 + n % 32, f64(k[b]), f64(v[b]))
            held[b] = np.concatenate([held[b], K.values(f64(k[b:b + 1]))])
            lengths[b] += 1
        np.testing.assert_array_equal(kv.pool.cpu().numpy(), before)
        assert kv.seq_len.tolist() == lengths
        now = [max(0, (n - local) // 32) for n in lengths]
        assert kv.sealed.tolist() == now
        reps = kv.reps.cpu().numpy().astype(np.float64)
        for b in range(len(lengths)):
            for s in range(sealed[b], now[b]):
                block = held[b][32 * s:32 * s + 32]
                bound = 2.0 ** -24 * 34 * np.abs(block).mean(0)
                assert (np.abs(reps[b, :, :, s] - block.mean(0)) <= bound).all()
        sealed = now
    assert int(status) == 0


def test_append_without_room(hip):
    """A sequence whose table row is full, whose page is none, or whose lengths disagree is left as it is."""
    kv, _, table = sequences(hip, [64, 64, 64, 64], 2, 64)
    kv.seq_len[0] = table.shape[1] * 32
    kv.block_table[1, 2] = 10 ** 6
    kv.sealed[2] = 3
    kv.sealed[0] = 2
    before = kv.pool.clone()
    lens = kv.seq_len.clone()
    status = ints([0])
    x = torch.randn(4, 2, 64, device="cuda")
    hip.kv4_append_seal(kv, x, x, 0, status=status)
    assert int(status) == 12
    assert kv.seq_len.tolist() == [int(lens[0]), 64, 64, 65] and kv.sealed.tolist() == [2, 0, 3, 2]
    changed = (kv.pool != before).any(-1).any(-1).nonzero().flatten().tolist()
    assert changed == [int(table[3, 2])]


def test_seal_stops_at_a_missing_page(hip):
    kv, held, _ = sequences(hip, [200], 2, 128)
    kv.block_table[0, 3] = -1
    status = ints([0])
    hip.kv4_seal(kv, 0, status=status)
    assert int(status) == 8 and kv.sealed.tolist() == [3] and kv.generation.tolist() == [3]
