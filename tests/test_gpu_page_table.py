"""Pages handed out and taken back on the GPU (reserve_tokens, release_sequences) against a plain implementation:
whole numbers, so everything is equal."""
import numpy as np
import pytest
import torch

import kv4_oracle as K

pytestmark = pytest.mark.gpu


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()


def batch(seed, B, longest, spare=1):
    """A batch on a shuffled pool: table, lengths, free stack (with `spare` more pages than blocks held)."""
    rng = np.random.default_rng(seed)
    seq_len = rng.integers(0, longest + 1, B).astype(np.int32)
    blocks = -(-seq_len // 32)
    num_pages = int(blocks.sum()) + spare
    perm = rng.permutation(num_pages).astype(np.int32)
    stride = int(blocks.max()) + 3
    table = np.full((B, stride), -1, np.int32)
    at = 0
    for b in range(B):
        table[b, :blocks[b]] = perm[at:at + blocks[b]]
        at += blocks[b]
    free = np.zeros(num_pages, np.int32)
    free[:spare] = perm[at:]
    return rng, table, seq_len, free, spare, num_pages


def view(sa, table, seq_len, num_pages):
    kv = sa.PagedKV4(table.shape[0], 2, 1, table.shape[1], num_pages=num_pages, rep_stride=1, head_dim=64,
                     pool=torch.zeros((num_pages, 1, 40 * 64), dtype=torch.uint8, device="cuda"))
    kv.block_table = dev(table)
    kv.seq_len = dev(seq_len)
    return kv


def call(sa, kv, new, free, count, max_tokens, in_place=True, positions=True):
    B = kv.batch
    f = dev(free)
    c = dev([count])
    out = {"start": dev(np.full(B + 1, 77)), "slots": dev(np.full(max_tokens, 77)),
           "pos": dev(np.full(max_tokens, 77)) if positions else None,
           "len": kv.seq_len if in_place else dev(np.full(B, 77)), "count": c if in_place else dev([77]),
           "status": dev([0])}
    sa.reserve_tokens(kv, dev(new), f, c, out["start"], out["slots"], out["pos"],
                      seq_len_out=None if in_place else out["len"], free_count_out=None if in_place else out["count"],
                      status=out["status"])
    return {k: v.cpu().numpy() for k, v in out.items() if v is not None}


def same(got, kv, expect):
    ok, table, seq_len, count, start, slots, positions = expect
    np.testing.assert_array_equal(kv.block_table.cpu().numpy(), table)
    np.testing.assert_array_equal(got["len"], seq_len)
    assert got["count"][0] == count
    np.testing.assert_array_equal(got["start"], start)
    np.testing.assert_array_equal(got["slots"], slots)
    if "pos" in got:
        np.testing.assert_array_equal(got["pos"], positions)


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("B,longest,most", [(1, 0, 1), (1, 31, 1), (1, 64, 5000), (3, 70, 40), (64, 300, 1),
                                            (257, 90, 70), (1025, 40, 9), (3000, 33, 3)])
def test_reserve(hip, B, longest, most, in_place):
    rng, table, seq_len, free, spare, num_pages = batch(B + most, B, longest, spare=B * (most // 32 + 2))
    if table.shape[1] < (longest + most) // 32 + 2:
        table = np.pad(table, ((0, 0), (0, (longest + most) // 32 + 2 - table.shape[1])), constant_values=-1)
    new = rng.integers(0, most + 1, B).astype(np.int32)
    new[0] = most
    kv = view(hip, table, seq_len, num_pages)
    rows = int(new.sum()) + 5
    expect = K.reserve(table, seq_len, new, free, spare, rows, num_pages)
    assert expect[0]
    got = call(hip, kv, new, free, spare, rows, in_place=in_place, positions=B != 3)
    assert got["status"][0] == 0
    same(got, kv, expect)


def test_reserve_nothing_new(hip):
    _, table, seq_len, free, spare, num_pages = batch(5, 9, 100)
    kv = view(hip, table, seq_len, num_pages)
    got = call(hip, kv, np.zeros(9), free, spare, 0)
    same(got, kv, K.reserve(table, seq_len, np.zeros(9, np.int32), free, spare, 0, num_pages))
    assert got["status"][0] == 0


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("rows", [600, 9000])
@pytest.mark.parametrize("why,status", [("pages", 8), ("rows", 8), ("table", 8), ("negative length", 4),
                                        ("negative tokens", 4), ("past 32 bits", 4), ("count", 4)])
def test_reserve_all_or_nothing(hip, why, status, rows, in_place):
    """What does not fit hands out nothing, with one workgroup and with several."""
    rng, table, seq_len, free, spare, num_pages = batch(7, 20, 200, spare=rows // 32 + 40)
    new = np.full(20, (rows - 40) // 20, np.int32)
    table = np.pad(table, ((0, 0), (0, new[0] // 32 + 2)), constant_values=-1)
    count, cap = spare, rows
    if why == "pages":
        count = 3
    elif why == "rows":
        cap = int(new.sum()) - 1
    elif why == "table":
        seq_len[4] = table.shape[1] * 32 - 1
    elif why == "negative length":
        seq_len[3] = -1
    elif why == "negative tokens":
        new[19] = -2
    elif why == "past 32 bits":
        seq_len[2] = 2 ** 31 - 3
    else:
        count = num_pages + 1
    kv = view(hip, table, seq_len, num_pages)
    got = call(hip, kv, new, free, count, cap, in_place=in_place)
    assert got["status"][0] & status
    np.testing.assert_array_equal(kv.block_table.cpu().numpy(), table)
    np.testing.assert_array_equal(got["len"], seq_len)
    assert got["count"][0] == count
    assert not got["start"].any() and (got["slots"] == -1).all() and (got["pos"] == -1).all()


def test_reserve_bad_page_ids(hip):
    """A page id outside the pool, on the stack or in a partly filled block, gives its tokens slot -1."""
    table = np.array([[2, -1, -1], [9, -1, -1], [0, -1, -1]], np.int32)  # 9 is no page
    seq_len = np.array([30, 30, 30], np.int32)
    free = np.array([1, 50, 3, 0, 0], np.int32)  # the second page taken, 50, is none
    kv = view(hip, table, seq_len, 5)
    got = call(hip, kv, np.array([4, 4, 4]), free, 3, 12)
    assert got["status"][0] == 1
    same(got, kv, K.reserve(table, seq_len, np.array([4, 4, 4]), free, 3, 12, 5))


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("B,longest", [(1, 1), (5, 100), (200, 2000), (1500, 64)])
def test_release_then_reserve(hip, B, longest, in_place):
    rng, table, seq_len, free, spare, num_pages = batch(B, B, longest)
    finished = (rng.random(B) < 0.4).astype(np.int32)
    finished[-1] = 5
    kv = view(hip, table, seq_len, num_pages)
    kv.sealed.copy_(dev(seq_len // 32))
    f, c, status = dev(free), dev([spare]), dev([0])
    out_len, out_count = (kv.seq_len, c) if in_place else (dev(np.full(B, 9)), dev([9]))
    hip.release_sequences(kv, dev(finished), f, c, seq_len_out=None if in_place else out_len,
                          free_count_out=None if in_place else out_count, status=status)
    ok, lens, pages, count = K.release(table, seq_len, finished, free, spare, num_pages)
    assert ok and int(status) == 0
    np.testing.assert_array_equal(out_len.cpu().numpy(), lens)
    assert int(out_count) == count
    np.testing.assert_array_equal(f.cpu().numpy()[:count], pages[:count])
    np.testing.assert_array_equal(kv.sealed.cpu().numpy(), np.where(finished, 0, seq_len // 32))
    kv.seq_len = out_len
    new = np.where(finished, 33, 0).astype(np.int32)
    if table.shape[1] < 2:
        return
    got = call(hip, kv, new, pages, count, int(new.sum()))
    same(got, kv, K.reserve(table, lens, new, pages, count, int(new.sum()), num_pages))


def test_release_refuses_more_than_the_pool(hip):
    _, table, seq_len, free, spare, num_pages = batch(3, 6, 200)
    kv = view(hip, table, seq_len, num_pages)
    kv.sealed.fill_(1)
    for count, why in ((num_pages - 1, 8), (-3, 4)):
        f, c, status = dev(free), dev([count]), dev([0])
        hip.release_sequences(kv, dev(np.ones(6)), f, c, status=status)
        assert int(status) & why and int(c) == count
        np.testing.assert_array_equal(f.cpu().numpy(), free)
        np.testing.assert_array_equal(kv.seq_len.cpu().numpy(), seq_len)
        assert (kv.sealed == 1).all()


def test_captured_step(hip):
    """A captured reserve replays on new lengths; every replay equals the plain implementation."""
    rng, table, seq_len, free, spare, num_pages = batch(11, 40, 300, spare=60)
    kv = view(hip, table, seq_len, num_pages)
    f, c = dev(free), dev([spare])
    new = dev(np.ones(40))
    start, slots, pos, status = dev(np.zeros(41)), dev(np.zeros(40)), dev(np.zeros(40)), dev([0])
    hip.reserve_tokens(kv, dev(np.zeros(40)), f, c, start, slots, pos, status=status)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        hip.reserve_tokens(kv, new, f, c, start, slots, pos, status=status)
    count = spare
    for step in range(6):
        n = (rng.random(40) < 0.7).astype(np.int32)
        new.copy_(dev(n))
        ok, table, seq_len, count, s, sl, ps = K.reserve(table, seq_len, n, free, count, 40, num_pages)
        assert ok
        graph.replay()
        torch.cuda.synchronize()
        assert int(c) == count and int(status) == 0
        np.testing.assert_array_equal(kv.block_table.cpu().numpy(), table)
        np.testing.assert_array_equal(kv.seq_len.cpu().numpy(), seq_len)
        np.testing.assert_array_equal(start.cpu().numpy(), s)
        np.testing.assert_array_equal(slots.cpu().numpy(), sl)
        np.testing.assert_array_equal(pos.cpu().numpy(), ps)
