"""Attention over the 4-bit pages against 64-bit softmax attention over the values that the cache holds."""
import numpy as np
import pytest
import torch

import kv4_oracle as K

pytestmark = pytest.mark.gpu
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
EPS = {t: torch.finfo(d).eps / 2 for t, d in TYPES.items()}


def ints(a):
    return torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()


class Cache:
    """Sequences of the given lengths in a pool of random bytes (NaN halves among them), pages shuffled."""

    def __init__(self, sa, lengths, heads, d, group, seed=0, size=1.0, spare=0):
        self.lengths, self.heads, self.d, self.group = list(lengths), heads, d, group
        B = len(lengths)
        self.stride = max(lengths) // 32 + 2
        g = torch.Generator().manual_seed(seed + B)
        pages = B * self.stride + spare
        self.table = torch.randperm(pages, generator=g)[:B * self.stride].view(B, -1).numpy().astype(np.int32)
        self.kv = sa.PagedKV4(B, heads * group, heads, self.stride, num_pages=pages, head_dim=d)
        self.kv.pool.copy_(torch.randint(0, 256, self.kv.pool.shape, generator=g, dtype=torch.uint8))
        self.kv.block_table.copy_(ints(self.table))
        self.kv.seq_len.copy_(ints(lengths))
        self.kv.sealed.copy_(ints([n // 32 for n in lengths]))
        n = sum(lengths)
        if n:
            slots = np.concatenate([self.table[b, np.arange(m) // 32] * 32 + np.arange(m) % 32
                                    for b, m in enumerate(lengths)])
            k, v = torch.randn((n, heads, d), generator=g) * size, torch.randn((n, heads, d), generator=g) * size
            k[..., :4] *= 3.0
            v[..., 5] += 2.0
            sa.kv4_store(self.kv, k.cuda(), v.cuda(), ints(slots))
        self.refresh()

    def refresh(self):
        self.k, self.v = K.read(self.kv.pool.cpu().numpy())  # [pages][heads][32][d]

    def rows(self, b, h, blocks, n):
        """Keys and values of the tokens below n of the blocks given."""
        ids = self.table[b, blocks]
        at = (np.asarray(blocks)[:, None] * 32 + np.arange(32)).reshape(-1)
        k, v = self.k[ids, h].reshape(-1, self.d), self.v[ids, h].reshape(-1, self.d)
        return k[at < n], v[at < n]


def check(got, want, bound, what=""):
    err = np.abs(got - want)
    assert (err <= bound).all(), (what, float((err / bound).max()), float(err.max()))


def query(seed, n, heads, d, dtype, size=1.0):
    return (torch.randn((n, heads, d), generator=torch.Generator().manual_seed(seed)) * size).to(TYPES[dtype])


def check_decode(c, q, out, dtype, scale, selected=None, counts=None, groups=0):
    q, out = q.double().numpy(), out.double().cpu().numpy()
    for b, n in enumerate(c.lengths):
        for h in range(c.heads):
            if selected is None:
                blocks = list(range((n + 31) // 32))
            else:
                sg = h // (c.heads // groups)
                blocks = list(selected[b, sg, :counts[b, sg]]) + list(range(n // 32, (n + 31) // 32))
            k, v = c.rows(b, h, np.array(blocks, np.int64), n)
            rows = slice(h * c.group, (h + 1) * c.group)
            want, _ = K.attend(q[b, rows], k, v, scale)
            check(out[b, rows], want, K.error_bound(q[b, rows], k, v, scale, dtype, EPS[dtype]) + 1e-30, (b, h))


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("d,heads,group", [(64, 8, 2), (64, 1, 16), (128, 1, 1), (128, 8, 2), (128, 2, 8), (128, 3, 5),
                                           (256, 4, 1), (256, 1, 16)])
def test_decode_whole_sequences(hip, d, heads, group, dtype):
    c = Cache(hip, [0, 1, 31, 32, 33, 64, 500, 1999, 2], heads, d, group)
    q = query(d + group, len(c.lengths), heads * group, d, dtype)
    status = ints([0])
    ws = hip.kv4_attention_workspace(c.kv)
    for _ in range(2):  # the workspace serves one call after the other
        out = hip.kv4_decode_attention(c.kv, q.cuda(), d ** -0.5, workspace=ws, status=status)
        assert int(status) == 0
        check_decode(c, q, out, dtype, d ** -0.5)
    assert not out[0].any()  # a sequence without tokens


@pytest.mark.parametrize("B", [1, 2, 700])
def test_decode_batches(hip, B):
    """One long list over many workgroups, and more short lists than workgroups."""
    lengths = [9000] if B == 1 else [3000, 77] if B == 2 else [(b * 37) % 90 for b in range(B)]
    c = Cache(hip, lengths, 2 if B == 700 else 1, 128, 2)
    q = query(B, B, c.heads * 2, 128, "fp32")
    out = hip.kv4_decode_attention(c.kv, q.cuda(), 128 ** -0.5)
    check_decode(c, q, out, "fp32", 128 ** -0.5)


@pytest.mark.parametrize("d,lengths", [(64, [1, 512, 0, 40]), (128, [300] * 5), (128, [512, 511]), (256, [33, 64, 2]),
                                       (128, [513, 20]), (64, [2000] * 3), (128, [700] * 40),
                                       (64, [1536, 3, 900, 1100] * 13), (128, [1537, 40] * 26)])
def test_decode_short_and_equal_lists(hip, d, lengths):
    """Lists of up to 16 pages with a workgroup each, of up to 48 when there are many, one page more, and lists of one
    length, whose shares end with them; whole sequences and selected blocks."""
    c = Cache(hip, lengths, 4, d, 2, seed=7)
    q = query(8, len(lengths), 8, d, "fp32")
    status = ints([0])
    ws = hip.kv4_attention_workspace(c.kv)
    out = hip.kv4_decode_attention(c.kv, q.cuda(), 0.1, workspace=ws, status=status)
    check_decode(c, q, out, "fp32", 0.1)
    counts = np.stack([np.minimum(3, np.array(lengths) // 32)] * 2, 1)
    selected = np.tile(np.arange(3), (len(lengths), 2, 1))
    out = hip.kv4_decode_attention(c.kv, q.cuda(), 0.1, ints(selected), ints(counts), workspace=ws, status=status)
    check_decode(c, q, out, "fp32", 0.1, selected, counts, 2)
    assert int(status) == 0


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_prompt_short_lists(hip, d, dtype):
    """Tiles of up to 16 pages with a workgroup each, in tiles of few rows and of many, and tiles of one page more."""
    for lengths, new in (([512, 40, 3], [4, 2, 3]), ([512, 100], [512, 100]), ([513, 100], [3, 4]), ([530], [400]),
                         ([1536, 900] * 33, [3, 2] * 33), ([1537, 8] * 33, [2, 3] * 33)):
        c = Cache(hip, lengths, 2, d, 4, seed=6)
        start = np.concatenate([[0], np.cumsum(new)])
        q = query(9, int(start[-1]), 8, d, dtype)
        out = hip.kv4_prompt_attention(c.kv, q.cuda(), ints(start), d ** -0.5)
        check_prompt(c, q, start, out, dtype, d ** -0.5)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("d,heads,group,groups", [(64, 4, 2, 4), (128, 8, 2, 8), (128, 8, 4, 1), (128, 4, 1, 2),
                                                  (256, 2, 8, 2)])
def test_decode_selected_blocks(hip, d, heads, group, groups, dtype):
    lengths = [5, 32, 700, 1500, 64, 95]
    c = Cache(hip, lengths, heads, d, group, seed=3)
    rng = np.random.default_rng(d + heads)
    stride = 19
    selected = np.full((len(lengths), groups, stride), -7, np.int32)
    counts = np.zeros((len(lengths), groups), np.int32)
    for b, n in enumerate(lengths):
        for g in range(groups):
            m = int(rng.integers(0, min(stride, n // 32) + 1))
            selected[b, g, :m] = np.sort(rng.permutation(n // 32)[:m])
            counts[b, g] = m
    q = query(5, len(lengths), heads * group, d, dtype)
    status = ints([0])
    out = hip.kv4_decode_attention(c.kv, q.cuda(), d ** -0.5, ints(selected), ints(counts), status=status)
    assert int(status) == 0
    check_decode(c, q, out, dtype, d ** -0.5, selected, counts, groups)


def check_prompt(c, q, start, out, dtype, scale, untouched=None):
    qn, on = q.double().numpy(), out.double().cpu().numpy()
    for b, n in enumerate(c.lengths):
        m = start[b + 1] - start[b]
        blocks = np.arange((n + 31) // 32)
        for h in range(c.heads):
            k, v = c.rows(b, h, blocks, n)
            rows = slice(h * c.group, (h + 1) * c.group)
            for i in range(m):
                seen = n - m + i + 1
                qq, got = qn[start[b] + i, rows], on[start[b] + i, rows]
                want, _ = K.attend(qq, k[:max(seen, 0)], v[:max(seen, 0)], scale)
                bound = K.error_bound(qq, k[:max(seen, 0)], v[:max(seen, 0)], scale, dtype, EPS[dtype], rounded=True)
                check(got, want, bound + 1e-30, (b, h, i))


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("d,heads,group", [(64, 2, 2), (64, 1, 16), (128, 1, 1), (128, 2, 4), (128, 1, 3), (256, 1, 8)])
def test_prompt(hip, d, heads, group, dtype):
    """Chunks of one token to several hundred, at contexts of none to more than a thousand; some sequences idle."""
    lengths = [1, 40, 257, 32, 1100, 33, 300, 640]
    new = [1, 40, 257, 0, 5, 33, 17, 64]
    c = Cache(hip, lengths, heads, d, group, seed=1)
    start = np.concatenate([[0], np.cumsum(new)])
    rows = int(start[-1]) + 3  # rows behind the last sequence
    q = query(d, rows, heads * group, d, dtype)
    out = torch.full(q.shape, 9.0, dtype=q.dtype, device="cuda")
    status = ints([0])
    ws = hip.kv4_attention_workspace(c.kv, rows)
    for _ in range(2):
        hip.kv4_prompt_attention(c.kv, q.cuda(), ints(start), d ** -0.5, out=out, workspace=ws, status=status)
        assert int(status) == 0
        check_prompt(c, q, start, out, dtype, d ** -0.5)
        assert (out[start[-1]:] == 9.0).all()


def test_prompt_of_one_token_is_decode(hip):
    c = Cache(hip, [5, 64, 900, 1], 4, 128, 2)
    q = query(1, 4, 8, 128, "fp32").cuda()
    a = hip.kv4_decode_attention(c.kv, q, 0.1)
    b = hip.kv4_prompt_attention(c.kv, q, ints([0, 1, 2, 3, 4]), 0.1)
    check_decode(c, q.cpu(), a, "fp32", 0.1)
    check_decode(c, q.cpu(), b, "fp32", 0.1)


def test_prompt_more_rows_than_tokens(hip):
    """Rows before a sequence's first token see nothing: zeros, and a status bit."""
    c = Cache(hip, [3, 50], 2, 128, 2)
    q = query(2, 12, 4, 128, "fp32")
    status = ints([0])
    out = hip.kv4_prompt_attention(c.kv, q.cuda(), ints([0, 7, 12]), 0.1, status=status)
    assert int(status) == 4 and not out[:4].any()
    check_prompt(c, q, [0, 7, 12], out, "fp32", 0.1)


def test_prompt_bad_ranges(hip):
    """Ranges that do not ascend, or pass the rows, would share rows: nothing is written."""
    c = Cache(hip, [60, 50, 40], 1, 64, 1)
    q = query(2, 12, 1, 64, "fp32").cuda()
    ws = hip.kv4_attention_workspace(c.kv, 12)
    for start in ([0, 5, 3, 8], [-2, 5, 8, 12], [0, 5, 8, 13]):
        out = torch.full(q.shape, 4.0, device="cuda")
        status = ints([0])
        hip.kv4_prompt_attention(c.kv, q, ints(start), 0.1, out=out, workspace=ws, status=status)
        assert int(status) == 4 and (out == 4.0).all()
    hip.kv4_prompt_attention(c.kv, q, ints([0, 5, 8, 12]), 0.1, out=out, workspace=ws)
    check_prompt(c, q.cpu(), [0, 5, 8, 12], out, "fp32", 0.1)


@pytest.mark.parametrize("what", ["sharp", "flat", "tiny", "large", "one query"])
def test_extremes(hip, what):
    """Scores far apart, all alike, values near FP16's smallest, cache values near the limit, queries of 1e20."""
    size = {"tiny": 3e-6, "large": 6000.0}.get(what, 1.0)
    c = Cache(hip, [700, 33], 2, 128, 4, size=size)
    q = query(4, 2, 8, 128, "fp32", {"sharp": 40.0, "flat": 1e-6, "tiny": 1e5, "large": 1e-4, "one query": 1.0}[what])
    if what == "one query":
        q[1] *= 1e20
        q[0, 0] = 0.0
    out = hip.kv4_decode_attention(c.kv, q.cuda(), 128 ** -0.5)
    if what == "one query":  # the largest score takes it all
        on = out.double().cpu().numpy()
        for h in range(2):
            k, v = c.rows(1, h, np.arange(2), 33)
            s = q[1, 4 * h:4 * h + 4].double().numpy() @ k.T
            np.testing.assert_allclose(on[1, 4 * h:4 * h + 4], v[s.argmax(-1)], rtol=0, atol=2.0 ** -17 * np.abs(v).max())
        c.lengths = c.lengths[:1]
    check_decode(c, q, out, "fp32", 128 ** -0.5)


def test_long_flat_tail_keeps_its_mass(hip):
    """One token with nearly all the weight and thousands of others whose probabilities lie below FP16's smallest
    number: their sum is not lost."""
    n = 6000
    c = Cache(hip, [n], 1, 64, 1)
    g = torch.Generator().manual_seed(0)
    k = torch.zeros((n, 1, 64))
    k[0, 0, :] = 1.0  # q . k = 18 against 0: each of the others weighs 1.5e-8, together 9e-5
    v = torch.randn((n, 1, 64), generator=g) * 0.01 + 1.0
    v[0] = -1.0
    slots = c.table[0, np.arange(n) // 32] * 32 + np.arange(n) % 32
    hip.kv4_store(c.kv, k.cuda(), v.cuda(), ints(slots))
    c.refresh()
    for dtype in ("fp32", "fp16"):
        q = torch.full((1, 1, 64), 18.0 / 8, dtype=TYPES[dtype])
        out = hip.kv4_decode_attention(c.kv, q.cuda(), 0.125)
        check_decode(c, q, out, dtype, 0.125)
        kk, vv = c.rows(0, 0, np.arange(188), n)
        want, _ = K.attend(q[0].double().numpy(), kk, vv, 0.125)
        moved = (out[0].double().cpu().numpy() + 1.0)
        if dtype == "fp32":
            # The others move the output by 1.8e-4: within 2^-11 of that, besides the roundings of sums next to 1
            # (2^-23) and the 31 tokens of the large one's own page. Each weighs e^-18 < 2^-25, less than half the
            # last bit of a 32-bit sum that holds the 1, so that a matrix product over the page may keep none of them:
            # 31 e^-18 in the numerator (|v| <= 1.05 here) and as much in the denominator.
            assert np.abs(vv).max() < 1.05
            np.testing.assert_allclose(moved, want + 1.0, rtol=2.0 ** -11, atol=2.0 ** -23 + 2.05 * 31 * np.exp(-18.0))


def test_nan_reaches_only_those_who_see_it(hip):
    c = Cache(hip, [100, 70], 2, 128, 2)
    k, v = torch.randn(1, 2, 128), torch.randn(1, 2, 128)
    v[0, 0, 40] = float("nan")       # head 0, channels 32..63 of token 80
    slot = c.table[0, 2] * 32 + 16
    hip.kv4_store(c.kv, k.cuda(), v.cuda(), ints([slot]))
    k2 = torch.randn(1, 2, 128)
    k2[0, 1, 3] = float("nan")       # head 1's key of token 90
    hip.kv4_store(c.kv, k2.cuda(), torch.randn(1, 2, 128).cuda(), ints([c.table[0, 2] * 32 + 26]))
    c.refresh()
    q = query(3, 100 + 70, 4, 128, "fp32")
    out = hip.kv4_prompt_attention(c.kv, q.cuda(), ints([0, 100, 170]), 0.09).cpu()
    nan = torch.zeros(out.shape, dtype=torch.bool)
    nan[80:100, :2, 32:64] = True
    nan[90:100, 2:] = True
    assert torch.equal(out.isnan(), nan)
    clean = torch.where(nan, torch.zeros_like(out), out).double().numpy()
    for b, (n, at) in enumerate(((100, 0), (70, 100))):
        for h in range(2):
            k, v = c.rows(b, h, np.arange((n + 31) // 32), n)
            for i in range(n):
                kk, vv = np.nan_to_num(k[:i + 1]), np.nan_to_num(v[:i + 1])
                qq = q[at + i, 2 * h:2 * h + 2].double().numpy()
                want, _ = K.attend(qq, kk, vv, 0.09)
                keep = ~nan[at + i, 2 * h:2 * h + 2].numpy()
                err = np.abs(clean[at + i, 2 * h:2 * h + 2] - want)
                bound = np.broadcast_to(K.error_bound(qq, kk, vv, 0.09, "fp32", EPS["fp32"]), err.shape)
                assert (err[keep] <= bound[keep]).all(), (b, h, i)
    one = hip.kv4_decode_attention(c.kv, q[:2].cuda(), 0.09).cpu()
    assert one[0, :2, 32:64].isnan().all() and not one[0, :2, :32].isnan().any() and one[0, 2:].isnan().all()
    assert not one[1].isnan().any()


def test_bad_pages_and_lengths(hip):
    """Pages outside the pool and blocks outside the sealed range are flagged and passed over."""
    c = Cache(hip, [200, 100, 64], 2, 128, 2)
    q = query(6, 3, 4, 128, "fp32")
    c.kv.block_table[0, 2] = c.kv.num_pages
    c.kv.block_table[0, 4] = -3
    status = ints([0])
    out = hip.kv4_decode_attention(c.kv, q.cuda(), 0.1, status=status).double().cpu().numpy()
    assert int(status) == 1
    k, v = c.rows(0, 1, np.array([0, 1, 3, 5, 6]), 200)
    want, _ = K.attend(q[0, 2:4].double().numpy(), k, v, 0.1)
    check(out[0, 2:4], want, K.error_bound(q[0, 2:4].double().numpy(), k, v, 0.1, "fp32", EPS["fp32"]))
    selected = ints([[[1, 9, -1, 0]], [[0, 3, 2, 1]], [[1, 0, 0, 0]]])
    status.zero_()
    c.kv.seq_len[2] = -5
    out = hip.kv4_decode_attention(c.kv, q.cuda(), 0.1, selected, ints([[3], [5], [1]]), status=status)
    assert int(status) == 2 + 4
    out = out.double().cpu().numpy()
    k, v = c.rows(0, 0, np.array([1, 6]), 200)
    want, _ = K.attend(q[0, :2].double().numpy(), k, v, 0.1)
    check(out[0, :2], want, K.error_bound(q[0, :2].double().numpy(), k, v, 0.1, "fp32", EPS["fp32"]))
    k, v = c.rows(1, 0, np.array([3]), 100)  # a count past the stride: the tail alone
    want, _ = K.attend(q[1, :2].double().numpy(), k, v, 0.1)
    check(out[1, :2], want, K.error_bound(q[1, :2].double().numpy(), k, v, 0.1, "fp32", EPS["fp32"]))


def test_lengths_past_the_table(hip):
    """A length that no table row holds is flagged; its pages end with the row, and the others are as they were."""
    for lengths, new, dtype in (([60, 100, 33], [1, 1, 1], "fp32"), ([60, 100, 33], [3, 4, 2], "bf16"),
                                ([60, 100, 33], [60, 100, 33], "bf16")):
        c = Cache(hip, lengths, 2, 128, 4)
        c.kv.seq_len[1] = 2 ** 31 - 1
        start = np.concatenate([[0], np.cumsum(new)])
        q = query(6, int(start[-1]), 8, 128, dtype)
        status = ints([0])
        if max(new) == 1:
            out = hip.kv4_decode_attention(c.kv, q.cuda(), 0.1, status=status)
        else:
            out = hip.kv4_prompt_attention(c.kv, q.cuda(), ints(start), 0.1, status=status)
        assert int(status) == 2
        for b in (0, 2):
            rows = slice(start[b], start[b + 1])
            c.lengths = [lengths[b]]
            c.table = c.kv.block_table[b:b + 1].cpu().numpy()
            check_prompt(c, q[rows], [0, new[b]], out[rows], dtype, 0.1)


@pytest.mark.parametrize("d,dtype", [(64, "fp16"), (128, "fp16"), (64, "bf16"), (128, "bf16")])
def test_nan_in_tiles_of_many_rows(hip, d, dtype):
    """A NaN value reaches the channels of its group, a NaN key its head, in the rows that see the token."""
    lengths = [400, 70]
    c = Cache(hip, lengths, 2, d, 4)
    g = torch.Generator().manual_seed(3)
    k, v = torch.randn((1, 2, d), generator=g), torch.randn((1, 2, d), generator=g)
    v[0, 0, 40] = float("nan")       # head 0, channels 32..63 of token 80
    hip.kv4_store(c.kv, k.cuda(), v.cuda(), ints([c.table[0, 2] * 32 + 16]))
    k[0, 1, 3], v[0, 0, 40] = float("nan"), 0.5
    hip.kv4_store(c.kv, k.cuda(), v.cuda(), ints([c.table[0, 6] * 32 + 31]))  # head 1's key of token 223
    c.refresh()
    q = query(3, 470, 8, d, dtype)
    out = hip.kv4_prompt_attention(c.kv, q.cuda(), ints([0, 400, 470]), 0.09).cpu()
    nan = torch.zeros(out.shape, dtype=torch.bool)
    nan[80:400, :4, 32:64] = True
    nan[223:400, 4:] = True
    assert torch.equal(out.isnan(), nan)
    for b, at in ((0, 0), (1, 400)):
        for h in range(2):
            k, v = c.rows(b, h, np.arange((lengths[b] + 31) // 32), lengths[b])
            k, v = np.nan_to_num(k), np.nan_to_num(v)
            for i in range(0, lengths[b], 13):
                rows = slice(4 * h, 4 * h + 4)
                qq, on = q[at + i, rows].double().numpy(), out[at + i, rows].double().numpy()
                want, _ = K.attend(qq, k[:i + 1], v[:i + 1], 0.09)
                bound = K.error_bound(qq, k[:i + 1], v[:i + 1], 0.09, dtype, EPS[dtype], rounded=True)
                keep = ~nan[at + i, rows].numpy()
                assert (np.abs(on - want)[keep] <= np.broadcast_to(bound, on.shape)[keep]).all(), (b, h, i)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_nan_in_tiles_of_few_rows(hip, d, dtype):
    """The same among the last tokens of a sequence, whose rows see a part of their page."""
    c = Cache(hip, [400, 70], 2, d, 4)
    g = torch.Generator().manual_seed(3)
    k, v = torch.randn((1, 2, d), generator=g), torch.randn((1, 2, d), generator=g)
    v[0, 0, 40] = float("nan")       # head 0, channels 32..63 of token 395
    hip.kv4_store(c.kv, k.cuda(), v.cuda(), ints([c.table[0, 12] * 32 + 11]))
    k[0, 1, 3], v[0, 0, 40] = float("nan"), 0.5
    hip.kv4_store(c.kv, k.cuda(), v.cuda(), ints([c.table[0, 12] * 32 + 13]))  # head 1's key of token 397
    c.refresh()
    q = query(3, 14, 8, d, dtype)
    out = hip.kv4_prompt_attention(c.kv, q.cuda(), ints([0, 9, 14]), 0.09).cpu()  # tokens 391.., 65..
    nan = torch.zeros(out.shape, dtype=torch.bool)
    nan[4:9, :4, 32:64] = True
    nan[6:9, 4:] = True
    assert torch.equal(out.isnan(), nan)
    for b, at, m in ((0, 0, 9), (1, 9, 5)):
        n = c.lengths[b]
        for h in range(2):
            k, v = c.rows(b, h, np.arange((n + 31) // 32), n)
            k, v = np.nan_to_num(k), np.nan_to_num(v)
            for i in range(m):
                rows, seen = slice(4 * h, 4 * h + 4), n - m + i + 1
                qq, on = q[at + i, rows].double().numpy(), out[at + i, rows].double().numpy()
                want, _ = K.attend(qq, k[:seen], v[:seen], 0.09)
                bound = K.error_bound(qq, k[:seen], v[:seen], 0.09, dtype, EPS[dtype])
                keep = ~nan[at + i, rows].numpy()
                assert (np.abs(on - want)[keep] <= np.broadcast_to(bound, on.shape)[keep]).all(), (b, h, i)


def test_strided_query_own_buffer_and_stream(hip):
    """Rows inside a fused projection; out over the query; a stream other than the current one."""
    c = Cache(hip, [90, 300, 64], 2, 128, 4)
    fused = torch.randn((3, 8 + 4, 128)).to(torch.bfloat16)
    q = fused[:, :8]
    dev = fused.cuda()
    out = hip.kv4_decode_attention(c.kv, dev[:, :8], 0.08)
    check_decode(c, q, out, "bf16", 0.08)
    own = q.contiguous().cuda()
    hip.kv4_decode_attention(c.kv, own, 0.08, out=own)
    assert torch.equal(own, out)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    other = hip.kv4_decode_attention(c.kv, dev[:, :8], 0.08, stream=s)
    s.synchronize()
    assert torch.equal(other, out)


def test_same_bits_every_time(hip):
    c = Cache(hip, [4000, 31, 700], 2, 128, 2)
    q = query(8, 3, 4, 128, "fp32").cuda()
    a = hip.kv4_decode_attention(c.kv, q, 0.1)
    start = ints([0, 1, 1, 3])
    p = hip.kv4_prompt_attention(c.kv, q, start, 0.1)
    for _ in range(5):
        assert torch.equal(hip.kv4_decode_attention(c.kv, q, 0.1), a)
        assert torch.equal(hip.kv4_prompt_attention(c.kv, q, start, 0.1), p)


@pytest.mark.parametrize("d,heads,group", [(64, 2, 4), (128, 2, 4), (128, 1, 16)])
def test_long_chunks(hip, d, heads, group):
    """Chunks of hundreds of rows at contexts of several thousand: tiles over many pages, cut by shares, and the same
    bits every time; a page that is not there among them."""
    c = Cache(hip, [3000, 700, 2100], heads, d, group, seed=5)
    new = [300, 700, 65]
    start = np.concatenate([[0], np.cumsum(new)])
    q = query(9, int(start[-1]), heads * group, d, "bf16")
    ws = hip.kv4_attention_workspace(c.kv, q.shape[0])
    out = hip.kv4_prompt_attention(c.kv, q.cuda(), ints(start), d ** -0.5, workspace=ws)
    qn, on = q.double().numpy(), out.double().cpu().numpy()
    for b, n in enumerate(c.lengths):
        blocks = np.arange((n + 31) // 32)
        for h in range(heads):
            k, v = c.rows(b, h, blocks, n)
            rows = slice(h * group, (h + 1) * group)
            for i in list(range(0, new[b], 37)) + [new[b] - 1]:
                seen = n - new[b] + i + 1
                qq = qn[start[b] + i, rows]
                want, _ = K.attend(qq, k[:seen], v[:seen], d ** -0.5)
                check(on[start[b] + i, rows], want, K.error_bound(qq, k[:seen], v[:seen], d ** -0.5, "bf16",
                                                                  EPS["bf16"]), (b, h, i))
    for _ in range(4):
        assert torch.equal(hip.kv4_prompt_attention(c.kv, q.cuda(), ints(start), d ** -0.5, workspace=ws), out)
    c.kv.block_table[0, 50] = c.kv.num_pages + 7
    status = ints([0])
    on = hip.kv4_prompt_attention(c.kv, q.cuda(), ints(start), d ** -0.5, workspace=ws, status=status).double().cpu().numpy()
    assert int(status) == 1
    k, v = c.rows(0, 0, np.array([i for i in range(94) if i != 50]), 3000)
    for i in (0, 123, 299):
        seen = 3000 - 300 + i + 1 - 32
        want, _ = K.attend(qn[i, :group], k[:seen], v[:seen], d ** -0.5)
        check(on[i, :group], want, K.error_bound(qn[i, :group], k[:seen], v[:seen], d ** -0.5, "bf16", EPS["bf16"]))


def test_captured(hip):
    """Both calls in one graph, replayed on new queries and lengths."""
    c = Cache(hip, [600, 90, 333], 2, 128, 2)
    q = query(1, 3, 4, 128, "fp32").cuda()
    qp = query(2, 40, 4, 128, "fp32").cuda()
    start = ints([0, 30, 30, 40])
    wa, wb = hip.kv4_attention_workspace(c.kv, 3), hip.kv4_attention_workspace(c.kv, 40)
    a, b = torch.empty_like(q), torch.empty_like(qp)
    run = lambda: (hip.kv4_decode_attention(c.kv, q, 0.1, out=a, workspace=wa),
                   hip.kv4_prompt_attention(c.kv, qp, start, 0.1, out=b, workspace=wb))
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for step in range(4):
        q.copy_(query(10 + step, 3, 4, 128, "fp32"))
        qp.copy_(query(20 + step, 40, 4, 128, "fp32"))
        c.kv.seq_len.copy_(ints([600 - 50 * step, 90 - step, 333]))
        c.lengths = [600 - 50 * step, 90 - step, 333]
        graph.replay()
        torch.cuda.synchronize()
        ga, gb = a.clone(), b.clone()
        check_decode(c, q.cpu(), ga, "fp32", 0.1)
        check_prompt(c, qp.cpu(), [0, 30, 30, 40], gb, "fp32", 0.1)
