"""The page stack, the 4-bit cache, the selection and the attention as a serving loop uses them: prompts come in, every
sequence takes a token a step, some end and give their pages to the next.  Every step against 64-bit attention over
what was written."""
import numpy as np
import pytest
import torch

import kv4_oracle as K

pytestmark = pytest.mark.gpu
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
EPS = {t: torch.finfo(d).eps / 2 for t, d in TYPES.items()}
LOCAL = 64  # tokens a block stays out of the sealed ones


def ints(a):
    return torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()


class Loop:
    """A cache with its stack, and beside it each sequence's keys and values as the format holds them."""

    def __init__(self, sa, batch, heads, group, d, dtype, pages, stride, seed):
        self.sa, self.d, self.dtype, self.heads, self.group = sa, d, dtype, heads, group
        self.rng = np.random.default_rng(seed)
        self.kv = sa.PagedKV4(batch, heads * group, heads, stride, num_pages=pages, head_dim=d)
        self.kv.pool.fill_(0xFF)  # NaN scales and minima wherever nothing was written
        self.free = ints(self.rng.permutation(pages))
        self.count = ints([pages])
        self.start, self.status = ints(np.zeros(batch + 1)), ints([0])
        self.k = [np.zeros((0, heads, d)) for _ in range(batch)]
        self.v = [np.zeros((0, heads, d)) for _ in range(batch)]
        self.ws = sa.kv4_attention_workspace(self.kv, 512)
        self.scores = torch.zeros(batch, heads, self.kv.rep_stride).cuda()
        self.scale = d ** -0.5

    def rows(self, n, heads):
        return torch.from_numpy(self.rng.standard_normal((n, heads, self.d))).to(TYPES[self.dtype])

    def hold(self, b, k, v):
        """What the cache gives back for these tokens."""
        self.k[b] = np.concatenate([self.k[b], K.values(k.float().numpy())])
        self.v[b] = np.concatenate([self.v[b], K.values(v.float().numpy())])

    def prompts(self, new):
        """new[b] tokens into each sequence: pages, rows, seal, attention."""
        sa, kv, n = self.sa, self.kv, int(np.sum(new))
        slots, positions = ints(np.full(n + 3, 5)), ints(np.full(n + 3, 5))
        sa.reserve_tokens(kv, ints(new), self.free, self.count, self.start, slots, positions, status=self.status)
        k, v, q = self.rows(n, self.heads), self.rows(n, self.heads), self.rows(n, self.heads * self.group)
        sa.kv4_store(kv, k.cuda(), v.cuda(), slots[:n], status=self.status)
        sa.kv4_seal(kv, LOCAL, status=self.status)
        out = sa.kv4_prompt_attention(kv, q.cuda(), self.start, self.scale, workspace=self.ws, status=self.status)
        assert int(self.status) == 0
        at = np.concatenate([[0], np.cumsum(new)])
        assert self.start.cpu().tolist() == at.tolist()
        assert (slots[n:] == -1).all() and (positions[n:] == -1).all()
        for b, m in enumerate(new):
            before = len(self.k[b])
            assert positions[at[b]:at[b + 1]].cpu().tolist() == list(range(before, before + m))
            self.hold(b, k[at[b]:at[b + 1]], v[at[b]:at[b + 1]])
            for i in range(m):
                self.check(b, q[at[b] + i], out[at[b] + i], before + i + 1, None, rounded=True)

    def check(self, b, q, out, seen, blocks, rounded=False):
        """One token's output; blocks [heads]: the sealed blocks it attends besides the tail, or all tokens."""
        q, out = q.double().numpy(), out.double().cpu().numpy()
        for h in range(self.heads):
            at = np.arange(seen)
            if blocks is not None:
                sealed = int(self.kv.sealed[b])
                at = at[np.isin(at // 32, blocks[h]) | (at >= 32 * sealed)]
            rows = slice(h * self.group, (h + 1) * self.group)
            k, v = self.k[b][at, h], self.v[b][at, h]
            want, _ = K.attend(q[rows], k, v, self.scale)
            bound = K.error_bound(q[rows], k, v, self.scale, self.dtype, EPS[self.dtype],
                                  rounded)
            assert (np.abs(out[rows] - want) <= bound + 1e-30).all(), (b, h, seen)

    def step(self, budget):
        """A token for every sequence: pages, append and seal, selection, attention."""
        sa, kv, B = self.sa, self.kv, self.kv.batch
        slots, ahead = ints(np.zeros(B)), ints(np.zeros(B))
        sa.reserve_tokens(kv, ints(np.ones(B)), self.free, self.count, self.start, slots, seq_len_out=ahead,
                          status=self.status)
        k, v, q = self.rows(B, self.heads), self.rows(B, self.heads), self.rows(B, self.heads * self.group)
        sa.kv4_append_seal(kv, k.cuda(), v.cuda(), LOCAL, status=self.status)
        assert kv.seq_len.tolist() == ahead.tolist()
        selected = counts = None
        if budget:
            selected, counts = sa.score_select(kv, q.float().cuda(), self.heads, budget, 1, 1, scores=self.scores,
                                               status=self.status)
        out = sa.kv4_decode_attention(kv, q.cuda(), self.scale, selected, counts, workspace=self.ws,
                                      status=self.status)
        assert int(self.status) == 0
        for b in range(B):
            self.hold(b, k[b:b + 1], v[b:b + 1])
            blocks = None
            if budget:
                sel, n = selected[b].cpu().numpy(), counts[b].cpu().numpy()
                assert (n == min(budget, int(kv.sealed[b]))).all()
                blocks = [sel[h, :n[h]] for h in range(self.heads)]
            self.check(b, q[b], out[b], len(self.k[b]), blocks)

    def release(self, gone):
        before = int(self.count)
        finished = np.zeros(self.kv.batch)
        finished[gone] = 1
        self.sa.release_sequences(self.kv, ints(finished), self.free, self.count, status=self.status)
        assert int(self.status) == 0
        assert int(self.count) == before + sum(-(-len(self.k[b]) // 32) for b in gone)
        for b in gone:
            self.k[b], self.v[b] = self.k[b][:0], self.v[b][:0]

    def no_page_twice(self):
        held = [p for b in range(self.kv.batch)
                for p in self.kv.block_table[b, :-(-len(self.k[b]) // 32)].cpu().tolist()]
        free = self.free[:int(self.count)].cpu().tolist()
        assert sorted(held + free) == list(range(self.kv.num_pages))


@pytest.mark.parametrize("d,heads,group,dtype", [(64, 3, 1, "fp32"), (128, 2, 4, "bf16"), (128, 1, 2, "fp16"),
                                                 (256, 2, 2, "fp16")])
def test_serving_loop(hip, d, heads, group, dtype):
    loop = Loop(hip, 4, heads, group, d, dtype, pages=33, stride=12, seed=d + heads)
    loop.prompts([130, 1, 64, 31])
    loop.no_page_twice()
    for i in range(3):
        loop.step(2 if i else 0)
    loop.release([0, 2])
    loop.prompts([33, 0, 200, 2])  # two new prompts; one sequence takes two tokens at once, one none
    loop.no_page_twice()
    for i in range(2):
        loop.step(3)
    loop.release([0, 1, 2, 3])
    loop.no_page_twice()
    assert int(loop.count) == 33


def test_serving_step_in_a_graph(hip):
    """The decode step of four operators captured once and replayed, against the same steps called one by one."""
    B, heads, group, d = 3, 2, 2, 64
    runs = []
    for captured in (False, True):
        loop = Loop(hip, B, heads, group, d, "fp32", pages=40, stride=12, seed=1)
        loop.prompts([95, 30, 7])
        one, slots, ahead = ints(np.ones(B)), ints(np.zeros(B)), ints(np.zeros(B))
        k, v = torch.zeros(B, heads, d).cuda(), torch.zeros(B, heads, d).cuda()
        q, out = torch.zeros(B, heads * group, d).cuda(), torch.zeros(B, heads * group, d).cuda()
        selected, counts = ints(np.full((B, heads, 2), -1)), ints(np.zeros((B, heads)))
        status = ints([0])

        def step():
            hip.reserve_tokens(loop.kv, one, loop.free, loop.count, loop.start, slots, seq_len_out=ahead,
                               status=status)
            hip.kv4_append_seal(loop.kv, k, v, LOCAL, status=status)
            hip.score_select(loop.kv, q, heads, 2, 1, 1, selected=selected, counts=counts, scores=loop.scores,
                             status=status)
            hip.kv4_decode_attention(loop.kv, q, loop.scale, selected, counts, out=out, workspace=loop.ws,
                                     status=status)

        if captured:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):  # (captures only: nothing is written)
                step()
        outs = []
        g = torch.Generator().manual_seed(9)
        for i in range(70):  # past two block borders
            for x in (k, v, q):
                x.copy_(torch.randn(x.shape, generator=g))
            graph.replay() if captured else step()
            outs.append(out.cpu().numpy().copy())
            assert int(status) == 0
        runs.append((outs, loop.kv.seq_len.tolist(), loop.kv.sealed.tolist(), loop.kv.block_table.cpu().numpy(),
                     loop.kv.pool.cpu().numpy(), int(loop.count)))
    for a, b in zip(runs[0][0], runs[1][0]):
        assert np.array_equal(a, b)
    assert runs[0][1:3] == runs[1][1:3] and runs[0][5] == runs[1][5]
    assert np.array_equal(runs[0][3], runs[1][3]) and np.array_equal(runs[0][4], runs[1][4])
    assert runs[0][1] == [165, 100, 77]
