"""Calls of the page stack and the 4-bit cache that are refused before anything is launched (no GPU needed)."""
import ctypes as C

import pytest
import torch

import solidattention_amd as sa


def struct(**change):
    kv = sa.PagedKVStruct()
    kv.pool = kv.block_table = kv.seq_len = kv.sealed = kv.reps = 4096
    kv.num_pages, kv.batch, kv.table_stride = 8, 2, 4
    kv.rep_heads, kv.rep_stride, kv.query_heads, kv.kv_heads, kv.head_dim = 2, 4, 4, 2, 128
    kv.reserved = sa.POOL_KV4
    for name, value in change.items():
        setattr(kv, name, value)
    return kv


def refused(rc, what):
    message = sa.lib().sa_hip_last_error().decode()
    assert rc == -1 and what in message, (rc, message)


P = C.c_void_p(1 << 20)
Q = C.c_void_p(1 << 24)
O = C.c_void_p(1 << 28)
KV4_CALLS = {
    "store": lambda kv: sa.lib().sa_hip_kv4_store(C.byref(kv), P, Q, 1, 256, 256, P, 3, None, None),
    "load": lambda kv: sa.lib().sa_hip_kv4_load(C.byref(kv), P, Q, 1, 256, 256, P, 3, None, None),
    "append": lambda kv: sa.lib().sa_hip_kv4_append_seal(C.byref(kv), P, Q, 1, 256, 256, 0, None, None),
    "seal": lambda kv: sa.lib().sa_hip_kv4_seal(C.byref(kv), 0, None, None),
    "decode": lambda kv: sa.lib().sa_hip_kv4_decode_attention(C.byref(kv), P, 1, 512, None, None, 0, 0, C.c_float(1),
                                                              O, P, 1 << 40, None, None),
    "prompt": lambda kv: sa.lib().sa_hip_kv4_prompt_attention(C.byref(kv), P, 1, 512, P, 5, C.c_float(1), O, P,
                                                              1 << 40, None, None),
}


@pytest.mark.parametrize("name", KV4_CALLS)
@pytest.mark.parametrize("change,what", [
    ({"reserved": 0}, "does not hold 4-bit pages"), ({"head_dim": 96}, "head_dim 96"), ({"head_dim": 0}, "head_dim 0"),
    ({"query_heads": 3}, "3/2"), ({"kv_heads": 0}, "4/0"), ({"query_heads": 34}, "17 query heads"),
    ({"num_pages": 0}, "num_pages"), ({"num_pages": 1 << 26}, "num_pages"), ({"pool": None}, "pool"),
    ({"pool": 4100}, "pool")])
def test_cache_shapes(name, change, what):
    refused(KV4_CALLS[name](struct(**change)), what)


@pytest.mark.parametrize("name", ["append", "seal", "decode", "prompt"])
@pytest.mark.parametrize("change,what", [({"batch": 0}, "batch 0"), ({"batch": 65536}, "batch"),
                                         ({"table_stride": 0}, "table_stride"), ({"block_table": None}, "null table"),
                                         ({"seq_len": None}, "null table"), ({"sealed": None}, "null table")])
def test_cache_tables(name, change, what):
    refused(KV4_CALLS[name](struct(**change)), what)


@pytest.mark.parametrize("name", ["append", "seal"])
def test_representatives(name):
    refused(KV4_CALLS[name](struct(reps=None)), "reps")
    refused(KV4_CALLS[name](struct(rep_heads=3)), "rep_heads")
    refused(KV4_CALLS[name](struct(rep_stride=0)), "rep_stride")


def test_rows():
    L, kv = sa.lib(), C.byref(struct())
    odd = C.c_void_p((1 << 20) + 8)
    for k, v, type_, ks, vs, slots, n, what in (
            (None, P, 1, 256, 256, P, 3, "null k"), (P, None, 1, 256, 256, P, 3, "null v"),
            (odd, P, 1, 256, 256, P, 3, "aligned"), (P, P, 1, 260, 256, P, 3, "aligned"),
            (P, P, 0, 256, 258, P, 3, "aligned"), (P, P, 1, 255, 256, P, 3, "apart"), (P, P, 7, 256, 256, P, 3, "type 7"),
            (P, P, 1, 256, 256, None, 3, "slots"), (P, P, 1, 256, 256, P, -1, "-1 tokens"),
            (P, P, 1, 256, 256, P, 2 ** 31 - 1, "exceed")):
        refused(L.sa_hip_kv4_store(kv, k, v, type_, ks, vs, slots, n, None, None), what)
        refused(L.sa_hip_kv4_load(kv, k, v, type_, ks, vs, slots, n, None, None), what)
    assert L.sa_hip_kv4_store(kv, None, None, 1, 0, 0, None, 0, None, None) == 0  # no tokens: nothing to do
    assert L.sa_hip_kv4_page_bytes(8, 128) == 8 * 5120 and L.sa_hip_kv4_page_bytes(8, 96) == 0


def test_attention_arguments():
    L, kv = sa.lib(), C.byref(struct())
    one = C.c_float(1)
    decode = lambda q=P, t=1, qs=512, sel=None, cnt=None, g=0, ss=0, out=O, ws=P, n=1 << 40: \
        L.sa_hip_kv4_decode_attention(kv, q, t, qs, sel, cnt, g, ss, one, out, ws, n, None, None)
    refused(decode(q=None), "null query")
    refused(decode(t=3), "type 3")
    refused(decode(qs=511), "apart")
    refused(decode(qs=514), "aligned")
    refused(decode(out=None), "out")
    refused(decode(ws=None), "workspace")
    refused(decode(n=1000), "workspace")
    refused(decode(ws=C.c_void_p((1 << 20) + 4)), "workspace")
    refused(decode(sel=P), "counts")
    refused(decode(sel=P, cnt=P, g=0, ss=4), "select_groups")
    refused(decode(sel=P, cnt=P, g=3, ss=4), "select_groups")
    refused(decode(sel=P, cnt=P, g=2, ss=0), "sel_stride")
    refused(L.sa_hip_kv4_decode_attention(C.byref(struct(batch=64, table_stride=1 << 25)), P, 1, 512, None, None, 0, 0,
                                          one, O, P, 1 << 40, None, None), "2^31 page reads")
    refused(decode(out=C.c_void_p((1 << 20) + 512)), "overlap")
    prompt = lambda st=P, n=5, q=P, qs=512, out=O, ws=1 << 40: \
        L.sa_hip_kv4_prompt_attention(kv, q, 1, qs, st, n, one, out, P, ws, None, None)
    refused(prompt(st=None), "query_start")
    refused(prompt(n=-1), "-1 query_tokens")
    refused(prompt(q=None), "null query")
    refused(prompt(qs=520, out=P), "overlap")
    refused(prompt(ws=16), "workspace")
    assert prompt(n=0) == 0
    assert L.sa_hip_kv4_attention_workspace_bytes(kv, -1) == 0
    a, b = (L.sa_hip_kv4_attention_workspace_bytes(kv, n) for n in (2, 5000))
    assert 0 < a < b


def test_16_bit_pages_entry_points_refuse_the_4_bit_pool():
    L, kv = sa.lib(), C.byref(struct())
    p = sa.SelectParamsStruct(2, 4, 1, 1, 4, 0, None)
    f = C.c_float(1)
    for call in (lambda: L.sa_hip_append_seal(kv, P, P, 0, None, None),
                 lambda: L.sa_hip_append_seal_f16(kv, P, P, 0, None, None), lambda: L.sa_hip_seal(kv, 0, None, None),
                 lambda: L.sa_hip_sparse_decode_attention(kv, P, P, P, 2, 4, f, P, None, 0, 1, None, None),
                 lambda: L.sa_hip_sparse_decode_attention_chunked(kv, P, P, P, 2, 4, f, P, P, 1 << 30, 4, 4, None, None),
                 lambda: L.sa_hip_sparse_decode_attention_partial(kv, P, P, P, 2, 4, f, 1, P, 1 << 30, 0, 1, 2, None,
                                                                  None),
                 lambda: L.sa_hip_attention_merge(kv, P, 1 << 30, 2, P, None),
                 lambda: L.sa_hip_select_attend(kv, P, C.byref(p), f, P, P, P, None, 0, 1, None, None),
                 lambda: L.sa_hip_decode_step(kv, P, P, 0, P, C.byref(p), f, P, P, P, P, 1 << 30, 1, None, None),
                 lambda: L.sa_hip_decode_step_f16(kv, P, P, 0, P, C.byref(p), f, P, P, P, P, 1 << 30, 1, None, None),
                 lambda: L.sa_hip_read_step_bytes(kv, P, P, 2, 4, P, None, None)):
        refused(call(), "4-bit pages")


def test_page_stack_arguments():
    L = sa.lib()

    def reserve(kv, new=P, free=P, count=P, n=4, start=P, slots=P, out_len=Q, out_count=O):
        return L.sa_hip_reserve_tokens(C.byref(kv), new, free, count, n, start, slots, None, out_len, out_count, None, None)

    def release(kv, gone=P, free=P, count=P, out_len=Q, out_count=O):
        return L.sa_hip_release_sequences(C.byref(kv), gone, free, count, out_len, out_count, None, None)

    for call in (reserve, release):
        refused(call(struct(batch=0)), "batch 0")
        refused(call(struct(table_stride=0)), "table_stride")
        refused(call(struct(num_pages=1 << 26)), "num_pages")
        refused(call(struct(block_table=None)), "null table")
        refused(call(struct(), free=None), "null")
        refused(call(struct(), count=None), "null")
        refused(call(struct(), out_len=None), "null")
        refused(call(struct(), out_count=None), "null")
        refused(call(struct(), out_len=C.c_void_p(4096 + 4)), "overlap")
        refused(call(struct(), count=P, out_count=C.c_void_p((1 << 20) + 2)), "overlap")
    refused(reserve(struct(), new=None), "null")
    refused(reserve(struct(), start=None), "null")
    refused(reserve(struct(), slots=None), "slots")
    refused(reserve(struct(), n=-1), "slots")
    refused(release(struct(), gone=None), "null")
    refused(release(struct(sealed=None)), "null")


def test_python_checks():
    """Tensors of another dtype, shape, layout or device than the call takes."""
    with pytest.raises(ValueError, match="head_dim 96"):
        sa.PagedKV4(1, 2, 2, 4, head_dim=96, device="cpu")
    with pytest.raises(ValueError, match="pool must be"):
        sa.PagedKV4(1, 2, 2, 4, pool=torch.zeros((4, 2, 100), dtype=torch.uint8))
    kv = sa.PagedKV4(1, 4, 2, 4, device="cpu")
    assert kv.page_bytes * kv.num_pages == kv.pool.numel() and kv.struct().reserved == sa.POOL_KV4
    x = torch.zeros((3, 2, 128))
    slots = torch.zeros(3, dtype=torch.int32)
    for k, v, s in ((x.double(), x.double(), slots), (x, x.half(), slots), (x[:2], x[:2], slots), (x[:, :1], x, slots),
                    (x.transpose(1, 2), x, slots), (x.expand(3, 2, 128)[..., ::2], x, slots), (x, x, slots.long()),
                    (torch.zeros(1, 2, 128).expand(3, 2, 128), x, slots)):
        with pytest.raises(ValueError):
            sa.kv4_store(kv, k, v, s)
    q = torch.zeros((1, 4, 128))
    for args, keys in (((q[:, :3], 1.0), {}), ((torch.zeros((2, 4, 128)), 1.0), {}),
                       ((q, 1.0), {"selected": torch.zeros((1, 2, 4), dtype=torch.int64)})):
        with pytest.raises(ValueError):
            sa.kv4_decode_attention(kv, *args, **keys)
    with pytest.raises(ValueError, match="query_start"):
        sa.kv4_prompt_attention(kv, q, torch.zeros(1, dtype=torch.int32), 1.0)
    one = torch.zeros(1, dtype=torch.int32)
    free = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError, match="new_tokens"):
        sa.reserve_tokens(kv, one.long(), free, one, torch.zeros(2, dtype=torch.int32), slots)
    with pytest.raises(ValueError, match="free_pages"):
        sa.reserve_tokens(kv, one, one, one, torch.zeros(2, dtype=torch.int32), slots)
    with pytest.raises(ValueError, match="finished"):
        sa.release_sequences(kv, one[:0], free, one)
