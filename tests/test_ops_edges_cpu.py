"""The serving operators' plans and refusals, through the C entry points, without a GPU (addresses are made up, nothing is launched)."""
import ctypes as C

import pytest

from chatterbox_amd import _lib
from tests.host_runtime import run
from tests.test_ops_cpu import P, append, attention, cache, refused


def split(c, **kw):
    """Whether a call's keys are shared among blocks: it asks for a workspace then."""
    n = C.c_size_t(0)
    assert _lib.load().t3mi_paged_attention_workspace(c, attention(**kw), C.byref(n)) == _lib.OK
    return n.value > 0


def long_cache(n_seqs, kv_heads, dim, dtype):
    c = cache(n_seqs=n_seqs, max_pages=2048, n_pages=10000, page_size=64, kv_heads=kv_heads, head_dim=dim, dtype=dtype)
    c.k_stride[:] = c.v_stride[:] = (64 * kv_heads * dim, kv_heads * dim, dim)
    return c


@pytest.mark.parametrize("heads,kv_heads,dim,dtype", [(32, 8, 128, _lib.W_BF16), (16, 16, 64, _lib.W_BF16), (16, 16, 64, _lib.W_F32), (8, 1, 128, _lib.W_BF16)])
@pytest.mark.parametrize("prompt", [0, 1])
def test_a_few_rows_of_a_long_sequence_are_split(heads, kv_heads, dim, dtype, prompt):
    """Draft tokens, a short chunk: rows that share their keys would be a handful of blocks that each walk 131072 keys.  Enough of them are left together."""
    c = long_cache(1, kv_heads, dim, dtype)
    kw = dict(q_heads=heads, seq=P, q_stride=(heads * dim, dim), out_stride=(heads * dim, dim), prompt=prompt)
    for rows in (1, 4, 8):
        assert split(c, rows=rows, **kw)
    assert not split(c, rows=512, **kw)


def test_rows_in_unknown_order_share_keys_where_that_gains_more_than_it_may_lose():
    """Rows as [step][sequence] look like rows as [sequence][step] to the host."""
    c = long_cache(16, 4, 64, _lib.W_BF16)
    kw = dict(q_heads=4, seq=P, q_stride=(256, 64), out_stride=(256, 64))
    assert split(c, rows=64, prompt=0, **kw) and not split(c, rows=64, prompt=1, **kw) and split(c, rows=64, prompt=-1, **kw)
    assert not split(c, rows=512, prompt=0, **kw)


# (everything on a stand-in for the HIP runtime: calls that pass the checks launch nothing there)
CALLS = """
P = 1 << 24
def attend(q, out, qs, os, rows=3, heads=4, qd=0, od=0, dim=64):
    c = _lib.PagedCache(k=P << 8, v=P << 9, block_table=P << 10, table_stride=4, n_seqs=rows, max_pages=4, n_pages=9, page_size=16, kv_heads=2, head_dim=dim, dtype=qd, device=0)
    c.k_stride[:] = c.v_stride[:] = (16 * 2 * dim, 2 * dim, dim)
    a = _lib.AttentionArgs(q=q, out=out, lengths=P << 10, workspace=P << 11, workspace_bytes=1 << 40, scale=0.125, rows=rows, q_heads=heads, q_dtype=qd, out_dtype=od)
    a.q_stride[:], a.out_stride[:] = qs, os
    return L.t3mi_paged_attention(C.byref(c), C.byref(a), None)

def append(k, v, q, out, ks, vs, qs, os, rows=3, heads=4):
    c = _lib.PagedCache(k=P << 8, v=P << 9, block_table=P << 10, table_stride=4, n_seqs=rows, max_pages=4, n_pages=9, page_size=16, kv_heads=2, head_dim=64, dtype=0, device=0)
    c.k_stride[:] = c.v_stride[:] = (16 * 2 * 64, 2 * 64, 64)
    a = _lib.AppendArgs(k=k, v=v, q=q, q_out=out, positions=P << 10, rows=rows, q_heads=heads, dtype=0)
    a.k_stride[:], a.v_stride[:], a.q_stride[:], a.q_out_stride[:] = ks, vs, qs, os
    return L.t3mi_paged_append(C.byref(c), C.byref(a), None)

def rules(logits, out, ls, os, uncond=None, us=0, rows=3, vocab=100, dtype=0):
    a = _lib.LogitsArgs(logits=logits, out=out, uncond=uncond, logits_stride=ls, uncond_stride=us, out_stride=os, repetition=1.0, rows=rows, vocab=vocab, dtype=dtype, device=0)
    return L.t3mi_process_logits(C.byref(a), None)

def refused(rc):
    assert rc == _lib.ERR_ARG and b"share memory" in L.t3mi_last_error(), (rc, L.t3mi_last_error())

def taken(rc):
    assert rc == _lib.OK, (rc, L.t3mi_last_error())
"""


def test_outputs_that_share_memory_with_inputs_are_refused():
    """At another address, that is: a row later, half a head further, in other steps, in the other type.  Woven views of one buffer are taken."""
    run(CALLS + """
row, F = 4 * 64, 4                                      # elements of a row of q, bytes of one
s = (row, 64)
taken(attend(P, P, s, s))
taken(attend(P, P + 3 * row * F, s, s))
for off in (16, 64 * F, row * F, 2 * row * F, 3 * row * F - 16):
    refused(attend(P, P + off, s, s))
    refused(attend(P + off, P, s, s))
wide = (3 * row, 64)
taken(attend(P, P + row * F, wide, wide))               # q and out beside each other in one buffer, either way round, and rows later
taken(attend(P + 2 * row * F, P, wide, wide))
taken(attend(P, P + 7 * row * F, wide, wide))
refused(attend(P, P + row * F // 2, wide, wide))
refused(attend(P, P + 3 * row * F, wide, wide))
refused(attend(P, P + row * F, wide, (3 * row, 128)))   # (other steps in the same place)
taken(attend(P, P + 64 * F, (2 * row, 128), (2 * row, 128)))    # heads in turn
taken(attend(P, P + 5 * 64 * F, (4 * row, 128), (4 * row, 128)))
refused(attend(P, P + 4 * 64 * F, (4 * row, 128), (4 * row, 128)))
taken(attend(P, P + 64 * F, (64 * 2, 64 * 8), (64 * 2, 64 * 8)))  # heads outside, rows inside
refused(attend(P, P + 64 * 2 * F, (64 * 2, 64 * 8), (64 * 2, 64 * 8)))
taken(attend(P, P + row * F, (0, 64), (0, 64), rows=1))
refused(attend(P, P + 64 * F, (0, 64), (0, 64), rows=1))
refused(attend(P, P + 2 * row, s, s, qd=1, od=0))       # a bf16 row later, in fp32
taken(attend(P, P + 3 * row * 2, s, s, qd=1, od=0))

kv = (2 * 64, 64)
k, v, q, o = P, P << 1, P << 2, P << 3
taken(append(k, v, q, o, kv, kv, s, s))
taken(append(k, v, q, q, kv, kv, s, s))
packed = (8 * 64, 64)                                   # q, k and v of a row beside each other, q_out in q's place
taken(append(P + row * F, P + (row + 128) * F, P, P, packed, packed, packed, packed))
refused(append(P + row * F, P + (row + 128) * F, P, P + 64 * F, packed, packed, packed, packed))
refused(append(k, v, q, k, kv, kv, s, s))
refused(append(k, v, q, v + 128 * F, kv, kv, s, s))
refused(append(k, v, q, q + row * F, kv, kv, s, s))

taken(rules(P, P, 100, 100))
taken(rules(P, P + 300 * F, 100, 100))
taken(rules(P, P + 100 * F, 200, 200))
for off in (F, 100 * F, 299 * F):
    refused(rules(P, P + off, 100, 100))
refused(rules(P, P + 100 * F, 200, 100))
refused(rules(P << 1, P, 100, 100, P + F, 100))
refused(rules(P << 1, P, 100, 100, P, 100))
taken(rules(P << 1, P, 100, 100, P << 2, 100))
taken(rules(P, P + 100 * F, 0, 100, P, 0))              # (a broadcast row before it)
refused(rules(P + 100 * F, P, 0, 100))
""")


def test_keys_and_values_of_a_cache_that_share_memory_are_refused_by_the_append():
    """Equal addresses alone were compared.  Keys and values of a page side by side, heads of both in turn, or one pool cut in two are taken."""
    run(CALLS + """
def put(k, v, strides, n_pages=9, page=16, heads=2, vs=None):
    c = _lib.PagedCache(k=k, v=v, block_table=P << 10, table_stride=4, n_seqs=3, max_pages=4, n_pages=n_pages, page_size=page, kv_heads=heads, head_dim=64, dtype=0, device=0)
    c.k_stride[:], c.v_stride[:] = strides, vs or strides
    a = _lib.AppendArgs(k=P << 5, v=P << 6, positions=P << 10, rows=3, dtype=0)
    a.k_stride[:] = a.v_stride[:] = (128, 64)
    return L.t3mi_paged_append(C.byref(c), C.byref(a), None)

def no(rc):
    assert rc == _lib.ERR_ARG and b"must not overlap" in L.t3mi_last_error(), (rc, L.t3mi_last_error())

page, F = 16 * 2 * 64, 4
plain, side = (page, 128, 64), (2 * page, 128, 64)
taken(put(P, P + 9 * page * F, plain))
taken(put(P + 9 * page * F, P, plain))
taken(put(P, P + page * F, side))                        # [pages, 2, slots, heads, 64]
taken(put(P + page * F, P, side))
taken(put(P, P + 2 * 64 * F, (2 * page, 256, 64)))       # [pages, slots, 2, heads, 64]
taken(put(P, P + 64 * F, (2 * page, 256, 128)))          # [pages, slots, heads, 2, 64]
taken(put(P, P + 16 * 64 * F, (2 * page, 64, 2 * 16 * 64)))   # [pages, heads, 2, slots, 64]
for off in (0, 16, 64 * F, 128 * F, page * F, 8 * page * F, 9 * page * F - 16):
    no(put(P, P + off, plain))
for off in (0, 64 * F, page * F // 2, page * F + 128 * F, 2 * page * F):
    no(put(P, P + off, side))
no(put(P, P + page * F, side, vs=(2 * page, 64, 16 * 64)))    # (another order in the same place)
""")


@pytest.mark.parametrize("which", ["lengths", "starts", "seq", "positions"])
def test_misaligned_lists_are_refused(which):
    """(a scalar load would drop the low bits of the address and read a neighbour)"""
    L, kw = _lib.load(), {which: P + 2}
    if which != "positions":
        n = C.c_size_t(0)
        refused(L.t3mi_paged_attention_workspace(cache(), attention(**kw), n), "4 bytes")
    if which in ("positions", "seq"):
        refused(L.t3mi_paged_append(cache(v=2 * P), append(q_out=P, **kw), None), "4 bytes")
