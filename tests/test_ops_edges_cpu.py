"""The serving operators' plans and refusals, through the C entry points, without a GPU (addresses are made up, nothing is launched)."""
import ctypes as C

import pytest

from chatterbox_amd import _lib
from tests.test_ops_cpu import P, attention, cache


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
