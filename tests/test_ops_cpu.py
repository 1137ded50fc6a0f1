"""The serving operators' argument checks, through the C entry points, without a GPU: every refusal comes before any GPU work.
Addresses are made up; a call that passed its checks would fail for want of a device, which is told apart by its code."""
import ctypes as C

import pytest

from chatterbox_amd import _lib

P = 1 << 20        # an address, aligned


def cache(**kw):
    c = _lib.PagedCache(k=P, v=P, block_table=P, table_stride=4, n_seqs=3, max_pages=4, n_pages=9, page_size=16, kv_heads=2, head_dim=64,
                        dtype=_lib.W_F32, device=0)
    c.k_stride[:] = c.v_stride[:] = (16 * 2 * 64, 2 * 64, 64)
    return put(c, kw)


def put(c, kw):
    for n, v in kw.items():
        if isinstance(v, (tuple, list)):
            getattr(c, n)[:] = v
        else:
            setattr(c, n, v)
    return c


def append(**kw):
    a = _lib.AppendArgs(k=P, v=P, q=P, q_out=P, cos=P, sin=P, rope_stride=32, positions=P, rows=3, q_heads=4, rope_len=10, dtype=_lib.W_F32)
    a.k_stride[:] = a.v_stride[:] = (128, 64)
    a.q_stride[:] = a.q_out_stride[:] = (256, 64)
    return put(a, kw)


def attention(**kw):
    a = _lib.AttentionArgs(q=P, out=P, lengths=P, workspace=P, workspace_bytes=1 << 30, scale=0.125, rows=3, q_heads=4, q_dtype=_lib.W_F32, out_dtype=_lib.W_F32)
    a.q_stride[:] = a.out_stride[:] = (256, 64)
    return put(a, kw)


def logits(**kw):
    a = _lib.LogitsArgs(logits=P, out=P, logits_stride=100, out_stride=100, tokens=P, n_tokens=P, tokens_stride=8, repetition=1.0, rows=3, vocab=100,
                        dtype=_lib.W_F32, token_cap=8, device=0)
    return put(a, kw)


def refused(rc, word):
    msg = _lib.load().t3mi_last_error().decode()
    assert rc == _lib.ERR_ARG, (rc, msg)
    assert word in msg, (word, msg)


@pytest.mark.parametrize("kw,word", [(dict(k=None), "null"), (dict(block_table=None), "null"), (dict(dtype=2), "dtype"), (dict(head_dim=96), "head_dim"),
                                     (dict(page_size=0), "page_size"), (dict(page_size=24), "page_size"), (dict(page_size=1 << 17), "page_size"),
                                     (dict(n_pages=0), "positive"), (dict(kv_heads=0), "positive"), (dict(max_pages=-1), "positive"),
                                     (dict(k=P + 4), "16 bytes"), (dict(v_stride=(2048, 126, 64)), "16 bytes"), (dict(k_stride=(-2048, 128, 64)), "16 bytes"),
                                     (dict(max_pages=1 << 28), "keys"), (dict(table_stride=-1), "block table")])
def test_bad_caches_are_refused(kw, word):
    L = _lib.load()
    refused(L.t3mi_paged_append(cache(**kw), append(), None), word)
    refused(L.t3mi_paged_attention(cache(**kw), attention(), None), word)


@pytest.mark.parametrize("kw,word", [(dict(rows=-1), "rows"), (dict(dtype=7), "dtype"), (dict(q_out=None), "together"), (dict(q_heads=0), "q_heads"),
                                     (dict(sin=None), "together"), (dict(rope_len=0), "tables"), (dict(k=None), "null"), (dict(positions=None), "null"),
                                     (dict(v=P + 8), "16 bytes"), (dict(q_stride=(255, 64)), "16 bytes"), (dict(cos=P + 2), "4 bytes"),
                                     (dict(q_out_stride=(512, 64)), "same strides"), (dict(rows=4), "sequences"), (dict(rows=1 << 27, seq=P), "pairs")])
def test_bad_appends_are_refused(kw, word):
    refused(_lib.load().t3mi_paged_append(cache(), append(**kw), None), word)


def test_outputs_that_overlap_are_refused():
    """Written tensors whose strides put two elements in one place: a broadcast row or head, heads closer than head_dim, a shared page."""
    L = _lib.load()
    for stride in ((0, 64), (256, 0), (64, 64), (128, 64), (32, 256)):
        refused(L.t3mi_paged_attention(cache(), attention(rows=3, q_heads=4, out=2 * P, out_stride=stride), None), "out must not overlap")
        refused(L.t3mi_paged_append(cache(v=2 * P), append(rows=3, q_heads=4, q_out=2 * P, q_out_stride=stride), None), "q_out must not overlap")
    for kw in (dict(k_stride=(0, 128, 64)), dict(v_stride=(1024, 64, 64)), dict(k_stride=(2048, 128, 32)), dict(v=P)):
        refused(L.t3mi_paged_append(cache(**{"v": 2 * P, **kw}), append(), None), "cache must not overlap")


@pytest.mark.parametrize("kw,word", [(dict(rows=-2), "q_heads"), (dict(q_heads=3), "multiple"), (dict(q_heads=0), "multiple"), (dict(q_dtype=5), "dtypes"),
                                     (dict(q_dtype=_lib.W_BF16), "bf16 cache"), (dict(length_add=2), "length_add"), (dict(prompt=2), "prompt"), (dict(prompt=-2), "prompt"), (dict(max_length=-1), "max_length"),
                                     (dict(scale=float("inf")), "finite"), (dict(q=None), "null"), (dict(lengths=None), "null"), (dict(out=P + 4), "16 bytes"),
                                     (dict(out_stride=(256, 63)), "16 bytes"), (dict(rows=4), "sequences"), (dict(rows=1 << 23, seq=P), "pairs"), (dict(out_stride=(512, 64)), "same strides"),
                                     (dict(out_dtype=_lib.W_BF16), "same strides")])
def test_bad_attentions_are_refused(kw, word):
    L = _lib.load()
    refused(L.t3mi_paged_attention(cache(), attention(**kw), None), word)
    n = C.c_size_t(0)
    refused(L.t3mi_paged_attention_workspace(cache(), attention(**kw), n), word)


@pytest.mark.parametrize("kw,word", [(dict(rows=-1), "rows"), (dict(rows=65536), "rows"), (dict(vocab=0), "vocab"), (dict(vocab=(1 << 28) + 1), "vocab"), (dict(dtype=3), "dtype"), (dict(out=None), "null"),
                                     (dict(logits=P + 2), "aligned"), (dict(out_stride=99), "overlap"), (dict(logits_stride=128, out=P, out_stride=100), "same stride"),
                                     (dict(n_tokens=None), "n_tokens"), (dict(token_cap=1 << 20), "token_cap"), (dict(n_bias=5), "n_bias"),
                                     (dict(n_bias=4095, bias_ids=P, bias_values=P), "n_bias"), (dict(repetition=0.0), "repetition"),
                                     (dict(repetition=float("nan")), "repetition"), (dict(allowed=P + 1), "4 bytes"), (dict(tokens_stride=-1), "strides")])
def test_bad_logits_calls_are_refused(kw, word):
    refused(_lib.load().t3mi_process_logits(logits(**kw), None), word)


def test_null_structs_are_refused():
    L = _lib.load()
    refused(L.t3mi_set_paged_kv(None, 16, 0), "null")
    refused(L.t3mi_set_logit_rules(None, None), "null")
    refused(L.t3mi_session_logit_rules(None, 0, None), "null")
    refused(L.t3mi_session_pages(None, None, None), "null")
    refused(L.t3mi_paged_append(None, append(), None), "null")
    refused(L.t3mi_paged_append(cache(), None, None), "null")
    refused(L.t3mi_paged_attention(cache(), None, None), "null")
    refused(L.t3mi_paged_attention_workspace(cache(), attention(), None), "null")
    refused(L.t3mi_process_logits(None, None), "null")


def test_no_rows_is_nothing_to_do():
    L = _lib.load()
    assert L.t3mi_paged_append(cache(), append(rows=0), None) == _lib.OK
    assert L.t3mi_paged_attention(cache(), attention(rows=0), None) == _lib.OK
    assert L.t3mi_process_logits(logits(rows=0), None) == _lib.OK


def test_tensors_off_the_gpu_are_refused():
    torch = pytest.importorskip("torch")
    import chatterbox_amd as cb
    k = torch.zeros(2, 16, 2, 64)
    table, lens = torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="run on the GPU"):
        cb.paged_attention(torch.zeros(1, 4, 64), k, k, table, lens)
    with pytest.raises(ValueError, match="run on the GPU"):
        cb.paged_kv_append(torch.zeros(1, 2, 64), torch.zeros(1, 2, 64), k, k, table, lens)
    with pytest.raises(ValueError, match="run on the GPU"):
        cb.process_logits(torch.zeros(1, 5))
