"""Sessions on a paged cache and under logit rules: settings that meet each other."""
import ctypes as C

import numpy as np
import pytest

import chatterbox_amd as cb
from chatterbox_amd import _lib, synth, t3

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tiny():
    dims = synth.TINY
    m = cb.load_t3(synth.ensure_checkpoint(dims, 1234), device=0, start_speech_token=dims.start_speech_token, stop_speech_token=dims.stop_speech_token)
    yield dims, m
    m.close()


@pytest.fixture(autouse=True)
def plain_afterwards(tiny):
    yield
    tiny[1].set_paged_kv(0)
    tiny[1].set_logit_rules()


def _emb(dims, s0, seed):
    return synth.synth_embeds(2, s0, dims.hidden_size, seed)


def continuous(model, embs, limits, slots, cache_len):
    """t3mi_generate_continuous with a cache length of the caller's; tokens, and the slots it opened."""
    n, cap = len(embs), max(limits)
    es = [np.ascontiguousarray(e, dtype=np.float32) for e in embs]
    p = t3._params(model, cap, 0.8, 0.5, 0.9, 0.05, 1.2, _lib.SAMPLER_R, cache_len, 4, True)
    out, n_out, st = np.zeros((n, cap), np.int32), (C.c_int32 * n)(), (C.c_int32 * 4)()
    _lib.check(model._lib.t3mi_generate_continuous(model._h, n, 2, (C.c_void_p * n)(*[e.ctypes.data for e in es]), (C.c_int32 * n)(*[e.shape[1] for e in es]),
                                                   (C.c_int32 * n)(*limits), slots, 5, 0, C.byref(p), out.ctypes.data_as(C.POINTER(C.c_int32)), cap, n_out, st))
    return [list(out[u, : n_out[u]]) for u in range(n)], st[3]


@pytest.mark.parametrize("page,pages,cache", [(8, 40, 40), (16, 12, 45), (4, 18, 34), (8, 0, 40)])
def test_a_small_pool_under_max_cache_len(tiny, page, pages, cache):
    """max_cache_len ends utterances long before their token limits: the pool has to hold what the cache rows have room for, not the limits."""
    dims, model = tiny
    embs = [_emb(dims, 6 + (u * 5) % 9, 700 + u) for u in range(7)]
    lim = [200 + u for u in range(7)]
    ref, _ = continuous(model, embs, lim, 3, cache)
    model.set_paged_kv(page, pages)
    got, slots = continuous(model, embs, lim, 3, cache)
    for u in range(7):
        assert got[u] == ref[u] and len(got[u]) == cache - embs[u].shape[1] - 1
    assert slots == (min(3, pages // (2 * -(-cache // page))) if pages else 3)   # an utterance has two rows of `cache` positions
