"""Sessions on a paged key-value cache (T3Model.set_paged_kv) and under logit rules (T3Model.set_logit_rules, Session.logit_rules).

The paged path is held to the same bars as the slab path: fp32 logits within 1e-3 of the oracle's under teacher forcing and identical greedy
tokens; bf16 as far from the fp32 model as the slab path; continuous batching equal to the one-call batch."""
import numpy as np
import pytest

import chatterbox_amd as cb
from chatterbox_amd import _lib, synth
from oracle import t3_oracle as O
from tests.helpers import oracle_model, rel_err, turbo_oracle

pytestmark = pytest.mark.gpu

LOGIT_TOL = 1e-3


@pytest.fixture(scope="module")
def tiny():
    dims = synth.TINY
    m = cb.load_t3(synth.ensure_checkpoint(dims, 1234), device=0, start_speech_token=dims.start_speech_token, stop_speech_token=dims.stop_speech_token)
    yield dims, m
    m.close()


@pytest.fixture(scope="module")
def turbo():
    dims = synth.TURBO_TINY
    m = cb.load_t3_turbo(synth.ensure_turbo_checkpoint(dims, 4321), device=0, start_speech_token=dims.start_speech_token,
                         stop_speech_token=dims.stop_speech_token)
    yield dims, m
    m.close()


@pytest.fixture(autouse=True)
def plain_afterwards(tiny, turbo):
    yield
    for _, m in (tiny, turbo):
        m.set_paged_kv(0)
        m.set_logit_rules()


def _emb(dims, s0, seed, rows=2):
    return synth.synth_embeds(rows, s0, dims.hidden_size, seed)


# ---- paged cache ------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("page", [4, 16, 128])
def test_one_utterance_matches_the_oracle(tiny, page):
    """Prompt that ends inside a page, decode across several pages; logits of every step, greedy tokens."""
    dims, model = tiny
    emb, n = _emb(dims, 13, 99), 24
    ref = O.t3_inference(oracle_model(dims), emb, O.SampleParams(max_new_tokens=n, top_p=0.0), mask_stop=True)
    model.set_paged_kv(page)
    with cb.Session(model, [emb], max_new_tokens=n, top_p=0.0, mask_stop=True) as s:
        for i in range(n):
            assert rel_err(s.logits(), ref.raw_logits[i]) < LOGIT_TOL, f"step {i}"
            s.decode(1)
        assert list(s.tokens(0)) == list(ref.tokens)
        total, free = s.pages()
        assert total >= 2 * -(-(13 + n) // page) and free >= 0
    assert list(cb.t3_inference(model, emb, max_new_tokens=n, top_p=0.0)) == list(
        O.t3_inference(oracle_model(dims), emb, O.SampleParams(max_new_tokens=n, top_p=0.0)).tokens)


def test_turbo_matches_the_oracle(turbo):
    dims, model = turbo
    emb, n = _emb(dims, 13, 3, 1), 18
    ref = O.t3_inference_turbo(turbo_oracle(dims, 4321), emb, O.TurboParams(max_new_tokens=n, top_k=100, top_p=0.9, seed=7), mask_stop=True)
    model.set_paged_kv(16)
    with cb.Session(model, [emb], max_new_tokens=n, top_k=100, top_p=0.9, seed=7, mask_stop=True, forced=np.array(ref.tokens)) as s:
        for i in range(n + 1):
            assert rel_err(s.logits(), ref.raw_logits[i]) < LOGIT_TOL, f"step {i}"
            s.decode(1)
        assert list(s.tokens(0)) == ref.tokens


@pytest.mark.parametrize("U", [1, 3, 9])
def test_ragged_batch_equals_slabs(tiny, U):
    """Greedy tokens of a ragged batch, and its logits after 30 steps, from pages and from slabs."""
    dims, model = tiny
    embs = [_emb(dims, 5 + (u * 5) % 17, 100 + u) for u in range(U)]
    kw = dict(max_new_tokens=40, top_p=0.0, mask_stop=True)
    got = {}
    for page in (0, 16):
        model.set_paged_kv(page)
        with cb.Session(model, embs, **kw) as s:
            s.decode(30)
            got[page] = [list(s.tokens(u)) for u in range(U)], s.logits()
    assert got[0][0] == got[16][0]
    assert rel_err(got[16][1], got[0][1]) < LOGIT_TOL


def test_full_size_bf16_many_rows():
    """Full-size model, bf16 weights and cache, 20 utterances of different length: logits after the prefill and under forced tokens.  Both
    paths round at the same four places of each of 30 layers (two independent roundings of a row differ by as much as each is off, so
    their difference says little): the paged path's distance from the fp32 model -- over 40 x 8194 logits -- may be a tenth above the slab path's,
    and is far inside what 120 roundings of at most 2^-8 come to where none cancels, sqrt(120) 2^-8 of the logits' size."""
    dims = synth.FULL
    embs = [_emb(dims, 20 + (u * 7) % 50, 600 + u) for u in range(20)]
    forced = np.random.default_rng(0).integers(0, 6561, (20, 40)).astype(np.int32)
    lg = {}
    for dtype, page in (("f32", 0), ("bf16", 0), ("bf16", 64)):
        model = cb.load_t3(synth.ensure_checkpoint(dims, 1234), device=0, dtype=dtype)
        try:
            model.set_paged_kv(page)
            with cb.Session(model, embs, max_new_tokens=48, top_p=0.0, mask_stop=True, forced=forced) as s:
                first = s.logits()
                s.decode(40)
                lg[dtype, page] = first, s.logits()
        finally:
            model.close()
    for i in range(2):
        ref = lg["f32", 0][i].astype(np.float64)
        slab, paged = (float(np.sqrt(np.mean((lg["bf16", p][i] - ref) ** 2) / np.mean(ref ** 2))) for p in (0, 64))
        assert paged < 1.1 * slab and paged < np.sqrt(120) * 2.0 ** -8, (i, slab, paged)


@pytest.mark.parametrize("turbo_model", [False, True])
@pytest.mark.parametrize("dtype,U,page", [("f32", 3, 32), ("f32", 40, 4), ("f32", 72, 64), ("bf16", 2, 4), ("bf16", 10, 128), ("bf16", 70, 16), ("bf16", 290, 8)])
def test_every_product_writes_into_the_pages(dtype, U, page, turbo_model):
    """Row counts that take each kernel of the qkv product (fp32 below 64 rows: product and append apart), Llama and Turbo, ragged, teacher-forced, from
    pages and from slabs.  fp32: the slab path's bar.  bf16: the distance from the fp32 model, over U x vocabulary logits, at most a tenth above the
    slab path's (the two round at the same places; only the attention's sums differ) and below what the 8 roundings of two layers come to.  Up to 4 rows
    the slab session computes in fp32 on bf16 weights and rounds at none of those places, so there the second bar alone says something."""
    dims = synth.TURBO_TINY if turbo_model else synth.TINY
    rows = 1 if turbo_model else 2
    path = synth.ensure_turbo_checkpoint(dims, 4321) if turbo_model else synth.ensure_checkpoint(dims, 1234)
    load = cb.load_t3_turbo if turbo_model else cb.load_t3
    embs = [_emb(dims, 4 + (u * 5) % 13, 900 + u, rows) for u in range(U)]
    forced = np.random.default_rng(U).integers(0, 600, (U, 24)).astype(np.int32)
    kw = dict(max_new_tokens=24, mask_stop=True, forced=forced, **(dict(top_k=50, top_p=0.9) if turbo_model else dict(top_p=0.0)))
    got = {}
    for dt in {"f32", dtype}:
        m = load(path, device=0, dtype=dt, start_speech_token=dims.start_speech_token, stop_speech_token=dims.stop_speech_token)
        try:
            for p in (0, page):
                m.set_paged_kv(p)
                with cb.Session(m, embs, **kw) as s:
                    first = s.logits()
                    s.decode(20)
                    got[dt, p] = first, s.logits()
        finally:
            m.close()
    for i in range(2):
        ref = got["f32", 0][i].astype(np.float64)
        if dtype == "f32":
            assert rel_err(got["f32", page][i], ref) < LOGIT_TOL, i
        else:
            slab, paged = (float(np.sqrt(np.mean((got["bf16", p][i] - ref) ** 2) / np.mean(ref ** 2))) for p in (0, page))
            assert (paged < 1.1 * slab or U * rows <= 4) and paged < np.sqrt(8) * 2.0 ** -8, (i, slab, paged)


def test_pool_is_shared_and_refill_takes_freed_pages(tiny):
    """A pool for less than the worst case: refill refuses what does not fit and leaves the session as it was; an ended utterance's pages serve
    the next; tokens are those of slabs."""
    dims, model = tiny
    embs = [_emb(dims, 7, 400), _emb(dims, 9, 401)]
    kw = dict(max_new_tokens=20, top_p=0.0, mask_stop=True, max_cache_len=64)
    new = _emb(dims, 30, 402)
    with cb.Session(model, embs, **kw) as s:
        s.decode(5)
        s.refill([0], [new], max_new_tokens=[10])
        s.decode(9)
        ref = [list(s.tokens(u)) for u in range(2)]
    need = 2 * (-(-(7 + 20) // 8) + -(-(9 + 20) // 8))
    model.set_paged_kv(8, need + 1)
    with cb.Session(model, embs, **kw) as s:
        assert s.pages() == (need + 1, 1)
        s.decode(5)
        with pytest.raises(_lib.T3miError, match="pages"):
            s.refill([0], [new], max_new_tokens=[20])        # 14 pages; 8 of the slot's own and the spare one
        assert s.pages() == (need + 1, 1)
        s.refill([0], [new], max_new_tokens=[2])             # 8 pages
        assert s.pages()[1] == 1
        s.decode(2)                                          # its two tokens: ended
        s.refill([0], [_emb(dims, 5, 403)], max_new_tokens=[3])
        assert s.pages()[1] == 1 + 8 - 2 * -(-(5 + 3) // 8)
        s.decode(7)
        assert list(s.tokens(1)) == ref[1][:14]
    model.set_paged_kv(8, need - 1)
    with pytest.raises(_lib.T3miError, match="pool"):
        cb.Session(model, embs, **kw)
    model.set_paged_kv(8, 2 * (-(-(30 + 10) // 8) + -(-(9 + 20) // 8)))
    with cb.Session(model, [_emb(dims, 3, 1), embs[1]], **kw) as s:      # the refilled prompt alone decides its tokens
        s.decode(5)
        s.refill([0], [new], max_new_tokens=[10])
        s.decode(9)
        assert list(s.tokens(0)) == ref[0]


@pytest.mark.parametrize("pages", [0, 24, 40])
def test_continuous_batching_on_a_small_pool_equals_the_batch(tiny, pages):
    """Eleven ragged utterances through four slots; 24 pages of 8 hold barely two of the largest."""
    dims, model = tiny
    n = 11
    embs = [_emb(dims, 5 + (u * 3) % 7, 300 + u) for u in range(n)]
    lim = [5 + (u * 7) % 23 for u in range(n)]
    kw = dict(top_p=0.9, seed=4, mask_stop=True, first_utterance_id=1000)
    ref = cb.t3_inference_batch(model, embs, max_new_tokens=max(lim), **kw)
    model.set_paged_kv(8, pages)
    for longest in (False, True):
        st = {}
        got = cb.t3_inference_continuous(model, embs, slots=4, poll_steps=3, max_new_tokens=lim, stats=st, longest_first=longest, **kw)
        assert st["slots"] <= 4
        for u in range(n):
            assert list(got[u]) == list(ref[u][: lim[u]]), (u, got[u], ref[u][: lim[u]])
    model.set_paged_kv(8, 6)
    with pytest.raises(_lib.T3miError, match="pages"):
        cb.t3_inference_continuous(model, embs, slots=4, max_new_tokens=lim, **kw)


def test_turbo_continuous_on_pages(turbo):
    dims, model = turbo
    embs = [_emb(dims, 9 + u, 40 + u, 1) for u in range(6)]
    lim = [6, 11, 4, 9, 12, 7]
    ref = cb.t3_inference_turbo_batch(model, embs, max_new_tokens=12, top_k=1, mask_stop=True, keep_stop=True)
    model.set_paged_kv(4, 16)
    got = cb.t3_inference_continuous(model, embs, slots=3, poll_steps=3, max_new_tokens=lim, top_k=1, mask_stop=True, keep_stop=True)
    for u in range(6):
        assert list(got[u]) == list(ref[u][: lim[u] + 1])


def test_bad_page_settings_are_refused(tiny):
    _, model = tiny
    for args in ((3, 0), (12, 0), (2048, 0), (-4, 0), (16, -1), (0, 5), (2, 0)):
        with pytest.raises(_lib.T3miError):
            model.set_paged_kv(*args)


# ---- logit rules -------------------------------------------------------------------------------------------------------------------

def _filtered(raw, tokens, prm, bias, allowed, fre, pre, seen):
    """The row the sampler sees, in 64 bits: guidance, rules, the R sampler's penalty on `seen`, temperature."""
    z = raw[0] + prm["cfg_weight"] * (raw[0] - raw[1])
    for t, b in bias.items():
        z[t] += b
    for t in set(tokens):
        z[t] -= fre * tokens.count(t) + pre
    if allowed is not None:
        z[~allowed] = -np.inf
    for t in seen:
        z[t] /= prm["repetition_penalty"]
    return z / prm["temperature"]


@pytest.mark.parametrize("paged", [0, 16])
def test_rules_change_the_row_the_sampler_sees(tiny, paged):
    """Every step's row against the 64-bit formula: biases, penalties growing with the tokens, a token set, CFG before all of them."""
    dims, model = tiny
    model.set_paged_kv(paged)
    rng = np.random.default_rng(5)
    allowed = np.zeros(dims.speech_vocab, bool)
    allowed[rng.choice(dims.speech_vocab, 40, replace=False)] = True
    bias = {int(t): float(b) for t, b in zip(rng.choice(dims.speech_vocab, 30, replace=False), rng.normal(0, 3, 30))}
    prm = dict(cfg_weight=0.5, repetition_penalty=1.3, temperature=0.7)
    with cb.Session(model, [_emb(dims, 9, 11)], max_new_tokens=30, top_p=0.8, seed=3, mask_stop=True, **prm) as s:
        s.keep_filtered()
        s.logit_rules(0, bias=bias, allowed=allowed, frequency_penalty=0.4, presence_penalty=0.7)
        tokens = []
        for i in range(20):
            raw = s.logits().astype(np.float64)
            want = _filtered(raw, tokens, prm, bias, allowed, 0.4, 0.7, set(tokens) | {dims.start_speech_token - 1})
            want[dims.stop_speech_token] = -np.inf
            s.decode(1)
            got = s.filtered_logits(0).astype(np.float64)
            off = np.isneginf(want)
            assert (np.isneginf(got) == off).all()
            # up to 8 fp32 operations on values below the magnitude of what they combine
            mag = (3 * np.abs(raw).max() + max(abs(b) for b in bias.values()) + 0.4 * 20 + 0.7) / 0.7
            assert np.abs(got[~off] - want[~off]).max() < 8 * 2.0 ** -24 * mag
            tokens = list(s.tokens(0))
            assert allowed[tokens[-1]]


def test_rules_set_and_removed_between_steps(tiny):
    """No rules and neutral ones draw the same tokens; rules from step 6 to step 12 change those steps and their graph is recaptured twice
    (more biases than the buffers held)."""
    dims, model = tiny
    embs = [_emb(dims, 8, 21), _emb(dims, 6, 22)]
    kw = dict(max_new_tokens=30, top_p=0.0, mask_stop=True)
    with cb.Session(model, embs, **kw) as s:
        s.decode(6)
        head = [list(s.tokens(u)) for u in range(2)]
        s.decode(20)
        base = [list(s.tokens(u)) for u in range(2)]
    with cb.Session(model, embs, **kw) as s:
        s.logit_rules(0, bias={3: 0.0})
        s.decode(26)
        assert [list(s.tokens(u)) for u in range(2)] == base
    forced = 123
    with cb.Session(model, embs, **kw) as s:
        s.decode(6)
        s.logit_rules(1, allowed=[forced])
        s.decode(3)
        s.logit_rules(1, bias={t: (1e4 if t == 77 else 0.0) for t in range(200)})
        s.decode(3)
        s.logit_rules(1)
        s.decode(3)
        assert list(s.tokens(1)[:12]) == head[1] + [forced] * 3 + [77] * 3
        assert list(s.tokens(0)) == base[0][:15]             # the other slot never noticed
        s.refill([1], [embs[1]])
        s.decode(6)
        assert list(s.tokens(1)) == head[1]                  # a new utterance, no rules of the old one


def test_model_rules_hold_in_the_generate_calls(tiny, turbo):
    """Tokens stay inside the allowed set through batch, continuous batching and Turbo; a frequency penalty keeps a greedy stream from
    repeating itself."""
    dims, model = tiny
    embs = [_emb(dims, 6 + u, 50 + u) for u in range(5)]
    allowed = np.arange(dims.speech_vocab) < 300
    model.set_logit_rules(allowed=allowed)
    out = cb.t3_inference_batch(model, embs, max_new_tokens=25, seed=1)
    cont = cb.t3_inference_continuous(model, embs, slots=2, poll_steps=4, max_new_tokens=25, seed=1)
    assert all(len(o) == 25 and (o < 300).all() for o in out)     # the stop token is not among them: nobody ends early
    for a, b in zip(out, cont):
        assert (b < 300).all() and len(b) == 25
    model.set_logit_rules(frequency_penalty=1e4)
    for o in cb.t3_inference_batch(model, embs, max_new_tokens=60, top_p=0.0, mask_stop=True):
        assert len(set(o)) == 60
    model.set_logit_rules()
    tdims, tm = turbo
    tm.set_logit_rules(allowed=list(range(10)), presence_penalty=1e4)
    o = cb.t3_inference_turbo(tm, _emb(tdims, 9, 60, 1), max_new_tokens=9, seed=0)
    assert sorted(o) == list(range(10))                      # each of the ten once


def test_bad_rules_are_refused(tiny):
    dims, model = tiny
    V = dims.speech_vocab
    for kw in (dict(bias={V: 1.0}), dict(bias={-1: 1.0}), dict(bias={1: float("nan")}), dict(bias={1: float("inf")}), dict(frequency_penalty=float("nan")),
               dict(presence_penalty=float("inf")), dict(allowed=[]), dict(allowed=np.zeros(V, bool))):
        with pytest.raises(_lib.T3miError, match="logit rules"):
            model.set_logit_rules(**kw)
    for kw in (dict(allowed=[V]), dict(allowed=[-1]), dict(allowed=np.ones(V - 1, bool))):
        with pytest.raises(ValueError):
            model.set_logit_rules(**kw)
    with cb.Session(model, [_emb(dims, 5, 1)], max_new_tokens=4, top_p=0.0) as s:
        with pytest.raises(_lib.T3miError, match="slot"):
            s.logit_rules(1)
        s.decode(2)
    with pytest.raises(_lib.T3miError):
        _lib.check(_lib.load().t3mi_session_logit_rules(model._h, 0, None))   # no session
