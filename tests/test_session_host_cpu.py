"""What sessions do on the host -- pages, rules, allocations, refusals -- on a stand-in for the HIP runtime, without a GPU."""
from tests.host_runtime import run

# a step's launches go out one by one, and the arguments of the last logits-rules launch can be read: "device" memory is the process's own
RULES = """
import os
os.environ["T3MI_GRAPH"] = "0"

class LogitsArgs(C.Structure):   # t3k::LogitsArgs
    _fields_ = [(n, C.c_void_p) for n in ("logits", "uncond", "out")] + [(n, C.c_int64) for n in ("lr", "ur", "outr")] + \\
               [(n, C.c_int) for n in ("bf16", "rows", "vocab")] + [("cfg", C.c_float), ("tokens", C.c_void_p), ("n_tokens", C.c_void_p), ("tr", C.c_int64), ("cap", C.c_int)] + \\
               [(n, C.c_void_p) for n in ("repetition", "frequency", "presence")] + [(n, C.c_float) for n in ("rep", "fre", "pre")] + \\
               [("ids", C.c_void_p), ("values", C.c_void_p), ("br", C.c_int64), ("bvr", C.c_int64), ("n_bias", C.c_int), ("allowed", C.c_void_p), ("ar", C.c_int64)]

def step(s):
    # the biases, penalties and numbers of allowed tokens of every slot in the next step; None: no rules
    rt.hostrt_forget()
    s.decode(1)
    if not rt.hostrt_launches(b"process_logits"):
        return None
    a = LogitsArgs()
    assert rt.hostrt_last(b"process_logits", C.byref(a), C.c_size_t(C.sizeof(a)))
    got = []
    for u in range(a.rows):
        ids = np.ctypeslib.as_array((C.c_int32 * a.n_bias).from_address(a.ids + u * a.br * 4))
        vals = np.ctypeslib.as_array((C.c_float * a.n_bias).from_address(a.values + u * a.bvr * 4))
        words = np.ctypeslib.as_array((C.c_uint32 * ((a.vocab + 31) // 32)).from_address(a.allowed + u * a.ar * 4))
        got.append(({int(i): float(v) for i, v in zip(ids, vals) if i >= 0}, C.c_float.from_address(a.frequency + 4 * u).value,
                    int(np.unpackbits(words.view(np.uint8), bitorder="little")[:a.vocab].sum())))
    return got
"""


def test_rules_that_find_no_memory_leave_the_old_ones():
    """Each allocation of a growing rule set fails in turn: the error comes back, every slot keeps its rules, and nothing is lost or kept."""
    run(RULES + """
m = model()
with cb.Session(m, [prompt(9), prompt(5)], max_new_tokens=20, top_p=0.0) as s:
    assert step(s) is None
    wide = {t: 0.5 for t in range(100)}
    for first in (True, False):
        held, failed = rt.hostrt_held(), 0
        before = step(s)
        for k in range(20):
            rt.hostrt_fail_malloc(k)
            try:
                s.logit_rules(1, bias={7: 2.0} if first else wide, frequency_penalty=0.25)
                break
            except _lib.T3miError as e:
                assert "memory" in str(e)
                failed += 1
            rt.hostrt_fail_malloc(-1)
            assert rt.hostrt_held() == held and step(s) == before, (first, k, step(s), before)
        rt.hostrt_fail_malloc(-1)
        assert failed >= 5
        s.logit_rules(0, bias={3: 1.0}, allowed=[1, 2, 3])
    assert step(s) == [({3: 1.0}, 0.0, 3), (wide, 0.25, m.vocab)]
m.close()
""")


def test_a_refill_that_finds_no_memory_for_rules_changes_nothing():
    run(RULES + """
m = model()
m.set_paged_kv(8, 14)
with cb.Session(m, [prompt(9), prompt(5)], max_new_tokens=16, top_p=0.0) as s:
    m.set_logit_rules(bias={t: 0.5 for t in range(70)})
    pages, held = s.pages(), rt.hostrt_held()
    assert pages == (14, 14 - 2 * 4 - 2 * 3)
    for k in range(6):
        rt.hostrt_fail_malloc(k)
        try:
            s.refill([0], [prompt(3)], max_new_tokens=[4])
            raise SystemExit("no error")
        except _lib.T3miError as e:
            assert "memory" in str(e)
        rt.hostrt_fail_malloc(-1)
        assert s.pages() == pages and rt.hostrt_held() == held and step(s) is None, (k, s.pages(), pages)
    s.refill([0], [prompt(3)], max_new_tokens=[4])
    assert s.pages() == (14, 6) and [len(r[0]) for r in step(s)] == [70, 0]
m.close()
""")


def test_no_exception_leaves_the_session_calls():
    """Every allocation of a begin, a refill and a continuous job fails in turn with std::bad_alloc: an error comes back, and what follows is a session like any
    other (its own pages, no limits of the job that failed)."""
    run("""
m = model()
m.set_paged_kv(8, 60)
kw = dict(max_new_tokens=40, top_p=0.0)
embs = [prompt(9), prompt(5), prompt(7)]

def fails(call, limit=4000):
    n = 0
    for k in range(limit):
        rt.hostrt_fail_new(C.c_long(k))
        try:
            call()
        except _lib.T3miError as e:
            rt.hostrt_fail_new(C.c_long(-1))
            if "memory" not in str(e):
                return n                        # (the job's own end)
            n += 1
            continue
        rt.hostrt_fail_new(C.c_long(-1))
        return n
    raise SystemExit("no end")

def begin():
    cb.Session(m, embs, **kw).__enter__().__exit__(None, None, None)

def plain():
    with cb.Session(m, embs, **kw) as s:
        assert s.pages() == (42, 42 - 2 * (7 + 6 + 6)), s.pages()   # (never more than the worst case)

assert fails(begin) > 10
plain()
s = cb.Session(m, embs, **kw)
assert fails(lambda: s.refill([1], [prompt(6)], max_new_tokens=[5])) > 5
total, free = s.pages()
assert (total, free) == (42, 42 - 2 * (7 + 2 + 6))
s.close() if hasattr(s, "close") else s.__exit__(None, None, None)

def job():
    rt.hostrt_fail_copy(C.c_long(200))           # (no token is ever drawn here: the job ends with this error)
    try:
        cb.t3_inference_continuous(m, embs + [prompt(4)], slots=3, poll_steps=3, max_new_tokens=[2, 3, 4, 5], top_p=0.0)
    finally:
        rt.hostrt_fail_copy(C.c_long(-1))
        rt.hostrt_fail_new(C.c_long(-1))
        plain()

assert fails(job) > 10
plain()
m.close()
""")


def test_projections_take_memory_only_where_they_are_read():
    """The qkv product writes into the pages itself in bf16 and from 64 fp32 rows on: no buffer for its projections then (402 MB for the largest prefill of
    the full-size model), and one for the few rows that need it."""
    run("""
d = synth.TINY.hidden_size
for dtype, lens, decode_rows, prefill_rows in (("bf16", [40] * 5, 0, 0), ("bf16", [5], 0, 0), ("f32", [9, 20], 4, 58), ("f32", [200] * 2, 4, 0), ("f32", [200] * 40, 0, 0)):
    m = model(dtype=dtype)
    m.set_paged_kv(16)
    rt.hostrt_forget()
    with cb.Session(m, [prompt(n) for n in lens], max_new_tokens=11, top_p=0.0) as s:
        s.decode(1)
        got = sizes()
        for rows, needed in ((2 * len(lens), decode_rows), (2 * sum(lens), prefill_rows)):
            assert got.count(rows * 3 * d * 4) == (1 if needed else 0), (dtype, lens, rows, got)
    m.close()
""")


def test_rules_that_leave_no_token_under_mask_stop_are_refused():
    """The stop token alone allowed, and mask_stop: nothing could be drawn, and the sampler would have emitted the stop token all the same.  Refused where both are
    known: at begin, at a slot's rules, at a refill; the session goes on as it was."""
    run(RULES + """
m = model()
stop = m.stop_speech_token
kw = dict(max_new_tokens=20, top_p=0.0)

def refused(call):
    try:
        call()
    except _lib.T3miError as e:
        assert e.code == _lib.ERR_ARG and "mask_stop" in str(e), e
        return
    raise SystemExit("taken")

with cb.Session(m, [prompt(9), prompt(5)], mask_stop=True, **kw) as s:
    s.logit_rules(0, allowed=[5, stop])
    before = step(s)
    refused(lambda: s.logit_rules(1, allowed=[stop]))
    assert step(s) == before
    m.set_logit_rules(allowed=[stop])
    refused(lambda: s.refill([1], [prompt(4)]))
    assert step(s) == before
    refused(lambda: cb.Session(m, [prompt(9)], mask_stop=True, **kw).__enter__())
    assert step(s) == before                     # (refused before the running session is given up)
    refused(lambda: cb.t3_inference_batch(m, [prompt(9)], mask_stop=True, **kw))
refused(lambda: cb.t3_inference_continuous(m, [prompt(9)], mask_stop=True, **kw))
with cb.Session(m, [prompt(9)], **kw) as s:      # without mask_stop the stop token may be all there is
    assert step(s)[0][2] == 1
m.set_logit_rules(allowed=[5])
with cb.Session(m, [prompt(9)], mask_stop=True, **kw) as s:
    assert step(s)[0][2] == 1
# bits of the last word past the vocabulary are no tokens
words = (C.c_uint32 * ((m.vocab + 31) // 32))()
words[stop // 32] = 1 << (stop % 32)
words[len(words) - 1] |= 0xFFFFFFFF << (m.vocab % 32) & 0xFFFFFFFF
r = _lib.LogitRules(allowed=words)
_lib.check(L.t3mi_set_logit_rules(m._h, C.byref(r)))
refused(lambda: cb.Session(m, [prompt(9)], mask_stop=True, **kw).__enter__())
m.close()
""")


def test_token_ids_of_rules_are_taken_as_they_are():
    """An id past 32 bits used to wrap round to another token, a fractional one to be cut."""
    run("""
m = model()
for bad in ({2 ** 32 + 3: 1.0}, {-2 ** 32 + 5: 1.0}, {m.vocab: 1.0}, {3.7: 1.0}, {"3": 1.0}):
    try:
        m.set_logit_rules(bias=bad)
        raise SystemExit(f"taken: {bad}")
    except (ValueError, TypeError, _lib.T3miError):
        pass
for bad in ([1.7], np.array([1.0, 2.0]), ["3"], [m.vocab], [-1], [2 ** 70], [True, False]):
    try:
        m.set_logit_rules(allowed=bad)
        raise SystemExit(f"taken: {bad}")
    except (ValueError, OverflowError):
        pass
for good in ([3, 5], (3, 5), {3, 5}, np.array([3, 5], np.uint8), range(3, 6), np.arange(m.vocab) < 4):
    m.set_logit_rules(allowed=good, bias={np.int64(7): np.float32(1.0)})
m.close()
""")
