"""Paged attention where precision and special values can go wrong, against plain 64-bit numpy on the same inputs.

Tolerances as in test_gpu_ops: u = 2^-24; |out - ref| <= 2 (2 e + 2^-21 + n u) sum p |v| / sum p with e the error of a score, then half a step of the
result's type, 2^-8 of a bf16 value."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
import chatterbox_amd as cb  # noqa: E402
from tests.test_gpu_ops import DT, U, make_cache, np64, ref_attention  # noqa: E402

pytestmark = pytest.mark.gpu


def t32(x):
    return torch.tensor(x, dtype=torch.int32).cuda()


@pytest.mark.parametrize("q_t", ["f32", "bf16"])
@pytest.mark.parametrize("prompt,heads,kv_heads,dim,page", [(False, 16, 16, 64, 64), (False, 32, 8, 128, 16), (False, 6, 2, 64, 2), (True, 8, 2, 128, 64), (True, 4, 4, 64, 8),
                                                               (True, 24, 8, 128, 64), (True, 12, 12, 64, 8)])
def test_weights_under_a_bf16_result_are_not_rounded_to_it(q_t, prompt, heads, kv_heads, dim, page):
    """A bf16 result is off by its own rounding, 2^-8 of itself, and by next to nothing else: a weight held in two bf16 parts, each rounded to the nearest,
    is off by at most 2^-8 2^-8 of itself, a 256th of what one part would be.  Sums of many keys are small against sum p |v|, which one part's error goes with."""
    lens = [700, 33, 512, 1500]
    k, v, table, keys, vals = make_cache(lens, page, kv_heads, dim, "bf16", 7)
    seq = [s for s in range(4) for _ in range(9)] if prompt else list(range(4))
    rows = [(s, lens[s] - i % 9) for i, s in enumerate(seq)] if prompt else list(zip(seq, lens))
    q = torch.randn(len(rows), heads, dim, generator=torch.Generator().manual_seed(3)).to(DT[q_t]).cuda()
    got = np64(cb.paged_attention(q, k, v, table, t32([n for _, n in rows]), seq=t32(seq), out_dtype=torch.bfloat16, prompt=prompt))
    for r, (s, n) in enumerate(rows):
        ref, mag, err = ref_attention(np64(q[r]), keys[s][:n], vals[s][:n], 0, dim ** -0.5)
        tol = (2 * (2 * err * U + 2.0 ** -21 + n * U) + 2.0 ** -16) * mag
        tol += 2.0 ** -8 * (np.abs(ref) + tol)
        assert (np.abs(got[r] - ref) <= tol).all(), (r, n, float((np.abs(got[r] - ref) / tol).max()))


def ref_row(q, k, v, scale):
    """One row and key head: q [G, D], k, v [n, D] in 64 bits -> out [G, D], sum p |v| over the finite values, largest finite score error / U."""
    with np.errstate(all="ignore"):
        s = (q[:, None] * k[None]).sum(-1) * scale
        err = np.where(np.isfinite(s), (q.shape[1] + 2) * (np.abs(q)[:, None] * np.where(np.isfinite(k), np.abs(k), 0)[None]).sum(-1) * abs(scale), 0).max()
        p = np.exp(s - s.max(1, keepdims=True))
        p = p / p.sum(1, keepdims=True)
        return (p[:, :, None] * v[None]).sum(1), (p[:, :, None] * np.where(np.isfinite(v), np.abs(v), 0)[None]).sum(1), err


@pytest.mark.parametrize("q_t,kv_t,out_t", [("f32", "bf16", "f32"), ("f32", "bf16", "bf16"), ("bf16", "bf16", "f32"), ("bf16", "bf16", "bf16"), ("f32", "f32", "f32")])
@pytest.mark.parametrize("prompt,heads,kv_heads,dim,page,most", [(False, 4, 2, 64, 64, 0), (False, 6, 2, 128, 8, 0), (False, 4, 2, 64, 1, 0), (False, 8, 2, 128, 64, 20000),
                                                                 (False, 40, 2, 64, 32, 0), (True, 4, 2, 64, 64, 0), (True, 6, 2, 128, 8, 0), (True, 2, 2, 64, 16, 0),
                                                                 (True, 16, 8, 64, 64, 0), (True, 24, 8, 128, 8, 0), (True, 6, 6, 64, 16, 0), (True, 32, 8, 128, 32, 0)])
def test_infinities(q_t, kv_t, out_t, prompt, heads, kv_heads, dim, page, most):
    """Queries that bf16 holds exactly against keys and values with infinities in them.  A key of -inf score has no weight, one of +inf makes its rows NaN, an
    infinite value comes out in its element wherever its key is seen (also alone, with weight 1); everything else is as the formula has it, to the
    tolerance; key heads without infinities keep their bits."""
    lens = [400, 130, 1, 33, 2000]
    k, v, table, keys, vals = make_cache(lens, page, kv_heads, dim, kv_t, 17)
    inf = float("inf")

    def put(which, held, s, j, e, x):
        which[int(table[s, j // page]), j % page, 0, e] = x
        held[s][j, 0, e] = x

    g = np.random.default_rng(2)
    sign = np.sign(g.standard_normal(dim))
    for s, j in ((0, 7), (0, 333), (1, 129), (4, 1999), (4, 31)):
        put(k, keys, s, j, 5, -inf * sign[5])               # (every query has this sign there: score -inf)
    put(k, keys, 3, 20, 9, inf * sign[9])                   # score +inf
    for s, j, e, x in ((0, 100, 3, inf), (0, 200, 4, -inf), (1, 50, 3, -inf), (2, 0, 6, inf), (4, 1500, 1, inf), (4, 1501, 1, -inf)):
        put(v, vals, s, j, e, x)
    seen = [(s, n) for s in range(5) for n in (range(max(1, lens[s] - 12), lens[s] + 1) if prompt else [lens[s]])]
    q = torch.from_numpy(np.abs(g.standard_normal((len(seen), heads, dim))) * sign + 0.25 * sign).float().bfloat16().to(DT[q_t]).cuda()   # (no zero among them)
    args = dict(seq=t32([s for s, _ in seen]), out_dtype=DT[out_t], prompt=prompt, max_length=most)
    n = t32([n for _, n in seen])
    got = cb.paged_attention(q, k, v, table, n, **args)
    group = heads // kv_heads
    for r, (s, m) in enumerate(seen):
        for h in range(kv_heads):
            at = slice(h * group, (h + 1) * group)
            ref, mag, err = ref_row(np64(q[r, at]), keys[s][:m, h], vals[s][:m, h], dim ** -0.5)
            x = np64(got[r, at])
            fine = np.isfinite(ref)
            assert np.array_equal(np.isnan(x), np.isnan(ref)) and np.array_equal(x[np.isinf(ref)], ref[np.isinf(ref)]), (r, s, m, h)
            tol = 2 * (2 * err * U + 2.0 ** -21 + m * U) * mag
            if out_t == "bf16":
                tol = (tol + 2.0 ** -16 * mag) * (1 + 2.0 ** -8) + 2.0 ** -8 * np.abs(np.where(fine, ref, 0))
            assert (np.abs(x - ref)[fine] <= tol[fine]).all(), (r, s, m, h)
    clean = cb.paged_attention(q, torch.nan_to_num(k, posinf=1.0, neginf=1.0), torch.nan_to_num(v, posinf=1.0, neginf=1.0), table, n, **args)
    assert torch.equal(got[:, group:], clean[:, group:])


@pytest.mark.parametrize("q_t,kv_t,out_t", [("f32", "bf16", "f32"), ("f32", "bf16", "bf16"), ("bf16", "bf16", "bf16"), ("f32", "f32", "f32")])
@pytest.mark.parametrize("prompt", [False, True])
def test_infinite_queries(q_t, kv_t, out_t, prompt):
    """An infinite element makes every score +-inf: NaN where one is +inf, nothing seen (zeros) where all are -inf; a NaN element gives NaN; the other rows and
    heads keep their bits."""
    lens = [70, 300]
    k, v, table, _, _ = make_cache(lens, 16, 2, 64, kv_t, 19)
    k[:, :, 0, 3] = -k[:, :, 0, 3].abs()
    seq = t32([0, 1, 1, 0, 1])
    n = t32([70, 300, 299, 69, 298])
    q = torch.randn(5, 4, 64, generator=torch.Generator().manual_seed(3)).to(DT[q_t]).cuda()
    args = dict(seq=seq, out_dtype=DT[out_t], prompt=prompt)
    clean = cb.paged_attention(q, k, v, table, n, **args)
    q[1, 0, 3], q[2, 1, 3], q[3, 2, 3], q[4, 3, 7] = float("inf"), float("-inf"), float("inf"), float("nan")
    got = cb.paged_attention(q, k, v, table, n, **args)
    assert bool((got[1, 0] == 0).all()) and bool(got[2, 1].isnan().all()) and bool(got[3, 2].isnan().all()) and bool(got[4, 3].isnan().all())
    for r, h in ((1, 0), (2, 1), (3, 2), (4, 3)):
        got[r, h] = clean[r, h]
    assert torch.equal(got, clean)


@pytest.mark.parametrize("q_t,kv_t,out_t", [("f32", "f32", "f32"), ("f32", "bf16", "bf16"), ("bf16", "bf16", "bf16")])
@pytest.mark.parametrize("rows,heads,kv_heads,dim", [(4, 8, 2, 128), (12, 4, 4, 64), (40, 8, 2, 128), (64, 6, 6, 64), (96, 4, 2, 64)])
def test_rows_of_long_sequences_in_any_order(q_t, kv_t, out_t, rows, heads, kv_heads, dim):
    """Few and many rows of one and of four long sequences, one sequence after the other and in turn: the same values however they are planned."""
    lens = [5000, 3001, 4100, 4999]
    k, v, table, keys, vals = make_cache(lens, 64, kv_heads, dim, kv_t, 23)
    q = torch.randn(rows, heads, dim, generator=torch.Generator().manual_seed(4)).to(DT[q_t]).cuda()
    for seqs, order in ((1, "after"), (4, "after"), (4, "turn")):
        each = rows // seqs
        at = [(s, lens[s] - each + 1 + i) for s in range(seqs) for i in range(each)]
        if order == "turn":
            at = [at[s * each + i] for i in range(each) for s in range(seqs)]
        some = [r for r in range(rows) if r % 7 == 0 or r == rows - 1]
        want = [ref_attention(np64(q[r]), keys[s][:n], vals[s][:n], 0, dim ** -0.5) for r, (s, n) in ((r, at[r]) for r in some)]
        for prompt in (None, True, False):
            got = np64(cb.paged_attention(q, k, v, table[:seqs], t32([n for _, n in at]), seq=t32([s for s, _ in at]), out_dtype=DT[out_t], prompt=prompt))
            for r, (ref, mag, err) in zip(some, want):
                tol = 2 * (2 * err * U + 2.0 ** -21 + at[r][1] * U) * mag
                if out_t == "bf16":
                    tol = (tol + 2.0 ** -16 * mag) * (1 + 2.0 ** -8) + 2.0 ** -8 * np.abs(ref)
                assert (np.abs(got[r] - ref) <= tol).all(), (seqs, order, prompt, r)


@pytest.mark.parametrize("q_t,out_t", [("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16")])
@pytest.mark.parametrize("order", ["slots", "heads"])
def test_infinities_in_one_of_neighbouring_heads(q_t, out_t, order):
    """Enough rows that blocks take four neighbouring key heads (heads beside each other) or one (heads apart), in a graph that is replayed as the values come and
    go: head 2 sees an infinite value and a key of -inf score, the others keep their bits."""
    lens = [70, 33, 90]
    k, v, table, keys, vals = make_cache(lens, 16, 16, 64, "bf16", 29, order)
    rows = [(i % 3, lens[i % 3]) for i in range(120)]
    q = torch.randn(120, 16, 64, generator=torch.Generator().manual_seed(5)).bfloat16().abs().to(DT[q_t]).cuda() + 0.5
    seq, n = t32([s for s, _ in rows]), t32([m for _, m in rows])
    call = lambda: cb.paged_attention(q, k, v, table, n, seq=seq, out_dtype=DT[out_t], prompt=False)  # noqa: E731
    clean = call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    at = [(s, lens[s] - 5) for s in range(3)]
    places = [(int(table[s, j // 16]), j % 16) for s, j in at]
    held = [(k[p, i, 2, 3].clone(), v[p, i, 2, 7].clone()) for p, i in places]
    for turn in range(4):
        for (p, i), (hk, hv), (s, j) in zip(places, held, at):
            k[p, i, 2, 3] = float("-inf") if turn == 1 else hk
            v[p, i, 2, 7] = float("inf") if turn == 2 else hv
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, call())
        rest = [h for h in range(16) if h != 2]
        assert torch.equal(out[:, rest], clean[:, rest])
        if turn == 1:
            assert bool(out.isfinite().all())
            for r in (0, 1, 2, 119):
                s, m = rows[r]
                keep = [x for x in range(m) if x != at[s][1]]
                ref, mag, err = ref_attention(np64(q[r, 2:3]), keys[s][keep, 2:3], vals[s][keep, 2:3], 0, 0.125)
                tol = 2 * (2 * err * U + 2.0 ** -21 + m * U) * mag
                if out_t == "bf16":
                    tol = (tol + 2.0 ** -16 * mag) * (1 + 2.0 ** -8) + 2.0 ** -8 * np.abs(ref)
                assert (np.abs(np64(out[r, 2:3]) - ref) <= tol).all(), r
        elif turn == 2:
            assert bool((out[:, 2, 7] == float("inf")).all()) and bool(out[:, 2, :7].isfinite().all()) and bool(out[:, 2, 8:].isfinite().all())
        else:
            assert torch.equal(out, clean)
