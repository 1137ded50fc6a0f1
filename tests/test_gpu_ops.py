"""Serving operators (paged append, paged attention, logits rules) against plain 64-bit numpy on the same inputs.

Tolerances are derived, not tuned.  u = 2^-24 is half an fp32 step.  Attention: a score is a dot product of D products, its error at
most (D + 2) u sum |q_i k_i| scale =: e; each weight is then off by a factor of at most 1 + 2 e + 2^-21 (the maximum cancels,
the exponential is good to 2^-22), the weighted sum over n keys by n u more, and so is the sum of weights: |out - ref| <=
2 (2 e + 2^-21 + n u) sum p |v| / sum p.  Weights that enter a bf16 matrix product are rounded by at most 2^-8 each; a bf16 result by 2^-8
of itself (half a step of its 8 significant bits)."""
import ctypes as C

import numpy as np
import pytest

torch = pytest.importorskip("torch")
import chatterbox_amd as cb  # noqa: E402
from chatterbox_amd import _lib  # noqa: E402

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def np64(t):
    return t.detach().to("cpu", torch.float64).numpy()


def make_cache(lengths, page, heads, dim, kv, seed, order="slots", spare=3, fill=None):
    """Pool, table and contiguous 64-bit copies of every sequence's keys and values.  Slots no sequence owns hold `fill` (NaN)."""
    rng = np.random.default_rng(seed)
    need = [max(0, -(-n // page)) for n in lengths]
    pool = sum(need) + spare
    shape = (pool, page, heads, dim)
    if order == "slots":
        k, v = (torch.full(shape, float("nan"), dtype=DT[kv]) for _ in range(2))
    elif order == "heads":          # [pages, heads, slots, dim] in memory
        k, v = (torch.full((pool, heads, page, dim), float("nan"), dtype=DT[kv]).transpose(1, 2) for _ in range(2))
    else:                           # keys and values of a page side by side, rows padded
        both = torch.full((pool, 2, page, heads, dim + 8), float("nan"), dtype=DT[kv])
        k, v = both[:, 0, ..., :dim], both[:, 1, ..., :dim]
    ids = rng.permutation(pool)
    table = np.full((len(lengths), max(1, max(need))), -7, np.int32)
    keys, vals, at = [], [], 0
    for s, n in enumerate(lengths):
        n = max(n, 0)
        table[s, :need[s]] = ids[at:at + need[s]]
        at += need[s]
        ks, vs = (torch.from_numpy(rng.standard_normal((n, heads, dim)).astype(np.float32)).to(DT[kv]) for _ in range(2))
        for j in range(n):
            k[table[s, j // page], j % page] = ks[j]
            v[table[s, j // page], j % page] = vs[j]
        keys.append(np64(ks))
        vals.append(np64(vs))
    if order == "slots" or order == "heads":
        place = (lambda t: t.cuda()) if order == "slots" else (lambda t: t.transpose(1, 2).contiguous().cuda().transpose(1, 2))
        k, v = place(k), place(v)
    else:
        both = both.cuda()
        k, v = both[:, 0, ..., :dim], both[:, 1, ..., :dim]
    return k, v, torch.from_numpy(table).cuda(), keys, vals


def ref_attention(q, keys, vals, first, scale):
    """One row: q [H, D], keys [n, Hk, D] -> out [H, D], sum p |v| / sum p, largest score error / U."""
    H, D = q.shape
    n, Hk, _ = keys.shape
    out, mag, err = np.zeros((H, D)), np.zeros((H, D)), 0.0
    if n <= first:
        return out, mag, err
    for h in range(H):
        kk, vv = keys[first:, h // (H // Hk)], vals[first:, h // (H // Hk)]
        s = kk @ q[h] * scale
        err = max(err, (D + 2) * float((np.abs(kk) @ np.abs(q[h])).max()) * abs(scale))
        p = np.exp(s - s.max())
        out[h], mag[h] = p @ vv / p.sum(), p @ np.abs(vv) / p.sum()
    return out, mag, err


def check_rows(got, q, keys, vals, starts, seq, lengths, scale, out_dtype, weights_bf16):
    got = np64(got)
    for r, n in enumerate(lengths):
        if n < 0:
            continue
        s = seq[r]
        ref, mag, err = ref_attention(np64(q[r]), keys[s][:n], vals[s][:n], 0 if starts is None else max(0, starts[r]), scale)
        tol = 2 * (2 * err * U + 2.0 ** -21 + max(n, 1) * U) * mag
        if weights_bf16:
            tol += 2.0 ** -8 * mag
        if out_dtype == "bf16":
            tol += 2.0 ** -8 * (np.abs(ref) + tol)
        bad = np.abs(got[r] - ref) > tol + 1e-30
        assert not bad.any() and np.isfinite(got[r]).all(), (r, n, np.abs(got[r] - ref).max(), tol.max())


LENGTHS = [1, 2, 0, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 300, 511, 513, 777, -1, 1030]
TYPES = [("f32", "f32", "f32"), ("f32", "bf16", "f32"), ("f32", "bf16", "bf16"), ("f32", "f32", "bf16"), ("bf16", "bf16", "bf16"), ("bf16", "bf16", "f32")]


@pytest.mark.parametrize("q_t,kv_t,out_t", TYPES)
@pytest.mark.parametrize("heads,kv_heads,dim,page,order", [(16, 16, 64, 16, "slots"), (8, 2, 128, 64, "heads"), (15, 5, 64, 1, "pairs"),
                                                           (7, 1, 128, 8, "slots"), (40, 1, 64, 128, "pairs"), (3, 3, 128, 4096, "heads")])
def test_attention_matches_64_bits(q_t, kv_t, out_t, heads, kv_heads, dim, page, order):
    k, v, table, keys, vals = make_cache(LENGTHS, page, kv_heads, dim, kv_t, 11 + heads, order)
    rows = len(LENGTHS)
    q = (torch.randn(rows, heads, dim, generator=torch.Generator().manual_seed(5)) * 2).to(DT[q_t]).cuda()
    lengths = torch.tensor(LENGTHS, dtype=torch.int32).cuda()
    out = torch.full((rows, heads, dim), 77.0, dtype=DT[out_t], device="cuda")
    got = cb.paged_attention(q, k, v, table, lengths, out=out)
    assert got is out
    check_rows(got, q, keys, vals, None, range(rows), LENGTHS, dim ** -0.5, out_t, out_t == "bf16")
    assert bool((got[LENGTHS.index(0)] == 0).all()) and bool((got[LENGTHS.index(-1)] == 77).all())
    again = cb.paged_attention(q, k, v, table, lengths, out_dtype=DT[out_t])
    live = lengths >= 0
    assert torch.equal(again[live], got[live])          # the same call, the same bits


@pytest.mark.parametrize("max_length", [0, 1, 64, 400, 1030, 5000])
@pytest.mark.parametrize("q_t,kv_t", [("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16")])
def test_attention_plan_does_not_change_what_is_computed(max_length, q_t, kv_t):
    """max_length plans the split alone: rows above it come out right; first keys inside, at and past the end; scale given."""
    lens = [1030, 5, 640, 0, 129, 1000, 33]
    starts = [1000, 5, -3, 4, 128, 0, 40]
    k, v, table, keys, vals = make_cache(lens, 32, 4, 64, kv_t, 3)
    q = torch.randn(len(lens), 12, 64, generator=torch.Generator().manual_seed(6)).to(DT[q_t]).cuda()
    got = cb.paged_attention(q, k, v, table, torch.tensor(lens, dtype=torch.int32).cuda(), starts=torch.tensor(starts, dtype=torch.int32).cuda(),
                             scale=0.3, max_length=max_length)
    check_rows(got, q, keys, vals, starts, range(len(lens)), lens, np.float64(np.float32(0.3)), q_t, q_t == "bf16")
    for r in (1, 3, 6):
        assert bool((got[r] == 0).all())


@pytest.mark.parametrize("q_t,out_t", [("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16")])
@pytest.mark.parametrize("heads,kv_heads,order", [(15, 5, "slots"), (16, 16, "pairs")])
def test_attention_many_rows_of_neighbouring_heads(q_t, out_t, heads, kv_heads, order):
    """Enough rows of 128-byte keys that blocks take four neighbouring heads (the last block of 5 heads takes one), whole and split."""
    rng = np.random.default_rng(kv_heads)
    rows = 1100 // kv_heads
    lens = [int(n) for n in rng.integers(0, 80, rows)]
    lens[3], lens[4], lens[-1] = 0, -1, 700
    k, v, table, keys, vals = make_cache(lens, 16, kv_heads, 64, "bf16", 21, order)
    q = torch.randn(rows, heads, 64, generator=torch.Generator().manual_seed(3)).to(DT[q_t]).cuda()
    lengths = torch.tensor(lens, dtype=torch.int32).cuda()
    for most in (700, 80):
        out = torch.full((rows, heads, 64), 5.0, dtype=DT[out_t], device="cuda")
        cb.paged_attention(q, k, v, table, lengths, out=out, max_length=most)
        check_rows(out, q, keys, vals, None, range(rows), lens, 0.125, out_t, out_t == "bf16")
        assert bool((out[4] == 5).all()) and bool((out[3] == 0).all())


@pytest.mark.parametrize("q_t,kv_t", [("f32", "f32"), ("bf16", "bf16")])
@pytest.mark.parametrize("heads", [16, 17, 33])
def test_attention_wide_groups_over_a_long_row(q_t, kv_t, heads):
    """One key head for 16 and more query heads of 128: the largest blocks, and groups that end inside a tile of 16."""
    lens = [9001, 0, 130]
    k, v, table, keys, vals = make_cache(lens, 128, 1, 128, kv_t, 31)
    q = torch.randn(3, heads, 128, generator=torch.Generator().manual_seed(4)).to(DT[q_t]).cuda()
    got = cb.paged_attention(q, k, v, table, torch.tensor(lens, dtype=torch.int32).cuda(), max_length=2 ** 17)
    check_rows(got, q, keys, vals, None, range(3), lens, 128 ** -0.5, q_t, q_t == "bf16")
    assert torch.equal(cb.paged_attention(q, k, v, table, torch.tensor(lens, dtype=torch.int32).cuda(), max_length=2 ** 17, out=q), got)   # in place


@pytest.mark.parametrize("q_t,kv_t", [("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16")])
@pytest.mark.parametrize("most", [64, 20000])
def test_attention_passes_on_nan(q_t, kv_t, most):
    """NaN in a query, a live key or a live value comes out, as the formula has it, in one block and split over many; other rows and heads keep theirs."""
    lens = [3000, 33, 3000, 700, 1]
    k, v, table, keys, vals = make_cache(lens, 16, 2, 64, kv_t, 41)
    q = torch.randn(5, 4, 64, generator=torch.Generator().manual_seed(5)).to(DT[q_t])
    q[0, 1, 7] = float("nan")
    q[1, 2] = float("nan")
    q[4, 3, 0] = float("nan")
    q = q.cuda()
    at = 2900
    page, slot = int(table[2, at // 16]), at % 16
    k[page, slot, 0, 3] = float("nan")
    v[page, slot, 1, 5] = float("nan")
    lengths = torch.tensor(lens, dtype=torch.int32).cuda()
    got = cb.paged_attention(q, k, v, table, lengths, max_length=most)
    for r, h in ((0, 1), (1, 2), (4, 3), (2, 0), (2, 1)):
        assert bool(got[r, h].isnan().all()), (r, h)
    for h in (2, 3):
        nan = got[2, h].isnan()
        assert bool(nan[5]) and int(nan.sum()) == 1
    rest = torch.ones(5, 4, dtype=torch.bool)
    for r, h in ((0, 1), (1, 2), (4, 3), (2, 0), (2, 1), (2, 2), (2, 3)):
        rest[r, h] = False
    clean = torch.nan_to_num(q)
    k[page, slot, 0, 3] = 0
    v[page, slot, 1, 5] = 0
    assert torch.equal(got[rest], cb.paged_attention(clean, k, v, table, lengths, max_length=most)[rest])


@pytest.mark.parametrize("rows,heads,kv_heads,dim,q_t,kv_t,longest", [
    (220, 15, 5, 64, "f32", "bf16", 1500),     # blocks of four heads, rows in four parts
    (2, 40, 1, 128, "bf16", "bf16", 9000),     # three blocks to a key head, many parts
    (70, 4, 1, 64, "f32", "f32", 900),         # eight parts of four waves
    (300, 8, 4, 128, "f32", "f32", 700),       # two parts of four waves
    (40, 8, 8, 64, "f32", "bf16", 20000),      # much work: parts of eight waves
    (128, 2, 1, 128, "bf16", "bf16", 500),     # one block of two waves
    (12, 12, 2, 128, "f32", "bf16", 2500)])    # parts of two waves
def test_attention_plans(rows, heads, kv_heads, dim, q_t, kv_t, longest):
    """Each way to share a call's keys among blocks and waves, with rows of every length below the longest, none and padding among them."""
    rng = np.random.default_rng(longest)
    lens = [int(n) for n in rng.integers(0, min(longest, 200), rows)]
    lens[0], lens[1 % rows], lens[-1] = (0, -3, longest) if rows > 2 else (longest, longest - 1, longest)
    k, v, table, keys, vals = make_cache(lens, 32, kv_heads, dim, kv_t, 51)
    q = torch.randn(rows, heads, dim, generator=torch.Generator().manual_seed(6)).to(DT[q_t]).cuda()
    out = torch.full((rows, heads, dim), 5.0, dtype=DT[q_t], device="cuda")
    cb.paged_attention(q, k, v, table, torch.tensor(lens, dtype=torch.int32).cuda(), out=out)
    check_rows(out, q, keys, vals, None, range(rows), lens, dim ** -0.5, q_t, q_t == "bf16")
    if rows > 2:
        assert bool((out[1] == 5).all()) and bool((out[0] == 0).all())


@pytest.mark.parametrize("heads,kv_heads,dim", [(16, 16, 64), (16, 8, 128)])
def test_attention_of_the_most_rows(heads, kv_heads, dim):
    """2^24 (row, head) pairs, the most a call takes: rows of one key give its value exactly, rows of none zeros; one more row is refused."""
    rows = 1 << 20
    k, v, table, _, vals = make_cache([1, 1, 1], 16, kv_heads, dim, "bf16", 61)
    q = torch.zeros(rows, heads, dim, dtype=torch.bfloat16, device="cuda")
    seq = (torch.arange(rows, device="cuda", dtype=torch.int32) * 7) % 3
    lengths = (torch.arange(rows, device="cuda", dtype=torch.int32) % 5 != 0).int()
    out = cb.paged_attention(q, k, v, table, lengths, seq=seq)
    want = torch.from_numpy(np.stack(vals)[:, 0]).to(torch.bfloat16).cuda().repeat_interleave(heads // kv_heads, 1)
    for r0 in range(0, rows, 1 << 17):
        part = slice(r0, r0 + (1 << 17))
        assert torch.equal(out[part], want[seq[part].long()] * lengths[part].view(-1, 1, 1))
    more = torch.zeros(rows + 1, dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="pairs"):
        cb.paged_attention(q[:1].expand(rows + 1, heads, dim), k, v, table, more, seq=more, out=torch.empty(rows + 1, heads, dim, dtype=torch.bfloat16, device="cuda"))


def test_attention_prompt_rows_share_a_sequence():
    """Rows of a prompt: the same sequence at lengths 1, 2, 3, ... , in any order, through `seq`; q and out as strided views."""
    k, v, table, keys, vals = make_cache([70, 9], 16, 2, 64, "bf16", 4)
    seq = [0] * 70 + [1] * 9
    lens = list(range(1, 71)) + list(range(1, 10))
    perm = np.random.default_rng(0).permutation(79)
    seq, lens = [seq[i] for i in perm], [lens[i] for i in perm]
    wide = torch.randn(79, 3, 6, 64, generator=torch.Generator().manual_seed(1)).cuda()
    q, out = wide[:, 1], torch.zeros(6, 79, 64, device="cuda").transpose(0, 1)
    got = cb.paged_attention(q, k, v, table, torch.tensor(lens, dtype=torch.int32).cuda(), seq=torch.tensor(seq, dtype=torch.int32).cuda(), out=out)
    check_rows(got, q, keys, vals, None, seq, lens, 0.125, "f32", False)


@pytest.mark.parametrize("kv_t,q_t", [("f32", "f32"), ("bf16", "f32"), ("bf16", "bf16")])
def test_attention_long_row_is_split_and_joined(kv_t, q_t):
    """One row of many keys (peaked scores), one short: far more blocks than rows."""
    n, hk, d = 20011, 2, 128
    g = torch.Generator().manual_seed(8)
    kk, vv = (torch.randn(n, hk, d, generator=g).to(DT[kv_t]) for _ in range(2))
    page = 64
    pages = -(-n // page)
    k, v = (torch.full((pages + 1, page, hk, d), float("inf"), dtype=DT[kv_t]) for _ in range(2))
    k[:pages].view(-1, hk, d)[:n], v[:pages].view(-1, hk, d)[:n] = kk, vv
    table = torch.stack([torch.arange(pages, dtype=torch.int32)] * 2).cuda()
    q = (torch.randn(2, 8, d, generator=g) * 3).to(DT[q_t]).cuda()
    lens = [n, 50]
    got = cb.paged_attention(q, k.cuda(), v.cuda(), table, torch.tensor(lens, dtype=torch.int32).cuda())
    keys, vals = [np64(kk)] * 2, [np64(vv)] * 2
    check_rows(got, q, keys, vals, None, range(2), lens, d ** -0.5, q_t, q_t == "bf16")


def test_attention_bad_pages_and_sequences_are_absent():
    """Table entries that name no page, sequences outside the table and lengths past it: those keys are absent, nothing else changes."""
    lens = [100, 100, 100, 64]
    k, v, table, keys, vals = make_cache(lens, 32, 2, 64, "f32", 9)
    table[0, 1], table[1, 0], table[2, :] = 10 ** 6, -1, -1
    q = torch.randn(6, 4, 64, generator=torch.Generator().manual_seed(2)).cuda()
    got = cb.paged_attention(q, k, v, table, torch.tensor([100, 100, 100, 2 ** 31 - 1, 5, 5], dtype=torch.int32).cuda(),
                             seq=torch.tensor([0, 1, 2, 3, 4, -1], dtype=torch.int32).cuda())
    keep0 = [i for i in range(100) if not 32 <= i < 64]
    k0, v0 = keys[0][keep0], vals[0][keep0]
    check_rows(got[:1], q[:1], [k0], [v0], None, [0], [len(keep0)], 0.125, "f32", False)
    check_rows(got[1:2], q[1:2], [keys[1][32:]], [vals[1][32:]], None, [0], [68], 0.125, "f32", False)
    assert bool((got[2] == 0).all()) and bool((got[4:] == 0).all())
    check_rows(got[3:4], q[3:4], [keys[3]], [vals[3]], None, [0], [64], 0.125, "f32", False)    # (its other table entries name no page)


def test_attention_extreme_values():
    """Scores of +-1e30 and of zero: one key takes everything, equal keys share; keys of -inf score are as good as absent."""
    k = torch.zeros(1, 8, 1, 64)
    v = torch.arange(8.0).view(1, 8, 1, 1).expand(1, 8, 1, 64).contiguous()
    k[0, 3, 0, 0] = 1e30
    k[0, 5, 0, 1] = float("-inf")
    q = torch.zeros(3, 1, 64)
    q[0, 0, 0] = 1.0          # key 3 wins
    q[1, 0, 0] = -1.0         # key 3 loses, the others share
    q[2, 0, 2] = 1.0          # all equal
    q[:, 0, 1] = 1e-9         # key 5 scores -inf in every row
    table = torch.zeros(3, 1, dtype=torch.int32).cuda()
    got = cb.paged_attention(q.cuda(), k.cuda(), v.cuda(), table, torch.full((3,), 8, dtype=torch.int32).cuda()).cpu()
    want = torch.tensor([3.0, (28 - 3 - 5) / 6, (28 - 5) / 7])
    assert torch.allclose(got[:, 0, 0], want, rtol=8 * U, atol=0), got[:, 0, 0]


def prompt_rows(lens, shuffled, seed):
    """Rows (sequence, length, start) of prompts over sequences of `lens` keys: all positions of the first, the last 40 of each other, causal; padding,
    rows of no sequence and rows past the end among them; in order or shuffled."""
    rng = np.random.default_rng(seed)
    rows = [(0, n, 0) for n in range(1, lens[0] + 1)]
    for s in range(1, len(lens)):
        rows += [(s, n, int(rng.integers(0, 30)) if s % 2 else 0) for n in range(max(0, lens[s] - 40), lens[s] + 1)]
    rows[5] = (0, -1, 0)
    rows.insert(20, (-4, 9, 0))
    rows.insert(37, (len(lens) + 3, 50, 0))
    rows.insert(50, (0, 12, 12))
    if shuffled:
        rng.shuffle(rows)
    return [tuple(int(x) for x in r) for r in rows]


@pytest.mark.parametrize("q_t,kv_t,out_t", TYPES)
@pytest.mark.parametrize("heads,kv_heads,dim,page,order,shuffled", [(16, 16, 64, 16, "slots", False), (8, 2, 128, 64, "heads", False), (15, 5, 64, 1, "pairs", False),
                                                                    (7, 1, 128, 8, "slots", False), (12, 2, 128, 32, "slots", True), (5, 1, 64, 128, "heads", True),
                                                                    (2, 2, 64, 4, "pairs", True), (16, 2, 64, 2, "slots", False), (48, 4, 64, 32, "slots", False)])
def test_attention_of_prompts(q_t, kv_t, out_t, heads, kv_heads, dim, page, order, shuffled):
    """Rows that share the keys they read, with whatever else the call allows among them, against 64 bits; padding rows stay as they were."""
    lens = [75, 131, 0, 40, 300]
    k, v, table, keys, vals = make_cache(lens, page, kv_heads, dim, kv_t, 71, order)
    rows = prompt_rows(lens, shuffled, heads)
    seq, n, start = (torch.tensor([r[i] for r in rows], dtype=torch.int32).cuda() for i in range(3))
    q = (torch.randn(len(rows), heads, dim, generator=torch.Generator().manual_seed(8)) * 2).to(DT[q_t]).cuda()
    out = torch.full((len(rows), heads, dim), 5.0, dtype=DT[out_t], device="cuda")
    cb.paged_attention(q, k, v, table, n, seq=seq, starts=start, out=out, prompt=True)
    lengths = [r[1] if 0 <= r[0] < len(lens) else min(r[1], 0) for r in rows]
    sq = [r[0] if 0 <= r[0] < len(lens) else 0 for r in rows]
    check_rows(out, q, keys, vals, [r[2] for r in rows], sq, lengths, dim ** -0.5, out_t, out_t == "bf16")
    assert bool((out[[i for i, r in enumerate(rows) if r[1] < 0]] == 5).all())
    if not shuffled:                                       # a prompt without starts: by the sizes' rule, and in place
        own = [i for i, r in enumerate(rows) if r[0] == 0]
        qs = q[own].contiguous()
        want = cb.paged_attention(qs, k, v, table[:1], n[own], seq=seq[own], prompt=True)
        live = n[own] >= 0                                 # (a padding row of a new tensor holds anything)
        assert torch.equal(cb.paged_attention(qs, k, v, table[:1], n[own], seq=seq[own])[live], want[live])
        alone = cb.paged_attention(qs, k, v, table[:1], n[own], seq=seq[own], prompt=False)
        check_rows(want, qs, keys, vals, None, [0] * len(own), [int(x) for x in n[own]], dim ** -0.5, q_t, q_t == "bf16")
        check_rows(alone, qs, keys, vals, None, [0] * len(own), [int(x) for x in n[own]], dim ** -0.5, q_t, q_t == "bf16")
        assert torch.equal(cb.paged_attention(qs, k, v, table[:1], n[own], seq=seq[own], out=qs, prompt=True)[live], want[live])


@pytest.mark.parametrize("q_t,kv_t", [("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16")])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_attention_of_prompts_keeps_later_values_out(q_t, kv_t, bad):
    """A value that is not finite reaches the rows that see its key, in its element, and no other row of the tiles it lies in; keys off the pool likewise."""
    lens, at = [200], 133
    k, v, table, keys, vals = make_cache(lens, 16, 4, 64, kv_t, 81)
    page, slot = int(table[0, at // 16]), at % 16
    n = torch.arange(1, 201, dtype=torch.int32).cuda()
    seq = torch.zeros(200, dtype=torch.int32).cuda()
    q = torch.randn(200, 8, 64, generator=torch.Generator().manual_seed(9)).to(DT[q_t]).cuda()
    want = cb.paged_attention(q, k, v, table, n, seq=seq, prompt=True)
    v[page, slot, 2, 11] = bad
    got = cb.paged_attention(q, k, v, table, n, seq=seq, prompt=True)
    hit = torch.zeros(200, 8, 64, dtype=torch.bool)
    hit[at:, 4:6, 11] = True
    assert not bool(got[hit].isfinite().any())
    got[hit] = want[hit]                                  # (every other element as if the value were finite; summed in another order, so not bit for bit)
    check_rows(got, q, keys, vals, None, [0] * 200, list(range(1, 201)), 0.125, q_t, q_t == "bf16")
    v[page, slot, 2, 11] = 0
    k[page, slot, 1, 5] = float("nan")
    got = cb.paged_attention(q, k, v, table, n, seq=seq, prompt=True)
    assert bool(got[at:, 2:4].isnan().all()) and torch.equal(got[:at], want[:at]) and bool(got[at:, 4:].isfinite().all())
    k[page, slot, 1, 5] = 0
    table[0, 6] = -1                                     # keys 96..111 are absent: their values do not matter
    got = cb.paged_attention(q, k, v, table, n, seq=seq, prompt=True)
    for r in (95, 96, 111, 112, 199):
        there = [j for j in range(r + 1) if not 96 <= j < 112]
        kk, vv = k[table[0].clamp(min=0).long()].flatten(0, 1)[there], v[table[0].clamp(min=0).long()].flatten(0, 1)[there]
        check_rows(got[r:r + 1], q[r:r + 1], [np64(kk)], [np64(vv)], None, [0], [len(there)], 0.125, q_t, q_t == "bf16")


@pytest.mark.parametrize("q_t,kv_t,heads,kv_heads,dim,prompts", [("bf16", "bf16", 16, 8, 128, [700, 500]), ("bf16", "bf16", 16, 4, 64, [1500, 40, 1460, 1000]),
                                                                  ("f32", "bf16", 8, 8, 64, [2050, 2000]), ("f32", "f32", 16, 16, 64, [300] * 30), ("f32", "f32", 8, 1, 128, [901])])
def test_attention_of_long_prompts(q_t, kv_t, heads, kv_heads, dim, prompts):
    """Enough rows for blocks of one and of two waves; every 61st row and the ends of each prompt against 64 bits."""
    k, v, table, keys, vals = make_cache(prompts, 64, kv_heads, dim, kv_t, 91)
    lens = [n for p in prompts for n in range(1, p + 1)]
    sq = [i for i, p in enumerate(prompts) for _ in range(p)]
    q = torch.randn(len(lens), heads, dim, generator=torch.Generator().manual_seed(10)).to(DT[q_t]).cuda()
    got = cb.paged_attention(q, k, v, table, torch.tensor(lens, dtype=torch.int32).cuda(), seq=torch.tensor(sq, dtype=torch.int32).cuda())
    some = [r for r in range(len(lens)) if r % 61 == 0 or (r % 7 == 0 and lens[r] <= 2) or (r + 1 < len(lens) and sq[r] != sq[r + 1] and sq[r] % 5 == 0)] + [len(lens) - 1]
    check_rows(got[some], q[some], keys, vals, None, [sq[r] for r in some], [lens[r] for r in some], dim ** -0.5, q_t, q_t == "bf16")


def test_attention_offsets_past_32_bits():
    """A pool of more than 2^31 elements: pages at both ends."""
    page, hk, d = 256, 8, 128
    pages = (2 ** 31 + 2 ** 28) // (page * hk * d)
    k, v = (torch.empty(pages, page, hk, d, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    g = torch.Generator(device="cuda").manual_seed(3)
    ends = [0, pages - 1, pages - 2]
    for i in ends:
        k[i], v[i] = (torch.randn(page, hk, d, generator=g, device="cuda").bfloat16() for _ in range(2))
    table = torch.tensor([ends], dtype=torch.int32).cuda()
    q = torch.randn(1, 8, d, generator=g, device="cuda").bfloat16()
    got = cb.paged_attention(q, k, v, table, torch.tensor([700], dtype=torch.int32).cuda())
    keys, vals = ([np64(torch.cat([t[i] for i in ends])[:700])] for t in (k, v))
    check_rows(got, q, keys, vals, None, [0], [700], d ** -0.5, "bf16", True)
    # and the append at the far end of it
    new = torch.randn(1, hk, d, generator=g, device="cuda").bfloat16()
    cb.paged_kv_append(new, new * 2, k, v, torch.tensor([[0, 0, pages - 1]], dtype=torch.int32).cuda(), torch.tensor([2 * page + 255], dtype=torch.int32).cuda())
    assert torch.equal(k[pages - 1, 255], new[0]) and torch.equal(v[pages - 1, 255], new[0] * 2)


# ---- append -----------------------------------------------------------------------------------------------------------------

def rotated(x, cos, sin):
    half = x.shape[-1] // 2
    a, b = x[..., :half], x[..., half:]
    return np.concatenate([a * cos - b * sin, b * cos + a * sin], -1), np.concatenate([np.abs(a * cos) + np.abs(b * sin), np.abs(b * cos) + np.abs(a * sin)], -1)


def half_step(t):
    return 2.0 ** -8 if t == "bf16" else U


@pytest.mark.parametrize("x_t,kv_t", [("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("heads,kv_heads,dim,page,rotate,with_q", [(16, 16, 64, 16, True, True), (8, 2, 128, 64, True, True), (3, 1, 64, 1, False, True),
                                                                   (5, 5, 128, 8, True, False), (12, 4, 128, 32, False, False)])
def test_append_matches_64_bits(x_t, kv_t, heads, kv_heads, dim, page, rotate, with_q):
    """Rows of several sequences in mixed order, some skipped (negative position, past the rotation tables, past or off the block
    table, no such sequence): every slot and every q_out row that is not named keeps its bits."""
    rng = np.random.default_rng(heads * dim + page)
    n_seqs, width = 4, -(-70 // page)
    pool = n_seqs * width + 2
    table = rng.permutation(pool)[: n_seqs * width].reshape(n_seqs, width).astype(np.int32)
    table[2, 0] = pool                       # names no page
    pos = np.concatenate([np.arange(61), np.arange(7), [3, -1, -5, width * page, 64, 2, 5]]).astype(np.int32)
    seq = np.concatenate([np.zeros(61), np.full(7, 1), [3, 0, 1, 0, 3, 4, -1]]).astype(np.int32)
    extra = [(2, 0)] if page > 1 else []
    seq, pos = np.append(seq, [s for s, _ in extra]).astype(np.int32), np.append(pos, [p for _, p in extra]).astype(np.int32)
    order = rng.permutation(len(pos))
    pos, seq = pos[order], seq[order]
    rope_len = 64                            # position 64 is past it
    rows = len(pos)
    # inputs as views of one packed projection; the cache heads-first in memory; q_out padded
    packed = torch.from_numpy(rng.standard_normal((rows, heads + 2 * kv_heads, dim)).astype(np.float32)).to(DT[x_t]).cuda()
    q, k, v = packed[:, :heads], packed[:, heads:heads + kv_heads], packed[:, heads + kv_heads:]
    kc, vc = (torch.full((pool, kv_heads, page, dim), -3.0, dtype=DT[kv_t], device="cuda").transpose(1, 2) for _ in range(2))
    angle = np.arange(rope_len)[:, None] * 500000.0 ** (-np.arange(0, dim, 2) / dim)
    cos, sin = (torch.from_numpy(np.concatenate([f(angle)] * 2, 1).astype(np.float32)).cuda() for f in (np.cos, np.sin))
    q_out = torch.full((rows, heads + 1, dim), 9.0, dtype=DT[x_t], device="cuda")[:, 1:]
    got_q = cb.paged_kv_append(k, v, kc, vc, torch.from_numpy(table).cuda(), torch.from_numpy(pos).cuda(), seq=torch.from_numpy(seq).cuda(),
                               q=q if with_q else None, q_out=q_out if with_q else None, rope=(cos, sin) if rotate else None)
    want_k, want_v = np.full(kc.shape, -3.0), np.full(vc.shape, -3.0)
    tol_k, tol_v = np.zeros(kc.shape), np.zeros(vc.shape)
    want_q, tol_q = np.full(q.shape, 9.0), np.zeros(q.shape)
    kn, vn, qn, cn, sn = np64(k), np64(v), np64(q), np64(cos)[:, : dim // 2], np64(sin)[:, : dim // 2]
    for r in range(rows):
        p, s = int(pos[r]), int(seq[r])
        if p < 0 or not 0 <= s < n_seqs or p >= width * page or (rotate and p >= rope_len) or not 0 <= table[s, p // page] < pool:
            continue
        if rotate:
            (kk, km), (qq, qm) = rotated(kn[r], cn[p], sn[p]), rotated(qn[r], cn[p], sn[p])
            kt, qt = 3 * U * km, 3 * U * qm        # two products and a sum
        else:
            kk, qq, kt, qt = kn[r], qn[r], 0.0, 0.0
        at = table[s, p // page], p % page
        want_k[at], want_v[at] = kk, vn[r]
        step = 0.0 if (x_t == kv_t and not rotate) else half_step(kv_t)
        tol_k[at] = kt + step * (np.abs(kk) + kt)
        tol_v[at] = 0.0 if x_t == kv_t or kv_t == "f32" else half_step("bf16") * np.abs(vn[r])
        want_q[r], tol_q[r] = qq, qt + (half_step(x_t) * (np.abs(qq) + qt) if rotate else 0.0)
    assert (np.abs(np64(kc) - want_k) <= tol_k).all()
    assert (np.abs(np64(vc) - want_v) <= tol_v).all()
    if with_q:
        assert got_q is q_out and (np.abs(np64(got_q) - want_q) <= tol_q).all()
    else:
        assert got_q is None


def test_append_rotates_q_in_place():
    rows, d = 5, 64
    x = torch.randn(rows, 4, d, generator=torch.Generator().manual_seed(0)).cuda()
    k = torch.randn(rows, 2, d, generator=torch.Generator().manual_seed(1)).cuda()
    kc, vc = (torch.zeros(rows, 16, 2, d, device="cuda") for _ in range(2))
    table, pos = torch.arange(rows, dtype=torch.int32).view(rows, 1).cuda(), torch.tensor([0, 3, 15, 7, 1], dtype=torch.int32).cuda()
    a = torch.arange(16.0)[:, None] * 10000.0 ** (-torch.arange(0, d, 2) / d)
    rope = (a.cos().cuda(), a.sin().cuda())
    want = cb.paged_kv_append(k, k, kc, vc, table, pos, q=x.clone(), rope=rope)
    got = cb.paged_kv_append(k, k, kc, vc, table, pos, q=x, q_out=x, rope=rope)
    assert got is x and torch.equal(got, want)


def test_append_then_attention_as_a_step():
    """The two as a decode step uses them: prompts appended, then steps of one token, each against plain attention over everything
    appended so far; replayed as one captured graph with its lengths updated in place."""
    rng = np.random.default_rng(1)
    B, H, Hk, d, page, width = 3, 6, 2, 64, 16, 8
    kc, vc = (torch.full((B * width, page, Hk, d), float("nan"), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    table = torch.from_numpy(rng.permutation(B * width).reshape(B, width).astype(np.int32)).cuda()
    a = np.arange(width * page)[:, None] * 10000.0 ** (-np.arange(0, d, 2) / d)
    rope = tuple(torch.from_numpy(f(a).astype(np.float32)).cuda() for f in (np.cos, np.sin))
    cn, sn = np64(rope[0]), np64(rope[1])
    prompt = [37, 1, 16]
    pos = [p for n in prompt for p in range(n)]
    seq = [s for s, n in enumerate(prompt) for _ in range(n)]
    rows = len(pos)

    def rnd(*s):
        return torch.from_numpy(rng.standard_normal(s).astype(np.float32)).bfloat16().cuda()

    def t32(x):
        return torch.tensor(x, dtype=torch.int32).cuda()

    keys, vals = [np.zeros((0, Hk, d))] * B, [np.zeros((0, Hk, d))] * B

    def remember(k, v, seqs, positions):
        for r, (s, p) in enumerate(zip(seqs, positions)):
            kr = torch.from_numpy(rotated(np64(k[r]), cn[p], sn[p])[0].astype(np.float32)).bfloat16()
            keys[s] = np.concatenate([keys[s], np64(kr)[None]])
            vals[s] = np.concatenate([vals[s], np64(v[r])[None]])

    k, v = rnd(rows, Hk, d), rnd(rows, Hk, d)
    cb.paged_kv_append(k, v, kc, vc, table, t32(pos), seq=t32(seq), rope=rope)
    remember(k, v, seq, pos)
    q, k, v = rnd(B, H, d), rnd(B, Hk, d), rnd(B, Hk, d)
    at, lens = t32(prompt), t32([n + 1 for n in prompt])

    def step():
        qr = cb.paged_kv_append(k, v, kc, vc, table, at, q=q, rope=rope)
        return qr, cb.paged_attention(qr, kc, vc, table, lens)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        qr, out = step()
    for i in range(20):
        q.copy_(rnd(B, H, d)), k.copy_(rnd(B, Hk, d)), v.copy_(rnd(B, Hk, d))
        graph.replay()
        torch.cuda.synchronize()
        remember(k, v, range(B), [n + i for n in prompt])
        # the key of this step as the cache holds it (a rounding to bf16 may fall either way): taken from the cache, checked within half a step
        for s in range(B):
            p = prompt[s] + i
            held = np64(kc[int(table[s, p // page]), p % page])
            assert (np.abs(held - keys[s][-1]) <= 2.0 ** -7 * np.abs(held) + 1e-30).all()
            keys[s][-1] = held
        now = [n + i + 1 for n in prompt]
        eager = cb.paged_attention(qr, kc, vc, table, lens)
        assert torch.equal(eager, out)
        check_rows(out, qr, keys, vals, None, range(B), now, d ** -0.5, "bf16", True)
        at += 1
        lens += 1
    torch.cuda.synchronize()


def test_two_graphs_and_two_streams_do_not_share_a_workspace():
    """Two captured attentions replayed at once on two streams, and eager calls between them: each equals its eager result."""
    g = torch.Generator(device="cuda").manual_seed(0)
    page, hk, d, n = 64, 2, 128, 6000
    pages = -(-n // page)
    k, v = (torch.randn(pages, page, hk, d, generator=g, device="cuda").bfloat16() for _ in range(2))
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None]
    qs = [torch.randn(1, 8, d, generator=g, device="cuda").bfloat16() for _ in range(2)]
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    eager = [cb.paged_attention(q, k, v, table, lens) for q in qs]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for q in qs:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(cb.paged_attention(q, k, v, table, lens))
        graphs.append(gr)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(10):
        for gr, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
        third = cb.paged_attention(qs[0], k, v, table, lens)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], eager[0]) and torch.equal(outs[1], eager[1]) and torch.equal(third, eager[0])


# ---- logits -----------------------------------------------------------------------------------------------------------------

def ref_logits(l, u, w, tokens, n_tokens, rep, fre, pre, ids, vals, allowed):
    """64-bit values and the magnitude that bounds the fp32 rounding of each entry."""
    B, V = l.shape
    z, mag = l.astype(np.float64).copy(), np.abs(l).astype(np.float64)
    if u is not None:
        mag = np.abs(z) + abs(w) * (np.abs(z) + np.abs(u)) * 2
        z = z + w * (z - u)
    for r in range(B):
        if ids is not None:
            row = r if len(ids) > 1 else 0
            for t, b in dict((int(t), float(b)) for t, b in zip(ids[row], vals[row])).items():
                if 0 <= t < V:
                    z[r, t] += b
                    mag[r, t] += abs(b)
        if tokens is not None:
            n = min(max(int(n_tokens[r]), 0), tokens.shape[1])
            seen, count = np.unique(tokens[r, :n], return_counts=True)
            for t, c in zip(seen, count):
                if 0 <= t < V:
                    z[r, t] = z[r, t] / rep[r] if z[r, t] > 0 else z[r, t] * rep[r]
                    z[r, t] -= fre[r] * c + pre[r]
                    mag[r, t] = mag[r, t] * max(rep[r], 1 / rep[r]) + abs(fre[r]) * c * 2 + abs(pre[r])
        if allowed is not None:
            words = allowed[r if len(allowed) > 1 else 0].view(np.uint32)
            for t in range(V):
                if not (words[t >> 5] >> np.uint32(t & 31)) & 1:
                    z[r, t] = -np.inf
    return z, mag


@pytest.mark.parametrize("x_t", ["f32", "bf16"])
@pytest.mark.parametrize("rows,vocab,cap,n_bias,mask,guide,each", [(1, 8194, 300, 0, "none", True, False), (3, 1, 4, 2, "rows", False, True),
                                                                   (5, 31, 9, 3, "shared", True, True), (2, 4096, 50, 1, "rows", True, False),
                                                                   (4, 4097, 1000, 300, "shared", False, True), (7, 12289, 2500, 24, "rows", True, True),
                                                                   (2, 100, 0, 0, "none", False, False), (300, 65, 3, 4, "rows", False, True)])
def test_logits_match_64_bits(x_t, rows, vocab, cap, n_bias, mask, guide, each):
    rng = np.random.default_rng(vocab + rows)
    wide = vocab + 3                                     # rows that start at odd addresses
    l, u = (torch.from_numpy((rng.standard_normal((rows, wide)) * 3).astype(np.float32)).to(DT[x_t])[:, 1:vocab + 1].cuda() for _ in range(2))
    l = torch.cat([torch.zeros(rows, 1, dtype=DT[x_t], device="cuda"), l], 1)[:, 1:]
    tokens = rng.integers(-2, vocab + 2, (rows, cap)).astype(np.int32) if cap else None
    if cap:
        tokens[:, ::3] = rng.integers(0, min(vocab, 7), tokens[:, ::3].shape)     # repeats
    n_tokens = rng.integers(-1, cap + 3, rows).astype(np.int32) if cap else None
    rep, fre, pre = (rng.uniform(lo, hi, rows).astype(np.float32) for lo, hi in ((0.5, 2.0), (-0.5, 1.0), (-1.0, 1.0)))
    if not each:
        rep[:], fre[:], pre[:] = rep[0], fre[0], pre[0]
    ids = vals = allowed = None
    if n_bias:
        ids = rng.integers(-1, vocab + 1, (rows, n_bias)).astype(np.int32)
        ids[:, -1] = ids[:, 0]                                                   # named twice: the last counts
        vals = (rng.standard_normal((rows, n_bias)) * 5).astype(np.float32)
    if mask != "none":
        allowed = rng.integers(-2 ** 31, 2 ** 31, (1 if mask == "shared" else rows, (vocab + 31) // 32 + 1)).astype(np.int32)
        if mask == "rows":
            allowed[-1] = 0                                                      # nothing allowed
            with torch.no_grad():
                l[0, : min(vocab, 32)] = torch.tensor([float("nan"), float("inf"), float("-inf")] * 11)[: min(vocab, 32)].to(l)
            allowed[0, 0] = 0                                                    # NaN and infinities in masked places

    def dev(x):
        return None if x is None else torch.from_numpy(x).cuda()

    kw = dict(uncond=u if guide else None, cfg_weight=0.5, tokens=dev(tokens), n_tokens=dev(n_tokens), bias_ids=dev(ids), bias_values=dev(vals), allowed=dev(allowed))
    kw.update(dict(repetition_penalty=dev(rep), frequency_penalty=dev(fre), presence_penalty=dev(pre)) if each else
              dict(repetition_penalty=float(rep[0]), frequency_penalty=float(fre[0]), presence_penalty=float(pre[0])))
    got = cb.process_logits(l, **kw)
    with np.errstate(invalid="ignore"):
        want, mag = ref_logits(np64(l), np64(u) if guide else None, 0.5, tokens, n_tokens, rep.astype(np.float64), fre.astype(np.float64),
                               pre.astype(np.float64), ids, vals, allowed)
    g = np64(got)
    off = np.isneginf(want)
    assert (np.isneginf(g) == off).all()
    # at most 7 fp32 operations follow each other, each within U of a value below mag; then the rounding to the type
    tol = 8 * U * mag + (2.0 ** -8 * (np.abs(want) + 8 * U * mag) if x_t == "bf16" else 0.0)
    assert (np.abs(g[~off] - want[~off]) <= tol[~off]).all()
    cb.process_logits(l, **kw, out=l)                    # in place
    assert torch.equal(l, got)


@pytest.mark.parametrize("x_t", ["f32", "bf16"])
@pytest.mark.parametrize("rows,vocab,cap,n_bias", [(300, 12289, 700, 40), (90, 33000, 17000, 1500), (3, 9000, 9000, 4094), (70, 40960, 0, 3)])
def test_logits_of_many_chunks(x_t, rows, vocab, cap, n_bias):
    """Blocks of several chunks (tokens sorted, or too many to be), token lists and biases longer than a block holds; vectorised reference."""
    rng = np.random.default_rng(rows)
    l = torch.from_numpy((rng.standard_normal((rows, vocab)) * 3).astype(np.float32)).to(DT[x_t]).cuda()
    tokens = rng.integers(0, vocab, (rows, cap)).astype(np.int32) if cap else None
    n_tokens = rng.integers(0, cap + 1, rows).astype(np.int32) if cap else None
    if cap:
        n_tokens[0] = cap
    rep, fre, pre = (rng.uniform(lo, hi, rows).astype(np.float32) for lo, hi in ((0.5, 2.0), (0.0, 1.0), (-1.0, 1.0)))
    ids = rng.integers(0, vocab, (rows, n_bias)).astype(np.int32)
    ids[:, -1], ids[:, n_bias // 2] = ids[:, 0], ids[:, 0]
    vals = (rng.standard_normal((rows, n_bias)) * 5).astype(np.float32)
    allowed = rng.integers(-2 ** 31, 2 ** 31, (rows, (vocab + 31) // 32)).astype(np.int32)

    def dev(x):
        return None if x is None else torch.from_numpy(x).cuda()

    got = np64(cb.process_logits(l, tokens=dev(tokens), n_tokens=dev(n_tokens), repetition_penalty=dev(rep), frequency_penalty=dev(fre), presence_penalty=dev(pre),
                                 bias_ids=dev(ids), bias_values=dev(vals), allowed=dev(allowed)))
    x = np64(l)
    for r in range(rows):
        z = x[r].copy()
        b = dict(zip(ids[r].tolist(), vals[r].tolist()))
        at = np.fromiter(b, np.int64)
        z[at] += np.fromiter(b.values(), np.float64)
        mag = np.abs(x[r]).max() + np.abs(vals).max()
        if cap:
            c = np.bincount(tokens[r, : n_tokens[r]], minlength=vocab).astype(np.float64)
            z = np.where(c > 0, np.where(z > 0, z / np.float64(rep[r]), z * np.float64(rep[r])) - np.float64(fre[r]) * c - np.float64(pre[r]), z)
            mag = 2 * mag + np.abs(fre[r]) * c.max() * 2 + 1
        bits = np.unpackbits(allowed[r].view(np.uint8), bitorder="little")[:vocab].astype(bool)
        tol = 8 * U * mag + (2.0 ** -8 * (np.abs(z) + 8 * U * mag) if x_t == "bf16" else 0.0)
        assert (np.isneginf(got[r]) == ~bits).all(), r
        assert (np.abs(got[r] - z)[bits] <= (tol[bits] if x_t == "bf16" else tol)).all(), r


def test_logits_without_rules_are_copied_bit_for_bit():
    l = torch.randn(3, 1000, generator=torch.Generator().manual_seed(0)).cuda()
    l[0, 0], l[1, 5], l[2, 7] = float("nan"), float("inf"), -0.0
    for x in (l, l.bfloat16()):
        got = cb.process_logits(x)
        assert torch.equal(got.view(torch.int32 if x.dtype == torch.float32 else torch.int16), x.view(torch.int32 if x.dtype == torch.float32 else torch.int16))


def test_logits_captured_and_replayed():
    """A captured call replayed with its token list growing in place equals the eager call every time."""
    g = torch.Generator(device="cuda").manual_seed(0)
    l = torch.randn(4, 5001, generator=g, device="cuda")
    tokens, n = torch.zeros(4, 64, dtype=torch.int32, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    kw = dict(tokens=tokens, n_tokens=n, repetition_penalty=1.3, frequency_penalty=0.2, presence_penalty=0.1)
    cb.process_logits(l, **kw)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cb.process_logits(l, **kw)
    for i in range(12):
        tokens[:, i] = torch.randint(0, 5001, (4,), generator=g, device="cuda", dtype=torch.int32)
        n += 1
        graph.replay()
        assert torch.equal(out, cb.process_logits(l, **kw))
    torch.cuda.synchronize()


# ---- no rows, no tokens -------------------------------------------------------------------------------------------------------

def test_empty_calls():
    k, v = (torch.zeros(2, 16, 2, 64, device="cuda") for _ in range(2))
    table = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    assert cb.paged_attention(torch.zeros(0, 4, 64, device="cuda"), k, v, table, none).shape == (0, 4, 64)
    e = torch.zeros(0, 2, 64, device="cuda")
    assert cb.paged_kv_append(e, e, k, v, table, none, q=torch.zeros(0, 4, 64, device="cuda")).shape == (0, 4, 64)
    assert cb.process_logits(torch.zeros(0, 50, device="cuda")).shape == (0, 50)


def test_refusals_name_what_is_wrong():
    k, v = (torch.zeros(2, 16, 2, 64, device="cuda") for _ in range(2))
    table, lens = torch.zeros(3, 1, dtype=torch.int32, device="cuda"), torch.ones(3, dtype=torch.int32, device="cuda")
    q = torch.zeros(3, 4, 64, device="cuda")
    for bad, word in ((dict(q=q[..., :32]), "head_dim"), (dict(q=q.double()), "dtype"), (dict(q=q.cpu()), "is on"), (dict(q=q.bfloat16()), "bf16"),
                      (dict(q=q[:, :3]), "multiple"), (dict(lengths=lens.long()), "int32"), (dict(lengths=lens[:2]), "shape"),
                      (dict(q=q.clone().requires_grad_()), "gradients"), (dict(block_table=table[0]), "shape"), (dict(v_pages=v.bfloat16()), "dtype"),
                      (dict(out=q[:2]), "shape"), (dict(starts=lens.float()), "int32"), (dict(block_table=table[:2]), "sequences"),
                      (dict(scale=float("nan")), "finite"), (dict(k_pages=k[..., :63]), "differ")):
        args = dict(q=q, k_pages=k, v_pages=v, block_table=table, lengths=lens)
        args.update(bad)
        with pytest.raises((ValueError, _lib.T3miError), match=word):
            cb.paged_attention(**args)
    shifted = torch.zeros(3 * 4 * 64 + 1, device="cuda")[1:].view(3, 4, 64)
    with pytest.raises(_lib.T3miError, match="16 bytes"):
        cb.paged_attention(shifted, k, v, table, lens)
    with pytest.raises(_lib.T3miError, match="power of two"):
        cb.paged_attention(q, k[:, :12], v[:, :12], table, lens)


def test_work_on_another_stream_is_ordered_with_it():
    """Called under torch.cuda.stream: the operator runs on that stream, after what it holds and before what follows."""
    k, v = (torch.zeros(64, 64, 2, 64, device="cuda") for _ in range(2))
    table = torch.arange(64, dtype=torch.int32, device="cuda")[None]
    lens = torch.tensor([4096], dtype=torch.int32, device="cuda")
    q = torch.ones(1, 4, 64, device="cuda")
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        for i in range(1, 6):
            v.fill_(float(i))
            out = cb.paged_attention(q, k, v, table, lens)
            kept = out.clone()
            v.fill_(-1.0)
            st.synchronize()
            assert torch.allclose(kept, torch.full_like(kept, float(i)), rtol=4100 * U, atol=0)


def small_calls(seed):
    """One call of each operator over a ragged cache, and what they give."""
    k, v, table, _, _ = make_cache([700, 3, 1200], 16, 2, 64, "bf16", seed)
    gen = torch.Generator().manual_seed(seed)
    q, kn, vn = (torch.randn(3, h, 64, generator=gen).cuda() for h in (4, 2, 2))
    lengths = torch.tensor([700, 3, 1200], dtype=torch.int32).cuda()
    pos = lengths - 1
    l = torch.randn(5, 9001, generator=gen).cuda()
    tok = torch.randint(0, 9001, (5, 40), generator=gen).int().cuda()
    n_tok = torch.tensor([40, 0, 7, 1, 40], dtype=torch.int32).cuda()

    def run():
        turned = cb.paged_kv_append(kn, vn, k, v, table, pos, q=q)
        out = cb.paged_attention(turned, k, v, table, lengths, max_length=1200)
        return out, cb.process_logits(l, tokens=tok, n_tokens=n_tok, repetition_penalty=1.3, frequency_penalty=0.25)

    return run, (q, kn, vn, k, v, table, pos, lengths, l, tok, n_tok)


def test_calls_from_two_threads_on_two_streams():
    """The lock of the interpreter is given up while a call enqueues: two loops side by side get what each gets alone."""
    import threading
    runs = [small_calls(s)[0] for s in (1, 2)]
    want = [r() for r in runs]
    torch.cuda.synchronize()
    streams, wrong = [torch.cuda.Stream() for _ in runs], []

    def loop(i):
        try:
            with torch.cuda.stream(streams[i]):
                for _ in range(200):
                    got = runs[i]()
                streams[i].synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                    wrong.append(i)
                for _ in range(20):
                    try:
                        cb.process_logits(torch.zeros(2, 10, device="cuda"), repetition_penalty=0.0)
                        wrong.append("no refusal")
                    except RuntimeError as e:
                        if "repetition" not in str(e):
                            wrong.append(str(e))
        except BaseException as e:
            wrong.append(repr(e))

    threads = [threading.Thread(target=loop, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong


def test_calls_and_refusals_keep_no_reference():
    import sys
    run, tensors = small_calls(3)
    q, kn, vn, k, v, table, pos, lengths, l, tok, n_tok = tensors
    objects = list(tensors) + [torch.float32, torch.bfloat16, torch.int32, torch.uint8, q.device]

    def refusals():
        for bad in (lambda: cb.paged_attention(q, k, v, table, lengths[:2]), lambda: cb.paged_attention(q, k, v, table, lengths, out=q[:2]),
                    lambda: cb.paged_attention(q, k, v, table, lengths, out_dtype=torch.float16), lambda: cb.paged_attention(q[:, :3], k, v, table, lengths),
                    lambda: cb.paged_attention(q, k, v, table, lengths, scale=float("nan")), lambda: cb.paged_kv_append(kn, vn, k, v, table, pos, q=q, q_out=q[:1]),
                    lambda: cb.paged_kv_append(kn, vn, k, v, table, pos.cpu()), lambda: cb.process_logits(l, tokens=tok), lambda: cb.process_logits(l, out=l[:2]),
                    lambda: cb.process_logits(l, repetition_penalty=0.0), lambda: cb.process_logits(l, allowed=tok)):
            with pytest.raises((ValueError, RuntimeError)):
                bad()

    for _ in range(3):
        run()
        refusals()
    torch.cuda.synchronize()
    before, memory = [sys.getrefcount(o) for o in objects], torch.cuda.memory_allocated()
    for _ in range(30):
        run()
        refusals()
    torch.cuda.synchronize()
    after = [sys.getrefcount(o) for o in objects]
    assert all(abs(a - b) <= 5 for a, b in zip(after, before)), list(zip(before, after))   # (30 turns: a reference kept once a turn shows)
    assert torch.cuda.memory_allocated() == memory


def test_tensors_are_read_alike_without_the_exchange_table(monkeypatch):
    """torch versions without the DLPack exchange table: the tensors' own methods say the same of them, strides, refusals and all."""
    from chatterbox_amd import ops
    run, tensors = small_calls(4)
    q, _, _, k, v, table, _, lengths, l, _, _ = tensors
    wide = torch.randn(3, 8, 64, device="cuda")
    calls = [lambda: cb.paged_attention(wide[:, ::2], k, v, table, lengths), lambda: cb.paged_attention(wide[:, 1::2].bfloat16(), k, v, table, lengths),
             lambda: cb.process_logits(l[1:2, 5:], bias_ids=torch.tensor([[3, 7]], dtype=torch.int32, device="cuda"), bias_values=torch.ones(1, 2, device="cuda")),
             lambda: cb.process_logits(l.t()[:5].t(), frequency_penalty=torch.ones(5, device="cuda"))]
    bad = [lambda: cb.paged_attention(wide.transpose(1, 2), k, v, table, lengths), lambda: cb.paged_attention(q.double(), k, v, table, lengths),
           lambda: cb.paged_attention(q, k, v, table.cpu(), lengths), lambda: cb.paged_attention(q[0], k, v, table, lengths),
           lambda: cb.paged_attention(q.clone().requires_grad_(), k, v, table, lengths), lambda: cb.process_logits(l, tokens=l.long(), n_tokens=lengths)]

    def all_of_them():
        out, words = list(run()), []
        for c in calls:
            try:
                out.append(c())
            except ValueError as e:
                words.append(str(e))
        for c in bad:
            with pytest.raises(ValueError) as e:
                c()
            words.append(str(e.value))
        return out, words

    with_table = all_of_them()
    try:
        with monkeypatch.context() as m:
            m.delattr(torch.Tensor, "__dlpack_c_exchange_api__", raising=False)
            ops._bind()
            without = all_of_them()
    finally:
        ops._bind()
    assert with_table[1] == without[1] and len(with_table[0]) == len(without[0])
    for a, b in zip(with_table[0], without[0]):
        assert a.dtype == b.dtype and torch.equal(a, b)
