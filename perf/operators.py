"""The serving operators' cases: attention of new tokens over a paged key-value cache, the append that fills it, and the
rules a logits row goes through before it is sampled.  `run` computes each in its plain form (elementary torch operations in
32 bits, rounded once at the end) or, with `own`, through the framework's entry points."""
import math
import random

import torch

own = False

_DT = {"f32": torch.float32, "bf16": torch.bfloat16}
_MOST_BYTES = 1.9e9     # what the largest listed case moves, about


def listed():
    return [
        # one utterance and its guidance row, the 350-slot fp32 cache of the fixed-cache decode loop: latency alone counts
        _attend("attend-1-utterance", rows=2, heads=16, kv_heads=16, dim=64, page=16, low=349, high=350, q="f32", kv="f32"),
        # 64 utterances with their guidance rows in mid-flight, bf16 cache, fp32 query rows: the batched decode step
        _attend("attend-64-utterances", rows=128, heads=16, kv_heads=16, dim=64, page=64, low=60, high=1100, q="f32", kv="bf16"),
        # a few very long contexts with shared key heads: the keys have to be split to fill the card
        _attend("attend-long-contexts", rows=3, heads=32, kv_heads=8, dim=128, page=128, low=100003, high=131071, q="bf16", kv="bf16"),
        # a full serving batch of ragged contexts, shared key heads
        _attend("attend-full-batch", rows=96, heads=32, kv_heads=8, dim=128, page=64, low=1000, high=8190, q="bf16", kv="bf16"),
        # left-padded rows (each starts at its own key), fp32 cache, an odd number of heads and rows
        _attend("attend-left-padded", rows=37, heads=15, kv_heads=5, dim=64, page=32, low=500, high=3001, q="f32", kv="f32", padded=True),
        # the append of that single utterance's step
        _append("append-1-utterance", rows=2, seqs=2, heads=16, kv_heads=16, dim=64, page=16, past=349, x="f32", kv="f32"),
        # one step of 512 utterances with guidance rows into a bf16 cache
        _append("append-512-utterances", rows=1024, seqs=1024, heads=16, kv_heads=16, dim=64, page=64, past=463, x="f32", kv="bf16"),
        # one prefill group: all prompt positions of the utterances as one list of rows
        _append("append-prefill", rows=32768, seqs=80, heads=16, kv_heads=16, dim=64, page=64, past=0, x="f32", kv="bf16"),
        # bf16 prompts with shared key heads, an odd number of rows
        _append("append-prefill-shared", rows=20011, seqs=7, heads=32, kv_heads=8, dim=128, page=128, past=0, x="bf16", kv="bf16"),
        # one utterance's logits: guidance pair, penalties over the tokens so far
        _logits("logits-1-utterance", rows=1, vocab=8194, past=300, bias=0, mask="none", guide=True, x="f32"),
        # 64 utterances' logits with every rule, a token set shared by the rows
        _logits("logits-64-utterances", rows=64, vocab=8194, past=1000, bias=24, mask="shared", guide=True, x="f32"),
        # a full batch over a large vocabulary, a grammar's mask for every row
        _logits("logits-large-vocabulary", rows=256, vocab=131072, past=4000, bias=300, mask="rows", guide=False, x="f32"),
    ]


def _attend(name, rows, heads, kv_heads, dim, page, low, high, q, kv, padded=False):
    return {"name": name, "kind": "attend", "rows": rows, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page,
            "low": low, "high": high, "q": q, "kv": kv, "padded": padded}


def _append(name, rows, seqs, heads, kv_heads, dim, page, past, x, kv, rotate=True):
    return {"name": name, "kind": "append", "rows": rows, "seqs": seqs, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "page": page, "past": past, "x": x, "kv": kv, "rotate": rotate}


def _logits(name, rows, vocab, past, bias, mask, guide, x):
    return {"name": name, "kind": "logits", "rows": rows, "vocab": vocab, "past": past, "bias": bias, "mask": mask,
            "guide": guide, "x": x}


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(("attend", "attend", "append", "logits"))
    q, kv = rng.choice((("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16")))
    heads, kv_heads = rng.choice(((16, 16), (8, 8), (32, 8), (15, 5), (24, 2), (12, 1), (7, 7), (64, 4)))
    dim, page = rng.choice((64, 128)), rng.choice((8, 16, 32, 64, 128, 256))
    if kind == "attend":
        rows, high = _log(rng, 1, 256), _log(rng, 1, 131071)
        high = max(1, min(high, int(_MOST_BYTES / (rows * _row_bytes(kv_heads, dim, kv)))))
        c = _attend("", rows, heads, kv_heads, dim, page, max(1, int(high * rng.uniform(0.0, 1.0))), high, q, kv, rng.random() < 0.25)
    elif kind == "append":
        rows = min(_log(rng, 1, 32768), int(_MOST_BYTES / 4 / ((heads + 2 * kv_heads) * dim * 8)))
        seqs = rows if rng.random() < 0.5 and rows <= 1024 else max(1, min(rows, _log(rng, 1, 96)))
        c = _append("", rows, seqs, heads, kv_heads, dim, page, _log(rng, 1, 2000) - 1 if seqs == rows else 0, q, kv, rng.random() < 0.8)
    else:
        vocab = _log(rng, 100, 262144)
        rows = min(_log(rng, 1, 512), max(1, 256 * 131072 // vocab // 2))
        c = _logits("", rows, vocab, _log(rng, 1, 4000), rng.choice((0, 1, 24, 300)), rng.choice(("none", "shared", "rows")), rng.random() < 0.5, q)
    del c["name"]
    return c


def _row_bytes(kv_heads, dim, kv):
    return 2 * kv_heads * dim * _DT[kv].itemsize


def _lengths(case, seed):
    r = random.Random(seed * 7919 + 13)
    n = [r.randint(case["low"], case["high"]) for _ in range(case["rows"])]
    n[0] = case["high"]
    if case["rows"] >= 8:
        n[-1] = 0          # a padding row of the batch
    return n


def _table(counts, page, pool, r, dev):
    """Block table for sequences of `counts` keys: a pool's pages dealt in random order, unused entries -1."""
    need = [-(-n // page) for n in counts]
    ids = list(range(pool))
    r.shuffle(ids)
    wide = max(1, max(need))
    rows, at = [], 0
    for k in need:
        rows.append(ids[at:at + k] + [-1] * (wide - k))
        at += k
    return torch.tensor(rows, dtype=torch.int32).to(dev)


def prepare(case, seed):
    dev = "cuda"
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    r = random.Random(seed)

    def rnd(*shape, dt="f32", std=1.0):
        return (torch.randn(*shape, generator=g, device=dev, dtype=_DT[dt]) * std) if std != 1.0 else torch.randn(*shape, generator=g, device=dev, dtype=_DT[dt])

    s = dict(case)
    if case["kind"] == "attend":
        lens = _lengths(case, seed)
        pool = sum(-(-n // case["page"]) for n in lens) + 3
        table = _table(lens, case["page"], pool, r, dev)
        s["k"] = rnd(pool, case["page"], case["kv_heads"], case["dim"], dt=case["kv"])
        s["v"] = rnd(pool, case["page"], case["kv_heads"], case["dim"], dt=case["kv"])
        s["qx"] = rnd(case["rows"], case["heads"], case["dim"], dt=case["q"], std=2.0)
        s["table"], s["lengths"], s["longest"] = table, torch.tensor(lens, dtype=torch.int32).to(dev), max(lens)
        s["starts"] = torch.tensor([r.randint(0, n // 2) for n in lens], dtype=torch.int32).to(dev) if case["padded"] else None
    elif case["kind"] == "append":
        rows, seqs, h, hk, d = case["rows"], case["seqs"], case["heads"], case["kv_heads"], case["dim"]
        if seqs == rows:                                        # one new token for every sequence
            pos = [r.randint(case["past"] // 2, case["past"]) for _ in range(rows)]
            pool = rows * -(-(case["past"] + 1) // case["page"]) + 3
            counts, seq = [p + 1 for p in pos], None
        else:                                                   # prompts of different lengths, all their positions
            cuts = sorted(r.sample(range(1, rows), seqs - 1)) if seqs > 1 else []
            counts = [b - a for a, b in zip([0] + cuts, cuts + [rows])]
            pos = [p for n in counts for p in range(n)]
            pool = rows // case["page"] + seqs + 3
            seq = torch.tensor([i for i, n in enumerate(counts) for _ in range(n)], dtype=torch.int32).to(dev)
        table = _table(counts, case["page"], pool, r, dev)
        s["kx"], s["vx"], s["qx"] = rnd(rows, hk, d, dt=case["x"]), rnd(rows, hk, d, dt=case["x"]), rnd(rows, h, d, dt=case["x"])
        s["k"] = torch.zeros(pool, case["page"], hk, d, device=dev, dtype=_DT[case["kv"]])
        s["v"] = torch.zeros_like(s["k"])
        s["table"], s["positions"], s["seq"] = table, torch.tensor(pos, dtype=torch.int32).to(dev), seq
        s["rope"] = None
        if case["rotate"]:
            angle = torch.arange(max(pos) + 1, device=dev, dtype=torch.float64)[:, None] * 500000.0 ** (-torch.arange(0, d, 2, device=dev, dtype=torch.float64) / d)
            s["rope"] = (angle.cos().float(), angle.sin().float())
    else:
        b, v = case["rows"], case["vocab"]
        s["logits"] = rnd(b, v, dt=case["x"], std=3.0)
        s["uncond"] = rnd(b, v, dt=case["x"], std=3.0) if case["guide"] else None
        # tokens so far repeat themselves: a third of them comes from a few ids
        few = torch.randint(0, v, (b, 16), generator=g, device=dev, dtype=torch.int32)
        s["tokens"] = torch.randint(0, v, (b, case["past"]), generator=g, device=dev, dtype=torch.int32)
        pick = torch.randint(0, 48, (b, case["past"]), generator=g, device=dev)
        s["tokens"] = torch.where(pick < 16, few.gather(1, pick.clamp(max=15)), s["tokens"]).contiguous()
        s["n_tokens"] = torch.randint(0, case["past"] + 1, (b,), generator=g, device=dev, dtype=torch.int32)
        s["repetition"] = 1.0 + torch.rand(b, generator=g, device=dev)
        s["frequency"] = torch.rand(b, generator=g, device=dev)
        s["presence"] = torch.rand(b, generator=g, device=dev)
        s["ids"] = s["values"] = s["allowed"] = None
        if case["bias"]:
            s["ids"] = torch.randint(0, v, (b, case["bias"]), generator=g, device=dev, dtype=torch.int32)
            s["values"] = rnd(b, case["bias"], std=4.0)
        if case["mask"] != "none":
            n = 1 if case["mask"] == "shared" else b
            s["allowed"] = torch.randint(-2**31, 2**31, (n, (v + 31) // 32), generator=g, device=dev, dtype=torch.int32)
    return s


def run(state):
    if own:
        return {"attend": _own_attend, "append": _own_append, "logits": _own_logits}[state["kind"]](state)
    return {"attend": _plain_attend, "append": _plain_append, "logits": _plain_logits}[state["kind"]](state)


# ---- the framework's calls ----------------------------------------------------------------------------------------------

def _own_attend(s):
    import chatterbox_amd as cb
    return cb.paged_attention(s["qx"], s["k"], s["v"], s["table"], s["lengths"], starts=s["starts"], max_length=s["longest"])


def _own_append(s):
    import chatterbox_amd as cb
    q = cb.paged_kv_append(s["kx"], s["vx"], s["k"], s["v"], s["table"], s["positions"], seq=s["seq"], q=s["qx"], rope=s["rope"])
    return q, s["k"], s["v"]


def _own_logits(s):
    import chatterbox_amd as cb
    return cb.process_logits(s["logits"], uncond=s["uncond"], cfg_weight=0.5, tokens=s["tokens"], n_tokens=s["n_tokens"],
                             repetition_penalty=s["repetition"], frequency_penalty=s["frequency"], presence_penalty=s["presence"],
                             bias_ids=s["ids"], bias_values=s["values"], allowed=s["allowed"])


# ---- the plain forms ----------------------------------------------------------------------------------------------------

def _plain_attend(s):
    q, k, v, lens = s["qx"], s["k"], s["v"], s["lengths"]
    b, h, d = q.shape
    hk = k.shape[2]
    pages = s["table"].clamp(min=0).long()
    k = k[pages].flatten(1, 2).float()                                   # [b, keys, hk, d]
    v = v[pages].flatten(1, 2).float()
    at = torch.arange(k.shape[1], device=q.device)
    live = at[None] < lens[:, None]
    if s["starts"] is not None:
        live &= at[None] >= s["starts"][:, None]
    v = torch.where(live[:, :, None, None], v, 0.0)
    scores = torch.matmul(q.float().view(b, hk, h // hk, d), k.permute(0, 2, 3, 1)) * (1.0 / math.sqrt(d))
    scores = torch.where(live[:, None, None], scores, -torch.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -torch.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v.permute(0, 2, 1, 3)) / torch.where(total == 0, 1.0, total)
    return out.reshape(b, h, d).to(q.dtype)


def _rotate(x, cos, sin):
    half = x.shape[-1] // 2
    a, b = x[..., :half], x[..., half:]
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)


def _plain_append(s):
    k, v, q, at = s["kx"].float(), s["vx"].float(), s["qx"].float(), s["positions"].long()
    page = s["k"].shape[1]
    if s["rope"] is not None:
        cos, sin = (t[at][:, None] for t in s["rope"])
        k, q = _rotate(k, cos, sin), _rotate(q, cos, sin)
    seq = torch.arange(len(at), device=at.device) if s["seq"] is None else s["seq"].long()
    where = s["table"][seq, at // page].long()
    s["k"][where, at % page] = k.to(s["k"].dtype)
    s["v"][where, at % page] = v.to(s["v"].dtype)
    return q.to(s["qx"].dtype), s["k"], s["v"]


def _rules(s, z, kind):
    """The rules on a copy of the logits in `kind` bits; the id that a list names twice takes its last value."""
    b, v = z.shape
    dev = z.device
    if s["uncond"] is not None:
        z = z + 0.5 * (z - s["uncond"].to(kind))
    if s["ids"] is not None:
        n = s["ids"].shape[1]
        last = torch.zeros(b, v, dtype=torch.int64, device=dev)
        last.scatter_reduce_(1, s["ids"].long(), torch.arange(1, n + 1, device=dev).expand(b, n), "amax")
        z = z + torch.where(last > 0, s["values"].to(kind).gather(1, (last - 1).clamp(min=0)), 0.0)
    live = torch.arange(s["tokens"].shape[1], device=dev)[None] < s["n_tokens"][:, None]
    count = torch.zeros(b, v, dtype=torch.int32, device=dev)
    count.scatter_add_(1, s["tokens"].long(), live.to(torch.int32))
    r = s["repetition"].to(kind)[:, None]
    z = torch.where(count > 0, torch.where(z > 0, z / r, z * r), z)
    z = z - s["frequency"].to(kind)[:, None] * count - s["presence"].to(kind)[:, None] * (count > 0)
    if s["allowed"] is not None:
        at = torch.arange(v, device=dev)
        z = torch.where((s["allowed"][:, at // 32] >> (at % 32)) & 1 > 0, z, -torch.inf)
    return z


def _plain_logits(s):
    return _rules(s, s["logits"].float(), torch.float32).to(s["logits"].dtype)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------

def work(case):
    if case["kind"] == "attend":
        lens = [n * (0.75 if case["padded"] else 1.0) for n in _lengths(case, 0)]
        keys, rows = sum(lens), case["rows"]
        io = rows * case["heads"] * case["dim"] * _DT[case["q"]].itemsize
        return {"bytes": keys * _row_bytes(case["kv_heads"], case["dim"], case["kv"]) + 2 * io + sum(-(-int(n) // case["page"]) for n in lens) * 4 + 4 * rows,
                "flops": 4.0 * keys * case["heads"] * case["dim"]}
    if case["kind"] == "append":
        rows, d = case["rows"], case["dim"]
        x, c = _DT[case["x"]].itemsize, _DT[case["kv"]].itemsize
        angles = min(rows, case["past"] // 2 + 1 if case["seqs"] == rows else 2 * rows // case["seqs"]) * d * 4 if case["rotate"] else 0
        return {"bytes": rows * d * (case["heads"] * 2 * x + 2 * case["kv_heads"] * (x + c)) + angles + 4 * rows,
                "flops": 3.0 * rows * d * (case["heads"] + case["kv_heads"]) if case["rotate"] else 0.0}
    b, v, x = case["rows"], case["vocab"], _DT[case["x"]].itemsize
    n = b * v
    words = (v + 31) // 32 * 4 * {"none": 0, "shared": 1, "rows": b}[case["mask"]]
    return {"bytes": n * x * (3 if case["guide"] else 2) + words + b * (case["past"] // 2 * 4 + case["bias"] * 8 + 16), "flops": 6.0 * n}


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "attend":
        q, k, v, table, page = s["qx"], s["k"], s["v"], s["table"].tolist(), case["page"]
        group = case["heads"] // case["kv_heads"]
        out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
        starts = s["starts"].tolist() if s["starts"] is not None else [0] * case["rows"]
        for i, n in enumerate(s["lengths"].tolist()):
            if n <= starts[i]:
                continue
            ids = torch.tensor(table[i][:-(-n // page)], device=q.device)
            for j in range(case["kv_heads"]):
                kj = k[ids, :, j].reshape(-1, case["dim"])[starts[i]:n].double()
                vj = v[ids, :, j].reshape(-1, case["dim"])[starts[i]:n].double()
                w = torch.softmax(q[i, j * group:(j + 1) * group].double() @ kj.t().contiguous() / case["dim"] ** 0.5, -1)
                out[i, j * group:(j + 1) * group] = w @ vj
        return out
    if case["kind"] == "append":
        at = s["positions"].long()
        rows = torch.arange(len(at), device=at.device) if s["seq"] is None else s["seq"].long()

        def turned(x):
            x = x.double()
            if s["rope"] is None:
                return x
            cos, sin = (t[at].double()[:, None] for t in s["rope"])
            z = torch.complex(x[..., : case["dim"] // 2], x[..., case["dim"] // 2:]) * torch.complex(cos, sin)
            return torch.cat((z.real, z.imag), -1)

        flat = s["table"][rows, torch.div(at, case["page"], rounding_mode="floor")].long() * case["page"] + at % case["page"]
        k, v = (torch.zeros(s["k"].shape, dtype=torch.float64, device=at.device) for _ in range(2))
        k.view(-1, *k.shape[2:]).index_copy_(0, flat, turned(s["kx"]))
        v.view(-1, *v.shape[2:]).index_copy_(0, flat, s["vx"].double())
        return turned(s["qx"]), k, v
    out, v = [], case["vocab"]
    shift = torch.arange(32, device=s["logits"].device)
    for i in range(case["rows"]):
        z = s["logits"][i].double()
        if s["uncond"] is not None:
            z = 1.5 * z - 0.5 * s["uncond"][i].double()
        if s["ids"] is not None:
            named = dict(zip(s["ids"][i].tolist(), s["values"][i].tolist()))
            at = torch.tensor(list(named), device=z.device)
            z[at] += torch.tensor(list(named.values()), dtype=torch.float64, device=z.device)
        count = torch.bincount(s["tokens"][i, : int(s["n_tokens"][i])].long(), minlength=v).double()
        r = float(s["repetition"][i])
        z = torch.where(count > 0, z * torch.where(z > 0, 1.0 / r, r), z)
        z -= float(s["frequency"][i]) * count + float(s["presence"][i]) * (count > 0).double()
        if s["allowed"] is not None:
            words = s["allowed"][i if len(s["allowed"]) > 1 else 0]
            z[((words[:, None] >> shift) & 1).flatten()[:v] == 0] = -torch.inf
        out.append(z)
    return torch.stack(out)
