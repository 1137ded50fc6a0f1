"""Serving operators on torch tensors resident on the GPU: a key-value cache in pages (append, attention) and the rules a
logits row goes through before it is sampled.  A thin layer over the C entry points t3mi_paged_append, t3mi_paged_attention and
t3mi_process_logits (include/t3mi.h), for serving loops of one's own; the sessions of this package call the same kernels
(T3Model.set_paged_kv, T3Model.set_logit_rules).  The reference has no counterpart: its caches are contiguous
(R/llama_traced.R:274-297) and its sampling tail knows the repetition penalty alone (R/t3.R:529-537).

The calls enqueue on torch's current stream of the tensors' device and return; they may be captured into a graph.  Results and
workspaces are torch allocations of that stream.  There is no backward pass: inputs that require gradients are refused.
torch is imported by the first call, not with the package."""
from __future__ import annotations

import ctypes as C
from typing import Optional

from . import _lib

__all__ = ["paged_kv_append", "paged_attention", "process_logits"]

_torch = None
_raw_stream = None
_F32 = _BF16 = _I32 = None
_CODE: dict = {}


def _setup():
    global _torch, _raw_stream, _F32, _BF16, _I32
    import torch
    _torch, _F32, _BF16, _I32 = torch, torch.float32, torch.bfloat16, torch.int32
    _CODE[_F32], _CODE[_BF16] = _lib.W_F32, _lib.W_BF16
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    _raw_stream = raw if raw is not None else (lambda i: torch.cuda.current_stream(i).cuda_stream)


def _bad(msg: str):
    raise ValueError(msg)


def _rows(name: str, t, device, dtypes, dims: int):
    """A floating operand: on the device, of an admitted type, last dimension contiguous, without gradients."""
    if t.device != device:
        _bad(f"{name} is on {t.device}, not on {device}")
    if t.dtype not in dtypes:
        _bad(f"{name} has dtype {t.dtype}: float32 or bfloat16 wanted")
    if t.dim() != dims:
        _bad(f"{name} must have {dims} dimensions, got {tuple(t.shape)}")
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        _bad(f"{name}: the last dimension must be contiguous")
    if t.requires_grad and _torch.is_grad_enabled():
        _bad(f"{name} requires gradients: this operator has no backward pass")
    return t.data_ptr()


def _ints(name: str, t, device, shape):
    """An int32 array, last dimension contiguous; shape entries of None are free."""
    if t is None:
        return None
    if t.device != device or t.dtype != _I32:
        _bad(f"{name} must be int32 on {device}, got {t.dtype} on {t.device}")
    if t.dim() != len(shape) or any(w is not None and n != w for n, w in zip(t.shape, shape)):
        _bad(f"{name} has shape {tuple(t.shape)}, wanted {shape}")
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        _bad(f"{name}: the last dimension must be contiguous")
    return t.data_ptr()


def _cache(k_pages, v_pages, block_table):
    if _torch is None:
        _setup()
    device = k_pages.device
    if device.type != "cuda":
        _bad(f"k_pages is on {device}: the operators run on the GPU")
    dt = k_pages.dtype
    kp = _rows("k_pages", k_pages, device, _CODE, 4)
    vp = _rows("v_pages", v_pages, device, (dt,), 4)
    if v_pages.shape != k_pages.shape:
        _bad(f"v_pages {tuple(v_pages.shape)} and k_pages {tuple(k_pages.shape)} differ in shape")
    n_pages, page, heads, dim = k_pages.shape
    tp = _ints("block_table", block_table, device, (None, None))
    return device, _lib.PagedCache(kp, vp, k_pages.stride()[:3], v_pages.stride()[:3], tp, block_table.stride(0), block_table.shape[0],
                                   block_table.shape[1], n_pages, page, heads, dim, _CODE[dt], device.index)


def paged_kv_append(k, v, k_pages, v_pages, block_table, positions, *, seq=None, q=None, q_out=None, rope=None):
    """Write the keys and values of new tokens into a paged cache, rotated to their positions on the way.

    k, v: [rows, kv_heads, head_dim], float32 or bfloat16.  k_pages, v_pages: [pages, page_size, kv_heads, head_dim] (float32 or
    bfloat16, any strides with a contiguous last dimension; page_size a power of two, head_dim 64 or 128).  block_table: int32
    [sequences, pages of a sequence].  Row r goes to position positions[r] (int32) of sequence seq[r] (None: sequence r); a row whose
    position is negative, past the tables, or on no page of the pool is skipped.  rope = (cos, sin), float32 [positions,
    >= head_dim / 2]: keys and queries are rotated by halves, (a, b) -> (a cos - b sin, b cos + a sin); None: not rotated.  q:
    [rows, heads, head_dim] of k's type; the rotated queries are returned (in q_out, which may be q), rows that were skipped are
    left as they were in q_out.  No two rows may name the same place of the cache."""
    device, cache = _cache(k_pages, v_pages, block_table)
    dt = k.dtype
    kp = _rows("k", k, device, _CODE, 3)
    vp = _rows("v", v, device, (dt,), 3)
    rows = k.shape[0]
    heads, dim = k_pages.shape[2:]
    if k.shape != v.shape or k.shape[1] != heads or k.shape[2] != dim:
        _bad(f"k {tuple(k.shape)} and v {tuple(v.shape)} must be [rows, {heads}, {dim}]")
    pp = _ints("positions", positions, device, (rows,))
    sp = _ints("seq", seq, device, (rows,))
    qp = op = cp = np_ = None
    qs = os = (0, 0)
    q_heads = rope_stride = rope_len = 0
    if q is not None:
        qp = _rows("q", q, device, (dt,), 3)
        if q.shape[0] != rows or q.shape[2] != dim:
            _bad(f"q {tuple(q.shape)} must be [{rows}, heads, {dim}]")
        q_heads = q.shape[1]
        if q_out is None:
            q_out = _torch.empty((rows, q_heads, dim), dtype=dt, device=device)
        elif q_out.shape != q.shape:
            _bad(f"q_out {tuple(q_out.shape)} must have q's shape {tuple(q.shape)}")
        op = _rows("q_out", q_out, device, (dt,), 3)
        qs, os = q.stride()[:2], q_out.stride()[:2]
    elif q_out is not None:
        _bad("q_out without q")
    if rope is not None:
        cos, sin = rope
        cp = _rows("cos", cos, device, (_F32,), 2)
        np_ = _rows("sin", sin, device, (_F32,), 2)
        if cos.shape != sin.shape or cos.stride() != sin.stride() or cos.shape[1] < dim // 2:
            _bad(f"cos {tuple(cos.shape)} and sin {tuple(sin.shape)} must be alike, [positions, >= {dim // 2}]")
        rope_stride, rope_len = cos.stride(0), cos.shape[0]
    args = _lib.AppendArgs(kp, vp, qp, op, k.stride()[:2], v.stride()[:2], qs, os, cp, np_, rope_stride, pp, sp, rows, q_heads, rope_len, _CODE[dt])
    rc = _lib.load().t3mi_paged_append(cache, args, _raw_stream(device.index))
    if rc:
        _lib.check(rc)
    return q_out


def paged_attention(q, k_pages, v_pages, block_table, lengths, *, seq=None, starts=None, scale: Optional[float] = None,
                    max_length: Optional[int] = None, out=None, out_dtype=None):
    """Attention of one new token per row over a paged cache: out[r, h] = sum_j softmax_j(scale q[r, h] . k_j) v_j over the keys
    j in [starts[r], lengths[r]) of sequence seq[r] (None: sequence r; starts None: 0).

    q: [rows, heads, head_dim], float32 (cache float32 or bfloat16) or bfloat16 (cache bfloat16); heads a multiple of the cache's,
    head h reads key head h // (heads // kv_heads).  Cache and block_table as in paged_kv_append; lengths, starts, seq: int32 [rows].
    scale: 1 / sqrt(head_dim) by default.  max_length: about the longest length, where the host knows it (the call is planned by it;
    rows that are longer come out right too).  A row with no key gives zeros; a row of negative length is left as it was in out.
    out: [rows, heads, head_dim], float32 or bfloat16 (new, in out_dtype or q's type, by default).  Many rows of one sequence
    (a prompt, causal) are rows with the same seq and lengths 1, 2, 3, ..."""
    device, cache = _cache(k_pages, v_pages, block_table)
    qp = _rows("q", q, device, _CODE, 3)
    rows, q_heads, dim = q.shape
    if dim != k_pages.shape[3]:
        _bad(f"q has head_dim {dim}, the cache {k_pages.shape[3]}")
    lp = _ints("lengths", lengths, device, (rows,))
    bp = _ints("starts", starts, device, (rows,))
    sp = _ints("seq", seq, device, (rows,))
    if out is None:
        out = _torch.empty((rows, q_heads, dim), dtype=out_dtype or q.dtype, device=device)
    elif out.shape != q.shape or (out_dtype is not None and out.dtype != out_dtype):
        _bad(f"out {tuple(out.shape)} {out.dtype} must have q's shape {tuple(q.shape)}, and out_dtype where that is given")
    op = _rows("out", out, device, _CODE, 3)
    args = _lib.AttentionArgs(qp, op, q.stride()[:2], out.stride()[:2], lp, bp, sp, None, 0, dim ** -0.5 if scale is None else scale, rows, q_heads,
                              _CODE[q.dtype], _CODE[out.dtype], 0, max_length or 0)
    lib = _lib.load()
    need = C.c_size_t(0)
    rc = lib.t3mi_paged_attention_workspace(cache, args, need)
    if rc:
        _lib.check(rc)
    if need.value:
        ws = _torch.empty(need.value, dtype=_torch.uint8, device=device)
        args.workspace, args.workspace_bytes = ws.data_ptr(), need.value
    rc = lib.t3mi_paged_attention(cache, args, _raw_stream(device.index))
    if rc:
        _lib.check(rc)
    return out


def _each(name: str, x, device, rows: int):
    """A penalty: one number, or a float32 tensor with one for every row -> (scalar, pointer)."""
    if isinstance(x, (int, float)):
        return float(x), None
    p = _rows(name, x, device, (_F32,), 1)
    if x.shape[0] != rows:
        _bad(f"{name} has {x.shape[0]} entries for {rows} rows")
    return 1.0, p


def process_logits(logits, *, uncond=None, cfg_weight: float = 0.0, tokens=None, n_tokens=None, repetition_penalty=1.0,
                   frequency_penalty=0.0, presence_penalty=0.0, bias_ids=None, bias_values=None, allowed=None, out=None):
    """The rules on logits [rows, vocab] (float32 or bfloat16), row by row in this order, in float32:

    guidance with `uncond` (rows of the unconditional pass): z = l + cfg_weight (l - u);
    biases: bias_values[r, i] is added to token bias_ids[r, i] (a token named twice takes the last; ids outside the vocabulary name none);
    penalties over the tokens so far, tokens[r, :n_tokens[r]] (int32): z / repetition if z > 0 else z * repetition for a token that
    occurs, then z - frequency * occurrences - presence (each penalty a number, or float32 [rows]);
    allowed: bit t % 32 of allowed[r, t // 32] (int32 words) is 0: z = -inf, whatever it was.

    bias_ids / bias_values [rows or 1, n] and allowed [rows or 1, words]: one row serves all.  A row that allows nothing is all -inf.
    Returns out (new by default; may be logits itself)."""
    if _torch is None:
        _setup()
    device = logits.device
    if device.type != "cuda":
        _bad(f"logits is on {device}: the operators run on the GPU")
    dt = logits.dtype
    lp = _rows("logits", logits, device, _CODE, 2)
    rows, vocab = logits.shape
    up, us = None, 0
    if uncond is not None:
        up, us = _rows("uncond", uncond, device, (dt,), 2), uncond.stride(0)
        if uncond.shape != logits.shape:
            _bad(f"uncond {tuple(uncond.shape)} must have the shape of logits {tuple(logits.shape)}")
    if out is None:
        out = _torch.empty((rows, vocab), dtype=dt, device=device)
    elif out.shape != logits.shape:
        _bad(f"out {tuple(out.shape)} must have the shape of logits {tuple(logits.shape)}")
    op = _rows("out", out, device, (dt,), 2)
    tp = np_ = None
    ts = cap = 0
    if (tokens is None) != (n_tokens is None):
        _bad("tokens and n_tokens go together")
    if tokens is not None:
        tp, np_ = _ints("tokens", tokens, device, (rows, None)), _ints("n_tokens", n_tokens, device, (rows,))
        ts, cap = tokens.stride(0), tokens.shape[1]
    rep, rp = _each("repetition_penalty", repetition_penalty, device, rows)
    fre, fp = _each("frequency_penalty", frequency_penalty, device, rows)
    pre, pp = _each("presence_penalty", presence_penalty, device, rows)
    ip = vp = ap = None
    n_bias = bis = bvs = als = 0
    if (bias_ids is None) != (bias_values is None):
        _bad("bias_ids and bias_values go together")
    if bias_ids is not None:
        ip, vp = _ints("bias_ids", bias_ids, device, (None, None)), _rows("bias_values", bias_values, device, (_F32,), 2)
        if bias_ids.shape != bias_values.shape or bias_ids.shape[0] not in (1, rows):
            _bad(f"bias_ids {tuple(bias_ids.shape)} and bias_values {tuple(bias_values.shape)} must be [{rows} or 1, n]")
        n_bias = bias_ids.shape[1]
        if bias_ids.shape[0] > 1:
            bis, bvs = bias_ids.stride(0), bias_values.stride(0)
    if allowed is not None:
        ap = _ints("allowed", allowed, device, (None, None))
        if allowed.shape[0] not in (1, rows) or allowed.shape[1] < (vocab + 31) // 32:
            _bad(f"allowed {tuple(allowed.shape)} must be [{rows} or 1, >= {(vocab + 31) // 32}]")
        als = allowed.stride(0) if allowed.shape[0] > 1 else 0
    args = _lib.LogitsArgs(lp, up, op, logits.stride(0), us, out.stride(0), tp, np_, ts, rp, fp, pp, ip, vp, bis, bvs, ap, als, cfg_weight, rep, fre,
                           pre, rows, vocab, _CODE[dt], cap, n_bias, device.index)
    rc = _lib.load().t3mi_process_logits(args, _raw_stream(device.index))
    if rc:
        _lib.check(rc)
    return out
