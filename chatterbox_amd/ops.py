"""Serving operators on torch tensors resident on the GPU: a key-value cache in pages (append, attention) and the rules a
logits row goes through before it is sampled.  A thin layer over the C entry points t3mi_paged_append, t3mi_paged_attention and
t3mi_process_logits (include/t3mi.h), for serving loops of one's own; the sessions of this package call the same kernels
(T3Model.set_paged_kv, T3Model.set_logit_rules).  The reference has no counterpart: its caches are contiguous
(R/llama_traced.R:274-297) and its sampling tail knows the repetition penalty alone (R/t3.R:529-537).

The calls enqueue on torch's current stream of the tensors' device and return; they may be captured into a graph.  Results and
workspaces are torch allocations of that stream.  There is no backward pass and no forward-mode gradient: inputs that ask for either are refused.
torch is imported by the first call, not with the package."""
from __future__ import annotations

import ctypes as C
from typing import Optional

from . import _lib

__all__ = ["paged_kv_append", "paged_attention", "process_logits"]

_ops = None


def _bind():
    """The compiled half of this module (csrc/py_ops.c: tensors to structs), bound to the library and to torch at the first call."""
    global _ops
    import torch
    from torch.autograd import forward_ad
    try:
        from . import _ops as ext
    except ImportError as e:
        raise ImportError("chatterbox_amd/_ops is missing: build it with `make -C chatterbox_amd/csrc`") from e
    lib = _lib.load()
    entry = [C.cast(getattr(lib, n), C.c_void_p).value
             for n in ("t3mi_paged_append", "t3mi_paged_attention_workspace", "t3mi_paged_attention", "t3mi_process_logits")]
    # the raw handle of torch's current stream; the spelled-out way where this torch has no short one
    stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)
    ext.bind(*entry, torch.float32, torch.bfloat16, torch.int32, torch.empty, torch.empty_like, stream, torch.is_grad_enabled, _lib.check,
             forward_ad, forward_ad.unpack_dual, torch.Tensor, getattr(torch.Tensor, "__dlpack_c_exchange_api__", None))
    _ops = ext
    return ext


def paged_kv_append(k, v, k_pages, v_pages, block_table, positions, *, seq=None, q=None, q_out=None, rope=None):
    """Write the keys and values of new tokens into a paged cache, rotated to their positions on the way.

    k, v: [rows, kv_heads, head_dim], float32 or bfloat16.  k_pages, v_pages: [pages, page_size, kv_heads, head_dim] (float32 or
    bfloat16, any strides with a contiguous last dimension; page_size a power of two, head_dim 64 or 128).  block_table: int32
    [sequences, pages of a sequence].  Row r goes to position positions[r] (int32) of sequence seq[r] (None: sequence r); a row whose
    position is negative, past the tables, or on no page of the pool is skipped.  rope = (cos, sin), float32 [positions,
    >= head_dim / 2]: keys and queries are rotated by halves, (a, b) -> (a cos - b sin, b cos + a sin); None: not rotated.  q:
    [rows, heads, head_dim] of k's type; the rotated queries are returned (in q_out, which may be q and shares no memory with q, k or v
    otherwise), rows that were skipped are left as they were in q_out.  No two rows may name the same place of the cache."""
    cos, sin = (None, None) if rope is None else rope
    return (_ops or _bind()).append(k, v, k_pages, v_pages, block_table, positions, seq, q, q_out, cos, sin)


def paged_attention(q, k_pages, v_pages, block_table, lengths, *, seq=None, starts=None, scale: Optional[float] = None,
                    max_length: Optional[int] = None, out=None, out_dtype=None, prompt: Optional[bool] = None):
    """Attention of one new token per row over a paged cache: out[r, h] = sum_j softmax_j(scale q[r, h] . k_j) v_j over the keys
    j in [starts[r], lengths[r]) of sequence seq[r] (None: sequence r; starts None: 0).

    q: [rows, heads, head_dim], float32 (cache float32 or bfloat16) or bfloat16 (cache bfloat16); heads a multiple of the cache's,
    head h reads key head h // (heads // kv_heads).  Cache and block_table as in paged_kv_append; lengths, starts, seq: int32 [rows].
    scale: 1 / sqrt(head_dim) by default.  max_length: about the longest length, where the host knows it (the call is planned by it;
    rows that are longer come out right too; with starts, about the most keys a row sees).  A row with no key, or whose scores are all
    -inf, gives zeros; a row of negative length is left as it was in out.
    out: [rows, heads, head_dim], float32 or bfloat16 (new, in out_dtype or q's type, by default; may be q, and shares no memory with it
    otherwise).  Many rows of one sequence (a prompt, causal) are rows with the same seq and lengths 1, 2, 3, ...; prompt says whether
    neighbouring rows mostly share a sequence: such rows share the keys they read where there are enough of them for that to pay (None:
    four rows to a sequence of the table, and more of them, since their order is not known; the results are the same up to rounding)."""
    return (_ops or _bind()).attention(q, k_pages, v_pages, block_table, lengths, seq, starts, scale, max_length or 0, out, out_dtype,
                                       0 if prompt is None else 1 if prompt else -1)


def process_logits(logits, *, uncond=None, cfg_weight: float = 0.0, tokens=None, n_tokens=None, repetition_penalty=1.0,
                   frequency_penalty=0.0, presence_penalty=0.0, bias_ids=None, bias_values=None, allowed=None, out=None):
    """The rules on logits [rows, vocab] (float32 or bfloat16), row by row in this order, in float32:

    guidance with `uncond` (rows of the unconditional pass): z = l + cfg_weight (l - u);
    biases: bias_values[r, i] is added to token bias_ids[r, i] (a token named twice takes the last; ids outside the vocabulary name none);
    penalties over the tokens so far, tokens[r, :n_tokens[r]] (int32): z / repetition if z > 0 else z * repetition for a token that
    occurs, then z - frequency * occurrences - presence (each penalty a number, or float32 [rows]);
    allowed: bit t % 32 of allowed[r, t // 32] (int32 words) is 0: z = -inf, whatever it was.

    bias_ids / bias_values [rows or 1, n] and allowed [rows or 1, words]: one row serves all.  A row that allows nothing is all -inf.
    Returns out (new by default; may be logits itself, and shares memory with no other argument)."""
    return (_ops or _bind()).logits(logits, uncond, cfg_weight, tokens, n_tokens, repetition_penalty, frequency_penalty, presence_penalty,
                                    bias_ids, bias_values, allowed, out)
