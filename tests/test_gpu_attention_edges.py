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
@pytest.mark.parametrize("prompt,heads,kv_heads,dim,page", [(False, 16, 16, 64, 64), (False, 32, 8, 128, 16), (False, 6, 2, 64, 2), (True, 8, 2, 128, 64), (True, 4, 4, 64, 8)])
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
