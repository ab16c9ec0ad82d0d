"""bread_spec_verify: a signalling NaN logit counts as -inf, as any other NaN.

Which bits a NaN has is left to whoever wrote it; the rows below hold both kinds next to the largest logit, in
its place, in whole chunks and at drafts, for every number of logits a thread takes.
"""
import numpy as np
import pytest

from test_gpu_spec_verify import check, round_of

pytestmark = pytest.mark.gpu
SIGNALLING = {np.float16: [0x7C01, 0x7DFF, 0xFC01, 0xFDFF], np.float32: [0x7F800001, 0x7FBFFFFF, 0xFF800001, 0xFFBFFFFF]}


def plant(z, kind, rng):
    """NaN bits, by row: around the largest, alternating with everything, all but one, a few here and there."""
    bits = z.view({np.float16: np.uint16, np.float32: np.uint32}[kind])
    nan = np.array(SIGNALLING[kind] + [0x7E00 if kind is np.float16 else 0x7FC00000], bits.dtype)
    V = z.shape[1]
    for r in range(len(z)):
        top = int(np.argmax(z[r]))
        if r % 4 == 0:
            at = np.arange(max(0, top - 70), min(V, top + 71))
        elif r % 4 == 1:
            at = np.arange((top + 1) % 2, V, 2)
        elif r % 4 == 2:
            at = np.arange(V)
        else:
            at = rng.integers(0, V, 20)
        at = at[at != top]
        bits[r, at] = nan[rng.integers(0, len(nan), len(at))]
    assert np.isnan(z).any()


@pytest.mark.parametrize("kind", [np.float16, np.float32], ids=["f16", "f32"])
@pytest.mark.parametrize("probs", [True, False], ids=["model", "lookup"])
@pytest.mark.parametrize("V", [40, 2048, 8292])
def test_signalling_nan_is_minus_infinity(V, probs, kind):
    for seed, counts in enumerate(([0], [3, 0, 5], [7, 7])):
        rng = np.random.default_rng(seed)
        z, tokens, off, u, q = round_of(counts, V, 40 * V + seed, kind is np.float16, probs)
        plant(z, kind, rng)
        if seed == 2:
            z[4] = np.nan  # a row of nothing
        check(z, tokens, off, u, q)
        check(z, tokens, off, u, q, temp=np.array([0.7, 0.0, 40.0])[: len(counts)], eos=int(tokens[-1]))


def test_signalling_nan_in_large_chunks():
    """Rows enough for 32 logits a thread."""
    for kind in (np.float16, np.float32):
        rng = np.random.default_rng(3)
        z, tokens, off, u, _ = round_of([4] * 700, 9000, 77, kind is np.float16, False)
        assert len(z) * -(-9000 // 2048) > 16384
        plant(z, kind, rng)
        check(z, tokens, off, u, temp=np.tile([0.7, 0.0, 40.0, 1.0, 1.3], 140))
