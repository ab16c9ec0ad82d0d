"""bread_spec_verify with 32 logits a thread (chunks of 8192) and with 8 (chunks of 2048), every type of logits with
and without draft probabilities, vocabularies around a chunk's borders.  A round takes the small chunks up to 16384
of them in all, where a row has at most 2048."""
import numpy as np
import pytest

from test_gpu_spec_verify import check, round_of

pytestmark = pytest.mark.gpu
TEMP = np.array([0.0, 0.7, 1.3, -1.0, 2.0, 0.01, 60.0])


def many(V):
    """Requests with 0 to 12 drafts, rows enough for the large chunks."""
    rows = 16384 // -(-V // 2048) + 1
    counts = []
    while sum(counts) + len(counts) < rows:
        counts += [4, 0, 7, 1, 12]
    return counts


@pytest.mark.parametrize("half", [True, False], ids=["f16", "f32"])
@pytest.mark.parametrize("probs", [True, False], ids=["model", "lookup"])
@pytest.mark.parametrize("V", [100, 8191, 8192, 8193, 24653])
def test_large_chunks(V, probs, half):
    counts = many(V)
    z, tokens, off, u, q = round_of(counts, V, 7 * V, half, probs)
    assert len(tokens) * -(-V // 2048) > 16384
    z[3, : V // 2] = -np.inf
    z[9, 5:] = -np.inf
    z[11] = np.finfo(z.dtype).min
    z[15, V - 1] = np.inf
    z[17] = np.nan
    check(z, tokens, off, u, q, temp=np.resize(TEMP, len(counts)), eos=int(tokens[-1]))


@pytest.mark.parametrize("half", [True, False], ids=["f16", "f32"])
@pytest.mark.parametrize("probs", [True, False], ids=["model", "lookup"])
def test_the_last_small_chunks_and_the_first_large_ones(probs, half):
    """16384 small chunks, and one request more."""
    for n, small in ((1024, True), (1025, False)):
        z, tokens, off, u, q = round_of([3] * n, 7000, n, half, probs)
        assert (len(tokens) * 4 <= 16384) == small
        check(z, tokens, off, u, q, temp=np.resize(TEMP, n))


@pytest.mark.parametrize("counts,probs", [([0], False), ([1], True)])
def test_a_row_of_more_small_chunks_than_a_workgroup_holds(counts, probs):
    V = 2048 * 2048 + 777
    z, tokens, off, u, q = round_of(counts, V, 5, True, probs)
    check(z, tokens, off, u, q)
    u[-1] = np.float32(1) - np.float32(2.0 ** -24)
    u[0] = u[-1]
    check(z, tokens, off, u, q, temp=[1.5])
