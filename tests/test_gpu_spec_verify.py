"""bread_spec_verify against the definition in 64 bits, request by request.

Accepted counts and tokens are compared exactly: both sides hold probabilities
and sums in 64 bits, so that a uniform number would have to fall within 1e-13
of a border to tell them apart.  Log-probabilities are computed in 64 bits and
rounded once: 2^-24 of themselves, plus 1e-12 for the 64-bit sums.
"""
import numpy as np
import pytest
import torch

import breadv2_amd as B
from breadv2_amd import api

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
CHUNK = 8192  # logits a workgroup


def target(z, t):
    """(p, log p) of a row; log p at temperature 1 for greedy."""
    z = np.where(np.isnan(z), -np.inf, z.astype(np.float64))
    m = z.max()
    if m == -np.inf:
        return np.zeros_like(z), np.full_like(z, -np.inf)
    with np.errstate(invalid="ignore"):
        d = np.where(z == m, 0.0, np.where(z == -np.inf, -np.inf, (z - m) / (t if t > 0 else 1.0)))
    d = np.where((z == -np.inf) | ((m == np.inf) & (z != m)), -np.inf, d)
    e = np.exp(d)
    logp = d - np.log(e.sum())
    if not t > 0:
        p = np.zeros_like(z)
        p[int(np.argmax(z == m))] = 1.0
        return p, logp
    return e / e.sum(), logp


def plain(z, tokens, off, u, q=None, temp=None, eos=-1):
    nb = len(off) - 1
    n_acc, nxt, lp = np.zeros(nb, np.int32), np.zeros(nb, np.int32), np.zeros(len(tokens))
    for b in range(nb):
        t = 1.0 if temp is None else float(temp[b])
        stop = None
        for r in range(off[b], off[b + 1]):
            p, logp = target(z[r], t)
            if r + 1 == off[b + 1]:
                if stop is None:
                    stop = (r, p, logp, np.zeros_like(p), None)
                break
            d = int(tokens[r + 1])
            ok_id = 0 <= d < z.shape[1]
            lp[r] = logp[d] if ok_id else -np.inf
            if stop is not None:
                continue
            if q is None:
                qr = np.zeros_like(p)
                if ok_id:
                    qr[d] = 1.0
            else:
                qr = q[r - b].astype(np.float64)
                qr = np.where(qr > 0, qr, 0.0)
            qd = (qr[d] if q is not None else 1.0) if ok_id else 1.0
            stands = float(np.float64(u[r])) * qd < (p[d] if ok_id else 0.0)
            if not stands:
                stop = (r, p, logp, qr, None)
            elif d == eos:
                stop = (r, p, logp, None, d)
        r, p, logp, qr, end = stop
        n_acc[b] = r - off[b]
        if end is not None:
            nxt[b] = end
        elif p.sum() > 0:
            w = np.maximum(p - qr, 0.0)
            if not w.sum() > 0:
                w = p
            cum = np.cumsum(w)
            hit = np.nonzero(cum > float(np.float64(u[off[b + 1] - 1])) * cum[-1])[0]
            nxt[b] = hit[0] if len(hit) else np.nonzero(w > 0)[0][-1]
        lp[off[b + 1] - 1] = logp[nxt[b]]
    return n_acc, nxt, lp


def dev(a):
    return None if a is None else torch.from_numpy(np.ascontiguousarray(a)).to(DEV)


CTX = {}


def context(rows):
    n = max(64, rows)
    if n not in CTX:
        CTX[n] = B.MoeContext(B.shape(), max_tokens=n)
    return CTX[n]


def check(z, tokens, off, u, q=None, temp=None, eos=-1):
    ctx = context(len(tokens))
    a, n, lp = ctx.spec_verify(dev(z), dev(np.asarray(tokens, np.int32)), dev(np.asarray(off, np.int32)),
                               dev(np.asarray(u, np.float32)), draft_probs=dev(q),
                               temperature=dev(None if temp is None else np.asarray(temp, np.float32)), eos=eos)
    torch.cuda.synchronize()
    assert ctx.check_device() == 0
    ra, rn, rl = plain(z, tokens, off, np.asarray(u, np.float32), q, None if temp is None else np.asarray(temp, np.float32), eos)
    assert np.array_equal(a.cpu().numpy(), ra), (a.cpu().numpy(), ra)
    assert np.array_equal(n.cpu().numpy(), rn), (n.cpu().numpy(), rn)
    got = lp.cpu().numpy().astype(np.float64)
    fin = np.isfinite(rl)
    assert np.array_equal(fin, np.isfinite(got)) and np.all(got[~fin] == rl[~fin])
    assert np.all(np.abs(got[fin] - rl[fin]) <= 2.0 ** -24 * np.abs(rl[fin]) + 1e-12)
    return ra, rn


def softmax(z):
    e = np.exp(z - z.max(1, keepdims=True))
    return e / e.sum(1, keepdims=True)


def round_of(counts, V, seed, half=True, probs=True, spread=3.0):
    """Logits of a target, and drafts drawn from a noisy copy of it (or likely tokens without probabilities)."""
    rng = np.random.default_rng(seed)
    off = np.concatenate([[0], np.cumsum(np.asarray(counts) + 1)])
    R, nb = int(off[-1]), len(counts)
    z = (spread * rng.standard_normal((R, V))).astype(np.float16 if half else np.float32)
    tokens = rng.integers(0, V, R)
    q = np.zeros((R - nb, V), np.float32) if probs else None
    for b in range(nb):
        for r in range(off[b], off[b + 1] - 1):
            if probs:
                q[r - b] = softmax((0.9 * z[r] + 0.5 * rng.standard_normal(V))[None].astype(np.float64))[0]
                tokens[r + 1] = rng.choice(V, p=q[r - b].astype(np.float64) / q[r - b].astype(np.float64).sum())
            else:
                tokens[r + 1] = np.argmax(z[r]) if rng.random() < 0.7 else rng.integers(0, V)
    return z, tokens, off, rng.random(R).astype(np.float32), q


@pytest.mark.parametrize("half", [True, False], ids=["f16", "f32"])
@pytest.mark.parametrize("probs", [True, False], ids=["model", "lookup"])
@pytest.mark.parametrize("V", [1, 2, 7, 255, 1000, CHUNK - 1, CHUNK, CHUNK + 1, 3 * CHUNK + 77])
def test_rounds(V, probs, half):
    for seed, counts in enumerate(([0], [1], [4], [0, 3, 0, 1, 6], [2] * 9, [9, 0, 0])):
        z, tokens, off, u, q = round_of(counts, V, 31 * V + seed, half, probs)
        check(z, tokens, off, u, q)
        temp = np.array([0.0, 0.7, 1.3, -1.0, 2.0] * 4)[: len(counts)]
        check(z, tokens, off, u, q, temp=temp, eos=int(tokens[-1]))


def test_many_requests():
    counts = np.random.default_rng(0).integers(0, 9, 150)
    z, tokens, off, u, q = round_of(counts, 300, 5)
    check(z, tokens, off, u, q, temp=np.linspace(0.3, 2.0, 150), eos=7)


def test_long_drafts():
    """More rows in one request than the workgroup has waves, several times over."""
    z, tokens, off, u, _ = round_of([100, 3], 500, 6, probs=False)
    for r in range(100):
        tokens[r + 1] = int(np.argmax(z[r]))
        z[r, tokens[r + 1]] = 60.0
    ra, _ = check(z, tokens, off, u)
    assert ra[0] == 100


@pytest.mark.parametrize("half", [True, False], ids=["f16", "f32"])
@pytest.mark.parametrize("probs", [True, False], ids=["model", "lookup"])
def test_enough_rows_for_the_large_chunks(probs, half):
    counts = [4, 0, 7, 1, 12] * 7
    z, tokens, off, u, q = round_of(counts, 3 * CHUNK + 77, 61, half, probs)
    assert len(tokens) * (3 * CHUNK + 77) > 2048 * 2048
    temp = np.array([0.0, 0.7, 1.3, -1.0, 2.0, 0.01, 60.0] * 5)
    z[3, :CHUNK] = -np.inf
    z[9, 5:] = -np.inf
    check(z, tokens, off, u, q)
    check(z, tokens, off, u, q, temp=temp, eos=int(tokens[-1]))


@pytest.mark.parametrize("probs,half", [(True, False), (False, True)], ids=["model-f32", "lookup-f16"])
def test_many_rows_of_several_large_chunks(probs, half):
    counts = [4, 0, 7, 1, 12] * 46
    V = 3 * CHUNK + 77
    z, tokens, off, u, q = round_of(counts, V, 63, half, probs)
    assert len(tokens) * -(-V // 2048) > 16384
    temp = np.array([0.0, 0.7, 1.3, -1.0, 2.0, 0.01, 60.0] * 33)[: len(counts)]
    z[3, :CHUNK] = -np.inf
    z[9, 5:] = -np.inf
    check(z, tokens, off, u, q, temp=temp, eos=int(tokens[-1]))


@pytest.mark.parametrize("V,counts", [(300_001, [0, 2]), (1_100_000, [4])])
def test_more_chunks_than_two_a_lane(V, counts):
    z, tokens, off, u, _ = round_of(counts, V, 62, probs=False)
    check(z, tokens, off, u, temp=[0.9, 1.1][: len(counts)])


@pytest.mark.parametrize("V", [50, 2 * CHUNK + 5])
def test_greedy_is_spec_accept(V):
    """Temperature 0 gives bread_spec_accept's count and token on the rows' greedy predictions."""
    rng = np.random.default_rng(V)
    for seed in range(20):
        n = int(rng.integers(0, 7))
        z = rng.integers(-3, 3, (n + 1, V)).astype(np.float16)  # many equal logits
        pred = list(np.argmax(z, 1))
        draft = [int(pred[i]) if rng.random() < 0.8 else int(rng.integers(0, V)) for i in range(n)]
        eos = int(pred[n // 2]) if seed % 3 == 0 else -1
        ra, rn = check(z, [0] + draft, [0, n + 1], rng.random(n + 1), temp=[0.0], eos=eos)
        want = B.spec_accept([int(p) for p in pred], draft, eos, n + 1)
        assert (int(ra[0]), int(rn[0])) == want


def test_equal_models_accept_everything():
    """p = q: u q < p for every u < 1 (q rounded down to fp32)."""
    V = 4096
    rng = np.random.default_rng(3)
    z = rng.standard_normal((6, V)).astype(np.float32)
    p = np.array([target(r, 1.0)[0] for r in z])
    q = np.nextafter(p.astype(np.float32), np.float32(0))[:5]
    u = np.full(6, np.float32(1) - np.float32(2.0 ** -24), np.float32)
    ra, _ = check(z, rng.integers(0, V, 6), [0, 6], u, q)
    assert ra[0] == 5


def test_uniforms_at_their_ends():
    z, tokens, off, u, q = round_of([3, 3, 3, 3], 9000, 8)
    top = np.float32(1) - np.float32(2.0 ** -24)
    for lo in (np.float32(0), np.float32(1e-30), top):
        for final in (np.float32(0), top):
            v = np.full(len(u), lo, np.float32)
            v[off[1:] - 1] = final
            check(z, tokens, off, v, q)


def test_every_token_can_be_drawn():
    """Uniform numbers over [0, 1) in even steps draw each token as often as its weight says."""
    V, n = 64, 4096
    z = np.tile(np.random.default_rng(4).standard_normal((1, V)).astype(np.float16), (n, 1))
    u = ((np.arange(n) + 0.5) / n).astype(np.float32)
    _, rn = check(z, np.zeros(n, np.int32), np.arange(n + 1), u)
    p = target(z[0], 1.0)[0]
    assert np.all(np.abs(np.bincount(rn, minlength=V) - n * p) <= 1.0 + 1e-6)


def test_masked_rows():
    """-inf masks, a row of nothing, NaN, the type's lowest value, +inf, for both types."""
    inf = np.inf
    for kind in (np.float16, np.float32):
        V = CHUNK + 100
        rng = np.random.default_rng(9)
        z = rng.standard_normal((14, V)).astype(kind)
        z[0] = -inf
        z[2, :CHUNK] = -inf                    # a whole chunk masked
        z[4, 1:] = -inf                        # one token left
        z[6, :] = np.nan
        z[6, 77] = 1.0
        z[8] = np.finfo(kind).min
        z[8, 5] = 0.0
        z[10, [3, CHUNK + 3]] = inf
        z[12] = np.finfo(kind).min             # nothing but the lowest value: an even row
        off = np.arange(0, 15, 2)
        tokens = np.zeros(14, np.int32)
        tokens[1::2] = [0, CHUNK + 5, 0, 77, 5, 3, 9]
        for temp in (None, [0.5] * 7, [0.0] * 7, [1e30] * 7, [inf] * 7, [1e-30] * 7):
            check(z, tokens, off, rng.random(14), temp=temp)
        q = np.zeros((7, V), np.float32)
        q[:, :10] = 0.1
        check(z, tokens, off, rng.random(14), q)


def test_drafts_and_probabilities_out_of_the_ordinary():
    z, tokens, off, u, q = round_of([2, 2, 2, 2, 2], 1000, 11)
    tokens[1], tokens[4], tokens[8] = -1, 1000, 2 ** 30     # no tokens: they fall
    q[3, int(tokens[5])] = 0.0                              # a draft its model would not draw
    q[6] = np.nan
    q[7] = -1.0
    check(z, tokens, off, u, q)
    check(z, tokens, off, u)


def test_draft_probabilities_that_cover_the_targets():
    """Nothing is left over: the token comes from p itself."""
    z = np.zeros((2, 500), np.float32)
    q = np.full((1, 500), 1.0, np.float32)
    ra, rn = check(z, [0, 9], [0, 2], [0.9, 0.5], q)
    assert ra[0] == 0 and rn[0] == 250


def test_strided_rows_and_no_logprob():
    z, tokens, off, u, q = round_of([2, 0, 3], 777, 12)
    wide = torch.zeros(len(tokens), 1001, dtype=torch.float16, device=DEV)
    wide[:, 3:780] = dev(z)
    wq = torch.zeros(q.shape[0], 900, device=DEV)
    wq[:, 100:877] = dev(q)
    ctx = context(16)
    args = (dev(tokens.astype(np.int32)), dev(off.astype(np.int32)), dev(u))
    a, n, lp = ctx.spec_verify(wide[:, 3:780], *args, draft_probs=wq[:, 100:877], want_logprob=False)
    ra, rn, _ = plain(z, tokens, off, u, q)
    assert lp is None and np.array_equal(a.cpu().numpy(), ra) and np.array_equal(n.cpu().numpy(), rn)


def test_offsets_that_do_not_fit_are_flagged():
    z, tokens, off, u, q = round_of([2, 2], 400, 13)
    ctx = B.MoeContext(B.shape(), max_tokens=8)
    for bad in ([0, 3, 7], [0, 0, 6], [3, 1, 6], [0, -5, 6], [-1, 3, 6], [0, 2 ** 31 - 1, 6], [0, 6, 6]):
        a, n, _ = ctx.spec_verify(dev(z), dev(tokens.astype(np.int32)), dev(np.asarray(bad, np.int32)), dev(u),
                                  draft_probs=dev(q))
        with pytest.raises(B.BreadError) as e:
            ctx.check_device()
        assert e.value.device_error == 64, bad
    a, n, _ = ctx.spec_verify(dev(z), dev(tokens.astype(np.int32)), dev(off.astype(np.int32)), dev(u), draft_probs=dev(q))
    assert ctx.check_device() == 0
    ra, rn, _ = plain(z, tokens, off, u, q)
    assert np.array_equal(a.cpu().numpy(), ra) and np.array_equal(n.cpu().numpy(), rn)


def test_refusals():
    ctx = B.MoeContext(api.shape(256, 256, 256, 8, 1), max_tokens=4)
    i = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    z = torch.zeros(5, 64, dtype=torch.float16, device=DEV)
    u = torch.zeros(5, device=DEV)
    with pytest.raises(B.BreadError) as e:  # more rows than the context holds
        ctx.spec_verify(z, i(0, 0, 0, 0, 0), i(0, 5), u)
    assert e.value.status == api._lib.ERR_CAPACITY
    with pytest.raises(B.BreadError) as e:  # a vocabulary too large for its scratch
        ctx.spec_verify(torch.zeros(4, 1 << 21, dtype=torch.float16, device=DEV), i(0, 0, 0, 0), i(0, 4), u[:4])
    assert e.value.status == api._lib.ERR_CAPACITY
    with pytest.raises(B.BreadError) as e:  # more requests than rows
        ctx.spec_verify(z[:2], i(0, 0), i(0, 1, 2, 3), u[:2])
    assert e.value.status == api._lib.ERR_ARG
    with pytest.raises(ValueError):
        ctx.spec_verify(z[:4].to(torch.bfloat16), i(0, 0, 0, 0), i(0, 4), u[:4])
    with pytest.raises(ValueError):
        ctx.spec_verify(z[:4], i(0, 0, 0, 0).long(), i(0, 4), u[:4])
    with pytest.raises(ValueError):
        ctx.spec_verify(z[:4], i(0, 0, 0, 0), i(0, 4), u[:4], draft_probs=torch.zeros(2, 64, device=DEV))
    with pytest.raises(ValueError):
        ctx.spec_verify(z[:4], i(0, 0, 0, 0).cpu(), i(0, 4), u[:4])
    a, n, lp = ctx.spec_verify(z[:0], i(), i(0), u[:0])
    assert a.numel() == 0 and lp.numel() == 0


def test_repeats_stream_and_graph():
    """The same answers call after call, on another stream, and from a graph replayed between other calls of the context."""
    z, tokens, off, u, q = round_of([3, 0, 5, 1], 3 * CHUNK + 9, 14)
    ctx = B.MoeContext(B.shape(), max_tokens=16)
    args = [dev(z), dev(tokens.astype(np.int32)), dev(off.astype(np.int32)), dev(u)]
    qd = dev(q)
    ra, rn, _ = plain(z, tokens, off, u, q)
    for _ in range(5):
        a, n, _ = ctx.spec_verify(*args, draft_probs=qd)
        assert np.array_equal(a.cpu().numpy(), ra) and np.array_equal(n.cpu().numpy(), rn)
    s = torch.cuda.Stream()
    a, n, _ = ctx.spec_verify(*args, draft_probs=qd, stream=s)
    s.synchronize()
    assert np.array_equal(a.cpu().numpy(), ra) and np.array_equal(n.cpu().numpy(), rn)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        a, n, lp = ctx.spec_verify(*args, draft_probs=qd)
    rng = np.random.default_rng(0)
    for k in range(4):
        v = rng.random(len(u)).astype(np.float32)
        args[3].copy_(dev(v))
        g.replay()
        torch.cuda.synchronize()
        ra, rn, _ = plain(z, tokens, off, v, q)
        assert np.array_equal(a.cpu().numpy(), ra) and np.array_equal(n.cpu().numpy(), rn)
        a2, n2, _ = ctx.spec_verify(*args, draft_probs=qd)
        assert torch.equal(a, a2) and torch.equal(n, n2)
