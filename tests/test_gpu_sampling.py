"""Probabilities of logits and the verification of drafted tokens against plain 64-bit forms."""
from __future__ import annotations

import numpy as np
import pytest

import qraf_b200 as qb

pytestmark = pytest.mark.gpu


def _tensor(a, cuda):
    import torch

    return torch.from_numpy(np.ascontiguousarray(a)).to(cuda)


# ── probabilities ───────────────────────────────────────────────────────────
def probs64(x, temperature):
    """(probabilities, tolerance).  The argument (x - max) / T is rounded three times
    (difference, factor, product), 2^-24 of itself each, exp2 is within 2^-22, the sum of
    n terms in strips and trees within 64 of its last bits, the division and product one each."""
    x = np.asarray(x, np.float64)
    m = x.max(-1, keepdims=True)
    a = (x - np.where(np.isinf(m), 0, m)) / temperature
    e = np.exp(a)
    l = e.sum(-1, keepdims=True)
    p = e / np.where(l == 0, 1, l)
    reach = np.where(e > 0, np.abs(a), 0.0)
    mean = (p * reach).sum(-1, keepdims=True)
    return p, p * ((reach + mean) * 4 * 2.0 ** -24 + 2.0 ** -21 + 66 * 2.0 ** -24) + 2.0 ** -126


def _near(got, want, tol):
    bad = ~(np.abs(got.cpu().numpy().astype(np.float64) - want) <= tol)
    assert not bad.any(), f"{int(bad.sum())} values off"


@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (5, 17), (2, 511), (7, 4097), (160, 2049), (3, 32003), (2, 151936),
                                        (300, 16385), (1, 262147), (2, 500009)])
@pytest.mark.parametrize("temperature", [1.0, 0.35])
def test_token_probs(cuda, rows, vocab, temperature):
    """Vocabularies that end inside every vector and slice, one that no cluster keeps on chip."""
    x = np.random.default_rng(vocab).standard_normal((rows, vocab)).astype(np.float32) * 4
    got = qb.token_probs(_tensor(x, cuda), temperature)
    _near(got, *probs64(x, np.float64(np.float32(temperature))))
    assert qb.device_status() == qb.OK


def test_token_probs_masks_and_infinities(cuda):
    """-inf is 0 and a row of it zeros; the type's lowest value is not -inf; NaN and +inf make
    their own row NaN and no other."""
    low = np.finfo(np.float32).min
    x = np.random.default_rng(1).standard_normal((6, 1000)).astype(np.float32)
    x[0, ::2] = -np.inf
    x[1] = -np.inf
    x[2] = low
    x[2, 5] = 0.0
    x[3] = low
    got = qb.token_probs(_tensor(x, cuda))
    _near(got, *probs64(x, 1.0))
    assert not got[1].any() and (got[3] == got[3, 0]).all() and got[2, 5] == 1.0
    x[4, 7], x[5, 9] = np.nan, np.inf
    got = qb.token_probs(_tensor(x, cuda)).cpu().numpy()
    assert np.isnan(got[4]).all() and np.isnan(got[5]).all() and not np.isnan(got[:4]).any()


def test_token_probs_strides_in_place_and_streams(cuda):
    import torch

    x = np.random.default_rng(2).standard_normal((9, 5003)).astype(np.float32)
    want, tol = probs64(x, 0.5)
    wide = torch.zeros(9, 6001, device=cuda)
    wide[:, 3:5006] = _tensor(x, cuda)
    out = torch.zeros(9, 5011, device=cuda)
    qb.token_probs(wide[:, 3:5006], 0.5, out=out[:, 1:5004])
    _near(out[:, 1:5004], want, tol)
    assert not out[:, 0].any() and not out[:, 5004:].any()
    y = _tensor(x, cuda)
    torch.cuda.synchronize()
    s = torch.cuda.Stream(cuda)
    assert qb.token_probs(y, 0.5, out=y, stream=s) is y
    s.synchronize()
    _near(y, want, tol)
    big = torch.randn(2, 450000, device=cuda)   # re-read path, in place
    want, tol = probs64(big.cpu().numpy(), 1.0)
    qb.token_probs(big, out=big)
    _near(big, want, tol)
    assert qb.token_probs(_tensor(x[0], cuda)).shape == (5003,)
    assert qb.token_probs(torch.zeros(0, 5, device=cuda)).shape == (0, 5)


# ── verification ────────────────────────────────────────────────────────────
def verify64(target, draft, tokens, u, u_last, counts=None):
    b, k = tokens.shape
    out, acc = np.full((b, k + 1), -1, np.int32), np.zeros(b, np.int32)
    for s in range(b):
        m = k if counts is None else int(counts[s])
        a = 0
        while a < m and float(u[s, a]) * float(draft[s, a, tokens[s, a]]) < float(target[s, a, tokens[s, a]]):
            out[s, a] = tokens[s, a]
            a += 1
        p = target[s, a].astype(np.float64)
        w = np.maximum(p - draft[s, a].astype(np.float64), 0) if a < m else p
        if w.sum() == 0:
            w = p
        c = np.cumsum(w)
        hit = np.nonzero(c > float(u_last[s]) * c[-1])[0]
        out[s, a] = hit[0] if len(hit) else np.nonzero(w > 0)[0][-1]
        acc[s] = a
    return out, acc


def _case(rng, b, k, vocab, sharp=2.0, near=0.7):
    def soft(x):
        e = np.exp(x - x.max(-1, keepdims=True))
        return (e / e.sum(-1, keepdims=True)).astype(np.float32)

    x = rng.standard_normal((b, k + 1, vocab)) * sharp
    draft, target = soft(x[:, :k]), soft(x + near * rng.standard_normal(x.shape))
    tokens = np.stack([[rng.choice(vocab, p=d.astype(np.float64) / d.astype(np.float64).sum()) for d in s] for s in draft]) \
        if k else np.zeros((b, 0))
    return target, draft, tokens.astype(np.int32).reshape(b, k), rng.random((b, k)).astype(np.float32), \
        rng.random(b).astype(np.float32)


def _run(cuda, case, counts=None):
    got = qb.verify_drafts(*(_tensor(a, cuda) for a in case), counts=None if counts is None else _tensor(counts, cuda))
    return [t.cpu().numpy() for t in got]


@pytest.mark.parametrize("b,k,vocab", [(1, 1, 1), (1, 1, 2), (5, 3, 17), (64, 8, 1000), (3, 4, 4099), (16, 5, 32003),
                                       (2, 2, 151936), (4, 0, 777), (2, 200, 300)])
def test_verify_drafts(cuda, b, k, vocab):
    case = _case(np.random.default_rng(vocab + k), b, k, vocab)
    want = verify64(*case)
    got = _run(cuda, case)
    assert np.array_equal(got[1], want[1]) and np.array_equal(got[0], want[0])
    if k:
        counts = np.random.default_rng(k).integers(0, k + 1, b).astype(np.int32)
        got, want = _run(cuda, case, counts), verify64(*case, counts)
        assert np.array_equal(got[1], want[1]) and np.array_equal(got[0], want[0])
    assert qb.device_status() == qb.OK


def test_verify_at_the_borders(cuda):
    """u of 0 and just below 1; drafts of probability 0 on either side; a residual that is zero
    everywhere (target below the draft in every rounding): the draw falls back to the target; all
    the weight on the first or last token."""
    v = 9000
    rng = np.random.default_rng(3)
    target, draft, tokens, u, u_last = _case(rng, 8, 2, v)
    one = np.float32(1) - np.float32(2.0 ** -24)
    u_last[:] = [0, one, 0.5, 0, one, 0.5, 0.25, one]
    u[:4] = one
    u[4:] = 0
    target[0, 0, tokens[0, 0]] = 0                      # never accepted
    draft[1, 0, tokens[1, 0]] = 0                       # accepted although the draft says never
    target[2, 0] = draft[2, 0] * np.float32(0.5)        # residual zero everywhere
    tokens[2, 0] = int(np.argmax(draft[2, 0]))
    target[3, 0] = 0
    target[3, 0, -1] = 1
    tokens[3, 0] = 4
    target[5, 2] = 0
    target[5, 2, 0] = 1
    target[6, 2] = 0
    target[6, 2, v - 1] = 1e-30
    case = target, draft, tokens, u, u_last
    want, got = verify64(*case), _run(cuda, case)
    assert np.array_equal(got[1], want[1]) and np.array_equal(got[0], want[0])
    u_last[:] = 1.0                                     # outside the range: the last token with any weight
    want, got = verify64(*case), _run(cuda, case)
    assert np.array_equal(got[0], want[0])
    assert qb.device_status() == qb.OK


def test_verify_padding_errors_and_strides(cuda):
    import torch

    rng = np.random.default_rng(4)
    case = _case(rng, 3, 2, 5001)
    want = verify64(*case)
    t, d, tok, u, ul = (_tensor(a, cuda) for a in case)
    wide_t, wide_d = torch.zeros(3, 4, 5010, device=cuda), torch.zeros(3, 2, 5003, device=cuda)
    wide_t[:, 1:, 7:5008] = t
    wide_d[:, :, 1:5002] = d
    got = qb.verify_drafts(wide_t[:, 1:, 7:5008], wide_d[:, :, 1:5002], tok, u, ul)
    assert np.array_equal(got[0].cpu().numpy(), want[0])
    # a padded sequence raises nothing and does not disturb the others
    out = qb.verify_drafts(t, d, tok, u, ul, counts=_tensor(np.array([2, -1, 2], np.int32), cuda))
    assert np.array_equal(out[0].cpu().numpy()[[0, 2]], want[0][[0, 2]]) and qb.device_status() == qb.OK
    # a token outside the vocabulary falls and raises the status
    bad = tok.clone()
    bad[1, 0] = 5001
    out = qb.verify_drafts(t, d, bad, u, ul)
    assert qb.device_status() == qb.ERR_INVALID and out[1][1] == 0
    assert np.array_equal(out[0].cpu().numpy()[[0, 2]], want[0][[0, 2]])
    # a count above the drafts is cut
    out = qb.verify_drafts(t, d, tok, u, ul, counts=_tensor(np.array([2, 2, 3], np.int32), cuda))
    assert qb.device_status() == qb.ERR_INVALID and np.array_equal(out[0].cpu().numpy(), want[0])
    # a row without any weight
    t[2] = 0
    out = qb.verify_drafts(t, d, tok, u, ul)
    assert qb.device_status() == qb.ERR_INVALID and out[0][2].tolist() == [-1, -1, -1] and out[1][2] == 0
    t[2] = float("nan")
    out = qb.verify_drafts(t, d, tok, u, ul)
    assert qb.device_status() == qb.ERR_INVALID and out[0][2].tolist() == [-1, -1, -1]
    assert qb.device_status() == qb.OK


def test_accepted_tokens_follow_the_target(cuda):
    """Draft from q, verify against p, over many pairs of uniforms: the first token's frequencies
    are p's within five standard deviations."""
    import torch

    rng = np.random.default_rng(5)
    b, v = 40000, 6
    target, draft, _, _, _ = _case(rng, 1, 1, v, sharp=1.0)
    p, q = target[0, 0].astype(np.float64), draft[0, 0].astype(np.float64)
    tokens = rng.choice(v, b, p=q / q.sum()).astype(np.int32).reshape(b, 1)
    out, _ = qb.verify_drafts(_tensor(target, cuda).expand(b, 2, v).contiguous(), _tensor(draft, cuda).expand(b, 1, v).contiguous(),
                              _tensor(tokens, cuda), torch.from_numpy(rng.random((b, 1)).astype(np.float32)).to(cuda),
                              torch.from_numpy(rng.random(b).astype(np.float32)).to(cuda))
    seen = np.bincount(out[:, 0].cpu().numpy(), minlength=v) / b
    assert (np.abs(seen - p / p.sum()) <= 5 * np.sqrt(p * (1 - p) / b) + 1e-6).all()


def test_captured_verification(cuda):
    """Probabilities and verification captured in a graph, replayed with other logits."""
    import torch

    rng = np.random.default_rng(6)
    b, k, v = 4, 3, 2000
    logits, draft = torch.zeros(b * (k + 1), v, device=cuda), torch.zeros(b, k, v, device=cuda)
    tokens, u, ul = torch.zeros(b, k, dtype=torch.int32, device=cuda), torch.zeros(b, k, device=cuda), torch.zeros(b, device=cuda)

    def step():
        probs = qb.token_probs(logits, 0.8)
        return probs, qb.verify_drafts(probs.view(b, k + 1, v), draft, tokens, u, ul)

    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        probs, out = step()
    for _ in range(3):
        case = _case(rng, b, k, v)
        logits.copy_(0.8 * torch.log(_tensor(case[0], cuda)).view(-1, v))
        for dst, src in zip((draft, tokens, u, ul), case[1:]):
            dst.copy_(_tensor(src, cuda))
        g.replay()
        torch.cuda.synchronize()
        want = verify64(probs.view(b, k + 1, v).cpu().numpy(), *case[1:])
        assert np.array_equal(out[0].cpu().numpy(), want[0]) and np.array_equal(out[1].cpu().numpy(), want[1])
    del g


def test_refusals(cuda):
    import torch

    x = torch.zeros(2, 8, device=cuda)
    for t in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(qb.QrafError, match="temperature"):
            qb.token_probs(x, t)
    with pytest.raises(ValueError):
        qb.token_probs(x.half())
    with pytest.raises(ValueError):
        qb.token_probs(x.t())
    with pytest.raises(ValueError):
        qb.token_probs(x, out=torch.zeros(2, 9, device=cuda))
    t, d = torch.zeros(2, 3, 8, device=cuda), torch.zeros(2, 2, 8, device=cuda)
    tok, u, ul = torch.zeros(2, 2, dtype=torch.int32, device=cuda), torch.zeros(2, 2, device=cuda), torch.zeros(2, device=cuda)
    with pytest.raises(ValueError, match="shapes"):
        qb.verify_drafts(t, d[:, :1], tok, u, ul)
    with pytest.raises(ValueError, match="int32"):
        qb.verify_drafts(t, d, tok.long(), u, ul)
    with pytest.raises(ValueError, match="float32"):
        qb.verify_drafts(t.double(), d, tok, u, ul)
    with pytest.raises(ValueError, match="contiguous"):
        qb.verify_drafts(t.transpose(1, 2).contiguous().transpose(1, 2), d, tok, u, ul)
    with pytest.raises(qb.QrafError, match="256 drafts"):
        qb.verify_drafts(torch.zeros(1, 258, 4, device=cuda), torch.zeros(1, 257, 4, device=cuda),
                         torch.zeros(1, 257, dtype=torch.int32, device=cuda), torch.zeros(1, 257, device=cuda), ul[:1])
    with pytest.raises(qb.QrafError, match="empty"):
        qb.verify_drafts(t[:, :, :0], d[:, :, :0], tok, u, ul)
    assert qb.verify_drafts(t[:0], d[:0], tok[:0], u[:0], ul[:0])[0].shape == (0, 3)
