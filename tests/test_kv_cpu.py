"""Host-side refusals of the KV-cache and sampling entries: what needs no GPU."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

import qraf_b200 as qb

A = 1 << 20   # a 16-byte-aligned address that is never read


def _kv(**kw):
    d = qb.qraf_kv_t(k=A, v=A, k_scale=A, v_scale=A, slot_rows=64, slots=4, rows=64, kv_heads=2, head_dim=64, device=0)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("args,code,text", [
    ((None, A, A, A, 4, 64, 64, 2, 64), qb.ERR_INVALID, "NULL"),
    ((A, A, A, A, 0, 64, 64, 2, 64), qb.ERR_INVALID, "positive"),
    ((A, A, A, A, 4, 0, 64, 2, 64), qb.ERR_INVALID, "positive"),
    ((A, A, A, A, 4, 64, 64, 0, 64), qb.ERR_INVALID, "positive"),
    ((A, A, A, A, 4, 64, 64, 2, 0), qb.ERR_UNSUPPORTED, "head_dim"),
    ((A, A, A, A, 4, 64, 64, 2, 72), qb.ERR_UNSUPPORTED, "head_dim"),
    ((A, A, A, A, 4, 64, 64, 2, 272), qb.ERR_UNSUPPORTED, "head_dim"),
    ((A, A, A, A, 4, 64, 63, 2, 64), qb.ERR_INVALID, "overlap"),
    ((A + 8, A, A, A, 4, 64, 64, 2, 64), qb.ERR_INVALID, "aligned"),
    ((A, A, A, A + 2, 4, 64, 64, 2, 64), qb.ERR_INVALID, "aligned"),
    ((A, A, A, A, 1 << 31, 64, 64, 2, 64), qb.ERR_UNSUPPORTED, "2^31"),
])
def test_wrap_refuses(args, code, text):
    out = _kv()
    assert qb.lib.qraf_cuda_kv_wrap(*args, C.byref(out)) == code
    assert text in qb.last_error() and not out.k


@pytest.mark.parametrize("name", ["qraf_cuda_kv_store", "qraf_cuda_kv_load"])
def test_store_and_load_refuse(name):
    fn, kv = getattr(qb.lib, name), _kv()

    def call(kv=kv, k=A, v=A, type=0, ld_k=128, ld_v=128, n=2, slots=A, starts=A, cu=None, count=2):
        return fn(C.byref(kv) if kv is not None else None, k, v, type, ld_k, ld_v, n, slots, starts, cu, count, None)

    assert call(type=3) == qb.ERR_UNSUPPORTED
    assert call(n=0) == qb.OK and call(count=0) == qb.OK
    for kw, text in (({"slots": None}, "NULL"), ({"starts": None}, "NULL"), ({"count": 3}, "without cu"), ({"k": None}, "NULL"),
                     ({"v": A + 2}, "aligned"), ({"type": 1, "k": A + 1}, "aligned"), ({"ld_k": 127}, "stride"),
                     ({"ld_v": 0}, "stride"), ({"kv": None}, "NULL")):
        assert call(**kw) == qb.ERR_INVALID, kw
        assert text in qb.last_error(), kw


def test_attention_refuses():
    kv = _kv()

    def call(kv=kv, prefix=None, prefix_slot=0, prefix_len=0, q=A, out=A, type=0, q_ld=256, out_ld=256, n=2, heads=4, slots=A,
             lens=A, cu=None, count=2, max_len=64, scale=1.0):
        return qb.lib.qraf_cuda_kv_attention(C.byref(kv) if kv is not None else None, prefix, prefix_slot, prefix_len, q, out,
                                             type, q_ld, out_ld, n, heads, slots, lens, cu, count, max_len, scale, None, 0, None)

    assert call(type=9) == qb.ERR_UNSUPPORTED
    assert call(prefix_len=1 << 31) == qb.ERR_UNSUPPORTED
    assert call(n=0) == qb.OK
    for kw, text in (({"kv": None}, "NULL"), ({"heads": 0}, "multiple"), ({"heads": 3}, "multiple"), ({"max_len": 65}, "max_len"),
                     ({"q": None}, "NULL"), ({"out": A + 1}, "aligned"), ({"q_ld": 255}, "stride"), ({"out_ld": 8}, "stride"),
                     ({"count": 1}, "without cu"), ({"lens": None}, "NULL"),
                     ({"scale": float("nan")}, "finite"), ({"scale": float("inf")}, "finite")):
        assert call(**kw) == qb.ERR_INVALID, kw
        assert text in qb.last_error(), kw


def test_sampling_refuses():
    lib = qb.lib
    for t in (0.0, -1.0, float("inf"), float("nan"), 1e-45):
        assert lib.qraf_cuda_token_probs(A, 8, A, 8, 1, 8, t, None) == qb.ERR_INVALID
    assert lib.qraf_cuda_token_probs(None, 8, A, 8, 1, 8, 1.0, None) == qb.ERR_INVALID
    assert lib.qraf_cuda_token_probs(A, 7, A, 8, 2, 8, 1.0, None) == qb.ERR_INVALID
    assert lib.qraf_cuda_token_probs(A + 2, 8, A, 8, 2, 8, 1.0, None) == qb.ERR_INVALID
    assert lib.qraf_cuda_token_probs(A, 8, A, 8, 0, 8, 1.0, None) == qb.OK

    def verify(target=A, t_seq=64, t_row=16, draft=A, d_seq=48, d_row=16, tokens=A, u=A, last=A, seqs=2, drafts=3, vocab=16,
               out=A, acc=A):
        return lib.qraf_cuda_verify_drafts(target, t_seq, t_row, draft, d_seq, d_row, tokens, u, last, None, seqs, drafts, vocab,
                                           out, acc, None)

    assert verify(drafts=257) == qb.ERR_UNSUPPORTED
    assert verify(seqs=0) == qb.OK
    for kw in ({"target": None}, {"draft": None}, {"tokens": None}, {"u": None}, {"last": None}, {"out": None}, {"acc": None},
               {"vocab": 0}, {"t_row": 15}, {"d_row": 15}, {"t_seq": 15}, {"d_seq": 15}, {"target": A + 2}):
        assert verify(**kw) == qb.ERR_INVALID, kw


def _prefix_stretch(scores, term, restart, lag=8.0):
    """A row's way through one stretch of kv_prefix_kernel in fp32: (maximum, sum) that its records are
    joined with.  scores: (maximum, sum of weights relative to it) of each tile, binary; restart: the
    maximum referred to from a new sum on, of the one before and the tile's."""
    f32 = np.float32

    def ex2(x):   # 2^x, flushed to zero below the normal range as on the device
        with np.errstate(over="ignore"):
            y = np.exp2(f32(x), dtype=np.float32)
        return y if y >= np.finfo(f32).tiny else f32(0)

    m = [f32(-np.inf)] * 2   # of the two warpgroups, which take the tiles in turn
    total = [f32(0)] * 2
    before, records = None, []
    for t, (mt, weight) in enumerate(scores):
        mt = f32(mt)
        if t == 0:
            now = mt
        elif t % term == 0:
            records.append((before, f32(0)))   # what was summed leaves; its weights stay in the sum
            now = f32(restart(before, mt))
        else:
            now = mt if mt > before + f32(lag) else before
        g = t & 1
        if now != m[g]:
            with np.errstate(over="ignore", invalid="ignore"):
                total[g] = f32(0) if m[g] == -np.inf else total[g] * ex2(m[g] - now)
        m[g] = before = now
        total[g] = total[g] + f32(weight) * ex2(mt - now)
    end = f32(0)
    with np.errstate(over="ignore", invalid="ignore"):
        for g in range(2):
            if m[g] > -np.inf:
                end = end + total[g] * ex2(m[g] - before)
        records.append((before, end))
        top = max(r[0] for r in records)
        return top, sum(ex2(r[0] - top) * r[1] for r in records)


@pytest.mark.parametrize("gap", [0, 90, 120, 126, 127, 128, 130, 300, 2000])
@pytest.mark.parametrize("tiles,term", [(40, 32), (40, 8), (71, 32), (9, 8)])
def test_a_sum_that_starts_anew_keeps_its_weights(gap, tiles, term):
    """A first tile `gap` binary orders above all later ones: the joined sum of weights is its own (and
    the others', where they are not too small), relative to its maximum.  With a maximum that falls to a
    tile's own the sum is zero or not a number once 2^-gap is below the normal range."""
    scores = [(gap, 1.0)] + [(0.0, 1.0)] * (tiles - 1)
    want = 1.0 + (tiles - 1) * 2.0 ** -gap
    top, total = _prefix_stretch(scores, term, max)
    assert top == gap and abs(total - want) < 1e-5 * want
    top, total = _prefix_stretch(scores[::-1], term, max)
    assert top == gap and abs(total - want) < 1e-5 * want
    _, wrong = _prefix_stretch(scores, term, lambda before, mt: mt)
    assert (gap <= 126) == (abs(wrong - want) < 1e-4 * want)
