"""Host-side refusals of the KV-cache and sampling entries: what needs no GPU."""
from __future__ import annotations

import ctypes as C

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
