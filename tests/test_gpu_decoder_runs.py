"""Decoder steps over runs of tokens (qraf_cuda_decoder_step_runs), a shared prefix, and the serving
loop that they make with token_probs and verify_drafts, against the decoder's own single-token steps
(which tests/test_gpu_decoder.py holds to the reference).

With one layer and EXACT projections both decoders form the same K and V, so their caches hold the
same codes and only the attention's rounding differs (about 1e-6 of an output): logits within 1e-4
of themselves and of the largest.  With more layers that rounding may move a later layer's code by
one step, 1/127 of its row's largest, and the bar is the one of the int8 cache's own test."""
from __future__ import annotations

import numpy as np
import pytest

import qraf_b200 as qb
import qraf_spec
from qraf_b200 import qraf_file as qf

pytestmark = pytest.mark.gpu


def _model(tmp_path, oracle_lib, arch="qwen2", dt=qb.Q8_0, **kw):
    spec = qraf_spec.tiny_decoder(arch, dt, **kw)
    w = qf.QrafFileWriter()
    qraf_spec.write_with(w, spec, oracle_lib.quantize_rows)
    path = str(tmp_path / f"{arch}_{dt}_{kw.get('layers', 2)}_{kw.get('heads', 4)}.qraf")
    w.write(path)
    return path, dict(spec["config"])["vocab_size"]


def _i32(vals, cuda):
    import torch

    return torch.tensor(vals, dtype=torch.int32, device=cuda)


def _close(got, want, label, rel=1e-4):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    tol = rel * np.abs(want) + rel * np.abs(want).max()
    assert (np.abs(got - want) <= tol).all(), f"{label}: worst {np.abs(got - want).max():.3g}"


def _sequential(path, cuda, seqs, max_seq, mode):
    """Logits of each sequence token by token, one slot at a time."""
    out = []
    dec = qb.Decoder(path, max_slots=1, max_seq=max_seq, kv_int8=True)
    for s in seqs:
        out.append([dec.step(_i32([t], cuda), _i32([p], cuda), _i32([0], cuda), mode=mode).cpu().numpy()[0]
                    for p, t in enumerate(s)])
    dec.close()
    return out


def _runs(dec, cuda, seqs, slots, starts, mode, **kw):
    cu = np.concatenate([[0], np.cumsum([len(s) for s in seqs])])
    return dec.step_runs(_i32([t for s in seqs for t in s], cuda), _i32(slots, cuda), _i32(starts, cuda), _i32(cu.tolist(), cuda),
                         mode=mode, **kw).cpu().numpy()


@pytest.mark.parametrize("arch,dt,heads,kv_heads", [("qwen2", qb.Q8_0, 4, 2), ("llama", qb.Q4_0, 8, 1), ("qwen2", qb.Q4_0, 16, 16)])
def test_prompts_in_runs_match_single_steps(tmp_path, cuda, oracle_lib, arch, dt, heads, kv_heads):
    """Three prompts of uneven lengths at once, then more runs behind them (one token, several)."""
    path, vocab = _model(tmp_path, oracle_lib, arch, dt, layers=1, heads=heads, kv_heads=kv_heads, max_seq=128)
    rng = np.random.default_rng(1)
    seqs = [[int(t) for t in rng.integers(0, vocab, n)] for n in (70, 33, 8)]
    want = _sequential(path, cuda, seqs, 128, qb.MODE_EXACT)
    dec = qb.Decoder(path, max_slots=96, max_seq=128, kv_int8=True)
    at, slots = [0, 0, 0], [5, 0, 95]
    for take in ((50, 30, 1), (1, 1, 1), (19, 2, 6)):
        parts = [s[a:a + n] for s, a, n in zip(seqs, at, take)]
        got = _runs(dec, cuda, parts, slots, at, qb.MODE_EXACT)
        row = 0
        for i, part in enumerate(parts):
            for j in range(len(part)):
                _close(got[row], want[i][at[i] + j], f"sequence {i} position {at[i] + j}")
                row += 1
        at = [a + len(p) for a, p in zip(at, parts)]
    dec.close()
    assert qb.device_status() == qb.OK


@pytest.mark.parametrize("mode", [qb.MODE_AUTO, qb.MODE_FAST])
def test_two_layers_stay_close(tmp_path, cuda, oracle_lib, mode):
    """The projections' other routes (rows, tensor cores): logits within 2e-2 of the largest and a
    cosine above 0.9999, the bar of the int8 cache against the f32 one."""
    path, vocab = _model(tmp_path, oracle_lib, max_seq=64)
    rng = np.random.default_rng(2)
    seqs = [[int(t) for t in rng.integers(0, vocab, n)] for n in (40, 7, 21)]
    want = _sequential(path, cuda, seqs, 64, qb.MODE_EXACT)
    dec = qb.Decoder(path, max_slots=80, max_seq=64, kv_int8=True)
    got = _runs(dec, cuda, seqs, [2, 0, 1], [0, 0, 0], mode)
    flat = [w for s in want for w in s]
    for g, w in zip(got.astype(np.float64), np.asarray(flat, np.float64)):
        assert np.abs(g - w).max() < 2e-2 * np.abs(w).max()
        assert g @ w / np.linalg.norm(g) / np.linalg.norm(w) > 0.9999
    dec.close()
    assert qb.device_status() == qb.OK


def test_a_shared_prefix_is_the_sequences_own(tmp_path, cuda, oracle_lib):
    """Sequences behind a shared prompt give the logits that each gives with the prompt in its own
    slot; their rows begin at row 0 of their slots; the prompt's slot takes no tokens; without the
    prefix the decoder is as before."""
    path, vocab = _model(tmp_path, oracle_lib, layers=1, heads=8, kv_heads=2, max_seq=160)
    rng = np.random.default_rng(3)
    prompt = [int(t) for t in rng.integers(0, vocab, 90)]
    tails = [[int(t) for t in rng.integers(0, vocab, n)] for n in (12, 1, 30, 5)]
    want = [w[90:] for w in _sequential(path, cuda, [prompt + t for t in tails], 160, qb.MODE_EXACT)]
    dec = qb.Decoder(path, max_slots=90, max_seq=160, kv_int8=True)
    first = _runs(dec, cuda, [prompt], [7], [0], qb.MODE_EXACT)
    dec.share_prefix(7, 90)
    got = _runs(dec, cuda, tails, [3, 8, 0, 50], [90] * 4, qb.MODE_EXACT)
    for g, w in zip(got, [x for s in want for x in s]):
        _close(g, w, "behind the prefix")
    cache = dec.layer_cache(0)
    assert cache.k_scale[3, :12].all() and not cache.k_scale[3, 12:].any() and cache.rows == 160
    back = qb.kv_load(cache, _i32([0], cuda), _i32([3], cuda), n=1)[0].cpu().numpy().reshape(-1)
    k, _, ks, _ = dec.kv_read(0, 0, 3, 2, 32)
    assert np.array_equal(back, (k.reshape(2, 32).astype(np.float32) * ks[:, None]).reshape(-1))
    for slots, starts in (([7], [90]), ([3], [89]), ([90], [95]), ([-2], [95]), ([3], [160])):
        dec.step_runs(_i32([1], cuda), _i32(slots, cuda), _i32(starts, cuda), mode=qb.MODE_FAST)
        assert qb.device_status() == qb.ERR_INVALID
    dec.step_runs(_i32([1], cuda), _i32([-1], cuda), _i32([0], cuda), mode=qb.MODE_FAST)   # padding
    assert qb.device_status() == qb.OK
    dec.share_prefix(0, 0)
    again = _runs(dec, cuda, [prompt], [1], [0], qb.MODE_EXACT)
    assert again.tobytes() == first.tobytes()
    dec.close()
    assert qb.device_status() == qb.OK


def test_the_serving_loop(tmp_path, cuda, oracle_lib):
    """Drafted decoding behind a shared prompt: every round drafts up to three tokens a sequence, one
    step over runs scores them, token_probs and verify_drafts accept or replace them from given random
    numbers; rejected rows are overwritten by the next round.  The tokens are those that the plain
    form picks from the probabilities, and every logit is that of the sequence that was accepted."""
    import torch

    from test_gpu_sampling import verify64

    path, vocab = _model(tmp_path, oracle_lib, layers=1, heads=8, kv_heads=2, max_seq=96)
    rng = np.random.default_rng(4)
    prompt = [int(t) for t in rng.integers(0, vocab, 40)]
    b, k = 3, 3
    dec = qb.Decoder(path, max_slots=40, max_seq=96, kv_int8=True)
    _runs(dec, cuda, [prompt], [0], [0], qb.MODE_EXACT)
    dec.share_prefix(0, 40)
    texts = [[int(rng.integers(0, vocab))] for _ in range(b)]     # each sequence's tokens; the last one not yet in the cache
    slots = [1, 5, 9]
    seen = []                                                      # (sequence, position, logits) of accepted tokens
    for _ in range(6):
        # a draft model that knows the temperature-flattened answer would be: here, noise around uniform
        q = np.exp(0.3 * rng.standard_normal((b, k, vocab)))
        q = (q / q.sum(-1, keepdims=True)).astype(np.float32)
        tokens = np.array([[rng.choice(vocab, p=d.astype(np.float64) / d.astype(np.float64).sum()) for d in s] for s in q], np.int32)
        runs = [[t[-1]] + d.tolist() for t, d in zip(texts, tokens)]
        starts = [40 + len(t) - 1 for t in texts]
        cu = _i32([0, k + 1, 2 * (k + 1), 3 * (k + 1)], cuda)
        logits = dec.step_runs(_i32([t for r in runs for t in r], cuda), _i32(slots, cuda), _i32(starts, cuda), cu, mode=qb.MODE_EXACT)
        probs = qb.token_probs(logits, 3.0).view(b, k + 1, vocab)
        u, last = rng.random((b, k)).astype(np.float32), rng.random(b).astype(np.float32)
        out, accepted = qb.verify_drafts(probs, torch.from_numpy(q).to(cuda), torch.from_numpy(tokens).to(cuda),
                                         torch.from_numpy(u).to(cuda), torch.from_numpy(last).to(cuda))
        want = verify64(probs.cpu().numpy(), q, tokens, u, last)
        assert np.array_equal(out.cpu().numpy(), want[0]) and np.array_equal(accepted.cpu().numpy(), want[1])
        rows = logits.view(b, k + 1, vocab).cpu().numpy()
        for i in range(b):
            n = int(accepted[i])
            for j in range(n + 1):
                seen.append((i, len(texts[i]) - 1 + j, rows[i, j]))
            texts[i] += [int(t) for t in out[i, :n + 1]]
    dec.close()
    assert any(len(t) > 7 for t in texts)   # something was accepted
    exact = _sequential(path, cuda, [prompt + t for t in texts], 96, qb.MODE_EXACT)
    for i, at, row in seen:
        _close(row, exact[i][40 + at], f"sequence {i} token {at}")
    assert qb.device_status() == qb.OK


def test_captured_steps_over_runs(tmp_path, cuda, oracle_lib):
    """A step over runs behind a prefix, captured and replayed with other tokens and positions."""
    import torch

    path, vocab = _model(tmp_path, oracle_lib, layers=1, heads=8, kv_heads=2, max_seq=64)
    rng = np.random.default_rng(5)
    prompt = [int(t) for t in rng.integers(0, vocab, 20)]
    tails = [[int(t) for t in rng.integers(0, vocab, 8)] for _ in range(2)]
    want = _sequential(path, cuda, [prompt + t for t in tails], 64, qb.MODE_FAST)
    dec = qb.Decoder(path, max_slots=20, max_seq=64, kv_int8=True)
    _runs(dec, cuda, [prompt], [0], [0], qb.MODE_FAST)
    dec.share_prefix(0, 20)
    tok, slots, starts, cu = _i32([0] * 4, cuda), _i32([1, 2], cuda), _i32([20, 20], cuda), _i32([0, 2, 4], cuda)
    logits = torch.empty((4, vocab), device=cuda)
    s = torch.cuda.Stream(cuda)
    with torch.cuda.stream(s):
        dec.step_runs(tok, slots, starts, cu, mode=qb.MODE_FAST, logits=logits, stream=s)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        dec.step_runs(tok, slots, starts, cu, mode=qb.MODE_FAST, logits=logits, stream=s)
    for p in range(0, 8, 2):
        tok.copy_(_i32(tails[0][p:p + 2] + tails[1][p:p + 2], cuda))
        starts.fill_(20 + p)
        g.replay()
        torch.cuda.synchronize()
        for row, (i, j) in enumerate(((0, 0), (0, 1), (1, 0), (1, 1))):
            _close(logits[row].cpu().numpy(), want[i][20 + p + j], f"sequence {i} position {20 + p + j}")
    del g
    dec.close()
    assert qb.device_status() == qb.OK


def test_refusals(tmp_path, cuda, oracle_lib):
    import torch

    path, vocab = _model(tmp_path, oracle_lib, layers=1, max_seq=32)
    dec = qb.Decoder(path, max_slots=4, max_seq=32)
    one = _i32([0], cuda)
    for call in (lambda: dec.step_runs(one, one, one), lambda: dec.share_prefix(0, 4), lambda: dec.layer_cache(0)):
        with pytest.raises(qb.QrafError, match="int8") as e:
            call()
        assert e.value.code == qb.ERR_UNSUPPORTED
    dec.close()
    dec = qb.Decoder(path, max_slots=4, max_seq=32, kv_int8=True)
    with pytest.raises(qb.QrafError, match="max_slots"):
        dec.step_runs(_i32([0] * 5, cuda), one, one, _i32([0, 5], cuda))
    with pytest.raises(qb.QrafError, match="out of range"):
        dec.share_prefix(4, 1)
    with pytest.raises(qb.QrafError, match="out of range"):
        dec.share_prefix(0, 33)
    with pytest.raises(qb.QrafError, match="layer 1"):
        dec.layer_cache(1)
    with pytest.raises(ValueError, match="int32"):
        dec.step_runs(one.long(), one, one)
    with pytest.raises(ValueError, match="logits"):
        dec.step_runs(one, one, one, logits=torch.zeros(1, vocab + 1, device=cuda))
    assert dec.step_runs(one[:0], one[:0], one[:0]).shape == (0, vocab)
    dec.close()


@pytest.mark.parametrize("prefix", [0, 20])
def test_a_refused_run_stores_nothing(tmp_path, cuda, oracle_lib, prefix):
    """A run that ends past the last position, by one or by many, with others in the same step: the
    status is raised, no row of its slot is written, not even those that would fit, and the others give
    what they give without it."""
    path, vocab = _model(tmp_path, oracle_lib, layers=1, heads=8, kv_heads=2, max_seq=64)
    rng = np.random.default_rng(6)
    prompt, good = ([int(t) for t in rng.integers(0, vocab, n)] for n in (20, 5))
    dec = qb.Decoder(path, max_slots=40, max_seq=64, kv_int8=True)
    if prefix:
        _runs(dec, cuda, [prompt], [9], [0], qb.MODE_EXACT)
        dec.share_prefix(9, prefix)
    want = _runs(dec, cuda, [good], [1], [prefix], qb.MODE_EXACT)
    cache = dec.layer_cache(0)
    for slot, (length, start) in enumerate(((5, 60), (9, 60), (2, 63)), 2):
        bad = [int(t) for t in rng.integers(0, vocab, length)]
        got = _runs(dec, cuda, [bad, good], [slot, 1], [start, prefix], qb.MODE_EXACT)
        assert qb.device_status() == qb.ERR_INVALID and qb.device_status() == qb.OK
        assert got[length:].tobytes() == want.tobytes()
        for t in (cache.k, cache.v, cache.k_scale, cache.v_scale):
            assert not t[slot].any()
    _runs(dec, cuda, [[1, 2, 3, 4]], [2], [60], qb.MODE_EXACT)   # one that fits to the last position
    assert cache.k_scale[2, 60 - prefix:64 - prefix].all() and qb.device_status() == qb.OK
    dec.close()


def test_the_guides_serving_example(tmp_path, cuda, oracle_lib, monkeypatch):
    """The serving example of the integration guide, run as it stands: what it calls `tokens` and
    `accepted` are those."""
    import re
    from pathlib import Path

    import torch

    from test_gpu_sampling import verify64

    text = (Path(__file__).resolve().parents[1] / "INTEGRATION.md").read_text()
    blocks = [b for b in re.findall(r"```python\n(.*?)```", text, re.S) if "verify_drafts(" in b]
    assert len(blocks) == 1
    path, vocab = _model(tmp_path, oracle_lib, layers=1, heads=8, kv_heads=2, max_seq=4096)
    Path(path).rename(tmp_path / "model-q8.qraf")
    monkeypatch.chdir(tmp_path)
    rng = np.random.default_rng(7)
    q = rng.random((2, 3, vocab)).astype(np.float32) + 0.1
    q /= q.sum(-1, keepdims=True)
    drafts = rng.integers(0, vocab, (2, 3)).astype(np.int32)
    u, last = (rng.random(n).astype(np.float32) for n in ((2, 3), 2))
    lines = np.concatenate([rng.integers(0, vocab, (2, 1)).astype(np.int32), drafts], 1)
    at = {"prompt": _i32([int(t) for t in rng.integers(0, vocab, 30)], cuda), "drafted": torch.from_numpy(lines.reshape(-1)).to(cuda),
          "starts": _i32([30, 33], cuda), "q": torch.from_numpy(q).to(cuda), "drafts": torch.from_numpy(drafts).to(cuda),
          "u": torch.from_numpy(u).to(cuda), "u_last": torch.from_numpy(last).to(cuda)}
    exec(compile(blocks[0], "INTEGRATION.md", "exec"), at)
    want = verify64(at["p"].view(2, 4, -1).cpu().numpy(), q, drafts, u, last)
    assert np.array_equal(at["tokens"].cpu().numpy(), want[0]) and np.array_equal(at["accepted"].cpu().numpy(), want[1])
    at["dec"].close()
    assert qb.device_status() == qb.OK


def test_a_closed_decoders_cache_is_refused(tmp_path, cuda, oracle_lib):
    """Views of a decoder's cache keep it; closing it takes their memory away, and every operator then
    refuses them, as cache or as prefix, and so does the library their descriptor."""
    import ctypes as C
    import gc

    import torch

    path, vocab = _model(tmp_path, oracle_lib, layers=2, heads=8, kv_heads=2, max_seq=32)
    dec = qb.Decoder(path, max_slots=4, max_seq=32, kv_int8=True)
    scales = dec.layer_cache(1).k_scale
    _runs(dec, cuda, [[1, 2, 3]], [1], [0], qb.MODE_EXACT)
    cache = dec.layer_cache(1)
    dim, one = cache.head_dim, _i32([1], cuda)
    q, k = torch.zeros(1, 8, dim, device=cuda), torch.zeros(1, 2, dim, device=cuda)
    want = cache.k_scale.clone()
    del dec, cache
    gc.collect()
    assert torch.equal(scales, want) and scales[1, :3].all()   # a tensor alone keeps the decoder too
    del scales
    dec = qb.Decoder(path, max_slots=4, max_seq=32, kv_int8=True)
    cache, own = dec.layer_cache(0), qb.KvCache(2, 8, 2, dim)
    qb.kv_attention(q, cache, one, one)
    dec.close()
    for call in (lambda: qb.kv_store(cache, k, k, one, one), lambda: qb.kv_load(cache, one, one),
                 lambda: qb.kv_attention(q, cache, one, one),
                 lambda: qb.kv_attention(q, own, one, one, prefix=cache, prefix_len=4)):
        with pytest.raises(ValueError, match="closed"):
            call()
    assert cache.k is None
    assert qb.lib.qraf_cuda_kv_store(C.byref(cache.desc), k.data_ptr(), k.data_ptr(), 0, 2 * dim, 2 * dim, 1, one.data_ptr(),
                                     one.data_ptr(), None, 1, None) == qb.ERR_INVALID
    assert qb.device_status() == qb.OK
