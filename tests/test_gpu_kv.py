"""The KV-cache operators (kv_store, kv_load, kv_attention) against plain 64-bit forms:
codes and scales bit for bit, attention within a bound that follows from its arithmetic."""
from __future__ import annotations

import numpy as np
import pytest

import qraf_b200 as qb

pytestmark = pytest.mark.gpu

DTYPES = ("float32", "float16", "bfloat16")


def _i32(v, cuda):
    import torch

    return torch.tensor(v, dtype=torch.int32, device=cuda)


def _gen(seed):
    return np.random.default_rng(seed)


def _tensor(a, cuda, dtype="float32"):
    import torch

    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.float32)).to(cuda).to(getattr(torch, dtype))


def quantise(x):
    """(codes, scales) of float32 rows [..., hd] by the definition: IEEE fp32 steps, halves away from zero,
    and the clamp min(127, .) gives 127 for a NaN (an infinity times its row's inverse scale 0)."""
    x = np.asarray(x, np.float32)
    with np.errstate(all="ignore"):
        most = np.fmax.reduce(np.abs(x), axis=-1, initial=np.float32(0))
        scale = (most / np.float32(127)).astype(np.float32)
        inv = np.where(scale > 0, np.float32(1) / scale, np.float32(0)).astype(np.float32)
        y = (x * inv[..., None]).astype(np.float32).astype(np.float64)
        r = np.trunc(y + np.copysign(0.5, y))
        return np.where(np.isnan(r), 127, np.clip(r, -127, 127)).astype(np.int8), scale


def _cu(runs, cuda):
    return _i32(np.concatenate([[0], np.cumsum(runs)]).tolist(), cuda)


# ── store and load ──────────────────────────────────────────────────────────
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,dim", [(1, 16), (2, 128), (5, 80), (3, 32), (8, 64), (7, 256), (2, 176)])
def test_store_writes_the_quantisers_bytes_and_load_reads_them(cuda, dtype, heads, dim):
    """Ragged runs (an empty one and one of a single row among them) into a permutation of
    slots: every code and scale by definition, every other row of the cache as it was."""
    import torch

    rng = _gen(dim * 10 + heads)
    runs, slots, starts, rows = [3, 0, 1, 37, 70], [4, 0, 2, 5, 1], [9, 3, 99, 0, 30], 100
    n = sum(runs)
    x = {s: _tensor(rng.standard_normal((n, heads, dim)) * np.exp(rng.standard_normal((n, heads, 1)) * 4), cuda, dtype)
         for s in "kv"}
    x["k"][1] = 0.0                # a row of zeros: scale 0, codes 0
    x["v"][2, 0, :3] = 0.5 * x["v"][2, 0].abs().max()   # halves among the codes
    cache = qb.KvCache(7, rows, heads, dim)
    cache.k.fill_(77)
    cache.v.fill_(-77)
    cache.k_scale.fill_(3.0)
    cache.v_scale.fill_(4.0)
    want = {"k": cache.k.cpu().numpy(), "v": cache.v.cpu().numpy(), "k_scale": cache.k_scale.cpu().numpy(),
            "v_scale": cache.v_scale.cpu().numpy()}
    args = _i32(slots, cuda), _i32(starts, cuda), _cu(runs, cuda)
    qb.kv_store(cache, x["k"], x["v"], *args)
    back = qb.kv_load(cache, *args, n=n, dtype=getattr(torch, dtype))
    t = 0
    for m, s, f in zip(runs, slots, starts):
        for name in "kv":
            codes, scale = quantise(x[name][t:t + m].float().cpu().numpy())
            want[name][s, f:f + m], want[name + "_scale"][s, f:f + m] = codes, scale
        t += m
    for name, w in want.items():
        assert getattr(cache, name).cpu().numpy().tobytes() == w.tobytes(), name
    for name, got in zip("kv", back):
        codes, scale = quantise(x[name].float().cpu().numpy())
        with np.errstate(invalid="ignore"):
            val = torch.from_numpy(codes.astype(np.float32) * scale[..., None]).to(got.dtype)
        assert torch.equal(got.cpu().nan_to_num(nan=-7.0), val.nan_to_num(nan=-7.0)), name
    assert qb.device_status() == qb.OK


def test_store_of_one_row_a_sequence_from_a_joined_projection(cuda):
    """Without cu each row is a run; k and v are column slices of one projection's output."""
    import torch

    heads, dim, b = 2, 128, 5
    qkv = _tensor(_gen(1).standard_normal((b, 3 + 2 * heads * dim + 2)), cuda)   # an odd stride: no wide loads
    k, v = qkv[:, 3:3 + heads * dim], qkv[:, 3 + heads * dim:3 + 2 * heads * dim]
    cache = qb.KvCache(8, 10, heads, dim)
    slots, starts = [7, 0, 3, 2, 5], [9, 0, 4, 4, 1]
    qb.kv_store(cache, k, v, _i32(slots, cuda), _i32(starts, cuda))
    for i, (s, r) in enumerate(zip(slots, starts)):
        codes, scale = quantise(k[i].reshape(heads, dim).cpu().numpy())
        assert np.array_equal(cache.k[s, r].cpu().numpy(), codes)
        assert np.array_equal(cache.k_scale[s, r].cpu().numpy(), scale)
    kk, vv = torch.full((b, 2 * heads * dim), 9.0, device=cuda).split(heads * dim, 1)   # read back into slices
    qb.kv_load(cache, _i32(slots, cuda), _i32(starts, cuda), k=kk, v=vv)
    codes, scale = quantise(v.reshape(b, heads, dim).cpu().numpy())
    assert np.array_equal(vv.cpu().numpy().reshape(b, heads, dim), codes * scale[..., None])


def test_store_special_values(cuda):
    """A NaN is never the largest and takes the code the clamp gives it; an infinity's row
    has an infinite scale; values of 1e-38 and 1e38 keep theirs."""
    rows = np.ones((5, 1, 16), np.float32)
    rows[0, 0, 3] = np.nan
    rows[1, 0, 4] = np.inf
    rows[2] *= 1e38
    rows[3] *= 1e-38
    rows[4] = np.nan
    x = _tensor(rows, cuda)
    cache = qb.KvCache(1, 5, 1, 16)
    qb.kv_store(cache, x, x, _i32([0], cuda), _i32([0], cuda), _i32([0, 5], cuda))
    scale = cache.k_scale.cpu().numpy().reshape(5)
    codes = cache.k.cpu().numpy().reshape(5, 16)
    fine = [0, 2, 3]
    want = quantise(np.nan_to_num(rows[fine], nan=1.0))
    assert np.array_equal(scale[fine], want[1].reshape(-1))
    assert np.array_equal(np.delete(codes[0], 3), np.delete(want[0][0, 0], 3))
    assert np.array_equal(codes[2:4], want[0][1:, 0])
    assert np.isinf(scale[1]) and scale[4] == 0.0


def test_padding_and_bounds_leave_the_cache_alone(cuda):
    """Slot -1 and rows behind the last run are left out silently; a slot out of range, a
    start below zero and rows past the end of a slot are not written and raise the status."""
    heads, dim = 2, 64
    x = _tensor(_gen(3).standard_normal((12, heads, dim)), cuda)
    cache = qb.KvCache(3, 4, heads, dim)
    qb.kv_store(cache, x, x, _i32([1, -1], cuda), _i32([0, 0], cuda), _i32([0, 2, 5], cuda))
    assert qb.device_status() == qb.OK
    touched = cache.k_scale.cpu().numpy() != 0
    want = np.zeros((3, 4, heads), bool)
    want[1, :2] = True
    assert np.array_equal(touched, want)
    for slots, starts, ok in (([3], [0], ()), ([-2], [0], ()), ([0], [-1], ()), ([2], [2], ((2, 2), (2, 3))),
                              ([0], [2 ** 31 - 1], ())):
        cache.k_scale.zero_()
        qb.kv_store(cache, x, x, _i32(slots, cuda), _i32(starts, cuda), _i32([0, 4], cuda))
        assert qb.device_status() == qb.ERR_INVALID
        assert qb.device_status() == qb.OK
        want = np.zeros((3, 4, heads), bool)
        for at in ok:
            want[at] = True
        assert np.array_equal(cache.k_scale.cpu().numpy() != 0, want), (slots, starts)


def test_the_later_run_wins(cuda):
    """Runs of one call that write the same rows leave what storing them one after another would."""
    heads, dim = 3, 48
    runs, slots, starts = [6, 4, 5, 1], [1, 0, 1, 1], [0, 0, 3, 4]
    x = _tensor(_gen(4).standard_normal((16, heads, dim)), cuda)
    y = _tensor(_gen(5).standard_normal((16, heads, dim)), cuda)
    one, many = qb.KvCache(2, 8, heads, dim), qb.KvCache(2, 8, heads, dim)
    qb.kv_store(one, x, y, _i32(slots, cuda), _i32(starts, cuda), _cu(runs, cuda))
    t = 0
    for m, s, f in zip(runs, slots, starts):
        qb.kv_store(many, x[t:t + m], y[t:t + m], _i32([s], cuda), _i32([f], cuda), _i32([0, m], cuda))
        t += m
    for name in ("k", "v", "k_scale", "v_scale"):
        assert getattr(one, name).cpu().numpy().tobytes() == getattr(many, name).cpu().numpy().tobytes(), name


# ── attention ───────────────────────────────────────────────────────────────
def _filled(rng, slots, rows, heads, dim, cuda, wide=0.6):
    import torch

    cache = qb.KvCache(slots, rows, heads, dim)
    for name in "kv":
        x = rng.standard_normal((slots, rows, heads, dim)) * np.exp(wide * rng.standard_normal((heads, dim)))
        codes, scale = quantise(x)
        getattr(cache, name).copy_(torch.from_numpy(codes))
        getattr(cache, name + "_scale").copy_(torch.from_numpy(scale))
    return cache


def attention64(q, cache, slots, lens, runs, prefix=None, prefix_slot=0, prefix_len=0, scale=None):
    """(out, tolerance) in 64 bits.  The tolerance: a score is off by at most
    A (2 hd / 16 + 8) 2^-23, A = scale sum |q| |k|: the query's rounding to its two parts and
    to fp32, each of the 2 hd / 16 accumulations' last bit, the exponent's argument.  A weight
    is then off by twice that (its own and the maximum's) and 2^-21; the weighted sum and the
    sum of weights lose 2^-23 of sum p |v| at each of their accumulations, two per 16 keys, and
    at each of up to 64 joins.  A weight p vs is held in two fp16 parts, scaled so that the largest
    vs weighs 2^6 at least where p = 1: the lower part's last bit is 2^-24, so beside its relative
    error each weight is off by up to 2^-25 2^-6 vs_max, times a code of at most 127, over a sum of
    weights of at least 1.  For bf16 a weight may be held in one part, off by 2^-12 of itself."""
    import torch

    one_part = 2.0 ** -12 if q.dtype == torch.bfloat16 and prefix_len else 0.0
    q = q.double()
    n, heads, dim = q.shape
    group = heads // cache.kv_heads
    scale = dim ** -0.5 if scale is None else scale
    out, tol = torch.zeros_like(q), torch.zeros_like(q)

    def values(c, name, slot, rows):
        return getattr(c, name)[slot, :rows].double() * getattr(c, name + "_scale")[slot, :rows].double().unsqueeze(-1)

    if prefix_len:
        far = values(prefix, "k", prefix_slot, prefix_len), values(prefix, "v", prefix_slot, prefix_len)
    t = 0
    for slot, length, m in zip(slots, lens, runs):
        for i in range(m):
            seen = max(0, length - m + 1 + i)
            if slot >= 0 and prefix_len + seen:
                k, v = values(cache, "k", slot, seen), values(cache, "v", slot, seen)
                if prefix_len:
                    k, v = torch.cat([far[0], k]), torch.cat([far[1], v])
                k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
                s = torch.einsum("hd,khd->hk", q[t], k) * scale
                a = (torch.einsum("hd,khd->hk", q[t].abs(), k.abs()) * abs(scale)).amax(1)
                p = torch.softmax(s, 1)
                out[t] = torch.einsum("hk,khd->hd", p, v)
                size = torch.einsum("hk,khd->hd", p, v.abs())
                floor = len(k) * v.abs().max() * 2.0 ** -31   # max |v| is 127 vs_max
                ds = a * (2 * dim / 16 + 8) * 2.0 ** -23
                tol[t] = size * (2 * ds.unsqueeze(1) + one_part + 2.0 ** -21 + (len(k) / 8 + 64) * 2.0 ** -23) + floor
            t += 1
    return out.cpu().numpy(), tol.cpu().numpy()


def check(got, want, tol, dtype="float32"):
    import torch

    got = got.double().cpu().numpy().reshape(want.shape)
    info = torch.finfo(getattr(torch, dtype))
    tol = tol + (np.abs(want) + tol) * info.eps / 2 + info.smallest_normal * info.eps / 2 + 1e-300
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.size} values off, worst {np.nanmax(np.abs(got - want) / tol):.3g} x the bound"


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 1, 128), (16, 2, 128), (6, 2, 64), (5, 5, 16), (7, 1, 80),
                                                (16, 1, 96), (12, 4, 256), (20, 4, 32), (48, 3, 240)])
@pytest.mark.parametrize("prefix_len", [0, 1, 333])
def test_one_token_a_sequence(cuda, dtype, heads, kv_heads, dim, prefix_len):
    """Head layouts of 1 to 16 query heads a KV head, sizes that fill no tile, own lengths from
    none to many, with and without a prefix."""
    rng = _gen(heads * dim + prefix_len)
    slots, lens, rows = [3, 0, 6, 1, 4], [0, 1, 31, 33, 300], 300
    cache = _filled(rng, 7, rows, kv_heads, dim, cuda)
    prefix = _filled(rng, 2, 340, kv_heads, dim, cuda) if prefix_len else None
    q = _tensor(rng.standard_normal((5, heads, dim)) * 2, cuda, dtype)
    got = qb.kv_attention(q, cache, _i32(slots, cuda), _i32(lens, cuda), prefix=prefix, prefix_slot=1 if prefix else 0,
                          prefix_len=prefix_len)
    check(got, *attention64(q, cache, slots, lens, [1] * 5, prefix, 1, prefix_len), dtype)
    if not prefix_len:
        assert not got[0].any()   # a row that sees nothing
    assert qb.device_status() == qb.OK


@pytest.mark.parametrize("dtype", ("float32", "bfloat16"))
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 1, 128), (8, 8, 64), (12, 4, 80), (4, 2, 256)])
@pytest.mark.parametrize("prefix_len", [0, 500])
def test_drafted_runs_are_causal(cuda, dtype, heads, kv_heads, dim, prefix_len):
    """Runs of 0 to 9 tokens: token i of m sees len - m + 1 + i rows, nothing where that is
    below one (a run longer than its slot's rows)."""
    rng = _gen(heads + dim + prefix_len)
    slots, runs, lens, rows = [2, 0, 4, 3, 1, 5], [5, 1, 0, 9, 4, 2], [200, 7, 9, 41, 2, 129], 210
    cache = _filled(rng, 6, rows, kv_heads, dim, cuda)
    prefix = _filled(rng, 1, 512, kv_heads, dim, cuda) if prefix_len else None
    q = _tensor(rng.standard_normal((sum(runs), heads, dim)) * 2, cuda, dtype)
    got = qb.kv_attention(q, cache, _i32(slots, cuda), _i32(lens, cuda), _cu(runs, cuda), prefix=prefix,
                          prefix_len=prefix_len)
    check(got, *attention64(q, cache, slots, lens, runs, prefix, 0, prefix_len), dtype)
    assert qb.device_status() == qb.OK


def _big(cuda, dtype, seqs, heads, kv_heads, dim, prefix_len, own, run, seed):
    """A batch with ragged lengths and runs, its arguments and its exact answer."""
    rng = _gen(seed)
    runs = [int(v) for v in rng.integers(1, run + 1, seqs)]
    lens = [int(v) for v in rng.integers(0, own + 1, seqs)]
    slots = [int(v) for v in rng.permutation(seqs)]
    cache = _filled(rng, seqs, own, kv_heads, dim, cuda)
    prefix = _filled(rng, 1, prefix_len, kv_heads, dim, cuda) if prefix_len else None
    q = _tensor(rng.standard_normal((sum(runs), heads, dim)) * 2, cuda, dtype)
    args = (q, cache, _i32(slots, cuda), _i32(lens, cuda), _cu(runs, cuda))
    return args, dict(prefix=prefix, prefix_len=prefix_len), attention64(q, cache, slots, lens, runs, prefix, 0, prefix_len)


# one launch: clusters; two: own rows (and a prefix, 16 rows at a time) and the join; three: the
# prefix on tiles of 128 rows, own rows, the join
@pytest.mark.parametrize("launches,dtype,seqs,heads,kv_heads,dim,prefix_len,own,run", [
    (1, "float32", 33, 8, 1, 128, 500, 64, 1), (1, "bfloat16", 3, 16, 2, 64, 3000, 40, 2), (1, "float32", 9, 4, 4, 256, 0, 777, 3),
    (1, "float16", 20, 6, 2, 96, 33, 90, 1),
    (2, "float32", 200, 16, 2, 64, 0, 300, 1), (2, "float32", 80, 10, 5, 128, 0, 333, 2), (2, "bfloat16", 300, 4, 2, 32, 0, 65, 1),
    (2, "float32", 200, 16, 2, 256, 700, 50, 1), (2, "float16", 2, 32, 8, 128, 9000, 40, 3),
    (3, "float32", 70, 16, 2, 128, 4111, 64, 1), (3, "float32", 64, 32, 4, 64, 2049, 100, 1), (3, "float16", 100, 24, 3, 96, 700, 64, 1),
    (3, "bfloat16", 90, 16, 4, 80, 1500, 130, 2), (3, "float32", 40, 28, 4, 112, 1023, 70, 3), (3, "bfloat16", 8, 64, 8, 128, 20000, 33, 1),
    (3, "float16", 150, 8, 2, 16, 1900, 20, 1),
    # one unit whose tiles are one or two for each CTA, and one with more tiles a CTA than one sum takes
    (3, "float32", 8, 8, 1, 128, 36993, 30, 1), (3, "float32", 7, 8, 1, 16, 640001, 20, 1), (3, "bfloat16", 7, 8, 1, 32, 630000, 20, 1)])
def test_every_plan(cuda, launches, dtype, seqs, heads, kv_heads, dim, prefix_len, own, run):
    """Each way a call is carried out (told by its launches), at head sizes that fill no tile and
    lengths that end inside one; the same call again gives the same bits."""
    import torch

    args, kw, (want, tol) = _big(cuda, dtype, seqs, heads, kv_heads, dim, prefix_len, own, run, seqs + dim)
    before = qb.launch_count()
    got = qb.kv_attention(*args, **kw)
    assert qb.launch_count() - before == launches
    check(got, want, tol, dtype)
    again = qb.kv_attention(*args, **kw)
    assert torch.equal(got, again)   # no order of arrival in the results
    assert qb.device_status() == qb.OK


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_prefix_that_keeps_raising_the_maximum(cuda, dtype):
    """Keys sorted by their scores, so that every tile of the prefix moves the rows' maxima (the
    outputs so far are scaled), and sorted the other way; a negative and a zero scale."""
    import torch

    rng = _gen(21)
    seqs, heads, kv_heads, dim, n = 70, 16, 2, 128, 2000
    cache, prefix = _filled(rng, seqs, 16, kv_heads, dim, cuda), _filled(rng, 1, n, kv_heads, dim, cuda)
    base = rng.standard_normal((1, 1, dim))
    q = _tensor(base + 0.1 * rng.standard_normal((seqs, heads, dim)), cuda, dtype)
    s = torch.einsum("d,nhd->nh", torch.from_numpy(base[0, 0]).to(cuda).float(), prefix.k[0].float() * prefix.k_scale[0].unsqueeze(-1))
    slots, lens = list(range(seqs)), [int(v) for v in rng.integers(0, 17, seqs)]
    for order in (False, True):
        at = s[:, 0].argsort(descending=order)
        for t in (prefix.k, prefix.k_scale, prefix.v, prefix.v_scale):
            t[0] = t[0][at]
        s = s[at]
        for scale in (1.0, -0.5, 0.0):
            got = qb.kv_attention(q, cache, _i32(slots, cuda), _i32(lens, cuda), prefix=prefix, prefix_len=n, scale=scale)
            check(got, *attention64(q, cache, slots, lens, [1] * seqs, prefix, 0, n, scale), dtype)
    assert qb.device_status() == qb.OK


def test_a_batch_whose_other_rows_are_wild(cuda):
    """Queries of NaN, infinities and 1e30 in some sequences (a padded batch's leftovers) do not
    reach the others' outputs, with the prefix on tiles of 128 rows; V scales over forty binary
    orders keep the bound."""
    import torch

    rng = _gen(22)
    seqs, heads, kv_heads, dim, n = 70, 16, 2, 128, 1500
    cache, prefix = _filled(rng, seqs, 16, kv_heads, dim, cuda), _filled(rng, 1, n, kv_heads, dim, cuda)
    prefix.v_scale.mul_(torch.exp2(torch.from_numpy(rng.integers(-20, 21, (1, n, kv_heads)).astype(np.float32)).to(cuda)))
    q = _tensor(rng.standard_normal((seqs, heads, dim)), cuda)
    slots, lens = list(range(seqs)), [9] * seqs
    want, tol = attention64(q, cache, slots, lens, [1] * seqs, prefix, 0, n)
    q[3] = float("nan")
    q[17, 5] = float("inf")
    q[40] = 1e30
    slots[3] = -1
    out = torch.full_like(q, 7.0)
    qb.kv_attention(q, cache, _i32(slots, cuda), _i32(lens, cuda), prefix=prefix, prefix_len=n, out=out)
    assert (out[3] == 7.0).all()
    keep = [i for i in range(seqs) if i not in (3, 17, 40)]
    check(out[keep], want[keep], tol[keep])
    assert qb.device_status() == qb.OK


def test_extreme_magnitudes(cuda):
    """Scales of K and V rows over sixty binary orders, queries of 1e-6 and 1e4, sharp
    softmaxes: the bound holds relative to what each row's own keys weigh."""
    import torch

    rng = _gen(8)
    heads, dim, rows = 8, 128, 96
    cache = _filled(rng, 4, rows, 1, dim, cuda)
    cache.k_scale.mul_(torch.exp2(torch.from_numpy(rng.integers(-6, 3, (4, rows, 1)).astype(np.float32)).to(cuda)))
    cache.v_scale[1].mul_(2.0 ** 30)
    cache.v_scale[2].mul_(2.0 ** -30)
    cache.v_scale[3, ::2].mul_(2.0 ** -12)
    q = _tensor(rng.standard_normal((4, heads, dim)) * np.array([1e-6, 1.0, 8.0, 0.3])[:, None, None], cuda)
    slots, lens = [0, 1, 2, 3], [96, 95, 64, 96]
    got = qb.kv_attention(q, cache, _i32(slots, cuda), _i32(lens, cuda))
    check(got, *attention64(q, cache, slots, lens, [1] * 4))
    # a scale of its own, and a negative one
    for scale in (0.5, -0.25, 0.0):
        got = qb.kv_attention(q, cache, _i32(slots, cuda), _i32(lens, cuda), scale=scale)
        check(got, *attention64(q, cache, slots, lens, [1] * 4, scale=scale))


def test_hidden_rows_may_hold_anything(cuda):
    """NaN and infinite scales behind a slot's length, in other slots, and in rows that only
    later tokens of the run see do not reach the rows that do not see them; nor do large ones."""
    rng = _gen(9)
    heads, dim, rows = 8, 128, 70
    cache = _filled(rng, 3, rows, 2, dim, cuda)
    prefix = _filled(rng, 2, 200, 2, dim, cuda)
    runs, slots, lens = [4, 1], [0, 2], [50, 20]
    q = _tensor(rng.standard_normal((5, heads, dim)), cuda)
    args = (_i32(slots, cuda), _i32(lens, cuda), _cu(runs, cuda))
    want, tol = attention64(q, cache, slots, lens, runs, prefix, 0, 150)
    for bad in (float("nan"), float("inf"), 1e30):
        cache.v_scale[0, 49] = bad      # only token 3 sees it
        cache.k_scale[0, 50:] = float("nan")
        cache.v_scale[0, 50:] = bad
        cache.k_scale[1] = cache.v_scale[1] = bad
        cache.v_scale[2, 20:] = bad
        prefix.v_scale[0, 150:] = bad
        prefix.k_scale[1] = bad
        got = qb.kv_attention(q, cache, *args, prefix=prefix, prefix_len=150).cpu()
        rows_of = [0, 1, 2, 4]
        check(got[rows_of], want[rows_of], tol[rows_of])


def test_padded_batch_and_bad_lengths(cuda):
    """Slot -1 and tokens behind the last run keep what out holds; so do a slot out of range
    and a length above max_len, which raise the status; the others get their values."""
    import torch

    rng = _gen(10)
    cache, prefix = _filled(rng, 4, 64, 2, 64, cuda), _filled(rng, 1, 300, 2, 64, cuda)
    q = _tensor(rng.standard_normal((6, 4, 64)), cuda)
    for pre in (0, 300):
        for slots, lens, status in (([2, -1, 0], [10, 5, 64], qb.OK), ([2, 4, 0], [10, 5, 64], qb.ERR_INVALID),
                                    ([2, 1, 0], [10, 65, 64], qb.ERR_INVALID), ([2, 1, 0], [10, -1, 64], qb.ERR_INVALID),
                                    ([2, -2, 0], [10, 3, 64], qb.ERR_INVALID)):
            out = torch.full((6, 4, 64), 7.0, device=cuda)
            qb.kv_attention(q, cache, _i32(slots, cuda), _i32(lens, cuda), _i32([0, 1, 3, 5], cuda),
                            prefix=prefix if pre else None, prefix_len=pre, out=out)
            assert qb.device_status() == status
            want, tol = attention64(q, cache, [2, -1, 0], [10, 0, 64], [1, 2, 2], prefix, 0, pre)
            rows_of = [0, 3, 4]
            check(out[rows_of], want[rows_of], tol[rows_of])
            assert (out[[1, 2, 5]] == 7.0).all()
    # the same with the prefix on tiles, and with one chunk a row (the first kernel writes the output)
    seqs = 160
    wide, far = _filled(rng, seqs, 40, 2, 64, cuda), _filled(rng, 1, 900, 2, 64, cuda)
    qq = _tensor(rng.standard_normal((seqs + 4, 8, 64)), cuda)
    slots, lens = list(range(seqs)), [int(v) for v in rng.integers(0, 41, seqs)]
    slots[5], slots[77], lens[100] = -1, seqs, 41
    for pre, launches in ((900, 3), (0, 1)):
        out = torch.full((seqs + 4, 8, 64), 7.0, device=cuda)
        n0 = qb.launch_count()
        qb.kv_attention(qq, wide, _i32(slots, cuda), _i32(lens, cuda), _i32(list(range(seqs + 1)), cuda),
                        prefix=far if pre else None, prefix_len=pre, max_len=40, out=out)
        assert qb.launch_count() - n0 == launches or not pre
        assert qb.device_status() == qb.ERR_INVALID
        left = [5, 77, 100] + list(range(seqs, seqs + 4))
        keep = [i for i in range(seqs) if i not in left]
        want, tol = attention64(qq[:seqs], wide, [s if i not in left else -1 for i, s in enumerate(slots)],
                                [min(v, 40) for v in lens], [1] * seqs, far, 0, pre)
        check(out[keep], want[keep], tol[keep])
        assert (out[left] == 7.0).all()
    out = torch.full((2, 4, 64), 7.0, device=cuda)
    qb.kv_attention(q[:2], cache, _i32([1, -1], cuda), _i32([60, 60], cuda), max_len=64, out=out)
    want, tol = attention64(q[:2], cache, [1, -1], [60, 0], [1, 1])
    check(out[:1], want[:1], tol[:1])
    assert (out[1] == 7.0).all() and qb.device_status() == qb.OK


def test_strided_queries_and_views_of_a_larger_cache(cuda):
    """q a column slice of a joined projection, out a slice with a stride of its own, the cache
    one layer of a [slots, layers, rows, heads, dim] tensor."""
    import torch

    rng = _gen(11)
    slots, layers, rows, heads, dim = 3, 4, 50, 2, 64
    k, v = (torch.from_numpy(rng.integers(-127, 128, (slots, layers, rows, heads, dim)).astype(np.int8)).to(cuda)
            for _ in range(2))
    ks, vs = (_tensor(rng.random((slots, layers, rows, heads)) * 0.02 + 0.001, cuda) for _ in range(2))
    layer = qb.KvCache.from_tensors(k[:, 2], v[:, 2], ks[:, 2], vs[:, 2])
    joined = _tensor(rng.standard_normal((3, 4 * heads * dim + 3)), cuda)
    q = joined[:, 1:1 + 2 * heads * dim]
    wide = torch.zeros(3, 2 * heads * dim + 5, device=cuda)
    out = wide[:, 5:]
    got = qb.kv_attention(q, layer, _i32([1, 2, 0], cuda), _i32([50, 9, 33], cuda), out=out)
    assert got.data_ptr() == out.data_ptr() and not wide[:, :5].any()
    check(out.reshape(3, 2 * heads, dim), *attention64(q.reshape(3, 2 * heads, dim), layer, [1, 2, 0], [50, 9, 33], [1] * 3))


def test_offsets_past_32_bits(cuda):
    """A cache of more than 2^32 codes: rows in its last slot are stored, read and attended."""
    import torch

    heads, dim, rows = 8, 128, 1 << 20
    k, v = (torch.empty((5, rows, heads, dim), dtype=torch.int8, device=cuda) for _ in range(2))
    ks, vs = (torch.empty((5, rows, heads), device=cuda) for _ in range(2))
    cache = qb.KvCache.from_tensors(k, v, ks, vs)
    rng = _gen(12)
    m, first = 100, rows - 100
    x, y = (_tensor(rng.standard_normal((m, heads, dim)), cuda) for _ in range(2))
    args = _i32([4], cuda), _i32([first], cuda), _i32([0, m], cuda)
    qb.kv_store(cache, x, y, *args)
    small = qb.KvCache(1, m, heads, dim)
    qb.kv_store(small, x, y, _i32([0], cuda), _i32([0], cuda), _i32([0, m], cuda))
    for name in ("k", "v", "k_scale", "v_scale"):
        assert torch.equal(getattr(cache, name)[4, first:], getattr(small, name)[0]), name
    assert torch.equal(qb.kv_load(cache, *args, n=m)[1], qb.kv_load(small, *(args[0] * 0, args[1] * 0), args[2], n=m)[1])
    # the slot's last rows as a prefix, through a view that starts before them
    q = _tensor(rng.standard_normal((2, heads, dim)), cuda)
    own = qb.KvCache(2, 4, heads, dim)
    ks[4, :first] = 0.0     # the rows before weigh as zeros: masked out by comparing with the exact answer
    tail = qb.KvCache.from_tensors(k[:, first:], v[:, first:], ks[:, first:], vs[:, first:])
    got = qb.kv_attention(q, own, _i32([0, 1], cuda), _i32([0, 0], cuda), prefix=tail, prefix_slot=4, prefix_len=m)
    check(got, *attention64(q, own, [0, 1], [0, 0], [1, 1], small, 0, m))
    del k, v, ks, vs, cache, tail
    torch.cuda.empty_cache()


def test_graphs_streams_and_the_three_together(cuda):
    """A serving step on a side stream (store the new rows, attend, read back), captured twice
    and replayed at the same time on two streams with other lengths: each graph has a
    workspace of its own, and both give what eager calls give."""
    import torch

    rng = _gen(13)
    heads, kv_heads, dim, b, rows = 16, 2, 128, 6, 400
    prefix = _filled(rng, 1, 900, kv_heads, dim, cuda)
    sides = []
    for i in range(2):
        cache = _filled(rng, b, rows, kv_heads, dim, cuda)
        slots = _i32([int(s) for s in rng.permutation(b)], cuda)
        state = {"cache": cache, "slots": slots, "starts": _i32([20 * j + i for j in range(b)], cuda),
                 "lens": _i32([20 * j + i + 1 for j in range(b)], cuda),
                 "q": _tensor(rng.standard_normal((b, heads, dim)), cuda),
                 "k": _tensor(rng.standard_normal((b, kv_heads, dim)), cuda),
                 "v": _tensor(rng.standard_normal((b, kv_heads, dim)), cuda)}
        sides.append(state)

    def step(s):
        qb.kv_store(s["cache"], s["k"], s["v"], s["slots"], s["starts"])
        out = qb.kv_attention(s["q"], s["cache"], s["slots"], s["lens"], prefix=prefix, prefix_len=900)
        return out, qb.kv_load(s["cache"], s["slots"], s["starts"])

    graphs, outs = [], []
    stream = torch.cuda.Stream(cuda)
    for s in sides:
        with torch.cuda.stream(stream):
            step(s)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            outs.append(step(s))
        graphs.append(g)
    streams = [torch.cuda.Stream(cuda) for _ in range(2)]
    for round_ in range(3):
        for s in sides:
            s["starts"].add_(7)
            s["lens"].add_(7)
            s["k"].normal_()
            s["v"].normal_()
            s["q"].normal_()
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                for _ in range(4):
                    g.replay()
        torch.cuda.synchronize()
        for s, (out, (kb, vb)) in zip(sides, outs):
            kept = out.clone(), kb.clone(), vb.clone()
            eager, (ke, ve) = step(s)
            for a, e in zip(kept, (eager, ke, ve)):
                assert torch.equal(a, e), round_
            check(kept[0], *attention64(s["q"], s["cache"], s["slots"].tolist(), s["lens"].tolist(), [1] * b, prefix, 0, 900))
            codes, scale = quantise(s["k"].cpu().numpy())
            assert np.array_equal(kept[1].cpu().numpy(), codes * scale[..., None])
    # an explicit stream
    s = sides[0]
    other = torch.cuda.Stream(cuda)
    out = qb.kv_attention(s["q"], s["cache"], s["slots"], s["lens"], prefix=prefix, prefix_len=900, stream=other)
    other.synchronize()
    assert torch.equal(out, outs[0][0])
    del graphs
    assert qb.device_status() == qb.OK


def test_refusals_on_the_device(cuda):
    import torch

    cache = qb.KvCache(2, 8, 2, 64)
    q, one = torch.zeros(1, 4, 64, device=cuda), _i32([0], cuda)
    with pytest.raises(qb.QrafError, match="multiple of 2 KV heads"):
        qb.kv_attention(torch.zeros(1, 3, 64, device=cuda), cache, one, one)
    with pytest.raises(qb.QrafError, match="max_len 9"):
        qb.kv_attention(q, cache, one, one, max_len=9)
    with pytest.raises(qb.QrafError, match="prefix slot 2"):
        qb.kv_attention(q, cache, one, one, prefix=cache, prefix_slot=2, prefix_len=4)
    with pytest.raises(qb.QrafError, match="prefix slot 0 or length 9"):
        qb.kv_attention(q, cache, one, one, prefix=cache, prefix_len=9)
    with pytest.raises(qb.QrafError, match="heads of 32"):
        qb.kv_attention(q, cache, one, one, prefix=qb.KvCache(1, 8, 2, 32), prefix_len=4)
    with pytest.raises(qb.QrafError, match="multiple of 16"):
        qb.KvCache(1, 4, 2, 24)
    lib, d = qb.lib, cache.desc
    import ctypes as C

    long, ints, many = qb.KvCache(1, 4096, 8, 64), _i32([0] * 64, cuda), torch.zeros(64, 64, 64, device=cuda)
    size = C.c_uint64()
    assert lib.qraf_cuda_kv_attention_workspace(C.byref(long.desc), 0, 64, 64, 64, 0, 4096, C.byref(size)) == qb.OK
    for given, at in ((size.value - 1, many.data_ptr()), (size.value, many.data_ptr() + 4), (size.value, None)):
        rc = lib.qraf_cuda_kv_attention(C.byref(long.desc), None, 0, 0, many.data_ptr(), many.data_ptr(), 0, 4096, 4096, 64, 64,
                                        ints.data_ptr(), ints.data_ptr(), None, 64, 4096, 1.0, at, given, None)
        assert rc == qb.ERR_INVALID and "workspace" in qb.last_error()
    with pytest.raises(ValueError, match="float64"):
        qb.kv_store(cache, torch.zeros(1, 2, 64, device=cuda).double(), torch.zeros(1, 2, 64, device=cuda).double(), one, one)
    with pytest.raises(ValueError, match="int32"):
        qb.kv_attention(q, cache, one.long(), one)
    with pytest.raises(ValueError, match="without cu"):
        qb.kv_attention(q, cache, _i32([0, 1], cuda), _i32([0, 1], cuda))
    with pytest.raises(ValueError, match="cu needs 2"):
        qb.kv_attention(q, cache, one, one, _i32([0, 1, 1], cuda))
    with pytest.raises(ValueError, match="contiguous"):
        qb.kv_attention(torch.zeros(1, 64, 4, device=cuda).transpose(1, 2), cache, one, one)
    assert qb.kv_attention(q[:0], cache, one[:0], one[:0]).shape == (0, 4, 64)
    assert qb.device_status() == qb.OK
