"""kv_attention's prefix tiles where a CTA has many of them: sums that start anew, widely spread and
peaked scores, against 64-bit forms."""
from __future__ import annotations

import numpy as np
import pytest

import qraf_b200 as qb
from test_gpu_kv import DTYPES, attention64, _filled, _gen, _i32, _tensor, check, quantise

pytestmark = pytest.mark.gpu

# 160 tokens of 16 query heads a KV head are 20 tiles of 128 rows, and with 7 KV heads 140 (tile, head)
# units: one CTA has a whole unit, so every key of the prefix
SEQS, KV_HEADS, GROUP, DIM = 160, 7, 16, 64


def prefix64(q, prefix, n, scale):
    """(out, tolerance) of the prefix alone, in 64 bits: attention64's bound, but the weighted sum is
    formed 16 keys and one of two parts at a time (n / 8 accumulations, each off by at most a last bit)
    and joined from at most 64 records, whatever the type."""
    import torch

    q64 = q.double().view(q.shape[0], KV_HEADS, GROUP, DIM)
    k, v = (getattr(prefix, s)[0, :n].double() * getattr(prefix, s + "_scale")[0, :n].double().unsqueeze(-1) for s in "kv")
    out, tol = torch.empty_like(q64), torch.empty_like(q64)
    for h in range(KV_HEADS):
        s = torch.einsum("tgd,kd->tgk", q64[:, h], k[:, h]) * scale
        a = (torch.einsum("tgd,kd->tgk", q64[:, h].abs(), k[:, h].abs()) * abs(scale)).amax(-1, keepdim=True)
        p = torch.softmax(s, -1)
        out[:, h] = p @ v[:, h]
        ds = a * (2 * DIM / 16 + 8) * 2.0 ** -23
        floor = n * v[:, h].abs().max() * 2.0 ** -31
        tol[:, h] = (p @ v[:, h].abs()) * (2 * ds + 2.0 ** -21 + (n / 8 + 64) * 2.0 ** -23) + floor
    return out.view(q.shape).cpu().numpy(), tol.view(q.shape).cpu().numpy()


def _attend(q, prefix, n, cuda, **kw):
    """The call with own slots of no rows; the prefix is on tiles: three launches."""
    cache = qb.KvCache(1, 16, KV_HEADS, DIM)
    slots = _i32([0] * len(q), cuda)
    before = qb.launch_count()
    got = qb.kv_attention(q, cache, slots, slots * 0, prefix=prefix, prefix_len=n, **kw)
    assert qb.launch_count() - before == 3
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [5120, 8970])
def test_sorted_scores_over_many_sums(cuda, dtype, n):
    """Keys sorted by their scores, falling (each new sum starts far below the maximum so far) and
    rising, over 40 and 71 tiles: the falls reach several hundred binary orders."""
    import torch

    rng = _gen(n)
    prefix = _filled(rng, 1, n, KV_HEADS, DIM, cuda)
    base = rng.standard_normal(DIM)
    q = _tensor(base + 0.1 * rng.standard_normal((SEQS, KV_HEADS * GROUP, DIM)), cuda, dtype)
    for falling in (True, False):
        s = torch.einsum("d,nhd->nh", torch.from_numpy(base).to(cuda).float(), prefix.k[0].float() * prefix.k_scale[0].unsqueeze(-1))
        for h in range(KV_HEADS):
            at = s[:, h].argsort(descending=falling)
            for t in (prefix.k, prefix.k_scale, prefix.v, prefix.v_scale):
                t[0, :, h] = t[0, at, h]
        for scale in (1.0, 2.0, 4.0):
            check(_attend(q, prefix, n, cuda, scale=scale), *prefix64(q, prefix, n, scale), dtype)
    assert qb.device_status() == qb.OK


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gap", [90, 120, 125, 126, 127, 128, 130, 300])
@pytest.mark.parametrize("place", [5, 5000])
def test_one_key_far_above_the_others(cuda, dtype, gap, place):
    """A key in the first or the last tile that scores `gap` binary orders above the level of the
    others: every row is that key's value."""
    import torch

    n, rng = 5120, _gen(gap)
    prefix = _filled(rng, 1, n, KV_HEADS, DIM, cuda)
    base = np.sign(rng.standard_normal(DIM))
    q = _tensor(base * (1 + 0.01 * rng.random((SEQS, KV_HEADS * GROUP, 1))), cuda, dtype)
    prefix.k_scale.mul_(0.01)
    prefix.k[0, place] = torch.from_numpy((127 * base).astype(np.int8)).to(cuda)
    prefix.k_scale[0, place] = gap * np.log(2.0) / (127 * DIM)
    check(_attend(q, prefix, n, cuda, scale=1.0), *prefix64(q, prefix, n, 1.0), dtype)
    assert qb.device_status() == qb.OK


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [float("inf"), 3e38])
@pytest.mark.parametrize("dead", [128, 200, 1500])
def test_a_prefix_that_begins_with_scores_of_minus_infinity(cuda, dtype, bad, dead):
    """Whole tiles whose scores are below every fp32 number, before keys some 300 binary orders below
    zero: the rows are what those keys give, as if the others were not there."""
    import torch

    n, rng = 2000, _gen(dead)
    prefix = _filled(rng, 1, n, KV_HEADS, DIM, cuda)
    base = np.sign(rng.standard_normal(DIM))
    k = torch.from_numpy((-127 * base).astype(np.int8)).to(cuda)
    prefix.k[0] = torch.where(prefix.k[0] % 3 == 0, 0, k)
    prefix.k_scale.fill_(300 * np.log(2.0) / (127 * DIM * 2 / 3))
    prefix.k[0, :dead] = k
    prefix.k_scale[0, :dead] = bad
    q = _tensor(base * (1 + 0.01 * rng.random((SEQS, KV_HEADS * GROUP, 1))), cuda, dtype)
    rest = qb.KvCache.from_tensors(*(t[:, dead:].clone() for t in (prefix.k, prefix.v, prefix.k_scale, prefix.v_scale)))
    check(_attend(q, prefix, n, cuda, scale=1.0), *prefix64(q, rest, n - dead, 1.0), dtype)
    assert qb.device_status() == qb.OK


def _peaked(cuda, dtype, n, places):
    """Queries that each attend to one key alone: (q, prefix, exact outputs).  Token t's key lies 300
    binary orders above its next, so the answer is that key's value."""
    import torch

    rng, m = _gen(n), len(places)
    prefix = _filled(rng, 1, n, KV_HEADS, DIM, cuda)
    prefix.k_scale.mul_(2.0 ** -12)
    base = np.sign(rng.standard_normal((m, DIM)))
    most = np.abs(base @ base.T - DIM * np.eye(m)).max()   # of another key's codes with a query
    assert most < 0.8 * DIM
    place = torch.tensor(places, device=cuda)
    prefix.k[0, place] = torch.from_numpy(127 * base).to(cuda).to(torch.int8).unsqueeze(1)
    prefix.k_scale[0, place] = 2000.0 / (127 * DIM)
    of = np.arange(SEQS) % m
    q = _tensor(np.broadcast_to(base[of, None], (SEQS, KV_HEADS * GROUP, DIM)), cuda, dtype)
    v = prefix.v[0, place].double() * prefix.v_scale[0, place].double().unsqueeze(-1)
    return q, prefix, v[torch.from_numpy(of).to(cuda)].repeat_interleave(GROUP, 1)


def _check_rounded(got, want, rel, floor):
    """got is want, off by at most rel of itself and floor, rounded once."""
    import torch

    tol = want.abs() * rel + floor
    low, high = ((want + s * tol).to(got.dtype) for s in (-1, 1))
    bad = ~((low <= got) & (got <= high))
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} values off, worst {float(((got.double() - want).abs() / want.abs()).max()):.3g} of itself"


@pytest.mark.parametrize("dtype", DTYPES)
def test_weights_of_peaked_rows_keep_22_bits(cuda, dtype):
    """Rows that attend to one key behind a short prefix.  A weight w = p vs is rounded to fp32 (2^-24)
    and split (the lower part's rounding: 2^-22 of w at most); its two products with a code are exact
    and their sum loses a last bit (2^-23) at both accumulations; p is the same number in the sum of
    weights, which the others do not reach; the join's division and two products round to 2^-24 each:
    below 2^-20 together, and as much again to spare.  Every weight's lower part may end at 2^-31 of
    the largest vs."""
    q, prefix, want = _peaked(cuda, dtype, 300, [0, 77, 128, 129, 200, 255, 256, 299])
    floor = 127 * float(prefix.v_scale.max()) * 2.0 ** -31
    _check_rounded(_attend(q, prefix, 300, cuda, scale=1.0), want, 2.0 ** -19, floor)
    assert qb.device_status() == qb.OK


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [300, 5120])
def test_peaked_rows_are_as_exact_as_their_weight(cuda, dtype, n):
    """One key has a row's weight, in the first tile, in the last, or between, and the tensor cores add
    exact zeros for the others: the same steps as above, with nothing for their accumulations, and a
    term's sum added to the record (2^-24)."""
    last = (n - 1) // 128 * 128
    q, prefix, want = _peaked(cuda, dtype, n, [0, 77, 127, 128, 200, n // 2, last, n - 1])
    floor = 127 * float(prefix.v_scale.max()) * 2.0 ** -31
    _check_rounded(_attend(q, prefix, n, cuda, scale=1.0), want, 2.0 ** -20, floor)
    assert qb.device_status() == qb.OK


@pytest.mark.parametrize("n", [5120, 20481])
def test_even_weights_lose_nothing_with_length(cuda, n):
    """Keys of about the same weight and positive values, so that nothing cancels.  In a term of 8 tiles
    O grows evenly over 8 x 16 accumulations, each losing at most a last bit of its size: 64 x 2^-23.
    The terms' additions, and the sum of weights' (64 pairs a tile, growing likewise, and a tile's sum
    to the ones before), round to nearest: at most (n / 1024 + 32 + n / 256) / 2 x 2^-23 in their mean
    growth.  Weights are off by 2^-21 and twice the scores' bound ((2 dim / 16 + 8) 2^-23 of sum |q| |k|
    here), the rest by 8 x 2^-23."""
    import torch

    rng = _gen(n)
    prefix = _filled(rng, 1, n, KV_HEADS, DIM, cuda)
    prefix.v.copy_(prefix.v.abs().clamp_(min=30))
    q = _tensor(0.02 * rng.standard_normal((SEQS, KV_HEADS * GROUP, DIM)), cuda)
    got = _attend(q, prefix, n, cuda, scale=DIM ** -0.5).double().cpu().numpy()
    want, _ = prefix64(q, prefix, n, DIM ** -0.5)
    k = prefix.k[0].double().abs() * prefix.k_scale[0].double().unsqueeze(-1)
    a = float((q.double().abs().amax(1).amax(0) @ k.amax(0).amax(0))) * DIM ** -0.5
    rel = (64 + (n / 1024 + 32 + n / 256) / 2 + 4 + 2 * a * (2 * DIM / 16 + 8) + 8) * 2.0 ** -23
    off = np.abs(got - want) / want
    assert off.max() <= rel, f"{off.max():.3g}, mean {off.mean():.3g}, against {rel:.3g}"
    assert qb.device_status() == qb.OK


@pytest.mark.parametrize("launches,seqs,heads,kv_heads,dim,rows,run", [
    (1, 1, 16, 2, 128, 1024, 1), (2, 1, 16, 2, 128, 1025, 1), (2, 1, 64, 8, 128, 20000, 1), (2, 4, 16, 2, 64, 5000, 1),
    (1, 16, 64, 8, 128, 2048, 1), (2, 16, 64, 8, 128, 9000, 1), (1, 1, 16, 2, 256, 1024, 1), (2, 1, 16, 2, 256, 1500, 1),
    (1, 4, 16, 2, 256, 500, 5), (2, 4, 16, 2, 256, 900, 5)])
def test_long_own_rows_use_every_sm(cuda, launches, seqs, heads, kv_heads, dim, rows, run):
    """Own rows without a prefix: one launch of clusters while they are short, or while the clusters
    leave no SM empty, else the chunked kernel and its join."""
    rng = _gen(rows)
    cache = _filled(rng, seqs, rows, kv_heads, dim, cuda)
    lens = [rows - 3 * b for b in range(seqs)]
    q = _tensor(rng.standard_normal((seqs * run, heads, dim)), cuda)
    args = q, cache, _i32(list(range(seqs)), cuda), _i32(lens, cuda), _i32([run * b for b in range(seqs + 1)], cuda) if run > 1 else None
    before = qb.launch_count()
    got = qb.kv_attention(*args)
    assert qb.launch_count() - before == launches
    check(got, *attention64(q, cache, list(range(seqs)), lens, [run] * seqs))
    assert qb.device_status() == qb.OK


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("launches,seqs,heads,kv_heads,dim,n", [(1, 70, 16, 2, 128, 700), (3, 90, 24, 3, 96, 1100), (1, 80, 16, 2, 48, 513),
                                                                (3, 70, 16, 2, 128, 4111), (3, 150, 8, 2, 48, 1900),
                                                                (2, 200, 16, 2, 256, 700), (2, 200, 16, 2, 64, 0)])
def test_rows_that_allow_no_wide_access(cuda, dtype, launches, seqs, heads, kv_heads, dim, n):
    """q and out column slices with odd offsets and odd strides, own slots and the prefix layers of a larger
    cache, on each plan; what lies around out stays."""
    import torch

    rng = _gen(dim)
    rows, layers, width = 40, 3, heads * dim

    def layer(slots, length):
        k, v = (torch.from_numpy(rng.integers(-127, 128, (slots, layers, length, kv_heads, dim)).astype(np.int8)).to(cuda) for _ in "kv")
        ks, vs = (_tensor(rng.random((slots, layers, length, kv_heads)) * 0.02 + 0.001, cuda) for _ in "kv")
        return qb.KvCache.from_tensors(k[:, 1], v[:, 1], ks[:, 1], vs[:, 1])

    cache, prefix = layer(seqs, rows), layer(3, n + 5) if n else None
    joined = _tensor(rng.standard_normal((seqs, width + 7)), cuda, dtype)
    q = joined[:, 1:1 + width]
    around = torch.full((seqs, width + 9), 7.0, device=cuda, dtype=q.dtype)
    out = around[:, 3:3 + width]
    slots, lens = [int(v) for v in rng.permutation(seqs)], [int(v) for v in rng.integers(0, rows + 1, seqs)]
    before = qb.launch_count()
    qb.kv_attention(q, cache, _i32(slots, cuda), _i32(lens, cuda), prefix=prefix, prefix_slot=2 if n else 0, prefix_len=n, out=out)
    assert qb.launch_count() - before == launches or not n
    assert (around[:, :3] == 7).all() and (around[:, 3 + width:] == 7).all()
    shape = (seqs, heads, dim)
    check(out.reshape(shape), *attention64(q.reshape(shape), cache, slots, lens, [1] * seqs, prefix, 2, n), dtype)
    assert qb.device_status() == qb.OK


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("seqs,heads,kv_heads,dim,n,rows", [(3, 16, 2, 128, 100, 20), (70, 16, 2, 128, 1500, 20), (200, 16, 2, 256, 700, 20),
                                                            (200, 16, 2, 64, 0, 300), (16, 16, 2, 128, 30000, 20)])
def test_what_is_not_a_number_stays_so(cuda, dtype, seqs, heads, kv_heads, dim, n, rows):
    """A query of NaN, one with an infinity, and a K scale of NaN that some rows see make those rows' heads
    NaN and leave every other one as it is, on each plan."""
    import torch

    rng = _gen(seqs)
    cache, prefix = _filled(rng, seqs, rows, kv_heads, dim, cuda), _filled(rng, 1, n, kv_heads, dim, cuda) if n else None
    q = _tensor(rng.standard_normal((seqs, heads, dim)), cuda, dtype)
    slots, lens = list(range(seqs)), [rows] * seqs
    want, tol = attention64(q, cache, slots, lens, [1] * seqs, prefix, 0, n)
    lost = torch.zeros(seqs, heads, dtype=torch.bool)
    q[0] = float("nan")
    lost[0] = True
    q[1, 3] = float("inf")
    lost[1, 3] = True
    q[2, 5, 7] = float("nan")
    lost[2, 5] = True
    cache.k_scale[1, rows - 1, 1] = float("nan")
    lost[1, heads // 2:] = True
    got = qb.kv_attention(q, cache, _i32(slots, cuda), _i32(lens, cuda), prefix=prefix, prefix_len=n).cpu()
    assert got[lost].isnan().all()
    keep = ~lost
    check(got[keep], want[keep.numpy()], tol[keep.numpy()], dtype)
    assert qb.device_status() == qb.OK


def test_two_streams_behind_one_prefix(cuda):
    """Two batches behind the same prefix, at the same time on two streams, eagerly and as captured
    calls, with several sums a stretch: each gives what it gives alone."""
    import torch

    rng = _gen(31)
    seqs, heads, kv_heads, dim, n = 64, 64, 8, 128, 9000
    prefix = _filled(rng, 1, n, kv_heads, dim, cuda)
    sides = []
    for i in range(2):
        cache = _filled(rng, seqs, 30, kv_heads, dim, cuda)
        q = _tensor(rng.standard_normal((seqs, heads, dim)), cuda, "float32" if i else "bfloat16")
        args = q, cache, _i32(list(range(seqs)), cuda), _i32([int(v) for v in rng.integers(0, 31, seqs)], cuda)
        sides.append((args, qb.kv_attention(*args, prefix=prefix, prefix_len=n)))
    streams = [torch.cuda.Stream(cuda) for _ in sides]
    torch.cuda.synchronize()
    outs = [[] for _ in sides]
    for _ in range(5):
        for (args, _), st, got in zip(sides, streams, outs):
            got.append(qb.kv_attention(*args, prefix=prefix, prefix_len=n, stream=st))
    torch.cuda.synchronize()
    graphs = []
    for (args, _), st in zip(sides, streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            out = qb.kv_attention(*args, prefix=prefix, prefix_len=n)
        graphs.append((g, out))
    for _ in range(5):
        for (g, _), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for (_, want), got, (_, replayed) in zip(sides, outs, graphs):
        assert all(torch.equal(g, want) for g in got) and torch.equal(replayed, want)
    del graphs
    assert qb.device_status() == qb.OK


@pytest.mark.parametrize("seqs,heads,kv_heads,dim,rows,n", [(1700, 8, 1, 64, 4096, 0), (1300, 16, 1, 128, 2048, 0), (900, 4, 2, 256, 2000, 0),
                                                            (400, 16, 4, 256, 16, 3000), (16, 64, 8, 128, 2000, 0)])
def test_own_rows_lose_nothing_with_length(cuda, seqs, heads, kv_heads, dim, rows, n):
    """Keys of about the same weight and positive values, in chunks of up to thousands of keys (every
    warp has work without cutting finer), in one launch, and behind a prefix by 16 rows.  Sums round to
    nearest, which has no preferred sign: over thousands of rows the mean of the signed errors is far
    below a last bit (2^-23).  Left in the tensor cores' accumulator, a sum of k keys loses some
    4e-9 k of itself."""
    import torch

    rng = _gen(dim)

    def cache_of(slots, length):
        c = qb.KvCache(slots, length, kv_heads, dim)
        c.k.random_(-127, 128)
        c.v.random_(30, 128)
        c.k_scale.uniform_(0.005, 0.01)
        c.v_scale.uniform_(0.005, 0.01)
        return c

    torch.manual_seed(dim)
    cache, prefix = cache_of(seqs, rows), cache_of(1, n) if n else None
    q = _tensor(0.02 * rng.standard_normal((seqs, heads, dim)), cuda)
    got = qb.kv_attention(q, cache, _i32(list(range(seqs)), cuda), _i32([rows] * seqs, cuda), prefix=prefix, prefix_len=n)
    off = []
    for t in range(0, seqs, max(1, seqs * heads // 2400)):
        k, v = (getattr(cache, s)[t].double() * getattr(cache, s + "_scale")[t].double().unsqueeze(-1) for s in "kv")
        if n:
            far = [getattr(prefix, s)[0].double() * getattr(prefix, s + "_scale")[0].double().unsqueeze(-1) for s in "kv"]
            k, v = torch.cat([far[0], k]), torch.cat([far[1], v])
        s = torch.einsum("hgd,khd->hgk", q[t].double().view(kv_heads, -1, dim), k) * dim ** -0.5
        want = torch.einsum("hgk,khd->hgd", torch.softmax(s, -1), v).reshape(heads, dim)
        off.append((got[t].double() - want) / want)
    off = torch.stack(off)
    assert off.mean().abs() < 2.0 ** -23, f"mean {float(off.mean()):.3g}, worst {float(off.abs().max()):.3g}"
    assert qb.device_status() == qb.OK


@pytest.mark.parametrize("seqs,heads,kv_heads,dim,rows", [(3, 8, 1, 256, 300), (200, 16, 2, 256, 300), (3, 16, 1, 128, 700), (300, 8, 2, 192, 64)])
def test_scores_of_sharp_rows(cuda, seqs, heads, kv_heads, dim, rows):
    """Scores of some 100 that are sums of like signs, where what a score loses counts in full: two keys
    of the same score but for a few last bits, and their values opposite, so that the output is the
    difference of two weights of a half.  A score is off by at most the 8 accumulations of each 64 of its
    products (2^-23 of their sum each), dim / 64 additions and four roundings beside (2^-24 each) and the
    queries' 22 bits (2^-22): (8 + dim / 128 + 6) 2^-23 of sum |q| |k| together."""
    import torch

    rng = _gen(dim)
    cache = qb.KvCache(seqs, rows, kv_heads, dim)
    codes = torch.from_numpy(rng.integers(90, 128, (seqs, 2, kv_heads, dim)).astype(np.int8)).to(cuda)
    at = [rows // 3, rows - 1]
    cache.k[:, at] = codes
    cache.k_scale.fill_(1e-6)
    cache.k_scale[:, at] = 100.0 / (108 * dim)
    v = torch.from_numpy(rng.integers(1, 128, (seqs, kv_heads, dim)).astype(np.int8)).to(cuda)
    cache.v[:, at[0]], cache.v[:, at[1]] = v, -v
    cache.v_scale.fill_(0.01)
    q = _tensor(1 + 0.05 * rng.random((seqs, heads, dim)), cuda)
    got = qb.kv_attention(q, cache, _i32(list(range(seqs)), cuda), _i32([rows] * seqs, cuda), scale=1.0).double()
    group = heads // kv_heads
    k = codes.double() * cache.k_scale[:, at].double().unsqueeze(-1)
    s = torch.einsum("thgd,tkhd->thgk", q.double().view(seqs, kv_heads, group, dim), k)
    w = torch.softmax(s, -1)
    size = (v.double() * float(cache.v_scale[0, 0, 0]))[:, :, None]
    want = ((w[..., 0] - w[..., 1]).unsqueeze(-1) * size).reshape(seqs, heads, dim)
    ds = s.max() * (8 + dim / 128 + 6) * 2.0 ** -23
    tol = (size * (ds + 2.0 ** -20)).expand(-1, -1, group, -1).reshape(seqs, heads, dim)
    assert ((got - want).abs() <= tol).all(), f"{float(((got - want).abs() / tol).max()):.3g} of the bound"
    assert qb.device_status() == qb.OK


@pytest.mark.parametrize("seqs,heads,kv_heads,dim,n", [(3, 16, 2, 128, 0), (500, 16, 2, 64, 0), (3, 16, 2, 128, 100), (64, 64, 8, 128, 9000),
                                                       (200, 16, 2, 256, 700), (7, 8, 1, 32, 300000)])
def test_a_prefix_and_no_own_rows_at_all(cuda, seqs, heads, kv_heads, dim, n):
    """max_len 0: the prefix alone on each plan, in a workspace of exactly the stated size that holds
    anything beforehand, and zeros without one."""
    import ctypes as C

    import torch

    rng = _gen(n)
    cache, prefix = _filled(rng, seqs, 4, kv_heads, dim, cuda), _filled(rng, 1, max(n, 1), kv_heads, dim, cuda)
    q = _tensor(rng.standard_normal((seqs, heads, dim)), cuda)
    slots, lens = _i32(list(range(seqs)), cuda), _i32([0] * seqs, cuda)
    want, tol = attention64(q, cache, list(range(seqs)), [0] * seqs, [1] * seqs, prefix, 0, n)
    check(qb.kv_attention(q, cache, slots, lens, prefix=prefix, prefix_len=n, max_len=0), want, tol)
    size = C.c_uint64()
    qb.check(qb.lib.qraf_cuda_kv_attention_workspace(C.byref(cache.desc), n, seqs, heads, seqs, 0, 0, C.byref(size)))
    room = torch.full((size.value + 512,), 0xFF, dtype=torch.uint8, device=cuda)   # NaN in every word
    out = torch.full_like(q, 7.0)
    qb.check(qb.lib.qraf_cuda_kv_attention(C.byref(cache.desc), C.byref(prefix.desc), 0, n, q.data_ptr(), out.data_ptr(), 0, heads * dim,
                                           heads * dim, seqs, heads, slots.data_ptr(), lens.data_ptr(), None, seqs, 0, dim ** -0.5,
                                           room.data_ptr() + 256, size.value, torch.cuda.current_stream().cuda_stream))
    check(out, want, tol)
    assert (room[:256] == 0xFF).all() and (room[256 + size.value:] == 0xFF).all()
    assert qb.device_status() == qb.OK
