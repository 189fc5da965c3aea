"""The serving operators around the int8 KV cache, with their inputs and their plain forms.

Four operators, in the order in which a serving loop runs them:

  kv      rows of K and V are quantised into a cache of int8 codes with one fp32 scale per
          (row, KV head) as they are written, and read back as numbers
  attn    attention of a batch whose sequences share a long prefix: the prefix's rows are read
          once for all of them, then each sequence's own rows of its slot (one new token a
          sequence, or a run of drafted tokens, causal among themselves)
  probs   probabilities of logits at a temperature
  verify  drafted tokens accepted or replaced against the target's probabilities, from given
          uniform random numbers

``own`` false: elementary torch operations.  ``own`` true: the calls of qraf_b200.
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # one new token for each of 32 sequences of a small decoder (2 KV heads of 128): the
        # store of every decode step, where latency counts
        _kv("kv decode 32x2x128", "f32", 32, 1, 2, 128, 256),
        # odd sizes in 16 bits: prompts of uneven lengths, 5 heads of 80
        _kv("kv ragged 7x~330x5x80 f16", "f16", 7, 437, 5, 80, 600),
        # prompts of eight sequences written at once, 8 KV heads of 128
        _kv("kv prefill 8x~1.5k x8x128", "f32", 8, 2048, 8, 128, 4096),
        # a few answers to one question: small batch, short prefix, odd lengths
        _attn("attn 4 seqs 16/2x128 p777", "f32", 4, 1, 16, 2, 128, 777, 93),
        # a continuous batch behind one system prompt, small decoder
        _attn("attn 32 seqs 16/2x128 p4096", "f32", 32, 1, 16, 2, 128, 4096, 512),
        # a long shared document, few readers, 16-bit activations
        _attn("attn 8 seqs 16/2x128 p65536", "bf16", 8, 1, 16, 2, 128, 65536, 300),
        # drafted runs (up to 5 tokens a sequence) behind a prefix, large decoder
        _attn("attn 16 seqs x5 64/8x128 p2011", "f32", 16, 5, 64, 8, 128, 2011, 700),
        # a full batch of the large decoder behind a long prompt
        _attn("attn 64 seqs 64/8x128 p8192", "f32", 64, 1, 64, 8, 128, 8192, 1024),
        # the target's distributions of one sequence's drafts, and of a batch's
        {"name": "probs 5x151936", "op": "probs", "rows": 5, "vocab": 151936, "temperature": 0.7},
        {"name": "probs 320x32003", "op": "probs", "rows": 320, "vocab": 32003, "temperature": 1.0},
        # four drafts of one sequence; six drafts of a batch with uneven counts
        {"name": "verify 1x4x151936", "op": "verify", "seqs": 1, "drafts": 4, "vocab": 151936, "ragged": False},
        {"name": "verify 64x6x151936", "op": "verify", "seqs": 64, "drafts": 6, "vocab": 151936, "ragged": True},
    ]


def _kv(name, dtype, seqs, run, kv_heads, head_dim, rows):
    return {"name": name, "op": "kv", "dtype": dtype, "seqs": seqs, "run": run, "kv_heads": kv_heads,
            "head_dim": head_dim, "rows": rows}


def _attn(name, dtype, seqs, run, heads, kv_heads, head_dim, prefix, own_rows):
    return {"name": name, "op": "attn", "dtype": dtype, "seqs": seqs, "run": run, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "prefix": prefix, "own_rows": own_rows}


def draw(rng):
    def log(lo, hi):
        return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.99))))))

    op = rng.choice(["kv", "attn", "attn", "probs", "verify"])
    dtype = rng.choice(["f32", "f32", "f16", "bf16"])
    if op == "kv":
        seqs, run = log(1, 64), log(1, 2048)
        kv_heads, head_dim = rng.choice([1, 2, 3, 4, 5, 8]), 16 * rng.randint(1, 16)
        while seqs * run * kv_heads * head_dim > 16 << 20:
            run = max(1, run // 2)
        c = _kv("", dtype, seqs, run, kv_heads, head_dim, run + log(1, 2048))
    elif op == "attn":
        seqs, run = log(1, 64), rng.choice([1, 1, 1, 2, 5, 9])
        kv_heads, head_dim = rng.choice([1, 2, 4, 8]), rng.choice([32, 64, 80, 96, 128, 128, 128, 256])
        heads = kv_heads * rng.choice([1, 3, 4, 5, 7, 8, 8, 16])
        prefix, own_rows = rng.choice([0, log(1, 32768), log(64, 16384)]), run + log(1, 1500)
        while (seqs * run * heads * head_dim * (prefix + own_rows) > 4 << 30
               or seqs * own_rows * kv_heads * head_dim > 64 << 20):
            seqs, prefix = max(1, seqs // 2), prefix // 2
        c = _attn("", dtype, seqs, run, heads, kv_heads, head_dim, prefix, own_rows)
    elif op == "probs":
        vocab = log(17, 200000)
        c = {"op": "probs", "rows": min(log(1, 512), max(1, (24 << 20) // vocab)), "vocab": vocab,
             "temperature": rng.choice([0.3, 0.7, 1.0, 1.5])}
    else:
        drafts, vocab = rng.randint(1, 8), log(17, 200000)
        c = {"op": "verify", "seqs": min(log(1, 64), max(1, (80 << 20) // vocab // (2 * drafts + 1))), "drafts": drafts,
             "vocab": vocab, "ragged": rng.choice([False, True])}
    c.pop("name", None)
    return c


# ── sizes that follow from a case alone ─────────────────────────────────────
def _spread(i):
    """A fixed fraction in [0, 1) for item i."""
    return (i * 2654435761 % (1 << 32)) / (1 << 32)


def _runs(c):
    """New rows of each sequence: 1, or between 1 and `run`."""
    return [c["run"] - int(_spread(b) * min(c["run"], 3 + c["run"] // 2)) for b in range(c["seqs"])]


def _own_lens(c):
    """Rows of each sequence's own slot after its new rows: from the run's length to `own_rows`."""
    return [n + int((1 - _spread(3 * b + 1) ** 2) * (c["own_rows"] - n)) for b, n in enumerate(_runs(c))]


def work(c):
    if c["op"] == "kv":
        n = sum(_runs(c)) * c["kv_heads"]
        e = _BYTES[c["dtype"]]
        # K and V in, codes and scales out, the values they stand for out
        return {"bytes": 2 * n * (c["head_dim"] * (e + 1 + e) + 4), "flops": 2 * n * c["head_dim"] * 4}
    if c["op"] == "attn":
        runs, lens = _runs(c), _own_lens(c)
        row = 2 * c["kv_heads"] * (c["head_dim"] + 4)
        io = 2 * sum(runs) * c["heads"] * c["head_dim"] * _BYTES[c["dtype"]]
        keys = sum(n * c["prefix"] + sum(m - n + 1 + i for i in range(n)) for n, m in zip(runs, lens))
        return {"bytes": row * (c["prefix"] + sum(lens)) + io, "flops": 4 * c["heads"] * c["head_dim"] * keys}
    if c["op"] == "probs":
        return {"bytes": 8 * c["rows"] * c["vocab"], "flops": 5 * c["rows"] * c["vocab"]}
    return {"bytes": 8 * c["seqs"] * c["vocab"], "flops": 3 * c["seqs"] * c["vocab"]}


# ── inputs ──────────────────────────────────────────────────────────────────
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _cu(runs):
    at = [0]
    for n in runs:
        at.append(at[-1] + n)
    return _ints(at)


def _rows(g, n, heads, dim):
    """Rows as a projection leaves them: some channels much wider than others."""
    wide = torch.exp(0.6 * torch.randn(heads, dim, generator=g, device="cuda"))
    return torch.randn(n, heads, dim, generator=g, device="cuda") * wide


def _cache(g, slots, rows, heads, dim):
    """A cache that earlier steps have filled: codes and scales of K and V."""
    out = []
    for _ in range(2):
        codes, scale = _quantise(_rows(g, slots * rows, heads, dim))
        out += [codes.view(slots, rows, heads, dim), scale.view(slots, rows, heads)]
    return {"k": out[0], "k_scale": out[1], "v": out[2], "v_scale": out[3]}


def prepare(c, seed):
    g = _generator(seed)
    s = {"op": c["op"], "case": c}
    if c["op"] == "kv":
        runs = _runs(c)
        slots = c["seqs"] + 2
        s["slots"] = torch.randperm(slots, generator=g, device="cuda")[:c["seqs"]].to(torch.int32)
        s["starts"] = _ints([int(_spread(5 * b + 2) * (c["rows"] - n + 1)) for b, n in enumerate(runs)])
        s["cu"], s["n"] = _cu(runs), sum(runs)
        for name in ("k", "v"):
            s[name] = _rows(g, s["n"], c["kv_heads"], c["head_dim"]).to(_TYPES[c["dtype"]])
        shape = (slots, c["rows"], c["kv_heads"])
        s["cache"] = {"k": torch.zeros(*shape, c["head_dim"], dtype=torch.int8, device="cuda"),
                      "v": torch.zeros(*shape, c["head_dim"], dtype=torch.int8, device="cuda"),
                      "k_scale": torch.zeros(shape, device="cuda"), "v_scale": torch.zeros(shape, device="cuda")}
    elif c["op"] == "attn":
        runs, lens = _runs(c), _own_lens(c)
        slots = c["seqs"] + 1
        s["slots"] = torch.randperm(slots, generator=g, device="cuda")[:c["seqs"]].to(torch.int32)
        s["lens"], s["cu"] = _ints(lens), _cu(runs)
        s["q"] = _rows(g, sum(runs), c["heads"], c["head_dim"]).to(_TYPES[c["dtype"]])
        s["cache"] = _cache(g, slots, c["own_rows"], c["kv_heads"], c["head_dim"])
        s["prefix"] = _cache(g, 1, c["prefix"], c["kv_heads"], c["head_dim"]) if c["prefix"] else None
    elif c["op"] == "probs":
        s["logits"] = 3.0 * torch.randn(c["rows"], c["vocab"], generator=g, device="cuda")
    else:
        b, k, v = c["seqs"], c["drafts"], c["vocab"]
        near = 2.5 * torch.randn(b, k + 1, v, generator=g, device="cuda")
        s["draft"] = torch.softmax(near[:, :k], -1)
        near += 0.7 * torch.randn(b, k + 1, v, generator=g, device="cuda")
        s["target"] = torch.softmax(near, -1)
        # drafts drawn from the draft's own distributions
        at = torch.rand(b, k, 1, generator=g, device="cuda") * 0.9999
        s["tokens"] = (s["draft"].double().cumsum(-1) <= at).sum(-1).clamp_(max=v - 1).to(torch.int32)
        s["u"] = torch.rand(b, k, generator=g, device="cuda")
        s["u_last"] = torch.rand(b, generator=g, device="cuda")
        s["counts"] = _ints([k - int(_spread(i) * (k + 1)) for i in range(b)]) if c["ragged"] else None
    return s


# ── one pass ────────────────────────────────────────────────────────────────
def run(s):
    return (_run_own if own else _run_plain)[s["op"]](s)


def _quantise(x):
    """(codes, scales) of rows: scale = max |x| / 127, codes = x / scale rounded half away from zero."""
    x = x.float()
    most = x.abs().amax(-1)
    scale = most / torch.full_like(most, 127.0)
    inv = torch.where(scale > 0, torch.ones_like(scale) / scale, torch.zeros_like(scale))
    y = (x * inv.unsqueeze(-1)).double()
    codes = torch.sign(y) * torch.floor(y.abs() + 0.5)
    return codes.clamp(-127, 127).to(torch.int8), scale


def _places(cu, firsts, n):
    """(sequence, row) of each of n new rows: rows follow firsts[b] within sequence b."""
    at = torch.arange(n, device=cu.device)
    seq = torch.searchsorted(cu[1:].long(), at, right=True)
    return seq, at - cu.long()[seq] + firsts.long()[seq]


def _plain_kv(s):
    cache, out = s["cache"], []
    seq, row = _places(s["cu"], s["starts"], s["n"])
    slot = s["slots"].long()[seq]
    for name in ("k", "v"):
        codes, scale = _quantise(s[name])
        cache[name][slot, row] = codes
        cache[name + "_scale"][slot, row] = scale
        back = cache[name][slot, row].float() * cache[name + "_scale"][slot, row].unsqueeze(-1)
        out.append(back.to(s[name].dtype))
    return tuple(out)


def _values(cache, name, slots=None):
    codes, scale = cache[name], cache[name + "_scale"]
    if slots is not None:
        codes, scale = codes[slots], scale[slots]
    return codes.float() * scale.unsqueeze(-1)


def _plain_attn(s):
    q, cache, prefix = s["q"].float(), s["cache"], s["prefix"]
    n, heads, dim = q.shape
    slots, rows, kv_heads, _ = cache["k"].shape
    group, seqs = heads // kv_heads, len(s["lens"])
    seq, i = _places(s["cu"], torch.zeros_like(s["lens"]), n)
    run = int(s["case"]["run"])
    scale = 1.0 / math.sqrt(dim)
    # queries by sequence, padded to the longest run: [seqs, kv head, run x group, dim]
    qp = torch.zeros(seqs, run, heads, dim, device=q.device)
    qp[seq, i] = q
    qp = qp.view(seqs, run, kv_heads, group, dim).permute(0, 2, 1, 3, 4).reshape(seqs, kv_heads, run * group, dim)
    k, v = (_values(cache, name, s["slots"].long()).permute(0, 2, 1, 3) for name in ("k", "v"))
    scores = torch.matmul(qp, k.transpose(-1, -2)) * scale
    runs = (s["cu"][1:] - s["cu"][:-1]).view(-1, 1)
    seen = s["lens"].view(-1, 1) - runs + 1 + torch.arange(run, device=q.device)
    hidden = torch.arange(rows, device=q.device) >= seen.unsqueeze(-1)
    hidden = hidden.view(seqs, 1, run, 1, rows).expand(-1, -1, -1, group, -1).reshape(seqs, 1, run * group, rows)
    scores = scores.masked_fill(hidden, -math.inf)
    most = scores.amax(-1, keepdim=True)
    if prefix is not None:
        kp, vp = (_values(prefix, name)[0].permute(1, 0, 2) for name in ("k", "v"))
        qf = qp.permute(1, 0, 2, 3).reshape(kv_heads, seqs * run * group, dim)
        far = torch.matmul(qf, kp.transpose(-1, -2)) * scale
        far_most = far.amax(-1, keepdim=True).view(kv_heads, seqs, run * group, 1).transpose(0, 1)
        most = torch.maximum(most, far_most)
        far = torch.exp(far - most.transpose(0, 1).reshape(kv_heads, -1, 1))
    weights = torch.exp(scores - most)
    out, total = torch.matmul(weights, v), weights.sum(-1, keepdim=True)
    if prefix is not None:
        out = out + torch.matmul(far, vp).view(kv_heads, seqs, run * group, dim).transpose(0, 1)
        total = total + far.sum(-1, keepdim=True).view(kv_heads, seqs, run * group, 1).transpose(0, 1)
    out = (out / total).view(seqs, kv_heads, run, group, dim).permute(0, 2, 1, 3, 4).reshape(seqs, run, heads, dim)
    return out[seq, i].to(s["q"].dtype)


def _plain_probs(s):
    x = s["logits"] / s["case"]["temperature"]
    e = torch.exp(x - x.amax(-1, keepdim=True))
    return e / e.sum(-1, keepdim=True)


def _plain_verify(s):
    target, draft, tokens = s["target"], s["draft"], s["tokens"].long()
    b, k = tokens.shape
    at = tokens.unsqueeze(-1)
    p = torch.gather(target[:, :k], 2, at).squeeze(-1).double()
    q = torch.gather(draft, 2, at).squeeze(-1).double()
    counts = s["counts"].long() if s["counts"] is not None else torch.full((b,), k, device=tokens.device)
    place = torch.arange(k, device=tokens.device)
    ok = (s["u"].double() * q < p) & (place < counts.view(-1, 1))
    accepted = ok.long().cumprod(1).sum(1)
    lines = torch.arange(b, device=tokens.device)
    row = target[lines, accepted].double()
    beaten = draft[lines, accepted.clamp(max=k - 1)].double()
    rest = (row - beaten).clamp(min=0)
    use_row = (accepted == counts) | (rest.sum(-1) == 0)
    weights = torch.where(use_row.view(-1, 1), row, rest)
    sums = weights.cumsum(-1)
    goal = s["u_last"].double() * sums[:, -1]
    drawn = torch.searchsorted(sums, goal.view(-1, 1), right=True).squeeze(-1)
    last = target.shape[-1] - 1 - (weights > 0).flip(-1).to(torch.int8).argmax(-1)
    drawn = torch.minimum(drawn, last)
    out = torch.full((b, k + 1), -1, dtype=torch.int64, device=tokens.device)
    out[:, :k] = torch.where(place < accepted.view(-1, 1), tokens, out[:, :k])
    out[lines, accepted] = drawn
    return out.to(torch.int32), accepted.to(torch.int32)


_run_plain = {"kv": _plain_kv, "attn": _plain_attn, "probs": _plain_probs, "verify": _plain_verify}


# ── the framework's calls ───────────────────────────────────────────────────
def _handle(s, name):
    """The cache's handle, made once as a serving program keeps it."""
    import qraf_b200 as qb

    key = name + " handle"
    if key not in s:
        c = s[name]
        s[key] = None if c is None else qb.KvCache.from_tensors(c["k"], c["v"], c["k_scale"], c["v_scale"])
    return s[key]


def _own_kv(s):
    import qraf_b200 as qb

    cache = _handle(s, "cache")
    qb.kv_store(cache, s["k"], s["v"], s["slots"], s["starts"], s["cu"])
    return qb.kv_load(cache, s["slots"], s["starts"], s["cu"], n=s["n"], dtype=s["k"].dtype)


def _own_attn(s):
    import qraf_b200 as qb

    return qb.kv_attention(s["q"], _handle(s, "cache"), s["slots"], s["lens"], s["cu"],
                           prefix=_handle(s, "prefix"), prefix_len=s["case"]["prefix"])


def _own_probs(s):
    import qraf_b200 as qb

    return qb.token_probs(s["logits"], temperature=s["case"]["temperature"])


def _own_verify(s):
    import qraf_b200 as qb

    return qb.verify_drafts(s["target"], s["draft"], s["tokens"], s["u"], s["u_last"], counts=s["counts"])


_run_own = {"kv": _own_kv, "attn": _own_attn, "probs": _own_probs, "verify": _own_verify}


# ── the definitions in 64 bits ──────────────────────────────────────────────
def exact(c, seed):
    if c["op"] == "verify":
        return None   # whole numbers only
    s = prepare(c, seed)
    if c["op"] == "probs":
        x = s["logits"].double() / c["temperature"]
        return torch.exp(x - torch.logsumexp(x, -1, keepdim=True))
    if c["op"] == "kv":
        return tuple(_exact_rows(s[name]) for name in ("k", "v"))
    return _exact_attn(c, s)


def _exact_rows(x):
    """The values a row's codes stand for.  The stored scale and the products that are rounded
    to codes are 32-bit numbers by definition; the values are not rounded."""
    import numpy as np

    x = x.float().cpu().numpy()
    scale = np.abs(x).max(-1, keepdims=True) / np.float32(127)
    inv = np.divide(np.float32(1), scale, out=np.zeros_like(scale), where=scale > 0)
    y = (x * inv).astype(np.float64)
    return torch.from_numpy(np.trunc(y + np.copysign(0.5, y)).clip(-127, 127) * scale.astype(np.float64)).cuda()


def _exact_attn(c, s):
    group = c["heads"] // c["kv_heads"]
    out, at = [], 0
    for b, (n, m) in enumerate(zip(_runs(c), _own_lens(c))):
        slot = int(s["slots"][b])
        parts = []
        for name in ("k", "v"):
            x = s["cache"][name][slot, :m].double() * s["cache"][name + "_scale"][slot, :m].double()[..., None]
            if s["prefix"] is not None:
                far = s["prefix"][name][0].double() * s["prefix"][name + "_scale"][0].double()[..., None]
                x = torch.cat([far, x])
            parts.append(x.repeat_interleave(group, 1))
        k, v = parts
        for i in range(n):
            seen = c["prefix"] + m - n + 1 + i
            w = torch.softmax(torch.einsum("hd,khd->hk", s["q"][at + i].double(), k[:seen]) / c["head_dim"] ** 0.5, -1)
            out.append(torch.einsum("hk,khd->hd", w, v[:seen]))
        at += n
    return torch.stack(out)
