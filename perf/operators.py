"""Sequences of spherical signals: the operators between a spherical network and an answer about signals in order.

A spherical network gives one feature vector per signal.  Where signals come in order (the rings of a sphere, the frames of a
panoramic recording, the shells of a volume), a model relates them by attention with a learned bias by relative position,
with layer norm before it and dropout behind it.  Kinds of work:

  attention   softmax attention with a bias by buckets of the relative position.  ``infer``: the output alone, of whole sequences
              or of a few new signals that look at kept keys and values; ``train``: the output and all gradients
  norm        layer norm over the last axis: ``infer`` or ``train`` (with the gradients of input, weight and bias)
  dropout     dropout with a counter-based mask that is never stored, optionally added to a residual; output and gradient

Lengths are those of this package's grids: rings of 2b = 12 ... 128 positions, spheres of 4b^2 = 3600 (b = 30), 4096 (b = 32)
and 16384 (b = 64) points; widths those of its models (40, 100, 200 features) and powers of two.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}


def _attention(name, mode, dtype, batch, lq, lk, heads, kv_heads, dim, causal, ragged, buckets=32, distance=128):
    return {"name": name, "kind": "attention", "mode": mode, "dtype": dtype, "batch": batch, "lq": lq, "lk": lk, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "causal": causal, "ragged": ragged, "buckets": buckets, "distance": distance}


def listed():
    return [
        # the twelve rings of one small sphere, 40 features: the latency of one answer
        _attention("ring of one sphere", "infer", "float32", 1, 12, 12, 4, 4, 10, False, False, 8, 6),
        # a training step over the 60 rings of a batch of b = 30 spheres
        _attention("rings, train", "train", "float32", 32, 60, 60, 4, 4, 10, False, False, 16, 30),
        # every point of a b = 30 sphere looks at every other one, in the package's own type
        _attention("sphere of points, train", "train", "float32", 1, 3600, 3600, 4, 4, 64, False, False),
        # recordings of different lengths, padded to the longest: each frame sees the frames before it
        _attention("recordings, train", "train", "bfloat16", 8, 1000, 1000, 8, 8, 64, True, True),
        # the largest training step: all points of two b = 32 spheres
        _attention("large spheres, train", "train", "bfloat16", 2, 4096, 4096, 16, 16, 128, False, False),
        # a first pass over recordings whose keys and values are kept: three query heads share one of them
        _attention("first pass, shared heads", "infer", "bfloat16", 4, 2049, 2049, 12, 4, 64, True, False),
        # one new frame of each of 16 recordings looks at all that has been kept of it
        _attention("one new frame", "infer", "bfloat16", 16, 1, 16384, 16, 4, 128, True, True),
        # the same for a single recording with 200 float32 features, eight heads of 25
        _attention("one new frame, float32", "infer", "float32", 1, 1, 3600, 8, 8, 25, True, False),
        # the norm of a wide model's training step
        {"name": "norm, train", "kind": "norm", "mode": "train", "dtype": "bfloat16", "rows": 16384, "cols": 1024},
        # the norm of 200 float32 features of the points of a sphere, one of them left over
        {"name": "norm, float32, train", "kind": "norm", "mode": "train", "dtype": "float32", "rows": 3601, "cols": 200},
        # behind attention in a wide model's training step, added to what went around it
        {"name": "dropout, train", "kind": "dropout", "dtype": "bfloat16", "rows": 16384, "cols": 1024, "p": 0.1, "residual": True},
        # float32 features of an odd count, nothing to add to
        {"name": "dropout, float32, odd", "kind": "dropout", "dtype": "float32", "rows": 2401, "cols": 41, "p": 0.5, "residual": False},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "attention", "attention", "norm", "dropout"])
    dtype = rng.choice(["float32", "bfloat16", "bfloat16"])
    if kind == "norm":
        cols = _log(rng, 8, 8192)
        return {"kind": kind, "mode": rng.choice(["infer", "train", "train"]), "dtype": dtype, "rows": _log(rng, 1, min(65536, (1 << 24) // cols)), "cols": cols}
    if kind == "dropout":
        cols = _log(rng, 8, 8192)
        return {"kind": kind, "dtype": dtype, "rows": _log(rng, 1, min(65536, (1 << 24) // cols)), "cols": cols,
                "p": rng.choice([0.05, 0.1, 0.2, 0.5]), "residual": rng.random() < 0.5}
    mode = rng.choice(["train", "train", "infer", "one"])
    kv_heads, group = rng.choice([1, 2, 3, 4, 5, 8]), rng.choice([1, 1, 2, 4])
    dim = rng.choice([10, 16, 20, 25, 32, 40, 50, 64, 64, 80, 100, 128, 128])
    heads = kv_heads * group
    batch = _log(rng, 1, 32)
    # queries times keys over all heads and signals: a quarter of the largest listed case's in bfloat16, a fifteenth in float32
    most = (1 << 27) if dtype == "bfloat16" else (1 << 25)
    if mode == "one":
        lq = rng.choice([1, 1, 1, 2, 3])
        lk = max(lq, _log(rng, 100, 16384))
        batch = max(1, min(batch, (1 << 20) // (lk * kv_heads) * 2))
    else:
        lk = _log(rng, 12, min(4096, int(math.sqrt(most / heads))))
        batch = max(1, min(batch, most // (heads * lk * lk)))
        lq = lk if mode == "train" or rng.random() < 0.5 else rng.randint(max(1, lk // 4), lk)
    case = _attention("", "train" if mode == "train" else "infer", dtype, batch, lq, lk, heads, kv_heads, dim, rng.random() < 0.5,
                      batch > 1 and rng.random() < 0.5, rng.choice([16, 32]), rng.choice([30, 64, 128]))
    del case["name"]
    return case


def _lengths(case):
    """How many of each signal's positions are filled: all, or between all of them and a part, evenly."""
    n, b = case["lk"], case["batch"]
    return [max(1, n - i * n // b) for i in range(b)] if case["ragged"] else [n] * b


def _starts(case):
    """The position of each signal's first query among the keys: the last queries of what is filled, or the first position."""
    return [max(0, n - case["lq"]) if case["lq"] < case["lk"] else 0 for n in _lengths(case)]


def _bucket_map(buckets, distance):
    """The bucket of each relative position -distance ... distance, as int32: half of the buckets for each side, half of a side's
    for single steps, the others growing as powers up to the distance."""
    side = buckets // 2
    exact = max(1, side // 2)
    edges = [exact * (distance / exact) ** (k / (side - exact)) for k in range(1, side - exact)]
    steps = [d if d < exact else exact + sum(d >= e for e in edges) for d in range(distance + 1)]
    return [steps[-d] if d <= 0 else side + steps[d] for d in range(-distance, distance + 1)]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = TYPES[case["dtype"]]

    def normal(*shape, scale=1.0, shift=0.0):
        return (torch.randn(shape, generator=gen, device="cuda") * scale + shift).to(dtype)

    if case["kind"] == "attention":
        b, lq, lk, h, hk, d = (case[k] for k in ("batch", "lq", "lk", "heads", "kv_heads", "dim"))
        if lq == lk:        # one projection gives all three
            packed = normal(b, lq, h + 2 * hk, d)
            q, k, v = packed[:, :, :h], packed[:, :, h:h + hk], packed[:, :, h + hk:]
        else:               # new queries, kept keys and values
            q, k, v = normal(b, lq, h, d), normal(b, lk, hk, d), normal(b, lk, hk, d)
        order = torch.randperm(b, generator=torch.Generator().manual_seed(seed)).tolist()
        ints = lambda values: torch.tensor([values[i] for i in order], dtype=torch.int32, device="cuda")  # noqa: E731
        state = {"case": dict(case), "q": q, "k": k, "v": v, "bias": normal(case["buckets"], h),
                 "buckets": torch.tensor(_bucket_map(case["buckets"], case["distance"]), dtype=torch.int32, device="cuda"),
                 "start": ints(_starts(case)) if lq < lk else None, "lengths": ints(_lengths(case)) if case["ragged"] else None}
        if case["mode"] == "train":
            state["grad"] = normal(b, lq, h, d)
            for name in ("q", "k", "v", "bias"):
                state[name].requires_grad_(True)
        return state
    x = normal(case["rows"], case["cols"], scale=1.5, shift=0.25)
    state = {"case": dict(case), "x": x}
    if case["kind"] == "norm":
        state |= {"weight": normal(case["cols"], scale=0.2, shift=1.0), "bias": normal(case["cols"], scale=0.2)}
        if case["mode"] == "train":
            state["grad"] = normal(case["rows"], case["cols"])
            for name in ("x", "weight", "bias"):
                state[name].requires_grad_(True)
        return state
    x.requires_grad_(True)
    residual = normal(case["rows"], case["cols"]) if case["residual"] else None
    return state | {"residual": residual, "grad": normal(case["rows"], case["cols"]), "seed": seed * 0x9E3779B97F4A7C15 % (1 << 63), "step": seed % 1000}


# ---- the plain forms --------------------------------------------------------------------------------------------------


def _plain_attention(s):
    case = s["case"]
    q, k, v = (s[n].detach().float().transpose(1, 2) for n in "qkv")         # [batch, heads, length, dim]
    group, dev = case["heads"] // case["kv_heads"], q.device
    k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    scale = 1 / math.sqrt(case["dim"])
    i, j = torch.arange(case["lq"], device=dev)[:, None], torch.arange(case["lk"], device=dev)[None, :]
    start = s["start"].long()[:, None, None] if s["start"] is not None else torch.zeros(1, 1, 1, dtype=torch.long, device=dev)
    away = j - i - start                                                      # [batch or 1, queries, keys]
    reach = (s["buckets"].numel() - 1) // 2
    bucket = s["buckets"].long()[away.clamp(-reach, reach) + reach]
    seen = away <= 0 if case["causal"] else torch.ones_like(away, dtype=torch.bool)
    if s["lengths"] is not None:
        seen = seen & (j < s["lengths"].long()[:, None, None])
    p = q @ k.transpose(2, 3) * scale + s["bias"].detach().float()[bucket].permute(0, 3, 1, 2)
    p = p.masked_fill(~seen[:, None], -math.inf)
    p = torch.exp(p - p.amax(-1, keepdim=True).clamp_min(-1e30))
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-30)
    out = p @ v
    result = {"out": out.transpose(1, 2).to(s["q"].dtype)}
    if case["mode"] == "train":
        g = s["grad"].float().transpose(1, 2)
        shared = lambda t: t.unflatten(1, (case["kv_heads"], group)).sum(2).transpose(1, 2)  # noqa: E731
        result["dv"] = shared(p.transpose(2, 3) @ g).to(s["v"].dtype)
        ds = p * (g @ v.transpose(2, 3) - (g * out).sum(-1, keepdim=True))
        result["dq"] = (ds @ k * scale).transpose(1, 2).to(s["q"].dtype)
        result["dk"] = shared(ds.transpose(2, 3) @ q * scale).to(s["k"].dtype)
        # rows turned round and one place longer each: the diagonals j - i come to stand one under the other
        ds = ds.sum(0).flip(1)
        lq, lk = case["lq"], case["lk"]
        ds = torch.cat((ds, ds.new_zeros(ds.size(0), lq, lq)), 2).flatten(1)[:, : lq * (lq + lk - 1)].unflatten(1, (lq, lq + lk - 1)).sum(1)
        which = s["buckets"].long()[(torch.arange(lq + lk - 1, device=dev) - (lq - 1)).clamp(-reach, reach) + reach]
        hot = (which[:, None] == torch.arange(case["buckets"], device=dev)).float()
        result["dbias"] = (ds @ hot).t().to(s["bias"].dtype)
    return result


def _plain_norm(s):
    case, dtype = s["case"], s["x"].dtype
    x, w = s["x"].detach().float(), s["weight"].detach().float()
    x = x - x.mean(-1, keepdim=True)
    rstd = torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-5)
    x = x * rstd
    result = {"out": (x * w + s["bias"].detach().float()).to(dtype)}
    if case["mode"] == "train":
        dy = s["grad"].float()
        g = dy * w
        result["dx"] = (rstd * (g - g.mean(-1, keepdim=True) - x * (g * x).mean(-1, keepdim=True))).to(dtype)
        result["dweight"], result["dbias"] = (dy * x).sum(0).to(dtype), dy.sum(0).to(dtype)
    return result


def _plain_words(n, seed, step, device):
    """Word i of the generator for i = 0 ... n - 1: block i // 4 of Philox-4x32 with seven rounds (Salmon, Moraes, Dror and
    Shaw, 2011), counter (block, step), key seed, low words first."""
    low = 0xFFFFFFFF
    block = torch.arange((n + 3) // 4, device=device)
    a, b, c, d = block & low, block >> 32, torch.full_like(block, step & low), torch.full_like(block, step >> 32)
    key = [seed & low, seed >> 32]
    rounds = [[(key[0] + r * 0x9E3779B9) & low, (key[1] + r * 0xBB67AE85) & low] for r in range(7)]

    def one(words, k):
        a, b, c, d = words
        x, y = a * 0xD2511F53, c * 0xCD9E8D57
        return (y >> 32) & low ^ b ^ k[0], y & low, (x >> 32) & low ^ d ^ k[1], x & low

    words = (a, b, c, d)
    for k in rounds:
        words = one(words, k)
    return torch.stack(words, 1).flatten()[:n]


def _plain_dropout(s):
    x, p = s["x"].detach(), s["case"]["p"]
    keep = _plain_words(x.numel(), s["seed"], s["step"], x.device).view(x.shape) >= int(p * 2 ** 32)
    out = torch.where(keep, x.float() / (1 - p), 0.0)
    if s["residual"] is not None:
        out = out + s["residual"].float()
    return {"out": out.to(x.dtype), "dx": torch.where(keep, s["grad"].float() / (1 - p), 0.0).to(x.dtype)}


def run(s):
    kind = s["case"]["kind"]
    if not own:
        return {"attention": _plain_attention, "norm": _plain_norm, "dropout": _plain_dropout}[kind](s)
    import s2cnn_b200 as S
    if kind == "dropout":
        out = S.dropout(s["x"], s["case"]["p"], s["seed"], s["step"], residual=s["residual"])
        return {"out": out.detach(), "dx": torch.autograd.grad(out, s["x"], s["grad"])[0]}
    if kind == "norm":
        out = S.layer_norm(s["x"], s["weight"], s["bias"])
        wanted, names = (s["x"], s["weight"], s["bias"]), ("dx", "dweight", "dbias")
    else:
        out = S.attention(s["q"], s["k"], s["v"], s["bias"], s["buckets"], causal=s["case"]["causal"],
                          q_start=0 if s["start"] is None else s["start"], kv_lengths=s["lengths"])
        wanted, names = (s["q"], s["k"], s["v"], s["bias"]), ("dq", "dk", "dv", "dbias")
    if s["case"]["mode"] != "train":
        return {"out": out}
    return {"out": out.detach()} | dict(zip(names, torch.autograd.grad(out, wanted, s["grad"])))


def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    if case["kind"] == "attention":
        train, b, lq, h, hk, d = case["mode"] == "train", case["batch"], case["lq"], case["heads"], case["kv_heads"], case["dim"]
        pairs, keys = 0, 0
        for n, start in zip(_lengths(case), _starts(case)):
            if case["causal"]:
                pairs += sum(min(n, start + i + 1) for i in range(lq))
                n = min(n, start + lq)
            else:
                pairs += n * lq
            keys += n
        kept = case["lk"] * b - keys          # gradients of unseen keys are written all the same
        values = b * lq * h * d * (4 if train else 2) + keys * hk * d * (4 if train else 2) + (kept * hk * d * 2 if train else 0)
        return {"bytes": values * size, "flops": (14 if train else 4) * d * h * pairs}
    n = case["rows"] * case["cols"]
    if case["kind"] == "norm":
        return {"bytes": n * size * (4 if case["mode"] == "train" else 2), "flops": n * (16 if case["mode"] == "train" else 8)}
    return {"bytes": n * size * (5 if case["residual"] else 4), "flops": n * 4}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------------


def _exact_attention(s):
    case = s["case"]
    b, lq, lk, h, hk, d = (case[k] for k in ("batch", "lq", "lk", "heads", "kv_heads", "dim"))
    train = case["mode"] == "train"
    dev = s["q"].device
    new = lambda *shape: torch.zeros(shape, dtype=torch.float64, device=dev)  # noqa: E731
    r = {"out": new(b, lq, h, d)}
    if train:
        r |= {"dq": new(b, lq, h, d), "dk": new(b, lk, hk, d), "dv": new(b, lk, hk, d), "dbias": new(case["buckets"], h)}
    table, reach = s["buckets"].long(), (s["buckets"].numel() - 1) // 2
    starts = [0] * b if s["start"] is None else s["start"].tolist()
    lengths = [lk] * b if s["lengths"] is None else s["lengths"].tolist()
    for n in range(b):
        rel = torch.arange(lengths[n], device=dev) - torch.arange(lq, device=dev).unsqueeze(1) - starts[n]
        bucket = table[(rel.clamp(min=-reach, max=reach) + reach)]
        for head in range(h):
            kh = head // (h // hk)
            q, k, v = s["q"][n, :, head].double(), s["k"][n, :lengths[n], kh].double(), s["v"][n, :lengths[n], kh].double()
            logits = torch.einsum("id,jd->ij", q, k) / d ** 0.5 + s["bias"][:, head].double()[bucket]
            if case["causal"]:
                logits[rel > 0] = -math.inf
            log_sum = torch.logsumexp(logits, 1, keepdim=True)
            prob = torch.exp(logits - log_sum)
            r["out"][n, :, head] = torch.einsum("ij,jd->id", prob, v)
            if train:
                g = s["grad"][n, :, head].double()
                dp = torch.einsum("id,jd->ij", g, v)
                dl = prob * (dp - torch.einsum("ij,ij->i", prob, dp).unsqueeze(1))
                r["dv"][n, :lengths[n], kh] += torch.einsum("ij,id->jd", prob, g)
                r["dq"][n, :, head] = torch.einsum("ij,jd->id", dl, k) / d ** 0.5
                r["dk"][n, :lengths[n], kh] += torch.einsum("ij,id->jd", dl, q) / d ** 0.5
                r["dbias"][:, head] += torch.stack([dl[bucket == which].sum() for which in range(case["buckets"])])
    return r


def _exact_dropout(s):
    x, p = s["x"].detach().double(), s["case"]["p"]
    mask32, n = np.uint64(0xFFFFFFFF), x.numel()
    counter = np.arange(-(-n // 4), dtype=np.uint64)
    v = [counter & mask32, counter >> np.uint64(32), np.full_like(counter, s["step"] & 0xFFFFFFFF), np.full_like(counter, s["step"] >> 32)]
    k0, k1 = s["seed"] & 0xFFFFFFFF, s["seed"] >> 32
    for _ in range(7):
        first, third = v[0] * np.uint64(0xD2511F53), v[2] * np.uint64(0xCD9E8D57)
        v = [(third >> np.uint64(32)) ^ v[1] ^ np.uint64(k0), third & mask32, (first >> np.uint64(32)) ^ v[3] ^ np.uint64(k1), first & mask32]
        k0, k1 = (k0 + 0x9E3779B9) % 2 ** 32, (k1 + 0xBB67AE85) % 2 ** 32
    keep = np.stack(v, 1).reshape(-1)[:n] >= np.uint64(math.floor(p * 2 ** 32))
    factor = torch.from_numpy(keep.astype(np.float64)).to(x.device).view(x.shape) / (1 - p)
    out = x * factor
    if s["residual"] is not None:
        out += s["residual"].double()
    return {"out": out, "dx": s["grad"].double() * factor}


def _exact_norm(s):
    x, w = s["x"].detach().double(), s["weight"].detach().double()
    var, mean = torch.var_mean(x, 1, unbiased=False, keepdim=True)
    hat = (x - mean) / torch.sqrt(var + 1e-5)
    r = {"out": hat * w + s["bias"].detach().double()}
    if s["case"]["mode"] == "train":
        dy, n = s["grad"].double(), x.size(1)
        dhat = dy * w
        r["dx"] = (n * dhat - dhat.sum(1, keepdim=True) - hat * (dhat * hat).sum(1, keepdim=True)) / (n * torch.sqrt(var + 1e-5))
        r["dweight"], r["dbias"] = torch.einsum("rc,rc->c", dy, hat), dy.sum(0)
    return r


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"attention": _exact_attention, "norm": _exact_norm, "dropout": _exact_dropout}[case["kind"]](s)
