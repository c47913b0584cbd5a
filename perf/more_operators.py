"""Positions that turn, and kept keys in pages: the operators of models over recordings that grow, differ in length and share beginnings.

A model over spherical signals in order keeps the keys and values of what it has seen and answers for each new signal.  Its queries
and keys are normed head by head and turned by their position; keys and values lie in pages of one pool, which sequences take as
they grow, share where they have a common beginning, and give back.  Kinds of work:

  rotate     norm of every head of queries and keys and rotation by position, ``infer`` or ``train`` (with all gradients)
  store      the same for new positions, whose keys and values go to their pages
  attention  softmax attention of a few new positions over the keys and values in their sequences' pages
  copy       pages of all layers copied within the pool: sequences that fork, a pool that is compacted

Lengths are those of this package's grids and sequences: rings of 2b = 12 ... 128 positions, spheres of 4b^2 = 3600 (b = 30) and 16384
(b = 64) points; widths those of its models (40, 100, 200 features) and powers of two.
"""
import math

import torch

own = False

TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}
EPS = 1e-6


def _rotate(name, mode, dtype, batch, length, heads, kv_heads, dim, turned, interleaved, norm, start=0, factor=1.0):
    return {"name": name, "kind": "rotate", "mode": mode, "dtype": dtype, "batch": batch, "length": length, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "turned": turned, "interleaved": interleaved, "norm": norm, "start": start, "factor": factor}


def _store(name, dtype, batch, new, room, heads, kv_heads, dim, turned, interleaved, norm, page, ragged):
    return {"name": name, "kind": "store", "dtype": dtype, "batch": batch, "length": new, "room": room, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "turned": turned, "interleaved": interleaved, "norm": norm, "page": page, "ragged": ragged, "factor": 1.0}


def _attention(name, dtype, batch, lq, lk, heads, kv_heads, dim, page, ragged, buckets=0, distance=0):
    return {"name": name, "kind": "attention", "dtype": dtype, "batch": batch, "lq": lq, "lk": lk, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "page": page, "ragged": ragged, "buckets": buckets, "distance": distance}


def _copy(name, dtype, copied, layers, kv_heads, page, dim):
    return {"name": name, "kind": "copy", "dtype": dtype, "copied": copied, "layers": layers, "kv_heads": kv_heads, "page": page, "dim": dim}


def listed():
    return [
        # a training step over the 60 rings of a batch of b = 30 spheres: the host's time counts
        _rotate("rotate, rings, train", "train", "float32", 32, 60, 4, 4, 10, 10, False, True),
        # long recordings in training, four query heads on one key head
        _rotate("rotate, recordings, train", "train", "bfloat16", 4, 4096, 16, 4, 128, 128, False, True),
        # neighbouring pairs of 24 of 25 values, no norm, far along a recording by frequencies scaled for it
        _rotate("rotate, far, odd heads", "infer", "float32", 1, 3601, 8, 8, 25, 24, True, False, 100000, 4.0),
        # one new frame of each of 16 recordings
        _store("store, one new frame", "bfloat16", 16, 1, 2048, 16, 4, 128, 128, False, True, 64, True),
        # a first pass over recordings whose keys and values are kept; half of each head is turned
        _store("store, first pass", "bfloat16", 4, 2049, 2100, 12, 4, 64, 32, True, True, 32, True),
        # the frame's look at all that has been kept of its recording
        _attention("paged, one new frame", "bfloat16", 16, 1, 16384, 16, 4, 128, 64, True),
        # the same for a single recording with 200 float32 features, eight heads of 25, and a bias by relative position
        _attention("paged, one new frame, float32", "float32", 1, 1, 3600, 8, 8, 25, 16, False, 32, 128),
        # four new frames each of 32 short recordings, shared heads and a bias
        _attention("paged, four new frames", "bfloat16", 32, 4, 1000, 12, 4, 64, 32, True, 32, 128),
        # as many full recordings as a busy server holds
        _attention("paged, many recordings", "bfloat16", 64, 1, 16384, 16, 4, 128, 64, False),
        # sixteen sequences fork: the page that they were writing to is copied
        _copy("copy, fork", "bfloat16", 16, 2, 4, 64, 128),
        # a pool is compacted
        _copy("copy, compaction", "bfloat16", 1024, 2, 4, 64, 128),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(["rotate", "rotate", "store", "attention", "attention", "attention", "copy"])
    dtype = rng.choice(["float32", "bfloat16", "bfloat16"])
    kv_heads, group = rng.choice([1, 2, 3, 4, 5, 8]), rng.choice([1, 1, 2, 4])
    dim = rng.choice([10, 16, 20, 25, 32, 40, 50, 64, 64, 80, 100, 128, 128])
    heads = kv_heads * group
    page = rng.choice([16, 32, 64, 128])
    most = (1 << 24) if dtype == "float32" else (1 << 25)          # values of a largest call, some
    if kind == "copy":
        case = _copy("", dtype, 1, rng.randint(1, 4), kv_heads, page, dim)
        values = case["layers"] * 2 * kv_heads * page * dim
        case["copied"] = _log(rng, 1, max(1, min(2048, 3 * most // values)))
    elif kind == "attention":
        lk = _log(rng, 1, 16384)
        batch = _log(rng, 1, max(1, min(64, 2 * most // (lk * kv_heads * dim))))
        lq = min(lk, rng.choice([1, 1, 1, 1, 2, 3, 4, 5, 8, 20]))
        buckets = rng.choice([0, 0, 16, 32])
        case = _attention("", dtype, batch, lq, lk, heads, kv_heads, dim, page, batch > 1 and rng.random() < 0.6, buckets, rng.choice([30, 64, 128]) if buckets else 0)
    else:
        turned = dim // 2 * 2 if rng.random() < 0.6 else 2 * rng.randint(1, dim // 2)
        interleaved, norm = rng.random() < 0.4, rng.random() < 0.7
        width = (heads + 2 * kv_heads) * dim
        batch = _log(rng, 1, 32)
        length = _log(rng, 1, max(1, min(16384, most // (width * batch))))
        if kind == "rotate":
            case = _rotate("", rng.choice(["train", "train", "infer"]), dtype, batch, length, heads, kv_heads, dim, turned, interleaved, norm,
                           rng.choice([0, 0, _log(rng, 1, 200000)]), rng.choice([1.0, 1.0, 4.0]))
        else:
            length = rng.choice([1, 1, length])
            case = _store("", dtype, batch, length, length + _log(rng, 1, 2000), heads, kv_heads, dim, turned, interleaved, norm, page, batch > 1 and rng.random() < 0.6)
    del case["name"]
    return case


def _frequencies(turned, factor, base=10000.0, length=4096, slow=1.0, fast=32.0):
    """Radians per position of each pair, in 64 bits.  Scaled by ``factor``: pairs that turn more than ``fast`` times over ``length``
    positions stay, those that turn less than ``slow`` times are slowed by the factor, between the two gradually."""
    result = []
    for i in range(turned // 2):
        f = base ** (-2 * i / turned)
        turns = f * length / (2 * math.pi)
        kept = min(1.0, max(0.0, (turns - slow) / (fast - slow)))
        result.append(f * (kept + (1 - kept) / factor))
    return result


def _counts(batch, most, ragged):
    """how many positions each sequence has: all, or evenly between all of them and a part"""
    return [max(1, most - i * most // batch) for i in range(batch)] if ragged else [most] * batch


def _row(case):
    """values from one position to the next in a page: rows start on 16-byte boundaries"""
    step = 16 // (4 if case["dtype"] == "float32" else 2)
    return (case["dim"] + step - 1) // step * step


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    dtype = TYPES[case["dtype"]]

    def normal(*shape, scale=1.0, shift=0.0):
        return (torch.randn(shape, generator=gen, device="cuda") * scale + shift).to(dtype)

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    if case["kind"] == "copy":
        n = case["copied"]
        pages = 2 * n + 3
        order = torch.randperm(pages, generator=host)
        shape = (pages, case["layers"], 2, case["kv_heads"], case["page"], _row(case))
        storage = torch.empty(shape, dtype=dtype, device="cuda")
        for part in storage.split(256):
            part.copy_(normal(*part.shape))
        return {"case": dict(case), "storage": storage, "source": ints(order[:n].tolist()), "target": ints(order[n:2 * n].tolist())}
    b, h, hk, d = (case[k] for k in ("batch", "heads", "kv_heads", "dim"))
    state = {"case": dict(case)}
    if case["kind"] != "attention":
        packed = normal(b, case["length"], h + 2 * hk, d, scale=1.5)         # one projection gives all three
        state |= {"q": packed[:, :, :h], "k": packed[:, :, h:h + hk], "v": packed[:, :, h + hk:],
                  "frequencies": torch.tensor(_frequencies(case["turned"], case["factor"]), dtype=torch.float64, device="cuda"),
                  "wq": normal(d, scale=0.2, shift=1.0) if case["norm"] else None, "wk": normal(d, scale=0.2, shift=1.0) if case["norm"] else None}
    if case["kind"] == "rotate":
        state["positions"] = ints([case["start"] + 7 * i for i in range(b)]) if case["start"] else 0
        if case["mode"] == "train":
            state |= {"gq": normal(b, case["length"], h, d), "gk": normal(b, case["length"], hk, d)}
            for name in ("q", "k") + (("wq", "wk") if case["norm"] else ()):
                state[name].requires_grad_(True)
        return state
    # a pool of which the sequences' pages are taken in no order, with some left over
    room = case["lk"] if case["kind"] == "attention" else case["room"]
    per = -(-room // case["page"])
    count = b * per + 5
    pool = torch.empty(count, 2, hk, case["page"], _row(case), dtype=dtype, device="cuda")
    for part in pool.split(max(1, (1 << 26) // pool[0].numel())):
        part.copy_(normal(*part.shape))
    state |= {"keys": pool[:, 0].transpose(1, 2)[..., :d], "values": pool[:, 1].transpose(1, 2)[..., :d],
              "pages": torch.randperm(count, generator=host)[:b * per].view(b, per).to(torch.int32).cuda()}
    order = torch.randperm(b, generator=host).tolist()
    counts = [_counts(b, case["lk"] if case["kind"] == "attention" else case["length"], case["ragged"])[i] for i in order]
    if case["kind"] == "store":
        return state | {"lengths": ints(counts) if case["ragged"] else None, "positions": ints([(room - n) * (i + 1) // b for i, n in enumerate(counts)])}
    state |= {"q": normal(b, case["lq"], h, d), "kv_lengths": ints(counts), "q_start": ints([n - case["lq"] for n in counts]), "bias": None, "buckets": None}
    if case["buckets"]:
        state |= {"bias": normal(case["buckets"], h), "buckets": ints(_bucket_map(case["buckets"], case["distance"]))}
    return state


def _bucket_map(buckets, distance):
    """The bucket of each relative position -distance ... distance: half of the buckets for each side, half of a side's for
    single steps, the others growing as powers up to the distance."""
    side = buckets // 2
    exact = max(1, side // 2)
    edges = [exact * (distance / exact) ** (k / (side - exact)) for k in range(1, side - exact)]
    steps = [d if d < exact else exact + sum(d >= e for e in edges) for d in range(distance + 1)]
    return [steps[-d] if d <= 0 else side + steps[d] for d in range(-distance, distance + 1)]


# ---- the plain forms --------------------------------------------------------------------------------------------------


def _plain_angles(s):
    """[batch or 1, length, 1, pairs]: cosines and sines in 32 bits, of angles in 64"""
    at, n = s["positions"], s["case"]["length"]
    first = at.long()[:, None] if torch.is_tensor(at) else torch.full((1, 1), at, dtype=torch.long, device=s["q"].device)
    angle = (first + torch.arange(n, device=s["q"].device)).double()[..., None] * s["frequencies"]
    return torch.cos(angle).float()[:, :, None], torch.sin(angle).float()[:, :, None]


def _plain_turn(x, cos, sin, interleaved):
    r = 2 * cos.size(-1)
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if interleaved else (x[..., :r // 2], x[..., r // 2:r])
    a, b = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((turned, x[..., r:]), -1)


def _plain_norm_rotate(s, x, w, cos, sin):
    x = x.detach().float()
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.detach().float()
    return _plain_turn(x, cos, sin, s["case"]["interleaved"])


def _plain_norm_rotate_grad(s, x, w, dy, cos, sin):
    g = _plain_turn(dy.float(), cos, -sin, s["case"]["interleaved"])
    if w is None:
        return g, None
    x = x.detach().float()
    rstd = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    x = x * rstd
    dw = (g * x).sum((0, 1, 2))
    g = g * w.detach().float()
    return rstd * (g - x * (g * x).mean(-1, keepdim=True)), dw


def _plain_rotate(s):
    cos, sin = _plain_angles(s)
    result = {}
    for x, w, g in (("q", "wq", "gq"), ("k", "wk", "gk")):
        dtype = s[x].dtype
        result[x] = _plain_norm_rotate(s, s[x], s[w], cos, sin).to(dtype)
        if s["case"]["mode"] == "train":
            dx, dw = _plain_norm_rotate_grad(s, s[x], s[w], s[g], cos, sin)
            result["d" + x] = dx.to(dtype)
            if dw is not None:
                result["d" + w] = dw.to(dtype)
    return result


def _plain_store(s):
    cos, sin = _plain_angles(s)
    case, dtype, dev = s["case"], s["q"].dtype, s["q"].device
    q, k = (_plain_norm_rotate(s, s[x], s[w], cos, sin).to(dtype) for x, w in (("q", "wq"), ("k", "wk")))
    new = torch.arange(case["length"], device=dev)
    at = s["positions"].long()[:, None] + new
    if s["lengths"] is not None:
        filled = new < s["lengths"].long()[:, None]
        q = q.masked_fill(~filled[:, :, None, None], 0)
        which = filled.nonzero(as_tuple=True)
        at, k, v = at[which], k[which], s["v"][which]
        page = s["pages"].long()[which[0], at // case["page"]]
    else:
        v = s["v"]
        page = s["pages"].long().gather(1, at // case["page"])
    s["keys"][page, at % case["page"]] = k
    s["values"][page, at % case["page"]] = v
    return {"q": q, "keys": s["keys"], "values": s["values"]}


def _plain_attention(s):
    case = s["case"]
    b, lq, h, hk, d = (case[k] for k in ("batch", "lq", "heads", "kv_heads", "dim"))
    dev = s["q"].device
    k, v = (s[n][s["pages"].long()].flatten(1, 2).float().transpose(1, 2) for n in ("keys", "values"))       # [batch, kv_heads, room, dim]
    q = s["q"].float().transpose(1, 2).reshape(b, hk, h // hk * lq, d)
    away = torch.arange(k.size(2), device=dev) - torch.arange(lq, device=dev)[:, None] - s["q_start"].long()[:, None, None]
    p = (q @ k.transpose(2, 3) / math.sqrt(d)).view(b, h, lq, -1)
    if s["bias"] is not None:
        reach = s["buckets"].numel() // 2
        p = p + s["bias"].float()[s["buckets"].long()[away.clamp(-reach, reach) + reach]].permute(0, 3, 1, 2)
    seen = (away <= 0) & (torch.arange(k.size(2), device=dev) < s["kv_lengths"].long()[:, None, None])
    p = p.masked_fill(~seen[:, None], -math.inf)
    p = torch.exp(p - p.amax(-1, keepdim=True).clamp_min(-1e30))
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-30)
    out = p.view(b, hk, h // hk * lq, -1) @ v
    return {"out": out.view(b, h, lq, d).transpose(1, 2).to(s["q"].dtype)}


def _plain_copy(s):
    s["storage"][s["target"].long()] = s["storage"][s["source"].long()]
    return {"storage": s["storage"]}


def run(s):
    case = s["case"]
    kind = case["kind"]
    if not own:
        return {"rotate": _plain_rotate, "store": _plain_store, "attention": _plain_attention, "copy": _plain_copy}[kind](s)
    import s2cnn_b200 as S
    if kind == "copy":
        S.copy_pages(s["storage"], s["source"], s["target"])
        return {"storage": s["storage"]}
    if kind == "attention":
        return {"out": S.paged_attention(s["q"], s["keys"], s["values"], s["pages"], s["bias"], s["buckets"], causal=True,
                                         q_start=s["q_start"], kv_lengths=s["kv_lengths"])}
    how = {"q_weight": s["wq"], "k_weight": s["wk"], "eps": EPS if case["norm"] else None, "positions": s["positions"], "interleaved": case["interleaved"]}
    if kind == "store":
        q = S.norm_rotate_store(s["q"], s["k"], s["v"], s["keys"], s["values"], s["pages"], s["frequencies"], lengths=s["lengths"], **how)
        return {"q": q, "keys": s["keys"], "values": s["values"]}
    q, k = S.norm_rotate(s["q"], s["k"], s["frequencies"], **how)
    if case["mode"] != "train":
        return {"q": q, "k": k}
    names = ("q", "k") + (("wq", "wk") if case["norm"] else ())
    grads = dict(zip(names, torch.autograd.grad((q, k), [s[n] for n in names], (s["gq"], s["gk"]))))
    result = {"q": q.detach(), "dq": grads["q"]}
    if case["norm"]:
        result["dwq"] = grads["wq"]
    result |= {"k": k.detach(), "dk": grads["k"]}
    if case["norm"]:
        result["dwk"] = grads["wk"]
    return result


def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    if case["kind"] == "copy":
        return {"bytes": 2 * case["copied"] * case["layers"] * 2 * case["kv_heads"] * case["page"] * _row(case) * size, "flops": 0}
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    if case["kind"] == "attention":
        keys = sum(_counts(case["batch"], case["lk"], case["ragged"]))
        queries = case["batch"] * case["lq"]
        return {"bytes": (2 * keys * hk + 2 * queries * h) * d * size, "flops": 4 * keys * case["lq"] * h * d}
    if case["kind"] == "store":
        new = sum(_counts(case["batch"], case["length"], case["ragged"]))
        return {"bytes": 2 * new * (h + 2 * hk) * d * size, "flops": 8 * new * (h + hk) * d}
    n = case["batch"] * case["length"] * (h + hk) * d
    train = case["mode"] == "train"
    return {"bytes": n * size * ((5 if case["norm"] else 4) if train else 2), "flops": n * (24 if train else 8)}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------------


def _exact_matrix(s, b):
    """[length, dim, dim] in 64 bits: what turns a head of each position of sequence b"""
    case, at = s["case"], s["positions"]
    n, r, d = case["length"], case["turned"], case["dim"]
    position = torch.arange(n, dtype=torch.float64, device="cuda") + (int(at[b]) if torch.is_tensor(at) else at)
    m = torch.eye(d, dtype=torch.float64, device="cuda").repeat(n, 1, 1)
    for pair, f in enumerate(_frequencies(r, case["factor"])):
        i, j = (2 * pair, 2 * pair + 1) if case["interleaved"] else (pair, pair + r // 2)
        c, t = torch.cos(position * f), torch.sin(position * f)
        m[:, i, i], m[:, j, j], m[:, i, j], m[:, j, i] = c, c, -t, t
    return m


def _exact_heads(s, x, w, dy=None):
    """(turned heads, and with dy: the gradients of x and w) of one kind of heads"""
    x = x.detach().double()
    weight = w.detach().double() if w is not None else None
    out, dx = torch.empty_like(x), torch.zeros_like(x)
    dw = torch.zeros(x.size(-1), dtype=torch.float64, device=x.device)
    for b in range(x.size(0)):
        m = None
        for lo in range(0, x.size(1), 512):
            sub = dict(s, case=dict(s["case"], length=min(512, x.size(1) - lo)), positions=(int(s["positions"][b]) if torch.is_tensor(s["positions"]) else s["positions"]) + lo)
            m = _exact_matrix(sub, b)
            part = x[b, lo:lo + 512]
            if weight is None:
                out[b, lo:lo + 512] = torch.einsum("nij,nhj->nhi", m, part)
            else:
                size = torch.sqrt(part.square().mean(-1, keepdim=True) + EPS)
                out[b, lo:lo + 512] = torch.einsum("nij,nhj->nhi", m, part / size * weight)
            if dy is not None:
                back = torch.einsum("nij,nhi->nhj", m, dy[b, lo:lo + 512].double())
                if weight is None:
                    dx[b, lo:lo + 512] = back
                else:
                    dw += (back * part / size).sum((0, 1))
                    back = back * weight
                    dx[b, lo:lo + 512] = back / size - part * (back * part).sum(-1, keepdim=True) / (x.size(-1) * size ** 3)
    return out, dx, dw


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["kind"] == "copy":
            before = s["storage"].clone()
            for a, b in zip(s["source"].tolist(), s["target"].tolist()):
                s["storage"][b].copy_(before[a])
            return {"storage": s["storage"]}
        if case["kind"] == "rotate":
            r = {}
            for x, w, g in (("q", "wq", "gq"), ("k", "wk", "gk")):
                r[x], dx, dw = _exact_heads(s, s[x], s[w], s.get(g))
                if case["mode"] == "train":
                    r["d" + x] = dx
                    if case["norm"]:
                        r["d" + w] = dw
            return r
        if case["kind"] == "store":
            q, k = _exact_heads(s, s["q"], s["wq"])[0], _exact_heads(s, s["k"], s["wk"])[0]
            keys, values = s["keys"].double(), s["values"].double()
            for b in range(case["batch"]):
                n = case["length"] if s["lengths"] is None else int(s["lengths"][b])
                q[b, n:] = 0
                at = torch.arange(n, device="cuda") + int(s["positions"][b])
                page, slot = s["pages"][b].long()[at // case["page"]], at % case["page"]
                keys[page, slot], values[page, slot] = k[b, :n], s["v"][b, :n].double()
            return {"q": q, "keys": keys, "values": values}
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        group = case["heads"] // case["kv_heads"]
        for b in range(case["batch"]):
            n, start = int(s["kv_lengths"][b]), int(s["q_start"][b])
            at = torch.arange(n, device="cuda")
            page, slot = s["pages"][b].long()[at // case["page"]], at % case["page"]
            k, v = s["keys"][page, slot].double(), s["values"][page, slot].double()
            away = at - torch.arange(case["lq"], device="cuda")[:, None] - start
            for h in range(case["heads"]):
                logits = s["q"][b, :, h].double() @ k[:, h // group].T / case["dim"] ** 0.5
                if s["bias"] is not None:
                    reach = (s["buckets"].numel() - 1) // 2
                    logits += s["bias"][:, h].double()[s["buckets"].long()[away.clamp(min=-reach, max=reach) + reach]]
                logits[away > 0] = -math.inf
                sees = (away <= 0).any(1)
                out[b, sees, h] = torch.exp(logits[sees] - torch.logsumexp(logits[sees], 1, keepdim=True)) @ v[:, h // group]
        return {"out": out}
