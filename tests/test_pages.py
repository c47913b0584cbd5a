"""Kept keys and values in pages: what is written where, attention over them, pages that are copied, and the account of a pool.

Tolerances.  Stored values and copies are bits.  Normed and turned heads: as in test_norm_rotate.py.  Attention: float32 5e-6 and
bfloat16 8e-3 as in test_sequence_ops.py, whose definition in 64 bits is used on keys and values gathered by indexing.
"""
import math

import pytest
import torch

import backends
import s2cnn_b200 as S
from test_norm_rotate import TOL as TURN_TOL
from test_norm_rotate import exact as exact_heads
from test_sequence_ops import TOL, exact_attention, normal, rel

F32, BF16 = torch.float32, torch.bfloat16


def ints(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def pool(gen, dev, dtype, count, page, Hk, D, how="heads"):
    """keys and values [count, page, Hk, D]: heads outside positions in rows of whole 16 bytes, positions outside heads, or odd rows"""
    if how == "heads":
        step = 16 // torch.empty(0, dtype=dtype).element_size()
        both = normal(gen, dev, dtype, count, 2, Hk, page, -(-D // step) * step)
        return both[:, 0].transpose(1, 2)[..., :D], both[:, 1].transpose(1, 2)[..., :D]
    if how == "positions":
        return normal(gen, dev, dtype, count, page, Hk, D), normal(gen, dev, dtype, count, page, Hk, D)
    both = normal(gen, dev, dtype, count, page, Hk, 2 * D + 3)
    return both[..., 1:D + 1], both[..., D + 2:2 * D + 2]


def shuffled(gen, dev, count, batch, columns):
    return torch.randperm(count, generator=gen)[:batch * columns].view(batch, columns).int().to(dev)


def gathered(keys, pages):
    """[batch, columns * page, heads, dim]; NaN where an entry is no page"""
    bad = (pages < 0) | (pages >= keys.size(0))
    out = keys[pages.long().masked_fill(bad, 0)]
    return out.masked_fill(bad[:, :, None, None, None], math.nan).flatten(1, 2)


# ---- attention ----------------------------------------------------------------------------------------------------------


def check_attention(dev, dtype, B, lq, room, H, Hk, D, page, bias=None, how="heads", seed=0, poison=True, **kw):
    gen = torch.Generator().manual_seed(seed)
    columns = -(-room // page)
    count = B * columns + 3
    keys, values = pool(gen, dev, dtype, count, page, Hk, D, how)
    pages = shuffled(gen, dev, count, B, columns)
    q = normal(gen, dev, dtype, B, lq, H + 1, D)[:, :, 1:]
    table = buckets = None
    if bias:
        table, buckets = normal(gen, dev, dtype, bias[0], H), S.relative_buckets(*bias, device=dev)
    kw = {n: ints(x, dev) if isinstance(x, list) else x for n, x in kw.items()}
    k, v = gathered(keys, pages), gathered(values, pages)
    want = exact_attention(q, k, v, table, buckets, **kw)[0]
    if poison:          # what is kept beyond a sequence's positions, and on pages that are nobody's
        seen = torch.zeros(count, page, dtype=torch.bool)
        for b in range(B):
            n = columns * page if "kv_lengths" not in kw else min(max(int(kw["kv_lengths"][b]), 0), columns * page)
            if kw.get("causal"):
                start = kw.get("q_start", 0)
                nq = lq if "q_lengths" not in kw else min(max(int(kw["q_lengths"][b]), 0), lq)
                n = min(n, max(0, (int(start[b]) if isinstance(start, torch.Tensor) else start) + nq))
            at = torch.arange(n)
            seen[pages[b].cpu().long()[at // page], at % page] = True
        keys[~seen.to(dev)], values[~seen.to(dev)] = math.nan, math.inf
    out = S.paged_attention(q, keys, values, pages, table, buckets, **kw)
    assert out.dtype == dtype and out.is_contiguous()
    assert rel(out, want) <= TOL[dtype], rel(out, want)
    return out


SMALL = [
    # B, lq, room, H, Hk, D, page, bias, kw
    (1, 1, 1, 1, 1, 1, 8, None, {}),
    (1, 1, 70, 4, 4, 10, 8, (8, 6), {"causal": True, "q_start": 69, "kv_lengths": [70]}),
    (2, 3, 100, 2, 1, 16, 16, (8, 3), {"kv_lengths": [41, 100], "causal": True, "q_start": [38, 97]}),
    (2, 1, 130, 4, 2, 25, 32, None, {"kv_lengths": [130, 17], "how": "positions"}),
    (3, 2, 64, 6, 3, 20, 16, (16, 30), {"kv_lengths": [64, 0, 33], "q_lengths": [2, 2, 1], "how": "odd"}),
    (2, 5, 48, 4, 1, 50, 8, (16, 64), {"causal": True, "q_start": [-2, 40], "kv_lengths": [45, 45]}),     # queries before the first key; 20 rows
    (1, 4, 90, 2, 2, 128, 64, None, {"causal": True, "q_start": 60, "kv_lengths": [200]}),               # more than the columns hold
    (2, 1, 40, 2, 2, 64, 128, None, {"kv_lengths": [-3, 1]}),
    (1, 33, 70, 2, 1, 32, 16, (8, 4), {"causal": True, "q_start": 30, "kv_lengths": [63]}),
    (1, 2, 64, 3, 1, 12, 32, None, {"how": "positions"}),                                                  # every position, without lengths
]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("case", SMALL, ids=lambda c: "x".join(map(str, c[:7])))
@pytest.mark.parametrize("backend", backends.BACKENDS)
def test_paged_attention(backend, case, dtype):
    with backends.active(backend) as (_, dev):
        B, lq, room, H, Hk, D, page, bias, kw = case
        check_attention(dev, dtype, B, lq, room, H, Hk, D, page, bias, **kw)


LARGE = [
    (16, 1, 2000, 16, 4, 128, 64, None, {"causal": True, "q_start": [1999 - 120 * i for i in range(16)], "kv_lengths": [2000 - 120 * i for i in range(16)]}),
    (3, 2, 777, 10, 2, 25, 16, (32, 64), {"kv_lengths": [777, 0, 513], "how": "positions"}),
    (1, 1, 9000, 8, 1, 128, 128, (32, 128), {"causal": True, "q_start": 8999}),
    (1, 1, 9000, 1, 1, 80, 8, None, {"kv_lengths": [8999]}),
    (2, 4, 1500, 12, 4, 64, 32, (32, 128), {"causal": True, "q_start": [1496, 3], "kv_lengths": [1500, 7]}),
    (1, 16, 600, 16, 1, 128, 64, (32, 2048), {"causal": True, "q_start": 500}),                            # 256 rows for one head of keys
    (40, 1, 300, 6, 6, 64, 16, None, {"kv_lengths": [300 - 7 * i for i in range(40)]}),
    (300, 1, 70, 2, 1, 40, 16, None, {"kv_lengths": [(37 * i) % 71 for i in range(300)]}),                 # more sequences than threads, empty ones among them
    (2, 3, 3000, 5, 1, 100, 64, (16, 64), {"causal": True, "q_start": [2900, 1000], "kv_lengths": [2903, 1003], "how": "odd"}),
    (2, 40, 900, 4, 2, 64, 64, None, {"causal": True, "q_start": [860, 200], "kv_lengths": [900, 240]}),
    (2, 70, 700, 8, 2, 64, 32, (16, 64), {"causal": True, "q_start": [600, 100], "kv_lengths": [650, 160], "q_lengths": [70, 33]}),   # one array for whole tiles
    (1, 100, 500, 6, 2, 25, 16, None, {"kv_lengths": [333], "how": "odd"}),
    (1, 300, 300, 2, 1, 128, 64, None, {"causal": True}),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("case", LARGE, ids=lambda c: "x".join(map(str, c[:7])))
def test_paged_attention_over_many_pages(case, dtype):
    B, lq, room, H, Hk, D, page, bias, kw = case
    a = check_attention("cuda", dtype, B, lq, room, H, Hk, D, page, bias, **kw)
    assert torch.equal(a, check_attention("cuda", dtype, B, lq, room, H, Hk, D, page, bias, **kw))        # the same in every call


@pytest.mark.parametrize("backend", backends.BACKENDS)
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_entries_that_are_no_page_read_as_nan(backend, dtype):
    """where a query sees them, and nowhere else"""
    with backends.active(backend) as (_, dev):
        gen = torch.Generator().manual_seed(1)
        keys, values = pool(gen, dev, dtype, 9, 16, 2, 24)
        pages = ints([[0, 1, 2], [3, -1, 4], [5, 6, 9], [7, 1 << 30, -(1 << 31)]], dev)
        q = normal(gen, dev, dtype, 4, 1, 4, 24)
        for lengths, bad in (([48, 48, 48, 48], [False, True, True, True]), ([48, 16, 32, 16], [False] * 4), ([1, 17, 33, 0], [False, True, True, False])):
            out = S.paged_attention(q, keys, values, pages, kv_lengths=ints(lengths, dev))
            for b in range(4):
                if bad[b]:
                    assert out[b].isnan().all()
                else:
                    n = lengths[b]
                    want = exact_attention(q[b:b + 1], gathered(keys, pages[b:b + 1])[:, :n], gathered(values, pages[b:b + 1])[:, :n])[0]
                    assert rel(out[b:b + 1], want) <= TOL[dtype]


@pytest.mark.parametrize("backend", backends.BACKENDS)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lq", [1, 20])
def test_bias_of_the_lowest_value(backend, dtype, lq):
    """A bucket of the type's lowest value or of -infinity takes no weight; a row of the lowest value alone is a plain mean."""
    with backends.active(backend) as (_, dev):
        gen = torch.Generator().manual_seed(2)
        keys, values = pool(gen, dev, dtype, 6, 16, 2, 16)
        pages, q = ints([[4, 0, 5, 2, 3]], dev), normal(gen, dev, dtype, 1, lq, 2, 16)
        buckets = S.relative_buckets(8, 4, device=dev)
        k, v = gathered(keys, pages), gathered(values, pages)
        for low in (torch.finfo(dtype).min, -math.inf):
            table = torch.zeros(8, 2, dtype=dtype, device=dev)
            table[4:] = low                                      # keys behind the query
            out = S.paged_attention(q, keys, values, pages, table, buckets, q_start=50)
            assert rel(out, exact_attention(q, k, v, causal=True, q_start=50)[0]) <= TOL[dtype]
        table = torch.full((8, 2), torch.finfo(dtype).min, dtype=dtype, device=dev)
        out = S.paged_attention(q, keys, values, pages, table, buckets)
        assert (out.double().cpu() - v.double().cpu().mean(1, keepdim=True)).abs().max() <= TOL[dtype] * 4
        # -infinity everywhere: nothing is seen
        out = S.paged_attention(q, keys, values, pages, torch.full_like(table, -math.inf), buckets)
        assert not out.any()


@pytest.mark.parametrize("backend", backends.BACKENDS)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows", [(1, 2), (2, 6), (20, 2)], ids=str)
def test_an_infinity_that_is_seen_stays_in_its_column(backend, dtype, rows):
    """and in the heads that share its key head"""
    with backends.active(backend) as (_, dev):
        gen = torch.Generator().manual_seed(3)
        lq, H = rows
        keys, values = pool(gen, dev, dtype, 8, 16, 2, 40)
        pages, q = ints([[4, 0, 5, 2, 3, 1]], dev), normal(gen, dev, dtype, 1, lq, H, 40)
        want = S.paged_attention(q, keys, values, pages)
        for bad in (math.inf, -math.inf, math.nan):
            w = values.clone()
            w[5, 3, 1, 5] = bad
            out = S.paged_attention(q, keys, w, pages)
            assert not torch.isfinite(out[0, :, H // 2:, 5]).any()
            out[0, :, H // 2:, 5] = want[0, :, H // 2:, 5]
            assert rel(out, want) <= TOL[dtype]
            k = keys.clone()
            k[5, 3, 1, 5] = bad
            out = S.paged_attention(q, k, values, pages)
            assert rel(out[:, :, :H // 2], want[:, :, :H // 2]) <= TOL[dtype]


@pytest.mark.parametrize("backend", backends.BACKENDS)
def test_paged_attention_without_positions(backend):
    with backends.active(backend) as (_, dev):
        keys = torch.ones(4, 8, 2, 16, device=dev)
        for B, lq, columns, count in ((0, 1, 2, 4), (2, 0, 2, 4), (2, 3, 0, 4), (2, 1, 0, 0)):
            out = S.paged_attention(torch.ones(B, lq, 4, 16, device=dev), keys[:count], keys[:count], torch.zeros(B, columns, dtype=torch.int32, device=dev))
            assert out.shape == (B, lq, 4, 16) and not out.any()
        out = S.paged_attention(torch.ones(1, 1, 2, 16, device=dev), keys[:0], keys[:0], ints([[0, 0]], dev))        # a pool without pages
        assert out.isnan().all()
        assert not S.paged_attention(torch.ones(1, 1, 2, 16, device=dev), keys[:0], keys[:0], ints([[0, 0]], dev), kv_lengths=ints([0], dev)).any()


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """A pool whose pages lie 2^22 elements apart: the last of 1500 lie 6.3e9 elements behind the first."""
    gen = torch.Generator().manual_seed(4)
    room = torch.empty(1500, 1 << 22, dtype=BF16, device="cuda")
    keys, values = (room[:, n * 4096:(n + 1) * 4096].unflatten(1, (2, 16, 128)).transpose(1, 2) for n in (0, 1000))
    small = [normal(gen, "cuda", BF16, 1500, 2, 16, 128).transpose(1, 2) for _ in range(2)]
    keys.copy_(small[0])
    values.copy_(small[1])
    pages, q = torch.randperm(1500, generator=gen)[None].int().cuda(), normal(gen, "cuda", BF16, 1, 1, 8, 128)
    assert torch.equal(S.paged_attention(q, keys, values, pages), S.paged_attention(q, *small, pages))
    k, v = normal(gen, "cuda", BF16, 1, 3, 2, 128), normal(gen, "cuda", BF16, 1, 3, 2, 128)
    for a, b in ((keys, values), small):
        S.norm_rotate_store(None, k, v, a, b, pages, positions=1500 * 16 - 3)
    assert torch.equal(keys, small[0]) and torch.equal(values, small[1])
    S.copy_pages(room, ints([1499, 0], "cuda"), ints([3, 1498], "cuda"))
    assert torch.equal(room[3], room[1499]) and torch.equal(room[1498], room[0])


# ---- storing ------------------------------------------------------------------------------------------------------------


STORE = [
    # B, new, H, Hk, D, pairs, page, columns, positions, lengths, how, kw
    (1, 1, 1, 1, 1, 0, 8, 1, 0, None, "positions", {}),
    (2, 1, 4, 2, 10, 5, 8, 3, [23, 7], None, "heads", {}),
    (3, 5, 4, 2, 25, 12, 16, 2, [0, 14, 27], [5, 0, 3], "heads", {"interleaved": True}),
    (2, 9, 6, 2, 64, 16, 8, 4, [30, 3], [2, 12], "positions", {"eps": None}),
    (1, 20, 2, 2, 128, 64, 16, 2, 12, None, "heads", {"magnitude": 1.5}),
    (2, 4, 3, 1, 32, 16, 32, 1, [[5, 0, 31, 9], [1, 2, 3, 20]], None, "odd", {}),
    (1, 3, 2, 1, 80, 40, 64, 1, 61, None, "heads", {"weights": False}),
]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("case", STORE, ids=lambda c: "x".join(map(str, c[:8])))
@pytest.mark.parametrize("backend", backends.BACKENDS)
def test_store(backend, case, dtype):
    """Keys and values in their places, all others as they were, and the queries of norm_rotate."""
    with backends.active(backend) as (_, dev):
        B, new, H, Hk, D, pairs, page, columns, positions, lengths, how, kw = case
        kw = dict(kw)
        gen = torch.Generator().manual_seed(10)
        count = B * columns + 2
        keys, values = pool(gen, dev, dtype, count, page, Hk, D, how)
        pages = shuffled(gen, dev, count, B, columns)
        q, k, v = normal(gen, dev, dtype, B, new, H + 2 * Hk, D).split((H, Hk, Hk), 2)
        eps = kw.pop("eps", 1e-6)
        wq, wk = (normal(gen, dev, dtype, D), normal(gen, dev, dtype, D)) if kw.pop("weights", True) and eps is not None else (None, None)
        f = S.rotary_frequencies(2 * pairs, device=dev) if pairs else None
        at = ints(positions, dev) if isinstance(positions, list) else positions
        want_q, want_k = (exact_heads(x, w, f, eps, at, kw.get("interleaved", False), kw.get("magnitude", 1.0)) for x, w in ((q, wq), (k, wk)))
        turned = S.norm_rotate(q, k, f, wq, wk, eps, positions=at, **kw)
        before = keys.clone(), values.clone()
        if lengths is not None:                     # what is not filled is not read
            for b in range(B):
                for t in (q, k, v):
                    t[b, max(0, lengths[b]):] = math.nan
        for queries in (q, None):
            keys.copy_(before[0])
            values.copy_(before[1])
            out = S.norm_rotate_store(queries, k, v, keys, values, pages, f, wq, wk, eps, positions=at, lengths=None if lengths is None else ints(lengths, dev), **kw)
            expect = before[0].clone(), before[1].clone()
            for b in range(B):
                for i in range(new):
                    where = positions + i if not isinstance(positions, list) else positions[b][i] if isinstance(positions[b], list) else positions[b] + i
                    filled, there = lengths is None or i < lengths[b], 0 <= where < columns * page
                    if filled and there:
                        place = int(pages[b, where // page]), where % page
                        expect[0][place], expect[1][place] = turned[1][b, i], v[b, i]
                        assert rel(turned[1][b, i], want_k[b, i]) <= 2 * TURN_TOL[dtype]
                    if queries is not None:
                        if filled and there:
                            assert torch.equal(out[b, i], turned[0][b, i]) and rel(out[b, i], want_q[b, i]) <= 2 * TURN_TOL[dtype]
                        else:
                            assert out[b, i].isnan().all() if filled else not out[b, i].any()
            assert torch.equal(keys, expect[0]) and torch.equal(values, expect[1])
            assert (out is None) == (queries is None)


@pytest.mark.parametrize("backend", backends.BACKENDS)
def test_store_beside_entries_that_are_no_page(backend):
    with backends.active(backend) as (_, dev):
        gen = torch.Generator().manual_seed(11)
        keys, values = pool(gen, dev, F32, 4, 8, 1, 16)
        before = keys.clone(), values.clone()
        q, k, v = (normal(gen, dev, F32, 5, 2, n, 16) for n in (2, 1, 1))
        pages = ints([[2, 0], [-1, 0], [4, 0], [1, 1 << 30], [3, 0]], dev)
        out = S.norm_rotate_store(q, k, v, keys, values, pages, positions=ints([0, 0, 0, 7, -1], dev))
        bad = torch.tensor([[0, 0], [1, 1], [1, 1], [0, 1], [1, 0]], dtype=torch.bool)
        assert torch.equal(out.isnan().all(-1).all(-1).cpu(), bad) and torch.equal(out[~bad.to(dev)], q[~bad.to(dev)])
        for b, i, page, at in ((0, 0, 2, 0), (0, 1, 2, 1), (3, 0, 1, 7), (4, 1, 3, 0)):
            assert torch.equal(keys[page, at], k[b, i]) and torch.equal(values[page, at], v[b, i])
            before[0][page, at], before[1][page, at] = k[b, i], v[b, i]
        assert torch.equal(keys, before[0]) and torch.equal(values, before[1])


# ---- copying ------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("backend", backends.BACKENDS)
@pytest.mark.parametrize("dtype", [torch.uint8, BF16, F32, torch.float64])
@pytest.mark.parametrize("shape", [(7, 1), (9, 3), (5, 4096), (6, 2, 4099), (1, 5)], ids=str)
def test_copy_pages(backend, dtype, shape):
    with backends.active(backend) as (_, dev):
        gen = torch.Generator().manual_seed(12)
        for gap in (0, 3):
            room = (torch.rand(shape[0], math.prod(shape[1:]) + gap, generator=gen) * 200).to(dtype).to(dev)
            storage = room[:, :math.prod(shape[1:])].unflatten(1, shape[1:])
            want = room.clone()
            n = shape[0]
            source, target = [0, 0, n - 1, -1, n, 2], [n - 2, 1, n - 3, 3, 3, n + 5]
            keep = [(a, b) for a, b in zip(source, target) if 0 <= a < n and 0 <= b < n and n > 4]
            if n <= 4:
                source, target = [0, 5], [1, 0]
            for a, b in keep:
                want[b, :math.prod(shape[1:])] = room[a, :math.prod(shape[1:])]
            S.copy_pages(storage, ints(source, dev), ints(target, dev))
            assert torch.equal(room, want)
            S.copy_pages(storage, ints([], dev), ints([], dev))
            assert torch.equal(room, want)


# ---- the account of a pool --------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("backend", backends.BACKENDS)
def test_paged_cache_follows_its_sequences(backend):
    """A few hundred steps, forks, cuts and compactions beside plain lists of what each sequence holds."""
    with backends.active(backend) as (_, dev):
        import random
        rng = random.Random(13)
        gen = torch.Generator().manual_seed(13)
        layers, Hk, D, slots = 2, 1, 10, 4
        cache = S.PagedCache(12, 8, Hk, D, slots, columns=5, layers=layers, device=dev)
        held = [[[] for _ in range(slots)] for _ in range(layers)]
        table, filled = cache.table.data_ptr(), cache.filled.data_ptr()
        refused = 0
        for step in range(150):
            what = rng.choice(["extend"] * 6 + ["fork", "truncate", "free", "compact"])
            s = rng.randrange(slots)
            if what == "extend":
                new = [rng.choice([0, 1, 1, 2, 5, 9]) for _ in range(slots)]
                account = cache.lengths[:], [p[:] for p in cache._pages], cache._uses[:], sorted(cache._free), cache.table.clone()
                try:
                    cache.extend(new)
                except MemoryError:
                    refused += 1
                    assert account[:4] == (cache.lengths, cache._pages, cache._uses, sorted(cache._free)) and torch.equal(account[4], cache.table)
                    continue
                if rng.random() < 0.2:                   # asked again for less
                    new = [n // 2 for n in new]
                    cache.extend(new)
                n = max(new)
                if n:
                    for layer in range(layers):
                        k, v = normal(gen, dev, F32, slots, n, Hk, D), normal(gen, dev, F32, slots, n, Hk, D)
                        S.norm_rotate_store(None, k, v, cache.keys(layer), cache.values(layer), cache.table, positions=cache.filled, lengths=ints(new, dev))
                        for i in range(slots):
                            held[layer][i] += [(k[i, j], v[i, j]) for j in range(new[i])]
                cache.advance()
            elif what == "fork":
                others = [i for i in range(slots) if i != s and not cache.lengths[i] and not cache._pages[i]]
                if others:
                    cache.fork(s, others[0])
                    for layer in range(layers):
                        held[layer][others[0]] = held[layer][s][:]
            elif what == "truncate":
                n = rng.randint(0, cache.lengths[s])
                cache.truncate(s, n)
                for layer in range(layers):
                    del held[layer][s][n:]
            elif what == "free":
                cache.free(s)
                for layer in range(layers):
                    held[layer][s] = []
            else:
                n = cache.compact()
                assert n == 12 - cache.free_pages and all(p < n for pages in cache._pages for p in pages)
            assert cache.lengths == [len(x) for x in held[0]] == cache.filled.tolist()
            users = [p for pages in cache._pages for p in pages]
            assert sorted(cache._free + sorted(set(users))) == list(range(12)) and cache._uses == [users.count(p) for p in range(12)]
            for layer in range(layers):
                for i in range(slots):
                    n = cache.lengths[i]
                    if n:
                        k, v = (gathered(t, cache.table[i:i + 1])[0, :n] for t in (cache.keys(layer), cache.values(layer)))
                        assert torch.equal(k, torch.stack([x[0] for x in held[layer][i]])) and torch.equal(v, torch.stack([x[1] for x in held[layer][i]]))
        assert refused and (table, filled) == (cache.table.data_ptr(), cache.filled.data_ptr())


@pytest.mark.parametrize("backend", backends.BACKENDS)
def test_paged_cache_refusals(backend):
    with backends.active(backend) as (_, dev):
        for kw in ({"page": 12}, {"page": 4}, {"pages": 0}, {"sequences": 0}):
            with pytest.raises(AssertionError):
                S.PagedCache(**{**dict(pages=4, page=8, kv_heads=1, dim=8, sequences=2, device=dev), **kw})
        cache = S.PagedCache(4, 8, 1, 8, 2, columns=3, device=dev)
        with pytest.raises(MemoryError):
            cache.extend([25, 0])                        # columns
        with pytest.raises(MemoryError):
            cache.extend([24, 9])                        # pages
        with pytest.raises(AssertionError):
            cache.extend([1])
        with pytest.raises(AssertionError):
            cache.extend(-1)
        cache.extend([5, 0])
        for call in (lambda: cache.fork(0, 1), lambda: cache.truncate(0, 0), lambda: cache.free(0), cache.compact):
            with pytest.raises(AssertionError):
                call()                                   # within a step
        cache.advance()
        for call in (lambda: cache.fork(0, 0), lambda: cache.truncate(0, 6), lambda: cache.truncate(0, -1)):
            with pytest.raises(AssertionError):
                call()
        cache.extend([0, 1])
        cache.advance()
        with pytest.raises(AssertionError):
            cache.fork(0, 1)


# ---- in a block ---------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("backend", backends.BACKENDS)
def test_steps_of_nothing(backend):
    """No new positions, no sequences, sequences of which some have none: shapes, zeros where nothing is filled, nothing written."""
    with backends.active(backend) as (_, dev):
        torch.manual_seed(23)
        block = S.SequenceBlock(16, 2, causal=True, p=0.0, rotary=8).to(dev).eval()
        cache = S.PagedCache(4, 8, 2, 8, 2, device=dev)
        args = cache.keys(), cache.values(), cache.table, cache.filled
        assert block.step_pages(torch.randn(2, 0, 16, device=dev), *args).shape == (2, 0, 16)
        assert block.step_pages(torch.randn(0, 1, 16, device=dev), *args[:2], cache.table[:0], cache.filled[:0]).shape == (0, 1, 16)
        cache.extend(0)
        cache.advance()
        assert cache.lengths == [0, 0] and cache.free_pages == 4 and not cache.storage.any()
        cache.extend([0, 2])
        x = torch.randn(2, 2, 16, device=dev)
        out = block.step_pages(x, *args, lengths=ints([0, 2], dev))
        cache.advance()
        alone = block(x[1:]).detach()
        assert torch.isfinite(out).all() and rel(out[1:], alone) <= 2e-5
        used = cache._pages[1][0]
        rest = [p for p in range(4) if p != used]
        assert cache.storage[used].any() and not cache.storage[rest].any()


@pytest.mark.parametrize("backend", backends.BACKENDS)
@pytest.mark.parametrize("how", ["bias", "rotary", "rotary, head norm"])
@pytest.mark.parametrize("page", [8, 16])
def test_block_in_pages_agrees_with_whole_sequences(backend, how, page):
    """A layer's answers position by position, and in chunks of different lengths, over a cache that forks and is compacted on the way, are
    those for whole sequences (float32; 2e-5 through norms, two linear layers and attention)."""
    with backends.active(backend) as (_, dev):
        torch.manual_seed(20)
        kw = {} if how == "bias" else {"rotary": 6, "head_norm": how != "rotary"}
        block = S.SequenceBlock(32, 4, 2, causal=True, p=0.0, num_buckets=8, reach=5, **kw).to(dev).eval()
        with torch.no_grad():
            for p in block.parameters():
                p.add_(torch.randn(p.shape).to(dev) * 0.1)
        x = torch.randn(2, 30, 32).to(dev)
        whole = block(x)
        cache = S.PagedCache(16, page, 2, 8, 3, device=dev)

        def step(parts):
            new = [p.size(0) for p in parts]
            cache.extend(new)
            padded = torch.full((3, max(new), 32), math.nan, device=dev)
            for row, p in zip(padded, parts):
                row[:p.size(0)] = p
            out = block.step_pages(padded, cache.keys(), cache.values(), cache.table, cache.filled, ints(new, dev))
            cache.advance()
            return [o[:n] for o, n in zip(out, new)]

        none = x[0, :0]
        a = step([x[0, :13], x[1, :20], none])
        assert rel(a[0], whole[0, :13]) <= 2e-5 and rel(a[1], whole[1, :20]) <= 2e-5
        cache.fork(0, 2)                                                     # goes on as another sequence would
        cache.truncate(2, 11)
        a = step([x[0, 13:14], x[1, 20:23], x[0, 11:15]])
        assert rel(a[0], whole[0, 13:14]) <= 2e-5 and rel(a[1], whole[1, 20:23]) <= 2e-5 and rel(a[2], whole[0, 11:15]) <= 2e-5
        cache.free(1)
        cache.compact()
        a = step([x[0, 14:30], none, x[0, 15:16]])
        assert rel(a[0], whole[0, 14:]) <= 2e-5 and rel(a[2], whole[0, 15:16]) <= 2e-5
        room_k, room_v = (torch.zeros(2, 30, 2, 8, device=dev) for _ in range(2))      # the padded room gives the same
        filled = ints([0, 0], dev)
        for i, j in ((0, 12), (12, 13), (13, 30)):
            out = block.step(x[:, i:j], room_k, room_v, filled).detach()
            assert rel(out, whole[:, i:j]) <= 2e-5
            filled += j - i


@pytest.mark.parametrize("backend", backends.BACKENDS)
def test_block_without_a_page_gives_nan(backend):
    with backends.active(backend) as (_, dev):
        torch.manual_seed(21)
        block = S.SequenceBlock(16, 2, causal=True, p=0.0, rotary=8).to(dev).eval()
        cache = S.PagedCache(3, 8, 2, 8, 2, device=dev)
        cache.extend([7, 8])
        cache.advance()
        out = block.step_pages(torch.randn(2, 1, 16, device=dev), cache.keys(), cache.values(), cache.table, cache.filled)
        assert torch.isfinite(out[0]).all() and out[1].isnan().all()


@pytest.mark.parametrize("backend", backends.BACKENDS)
def test_rotary_block_trains(backend):
    """Its gradients against differences (as in test_norm_rotate.py), its types, and frequencies that no cast changes."""
    with backends.active(backend) as (_, dev):
        torch.manual_seed(22)
        block = S.SequenceBlock(16, 2, causal=True, p=0.0, rotary=6, frequencies=S.rotary_frequencies(6, base=50.0), head_norm=True).to(dev)
        assert set(n for n, _ in block.named_parameters()) >= {"q_norm", "k_norm"} and "bias.weight" not in dict(block.named_parameters())
        assert "frequencies" not in block.state_dict()
        x, g = torch.randn(1, 6, 16).to(dev), torch.randn(1, 6, 16).to(dev) / 10
        f = lambda: (block(x).double() * g).sum()  # noqa: E731
        grads = torch.autograd.grad(f(), list(block.parameters()))
        for p, grad in zip(block.parameters(), grads):
            way = torch.randn(p.shape).to(dev)
            way /= way.norm()
            slopes = []
            with torch.no_grad():
                for s in (1, -2, 1):
                    p.add_(s * 1e-2 * way)
                    slopes.append(f().item())
            assert abs((slopes[0] - slopes[1]) / 2e-2 - (grad * way).sum().item()) <= 3e-4
        want = block.frequencies.clone()
        out = block.to(torch.bfloat16)(x.bfloat16())
        assert block.frequencies.dtype == torch.float64 and torch.equal(block.frequencies, want) and out.dtype == BF16
        with pytest.raises(AssertionError):
            S.SequenceBlock(16, 2, rotary=10)
        with pytest.raises(AssertionError):
            S.SequenceBlock(16, 2, head_norm=True)


# ---- refusals -----------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("backend", backends.BACKENDS)
def test_refusals(backend):
    with backends.active(backend) as (_, dev):
        new = lambda *shape: torch.zeros(*shape, device=dev)  # noqa: E731
        keys, q, k, pages = new(4, 8, 2, 16), new(1, 2, 4, 16), new(1, 2, 2, 16), ints([[0, 1]], dev)
        at = lambda q=q, keys=keys, values=None, pages=pages, *a, **kw: S.paged_attention(q, keys, keys if values is None else values, pages, *a, **kw)  # noqa: E731
        store = lambda q=q, k=k, v=None, keys=keys, values=None, pages=pages, **kw: S.norm_rotate_store(  # noqa: E731
            q, k, k if v is None else v, keys, keys.clone() if values is None else values, pages, **kw)
        leaf = new(1, 2, 4, 16).requires_grad_(True)
        for error, call in [
            (AssertionError, lambda: at(keys=new(4, 12, 2, 16))),                   # positions of a page
            (AssertionError, lambda: at(keys=new(4, 4, 2, 16))),
            (AssertionError, lambda: at(keys=new(4, 8, 3, 16))),
            (AssertionError, lambda: at(keys=new(4, 8, 2, 8))),
            (AssertionError, lambda: at(values=new(4, 8, 1, 16))),
            (AssertionError, lambda: at(keys=new(4, 8, 16, 2).transpose(2, 3))),    # last axis not contiguous
            (AssertionError, lambda: at(q=new(2, 2, 4, 16))),
            (AssertionError, lambda: at(q=new(2, 4, 16))),
            (RuntimeError, lambda: at(q=new(1, 1, 2, 129), keys=new(4, 8, 2, 129))),
            (AssertionError, lambda: at(pages=pages[0])),
            (AssertionError, lambda: at(pages=ints([[0, 1], [2, 3]], dev).t()[:1])),
            (TypeError, lambda: at(pages=pages.long())),
            (TypeError, lambda: at(q=q.bfloat16())),
            (TypeError, lambda: at(q=q.double(), keys=keys.double())),
            (TypeError, lambda: at(kv_lengths=torch.zeros(1, dtype=torch.int64, device=dev))),
            (AssertionError, lambda: at(kv_lengths=ints([1, 1], dev))),
            (AssertionError, lambda: at(bias=new(8, 4))),
            (RuntimeError, lambda: at(q=leaf)),
            (TypeError, lambda: store(k=None)),
            (AssertionError, lambda: store(v=new(1, 2, 1, 16))),
            (AssertionError, lambda: store(v=new(1, 3, 2, 16))),
            (AssertionError, lambda: store(k=new(1, 2, 1, 16), v=new(1, 2, 1, 16))),
            (AssertionError, lambda: store(keys=new(1, 8, 2, 16).expand(4, 8, 2, 16))),
            (AssertionError, lambda: store(pages=ints([[0], [1]], dev))),
            (AssertionError, lambda: store(lengths=ints([1, 1], dev))),
            (TypeError, lambda: store(keys=keys.bfloat16())),
            (RuntimeError, lambda: store(q=leaf)),
            (AssertionError, lambda: S.copy_pages(new(4), pages[0], pages[0])),
            (AssertionError, lambda: S.copy_pages(new(4, 6, 2).transpose(1, 2), pages[0], pages[0])),
            (AssertionError, lambda: S.copy_pages(new(1, 6).expand(4, 6), pages[0], pages[0])),
            (AssertionError, lambda: S.copy_pages(new(4, 6), pages[0], ints([1], dev))),
            (AssertionError, lambda: S.copy_pages(new(4, 6), pages, pages)),
            (TypeError, lambda: S.copy_pages(new(4, 6), pages[0].long(), pages[0].long())),
            (RuntimeError, lambda: S.copy_pages(leaf, pages[0], pages[0])),
        ]:
            with pytest.raises(error):
                call()
        with torch.no_grad():
            at(q=leaf)
        assert not keys.any()
