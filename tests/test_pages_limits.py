"""Turned heads and kept keys in pages where they could go wrong: numbers at the ends of float32, memory that is not there, widths, many items.

Tolerances: as in test_norm_rotate.py and test_pages.py; what is compared without one is bits.
"""
import ctypes
import math
import random

import pytest
import torch

import backends
import s2cnn_b200 as S
from s2cnn_b200 import _lib
from test_norm_rotate import normal
from test_pages import check_attention, gathered, ints, pool, shuffled
from test_pages_calls import attention_desc, page_desc
from test_sequence_ops import TOL, exact_attention, rel

F32, BF16 = torch.float32, torch.bfloat16


# ---- heads --------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("backend", backends.BACKENDS)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", [(24, 8, False), (24, 24, False), (40, 16, False), (80, 80, False), (128, 64, False), (20, 20, True), (44, 8, True), (25, 24, True)], ids=str)
def test_squares_that_overflow(backend, dtype, shape):
    """Where the sum of a head's squares is no float32 its inverse root is 0: the head is zeros, its gradient too, and it adds nothing to the
    weight's.  Other heads are as they were.  (1e20 is in the range of both types; its square is not.)"""
    with backends.active(backend) as (_, dev):
        D, turned, interleaved = shape
        gen = torch.Generator().manual_seed(60)
        f, w = S.rotary_frequencies(turned, device=dev), normal(gen, dev, dtype, D, scale=0.3, shift=1.0).requires_grad_(True)
        q, g = normal(gen, dev, dtype, 1, 7, 5, D), normal(gen, dev, dtype, 1, 7, 5, D)
        large, none = q.clone(), q.clone()
        for place in range(0, D, 3):
            i, h = place // 3 % 7, place // 3 % 5
            large[0, i, h, place] = 1e20
            none[0, i, h] = 0
        grads = []
        for x in (large, none):
            x.requires_grad_(True)
            y, _ = S.norm_rotate(x, None, f, w, eps=1e-6, positions=5, interleaved=interleaved)
            grads.append((y.detach(),) + torch.autograd.grad(y, (x, w), g))
        zeros = (none == 0).all(-1)
        for a, b in zip(grads[0][:2], grads[1][:2]):
            assert not a[zeros].any() and torch.equal(a[~zeros], b[~zeros])
        assert torch.equal(grads[0][2], grads[1][2])


@pytest.mark.parametrize("backend", backends.BACKENDS)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", [(24, 8, False), (64, 64, False), (20, 8, True), (25, 24, True)], ids=str)
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_frequencies_that_are_no_numbers(backend, dtype, shape, bad):
    """Their pair is NaN at every position (an infinity times position 0 is, too), in the gradient as well; other pairs are as they were."""
    with backends.active(backend) as (_, dev):
        D, turned, interleaved = shape
        gen = torch.Generator().manual_seed(61)
        f, w = S.rotary_frequencies(turned, device=dev), normal(gen, dev, dtype, D, scale=0.3, shift=1.0).requires_grad_(True)
        wrong, pair = f.clone(), turned // 4
        wrong[pair] = bad
        at = torch.zeros(D, dtype=torch.bool, device=dev)
        at[[2 * pair, 2 * pair + 1] if interleaved else [pair, pair + turned // 2]] = True
        q, g = normal(gen, dev, dtype, 2, 3, 3, D).requires_grad_(True), normal(gen, dev, dtype, 2, 3, 3, D)
        for eps in (None, 1e-6):
            for positions in (0, -4):
                results = []
                for x in (f, wrong):
                    y, _ = S.norm_rotate(q, None, x, None if eps is None else w, eps=eps, positions=positions, interleaved=interleaved)
                    results.append((y.detach(),) + torch.autograd.grad(y, (q,) if eps is None else (q, w), g))
                for n, (fine, out) in enumerate(zip(*results)):
                    if n == 1 and eps is not None:            # through the norm a pair reaches the whole head
                        assert out.isnan().all()
                    else:
                        assert out[..., at].isnan().all() and torch.equal(out[..., ~at], fine[..., ~at])
        keys, values = (torch.zeros(1, 8, 3, D, dtype=dtype, device=dev) for _ in range(2))
        with torch.no_grad():
            out = S.norm_rotate_store(q[:1], q[:1], q[:1], keys, values, torch.zeros(1, 1, dtype=torch.int32, device=dev), wrong, interleaved=interleaved)
        for t in (out[0], keys[0, :3]):
            assert t[..., at].isnan().all() and torch.isfinite(t[..., ~at]).all()
        assert torch.equal(values[0, :3], q[0])


# Rows behind `lengths` that are not there: q, k and v end where memory that may not be read begins.  Run in a process of its own, on the CPU.
_ENDS = """
import ctypes, mmap, sys
import torch
import backends, emul
import s2cnn_b200 as S
from test_pages import ints, pool, shuffled
from test_pages_calls import head_desc, page_desc
import s2cnn_b200.ops as ops_mod
ops_mod._cuda_ops = ops = emul.ops()
libc = ctypes.CDLL(None, use_errno=True)
D, dtype, interleaved = int(sys.argv[1]), getattr(torch, sys.argv[2]), sys.argv[3] == "True"
H, Hk, B, new, half = 12, 5, 3, 4, 1 << 16
size = torch.empty(0, dtype=dtype).element_size()
gen = torch.Generator().manual_seed(62)
f = S.rotary_frequencies(D // 4 * 2)
pages = shuffled(gen, "cpu", 8, B, 2)
# the filled rows of the middle sequence end where the closed part begins; those of the first one would lie in it altogether
lengths = ints([0, 2, 0], "cpu")
for backwards in (False, True):
    want, at = {}, {}
    for name, n in (("q", H), ("k", Hk), ("v", Hk)):
        room = mmap.mmap(-1, 2 * half)
        base = ctypes.addressof(ctypes.c_char.from_buffer(room))
        assert libc.mprotect(ctypes.c_void_p(base + half), half, 0) == 0
        rows = torch.randn(2, n, D, generator=gen).to(dtype)
        data = rows.flatten().view(torch.uint8).numpy().tobytes()
        ctypes.memmove(base + half - len(data), data, len(data))
        want[name], at[name] = rows, (room, base + half - len(data))
    q, k, v = (torch.zeros(B, new, n, D, dtype=dtype) for n in (H, Hk, Hk))
    for name, t in (("q", q), ("k", k), ("v", v)):
        t[1, :2] = want[name]
    results = []
    for there in (True, False):
        keys, values = pool(torch.Generator().manual_seed(63), "cpu", dtype, 8, 8, Hk, D)
        d = head_desc(q, k, v, f, norm=1, eps=1e-6, start=3, interleaved=int(interleaved), lengths=lengths.data_ptr())
        out = torch.full((B, new, H, D), 5.0, dtype=dtype)
        pointers = [t.data_ptr() for t in (q, k, v)]
        if not there:
            # sequence 1 lies at the end of what may be read, its unfilled rows, and sequences 0 and 2 (also before it: backwards), behind
            for name, n in (("q", H), ("k", Hk), ("v", Hk)):
                step = 4 * n * D
                getattr(d, name + "_stride")[0] = -step if backwards else 0
            pointers = [at[n][1] + (4 * w * D * size if backwards else 0) for n, w in (("q", H), ("k", Hk), ("v", Hk))]
        pd = page_desc(keys, values, pages)
        ops.lib.call("s2c_norm_rotate_store", ctypes.byref(d), ctypes.byref(pd), *pointers, None, None, out.data_ptr(), keys.data_ptr(), values.data_ptr(), None)
        results.append((out, keys, values))
    assert all(torch.equal(a, b) for a, b in zip(*results))
    assert not results[1][0][0].any() and not results[1][0][1, 2:].any() and results[1][0][1, :2].any()
print("done")
"""


@pytest.mark.parametrize("case", [(24, "float32", False), (128, "bfloat16", False), (20, "float32", True), (25, "bfloat16", True), (80, "float32", False)], ids=str)
def test_rows_that_are_not_there(case):
    import os
    import subprocess
    import sys
    import emul
    emul.build()
    here = os.path.dirname(os.path.abspath(__file__))
    done = subprocess.run([sys.executable, "-c", _ENDS] + [str(x) for x in case], cwd=here, env=dict(os.environ, PYTHONPATH=os.pathsep.join((here, os.path.dirname(here)))),
                          stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    assert done.returncode == 0 and "done" in done.stdout, done.stdout


@pytest.mark.parametrize("backend", backends.BACKENDS)
def test_first_positions_out_of_range(backend):
    """Numbers that are no 32-bit positions are refused, the least 64-bit one (whose magnitude is none) among them; 32-bit ones are not."""
    with backends.active(backend) as (_, dev):
        q, keys, pages = torch.ones(1, 1, 1, 8, device=dev), torch.ones(1, 8, 1, 8, device=dev), torch.zeros(1, 1, dtype=torch.int32, device=dev)
        for start in (1 << 31, -(1 << 31), (1 << 63) - 1, -(1 << 63)):
            for call in (lambda: S.norm_rotate(q, None, positions=start), lambda: S.norm_rotate_store(q, q, q, keys, keys, pages, positions=start),
                         lambda: S.paged_attention(q, keys, keys, pages, q_start=start), lambda: S.attention(q, q, q, q_start=start)):
                with pytest.raises((AssertionError, _lib.S2cError), match="range"):
                    call()
        for start in ((1 << 31) - 1, 1 - (1 << 31)):
            assert torch.equal(S.norm_rotate(q, None, positions=start)[0], q) and S.attention(q, q, q, q_start=start).shape == q.shape


# ---- attention ----------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("backend", backends.BACKENDS)
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_workspace_of_many_queries(backend, dtype):
    """Keys and values of as many sequences as 2^30 bytes hold, and packed copies of these and of the queries: of heads rounded up to 8 values,
    three bfloat16 parts in float32, one in bfloat16 where heads are no multiple of 8."""
    with backends.active(backend) as (ops, dev):
        q, keys = torch.zeros(1, 1, 1, 1, dtype=dtype, device=dev), torch.zeros(2, 64, 1, 1, dtype=dtype, device=dev)
        pages = torch.zeros(1, 1, dtype=torch.int32, device=dev)
        for Hk, D in ((4, 128), (1, 64), (3, 25)):
            for columns in (1, 40, 1000, 2500):
                sizes, batches = [], (1, 2, 3, 8, 9, 50, 1000, 100000)
                for batch in batches:
                    d = attention_desc(q, keys, batch=batch, lq=300, heads=2 * Hk, kv_heads=Hk, dim=D, q_stride=(ctypes.c_long * 3)(600 * Hk * D, 2 * Hk * D, D))
                    p = page_desc(keys, keys, pages, columns=columns)
                    sizes.append(ops.lib.s2c_paged_attention_workspace(ctypes.byref(d), ctypes.byref(p)))
                size, eight = dtype.itemsize, -(-D // 8) * 8
                copies = 6 if dtype == F32 else 2 if D % 8 else 0
                for batch, n in zip(batches, sizes):
                    assert 0 < n <= (1 << 30) + (1 << 30) // (D * size) * eight * copies + batch * 300 * 2 * Hk * eight * copies + 4096, (Hk, D, columns, batch, n)


@pytest.mark.parametrize("backend", backends.BACKENDS)
@pytest.mark.parametrize("dtype, Hk", [(F32, 1), (F32, 2), (BF16, 4)])
def test_many_queries_over_wide_tables(backend, dtype, Hk):
    """Columns that nobody has filled, 2^18 positions for each of five sequences: what a table of seven columns gives to the type's exactness.  Keys
    and values of one sequence take 2 x 2^18 x 128 x 4 = 2.7e8 bytes in float32 with one key head, four of them fit in 2^30, and 5.4e8 in
    bfloat16 with four: the calls on single sequences give the same bits.  In float32 with two key heads one fits, but its 8 heads have too
    few tiles of queries for the device: all rows go over the pages, with shares of the work that depend on the batch."""
    with backends.active(backend) as (_, dev):
        gen = torch.Generator().manual_seed(64)
        B, lq, H, D, page, columns = 5, 70, 80 if dev.type == "cuda" and Hk != 2 else 8, 128, 128, 2048       # (80 tiles of a group: half of 148 SMs)
        keys, values = pool(gen, dev, dtype, 7 * B + 1, page, Hk, D)
        narrow = shuffled(gen, dev, 7 * B, B, 7)
        pages = torch.full((B, columns), -1, dtype=torch.int32, device=dev)
        pages[:, :7] = narrow
        q = normal(gen, dev, dtype, B, lq, H, D)
        table, buckets = normal(gen, dev, dtype, 16, H), S.relative_buckets(16, 30, device=dev)
        kept = [800, 0, 1, 333, 100]
        kw = {"causal": True, "q_start": ints([730, 5, 0, 263, 60], dev), "q_lengths": ints([70, 70, 1, 70, 40], dev), "kv_lengths": ints(kept, dev)}
        out = S.paged_attention(q, keys, values, pages, table, buckets, **kw)
        k, v = gathered(keys, narrow), gathered(values, narrow)
        assert rel(out, exact_attention(q, k, v, table, buckets, **kw)[0]) <= TOL[dtype]
        assert rel(S.paged_attention(q, keys, values, narrow, table, buckets, **kw), out) <= 2 * TOL[dtype]
        for b in range(B):
            one = {n: t if n == "causal" else t[b:b + 1] for n, t in kw.items()}
            alone = S.paged_attention(q[b:b + 1], keys, values, pages[b:b + 1], table, buckets, **one)
            assert torch.equal(out[b:b + 1], alone) if Hk != 2 else rel(out[b:b + 1], alone) <= 2 * TOL[dtype]


def lengths_of(batch, most):
    """from none and one to all, in no order"""
    return [0, 1, most] + [(37 * i * i + 11 * i) % (most + 1) for i in range(batch - 3)]


MANY = [
    # B, lq, room, H, Hk, D, page, bias, kept; with 148 SMs at most 444 blocks share the items (sequence, key head, 8 or 16 rows)
    (64, 1, 700, 16, 8, 64, 16, None, lengths_of(64, 700)),                      # 512 items
    (64, 3, 500, 32, 8, 64, 32, (16, 30), lengths_of(64, 500)),                  # 512, of 12 rows
    (200, 1, 6000, 8, 4, 32, 64, None, [6000] + [(7 * i) % 50 for i in range(199)]),     # 800, one long sequence among short ones
    (150, 24, 200, 2, 2, 128, 16, None, lengths_of(150, 200)),                   # 600: 24 rows are two times 16
    (70, 2, 900, 16, 8, 128, 64, (8, 20), lengths_of(70, 900)),                  # 560
    (500, 1, 40, 3, 1, 25, 8, None, lengths_of(500, 40)),                        # 500, of one step each; four sequences to a thread that adds up
    (3, 200, 1500, 8, 8, 40, 16, None, [1500, 700, 0]),                          # 312 of 16 rows in float32; in bfloat16 200 rows take the kernels of whole tiles
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("case", MANY, ids=lambda c: "x".join(map(str, c[:7])))
def test_more_items_than_blocks(case, causal, dtype):
    """Each item's share is found, joined and written, with a workspace full of NaN; the same in every call."""
    B, lq, room, H, Hk, D, page, bias, kept = case
    kw = {"kv_lengths": kept}
    if causal:
        kw |= {"causal": True, "q_start": [n - lq for n in kept]}
    else:
        kw |= {"q_lengths": [(i * 5) % (lq + 1) for i in range(B)]}
    results = []
    for _ in range(2):
        stale = torch.full((1 << 26,), math.nan, device="cuda")
        del stale
        results.append(check_attention("cuda", dtype, B, lq, room, H, Hk, D, page, bias, seed=65, **kw))
    assert torch.equal(*results)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_ragged_new_positions(dtype):
    """A step in which one of sixteen sequences brings 30 positions, one none and the others one: a row of the call on each sequence alone."""
    gen = torch.Generator().manual_seed(66)
    B, new, H, Hk, D, page = 16, 30, 16, 4, 64, 32
    counts = [30, 0] + [1] * 14
    filled = [100 + 61 * i for i in range(B)]
    keys, values = pool(gen, "cuda", dtype, B * 36 + 2, page, Hk, D)
    pages = shuffled(gen, "cuda", B * 36 + 2, B, 36)
    q, k, v = normal(gen, "cuda", dtype, B, new, H + 2 * Hk, D).split((H, Hk, Hk), 2)
    f, lengths, at = S.rotary_frequencies(32, device="cuda"), ints(counts, "cuda"), ints(filled, "cuda")
    turned = S.norm_rotate_store(q, k, v, keys, values, pages, f, positions=at, lengths=lengths)
    kw = {"causal": True, "q_start": at, "q_lengths": lengths, "kv_lengths": at + lengths}
    out = S.paged_attention(turned, keys, values, pages, **kw)
    assert rel(out, exact_attention(turned, gathered(keys, pages), gathered(values, pages), **kw)[0]) <= TOL[dtype]
    for b, n in enumerate(counts):
        assert not out[b, n:].any()
        if n:
            alone = S.paged_attention(turned[b:b + 1, :n], keys, values, pages[b:b + 1], causal=True, q_start=filled[b], kv_lengths=ints([filled[b] + n], "cuda"))
            assert rel(out[b:b + 1, :n], alone) <= 2 * TOL[dtype]


# ---- the account of a pool ----------------------------------------------------------------------------------------------


def account(cache, table, filled):
    """the table and the lengths on the device are the host's"""
    want = torch.full(table.shape, -1, dtype=torch.int32)
    for row, pages in zip(want, cache._pages):
        row[:len(pages)] = torch.tensor(pages, dtype=torch.int32)
    assert torch.equal(table.cpu(), want) and filled.tolist() == cache.lengths


@pytest.mark.parametrize("backend", backends.BACKENDS)
def test_the_table_follows_the_account(backend):
    with backends.active(backend) as (_, dev):
        rng = random.Random(70)
        for columns in (6, 300):
            cache = S.PagedCache(40, 8, 1, 4, 7, columns=columns, device=dev)
            for _ in range(120):
                what, s, t = rng.choice(["extend", "extend", "extend", "fork", "truncate", "free", "compact"]), rng.randrange(7), rng.randrange(7)
                if what == "extend":
                    try:
                        cache.extend([rng.choice([0, 0, 1, 3, 17]) for _ in range(7)])
                        if rng.random() < 0.3:
                            cache.extend([rng.choice([0, 1, 5]) for _ in range(7)])
                    except MemoryError:
                        pass
                    cache.advance()
                elif what == "fork" and s != t:
                    cache.free(t)
                    cache.fork(s, t)
                elif what == "truncate":
                    cache.truncate(s, rng.randint(0, cache.lengths[s]))
                elif what == "free":
                    cache.free(s - 7)                        # (counted from the end)
                elif what == "compact":
                    held = cache.compact()
                    assert all(p < held for pages in cache._pages for p in pages)
                account(cache, cache.table, cache.filled)


@pytest.mark.gpu
def test_the_account_does_not_wait_for_the_device():
    """Steps, forks and the rest come back while work that was queued before them still runs, whatever the table's width."""
    a = torch.randn(8192, 8192, device="cuda", dtype=BF16)
    for turn in range(2):                                        # (the first one has memory pinned)
        cache = S.PagedCache(30000, 8, 1, 8, 64, columns=16384, dtype=BF16)
        cache.extend([8 * n for n in range(64)])
        cache.advance()
        torch.cuda.synchronize()
        for _ in range(300):
            b = a @ a
        done = torch.cuda.Event()
        done.record()
        for step in range(5):
            cache.extend(9)
            cache.advance()
            cache.free(step)
            cache.fork(60, step)
            cache.truncate(50 + step, 20)
            cache.compact()
        waited = done.query()
        account(cache, cache.table, cache.filled)
        assert not (turn and waited)
        del b


# ---- blocks -------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("backend", backends.BACKENDS)
@pytest.mark.parametrize("rotary", [None, 8])
def test_lengths_beyond_the_new_positions(backend, rotary):
    """Count as all of them, and below 0 as none: what a page holds behind the new positions is not looked at."""
    with backends.active(backend) as (_, dev):
        torch.manual_seed(72)
        block = S.SequenceBlock(32, 4, 2, causal=False, p=0.0, rotary=rotary).to(dev).eval()
        x, results = torch.randn(3, 4, 32, device=dev), []
        pages, filled = ints([[0, 1], [2, 3], [4, 5]], dev), ints([5, 3, 1], dev)
        for lengths in ([4, 2, 0], [9, 2, -3]):
            keys, values = (torch.randn(6, 8, 2, 8, generator=torch.Generator().manual_seed(73 + n)).to(dev) for n in (0, 1))
            results.append((block.step_pages(x, keys, values, pages, filled, lengths=ints(lengths, dev)), keys, values))
        for a, b in zip(*results):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_the_account_is_not_captured():
    """A replay would copy from memory that has long been used for something else: refused before anything changes."""
    cache = S.PagedCache(20, 8, 1, 8, 3)
    cache.extend(5)
    cache.advance()
    x = torch.ones(1, device="cuda")
    for call in (lambda: cache.extend(9), cache.advance, lambda: cache.fork(0, 2), lambda: cache.truncate(0, 2), lambda: cache.free(1), cache.compact):
        before = list(cache.lengths), [list(p) for p in cache._pages], list(cache._free)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            x.add_(1)
            with pytest.raises(AssertionError, match="captured"):
                call()
        assert before == (cache.lengths, cache._pages, cache._free)
        account(cache, cache.table, cache.filled)
        del graph
    cache.extend(9)
    cache.advance()
    account(cache, cache.table, cache.filled)
