"""The operators on pages and on turned heads as they are called in earnest: by the C entry points, on streams, captured and replayed,
two at once, fused and recorded, in bfloat16 blocks."""
import ctypes
import math

import pytest
import torch

import backends
import s2cnn_b200 as S
from s2cnn_b200 import _lib
from test_pages import gathered, ints, pool, shuffled
from test_sequence_c_abi import Desc as AttentionDesc
from test_sequence_c_abi import off_by, stream_of
from test_sequence_ops import TOL, exact_attention, normal, rel

F32, BF16 = torch.float32, torch.bfloat16


class HeadDesc(ctypes.Structure):
    """s2c_head_desc"""
    _fields_ = ([(n, ctypes.c_int) for n in ("dtype", "batch", "length", "heads", "kv_heads", "dim")] +
                [(n, ctypes.c_long * 3) for n in ("q_stride", "k_stride", "v_stride")] +
                [("frequencies", ctypes.c_void_p), ("pairs", ctypes.c_int), ("interleaved", ctypes.c_int), ("magnitude", ctypes.c_float),
                 ("norm", ctypes.c_int), ("eps", ctypes.c_float), ("start", ctypes.c_int), ("each", ctypes.c_int), ("positions", ctypes.c_void_p),
                 ("lengths", ctypes.c_void_p)])


class PageDesc(ctypes.Structure):
    """s2c_page_desc"""
    _fields_ = ([("table", ctypes.c_void_p)] + [(n, ctypes.c_int) for n in ("columns", "count", "page")] +
                [(n, ctypes.c_long * 3) for n in ("key_stride", "value_stride")])


def three(t):
    return (ctypes.c_long * 3)(*t.stride()[:3])


def page_desc(keys, values, pages, **kw):
    d = PageDesc(table=pages.data_ptr(), columns=pages.size(1), count=keys.size(0), page=keys.size(1), key_stride=three(keys), value_stride=three(values))
    for name, value in kw.items():
        setattr(d, name, value)
    return d


def attention_desc(q, keys, **kw):
    d = AttentionDesc(dtype=int(q.dtype == BF16), batch=q.size(0), lq=q.size(1), heads=q.size(2), kv_heads=keys.size(2), dim=q.size(3),
                      scale=q.size(3) ** -0.5, q_stride=three(q))
    for name, value in kw.items():
        setattr(d, name, value.data_ptr() if isinstance(value, torch.Tensor) else value)
    return d


def head_desc(q, k, v, f, **kw):
    d = HeadDesc(dtype=int(q.dtype == BF16), batch=q.size(0), length=q.size(1), heads=q.size(2), kv_heads=k.size(2), dim=q.size(3), q_stride=three(q),
                 k_stride=three(k), v_stride=three(v), frequencies=f.data_ptr(), pairs=f.numel(), magnitude=1.0)
    for name, value in kw.items():
        setattr(d, name, value)
    return d


@pytest.mark.parametrize("backend", backends.BACKENDS)
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_c_entry_points(backend, dtype):
    """Arrays off every boundary but their type's give what aligned ones give; guards before and behind what is written stay."""
    with backends.active(backend) as (ops, dev):
        gen = torch.Generator().manual_seed(50)
        lib, stream = ops.lib, stream_of(dev)
        B, new, H, Hk, D, page, columns = 2, 3, 4, 2, 24, 8, 4
        f = S.rotary_frequencies(16, device=dev)
        pages = shuffled(gen, dev, 10, B, columns)
        for off in (0, 1):
            gen.manual_seed(51)
            q, k, v = (off_by(normal(gen, dev, dtype, B, new, n, D), off) for n in (H, Hk, Hk))
            keys, values = (off_by(normal(gen, dev, dtype, 10, page, Hk, D), off) for _ in range(2))
            w, gq, gk = (off_by(normal(gen, dev, dtype, *s), off) for s in ((D,), (B, new, H, D), (B, new, Hk, D)))
            guard = lambda *shape: torch.full((math.prod(shape) + 32,), 77.0, dtype=dtype, device=dev)  # noqa: E731
            inside = lambda room, *shape: room[16 + off:16 + off + math.prod(shape)].view(shape)  # noqa: E731
            rooms = {n: guard(*s) for n, s in (("q", (B, new, H, D)), ("k", (B, new, Hk, D)), ("dq", (B, new, H, D)), ("dk", (B, new, Hk, D)), ("dw", (D,)),
                                               ("dv", (D,)), ("out", (B, new, H, D)))}
            at = {n: inside(r, *s.shape) for (n, r), s in zip(rooms.items(), (q, k, q, k, w, w, q))}
            d = head_desc(q, k, v, f, norm=1, eps=1e-6, start=20)
            p = ctypes.byref(d)
            lib.call("s2c_norm_rotate", p, q.data_ptr(), k.data_ptr(), w.data_ptr(), None, at["q"].data_ptr(), at["k"].data_ptr(), stream)
            need = lib.s2c_norm_rotate_backward_workspace(p)
            ws = torch.full((need + 64,), 0x5A, dtype=torch.uint8, device=dev)
            lib.call("s2c_norm_rotate_backward", p, q.data_ptr(), k.data_ptr(), w.data_ptr(), w.data_ptr(), gq.data_ptr(), gk.data_ptr(), at["dq"].data_ptr(),
                     at["dk"].data_ptr(), at["dw"].data_ptr(), at["dv"].data_ptr(), ws.data_ptr(), need, stream)
            assert bool((ws[need:] == 0x5A).all())
            pd = page_desc(keys, values, pages)
            pp = ctypes.byref(pd)
            lib.call("s2c_norm_rotate_store", p, pp, q.data_ptr(), k.data_ptr(), v.data_ptr(), w.data_ptr(), None, at["q"].data_ptr(), keys.data_ptr(), values.data_ptr(), stream)
            a = attention_desc(at["q"], keys, causal=1, q_start=20)
            pa = ctypes.byref(a)
            need = lib.s2c_paged_attention_workspace(pa, pp)
            ws = torch.full((need + 64,), 0x5A, dtype=torch.uint8, device=dev)
            lib.call("s2c_paged_attention", pa, pp, at["q"].data_ptr(), keys.data_ptr(), values.data_ptr(), None, at["out"].data_ptr(), ws.data_ptr(), need, stream)
            assert bool((ws[need:] == 0x5A).all())
            for room, t in zip(rooms.values(), at.values()):
                n = t.numel()
                assert bool((room[:16 + off] == 77).all()) and bool((room[16 + off + n:] == 77).all())
            result = {n: t.clone() for n, t in at.items()} | {"keys": keys.clone(), "values": values.clone()}
            if off == 0:
                want = result
                leaves = [t.clone().requires_grad_(True) for t in (q, k, w, w)]
                turned = S.norm_rotate(leaves[0], leaves[1], f, leaves[2], None, eps=1e-6, positions=20)
                assert torch.equal(turned[0], at["q"]) and torch.equal(turned[1], at["k"])
                grads = torch.autograd.grad(S.norm_rotate(leaves[0], leaves[1], f, leaves[2], leaves[3], eps=1e-6, positions=20), leaves, (gq, gk))
                assert all(torch.equal(x, at[n]) for x, n in zip(grads, ("dq", "dk", "dw", "dv")))
                ref = exact_attention(at["q"], gathered(keys, pages), gathered(values, pages), causal=True, q_start=20)[0]
                assert rel(at["out"], ref) <= TOL[dtype]
        for n in want:
            assert torch.equal(want[n], result[n]), n


@pytest.mark.parametrize("backend", backends.BACKENDS)
def test_c_refusals(backend):
    """Status codes with a message; nothing is launched."""
    with backends.active(backend) as (ops, dev):
        lib, stream = ops.lib, stream_of(dev)
        q, keys = torch.zeros(1, 2, 4, 16, device=dev), torch.zeros(4, 8, 2, 16, device=dev)
        k, pages, f = torch.zeros(1, 2, 2, 16, device=dev), ints([[0, 1]], dev), S.rotary_frequencies(16, device=dev)
        out, ws = torch.full_like(q, 5.0), torch.zeros(1 << 20, dtype=torch.uint8, device=dev)
        ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
        attend = lambda a, p, q=q, ws=ws, n=1 << 20, out=out: lib.s2c_paged_attention(  # noqa: E731
            ctypes.byref(a) if a else None, ctypes.byref(p) if p else None, ptr(q), ptr(keys), ptr(keys), None, ptr(out), ptr(ws), n, stream)
        good_a, good_p = lambda **kw: attention_desc(q, keys, **kw), lambda **kw: page_desc(keys, keys, pages, **kw)  # noqa: E731
        BAD, SMALL, UNSUPPORTED = 1, 3, 4
        assert attend(None, good_p()) == BAD and attend(good_a(), None) == BAD
        assert attend(good_a(dtype=2), good_p()) == BAD and attend(good_a(kv_heads=3), good_p()) == BAD
        assert attend(good_a(dim=129), good_p()) == UNSUPPORTED and attend(good_a(scale=math.nan), good_p()) == BAD
        assert attend(good_a(), good_p(table=None)) == BAD and attend(good_a(), good_p(page=12)) == UNSUPPORTED and attend(good_a(), good_p(page=4)) == UNSUPPORTED
        assert attend(good_a(), good_p(columns=-1)) == BAD and attend(good_a(), good_p(columns=1 << 26)) == UNSUPPORTED
        assert attend(good_a(), good_p(count=1 << 29)) == UNSUPPORTED
        assert attend(good_a(), good_p(), q=None) == BAD and attend(good_a(), good_p(), out=None) == BAD
        need = lib.s2c_paged_attention_workspace(ctypes.byref(good_a()), ctypes.byref(good_p()))
        assert attend(good_a(), good_p(), n=need - 1) == SMALL and attend(good_a(), good_p(), ws=None) == SMALL and attend(good_a(), good_p(), ws=ws[1:]) == BAD
        assert "boundary" in lib.last_error()
        assert lib.s2c_paged_attention_workspace(ctypes.byref(good_a(dim=0)), ctypes.byref(good_p())) == 0
        turn = lambda d, q=q, qo=out: lib.s2c_norm_rotate(ctypes.byref(d) if d else None, ptr(q), None, None, None, ptr(qo), None, stream)  # noqa: E731
        good_h = lambda **kw: head_desc(q, k, k, f, **kw)  # noqa: E731
        assert turn(None) == BAD and turn(good_h(dtype=3)) == BAD and turn(good_h(dim=129)) == UNSUPPORTED and turn(good_h(pairs=9)) == BAD
        assert turn(good_h(frequencies=None)) == BAD and turn(good_h(magnitude=math.inf)) == BAD and turn(good_h(norm=1, eps=-1.0)) == BAD
        assert turn(good_h(norm=1, eps=math.nan)) == BAD and turn(good_h(batch=-1)) == BAD and turn(good_h(), qo=None) == BAD
        back = lambda d, dw=None, w=None, n=0: lib.s2c_norm_rotate_backward(  # noqa: E731
            ctypes.byref(d), ptr(q), ptr(k), ptr(w), None, ptr(q), ptr(k), ptr(out), None, ptr(dw), None, ptr(ws), n, stream)
        w = torch.ones(16, device=dev)
        assert back(good_h(), dw=w) == BAD and back(good_h(norm=1), dw=w) == BAD and back(good_h(norm=1), dw=w, w=w) == SMALL
        store = lambda d, p, k=k, q=None: lib.s2c_norm_rotate_store(  # noqa: E731
            ctypes.byref(d), ctypes.byref(p), ptr(q), ptr(k), ptr(k), None, None, None, ptr(keys), ptr(keys), stream)
        assert store(good_h(), good_p(), k=None) == BAD and store(good_h(), good_p(page=3)) == UNSUPPORTED and store(good_h(), good_p(), q=q) == BAD
        copy = lambda stride, n, count, t=keys: lib.s2c_copy_pages(ptr(t), stride, n, count, ptr(pages), ptr(pages), 2, stream)  # noqa: E731
        assert copy(10, 16, 4) == BAD and copy(16, 16, -1) == BAD and copy(16, -16, 4) == BAD and copy(16, 16, 4, None) == BAD
        assert bool((out == 5).all()) and not keys.any()


@pytest.mark.gpu
def test_captured_step_follows_a_growing_cache():
    """One captured step of a layer, replayed while the cache grows from page to page and forks: what the uncaptured layer gives."""
    torch.manual_seed(52)
    block = S.SequenceBlock(64, 4, 2, causal=True, p=0.0, rotary=16, head_norm=True).cuda().eval()
    x = torch.randn(2, 40, 64, device="cuda")
    whole = block(x).detach()
    cache = S.PagedCache(24, 8, 2, 16, 3)
    xs = torch.zeros(3, 1, 64, device="cuda")
    run = lambda: block.step_pages(xs, cache.keys(), cache.values(), cache.table, cache.filled)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    cache.storage.zero_()
    got = []
    for i in range(40):
        cache.extend([1, 1, 1 if i >= 20 else 0])
        xs[:2, 0] = x[:, i]
        xs[2, 0] = x[0, i]
        graph.replay()
        got.append(out.clone())
        cache.advance()
        if i == 19:
            cache.fork(0, 2)                                     # continues as sequence 0 does
    got = torch.cat(got, 1)
    assert rel(got[:2], whole) <= 2e-5
    assert torch.equal(got[2, 20:], got[0, 20:])
    del graph


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_two_calls_at_once(dtype):
    """On two streams, in graphs that share a memory pool replayed one after the other, and on a stream that is not the current one's default."""
    gen = torch.Generator().manual_seed(53)
    keys, values = pool(gen, "cuda", dtype, 300, 16, 4, 128)
    pages = shuffled(gen, "cuda", 300, 2, 140)
    qs = [normal(gen, "cuda", dtype, 2, 1, n, 128) for n in (16, 64)]
    kw = {"kv_lengths": ints([2240, 777], "cuda")}
    want = [S.paged_attention(q, keys, values, pages, **kw) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    outs = [[], []]
    for _ in range(20):
        for n, (s, q) in enumerate(zip(streams, qs)):
            with torch.cuda.stream(s):
                outs[n].append(S.paged_attention(q, keys, values, pages, **kw))
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for os, w in zip(outs, want) for o in os)
    shared = torch.cuda.graph_pool_handle()
    graphs, results = [], []
    for q in qs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=shared):
            results.append(S.paged_attention(q, keys, values, pages, **kw))
        graphs.append(g)
    for n in (0, 1, 1, 0):
        graphs[n].replay()
        torch.cuda.synchronize()
        assert torch.equal(results[n], want[n])
    del graphs


@pytest.mark.gpu
def test_captured_training_step():
    """Forward and backward of turned heads captured and replayed on new inputs."""
    gen = torch.Generator().manual_seed(54)
    f, w = S.rotary_frequencies(32, device="cuda"), normal(gen, "cuda", F32, 32).requires_grad_(True)
    x, g = normal(gen, "cuda", F32, 2, 50, 6, 32).requires_grad_(True), normal(gen, "cuda", F32, 2, 50, 4, 32)
    step = lambda: torch.autograd.grad(S.norm_rotate(x[:, :, :4], x[:, :, 4:], f, w, w, eps=1e-6)[0], (x, w), g)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in (1, 2):
        with torch.no_grad():
            x.copy_(normal(torch.Generator().manual_seed(seed), "cuda", F32, 2, 50, 6, 32))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, step()))
    del graph


@pytest.mark.parametrize("backend", backends.BACKENDS)
def test_recorded_calls_are_refused(backend):
    with backends.active(backend) as (_, dev):
        gen = torch.Generator().manual_seed(55)
        keys, values = pool(gen, dev, F32, 4, 8, 1, 16)
        pages, q, f = ints([[0, 1]], dev), normal(gen, dev, F32, 1, 1, 2, 16), S.rotary_frequencies(16, device=dev)
        leaf = q.clone().requires_grad_(True)
        for call in (lambda: S.paged_attention(leaf, keys, values, pages), lambda: S.paged_attention(q, keys.clone().requires_grad_(True), values, pages),
                     lambda: S.norm_rotate_store(leaf, q[:, :, :1], q[:, :, :1], keys, values, pages), lambda: S.copy_pages(leaf, pages[0, :0], pages[0, :0]),
                     lambda: S.norm_rotate(q, None, f.clone().requires_grad_(True))):
            with pytest.raises(RuntimeError, match="gradient"):
                call()
        with torch.no_grad():
            assert torch.equal(S.paged_attention(leaf, keys, values, pages), S.paged_attention(q, keys, values, pages))
        with pytest.raises(RuntimeError):
            torch.jit.trace(lambda x: S.paged_attention(x, keys, values, pages), q, check_trace=False)
        saved = keys.clone().requires_grad_(True)                # an array that a backward pass will read is out of date once it is written
        kept = saved * 1
        loss = (kept * kept).sum()
        with torch.no_grad():
            S.norm_rotate_store(None, q[:, :, :1], q[:, :, :1], kept.detach(), values, pages)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()


@pytest.mark.parametrize("backend", backends.BACKENDS)
def test_fused_network_with_turned_heads(backend):
    """The rotary network's answers and gradients, fused and plain (2e-5: as test_sequence_fuse.py)."""
    with backends.active(backend) as (_, dev):
        torch.manual_seed(56)
        m = S.models.SphereSequenceNet(f1=2, f2=8, f_output=3, b_in=4, b_l1=3, b_l2=2, heads=2, p=0.0, rotary=4, head_norm=True).to(dev)
        x = torch.randn(2, 5, 1, 8, 8, device=dev)
        results = []
        for net in (m, S.fuse(m)):
            m.zero_grad()
            y = net(x)
            y.square().sum().backward()
            results.append([y.detach()] + [p.grad.clone() for p in m.parameters()])
        for a, b in zip(*results):
            assert (a - b).norm() <= 2e-5 * a.norm().clamp_min(1e-6)

        class Own(torch.nn.Module):
            def __init__(self):
                super().__init__()
                self.register_buffer("f", S.rotary_frequencies(4))

            def forward(self, q):
                a, b = S.norm_rotate(q, q, self.f)
                return a + b

        own, q = Own().to(dev), torch.randn(1, 3, 2, 4, device=dev)
        assert torch.equal(S.fuse(own)(q), own(q))


@pytest.mark.parametrize("backend", backends.BACKENDS)
def test_bfloat16_block_in_pages(backend):
    """A bfloat16 layer step by step and whole (3e-2: some ten roundings of 2^-8 on the way, as in test_sequence_bfloat16_network.py), and
    under autocast with a float32 stream."""
    with backends.active(backend) as (_, dev):
        torch.manual_seed(57)
        block = S.SequenceBlock(32, 4, 2, causal=True, p=0.0, rotary=8, head_norm=True).to(dev).eval()
        x = torch.randn(1, 12, 32, device=dev)
        want = block(x).detach()

        def steps(block, x):
            cache = S.PagedCache(4, 8, 2, 8, 1, dtype=BF16, device=dev)
            out = []
            for i in range(12):
                cache.extend(1)
                out.append(block.step_pages(x[:, i:i + 1], cache.keys(), cache.values(), cache.table, cache.filled))
                cache.advance()
            return torch.cat(out, 1)

        with torch.autocast(dev.type, torch.bfloat16):
            assert rel(steps(block, x), want) <= 3e-2
        block = block.to(BF16)
        out = steps(block, x.to(BF16))
        assert out.dtype == BF16 and rel(out, want) <= 3e-2 and rel(out, block(x.to(BF16))) <= 3e-2


@pytest.mark.parametrize("backend", backends.BACKENDS)
def test_error_type(backend):
    with backends.active(backend) as (_, dev):
        if dev.type == "cuda":
            with pytest.raises(_lib.S2cError):
                S.norm_rotate(torch.zeros(1, 1, 1, 8))
            with pytest.raises(_lib.S2cError):
                S.copy_pages(torch.zeros(4, 8), torch.zeros(1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))
