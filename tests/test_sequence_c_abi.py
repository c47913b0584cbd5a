"""The C entry points of attention as a C caller uses them: arrays aligned to their type alone, what of a workspace is written, what
is refused."""
import ctypes
import math

import pytest
import torch

import backends
import s2cnn_b200 as S
from s2cnn_b200 import _lib

F32, BF16 = torch.float32, torch.bfloat16


class Desc(ctypes.Structure):
    """s2c_attention_desc"""
    _fields_ = ([(n, ctypes.c_int) for n in ("dtype", "batch", "lq", "lk", "heads", "kv_heads", "dim")] +
                [(n, ctypes.c_long * 3) for n in ("q_stride", "k_stride", "v_stride")] +
                [("causal", ctypes.c_int), ("scale", ctypes.c_float), ("q_start", ctypes.c_int)] +
                [(n, ctypes.c_void_p) for n in ("q_starts", "q_lengths", "kv_lengths", "bucket_of")] +
                [(n, ctypes.c_int) for n in ("n_buckets", "reach", "bias_grad")])


def describe(q, k, v, **kw):
    d = Desc(dtype=int(q.dtype == BF16), batch=q.size(0), lq=q.size(1), lk=k.size(1), heads=q.size(2), kv_heads=k.size(2), dim=q.size(3),
             scale=1 / math.sqrt(q.size(3)))
    for name, t in (("q_stride", q), ("k_stride", k), ("v_stride", v)):
        setattr(d, name, (ctypes.c_long * 3)(*t.stride()[:3]))
    for name, value in kw.items():
        setattr(d, name, value.data_ptr() if isinstance(value, torch.Tensor) else value)
    return d


def stream_of(dev):
    return torch.cuda.current_stream().cuda_stream if dev.type == "cuda" else None


def off_by(t, n):
    """The same values, contiguous, n elements past a 16-byte boundary."""
    room = torch.empty(t.numel() + n + 8, dtype=t.dtype, device=t.device)
    assert room.data_ptr() % 16 == 0
    return room[n:n + t.numel()].view(t.shape).copy_(t)


def call(ops, dev, q, k, v, dout, off=0, fill=None, **kw):
    """(out, dq, dk, dv) by the C entry points, results and dout `off` elements past a 16-byte boundary."""
    d = describe(q, k, v, **kw)
    p = ctypes.byref(d)
    new = lambda n: torch.full((max(1, n),), 0x5A, dtype=torch.uint8, device=dev)  # noqa: E731
    out, dq, dk, dv = (off_by(torch.zeros(t.shape, dtype=t.dtype, device=dev), off) for t in (q, q, k, v))
    dout = off_by(dout, off)
    saved, ws = new(ops.lib.s2c_attention_saved_bytes(p)), new(ops.lib.s2c_attention_workspace(p))
    ops.lib.call("s2c_attention", p, q.data_ptr(), k.data_ptr(), v.data_ptr(), None, out.data_ptr(), saved.data_ptr(), ws.data_ptr(),
                 ops.lib.s2c_attention_workspace(p), stream_of(dev))
    back = new(ops.lib.s2c_attention_backward_workspace(p))
    ops.lib.call("s2c_attention_backward", p, q.data_ptr(), k.data_ptr(), v.data_ptr(), None, out.data_ptr(), saved.data_ptr(), dout.data_ptr(),
                 dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), None, back.data_ptr(), ops.lib.s2c_attention_backward_workspace(p), stream_of(dev))
    return (out, dq, dk, dv), ws, back


def operands(dev, dtype, B, Lq, Lk, H, D, gap):
    """Rows `gap` elements apart from one another."""
    gen = torch.Generator().manual_seed(40)
    q, k, v = (torch.randn(B, n, H * D + gap, generator=gen).to(dtype).to(dev)[..., :H * D].unflatten(2, (H, D)) for n in (Lq, Lk, Lk))
    return q, k, v, torch.randn(B, Lq, H, D, generator=gen).to(dtype).to(dev)


@pytest.mark.parametrize("backend", backends.BACKENDS)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("gap", [0, 4])
def test_arrays_aligned_to_their_type(backend, dtype, gap):
    """Results and their gradients off a 16-byte boundary, with rows that are fetched in pieces and rows that are packed.  Packed rows
    take the same kernels either way; others may go to the FP32 pipes (8e-3 and 5e-6: see test_sequence_ops.py)."""
    with backends.active(backend) as (ops, dev):
        for D in (64, 128):
            q, k, v, g = operands(dev, dtype, 1, 130, 140, 2, D, gap)
            want, _, _ = call(ops, dev, q, k, v, g)
            got, _, _ = call(ops, dev, q, k, v, g, off=1)
            for a, b in zip(want, got):
                if gap or dtype == F32:
                    assert torch.equal(a, b)
                else:
                    assert (a.double() - b.double()).norm() <= 8e-3 * a.double().norm()


@pytest.mark.parametrize("backend", backends.BACKENDS)
def test_saved_and_workspace_are_aligned(backend):
    with backends.active(backend) as (ops, dev):
        q, k, v, g = operands(dev, F32, 1, 130, 140, 2, 64, 0)
        d = describe(q, k, v)
        p = ctypes.byref(d)
        room = torch.zeros(1 << 22, dtype=torch.uint8, device=dev)
        out = torch.zeros_like(q)
        for saved, ws in ((room.data_ptr() + 4, room.data_ptr()), (room.data_ptr(), room.data_ptr() + 8)):
            with pytest.raises(_lib.S2cError, match="status 1"):
                ops.lib.call("s2c_attention", p, q.data_ptr(), k.data_ptr(), v.data_ptr(), None, out.data_ptr(), saved, ws, 1 << 20, stream_of(dev))
            with pytest.raises(_lib.S2cError, match="status 1"):
                ops.lib.call("s2c_attention_backward", p, q.data_ptr(), k.data_ptr(), v.data_ptr(), None, out.data_ptr(), saved, g.data_ptr(), out.data_ptr(),
                             k.data_ptr(), v.data_ptr(), None, ws, 1 << 21, stream_of(dev))


@pytest.mark.parametrize("backend", backends.BACKENDS)
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_gradient_off_a_boundary_takes_the_same_kernels(backend, dtype):
    """What comes back for dout is the same to the last bit wherever dout lies."""
    with backends.active(backend) as (_, dev):
        q, k, v, g = operands(dev, dtype, 1, 130, 140, 2, 64, 0)
        args = [t.requires_grad_(True) for t in (q, k, v)]
        off = off_by(g, 1)
        assert off.is_contiguous() and off.data_ptr() % 16
        a, b = (torch.autograd.grad(S.attention(*args), args, t) for t in (g, off))
        assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("causal", [0, 1])
def test_rows_that_nobody_sees_are_not_packed(dtype, causal):
    """A workspace keeps what it held where the packed copies of rows beyond the lengths, and of keys behind all queries, would
    be: [tensor][part][batch][head][position][values], each tensor from a 256-byte boundary on."""
    ops, dev = backends.get("cuda")
    B, Lq, Lk, H, D = 3, 130, 300, 2, 20
    q, k, v, g = operands(dev, dtype, B, Lq, Lk, H, D, 0)
    q_lengths, kv_lengths = [130, 0, 70], [200, 300, 40]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    starts = i32([-60, 0, 10])
    keep = i32(q_lengths), i32(kv_lengths)
    _, ws, back = call(ops, dev, q, k, v, g, q_lengths=keep[0], kv_lengths=keep[1], q_starts=starts, causal=causal)
    keys = [min(n, max(0, s + m)) if causal else n for n, m, s in zip(kv_lengths, q_lengths, [-60, 0, 10])]

    def untouched(rows, lengths):
        t = torch.zeros((3 if dtype == F32 else 1, B, H, rows, 24 * 2), dtype=torch.bool)
        for b, n in enumerate(lengths):
            t[:, b, :, n:] = True
        t = t.flatten()
        return torch.cat((t, torch.zeros(-len(t) % 256, dtype=torch.bool)))

    parts = [untouched(Lq, q_lengths), untouched(Lk, keys), untouched(Lk, keys), untouched(Lq, q_lengths)]
    for space, of in ((ws, parts[:3]), (back, parts)):
        mask = torch.cat(of)
        assert len(mask) <= len(space)
        mask = torch.cat((torch.zeros(len(space) - len(mask), dtype=torch.bool), mask))
        assert mask.any() and bool((space.cpu()[mask] == 0x5A).all())
        assert bool((space.cpu()[~mask] != 0x5A).any())


@pytest.mark.parametrize("backend", backends.BACKENDS)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lq", [3, 200])
def test_output_is_the_same_recorded_or_not(backend, dtype, lq):
    """To the last bit, where the bias itself wants no gradient."""
    with backends.active(backend) as (_, dev):
        q, k, v, _ = operands(dev, dtype, 2, lq, 200, 2, 64, 0)
        table, buckets = torch.randn(16, 2, generator=torch.Generator().manual_seed(41)).to(dtype).to(dev), S.relative_buckets(16, 30, device=dev)
        plain = S.attention(q, k, v, table, buckets)
        leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
        recorded = S.attention(*leaves, table, buckets)
        assert recorded.requires_grad and torch.equal(plain, recorded)
