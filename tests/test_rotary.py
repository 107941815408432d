"""Rotary positions against the definition in 64 bits.  An element is rounded once, by half a step of its type at most; sine and cosine are good to 2^-22 and the
products and sums are fp32, 2^-22 of the terms with them."""
import ctypes
import math

import pytest
import torch

from lego_amd import ops, runtime

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def oracle(x, positions, frequencies, interleaved, magnitude, inverse=False):
    """The turned tensor in 64 bits and a bound of the error."""
    u = U[x.dtype]
    x = x.detach().cpu().double()
    if positions.dim() == 1:
        positions = positions.expand(x.shape[0], -1)
    t = positions.cpu().double()[:, :, None, None] * frequencies.cpu() * (-1 if inverse else 1)
    part = 2 * frequencies.shape[0]
    pair = (slice(0, part, 2), slice(1, part, 2)) if interleaved else (slice(0, part // 2), slice(part // 2, part))
    a, b = x[..., pair[0]], x[..., pair[1]]
    y, off = x.clone(), torch.zeros_like(x)
    y[..., pair[0]] = magnitude * (a * t.cos() - b * t.sin())
    y[..., pair[1]] = magnitude * (b * t.cos() + a * t.sin())
    terms = abs(magnitude) * (a.abs() + b.abs())
    for s in pair:
        off[..., s] = u * y[..., s].abs() + (2.0 ** -21 + 1e-15 * float(positions.abs().max())) * terms + (2.0 ** -25 if x.dtype != torch.float32 and u == 2.0 ** -11 else 0.0)
    return y, off


def close(got, x, *how, **more):
    want, off = oracle(x, *how, **more)
    assert got.dtype == x.dtype and got.shape == x.shape
    assert ((got.detach().cpu().double() - want).abs() <= off + (2.0 ** -25 if x.dtype == torch.float16 else 0.0)).all()


SHAPES = [      # batch, tokens, heads, key heads, head, part
    (1, 1, 1, 1, 2, 2), (2, 7, 4, 2, 64, 64), (1, 33, 8, 8, 128, 64), (3, 5, 2, 1, 80, 32), (2, 3, 3, 3, 77, 50), (1, 9, 4, 1, 256, 256), (1, 300, 2, 2, 96, 24), (5, 1, 40, 8, 128, 128),
]


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", list(U))
@pytest.mark.parametrize("shape", SHAPES)
def test_turns_and_gradients(shape, dtype, interleaved):
    batch, tokens, heads, key_heads, head, part = shape
    g = torch.Generator().manual_seed(1)
    q, k, dq, dk = (torch.randn(batch, tokens, h, head, generator=g).to(dtype).cuda() for h in (heads, key_heads) * 2)
    positions = torch.randint(0, 4096, (batch, tokens), generator=g, dtype=torch.int32).cuda()
    frequencies = ops.rotary_frequencies(part)
    q, k = q.requires_grad_(), k.requires_grad_()
    out = ops.rotary(q, k, positions, frequencies, interleaved=interleaved, magnitude=1.25)
    grads = torch.autograd.grad(out, (q, k), (dq, dk))
    for x, y, dx, dy in zip((q, k), out, grads, (dq, dk)):
        close(y, x, positions, frequencies, interleaved, 1.25)
        close(dx, dy, positions, frequencies, interleaved, 1.25, inverse=True)


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("wide", [False, True])
def test_far_positions(wide, interleaved):
    first = 3_000_000_000 if wide else 2_000_000_000
    positions = torch.arange(first, first + 20, dtype=torch.int64 if wide else torch.int32, device="cuda")
    if not wide:
        positions = torch.cat((positions[:10], -positions[10:]))
    q = torch.randn(2, 20, 2, 64, device="cuda")
    close(ops.rotary(q, None, positions, ops.rotary_frequencies(64), interleaved)[0], q, positions, ops.rotary_frequencies(64), interleaved, 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_layouts(dtype, interleaved):
    """Slices of a fused projection, heads before tokens, rows at any element, an element apart, shared rows."""
    f = ops.rotary_frequencies(32)
    p = torch.arange(11, device="cuda")
    qkv = torch.randn(2, 11, 8, 64, device="cuda").to(dtype)
    for q, k in ((qkv[:, :, :4], qkv[:, :, 4:6]), (qkv.transpose(1, 2).contiguous().transpose(1, 2)[:, :, :4], qkv[:, :, 4:6]), (qkv[..., 1:50], qkv[:, :, :2, 3:52]),
                 (qkv[..., ::2], qkv[:, :, 2:3, ::2]), (qkv[:, :, :1].expand(-1, -1, 4, -1), qkv[:1, :, 4:6].expand(2, -1, -1, -1))):
        out = ops.rotary(q, k, p, f, interleaved)
        for x, y in zip((q, k), out):
            close(y, x, p, f, interleaved, 1.0)


@pytest.mark.gpu
def test_one_of_the_two():
    f, p = ops.rotary_frequencies(64), torch.arange(6, device="cuda", dtype=torch.int32)
    q, k = (torch.randn(1, 6, 2, 64, device="cuda", requires_grad=True) for _ in range(2))
    a, b = ops.rotary(q, k, p, f)
    (dq,) = torch.autograd.grad(a, q, torch.ones_like(a))
    a, b = ops.rotary(q, k, p, f)
    (dk,) = torch.autograd.grad(b, k, torch.ones_like(b))
    alone, none = ops.rotary(q, None, p, f)
    assert none is None and torch.equal(alone, a)
    close(dq, torch.ones_like(a), p, f, False, 1.0, inverse=True)
    close(dk, torch.ones_like(a), p, f, False, 1.0, inverse=True)
    a, b = ops.rotary(q.detach(), k, p, f)
    assert torch.equal(torch.autograd.grad(b, k, torch.ones_like(b))[0], dk)


@pytest.mark.gpu
def test_there_and_back():
    f, p = ops.rotary_frequencies(128), torch.arange(100, device="cuda")
    q, k = torch.randn(2, 100, 4, 128, device="cuda"), torch.randn(2, 100, 2, 128, device="cuda")
    q2, k2 = ops.rotary(*ops.rotary(q, k, p, f), -p, f)
    assert (q2 - q).abs().max() < 1e-5 and (k2 - k).abs().max() < 1e-5


@pytest.mark.gpu
def test_empty_and_graph():
    f, p = ops.rotary_frequencies(64), torch.arange(6, device="cuda")
    q, k = torch.randn(1, 6, 4, 64, device="cuda"), torch.randn(1, 6, 2, 64, device="cuda")
    for a, b in ((q[:0], k[:0]), (q[:, :0], k[:, :0])):
        got = ops.rotary(a, b, p[:a.shape[1]], f)
        assert got[0].shape == a.shape and got[1].shape == b.shape
    assert torch.equal(ops.rotary(q[:, :, :0], k, p, f)[1], ops.rotary(q, k, p, f)[1])
    assert torch.equal(ops.rotary(q, k[:, :, :0], p, f)[0], ops.rotary(q, k, p, f)[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = ops.rotary(q, k, p, f)
    for _ in range(3):
        q.normal_()
        p.add_(1000)
        want = ops.rotary(q, k, p, f)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held[0], want[0]) and torch.equal(held[1], want[1])


def test_frequencies():
    f = ops.rotary_frequencies(8, base=100.0, device="cpu")
    assert f.dtype == torch.float64 and torch.allclose(f, torch.tensor([1.0, 100 ** -0.25, 0.1, 100 ** -0.75], dtype=torch.float64))
    assert torch.equal(ops.rotary_frequencies(8, base=100.0, stretch=4.0, device="cpu"), f / 4)
    # 100 positions: 15.9, 5.0, 1.59 and 0.5 turns; whole ones from 10 on, none below 1
    g = ops.rotary_frequencies(8, base=100.0, stretch=4.0, original=100, slow=1.0, fast=10.0, device="cpu")
    turns = 100 * f / (2 * math.pi)
    keep = ((turns - 1) / 9).clamp(0, 1)
    assert torch.allclose(g, f * keep + f / 4 * (1 - keep)) and g[0] == f[0] and g[3] == f[3] / 4
    for bad in (dict(part=7), dict(part=0), dict(part=258), dict(part=8, base=0.0), dict(part=8, stretch=-1.0), dict(part=8, stretch=2.0, original=10, slow=2.0, fast=2.0)):
        with pytest.raises(ValueError):
            ops.rotary_frequencies(device="cpu", **bad)


def test_refusals_of_the_entry_point():
    lib = runtime.load_library()
    p = ctypes.c_void_p
    longs = lambda *v: (ctypes.c_longlong * len(v))(*v)      # noqa: E731
    good, st = (1, 4, 2, 2, 64, 64), (512, 128, 64) * 4 + (4, 1)

    def call(ptrs=(4096, 8192, 12288, 16384, 20480, 24576), sizes=good, strides=st, interleaved=0, inverse=0, element=1, wide=0):
        return lib.lego_hip_rotary(*[p(x) if x else None for x in ptrs], longs(*sizes), longs(*strides), interleaved, 1.0, inverse, element, wide, None)

    for i in range(6):
        assert call(tuple(0 if j == i else x for j, x in enumerate((4096, 8192, 12288, 16384, 20480, 24576)))) == 1
        assert call(tuple(x + 1 if j == i else x for j, x in enumerate((4096, 8192, 12288, 16384, 20480, 24576)))) == 1
    for bad in ((0, 4, 2, 2, 64, 64), (1, 0, 2, 2, 64, 64), (1, 4, 0, 2, 64, 64), (1, 4, 2, -1, 64, 64), (1, 4, 2, 0, 64, 64), (1, 4, 2, 2, 64, 66), (1, 4, 2, 2, 64, 7), (1, 4, 2, 2, 64, 0),
                (1, 4, 2, 2, 512, 258), (1 << 20, 1 << 20, 2, 2, 64, 64), (1, 4, 1 << 25, 2, 64, 64)):
        assert call(sizes=bad) == 1, bad
    assert call(strides=(-1,) + st[1:]) == 1 and call(element=3) == 1 and call(interleaved=2) == 1 and call(inverse=-1) == 1 and call(wide=2) == 1


@pytest.mark.gpu
def test_second_derivatives_and_saved_tensors():
    """What would need the gradient's own gradient raises; saved tensors that come back as others are an error before anything is launched."""
    q, k = (torch.randn(2, 9, h, 16, device="cuda", dtype=torch.float32).requires_grad_() for h in (4, 2))
    at, f = torch.arange(9, device="cuda"), ops.rotary_frequencies(16)
    turned = ops.rotary(q, k, at, f)
    dq, dk = torch.autograd.grad(turned[0].square().sum() + turned[1].square().sum(), (q, k), create_graph=True)
    assert torch.allclose(dq, 2 * q, atol=1e-4) and torch.allclose(dk, 2 * k, atol=1e-4)      # lengths stay: 32-bit roundings of numbers below 8
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dq.square().sum() + turned[0].sum(), q)
    for other in (lambda t: t.cpu(), lambda t: t[:5], lambda t: t.float()):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, other):
            turned = ops.rotary(q, k, at, f)
        with pytest.raises((RuntimeError, ValueError)):
            torch.autograd.grad(turned[0].sum() + turned[1].sum(), (q, k))


@pytest.mark.gpu
def test_refusals():
    q, k = torch.randn(2, 6, 4, 64, device="cuda"), torch.randn(2, 6, 2, 64, device="cuda")
    p, f = torch.arange(6, device="cuda"), ops.rotary_frequencies(64)
    for args, how in (((q.double(), k, p, f), {}), ((q, k.half(), p, f), {}), ((q[0], k, p, f), {}), ((q, k[:1], p, f), {}), ((q, k[..., :62], p, f), {}), ((q.cpu(), k, p, f), {}),
                      ((q, k, p[:5], f), {}), ((q, k, p.float(), f), {}), ((q, k, p.cpu(), f), {}), ((q, k, p, f.float()), {}), ((q, k, p, f.cpu()), {}), ((q, k, p, f[:0]), {}),
                      ((q, k, p, ops.rotary_frequencies(66)), {}), ((q, k, p, f), dict(magnitude=math.nan))):
        with pytest.raises(ValueError):
            ops.rotary(*args, **how)
