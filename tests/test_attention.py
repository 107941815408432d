"""Attention and its gradient against the definition in 64 bits, and what the entry points refuse.

Tolerances count roundings.  With u half a step of the type (bf16 2^-8, fp16 2^-11), P and dS are rounded once as operands of a product and a result once as it is
stored; scores and sums are fp32, whose errors are counted as ``e`` for the relative error of P: (head + 8) products and sums of 2^-24 each of the scores' absolute
terms, 2^-21 for exponential, sum and division.  A value also loses what lies below its
type's smallest numbers: half of 2^-24 in fp16, and in bf16, as in fp32, all of a value below 2^-126 (exponentials of less are zeros).
"""
import ctypes
import math

import pytest
import torch

from lego_amd import ops, runtime

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
SINK = {torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}


def seen_by(queries, keys, causal, documents, prefix):
    """[batch or 1, 1, query, key]"""
    place = torch.arange(queries)[:, None] + keys - queries
    at = torch.arange(keys)
    seen = torch.ones(1, 1, queries, keys, dtype=torch.bool)
    if causal:
        seen = (at <= place)[None, None]
        if prefix is not None:
            seen = seen | (at < prefix[:, None, None, None])
    if documents is not None:
        own = documents[:, keys - queries:]
        seen = seen & ((own[:, None, :, None] == documents[:, None, None, :]) & (documents >= 0)[:, None, None, :])
    return seen


def oracle(q, k, v, dout, causal=False, scale=None, softcap=0.0, slopes=None, documents=None, prefix=None):
    """out, lse, dq, dk, dv in 64 bits and a bound of each one's error, as the module's text counts it."""
    u, sink = U[q.dtype], SINK[q.dtype]
    group = q.shape[2] // k.shape[2]
    dim = q.shape[3]
    scale = 1 / math.sqrt(dim) if scale is None else scale
    documents, prefix, slopes = (None if t is None else t.cpu() for t in (documents, prefix, slopes))
    q, dout = (t.detach().cpu().double().transpose(1, 2) for t in (q, dout))
    k, v = (t.detach().cpu().double().transpose(1, 2).repeat_interleave(group, 1) for t in (k, v))
    seen = seen_by(q.shape[2], k.shape[2], causal, documents, prefix).expand(q.shape[0], q.shape[1], -1, -1)
    s = scale * q @ k.transpose(2, 3)
    terms = abs(scale) * q.abs() @ k.abs().transpose(2, 3)
    bend = torch.ones_like(s)
    if softcap:
        bend = 1 - torch.tanh(s / softcap) ** 2
        s = softcap * torch.tanh(s / softcap)
        terms = terms + softcap
    if slopes is not None:
        place = torch.arange(q.shape[2])[:, None] + k.shape[2] - q.shape[2]
        away = slopes.double()[:, None, None] * (place - torch.arange(k.shape[2])).abs()
        s, terms = s - away, terms + away
    s = s.masked_fill(~seen, -math.inf)
    lse = torch.logsumexp(s, 3)
    p = torch.exp(s - lse.masked_fill(lse == -math.inf, 0.0)[..., None]).masked_fill(~seen, 0.0)
    full = seen.any(3)
    v, k = (t.nan_to_num(0.0, 0.0, 0.0) for t in (v, k))
    q, dout = (t.masked_fill(~full[..., None], 0.0) for t in (q, dout))
    e = ((dim + 8) * 2.0 ** -24 * terms.nan_to_num(0.0).masked_fill(~seen, 0.0)).amax((2, 3), keepdim=True) + 2.0 ** -21
    out = p @ v
    out_off = u * out.abs() + (u + 2 * e) * (p @ v.abs()) + sink * (1 + seen.double() @ v.abs())
    lse_off = e.amax(3) * 2 + 2.0 ** -22 * lse.abs().masked_fill(~full, 0.0) + 2.0 ** -21
    # the kernels' own out stands in delta
    delta, delta_off = (dout * out).sum(3, keepdim=True), (dout.abs() * out_off).sum(3, keepdim=True)
    dp = dout @ v.transpose(2, 3)
    dp_terms = dout.abs() @ v.abs().transpose(2, 3)
    ds = (p * (dp - delta) * bend).masked_fill(~seen, 0.0)
    up = sink * 2 * dout.abs().amax((2, 3), keepdim=True)
    ds_off = (u * ds.abs() + p * (delta_off + (3 * e + (dim + 8) * 2.0 ** -24) * (dp_terms + delta.abs()) + 2.0 ** -21 * (dp_terms + delta.abs())) + up).masked_fill(~seen, 0.0)
    if softcap:      # 4 r (1 - r): r has an absolute error of 2^-22
        ds_off = ds_off + (2.0 ** -19 * p * (dp - delta).abs()).masked_fill(~seen, 0.0)
    dq, dq_off = scale * ds @ k, abs(scale) * ds_off @ k.abs()
    dk, dk_off = scale * ds.transpose(2, 3) @ q, abs(scale) * ds_off.transpose(2, 3) @ q.abs()
    dv = p.transpose(2, 3) @ dout
    dv_off = ((u + 2 * e) * p + sink * seen.double()).transpose(2, 3) @ dout.abs()
    dk, dk_off, dv, dv_off = (t.unflatten(1, (-1, group)).sum(2) for t in (dk, dk_off, dv, dv_off))
    dq_off, dk_off, dv_off = (off + u * x.abs() + sink + 2.0 ** -19 * off for off, x in ((dq_off, dq), (dk_off, dk), (dv_off, dv)))
    back = lambda t: t.transpose(1, 2)      # noqa: E731
    return (back(out), lse, back(dq), back(dk), back(dv)), (back(out_off), lse_off, back(dq_off), back(dk_off), back(dv_off))


NAMES = ("out", "lse", "dq", "dk", "dv")


def close(got, want, off):
    for name, g, w, o in zip(NAMES, got, want, off):
        g = g.detach().cpu().double()
        assert g.shape == w.shape, name
        assert torch.equal(g == -math.inf, w == -math.inf), name
        w = w.masked_fill(w == -math.inf, 0.0)
        g = g.masked_fill(g == -math.inf, 0.0)
        assert torch.isfinite(g).all(), name
        worst = ((g - w).abs() / (o + 1e-300)).max()
        assert worst <= 1.0, (name, float(worst), float((g - w).abs().max()))


def make(batch, queries, keys, heads, key_heads, dim, dtype, seed=0, layout="own"):
    g = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g).to(dtype).cuda()      # noqa: E731
    if layout == "fused":        # slices of one projection
        qkv = rand(batch, keys, heads + 2 * key_heads, dim)
        q, k, v = qkv[:, keys - queries:, :heads] if queries <= keys else rand(batch, queries, heads, dim), qkv[:, :, heads:heads + key_heads], qkv[:, :, heads + key_heads:]
    elif layout == "heads_first":
        q, k, v = (rand(batch, h, t, dim).transpose(1, 2) for h, t in ((heads, queries), (key_heads, keys), (key_heads, keys)))
    elif layout == "odd_base":       # rows that start at any element: copied
        q, k, v = (rand(batch * t * h * dim + 1)[1:].view(batch, t, h, dim) for h, t in ((heads, queries), (key_heads, keys), (key_heads, keys)))
    elif layout == "shared":         # one key and value for all heads and batches
        q = rand(batch, queries, heads, dim)
        k, v = (rand(1, keys, 1, dim).expand(batch, -1, key_heads, -1) for _ in range(2))
    else:
        q, k, v = (rand(batch, t, h, dim) for h, t in ((heads, queries), (key_heads, keys), (key_heads, keys)))
    return q, k, v, rand(batch, queries, heads, dim)


def both(q, k, v, dout, **how):
    out, lse, rest = ops.attention_fwd(q, k, v, **how, with_rest=True)
    grads = ops.attention_bwd(dout, q, k, v, out, lse, **how, rest=rest)
    return (out, lse, *grads)


def check(q, k, v, dout, **how):
    got = both(q, k, v, dout, **how)
    want = oracle(q, k, v, dout, **how)
    close(got, *want)
    out, _, rest = ops.attention_fwd(q, k, v, **how, with_rest=True)      # what rounding took is at most a rounding
    assert (rest.float().abs() <= U[out.dtype] * out.float().abs() + 2.0 ** -24).all()
    without = ops.attention_fwd(q, k, v, **how)
    assert torch.equal(without[0], got[0]) and torch.equal(without[1], got[1])
    close(without + ops.attention_bwd(dout, q, k, v, *without, **how), *want)
    return got


SHAPES = [      # batch, queries, keys, heads, key heads, head
    (1, 1, 1, 1, 1, 8), (2, 1, 1, 4, 2, 64), (1, 63, 63, 2, 1, 64), (1, 64, 64, 2, 2, 128), (2, 65, 65, 4, 1, 96), (1, 77, 77, 3, 3, 40),
    (1, 128, 128, 2, 2, 64), (1, 129, 129, 6, 2, 80), (2, 200, 333, 4, 4, 128), (1, 1, 500, 8, 2, 128), (1, 193, 40, 2, 1, 64), (1, 577, 577, 2, 1, 104), (3, 31, 700, 2, 2, 24),
]


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES)
def test_attention_and_gradients(shape, dtype, causal):
    check(*make(*shape, dtype), causal=causal)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["fused", "heads_first", "odd_base", "shared"])
@pytest.mark.parametrize("shape", [(2, 150, 150, 4, 2, 64), (1, 70, 201, 6, 3, 128), (2, 97, 97, 4, 4, 72)])
def test_layouts(shape, layout):
    check(*make(*shape, torch.bfloat16, layout=layout), causal=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 96, 128])
@pytest.mark.parametrize("queries,keys", [(150, 150), (65, 260), (260, 65)])
@pytest.mark.parametrize("how", ["capped", "slopes", "both", "both_ways"])
def test_scores(dtype, dim, queries, keys, how):
    q, k, v, dout = make(2, queries, keys, 4, 2, dim, dtype, seed=3)
    slopes = torch.tensor([0.5, 0.125, 0.03, 0.0], device="cuda")
    check(3 * q, 3 * k, v, dout, causal=how != "both_ways", scale=0.2 if how == "both" else None, softcap=5.0 if how in ("capped", "both") else 0.0,
          slopes=None if how == "capped" else slopes)


def pack(lengths, padding=0):
    ids = [i for i, n in enumerate(lengths) for _ in range(n)]
    return ids + [-1] * padding


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("queries", [400, 130])
@pytest.mark.parametrize("kind", ["packed", "many", "unordered", "padded", "all_padding"])
def test_documents(kind, queries, causal):
    g = torch.Generator().manual_seed(5)
    rows = {"packed": [pack([100, 200, 100]), pack([1, 335, 64])], "many": [pack([8] * 50), pack([1] * 400)], "unordered": torch.randint(0, 3, (2, 400), generator=g).tolist(),
            "padded": [pack([100, 111], 189), [-1] * 70 + pack([330])], "all_padding": [[-1] * 400, pack([400])]}[kind]
    documents = torch.tensor(rows, dtype=torch.int32, device="cuda")
    q, k, v, dout = make(2, queries, 400, 4, 2, 64, torch.bfloat16, seed=7)
    hidden = (documents < 0)
    k[hidden], v[hidden] = math.nan, math.inf      # whatever padding holds
    q[hidden[:, 400 - queries:]], dout[hidden[:, 400 - queries:]] = math.nan, math.nan
    got = check(q, k, v, dout, causal=causal, documents=documents)
    for name, t in zip(NAMES[2:], got[2:]):
        assert (t[hidden if t.shape[1] == 400 else hidden[:, 400 - queries:]] == 0).all(), name


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("queries,keys", [(200, 200), (60, 300), (300, 60)])
@pytest.mark.parametrize("documents", [False, True])
def test_prefix(queries, keys, documents, dtype):
    if documents and queries > keys:
        pytest.skip("documents are the keys'")
    q, k, v, dout = make(4, queries, keys, 2, 1, 64, dtype, seed=11)
    prefix = torch.tensor([0, 33, keys, keys + 1000], dtype=torch.int32, device="cuda")
    ids = torch.tensor([pack([keys // 3, keys - keys // 3])] * 4, dtype=torch.int32, device="cuda") if documents else None
    check(q, k, v, dout, causal=True, prefix=prefix, documents=ids)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 96, 128])
@pytest.mark.parametrize("kind", ["all", "scores", "documents", "prefix"])
def test_more_heads_than_the_chip_holds(kind, dim, dtype):
    """From some number of workgroups on they are not cut in halves: two blocks of each of 264 heads."""
    q, k, v, dout = make(2, 150, 150, 132, 66, dim, dtype, seed=13)
    how = {"all": {}, "scores": dict(causal=True, softcap=6.0, slopes=torch.linspace(0, 0.5, 132).cuda()),
           "documents": dict(causal=True, documents=torch.tensor([pack([30, 71, 40], 9), pack([150])], dtype=torch.int32, device="cuda")),
           "prefix": dict(causal=True, prefix=torch.tensor([70, 0], dtype=torch.int32, device="cuda"))}[kind]
    check(q, k, v, dout, **how)


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("queries", [520, 390])
@pytest.mark.parametrize("kind", ["packed", "unordered", "padded"])
def test_documents_in_order_of_their_work(kind, queries, causal):
    """Five blocks (four of queries) of each of 66 heads, the ones with the most work first."""
    rows = {"packed": pack([200, 3, 300, 17]), "unordered": torch.randint(0, 4, (520,), generator=torch.Generator().manual_seed(5)).tolist(), "padded": pack([129, 200], 191)}[kind]
    documents = torch.tensor([rows], dtype=torch.int32, device="cuda")
    prefix = torch.tensor([250], dtype=torch.int32, device="cuda") if causal and kind == "packed" else None
    check(*make(1, queries, 520, 66, 66, 128, torch.bfloat16, seed=21), causal=causal, documents=documents, prefix=prefix)


@pytest.mark.gpu
def test_prefix_below_zero_is_none():
    q, k, v, _ = make(2, 70, 70, 2, 2, 64, torch.bfloat16)
    with_none = ops.attention(q, k, v, causal=True)
    assert torch.equal(ops.attention(q, k, v, causal=True, prefix=torch.tensor([-5, 0], dtype=torch.int32, device="cuda")), with_none)


@pytest.mark.gpu
def test_rows_that_see_nothing_take_and_give_nothing():
    """More queries than keys, causal: the first ones stand before every key, and hold anything."""
    q, k, v, dout = make(1, 150, 60, 2, 1, 64, torch.float16, seed=1)
    q[:, :90], dout[:, :90] = math.nan, math.nan
    got = check(q, k, v, dout, causal=True)
    assert (got[0][:, :90] == 0).all() and (got[2][:, :90] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("size", [1e-5, 1e3])
def test_small_and_large_gradients_in_fp16(size):
    """dS lies far below dout: P is about 1/keys.  dout below fp16's normal numbers has few digits itself, and is taken as it is."""
    q, k, v, dout = make(1, 300, 300, 2, 2, 64, torch.float16, seed=2)
    dout = (dout.float() * size).half()
    dout[:, 200:] *= 0.125      # tiles of other sizes
    check(q, k, v, dout, causal=True)


@pytest.mark.gpu
def test_large_scores():
    q, k, v, dout = make(1, 130, 130, 2, 2, 64, torch.bfloat16, seed=4)
    check(8 * q, 8 * k, v, dout, causal=True)
    check(q, k, v, dout, causal=False, scale=-0.3)


@pytest.mark.gpu
def test_autograd_gradients_and_repeats():
    q, k, v, dout = make(2, 200, 200, 8, 2, 64, torch.bfloat16, layout="fused")
    q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    first = None
    for _ in range(3):
        out = ops.attention(q, k, v, causal=True)
        grads = torch.autograd.grad(out, (q, k, v), dout)
        now = (out.detach(), *grads)
        first = first or now
        assert all(torch.equal(a, b) for a, b in zip(first, now))
    q0, k0, v0 = (t.detach() for t in (q, k, v))
    out, lse, rest = ops.attention_fwd(q0, k0, v0, causal=True, with_rest=True)
    got = ops.attention_bwd(dout, q0, k0, v0, out, lse, causal=True, rest=rest)
    assert torch.equal(out, first[0]) and all(torch.equal(a, b) for a, b in zip(got, first[1:]))
    # shared keys through expand: autograd sums what the kernel gives for each
    k1 = torch.randn(1, 200, 1, 64, device="cuda").bfloat16().requires_grad_()
    out = ops.attention(q.detach(), k1.expand(2, -1, 2, -1), v.detach(), causal=True)
    (dk,) = torch.autograd.grad(out, (k1,), dout)
    assert dk.shape == k1.shape and torch.isfinite(dk).all()


@pytest.mark.gpu
@pytest.mark.parametrize("node", ["call", "python"])
def test_no_second_derivative(node):
    """What would need one raises, and is no gradient with a part missing."""
    q, k, v, _ = make(1, 20, 20, 2, 2, 64, torch.bfloat16)
    q.requires_grad_()
    attend = (lambda: ops.attention(q, k, v, causal=True)) if node == "call" else (lambda: ops.LEGOAttention.apply(q, k, v, True, None, 0.0, None, None, None))
    out = attend()
    (dq,) = torch.autograd.grad(out.float().square().sum(), q, create_graph=True)
    (plain,) = torch.autograd.grad(attend().float().square().sum(), q)
    assert torch.equal(dq.detach(), plain)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dq.float().square().sum() + out.float().sum(), q)


@pytest.mark.gpu
def test_saved_tensors_that_come_back_as_others():
    """A hook that hands back what was not saved is an error before anything is launched; one that keeps them on the host is not."""
    q, k, v, dout = make(1, 20, 20, 2, 2, 64, torch.bfloat16, layout="fused")
    q = q.detach().requires_grad_()
    documents = torch.zeros(1, 20, dtype=torch.int32, device="cuda")
    how = dict(causal=True, slopes=torch.tensor([0.1, 0.2], device="cuda"), documents=documents)
    (want,) = torch.autograd.grad(ops.attention(q, k, v, **how), q, dout)
    with torch.autograd.graph.save_on_cpu():
        out = ops.attention(q, k, v, **how)
    assert torch.equal(torch.autograd.grad(out, q, dout)[0], want)
    for other in (lambda t: t.cpu(), lambda t: t[:, :10] if t.dim() > 1 else t[:1], lambda t: t.long() if t.dtype == torch.int32 else t):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, other):
            out = ops.attention(q, k, v, **how)
        with pytest.raises((RuntimeError, ValueError)):
            torch.autograd.grad(out, q, dout)


@pytest.mark.gpu
def test_gradient_against_differences():
    """A step along a random direction changes sum(out * dout) by the gradient's part in it.  fp32 sums of fp16 outputs: an output's rounding, 2^-11 relative, adds up like
    noise over the outputs, which a step of 2^-5 of values near one, over three directions, stands well above."""
    q, k, v, dout = make(1, 90, 90, 2, 1, 64, torch.float16, seed=9)
    how = dict(causal=True, softcap=4.0, slopes=torch.tensor([0.1, 0.3], device="cuda"))
    _, _, *grads = both(q, k, v, dout, **how)
    (want, *_), (off, *_) = oracle(q, k, v, dout, **how)
    noise = (off * dout.cpu().double().abs()).sum()
    for i in range(3):
        ins = [q, k, v]
        way = torch.randn(ins[i].shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(i)).half()
        way = way * 0 + grads[i].sign()      # uphill, so that the change stands above the noise
        step = 2.0 ** -6
        ends = []
        for sign in (1, -1):
            at = list(ins)
            at[i] = (ins[i] + sign * step * way).half()
            ends.append((ops.attention_fwd(*at, **how)[0].double() * dout.double()).sum().cpu())
        moved = ((ins[i] + step * way).half().double() - (ins[i] - step * way).half().double())
        expected = (grads[i].double() * moved).sum().cpu()
        # curvature: third order in the step; the bound is a quarter of the change and the roundings of both ends
        assert abs(ends[0] - ends[1] - expected) <= 0.25 * abs(expected) + 2 * noise


@pytest.mark.gpu
def test_empty_calls():
    q, k, v, dout = make(2, 5, 7, 4, 2, 64, torch.bfloat16)
    assert ops.attention(q[:, :0], k, v).shape == (2, 0, 4, 64)
    out, lse = ops.attention_fwd(q, k[:, :0], v[:, :0])
    assert (out == 0).all() and (lse == -math.inf).all()
    dq, dk, dv = ops.attention_bwd(dout, q, k[:, :0], v[:, :0], out, lse)
    assert (dq == 0).all() and dk.shape == (2, 0, 2, 64) and dv.shape == (2, 0, 2, 64)
    assert ops.attention(q[:0], k[:0], v[:0]).shape == (0, 5, 4, 64)


@pytest.mark.gpu
def test_other_stream_and_graph():
    q, k, v, dout = make(1, 260, 260, 4, 1, 64, torch.bfloat16)
    documents = torch.tensor([pack([100, 160])], dtype=torch.int32, device="cuda")
    how = dict(causal=True, documents=documents)
    want = both(q, k, v, dout, **how)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = both(q, k, v, dout, **how)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = []
    for _ in range(2):      # two graphs, each with workspaces of its own
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = both(q, k, v, dout, **how)
        graphs.append((graph, held))
    for turn in range(4):
        q.normal_()
        dout.normal_()
        want = both(q, k, v, dout, **how)
        torch.cuda.synchronize()
        for graph, held in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, held in graphs:
            assert all(torch.equal(a, b) for a, b in zip(held, want)), turn


@pytest.mark.gpu
def test_far_tokens():
    """Tokens 40000 elements apart, over 32 bits of bytes in all."""
    base = torch.empty(60000, 40000, dtype=torch.bfloat16, device="cuda")
    k, v = base[None, :, None, :64], base[None, :, None, 64:128]
    k.normal_()
    v.normal_()
    q = torch.randn(1, 40, 1, 64, device="cuda").bfloat16()
    dout = torch.randn_like(q)
    got = both(q, k, v, dout, causal=True)
    want = both(q, k.contiguous(), v.contiguous(), dout, causal=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals_of_the_entry_points():
    """Everything is looked at on the host, before anything touches a device."""
    lib = runtime.load_library()
    p = ctypes.c_void_p
    longs = lambda *v: (ctypes.c_longlong * len(v))(*v)      # noqa: E731
    need = ctypes.c_ulonglong(0)
    good = (2, 100, 100, 4, 2, 64)
    assert lib.lego_hip_attention_workspace_bytes(longs(*good), 0, 0, ctypes.byref(need)) == 0 and need.value == 0
    assert lib.lego_hip_attention_workspace_bytes(longs(*good), 1, 0, ctypes.byref(need)) == 0 and need.value == 2 * 2 * 8
    assert lib.lego_hip_attention_workspace_bytes(longs(*good), 0, 1, ctypes.byref(need)) == 0 and need.value >= 2 * 4 * 100 * 4
    for bad in ((0, 100, 100, 4, 2, 64), (2, 0, 100, 4, 2, 64), (2, 100, 0, 4, 2, 64), (2, 100, 100, 4, 3, 64), (2, 100, 100, 4, 2, 60), (2, 100, 100, 4, 2, 136),
                (1 << 20, 1 << 20, 4, 4, 4, 64), (2, 100, 100, 4, 0, 64), (2, 100, 100, 4, 2, 0), (1, 1 << 29, 100, 1, 1, 64)):
        assert lib.lego_hip_attention_workspace_bytes(longs(*bad), 0, 1, ctypes.byref(need)) == 1, bad
    strides = lambda n, **k: longs(*(k.get("s") or (25600, 256, 64) * n))      # noqa: E731
    at = lambda i: p(4096 * (i + 1))      # noqa: E731

    def fwd(ptrs=None, sizes=good, st=None, scale=0.1, cap=0.0, slopes=None, docs=None, prefix=None, causal=1, element=1, ws=None, room=0):
        return lib.lego_hip_attention_fwd(*(ptrs or [at(i) for i in range(6)]), longs(*sizes), st or strides(4), scale, cap, slopes, docs, prefix, causal, element, ws, room, None)

    for i in range(6):
        ptrs = [at(j) for j in range(6)]
        ptrs[i] = None
        assert i == 4 or fwd(ptrs) == 1      # (rest may be null)
        ptrs[i] = p(4096 + 2)
        assert fwd(ptrs) == 1
    assert fwd(scale=math.nan) == 1 and fwd(scale=math.inf) == 1 and fwd(cap=-1.0) == 1 and fwd(cap=math.nan) == 1 and fwd(element=2) == 1 and fwd(causal=2) == 1
    assert fwd(prefix=at(9), causal=0) == 1 and fwd(slopes=p(4097)) == 1 and fwd(docs=p(4098)) == 1
    assert fwd(docs=at(9)) == 1 and fwd(docs=at(9), ws=at(10), room=8) == 1      # no workspace, a short one
    assert fwd(sizes=(2, 101, 100, 4, 2, 64), docs=at(9), ws=at(10), room=1 << 20) == 1
    assert fwd(st=strides(4, s=(25600, 256, 60) * 4)) == 1 and fwd(st=strides(4, s=(25600, 1 << 25, 64) * 4)) == 1 and fwd(st=strides(4, s=(-8, 256, 64) * 4)) == 1
    bwd = lambda ptrs, ws, room: lib.lego_hip_attention_bwd(*ptrs, longs(*good), strides(8), 0.1, 0.0, None, None, None, 1, 1, ws, room, None)      # noqa: E731
    ptrs = [at(i) for i in range(10)]
    assert bwd(ptrs, None, 0) == 1 and bwd(ptrs, at(20), 16) == 1 and bwd(ptrs, p(4097), 1 << 30) == 1
    for i in (0, 1, 2, 3, 4, 6, 7, 8, 9):
        assert bwd([None if j == i else x for j, x in enumerate(ptrs)], at(20), 1 << 30) == 1


def test_refusals_on_the_cpu():
    q = torch.zeros(1, 4, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="GPU"):
        ops.attention(q, q, q)


@pytest.mark.gpu
def test_refusals():
    q, k, v, dout = make(2, 10, 10, 4, 2, 64, torch.bfloat16)
    ints = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")      # noqa: E731
    for args, how in (((q.float(), k, v), {}), ((q, k.half(), v), {}), ((q[0], k, v), {}), ((q, k[:1], v[:1]), {}), ((q, k, v[:, :9]), {}), ((q[:, :, :3], k, v), {}),
                      ((q[..., :60], k[..., :60], v[..., :60]), {}), ((q, k, v), dict(softcap=-1.0)), ((q, k, v), dict(scale=math.inf)), ((q, k, v), dict(prefix=ints(2))),
                      ((q, k, v), dict(causal=True, prefix=ints(3))), ((q, k, v), dict(documents=ints(2, 9))), ((q, k[:, :9], v[:, :9]), dict(documents=ints(2, 9))),
                      ((q, k, v), dict(documents=ints(2, 10).long())), ((q, k, v), dict(slopes=torch.zeros(2, device="cuda"))),
                      ((q, k, v), dict(slopes=torch.zeros(4, device="cuda", requires_grad=True))), ((q.cpu(), k, v), {}), ((q, k, v), dict(documents=ints(2, 10).cpu())),
                      ((q[:, :, :0], k[:, :, :0], v[:, :, :0]), {})):
        with pytest.raises(ValueError):
            ops.attention(*args, **how)
    out, lse = ops.attention_fwd(q, k, v)
    for bad in ((dout[:, :9], q, k, v, out, lse), (dout, q, k, v, out.float(), lse), (dout, q, k, v, out, lse[:, :, :9]), (dout, q, k, v, out, lse.double())):
        with pytest.raises(ValueError):
            ops.attention_bwd(*bad)
