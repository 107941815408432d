"""Attention of drafted tokens over a paged cache, against the definition in 64 bits, and what is refused.

An output is rounded once, by u (half a step) of its value; P once as an operand, and its relative error beside that is e: (head + 8) steps of 2^-24 of the scores' absolute
terms and 2^-20 for exponentials, sums and the joining of parts.  Values below the type's smallest numbers are lost (2^-25 in fp16, 2^-126 in bf16)."""
import ctypes
import math
import subprocess
from pathlib import Path

import pytest
import torch

from lego_amd import ops, runtime

CSRC = Path(__file__).resolve().parents[1] / "lego_amd" / "csrc"
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
SINK = {torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}


def oracle(q, k, v, k_cache, v_cache, pages, lengths, tree=None, scale=None, softcap=0.0, slopes=None, positions=None):
    u, sink = U[q.dtype], SINK[q.dtype]
    batch, drafts, heads, dim = q.shape
    rows, count = k_cache.shape[1], k_cache.shape[0]
    group = heads // k_cache.shape[2]
    scale = dim ** -0.5 if scale is None else scale
    cpu = lambda t: None if t is None else t.cpu()      # noqa: E731
    q, k, v, k_cache, v_cache, pages, lengths, tree, slopes, positions = map(cpu, (q, k, v, k_cache, v_cache, pages, lengths, tree, slopes, positions))
    out, off = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    for b in range(batch):
        length = max(0, min(int(lengths[b]), rows * pages.shape[1]))
        at = torch.arange(length)
        page = pages[b].long()[at // rows] if length else at
        good = (page >= 0) & (page < count)
        at, page = at[good], page[good]
        kk, vv = k_cache[page, at % rows].double(), v_cache[page, at % rows].double()
        place, seen = at.double(), torch.ones(drafts, len(at), dtype=torch.bool)
        own = torch.arange(drafts).double() + length if positions is None else positions[b].double()
        if k is not None:
            kk, vv, place = torch.cat((kk, k[b].double())), torch.cat((vv, v[b].double())), torch.cat((place, own))
            shown = torch.ones(drafts, drafts).tril().bool() if tree is None else tree if tree.dim() == 2 else tree[b]
            seen = torch.cat((seen, shown), 1)
        for h in range(heads):
            kh, vh, qh = kk[:, h // group], vv[:, h // group], q[b, :, h].double()
            s, terms = scale * qh @ kh.t(), abs(scale) * qh.abs() @ kh.abs().t()
            if softcap:
                s, terms = softcap * torch.tanh(s / softcap), terms + softcap
            if slopes is not None:
                away = float(slopes[h]) * (own[:, None] - place).abs()
                s, terms = s - away, terms + away
            s = s.masked_fill(~seen, -math.inf)
            p = torch.softmax(s, 1).nan_to_num(0.0) if s.shape[1] else torch.zeros_like(s)
            e = ((dim + 8) * 2.0 ** -24 * terms.masked_fill(~seen, 0.0)).max() + 2.0 ** -20 if terms.numel() else 0.0
            out[b, :, h] = p @ vh
            off[b, :, h] = u * out[b, :, h].abs() + (u + 2 * e) * (p @ vh.abs()) + sink * (1 + seen.double() @ vh.abs())
    return out, off


def close(got, want, off):
    assert got.shape == want.shape and torch.isfinite(got).all()
    worst = ((got.cpu().double() - want).abs() / (off + 1e-300)).max()
    assert worst <= 1.0, float(worst)


def make(lengths, drafts, heads, key_heads, dim, rows, dtype, seed=0, spare=3, trees=True):
    g = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g).to(dtype).cuda()      # noqa: E731
    batch = len(lengths)
    need = [-(-n // rows) for n in lengths]
    order = torch.randperm(sum(need) + spare, generator=g).tolist()
    width = max(1, max(need))
    pages = torch.full((batch, width), -1, dtype=torch.int32)
    for b, n in enumerate(need):
        pages[b, :n] = torch.tensor(order[:n], dtype=torch.int32)
        order = order[n:]
    caches = [rand(sum(need) + spare, rows, key_heads, dim) for _ in range(2)]
    used = torch.zeros(sum(need) + spare, rows, dtype=torch.bool)
    for b, n in enumerate(lengths):
        at = torch.arange(n)
        used[pages[b].long()[at // rows], at % rows] = True
    for c in caches:      # what no sequence holds: anything
        c[~used] = math.nan
    tree = torch.rand(batch, drafts, drafts, generator=g) < 0.4
    tree |= torch.eye(drafts, dtype=torch.bool)
    return dict(q=rand(batch, drafts, heads, dim), k=rand(batch, drafts, key_heads, dim), v=rand(batch, drafts, key_heads, dim), k_cache=caches[0], v_cache=caches[1],
                pages=pages.cuda(), lengths=torch.tensor(lengths, dtype=torch.int32).cuda(), tree=tree.cuda() if trees else None)


def check(**how):
    got = ops.tree_attention(**how)
    close(got, *oracle(**how))
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,key_heads,dim", [(1, 1, 8), (4, 1, 64), (8, 2, 128), (6, 6, 80), (3, 1, 96), (40, 1, 64)])
@pytest.mark.parametrize("lengths,rows", [([1], 16), ([0, 63, 64, 65], 16), ([100, 0, 1000, 7, 513], 64), ([2000], 7), ([129] * 70, 1)])
def test_single_tokens(lengths, rows, heads, key_heads, dim, dtype):
    check(**make(lengths, 1, heads, key_heads, dim, rows, dtype, trees=False))


@pytest.mark.gpu
@pytest.mark.parametrize("drafts", [2, 16, 33, 64, 65, 130])
@pytest.mark.parametrize("heads,key_heads,dim", [(4, 4, 64), (8, 2, 128), (2, 1, 40)])
@pytest.mark.parametrize("lengths", [[0], [5, 700, 0, 64]])
def test_trees(lengths, heads, key_heads, dim, drafts):
    how = make(lengths, drafts, heads, key_heads, dim, 32, torch.bfloat16, seed=drafts)
    check(**how)
    check(**{**how, "tree": how["tree"][0]})
    check(**{**how, "tree": None})


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("how", ["capped", "slopes", "both"])
def test_scores(how, dtype):
    x = make([300, 40, 1111], 9, 8, 2, 64, 16, dtype, seed=3)
    x["q"] = 3 * x["q"]
    if how != "slopes":
        x |= dict(softcap=5.0, scale=0.2)
    if how != "capped":
        x |= dict(slopes=torch.tensor([2.0 ** -i for i in range(8)], device="cuda"), positions=x["lengths"][:, None] + torch.tensor([0, 1, 1, 2, 2, 2, 3, 1, 0], dtype=torch.int32, device="cuda"))
    check(**x)
    if how != "capped":
        check(**{**x, "tree": None, "positions": None})


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("drafts", [3, 13, 40])
@pytest.mark.parametrize("dim", [64, 96, 128])
def test_scores_of_all_numbers_of_rows(dim, drafts, dtype):
    """12, 52 and 160 rows a key head."""
    x = make([300, 40, 1111, 0, 77], drafts, 8, 2, dim, 16, dtype, seed=4)
    slopes = torch.tensor([2.0 ** -i for i in range(8)], device="cuda")
    positions = x["lengths"][:, None] + torch.arange(drafts, dtype=torch.int32, device="cuda") // 2
    check(**x, softcap=6.0)
    check(**x, slopes=slopes, positions=positions)
    check(**x, softcap=6.0, scale=-0.3, slopes=slopes, positions=positions)
    check(**x, scale=-0.3)


@pytest.mark.gpu
@pytest.mark.parametrize("drafts", [1, 5, 20, 40])
def test_tables_longer_than_a_piece(drafts):
    """Pages of 1 to 3 rows: the kernels hold 256 or 1024 entries of a table at a time."""
    for rows, lengths in ((1, [2500, 3, 1100]), (2, [4200]), (3, [3, 3500])):
        check(**make(lengths, drafts, 8, 2, 64, rows, torch.bfloat16, seed=rows))


@pytest.mark.gpu
def test_many_sequences_side_by_side():
    """More than 64 of them, in runs that begin and end anywhere, with blocks of rows side by side."""
    lengths = [(37 * i) % 501 for i in range(130)]
    check(**make(lengths, 2, 4, 2, 64, 16, torch.bfloat16, seed=8))
    check(**make(lengths[:70], 70, 4, 2, 64, 16, torch.float16, seed=9))
    lengths = [(677 * i) % 2901 for i in range(70)]
    check(**make(lengths, 2, 4, 2, 64, 16, torch.bfloat16, seed=10))
    check(**make(lengths[:20], 20, 4, 1, 128, 32, torch.bfloat16, seed=11))


@pytest.mark.gpu
@pytest.mark.parametrize("lengths", [[0, 200, 64, 1], [0]])
def test_over_the_cache_alone(lengths):
    how = make(lengths, 3, 4, 2, 64, 16, torch.bfloat16, trees=False) | dict(k=None, v=None)
    got = check(**how)
    assert (got[torch.tensor(lengths) == 0] == 0).all()


@pytest.mark.gpu
def test_rows_that_see_nothing():
    how = make([0, 80], 5, 4, 2, 64, 16, torch.float16)
    how["tree"][:, 2] = False
    got = check(**how)
    assert (got[0, 2] == 0).all() and (got[1, 2] != 0).any()


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128])
def test_bad_pages_and_lengths_stand_for_no_keys(dim):
    how = make([500, 300, 64], 3, 4, 2, dim, 16, torch.bfloat16)
    how["pages"][0, 3], how["pages"][0, 7], how["pages"][1, 0] = -1, 1 << 30, how["k_cache"].shape[0]
    how["pages"][2] = -7
    check(**how)
    how = make([500, 300, 64], 3, 4, 2, dim, 16, torch.bfloat16)
    full = how["pages"].shape[1] * 16
    how["pages"][:] = how["pages"][0]
    how["k_cache"], how["v_cache"] = (t.nan_to_num(0.0) for t in (how["k_cache"], how["v_cache"]))
    how["lengths"] = torch.tensor([full + 1000, -5, 1 << 30], dtype=torch.int32, device="cuda")
    check(**how)


@pytest.mark.gpu
def test_nan_of_one_sequence_stays_there():
    """A workgroup goes from one sequence's keys to the next one's."""
    how = make([70 + 3 * i for i in range(200)], 1, 8, 8, 64, 16, torch.bfloat16, trees=False)
    clean = ops.tree_attention(**how)
    first = how["pages"][::2, 0].long()
    how["k_cache"][first] = math.nan
    how["v_cache"][first] = math.inf
    got = ops.tree_attention(**how)
    assert torch.equal(got[1::2], clean[1::2]) and not torch.isfinite(got[::2]).any()


@pytest.mark.gpu
def test_layouts():
    """Caches with heads before rows, keys and values in one tensor, drafts out of a fused projection, a sequence's cache in one page."""
    how = make([300, 77], 4, 4, 2, 64, 16, torch.bfloat16)
    want = check(**how)
    both = torch.stack((how["k_cache"], how["v_cache"]), 2)
    first = how["k_cache"].transpose(1, 2).contiguous().transpose(1, 2)
    qkv = torch.cat((how["q"], how["k"], how["v"]), 2)
    got = ops.tree_attention(**{**how, "k_cache": both[:, :, 0], "v_cache": both[:, :, 1], "q": qkv[:, :, :4], "k": qkv[:, :, 4:6], "v": qkv[:, :, 6:]})
    assert torch.equal(got, want)
    assert torch.equal(ops.tree_attention(**{**how, "k_cache": first}), want)
    whole = torch.randn(2, 1000, 2, 64, device="cuda").bfloat16()
    check(**{**how, "k_cache": whole, "v_cache": -whole, "pages": torch.tensor([[1], [0]], dtype=torch.int32, device="cuda"), "lengths": torch.tensor([1000, 333], dtype=torch.int32, device="cuda")})


@pytest.mark.gpu
def test_far_rows():
    """A cache whose rows pass 32 bits of elements."""
    pool = torch.empty(70000, 16, 2, 2048, dtype=torch.bfloat16, device="cuda")
    cache = pool[..., :64]
    pages = torch.tensor([[69999, 3, 40000]], dtype=torch.int32, device="cuda")
    cache[pages[0].long()] = torch.randn(3, 16, 2, 64, device="cuda").bfloat16()
    small = cache[pages[0].long()].contiguous()
    how = make([41], 2, 4, 2, 64, 16, torch.bfloat16, trees=False)
    lengths = torch.tensor([41], dtype=torch.int32, device="cuda")
    got = ops.tree_attention(**{**how, "k_cache": cache, "v_cache": cache, "pages": pages, "lengths": lengths})
    want = ops.tree_attention(**{**how, "k_cache": small, "v_cache": small, "pages": torch.tensor([[0, 1, 2]], dtype=torch.int32, device="cuda"), "lengths": lengths})
    assert torch.equal(got, want)


@pytest.mark.gpu
def test_empty_calls():
    how = make([30, 0], 3, 4, 2, 64, 16, torch.bfloat16)
    assert ops.tree_attention(**{n: t[:, :0] if n in "qkv" else t for n, t in how.items() if n != "tree"}).shape == (2, 0, 4, 64)
    no_cache = {**how, "k_cache": how["k_cache"][:0], "v_cache": how["v_cache"][:0]}
    check(**{**how, "lengths": how["lengths"] * 0})
    assert torch.equal(ops.tree_attention(**no_cache), ops.tree_attention(**{**how, "lengths": how["lengths"] * 0}))
    assert (ops.tree_attention(**{**no_cache, "k": None, "v": None, "tree": None}) == 0).all()


@pytest.mark.gpu
def test_a_step_of_verification():
    """Rotary, attention of the drafts, and the accepted ones written to the cache, against attention over the whole sequence."""
    torch.manual_seed(0)
    heads, key_heads, dim, rows = 4, 2, 64, 16
    lengths, path = [40, 13], [0, 2, 3]      # draft 1 is refused: 0 -> 2 -> 3
    tokens = [torch.randn(1, n + 4, heads + 2 * key_heads, dim, device="cuda").bfloat16() for n in lengths]
    frequencies = ops.rotary_frequencies(dim)
    k_cache, v_cache = (torch.zeros(10, rows, key_heads, dim, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    pages = torch.tensor([[7, 1, 4, 9], [0, 3, 2, 5]], dtype=torch.int32, device="cuda")
    depth = torch.tensor([0, 1, 1, 2], dtype=torch.int32, device="cuda")
    tree = torch.tensor([[1, 0, 0, 0], [1, 1, 0, 0], [1, 0, 1, 0], [1, 0, 1, 1]], dtype=torch.bool, device="cuda")
    count = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    for b, n in enumerate(lengths):
        _, k = ops.rotary(tokens[b][:, :n, :heads], tokens[b][:, :n, heads:heads + key_heads], torch.arange(n, device="cuda"), frequencies)
        at = torch.arange(n, device="cuda")
        k_cache[pages[b].long()[at // rows], at % rows] = k[0]
        v_cache[pages[b].long()[at // rows], at % rows] = tokens[b][0, :n, heads + key_heads:]
    drafts = torch.cat([t[:, -4:] for t in tokens])
    q, k = ops.rotary(drafts[:, :, :heads], drafts[:, :, heads:heads + key_heads], count[:, None] + depth, frequencies)
    out = ops.tree_attention(q, k, drafts[:, :, heads + key_heads:], k_cache, v_cache, pages, count, tree=tree)
    for b, n in enumerate(lengths):
        line = torch.cat((tokens[b][:, :n], tokens[b][:, n:][:, path]), 1)
        places = torch.arange(n + 3, device="cuda")
        lq, lk = ops.rotary(line[:, :, :heads], line[:, :, heads:heads + key_heads], places, frequencies)
        whole = ops.attention(lq, lk, line[:, :, heads + key_heads:], causal=True)
        # two orders of the same sums: each is within its own bound of the exact value, 2^-8 of the output and of P |v| (at most 5 here)
        assert (whole[0, n:].float() - out[b][path].float()).abs().max() <= 2 * 2.0 ** -8 * (out[b].float().abs().max() + 5)


@pytest.mark.gpu
@pytest.mark.parametrize("lengths", [[60], [900, 3000, 5]])
def test_other_stream_and_graph(lengths):
    how = make(lengths, 3, 8, 2, 64, 16, torch.bfloat16)
    want = ops.tree_attention(**how)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.tree_attention(**how)
    side.synchronize()
    assert torch.equal(got, want)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = ops.tree_attention(**how)
        graphs.append((graph, held))
    full = how["lengths"].clone()
    for turn in range(4):      # other tokens and other lengths on the same graph
        how["q"].normal_()
        how["lengths"].copy_((full * (turn + 1)) // 4)
        want = ops.tree_attention(**how)
        torch.cuda.synchronize()
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, held in graphs:
            assert torch.equal(held, want), turn


def test_page_lookup_on_the_host(tmp_path):
    """The kernels' own lookup, compiled for the host: no key is read where a table or a length names none."""
    (tmp_path / "p.cpp").write_text('''
typedef struct { int x, y; } int2; typedef struct { float x, y; } float2;
#define HIP_INCLUDE_HIP_HIP_RUNTIME_H
#include <stdint.h>
''' + (CSRC / "attention_args.h").read_text().replace("#include <hip/hip_runtime.h>", "").replace("#pragma once", "") + '''
extern "C" int lookup(const int* p, unsigned n, unsigned c, bool w, unsigned at) { return page_of(p, n, c, w, at); }
extern "C" unsigned long long wrong_quotients(unsigned d)
{
  unsigned factor, shift;
  quotients_by(d, factor, shift);
  const unsigned long long last = 0x7fffffffull;
  unsigned long long wrong = 0;
  for (unsigned long long i = 0; i < 4000; ++i) {      // around multiples of d from either end of the range, and the ends
    const unsigned long long near[] = {i * d, i * d - 1, last - last % d - i * d, last - last % d - i * d - 1, i, last - i};
    for (unsigned long long x : near)
      if (x <= last) wrong += quotient((unsigned)x, factor, shift) != x / d;
  }
  return wrong;
}
''')
    lib = tmp_path / "p.so"
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-o", str(lib), str(tmp_path / "p.cpp")], check=True, capture_output=True)
    loaded = ctypes.CDLL(str(lib))
    for d in list(range(1, 300)) + [(1 << i) + j for i in range(9, 31) for j in (-1, 0, 1)] + [(1 << 31) - 1]:
        assert loaded.wrong_quotients(ctypes.c_uint(d)) == 0, d
    look = loaded.lookup
    look.argtypes = [ctypes.POINTER(ctypes.c_int), ctypes.c_uint, ctypes.c_uint, ctypes.c_bool, ctypes.c_uint]
    table = (ctypes.c_int * 5)(5, -1, 9, 10, 1 << 30)
    assert [look(table, 5, 10, True, at) for at in range(5)] == [5, -1, 9, -1, -1]
    assert look(table, 5, 10, False, 0) == -1 and look(table, 2, 10, True, 2) == -1 and look(table, 5, 10, True, 0xffffffff) == -1


def test_refusals_of_the_entry_points():
    lib = runtime.load_library()
    longs = lambda *v: (ctypes.c_longlong * len(v))(*v)      # noqa: E731
    need = ctypes.c_ulonglong(0)
    good = (2, 3, 4, 2, 64, 16, 100, 200)
    assert lib.lego_hip_tree_attention_workspace_bytes(longs(*good), ctypes.byref(need)) == 0 and need.value > 0
    assert lib.lego_hip_tree_attention_workspace_bytes(longs(2, 3, 4, 2, 64, 16, 100, 8), ctypes.byref(need)) == 0 and need.value == 0
    bads = [tuple(0 if j == i else x for j, x in enumerate(good)) for i in range(8)] + [(2, 3, 4, 3, 64, 16, 100, 50), (2, 3, 4, 2, 60, 16, 100, 50), (2, 3, 4, 2, 136, 16, 100, 50),
            (2, 3, 4, 2, 64, 1 << 20, 100, 1 << 20), (1 << 20, 1 << 20, 4, 2, 64, 16, 100, 50), (1 << 20, 1, 64, 64, 64, 16, 100, 1 << 16)]
    for bad in bads:
        assert lib.lego_hip_tree_attention_workspace_bytes(longs(*bad), ctypes.byref(need)) == 1, bad
    at = [ctypes.c_void_p(4096 * (i + 1)) for i in range(12)]
    st = (768, 256, 64) + (384, 128, 64) * 2 + (2048, 128, 64) * 2 + (768, 256, 64, 9)

    def call(ptrs=at[:11], sizes=good, strides=st, scale=0.1, cap=0.0, element=1, ws=at[11], room=1 << 30):
        return lib.lego_hip_tree_attention(*ptrs, longs(*sizes), longs(*strides), scale, cap, element, ws, room, None)

    for i in range(8):      # q, k, v, the caches, out, pages, lengths: null alone
        assert call([None if j == i else x for j, x in enumerate(at[:11])]) == 1, i
        assert call([ctypes.c_void_p(4097) if j == i else x for j, x in enumerate(at[:11])]) == 1, i
    assert call([at[0], None, None] + at[3:11]) == 1      # a tree without drafts' keys
    assert call(at[:9] + [None, at[10]]) == 1              # positions without slopes
    assert call(scale=math.nan) == 1 and call(cap=-1.0) == 1 and call(cap=math.inf) == 1 and call(element=2) == 1
    assert call(ws=None) == 1 and call(room=64) == 1 and call(ws=ctypes.c_void_p(4097)) == 1
    assert call(strides=(768, 256, 60) + st[3:]) == 1 and call(strides=(-8,) + st[1:]) == 1 and call(strides=st[:18] + (-1,)) == 1
    assert call(strides=st[:9] + (1 << 34, 128, 64) + st[12:]) == 1      # over 64 GiB


@pytest.mark.gpu
def test_refusals():
    how = make([30, 100], 3, 4, 2, 64, 16, torch.bfloat16)
    slopes = torch.ones(4, device="cuda")
    for bad in (dict(k=None), dict(k=how["k"][:, :2]), dict(v=how["v"][..., :56]), dict(k_cache=how["k_cache"].half()), dict(k_cache=how["k_cache"][:, :, :1]), dict(v_cache=how["v_cache"][:-1]),
                dict(pages=how["pages"].long()), dict(pages=how["pages"][:1]), dict(pages=how["pages"][0]), dict(lengths=how["lengths"].cpu()), dict(lengths=how["lengths"][:1]),
                dict(tree=how["tree"].int()), dict(tree=how["tree"][:, :2]), dict(tree=how["tree"][:1]), dict(slopes=slopes), dict(slopes=slopes[:2], positions=how["pages"][:, :3]),
                dict(positions=torch.zeros(2, 3, dtype=torch.int32, device="cuda")), dict(softcap=-1.0), dict(scale=math.nan), dict(q=how["q"].float()), dict(q=how["q"][:, :, :3]),
                dict(k=None, v=None), dict(k_cache=how["k_cache"][..., 1:57], v_cache=how["v_cache"][..., 1:57], q=how["q"][..., :56], k=how["k"][..., :56], v=how["v"][..., :56])):
        with pytest.raises(ValueError):
            ops.tree_attention(**{**how, **bad})
