"""The attention operators of ``lego_amd.ops`` as cases that a timing harness runs: rotary positions, attention with its
gradient, and attention of drafted tokens over a paged cache, each beside its plain form in elementary torch operations.

``listed()`` names the sizes that stand for each operator; ``draw(rng)`` gives more cases of the same ranges, ``prepare`` makes
a case's inputs, ``run`` takes one pass through the operator (where ``own`` is true) or its plain form, and ``exact`` computes
the same from the definition in 64 bits.
"""
import math
import random

import torch

own = False

_DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # positions of one decoding step: 16 sequences, one token each, far into a context stretched to eight times its length
        {"name": "rotary_token", "op": "rotary", "dtype": "bf16", "b": 16, "t": 1, "hq": 32, "hk": 8, "d": 128, "part": 128,
         "interleaved": False, "stretch": 8.0, "far": 131072, "fused": False, "train": False},
        # queries and keys of a training step, both directions
        {"name": "rotary_train", "op": "rotary", "dtype": "bf16", "b": 4, "t": 4096, "hq": 32, "hk": 8, "d": 128, "part": 128,
         "interleaved": False, "stretch": 1.0, "far": 4096, "fused": False, "train": True},
        # interleaved pairs in part of a smaller head, queries and keys as slices of one fused projection, an odd length
        {"name": "rotary_part_fused", "op": "rotary", "dtype": "f16", "b": 2, "t": 2047, "hq": 16, "hk": 16, "d": 80, "part": 32,
         "interleaved": True, "stretch": 1.0, "far": 2047, "fused": True, "train": True},
        # a short prompt: what a launch costs
        {"name": "attention_short", "op": "attention", "dtype": "f16", "b": 4, "t": 77, "hq": 8, "hk": 8, "d": 64, "causal": True,
         "cap": 0.0, "slopes": False, "documents": 0, "prefix": False, "fused": True, "train": False},
        # a training step with capped scores, four query heads to a key head
        {"name": "attention_capped_train", "op": "attention", "dtype": "bf16", "b": 2, "t": 4096, "hq": 16, "hk": 4, "d": 128, "causal": True,
         "cap": 30.0, "slopes": False, "documents": 0, "prefix": False, "fused": False, "train": True},
        # a training step over documents packed into one long sequence
        {"name": "attention_documents_train", "op": "attention", "dtype": "bf16", "b": 1, "t": 8192, "hq": 16, "hk": 16, "d": 128, "causal": True,
         "cap": 0.0, "slopes": False, "documents": 7, "prefix": False, "fused": False, "train": True},
        # a training step with a bias by distance in place of positions: smaller heads, an odd length
        {"name": "attention_distance_train", "op": "attention", "dtype": "f16", "b": 3, "t": 1531, "hq": 12, "hk": 12, "d": 64, "causal": True,
         "cap": 0.0, "slopes": True, "documents": 0, "prefix": False, "fused": True, "train": True},
        # prefill of long prompts whose first part is seen from both sides
        {"name": "attention_prefix", "op": "attention", "dtype": "bf16", "b": 2, "t": 8192, "hq": 32, "hk": 8, "d": 128, "causal": True,
         "cap": 0.0, "slopes": False, "documents": 0, "prefix": True, "fused": False, "train": False},
        # the first token after a short prompt: what launches cost
        {"name": "tree_first_token", "op": "tree", "dtype": "f16", "b": 1, "t": 1, "hq": 16, "hk": 16, "d": 64, "page": 16,
         "shortest": 100, "longest": 100, "cap": 0.0, "slopes": False},
        # a decoding step of a batch of sequences of all lengths
        {"name": "tree_tokens", "op": "tree", "dtype": "bf16", "b": 32, "t": 1, "hq": 32, "hk": 8, "d": 128, "page": 16,
         "shortest": 37, "longest": 8192, "cap": 0.0, "slopes": False},
        # a verification step: trees of 48 drafted tokens
        {"name": "tree_drafts", "op": "tree", "dtype": "bf16", "b": 8, "t": 48, "hq": 32, "hk": 8, "d": 128, "page": 64,
         "shortest": 1021, "longest": 16384, "cap": 30.0, "slopes": False},
        # a few drafted tokens of one sequence far into a long context
        {"name": "tree_long", "op": "tree", "dtype": "f16", "b": 1, "t": 7, "hq": 16, "hk": 4, "d": 64, "page": 256,
         "shortest": 131000, "longest": 131000, "cap": 0.0, "slopes": True},
    ]


def _log(rng, lo, hi):
    """A whole number, its logarithm spread evenly."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    case = _any(rng)
    # no more work than the largest listed case of the operator has
    most = [work(c) for c in listed() if c["op"] == case["op"]]
    while any(work(case)[m] > max(w[m] for w in most) for m in ("bytes", "flops")):
        case |= {n: case[n] // 2 for n in (("shortest", "longest") if case["op"] == "tree" else ("t",))}
    return case


def _any(rng):
    op = rng.choice(("rotary", "attention", "attention", "tree"))
    dtype = rng.choice(("f16", "bf16"))
    hk, group = rng.choice((1, 2, 4, 8, 12, 16)), rng.choice((1, 1, 2, 4, 8))
    d = rng.choice((64, 64, 128, 128, 80, 96))
    if op == "rotary":
        tokens = _log(rng, 1, 16384)
        b = min(tokens, rng.choice((1, 1, 2, 4, 16)))
        t = max(1, tokens // b)
        part = rng.choice((d, d, d // 2, 32))
        return {"op": op, "dtype": dtype, "b": b, "t": t, "hq": hk * group, "hk": hk, "d": d, "part": part,
                "interleaved": rng.random() < 0.5, "stretch": rng.choice((1.0, 1.0, 4.0, 32.0)), "far": max(t, _log(rng, 64, 1 << 20)),
                "fused": rng.random() < 0.5, "train": rng.random() < 0.5}
    if op == "attention":
        hk = min(hk, 4) if group > 2 else hk
        t = _log(rng, 1, 8192)
        b = min(rng.choice((1, 2, 3, 8)), max(1, 16384 // t))
        mask = rng.choice(("", "", "documents", "prefix"))
        return {"op": op, "dtype": dtype, "b": b, "t": t, "hq": hk * group, "hk": hk, "d": d, "causal": mask == "prefix" or rng.random() < 0.8,
                "cap": rng.choice((0.0, 0.0, 30.0, 50.0)), "slopes": rng.random() < 0.3,
                "documents": rng.randint(2, 9) if mask == "documents" and t >= 64 else 0, "prefix": mask == "prefix",
                "fused": rng.random() < 0.5, "train": rng.random() < 0.6}
    longest = _log(rng, 16, 131072)
    b = max(1, min(_log(rng, 1, 64), (1 << 18) // longest))
    return {"op": op, "dtype": dtype, "b": b, "t": rng.choice((1, 1, 1, rng.randint(2, 8), rng.randint(9, 64))), "hq": hk * group, "hk": hk, "d": d,
            "page": rng.choice((16, 16, 32, 64, 128, 256)), "shortest": rng.randint(0, longest), "longest": longest,
            "cap": rng.choice((0.0, 0.0, 30.0)), "slopes": rng.random() < 0.25}


def _lengths(case):
    """The sequences' cached tokens: evenly from the shortest to the longest."""
    b, lo, hi = case["b"], case["shortest"], case["longest"]
    return [hi if b == 1 else lo + (hi - lo) * i // (b - 1) for i in range(b)]


def _documents(case):
    """Lengths of a sequence's documents, as 2 : 3 : 4 : ..."""
    n, t = case["documents"], case["t"]
    total = n * (n + 3) // 2
    cuts = [t * (i * (i + 3) // 2) // total for i in range(n + 1)]
    return [b - a for a, b in zip(cuts, cuts[1:])]


def _prefixes(case):
    """Tokens seen from both sides: evenly from an eighth to half of the sequence."""
    b, lo, hi = case["b"], case["t"] // 8, case["t"] // 2
    return [hi if b == 1 else lo + (hi - lo) * i // (b - 1) for i in range(b)]


def _slopes(heads):
    """A slope for each head, from 1/2 to 1/256."""
    return [2.0 ** (-1 - 7 * i / max(1, heads - 1)) for i in range(heads)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)
    dtype, op = _DTYPES[case["dtype"]], case["op"]
    b, t, hq, hk, d = (case[k] for k in ("b", "t", "hq", "hk", "d"))

    def randn(*shape, scale=1.0):
        return (scale * torch.randn(*shape, device="cuda", generator=g)).to(dtype)

    def ints(values):
        return torch.tensor(values, device="cuda", dtype=torch.int32)

    state = {"case": case}
    if op == "tree":
        lengths = _lengths(case)
        rng.shuffle(lengths)
        page = case["page"]
        width = max(1, -(-max(lengths) // page))
        count = sum(-(-n // page) for n in lengths) + 3      # of a pool that other sequences use as well
        order = list(range(count))
        rng.shuffle(order)
        rows = []
        for n in lengths:
            need = -(-n // page)
            rows.append(order[:need] + [0] * (width - need))
            order = order[need:]
        # a tree: every draft hangs below an earlier one, or below the last cached token
        tree = torch.zeros(b, t, t, dtype=torch.bool)
        depth = [[0] * t for _ in range(b)]
        for i in range(b):
            for j in range(t):
                parent = rng.randrange(max(-1, j - 6), j) if j else -1
                if parent >= 0:
                    tree[i, j] = tree[i, parent]
                    depth[i][j] = depth[i][parent] + 1
                tree[i, j, j] = True
        state |= {"q": randn(b, t, hq, d), "k": randn(b, t, hk, d), "v": randn(b, t, hk, d),
                  "k_cache": randn(count, page, hk, d), "v_cache": randn(count, page, hk, d), "pages": ints(rows), "lengths": ints(lengths),
                  "tree": tree.cuda() if t > 1 else None, "positions": None, "slopes": None}
        if case["slopes"]:
            state["slopes"] = torch.tensor(_slopes(hq), device="cuda")
            state["positions"] = ints([[n + x for x in depth[i]] for i, n in enumerate(lengths)])
        return state

    # queries, keys and values as tensors of their own or as slices of what one projection gives
    if case["fused"]:
        qkv = randn(b, t, hq + 2 * hk, d)
        state |= {"q": qkv[:, :, :hq], "k": qkv[:, :, hq:hq + hk], "v": qkv[:, :, hq + hk:]}
    else:
        state |= {"q": randn(b, t, hq, d), "k": randn(b, t, hk, d), "v": randn(b, t, hk, d)}
    if case["train"]:
        for name in ("q", "k", "v"):
            state[name] = state[name].detach().requires_grad_()
        state |= {"dq": randn(b, t, hq, d), "dk": randn(b, t, hk, d)}
    if op == "rotary":
        part, far = case["part"], case["far"]
        first = [rng.randint(0, far - t) for _ in range(b)]
        state["positions"] = ints([list(range(f, f + t)) for f in first])
        # what a program keeps: radians a position, slow ones divided by the stretch, fast ones kept, a ramp in between
        radians = 10000.0 ** (-torch.arange(0, part, 2, dtype=torch.float64) / part)
        turns = 4096 * radians / (2 * math.pi)
        keep = ((turns - 1) / 31).clamp(0, 1)
        state["frequencies"] = (radians * (keep + (1 - keep) / case["stretch"])).cuda()
        state["magnitude"] = 0.1 * math.log(case["stretch"]) + 1.0
        return state
    state["slopes"] = torch.tensor(_slopes(hq), device="cuda") if case["slopes"] else None
    state["documents"] = state["prefix"] = None
    if case["documents"]:
        ids = []
        for _ in range(b):
            lengths = _documents(case)
            rng.shuffle(lengths)
            ids.append([i for i, n in enumerate(lengths) for _ in range(n)])
        state["documents"] = ints(ids)
    if case["prefix"]:
        prefixes = _prefixes(case)
        rng.shuffle(prefixes)
        state["prefix"] = ints(prefixes)
    return state


def _rotate(x, cos, sin, part, interleaved):
    """Pairs of the first ``part`` elements turned, the others as they are, in 32 bits."""
    x = x.float()
    turned = x[..., :part]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        y = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = turned[..., :part // 2], turned[..., part // 2:]
        y = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((y, x[..., part:]), -1)


def _rotary(s):
    case = s["case"]
    if own:
        from lego_amd import ops
        q, k = ops.rotary(s["q"], s["k"], s["positions"], s["frequencies"], interleaved=case["interleaved"], magnitude=s["magnitude"])
        if not case["train"]:
            return q, k
        return (q.detach(), k.detach()) + torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
    dtype, shape = s["q"].dtype, (case["part"], case["interleaved"])
    angle = s["positions"].double()[:, :, None, None] * s["frequencies"]
    cos, sin = (s["magnitude"] * angle.cos()).float(), (s["magnitude"] * angle.sin()).float()
    out = tuple(_rotate(s[n].detach(), cos, sin, *shape).to(dtype) for n in ("q", "k"))
    if not case["train"]:
        return out
    return out + tuple(_rotate(s[n], cos, -sin, *shape).to(dtype) for n in ("dq", "dk"))


def _by_head(x, group=1):
    """``[batch, token, head, element]`` in 32 bits as ``[batch, head, token, element]``, each head ``group`` times."""
    return x.detach().float().transpose(1, 2).repeat_interleave(group, 1)


def _seen(s, tokens):
    """Which key each query sees, ``[batch or 1, 1, query, key]``."""
    case = s["case"]
    at = torch.arange(tokens, device="cuda")
    seen = torch.ones(1, 1, tokens, tokens, dtype=torch.bool, device="cuda")
    if case["causal"]:
        seen = (at <= at[:, None])[None, None]
        if s["prefix"] is not None:
            seen = seen | (at < s["prefix"][:, None, None, None])
    if s["documents"] is not None:
        ids = s["documents"]
        seen = seen & ((ids[:, None, :, None] == ids[:, None, None, :]) & (ids >= 0)[:, None, None, :])
    return seen


def _attention(s):
    case = s["case"]
    if own:
        from lego_amd import ops
        out = ops.attention(s["q"], s["k"], s["v"], causal=case["causal"], softcap=case["cap"], slopes=s["slopes"], documents=s["documents"], prefix=s["prefix"])
        if not case["train"]:
            return out
        return (out.detach(),) + torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["dq"])
    dtype, group, tokens, cap = s["q"].dtype, case["hq"] // case["hk"], case["t"], case["cap"]
    q, k, v = _by_head(s["q"]), _by_head(s["k"], group), _by_head(s["v"], group)
    scale = 1 / math.sqrt(case["d"])
    scores = (q @ k.transpose(2, 3)) * scale
    if cap:
        capped = torch.tanh(scores / cap)
        scores = cap * capped
    if s["slopes"] is not None:
        at = torch.arange(tokens, device="cuda")
        scores = scores - s["slopes"][:, None, None] * (at[:, None] - at).abs()
    scores = torch.where(_seen(s, tokens), scores, -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    out = p @ v
    rounded = out.transpose(1, 2).to(dtype)
    if not case["train"]:
        return rounded
    do = _by_head(s["dq"])
    dv = p.transpose(2, 3) @ do
    ds = p * (do @ v.transpose(2, 3) - (do * out).sum(-1, keepdim=True))
    if cap:
        ds = ds * (1 - capped * capped)
    dq, dk = ds @ k * scale, ds.transpose(2, 3) @ q * scale
    dk, dv = (x.unflatten(1, (case["hk"], group)).sum(2) for x in (dk, dv))
    return (rounded,) + tuple(x.transpose(1, 2).to(dtype) for x in (dq, dk, dv))


def _tree(s):
    case = s["case"]
    if own:
        from lego_amd import ops
        return ops.tree_attention(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["pages"], s["lengths"], tree=s["tree"],
                                  softcap=case["cap"], slopes=s["slopes"], positions=s["positions"])
    dtype, group, t = s["q"].dtype, case["hq"] // case["hk"], case["t"]
    # the cached tokens of every sequence side by side, its drafts behind them
    cached = [s[n][s["pages"].long()].flatten(1, 2) for n in ("k_cache", "v_cache")]
    room = cached[0].shape[1]
    k, v = (_by_head(torch.cat((c, s[n]), 1), group) for c, n in zip(cached, ("k", "v")))
    at = torch.arange(room, device="cuda")
    seen = (at < s["lengths"][:, None])[:, None, :].expand(-1, t, -1)
    tree = s["tree"] if s["tree"] is not None else torch.ones(case["b"], 1, 1, dtype=torch.bool, device="cuda")
    seen = torch.cat((seen, tree), 2)[:, None]
    scores = (_by_head(s["q"]) @ k.transpose(2, 3)) / math.sqrt(case["d"])
    if case["cap"]:
        scores = case["cap"] * torch.tanh(scores / case["cap"])
    if s["slopes"] is not None:
        place = torch.cat((at.expand(case["b"], -1), s["positions"]), 1)
        scores = scores - s["slopes"][:, None, None] * (s["positions"][:, :, None] - place[:, None, :]).abs()[:, None]
    scores = torch.where(seen, scores, -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    return ((p / p.sum(-1, keepdim=True)) @ v).transpose(1, 2).to(dtype)


_RUN = {"rotary": _rotary, "attention": _attention, "tree": _tree}


def run(state):
    return _RUN[state["case"]["op"]](state)


def _pairs(case):
    """Pairs of a query and a key that it sees, over the batch, for one query head."""
    b, t = case["b"], case["t"]
    spans = _documents(case) if case["documents"] else [t]
    pairs = b * sum(n * (n + 1) // 2 if case["causal"] else n * n for n in spans)
    if case["prefix"]:
        pairs += sum(p * (p - 1) // 2 for p in _prefixes(case))
    return pairs


def work(case):
    b, t, hq, hk, d = (case[k] for k in ("b", "t", "hq", "hk", "d"))
    if case["op"] == "rotary":
        # queries and keys in and out, in both directions; three operations an element turned
        n, passes = b * t * (hq + hk), 2 if case["train"] else 1
        return {"bytes": passes * (2 * n * d * 2 + 4 * b * t), "flops": passes * 3 * n * case["part"]}
    if case["op"] == "attention":
        # forward: q, k, v in, out out, two products; backward: q, k, v, out and its gradient in, three gradients out, five products
        q, kv = 2 * b * t * hq * d, 2 * b * t * hk * d
        pairs = _pairs(case) * hq
        return {"bytes": 2 * q + 2 * kv + (4 * q + 4 * kv if case["train"] else 0), "flops": pairs * d * (14 if case["train"] else 4)}
    keys = sum(_lengths(case))
    return {"bytes": 2 * (2 * b * t * hq * d + 2 * b * t * hk * d + 2 * keys * hk * d), "flops": 4 * d * hq * t * (keys + b * (t + 1) // 2)}


def _exact_rotary(s):
    case = s["case"]
    # each pair as a complex number times magnitude * exp(i angle)
    part = case["part"]
    turn = torch.polar(torch.full((), s["magnitude"], dtype=torch.float64, device="cuda"), s["positions"].double().unsqueeze(-1) * s["frequencies"]).unsqueeze(2)

    def through(x, turn):
        x = x.detach().double()
        head, rest = x.split((part, case["d"] - part), -1)
        pairs = head.unflatten(-1, (-1, 2)) if case["interleaved"] else head.unflatten(-1, (2, -1)).transpose(-1, -2)
        y = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        return torch.cat((y.flatten(-2) if case["interleaved"] else y.transpose(-1, -2).flatten(-2), rest), -1)

    out = (through(s["q"], turn), through(s["k"], turn))
    return out + (through(s["dq"], turn.conj()), through(s["dk"], turn.conj())) if case["train"] else out


def _exact_attention(s):
    case = s["case"]
    b, t, hq, hk, cap = (case[k] for k in ("b", "t", "hq", "hk", "cap"))
    q, k, v = (s[n].detach().double() for n in ("q", "k", "v"))
    out, scale = torch.zeros_like(q), case["d"] ** -0.5
    grads = [torch.zeros_like(x) for x in (q, k, v)]
    rows, cols = torch.meshgrid(torch.arange(t, device="cuda"), torch.arange(t, device="cuda"), indexing="ij")
    for i in range(b):
        hidden = torch.zeros(t, t, dtype=torch.bool, device="cuda")
        if case["causal"]:
            hidden = cols > rows
            if case["prefix"]:
                hidden &= cols >= int(s["prefix"][i])
        if case["documents"]:
            hidden = hidden | (s["documents"][i][rows] != s["documents"][i][cols])
        for h in range(hq):
            g = h // (hq // hk)
            x = scale * torch.mm(q[i, :, h], k[i, :, g].t())
            slope = 1.0
            if cap:
                x = cap * torch.tanh(x / cap)
                slope = 1 - (x / cap) ** 2
            if case["slopes"]:
                x = x - s["slopes"][h].double() * (rows - cols).abs()
            p = torch.softmax(x.masked_fill(hidden, -math.inf), 1)
            out[i, :, h] = torch.mm(p, v[i, :, g])
            if case["train"]:
                do = s["dq"][i, :, h].double()
                dp = torch.mm(do, v[i, :, g].t())
                ds = scale * slope * p * (dp - (p * dp).sum(1, keepdim=True))
                grads[0][i, :, h] = torch.mm(ds, k[i, :, g])
                grads[1][i, :, g] += torch.mm(ds.t(), q[i, :, h])
                grads[2][i, :, g] += torch.mm(p.t(), do)
    return (out, *grads) if case["train"] else out


def _exact_tree(s):
    case = s["case"]
    out = torch.zeros_like(s["q"], dtype=torch.float64)
    group, t = case["hq"] // case["hk"], case["t"]
    for i, n in enumerate(s["lengths"].tolist()):
        used = s["pages"][i, :-(-n // case["page"])].long()
        k, v = (torch.cat((s[c][used].flatten(0, 1)[:n], s[x][i])).double() for c, x in (("k_cache", "k"), ("v_cache", "v")))
        hidden = torch.zeros(t, n + t, dtype=torch.bool, device="cuda")
        if s["tree"] is not None:
            hidden[:, n:] = ~s["tree"][i]
        for h in range(case["hq"]):
            x = torch.mv(k[:, h // group], s["q"][i, 0, h].double())[None] if t == 1 else s["q"][i, :, h].double() @ k[:, h // group].t()
            x = x * case["d"] ** -0.5
            if case["cap"]:
                x = case["cap"] * torch.tanh(x / case["cap"])
            if case["slopes"]:
                place = torch.cat((torch.arange(n, device="cuda"), s["positions"][i].long()))
                x = x - s["slopes"][h].double() * (s["positions"][i].long()[:, None] - place).abs()
            out[i, :, h] = torch.softmax(x.masked_fill(hidden, -math.inf), 1) @ v[:, h // group]
    return out


def exact(case, seed):
    """What ``run`` returns for these inputs, from the operators' definitions in 64 bits."""
    s = prepare(case, seed)
    return {"rotary": _exact_rotary, "attention": _exact_attention, "tree": _exact_tree}[case["op"]](s)
