"""Operators of speculative decoding over the 4-bit cache, as a serving program calls them.

tree    attention.attention_fp4_tree: attention of a tree of drafted tokens (each row sees the
        context and its own ancestors) over the paged cache of 4-bit values.
probs   sampling.token_probs: a vocabulary's probabilities of logits, with a temperature a row.
verify  sampling.verify_drafts: which drafted tokens stand, by the target's probabilities and
        given random numbers, and the token that follows them.
move    attention.move_fp4: the accepted rows of each tree go to consecutive rows of the cache;
        attention.unpack_fp4 then reads all of the tree's rows back as BF16.

The plain forms compute in FP32 with elementary torch operations and round once at the end; which
drafts stand is computed in 64 bits, since whole vocabularies are summed and compared there.
"""

import math
import os
import sys

import torch

own = False

DEVICE = "cuda"
BLOCK = 32  # channels that share one scale

# (query heads, key heads, channels of a head)
HEADS = [(32, 8, 128), (24, 4, 256), (40, 8, 128), (64, 8, 128), (16, 16, 64), (14, 2, 64), (28, 4, 128)]


def _heads(i):
    hq, hkv, dim = HEADS[i]
    return dict(hq=hq, hkv=hkv, dim=dim)


def listed():
    return [
        # One conversation, seven drafted tokens and the certain one: the smallest attention call.
        dict(name="tree_s1_n8_c600_32x8x128", kind="tree", **_heads(0), seqs=1, nodes=8, c_min=600, c_max=600, page=16, window=0),
        # A batch of ragged conversations with small trees.
        dict(name="tree_s16_n16_c8000_32x8x128", kind="tree", **_heads(0), seqs=16, nodes=16, c_min=500, c_max=8000, page=16, window=0),
        # Wide trees, as a drafter with many heads gives: the most operations.
        dict(name="tree_s8_n64_c16000_40x8x128", kind="tree", **_heads(2), seqs=8, nodes=64, c_min=4000, c_max=16000, page=64, window=0),
        # Long documents: the most bytes.
        dict(name="tree_s4_n26_c131071_24x4x256", kind="tree", **_heads(1), seqs=4, nodes=26, c_min=40000, c_max=131071, page=64, window=0),
        # A full batch, a ragged number of drafts, of which each sees 1024 tokens.
        dict(name="tree_s32_n11_c9000_28x4x128_w1024", kind="tree", **_heads(6), seqs=32, nodes=11, c_min=300, c_max=9000, page=32, window=1024),
        # The next token of one conversation: the smallest call.
        dict(name="probs_t1_v32000_bf16", kind="probs", tokens=1, vocab=32000, bits=16),
        # A vocabulary of odd size, FP32 logits of a small batch of trees.
        dict(name="probs_t52_v50001_fp32", kind="probs", tokens=52, vocab=50001, bits=32),
        # All rows of a batch of trees.
        dict(name="probs_t512_v152000_bf16", kind="probs", tokens=512, vocab=152000, bits=16),
        # One conversation, a tree of certain choices (the drafter's best ones).
        dict(name="verify_s1_n26_v32000_tree", kind="verify", seqs=1, nodes=26, vocab=32000, tree=True, draft=False),
        # A batch of chains, eight tokens each, drawn from a drafter's probabilities.
        dict(name="verify_s64_n9_v152000_chain_drawn", kind="verify", seqs=64, nodes=9, vocab=152000, tree=False, draft=True),
        # Trees whose children were drawn from the drafter's probabilities.
        dict(name="verify_s16_n32_v128000_tree_drawn", kind="verify", seqs=16, nodes=32, vocab=128000, tree=True, draft=True),
        # What a batch of trees leaves in one layer's cache.
        dict(name="move_s32_n26_40x8x128", kind="move", **_heads(2), seqs=32, nodes=26, page=64),
    ]


def _log_int(rng, low, high):
    """An integer in [low, high], spread evenly over the logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49))))))


def draw(rng):
    kind = rng.choice(["tree", "tree", "tree", "probs", "verify", "verify", "move"])
    if kind == "probs":
        tokens, bits = _log_int(rng, 1, 700), rng.choice([16, 16, 32])
        vocab = min(_log_int(rng, 1000, 200000), 512 * 152000 * 6 // (tokens * (bits // 8 + 4)))
        return dict(kind=kind, tokens=tokens, vocab=vocab, bits=bits)
    if kind == "verify":
        seqs, nodes = _log_int(rng, 1, 64), _log_int(rng, 1, 64)
        vocab = max(500, min(_log_int(rng, 1000, 200000), 64 * 9 * 152000 // (seqs * nodes)))
        return dict(kind=kind, seqs=seqs, nodes=nodes, vocab=vocab, tree=rng.random() < 0.6, draft=rng.random() < 0.5)
    heads = _heads(rng.randrange(len(HEADS)))
    if kind == "move":
        return dict(kind=kind, **heads, seqs=_log_int(rng, 1, 32), nodes=rng.randint(2, 26), page=rng.choice([16, 32, 64, 128]))
    seqs, nodes = _log_int(rng, 1, 32), _log_int(rng, 2, 64)
    c = nodes + _log_int(rng, 60, 130000)
    # no more than the largest listed cases: products of wide trees, bytes of long contexts
    most = min(8 * 40 * 64 * 16000 * 128 / (seqs * heads["hq"] * nodes * heads["dim"]),
               4 * 4 * 256 * 131071 / (seqs * heads["hkv"] * heads["dim"]))
    c = max(nodes + 1, min(c, int(most)))
    return dict(kind=kind, **heads, seqs=seqs, nodes=nodes, c_min=max(nodes, c // 4), c_max=c, page=rng.choice([16, 32, 64, 128]),
                window=rng.choice([0, 0, 0, 40, 1024]))


# ---- sizes of a case, the same for every seed -------------------------------------------


def _spread(count, low, high):
    """`count` lengths between low and high, the first the longest, evenly spread."""
    return [high - int((high - low) * math.modf(i * 0.6180339887498949)[0]) for i in range(count)]


def work(case):
    if case["kind"] == "probs":
        values = case["tokens"] * case["vocab"]
        return {"bytes": values * (case["bits"] // 8 + 4) + case["tokens"] * 4, "flops": values * 5}
    if case["kind"] == "verify":
        rows, seqs, each = case["seqs"] * case["nodes"], case["seqs"], 2 if case["draft"] else 1
        # tokens, parents, numbers, path; the row at which each sequence ends, and one value a tested row
        return {"bytes": rows * (8 + 4 + 4 + 4 + 4 * each) + seqs * (4 + 4 + 8 + 4 * each * case["vocab"]),
                "flops": seqs * case["vocab"] * (3 if case["draft"] else 1)}
    hq, hkv, dim = case["hq"], case["hkv"], case["dim"]
    packed = dim // 2 + dim // BLOCK  # bytes of one head of one token
    if case["kind"] == "move":
        rows, moved = case["seqs"] * case["nodes"], case["seqs"] * len(_jumps(case["nodes"]))
        return {"bytes": rows * 12 + moved * 2 * hkv * packed * 2 + rows * (8 + 2 * hkv * (packed + 2 * dim)),
                "flops": rows * 2 * hkv * dim}
    read = pairs = 0
    n, window = case["nodes"], case["window"] or 1 << 30
    for c in _spread(case["seqs"], case["c_min"], case["c_max"]):
        harmonic = 0.0  # the expected depth of row i in these trees
        for i in range(n):
            harmonic += 1 / i if i else 0
            pairs += min(window, c - n + 1 + harmonic)
        read += min(c, window + n)
    return {"bytes": int(read * 2 * hkv * packed + case["seqs"] * n * (hq * (dim * 4 + 4) + 4)), "flops": int(4 * pairs * hq * dim)}


# ---- inputs -----------------------------------------------------------------------------


def _fp4_codes(x):
    """FP32 [..., dim] -> E2M1 codes of two channels a byte and E8M0 scale bytes: the scale is
    the smallest 2^e with amax <= 7 * 2^e, ties go to the even code."""
    x = x.unflatten(-1, (-1, BLOCK))
    mant, exp = torch.frexp(x.abs().amax(-1, keepdim=True))
    e = (exp - 3 + (mant > 0.875)).clamp(min=-125)
    y = x * ((127 - e) << 23).view(torch.float32)
    a = y.abs()
    code = ((a > 0.25).byte() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5)
            + torch.signbit(y).byte() * 8)
    code = code.flatten(-2)
    return code[..., 0::2] + code[..., 1::2] * 16, (e.squeeze(-1) + 127).byte()


_E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _fp4_values(codes, scales, dtype=torch.float32):
    """The values that E2M1 codes and E8M0 scale bytes stand for."""
    one = torch.tensor(_E2M1 + [-v for v in _E2M1], dtype=dtype, device=codes.device)
    pair = torch.stack([one.repeat(16), one.repeat_interleave(16)], 1)  # of a byte: low half first
    scale = (scales.int() << 23).view(torch.float32).to(dtype)
    values = pair[codes.int()].flatten(-2)
    return (values.unflatten(-1, (-1, BLOCK)) * scale.unsqueeze(-1)).flatten(-2)


def _filled_cache(pages, case, gen):
    """A cache of random keys and values whose channels differ in size, as trained ones do."""
    hkv, page, dim = case["hkv"], case["page"], case["dim"]
    cache = [torch.zeros(pages, hkv, page, dim // n, dtype=torch.uint8, device=DEVICE) for n in (2, BLOCK, 2, BLOCK)]
    gain = torch.exp(0.5 * torch.randn(2, hkv, 1, dim, device=DEVICE, generator=gen))
    step = max(1, (1 << 26) // (hkv * page * dim))
    for first in range(0, pages, step):
        n = min(step, pages - first)
        for i in range(2):
            x = torch.randn(n, hkv, page, dim, device=DEVICE, generator=gen) * gain[i]
            cache[2 * i][first:first + n], cache[2 * i + 1][first:first + n] = _fp4_codes(x)
    return cache


def _trees(seqs, nodes, gen):
    """INT32 parents [seqs * nodes]: a row's parent is any row before it."""
    u = torch.rand(seqs, nodes, device=DEVICE, generator=gen)
    i = torch.arange(nodes, device=DEVICE)
    return torch.minimum((u * i).int(), (i - 1).int()).flatten()  # -1 for the first row


def _starts(seqs, nodes):
    return torch.arange(0, (seqs + 1) * nodes, nodes, dtype=torch.int32, device=DEVICE)


def _jumps(nodes):
    """Rows that an accepted path of a few rows takes from further back."""
    length = min(nodes, 2 + nodes // 5)
    return [i for i in range(length) if i >= (length + 1) // 2 and length + (i - length // 2) * 2 + 1 < nodes]


def prepare(case, seed):
    gen = torch.Generator(DEVICE).manual_seed(seed)
    s = {"case": case}
    if case["kind"] == "probs":
        t, v = case["tokens"], case["vocab"]
        # a few tokens lead, most follow far behind
        logits = -1.5 * torch.log(torch.rand(t, v, device=DEVICE, generator=gen).clamp_(min=2.0 ** -24))
        s["logits"] = logits if case["bits"] == 32 else logits.bfloat16()
        # sampled rows, and greedy ones among them
        warm = 0.5 + torch.rand(t, device=DEVICE, generator=gen)
        s["temperature"] = torch.where(torch.rand(t, device=DEVICE, generator=gen) < 0.1, 0.0, warm)
        s["probs"] = torch.empty(t, v, device=DEVICE)
        s["workspace"] = torch.empty(1 << 18, device=DEVICE)
        return s
    seqs, nodes = case["seqs"], case["nodes"]
    rows = seqs * nodes
    s["q_starts"] = _starts(seqs, nodes)
    if case["kind"] == "verify":
        v = case["vocab"]
        s["parents"] = _trees(seqs, nodes, gen) if case["tree"] else None
        logits = -1.3 * torch.log(torch.rand(rows, v, device=DEVICE, generator=gen).clamp_(min=2.0 ** -24))
        guess = logits + 0.7 * torch.randn(rows, v, device=DEVICE, generator=gen)
        s["target"] = torch.softmax(logits, -1)
        guess = torch.softmax(guess, -1)
        at = torch.arange(rows, device=DEVICE)
        parent = at - 1 if s["parents"] is None else at // nodes * nodes + s["parents"]
        # each row's token is drawn from what the drafter gave its parent
        race = torch.empty(rows, v, device=DEVICE).exponential_(generator=gen)
        s["tokens"] = (guess[parent.clamp(min=0)] / race).argmax(-1)
        s["draft"] = guess if case["draft"] else None
        s["uniforms"] = torch.rand(rows, device=DEVICE, generator=gen)
        s["path"] = torch.empty(rows, dtype=torch.int32, device=DEVICE)
        s["accepted"] = torch.empty(seqs, dtype=torch.int32, device=DEVICE)
        s["next"] = torch.empty(seqs, dtype=torch.int64, device=DEVICE)
        s["workspace"] = torch.empty(1 << 18, device=DEVICE)
        return s
    hq, hkv, dim, page = case["hq"], case["hkv"], case["dim"], case["page"]
    if case["kind"] == "move":
        # each sequence's rows lie in two pages of its own, from some row of the first on
        used = 1 + (nodes + page - 1) // page
        pages = seqs * used + 3
        s["cache"] = _filled_cache(pages, case, gen)
        order = torch.randperm(pages, device=DEVICE, generator=gen)[:seqs * used].view(seqs, used)
        at = torch.randint(0, page, (seqs, 1), device=DEVICE, generator=gen) + torch.arange(nodes, device=DEVICE)
        s["slots"] = (order.gather(1, at // page) * page + at % page).flatten()
        # the first accepted rows are where they belong, the others come from behind the path
        length, jumps = min(nodes, 2 + nodes // 5), _jumps(nodes)
        path = torch.full((seqs, nodes), -1, dtype=torch.int32, device=DEVICE)
        path[:, :length] = torch.arange(length, device=DEVICE)
        step = torch.randint(0, 2, (seqs, 1), device=DEVICE, generator=gen)
        for i in jumps:
            path[:, i] = (length + (i - length // 2) * 2 + 1 - step[:, 0]).int()
        s["rows"] = path.flatten()
        s["k_values"], s["v_values"] = (torch.empty(rows, hkv, dim, dtype=torch.bfloat16, device=DEVICE) for _ in "kv")
        return s
    cs = _spread(seqs, case["c_min"], case["c_max"])
    used = [(c + page - 1) // page for c in cs]
    pages = sum(used) + max(2, sum(used) // 16)
    s["cache"] = _filled_cache(pages, case, gen)
    order = torch.randperm(pages, device=DEVICE, generator=gen).int()
    width = max(used)
    ends = torch.tensor(used, device=DEVICE).cumsum(0)
    col = torch.arange(width, device=DEVICE)
    start = (ends - torch.tensor(used, device=DEVICE))[:, None]
    s["page_table"] = torch.where(start + col < ends[:, None], order[(start + col).clamp(max=pages - 1)], -1)
    s["context_lens"] = torch.tensor(cs, dtype=torch.int32, device=DEVICE)
    s["parents"] = _trees(seqs, nodes, gen)
    # rows of the projected tokens' buffer; scores of a few units, as trained heads have
    qkv = 2 * torch.randn(rows, (hq + 2 * hkv) * dim, device=DEVICE, generator=gen).bfloat16()
    s["q"] = qkv[:, :hq * dim].unflatten(1, (hq, dim))
    s["scale"] = dim ** -0.5
    s["out"] = torch.empty(rows, hq, dim, dtype=torch.bfloat16, device=DEVICE)
    s["lse"] = torch.empty(rows, hq, dtype=torch.float32, device=DEVICE)
    s["workspace"] = torch.empty(65536, dim + 2, dtype=torch.float32, device=DEVICE)
    return s


# ---- the operators ----------------------------------------------------------------------


def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    path = os.path.join(os.getcwd(), "consumer-int8-kernels_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from consumer_int8 import attention, sampling

    case = s["case"]
    if case["kind"] == "tree":
        attention.attention_fp4_tree(s["q"], *s["cache"], s["page_table"], s["context_lens"], s["q_starts"], s["parents"],
                                     s["workspace"], s["out"], s["lse"], s["scale"], case["nodes"], case["window"])
        return {"out": s["out"], "lse": s["lse"]}
    if case["kind"] == "probs":
        sampling.token_probs(s["logits"], s["temperature"], s["workspace"], s["probs"])
        return {"probs": s["probs"]}
    if case["kind"] == "verify":
        sampling.verify_drafts(s["target"], s["draft"], s["tokens"], s["parents"], s["q_starts"], s["uniforms"],
                               s["workspace"], s["path"], s["accepted"], s["next"])
        return {"path": s["path"], "accepted": s["accepted"], "next": s["next"]}
    attention.move_fp4(*s["cache"], s["rows"], s["slots"], s["q_starts"])
    attention.unpack_fp4(*s["cache"], s["slots"], s["k_values"], s["v_values"])
    return {"k": s["k_values"], "v": s["v_values"]}


def _run_plain(s):
    return {"tree": _plain_tree, "probs": _plain_probs, "verify": _plain_verify, "move": _plain_move}[s["case"]["kind"]](s)


def _ancestors(parents):
    """Parents [S, N] -> [S, N, N], whether row i is or descends from row j: powers of the parent relation."""
    n = parents.shape[1]
    i = torch.arange(n, device=DEVICE)
    reach = (parents[:, :, None] == i) | (i[:, None] == i)
    steps = reach.float()
    for _ in range(max(1, n - 1).bit_length()):  # twice as far each time
        steps = (torch.matmul(steps, steps) > 0).float()
    return steps > 0


def _plain_tree(s):
    case = s["case"]
    hq, hkv, n, seqs = case["hq"], case["hkv"], case["nodes"], case["seqs"]
    group, most_c, window, lens = hq // hkv, case["c_max"], case["window"], s["context_lens"]

    def gathered(codes, scales):  # [S, Hkv, C, dim]
        at = s["page_table"].clamp(min=0)
        c, e = (x[at].transpose(1, 2).flatten(2, 3)[:, :, :most_c] for x in (codes, scales))
        return _fp4_values(c, e)

    above = _ancestors(s["parents"].view(seqs, n))
    depth = above.sum(-1) - 1
    first = (lens - n)[:, None]                                                # the tree's first token
    at = torch.arange(most_c, device=DEVICE)
    node = at - first                                                          # [S, C], the row that a token is
    in_tree = (node >= 0) & (node < n)
    node = node.clamp(0, n - 1)
    seen = torch.where(in_tree[:, None], above.gather(2, node[:, None].expand(-1, n, -1)), (at < first)[:, None])
    if window:
        position = torch.where(in_tree, first + depth.gather(1, node), at)
        seen = seen & (position[:, None] > (first + depth)[:, :, None] - window)
    keys = gathered(*s["cache"][:2])
    q = s["q"].float().view(seqs, n, hkv, group, -1).permute(0, 2, 1, 3, 4).flatten(2, 3)  # [S, Hkv, N * group, dim]
    scores = torch.matmul(q, keys.transpose(-1, -2)) * s["scale"]
    del keys
    scores = torch.where(seen.repeat_interleave(group, 1)[:, None], scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - top)
    del scores
    total = p.sum(-1, keepdim=True)
    values = torch.where((at < lens[:, None])[:, None, :, None], gathered(*s["cache"][2:]), 0)
    out = torch.matmul(p, values) / total
    lse = torch.log(total) + top
    out, lse = (x.unflatten(2, (n, group)).permute(0, 2, 1, 3, 4).flatten(0, 1).flatten(1, 2) for x in (out, lse))
    return {"out": out.bfloat16(), "lse": lse.squeeze(-1)}


def _plain_probs(s):
    x, t = s["logits"].float(), s["temperature"][:, None]
    top = x.amax(-1, keepdim=True)
    e = torch.exp((x - top) / torch.where(t == 0, 1.0, t))
    drawn = e / e.sum(-1, keepdim=True)
    index = torch.arange(x.shape[1], device=DEVICE)
    best = torch.where(x == top, index, x.shape[1]).amin(-1, keepdim=True)
    return {"probs": torch.where(t == 0, (index == best).float(), drawn)}


def _plain_verify(s):
    case = s["case"]
    seqs, n, v = case["seqs"], case["nodes"], case["vocab"]
    target = s["target"].view(seqs, n, v)
    draft = None if s["draft"] is None else s["draft"].view(seqs, n, v)
    tokens, u = s["tokens"].view(seqs, n), s["uniforms"].view(seqs, n).double()
    every = torch.arange(seqs, device=DEVICE)
    parents = torch.arange(-1, n - 1, device=DEVICE).expand(seqs, n) if s["parents"] is None else s["parents"].view(seqs, n)
    node = torch.zeros(seqs, dtype=torch.int64, device=DEVICE)
    accepted = torch.ones(seqs, dtype=torch.int64, device=DEVICE)
    path = torch.full((seqs, n), -1, dtype=torch.int64, device=DEVICE)
    path[:, 0] = 0
    weights = target[:, 0].double()  # of what the tokens after `node` are drawn from
    total = torch.ones(seqs, dtype=torch.float64, device=DEVICE)
    taken = torch.zeros(seqs, dtype=torch.float64, device=DEVICE)
    # Rows in order: a row's children come after it, in the order in which they are tried.
    for i in range(1, n):
        tried = parents[:, i] == node
        x = tokens[:, i]
        w = weights.gather(1, x[:, None])[:, 0]
        chance = total if draft is None else total * draft[every, node, x].double()
        stands = tried & (u[:, i] * chance < w)
        fails = tried & ~stands
        if draft is None:
            weights = weights.scatter(1, x[:, None], torch.where(fails, 0.0, w)[:, None])
            total = torch.where(fails, total - w, total)
        else:
            taken = torch.where(fails, taken + total, taken)
            left = (target[every, node].double() - taken[:, None] * draft[every, node].double()).clamp(min=0)
            weights = torch.where(fails[:, None], left, weights)
            total = torch.where(fails, left.sum(-1), total)
        node = torch.where(stands, i, node)
        path[every, accepted.clamp(max=n - 1)] = torch.where(stands, i, path[every, accepted.clamp(max=n - 1)])
        accepted = accepted + stands.long()
        weights = torch.where(stands[:, None], target[:, i].double(), weights)
        total = torch.where(stands, 1.0, total)
        taken = torch.where(stands, 0.0, taken)
    weights = torch.where((weights > 0).any(-1, keepdim=True), weights, target[every, node].double())
    sums = weights.cumsum(-1)
    following = (sums > u[:, :1] * sums[:, -1:]).int().argmax(-1)
    return {"path": path.flatten().int(), "accepted": accepted.int(), "next": following}


def _plain_move(s):
    case = s["case"]
    n, page = case["nodes"], case["page"]
    path, slots = s["rows"].view(-1, n).long(), s["slots"].view(-1, n)
    moved = path > torch.arange(n, device=DEVICE)
    source = torch.where(moved, slots.gather(1, path.clamp(min=0)), slots).flatten()
    to = slots.flatten()

    def rows_of(x, at):
        return x[at // page, :, at % page]

    for x in s["cache"]:
        x[to // page, :, to % page] = rows_of(x, source)
    (k, ks), (v, vs) = s["cache"][:2], s["cache"][2:]
    return {"k": _fp4_values(rows_of(k, to), rows_of(ks, to)).bfloat16(),
            "v": _fp4_values(rows_of(v, to), rows_of(vs, to)).bfloat16()}


# ---- the same from the definitions, in 64 bits --------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    n = case.get("nodes")
    if case["kind"] == "verify":
        path, accepted, following = [], [], []
        tokens, numbers = s["tokens"].tolist(), s["uniforms"].tolist()
        parents = list(range(-1, n - 1)) * case["seqs"] if s["parents"] is None else s["parents"].tolist()
        for first in range(0, case["seqs"] * n, n):
            chain, node, left = [0], 0, s["target"][first].double()
            left = left / left.sum()
            for i in range(1, n):
                if parents[first + i] != node:
                    continue
                x = tokens[first + i]
                if s["draft"] is None:  # a certain choice
                    guess = torch.zeros_like(left)
                    guess[x] = 1
                else:
                    guess = s["draft"][first + node].double()
                if numbers[first + i] * guess[x].item() < left[x].item():
                    chain.append(i)
                    node, left = i, s["target"][first + i].double()
                else:
                    left = (left - guess).clamp(min=0)
                left = left / left.sum()
            path += chain + [-1] * (n - len(chain))
            accepted.append(len(chain))
            following.append(int((left.cumsum(0) > numbers[first]).nonzero()[0, 0]))
        return {"path": torch.tensor(path, dtype=torch.int32, device=DEVICE),
                "accepted": torch.tensor(accepted, dtype=torch.int32, device=DEVICE),
                "next": torch.tensor(following, device=DEVICE)}
    if case["kind"] == "probs":
        rows = []
        for x, t in zip(s["logits"].double(), s["temperature"].double().tolist()):
            if t == 0:
                one = torch.zeros_like(x)
                one[(x == x.max()).nonzero()[0, 0]] = 1
                rows.append(one)
            else:
                rows.append(torch.softmax(x / t, -1))
        return {"probs": torch.stack(rows)}
    page = case["page"]
    if case["kind"] == "move":
        path, slots = s["rows"].tolist(), s["slots"].tolist()
        source = list(slots)
        for i, row in enumerate(path):
            if row > i % n:
                source[i] = slots[i // n * n + row]
        at = torch.tensor(source, device=DEVICE)
        return {name: _fp4_values(s["cache"][j][at // page, :, at % page], s["cache"][j + 1][at // page, :, at % page],
                                  torch.float64) for name, j in (("k", 0), ("v", 2))}
    hq, hkv, window = case["hq"], case["hkv"], case["window"] or 1 << 30
    group, parents = hq // hkv, s["parents"].tolist()
    out = torch.empty(case["seqs"] * n, hq, case["dim"], dtype=torch.float64, device=DEVICE)
    lse = torch.empty(case["seqs"] * n, hq, dtype=torch.float64, device=DEVICE)
    for i, c in enumerate(_spread(case["seqs"], case["c_min"], case["c_max"])):
        hidden = torch.zeros(n, 1, c, dtype=torch.bool)
        for row in range(n):
            chain = [row]
            while parents[i * n + chain[-1]] >= 0:
                chain.append(parents[i * n + chain[-1]])
            hidden[row, 0, c - n:] = True
            for a in chain[:window]:
                hidden[row, 0, c - n + a] = False
            hidden[row, 0, :min(c - n, max(0, c - n + len(chain) - window))] = True
        hidden = hidden.to(DEVICE)
        table = s["page_table"][i, :(c + page - 1) // page].long()
        for h in range(hkv):
            k, v = (_fp4_values(s["cache"][j][table, h], s["cache"][j + 1][table, h], torch.float64).flatten(0, 1)[:c]
                    for j in (0, 2))
            heads, mine = slice(h * group, (h + 1) * group), slice(i * n, (i + 1) * n)
            t = torch.matmul(s["q"][mine, heads].double().flatten(0, 1), k.T).unflatten(0, (n, -1)) * s["scale"]
            t = t.masked_fill(hidden, -math.inf)
            lse[mine, heads] = torch.logsumexp(t, -1)
            out[mine, heads] = torch.matmul(torch.softmax(t, -1).flatten(0, 1), v).unflatten(0, (n, -1))
    return {"out": out, "lse": lse}
