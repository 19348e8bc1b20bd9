"""The attention operators of `consumer_int8.attention`, as a serving program calls them.

norm_rope  attention.qk_norm_rope: RMS norm of each query and key head with the position
           rotation, in one pass over a layer's projected tokens.
append     attention.append_fp4: the same for the queries, while keys (normed, rotated) and
           values go to a paged cache of 4-bit values (E2M1 codes, one power-of-two scale for
           32 channels); then attention.unpack_fp4 reads the rows back as BF16.
attend     attention.attention_fp4: causal attention of BF16 queries over that cache, from one
           new token a sequence to whole prompts.

The plain forms compute in FP32 with elementary torch operations and round once at the end.
"""

import math
import os
import sys

import torch

own = False

DEVICE = "cuda"
BLOCK = 32  # channels that share one scale

# (query heads, key heads, channels of a head, rotated channels)
HEADS = [(32, 8, 128, 128), (24, 4, 256, 64), (40, 8, 128, 128), (64, 8, 128, 128),
         (16, 16, 64, 64), (14, 2, 64, 64), (28, 4, 128, 128)]


def _case(kind, heads, **more):
    hq, hkv, dim, rot = HEADS[heads]
    return dict(kind=kind, hq=hq, hkv=hkv, dim=dim, rot=rot, **more)


def listed():
    return [
        # One token of one sequence, eight key heads of 128: the smallest call.
        dict(name="norm_rope_t1_32x8x128", **_case("norm_rope", 0, tokens=1, axes=1, norm=True, interleaved=False)),
        # A prompt; 64 of 256 channels rotate.
        dict(name="norm_rope_t4096_24x4x256", **_case("norm_rope", 1, tokens=4096, axes=1, norm=True, interleaved=False)),
        # The patches of a video: time, height and width each turn a third of the pairs.
        dict(name="norm_rope_t9261_16x16x64_3axes", **_case("norm_rope", 4, tokens=9261, axes=3, norm=False, interleaved=True)),
        # A decode batch: one token for each of 64 sequences, small pages.
        dict(name="append_t64_32x8x128", **_case("append", 0, tokens=64, page=16, prompt=False, norm=True)),
        # A ragged prompt chunk into large pages.
        dict(name="append_t8191_24x4x256", **_case("append", 1, tokens=8191, page=64, prompt=True, norm=True)),
        # One short conversation: the smallest attention call.
        dict(name="attend_s1_c517_32x8x128", **_case("attend", 0, seqs=1, q_min=1, q_max=1, c_min=517, c_max=517, page=16, window=0)),
        # A decode batch of ragged conversations.
        dict(name="attend_s32_c8000_32x8x128", **_case("attend", 0, seqs=32, q_min=1, q_max=1, c_min=200, c_max=8000, page=16, window=0)),
        # One very long document.
        dict(name="attend_s1_c131071_24x4x256", **_case("attend", 1, seqs=1, q_min=1, q_max=1, c_min=131071, c_max=131071, page=64, window=0)),
        # A full decode batch with long contexts: the most bytes.
        dict(name="attend_s64_c32768_64x8x128", **_case("attend", 3, seqs=64, q_min=1, q_max=1, c_min=8192, c_max=32768, page=64, window=0)),
        # Four drafted tokens a sequence are verified.
        dict(name="attend_s16_q4_c16000_24x4x256", **_case("attend", 1, seqs=16, q_min=4, q_max=4, c_min=3000, c_max=16000, page=32, window=0)),
        # A whole prompt over its own cache: the most operations.
        dict(name="attend_s1_q4096_c4096_40x8x128", **_case("attend", 2, seqs=1, q_min=4096, q_max=4096, c_min=4096, c_max=4096, page=64, window=0)),
        # Ragged prompt chunks behind long contexts, of which a window of 4096 tokens is seen.
        dict(name="attend_s3_q1000_c15000_28x4x128_w4096", **_case("attend", 6, seqs=3, q_min=300, q_max=1000, c_min=9000, c_max=15000, page=32, window=4096)),
    ]


def _log_int(rng, low, high):
    """An integer in [low, high], spread evenly over the logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49))))))


def _attend_cost(c):
    """Multiply-adds of the padded plain form."""
    return c["seqs"] * c["hq"] * c["q_max"] * c["c_max"] * c["dim"]


def draw(rng):
    kind = rng.choice(["norm_rope", "append", "attend", "attend", "attend"])
    heads = rng.randrange(len(HEADS))
    if kind == "norm_rope":
        return _case(kind, heads, tokens=_log_int(rng, 1, 9000 if heads != 3 else 4096), axes=rng.choice([1, 3]),
                     norm=rng.random() < 0.7, interleaved=rng.random() < 0.5)
    if kind == "append":
        prompt = rng.random() < 0.5
        return _case(kind, heads, tokens=_log_int(rng, 200, 8000) if prompt else _log_int(rng, 1, 256),
                     page=rng.choice([16, 32, 64, 128]), prompt=prompt, norm=rng.random() < 0.7)
    page, window = rng.choice([16, 32, 64, 128]), rng.choice([0, 0, 0, 1024, 4096])
    form = rng.choice(["decode", "decode", "verify", "prompt"])
    if form == "decode":
        seqs, q = _log_int(rng, 1, 64), 1
        c = _log_int(rng, 100, 131072)
    elif form == "verify":
        seqs, q = _log_int(rng, 1, 24), rng.randint(2, 8)
        c = _log_int(rng, 100, 32768)
    else:
        seqs, q = rng.randint(1, 4), _log_int(rng, 64, 4000)
        c = q + _log_int(rng, 1, 12000)
    case = _case(kind, heads, seqs=seqs, q_min=q if q <= 8 else max(1, q // 2), q_max=q,
                 c_min=max(q, c // 4), c_max=c, page=page, window=window)
    # no more than the largest listed case: bytes of a decode batch, products of a prompt
    most = 64 * 32768 * 8 * 128 if q <= 8 else 40 * 4096 * 4096 * 128
    cost = seqs * c * case["hkv"] * case["dim"] if q <= 8 else _attend_cost(case)
    if cost > most:
        shrink = most / cost
        case["c_max"] = max(q, int(c * shrink))
        case["c_min"] = max(q, case["c_max"] // 4)
        if q > 8 and _attend_cost(case) > most:
            case["seqs"] = 1
    return case


# ---- sizes of a case, the same for every seed -------------------------------------------


def _spread(count, low, high):
    """`count` lengths between low and high, the first the longest, evenly spread."""
    return [high - int((high - low) * math.modf(i * 0.6180339887498949)[0]) for i in range(count)]


def _lens(case):
    qs, cs = _spread(case["seqs"], case["q_min"], case["q_max"]), _spread(case["seqs"], case["c_min"], case["c_max"])
    return qs, [max(q, c) for q, c in zip(qs, cs)]


def work(case):
    hq, hkv, dim = case["hq"], case["hkv"], case["dim"]
    if case["kind"] == "norm_rope":
        t = case["tokens"]
        return {"bytes": t * ((hq + hkv) * dim * 4 + case["rot"] * 4 + 8 * case["axes"]), "flops": t * (hq + hkv) * dim * 8}
    packed = dim // 2 + dim // BLOCK  # bytes of one head of one token
    if case["kind"] == "append":
        t = case["tokens"]
        bytes_ = t * (hq * dim * 4 + 2 * hkv * dim * 2 + case["rot"] * 4 + 16)  # q in and out, k and v in
        bytes_ += t * 2 * hkv * (2 * packed + dim * 2)                          # packed out, packed in, values out
        return {"bytes": bytes_, "flops": t * (hq + 3 * hkv) * dim * 8}
    qs, cs = _lens(case)
    window = case["window"] or max(cs)
    tokens = sum(qs)
    read = pairs = 0
    for q, c in zip(qs, cs):
        read += min(c, window + q - 1)
        # positions c-q .. c-1, each seeing min(position + 1, window) tokens
        full = max(0, min(q, c - max(window, c - q + 1) + 1))
        short = q - full
        pairs += full * window + sum(range(c - q + 1, c - q + 1 + short))
    return {"bytes": read * 2 * hkv * packed + tokens * hq * (dim * 4 + 4), "flops": 4 * pairs * hq * dim}


# ---- inputs -----------------------------------------------------------------------------


def _rope_table(rows, rot):
    """FP32 [rows, rot]: the cosines of a position's rot/2 angles, then their sines."""
    freq = 1e6 ** (-torch.arange(rot // 2, dtype=torch.float64) * 2 / rot)
    angle = torch.arange(rows, dtype=torch.float64)[:, None] * freq
    return torch.cat([angle.cos(), angle.sin()], 1).float().to(DEVICE)


def _projected(case, gen):
    """One layer's projected tokens, BF16 [T, (Hq + 2 Hkv) * dim], and its heads as views."""
    t, hq, hkv, dim = case["tokens"], case["hq"], case["hkv"], case["dim"]
    # channels differ in size, as those of keys do
    gain = torch.exp(0.7 * torch.randn((hq + 2 * hkv) * dim, device=DEVICE, generator=gen))
    qkv = (torch.randn(t, (hq + 2 * hkv) * dim, device=DEVICE, generator=gen) * gain).bfloat16()
    q, k, v = qkv.split([hq * dim, hkv * dim, hkv * dim], 1)
    return q.unflatten(1, (hq, dim)), k.unflatten(1, (hkv, dim)), v.unflatten(1, (hkv, dim))


def _norm_weights(case, gen):
    if not case["norm"]:
        return None, None
    return tuple(torch.exp(0.3 * torch.randn(case["dim"], device=DEVICE, generator=gen)) for _ in "qk")


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


def _empty_cache(pages, case):
    shape = (pages, case["hkv"], case["page"])
    return [torch.zeros(*shape, case["dim"] // n, dtype=torch.uint8, device=DEVICE) for n in (2, BLOCK, 2, BLOCK)]


def prepare(case, seed):
    gen = torch.Generator(DEVICE).manual_seed(seed)
    hq, hkv, dim, rot = case["hq"], case["hkv"], case["dim"], case["rot"]
    s = {"case": case}
    if case["kind"] != "attend":
        t, rows = case["tokens"], 16384
        s["q"], s["k"], s["v"] = _projected(case, gen)
        s["q_weight"], s["k_weight"] = _norm_weights(case, gen)
        s["rope"] = _rope_table(rows, rot)
        s["q_out"] = torch.empty(t, hq, dim, dtype=torch.bfloat16, device=DEVICE)
    if case["kind"] == "norm_rope":
        s["k_out"] = torch.empty(t, hkv, dim, dtype=torch.bfloat16, device=DEVICE)
        if case["axes"] == 1:
            first = int(torch.randint(0, rows - t, (1,), device=DEVICE, generator=gen))
            s["positions"] = first + torch.arange(t, device=DEVICE)
            s["axes"] = None
        else:
            side = max(1, round(t ** (1 / 3)))
            at = torch.arange(t, device=DEVICE)
            s["positions"] = torch.stack([at // (side * side), at // side % side, at % side])
            s["axes"] = (torch.arange(rot // 2, device=DEVICE) % 3).int()
    elif case["kind"] == "append":
        page = case["page"]
        pages = (t + page - 1) // page + 3 if case["prompt"] else t + t // 4 + 3
        order = torch.randperm(pages, device=DEVICE, generator=gen)
        if case["prompt"]:
            s["positions"] = torch.arange(t, device=DEVICE)
            s["slots"] = order[s["positions"] // page] * page + s["positions"] % page
        else:  # each token in the newest page of its own sequence
            s["positions"] = torch.randint(0, rows, (t,), device=DEVICE, generator=gen)
            s["slots"] = order[:t] * page + s["positions"] % page
        s["cache"] = _empty_cache(pages, case)
        s["k_values"], s["v_values"] = (torch.empty(t, hkv, dim, dtype=torch.bfloat16, device=DEVICE) for _ in "kv")
    else:
        page = case["page"]
        qs, cs = _lens(case)
        used = [(c + page - 1) // page for c in cs]
        pages = sum(used) + max(2, sum(used) // 16)
        s["cache"] = _empty_cache(pages, case)
        gain = torch.exp(0.5 * torch.randn(2, hkv, 1, dim, device=DEVICE, generator=gen))
        step = max(1, (1 << 26) // (hkv * page * dim))
        for first in range(0, pages, step):
            n = min(step, pages - first)
            for i in range(2):
                x = torch.randn(n, hkv, page, dim, device=DEVICE, generator=gen) * gain[i]
                s["cache"][2 * i][first:first + n], s["cache"][2 * i + 1][first:first + n] = _fp4_codes(x)
        order = torch.randperm(pages, device=DEVICE, generator=gen).int()
        width = max(used)
        ends = torch.tensor(used, device=DEVICE).cumsum(0)
        col = torch.arange(width, device=DEVICE)
        start = (ends - torch.tensor(used, device=DEVICE))[:, None]
        s["page_table"] = torch.where(start + col < ends[:, None], order[(start + col).clamp(max=pages - 1)], -1)
        s["context_lens"] = torch.tensor(cs, dtype=torch.int32, device=DEVICE)
        s["q_starts"] = torch.tensor([0] + qs, device=DEVICE).cumsum(0).int()
        tokens = sum(qs)
        # rows of the projected tokens' buffer; scores of a few units, as trained heads have
        qkv = 2 * torch.randn(tokens, (hq + 2 * hkv) * dim, device=DEVICE, generator=gen).bfloat16()
        s["q"] = qkv[:, :hq * dim].unflatten(1, (hq, dim))
        s["scale"] = dim ** -0.5
        s["out"] = torch.empty(tokens, hq, dim, dtype=torch.bfloat16, device=DEVICE)
        s["lse"] = torch.empty(tokens, hq, dtype=torch.float32, device=DEVICE)
        s["workspace"] = torch.empty(65536, dim + 2, dtype=torch.float32, device=DEVICE)
    return s


# ---- the operators ----------------------------------------------------------------------


def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    path = os.path.join(os.getcwd(), "consumer-int8-kernels_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from consumer_int8 import attention

    case = s["case"]
    if case["kind"] == "norm_rope":
        attention.qk_norm_rope(s["q"], s["k"], s["q_weight"], s["k_weight"], s["rope"], s["positions"], s["axes"],
                               s["q_out"], s["k_out"], 1e-6, case["interleaved"])
        return {"q": s["q_out"], "k": s["k_out"]}
    if case["kind"] == "append":
        attention.append_fp4(s["q"], s["k"], s["v"], s["q_weight"], s["k_weight"], s["rope"], s["positions"], None,
                             s["slots"], s["q_out"], *s["cache"], 1e-6, False)
        attention.unpack_fp4(*s["cache"], s["slots"], s["k_values"], s["v_values"])
        return {"q": s["q_out"], "k": s["k_values"], "v": s["v_values"]}
    attention.attention_fp4(s["q"], *s["cache"], s["page_table"], s["context_lens"], s["q_starts"], s["workspace"],
                            s["out"], s["lse"], s["scale"], case["q_max"], case["window"])
    return {"out": s["out"], "lse": s["lse"]}


def _pairs(x):
    return x[..., 0::2] + x[..., 1::2]


def _plain_norm(x, weight):
    """x / rms(x) * weight over the last axis; neighbours are summed first, then pairs of them."""
    if weight is None:
        return x
    squares = torch.nn.functional.pad(x * x, (0, 256 - x.shape[-1]))
    total = _pairs(_pairs(_pairs(_pairs(_pairs(_pairs(_pairs(_pairs(squares))))))))
    return x * (1 / torch.sqrt(total * (1 / x.shape[-1]) + 1e-6)) * weight


def _plain_rope(x, s):
    """Pairs of the first rot channels turn by their position's angles."""
    rot, half, at = s["case"]["rot"], s["case"]["rot"] // 2, s["positions"]
    if s.get("axes") is None:
        cos, sin = s["rope"][at, :half], s["rope"][at, half:]
    else:
        row = at[s["axes"].long()].T  # [T, half]
        col = torch.arange(half, device=row.device)
        cos, sin = s["rope"][row, col], s["rope"][row, half + col]
    cos, sin = cos[:, None], sin[:, None]
    turned, rest = x[..., :rot], x[..., rot:]
    if s["case"].get("interleaved"):
        a, b = turned[..., 0::2], turned[..., 1::2]
        return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), rest], -1)
    a, b = turned[..., :half], turned[..., half:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)


def _run_plain(s):
    case = s["case"]
    if case["kind"] != "attend":
        q = _plain_rope(_plain_norm(s["q"].float(), s["q_weight"]), s).bfloat16()
        k = _plain_rope(_plain_norm(s["k"].float(), s["k_weight"]), s)
        if case["kind"] == "norm_rope":
            return {"q": q, "k": k.bfloat16()}
        page, row = s["slots"] // case["page"], s["slots"] % case["page"]
        for_k, for_v = s["cache"][:2], s["cache"][2:]
        for_k[0][page, :, row], for_k[1][page, :, row] = _fp4_codes(k)
        for_v[0][page, :, row], for_v[1][page, :, row] = _fp4_codes(s["v"].float())
        back = (_fp4_values(c[page, :, row], e[page, :, row]).bfloat16() for c, e in (for_k, for_v))
        return {"q": q, "k": next(back), "v": next(back)}

    hq, hkv, dim = case["hq"], case["hkv"], case["dim"]
    group, tokens = hq // hkv, s["q"].shape[0]
    lens, starts, window = s["context_lens"], s["q_starts"], case["window"]
    seqs, most_q, most_c = case["seqs"], case["q_max"], case["c_max"]

    def gathered(codes, scales):  # [S, Hkv, C, dim]
        at = s["page_table"].clamp(min=0)
        c, e = (x[at].transpose(1, 2).flatten(2, 3)[:, :, :most_c] for x in (codes, scales))
        return _fp4_values(c, e)

    keys = gathered(*s["cache"][:2])
    i = torch.arange(most_q, device=DEVICE)
    q_len = starts[1:] - starts[:-1]
    rows = (starts[:-1, None] + i).clamp(max=tokens - 1)
    q = s["q"].float()[rows]                                                    # [S, Q, Hq, dim]
    q = q.unflatten(2, (hkv, group)).permute(0, 2, 1, 3, 4).flatten(2, 3)      # [S, Hkv, Q * group, dim]
    scores = torch.matmul(q, keys.transpose(-1, -2)) * s["scale"]
    del keys
    pos = ((lens - q_len)[:, None] + i).repeat_interleave(group, 1)[:, None, :, None]
    at = torch.arange(most_c, device=DEVICE)
    seen = at <= pos
    if window:
        seen = seen & (at > pos - window)
    scores = torch.where(seen, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0, top)
    p = torch.exp(scores - top)
    del scores
    total = p.sum(-1, keepdim=True)
    values = gathered(*s["cache"][2:])
    values = torch.where((at < lens[:, None])[:, None, :, None], values, 0)
    out = torch.matmul(p, values) / torch.where(total == 0, 1, total)
    lse = torch.log(total) + top
    out, lse = (x.unflatten(2, (most_q, group)).permute(0, 2, 1, 3, 4).flatten(2, 3) for x in (out, lse))
    real = i < q_len[:, None]
    return {"out": out[real].bfloat16(), "lse": lse[real].squeeze(-1)}


# ---- the same from the definitions, in 64 bits --------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] != "attend":
        rot, half = case["rot"], case["rot"] // 2
        pos = s["positions"][None] if s["positions"].dim() == 1 else s["positions"]
        which = s["axes"].long() if s.get("axes") is not None else torch.zeros(half, dtype=torch.int64, device=DEVICE)
        angle_row = pos[which]  # [half, T]
        cs = torch.stack([s["rope"][angle_row[j], j] for j in range(half)], 1).double()
        sn = torch.stack([s["rope"][angle_row[j], half + j] for j in range(half)], 1).double()

        def turned(x, w):
            x = x.double()
            if w is not None:
                x = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
            y = x.clone()
            for j in range(half):
                a, b = (2 * j, 2 * j + 1) if case.get("interleaved") else (j, j + half)
                c, d = cs[:, j, None], sn[:, j, None]
                y[..., a] = x[..., a] * c - x[..., b] * d
                y[..., b] = x[..., a] * d + x[..., b] * c
            return y

        q, k = turned(s["q"], s["q_weight"]), turned(s["k"], s["k_weight"])
        if case["kind"] == "norm_rope":
            return {"q": q, "k": k}

        def stored(x):  # the nearest E2M1 multiple of the block's scale, ties to the even code
            b = x.unflatten(-1, (-1, BLOCK))
            top = b.abs().amax(-1, keepdim=True)
            e = torch.ceil(torch.log2(torch.where(top > 0, top, 2.0 ** -122) / 7)).clamp(min=-125)
            e = e + (top > 7 * torch.exp2(e)).double() - ((top <= 7 * torch.exp2(e - 1)) & (e > -125)).double()
            unit = torch.exp2(e)
            y = b / unit
            low = torch.floor(torch.log2(y.abs().clamp(min=1))).clamp(max=2)
            step = torch.exp2(low - 1)
            return ((torch.round(y / step) * step).clamp(-6, 6) * unit).flatten(-2)

        return {"q": q, "k": stored(k), "v": stored(s["v"].double())}

    hq, hkv, page, window = case["hq"], case["hkv"], case["page"], case["window"]
    qs, cs = _lens(case)
    out = torch.empty(sum(qs), hq, case["dim"], dtype=torch.float64, device=DEVICE)
    lse = torch.empty(sum(qs), hq, dtype=torch.float64, device=DEVICE)
    begin = 0
    for i, (nq, c) in enumerate(zip(qs, cs)):
        table = s["page_table"][i, :(c + page - 1) // page].long()
        for h in range(hkv):
            k, v = (_fp4_values(s["cache"][j][table, h], s["cache"][j + 1][table, h], torch.float64).flatten(0, 1)[:c]
                    for j in (0, 2))
            heads = slice(h * (hq // hkv), (h + 1) * (hq // hkv))
            q = s["q"][begin:begin + nq, heads].double()
            t = torch.matmul(q.flatten(0, 1), k.T).unflatten(0, (nq, -1)) * s["scale"]
            pos = torch.arange(c - nq, c, device=DEVICE)[:, None, None]
            at = torch.arange(c, device=DEVICE)
            hidden = (at > pos) | ((at <= pos - window) if window else False)
            t = t.masked_fill(hidden, -math.inf)
            lse[begin:begin + nq, heads] = torch.logsumexp(t, -1)
            out[begin:begin + nq, heads] = torch.matmul(torch.softmax(t, -1).flatten(0, 1), v).unflatten(0, (nq, -1))
        begin += nq
    return {"out": out, "lse": lse}
