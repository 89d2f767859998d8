"""What the serving and position operators are measured on: per-head q / k norm with rotary positions (`qk_rope`, forward and backward),
appending keys and values to a paged cache with the rotation applied on the way (`kv_append`), and attention of new tokens over the
paged cache (`attn_paged`).

A case is a dict of plain values.  Ragged lengths follow from the case alone (`_lengths`), values and the order of the pages from the
seed.  With `own` false `run` computes the plain forms in 32 bits (angles in 64); with `own` true it makes the package's calls."""
import math
import random

import torch

own = False

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
F8 = torch.float8_e4m3fn
F8_MAX = 448.0


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # training step of a qk-normed block on the framework's own token grid: 16 samples x 16 frames x 320 tokens, 8 heads of 32,
        # LayerNorm with the shared affine, (frame, row, column) positions on one third of the pairs each
        dict(name="rope train frames", op="rope", grad=True, tokens=81920, hq=8, hk=8, d=32, rot=32, inter=False, norm="layer", type="bf16",
             wtype="fp32", axes=3, far=16, scaled=False),
        # training step with grouped heads on one ragged-packed batch of an odd number of tokens, frequencies scaled for a long context
        dict(name="rope train grouped", op="rope", grad=True, tokens=8191, hq=32, hk=8, d=128, rot=128, inter=True, norm="rms", type="bf16",
             wtype="bf16", axes=1, far=131072, scaled=True),
        # a handful of decoded tokens at far positions, half of each head rotated, no norm: a latency-bound call
        dict(name="rope decode", op="rope", grad=False, tokens=7, hq=32, hk=8, d=128, rot=64, inter=False, norm="none", type="fp16",
             wtype="fp32", axes=1, far=1000000, scaled=False),
        # one decode step of 64 running sequences: q and k normed and rotated, k and v put into their pages, in one call
        dict(name="append decode", op="append", seqs=64, past_lo=0, past_hi=8192, new_lo=1, new_hi=1, hq=32, hk=8, d=128, rot=128, inter=False,
             norm="rms", type="bf16", wtype="bf16", cache="same", page=16, axes=1, with_q=True, pad=0),
        # prompts going into an 8-bit cache; queries are handled elsewhere
        dict(name="append prompts e4m3", op="append", seqs=4, past_lo=0, past_hi=3000, new_lo=1000, new_hi=3001, hq=32, hk=8, d=128, rot=128,
             inter=False, norm="none", type="bf16", wtype="fp32", cache="e4m3", page=64, axes=1, with_q=False, pad=0),
        # one new frame (256 image + 64 action tokens) of 8 rollouts of the video model, a page per 64 tokens, a padded batch
        dict(name="append frame", op="append", seqs=8, past_lo=0, past_hi=20160, new_lo=320, new_hi=320, hq=8, hk=8, d=32, rot=32, inter=False,
             norm="layer", type="bf16", wtype="fp32", cache="same", page=64, axes=3, with_q=True, pad=64),
        # a single interactive sequence, one token
        dict(name="attn one token", op="attn", seqs=1, past_lo=700, past_hi=700, new_lo=1, new_hi=1, hq=32, hk=8, d=128, type="bf16", cache="same",
             page=16, causal=True, window=0, pad=0),
        # a decode step of a batch whose sequences have very different lengths
        dict(name="attn decode ragged", op="attn", seqs=64, past_lo=0, past_hi=16384, new_lo=1, new_hi=1, hq=32, hk=8, d=128, type="bf16",
             cache="same", page=16, causal=True, window=0, pad=0),
        # few long sequences out of an 8-bit cache
        dict(name="attn decode long e4m3", op="attn", seqs=4, past_lo=65536, past_hi=131071, new_lo=1, new_hi=1, hq=64, hk=8, d=128, type="bf16",
             cache="e4m3", page=64, causal=True, window=0, pad=0),
        # a frame of the video model over the frames so far: its 320 tokens see each other and the whole past, a page per frame
        dict(name="attn frame", op="attn", seqs=4, past_lo=5120, past_hi=20160, new_lo=320, new_hi=320, hq=8, hk=8, d=32, type="bf16",
             cache="same", page=320, causal=False, window=0, pad=0),
        # whole prompts
        dict(name="attn prompts", op="attn", seqs=2, past_lo=0, past_hi=0, new_lo=5003, new_hi=8191, hq=32, hk=8, d=128, type="bf16",
             cache="same", page=32, causal=True, window=0, pad=0),
        # chunks of prompts and decoded tokens in one batch, a sliding window, a padded batch
        dict(name="attn mixed window", op="attn", seqs=8, past_lo=0, past_hi=12000, new_lo=1, new_hi=512, hq=16, hk=2, d=64, type="fp16",
             cache="same", page=16, causal=True, window=4096, pad=24),
    ]


def _log(rng, lo, hi):
    """A whole number whose logarithm is uniform in [lo, hi]."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.999)))))))


def draw(rng):
    op = rng.choice(["rope", "append", "attn", "attn"])
    hk, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 8])
    if op != "attn":
        d = rng.choice([32, 64, 80, 96, 128])
        rot = rng.choice([d, d, d // 2, d // 4])
        c = dict(op=op, hq=hk * group, hk=hk, d=d, rot=rot, inter=rng.random() < 0.5, norm=rng.choice(["none", "rms", "layer"]),
                 type=rng.choice(["bf16", "bf16", "fp16"]), wtype=rng.choice(["fp32", "same"]), axes=rng.choice([1, 1, 3]))
        c["wtype"] = c["type"] if c["wtype"] == "same" else "fp32"
        if op == "rope":
            most = 8191 * 40 * 128 // ((c["hq"] + hk) * d)
            return c | dict(grad=rng.random() < 0.6, tokens=_log(rng, 1, min(81920, most)), far=_log(rng, 16, 1000000), scaled=rng.random() < 0.3)
        seqs = _log(rng, 1, 64)
        new_hi = _log(rng, 1, 2048 // seqs)
        return c | dict(seqs=seqs, past_lo=0, past_hi=_log(rng, 1, 8192), new_lo=rng.choice([1, new_hi]), new_hi=new_hi,
                        cache=rng.choice(["same", "same", "e4m3"]), page=rng.choice([16, 32, 48, 64, 128]), with_q=rng.random() < 0.7,
                        pad=rng.choice([0, 0, 5, 32]))
    d = rng.choice([32, 64, 128])
    hq = hk * group
    c = dict(op=op, hq=hq, hk=hk, d=d, type=rng.choice(["bf16", "bf16", "fp16"]), cache=rng.choice(["same", "same", "e4m3"]),
             page=rng.choice([8, 16, 32, 48, 64, 128, 320]), pad=rng.choice([0, 0, 3, 17]))
    c["causal"] = rng.random() < 0.7
    c["window"] = _log(rng, 64, 4096) if c["causal"] and rng.random() < 0.3 else 0
    seqs = _log(rng, 1, 48)
    new_hi = min(rng.choice([1, 1, _log(rng, 2, 64), _log(rng, 64, 2048)]), max(1, 8192 // seqs))
    # at most 1.2e9 pairs of a query and a key over all heads, and the cache no larger than the listed ones
    most = min(40000, 1_200_000_000 // (seqs * new_hi * hq) - new_hi, 500_000_000 // (seqs * hk * d) - new_hi)
    past_hi = _log(rng, 1, max(1, most))
    return c | dict(seqs=seqs, past_lo=rng.choice([0, past_hi // 2]), past_hi=past_hi, new_lo=rng.choice([1, new_hi]), new_hi=new_hi)


def _lengths(c):
    """(new tokens, tokens in the cache with them) of each sequence.  Ragged ranges are spread evenly in a fixed order; the extremes occur."""
    n, r = c["seqs"], random.Random(7 * c["seqs"] + c["new_hi"])

    def spread(lo, hi):
        v = [lo + (hi - lo) * i // max(1, n - 1) for i in range(n)] if n > 1 else [hi]
        r.shuffle(v)
        return v

    new, past = spread(c["new_lo"], c["new_hi"]), spread(c["past_lo"], c["past_hi"])
    return new, [a + b for a, b in zip(new, past)]


# ------------------------------------------------------------------------------------------------ inputs
def _frequencies(c):
    """Radians per position of each rotated pair, 64 bits.  `scaled`: pairs that turn less than once over 8192 positions are slowed down
    eight times, those that turn over 32 times are left, a ramp between them; the amplitude grows with the logarithm of the scale."""
    i = torch.arange(c["rot"] // 2, dtype=torch.float64, device="cuda")
    f, amp = 10000.0 ** (-2.0 * i / c["rot"]), 1.0
    if c.get("scaled"):
        keep = ((8192.0 * f / (2 * math.pi) - 1.0) / 31.0).clamp(0, 1)
        f, amp = f * (keep + (1 - keep) / 8.0), 1.0 + 0.1 * math.log(8.0)
    return f, amp


def _rotary_state(c, g, tokens, s):
    """Norm weights, frequencies and positions."""
    s["freqs"], s["amp"] = _frequencies(c)
    s["axes"] = (torch.arange(c["rot"] // 2, device="cuda") % 3).to(torch.int32) if c["axes"] == 3 else None
    wt = DT[c["wtype"]]
    for h in ("q", "k"):
        s[h + "w"] = (1 + 0.2 * torch.randn(c["d"], generator=g, device="cuda")).to(wt) if c["norm"] != "none" else None
        s[h + "b"] = (0.1 * torch.randn(c["d"], generator=g, device="cuda")).to(wt) if c["norm"] == "layer" else None
    s["eps"] = 1e-5
    if c["axes"] == 3:  # (frame, row, column) of a 16 x 20 token grid per frame
        at = torch.arange(tokens, device="cuda")
        s["pos"] = torch.stack([at // 320 % c.get("far", 64), at % 320 // 20, at % 20])
    elif c["op"] == "rope":
        s["pos"] = torch.randint(0, c["far"], (tokens,), generator=g, device="cuda")
    else:
        s["pos"] = None  # the tokens' places in the cache


def _packed(c, g, tokens, t):
    """q, k, v as views of the packed rows that a projection writes."""
    hq, hk, d = c["hq"], c["hk"], c["d"]
    x = (1.5 * torch.randn(tokens, (hq + 2 * hk) * d, generator=g, device="cuda") + 0.1).to(t)
    return (x[:, : hq * d].view(tokens, hq, d), x[:, hq * d : (hq + hk) * d].view(tokens, hk, d), x[:, (hq + hk) * d :].view(tokens, hk, d))


def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = DT[c["type"]]
    s = dict(c)
    if c["op"] == "rope":
        n = c["tokens"]
        s["q"], s["k"], _ = _packed(c, g, n, t)
        _rotary_state(c, g, n, s)
        if c["grad"]:
            s["gq"] = torch.randn(n, c["hq"], c["d"], generator=g, device="cuda").to(t)
            s["gk"] = torch.randn(n, c["hk"], c["d"], generator=g, device="cuda").to(t)
            s["leaves"] = [x.detach().requires_grad_() for x in (s["q"], s["k"], s["qw"], s["qb"], s["kw"], s["kb"]) if x is not None]
        return s
    new, lens = _lengths(c)
    page, hk, d = c["page"], c["hk"], c["d"]
    need = [-(-n // page) for n in lens]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((c["seqs"], max(need) + 1), -1, dtype=torch.int32, device="cuda")  # the entries behind a sequence's pages hold no page
    at = 0
    for b, k in enumerate(need):
        table[b, :k] = order[at : at + k]
        at += k
    s["table"] = table
    s["cu"] = torch.tensor([sum(new[:b]) for b in range(c["seqs"] + 1)], dtype=torch.int32, device="cuda")
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    s["most_new"], s["most_len"] = max(new), max(lens)
    tokens = sum(new) + c["pad"]
    shape = (pages, hk, page, d)  # a page holds each head's tokens one behind the other
    if c["cache"] == "e4m3":
        s["ks"] = 0.012 + 0.004 * torch.rand(hk, generator=g, device="cuda")
        s["vs"] = 0.012 + 0.004 * torch.rand(hk, generator=g, device="cuda")
        s["kc"] = (torch.randn(shape, generator=g, device="cuda") / s["ks"][:, None, None]).clamp(-F8_MAX, F8_MAX).to(F8)
        s["vc"] = (torch.randn(shape, generator=g, device="cuda") / s["vs"][:, None, None]).clamp(-F8_MAX, F8_MAX).to(F8)
    else:
        s["ks"] = s["vs"] = None
        s["kc"] = torch.randn(shape, generator=g, device="cuda", dtype=t)
        s["vc"] = torch.randn(shape, generator=g, device="cuda", dtype=t)
    if c["op"] == "append":
        s["q"], s["k"], s["v"] = _packed(c, g, tokens, t)
        _rotary_state(c, g, tokens, s)
    else:
        s["q"] = torch.randn(tokens, c["hq"], d, generator=g, device="cuda").to(t)
        s["scale"] = d ** -0.5
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _angles(s, pos):
    """(cos, sin) of each token and pair times the amplitude; the angle in 64 bits."""
    p = pos.double()
    a = (p[:, None] if p.dim() == 1 else p.t()[:, s["axes"].long()]) * s["freqs"]
    return (a.cos() * s["amp"]).float()[:, None], (a.sin() * s["amp"]).float()[:, None]


def _turn(s, x, cos, sin):
    r, h = s["rot"], s["rot"] // 2
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if s["inter"] else (x[..., :h], x[..., h:r])
    u, w = a * cos - b * sin, a * sin + b * cos
    y = torch.stack([u, w], -1).flatten(-2) if s["inter"] else torch.cat([u, w], -1)
    return torch.cat([y, x[..., r:]], -1)


def _unit(s, x):
    """(normalised x, 1 / deviation): nothing, root mean square, or mean and deviation."""
    if s["norm"] == "none":
        return x, None
    if s["norm"] == "layer":
        x = x - x.mean(-1, keepdim=True)
    r = (x.square().mean(-1, keepdim=True) + s["eps"]).rsqrt()
    return x * r, r


def _affine(s, x, h):
    x = x if s[h + "w"] is None else x * s[h + "w"].float()
    return x if s[h + "b"] is None else x + s[h + "b"].float()


def _rotated(s, x, h, cos, sin):
    return _turn(s, _affine(s, _unit(s, x.float())[0], h), cos, sin)


def _rotated_grad(s, x, g, h, cos, sin):
    """[d x, d weight, d bias] from the gradient `g` of the rotated rows."""
    u, r = _unit(s, x.float())
    g = _turn(s, g.float(), cos, -sin)  # the rotation back
    dw = None if s[h + "w"] is None else (g * u).sum((0, 1)).to(s[h + "w"].dtype)
    db = None if s[h + "b"] is None else g.sum((0, 1)).to(s[h + "b"].dtype)
    if s["norm"] != "none":
        g = g * s[h + "w"].float()
        d = g - u * (g * u).mean(-1, keepdim=True)
        g = (d - g.mean(-1, keepdim=True) if s["norm"] == "layer" else d) * r
    return [g.to(x.dtype), dw, db]


def _plain_rope(s):
    cos, sin = _angles(s, s["pos"])
    out = [_rotated(s, s["q"], "q", cos, sin).to(s["q"].dtype), _rotated(s, s["k"], "k", cos, sin).to(s["k"].dtype)]
    if s["grad"]:
        out += _rotated_grad(s, s["q"], s["gq"], "q", cos, sin) + _rotated_grad(s, s["k"], s["gk"], "k", cos, sin)
    return [x for x in out if x is not None]


def _places(s, tokens):
    """(sequence, place in the cache, whether it belongs to a sequence) of each row of the batch."""
    row = torch.arange(tokens, device="cuda")
    live = row < s["cu"][-1]
    b = torch.searchsorted(s["cu"][1:].long(), row, right=True).clamp(max=s["seqs"] - 1)
    return b, s["lens"].long()[b] - s["cu"].long()[b + 1] + row, live


def _stored(x, scale, like):
    x = x if scale is None else (x / scale[:, None]).clamp(-F8_MAX, F8_MAX)
    return x.to(like)


def _plain_append(s):
    b, at, live = _places(s, s["k"].shape[0])
    cos, sin = _angles(s, at if s["pos"] is None else s["pos"])
    k = _stored(_rotated(s, s["k"], "k", cos, sin), s["ks"], s["kc"].dtype)
    v = _stored(s["v"].float(), s["vs"], s["vc"].dtype)
    rows = int(live.shape[0]) - s["pad"]  # the rows behind the last sequence go nowhere
    page, off = s["table"].long()[b[:rows], at[:rows] // s["page"]], at[:rows] % s["page"]
    s["kc"].view(_bits(s["kc"]))[page, :, off] = k[:rows].view(_bits(k))
    s["vc"].view(_bits(s["vc"]))[page, :, off] = v[:rows].view(_bits(v))
    out = [s["kc"], s["vc"]]
    if s["with_q"]:
        out.append(torch.where(live[:, None, None], _rotated(s, s["q"], "q", cos, sin), 0.0).to(s["q"].dtype))
    return out


def _bits(x):
    return torch.uint8 if x.element_size() == 1 else torch.int16


def _cached(s, name, scale):
    """The cache's rows of each sequence in order, (sequence, head, place, value) in 32 bits, nothing behind a sequence's end."""
    at = torch.arange(s["most_len"], device="cuda")
    c = s[name]
    x = c.view(_bits(c))[s["table"].long()[:, at // s["page"]].clamp(min=0), :, at % s["page"]].view(c.dtype).float()
    x = torch.where((at < s["lens"][:, None])[:, :, None, None], x, 0.0).permute(0, 2, 1, 3).contiguous()
    return x if scale is None else x * scale[:, None, None]


def _plain_attn(s):
    hq, hk, d, tokens, n = s["hq"], s["hk"], s["d"], s["q"].shape[0], s["most_new"]
    b, at, live = _places(s, tokens)
    k, v = _cached(s, "kc", s["ks"]), _cached(s, "vc", s["vs"])
    i = torch.arange(n, device="cuda")
    rows = (s["cu"].long()[:-1, None] + i).clamp(max=max(0, tokens - 1))  # (sequence, new token)
    q = s["q"].float()[rows].view(-1, n, hk, hq // hk, d).permute(0, 2, 3, 1, 4).reshape(-1, hk, hq // hk * n, d)
    z = torch.matmul(q, k.transpose(-1, -2).contiguous()).view(-1, hk, hq // hk, n, s["most_len"]) * s["scale"]
    new = (s["cu"][1:] - s["cu"][:-1])[:, None]
    place = (s["lens"][:, None] - new + i)[:, :, None]  # (sequence, new token, 1)
    key = torch.arange(s["most_len"], device="cuda")
    seen = (key < s["lens"][:, None])[:, None, :] & ((key <= place) if s["causal"] else (place > -(1 << 30)))
    seen = seen & (key > place - s["window"]) if s["window"] else seen
    z = z.masked_fill_(~seen[:, None, None], -math.inf)
    m = z.amax(-1, keepdim=True)
    p = (z.sub_(torch.where(m == -math.inf, 0.0, m))).exp_()
    l = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(-1, hk, hq // hk * n, s["most_len"]), v).view(-1, hk, hq // hk, n, d) / torch.where(l > 0, l, 1.0)
    lse = (m + l.log()).squeeze(-1)
    o = o.permute(0, 3, 1, 2, 4).reshape(-1, n, hq, d)
    lse = lse.permute(0, 3, 1, 2).reshape(-1, n, hq)
    off = (torch.arange(tokens, device="cuda") - s["cu"].long()[b]).clamp(max=n - 1)
    return [torch.where(live[:, None, None], o[b, off], 0.0).to(s["q"].dtype), torch.where(live[:, None], lse[b, off], -math.inf)]


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    if own:
        return _own(s)
    return {"rope": _plain_rope, "append": _plain_append, "attn": _plain_attn}[s["op"]](s)


def _own(s):
    from hma_amd import ops
    from hma_amd import torch_ops  # noqa: F401

    if s["op"] == "attn":
        return ops.attn_paged_fwd(s["q"], s["kc"], s["vc"], s["table"], s["cu"], s["lens"], s["scale"], causal=s["causal"], window=s["window"],
                                  k_scale=s["ks"], v_scale=s["vs"])
    if s["op"] == "append":
        of_q = dict(q=s["q"], q_weight=s["qw"], q_bias=s["qb"]) if s["with_q"] else {}  # (its weights without it are refused)
        q = ops.kv_append(s["k"], s["v"], s["kc"], s["vc"], s["table"], s["cu"], s["lens"], **of_q, freqs=s["freqs"], positions=s["pos"],
                          axes=s["axes"], interleaved=s["inter"], amplitude=s["amp"], norm=s["norm"], k_weight=s["kw"], k_bias=s["kb"],
                          eps=s["eps"], k_scale=s["ks"], v_scale=s["vs"])
        return [s["kc"], s["vc"]] + ([q] if s["with_q"] else [])
    if not s["grad"]:
        return ops.qk_rope_fwd(s["q"], s["k"], s["freqs"], s["pos"], axes=s["axes"], interleaved=s["inter"], amplitude=s["amp"], norm=s["norm"],
                               q_weight=s["qw"], q_bias=s["qb"], k_weight=s["kw"], k_bias=s["kb"], eps=s["eps"])
    leaves = iter(s["leaves"])
    q, k = next(leaves), next(leaves)
    qw, qb, kw, kb = (None if s[n] is None else next(leaves) for n in ("qw", "qb", "kw", "kb"))
    y = torch.ops.hma.qk_rope(q, k, s["freqs"], s["pos"], s["axes"], s["inter"], s["amp"], s["norm"], qw, qb, kw, kb, s["eps"])
    d = torch.autograd.grad(y, s["leaves"], [s["gq"], s["gk"]])
    n = 1 + (s["qw"] is not None) + (s["qb"] is not None)  # in the plain form's order: all of q's, then all of k's
    return [x.detach() for x in y] + [d[0], *d[2 : 1 + n], d[1], *d[1 + n :]]


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(c):
    e, row = (4 if c["type"] == "fp32" else 2), c["d"]
    if c["op"] == "rope":
        one = c["tokens"] * (c["hq"] + c["hk"]) * row * e
        return {"bytes": one * (4 if c["grad"] else 2) + 8 * c["axes"] * c["tokens"], "flops": one // e * (30 if c["grad"] else 10)}
    new, lens = _lengths(c)
    kept = 1 if c["cache"] == "e4m3" else e
    if c["op"] == "append":
        n = sum(new)
        return {"bytes": n * row * (2 * c["hk"] * (e + kept) + (2 * c["hq"] * e if c["with_q"] else 0)), "flops": n * row * 10 * (c["hq"] + c["hk"])}
    pairs = read = 0
    for n, m in zip(new, lens):
        lo, hi = m - n, m  # places of the new tokens
        w = c["window"] or m
        pairs += sum(min(p + 1, w) for p in range(lo, hi)) if c["causal"] else n * m
        read += m - max(0, lo + 1 - w) if n else 0
    return {"bytes": read * 2 * c["hk"] * row * kept + sum(new) * c["hq"] * (2 * row * e + 4), "flops": 4 * row * c["hq"] * pairs}


# ------------------------------------------------------------------------------------------------ from the definitions, in 64 bits
def _exact_rows(s, x, h, pos):
    """One head's rows (tokens, d) at positions (tokens, pairs), each normed and rotated as complex numbers."""
    x = x.double()
    if s["norm"] == "layer":
        x = (x - x.mean(-1, keepdim=True)) / (x.var(-1, unbiased=False, keepdim=True) + s["eps"]).sqrt()
    elif s["norm"] == "rms":
        x = x / (x.pow(2).mean(-1, keepdim=True) + s["eps"]).sqrt()
    if s[h + "w"] is not None:
        x = x * s[h + "w"].double()
    if s[h + "b"] is not None:
        x = x + s[h + "b"].double()
    r = s["rot"]
    pair = x[:, :r].reshape(-1, r // 2, 2) if s["inter"] else x[:, :r].reshape(-1, 2, r // 2).transpose(1, 2)
    z = torch.view_as_complex(pair.contiguous()) * torch.polar(torch.full_like(pos, s["amp"]), pos)
    z = torch.view_as_real(z)
    z = z.reshape(-1, r) if s["inter"] else z.transpose(1, 2).reshape(-1, r)
    return torch.cat([z, x[:, r:]], 1)


def _exact_positions(s, pos):
    pos = pos.double()
    if pos.dim() == 2:
        return torch.stack([pos[int(a)] for a in s["axes"]], 1) * s["freqs"]
    return pos[:, None] * s["freqs"][None]


def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] == "rope":
        pos = _exact_positions(s, s["pos"])
        out, grads = [], []
        for h, g in (("q", "gq"), ("k", "gk")):
            for n in (h, h + "w", h + "b"):
                if s[n] is not None:
                    s[n] = s[n].double().requires_grad_(c["grad"])
            y = torch.stack([_exact_rows(s, s[h][:, j], h, pos) for j in range(s[h].shape[1])], 1)
            if c["grad"]:
                grads += torch.autograd.grad(y, [s[n] for n in (h, h + "w", h + "b") if s[n] is not None], s[g].double())
            out.append(y.detach())
        return out + grads
    new, lens = _lengths(c)
    page, table = c["page"], s["table"].tolist()
    if c["op"] == "append":
        kc, vc = s["kc"].double(), s["vc"].double()
        qo, at = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), 0
        for b, (n, m) in enumerate(zip(new, lens)):
            place = torch.arange(m - n, m, device="cuda")
            pos = _exact_positions(s, place if s["pos"] is None else s["pos"][..., at : at + n])
            pg, off = s["table"][b].long()[place // page], place % page
            for j in range(c["hk"]):
                k, v = _exact_rows(s, s["k"][at : at + n, j], "k", pos), s["v"][at : at + n, j].double()
                if s["ks"] is not None:
                    k, v = (k / s["ks"][j].double()).clamp(-F8_MAX, F8_MAX), (v / s["vs"][j].double()).clamp(-F8_MAX, F8_MAX)
                kc[pg, j, off], vc[pg, j, off] = k, v
            if c["with_q"]:
                for j in range(c["hq"]):
                    qo[at : at + n, j] = _exact_rows(s, s["q"][at : at + n, j], "q", pos)
            at += n
        return [kc, vc] + ([qo] if c["with_q"] else [])
    o = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    at, group = 0, c["hq"] // c["hk"]
    for b, (n, m) in enumerate(zip(new, lens)):
        pg = torch.tensor(table[b][: -(-m // page)], dtype=torch.long, device="cuda")
        key = torch.arange(m, device="cuda")[None]
        me = torch.arange(m - n, m, device="cuda")[:, None]
        hidden = key > me if c["causal"] else key < 0
        hidden = hidden | (me - key >= c["window"]) if c["window"] else hidden
        for j in range(c["hk"]):
            k, v = (s[x][pg, j].double().reshape(-1, c["d"])[:m] * (1.0 if z is None else z[j].double()) for x, z in (("kc", s["ks"]), ("vc", s["vs"])))
            for h in range(j * group, (j + 1) * group):
                z = (s["q"][at : at + n, h].double() @ k.t() * s["scale"]).masked_fill(hidden, -math.inf)
                lse[at : at + n, h] = torch.logsumexp(z, 1)
                o[at : at + n, h] = torch.softmax(z, 1) @ v
        at += n
    return [o, lse]
