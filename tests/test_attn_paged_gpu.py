"""hma_amd.ops.attn_paged_fwd on the GPU against softmax attention in 64 bits, and a run of kv_append + attn_paged as a rollout makes it."""
import ctypes as C
import math

import pytest
import torch

import hma_amd.torch_ops  # noqa: F401
from hma_amd import _lib, ops
from tests import rope_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF = torch.bfloat16, torch.float16
F8 = torch.float8_e4m3fn


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def batch(new, lens, page, hq, hk, d, dtype, f8=False, tail=0, seed=0, extra=3, poison=True):
    """A cache whose every place that is no sequence's own holds a NaN."""
    g = gen(seed)
    need = [-(-max(n, 0) // page) for n in lens]
    pages = sum(need) + extra
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    table = torch.full((len(lens), max(need + [1]) + 1), -1, dtype=torch.int32, device=DEV)
    kc = torch.full((pages, hk, page, d), float("nan") if poison else 0.0, device=DEV)
    vc = kc.clone()
    at, ks, vs = 0, [], []
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
        m = max(lens[b], 0)
        k, v = (torch.randn(hk, m, d, generator=g, device=DEV) for _ in range(2))
        if m:
            pl = torch.arange(m, device=DEV)
            pg = table[b].long()[pl // page]
            kc[pg, :, pl % page], vc[pg, :, pl % page] = k.transpose(0, 1), v.transpose(0, 1)
    s = dict(table=table, cu=torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32, device=DEV),
             lens=torch.tensor(lens, dtype=torch.int32, device=DEV), new=new, lengths=lens, page=page)
    if f8:
        s["k_scale"], s["v_scale"] = (0.01 + 0.01 * torch.rand(hk, generator=g, device=DEV) for _ in range(2))
        kc, vc = ((c / s[n][:, None, None]).to(F8) for c, n in ((kc, "k_scale"), (vc, "v_scale")))
    else:
        kc, vc = kc.to(dtype), vc.to(dtype)
        s["k_scale"] = s["v_scale"] = None
    s["kc"], s["vc"] = kc, vc
    s["q"] = torch.randn(sum(new) + tail, hq, d, generator=g, device=DEV).to(dtype)
    return s


def call(s, scale, causal=True, window=0, **kw):
    return ops.attn_paged_fwd(s["q"], s["kc"], s["vc"], s["table"], s["cu"], s["lens"], scale, causal=causal, window=window, k_scale=s["k_scale"],
                              v_scale=s["v_scale"], **kw)


def check(s, got, scale, causal, window):
    o, lse = got
    q, page = s["q"], s["page"]
    hq, d, hk = q.shape[1], q.shape[2], s["kc"].shape[1]
    u = R.U[q.dtype]
    at = 0
    for b, (n, m) in enumerate(zip(s["new"], s["lengths"])):
        if n == 0:
            continue
        pl = torch.arange(max(m, 0), device=DEV)
        pg = s["table"][b].long()[pl // page] if m > 0 else pl
        here = (pg >= 0) & (pg < s["kc"].shape[0])
        pg = torch.where(here, pg, 0)
        k, v = (s[c][pg, :, pl % page].double().transpose(0, 1) for c in ("kc", "vc"))  # (hk, m, d)
        k, v = (torch.where(here[None, :, None], x, 0.0) for x in (k, v))
        if s["k_scale"] is not None:
            k, v = k * s["k_scale"].double()[:, None, None], v * s["v_scale"].double()[:, None, None]
        place = torch.arange(m - n, m, device=DEV)[:, None]
        seen = (pl[None] <= place) if causal else torch.ones(n, max(m, 0), dtype=torch.bool, device=DEV)
        if window:
            seen = seen & (pl[None] > place - window)
        seen = seen & here[None]
        for h in range(hq):
            j = h // (hq // hk)
            x = q[at:at + n, h].double()
            z = (x @ k[j].t() * scale).masked_fill(~seen, -math.inf)
            big = x.abs() @ k[j].abs().t() * scale
            none = ~seen.any(1)
            p = torch.softmax(z, 1).masked_fill(none[:, None], 0.0) if m > 0 else z
            ref, rl = p @ v[j], torch.logsumexp(z, 1) if m > 0 else torch.full((n,), -math.inf, dtype=torch.float64, device=DEV)
            # a score: d products summed in 32 bits, scaled twice; its exponential: the hardware's 1 ulp and the argument's rounding; the
            # row sum: chains of a fourth of the keys.  Relative error of a probability / absolute error of lse:
            count = seen.sum(1)
            e32 = (d + 8) * R.F32U * big.masked_fill(~seen, 0.0).amax(1) + 8 * R.F32U * rl.abs().masked_fill(none, 0.0) + (count / 4 + 128) * R.F32U if m > 0 else torch.zeros(n, device=DEV, dtype=torch.float64)
            pv = p @ v[j].abs()
            bound = u * ref.abs() + (u + 2 * e32)[:, None] * pv * (1 + u)
            if q.dtype == HF:  # probabilities below 2^-14 of the largest are fp16 subnormals: off by 2^-25 each
                bound = bound + 2.0 ** -25 * (seen.double() @ v[j].abs()) + 2.0 ** -25
            # a value over 448 scales is a NaN in e4m3 (the cast does not clamp): where the definition gives a NaN, a NaN is wanted
            mine = o[at:at + n, h].double()
            assert torch.equal(mine.isnan(), ref.isnan()), (b, h)
            off = ((mine - ref).abs() - bound).masked_fill(ref.isnan(), 0.0)
            assert bool((off <= 0).all()), (b, h, float(off.max()))
            gl = lse[at:at + n, h].double()
            assert torch.equal(gl == -math.inf, none) and torch.equal(gl.isnan(), rl.isnan()), (b, h)
            some = ~none & ~rl.isnan()
            assert bool(((gl - rl).abs()[some] <= e32[some]).all()), (b, h, float((gl - rl).abs()[some].max()))
            assert not o[at:at + n, h][none].any()
        at += n
    assert not o[at:].any() and bool((lse[at:] == -math.inf).all())


CASES = {  # new, lens, page, hq, hk, causal, window, tail
    "one": ([1], [1], 16, 8, 8, True, 0, 0),
    "one long": ([1], [3001], 16, 8, 2, True, 0, 0),
    "decode": ([1] * 9, [1, 2, 31, 32, 33, 127, 128, 129, 700], 16, 8, 1, True, 0, 3),
    "idle and empty": ([1, 0, 1, 1, 0], [64, 9, 0, 513, 0], 64, 4, 2, True, 0, 2),
    "all empty": ([1, 1], [0, 0], 8, 2, 2, True, 0, 0),
    "group of 3": ([2, 3, 1], [77, 3, 260], 7, 6, 2, True, 0, 0),
    "group of 32": ([1, 1], [300, 45], 16, 32, 1, True, 0, 1),
    "window": ([1, 1, 5], [300, 40, 500], 16, 4, 4, True, 64, 0),
    "window of 1": ([1, 40], [300, 90], 16, 4, 4, True, 1, 0),
    "chunks": ([130, 1, 64, 257], [130, 400, 64, 1000], 16, 4, 2, True, 0, 5),
    "chunk window": ([200, 33], [700, 33], 32, 3, 3, True, 50, 0),
    "frame": ([320, 320], [320, 1600], 320, 8, 8, False, 0, 0),
    "frame few": ([4, 4, 4], [4, 300, 77], 1, 2, 2, False, 0, 1),
    "more new than cached": ([40, 3], [25, 1], 16, 4, 2, True, 0, 0),
    "pages of 48": ([17, 90], [500, 91], 48, 5, 1, True, 0, 0),
}


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("name", list(CASES))
def test_values(name, d):
    new, lens, page, hq, hk, causal, window, tail = CASES[name]
    for dtype, f8 in ((BF, False), (HF, False), (BF, True), (HF, True)):
        s = batch(new, lens, page, hq, hk, d, dtype, f8, tail, seed=d)
        scale = d ** -0.5
        got = call(s, scale, causal, window)
        assert got[0].is_contiguous() and got[0].dtype == dtype and got[1].dtype == torch.float32
        check(s, got, scale, causal, window)
        again = call(s, scale, causal, window)
        assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])


@pytest.mark.parametrize("d,hq,hk,new,lens", [(128, 32, 8, [3000, 1300], [3000, 1900]), (32, 64, 64, [700, 1], [700, 900]), (64, 20, 10, [7001], [7001])])
def test_whole_prompts(d, hq, hk, new, lens):
    """Enough row tiles that nothing is split."""
    s = batch(new, lens, 32, hq, hk, d, BF, seed=3)
    check(s, call(s, d ** -0.5), d ** -0.5, True, 0)


def test_large_scores_and_ties():
    s = batch([1, 70], [500, 300], 16, 4, 2, 64, BF, seed=5)
    s["q"] = s["q"] * 30  # scores of +-100s: one key takes nearly everything, the running maximum jumps
    check(s, call(s, 0.5), 0.5, True, 0)
    s["q"].zero_()
    check(s, call(s, 0.5), 0.5, True, 0)


def test_pages_outside_the_cache():
    s = batch([1, 130, 2], [200, 260, 90], 16, 4, 2, 64, BF, seed=6)
    s["table"][0, 3] = -7
    s["table"][1, 0] = 10 ** 9
    s["table"][1, 16] = s["kc"].shape[0]
    s["table"][2] = -1  # nothing of this sequence is there
    check(s, call(s, 0.125), 0.125, True, 0)
    short = dict(s, table=s["table"][:, :10].contiguous())  # places from 160 on have no page
    o, lse = call(short, 0.125)
    ref = dict(s, table=torch.cat([s["table"][:, :10], torch.full_like(s["table"][:, 10:], -1)], 1))
    check(ref, (o, lse), 0.125, True, 0)


def test_what_no_row_of_a_tile_sees_is_not_read():
    """Keys and values left of the window, and all of another sequence, hold NaN and infinities."""
    for f8 in (False, True):
        s = batch([1, 1], [600, 90], 16, 8, 2, 64, BF, f8, seed=7)
        want = call(s, 0.125, True, 100)
        for c in ("kc", "vc"):
            pg = s["table"][0].long()[:31]  # places 0 .. 495; the row at 599 sees 500 .. 599
            s[c].view(torch.uint8 if f8 else torch.int16)[pg] = -1  # NaN in both types
            if not f8:
                s[c][pg[::2]] = float("inf")
        got = call(s, 0.125, True, 100)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("tokens", [1, 3, 300])
def test_no_sequences(tokens):
    s = batch([], [], 16, 4, 2, 32, BF, tail=tokens)
    o, lse = call(s, 0.2)
    assert o.shape == (tokens, 4, 32) and not o.any() and bool((lse == -math.inf).all())
    mine = torch.full_like(o, 3.0), torch.full_like(lse, 3.0)
    call(s, 0.2, out=mine[0], lse=mine[1])
    assert bool((mine[0] == 3).all() and (mine[1] == 3).all())


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("new,lens", [([1, 1], [300, 77]), ([200, 70], [500, 70]), ([3000], [3000])])
def test_rows_that_are_no_numbers_stay_their_own(new, lens, d):
    """A query row with a NaN or an infinity: NaN there (one key's score is a NaN or both signs are infinite), every other row as without."""
    s = batch(new, lens, 16, 4, 2, d, BF, seed=13)
    want = call(s, 0.125)
    q = s["q"].clone()
    q[0, 0], q[-1, 3], q[-1, 1, 5] = float("nan"), float("inf"), float("nan")
    o, lse = call(dict(s, q=q), 0.125)
    odd = torch.zeros(q.shape[:2], dtype=torch.bool, device=DEV)
    odd[0, 0] = odd[-1, 3] = odd[-1, 1] = True
    assert bool(o[odd].isnan().all()) and bool(lse[odd].isnan().all())
    assert torch.equal(o[~odd], want[0][~odd]) and torch.equal(lse[~odd], want[1][~odd])


def test_two_calls_at_once():
    a, b = batch([1, 1, 1], [700, 900, 333], 16, 8, 2, 128, BF, seed=14), batch([140, 2], [700, 500], 16, 8, 2, 128, BF, seed=15)
    want = [call(x, 0.09) for x in (a, b)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, x in enumerate((a, b)):
            with torch.cuda.stream(streams[i]):
                got[i].append(call(x, 0.09))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g[0], want[i][0]) and torch.equal(g[1], want[i][1]) for g in got[i])


def test_strides_and_streams():
    s = batch([3, 1, 200], [70, 300, 333], 16, 8, 4, 64, BF, seed=8)
    want = call(s, 0.125)
    packed = torch.randn(204, 8 * 64 * 2, device=DEV).to(BF)
    packed[:, :512] = s["q"].reshape(204, 512)
    by_token = {c: s[c].transpose(1, 2).contiguous().transpose(1, 2) for c in ("kc", "vc")}  # pages of (token, head) order
    wide = torch.full((3, 40), 99, dtype=torch.int32, device=DEV)
    wide[:, :s["table"].shape[1]] = s["table"]
    for t in (dict(s, q=packed[:, :512].view(204, 8, 64)), dict(s, **by_token), dict(s, table=wide[:, :s["table"].shape[1]]),
              dict(s, q=s["q"].transpose(0, 1).contiguous().transpose(0, 1))):
        got = call(t, 0.125)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    both = torch.stack([s["kc"], s["vc"]], 1)  # one buffer, pages of [keys | values]
    got = call(dict(s, kc=both[:, 0], vc=both[:, 1]), 0.125)
    assert torch.equal(got[0], want[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call(s, 0.125)
    side.synchronize()
    assert torch.equal(got[0], want[0])
    out, lse = torch.full_like(want[0], 5.0), torch.full_like(want[1], 5.0)
    t = dict(s, cu=torch.tensor([0, 3, 4, 4], dtype=torch.int32, device=DEV))  # the third sequence is gone: 200 rows behind the last
    call(t, 0.125, out=out, lse=lse)
    assert torch.equal(out[:4], want[0][:4]) and bool((out[4:] == 5).all()) and bool((lse[4:] == 5).all())
    o, l = call(dict(s, q=s["q"][:0], cu=torch.zeros(4, dtype=torch.int32, device=DEV)), 0.125)
    assert o.shape == (0, 8, 64) and l.shape == (0, 8)
    o, l = ops.attn_paged_fwd(s["q"], s["kc"], s["vc"], s["table"][:0], s["cu"][:1], s["lens"][:0], 0.125)
    assert not o.any() and bool((l == -math.inf).all())


def test_custom_op_and_two_graphs():
    s = batch([1, 1, 1], [70, 900, 333], 16, 8, 2, 128, BF, seed=9, poison=False)
    t = batch([40, 2], [70, 500], 16, 8, 2, 128, BF, seed=10, poison=False)

    def run(x):
        return torch.ops.hma.attn_paged(x["q"], x["kc"], x["vc"], x["table"], x["cu"], x["lens"], 0.09, True, 0, None, None)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(s), run(t)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for x in (s, t):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(run(x))
        graphs.append(g)
    for i in range(3):
        for x in (s, t):
            x["lens"].sub_(7)
            x["q"].mul_(1.5)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for x, y in zip((s, t), outs):
            want = run(x)
            torch.cuda.synchronize()
            assert torch.equal(y[0], want[0]) and torch.equal(y[1], want[1])


@pytest.mark.parametrize("f8", [False, True])
def test_many_sequences(f8):
    lens = [(37 * i) % 211 for i in range(1500)]
    s = batch([1 if i % 5 else 0 for i in range(1500)], lens, 16, 2, 1, 32, BF, f8, seed=11)
    check(s, call(s, 0.2), 0.2, True, 0)


def test_offsets_past_32_bits():
    """A cache of more than 2^32 elements a tensor, the sequence's pages at its far end."""
    page, hk, d = 64, 8, 128
    pages = 2 ** 32 // (page * hk * d) + 40
    kc = torch.empty(pages, hk, page, d, dtype=F8, device=DEV)
    vc = torch.empty(pages, hk, page, d, dtype=F8, device=DEV)
    s = batch([2, 100], [300, 900], page, 16, hk, d, BF, True, seed=12)
    n = s["kc"].shape[0]
    kc[-n:].view(torch.uint8).copy_(s["kc"].view(torch.uint8))
    vc[-n:].view(torch.uint8).copy_(s["vc"].view(torch.uint8))
    want = call(s, 0.09)
    far = dict(s, kc=kc, vc=vc, table=torch.where(s["table"] >= 0, s["table"] + (pages - n), s["table"]))
    got = call(far, 0.09)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    k = torch.randn(102, hk, d, device=DEV).to(BF)
    ops.kv_append(k, k, kc, vc, far["table"], s["cu"], s["lens"], k_scale=s["k_scale"], v_scale=s["v_scale"])
    ops.kv_append(k, k, s["kc"], s["vc"], s["table"], s["cu"], s["lens"], k_scale=s["k_scale"], v_scale=s["v_scale"])
    assert torch.equal(kc[-n:].view(torch.uint8), s["kc"].view(torch.uint8)) and torch.equal(vc[-n:].view(torch.uint8), s["vc"].view(torch.uint8))


# ------------------------------------------------------------------------------------------------ as a rollout makes it
def test_rollout():
    """Three rollouts of different lengths: a prompt each, two frames whose tokens see each other, then single tokens, all through kv_append +
    attn_paged; against dense attention in 64 bits over the normed, rotated rows of the whole history."""
    g, page, hq, hk, d, frame = gen(20), 16, 8, 2, 64, 24
    freqs, amp = ops.rope_freqs(32, scaling="parts", factor=4.0, trained=64, device=DEV)
    qw, kw = (1 + 0.1 * torch.randn(d, generator=g, device=DEV) for _ in range(2))
    B, lens = 3, [0, 0, 0]
    table = torch.randperm(64, generator=g, device=DEV).to(torch.int32)[:48].view(B, 16).contiguous()
    kc, vc = (torch.full((64, hk, page, d), float("nan"), dtype=BF, device=DEV) for _ in range(2))
    hist = [[] for _ in range(B)]
    for step, (news, causal) in enumerate([([33, 5, 70], True), ([frame] * 3, False), ([frame] * 3, False), ([1, 1, 1], True), ([1, 0, 1], True)]):
        n = sum(news)
        qkv = torch.randn(n, (hq + 2 * hk) * d, generator=g, device=DEV).to(BF)
        q, k, v = qkv[:, :hq * d].view(n, hq, d), qkv[:, hq * d:(hq + hk) * d].view(n, hk, d), qkv[:, (hq + hk) * d:].view(n, hk, d)
        lens = [a + b for a, b in zip(lens, news)]
        cu = torch.tensor([sum(news[:b]) for b in range(B + 1)], dtype=torch.int32, device=DEV)
        kv = torch.tensor(lens, dtype=torch.int32, device=DEV)
        qr = ops.kv_append(k, v, kc, vc, table, cu, kv, q=q, freqs=freqs, amplitude=amp, norm="rms", q_weight=qw, k_weight=kw)
        o, lse = ops.attn_paged_fwd(qr, kc, vc, table, cu, kv, d ** -0.5, causal=causal)
        at = 0
        for b in range(B):
            hist[b].append((k[at:at + news[b]], v[at:at + news[b]]))
            m, x = lens[b], q[at:at + news[b]]
            if news[b]:
                kk, vv = (torch.cat([h[i] for h in hist[b]]).double() for i in (0, 1))
                cs = R.table(freqs, torch.arange(m, device=DEV), None, m, DEV)
                kk = R.qk_rope(kk, cs, False, amp, "rms", kw, None, 1e-5)
                tail = tuple(t[m - news[b]:] for t in cs)
                xx = R.qk_rope(x.double(), tail, False, amp, "rms", qw, None, 1e-5)
                seen = torch.arange(m, device=DEV)[None] <= torch.arange(m - news[b], m, device=DEV)[:, None] if causal else torch.ones(news[b], m, dtype=torch.bool, device=DEV)
                for h in range(hq):
                    z = (xx[:, h] @ kk[:, h // 4].t() * d ** -0.5).masked_fill(~seen, -math.inf)
                    p = torch.softmax(z, 1)
                    ref, pv = p @ vv[:, h // 4], p @ vv[:, h // 4].abs()
                    # q and k are rounded to bf16 (2^-8 each): a score moves by at most 2.1 * 2^-8 * scale |q| |k|; p by that, relative, twice
                    e = 2.1 * 2.0 ** -8 * (xx[:, h].abs() @ kk[:, h // 4].abs().t() * d ** -0.5).amax(1)
                    bound = 2.0 ** -8 * ref.abs() + (2 * e.exp().sub(1) + 2.0 ** -8 + 1e-4)[:, None] * pv * 1.01
                    assert bool(((o[at:at + news[b], h].double() - ref).abs() <= bound).all()), (step, b, h)
                    rms = float((o[at:at + news[b], h].double() - ref).norm() / ref.norm())
                    assert rms < 2e-2, (step, b, h, rms)  # what independent roundings of that size leave of the bound
            at += news[b]


@pytest.mark.parametrize("hq,new,lens", [(64, [1, 3], [70, 300]), (160, [2, 1, 9], [40, 130, 9]), (160, [1], [1])])
def test_groups_larger_than_a_tile_of_rows(hq, new, lens):
    for window in (0, 20):
        s = batch(new, lens, 16, hq, 1, 64, BF, seed=30, tail=1)
        check(s, call(s, 0.125, True, window), 0.125, True, window)


def test_the_most_sequences():
    lens = [(13 * i) % 70 for i in range(4096)]
    s = batch([1] * 4096, lens, 16, 1, 1, 64, HF, seed=31)
    got = call(s, 0.125)
    for lo in (0, 2040, 4090):  # against calls of six sequences each
        part = dict(s, q=s["q"][lo:lo + 6], table=s["table"][lo:lo + 6], lens=s["lens"][lo:lo + 6], cu=torch.arange(7, dtype=torch.int32, device=DEV),
                    new=[1] * 6, lengths=lens[lo:lo + 6])
        check(part, (got[0][lo:lo + 6], got[1][lo:lo + 6]), 0.125, True, 0)
    with pytest.raises(RuntimeError):
        call(batch([1] * 4097, [1] * 4097, 16, 1, 1, 64, HF), 0.125)


def test_windows_beyond_every_length():
    for new, lens in (([1, 3], [700, 90]), ([200, 70], [500, 70])):
        s = batch(new, lens, 16, 4, 2, 64, BF, seed=42)
        want = call(s, 0.125)
        for window in (10 ** 6, 2 ** 31 - 1, 2 ** 31, 2 ** 40):
            got = call(s, 0.125, True, window)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), window


# (heads, key heads, sequences, new tokens of each, keys): few rows in many shares and in few, many rows split along the keys, unsplit
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("hq,hk,seqs,n,m", [(4, 1, 1, 1, 131072), (8, 8, 96, 1, 131072), (8, 8, 30, 40, 131072), (96, 96, 1, 2700, 40000)])
@pytest.mark.parametrize("sink", ["first", "last", "inside"])
def test_what_a_far_larger_score_leaves_of_fp16(d, hq, hk, seqs, n, m, sink):
    """One key takes nearly all of the weight and has a value of zero: the output is what the others, up to 20 powers of e behind it, add up to.
    All rows are alike: with w = e^-gap, o = w sum v / (1 + (m - 1) w)."""
    at = {"first": 0, "last": m - 1, "inside": m // 3}[sink]
    g, page = gen(40), 64
    for f8 in (False, True):
        pages = -(-m // page)
        kc = torch.zeros(pages, hk, page, d, dtype=HF, device=DEV)
        vc = (0.5 + torch.rand(pages, 1, page, d, generator=g, device=DEV)).to(HF)
        vc = (vc.to(F8) if f8 else vc).expand(pages, hk, page, d).contiguous()
        kc[at // page, :, at % page, 0] = 16.0
        vc.view(torch.uint8 if f8 else torch.int16)[at // page, :, at % page] = 0
        kc = kc.to(F8) if f8 else kc
        one = dict(k_scale=torch.ones(hk, device=DEV), v_scale=torch.ones(hk, device=DEV)) if f8 else {}
        q = torch.zeros(seqs * n, hq, d, dtype=HF, device=DEV)
        q[..., 0] = 1.0
        table = torch.arange(pages, dtype=torch.int32, device=DEV)[None].expand(seqs, pages)  # the same history
        cu, lens = torch.arange(seqs + 1, dtype=torch.int32, device=DEV) * n, torch.full((seqs,), m, dtype=torch.int32, device=DEV)
        v = vc[:, 0].reshape(-1, d)[:m].double()
        for gap in (8.0, 14.0, 17.0, 20.0):
            o, lse = ops.attn_paged_fwd(q, kc, vc, table, cu, lens, gap / 16, causal=False, **one)
            w = math.exp(-gap)
            ref, rl = w * v.sum(0) / (1 + (m - 1) * w), gap + math.log1p((m - 1) * w)
            # check()'s bound, with probabilities held down to 2^-24 of fp16 at 2^10 for the largest: off by 2^-35 of it each
            e32 = (d + 8) * R.F32U * gap + 8 * R.F32U * rl + (m / 4 + 128) * R.F32U
            bound = (2 * R.U[HF] + 2 * e32) * ref * (1 + R.U[HF]) + 2.0 ** -35 * v.sum(0) + 2.0 ** -25
            off = (o.double() - ref).abs() - bound
            assert bool((off <= 0).all()), (f8, gap, float(((o.double() - ref).abs() / ref).max()))
            assert float((lse.double() - rl).abs().max()) <= e32, (f8, gap)


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("new,lens", [([1, 2], [700, 500]), ([200, 70], [900, 700]), ([300] * 60, [300 + 7 * i for i in range(60)])])
def test_fp16_scores_that_rise_along_the_keys(new, lens, d):
    """Every block's largest score exceeds all before it, by less and by more than what the running maximum tolerates."""
    for hk, f8 in ((2, False), (8, False), (2, True)):
        for slope in (0.002, 0.03, 0.3, 3.0):
            s = batch(new, lens, 16, 2 * hk, hk, d, HF, f8, seed=41)
            s["q"][..., 0] = 1.0
            for b, m in enumerate(lens):
                pl = torch.arange(m, device=DEV)
                rise = (slope * pl / d ** -0.5).clamp(max=400.0 if f8 else 3e4)
                if f8:
                    s["kc"][s["table"][b].long()[pl // 16], :, pl % 16, 0] = (rise[:, None] / s["k_scale"]).clamp(max=448).to(F8)
                else:
                    s["kc"][s["table"][b].long()[pl // 16], :, pl % 16, 0] = rise[:, None].to(HF)
            check(s, call(s, d ** -0.5), d ** -0.5, True, 0)


def workspace(s, causal=True, window=0):
    """Bytes that a call wants; none: its row tiles are not split along the keys."""
    q, kc, n = s["q"], s["kc"], C.c_int64()
    p = _lib.AttnPaged(tokens=q.shape[0], hq=q.shape[1], hk=kc.shape[1], d=q.shape[2], dtype=0 if q.dtype == BF else 1, seqs=len(s["new"]),
                       table_w=s["table"].shape[1], pages=kc.shape[0], page=kc.shape[2], cache_e4m3=kc.dtype == F8, causal=causal, window=window, scale=1.0)
    _lib.check(_lib.load().hma_attn_paged_ws(C.byref(p), C.byref(n)), "hma_attn_paged_ws")
    return n.value


UNSPLIT = {  # heads, key heads, new, lens, page, causal, window, tail
    "one prompt": (140, 140, [1950], [1950], 32, True, 0, 0),
    "a prompt behind a past": (160, 160, [1801, 1], [2500, 70], 16, True, 0, 3),
    "many sequences, some idle": (17, 17, [0, 45, 80, 0, 45] * 24, [900, 45, 300, 0, 150] * 24, 16, True, 0, 5),
    "odd pages": (34, 17, [33, 47, 0] * 40, [33, 130, 12] * 40, 7, True, 0, 0),
    "window": (17, 17, [90, 45] * 60, [400, 45] * 60, 16, True, 30, 1),
    "frames": (17, 17, [64] * 120, [64 * (1 + i % 5) for i in range(120)], 64, False, 0, 2),
    "more new than cached": (17, 17, [70, 40] * 60, [50, 1] * 60, 48, True, 0, 0),
}


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("name", list(UNSPLIT))
def test_row_tiles_that_are_not_split(name, d):
    hq, hk, new, lens, page, causal, window, tail = UNSPLIT[name]
    for dtype, f8 in ((BF, False), (HF, False), (BF, True), (HF, True)):
        s = batch(new, lens, page, hq, hk, d, dtype, f8, tail, seed=50 + d)
        assert workspace(s, causal, window) == 0
        o, lse = call(s, d ** -0.5, causal, window)
        some = [0, hk // 2, hk - 1]  # key heads looked at, with the heads that share them
        rows = [j * (hq // hk) + i for j in some for i in range(hq // hk)]
        part = dict(s, q=s["q"][:, rows], kc=s["kc"].view(torch.uint8 if f8 else dtype)[:, some].view(s["kc"].dtype),
                    vc=s["vc"].view(torch.uint8 if f8 else dtype)[:, some].view(s["vc"].dtype))
        if f8:
            part |= dict(k_scale=s["k_scale"][some], v_scale=s["v_scale"][some])
        check(part, (o[:, rows], lse[:, rows]), d ** -0.5, causal, window)
