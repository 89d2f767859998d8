"""hma_amd.ops.qk_rope_fwd / qk_rope_bwd / kv_append and their custom ops on the GPU, against the formulas in 64 bits."""
import itertools

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

import hma_amd.torch_ops  # noqa: F401
from hma_amd import ops
from tests import rope_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
F8 = torch.float8_e4m3fn


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def make(tokens, hq, hk, d, rot, kind, dtype, wdtype=None, axes=1, far=5000, seed=0, int32=False, freqs=True):
    g = gen(seed)
    x = (1.3 * torch.randn(tokens, (hq + 2 * hk) * d, generator=g, device=DEV) + 0.3).to(dtype)
    q, k, v = x[:, :hq * d].view(tokens, hq, d), x[:, hq * d:(hq + hk) * d].view(tokens, hk, d), x[:, (hq + hk) * d:].view(tokens, hk, d)
    s = dict(q=q, k=k, v=v, freqs=ops.rope_freqs(rot, device=DEV)[0] if rot and freqs else None, axes=None)
    pos = torch.randint(-3, far, (axes, tokens), generator=g, device=DEV)
    s["positions"] = (pos if axes > 1 else pos[0]).to(torch.int32 if int32 else torch.int64)
    if axes > 1:
        s["axes"] = torch.randint(0, axes, (rot // 2,), generator=g, device=DEV).to(torch.int32)
    wdtype = wdtype or F32
    for n in ("q_weight", "k_weight"):
        s[n] = (1 + 0.3 * torch.randn(d, generator=g, device=DEV)).to(wdtype) if kind != "none" else None
    for n in ("q_bias", "k_bias"):
        s[n] = (0.2 * torch.randn(d, generator=g, device=DEV)).to(wdtype) if kind == "layer" else None
    return s


def kwargs(s, kind, inter, amp):
    return dict(axes=s["axes"], interleaved=inter, amplitude=amp, norm=kind, eps=1e-5, **{n: s[n] for n in ("q_weight", "q_bias", "k_weight", "k_bias")})


def close(got, ref, bound):
    assert got.shape == ref.shape
    off = (got.double() - ref).abs() - bound
    assert bool((off <= 0).all()), float(off.max())  # a NaN fails


SHAPES = [  # tokens, hq, hk, d, rot, axes
    (1, 1, 1, 8, 8, 1), (1, 8, 8, 32, 32, 1), (7, 32, 8, 128, 64, 1), (3, 5, 1, 64, 24, 1), (130, 8, 8, 32, 32, 3), (333, 6, 2, 80, 20, 1),
    (65, 3, 3, 96, 96, 2), (19, 2, 1, 256, 250, 1), (17, 4, 2, 16, 2, 1), (9, 40, 8, 128, 128, 1), (5000, 8, 8, 32, 32, 3), (2500, 12, 4, 128, 128, 1),
    (64, 3, 1, 40, 0, 1)]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("kind,inter", list(itertools.product(["none", "rms", "layer"], [False, True])))
def test_forward(shape, kind, inter):
    tokens, hq, hk, d, rot, axes = shape
    for dtype in (BF, HF, F32):
        s = make(tokens, hq, hk, d, rot, kind, dtype, wdtype=dtype if tokens % 2 else F32, axes=axes, int32=tokens % 3 == 0)
        amp = 1.25 if rot else 1.0
        kw = kwargs(s, kind, inter, amp)
        got = ops.qk_rope_fwd(s["q"], s["k"], s["freqs"], s["positions"], **kw)
        cs = R.table(s["freqs"], s["positions"], s["axes"], tokens, DEV)
        for x, y, h in ((s["q"], got[0], "q"), (s["k"], got[1], "k")):
            w, b = s[h + "_weight"], s[h + "_bias"]
            ref = R.qk_rope(x.double(), cs, inter, amp, kind, w, b, 1e-5)
            assert y.is_contiguous() and y.dtype == dtype
            close(y, ref, R.out_bound(x.double(), amp, kind, w, b, 1e-5, dtype, ref))


@pytest.mark.parametrize("shape", [s for s in SHAPES if s[0] not in (64,)] + [(64, 3, 1, 40, 0, 1), (20000, 8, 8, 32, 32, 3)], ids=str)
@pytest.mark.parametrize("kind,inter", list(itertools.product(["none", "rms", "layer"], [False, True])))
def test_backward(shape, kind, inter):
    tokens, hq, hk, d, rot, axes = shape
    for dtype in (BF, HF, F32):
        wd = dtype if tokens % 2 else F32
        s = make(tokens, hq, hk, d, rot, kind, dtype, wdtype=wd, axes=axes, seed=1)
        amp = 0.75 if rot else 1.0
        g = gen(2)
        gy = [torch.randn(tokens, h, d, generator=g, device=DEV).to(dtype) for h in (hq, hk)]
        got = ops.qk_rope_bwd(*gy, s["q"], s["k"], s["freqs"], s["positions"], **kwargs(s, kind, inter, amp))
        cs = R.table(s["freqs"], s["positions"], s["axes"], tokens, DEV)
        for i, h in enumerate("qk"):
            leaf = [None if t is None else t.double().requires_grad_() for t in (s[h], s[h + "_weight"], s[h + "_bias"])]
            y = R.qk_rope(leaf[0], cs, inter, amp, kind, leaf[1], leaf[2], 1e-5)
            ref = torch.autograd.grad(y, [t for t in leaf if t is not None], gy[i].double())
            x, w = s[h].double(), leaf[1]
            rot_g = R.rotate(gy[i].double(), cs[0], -cs[1], inter, amp)  # the gradient behind the rotation
            du = rot_g if w is None else rot_g * w.detach()
            sig = torch.ones_like(x[..., :1])
            xm = x.abs().amax(-1, keepdim=True)
            if kind != "none":
                c = x - x.mean(-1, keepdim=True) if kind == "layer" else x
                sig = (c.square().mean(-1, keepdim=True) + 1e-5).sqrt()
            # du carries the rotation's 16 u of the largest |g| of its row; u = x / sigma 12 u of max|x| / sigma; the row mean of du u is
            # a sum of such products, then multiplied by u once more: below 64 u max|g| max|w| (1 + max|x| / sigma)^2 / sigma
            gm = gy[i].double().abs().amax(-1, keepdim=True) * max(1.0, amp) * (1.0 if w is None else float(w.abs().max()))
            big = gm if kind == "none" else gm * (1 + xm / sig).square() / sig
            close(got[i], ref[0], R.U[dtype] * ref[0].abs() + 64 * R.F32U * big)
            u = None if kind == "none" else (c / sig)
            rows_per_lane = tokens * h_count(s, h) / 64 + 200  # an upper bound on the length of any chain of additions (64 lanes, 16 x 64 partial sums)
            for n, name in ((2 + 2 * i, "_weight"), (3 + 2 * i, "_bias")):
                if s[h + name] is None:
                    assert got[n] is None
                    continue
                assert got[n].dtype == wd
                term = (rot_g * u) if name == "_weight" else rot_g
                r = ref[1] if name == "_weight" else ref[2]
                mag = term.abs().sum((0, 1)) + 30 * (gm * (xm / sig)).sum((0, 1)) / 8  # the terms' own errors: 30 u of their row's largest, an eighth of
                # which is what independent signs over any count of rows leave; the chain of additions: rounding grows like its root
                close(got[n], r, R.U[wd] * r.abs() + R.F32U * (rows_per_lane ** 0.5 + 8) * mag)


def h_count(s, h):
    return s[h].shape[1]


@pytest.mark.parametrize("kind,inter", [("none", False), ("rms", True), ("layer", False)])
def test_backward_against_differences(kind, inter):
    s = make(5, 3, 2, 32, 24, kind, F32, seed=4)
    kw = kwargs(s, kind, inter, 1.1)
    g = gen(5)
    gy = [torch.randn(5, h, 32, generator=g, device=DEV) for h in (3, 2)]
    grads = ops.qk_rope_bwd(*gy, s["q"], s["k"], s["freqs"], s["positions"], **kw)
    cs = R.table(s["freqs"], s["positions"], s["axes"], 5, DEV)

    def loss(x, h, fn):
        return float((fn(x, h).double() * gy["qk".index(h)].double()).sum())

    def kernel(x, h):
        q, k = (x, s["k"]) if h == "q" else (s["q"], x)
        return ops.qk_rope_fwd(q, k, s["freqs"], s["positions"], **kw)["qk".index(h)]

    def exact(x, h):
        return R.qk_rope(x.double(), cs, inter, 1.1, kind, s[h + "_weight"], s[h + "_bias"], 1e-5)

    step = 2.0 ** -7
    for i, h in enumerate("qk"):
        d = torch.randn(s[h].shape, generator=g, device=DEV)
        a, b = (s[h] + step * d).contiguous(), (s[h] - step * d).contiguous()
        span = ((a.double() - b.double()) / 2)  # the step as it was rounded
        slope = (loss(a, h, kernel) - loss(b, h, kernel)) / 2
        slope64 = (loss(a, h, exact) - loss(b, h, exact)) / 2
        mine = float((grads[i].double() * span).sum())
        x = s[h].double().requires_grad_()
        exact_mine = float((torch.autograd.grad(exact(x, h), x, gy[i].double())[0] * span).sum())
        ref = exact(a, h)
        rounding = float((R.out_bound(a.double(), 1.1, kind, s[h + "_weight"], s[h + "_bias"], 1e-5, F32, ref) * gy[i].abs().double()).sum())
        # the difference quotient's own curvature (known in 64 bits), the roundings of the outputs on both sides, the gradient's 1e-5
        assert abs(mine - slope) <= abs(slope64 - exact_mine) + rounding + 1e-5 * float((grads[i].double() * span).abs().sum())


def test_far_positions_and_amplitude():
    s = make(6, 2, 1, 64, 64, "none", F32, seed=7)
    s["positions"] = torch.tensor([0, 1, 10 ** 6, 2 ** 30, -2 ** 30, 123456789], device=DEV)
    q, k = ops.qk_rope_fwd(s["q"], s["k"], s["freqs"], s["positions"])
    cs = R.table(s["freqs"], s["positions"], None, 6, DEV)
    ref = R.qk_rope(s["q"].double(), cs, False, 1.0, "none", None, None, 0)
    # 2^30 f is rounded to 2^-53 twice and once by the reference: 3 * 2^30 * 2^-53 rad more than out_bound has
    close(q, ref, R.out_bound(s["q"].double(), 1.0, "none", None, None, 0, F32, ref) + 3 * 2.0 ** -23 * s["q"].double().abs().amax(-1, keepdim=True) * 2)
    assert torch.equal(q[0], s["q"][0])


def test_autograd_and_graph_replays():
    s = make(300, 4, 2, 64, 32, "layer", BF, wdtype=F32, seed=8)
    leaves = [t.detach().clone().requires_grad_() for t in (s["q"], s["k"], s["q_weight"], s["q_bias"], s["k_weight"], s["k_bias"])]
    gy = [torch.randn(300, h, 64, generator=gen(9), device=DEV).to(BF) for h in (4, 2)]

    def step():
        y = torch.ops.hma.qk_rope(leaves[0], leaves[1], s["freqs"], s["positions"], None, False, 1.0, "layer", *leaves[2:], 1e-5)
        return list(torch.autograd.grad(y, leaves, gy)) + [t.detach() for t in y]

    want = [t.clone() for t in step()]
    direct = ops.qk_rope_bwd(*gy, *(t.detach() for t in leaves[:2]), s["freqs"], s["positions"], **kwargs(s, "layer", False, 1.0))
    for a, b in zip(want[:6], (direct[0], direct[1], *direct[2:])):
        assert torch.equal(a, b)
    # k unused: its gradient comes in as zeros and goes out as zeros
    y = torch.ops.hma.qk_rope(leaves[0], leaves[1], s["freqs"], s["positions"], None, False, 1.0, "layer", *leaves[2:], 1e-5)
    gk = torch.autograd.grad(y[0], [leaves[0], leaves[1]], gy[0])
    assert torch.equal(gk[0], want[0]) and not gk[1].any()
    del y, gk  # no eager graph of these leaves lives while a step is captured
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(3):
        with torch.no_grad():
            leaves[0].copy_((s["q"].float() * (1 + i)).to(BF))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


def test_strides_streams_and_broadcast():
    s = make(50, 4, 2, 32, 32, "rms", BF, seed=10)
    kw = kwargs(s, "rms", False, 1.0)
    want = ops.qk_rope_fwd(s["q"].contiguous(), s["k"].contiguous(), s["freqs"], s["positions"], **kw)
    assert all(torch.equal(a, b) for a, b in zip(want, ops.qk_rope_fwd(s["q"], s["k"], s["freqs"], s["positions"], **kw)))
    odd = torch.empty(50 * 4 * 32 + 1, dtype=BF, device=DEV)[1:].view(50, 4, 32)  # two bytes off
    odd.copy_(s["q"])
    by_head = s["k"].permute(1, 0, 2).contiguous().permute(1, 0, 2)
    assert all(torch.equal(a, b) for a, b in zip(want, ops.qk_rope_fwd(odd, by_head, s["freqs"], s["positions"], **kw)))
    wide = torch.empty(50, 2, 64, dtype=BF, device=DEV)[..., ::2]  # every second value
    wide.copy_(s["k"])
    assert torch.equal(want[1], ops.qk_rope_fwd(s["q"], wide, s["freqs"], s["positions"], **kw)[1])
    one = s["k"][:, :1].expand(50, 6, 32)
    assert torch.equal(ops.qk_rope_fwd(s["q"], one, s["freqs"], s["positions"], **kw)[1], want[1][:, :1].expand(50, 6, 32))
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = ops.qk_rope_fwd(s["q"], s["k"], s["freqs"], s["positions"], **kw)
    side.synchronize()
    assert torch.equal(got[0], want[0])
    empty = ops.qk_rope_fwd(s["q"][:0], s["k"][:0], s["freqs"], s["positions"][:0], **kw)
    assert empty[0].shape == (0, 4, 32)
    grads = ops.qk_rope_bwd(s["q"][:0], s["k"][:0], s["q"][:0], s["k"][:0], s["freqs"], s["positions"][:0], **kw)
    assert grads[0].shape == (0, 4, 32) and not grads[2].any() and not grads[4].any()


def test_extremes():
    """A row of zeros, of the type's largest values, with an infinity and with a NaN: each stays its own row's matter."""
    s = make(4, 1, 1, 64, 64, "rms", BF, seed=11)
    q = s["q"].clone()
    q[0], q[1] = 0, torch.finfo(BF).max
    q[2, 0, 5], q[3, 0, 7] = float("inf"), float("nan")
    y, _ = ops.qk_rope_fwd(q, s["k"], s["freqs"], s["positions"], **kwargs(s, "rms", False, 1.0))
    assert not y[0].any() and y[3].isnan().all()
    assert y[2].isnan().any()
    clean, _ = ops.qk_rope_fwd(s["q"], s["k"], s["freqs"], s["positions"], **kwargs(s, "none", False, 1.0) | dict(q_weight=None, k_weight=None))
    q[3] = s["q"][3]
    z, _ = ops.qk_rope_fwd(q, s["k"], s["freqs"], s["positions"], **kwargs(s, "none", False, 1.0) | dict(q_weight=None, k_weight=None))
    assert torch.equal(z[3], clean[3])


@pytest.mark.parametrize("rot,inter", [(0, False), (24, False), (20, False), (20, True), (24, True), (2, True)])
def test_values_behind_the_rotation_pass(rot, inter):
    """An infinity, a NaN and the largest value behind `rot` come out as they went in and reach no other value, forward and backward."""
    s = make(9, 3, 2, 64, rot, "none", BF, seed=12)
    kw = dict(interleaved=inter)
    clean = ops.qk_rope_fwd(s["q"], s["k"], s["freqs"], s["positions"], **kw)
    q, k = s["q"].clone(), s["k"].clone()
    for x in (q, k):
        x[0, 0, rot], x[1, 1, rot + 1], x[2, 0, 63], x[3, 1, 63] = float("inf"), -float("inf"), float("nan"), torch.finfo(BF).max
    odd = [x.float() != y.float() for x, y in ((q, s["q"]), (k, s["k"]))]
    assert [int(o.sum()) for o in odd] == [4, 4]
    clean_b = ops.qk_rope_bwd(s["q"], s["k"], s["q"], s["k"], s["freqs"], s["positions"], **kw)
    got = ops.qk_rope_fwd(q, k, s["freqs"], s["positions"], **kw), ops.qk_rope_bwd(q, k, s["q"], s["k"], s["freqs"], s["positions"], **kw)
    for ys, zs in zip(got, (clean, clean_b)):
        for y, z, x, o in zip(ys, zs, (q, k), odd):
            torch.testing.assert_close(y[o], x[o], rtol=0, atol=0, equal_nan=True)
            assert torch.equal(y[~o], z[~o])


def test_gradients_of_gradients_are_refused_and_broadcast_gradients_taken():
    s = make(5, 2, 1, 32, 32, "rms", F32, seed=13)
    q, k = s["q"].clone().requires_grad_(), s["k"].clone().requires_grad_()
    y = torch.ops.hma.qk_rope(q, k, s["freqs"], s["positions"], None, False, 1.0, "rms", s["q_weight"], None, s["k_weight"], None, 1e-5)
    gq, gk = torch.autograd.grad(y[0].sum() + y[1].sum(), [q, k], create_graph=True)  # a gradient with strides of zero
    ones = [torch.ones_like(t) for t in y]
    want = ops.qk_rope_bwd(*ones, s["q"], s["k"], s["freqs"], s["positions"], **kwargs(s, "rms", False, 1.0))
    assert torch.equal(gq, want[0]) and torch.equal(gk, want[1])
    y = torch.ops.hma.qk_rope(q, k, s["freqs"], s["positions"], None, False, 1.0, "rms", s["q_weight"], None, s["k_weight"], None, 1e-5)
    gq, = torch.autograd.grad(y[0].square().sum() + y[1].sum(), [q], create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate twice"):
        gq.square().sum().backward()


# ------------------------------------------------------------------------------------------------ kv_append
def paged(new, lens, page, hk, d, dtype, g, extra=2, tail=0):
    need = [-(-max(n, 0) // page) for n in lens]
    pages = sum(need) + extra
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    table = torch.full((len(lens), max(need + [1])), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    cu = torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32, device=DEV)
    kc = torch.randn(pages, hk, page, d, generator=g, device=DEV).to(dtype)
    vc = torch.randn(pages, hk, page, d, generator=g, device=DEV).to(dtype)
    return table, cu, torch.tensor(lens, dtype=torch.int32, device=DEV), kc, vc, sum(new) + tail


APPENDS = [  # new, lens, page, hq, hk, d, rot, kind, tail
    ([1], [1], 16, 8, 8, 32, 32, "layer", 0), ([1, 1, 1], [5, 1, 77], 16, 32, 8, 128, 128, "rms", 2), ([3, 0, 9, 1], [3, 40, 70, 64], 7, 6, 2, 64, 20, "none", 5),
    ([320, 320], [320, 1600], 64, 8, 8, 32, 32, "layer", 64), ([1500], [1777], 1, 4, 1, 80, 80, "rms", 0), ([0, 0], [0, 9], 16, 2, 2, 16, 8, "none", 3),
    ([1] * 70, list(range(1, 71)), 32, 4, 2, 64, 64, "rms", 1), ([1] * 300, [(7 * i) % 90 + 1 for i in range(300)], 16, 2, 1, 32, 16, "rms", 0)]


@pytest.mark.parametrize("case", APPENDS, ids=lambda c: f"{len(c[0])}seqs-{sum(c[0])}tok-page{c[2]}-d{c[5]}")
@pytest.mark.parametrize("f8", [False, True])
def test_append(case, f8):
    new, lens, page, hq, hk, d, rot, kind, tail = case
    for dtype, inter, axes in ((BF, False, 1), (HF, True, 3)):
        g = gen(20)
        table, cu, kv, kc, vc, tokens = paged(new, lens, page, hk, d, dtype, g, tail=tail)
        s = make(tokens, hq, hk, d, rot, kind, dtype, axes=axes, seed=21)
        scales = {}
        if f8:
            scales = dict(k_scale=0.01 + 0.01 * torch.rand(hk, generator=g, device=DEV), v_scale=0.01 + 0.01 * torch.rand(hk, generator=g, device=DEV))
            kc, vc = kc.to(F8), vc.to(F8)
        # strided caches: pages of (token, head) order
        if page == 16:
            kc = kc.transpose(1, 2).contiguous().transpose(1, 2)
        k0, v0 = kc.clone(), vc.clone()
        pos = s["positions"] if axes > 1 else None
        kw = kwargs(s, kind, inter, 1.0)
        q_out = ops.kv_append(s["k"], s["v"], kc, vc, table, cu, kv, q=s["q"], freqs=s["freqs"], positions=pos, **kw, **scales)
        seq = [b for b, n in enumerate(new) for _ in range(n)]
        place = [lens[b] - new[b] + i for b in range(len(new)) for i in range(new[b])]
        n = len(place)
        pl = torch.tensor(place, dtype=torch.int64, device=DEV)
        cs = R.table(s["freqs"], pl if pos is None else pos[:, :n], s["axes"], n, DEV)
        pg = torch.tensor([int(t) for t in table[seq, [p // page for p in place]]] if n else [], dtype=torch.int64, device=DEV)
        off = pl % page
        ref = R.qk_rope(s["q"][:n].double(), cs, inter, 1.0, kind, s["q_weight"], s["q_bias"], 1e-5)
        close(q_out[:n], ref, R.out_bound(s["q"][:n].double(), 1.0, kind, s["q_weight"], s["q_bias"], 1e-5, dtype, ref))
        assert not q_out[n:].any()
        k_ref = R.qk_rope(s["k"][:n].double(), cs, inter, 1.0, kind, s["k_weight"], s["k_bias"], 1e-5)
        kb = R.out_bound(s["k"][:n].double(), 1.0, kind, s["k_weight"], s["k_bias"], 1e-5, dtype, k_ref)
        got_k, got_v = kc[pg, :, off].double(), vc[pg, :, off].double()
        if f8:
            ks, vs = scales["k_scale"].double()[:, None], scales["v_scale"].double()[:, None]
            r = (k_ref / ks).clamp(-448, 448)
            # half a step of e4m3 (2^-4 relative, 2^-10 among the subnormals) of the value with its 32-bit error and the division's
            e32 = (kb - R.U[dtype] * k_ref.abs() + 4 * R.F32U * k_ref.abs()) / ks
            close(got_k, r, 2.0 ** -4 * r.abs() + 2.0 ** -10 + e32 * (1 + 2.0 ** -4))
            rv = (s["v"][:n].double() / vs).clamp(-448, 448)
            close(got_v, rv, 2.0 ** -4 * rv.abs() * (1 + 2.0 ** -20) + 2.0 ** -10)
        else:
            close(got_k, k_ref, kb)
            assert torch.equal(vc[pg, :, off], s["v"][:n])
        # nothing else has changed
        bits = torch.uint8 if f8 else torch.int16
        for now, before in ((kc, k0), (vc, v0)):
            now, before = now.view(bits).clone(), before.view(bits)
            if n:
                now[pg, :, off] = before[pg, :, off]
            assert torch.equal(now, before)
        # without q: the same caches; q_out given: rows behind the last sequence stay
        k2, v2 = k0.clone(), v0.clone()
        kw.pop("q_weight"), kw.pop("q_bias")
        assert ops.kv_append(s["k"], s["v"], k2, v2, table, cu, kv, freqs=s["freqs"], positions=pos, **kw, **scales) is None
        assert torch.equal(k2.view(bits), kc.view(bits)) and torch.equal(v2.view(bits), vc.view(bits))
        mine = torch.full_like(q_out, 7.0)
        ops.kv_append(s["k"], s["v"], k2, v2, table, cu, kv, q=s["q"], q_out=mine, q_weight=s["q_weight"], q_bias=s["q_bias"], freqs=s["freqs"], positions=pos,
                      **kw, **scales)
        assert torch.equal(mine[:n], q_out[:n]) and bool((mine[n:] == 7).all())


def test_append_skips_what_has_no_place():
    """Page numbers outside the cache, a table that is too short, lengths smaller than the new tokens: not stored, all else is."""
    g = gen(30)
    new, lens = [4, 4, 4, 4], [4, 20, 2, 12]
    table, cu, kv, kc, vc, tokens = paged(new, lens, 4, 2, 32, BF, g)
    kc.zero_(), vc.zero_()
    table[0, 0] = 10 ** 6           # outside
    table[3, 2] = -5                # sequence 3: its four new tokens are places 8 .. 11, page 2
    short = table[:, :4].contiguous()  # sequence 1: places 16 .. 19 need page 4
    s = make(tokens, 2, 2, 32, 32, "none", BF, seed=31)
    ops.kv_append(s["k"], s["v"], kc, vc, short, cu, kv, freqs=s["freqs"])
    stored = vc.abs().sum((1, 3)) > 0  # (page, row)
    want = torch.zeros_like(stored)
    want[int(table[2, 0]), :2] = True  # sequence 2: places -2 .. 1
    assert torch.equal(stored, want)
    assert torch.equal(vc[int(table[2, 0]), :, 0], s["v"][10]) and torch.equal(vc[int(table[2, 0]), :, 1], s["v"][11])


def test_append_custom_op_and_graph():
    g = gen(40)
    new, lens = [1, 1, 1], [9, 33, 17]
    table, cu, kv, kc, vc, tokens = paged(new, lens, 16, 2, 64, BF, g)
    s = make(tokens, 4, 2, 64, 64, "rms", BF, seed=41)
    args = (s["q"], s["freqs"], None, None, False, 1.0, "rms", s["q_weight"], None, s["k_weight"], None, 1e-5, None, None)
    want_k, want_v = kc.clone(), vc.clone()
    want_q = ops.kv_append(s["k"], s["v"], want_k, want_v, table, cu, kv, q=s["q"], freqs=s["freqs"], norm="rms", q_weight=s["q_weight"], k_weight=s["k_weight"])
    got = torch.ops.hma.kv_append(s["k"], s["v"], kc, vc, table, cu, kv, *args)
    assert torch.equal(got, want_q) and torch.equal(kc, want_k) and torch.equal(vc, want_v)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.ops.hma.kv_append(s["k"], s["v"], kc, vc, table, cu, kv, *args)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = torch.ops.hma.kv_append(s["k"], s["v"], kc, vc, table, cu, kv, *args)
    for i in range(3):
        kv.sub_(1)  # other places on each replay
        k2, v2 = kc.clone(), vc.clone()
        graph.replay()
        q2 = ops.kv_append(s["k"], s["v"], k2, v2, table, cu, kv, q=s["q"], freqs=s["freqs"], norm="rms", q_weight=s["q_weight"], k_weight=s["k_weight"])
        torch.cuda.synchronize()
        assert torch.equal(out, q2) and torch.equal(kc, k2) and torch.equal(vc, v2)


def test_append_in_place():
    """q_out may be q: every row is read before the wave that read it writes it."""
    g = gen(50)
    new, lens = [700, 1, 40], [700, 90, 400]
    table, cu, kv, kc, vc, tokens = paged(new, lens, 16, 2, 64, BF, g)
    s = make(tokens, 12, 2, 64, 64, "rms", BF, seed=51)
    kw = dict(freqs=s["freqs"], norm="rms", q_weight=s["q_weight"], k_weight=s["k_weight"])
    want = ops.kv_append(s["k"], s["v"], kc, vc, table, cu, kv, q=s["q"], **kw)
    q = s["q"].contiguous()
    assert ops.kv_append(s["k"], s["v"], kc, vc, table, cu, kv, q=q, q_out=q, **kw) is q and torch.equal(q, want)


def test_append_what_is_no_number_into_e4m3():
    """Beyond the type's largest value: that value; a NaN stays one; the others of the row are as without."""
    g = gen(60)
    table, cu, kv, kc, vc, tokens = paged([5, 2], [5, 30], 16, 2, 64, BF, g)
    s = make(tokens, 2, 2, 64, 0, "none", BF, seed=61)
    scales = dict(k_scale=torch.full((2,), 0.02, device=DEV), v_scale=torch.full((2,), 0.03, device=DEV))
    k, v = s["k"].clone(), s["v"].clone()
    for x in (k, v):
        x[0, 0, 3], x[1, 1, 63], x[5, 0, 0], x[6, 1, 8] = float("inf"), -float("inf"), float("nan"), 1e4
    got = []
    for a, b in ((s["k"], s["v"]), (k, v)):
        c = torch.zeros_like(kc).to(F8), torch.zeros_like(vc).to(F8)
        ops.kv_append(a, b, *c, table, cu, kv, **scales)
        got.append(c)
    place = [0, 1, 2, 3, 4, 28, 29]
    seq = [0] * 5 + [1] * 2
    pg = table[seq, [p // 16 for p in place]].long()
    off = torch.tensor(place, device=DEV) % 16
    for clean, odd, x, y in zip(*got, (k, v), (s["k"], s["v"])):
        a, b = clean[pg, :, off].float(), odd[pg, :, off].float()
        same = x.float() == y.float()
        assert int((~same).sum()) == 4 and torch.equal(a[same], b[same])
        assert b[0, 0, 3] == 448 and b[1, 1, 63] == -448 and b[5, 0, 0].isnan() and b[6, 1, 8] == 448


@pytest.mark.parametrize("dtype", [BF, HF])
def test_append_rounds_the_quotient(dtype):
    """What goes into an e4m3 cache is x / scale in 32 bits, rounded: every finite value of the rows' type, against scales whose quotients
    lie on the borders between two e4m3 values (odd multiples of powers of two) and others; exact, zeros' signs too."""
    g = torch.Generator().manual_seed(70)
    scales = torch.cat([(2 * torch.arange(32) + 1) * 2.0 ** -11, 0.001 + 0.02 * torch.rand(28, generator=g), torch.tensor([1.0, 448.0, 3e-20, 5e15])]).float()
    x = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype)
    x = torch.where(x.isnan(), torch.zeros_like(x), x).view(512, 1, 128).expand(512, 64, 128)
    page = 64
    kc, vc = (torch.zeros(8, 64, page, 128, dtype=F8, device=DEV) for _ in range(2))
    table = torch.arange(8, dtype=torch.int32, device=DEV)[None]
    cu, lens = torch.tensor([0, 512], dtype=torch.int32, device=DEV), torch.tensor([512], dtype=torch.int32, device=DEV)
    ops.kv_append(x.to(DEV), x.flip(1).to(DEV), kc, vc, table, cu, lens, k_scale=scales.to(DEV), v_scale=scales.flip(0).to(DEV))
    for cache, s in ((kc, scales), (vc, scales.flip(0))):
        got = cache.transpose(1, 2).reshape(512, 64, 128).cpu()
        want = (x.float() / s[:, None]).clamp(-448, 448).to(F8)
        off = got.view(torch.uint8) != want.view(torch.uint8)
        assert not off.any(), (int(off.sum()), s[off.any(0).any(-1)].tolist(), x[off][:4].tolist(), got[off][:4].float().tolist(), want[off][:4].float().tolist())


def test_traced_graph_on_the_gpu():
    """A graph traced with real tensors launches what the eager pass launches, forward and back, on inputs other than the trace's."""
    def step(q, k, w, freqs, positions):
        leaves = [t.detach().requires_grad_() for t in (q, k, w)]
        y = torch.ops.hma.qk_rope(leaves[0], leaves[1], freqs, positions, None, True, 1.0, "rms", leaves[2], None, leaves[2], None, 1e-5)
        return [t.detach() for t in y] + list(torch.autograd.grad(y, leaves, [y[0].detach() * 2, y[1].detach()]))

    a, b = (make(40, 6, 2, 64, 32, "rms", BF, seed=s) for s in (80, 81))
    graph = make_fx(step)(a["q"], a["k"], a["q_weight"], a["freqs"], a["positions"])
    called = [n.target for n in graph.graph.nodes if n.op == "call_function"]
    assert called.count(torch.ops.hma.qk_rope.default) == 1 and called.count(torch.ops.hma.qk_rope_bwd.default) == 1
    for s in (a, b):
        args = (s["q"], s["k"], s["q_weight"], s["freqs"], s["positions"])
        got, want = graph(*args), step(*args)
        assert len(got) == len(want) == 5 and all(torch.equal(x, y) for x, y in zip(got, want))
