"""qk_rope, kv_append, attn_paged without a GPU: what the wrappers and the C entry points refuse, the shapes that tracing sees, the
frequencies."""
import contextlib
import ctypes as C
import math
import os
import subprocess

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode

import hma_amd.torch_ops as T
from hma_amd import _lib, ops

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
F8 = torch.float8_e4m3fn
EINVAL = -10001


class Launched(Exception):
    pass


@pytest.fixture
def host(monkeypatch):
    """The wrappers on host tensors, up to the launch."""
    monkeypatch.setattr(ops, "_device", lambda *a: contextlib.nullcontext())
    monkeypatch.setattr(ops, "_stream", lambda t: 0)

    def call(name, *a):
        if name.endswith("_ws"):
            return _lib.check(getattr(_lib.load(), name)(*a), name)
        raise Launched(name)

    monkeypatch.setattr(ops._lib, "call", call)


def rope_args(**over):
    a = dict(q=torch.zeros(5, 4, 32, dtype=BF), k=torch.zeros(5, 2, 32, dtype=BF), freqs=torch.ones(8, dtype=torch.float64), positions=torch.arange(5))
    kw = dict(norm="rms", q_weight=torch.ones(32), k_weight=torch.ones(32))
    for n, v in over.items():
        (a if n in a else kw)[n] = v
    return list(a.values()), kw


ROPE_BAD = [dict(k=torch.zeros(6, 2, 32, dtype=BF)), dict(k=torch.zeros(5, 2, 16, dtype=BF)), dict(k=torch.zeros(5, 2, 32, dtype=HF)),
            dict(q=torch.zeros(5, 4, 32, dtype=torch.float64), k=torch.zeros(5, 2, 32, dtype=torch.float64)), dict(q=torch.zeros(5, 128, dtype=BF)),
            dict(freqs=torch.ones(8)), dict(freqs=torch.ones(17, dtype=torch.float64)), dict(freqs=torch.ones(4, 2, dtype=torch.float64)),
            dict(positions=None), dict(positions=torch.arange(4)), dict(positions=torch.arange(5).float()),
            dict(positions=torch.zeros(2, 5, dtype=torch.int64)), dict(positions=torch.arange(10)[::2]),
            dict(axes=torch.zeros(8, dtype=torch.int64)), dict(axes=torch.zeros(7, dtype=torch.int32)),
            dict(norm="batch"), dict(norm="none"), dict(q_weight=torch.ones(31)), dict(q_weight=torch.ones(32, dtype=HF), k_weight=None),
            dict(q_weight=torch.ones(32, dtype=BF)), dict(q_bias=torch.zeros(32)), dict(q_weight=torch.ones(64)[::2])]


@pytest.mark.parametrize("over", ROPE_BAD, ids=lambda o: "-".join(o))
def test_qk_rope_refuses(host, over):
    a, kw = rope_args(**over)
    with pytest.raises(ValueError):
        ops.qk_rope_fwd(*a, **kw)
    a, kw = rope_args(**over)
    with pytest.raises(ValueError):
        ops.qk_rope_bwd(torch.zeros_like(a[0]), torch.zeros_like(a[1]), *a, **kw)


def test_qk_rope_launches(host):
    for over in (dict(), dict(norm="layer", q_bias=torch.zeros(32)), dict(norm="none", q_weight=None, k_weight=None, freqs=None, positions=None),
                 dict(positions=torch.zeros(3, 5, dtype=torch.int32), axes=torch.zeros(8, dtype=torch.int32))):
        a, kw = rope_args(**over)
        with pytest.raises(Launched):
            ops.qk_rope_fwd(*a, **kw)
    a, kw = rope_args()
    with pytest.raises(ValueError):
        ops.qk_rope_bwd(torch.zeros(5, 4, 32), torch.zeros(5, 2, 32, dtype=BF), *a, **kw)


def cache_args(**over):
    a = dict(k=torch.zeros(3, 2, 32, dtype=BF), v=torch.zeros(3, 2, 32, dtype=BF), k_cache=torch.zeros(4, 2, 16, 32, dtype=BF),
             v_cache=torch.zeros(4, 2, 16, 32, dtype=BF), page_table=torch.zeros(2, 3, dtype=torch.int32), cu_seqlens=torch.zeros(3, dtype=torch.int32),
             kv_lens=torch.zeros(2, dtype=torch.int32))
    kw = {}
    for n, v in over.items():
        (a if n in a else kw)[n] = v
    return a, kw


CACHE_BAD = [dict(k_cache=torch.zeros(4, 2, 16, 32, dtype=HF)), dict(v_cache=torch.zeros(4, 2, 8, 32, dtype=BF)),
             dict(k_cache=torch.zeros(4, 2, 16, 32, dtype=F8), v_cache=torch.zeros(4, 2, 16, 32, dtype=F8)),  # no scales
             dict(k_scale=torch.ones(2), v_scale=torch.ones(2)), dict(page_table=torch.zeros(2, 3, dtype=torch.int64)),
             dict(page_table=torch.zeros(6, dtype=torch.int32)), dict(page_table=torch.zeros(3, 2, dtype=torch.int32).t()),
             dict(cu_seqlens=torch.zeros(2, dtype=torch.int32)), dict(kv_lens=torch.zeros(3, dtype=torch.int32)),
             dict(cu_seqlens=torch.zeros(3, dtype=torch.int64)), dict(kv_lens=torch.zeros(4, dtype=torch.int32)[::2]),
             dict(k_cache=torch.zeros(4, 2, 32, 16, dtype=BF).transpose(2, 3), v_cache=torch.zeros(4, 2, 32, 16, dtype=BF).transpose(2, 3))]
E4M3 = dict(k_cache=torch.zeros(4, 2, 16, 32, dtype=F8), v_cache=torch.zeros(4, 2, 16, 32, dtype=F8))


@pytest.mark.parametrize("over", CACHE_BAD + [dict(v=torch.zeros(3, 2, 16, dtype=BF)), dict(k=torch.zeros(3, 1, 32, dtype=BF), v=torch.zeros(3, 1, 32, dtype=BF)),
                                              dict(k=torch.zeros(3, 2, 32), v=torch.zeros(3, 2, 32)), dict(q=torch.zeros(2, 4, 32, dtype=BF)),
                                              dict(q=torch.zeros(3, 4, 32, dtype=HF)), dict(q_out=torch.zeros(3, 4, 32, dtype=BF)),
                                              dict(q=torch.zeros(3, 4, 32, dtype=BF), q_out=torch.zeros(3, 4, 64, dtype=BF)[..., ::2]),
                                              dict(norm="rms", q_weight=torch.ones(32)), dict(norm="rms", k_weight=torch.ones(16)),
                                              E4M3 | dict(k_scale=torch.ones(2), v_scale=torch.ones(3)), E4M3 | dict(k_scale=torch.ones(2))],
                         ids=lambda o: "-".join(o))
def test_kv_append_refuses(host, over):
    a, kw = cache_args(**over)
    with pytest.raises(ValueError):
        ops.kv_append(*a.values(), **kw)


@pytest.mark.parametrize("over", CACHE_BAD + [dict(window=-1), dict(window=5, causal=False), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan),
                                              dict(scale=math.inf), dict(q=torch.zeros(3, 3, 32, dtype=BF)), dict(q=torch.zeros(3, 4, 32)),
                                              dict(q=torch.zeros(3, 4, 64, dtype=BF)), dict(out=torch.zeros(3, 4, 32, dtype=BF)),
                                              dict(lse=torch.zeros(3, 4)), dict(out=torch.zeros(3, 4, 32, dtype=BF), lse=torch.zeros(3, 5)),
                                              dict(out=torch.zeros(3, 4, 32, dtype=HF), lse=torch.zeros(3, 4))], ids=lambda o: "-".join(o))
def test_attn_paged_refuses(host, over):
    a, kw = cache_args(**over)
    del a["k"], a["v"]
    q, scale = kw.pop("q", torch.zeros(3, 4, 32, dtype=BF)), kw.pop("scale", 0.2)
    with pytest.raises(ValueError):
        ops.attn_paged_fwd(q, *a.values(), scale, **kw)


def test_the_good_calls_launch(host):
    a, kw = cache_args()
    with pytest.raises(Launched):
        ops.kv_append(*a.values())
    a, kw = cache_args(**E4M3, k_scale=torch.ones(2), v_scale=torch.ones(2))
    with pytest.raises(Launched):
        ops.kv_append(*a.values(), **kw, q=torch.zeros(3, 4, 32, dtype=BF), norm="rms", q_weight=torch.ones(32))
    del a["k"], a["v"]
    with pytest.raises(Launched):
        ops.attn_paged_fwd(torch.zeros(3, 4, 32, dtype=BF), *a.values(), 0.2, **kw)
    with pytest.raises(NotImplementedError):
        ops.attn_paged_fwd(torch.zeros(3, 4, 48, dtype=BF), *(torch.zeros(4, 2, 16, 48, dtype=BF),) * 2, *list(a.values())[2:], 0.2)


def test_windows_of_any_size_launch(host, monkeypatch):
    """A window larger than a 32-bit number is one that no sequence reaches, not an error of the argument structure."""
    a, _ = cache_args()
    del a["k"], a["v"]
    passed = []
    monkeypatch.setattr(ops._lib, "call", lambda name, *p: passed.append((name, [x._obj for x in p if hasattr(x, "_obj")][0])))
    for window in (0, 5, 2 ** 31 - 1, 2 ** 31, 2 ** 63 - 1, 2 ** 70):
        ops.attn_paged_fwd(torch.zeros(3, 4, 32, dtype=BF), *a.values(), 0.2, window=window)
        assert passed[-1][0] == "hma_attn_paged_fwd" and passed[-1][1].window == min(window, 2 ** 31 - 1)


def test_host_tensors_are_refused():
    a, kw = rope_args()
    with pytest.raises(RuntimeError):
        ops.qk_rope_fwd(*a, **kw)
    b, _ = cache_args()
    with pytest.raises(RuntimeError):
        ops.kv_append(*b.values())
    with pytest.raises(RuntimeError):
        ops.attn_paged_fwd(torch.zeros(3, 4, 32, dtype=BF), *list(b.values())[2:], 0.2)
    with pytest.raises(NotImplementedError):
        torch.ops.hma.qk_rope(a[0], a[1], a[2], a[3], None, False, 1.0, "none", None, None, None, None, 1e-5)


# ------------------------------------------------------------------------------------------------ the C entry points
def attn_struct(**over):
    p = _lib.AttnPaged()
    v = dict(q=16, o=16, lse=16, kc=16, vc=16, table=16, cu=16, lens=16, ws=16, ws_bytes=1 << 40, tokens=4, q_tok=128, q_head=32, kc_page=1024, kc_head=512,
             kc_tok=32, vc_page=1024, vc_head=512, vc_tok=32, table_stride=4, hq=4, hk=2, d=32, dtype=0, seqs=2, table_w=4, pages=8, page=16, causal=1,
             scale=0.2)
    v.update(over)
    for n, x in v.items():
        setattr(p, n, x)
    return p


@pytest.mark.parametrize("over", [dict(q=None), dict(q=18), dict(o=None), dict(o=8), dict(kc=None), dict(vc=8), dict(table=None), dict(cu=None), dict(lens=None),
                                  dict(ws=None), dict(ws=8), dict(ws_bytes=64), dict(q_tok=4), dict(q_head=-32), dict(kc_page=1023), dict(vc_tok=4),
                                  dict(kc_head=-512), dict(d=48), dict(d=256), dict(dtype=2), dict(hq=3), dict(hq=0), dict(hk=0), dict(seqs=-1),
                                  dict(seqs=4097), dict(page=0), dict(pages=-1), dict(table_w=-1), dict(tokens=-1), dict(window=-1),
                                  dict(window=4, causal=0), dict(scale=0.0), dict(scale=math.nan), dict(cache_e4m3=1),
                                  dict(cache_e4m3=1, k_scale=16, v_scale=16, kc_tok=40)], ids=str)
def test_attn_paged_entry_refuses(over):
    assert _lib.load().hma_attn_paged_fwd(None, attn_struct(**over)) == EINVAL


def test_attn_paged_workspace():
    lib, n = _lib.load(), C.c_int64(-1)
    assert lib.hma_attn_paged_ws(attn_struct(), None) == EINVAL and lib.hma_attn_paged_ws(None, C.byref(n)) == EINVAL
    assert lib.hma_attn_paged_ws(attn_struct(), C.byref(n)) == 0 and n.value > 0
    few = n.value
    assert lib.hma_attn_paged_ws(attn_struct(table_w=4000), C.byref(n)) == 0 and n.value > few
    assert lib.hma_attn_paged_ws(attn_struct(tokens=1 << 20), C.byref(n)) == 0 and n.value == 0  # nothing is split
    assert lib.hma_attn_paged_fwd(None, attn_struct(tokens=0)) == 0  # nothing to do: no launch


def rope_struct(cls, **over):
    p = cls()
    v = dict(tokens=4, hq=4, hk=2, q=16, k=16, q_tok=128, q_head=32, k_tok=64, k_head=32, q_out=16)
    if cls is _lib.QkRope:
        v |= dict(k_out=16, dy_q=16, dy_k=16, dyq_tok=128, dyq_head=32, dyk_tok=64, dyk_head=32, dq=16, dk=16)
    else:
        v |= dict(v=16, v_tok=64, v_head=32, kc=16, vc=16, kc_page=1024, kc_head=512, kc_tok=32, vc_page=1024, vc_head=512, vc_tok=32, table=16, cu=16,
                  lens=16, table_stride=4, seqs=2, table_w=4, pages=8, page=16)
    r = dict(freqs=16, positions=16, pos_stride=4, d=32, rot=16, norm=1, dtype=0, w_f32=1, pos_64=1, n_axes=1, eps=1e-5, amplitude=1.0)
    for n, x in over.items():
        (r if n in r or n in ("axes", "q_w", "q_b") else v)[n] = x
    for n, x in v.items():
        setattr(p, n, x)
    for n, x in r.items():
        setattr(p.r, n, x)
    return p


BAD_ROPE = [dict(d=12), dict(d=264), dict(d=0), dict(rot=15), dict(rot=34), dict(rot=-2), dict(freqs=None), dict(norm=3), dict(dtype=3), dict(hk=0), dict(tokens=-1),
            dict(n_axes=0), dict(n_axes=2), dict(n_axes=2, axes=16, pos_stride=3), dict(norm=0, q_w=16), dict(k=None), dict(k=8), dict(k_tok=60), dict(k_head=-32),
            dict(q=24), dict(q_tok=3), dict(q_out=None)]


@pytest.mark.parametrize("over", BAD_ROPE, ids=str)
def test_rope_entries_refuse(over):
    lib = _lib.load()
    assert lib.hma_qk_rope_fwd(None, rope_struct(_lib.QkRope, **over)) == EINVAL
    if "q_out" not in over:
        assert lib.hma_qk_rope_bwd(None, rope_struct(_lib.QkRope, **over)) == EINVAL
    assert lib.hma_kv_append(None, rope_struct(_lib.KvAppend, **over)) == EINVAL


def test_rope_entries_refuse_their_own():
    lib = _lib.load()
    assert lib.hma_qk_rope_fwd(None, rope_struct(_lib.QkRope, positions=None)) == EINVAL
    assert lib.hma_qk_rope_fwd(None, rope_struct(_lib.QkRope, hq=0)) == EINVAL
    assert lib.hma_qk_rope_fwd(None, None) == EINVAL and lib.hma_qk_rope_bwd(None, None) == EINVAL and lib.hma_kv_append(None, None) == EINVAL
    for over in (dict(dq_w=16), dict(dq_w=16, ws=16, ws_floats=100), dict(dk=None), dict(dy_q=None), dict(dyk_tok=1), dict(norm=0, dq_b=16, ws=16, ws_floats=1 << 30)):
        assert lib.hma_qk_rope_bwd(None, rope_struct(_lib.QkRope, **over)) == EINVAL
    for over in (dict(dtype=2), dict(v=None), dict(v_tok=60), dict(page=0), dict(pages=-1), dict(seqs=-1), dict(table=None), dict(cu=None), dict(lens=None),
                 dict(kc=None), dict(vc=8), dict(kc_tok=36), dict(vc_page=-8), dict(cache_e4m3=1), dict(cache_e4m3=1, k_scale=16, v_scale=16, kc=20)):
        assert lib.hma_kv_append(None, rope_struct(_lib.KvAppend, **over)) == EINVAL, over
    assert lib.hma_qk_rope_fwd(None, rope_struct(_lib.QkRope, tokens=0, positions=None)) == 0
    assert lib.hma_kv_append(None, rope_struct(_lib.KvAppend, tokens=0)) == 0


def test_struct_sizes_match_the_header():
    assert C.sizeof(_lib.Rope) == 104 and C.sizeof(_lib.KvAppend) == 336 and C.sizeof(_lib.AttnPaged) == 232 and C.sizeof(_lib.QkRope) == 296


def test_struct_layouts_are_the_header_s(tmp_path):
    """Every field of the argument structures where the C header has it, asked of a C compiler."""
    structs = {"hma_rope_t": _lib.Rope, "hma_qk_rope_t": _lib.QkRope, "hma_kv_append_t": _lib.KvAppend, "hma_attn_paged_t": _lib.AttnPaged}
    lines = []
    for name, cls in structs.items():
        lines.append(f'printf("{name} - %zu\\n", sizeof({name}));')
        lines += [f'printf("{name} {f} %zu %zu\\n", offsetof({name}, {f}), sizeof((({name}*)0)->{f}));' for f, _ in cls._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("#include <stddef.h>\n#include <stdio.h>\n#include \"hma_hip.h\"\nint main(void) {\n" + "\n".join(lines) + "\nreturn 0;\n}\n")
    subprocess.run(["gcc", "-I", os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include"), str(src), "-o", str(exe)], check=True)
    for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines():
        name, field, *n = line.split()
        if field == "-":
            assert C.sizeof(structs[name]) == int(n[0]), line
        else:
            f = getattr(structs[name], field)
            assert [f.offset, f.size] == [int(x) for x in n], line


# ------------------------------------------------------------------------------------------------ tracing, frequencies
def test_fake_shapes():
    assert {"qk_rope", "qk_rope_bwd", "kv_append", "attn_paged"} <= set(T.OPS)
    with FakeTensorMode():
        q, k = (torch.empty(5, h, 32, dtype=BF, device="cuda") for h in (4, 2))
        f, w = torch.empty(8, dtype=torch.float64, device="cuda"), torch.empty(32, device="cuda")
        pos = torch.empty(5, dtype=torch.int64, device="cuda")
        y = torch.ops.hma.qk_rope(q, k, f, pos, None, False, 1.0, "rms", w, None, w, None, 1e-5)
        assert [t.shape for t in y] == [q.shape, k.shape] and y[0].dtype == BF
        y = torch.ops.hma.qk_rope(q.clone().requires_grad_(), k, f, pos, None, False, 1.0, "rms", w, None, w, None, 1e-5)
        assert y[0].requires_grad
        d = torch.ops.hma.qk_rope_bwd(q, k, q, k, f, pos, None, False, 1.0, "rms", w, None, w, None, 1e-5)
        assert [t.shape for t in d] == [q.shape, k.shape, w.shape, w.shape]
        kc = torch.empty(4, 2, 16, 32, dtype=BF, device="cuda")
        tab, cu, lens = (torch.empty(s, dtype=torch.int32, device="cuda") for s in ((2, 3), (3,), (2,)))
        out = torch.ops.hma.kv_append(k, k, kc, kc.clone(), tab, cu, lens, q, f, None, None, False, 1.0, "none", None, None, None, None, 1e-5, None, None)
        assert out.shape == q.shape
        o, lse = torch.ops.hma.attn_paged(q, kc, kc, tab, cu, lens, 0.2, True, 0, None, None)
        assert o.shape == q.shape and lse.shape == (5, 4) and lse.dtype == F32


@pytest.fixture
def on_the_host(monkeypatch):
    """qk_rope and its backward registered for host tensors with a stand-in for the launches: x 3 + w, and gradients of their own shapes."""
    def fwd(q, k, freqs, positions, *, q_weight=None, k_weight=None, **kw):
        return tuple(t * 3 + (0 if w is None else w.to(t.dtype)) for t, w in ((q, q_weight), (k, k_weight)))

    def bwd(dy_q, dy_k, q, k, freqs, positions, *, q_weight=None, k_weight=None, **kw):
        return (dy_q * 3, dy_k * 3, *(None if w is None else d.to(w.dtype).sum((0, 1)) for d, w in ((dy_q, q_weight), (dy_q, None), (dy_k, k_weight), (dy_k, None))))

    monkeypatch.setattr(ops, "qk_rope_fwd", fwd)
    monkeypatch.setattr(ops, "qk_rope_bwd", bwd)
    lib = torch.library.Library("hma", "IMPL")
    lib.impl("qk_rope", T._qk_rope, "CPU")
    lib.impl("qk_rope_bwd", T._qk_rope_bwd, "CPU")
    lib.impl("qk_rope", lambda *a: T._QkRope.apply(*a), "AutogradCPU")
    yield
    lib._destroy()


def rope_and_gradients(q, k, w):
    f, pos = torch.ones(8, dtype=torch.float64), torch.arange(5)
    leaves = [t.detach().requires_grad_() for t in (q, k, w)]
    y = torch.ops.hma.qk_rope(leaves[0], leaves[1], f, pos, None, False, 1.0, "rms", leaves[2], None, leaves[2], None, 1e-5)
    return [t.detach() for t in y] + list(torch.autograd.grad(y, leaves, [y[0].detach() * 2, y[1].detach()]))


def rope_inputs(seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(*s, generator=g) for s in ((5, 4, 32), (5, 2, 32), (32,))]


@pytest.mark.parametrize("mode", ["real", "fake"])
def test_traced_graphs_hold_the_op_and_its_backward(on_the_host, mode):
    graph = make_fx(rope_and_gradients, tracing_mode=mode)(*rope_inputs(0))
    called = [n.target for n in graph.graph.nodes if n.op == "call_function"]
    assert called.count(torch.ops.hma.qk_rope.default) == 1 and called.count(torch.ops.hma.qk_rope_bwd.default) == 1
    for seed in (0, 1):  # the inputs of the trace and others
        got, want = graph(*rope_inputs(seed)), rope_and_gradients(*rope_inputs(seed))
        assert len(got) == len(want) == 5 and all(torch.equal(a, b) for a, b in zip(got, want))


def test_dispatch_modes_see_the_op_and_its_backward(on_the_host):
    seen = []

    class Record(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(func)
            return func(*args, **(kwargs or {}))

    with Record():
        got = rope_and_gradients(*rope_inputs(2))
    assert seen.count(torch.ops.hma.qk_rope.default) == 1 and seen.count(torch.ops.hma.qk_rope_bwd.default) == 1
    assert all(torch.equal(a, b) for a, b in zip(got, rope_and_gradients(*rope_inputs(2))))


def test_negated_views_are_resolved(on_the_host, monkeypatch):
    """A view whose values are the negatives of its memory reaches the kernels as the values, in whichever place it is given."""
    fwd, bwd = ops.qk_rope_fwd, ops.qk_rope_bwd

    def plain(fn):
        def f(*a, **kw):
            assert not any(t.is_neg() for t in (*a, *kw.values()) if isinstance(t, torch.Tensor))
            return fn(*a, **kw)
        return f

    monkeypatch.setattr(ops, "qk_rope_fwd", plain(fwd))
    monkeypatch.setattr(ops, "qk_rope_bwd", plain(bwd))
    q, k, w = rope_inputs(3)
    for i in range(3):
        a, b = [q, k, w], [q, k, w]
        a[i], b[i] = torch._neg_view(a[i]), -b[i]
        assert all(torch.equal(x, y) for x, y in zip(rope_and_gradients(*a), rope_and_gradients(*b)))


def test_frequencies():
    f, amp = ops.rope_freqs(64, 10000.0, device="cpu")
    i = torch.arange(32, dtype=torch.float64)
    assert torch.allclose(f, 10000.0 ** (-2 * i / 64), rtol=1e-14, atol=0) and amp == 1.0
    assert torch.allclose(ops.rope_freqs(64, scaling="linear", factor=4.0, device="cpu")[0], f / 4, rtol=1e-14, atol=0)
    base, _ = ops.rope_freqs(64, scaling="base", factor=4.0, device="cpu")
    assert float(base[0]) == 1.0 and abs(float(base[-1] / f[-1]) - 0.25) < 1e-12
    parts, amp = ops.rope_freqs(64, scaling="parts", factor=4.0, trained=4096, device="cpu")
    turns = 4096 * f / (2 * math.pi)
    assert torch.equal(parts[turns >= 32], f[turns >= 32]) and torch.allclose(parts[turns <= 1], f[turns <= 1] / 4, rtol=1e-14, atol=0)
    assert bool((parts[1:] < parts[:-1]).all()) and abs(amp - (1 + 0.1 * math.log(4))) < 1e-12
    for bad in (dict(rot=7), dict(rot=0), dict(rot=8, base=1.0), dict(rot=8, factor=0.0), dict(rot=8, scaling="other"), dict(rot=8, slow=4.0, fast=2.0)):
        with pytest.raises(ValueError):
            ops.rope_freqs(**bad, device="cpu")
