"""The rotation, the per-head norms and the paged cache restated in 64 bits for the tests of hma_amd.ops.qk_rope_* / kv_append /
attn_paged_fwd."""
import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}  # half a step, relative
F32U = 2.0 ** -24


def table(freqs, positions, axes, tokens, device):
    """(cos, sin), (tokens, 1, rot / 2), float64"""
    if freqs is None:
        z = torch.zeros(tokens, 1, 0, dtype=torch.float64, device=device)
        return z, z
    p = positions.double()
    a = (p[axes.long()].t() if p.dim() == 2 and axes is not None else (p[0] if p.dim() == 2 else p)[:, None]) * freqs
    return a.cos()[:, None], a.sin()[:, None]


def norm(x, kind, w, b, eps):
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    if kind != "none":
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    x = x if w is None else x * w.double()
    return x if b is None else x + b.double()


def rotate(x, cos, sin, interleaved, amp):
    h = cos.shape[-1]
    lo, hi = (x[..., 0:2 * h:2], x[..., 1:2 * h:2]) if interleaved else (x[..., :h], x[..., h:2 * h])
    u, v = (lo * cos - hi * sin) * amp, (hi * cos + lo * sin) * amp
    y = torch.stack([u, v], -1).flatten(-2) if interleaved else torch.cat([u, v], -1)
    return torch.cat([y, x[..., 2 * h:]], -1)


def qk_rope(x, cs, interleaved, amp, kind, w, b, eps):
    """x (tokens, heads, d) double"""
    return rotate(norm(x, kind, w, b, eps), *cs, interleaved, amp)


def out_bound(x, amp, kind, w, b, eps, dtype, ref):
    """Bound on |got - ref| of one rounded output: half a step of its type, and the 32-bit arithmetic before that.  With M the largest
    magnitude a row's values reach in it -- amp (max|x| / sigma max|w| + max|b|) -- every value is two products of such numbers with a
    cosine and a sine: their own errors (the angle rounded to 2^-25 turns / pi ~ 1e-7 rad, the functions 2 ulp: 5 u each), 1 / sigma and
    the sums behind it (8 u), subtraction, weight, bias, amplitude, two products and a sum (8 u): below 32 u M, u = 2^-24."""
    m = x.abs().amax(-1, keepdim=True)
    if kind != "none":
        c = x - x.mean(-1, keepdim=True) if kind == "layer" else x
        m = m / (c.square().mean(-1, keepdim=True) + eps).sqrt()
    m = m * (1.0 if w is None else float(w.abs().max())) + (0.0 if b is None else float(b.abs().max()))
    return U[dtype] * ref.abs() + 32 * F32U * max(1.0, amp) * m
