"""Tensor-level wrappers over the C ABI (include/hma_hip.h).

PyTorch here is plumbing only: device memory, streams.  Every function enqueues HIP kernels on
the current stream through libhma_hip.so and raises if the library is missing -- there is no
eager / CPU fallback anywhere in this package.
"""
from __future__ import annotations

import contextlib
import ctypes as C
import math
from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import (A_BF16, A_BF16_AFFINE, A_F32, EPI_ATOMIC_F32, EPI_BF16, EPI_DGELU, EPI_DSILU, EPI_F32, EPI_GELU2,
                   EPI_RESID, EPI_SILU2, ChainABFwd, ChainABwd, ChainAFwd, ChainBFwd, ChainSBwd, ChainTBwd, AttnPaged, GemmNT, GemmTN, KvAppend, MlpBwd, MlpFwd, QkRope,
                   ReadoutCE)

BF16 = torch.bfloat16
F32 = torch.float32


def stream_ptr() -> int:
    return torch.cuda.current_stream().cuda_stream


def ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _kind(t: torch.Tensor, affine: bool = False) -> int:
    if t.dtype == F32:
        assert not affine
        return A_F32
    assert t.dtype == BF16, t.dtype
    return A_BF16_AFFINE if affine else A_BF16


def make_gemm_nt(*, A: int, lda: int, a_kind: int, W: int, ldw: int, M: int, N: int, K: int, epi: int, Cp: int, ldc: int,
                 bias: Optional[int] = None, gamma: Optional[int] = None, beta: Optional[int] = None,
                 a_group=(0, 0), c_group=(0, 0), C2: Optional[int] = None, ldc2: int = 0, U: Optional[int] = None,
                 ldu: int = 0, batch: int = 1, sA: int = 0, sW: int = 0, sBias: int = 0, sC: int = 0, sC2: int = 0,
                 sU: int = 0, ln_xhat: Optional[int] = None, ln_rstd: Optional[int] = None, ln_eps: float = 0.0,
                 ln_ss: Optional[int] = None, ln_xm: Optional[int] = None, ln_rows_per_frame: int = 0, drop_p: float = 0.0,
                 drop_salt: int = 0, drop_seed: Optional[int] = None) -> GemmNT:
    g = GemmNT()
    g.A, g.lda, g.a_kind = A, lda, a_kind
    g.a_group_rows, g.a_group_stride = a_group
    g.gamma, g.beta = gamma, beta
    g.W, g.ldw = W, ldw
    g.M, g.N, g.K = M, N, K
    g.epi, g.bias = epi, bias
    g.C, g.ldc = Cp, ldc
    g.c_group_rows, g.c_group_stride = c_group
    g.C2, g.ldc2, g.U, g.ldu = C2, ldc2, U, ldu
    g.batch, g.sA, g.sW, g.sBias, g.sC, g.sC2, g.sU = batch, sA, sW, sBias, sC, sC2, sU
    g.ln_xhat, g.ln_rstd, g.ln_ss, g.ln_xm = ln_xhat, ln_rstd, ln_ss, ln_xm
    g.ln_eps, g.ln_rows_per_frame = ln_eps, ln_rows_per_frame
    g.drop_p, g.drop_salt, g.drop_seed = drop_p, drop_salt, drop_seed
    return g


def make_gemm_tn(*, dY: int, ldy: int, y_kind: int, A: int, lda: int, a_kind: int, M: int, N: int, K: int, dW: int,
                 lddw: int, dBias: Optional[int] = None, gamma: Optional[int] = None, beta: Optional[int] = None,
                 y_group=(0, 0), a_group=(0, 0), splits: int = 0, batch: int = 1, sY: int = 0, sA: int = 0, sdW: int = 0,
                 sdBias: int = 0, ws: Optional[int] = None, ws_elems: int = 0, w_master: Optional[int] = None,
                 dgamma: Optional[int] = None, dbeta: Optional[int] = None) -> GemmTN:
    g = GemmTN()
    g.dY, g.ldy, g.y_kind = dY, ldy, y_kind
    g.y_group_rows, g.y_group_stride = y_group
    g.A, g.lda, g.a_kind = A, lda, a_kind
    g.a_group_rows, g.a_group_stride = a_group
    g.gamma, g.beta = gamma, beta
    g.M, g.N, g.K = M, N, K
    g.dW, g.lddw, g.dBias = dW, lddw, dBias
    if splits <= 0:
        tiles = (N // 128) * (K // 128) * max(batch, 1)
        splits = max(1, min((M + 63) // 64, 1024 // max(tiles, 1)))
    g.splits, g.batch = splits, batch
    g.sY, g.sA, g.sdW, g.sdBias = sY, sA, sdW, sdBias
    g.ws, g.ws_elems = ws, ws_elems
    g.w_master, g.dgamma, g.dbeta = w_master, dgamma, dbeta
    return g


def make_mlp_fwd(*, M: int, xhat: int, x: int, w1p: int, w2p: int, b1: int, b2: Optional[int] = None,
                 ln_xhat: Optional[int] = None, ln_rstd: Optional[int] = None, ln_eps: float = 1e-5) -> MlpFwd:
    g = MlpFwd()
    g.xhat, g.x, g.w1p, g.w2p, g.b1, g.b2 = xhat, x, w1p, w2p, b1, b2
    g.ln_xhat, g.ln_rstd, g.ln_eps, g.M = ln_xhat, ln_rstd, ln_eps, M
    return g


def make_mlp_bwd(*, M: int, xhat: int, rstd: int, dy: int, dx: int, dx_bf16: int, w1p: int, w2tp: int, w1tp: int, b1: int,
                 hg: int, du: int, drop_p: float = 0.0, drop_salt: int = 0, drop_seed: Optional[int] = None,
                 dy_drop: Optional[int] = None) -> MlpBwd:
    g = MlpBwd()
    g.xhat, g.rstd, g.dy, g.dx, g.dx_bf16 = xhat, rstd, dy, dx, dx_bf16
    g.w1p, g.w2tp, g.w1tp, g.b1, g.hg, g.du, g.M = w1p, w2tp, w1tp, b1, hg, du, M
    g.drop_p, g.drop_salt, g.drop_seed, g.dy_drop = drop_p, drop_salt, drop_seed, dy_drop
    return g


def chain_pack(src: torch.Tensor, *, kind: int, rows: int, cols: int, row_stride: int, col_stride: int,
               row_scale: Optional[torch.Tensor] = None, col_scale: Optional[torch.Tensor] = None,
               out: Optional[torch.Tensor] = None, bundle_stride: int = 1, bundle_offset: int = 0) -> torch.Tensor:
    """Bundles of one logical [rows][cols] matrix (hma_chain_pack) in the chains' streaming order; bf16, 8192 elements per bundle.
    Bundle b lands at bundle slot bundle_offset + b * bundle_stride of `out`."""
    nb = (rows if kind == 0 else cols) // 32
    if out is None:
        out = torch.empty((bundle_offset + (nb - 1) * bundle_stride + 1) * 8192, dtype=BF16, device=src.device)
    _lib.call("hma_chain_pack", stream_ptr(), ptr(src), row_stride, col_stride, ptr(row_scale), ptr(col_scale),
              out.data_ptr() + 2 * 8192 * bundle_offset, kind, rows, cols, 1, 0, 0, bundle_stride)
    return out


def _chain_weights(w, segs) -> None:
    for i in range(4):
        w.seg[i] = segs[i][0] if i < len(segs) else None
        w.bundles[i] = segs[i][1] if i < len(segs) else 0


def make_chain_a_fwd(*, M: int, segs, o: int, x: int, qkv: int, ldq: int = 768, ss: Optional[int] = None,
                     b_proj: Optional[int] = None, b_lin: Optional[int] = None, b_qkv: Optional[int] = None,
                     xhat: Optional[int] = None, xm: Optional[int] = None, rstd: Optional[int] = None,
                     x_bf16: Optional[int] = None, q_group=(0, 0), rows_per_frame: int = 0, use_mod: bool = True) -> ChainAFwd:
    """segs: [(device pointer, bundles)] of the packed proj (8), linear_out (8, use_mod only) and qkv (24) weights."""
    g = ChainAFwd()
    _chain_weights(g.w, segs)
    g.o, g.x, g.ss = o, x, ss
    g.b_proj, g.b_lin, g.b_qkv = b_proj, b_lin, b_qkv
    g.xhat, g.xm, g.rstd, g.x_bf16 = xhat, xm, rstd, x_bf16
    g.qkv, g.ldq = qkv, ldq
    g.q_group_rows, g.q_group_stride = q_group
    g.M, g.rows_per_frame, g.use_mod = M, rows_per_frame, 1 if use_mod else 0
    return g


def make_chain_b_fwd(*, M: int, segs, o: int, x: int, b1: int, b_proj: Optional[int] = None, b2: Optional[int] = None,
                     b_qkv: Optional[int] = None, qkv: Optional[int] = None, ldq: int = 768, ln_eps: float = 1e-5,
                     xhat2: Optional[int] = None, rstd2: Optional[int] = None, xhat1n: Optional[int] = None,
                     rstd1n: Optional[int] = None, drop_p: float = 0.0, drop_salt: int = 0,
                     drop_seed: Optional[int] = None) -> ChainBFwd:
    """segs: packed proj (8), the 64 alternating fc1 / fc2 bundles, and -- with `qkv` -- the next block's folded qkv (24)."""
    g = ChainBFwd()
    _chain_weights(g.w, segs)
    g.o, g.x = o, x
    g.b_proj, g.b1, g.b2, g.b_qkv = b_proj, b1, b2, b_qkv
    g.qkv, g.ldq, g.M, g.ln_eps = qkv, ldq, M, ln_eps
    g.xhat2, g.rstd2, g.xhat1n, g.rstd1n = xhat2, rstd2, xhat1n, rstd1n
    g.drop_p, g.drop_salt, g.drop_seed = drop_p, drop_salt, drop_seed
    return g


def make_readout_ce(*, rows: int, segs, x: int, bias: Optional[int], input_ids: int, labels: int, stats: int, dlogits: Optional[int],
                    grad_scale_dev: Optional[int], grad_scale: float, S: int, SA: int, T: int, mask_id: int,
                    label_smoothing: float) -> ReadoutCE:
    """segs: the 32 N-block bundles of out_x_proj.weight (chain_pack kind 0)."""
    g = ReadoutCE()
    _chain_weights(g.w, segs)
    g.x, g.bias, g.input_ids, g.labels, g.stats, g.dlogits, g.grad_scale_dev = x, bias, input_ids, labels, stats, dlogits, grad_scale_dev
    g.rows, g.mask_id, g.S, g.SA, g.T, g.grad_scale, g.label_smoothing = rows, mask_id, S, SA, T, grad_scale, label_smoothing
    return g


def make_chain_a_bwd(*, M: int, segs, dqkv: int, dx: int, dx1_bf16: int, d_o: int, ldq: int = 768, xhat: Optional[int] = None,
                     rstd: Optional[int] = None, ss: Optional[int] = None, dx2_bf16: Optional[int] = None,
                     dss: Optional[int] = None, rows_per_frame: int = 0, use_mod: bool = True) -> ChainABwd:
    """segs: packed qkv^T (3 x 8), linear_out^T (8, use_mod only), proj^T (8)."""
    g = ChainABwd()
    _chain_weights(g.w, segs)
    g.dqkv, g.ldq, g.dx = dqkv, ldq, dx
    g.xhat, g.rstd, g.ss = xhat, rstd, ss
    g.dx2_bf16, g.dx1_bf16, g.d_o, g.dss = dx2_bf16, dx1_bf16, d_o, dss
    g.M, g.rows_per_frame, g.use_mod = M, rows_per_frame, 1 if use_mod else 0
    return g


def make_chain_ab_fwd(*, B: int, SA: int, segs, o_s: int, x: int, b1: int, x2b: int, qkv_t: int, o_t: int, xhat2: int, rstd2: int,
                      attn_scale: float, ss: Optional[int] = None, xhat_m: Optional[int] = None, xm: Optional[int] = None,
                      rstd_m: Optional[int] = None, b_proj_s: Optional[int] = None, b_lin: Optional[int] = None,
                      b_qkv_t: Optional[int] = None, b_proj_t: Optional[int] = None, b2: Optional[int] = None, b_qkv_s: Optional[int] = None,
                      xhat1n: Optional[int] = None, rstd1n: Optional[int] = None, qkv_s: Optional[int] = None, ln_eps: float = 1e-5,
                      T: int = 16, drop_p: float = 0.0, drop_salt: int = 0, drop_seed: Optional[int] = None) -> ChainABFwd:
    """segs: [(pointer, bundles)] x 6 = proj_s (8), linear_out (8; (None, 0) for blocks without action tokens: then ss / xhat_m / xm /
    rstd_m are not used), temporal qkv (24), proj_t (8), the 64 fc1 / fc2 bundles, the next block's folded spatial qkv (24; (None, 0)
    for the last block).  drop_p > 0: the two nn.Dropout sites of the MLP (salts drop_salt, drop_salt + 1)."""
    g = ChainABFwd()
    for i in range(6):
        g.seg[i] = segs[i][0] if i < len(segs) else None
        g.bundles[i] = segs[i][1] if i < len(segs) else 0
    g.o_s, g.x, g.ss = o_s, x, ss
    g.b_proj_s, g.b_lin, g.b_qkv_t, g.b_proj_t, g.b1, g.b2, g.b_qkv_s = b_proj_s, b_lin, b_qkv_t, b_proj_t, b1, b2, b_qkv_s
    g.xhat_m, g.xm, g.rstd_m, g.x2b, g.qkv_t, g.o_t = xhat_m, xm, rstd_m, x2b, qkv_t, o_t
    g.xhat2, g.rstd2, g.xhat1n, g.rstd1n, g.qkv_s = xhat2, rstd2, xhat1n, rstd1n, qkv_s
    g.B, g.T, g.SA, g.attn_scale, g.ln_eps = B, T, SA, attn_scale, ln_eps
    g.drop_p, g.drop_salt, g.drop_seed = drop_p, drop_salt, drop_seed
    return g


def make_chain_s_bwd(*, M: int, segs, dqkv: int, dx: int, xhat: int, rstd: int, dx_bf16: int, ldq: int = 768, hb_rows: int = 0) -> ChainSBwd:
    """segs: packed qkv^T (3 x 8) of the spatial attention with norm1's gamma folded into the output rows.  hb_rows > 0: dqkv in the
    head-blocked order of hma_attn_spatial_bwd_blocked (rows per frame)."""
    g = ChainSBwd()
    _chain_weights(g.w, segs)
    g.dqkv, g.ldq, g.dx = dqkv, ldq, dx
    g.xhat, g.rstd, g.dx_bf16 = xhat, rstd, dx_bf16
    g.M, g.hb_rows = M, hb_rows
    return g


def make_chain_t_bwd(*, B: int, SA: int, segs, dy_bf16: int, qkv: int, dqkv: int, attn_scale: float, T: int = 16) -> ChainTBwd:
    """segs: the packed transposed temporal projection (8 bundles).  Rows (b, t, s), M = T B SA, 1 <= T <= 16."""
    g = ChainTBwd()
    _chain_weights(g.w, segs)
    g.dy_bf16, g.qkv, g.dqkv = dy_bf16, qkv, dqkv
    g.B, g.T, g.SA, g.attn_scale = B, T, SA, attn_scale
    return g


# ----------------------------------------------------------------------------------------------
# tensor conveniences (used by the module-level API and the parity tests)
# ----------------------------------------------------------------------------------------------
def linear(x: torch.Tensor, w_bf16: torch.Tensor, bias: Optional[torch.Tensor] = None, *, epi: int = EPI_F32,
           gamma=None, beta=None, out: Optional[torch.Tensor] = None, out2: Optional[torch.Tensor] = None,
           aux: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y = x' @ w^T (+ bias) with x (M, K) bf16/f32 and w (N, K) bf16; epilogue per `epi`."""
    assert x.dim() == 2 and w_bf16.dim() == 2 and w_bf16.dtype == BF16 and x.is_contiguous() and w_bf16.is_contiguous()
    M, K = x.shape
    N = w_bf16.shape[0]
    if out is None:
        dt = F32 if epi in (EPI_F32, EPI_RESID, EPI_ATOMIC_F32) else BF16
        out = torch.empty(M, N, dtype=dt, device=x.device)
    g = make_gemm_nt(A=ptr(x), lda=K, a_kind=_kind(x, gamma is not None), W=ptr(w_bf16), ldw=K, M=M, N=N, K=K, epi=epi,
                     Cp=ptr(out), ldc=N, bias=ptr(bias), gamma=ptr(gamma), beta=ptr(beta), C2=ptr(out2), ldc2=N,
                     U=ptr(aux), ldu=N)
    _lib.call("hma_gemm_nt", stream_ptr(), C.byref(g))
    return out


def linear_wgrad(dy: torch.Tensor, x: torch.Tensor, dW: torch.Tensor, dbias: Optional[torch.Tensor] = None, *,
                 gamma=None, beta=None, splits: int = 0, ws: Optional[torch.Tensor] = None) -> None:
    """dW (N, K) fp32 += dy^T x' ; dbias += column sums of dy."""
    M, N = dy.shape
    K = x.shape[1]
    g = make_gemm_tn(dY=ptr(dy), ldy=N, y_kind=_kind(dy), A=ptr(x), lda=K, a_kind=_kind(x, gamma is not None), M=M, N=N,
                     K=K, dW=ptr(dW), lddw=K, dBias=ptr(dbias), gamma=ptr(gamma), beta=ptr(beta), splits=splits,
                     ws=ptr(ws), ws_elems=0 if ws is None else ws.numel())
    _lib.call("hma_gemm_tn", stream_ptr(), C.byref(g))


def ln_fwd(x: torch.Tensor, eps: float):
    rows = x.numel() // 256
    xhat = torch.empty(x.shape, dtype=BF16, device=x.device)
    rstd = torch.empty(rows, dtype=F32, device=x.device)
    _lib.call("hma_ln_fwd", stream_ptr(), ptr(x), ptr(xhat), ptr(rstd), rows, eps)
    return xhat, rstd


def qknorm_fwd(qkv: torch.Tensor, gamma: torch.Tensor, beta: torch.Tensor, eps: float = 1e-5, save_raw: bool = True):
    """qk_norm=True (hma/model/attention.py:31-35,44-48): per-head LayerNorm of the q | k parts of a packed (rows, 768) bf16 qkv.
    Returns (normalised copy, pre-norm q | k (rows, 512) for the backward or None)."""
    out = qkv.clone()
    raw = torch.empty(qkv.shape[0], 512, dtype=BF16, device=qkv.device) if save_raw else None
    _lib.call("hma_qknorm_fwd", stream_ptr(), ptr(out), 768, ptr(raw), ptr(gamma), ptr(beta), eps, qkv.shape[0], 0, 0)
    return out, raw


def qknorm_bwd(dqkv: torch.Tensor, raw: torch.Tensor, gamma: torch.Tensor, eps: float = 1e-5):
    """(gradient wrt the raw qkv, dgamma [32], dbeta [32]) from the gradient wrt the normalised one."""
    out = dqkv.clone()
    dg = torch.zeros(32, dtype=F32, device=dqkv.device)
    db = torch.zeros(32, dtype=F32, device=dqkv.device)
    _lib.call("hma_qknorm_bwd", stream_ptr(), ptr(out), 768, ptr(raw), ptr(gamma), eps, ptr(dg), ptr(db), dqkv.shape[0])
    return out, dg, db


def attn_spatial_fwd(qkv: torch.Tensor, frames: int, n: int, scale: float):
    o = torch.empty(frames * n, 256, dtype=BF16, device=qkv.device)
    lse = torch.empty(frames * n, 8, dtype=F32, device=qkv.device)
    _lib.call("hma_attn_spatial_fwd", stream_ptr(), ptr(qkv), ptr(o), ptr(lse), frames, n, scale)
    return o, lse


def attn_spatial_bwd(qkv, o, d_o, lse, frames: int, n: int, scale: float, blocked: bool = False):
    """dqkv [frames * n, 768] row-major; `blocked`: in the head-blocked order (`headblk_to_rows` turns it back)."""
    delta = torch.empty_like(lse)
    dqkv = torch.empty_like(qkv)
    _lib.call("hma_attn_spatial_bwd_blocked" if blocked else "hma_attn_spatial_bwd", stream_ptr(), ptr(qkv), ptr(o), ptr(d_o), ptr(lse),
              ptr(delta), ptr(dqkv), frames, n, scale)
    return dqkv


def headblk_to_rows(t: torch.Tensor, n: int) -> torch.Tensor:
    """[M, 256 W] head-blocked (HMA_A_BF16_HEADBLK: [frame][head][part][n][32]) -> row-major [M, 256 W]."""
    M, C = t.shape
    W = C // 256
    return t.reshape(M // n, 8, W, n, 32).permute(0, 3, 2, 1, 4).reshape(M, C).contiguous()


def rows_to_headblk(t: torch.Tensor, n: int) -> torch.Tensor:
    M, C = t.shape
    W = C // 256
    return t.reshape(M // n, n, W, 8, 32).permute(0, 3, 2, 1, 4).reshape(M, C).contiguous()


def attn_temporal_fwd(qkv: torch.Tensor, batch: int, T: int, n_s: int, scale: float):
    o = torch.empty(batch * T * n_s, 256, dtype=BF16, device=qkv.device)
    _lib.call("hma_attn_temporal_fwd", stream_ptr(), ptr(qkv), ptr(o), batch, T, n_s, scale)
    return o


def attn_temporal_bwd(qkv, o, d_o, batch: int, T: int, n_s: int, scale: float):
    dqkv = torch.empty_like(qkv)
    _lib.call("hma_attn_temporal_bwd", stream_ptr(), ptr(qkv), ptr(o), ptr(d_o), ptr(dqkv), batch, T, n_s, scale)
    return dqkv


# ----------------------------------------------------------------------------------------------
# positions, norms of queries / keys, paged cache (csrc/rope.hip)
# ----------------------------------------------------------------------------------------------
F8 = torch.float8_e4m3fn
_DTYPE = {BF16: 0, torch.float16: 1, F32: 2}
_NORM = {"none": 0, "rms": 1, "layer": 2}
_QK_ROPE_WS_GROUPS = 768


# These wrappers stand in front of launches of a few microseconds: an argument structure is filled in one call (setting its 50 fields one by
# one took longer than the launch)
_QK_ROPE, _KV_APPEND, _ATTN_PAGED = (_lib.packer(c) for c in (QkRope, KvAppend, AttnPaged))
_NO_GRADIENTS = (0,) * 14  # the fields of QkRope behind k_out
_HERE = contextlib.nullcontext()


def _device(*ts: Optional[torch.Tensor]):
    """Every tensor on the first one's GPU; the context in which its kernels are launched (nothing where that GPU is the current one).
    These wrappers stand in front of launches of a few microseconds: they look at each tensor once and hold their tests to plain
    comparisons."""
    i = ts[0].get_device()
    if i < 0:
        raise RuntimeError("hma ops run on the HIP kernels only (got a %s tensor)" % ts[0].device.type)
    for t in ts:
        if t is not None and t.get_device() != i:
            raise ValueError(f"tensors on {ts[0].device} and {t.device}")
    return _HERE if i == torch._C._cuda_getDevice() else torch.cuda.device(i)


def _stream(t: torch.Tensor) -> int:
    return torch._C._cuda_getCurrentRawStream(t.get_device())


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _at(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _like(t: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _rows16(t: torch.Tensor) -> torch.Tensor:
    """(tokens, heads, d) with contiguous 16-byte aligned rows: t itself, or a contiguous copy where its strides are others."""
    s0, s1, s2 = t.stride()
    if s2 == 1 and not (s0 | s1) & (3 if t.dtype == F32 else 7) and not t.data_ptr() & 15:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def rope_freqs(rot: int, base: float = 10000.0, *, scaling: str = "none", factor: float = 1.0, trained: int = 8192, slow: float = 1.0,
               fast: float = 32.0, device="cuda") -> Tuple[torch.Tensor, float]:
    """(frequencies, float64 (rot / 2,) radians per position, amplitude) of rotary positions: base ** (-2 i / rot), for contexts `factor`
    times the `trained` length
      "linear": every frequency divided by the factor;
      "base":   the base raised so that the slowest pair is slowed by the factor and the fastest is not;
      "parts":  pairs that turn at most `slow` times over the trained length divided by the factor, those that turn `fast` times or more
                left, a linear ramp between; the amplitude is 1 + 0.1 ln(factor)."""
    _need(rot > 0 and rot % 2 == 0 and base > 1 and factor > 0 and trained > 0 and fast > slow, "rope_freqs: rot even and positive, base > 1, factor > 0, fast > slow")
    _need(scaling in ("none", "linear", "base", "parts"), f"rope_freqs: scaling {scaling!r}")
    if scaling == "base" and rot > 2:
        base = base * factor ** (rot / (rot - 2))
    f = base ** (-2.0 * torch.arange(rot // 2, dtype=torch.float64) / rot)
    amplitude = 1.0
    if scaling == "linear":
        f = f / factor
    elif scaling == "parts":
        keep = ((trained * f / (2 * math.pi) - slow) / (fast - slow)).clamp(0, 1)
        f = f * (keep + (1 - keep) / factor)
        amplitude = 1.0 + 0.1 * math.log(factor) if factor > 1 else 1.0
    return f.to(device), amplitude


# hma_rope_t in the order of its fields
def _rope_values(dtype, d: int, tokens: int, freqs, positions, axes, interleaved, amplitude, norm, q_weight, q_bias, k_weight, k_bias, eps) -> tuple:
    rot, f, a, at, pos64, n_axes, pos_stride = 0, 0, 0, 0, 0, 1, 0
    if freqs is not None:
        rot = 2 * freqs.numel()
        _need(freqs.dtype == torch.float64 and freqs.dim() == 1 and freqs.is_contiguous() and rot <= d, "freqs: float64 (rot / 2,) contiguous, rot <= head size")
        f = freqs.data_ptr()
    if positions is not None and rot:
        shape, stride, kind = positions.shape, positions.stride(), positions.dtype
        pos64 = kind == torch.int64
        _need((pos64 or kind == torch.int32) and len(shape) in (1, 2) and shape[-1] == tokens and (tokens <= 1 or stride[-1] == 1),
              "positions: int64 or int32, (tokens,) or (axes, tokens), contiguous over the tokens")
        at = positions.data_ptr()
        if len(shape) == 2:
            n_axes, pos_stride = shape[0], stride[0]
            _need(n_axes >= 1 and (axes is not None or n_axes == 1) and (n_axes == 1 or pos_stride >= tokens),
                  "positions of several axes need `axes` and rows that do not overlap")
    if axes is not None and rot:
        _need(axes.dtype == torch.int32 and axes.shape == freqs.shape and axes.is_contiguous(), "axes: int32 (rot / 2,) contiguous")
        a = axes.data_ptr()
    kind = _NORM.get(norm)
    if kind is None:
        raise ValueError(f"norm {norm!r}: none, rms or layer")
    w, wt = [0, 0, 0, 0], None
    for i, t in enumerate((q_weight, q_bias, k_weight, k_bias)):
        if t is not None:
            _need(kind and t.shape == (d,) and t.is_contiguous() and t.dtype in (F32, dtype) and wt in (None, t.dtype),
                  "norm weights: (head size,) contiguous, all fp32 or all of the rows' type, with a norm")
            wt = t.dtype
            w[i] = t.data_ptr()
    _need(kind == 2 or (q_bias is None and k_bias is None), "a bias goes with norm 'layer'")
    return f, a, at, pos_stride, *w, d, rot, bool(interleaved), kind, _DTYPE[dtype], wt in (None, F32), pos64, n_axes, eps, amplitude


def _qk_values(q, k, freqs, positions, axes, interleaved, amplitude, norm, q_weight, q_bias, k_weight, k_bias, eps):
    """q, k as the kernels read them, and the first fields of hma_qk_rope_t"""
    kind, qs, ks = q.dtype, q.shape, k.shape
    _need(len(qs) == 3 and len(ks) == 3 and qs[0] == ks[0] and qs[2] == ks[2] and kind == k.dtype and kind in _DTYPE,
          "q (tokens, heads, d) and k (tokens, kv heads, d) of one type: bf16, fp16 or fp32")
    _need(freqs is None or positions is not None, "a rotation needs positions")
    q, k = _rows16(q), _rows16(k)
    rope = _rope_values(kind, qs[2], qs[0], freqs, positions, axes, interleaved, amplitude, norm, q_weight, q_bias, k_weight, k_bias, eps)
    return q, k, (*rope, qs[0], qs[1], ks[1], q.data_ptr(), k.data_ptr(), *q.stride()[:2], *k.stride()[:2])


def qk_rope_fwd(q: torch.Tensor, k: torch.Tensor, freqs: Optional[torch.Tensor], positions: Optional[torch.Tensor], *, axes: Optional[torch.Tensor] = None,
                interleaved: bool = False, amplitude: float = 1.0, norm: str = "none", q_weight=None, q_bias=None, k_weight=None, k_bias=None,
                eps: float = 1e-5) -> Tuple[torch.Tensor, torch.Tensor]:
    """Norm of each head of q (tokens, heads, d) and k (tokens, kv heads, d) -- none, "rms" or "layer", weights (d,) -- and the rotation of
    its first 2 * len(freqs) values by positions * freqs, in one pass (hma_qk_rope_fwd).  bf16, fp16 or fp32; d a multiple of 8 up to 256;
    views of a packed projection need no copy.  positions (tokens,) or (axes, tokens) with `axes` int32 naming each pair's axis.  Returns
    contiguous (q, k)."""
    with _device(q, k, freqs, positions, axes, q_weight, q_bias, k_weight, k_bias):
        qr, kr, values = _qk_values(q, k, freqs, positions, axes, interleaved, amplitude, norm, q_weight, q_bias, k_weight, k_bias, eps)
        qo, ko = _like(q), _like(k)
        p = QkRope()
        _QK_ROPE.pack_into(p, 0, *values, qo.data_ptr(), ko.data_ptr(), *_NO_GRADIENTS)
        _lib.call("hma_qk_rope_fwd", _stream(q), C.byref(p))
    return qo, ko


def qk_rope_bwd(dy_q: torch.Tensor, dy_k: torch.Tensor, q: torch.Tensor, k: torch.Tensor, freqs, positions, *, axes=None, interleaved: bool = False,
                amplitude: float = 1.0, norm: str = "none", q_weight=None, q_bias=None, k_weight=None, k_bias=None, eps: float = 1e-5):
    """(dq, dk, d q_weight, d q_bias, d k_weight, d k_bias) of qk_rope_fwd from its inputs and the gradients of its outputs; the weights'
    gradients (None where there is no weight) are summed in 32 bits in a fixed order (hma_qk_rope_bwd)."""
    with _device(q, k, freqs, positions, axes, q_weight, q_bias, k_weight, k_bias, dy_q, dy_k):
        _need(dy_q.shape == q.shape and dy_k.shape == k.shape and dy_q.dtype == q.dtype and dy_k.dtype == k.dtype, "gradients of the shapes and type of q and k")
        qr, kr, values = _qk_values(q, k, freqs, positions, axes, interleaved, amplitude, norm, q_weight, q_bias, k_weight, k_bias, eps)
        gq, gk = _rows16(dy_q), _rows16(dy_k)
        dq, dk = _like(q), _like(k)
        dw = [None if w is None else torch.empty_like(w) for w in (q_weight, q_bias, k_weight, k_bias)]
        ws = torch.empty(_QK_ROPE_WS_GROUPS * 4 * q.shape[2], dtype=F32, device=q.device) if any(w is not None for w in dw) else None
        p = QkRope()
        _QK_ROPE.pack_into(p, 0, *values, 0, 0, gq.data_ptr(), gk.data_ptr(), *gq.stride()[:2], *gk.stride()[:2], dq.data_ptr(), dk.data_ptr(),
                           *(_at(w) for w in dw), _at(ws), 0 if ws is None else ws.numel())
        _lib.call("hma_qk_rope_bwd", _stream(q), C.byref(p))
    return (dq, dk, *dw)


def _cache_values(k_cache, v_cache, page_table, cu_seqlens, kv_lens, k_scale, v_scale, dtype) -> tuple:
    """The paged cache of hma_kv_append / hma_attn_paged_fwd: caches (pages, kv heads, page size, d), table int32 (sequences, pages of one).
    ((both caches, table, cu, lens, scales), (strides of both caches), stride of the table, (sequences, table's width, pages, page size, e4m3))"""
    shape, kind, table = k_cache.shape, k_cache.dtype, page_table.shape
    f8 = kind == F8
    _need(len(shape) == 4 and v_cache.shape == shape and v_cache.dtype == kind and (f8 or kind == dtype) and shape[2] > 0,
          "caches: (pages, kv heads, page size, d), both of the rows' type or both float8_e4m3fn")
    _need(len(table) == 2 and cu_seqlens.shape == (table[0] + 1,) and kv_lens.shape == (table[0],) and
          page_table.dtype == cu_seqlens.dtype == kv_lens.dtype == torch.int32 and cu_seqlens.is_contiguous() and kv_lens.is_contiguous(),
          "page_table (sequences, n), cu_seqlens (sequences + 1,), kv_lens (sequences,): int32")
    t0, t1 = page_table.stride()
    _need(table[1] <= 1 or t1 == 1, "page_table: a sequence's pages one behind the other")
    _need((k_scale is None) == (v_scale is None) == (not f8), "scales go with a float8_e4m3fn cache, and only with it")
    if f8:
        for s in (k_scale, v_scale):
            _need(s.dtype == F32 and s.shape == shape[1:2] and s.is_contiguous(), "k_scale, v_scale: fp32 (kv heads,) contiguous")
    k0, k1, k2, k3 = k_cache.stride()
    v0, v1, v2, v3 = v_cache.stride()
    _need(k3 == 1 and v3 == 1, "the caches' last dimension is contiguous")
    return ((k_cache.data_ptr(), v_cache.data_ptr(), page_table.data_ptr(), cu_seqlens.data_ptr(), kv_lens.data_ptr(), _at(k_scale), _at(v_scale)),
            (k0, k1, k2, v0, v1, v2), t0, (table[0], table[1], shape[0], shape[2], f8))


def kv_append(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor, cu_seqlens: torch.Tensor,
              kv_lens: torch.Tensor, *, q: Optional[torch.Tensor] = None, freqs=None, positions=None, axes=None, interleaved: bool = False,
              amplitude: float = 1.0, norm: str = "none", q_weight=None, q_bias=None, k_weight=None, k_bias=None, eps: float = 1e-5,
              k_scale=None, v_scale=None, q_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Puts the new keys (normed and rotated like qk_rope_fwd's) and values (tokens, kv heads, d) of a batch of sequences into the pages of
    k_cache / v_cache (pages, kv heads, page size, d), in place and in one launch (hma_kv_append).  Rows cu_seqlens[b] .. cu_seqlens[b + 1]
    belong to sequence b and become its last places: kv_lens[b] counts its tokens with the new ones; place p is row p % page size of page
    page_table[b, p // page size].  positions None: a token's place.  float8_e4m3fn caches store x / scale[head].  With q (tokens, heads,
    d): returns q normed and rotated (rows behind the last sequence zero; with q_out given they are left as they were).  A token without a
    place (kv_lens too small, a page number outside the cache) is not stored.  Pages written by one call belong to one sequence each."""
    with _device(k, v, k_cache, v_cache, page_table, cu_seqlens, kv_lens, q, freqs, positions, axes, q_weight, q_bias, k_weight, k_bias, k_scale,
                 v_scale, q_out):
        kind, shape = k.dtype, k.shape
        _need(len(shape) == 3 and v.shape == shape and v.dtype == kind and (kind == BF16 or kind == torch.float16), "k, v: (tokens, kv heads, d) of one type, bf16 or fp16")
        tokens, hk, d = shape
        (kc, vc, *lists), strides, table_stride, sizes = _cache_values(k_cache, v_cache, page_table, cu_seqlens, kv_lens, k_scale, v_scale, kind)
        _need(k_cache.shape[1] == hk and k_cache.shape[3] == d, "caches of k's heads and head size")
        rope = _rope_values(kind, d, tokens, freqs, positions, axes, interleaved, amplitude, norm, q_weight, q_bias, k_weight, k_bias, eps)
        _need(q is not None or (q_weight is None and q_bias is None and q_out is None), "q's weights and output without q")
        k, v = _rows16(k), _rows16(v)
        hq, q_at, q_to, q_tok, q_head, zero_tail = 0, 0, 0, 0, 0, 0
        if q is not None:
            qs = q.shape
            _need(len(qs) == 3 and qs[0] == tokens and qs[2] == d and q.dtype == kind, "q: (tokens, heads, d) of k's type")
            if q_out is None:
                q_out, zero_tail = _like(q), 1
            else:
                _need(q_out.shape == qs and q_out.dtype == kind and q_out.is_contiguous(), "q_out: q's shape and type, contiguous")
            q = _rows16(q)
            hq, q_at, q_to = qs[1], q.data_ptr(), q_out.data_ptr()
            q_tok, q_head, _ = q.stride()
        p = KvAppend()
        _KV_APPEND.pack_into(p, 0, *rope, tokens, hq, hk, q_at, k.data_ptr(), v.data_ptr(), q_tok, q_head, *k.stride()[:2], *v.stride()[:2], q_to,
                             kc, vc, *strides, *lists[:3], table_stride, *lists[3:], *sizes, zero_tail)
        _lib.call("hma_kv_append", _stream(k), C.byref(p))
    return q_out


def attn_paged_fwd(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor, cu_seqlens: torch.Tensor,
                   kv_lens: torch.Tensor, scale: float, *, causal: bool = True, window: int = 0, k_scale=None, v_scale=None,
                   out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(o, lse) of the new tokens q (tokens, heads, d) of a batch of sequences over the paged cache that kv_append filled (the same
    page_table, cu_seqlens and kv_lens): each is at its place and sees the places up to it (causal), the last `window` of them, or its whole
    sequence (causal=False: a chunk whose tokens see each other, such as a frame).  bf16 or fp16, d 32, 64 or 128, heads a multiple of
    the cache's; a cache of q's type or float8_e4m3fn with scales (hma_attn_paged_fwd).  lse fp32 (tokens, heads); a row that sees no key has o = 0,
    lse = -inf, and so have rows behind the last sequence (with out / lse given those are left as they were)."""
    with _device(q, k_cache, v_cache, page_table, cu_seqlens, kv_lens, k_scale, v_scale, out, lse):
        kind, shape, cache = q.dtype, q.shape, k_cache.shape
        _need(len(shape) == 3 and (kind == BF16 or kind == torch.float16) and len(cache) == 4 and cache[3] == shape[2] and cache[1] > 0 and
              shape[1] % cache[1] == 0, "q: (tokens, heads, d) bf16 or fp16, heads a multiple of the cache's, d the cache's")
        tokens, hq, d = shape
        if d not in (32, 64, 128):
            raise NotImplementedError("attn_paged is built for heads of 32, 64 and 128")
        _need(window >= 0 and (causal or window == 0), "a window goes with causal")
        _need(0 < scale < 3e38, "scale > 0")
        lists, strides, table_stride, sizes = _cache_values(k_cache, v_cache, page_table, cu_seqlens, kv_lens, k_scale, v_scale, kind)
        q = _rows16(q)
        _need((out is None) == (lse is None), "out and lse together")
        zero_tail = out is None
        if zero_tail:
            out, lse = _like(q), torch.empty(shape[:2], dtype=F32, device=q.device)
        else:
            _need(out.shape == shape and out.dtype == kind and out.is_contiguous() and lse.shape == shape[:2] and lse.dtype == F32 and
                  lse.is_contiguous(), "out: q's shape and type, lse: fp32 (tokens, heads), contiguous")
        q_tok, q_head, _ = q.stride()
        p, n = AttnPaged(), C.c_int64()
        _ATTN_PAGED.pack_into(p, 0, q.data_ptr(), out.data_ptr(), lse.data_ptr(), *lists, 0, 0, tokens, q_tok, q_head, *strides, table_stride, hq, cache[1], d,
                              _DTYPE[kind], *sizes, causal, min(window, 0x7fffffff), zero_tail, scale, 0)  # (lengths are below 2^31)
        _lib.call("hma_attn_paged_ws", C.byref(p), C.byref(n))
        if n.value:
            ws = torch.empty(n.value, dtype=torch.uint8, device=q.device)
            p.ws, p.ws_bytes = ws.data_ptr(), n.value
        _lib.call("hma_attn_paged_fwd", _stream(q), C.byref(p))
    return out, lse
