// Per-head norms of queries and keys with the rotary position rotation in the same pass, forward and backward, and the same pass
// with its keys (and the values) going into the pages of a cache.
//
// One row = one head of one token, D values:  y = R(pos) (u w + b),
//   u = x  |  x / sqrt(mean x^2 + eps)  |  (x - mean x) / sqrt(var x + eps),
// R rotates the first `rot` values in pairs -- (2 i, 2 i + 1) or (i, i + rot / 2) -- by the angle pos f_i and multiplies them by an
// amplitude.  Written per value e with its pair's other value p(e):  R x[e] = x[e] C[e] + x[p(e)] S[e], S carrying the sign; the values
// behind `rot` have C = 1, S = 0, so no lane branches.  R^T is the same with -S.
//
// Bound by the HBM bytes of the rows.  A lane holds 8 consecutive values of a row (16-byte loads and stores of 16-bit types), D / 8
// lanes (rounded up to a power of two) hold a row, 64 lanes several heads.  What would bound it instead is the angles: a sine and a
// cosine cost more than everything else that happens to a value, and every head of a token needs the same ones.  So a workgroup takes
// a tile of tokens, its threads first compute the tile's C / S table once (about one angle per thread) into LDS, and the heads read it.
// Angles: position times frequency in 64 bits, reduced to a fraction of a turn there, rounded to 32 bits after that -- a 32-bit product
// at position 10^6 is off by 0.03 rad.
// Reductions: everything in 32 bits; each output is rounded once.
#include "hma_common.h"
#include "../../include/hma_hip.h"

using namespace hma;

namespace {

constexpr int TPB = 256;    // threads of a workgroup
constexpr int WAVES = TPB / 64;
constexpr int TABLE = 512;  // C and S values (tokens x D) of a tile: two per thread each
constexpr int MAX_TT = 16;  // tokens of a tile

struct Bf16 { uint16_t v; };
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));

template <typename T> struct Io;
template <> struct Io<Bf16> {
  typedef uint4 raw;
  static __device__ __forceinline__ raw load(const void* p, int64_t i) { return *reinterpret_cast<const uint4*>((const uint16_t*)p + i); }
  static __device__ __forceinline__ void unpack(const raw& r, float* f) { unpack8(r, f); }
  static __device__ __forceinline__ void store(void* p, int64_t i, const float* f) { *reinterpret_cast<uint4*>((uint16_t*)p + i) = pack8(f); }
  static __device__ __forceinline__ float one(const void* p, int64_t i) { return from_bf16(((const uint16_t*)p)[i]); }
  static __device__ __forceinline__ void put(void* p, int64_t i, float v) { ((uint16_t*)p)[i] = to_bf16(v); }
};
template <> struct Io<_Float16> {
  typedef uint4 raw;
  static __device__ __forceinline__ raw load(const void* p, int64_t i) { return *reinterpret_cast<const uint4*>((const _Float16*)p + i); }
  static __device__ __forceinline__ void unpack(const raw& r, float* f) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const half2_t h = __builtin_bit_cast(half2_t, w[i]);
      f[2 * i] = (float)h[0];
      f[2 * i + 1] = (float)h[1];
    }
  }
  static __device__ __forceinline__ void store(void* p, int64_t i, const float* f) {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const half2_t h = {(_Float16)f[2 * j], (_Float16)f[2 * j + 1]};
      w[j] = __builtin_bit_cast(uint32_t, h);
    }
    *reinterpret_cast<uint4*>((_Float16*)p + i) = make_uint4(w[0], w[1], w[2], w[3]);
  }
  static __device__ __forceinline__ float one(const void* p, int64_t i) { return (float)((const _Float16*)p)[i]; }
  static __device__ __forceinline__ void put(void* p, int64_t i, float v) { ((_Float16*)p)[i] = (_Float16)v; }
};
template <> struct Io<float> {
  struct raw { float4 a, b; };
  static __device__ __forceinline__ raw load(const void* p, int64_t i) {
    const float4* q = reinterpret_cast<const float4*>((const float*)p + i);
    return raw{q[0], q[1]};
  }
  static __device__ __forceinline__ void unpack(const raw& r, float* f) {
    f[0] = r.a.x; f[1] = r.a.y; f[2] = r.a.z; f[3] = r.a.w;
    f[4] = r.b.x; f[5] = r.b.y; f[6] = r.b.z; f[7] = r.b.w;
  }
  static __device__ __forceinline__ void store(void* p, int64_t i, const float* f) {
    float4* q = reinterpret_cast<float4*>((float*)p + i);
    q[0] = make_float4(f[0], f[1], f[2], f[3]);
    q[1] = make_float4(f[4], f[5], f[6], f[7]);
  }
  static __device__ __forceinline__ float one(const void* p, int64_t i) { return ((const float*)p)[i]; }
  static __device__ __forceinline__ void put(void* p, int64_t i, float v) { ((float*)p)[i] = v; }
};

// 8 values -> 8 e4m3 bytes, nearest even, clamped to the type's largest value (a NaN stays one)
__device__ __forceinline__ float sat8(float x) { return x != x ? x : __builtin_amdgcn_fmed3f(x, -448.f, 448.f); }
__device__ __forceinline__ void store_e4m3(void* p, int64_t i, const float* f, float mul) {
  uint2 w;
  int a = 0, b = 0;
  a = __builtin_amdgcn_cvt_pk_fp8_f32(sat8(f[0] * mul), sat8(f[1] * mul), a, false);
  a = __builtin_amdgcn_cvt_pk_fp8_f32(sat8(f[2] * mul), sat8(f[3] * mul), a, true);
  b = __builtin_amdgcn_cvt_pk_fp8_f32(sat8(f[4] * mul), sat8(f[5] * mul), b, false);
  b = __builtin_amdgcn_cvt_pk_fp8_f32(sat8(f[6] * mul), sat8(f[7] * mul), b, true);
  w.x = (uint32_t)a;
  w.y = (uint32_t)b;
  *reinterpret_cast<uint2*>((uint8_t*)p + i) = w;
}

// Sum over the lg (1, 2, .. 32) lanes that hold a row, in each of them
__device__ __forceinline__ float row_sum(float v, int lg) {
  if (lg > 1) v += dpp_f32<0xB1>(v);
  if (lg > 2) v += dpp_f32<0x4E>(v);
  if (lg > 4) v += dpp_f32<0x141>(v);
  if (lg > 8) v += dpp_f32<0x140>(v);
  if (lg > 16) v += __shfl_xor(v, 16, 64);
  return v;
}
__device__ __forceinline__ void wave_lds_order() {  // this wave's LDS writes before its LDS reads
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// What the three kernels share of their arguments
struct Shape {
  const double* freqs;
  const int32_t* axes;
  const void* positions;
  const void* w[2][2];  // [q | k][weight | bias]
  int64_t tokens, pos_stride;
  int32_t hq, hk, d, rot, inter, norm, w_f32, pos64, n_axes, lg, hp, tt, passes, py;
  float eps, amp;
};

struct Lds {
  float c[TABLE], s[TABLE];
  float w[2][2][256];
  float xch[WAVES][64 * 8];
  int32_t page[MAX_TT], off[MAX_TT];
  int64_t pos[MAX_TT];
};

__device__ __forceinline__ float weight_at(const Shape& a, const void* p, int i, bool is_bf16) {
  if (a.w_f32) return ((const float*)p)[i];
  return is_bf16 ? Io<Bf16>::one(p, i) : Io<_Float16>::one(p, i);
}
template <typename T> struct IsBf16 { static constexpr bool value = false; };
template <> struct IsBf16<Bf16> { static constexpr bool value = true; };

// The norms' weights into LDS (1 and 0 where there are none)
template <typename T>
__device__ __forceinline__ void stage_weights(const Shape& a, Lds& L) {
  for (int i = threadIdx.x; i < 4 * a.d; i += TPB) {
    const int kind = i / (2 * a.d), which = (i / a.d) & 1, e = i % a.d;
    const void* p = a.w[kind][which];
    L.w[kind][which][e] = p ? weight_at(a, p, e, IsBf16<T>::value) : (which ? 0.f : 1.f);
  }
}

// The tile's table: C and S of every token and value.  `own` = positions come from L.pos (already in LDS).
__device__ __forceinline__ void stage_angles(const Shape& a, Lds& L, int64_t tok0, int nt, bool own) {
  const int half = a.rot >> 1, hd = a.d >> 1;
  for (int i = threadIdx.x; i < nt * hd; i += TPB) {
    const int t = i / hd, p = i - t * hd;
    float c = 1.f, s = 0.f;
    int e0 = 2 * p, e1 = 2 * p + 1;  // where the pair's two values sit
    if (p < half) {
      double pos;
      if (own) {
        pos = (double)L.pos[t];
      } else {
        int ax = a.axes ? a.axes[p] : 0;
        ax = min(max(ax, 0), a.n_axes - 1);
        const int64_t at = ax * a.pos_stride + tok0 + t;
        pos = a.pos64 ? (double)((const int64_t*)a.positions)[at] : (double)((const int32_t*)a.positions)[at];
      }
      double x = pos * (a.freqs[p] * 0.15915494309189533577);  // turns
      x -= rint(x);
      sincospif((float)(2.0 * x), &s, &c);
      c *= a.amp;
      s *= a.amp;
      if (!a.inter) e0 = p, e1 = p + half;
    }
    float* C = L.c + t * a.d;
    float* S = L.s + t * a.d;
    C[e0] = c; C[e1] = c;
    S[e0] = -s; S[e1] = s;
  }
}

__device__ __forceinline__ void read8(const float* p, float* f) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
  f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
}

// y = x C + x[partner] S (sgn = -1: the transposed rotation) for the 8 values e0 .. e0 + 7 of each lane's row
__device__ __forceinline__ void rotate(const Shape& a, float* xch, int lane, int e0, const float* x, const float* c, const float* s, float sgn, float* y) {
  float p[8];
  if (a.inter) {
#pragma unroll
    for (int e = 0; e < 8; ++e) p[e] = x[e ^ 1];
  } else {
    float* mine = xch + lane * 8;
    *reinterpret_cast<float4*>(mine) = make_float4(x[0], x[1], x[2], x[3]);
    *reinterpret_cast<float4*>(mine + 4) = make_float4(x[4], x[5], x[6], x[7]);
    wave_lds_order();
    const int half = a.rot >> 1;
    const float* row = mine - e0;
    if ((half & 3) == 0) {
#pragma unroll
      for (int q = 0; q < 8; q += 4) {
        const int e = e0 + q, at = e < half ? e + half : e < a.rot ? e - half : e;
        const float4 v = *reinterpret_cast<const float4*>(row + at);
        p[q] = v.x; p[q + 1] = v.y; p[q + 2] = v.z; p[q + 3] = v.w;
      }
    } else {
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const int e = e0 + q, at = e < half ? e + half : e < a.rot ? e - half : e;
        p[q] = row[at];
      }
    }
    wave_lds_order();  // the next rows are written behind these reads
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) y[e] = __builtin_fmaf(p[e] * sgn, s[e], x[e] * c[e]);
}

// mean (layer) and 1 / deviation of a row; lanes behind the row hold zeros
__device__ __forceinline__ void row_stats(const Shape& a, const float* x, bool in_row, float inv_d, float& mean, float& rstd) {
  mean = 0.f;
  if (a.norm == HMA_NORM_LAYER) {
    float t = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) t += x[e];
    mean = row_sum(t, a.lg) * inv_d;
  }
  float q = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) q = __builtin_fmaf(x[e] - mean, x[e] - mean, q);
  q = row_sum(in_row ? q : 0.f, a.lg);
  rstd = rsqrtf(q * inv_d + a.eps);
}

// ------------------------------------------------------------------------------------- forward, and appending to a paged cache
struct FwdArgs {
  Shape s;
  const void *q, *k, *v;
  void *q_out, *k_out, *kc, *vc;
  int64_t q_tok, q_head, k_tok, k_head, v_tok, v_head;
  // cache
  const int32_t *table, *cu, *lens;
  const float *k_scale, *v_scale;
  int64_t table_stride, kc_page, kc_head, kc_tok, vc_page, vc_head, vc_tok;
  int32_t seqs, table_w, pages, page, zero_tail;
};

// Sequence of a row: how many of cu[1 .. n] are <= row, by the whole wave (64 candidates a step)
__device__ __forceinline__ int find_seq(const int32_t* cu, int n, int64_t row, int lane) {
  int lo = 0;
  while (n > 64) {
    const int st = (n + 63) >> 6, i = (lane + 1) * st;
    const int c = __popcll(__ballot(i <= n && cu[lo + min(i, n)] <= row));
    lo += c * st;
    n = min(st, n - c * st);
  }
  if (n <= 0) return lo;
  return lo + __popcll(__ballot(lane < n && cu[lo + min(lane + 1, n)] <= row));
}

template <typename T, bool APPEND, bool F8>
__global__ __launch_bounds__(TPB) void rope_fwd_kernel(const FwdArgs g) {
  __shared__ Lds L;
  const Shape& a = g.s;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t tok0 = (int64_t)blockIdx.x * a.tt;
  const int nt = (int)min((int64_t)a.tt, a.tokens - tok0);
  // this wave's units: a unit is one token's group of hp heads; blockIdx.y takes a share of every token's groups
  const int pp = (a.passes + a.py - 1) / a.py, p_lo = blockIdx.y * pp, np = min(pp, a.passes - p_lo);
  if (np <= 0) return;
  const int units = nt * np, per = (units + WAVES - 1) / WAVES, u_lo = wave * per, u_hi = min(units, u_lo + per);
  const int dl = lane & (a.lg - 1), sub = lane / a.lg, e0 = dl * 8;
  const bool in_row = e0 < a.d;
  const int heads = a.hq + a.hk + (APPEND ? a.hk : 0);
  const float inv_d = 1.0f / (float)a.d;

  auto fetch = [&](int u) {
    const int t = u / np, h = min((p_lo + u - t * np) * a.hp + sub, heads - 1);
    const int64_t tok = tok0 + t;
    const int e = in_row ? e0 : 0;
    if (h < a.hq) return Io<T>::load(g.q, tok * g.q_tok + h * g.q_head + e);
    if (!APPEND || h < a.hq + a.hk) return Io<T>::load(g.k, tok * g.k_tok + (h - a.hq) * g.k_head + e);
    return Io<T>::load(g.v, tok * g.v_tok + (h - a.hq - a.hk) * g.v_head + e);
  };
  typename Io<T>::raw nx;
  if (u_lo < u_hi) nx = fetch(u_lo);

  if (APPEND) {
    for (int t = wave; t < nt; t += WAVES) {
      const int64_t row = tok0 + t;
      const int b = find_seq(g.cu, g.seqs, row, lane);
      int32_t page = -1, off = 0;
      int64_t place = 0;
      if (b < g.seqs && row >= g.cu[b]) {
        place = (int64_t)g.lens[b] - g.cu[b + 1] + row;
        const int64_t pi = place / g.page;
        if (place >= 0 && pi < g.table_w) {
          page = g.table[b * g.table_stride + pi];
          if (page < 0 || page >= g.pages) page = -1;
          off = (int32_t)(place - pi * g.page);
        }
        if (page < 0) off = -1;  // belongs to a sequence, has no place in the cache
      } else {
        off = -2;  // behind the last sequence
      }
      if (lane == 0) L.page[t] = page, L.off[t] = off, L.pos[t] = place;
    }
    __syncthreads();
  }
  stage_weights<T>(a, L);
  stage_angles(a, L, tok0, nt, APPEND && !g.s.positions);
  __syncthreads();

  int t_cur = -1;
  bool first = true, k_cur = false;
  float c[8], s[8], w[8], b[8];
  for (int u = u_lo; u < u_hi; ++u) {
    const typename Io<T>::raw r = nx;
    if (u + 1 < u_hi) nx = fetch(u + 1);
    const int t = u / np, h = (p_lo + u - t * np) * a.hp + sub;
    const bool is_q = h < a.hq, is_v = APPEND && h >= a.hq + a.hk, is_k = !is_q && !is_v;
    if (t != t_cur) {
      t_cur = t;
      read8(L.c + t * a.d + (in_row ? e0 : 0), c);
      read8(L.s + t * a.d + (in_row ? e0 : 0), s);
    }
    if (first || __ballot(is_k != k_cur)) {
      first = false;
      k_cur = is_k;
      read8(&L.w[is_k][0][in_row ? e0 : 0], w);
      read8(&L.w[is_k][1][in_row ? e0 : 0], b);
    }
    float x[8], y[8];
    Io<T>::unpack(r, x);
    if (!in_row) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = 0.f;
    }
    float n[8];
    if (a.norm != HMA_NORM_NONE) {
      float mean, rstd;
      row_stats(a, x, in_row, inv_d, mean, rstd);
#pragma unroll
      for (int e = 0; e < 8; ++e) n[e] = __builtin_fmaf((x[e] - mean) * rstd, w[e], b[e]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) n[e] = x[e];
    }
    rotate(a, L.xch[wave], lane, e0, n, c, s, 1.f, y);
    if (!in_row || h >= heads) continue;
    const int64_t tok = tok0 + t;
    if (!APPEND) {
      if (is_q)
        Io<T>::store(g.q_out, (tok * a.hq + h) * a.d + e0, y);
      else
        Io<T>::store(g.k_out, (tok * a.hk + (h - a.hq)) * a.d + e0, y);
      continue;
    }
    const int off = L.off[t];
    if (is_q) {
      if (off == -2) {
        if (!g.zero_tail) continue;
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = 0.f;
      }
      Io<T>::store(g.q_out, (tok * a.hq + h) * a.d + e0, y);
      continue;
    }
    if (off < 0) continue;
    const int64_t page = L.page[t];
    const int hk = is_v ? h - a.hq - a.hk : h - a.hq;
    void* dst = is_v ? g.vc : g.kc;
    const int64_t at = is_v ? page * g.vc_page + hk * g.vc_head + off * g.vc_tok + e0 : page * g.kc_page + hk * g.kc_head + off * g.kc_tok + e0;
    if (is_v) {
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = x[e];
    }
    if (F8)
      store_e4m3(dst, at, y, 1.0f / (is_v ? g.v_scale : g.k_scale)[hk]);
    else
      Io<T>::store(dst, at, y);
  }
}

// ------------------------------------------------------------------------------------- backward
struct BwdArgs {
  Shape s;
  const void *q, *k, *gq, *gk;
  void *dq, *dk;
  float* part;  // [workgroup][q | k][weight | bias][d]
  int64_t q_tok, q_head, k_tok, k_head, gq_tok, gq_head, gk_tok, gk_head, tiles;
};

// dx of every row; the sums for the weights per workgroup (a lane adds its 8 columns over all its rows in registers, the workgroup adds
// its lanes in a fixed order), so no atomics and the same bits every time.
template <typename T>
__global__ __launch_bounds__(TPB) void rope_bwd_kernel(const BwdArgs g) {
  __shared__ Lds L;
  const Shape& a = g.s;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int dl = lane & (a.lg - 1), sub = lane / a.lg, e0 = dl * 8;
  const bool in_row = e0 < a.d;
  const int er = in_row ? e0 : 0, heads = a.hq + a.hk, np = a.passes;
  const float inv_d = 1.0f / (float)a.d;
  float dw[2][8], db[2][8];
#pragma unroll
  for (int e = 0; e < 8; ++e) dw[0][e] = dw[1][e] = db[0][e] = db[1][e] = 0.f;
  stage_weights<T>(a, L);

  for (int64_t tile = blockIdx.x; tile < g.tiles; tile += gridDim.x) {
    const int64_t tok0 = tile * a.tt;
    const int nt = (int)min((int64_t)a.tt, a.tokens - tok0);
    const int units = nt * np, per = (units + WAVES - 1) / WAVES, u_lo = wave * per, u_hi = min(units, u_lo + per);
    auto fetch = [&](int u, typename Io<T>::raw& x, typename Io<T>::raw& d) {
      const int t = u / np, h = min((u - t * np) * a.hp + sub, heads - 1);
      const int64_t tok = tok0 + t;
      const bool is_q = h < a.hq;
      x = is_q ? Io<T>::load(g.q, tok * g.q_tok + h * g.q_head + er) : Io<T>::load(g.k, tok * g.k_tok + (h - a.hq) * g.k_head + er);
      d = is_q ? Io<T>::load(g.gq, tok * g.gq_tok + h * g.gq_head + er) : Io<T>::load(g.gk, tok * g.gk_tok + (h - a.hq) * g.gk_head + er);
    };
    typename Io<T>::raw nx, nd;
    if (u_lo < u_hi) fetch(u_lo, nx, nd);
    __syncthreads();  // the last tile's readers of the table are done
    stage_angles(a, L, tok0, nt, false);
    __syncthreads();
    int t_cur = -1;
    bool first = true, k_cur = false;
    float c[8], s[8], w[8];
    for (int u = u_lo; u < u_hi; ++u) {
      const typename Io<T>::raw rx = nx, rd = nd;
      if (u + 1 < u_hi) fetch(u + 1, nx, nd);
      const int t = u / np, h = (u - t * np) * a.hp + sub;
      const bool is_k = h >= a.hq, live = in_row && h < heads;
      if (t != t_cur) {
        t_cur = t;
        read8(L.c + t * a.d + er, c);
        read8(L.s + t * a.d + er, s);
      }
      if (first || __ballot(is_k != k_cur)) {
        first = false;
        k_cur = is_k;
        read8(&L.w[is_k][0][er], w);
      }
      float x[8], d[8], y[8];
      Io<T>::unpack(rx, x);
      Io<T>::unpack(rd, d);
      if (!live) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = 0.f, d[e] = 0.f;
      }
      rotate(a, L.xch[wave], lane, e0, d, c, s, -1.f, y);
      if (a.norm != HMA_NORM_NONE) {
        float mean, rstd;
        row_stats(a, x, in_row, inv_d, mean, rstd);
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          x[e] = (x[e] - mean) * rstd;
          const float gu = y[e] * x[e];
          dw[0][e] += is_k ? 0.f : gu;
          dw[1][e] += is_k ? gu : 0.f;
          db[0][e] += is_k ? 0.f : y[e];
          db[1][e] += is_k ? y[e] : 0.f;
          y[e] *= w[e];
          s1 += y[e];
          s2 = __builtin_fmaf(y[e], x[e], s2);
        }
        if (!in_row) s1 = s2 = 0.f;
        s1 = a.norm == HMA_NORM_LAYER ? row_sum(s1, a.lg) * inv_d : 0.f;
        s2 = row_sum(s2, a.lg) * inv_d;
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = rstd * (y[e] - s1 - x[e] * s2);
      }
      if (!live) continue;
      const int64_t tok = tok0 + t;
      if (!is_k)
        Io<T>::store(g.dq, (tok * a.hq + h) * a.d + e0, y);
      else
        Io<T>::store(g.dk, (tok * a.hk + (h - a.hq)) * a.d + e0, y);
    }
  }
  if (!g.part) return;
  // lanes of the same columns: sub groups first (by shuffles), then the waves through LDS
  for (int kind = 0; kind < 2; ++kind)
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float v = kind ? (which ? db[1][e] : dw[1][e]) : (which ? db[0][e] : dw[0][e]);
        for (int o = a.lg; o < 64; o <<= 1) v += __shfl_xor(v, o, 64);
        if (sub == 0) L.xch[wave][e0 + e] = v;  // e0 + 7 < 256
      }
      __syncthreads();
      for (int e = threadIdx.x; e < a.d; e += TPB) {
        float v = 0.f;
#pragma unroll
        for (int k = 0; k < WAVES; ++k) v += L.xch[k][e];
        g.part[(((int64_t)blockIdx.x * 2 + kind) * 2 + which) * a.d + e] = v;
      }
    }
}

// out[i] = sum over the workgroups' partial sums, i over [q | k][weight | bias][d]: 16 threads a value, in a fixed order
__global__ __launch_bounds__(TPB) void rope_wsum_kernel(const float* part, int n, int width, void* qw, void* qb, void* kw, void* kb, int d, int w_f32, int bf16) {
  __shared__ float sum[16][17];
  const int col = threadIdx.x & 15, row = threadIdx.x >> 4, i = blockIdx.x * 16 + col;
  float v = 0.f;
  if (i < width)
    for (int k = row; k < n; k += 16) v += part[(int64_t)k * width + i];
  sum[row][col] = v;
  __syncthreads();
  if (row || i >= width) return;
  v = 0.f;
#pragma unroll
  for (int k = 0; k < 16; ++k) v += sum[k][col];
  const int which = i / d, e = i - which * d;
  void* out = which == 0 ? qw : which == 1 ? qb : which == 2 ? kw : kb;
  if (!out) return;
  if (w_f32)
    ((float*)out)[e] = v;
  else if (bf16)
    Io<Bf16>::put(out, e, v);
  else
    Io<_Float16>::put(out, e, v);
}

int pow2_up(int v) {
  int p = 1;
  while (p < v) p <<= 1;
  return p;
}
bool aligned(const void* p, int64_t a, int64_t b, int size) {
  return p && ((uintptr_t)p & 15) == 0 && (a * size) % 16 == 0 && (b * size) % 16 == 0 && a >= 0 && b >= 0;
}

// Checks and fills what the kernels share; 0 or HMA_EINVAL
int fill_shape(Shape& s, const hma_rope_t& r, int32_t hq, int32_t hk, int64_t tokens, int extra_heads, bool needs_pos) {
  if (r.d < 8 || r.d > 256 || (r.d & 7) || r.rot < 0 || r.rot > r.d || (r.rot & 1)) return HMA_EINVAL;
  if (hq < 0 || hk < 1 || hq > 4096 || hk > 4096 || tokens < 0 || r.norm < 0 || r.norm > 2 || r.dtype < 0 || r.dtype > 2) return HMA_EINVAL;
  if (r.rot > 0 && (!r.freqs || (needs_pos && tokens > 0 && !r.positions))) return HMA_EINVAL;
  if (r.n_axes < 1 || (r.positions && r.pos_stride < tokens && r.n_axes > 1)) return HMA_EINVAL;
  if (r.n_axes > 1 && (!r.axes || (tokens > 0 && !r.positions))) return HMA_EINVAL;
  if (r.norm == HMA_NORM_NONE && (r.q_w || r.q_b || r.k_w || r.k_b)) return HMA_EINVAL;
  if (r.dtype == HMA_F32 && !r.w_f32 && (r.q_w || r.q_b || r.k_w || r.k_b)) return HMA_EINVAL;
  s.freqs = r.freqs;
  s.axes = r.axes;
  s.positions = r.positions;
  s.w[0][0] = r.q_w; s.w[0][1] = r.q_b; s.w[1][0] = r.k_w; s.w[1][1] = r.k_b;
  s.tokens = tokens;
  s.pos_stride = r.pos_stride;
  s.hq = hq; s.hk = hk; s.d = r.d; s.rot = r.rot; s.inter = r.interleaved; s.norm = r.norm; s.w_f32 = r.w_f32; s.pos64 = r.pos_64; s.n_axes = r.n_axes;
  s.lg = pow2_up(r.d / 8);
  s.hp = 64 / s.lg;
  s.passes = (hq + hk + extra_heads + s.hp - 1) / s.hp;
  s.eps = r.eps;
  s.amp = r.amplitude;
  // tokens of a tile: as many as the table holds (one angle per thread), fewer where the chip would not be filled; then the heads of a
  // token over several workgroups, a unit per wave.  1024 workgroups = four on each compute unit.
  s.tt = TABLE / r.d;
  if (s.tt > MAX_TT) s.tt = MAX_TT;
  while (s.tt > 1 && (tokens + s.tt - 1) / s.tt < 1024) s.tt >>= 1;
  s.py = 1;
  const int most = (s.passes + WAVES - 1) / WAVES;
  while (s.py < most && (tokens + s.tt - 1) / s.tt * s.py < 1024) s.py <<= 1;
  if (s.py > most) s.py = most;
  return 0;
}

}  // namespace

extern "C" int hma_qk_rope_fwd(void* stream, const hma_qk_rope_t* p) {
  if (!p) return HMA_EINVAL;
  FwdArgs g = {};
  const int rc = fill_shape(g.s, p->r, p->hq, p->hk, p->tokens, 0, true);
  if (rc) return rc;
  if (p->tokens == 0) return 0;
  const int size = p->r.dtype == HMA_F32 ? 4 : 2;
  if (p->hq < 1 || !aligned(p->q, p->q_tok, p->q_head, size) || !aligned(p->k, p->k_tok, p->k_head, size) || !aligned(p->q_out, 0, 0, size) ||
      !aligned(p->k_out, 0, 0, size))
    return HMA_EINVAL;
  g.q = p->q; g.k = p->k; g.q_out = p->q_out; g.k_out = p->k_out;
  g.q_tok = p->q_tok; g.q_head = p->q_head; g.k_tok = p->k_tok; g.k_head = p->k_head;
  const int64_t tiles = (p->tokens + g.s.tt - 1) / g.s.tt;
  if (tiles > 0x7fffffff) return HMA_EINVAL;
  const dim3 grid((unsigned)tiles, (unsigned)g.s.py);
  if (p->r.dtype == HMA_BF16)
    hipLaunchKernelGGL((rope_fwd_kernel<Bf16, false, false>), grid, dim3(TPB), 0, (hipStream_t)stream, g);
  else if (p->r.dtype == HMA_F16)
    hipLaunchKernelGGL((rope_fwd_kernel<_Float16, false, false>), grid, dim3(TPB), 0, (hipStream_t)stream, g);
  else
    hipLaunchKernelGGL((rope_fwd_kernel<float, false, false>), grid, dim3(TPB), 0, (hipStream_t)stream, g);
  HMA_CHECK_LAUNCH();
  return 0;
}

extern "C" int hma_qk_rope_bwd(void* stream, const hma_qk_rope_t* p) {
  if (!p) return HMA_EINVAL;
  BwdArgs g = {};
  const int rc = fill_shape(g.s, p->r, p->hq, p->hk, p->tokens, 0, true);
  if (rc) return rc;
  const int size = p->r.dtype == HMA_F32 ? 4 : 2;
  const bool sums = p->dq_w || p->dq_b || p->dk_w || p->dk_b;
  if (p->hq < 1 || (sums && (!p->ws || p->ws_floats < (int64_t)HMA_QK_ROPE_WS_GROUPS * 4 * p->r.d || p->r.norm == HMA_NORM_NONE))) return HMA_EINVAL;
  if (p->tokens > 0 && (!aligned(p->q, p->q_tok, p->q_head, size) || !aligned(p->k, p->k_tok, p->k_head, size) ||
                        !aligned(p->dy_q, p->dyq_tok, p->dyq_head, size) || !aligned(p->dy_k, p->dyk_tok, p->dyk_head, size) ||
                        !aligned(p->dq, 0, 0, size) || !aligned(p->dk, 0, 0, size)))
    return HMA_EINVAL;
  g.q = p->q; g.k = p->k; g.gq = p->dy_q; g.gk = p->dy_k; g.dq = p->dq; g.dk = p->dk;
  g.part = sums ? p->ws : nullptr;
  g.q_tok = p->q_tok; g.q_head = p->q_head; g.k_tok = p->k_tok; g.k_head = p->k_head;
  g.gq_tok = p->dyq_tok; g.gq_head = p->dyq_head; g.gk_tok = p->dyk_tok; g.gk_head = p->dyk_head;
  g.tiles = (p->tokens + g.s.tt - 1) / g.s.tt;
  // no tokens: no workgroup, and the sums over nothing are zero
  const unsigned groups = (unsigned)(g.tiles < HMA_QK_ROPE_WS_GROUPS ? g.tiles : HMA_QK_ROPE_WS_GROUPS);
  if (groups) {
    if (p->r.dtype == HMA_BF16)
      hipLaunchKernelGGL((rope_bwd_kernel<Bf16>), dim3(groups), dim3(TPB), 0, (hipStream_t)stream, g);
    else if (p->r.dtype == HMA_F16)
      hipLaunchKernelGGL((rope_bwd_kernel<_Float16>), dim3(groups), dim3(TPB), 0, (hipStream_t)stream, g);
    else
      hipLaunchKernelGGL((rope_bwd_kernel<float>), dim3(groups), dim3(TPB), 0, (hipStream_t)stream, g);
    HMA_CHECK_LAUNCH();
  }
  if (sums) {
    const int width = 4 * p->r.d;
    hipLaunchKernelGGL(rope_wsum_kernel, dim3((width + 15) / 16), dim3(TPB), 0, (hipStream_t)stream, p->ws, (int)groups, width, p->dq_w, p->dq_b,
                       p->dk_w, p->dk_b, p->r.d, p->r.w_f32, p->r.dtype == HMA_BF16);
    HMA_CHECK_LAUNCH();
  }
  return 0;
}

extern "C" int hma_kv_append(void* stream, const hma_kv_append_t* p) {
  if (!p) return HMA_EINVAL;
  FwdArgs g = {};
  const int rc = fill_shape(g.s, p->r, p->q ? p->hq : 0, p->hk, p->tokens, p->hk, false);
  if (rc) return rc;
  if (p->r.dtype == HMA_F32 || p->seqs < 0 || p->page < 1 || p->pages < 0 || p->table_w < 0) return HMA_EINVAL;
  if (p->tokens == 0) return 0;
  if (p->tokens > 0x7fffffff || !p->cu || (p->seqs > 0 && (!p->lens || (p->table_w > 0 && !p->table)))) return HMA_EINVAL;
  const bool f8 = p->cache_e4m3 != 0;
  if (f8 && (!p->k_scale || !p->v_scale)) return HMA_EINVAL;
  if (!aligned(p->k, p->k_tok, p->k_head, 2) || !aligned(p->v, p->v_tok, p->v_head, 2)) return HMA_EINVAL;
  if (p->q && (p->hq < 1 || !aligned(p->q, p->q_tok, p->q_head, 2) || !aligned(p->q_out, 0, 0, 2))) return HMA_EINVAL;
  if (p->pages > 0) {
    const int m = f8 ? 7 : 15, e = f8 ? 1 : 2;  // a lane writes 8 values
    const int64_t st[6] = {p->kc_page, p->kc_head, p->kc_tok, p->vc_page, p->vc_head, p->vc_tok};
    for (int i = 0; i < 6; ++i)
      if (st[i] < 0 || ((st[i] * e) & m)) return HMA_EINVAL;
    if (!p->kc || !p->vc || ((uintptr_t)p->kc & m) || ((uintptr_t)p->vc & m)) return HMA_EINVAL;
  }
  g.q = p->q; g.k = p->k; g.v = p->v; g.q_out = p->q_out; g.kc = p->kc; g.vc = p->vc;
  g.q_tok = p->q_tok; g.q_head = p->q_head; g.k_tok = p->k_tok; g.k_head = p->k_head; g.v_tok = p->v_tok; g.v_head = p->v_head;
  g.table = p->table; g.cu = p->cu; g.lens = p->lens; g.k_scale = p->k_scale; g.v_scale = p->v_scale;
  g.table_stride = p->table_stride;
  g.kc_page = p->kc_page; g.kc_head = p->kc_head; g.kc_tok = p->kc_tok; g.vc_page = p->vc_page; g.vc_head = p->vc_head; g.vc_tok = p->vc_tok;
  g.seqs = p->seqs; g.table_w = p->table_w; g.pages = p->pages; g.page = p->page; g.zero_tail = p->zero_tail;
  const dim3 grid((unsigned)((p->tokens + g.s.tt - 1) / g.s.tt), (unsigned)g.s.py);
  if (p->r.dtype == HMA_BF16) {
    if (f8)
      hipLaunchKernelGGL((rope_fwd_kernel<Bf16, true, true>), grid, dim3(TPB), 0, (hipStream_t)stream, g);
    else
      hipLaunchKernelGGL((rope_fwd_kernel<Bf16, true, false>), grid, dim3(TPB), 0, (hipStream_t)stream, g);
  } else {
    if (f8)
      hipLaunchKernelGGL((rope_fwd_kernel<_Float16, true, true>), grid, dim3(TPB), 0, (hipStream_t)stream, g);
    else
      hipLaunchKernelGGL((rope_fwd_kernel<_Float16, true, false>), grid, dim3(TPB), 0, (hipStream_t)stream, g);
  }
  HMA_CHECK_LAUNCH();
  return 0;
}
