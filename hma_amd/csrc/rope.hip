// Per-head norms of queries and keys with the rotary position rotation in the same pass, forward and backward, and the same pass
// with its keys (and the values) going into the pages of a cache.
//
// One row = one head of one token, D values:  y = R(pos) (u w + b),
//   u = x  |  x / sqrt(mean x^2 + eps)  |  (x - mean x) / sqrt(var x + eps),
// R rotates the first `rot` values in pairs -- (2 i, 2 i + 1) or (i, i + rot / 2) -- by the angle pos f_i and multiplies them by an
// amplitude.  Written per value e with its pair's other value p(e):  R x[e] = x[e] C[e] + x[p(e)] S[e], S carrying the sign; the values
// behind `rot` have C = 1, S = 0 and a zero as partner (an infinity behind `rot` stays one), so no lane branches.  R^T is the same with -S.
//
// Bound by the HBM bytes of the rows.  A lane holds 8 consecutive values of a row (16-byte loads and stores of 16-bit types), D / 8
// lanes (rounded up to a power of two) hold a row, 64 lanes several heads: a unit, one load a lane.  What would bound it instead is the
// angles: a sine and a cosine cost more than everything else that happens to a value, and every head of a token needs the same ones.  So
// a wave takes the tokens whose pairs are about 64 (four at D = 32, one at D = 128), computes one angle per lane into its own C / S table
// in LDS and walks the tokens' heads with it.  Waves share nothing but the norms' weights, so there is one barrier in a launch; a wave
// fetches its next units (and the next tokens' positions) before it works on the current ones.
// Angles: position times frequency in 64 bits, reduced to a fraction of a turn there, rounded to 32 bits after that -- a 32-bit product
// at position 10^6 is off by 0.03 rad.
// Reductions: everything in 32 bits; each output is rounded once.
// Measured (bf16): forward of 81920 tokens x 16 heads of 32, three axes, layer norm: 40 us = 4.2 TB/s of 168 MB; of 8191 x 40 heads of 128,
// RMS norm: 34 us = 4.9 TB/s.  fp32: 80 us = 4.2 TB/s and 71 us = 4.7 TB/s.
// 7 tokens x 40 heads of 128: 4.9 us, a launch and one trip to memory.  The cache form: 8 frames of 320 tokens x 32
// rows of 32: 12 us; 7.9 thousand tokens x 16 rows of 128 into e4m3: 21 us = 2.3 TB/s (what a wave does once, and four dependent loads in front
// of its first store -- sequence, length, page, row -- for two tokens); 128 thousand such tokens: 252 us = 3.1 TB/s, into bf16 224 us =
// 4.7 TB/s; one token of 64 sequences x 48 rows of 128: 7.4 us.
#include "hma_common.h"
#include "../../include/hma_hip.h"

using namespace hma;

namespace {

constexpr int TPB = 256;    // threads of a workgroup
constexpr int WAVES = TPB / 64;
constexpr int MAX_WT = 16;  // tokens of a wave's batch

struct Bf16 { uint16_t v; };
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));

template <typename T> struct Io;
template <> struct Io<Bf16> {
  typedef uint4 raw;
  static constexpr int SIZE = 2;
  static __device__ __forceinline__ raw load(const uint8_t* p) { return *reinterpret_cast<const uint4*>(p); }
  static __device__ __forceinline__ void unpack(const raw& r, float* f) { unpack8(r, f); }
  static __device__ __forceinline__ void store(uint8_t* p, const float* f) { *reinterpret_cast<uint4*>(p) = pack8(f); }
  static __device__ __forceinline__ float one(const void* p, int64_t i) { return from_bf16(((const uint16_t*)p)[i]); }
  static __device__ __forceinline__ void put(void* p, int64_t i, float v) { ((uint16_t*)p)[i] = to_bf16(v); }
};
template <> struct Io<_Float16> {
  typedef uint4 raw;
  static constexpr int SIZE = 2;
  static __device__ __forceinline__ raw load(const uint8_t* p) { return *reinterpret_cast<const uint4*>(p); }
  static __device__ __forceinline__ void unpack(const raw& r, float* f) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const half2_t h = __builtin_bit_cast(half2_t, w[i]);
      f[2 * i] = (float)h[0];
      f[2 * i + 1] = (float)h[1];
    }
  }
  static __device__ __forceinline__ void store(uint8_t* p, const float* f) {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const half2_t h = {(_Float16)f[2 * j], (_Float16)f[2 * j + 1]};
      w[j] = __builtin_bit_cast(uint32_t, h);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
  static __device__ __forceinline__ float one(const void* p, int64_t i) { return (float)((const _Float16*)p)[i]; }
  static __device__ __forceinline__ void put(void* p, int64_t i, float v) { ((_Float16*)p)[i] = (_Float16)v; }
};
template <> struct Io<float> {
  struct raw { float4 a, b; };
  static constexpr int SIZE = 4;
  static __device__ __forceinline__ raw load(const uint8_t* p) {
    const float4* q = reinterpret_cast<const float4*>(p);
    return raw{q[0], q[1]};
  }
  static __device__ __forceinline__ void unpack(const raw& r, float* f) {
    f[0] = r.a.x; f[1] = r.a.y; f[2] = r.a.z; f[3] = r.a.w;
    f[4] = r.b.x; f[5] = r.b.y; f[6] = r.b.z; f[7] = r.b.w;
  }
  static __device__ __forceinline__ void store(uint8_t* p, const float* f) {
    float4* q = reinterpret_cast<float4*>(p);
    q[0] = make_float4(f[0], f[1], f[2], f[3]);
    q[1] = make_float4(f[4], f[5], f[6], f[7]);
  }
  static __device__ __forceinline__ float one(const void* p, int64_t i) { return ((const float*)p)[i]; }
  static __device__ __forceinline__ void put(void* p, int64_t i, float v) { ((float*)p)[i] = v; }
};

// 8 values -> 8 e4m3 bytes of x / scale: nearest even, clamped to the type's largest value (a NaN stays one).  The product with the hardware's
// reciprocal (one step off) alone lands on the wrong side of a border between two e4m3 values where the quotient lies on it or next to it
// (an odd multiple of a power of two for a scale: one value in twenty thousand); its remainder q scale - x, exact in one fma, puts that
// right.  128 thousand tokens x 16 rows: 250 -> 252 us, with the compiler's division 311.  x is clamped, not q: an infinity has no remainder.
__device__ __forceinline__ void store_e4m3(uint8_t* p, const float* f, float scale) {
  const float inv = __builtin_amdgcn_rcpf(scale), lim = fminf(448.f * scale, 3.4e38f);
  float q[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float x = __builtin_elementwise_maximum(__builtin_elementwise_minimum(f[e], lim), -lim);
    q[e] = x * inv;
    q[e] = __builtin_fmaf(-__builtin_fmaf(q[e], scale, -x), inv, q[e]);  // (in this order a zero keeps its sign)
  }
  uint2 w;
  int a = 0, b = 0;
  a = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], a, false);
  a = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], a, true);
  b = __builtin_amdgcn_cvt_pk_fp8_f32(q[4], q[5], b, false);
  b = __builtin_amdgcn_cvt_pk_fp8_f32(q[6], q[7], b, true);
  w.x = (uint32_t)a;
  w.y = (uint32_t)b;
  *reinterpret_cast<uint2*>(p) = w;
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

// What the kernels share of their arguments
struct Shape {
  const double* freqs;
  const int32_t* axes;
  const void* positions;
  const void* w[2][2];  // [q | k][weight | bias]
  int64_t tokens, pos_stride, batches;
  int32_t hq, hk, d, rot, inter, norm, w_f32, pos64, n_axes, lg, hp, wt, passes, py;
  float eps, amp;
};

struct WaveLds {
  float c[256], s[256];  // [token of the batch][d]
  float xch[64 * 8];
  int32_t page[MAX_WT], off[MAX_WT];
};
struct Lds {
  float w[2][2][256];
  WaveLds wave[WAVES];
};
struct BwdLds : Lds {
  float acc[WAVES][2][2][64 * 8];  // [wave][q | k][weight | bias]: each lane's 8 columns, parked while the wave works on the other tensor
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

// The angles of a wave's batch: lane l computes those of pair numbers l and l + 64 of its wt * d / 2 (two only where d > 128)
struct Angles {
  double f[2];      // turns per position
  int32_t t[2], e[2][2];  // token of the batch (-1: none), where the pair's values sit in the table
  const uint8_t* pos[2];
  bool turn[2];

  __device__ __forceinline__ void begin(const Shape& a, int lane) {
    const int half = a.rot >> 1, hd = a.d >> 1;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int i = lane + 64 * k;
      t[k] = i < a.wt * hd ? i / hd : -1;
      const int p = i % hd;
      turn[k] = t[k] >= 0 && p < half;
      f[k] = turn[k] ? a.freqs[p] * 0.15915494309189533577 : 0.0;
      const int ax = turn[k] && a.axes ? min(max(a.axes[p], 0), a.n_axes - 1) : 0;
      pos[k] = (const uint8_t*)a.positions + ax * a.pos_stride * (a.pos64 ? 8 : 4);
      const bool inter = a.inter || !turn[k];
      e[k][0] = max(t[k], 0) * a.d + (inter ? 2 * p : p);
      e[k][1] = max(t[k], 0) * a.d + (inter ? 2 * p + 1 : p + half);
    }
  }
  __device__ __forceinline__ void position(const Shape& a, int64_t tok0, double* at) const {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (k == 1 && a.wt * a.d <= 128) break;
      const int64_t tok = tok0 + t[k];
      at[k] = 0.0;
      if (turn[k] && tok < a.tokens) at[k] = a.pos64 ? (double)((const int64_t*)pos[k])[tok] : (double)((const int32_t*)pos[k])[tok];
    }
  }
  __device__ __forceinline__ void stage(const Shape& a, WaveLds& L, const double* at) const {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (k == 1 && a.wt * a.d <= 128) break;
      if (t[k] < 0) continue;
      float c = 1.f, s = 0.f;
      if (turn[k]) {
        double x = at[k] * f[k];
        x -= rint(x);
        sincospif((float)(2.0 * x), &s, &c);
        c *= a.amp;
        s *= a.amp;
      }
      L.c[e[k][0]] = c; L.c[e[k][1]] = c;
      L.s[e[k][0]] = -s; L.s[e[k][1]] = s;
    }
  }
};

__device__ __forceinline__ void read8(const float* p, float* f) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
  f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
}

// y = x C + x[partner] S (sgn = -1: the transposed rotation) for the 8 values e0 .. e0 + 7 of each lane's row
template <bool INTER>
__device__ __forceinline__ void rotate(const Shape& a, float* xch, int lane, int e0, const float* x, const float* c, const float* s, float sgn, float* y) {
  float p[8];
  if (INTER) {
#pragma unroll
    for (int e = 0; e < 8; ++e) p[e] = e0 + e < a.rot ? x[e ^ 1] : 0.f;
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
        const bool in = e < a.rot;
        p[q] = in ? v.x : 0.f; p[q + 1] = in ? v.y : 0.f; p[q + 2] = in ? v.z : 0.f; p[q + 3] = in ? v.w : 0.f;
      }
    } else {
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const int e = e0 + q, at = e < half ? e + half : e < a.rot ? e - half : e;
        p[q] = e < a.rot ? row[at] : 0.f;
      }
    }
    wave_lds_order();  // the next rows are written behind these reads
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) y[e] = __builtin_fmaf(p[e] * sgn, s[e], x[e] * c[e]);
}

// mean (layer) and 1 / deviation of a row; what lanes behind the row hold does not count
template <int NORM>
__device__ __forceinline__ void row_stats(const Shape& a, const float* x, bool in_row, float inv_d, float& mean, float& rstd) {
  mean = 0.f;
  if (NORM == HMA_NORM_LAYER) {
    float t = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) t += x[e];
    mean = row_sum(in_row ? t : 0.f, a.lg) * inv_d;
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

// Where the batch's rows go: lane t finds the sequence and place of row tok0 + t.  `sample`: cu at every st-th sequence (lane + 1) * st.
struct Target {
  int32_t page, off;  // off -1: belongs to a sequence, has no place in the cache; -2: behind the last sequence
  int64_t place;
};
__device__ __forceinline__ Target find_target(const FwdArgs& g, int64_t tok0, int nt, int lane, int st, int sample) {
  int mine = 0;
  for (int t = 0; t < nt; ++t) {  // how many of cu[1 .. seqs] are <= the row: 64 candidates a step
    const int64_t row = tok0 + t;
    const int c = __popcll(__ballot((lane + 1) * st <= g.seqs && sample <= row));
    int lo = c * st, n = min(st, g.seqs - lo);
    if (st == 1) n = 0;
    while (n > 0) {
      const int s2 = (n + 63) >> 6, i = (lane + 1) * s2;
      const int k = __popcll(__ballot(i <= n && g.cu[lo + min(i, n)] <= row));
      lo += k * s2;
      n = s2 == 1 ? 0 : min(s2, n - k * s2);
    }
    if (lane == t) mine = lo;
  }
  Target r = {-1, -2, 0};
  if (lane < nt && mine < g.seqs) {
    const int64_t row = tok0 + lane;
    const int c0 = g.cu[mine], c1 = g.cu[mine + 1], len = g.lens[mine];
    if (row >= c0) {
      r.off = -1;
      r.place = (int64_t)len - c1 + row;
      const int64_t pi = r.place >= 0 ? r.place / g.page : g.table_w;
      if (pi < g.table_w) {
        r.page = g.table[mine * g.table_stride + pi];
        if (r.page >= 0 && r.page < g.pages) r.off = (int32_t)(r.place - pi * g.page);
      }
    }
  }
  return r;
}

// Addresses of a unit: the token and the first head of the group are the wave's, so all but a lane's head of the group and its columns is
// scalar arithmetic.  `at` = heads of this tensor in front of the group (negative: the group begins before the tensor's first).
struct Part {
  const uint8_t* p;
  int64_t tok, head, lane;  // bytes per token, per head, of this lane
  __device__ __forceinline__ void begin(const void* base, int64_t tok_, int64_t head_, int size, int sub, int e) {
    p = (const uint8_t*)base;
    tok = tok_ * size;
    head = head_ * size;
    lane = sub * head + e * size;
  }
  __device__ __forceinline__ const uint8_t* of(int64_t t, int at) const { return p + t * tok + at * head; }
};

template <typename T, bool APPEND, bool F8, int NORM, bool INTER>
__global__ __launch_bounds__(TPB, (APPEND && NORM != HMA_NORM_NONE) || Io<T>::SIZE == 4 ? 3 : 4) void rope_fwd_kernel(const FwdArgs g) {
  constexpr int U = 2, SZ = Io<T>::SIZE, CS = F8 ? 1 : SZ;  // units in flight, bytes of a value and of a cached one
  __shared__ Lds L;
  const Shape& a = g.s;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  WaveLds& W = L.wave[wave];
  // this wave: a share (1 / py) of the heads of batches gw / py, + the grid's stride, ...
  const int gw = blockIdx.x * WAVES + wave, step = gridDim.x * WAVES / a.py;
  const int share = gw % a.py, pp = (a.passes + a.py - 1) / a.py, p_lo = share * pp, np = min(pp, a.passes - p_lo);
  int64_t batch = gw / a.py;
  const int dl = lane & (a.lg - 1), sub = lane / a.lg, e0 = dl * 8;
  const bool in_row = e0 < a.d;
  const int er = in_row ? e0 : 0, hqk = a.hq + a.hk, heads = hqk + (APPEND ? a.hk : 0);
  const float inv_d = 1.0f / (float)a.d;
  const bool places = APPEND && !a.positions;
  const int64_t k_lane = APPEND ? (sub * g.kc_head + e0) * CS : 0, v_lane = APPEND ? (sub * g.vc_head + e0) * CS : 0;  // this lane's part of a cache address
  Part pq, pk, pv;
  pq.begin(g.q, g.q_tok, g.q_head, SZ, sub, er);
  pk.begin(g.k, g.k_tok, g.k_head, SZ, sub, er);
  if (APPEND) pv.begin(g.v, g.v_tok, g.v_head, SZ, sub, er);

  // the next U units from (token t of batch bt, group p) on, with their heads' scales; a unit behind the batch's last is loaded as that one
  auto fetch = [&](int64_t bt, int t, int p, typename Io<T>::raw* r, float* scale) {
    const int64_t tok0 = bt * a.wt;
    const int nt = (int)min((int64_t)a.wt, a.tokens - tok0);
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int64_t tok = tok0 + t;
      const int h0 = (p_lo + p) * a.hp, h = h0 + sub;
      const uint8_t* at = pk.of(tok, h0 - a.hq) + pk.lane;
      if (h < a.hq) at = pq.of(tok, h0) + pq.lane;
      if (APPEND && h >= hqk) at = pv.of(tok, h0 - hqk) + pv.lane;
      if (h >= heads) at = pk.of(tok, 0) + er * SZ;
      r[i] = Io<T>::load(at);
      if (F8) scale[i] = h >= hqk && h < heads ? g.v_scale[h - hqk] : g.k_scale[h >= a.hq && h < hqk ? h - a.hq : 0];
      if (++p == np) {
        if (t + 1 < nt) p = 0, ++t; else p = np - 1;
      }
    }
  };
  const bool mine = np > 0 && batch < a.batches;
  typename Io<T>::raw nx[U];
  float ns[U];
  double pos[2] = {0.0, 0.0};
  Angles an;
  const int st = APPEND ? max((g.seqs + 63) >> 6, 1) : 1;
  int sample = 0x7fffffff;
  if (mine) {
    fetch(batch, 0, 0, nx, ns);
    if (APPEND && (lane + 1) * st <= g.seqs) sample = g.cu[(lane + 1) * st];
    an.begin(a, lane);
    if (!places) an.position(a, batch * a.wt, pos);
  }
  if (NORM != HMA_NORM_NONE) {
    stage_weights<T>(a, L);
    __syncthreads();
  }
  if (!mine) return;

  int k_cur = -1;
  float c[8], s[8], w[8], b[8];
  while (batch < a.batches) {
    const int64_t tok0 = batch * a.wt, nb = batch + step;
    const int nt = (int)min((int64_t)a.wt, a.tokens - tok0);
    if (APPEND) {
      const Target tg = find_target(g, tok0, nt, lane, st, sample);
      if (lane < nt) W.page[lane] = tg.page, W.off[lane] = tg.off;
      if (places) {
        const double pl = (double)tg.place;
        pos[0] = __shfl(pl, max(an.t[0], 0), 64);
        pos[1] = __shfl(pl, max(an.t[1], 0), 64);
      }
    }
    an.stage(a, W, pos);
    wave_lds_order();
    if (!places && nb < a.batches) an.position(a, nb * a.wt, pos);
    int t_cur = -1;
    for (int t = 0, p = 0; t < nt;) {
      typename Io<T>::raw r[U];
      float scale[U];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        r[i] = nx[i];
        if (F8) scale[i] = ns[i];
      }
      {
        int t2 = t, p2 = p + U;
        while (p2 >= np && t2 < nt) p2 -= np, ++t2;
        if (t2 < nt)
          fetch(batch, t2, p2, nx, ns);
        else if (nb < a.batches)
          fetch(nb, 0, 0, nx, ns);
      }
#pragma unroll
      for (int i = 0; i < U; ++i) {
        if (t >= nt) break;
        const int64_t tok = tok0 + t;
        const int h0 = (p_lo + p) * a.hp, h = h0 + sub;
        const bool is_q = h < a.hq, is_v = APPEND && h >= hqk, live = in_row && h < heads;
        if (t != t_cur) {
          t_cur = t;
          read8(W.c + t * a.d + er, c);
          read8(W.s + t * a.d + er, s);
        }
        if (NORM != HMA_NORM_NONE) {  // the weights of this group's rows: q's, k's, or both (a lane's own)
          const int kind = h0 + a.hp <= a.hq ? 0 : h0 >= a.hq ? 1 : 2;
          if (kind != k_cur) {
            k_cur = kind;
            read8(&L.w[!is_q][0][er], w);
            read8(&L.w[!is_q][1][er], b);
          }
        }
        float x[8], y[8] = {}, n[8];
        Io<T>::unpack(r[i], x);
        if (!APPEND || h0 < hqk) {  // (a group of values alone has neither norm nor rotation)
          if (NORM != HMA_NORM_NONE) {
            float mean, rstd;
            row_stats<NORM>(a, x, in_row, inv_d, mean, rstd);
#pragma unroll
            for (int e = 0; e < 8; ++e) n[e] = __builtin_fmaf((x[e] - mean) * rstd, w[e], b[e]);
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) n[e] = x[e];
          }
          rotate<INTER>(a, W.xch, lane, e0, n, c, s, 1.f, y);
        }
        if (!APPEND) {
          uint8_t* dst = (uint8_t*)(is_q ? g.q_out : g.k_out) + (is_q ? (tok * a.hq + h0) * a.d : (tok * a.hk + h0 - a.hq) * a.d) * SZ + (sub * a.d + e0) * SZ;
          if (live) Io<T>::store(dst, y);
        } else {
          const int off = __builtin_amdgcn_readfirstlane(W.off[t]), page = __builtin_amdgcn_readfirstlane(W.page[t]);
          if (h0 + a.hp > hqk) {  // some of the group's rows are values
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = is_v ? x[e] : y[e];
          }
          if (off == -2) {  // (nothing but zeros is stored of it)
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = 0.f;
          }
          if (live && is_q && (off != -2 || g.zero_tail)) Io<T>::store((uint8_t*)g.q_out + (tok * a.hq + h0) * a.d * SZ + (sub * a.d + e0) * SZ, y);
          if (live && !is_q && off >= 0) {
            const int64_t ks = page * g.kc_page + off * g.kc_tok + (h0 - a.hq) * g.kc_head, vs = page * g.vc_page + off * g.vc_tok + (h0 - hqk) * g.vc_head;
            uint8_t* dst = is_v ? (uint8_t*)g.vc + vs * CS + v_lane : (uint8_t*)g.kc + ks * CS + k_lane;
            if (F8)
              store_e4m3(dst, y, scale[i]);
            else
              Io<T>::store(dst, y);
          }
        }
        if (++p == np) p = 0, ++t;
      }
    }
    batch = nb;
  }
}

// ------------------------------------------------------------------------------------- backward
struct BwdArgs {
  Shape s;
  const void *q, *k, *gq, *gk;
  void *dq, *dk;
  float* part;  // [workgroup][q | k][weight | bias][d]
  int64_t q_tok, q_head, k_tok, k_head, gq_tok, gq_head, gk_tok, gk_head;
};

// dx of every row; the sums for the weights per workgroup (a lane adds its 8 columns over all its rows in registers, the workgroup adds
// its lanes in a fixed order), so no atomics and the same bits every time.  The sums of the tensor that a wave does not work on wait in
// LDS: in registers they cost a wave of occupancy.  81920 tokens x 16 heads of 32, layer norm: 69 us = 3.7 TB/s of 252 MB; 8191 x 40 heads of
// 128, RMS norm: 60 us = 4.2 TB/s; the second launch adds 768 partial sums in 4 us.  fp32, both launches:
// 113 us = 4.5 TB/s and 107 us = 4.7 TB/s.
template <typename T, int NORM, bool INTER>
__global__ __launch_bounds__(TPB, Io<T>::SIZE == 2 ? 3 : 2) void rope_bwd_kernel(const BwdArgs g) {
  constexpr int U = 2, SZ = Io<T>::SIZE;
  __shared__ BwdLds L;
  const Shape& a = g.s;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  WaveLds& W = L.wave[wave];
  const int dl = lane & (a.lg - 1), sub = lane / a.lg, e0 = dl * 8;
  const bool in_row = e0 < a.d;
  const int er = in_row ? e0 : 0, heads = a.hq + a.hk, np = a.passes;
  const float inv_d = 1.0f / (float)a.d;
  float dw[8], db[8];  // this lane's columns of the tensor that its rows belong to now
  bool acc_k = false;
  if (NORM != HMA_NORM_NONE) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      dw[e] = db[e] = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) L.acc[wave][k >> 1][k & 1][lane * 8 + e] = 0.f;
    }
  }
  auto park = [&]() {
    float* pw = &L.acc[wave][acc_k][0][lane * 8];
    float* pb = &L.acc[wave][acc_k][1][lane * 8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      pw[e] += dw[e];
      dw[e] = 0.f;
      if (NORM == HMA_NORM_LAYER) pb[e] += db[e], db[e] = 0.f;
    }
  };
  int64_t batch = (int64_t)blockIdx.x * WAVES + wave;
  const int64_t step = (int64_t)gridDim.x * WAVES;
  Part pq, pk, gq, gk;
  pq.begin(g.q, g.q_tok, g.q_head, SZ, sub, er);
  pk.begin(g.k, g.k_tok, g.k_head, SZ, sub, er);
  gq.begin(g.gq, g.gq_tok, g.gq_head, SZ, sub, er);
  gk.begin(g.gk, g.gk_tok, g.gk_head, SZ, sub, er);

  auto fetch = [&](int64_t bt, int t, int p, typename Io<T>::raw* x, typename Io<T>::raw* d) {
    const int64_t tok0 = bt * a.wt;
    const int nt = (int)min((int64_t)a.wt, a.tokens - tok0);
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int64_t tok = tok0 + t;
      const int h0 = p * a.hp, h = h0 + sub;
      const bool q = h < a.hq, none = h >= heads;
      if (NORM != HMA_NORM_NONE) x[i] = Io<T>::load(none ? pk.of(tok, 0) + er * SZ : q ? pq.of(tok, h0) + pq.lane : pk.of(tok, h0 - a.hq) + pk.lane);
      d[i] = Io<T>::load(none ? gk.of(tok, 0) + er * SZ : q ? gq.of(tok, h0) + gq.lane : gk.of(tok, h0 - a.hq) + gk.lane);
      if (++p == np) {
        if (t + 1 < nt) p = 0, ++t; else p = np - 1;
      }
    }
  };
  typename Io<T>::raw nx[U], nd[U];
  double pos[2] = {0.0, 0.0};
  Angles an;
  if (batch < a.batches) {
    fetch(batch, 0, 0, nx, nd);
    an.begin(a, lane);
    an.position(a, batch * a.wt, pos);
  }
  if (NORM != HMA_NORM_NONE) {
    stage_weights<T>(a, L);
    __syncthreads();
  }
  int k_cur = -1;
  float c[8], s[8], w[8];
  while (batch < a.batches) {
    const int64_t tok0 = batch * a.wt, nb = batch + step;
    const int nt = (int)min((int64_t)a.wt, a.tokens - tok0);
    an.stage(a, W, pos);
    wave_lds_order();
    if (nb < a.batches) an.position(a, nb * a.wt, pos);
    int t_cur = -1;
    for (int t = 0, p = 0; t < nt;) {
      typename Io<T>::raw rx[U], rd[U];
#pragma unroll
      for (int i = 0; i < U; ++i) rx[i] = nx[i], rd[i] = nd[i];
      {
        int t2 = t, p2 = p + U;
        while (p2 >= np && t2 < nt) p2 -= np, ++t2;
        if (t2 < nt)
          fetch(batch, t2, p2, nx, nd);
        else if (nb < a.batches)
          fetch(nb, 0, 0, nx, nd);
      }
#pragma unroll
      for (int i = 0; i < U; ++i) {
        if (t >= nt) break;
        const int64_t tok = tok0 + t;
        const int h0 = p * a.hp, h = h0 + sub;
        const bool is_k = h >= a.hq, live = in_row && h < heads;
        const int kind = h0 + a.hp <= a.hq ? 0 : h0 >= a.hq ? 1 : 2;
        if (t != t_cur) {
          t_cur = t;
          read8(W.c + t * a.d + er, c);
          read8(W.s + t * a.d + er, s);
        }
        if (NORM != HMA_NORM_NONE && kind != k_cur) {
          if (k_cur >= 0) park();
          k_cur = kind;
          acc_k = is_k;
          read8(&L.w[is_k][0][er], w);
        }
        float d[8], y[8];
        Io<T>::unpack(rd[i], d);
        rotate<INTER>(a, W.xch, lane, e0, d, c, s, -1.f, y);
        if (NORM != HMA_NORM_NONE) {
          float x[8], mean, rstd;
          Io<T>::unpack(rx[i], x);
          row_stats<NORM>(a, x, in_row, inv_d, mean, rstd);
          float s1 = 0.f, s2 = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = (x[e] - mean) * rstd;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            dw[e] += live ? y[e] * x[e] : 0.f;
            if (NORM == HMA_NORM_LAYER) db[e] += live ? y[e] : 0.f;
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            y[e] *= w[e];
            s1 += y[e];
            s2 = __builtin_fmaf(y[e], x[e], s2);
          }
          s1 = NORM == HMA_NORM_LAYER ? row_sum(in_row ? s1 : 0.f, a.lg) * inv_d : 0.f;
          s2 = row_sum(in_row ? s2 : 0.f, a.lg) * inv_d;
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] = rstd * (y[e] - s1 - x[e] * s2);
        }
        uint8_t* dst = (uint8_t*)(is_k ? g.dk : g.dq) + (is_k ? (tok * a.hk + h0 - a.hq) * a.d : (tok * a.hq + h0) * a.d) * SZ + (sub * a.d + e0) * SZ;
        if (live) Io<T>::store(dst, y);
        if (++p == np) p = 0, ++t;
      }
    }
    batch = nb;
  }
  if (NORM == HMA_NORM_NONE || !g.part) return;
  park();
  __syncthreads();
  for (int i = threadIdx.x; i < 4 * a.d; i += TPB) {  // the lanes of the same columns, wave by wave
    const int which = i / a.d, e = i - which * a.d, at = (e >> 3) * 8 + (e & 7);
    float v = 0.f;
    for (int k = 0; k < WAVES; ++k)
      for (int j = 0; j < a.hp; ++j) v += L.acc[k][which >> 1][which & 1][j * a.lg * 8 + at];
    g.part[(int64_t)blockIdx.x * 4 * a.d + i] = v;
  }
}

// out[i] = sum over the n workgroups' partial sums, i over [q | k][weight | bias][d]: 64 threads a value, each adding every 64th (8 loads
// in flight), then in order
__global__ __launch_bounds__(1024) void rope_wsum_kernel(const float* part, int n, int width, void* qw, void* qb, void* kw, void* kb, int d, int w_f32, int bf16) {
  __shared__ float sum[64][17];
  const int col = threadIdx.x & 15, row = threadIdx.x >> 4, i = blockIdx.x * 16 + col;
  float v = 0.f;
  if (i < width)
    for (int k = row; k < n; k += 512) {
      float x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = k + 64 * j < n ? part[(int64_t)(k + 64 * j) * width + i] : 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) v += x[j];
    }
  sum[row][col] = v;
  __syncthreads();
  if (row || i >= width) return;
  v = 0.f;
#pragma unroll
  for (int k = 0; k < 64; ++k) v += sum[k][col];
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

// Workgroups of a forward launch: a wave per (batch, share of the heads), at most what is resident (4 a compute unit, 3 with the cache's
// addresses and a norm); a wave then walks several batches.  With a third more than resident the last quarter of a launch runs on a third of the
// chip: the backward of 81920 x 16 heads of 32 took 87 us instead of 68.
unsigned fwd_groups(const Shape& s, bool append) {
  const int64_t want = (s.batches * s.py + WAVES - 1) / WAVES, most = 256 * (append && s.norm != HMA_NORM_NONE ? 3 : 4);
  return (unsigned)(want < most || s.py > 1 ? want : most);
}
template <typename T, bool APPEND, bool F8, int NORM>
void launch_fwd_n(hipStream_t st, const FwdArgs& g) {
  if (g.s.inter)
    hipLaunchKernelGGL((rope_fwd_kernel<T, APPEND, F8, NORM, true>), dim3(fwd_groups(g.s, APPEND)), dim3(TPB), 0, st, g);
  else
    hipLaunchKernelGGL((rope_fwd_kernel<T, APPEND, F8, NORM, false>), dim3(fwd_groups(g.s, APPEND)), dim3(TPB), 0, st, g);
}
template <typename T, bool APPEND, bool F8>
void launch_fwd(hipStream_t st, const FwdArgs& g) {
  if (g.s.norm == HMA_NORM_NONE)
    launch_fwd_n<T, APPEND, F8, HMA_NORM_NONE>(st, g);
  else if (g.s.norm == HMA_NORM_RMS)
    launch_fwd_n<T, APPEND, F8, HMA_NORM_RMS>(st, g);
  else
    launch_fwd_n<T, APPEND, F8, HMA_NORM_LAYER>(st, g);
}
template <typename T, int NORM>
void launch_bwd_n(hipStream_t st, const BwdArgs& g, unsigned groups) {
  if (g.s.inter)
    hipLaunchKernelGGL((rope_bwd_kernel<T, NORM, true>), dim3(groups), dim3(TPB), 0, st, g);
  else
    hipLaunchKernelGGL((rope_bwd_kernel<T, NORM, false>), dim3(groups), dim3(TPB), 0, st, g);
}
template <typename T>
void launch_bwd(hipStream_t st, const BwdArgs& g, unsigned groups) {
  if (g.s.norm == HMA_NORM_NONE)
    launch_bwd_n<T, HMA_NORM_NONE>(st, g, groups);
  else if (g.s.norm == HMA_NORM_RMS)
    launch_bwd_n<T, HMA_NORM_RMS>(st, g, groups);
  else
    launch_bwd_n<T, HMA_NORM_LAYER>(st, g, groups);
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
  // tokens of a wave's batch: as many as have 64 pairs together
  s.wt = 128 / r.d;
  if (s.wt > MAX_WT) s.wt = MAX_WT;
  if (s.wt < 1) s.wt = 1;
  s.batches = (tokens + s.wt - 1) / s.wt;
  // few tokens: the heads of a batch over several waves (each computes the angles again), until there are 4096 -- four a SIMD
  s.py = 1;
  while (s.py < s.passes && s.batches * s.py < 4096) s.py <<= 1;
  if (s.py > s.passes) s.py = s.passes;
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
  if (p->r.dtype == HMA_BF16)
    launch_fwd<Bf16, false, false>((hipStream_t)stream, g);
  else if (p->r.dtype == HMA_F16)
    launch_fwd<_Float16, false, false>((hipStream_t)stream, g);
  else
    launch_fwd<float, false, false>((hipStream_t)stream, g);
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
  // no tokens: no workgroup, and the sums over nothing are zero
  const int64_t want = (g.s.batches + WAVES - 1) / WAVES;
  const int64_t most = p->r.dtype == HMA_F32 ? 512 : 768;  // resident together (3, for fp32 2, a compute unit)
  static_assert(768 <= HMA_QK_ROPE_WS_GROUPS, "");
  const unsigned groups = (unsigned)(want < most ? want : most);
  if (groups) {
    if (p->r.dtype == HMA_BF16)
      launch_bwd<Bf16>((hipStream_t)stream, g, groups);
    else if (p->r.dtype == HMA_F16)
      launch_bwd<_Float16>((hipStream_t)stream, g, groups);
    else
      launch_bwd<float>((hipStream_t)stream, g, groups);
    HMA_CHECK_LAUNCH();
  }
  if (sums) {
    const int width = 4 * p->r.d;
    hipLaunchKernelGGL(rope_wsum_kernel, dim3((width + 15) / 16), dim3(1024), 0, (hipStream_t)stream, p->ws, (int)groups, width, p->dq_w, p->dq_b,
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
  if (p->r.dtype == HMA_BF16) {
    if (f8) launch_fwd<Bf16, true, true>((hipStream_t)stream, g);
    else launch_fwd<Bf16, true, false>((hipStream_t)stream, g);
  } else {
    if (f8) launch_fwd<_Float16, true, true>((hipStream_t)stream, g);
    else launch_fwd<_Float16, true, false>((hipStream_t)stream, g);
  }
  HMA_CHECK_LAUNCH();
  return 0;
}
