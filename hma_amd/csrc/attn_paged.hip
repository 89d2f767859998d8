// Attention of a batch's new tokens over a paged cache: from one token a sequence to whole prompts.
//
//   o = softmax(scale q K^T, over the keys the row sees) V,   lse = log sum exp of the scaled scores;
// the new tokens are the last places of their sequence; a row at place p sees the keys 0 .. p (causal), p - window + 1 .. p (window), or
// every key of its sequence (a frame whose tokens see each other).  A row that sees none: o = 0, lse = -inf.
//
// Rows.  The hq / hk query heads that share a key head are rows of one problem: row r of (sequence, key head) = token r / G, head r % G,
// so a tile of rows reads each key once for the whole group and one decoded token of 8 shared heads is an 8-row problem.
// Products.  S^T = K Q^T by v_mfma_f32_32x32x16: a lane then holds ONE row and 16 of 32 keys, the softmax is in-lane with one exchange
// between the half-waves, and the packed probabilities are the B operand of O^T = V^T P^T as they lie (the contraction index is permuted
// alike on both sides); V^T comes out of row-major LDS by transposing reads.  Scores, maxima, sums and O in 32 bits; probabilities are
// rounded once to the rows' 16-bit type for the second product, as the matrix instruction wants both operands of one type (2^-8 or 2^-11
// relative each, about as much as the output's own rounding adds: the error against 64 bits is 1.2 to 1.4 times that of a softmax in 32
// bits); the sums take them unrounded.  The running maximum is raised only when a row exceeds it by far (Range): that changes no relative
// rounding, and O is rescaled a few times instead of at every step.
// Pages.  A lane looks up the page of one key, the loads take it by a lane exchange.  A key outside what the tile sees, or in a page
// outside the cache, is loaded as zeros, so nothing that is not a sequence's own reaches a product.  e4m3 caches are widened to the rows'
// type (exactly) on their way into LDS; the scales join the scores' factor and the output's.
// Split.  Units of work -- (sequence, key head, row tile, key tile) in that order -- are dealt evenly over the workgroups, so one
// long sequence among short ones fills the chip; a workgroup's first and last row tile may be shared, their (max, sum, O) go to a
// workspace and a second launch joins them in unit order.  No atomics: the same bits every time.
#include <algorithm>
#include <atomic>

#include "hma_common.h"
#include "../../include/hma_hip.h"

using namespace hma;

namespace {

typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef short v4s16_t __attribute__((ext_vector_type(4)));
typedef short v8s16_t __attribute__((ext_vector_type(8)));
#define HMA_LDS(T) __attribute__((address_space(3))) T

constexpr int TPB = 256, WAVES = 4;
constexpr float LN2 = 0.69314718055994530942f, LOG2E = 1.44269504088896340736f;
constexpr int PAD = 16;       // few rows: LDS rows of D + 16 values (two-way conflicts of the transposing reads, which do not bound that kernel)

struct Args {
  const void* q;
  void* o;
  float* lse;
  const uint8_t *kc, *vc;
  const int32_t *table, *cu, *lens;
  const float *k_scale, *v_scale;
  float* part;     // [workgroup][first | last][row][D] then [..][row][max, sum]
  int64_t* units;  // [seqs + 1] first unit of each sequence, then the units of a workgroup
  int64_t tokens, q_tok, q_head, kc_page, kc_head, kc_tok, vc_page, vc_head, vc_tok, table_stride;  // cache strides in bytes
  uint32_t page_mul;
  int32_t page_shift, hq, hk, group, seqs, table_w, pages, page, causal, window, zero_tail, groups;
  float scale;
};

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// Probabilities are 2^(score - m), m = running maximum - LIFT; a row may exceed that maximum by LAZY powers of two before O is rescaled.  fp16 has
// 15 binades above 1 and, at full precision, 14 below: with the largest probability at 2^10 one keeps all its bits down to 2^-24 of it and is lost only
// below 2^-35 (at 1 it would be from 2^-25 on, and 131072 keys 17 powers of e behind one with a value of zero came out 20 % off).  bf16 has the
// range of 32 bits.  SUM: what no 16 probabilities together may exceed, so that none is over 2^LAZY or what the type holds.
template <typename T> struct Range;
template <> struct Range<__bf16> {
  static constexpr float LIFT = 0.f, LAZY = 8.f, SUM = 16.f * 256.f;
};
template <> struct Range<_Float16> {
  static constexpr float LIFT = 10.f, LAZY = 5.f, SUM = 65504.f;
};

template <typename T> struct Op;  // T: __bf16 or _Float16
template <> struct Op<__bf16> {
  static __device__ __forceinline__ f32x16_t mfma(uint4 a, uint4 b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) { return pack_bf16(a, b); }
  static __device__ __forceinline__ uint32_t widen(uint32_t w, bool hi) {  // two e4m3 values
    return __builtin_bit_cast(uint32_t, hi ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true) : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false));
  }
};
template <> struct Op<_Float16> {
  static __device__ __forceinline__ f32x16_t mfma(uint4 a, uint4 b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const half2_t h = {(_Float16)a, (_Float16)b};
    return __builtin_bit_cast(uint32_t, h);
  }
  static __device__ __forceinline__ uint32_t widen(uint32_t w, bool hi) {
    return __builtin_bit_cast(uint32_t, hi ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true) : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false));
  }
};

__device__ __forceinline__ void wave_lds_order() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// ------------------------------------------------------------------------------------- sequences, row tiles, units
struct Seq {
  int32_t row0, n, kv, len;  // first row of the batch, new tokens, keys that the table can hold, length
};
__device__ __forceinline__ Seq seq_from(const Args& a, int cu0, int cu1, int len) {
  Seq s;
  const int64_t c0 = min(max((int64_t)cu0, (int64_t)0), a.tokens), c1 = min(max((int64_t)cu1, c0), a.tokens);
  s.row0 = (int32_t)c0;
  s.n = (int32_t)(c1 - c0);
  s.len = max(len, -0x40000000);
  const int64_t room = min((int64_t)a.table_w * a.page, (int64_t)0x7fff0000);
  s.kv = a.pages > 0 ? (int32_t)min(max((int64_t)s.len, (int64_t)0), room) : 0;
  return s;
}
__device__ __forceinline__ Seq seq_of(const Args& a, int b) { return seq_from(a, a.cu[b], a.cu[b + 1], a.lens[b]); }
__device__ __forceinline__ int row_tiles(const Args& a, const Seq& s, int tr) { return (int)(((int64_t)s.n * a.group + tr - 1) / tr); }
// key tiles of a row tile: the most that any of the sequence's row tiles needs, one at least (a row that sees nothing is written too)
__device__ __forceinline__ int key_tiles(const Args& a, const Seq& s, int tr, int tk) {
  int t = (int)(((int64_t)s.kv + tk - 1) / tk);
  if (a.window > 0) t = (int)min((int64_t)t, ((int64_t)a.window + tr / a.group + 2 + tk - 1) / tk + 1);
  return max(t, 1);
}
// base[b] = units before sequence b, by the whole workgroup
template <int NW>
__device__ __forceinline__ void unit_table(const Args& a, int64_t* base, int64_t* wsum, int tr, int tk) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int64_t carry = 0;
  if (threadIdx.x == 0) base[0] = 0;
  for (int b0 = 0; b0 < a.seqs; b0 += 64 * NW) {
    const int b = b0 + threadIdx.x;
    int64_t v = 0;
    if (b < a.seqs) {
      const Seq s = seq_of(a, b);
      v = (int64_t)a.hk * row_tiles(a, s, tr) * key_tiles(a, s, tr, tk);
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int64_t up = __shfl_up(v, o, 64);
      if (lane >= o) v += up;
    }
    if (lane == 63) wsum[wave] = v;
    __syncthreads();
    int64_t before = carry;
    for (int w = 0; w < NW; ++w) {
      if (w < wave) before += wsum[w];
      carry += wsum[w];
    }
    if (b < a.seqs) base[b + 1] = before + v;
    __syncthreads();
  }
  __syncthreads();
}

// Row tile numbers: sequence b owns first_slot(b) .. first_slot(b + 1) - 1, at least as many as it needs, known without a sum over the
// sequences.  The sequence of a number by the whole wave, 64 candidates a step.
__device__ __forceinline__ int64_t slot_from(const Args& a, int cu, int b, int tr) { return (int64_t)cu * a.group / tr + b; }
__device__ __forceinline__ int64_t first_slot(const Args& a, int b, int tr) { return slot_from(a, a.cu[b], b, tr); }
__device__ __forceinline__ int seq_of_slot(const Args& a, int64_t slot, int tr) {
  const int lane = threadIdx.x & 63;
  int lo = 0, n = a.seqs;
  while (n > 0) {
    const int st = (n + 63) >> 6, i = (lane + 1) * st;
    const int c = __popcll(__ballot(i <= n && first_slot(a, lo + min(i, n), tr) <= slot));
    lo += c * st;
    n = st == 1 ? 0 : min(st, n - c * st);
  }
  return lo;  // seqs: behind the last sequence
}

// A row tile of a sequence: what its rows see
struct Tile {
  int32_t lo_min, lo_max, hi_min, hi_max, start;  // keys seen by any row: [lo_min, hi_max), by every row: [lo_max, hi_min); first key of key tile 0
};
__device__ __forceinline__ int32_t lo_of(const Args& a, const Seq& s, int tok) {
  return a.window > 0 ? (int32_t)max((int64_t)0, (int64_t)s.len - s.n + tok - a.window + 1) : 0;
}
__device__ __forceinline__ int32_t hi_of(const Args& a, const Seq& s, int tok) {
  return a.causal ? min(max(s.len - s.n + tok + 1, 0), s.kv) : s.kv;
}
__device__ __forceinline__ Tile tile_of(const Args& a, const Seq& s, int qt, int tr, int tk) {
  const int r0 = qt * tr, r1 = (int)min((int64_t)r0 + tr, (int64_t)s.n * a.group) - 1;
  const int t0 = r0 / a.group, t1 = r1 / a.group;
  Tile t;
  t.lo_min = lo_of(a, s, t0);
  t.lo_max = lo_of(a, s, t1);
  t.hi_min = hi_of(a, s, t0);
  t.hi_max = hi_of(a, s, t1);
  t.start = t.lo_min / tk * tk;
  return t;
}

// ------------------------------------------------------------------------------------- one wave: 32 rows against blocks of 32 keys
template <typename T, int D>
struct Rows {
  uint4 q[D / 16];
  f32x16_t o[D / 32];
  float m, l;       // running maximum less LIFT (powers of two), sum of this half-wave's keys
  int32_t lo, hi;   // keys that the row sees
  bool live;
  int64_t at;       // its row of o (tokens x heads)

  __device__ __forceinline__ void begin(const Args& a, const Seq& s, int hk, int r) {
    const int lane = threadIdx.x & 63;
    live = r < (int64_t)s.n * a.group;
    const int tok = live ? r / a.group : 0, h = hk * a.group + (live ? r - tok * a.group : 0);
    at = (int64_t)(s.row0 + tok) * a.hq + h;
    lo = live ? lo_of(a, s, tok) : 0;
    hi = live ? hi_of(a, s, tok) : 0x7fffffff;
    const uint16_t* p = (const uint16_t*)a.q + (int64_t)(s.row0 + tok) * a.q_tok + h * a.q_head + (lane >> 5) * 8;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) q[i] = live ? *reinterpret_cast<const uint4*>(p + i * 16) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[i][e] = 0.f;
    m = -INFINITY;
    l = 0.f;
  }

  // the rows' loads waited for here (the compiler, which does not count LDS DMA, would wait for them -- and for all in flight -- in the loop)
  __device__ __forceinline__ void arrive() {
#pragma unroll
    for (int i = 0; i < D / 16; ++i) asm volatile("" : "+v"(q[i].x), "+v"(q[i].y), "+v"(q[i].z), "+v"(q[i].w));
  }
  // scores of KB blocks of 32 keys; kt: their rows in LDS
  template <int KB>
  __device__ __forceinline__ void scores(const uint16_t* kt, f32x16_t (&s)[KB]) const {
    const int lane = threadIdx.x & 63;
    const uint16_t* p = kt + (lane & 31) * (D + PAD) + (lane >> 5) * 8;
#pragma unroll
    for (int k = 0; k < KB; ++k) {
#pragma unroll
      for (int e = 0; e < 16; ++e) s[k][e] = 0.f;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) s[k] = Op<T>::mfma(*reinterpret_cast<const uint4*>(p + k * 32 * (D + PAD) + i * 16), q[i], s[k]);
    }
  }
  // what a row does not see out of the scores
  template <int KB>
  __device__ __forceinline__ void mask(f32x16_t (&s)[KB], int key0) const {
    const uint32_t first = (uint32_t)(key0 - lo + 4 * ((threadIdx.x & 63) >> 5)), span = (uint32_t)max(hi - lo, 0);
#pragma unroll
    for (int k = 0; k < KB; ++k)
#pragma unroll
      for (int e = 0; e < 16; ++e) s[k][e] = first + (k * 32 + 8 * (e >> 2) + (e & 3)) < span ? s[k][e] : -INFINITY;
  }
  // keys without a page (bits of `bad`) out of the scores
  template <int KB>
  __device__ __forceinline__ void mask_bad(f32x16_t (&s)[KB], uint64_t bad) const {
#pragma unroll
    for (int k = 0; k < KB; ++k) {
      const uint32_t w = (uint32_t)(bad >> (k * 32)) >> (4 * ((threadIdx.x & 63) >> 5));
#pragma unroll
      for (int e = 0; e < 16; ++e) s[k][e] = w & (1u << (8 * (e >> 2) + (e & 3))) ? -INFINITY : s[k][e];
    }
  }
  // the largest score of a row's KB blocks in powers of two less LIFT (c: the scores' factor)
  template <int KB>
  __device__ __forceinline__ float largest(const f32x16_t (&s)[KB], float c) const {
    float x0 = -INFINITY, x1 = -INFINITY;
#pragma unroll
    for (int k = 0; k < KB; ++k)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        x0 = __builtin_fmaxf(__builtin_fmaxf(x0, s[k][e]), s[k][e + 1]);
        x1 = __builtin_fmaxf(__builtin_fmaxf(x1, s[k][e + 2]), s[k][e + 3]);
      }
    const uint32_t x = __float_as_uint(fmaxf(x0, x1));
    const auto both = __builtin_amdgcn_permlane32_swap(x, x, false, false);  // the two half-waves' values in every lane
    return __builtin_fmaf(fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1])), c, -Range<T>::LIFT);
  }
  // the running maximum raised where a row exceeds it by far (lazy: how far, in powers of two)
  __device__ __forceinline__ void raise(float x, float lazy) {
    if (__ballot(x > m + lazy)) {  // also where m is still -inf
      const float up = fmaxf(m, x), f = m == -INFINITY ? 0.f : fast_exp2(m - up);
      l *= f;
#pragma unroll
      for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[i][e] *= f;
      m = up;
    }
  }
  // a block of scores -> probabilities relative to the running maximum, packed as the second product's operand, and their sum
  __device__ __forceinline__ void weigh(f32x16_t& s, float c, uint4 (&p)[2]) {
    const float sub = m == -INFINITY ? 0.f : m;
    float l0 = 0.f, l1 = 0.f;
#pragma unroll
    for (int e = 0; e < 16; e += 2) {
      s[e] = fast_exp2(__builtin_fmaf(s[e], c, -sub));
      s[e + 1] = fast_exp2(__builtin_fmaf(s[e + 1], c, -sub));
      l0 += s[e];
      l1 += s[e + 1];
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
      p[h] = make_uint4(Op<T>::pack(s[8 * h], s[8 * h + 1]), Op<T>::pack(s[8 * h + 2], s[8 * h + 3]), Op<T>::pack(s[8 * h + 4], s[8 * h + 5]),
                        Op<T>::pack(s[8 * h + 6], s[8 * h + 7]));
    l += l0 + l1;
  }
  // o += V^T p; vt: the values' rows in LDS.  The transposing read gives lane (d = l & 31, half) the rows 4 half + {0..3} and those + 8 of
  // 16 -- the order in which pack left a row's probabilities.
  template <int KB>
  __device__ __forceinline__ void values(const uint16_t* vt, const uint4 (&p)[KB][2]) {
    const int lane = threadIdx.x & 63, i16 = lane & 15, g16 = lane >> 4;
    const uint16_t* base = vt + (4 * (g16 >> 1) + (i16 >> 2)) * (D + PAD) + 16 * (g16 & 1) + 4 * (i16 & 3);
#pragma unroll
    for (int k = 0; k < KB; ++k)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
          const uint16_t* v = base + (k * 32 + h * 16) * (D + PAD) + i * 32;
          const v4s16_t a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((HMA_LDS(v4s16_t)*)v);
          const v4s16_t b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((HMA_LDS(v4s16_t)*)(v + 8 * (D + PAD)));
          const v8s16_t w = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
          o[i] = Op<T>::mfma(__builtin_bit_cast(uint4, w), p[k][h], o[i]);
        }
  }
  // both half-waves' sums into each
  __device__ __forceinline__ void finish() { l += __shfl_xor(l, 32, 64); }

  // the rows' outputs: o / l, lse
  __device__ __forceinline__ void write(const Args& a, float vs) const {
    const int half = (threadIdx.x & 63) >> 5;
    const float f = l > 0.f ? vs / l : (l == 0.f ? 0.f : l);  // a NaN stays one
    uint16_t* row = (uint16_t*)a.o + at * D;
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
      for (int g = 0; g < 4; g += 2) {  // the half-waves trade quads: 16 contiguous bytes each
        const uint32_t ax = Op<T>::pack(o[i][4 * g] * f, o[i][4 * g + 1] * f), ay = Op<T>::pack(o[i][4 * g + 2] * f, o[i][4 * g + 3] * f);
        const uint32_t bx = Op<T>::pack(o[i][4 * g + 4] * f, o[i][4 * g + 5] * f), by = Op<T>::pack(o[i][4 * g + 6] * f, o[i][4 * g + 7] * f);
        const auto r0 = __builtin_amdgcn_permlane32_swap(ax, bx, false, false);
        const auto r1 = __builtin_amdgcn_permlane32_swap(ay, by, false, false);
        if (live) *reinterpret_cast<uint4*>(row + i * 32 + 8 * g + 8 * half) = make_uint4(r0[0], r1[0], r0[1], r1[1]);
      }
    if (live && half == 0 && a.lse) a.lse[at] = l == 0.f ? -INFINITY : (m + __log2f(l)) * LN2;
  }
  // a share of a row tile: unnormalised, for the second launch
  __device__ __forceinline__ void write_part(const Args& a, int64_t slot, int tr, int row) const {
    const int half = (threadIdx.x & 63) >> 5;
    float* p = a.part + (slot * tr + row) * D;
    if (live) {
#pragma unroll
      for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<float4*>(p + i * 32 + 8 * g + 4 * half) = make_float4(o[i][4 * g], o[i][4 * g + 1], o[i][4 * g + 2], o[i][4 * g + 3]);
      if (half == 0) {
        float* ml = a.part + (int64_t)a.groups * 2 * tr * D + (slot * tr + row) * 2;
        *reinterpret_cast<float2*>(ml) = make_float2(m, l);
      }
    }
  }
};

// ------------------------------------------------------------------------------------- loads of a block of keys
// THREADS threads load KEYS rows of 16-byte pieces, a wave RPW rows an instruction; lane l of each wave knows the page and the place in it
// of key l.  ALIGNED: the page size is a multiple of RPW, so the rows of an instruction lie in one page one behind the other and their
// address is scalar but for the lane's piece; otherwise each lane fetches its row's page by a lane exchange and multiplies by itself.
template <typename T, int D, bool F8, int KEYS, int THREADS, bool ALIGNED>
struct Loader {
  static constexpr int BYTES = F8 ? D : 2 * D, CPR = BYTES / 16, RPW = 64 / CPR, RPI = THREADS / CPR, NI = RPI < KEYS ? KEYS / RPI : 1;
  static_assert((KEYS % RPI == 0 || RPI % KEYS == 0) && KEYS <= 64, "");  // short rows: threads with nothing to load repeat what others do

  // tid = wave * 64 + lane
  static __device__ __forceinline__ void load(const uint8_t* c, int64_t page, int64_t tok, int pg, int off, int wave, int lane, uint4 (&r)[NI]) {
    if (ALIGNED) {
      const uint32_t mine = (uint32_t)(lane / CPR) * (uint32_t)tok + (lane % CPR) * 16;  // below 2^31: the host's check
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int row = (i * RPI + wave * RPW) % KEYS;
        const int p = __builtin_amdgcn_readlane(pg, row), f = __builtin_amdgcn_readlane(off, row);
        r[i] = *reinterpret_cast<const uint4*>(c + (p < 0 ? 0 : p * page + f * tok) + mine);
      }
    } else {
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int row = (i * RPI + wave * RPW + lane / CPR) % KEYS;
        const int p = __shfl(pg, row, 64), f = __shfl(off, row, 64);
        r[i] = *reinterpret_cast<const uint4*>(c + (p < 0 ? 0 : p * page + f * tok) + (lane % CPR) * 16);
      }
    }
  }
  // `gaps`: some key is not seen or has no page (`ok` false for lane = key): zeros
  static __device__ __forceinline__ void store(uint16_t* t, bool ok, bool gaps, int wave, int lane, uint4 (&r)[NI]) {
    if (gaps) {
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const bool have = __shfl((int)ok, (i * RPI + wave * RPW + lane / CPR) % KEYS, 64);
        r[i].x = have ? r[i].x : 0u; r[i].y = have ? r[i].y : 0u; r[i].z = have ? r[i].z : 0u; r[i].w = have ? r[i].w : 0u;
      }
    }
    uint16_t* p = t + ((wave * RPW + lane / CPR) % KEYS) * (D + PAD) + (lane % CPR) * (F8 ? 16 : 8);
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      uint16_t* w = p + i * RPI * (D + PAD);
      if (F8) {
        *reinterpret_cast<uint4*>(w) = make_uint4(Op<T>::widen(r[i].x, false), Op<T>::widen(r[i].x, true), Op<T>::widen(r[i].y, false), Op<T>::widen(r[i].y, true));
        *reinterpret_cast<uint4*>(w + 8) = make_uint4(Op<T>::widen(r[i].z, false), Op<T>::widen(r[i].z, true), Op<T>::widen(r[i].w, false), Op<T>::widen(r[i].w, true));
      } else {
        *reinterpret_cast<uint4*>(w) = r[i];
      }
    }
  }
};

// The page of key `key` of a sequence and its place there.  look() only issues the table's load (a key behind the sequence: its last
// page, row 0); what is asked of the page number waits for it, so it is asked a tile later.
struct Place {
  int32_t raw, off, key;
  __device__ __forceinline__ void look(const Args& a, const int32_t* table, int k, int kv) {  // kv > 0
    const int32_t i = (int32_t)(((uint64_t)(uint32_t)min(k, kv - 1) * a.page_mul) >> (31 + a.page_shift));
    key = k;
    off = k < kv ? k - i * a.page : 0;
    raw = table[i];
  }
  __device__ __forceinline__ bool good(const Args& a) const { return (uint32_t)raw < (uint32_t)a.pages; }
  __device__ __forceinline__ bool in(const Tile& t) const { return key >= t.lo_min && key < t.hi_max; }
  __device__ __forceinline__ bool seen(const Args& a, const Tile& t) const { return in(t) && good(a); }   // by some row of the tile, and in the cache
  __device__ __forceinline__ bool lost(const Args& a, const Tile& t) const { return in(t) && !good(a); }  // its page is none of the cache's
  // bytes from the head's first row to key's row
  __device__ __forceinline__ int64_t at(const Args& a, int64_t page, int64_t tok) const { return good(a) ? raw * page + off * tok : 0; }
};

// rows behind the last sequence
template <int D>
__device__ __forceinline__ void clear_tail(const Args& a) {
  if (!a.zero_tail) return;
  const int64_t end = min(max((int64_t)a.cu[a.seqs], (int64_t)0), a.tokens);
  const int64_t rows = (a.tokens - end) * a.hq, n = rows * (D / 8), at = end * a.hq;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
    *reinterpret_cast<uint4*>((uint16_t*)a.o + at * D + i * 8) = make_uint4(0, 0, 0, 0);
    if (a.lse && i % (D / 8) == 0) a.lse[at + i / (D / 8)] = -INFINITY;
  }
}

// first unit of this workgroup and the one behind its last; workgroups that run on one XCD (number % 8) take neighbouring shares
__device__ __forceinline__ int share_of(int groups) {
  const int b = blockIdx.x;
  return groups % 8 == 0 ? (b & 7) * (groups >> 3) + (b >> 3) : b;
}

// ------------------------------------------------------------------------------------- few rows: the waves take different keys
// Bound by the bytes of the cache.  Each wave has a block of keys of its own (no barrier among the waves until a row tile ends), fetches the
// next block's keys and values into registers while it multiplies, and looks the block after that up in the table; two workgroups a compute
// unit keep 8 x 16 KB in flight there.  64 sequences of up to 16 K tokens, 8 key heads of 128, bf16: 2.15 GB in 380 us = 5.6 TB/s; 4 of 66 to 131 K
// tokens in e4m3: 0.8 GB in 163 us = 4.9 TB/s; one of 700 tokens: 9 us + 4 us to join, all latency.
template <typename T, int D, bool F8, int KB, bool ALIGNED>
__global__ __launch_bounds__(TPB, 2) void attn_few_kernel(const Args a) {
  constexpr int TR = 32, KEYS = 32 * KB, TK = WAVES * KEYS, LD = D + PAD, NO = D / 32;
  typedef Loader<T, D, F8, KEYS, 64, ALIGNED> Ld;
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  __shared__ int64_t wsum[WAVES];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  uint16_t* tiles = (uint16_t*)smem;
  uint16_t* mine = tiles + wave * KEYS * LD;
  float* xch = (float*)smem;  // the waves' results on their way to wave 0
  int64_t* base = (int64_t*)(smem + WAVES * KEYS * LD * 2);
  clear_tail<D>(a);
  if (a.seqs == 0) return;
  unit_table<WAVES>(a, base, wsum, TR, TK);
  const int64_t total = base[a.seqs], each = (total + a.groups - 1) / a.groups;
  if (blockIdx.x == 0) {
    for (int i = threadIdx.x; i <= a.seqs; i += TPB) a.units[i] = base[i];
    if (threadIdx.x == 0) a.units[a.seqs + 1] = each;
  }
  const int64_t g = share_of(a.groups), u0 = g * each, u1 = min(total, u0 + each);
  if (u0 >= u1) return;
  int b = 0;
  for (int lo = 0, hi = a.seqs - 1; lo <= hi;) {  // the last sequence with base <= u0
    const int mid = (lo + hi) >> 1;
    if (base[mid] <= u0) b = mid, lo = mid + 1; else hi = mid - 1;
  }
  for (int64_t u = u0; u < u1;) {
    while (base[b + 1] <= u) ++b;
    const Seq s = seq_of(a, b);
    const int nt = key_tiles(a, s, TR, TK), nq = row_tiles(a, s, TR);
    const int64_t local = u - base[b], item = local / nt, first = u - (local - item * nt);
    const int j0 = (int)(local - item * nt), j1 = (int)min((int64_t)nt, j0 + (u1 - u));
    const int hk = (int)(item / nq), qt = (int)(item - (int64_t)hk * nq);
    const Tile t = tile_of(a, s, qt, TR, TK);
    const int32_t* table = a.table + b * a.table_stride;
    const uint8_t *kc = a.kc + hk * a.kc_head, *vc = a.vc + hk * a.vc_head;
    const float c = a.scale * LOG2E * (F8 ? a.k_scale[hk] : 1.0f);
    Rows<T, D> r;
    r.begin(a, s, hk, qt * TR + (lane & 31));

    // key blocks of this wave: start + j TK + wave KEYS; only those that the tile sees
    auto key_of = [&](int j) { return t.start + j * TK + wave * KEYS; };
    int j = j0, je = j1;
    while (j < je && key_of(j) + KEYS <= t.lo_min) ++j;
    while (je > j && (int64_t)t.start + (int64_t)(je - 1) * TK + wave * KEYS >= t.hi_max) --je;
    if (j < je) {
      const int kl = lane & (KEYS - 1);
      Place now, next;
      now.look(a, table, key_of(j) + kl, s.kv);
      next = now;
      int pg = now.good(a) ? now.raw : -1;
      uint4 kr[Ld::NI], vr[Ld::NI];
      Ld::load(kc, a.kc_page, a.kc_tok, pg, now.off, 0, lane, kr);
      Ld::load(vc, a.vc_page, a.vc_tok, pg, now.off, 0, lane, vr);
      if (j + 1 < je) next.look(a, table, key_of(j + 1) + kl, s.kv);
      for (; j < je; ++j) {
        const int key0 = key_of(j);
        const bool seen = now.seen(a, t), gaps = __ballot(!seen) != 0, more = j + 1 < je;
        const uint64_t bad = __ballot(now.lost(a, t));
        f32x16_t sc[KB];
        uint4 p[KB][2];
        Ld::store(mine, seen, gaps, 0, lane, kr);
        pg = next.good(a) ? next.raw : -1;
        if (more) Ld::load(kc, a.kc_page, a.kc_tok, pg, next.off, 0, lane, kr);
        wave_lds_order();
        r.template scores<KB>(mine, sc);
        if (key0 < t.lo_max || key0 + KEYS > t.hi_min) r.template mask<KB>(sc, key0);
        if (bad) r.template mask_bad<KB>(sc, bad);
        r.raise(r.template largest<KB>(sc, c), Range<T>::LAZY);
#pragma unroll
        for (int k = 0; k < KB; ++k) r.weigh(sc[k], c, p[k]);
        wave_lds_order();
        Ld::store(mine, seen, gaps, 0, lane, vr);
        if (more) {
          Ld::load(vc, a.vc_page, a.vc_tok, pg, next.off, 0, lane, vr);
          now = next;
          if (j + 2 < je) next.look(a, table, key_of(j + 2) + kl, s.kv);
        }
        wave_lds_order();
        r.template values<KB>(mine, p);
        wave_lds_order();
      }
    }
    r.finish();
    // waves 2, 3 -> 0, 1, then 1 -> 0
    for (int step = 2; step >= 1; step >>= 1) {
      __syncthreads();
      float* x = xch + (wave & (step - 1)) * (NO * 16 + 2) * 64 + lane;
      if (wave >= step && wave < 2 * step) {
#pragma unroll
        for (int i = 0; i < NO; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e) x[(i * 16 + e) * 64] = r.o[i][e];
        x[NO * 16 * 64] = r.m;
        x[(NO * 16 + 1) * 64] = r.l;
      }
      __syncthreads();
      if (wave < step) {
        const float m2 = x[NO * 16 * 64], l2 = x[(NO * 16 + 1) * 64], mm = fmaxf(r.m, m2);
        const float f1 = r.m == -INFINITY ? 0.f : fast_exp2(r.m - mm), f2 = m2 == -INFINITY ? 0.f : fast_exp2(m2 - mm);
#pragma unroll
        for (int i = 0; i < NO; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e) r.o[i][e] = r.o[i][e] * f1 + x[(i * 16 + e) * 64] * f2;
        r.l = r.l * f1 + l2 * f2;
        r.m = mm;
      }
    }
    if (wave == 0) {
      if (j0 == 0 && j1 == nt)
        r.write(a, F8 ? a.v_scale[hk] : 1.0f);
      else
        r.write_part(a, g * 2 + (first < u0 ? 0 : 1), TR, lane & 31);
    }
    __syncthreads();
    u += j1 - j0;
  }
}

// ------------------------------------------------------------------------------------- many rows: a wave takes 32 of the tile's 128
// The waves share tiles of 64 keys and values, two of each in LDS.  A wave has two companions at most on its SIMD and issues an
// instruction every five cycles or so, whatever its kind, so the instructions around the products and the exponentials are what there is
// to save: 16-bit tiles come by LDS DMA in pieces of 1 KB, whose addresses are scalar (two lane reads and two additions a piece) plus one
// register of lane offsets; a tile of keys is 16 such pieces at D = 128, four a wave.
// Layout of a tile: piece = 64 / CPR rows (CPR = D / 8 chunks of 16 bytes each), pieces 16 bytes further apart than their size, chunk c of
// row r at place c ^ turn(r) of its row.  A 16-byte read of 16 rows and a transposing read of 4 rows x 64 bytes then touch every bank once.
// Two prompts of 5 to 8 K tokens, 32 heads of 128 on 8, 755 GFLOP: 763 to 790 us a launch back to back = 0.96 to 0.99 PFLOP/s, two thirds of what
// a large matrix product reaches here (791 to 857 us apart from each other, under a trace).  Of a SIMD's cycles 49 % have a matrix instruction and 56 % a
// vector one in work; a wave waits 32 % of its own.  Heads of 32 have as many exponentials for a quarter of the products: 4 frames of 320
// tokens over 5 to 20 K, 17 GFLOP in 51 us, vector instructions in 69 % of the cycles (200 for 64 keys of 32 rows, 32 of them exponentials),
// matrix instructions in 18 %, waves waiting 42 %.
// Rejected, at the prompts: 64 rows a wave (one wave a SIMD) 862 us, 8 waves a workgroup the same, half tiles out of step slower.
template <int D>
struct Lay {
  static constexpr int CPR = D / 8, RPP = 64 / CPR, PIECE = 1024 + (D == 32 ? 0 : 16), PIECES = 64 / RPP, TILE = PIECES * PIECE;
  static __device__ __forceinline__ int turn(int r) { return D == 128 ? 4 * (r & 3) : D == 64 ? 4 * ((r >> 1) & 1) + 2 * ((r >> 2) & 1) : (r >> 2) & 3; }
  static __device__ __forceinline__ int at(int r, int c) { return r / RPP * PIECE + r % RPP * (2 * D) + (c ^ turn(r)) * 16; }
};
template <int D> struct ManyWaves { static constexpr int value = D == 128 ? 2 : D == 64 ? 3 : 4; };  // waves a SIMD

template <typename T, int D, bool F8, bool ALIGNED>
__global__ __launch_bounds__(TPB, ManyWaves<D>::value) void attn_many_kernel(const Args a, const int split) {
  typedef Lay<D> Y;
  constexpr int NW = WAVES, TR = 32 * NW, TK = 64, BUF = 2 * Y::TILE, NO = D / 32;
  constexpr bool DMA = !F8 && ALIGNED;
  constexpr int NP = Y::PIECES / NW;  // pieces of a tile per wave
  static_assert(Y::PIECES % NW == 0, "");
  // through registers: 16-byte pieces of the cache's rows, NI a thread
  constexpr int BYTES = F8 ? D : 2 * D, CPR = BYTES / 16, RPW = 64 / CPR, RPI = NW * RPW, NI = RPI < TK ? TK / RPI : 1;
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];  // [2][keys | values]
  __shared__ int64_t wsum[NW];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int64_t* base = (int64_t*)(smem + 2 * BUF);
  clear_tail<D>(a);
  if (a.seqs == 0) return;
  int64_t u0 = 0, u1 = 1, g = 0;
  int b = 0, slot_qt = 0;
  if (split) {
    unit_table<NW>(a, base, wsum, TR, TK);
    const int64_t total = base[a.seqs], each = (total + a.groups - 1) / a.groups;
    if (blockIdx.x == 0) {
      for (int i = tid; i <= a.seqs; i += 64 * NW) a.units[i] = base[i];
      if (tid == 0) a.units[a.seqs + 1] = each;
    }
    g = share_of(a.groups);
    u0 = g * each;
    u1 = min(total, u0 + each);
    if (u0 >= u1) return;
    for (int lo = 0, hi = a.seqs - 1; lo <= hi;) {
      const int mid = (lo + hi) >> 1;
      if (base[mid] <= u0) b = mid, lo = mid + 1; else hi = mid - 1;
    }
  } else {
    const int64_t slot = (int64_t)gridDim.x / a.hk - 1 - blockIdx.x / a.hk;  // the last tiles of a sequence, which see most, first
    b = __builtin_amdgcn_readfirstlane(seq_of_slot(a, slot, TR));
    if (b >= a.seqs) return;
    slot_qt = (int)(slot - first_slot(a, b, TR));
  }
  // lane constants: where this lane's operands lie in a tile
  const int half = lane >> 5, i16 = lane & 15, g16 = lane >> 4;
  constexpr int NKA = D == 128 ? 4 : D / 16;
  uint32_t ka[NKA], va[NO], va8 = 0;
#pragma unroll
  for (int s = 0; s < NKA; ++s) ka[s] = Y::at(lane & 31, (D == 128 ? 4 : 2) * s + half);
#pragma unroll
  for (int i = 0; i < NO; ++i) va[i] = Y::at(4 * (g16 >> 1) + (i16 >> 2), 4 * i + 2 * (g16 & 1) + ((i16 & 3) >> 1)) + 8 * (i16 & 1);
  if (D == 32) va8 = Y::at(8 + 4 * (g16 >> 1) + (i16 >> 2), 2 * (g16 & 1) + ((i16 & 3) >> 1)) + 8 * (i16 & 1);
  const int turned = ((lane % Y::CPR) ^ Y::turn(lane / Y::CPR)) * 16;  // DMA: the chunk that belongs in this lane's place
  const uint32_t k_off = lane / Y::CPR * (uint32_t)a.kc_tok + turned, v_off = lane / Y::CPR * (uint32_t)a.vc_tok + turned;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(HMA_LDS(uint8_t)*)smem;
  const bool alike = a.kc_page == a.vc_page && a.kc_tok == a.vc_tok;

  for (int64_t u = u0; u < u1;) {
    if (split)
      while (base[b + 1] <= u) ++b;
    const Seq s = seq_of(a, b);
    const int nq = row_tiles(a, s, TR);
    int nt, j0, j1, hk, qt;
    int64_t first = 0;
    Tile t;
    if (split) {
      nt = key_tiles(a, s, TR, TK);
      const int64_t local = u - base[b], item = local / nt;
      first = u - (local - item * nt);
      j0 = (int)(local - item * nt);
      j1 = (int)min((int64_t)nt, j0 + (u1 - u));
      hk = (int)(item / nq);
      qt = (int)(item - (int64_t)hk * nq);
      t = tile_of(a, s, qt, TR, TK);
    } else {
      qt = slot_qt;
      hk = blockIdx.x % a.hk;
      if (qt < 0 || qt >= nq) return;
      t = tile_of(a, s, qt, TR, TK);
      j0 = 0;
      nt = j1 = max((t.hi_max - t.start + TK - 1) / TK, 0);
    }
    const int32_t* table = a.table + b * a.table_stride;
    const uint8_t *kc = a.kc + hk * a.kc_head, *vc = a.vc + hk * a.vc_head;
    const float c = a.scale * LOG2E * (F8 ? a.k_scale[hk] : 1.0f);
    Rows<T, D> r;
    r.begin(a, s, hk, qt * TR + wave * 32 + (lane & 31));
    // what this wave's 32 rows see (rows that are none see nothing)
    const bool any = qt * TR + wave * 32 < (int64_t)s.n * a.group;
    Tile w = t;
    if (any) w = tile_of(a, s, qt * NW + wave, 32, TK);
    const int je = min(j1, max((t.hi_max - t.start + TK - 1) / TK, 0));

    uint4 kr[DMA ? 1 : NI], vr[DMA ? 1 : NI];
    // tile of `p` on its way: into LDS buffer `buf`, or into registers
    const auto fetch = [&](const Place& p, int buf) {
      if (DMA && NP <= 2) {  // few pieces a wave: their addresses by scalar products (D = 32, a frame: 52.7 -> 51.2 us)
        const int raw = p.good(a) ? p.raw : 0, off = p.good(a) ? p.off : 0;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          const int piece = i * NW + wave, row = piece * Y::RPP;
          const int64_t pg = __builtin_amdgcn_readlane(raw, row), of = __builtin_amdgcn_readlane(off, row);
          const uint32_t to = lds0 + buf * BUF + piece * Y::PIECE;
          const int64_t ko = pg * a.kc_page + of * a.kc_tok;
          glds16s(kc + ko, k_off, to);
          glds16s(vc + (alike ? ko : pg * a.vc_page + of * a.vc_tok), v_off, to + Y::TILE);
        }
      } else if (DMA) {
        const int64_t ko = p.at(a, a.kc_page, a.kc_tok);
        int64_t vo = ko;
        if (!alike) vo = p.at(a, a.vc_page, a.vc_tok);
        const int klo = (int)ko, khi = (int)(ko >> 32), vlo = (int)vo, vhi = (int)(vo >> 32);
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          const int piece = i * NW + wave, row = piece * Y::RPP;
          const uint32_t to = lds0 + buf * BUF + piece * Y::PIECE;
          glds16s(kc + (((int64_t)__builtin_amdgcn_readlane(khi, row) << 32) | (uint32_t)__builtin_amdgcn_readlane(klo, row)), k_off, to);
          glds16s(vc + (((int64_t)__builtin_amdgcn_readlane(vhi, row) << 32) | (uint32_t)__builtin_amdgcn_readlane(vlo, row)), v_off, to + Y::TILE);
        }
      } else {
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          const int row = (i * RPI + wave * RPW + lane / CPR) % TK;
          const int pg = __shfl(p.good(a) ? p.raw : -1, row, 64), f = __shfl(p.off, row, 64);
          kr[i] = *reinterpret_cast<const uint4*>(kc + (pg < 0 ? 0 : pg * a.kc_page + f * a.kc_tok) + (lane % CPR) * 16);
          vr[i] = *reinterpret_cast<const uint4*>(vc + (pg < 0 ? 0 : pg * a.vc_page + f * a.vc_tok) + (lane % CPR) * 16);
        }
      }
    };
    // the fetched tile into place: values of keys that no row sees are zeros (their scores are masked, but 0 x NaN is a NaN)
    const auto settle = [&](const Place& p, int buf) {
      const bool seen = p.seen(a, t), gaps = __ballot(!seen) != 0;
      uint8_t *kt = smem + buf * BUF, *vt = kt + Y::TILE;
      if (DMA) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        if (gaps) {
#pragma unroll
          for (int i = 0; i < NP; ++i) {
            const int piece = i * NW + wave;
            if (!__shfl((int)seen, piece * Y::RPP + lane / Y::CPR, 64)) *reinterpret_cast<uint4*>(vt + piece * Y::PIECE + lane * 16) = make_uint4(0, 0, 0, 0);
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          const int row = (i * RPI + wave * RPW + lane / CPR) % TK, ch = lane % CPR;
          const bool have = !gaps || __shfl((int)seen, row, 64);
          uint4 v = vr[i];
          v.x = have ? v.x : 0u; v.y = have ? v.y : 0u; v.z = have ? v.z : 0u; v.w = have ? v.w : 0u;
          if (F8) {
            const auto lo = [](const uint4& x) { return make_uint4(Op<T>::widen(x.x, false), Op<T>::widen(x.x, true), Op<T>::widen(x.y, false), Op<T>::widen(x.y, true)); };
            const auto hi = [](const uint4& x) { return make_uint4(Op<T>::widen(x.z, false), Op<T>::widen(x.z, true), Op<T>::widen(x.w, false), Op<T>::widen(x.w, true)); };
            *reinterpret_cast<uint4*>(kt + Y::at(row, 2 * ch)) = lo(kr[i]);
            *reinterpret_cast<uint4*>(kt + Y::at(row, 2 * ch + 1)) = hi(kr[i]);
            *reinterpret_cast<uint4*>(vt + Y::at(row, 2 * ch)) = lo(v);
            *reinterpret_cast<uint4*>(vt + Y::at(row, 2 * ch + 1)) = hi(v);
          } else {
            *reinterpret_cast<uint4*>(kt + Y::at(row, ch)) = kr[i];
            *reinterpret_cast<uint4*>(vt + Y::at(row, ch)) = v;
          }
        }
      }
    };
    if (j0 < je) {
      const auto look = [&](Place& p, int j) { p.look(a, table, t.start + j * TK + lane, s.kv); };
      Place now, next;
      look(now, j0);
      look(next, j0 + 1);
      r.arrive();
      fetch(now, 0);
      settle(now, 0);
      __syncthreads();
      int buf = 0;
      for (int j = j0; j < je; ++j, buf ^= 1) {
        const bool more = j + 1 < je;
        const uint64_t bad = __ballot(now.lost(a, t));
        Place after = next;
        if (more) {
          fetch(next, buf ^ 1);
          look(after, j + 2);
        }
        const int key0 = t.start + j * TK;
        if (any && key0 < w.hi_max && key0 + TK > w.lo_min) {
          const uint8_t *kt = smem + buf * BUF, *vt = kt + Y::TILE;
          // Two blocks of 32 keys.  The reads run AHEAD operands in front of the products that use them; the first block's exponentials stand
          // between the second's products, the second's between the first's values.  The barriers stop the compiler only: left alone it
          // puts each read right in front of its product and the exponentials behind the last, and the wave waits in both places.
          constexpr int NS = D / 16, AHEAD = 2;  // operands of a block of 32 keys, of a block of 32 values
          const auto key_operand = [&](int n) {
            const int at = D == 128 ? ka[(n % NS) >> 1] + (n & 1) * 32 : ka[n % NS % NKA];
            return *reinterpret_cast<const uint4*>(kt + at + n / NS * (32 / Y::RPP) * Y::PIECE);
          };
          const auto value_operand = [&](int n) {  // 16 keys, 32 columns n % NO
            const uint8_t* v = vt + n / NO * 16 / Y::RPP * Y::PIECE;
            const uint8_t* v8 = D == 32 ? v + va8 : v + va[n % NO] + 8 / Y::RPP * Y::PIECE;
            const v4s16_t x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((HMA_LDS(v4s16_t)*)(v + va[n % NO]));
            const v4s16_t y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((HMA_LDS(v4s16_t)*)v8);
            return __builtin_bit_cast(uint4, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
          };
          __builtin_amdgcn_s_setprio(1);  // ahead of the SIMD's waves that wait or fetch (a frame of 320 tokens over 20k: 63 -> 61 us)
          const bool edge = key0 < w.lo_max || key0 + TK > w.hi_min || bad != 0;
          f32x16_t sc[2];
          uint4 f[2 * NS], p[2];
          float sub = r.m == -INFINITY ? 0.f : r.m, sum = 0.f;
          // probabilities of elements e0 .. e1 - 1 in 32 bits; the scores stay, in case the running maximum turns out too low
          float x[16];
          const auto weigh = [&](const f32x16_t& s, int e0, int e1) {
#pragma unroll
            for (int e = e0; e < e1; ++e) {
              x[e] = fast_exp2(__builtin_fmaf(s[e], c, -sub));
              sum += x[e];
              if (e & 1) {
                uint32_t* to = &(&p[e >> 3].x)[(e & 7) >> 1];
                *to = Op<T>::pack(x[e - 1], x[e]);
                asm volatile("" : "+v"(*to));
              }
            }
            asm volatile("" : "+v"(sum));  // (here, not where the values are wanted)
          };
          // No maximum is sought as long as no row's probabilities of a block add up to more than SUM and every row has a maximum: the sum
          // is needed anyway.  Otherwise: the maximum, and the block again (fp16, whose SUM is reached below 2^LAZY each, takes any new maximum:
          // the next blocks would come here again).
          const auto settle_max = [&](int k) {
            if (__ballot(!(sum <= Range<T>::SUM) || r.m == -INFINITY)) {
              f32x16_t one[1] = {sc[k]};
              r.raise(r.template largest<1>(one, c), Range<T>::LIFT > 0.f ? 0.f : Range<T>::LAZY);
              sub = r.m == -INFINITY ? 0.f : r.m;
              sum = 0.f;
              weigh(sc[k], 0, 16);
            }
            r.l += sum;
            sum = 0.f;
          };
#pragma unroll
          for (int e = 0; e < 16; ++e) sc[0][e] = sc[1][e] = 0.f;
#pragma unroll
          for (int n = 0; n < AHEAD; ++n) f[n] = key_operand(n);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int n = 0; n < NS; ++n) {
            sc[0] = Op<T>::mfma(f[n], r.q[n], sc[0]);
            if (n + AHEAD < 2 * NS) f[n + AHEAD] = key_operand(n + AHEAD);
            __builtin_amdgcn_sched_barrier(0);
          }
          if (edge) {
            f32x16_t one[1] = {sc[0]};
            r.template mask<1>(one, key0);
            if ((uint32_t)bad) r.template mask_bad<1>(one, (uint32_t)bad);
            sc[0] = one[0];
          }
#pragma unroll
          for (int n = 0; n < NS; ++n) {
            sc[1] = Op<T>::mfma(f[n + NS], r.q[n], sc[1]);
            if (n + NS + AHEAD < 2 * NS) f[n + NS + AHEAD] = key_operand(n + NS + AHEAD);
            weigh(sc[0], n * 16 / NS, (n + 1) * 16 / NS);
            __builtin_amdgcn_sched_barrier(0);
          }
          if (edge) {
            f32x16_t one[1] = {sc[1]};
            r.template mask<1>(one, key0 + 32);
            if (bad >> 32) r.template mask_bad<1>(one, bad >> 32);
            sc[1] = one[0];
          }
#pragma unroll
          for (int n = 0; n < AHEAD; ++n) f[n] = value_operand(n);
          settle_max(0);
          uint4 p0[2] = {p[0], p[1]};
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int n = 0; n < NS; ++n) {
            r.o[n % NO] = Op<T>::mfma(f[n], p0[n / NO], r.o[n % NO]);
            if (n + AHEAD < 2 * NS) f[n + AHEAD] = value_operand(n + AHEAD);
            weigh(sc[1], n * 16 / NS, (n + 1) * 16 / NS);
            __builtin_amdgcn_sched_barrier(0);
          }
          settle_max(1);
#pragma unroll
          for (int n = NS; n < 2 * NS; ++n) {
            r.o[n % NO] = Op<T>::mfma(f[n], p[n % NS / NO], r.o[n % NO]);
            if (n + AHEAD < 2 * NS) f[n + AHEAD] = value_operand(n + AHEAD);
            __builtin_amdgcn_sched_barrier(0);
          }
        }
        __builtin_amdgcn_s_setprio(0);
        if (more) {
          settle(next, buf ^ 1);
          __syncthreads();  // the next tile is in LDS, and this one's readers are done
        }
        now = next;
        next = after;
      }
    }
    r.finish();
    if (!split || (j0 == 0 && j1 == nt))
      r.write(a, F8 ? a.v_scale[hk] : 1.0f);
    else
      r.write_part(a, g * 2 + (first < u0 ? 0 : 1), TR, wave * 32 + (lane & 31));
    if (!split) return;
    __syncthreads();  // the next row tile fills the buffers anew
    u += j1 - j0;
  }
}

// ------------------------------------------------------------------------------------- joining shared row tiles
// A workgroup joins as many rows of a (row tile, key head) as its threads hold, D / 4 threads a row; blockIdx.y walks the tile's rows.  The
// launch is short and all latency: where the row tile lies comes in one trip to memory, up to eight shares of a row are loaded together.
// 10 shares of 96 tiles of 128 rows x 32 (17 MB): 6.7 us; 4 or 16 at a time 7.0 and 7.3, shares that are not there loaded all the same 8.4.
template <typename T, int D>
__global__ __launch_bounds__(TPB) void attn_join_kernel(const Args a, int tr, int tk) {
  constexpr int TPR = D / 4, RPB = TPB / TPR, AT = 8;
  const int64_t slot = blockIdx.x / a.hk;
  const int hk = blockIdx.x % a.hk;
  const int64_t each = a.units[a.seqs + 1];
  int b, cu0, cu1, len;
  int64_t base;
  if (a.seqs <= 64) {  // every sequence in a lane: one trip to memory instead of three
    const int lane = threadIdx.x & 63, at = min(lane, max(a.seqs - 1, 0));
    const int c0 = a.cu[at], c1 = a.cu[min(at + 1, a.seqs)], l = a.lens[at];
    const int64_t u = a.units[at];
    b = __popcll(__ballot(lane < a.seqs && slot_from(a, c1, lane + 1, tr) <= slot));
    if (b >= a.seqs) return;
    cu0 = __builtin_amdgcn_readlane(c0, b);
    cu1 = __builtin_amdgcn_readlane(c1, b);
    len = __builtin_amdgcn_readlane(l, b);
    base = (int64_t)__builtin_amdgcn_readlane((int)(u >> 32), b) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)u, b);
  } else {
    b = seq_of_slot(a, slot, tr);
    if (b >= a.seqs) return;
    cu0 = a.cu[b];
    cu1 = a.cu[b + 1];
    len = a.lens[b];
    base = a.units[b];
  }
  const Seq s = seq_from(a, cu0, cu1, len);
  const int64_t qt = slot - slot_from(a, cu0, b, tr);
  const int nq = row_tiles(a, s, tr), nt = key_tiles(a, s, tr, tk);
  if (qt < 0 || qt >= nq) return;
  const int64_t u0 = base + ((int64_t)hk * nq + qt) * nt, g0 = u0 / each, g1 = (u0 + nt - 1) / each;
  if (g0 == g1) return;  // one workgroup had it all and wrote it
  const int rows = (int)min((int64_t)tr, (int64_t)s.n * a.group - qt * tr), d4 = threadIdx.x % TPR, row = blockIdx.y * RPB + threadIdx.x / TPR;
  if (row >= rows) return;
  const float* ml = a.part + (int64_t)a.groups * 2 * tr * D;
  const float vs = a.v_scale ? a.v_scale[hk] : 1.0f;
  float m = -INFINITY, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int64_t g = g0; g <= g1; g += AT) {
    float2 x[AT];
    float4 v[AT];
    float up = m;
#pragma unroll
    for (int i = 0; i < AT; ++i) {  // workgroup gi's share of this row tile: its first one unless the tile begins inside gi's units
      const int64_t gi = g + i, at = (gi * 2 + (u0 < gi * each ? 0 : 1)) * tr + row;
      x[i] = make_float2(-INFINITY, 0.f);
      v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (gi > g1) continue;
      x[i] = *reinterpret_cast<const float2*>(ml + at * 2);
      v[i] = *reinterpret_cast<const float4*>(a.part + at * D + d4 * 4);
    }
#pragma unroll
    for (int i = 0; i < AT; ++i) up = fmaxf(up, x[i].x);
    const float f0 = m == -INFINITY ? 0.f : fast_exp2(m - up);
    l *= f0;
    o.x *= f0; o.y *= f0; o.z *= f0; o.w *= f0;
#pragma unroll
    for (int i = 0; i < AT; ++i) {
      const float f = x[i].x == -INFINITY ? 0.f : fast_exp2(x[i].x - up);
      l = __builtin_fmaf(x[i].y, f, l);
      o.x = __builtin_fmaf(v[i].x, f, o.x); o.y = __builtin_fmaf(v[i].y, f, o.y);
      o.z = __builtin_fmaf(v[i].z, f, o.z); o.w = __builtin_fmaf(v[i].w, f, o.w);
    }
    m = up;
  }
  const float f = l > 0.f ? vs / l : (l == 0.f ? 0.f : l);
  const int64_t r = qt * tr + row, tok = r / a.group, at = (s.row0 + tok) * a.hq + hk * a.group + (r - tok * a.group);
  *reinterpret_cast<uint2*>((uint16_t*)a.o + at * D + d4 * 4) = make_uint2(Op<T>::pack(o.x * f, o.y * f), Op<T>::pack(o.z * f, o.w * f));
  if (d4 == 0 && a.lse) a.lse[at] = l == 0.f ? -INFINITY : (m + __log2f(l)) * LN2;
}

// ------------------------------------------------------------------------------------- host
struct Plan {
  bool few, split;
  int tr, tk, groups;
  int64_t slots, ws;
};
constexpr int CUS = 256;

bool usable(const hma_attn_paged_t* p) {
  if (!p || (p->d != 32 && p->d != 64 && p->d != 128) || (p->dtype != HMA_BF16 && p->dtype != HMA_F16)) return false;
  if (p->hq < 1 || p->hk < 1 || p->hq > 4096 || p->hq % p->hk || p->tokens < 0 || p->tokens > 0x3fffffff / p->hq * 1LL) return false;
  if (p->seqs < 0 || p->seqs > 4096 || p->table_w < 0 || p->pages < 0 || p->page < 1 || p->window < 0 || (p->window > 0 && !p->causal)) return false;
  return p->scale > 0.f && p->scale < 3e38f;
}
// Rule: sequences with at most 32 rows (tokens x shared heads) on average take the kernel whose waves share the keys, others the one
// whose waves share the rows.  The latter is split along the keys only where its row tiles do not give every compute unit its workgroups
// twice over.
Plan plan_of(const hma_attn_paged_t* p) {
  Plan r;
  const int64_t group = p->hq / p->hk, rows = p->tokens * group;
  r.few = rows <= 32LL * p->seqs;
  const int kb = p->d == 128 && !p->cache_e4m3 ? 1 : 2;
  r.tr = r.few ? 32 : 128;
  r.tk = r.few ? WAVES * 32 * kb : 64;
  r.slots = rows / r.tr + p->seqs;
  // as many workgroups as are resident together (their registers and LDS), each with one share, and no more than there are units: row
  // tiles x key tiles of the longest sequence that the table can hold
  const int64_t room = CUS * (r.few ? (p->d == 32 ? 3 : 2) : p->d == 128 ? 2 : p->d == 64 ? 3 : 4);
  r.split = r.few || r.slots * p->hk < 2 * room;
  const int64_t most = ((int64_t)p->table_w * p->page + r.tk - 1) / r.tk;
  const int64_t units = r.slots * p->hk * (most > 0 ? most : 1);
  r.groups = (int)(units < room ? (units > 0 ? units : 1) : room);
  r.ws = r.split ? (int64_t)r.groups * 2 * r.tr * (p->d + 2) * 4 + (p->seqs + 2) * 8 : 0;
  return r;
}

// One attribute call per kernel and process and device: the most LDS that any call asks for
template <auto Kern>
int allow_lds() {
  static std::atomic<uint64_t> done{0};  // a bit per device
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) return HMA_EINVAL;
  const uint64_t bit = 1ull << (dev & 63);
  if (done.load(std::memory_order_relaxed) & bit) return 0;
  const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(Kern), hipFuncAttributeMaxDynamicSharedMemorySize, WAVES * 64 * (128 + PAD) * 2 + 4097 * 8);
  if (e != hipSuccess) return -(int)e;
  done.fetch_or(bit, std::memory_order_relaxed);
  return 0;
}

template <typename T, int D, bool F8, bool ALIGNED>
int launch(hipStream_t st, const Args& a, const Plan& r) {
  constexpr int KB = D == 128 && !F8 ? 1 : 2, LD = D + PAD;
  const size_t units = (size_t)(a.seqs + 1) * 8;
  if (r.few) {
    const size_t lds = (size_t)WAVES * 32 * KB * LD * 2 + units;
    if (const int rc = allow_lds<attn_few_kernel<T, D, F8, KB, ALIGNED>>()) return rc;
    hipLaunchKernelGGL((attn_few_kernel<T, D, F8, KB, ALIGNED>), dim3((unsigned)r.groups), dim3(TPB), lds, st, a);
  } else {
    const size_t lds = (size_t)4 * Lay<D>::TILE + (r.split ? units : 0);
    const dim3 grid((unsigned)(r.split ? r.groups : r.slots * a.hk));
    if (const int rc = allow_lds<attn_many_kernel<T, D, F8, ALIGNED>>()) return rc;
    hipLaunchKernelGGL((attn_many_kernel<T, D, F8, ALIGNED>), grid, dim3(TPB), lds, st, a, (int)r.split);
  }
  HMA_CHECK_LAUNCH();
  if (r.split && a.seqs > 0) {
    const int most = (int)std::min<int64_t>(r.tr, a.tokens * a.group), per = TPB / (D / 4);
    hipLaunchKernelGGL((attn_join_kernel<T, D>), dim3((unsigned)(r.slots * a.hk), (unsigned)((most + per - 1) / per)), dim3(TPB), 0, st, a, r.tr, r.tk);
    HMA_CHECK_LAUNCH();
  }
  return 0;
}
template <typename T, int D, bool F8>
int launch_a(hipStream_t st, const Args& a, const Plan& r) {
  constexpr int RPW = 64 / ((F8 ? D : 2 * D) / 16);  // rows of a wave's load (Loader)
  const bool fits = a.kc_tok * RPW < 0x40000000 && a.vc_tok * RPW < 0x40000000;
  return a.page % RPW == 0 && fits ? launch<T, D, F8, true>(st, a, r) : launch<T, D, F8, false>(st, a, r);
}
template <typename T, int D>
int launch_f8(hipStream_t st, const Args& a, const Plan& r, bool e) {
  return e ? launch_a<T, D, true>(st, a, r) : launch_a<T, D, false>(st, a, r);
}
template <typename T>
int launch_d(hipStream_t st, const Args& a, const Plan& r, bool e, int d) {
  return d == 128 ? launch_f8<T, 128>(st, a, r, e) : d == 64 ? launch_f8<T, 64>(st, a, r, e) : launch_f8<T, 32>(st, a, r, e);
}

}  // namespace

extern "C" int hma_attn_paged_ws(const hma_attn_paged_t* p, int64_t* bytes) {
  if (!usable(p) || !bytes) return HMA_EINVAL;
  *bytes = plan_of(p).ws;
  return 0;
}

extern "C" int hma_attn_paged_fwd(void* stream, const hma_attn_paged_t* p) {
  if (!usable(p)) return HMA_EINVAL;
  if (p->tokens == 0) return 0;
  const bool e = p->cache_e4m3 != 0;
  if (!p->q || !p->o || ((uintptr_t)p->q & 15) || ((uintptr_t)p->o & 15) || p->q_tok < 0 || p->q_head < 0 || (p->q_tok & 7) || (p->q_head & 7)) return HMA_EINVAL;
  if (!p->cu || (p->seqs > 0 && (!p->lens || (p->table_w > 0 && !p->table))) || (e && (!p->k_scale || !p->v_scale))) return HMA_EINVAL;
  Args a = {};
  const int64_t es = e ? 1 : 2, st[6] = {p->kc_page, p->kc_head, p->kc_tok, p->vc_page, p->vc_head, p->vc_tok};
  if (p->pages > 0) {
    for (int i = 0; i < 6; ++i)
      if (st[i] < 0 || ((st[i] * es) & 15)) return HMA_EINVAL;
    if (!p->kc || !p->vc || ((uintptr_t)p->kc & 15) || ((uintptr_t)p->vc & 15)) return HMA_EINVAL;
  }
  const Plan r = plan_of(p);
  if (r.split && (!p->ws || ((uintptr_t)p->ws & 15) || p->ws_bytes < r.ws)) return HMA_EINVAL;
  if (r.slots * p->hk > 0x7fffffff) return HMA_EINVAL;
  a.q = p->q; a.o = p->o; a.lse = p->lse; a.kc = (const uint8_t*)p->kc; a.vc = (const uint8_t*)p->vc;
  a.table = p->table; a.cu = p->cu; a.lens = p->lens;
  a.k_scale = e ? p->k_scale : nullptr;
  a.v_scale = e ? p->v_scale : nullptr;
  a.tokens = p->tokens; a.q_tok = p->q_tok; a.q_head = p->q_head; a.table_stride = p->table_stride;
  a.kc_page = st[0] * es; a.kc_head = st[1] * es; a.kc_tok = st[2] * es; a.vc_page = st[3] * es; a.vc_head = st[4] * es; a.vc_tok = st[5] * es;
  // key / page = (key * page_mul) >> (31 + page_shift) for every key < 2^31: page_mul = ceil(2^(31 + s) / page), 2^s >= page
  while ((1LL << a.page_shift) < p->page) ++a.page_shift;
  a.page_mul = (uint32_t)(((1ULL << (31 + a.page_shift)) + p->page - 1) / p->page);
  a.hq = p->hq; a.hk = p->hk; a.group = p->hq / p->hk; a.seqs = p->seqs; a.table_w = p->table_w; a.pages = p->pages; a.page = p->page;
  a.causal = p->causal; a.window = p->window; a.zero_tail = p->zero_tail; a.groups = r.groups; a.scale = p->scale;
  a.part = (float*)p->ws;
  a.units = r.split ? (int64_t*)((uint8_t*)p->ws + (int64_t)r.groups * 2 * r.tr * (p->d + 2) * 4) : nullptr;
  return p->dtype == HMA_BF16 ? launch_d<__bf16>((hipStream_t)stream, a, r, e, p->d) : launch_d<_Float16>((hipStream_t)stream, a, r, e, p->d);
}
