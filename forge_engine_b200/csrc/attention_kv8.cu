// Causal grouped-query attention over the 8-bit cache (layout: kv8.cuh), compiled for one head size:
// -DFE_HEAD_DIM=<multiple of 16, 16..256>.  Single tokens of every head size and portions of head sizes other than 64
// and 128, which attention_kv8_portion.cu takes.
//
// A query at position i of a sequence sees the keys j <= i, or with a window those of the last `window`
// positions and the first `keep_first`.  With cached key code c_j, value code d_j and their scales 2^a_j, 2^b_j:
//
//   t_j = scale * log2(e) * (q . c_j) 2^a_j            out = sum_j 2^(t_j) 2^b_j d_j / sum_j 2^(t_j)
//
// Neither matrix is ever scaled element by element: 2^a_j is a factor of a finished score, and 2^b_j joins the
// exponent, u_j = t_j + b_j.  The running maximum M is that of u_j, the largest contribution to the output, so
// the weights 2^(u_j - M) of the value product lie in [0, 1] whatever the scales are, and the codes go into the
// tensor cores as the half-precision numbers they exactly are (one conversion instruction for two codes).  The
// denominator sums 2^(t_j - M) = 2^(u_j - M) 2^(-b_j) in 32 bits (small scales: see denominator_term).  Weights are rounded to half precision (11
// bits; what is below 2^-25 of the largest contribution vanishes).  A query row is scaled by a power of two so
// that its largest element lies in [2^14, 2^15): bfloat16's 8 bits stay whole down to 2^-31 of that.
//
// Upstream's counterparts read pages of the model's type: the eager attention of
// src/forge_engine/qwen3.py:187-206 and the decode kernel of src/forge_engine/kernels/cuda_paged.py:276-347.
#include <cuda_fp16.h>

#include <type_traits>

#include "attention_kv8.cuh"

#define CAT_(a, b) a##b
#define CAT(a, b) CAT_(a, b)
#define SYM(name) CAT(name, FE_HEAD_DIM)

using namespace kv8;

namespace {

constexpr int CHUNKS = D / 16;          // 16-byte pieces of a cached vector
constexpr int KEYS = 128;               // keys of a tile
constexpr int STEP = 32;                // keys a warp takes at a time
constexpr int ROWS = 16;                // rows a warp takes: the m of one mma
constexpr int WARPS = 4, THREADS = 32 * WARPS;
constexpr int STAGES = 2;
constexpr int MATRIX = STEP * D;        // bytes of one matrix of a stage
constexpr int STAGE = 2 * MATRIX + STEP * 16;      // codes, then of every key: 2^a, b, 2^-b
constexpr size_t RING = (size_t)WARPS * STAGES * STAGE;
constexpr size_t JOIN = (size_t)WARPS * ROWS * (D + 2) * sizeof(float);
constexpr size_t MMA_SMEM = RING > JOIN ? RING : JOIN;

__device__ __forceinline__ unsigned smem_addr(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void cp_async16(void* dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(smem_addr(dst)), "l"(src), "r"(valid ? 16 : 0));
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;\n" ::); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;\n" ::"n"(N)); }
__device__ __forceinline__ void mma_f16(float (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float exp2_fast(float x) {       // the weight is rounded to 11 bits anyway
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// What a key adds to the sum that divides: 2^(t - M) = w 2^(-b), with w = 2^(u - M) at hand and `back` 2^(-b).  But w is zero below
// 2^-126, and a value of zeros, whose b is the least, beside one with a b of 63 would not count at all.  So a warp that
// met a scale below 2^-32 walks its keys once more with SMALL, where that exponential is taken by itself and `back` is b.
// (Above it w vanishes only where t is 30 below that of the largest contribution, whose M is at most that t + 64.)
constexpr int SMALL_SCALE = KV8_BIAS - 32;
template <bool SMALL> __device__ __forceinline__ float denominator_term(float u, float base, float w, float back, float sum) {
  return SMALL ? sum + exp2_fast(u - base - back) : fmaf(w, back, sum);
}
// What sums with maximum `from` are worth with maximum `to`.  With SMALL the root of it: a sum may then be 2^64 of its weights
// and the maxima of keys that count alike 2^128 apart, so it goes its way in two halves.
template <bool SMALL> __device__ __forceinline__ float worth(float from, float to) {
  return from == -INFINITY ? 0.f : exp2f(SMALL ? 0.5f * (from - to) : from - to);
}
__device__ __forceinline__ unsigned pack_half(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const unsigned*>(&h);
}

// Where 16-byte piece c of row r lies.  Keys are read 8 rows x 4 pieces at a time (rows two by two in a phase
// of a shared-memory read), values the rows 2t, 2t + 1, 2t + 8, 2t + 9 x pieces of 8 lanes: each matrix has the
// exchange of pieces that keeps its reads apart.  Head sizes without a whole power of two of pieces take none.
__device__ __forceinline__ int key_piece(int r, int c) { return D % 128 == 0 ? c ^ ((r & 1) << 2) : c; }
__device__ __forceinline__ int value_piece(int r, int c) {
  return D % 128 == 0 ? c ^ (((r >> 1) & 3) << 1) : D % 64 == 0 ? c ^ ((r >> 1) & 3) : c;
}

// The queries of a warp's 16 rows as the A operand.  The order of the contraction is free as long as both
// operands keep it: in every stretch of 64 elements lane t of a quad holds elements 16 t .. 16 t + 15, which it
// reads of a key as one 16-byte piece; stretches of 32 and 16 at the end go by 8 and 4 elements.
struct Queries {
  unsigned a[D / 16][4];
  float factor[2];                 // what a product of row g / g + 8 is multiplied by to be a score in log2 units

  static __device__ __forceinline__ int element(int step, int t) {      // first of the lane's four elements of a k step
    constexpr int whole = D / 64 * 4;
    if (step < whole) return (step >> 2) * 64 + 16 * t + 4 * (step & 3);
    int base = D / 64 * 64, s = step - whole;
    if (D & 32) {
      if (s < 2) return base + 8 * t + 4 * s;
      base += 32;
    }
    return base + 4 * t;
  }

  __device__ __forceinline__ void load(const Kv8Attention& p, const Entry& e, int kvh, int row0, int rows_end, int lane) {
    const int t = lane & 3;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = row0 + (lane >> 2) + 8 * h;
      float x[D / 4];
      unsigned big = 0u;
#pragma unroll
      for (int i = 0; i < D / 4; ++i) x[i] = 0.f;
      if (row < rows_end) {
        const int token = row / p.groups, g = row - token * p.groups;
        const bf16* src = p.q + (size_t)(e.tok0 + token) * p.q_stride + (size_t)(kvh * p.groups + g) * D;
#pragma unroll
        for (int s = 0; s < D / 16; ++s) load4(src + element(s, t), x + 4 * s);
      }
#pragma unroll
      for (int i = 0; i < D / 4; ++i) big = max(big, __float_as_uint(x[i]) & 0x7fffffffu);
      big = max(big, __shfl_xor_sync(0xffffffffu, big, 1));
      big = max(big, __shfl_xor_sync(0xffffffffu, big, 2));
      const bool finite = big < 0x7f800000u;                     // a row that is not gives NaN, also where every score is minus infinity
      int e2 = (int)(big >> 23) - 127 - 14;                      // 2^e2 is taken out of the row
      e2 = big == 0u || !finite ? 0 : max(e2, -100);
      const float down = __int_as_float((127 - e2) << 23);
      factor[h] = finite ? p.scale_log2 * __int_as_float((127 + e2) << 23) : kv8_scale(KV8_NAN);
#pragma unroll
      for (int s = 0; s < D / 16; ++s) {
        a[s][h] = pack_half(x[4 * s] * down, x[4 * s + 1] * down);
        a[s][h + 2] = pack_half(x[4 * s + 2] * down, x[4 * s + 3] * down);
      }
    }
  }
};

// Running maximum, sum and value sums of a warp's 16 rows; lane (g, t) holds rows g and g + 8.  Value columns
// are taken in stretches of 128, 64, 32 and 16: in one of 8 W columns lane g of the B operand holds columns
// W g .. W g + W - 1, which are one read of W bytes of a value, and W products cover the stretch.
struct Sums {
  float m[2], l[2];
  float o[D / 8][4];
  __device__ __forceinline__ void clear() {
    m[0] = m[1] = -INFINITY;
    l[0] = l[1] = 0.f;
#pragma unroll
    for (int n = 0; n < D / 8; ++n) { o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f; }
  }
};

template <int W> struct Piece;
template <> struct Piece<16> { typedef uint4 type; };
template <> struct Piece<8> { typedef uint2 type; };
template <> struct Piece<4> { typedef unsigned type; };
template <> struct Piece<2> { typedef unsigned short type; };

// Value columns [BASE, BASE + 8 W): o += weights x values, 16 keys.
template <int BASE, int W>
__device__ __forceinline__ void value_stretch(const unsigned char* vs, int k0, const unsigned (&a)[4], float (&o)[D / 8][4], int lane) {
  const int g = lane >> 2, t = lane & 3;
  constexpr int WORDS = W < 4 ? 1 : W / 4;
  unsigned w[4][WORDS];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = k0 + 2 * t + (i & 1) + 8 * (i >> 1), byte = BASE + W * g;
    const typename Piece<W>::type x =
        *reinterpret_cast<const typename Piece<W>::type*>(vs + row * D + value_piece(row, byte >> 4) * 16 + (byte & 15));
    if constexpr (W == 16) { w[i][0] = x.x; w[i][1] = x.y; w[i][2] = x.z; w[i][3] = x.w; }
    else if constexpr (W == 8) { w[i][0] = x.x; w[i][1] = x.y; }
    else w[i][0] = x;
  }
#pragma unroll
  for (int c = 0; c < WORDS; ++c) {
    // bytes of two rows side by side: (row 2t column j, row 2t + 1 column j), ...
    const unsigned lo0 = __byte_perm(w[0][c], w[1][c], 0x5140), lo1 = __byte_perm(w[0][c], w[1][c], 0x7362);
    const unsigned hi0 = __byte_perm(w[2][c], w[3][c], 0x5140), hi1 = __byte_perm(w[2][c], w[3][c], 0x7362);
    constexpr int N0 = BASE / 8;
    unsigned b0[4], b1[4];
    kv8_halves(lo0, b0[0], b0[1]);
    kv8_halves(hi0, b1[0], b1[1]);
    mma_f16(o[N0 + 4 * c], a, b0[0], b1[0]);
    mma_f16(o[N0 + 4 * c + 1], a, b0[1], b1[1]);
    if constexpr (W > 2) {
      kv8_halves(lo1, b0[2], b0[3]);
      kv8_halves(hi1, b1[2], b1[3]);
      mma_f16(o[N0 + 4 * c + 2], a, b0[2], b1[2]);
      mma_f16(o[N0 + 4 * c + 3], a, b0[3], b1[3]);
    }
  }
}

// Column of element (n-tile, c) of Sums::o for quad lane t: n-tile BASE/8 + j holds columns W (2 t + c) + j.
__device__ __forceinline__ int value_column(int n, int c, int t) {
  int base = 0, left = D;
  if (n * 8 < D / 128 * 128) { base = n / 16 * 128; return base + 16 * (2 * t + c) + (n & 15); }
  base = D / 128 * 128; left = D - base;
  if (left & 64) { if (n * 8 < base + 64) return base + 8 * (2 * t + c) + (n * 8 - base) / 8; base += 64; }
  if (left & 32) { if (n * 8 < base + 32) return base + 4 * (2 * t + c) + (n * 8 - base) / 8; base += 32; }
  return base + 2 * (2 * t + c) + (n * 8 - base) / 8;
}

// The 32 keys of a stage, at positions from key0 on, against a warp's 16 rows.
template <bool SMALL>
__device__ __forceinline__ void take(const Queries& q, const unsigned char* stage, int key0, const Kv8Attention& p, bool clear,
                                     int pos_a, int pos_b, Sums& s, int lane) {
  const int g = lane >> 2, t = lane & 3;
  const float4* of_key = reinterpret_cast<const float4*>(stage + 2 * MATRIX);
  float c[STEP / 8][4];
  float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
  for (int n = 0; n < STEP / 8; ++n) {
    c[n][0] = c[n][1] = c[n][2] = c[n][3] = 0.f;
    const int row = 8 * n + g;
    unsigned w[D / 16];
#pragma unroll
    for (int b = 0; b < D / 64; ++b) {
      const uint4 x = *reinterpret_cast<const uint4*>(stage + row * D + key_piece(row, 4 * b + t) * 16);
      w[4 * b] = x.x; w[4 * b + 1] = x.y; w[4 * b + 2] = x.z; w[4 * b + 3] = x.w;
    }
    if constexpr ((D & 32) != 0) {
      const uint2 x = *reinterpret_cast<const uint2*>(stage + row * D + D / 64 * 64 + 8 * t);
      w[D / 64 * 4] = x.x; w[D / 64 * 4 + 1] = x.y;
    }
    if constexpr ((D & 16) != 0) w[D / 16 - 1] = *reinterpret_cast<const unsigned*>(stage + row * D + D - 16 + 4 * t);
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      unsigned b0, b1;
      kv8_halves(w[i], b0, b1);
      mma_f16(c[n], q.a[i], b0, b1);
    }
    // keys 8 n + 2 t and the next one
    const float4 k0 = of_key[8 * n + 2 * t], k1 = of_key[8 * n + 2 * t + 1];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      c[n][2 * h] = fmaf(c[n][2 * h] * k0.x, q.factor[h], k0.y);
      c[n][2 * h + 1] = fmaf(c[n][2 * h + 1] * k1.x, q.factor[h], k1.y);
    }
    if (!clear) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int key = key0 + 8 * n + 2 * t + (e & 1), pos = e < 2 ? pos_a : pos_b;
        const bool seen = key <= pos && (p.window <= 0 || pos - key < p.window || key < p.keep_first);
        if (!seen) c[n][e] = -INFINITY;
      }
    }
    mx[0] = fmaxf(mx[0], fmaxf(c[n][0], c[n][1]));
    mx[1] = fmaxf(mx[1], fmaxf(c[n][2], c[n][3]));
  }
  float corr[2], base[2], sum[2] = {0.f, 0.f};
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
    mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
    const float now = fmaxf(s.m[h], mx[h]);
    corr[h] = worth<SMALL>(s.m[h], now);
    s.m[h] = now;
    base[h] = now == -INFINITY ? 0.f : now;
  }
  if (__any_sync(0xffffffffu, corr[0] != 1.f || corr[1] != 1.f)) {
    const float by[2] = {SMALL ? corr[0] * corr[0] : corr[0], SMALL ? corr[1] * corr[1] : corr[1]};
#pragma unroll
    for (int n = 0; n < D / 8; ++n) { s.o[n][0] *= by[0]; s.o[n][1] *= by[0]; s.o[n][2] *= by[1]; s.o[n][3] *= by[1]; }
  }
#pragma unroll
  for (int k = 0; k < STEP / 16; ++k) {
    unsigned a[4];
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const float4 k0 = of_key[16 * k + 8 * n + 2 * t], k1 = of_key[16 * k + 8 * n + 2 * t + 1];
      const float2 back = make_float2(SMALL ? k0.y : k0.z, SMALL ? k1.y : k1.z);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float u0 = c[2 * k + n][2 * h], u1 = c[2 * k + n][2 * h + 1];
        const float w0 = exp2_fast(u0 - base[h]), w1 = exp2_fast(u1 - base[h]);
        sum[h] = denominator_term<SMALL>(u0, base[h], w0, back.x, denominator_term<SMALL>(u1, base[h], w1, back.y, sum[h]));
        a[2 * n + h] = pack_half(w0, w1);
      }
    }
    const unsigned char* vs = stage + MATRIX;
    value_stretch<0, D >= 128 ? 16 : D >= 64 ? 8 : D >= 32 ? 4 : 2>(vs, 16 * k, a, s.o, lane);
    if constexpr (D == 256) value_stretch<128, 16>(vs, 16 * k, a, s.o, lane);
    if constexpr (D > 128 && D < 256 && (D & 64) != 0) value_stretch<128, 8>(vs, 16 * k, a, s.o, lane);
    if constexpr (D > 64 && (D & 32) != 0) value_stretch<D / 64 * 64, 4>(vs, 16 * k, a, s.o, lane);
    if constexpr (D > 16 && (D & 16) != 0) value_stretch<D / 32 * 32, 2>(vs, 16 * k, a, s.o, lane);
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) s.l[h] = (SMALL ? s.l[h] * corr[h] : s.l[h]) * corr[h] + sum[h];       // this lane's keys; the quad's sums join at the end
}

// The codes of a step's 32 keys and values; lane l knows the row of key l in its cache (-1: none, zeros).  ALL: every key
// has one.
template <bool ALL>
__device__ __forceinline__ void copy_step(const Kv8Attention& p, unsigned char* stage, int mine, int lane) {
  if constexpr (32 % CHUNKS == 0) {
    // a lane's pieces lie STRIDE rows apart; their places in the stage differ by a constant, in the values' exchange of
    // pieces by a constant bit pattern
    constexpr int STRIDE = 32 / CHUNKS;
    const int row0 = lane / CHUNKS, c = lane % CHUNKS;
    const unsigned char* k = p.k + c * 16;
    const unsigned char* v = p.v + c * 16;
    const unsigned kd = smem_addr(stage) + row0 * D + key_piece(row0, c) * 16, vd = smem_addr(stage) + MATRIX + row0 * D + value_piece(row0, c) * 16;
#pragma unroll
    for (int j = 0; j < CHUNKS; ++j) {
      const int from = __shfl_sync(0xffffffffu, mine, row0 + STRIDE * j);
      const size_t offset = (size_t)(unsigned)(ALL ? from : max(from, 0)) * D;
      const unsigned turn = D % 128 == 0 ? (unsigned)((j * STRIDE / 2) & 3) << 5 : D % 64 == 0 ? (unsigned)((j * STRIDE / 2) & 3) << 4 : 0u;
      const int bytes = ALL || from >= 0 ? 16 : 0;
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(kd + j * STRIDE * D), "l"(k + offset), "r"(bytes));
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"((vd ^ turn) + j * STRIDE * D), "l"(v + offset), "r"(bytes));
    }
  } else {
#pragma unroll
    for (int j = 0; j < CHUNKS; ++j) {
      const int u = lane + 32 * j, row = u / CHUNKS, c = u - row * CHUNKS;
      const int from = __shfl_sync(0xffffffffu, mine, row);
      const size_t offset = (size_t)max(from, 0) * D + c * 16;
      cp_async16(stage + row * D + key_piece(row, c) * 16, p.k + offset, from >= 0);
      cp_async16(stage + MATRIX + row * D + value_piece(row, c) * 16, p.v + offset, from >= 0);
    }
  }
}

// A warp goes its own way through its keys: it copies them into a ring of its own, a step ahead, and waits for nobody (with
// a ring of the block and a barrier a tile, 64 keys of one head took 1.7 us a block whatever else ran).  A lane looks after
// one key of a step: its page, looked up two steps ahead, its place and its scales, asked for with the codes.
struct WarpRing {
  unsigned char* ring;
  const Kv8Attention& p;
  const int* table;
  int kvh, key_lo, key_end, lane, page, k_scale, v_scale;
  int least_scale;                   // of the lane's values so far
  __device__ __forceinline__ WarpRing(unsigned char* ring, const Kv8Attention& p, const int* table, int kvh, int key_lo, int key_end, int lane)
      : ring(ring), p(p), table(table), kvh(kvh), key_lo(key_lo), key_end(key_end), lane(lane), page(-1), k_scale(KV8_BIAS), v_scale(KV8_BIAS),
        least_scale(KV8_BIAS) {}
  __device__ __forceinline__ unsigned char* stage(int i) const { return ring + (i & 1) * STAGE; }
  __device__ __forceinline__ void look_up(int key0) { page = key_page(p, table, key0 + lane, key_end); }
  // The scales of step i, asked for with its codes.  A key whose value is not finite counts as not finite itself.
  __device__ __forceinline__ void put_scales(int i) {
    const bool bad = v_scale == KV8_NAN;
    least_scale = min(least_scale, v_scale);
    reinterpret_cast<float4*>(stage(i) + 2 * MATRIX)[lane] =
        make_float4(kv8_scale(bad ? KV8_NAN : k_scale), bad ? 0.f : (float)(v_scale - KV8_BIAS),
                    bad ? 1.f : __int_as_float((2 * KV8_BIAS - v_scale) << 23), 0.f);
  }
  // Ask for the codes and scales of step i, at positions from key0 on, and for the pages of the one after it.
  __device__ __forceinline__ void ask(int i, int key0, int next_key0) {
    const int key = key0 + lane;
    long long at;
    const bool there = key_row(p, page, kvh, key, &at);
    if (!there) tell_missing(p, key, key_lo, key_end);
    k_scale = v_scale = KV8_BIAS;
    if (there) {
      k_scale = __ldg(p.ks + at);
      v_scale = __ldg(p.vs + at);
    }
    look_up(next_key0);
    const int row = there ? (int)at : -1;             // the launcher holds the rows of a cache to 31 bits
    if (__all_sync(0xffffffffu, there)) copy_step<true>(p, stage(i), row, lane);
    else copy_step<false>(p, stage(i), row, lane);
  }
};

// ---- up to eight rows, head sizes of whole 32s ----
//
// Keys stand on the side of 16 of a product and the rows on the side of 8, so a GQA group of up to eight heads wastes
// nothing.  (Two eights of rows did not fit a thread's registers: 235 us for 48 windows of 15 rows, where the kernel of
// 16 rows takes 87.)  Scores are products of 8-bit numbers, the codes as they lie in shared memory against two e4m3
// numbers of a query element: a row times a power of two, rounded, and what the rounding left.  They hold bfloat16's 8
// bits down to 2^-11 of the row's largest element and what is smaller to within 2^-18 of it; the tensor core sums them
// to within 6e-8 of the sum of magnitudes.  Values go in as half-precision numbers, 16 of their elements on the side of
// 16, so an output comes out transposed too.  One sequence of 32768 keys, 32 heads on 8: 25.9 us, where 16 rows a
// product took 28.1; eight of 2048: 16.0 and 17.8 (21.6 and 14.3 since the cuts and launches below).  32 sequences of
// up to 8192 keys: 61 to 65 us, 0.70 of the copy peak; instructions issue in 47 % of the cycles, three warps a scheduler
// (registers and rings allow 12 an SM) wait for one another's latencies, not for memory.
struct RowQueries {
  unsigned b[2][D / 16];             // [part][four codes]
  float factor[2];                   // of rows 2t, 2t + 1: what a product is multiplied by to be a score in log2 units
  __device__ __forceinline__ void load(const Kv8Attention& p, const Entry& e, int kvh, int rows, int lane) {
    const int g = lane >> 2, t = lane & 3;
    float x[D / 4];
    unsigned big = 0u;
#pragma unroll
    for (int i = 0; i < D / 4; ++i) x[i] = 0.f;
    if (g < rows) {
      const int token = g / p.groups, head = g - token * p.groups;
      const bf16* src = p.q + (size_t)(e.tok0 + token) * p.q_stride + (size_t)(kvh * p.groups + head) * D;
#pragma unroll
      for (int s = 0; s < D / 16; ++s) load4(src + Queries::element(s, t), x + 4 * s);
    }
#pragma unroll
    for (int i = 0; i < D / 4; ++i) big = max(big, __float_as_uint(x[i]) & 0x7fffffffu);
    big = max(big, __shfl_xor_sync(0xffffffffu, big, 1));
    big = max(big, __shfl_xor_sync(0xffffffffu, big, 2));
    const bool finite = big < 0x7f800000u;
    const int ex = finite ? kv8_row_exponent(big) : 0;
    const float down = __int_as_float((127 - ex) << 23);
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
      unsigned word[2] = {0u, 0u};
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const __half2 v = __floats2half2_rn(x[4 * s + 2 * k] * down, x[4 * s + 2 * k + 1] * down);
        const unsigned hi = kv8_codes_of_half2(v), back = kv8_half2((unsigned short)hi);
        word[0] |= hi << (16 * k);
        word[1] |= kv8_codes_of_half2(__hsub2(v, *reinterpret_cast<const __half2*>(&back))) << (16 * k);
      }
      b[0][s] = word[0];
      b[1][s] = word[1];
    }
    const float up = finite ? p.scale_log2 * __int_as_float((127 + ex) << 23) : kv8_scale(KV8_NAN);
    factor[0] = __shfl_sync(0xffffffffu, up, 8 * t);             // row 2t lies with lanes 4 * 2t ..
    factor[1] = __shfl_sync(0xffffffffu, up, 8 * t + 4);
  }
};

__device__ __forceinline__ void mma_e4m3(float (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// A fragment of 8 x 8 half-precision numbers, transposed
__device__ __forceinline__ unsigned transposed(unsigned x) {
  unsigned y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

struct RowSums {
  float m[2], l[2];                  // rows 2t, 2t + 1; l: of this lane's keys
  float o[D / 16][4];                // m-tile i: elements (first, row 2t), (first, row 2t + 1), (second, ..), (second, ..)
};

// Value elements [BASE, BASE + 8 W): m-tile BASE/16 + 2c + h holds elements W g + 4 c + 2 h and the next one.
template <int BASE, int W>
__device__ __forceinline__ void row_values(const unsigned char* vs, int k0, const unsigned (&b)[2], RowSums& s, int lane) {
  const int g = lane >> 2, t = lane & 3;
  unsigned w[4][W / 4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = k0 + 2 * t + (i & 1) + 8 * (i >> 1), byte = BASE + W * g;
    const typename Piece<W>::type x = *reinterpret_cast<const typename Piece<W>::type*>(vs + row * D + value_piece(row, byte >> 4) * 16 + (byte & 15));
    if constexpr (W == 16) { w[i][0] = x.x; w[i][1] = x.y; w[i][2] = x.z; w[i][3] = x.w; }
    else if constexpr (W == 8) { w[i][0] = x.x; w[i][1] = x.y; }
    else w[i][0] = x;
  }
#pragma unroll
  for (int c = 0; c < W / 4; ++c) {
    unsigned a[2][4];
    kv8_halves(__byte_perm(w[0][c], w[1][c], 0x5140), a[0][0], a[0][1]);
    kv8_halves(__byte_perm(w[2][c], w[3][c], 0x5140), a[0][2], a[0][3]);
    kv8_halves(__byte_perm(w[0][c], w[1][c], 0x7362), a[1][0], a[1][1]);
    kv8_halves(__byte_perm(w[2][c], w[3][c], 0x7362), a[1][2], a[1][3]);
    mma_f16(s.o[BASE / 16 + 2 * c], a[0], b[0], b[1]);
    mma_f16(s.o[BASE / 16 + 2 * c + 1], a[1], b[0], b[1]);
  }
}

// The 32 keys of a stage against eight rows.
template <bool SMALL>
__device__ __forceinline__ void take_rows(const RowQueries& q, const unsigned char* stage, int key0, const Kv8Attention& p, bool clear,
                                          const int (&pos)[2], RowSums& s, int lane) {
  const int g = lane >> 2, t = lane & 3;
  const float4* of_key = reinterpret_cast<const float4*>(stage + 2 * MATRIX);
  float u[2][4];                     // [16 keys][(g, 2t), (g, 2t + 1), (g + 8, ..), (g + 8, ..)]
  float back[2][2], mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    unsigned w[2][D / 16];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = 16 * j + 8 * h + g;
#pragma unroll
      for (int b = 0; b < D / 64; ++b) {
        const uint4 x = *reinterpret_cast<const uint4*>(stage + row * D + key_piece(row, 4 * b + t) * 16);
        w[h][4 * b] = x.x; w[h][4 * b + 1] = x.y; w[h][4 * b + 2] = x.z; w[h][4 * b + 3] = x.w;
      }
      if constexpr ((D & 32) != 0) {
        const uint2 x = *reinterpret_cast<const uint2*>(stage + row * D + D / 64 * 64 + 8 * t);
        w[h][D / 64 * 4] = x.x; w[h][D / 64 * 4 + 1] = x.y;
      }
    }
    float c[2][4];
#pragma unroll
    for (int part = 0; part < 2; ++part) c[part][0] = c[part][1] = c[part][2] = c[part][3] = 0.f;
#pragma unroll
    for (int k = 0; k < D / 32; ++k) {
      const unsigned a[4] = {w[0][2 * k], w[1][2 * k], w[0][2 * k + 1], w[1][2 * k + 1]};
#pragma unroll
      for (int part = 0; part < 2; ++part) mma_e4m3(c[part], a, q.b[part][2 * k], q.b[part][2 * k + 1]);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float4 of = of_key[16 * j + 8 * h + g];
      back[j][h] = SMALL ? of.y : of.z;
      const int key = key0 + 16 * j + 8 * h + g;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float x = fmaf((c[0][2 * h + i] + c[1][2 * h + i]) * of.x, q.factor[i], of.y);
        if (!clear) {
          const bool seen = key <= pos[i] && (p.window <= 0 || pos[i] - key < p.window || key < p.keep_first);
          if (!seen) x = -INFINITY;
        }
        u[j][2 * h + i] = x;
        mx[i] = fmaxf(mx[i], x);
      }
    }
  }
  float corr[2], base[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], o));
    const float now = fmaxf(s.m[i], mx[i]);
    corr[i] = worth<SMALL>(s.m[i], now);
    s.m[i] = now;
    base[i] = now == -INFINITY ? 0.f : now;
  }
  if (__any_sync(0xffffffffu, corr[0] != 1.f || corr[1] != 1.f)) {
    const float by[2] = {SMALL ? corr[0] * corr[0] : corr[0], SMALL ? corr[1] * corr[1] : corr[1]};
    s.l[0] = (SMALL ? s.l[0] * corr[0] : s.l[0]) * corr[0];
    s.l[1] = (SMALL ? s.l[1] * corr[1] : s.l[1]) * corr[1];
#pragma unroll
    for (int d = 0; d < D / 16; ++d) { s.o[d][0] *= by[0]; s.o[d][1] *= by[1]; s.o[d][2] *= by[0]; s.o[d][3] *= by[1]; }
  }
  const unsigned char* vs = stage + MATRIX;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    unsigned b[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float w0 = exp2_fast(u[j][2 * h] - base[0]), w1 = exp2_fast(u[j][2 * h + 1] - base[1]);
      s.l[0] = denominator_term<SMALL>(u[j][2 * h], base[0], w0, back[j][h], s.l[0]);
      s.l[1] = denominator_term<SMALL>(u[j][2 * h + 1], base[1], w1, back[j][h], s.l[1]);
      b[h] = transposed(pack_half(w0, w1));
    }
    row_values<0, D >= 128 ? 16 : D >= 64 ? 8 : 4>(vs, 16 * j, b, s, lane);
    if constexpr (D == 256) row_values<128, 16>(vs, 16 * j, b, s, lane);
    if constexpr (D > 128 && D < 256 && (D & 64) != 0) row_values<128, 8>(vs, 16 * j, b, s, lane);
    if constexpr (D > 64 && (D & 32) != 0) row_values<D / 64 * 64, 4>(vs, 16 * j, b, s, lane);
  }
}

// First element of m-tile i (even i: four neighbouring ones, of m-tiles i and i + 1) for lane g.
__device__ __forceinline__ int row_element(int i, int g) {
  const int e0 = i * 16;
  if (e0 < D / 128 * 128) return e0 / 128 * 128 + 16 * g + (i % 8) * 2;
  int base = D / 128 * 128;
  if ((D - base) & 64) {
    if (e0 < base + 64) return base + 8 * g + (e0 - base) / 16 * 2;
    base += 64;
  }
  return base + 4 * g + (e0 - base) / 16 * 2;
}

// What the warps of a block (their maxima, sums and value sums in `acc` and `ml`) make of its rows: the output, or a piece.
__device__ __forceinline__ void finish_rows(const Kv8Attention& p, const Entry& e, int kvh, int n_rows, int pieces, const float* acc,
                                            const float* ml, float* ws) {
#pragma unroll 1
  for (int i = threadIdx.x; i < n_rows * (D / 4); i += THREADS) {
    const int r = i / (D / 4), d = (i - r * (D / 4)) * 4;
    float big = -INFINITY;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) big = fmaxf(big, ml[(w * ROWS + r) * 2]);
    float4 num = make_float4(0.f, 0.f, 0.f, 0.f);
    float den = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float l = ml[(w * ROWS + r) * 2 + 1], root = piece_share_root(ml[(w * ROWS + r) * 2], l, big), f = root * root;
      const float4 x = *reinterpret_cast<const float4*>(acc + (w * ROWS + r) * D + d);
      num.x += x.x * f; num.y += x.y * f; num.z += x.z * f; num.w += x.w * f;
      den += l * root * root;
    }
    if (pieces == 1) {
      const float inv = den == 0.f ? 0.f : 1.f / den;
      const float out[4] = {num.x * inv, num.y * inv, num.z * inv, num.w * inv};
      const int token = r / p.groups, gq = r - token * p.groups;
      store4(p.out + ((size_t)(e.tok0 + token) * p.nkv * p.groups + kvh * p.groups + gq) * D + d, out);
    } else {
      *reinterpret_cast<float4*>(ws + piece_element(p, r, d)) = num;
      if (d == 0) { ws[(size_t)p.ws_rows * D + 2 * r] = big; ws[(size_t)p.ws_rows * D + 2 * r + 1] = den; }
    }
  }
}

// grid: (kv heads, entries, spans); a block takes `span` key tiles of an entry, warp w the keys 32 w .. 32 w + 31 of each.
// Blocks past an entry's last piece come last.
// Registers: for heads of up to 128, what three blocks an SM leave (their rings do not leave room for more).
__global__ void __launch_bounds__(THREADS, D <= 128 ? 3 : 1) attn_kv8_rows_kernel(Kv8Attention p) {
  extern __shared__ __align__(128) unsigned char smem[];
  pdl_trigger();
  pdl_wait();
  const int kvh = blockIdx.x, entry = blockIdx.y, piece = blockIdx.z;
  const Entry e(p, entry);
  const int rows = e.n_new * p.groups;
  if (rows <= p.row_lo || rows > p.row_hi) {
    if (kvh == 0 && piece == 0 && threadIdx.x == 0 && left_out(p, rows)) atomicOr(p.status, FE_STATUS_LEFT_OUT);
    return;
  }
  const Walk<KEYS> walk(p, e.start, 0, rows);
  const int pieces = pieces_of(p, walk.count);
  if (piece >= pieces) return;
  const int begin = piece * p.span, end = piece == pieces - 1 ? walk.count : begin + p.span, steps = end - begin;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  auto key0_of = [&](int i) -> int { return walk.tile(begin + i) * KEYS + warp * STEP; };
  WarpRing mine(smem + warp * (STAGES * STAGE), p, p.block_table + (size_t)entry * p.max_pages, kvh, walk.key_lo, walk.key_end, lane);
  RowQueries q;
  RowSums s;
  int pos[2];                        // rows past the end take the last row's position; nobody reads them
#pragma unroll
  for (int i = 0; i < 2; ++i) pos[i] = e.start + min(2 * t + i, rows - 1) / p.groups;
  auto walk_keys = [&](auto small) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      s.m[i] = -INFINITY;
      s.l[i] = 0.f;
    }
#pragma unroll
    for (int d = 0; d < D / 16; ++d) { s.o[d][0] = s.o[d][1] = s.o[d][2] = s.o[d][3] = 0.f; }
    mine.look_up(key0_of(0));
#pragma unroll 1
    for (int i = -1; i < steps; ++i) {
      if (i >= 0) mine.put_scales(i);
      if (i + 1 < steps) mine.ask(i + 1, key0_of(i + 1), i + 2 < steps ? key0_of(i + 2) : walk.key_end);
      cp_async_commit();
      if (i < 0) {
        q.load(p, e, kvh, rows, lane);
        continue;
      }
      cp_async_wait<1>();
      __syncwarp();
      const int key0 = key0_of(i);
      if (key0 <= walk.pos_last) {
        const bool clear = key0 + STEP - 1 <= walk.pos_first && (p.window <= 0 || walk.pos_last - key0 < p.window);
        take_rows<decltype(small)::value>(q, mine.stage(i), key0, p, clear, pos, s, lane);
      }
      __syncwarp();
    }
  };
  walk_keys(std::false_type());
  if (__any_sync(0xffffffffu, mine.least_scale < SMALL_SCALE)) walk_keys(std::true_type());
  __syncthreads();                   // the rings' space takes the warps' sums
  float* acc = reinterpret_cast<float*>(smem);           // [WARPS][16][D]
  float* ml = acc + WARPS * ROWS * D;                    // [WARPS][16][2]
#pragma unroll
  for (int i = 0; i < 2; ++i) {
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) s.l[i] += __shfl_xor_sync(0xffffffffu, s.l[i], o);
    const int r = 2 * t + i;
    if (r >= rows) continue;
    float* to = acc + (warp * ROWS + r) * D;
#pragma unroll
    for (int d = 0; d < D / 16; d += 2)
      *reinterpret_cast<float4*>(to + row_element(d, g)) = make_float4(s.o[d][i], s.o[d][2 + i], s.o[d + 1][i], s.o[d + 1][2 + i]);
    if (g == 0) {
      ml[(warp * ROWS + r) * 2] = s.m[i];
      ml[(warp * ROWS + r) * 2 + 1] = s.l[i];
    }
  }
  __syncthreads();
  finish_rows(p, e, kvh, rows, pieces, acc, ml, piece_sums(p, entry, kvh, piece));
}

// ---- 9 to 16 rows, any number of head sizes that are no whole 32s, portions of head sizes other than 64 and 128 ----
//
// PORTION: a block takes 64 rows, 16 a warp, and every warp all keys of its tiles.  Otherwise it takes the (at most
// 16) rows of an entry, and warp w the keys 32 w .. 32 w + 31 of every tile; the warps' sums join at the end.
// grid: (kv heads, row tiles - single tokens: entries -, spans); a block takes `span` key tiles of its unit, the row tiles
// that see most keys first.
template <bool PORTION>
__global__ void __launch_bounds__(THREADS) attn_kv8_mma_kernel(Kv8Attention p) {
  extern __shared__ __align__(128) unsigned char smem[];
  constexpr int UNIT = PORTION ? ROWS * WARPS : ROWS;
  pdl_trigger();
  pdl_wait();
  const int kvh = blockIdx.x, piece = blockIdx.z;
  int slot = blockIdx.y, entry = slot, unit = 0;
  if constexpr (PORTION) {
    const Slot<UNIT, true> at(p, slot);
    if (at.entry < 0) return;
    slot = at.slot;
    entry = at.entry;
    unit = at.unit;
  }
  const Entry e(p, entry);
  const int rows = e.n_new * p.groups, row0 = unit * UNIT;
  if (rows <= p.row_lo || rows > p.row_hi || row0 < 0 || row0 >= rows) {
    if (!PORTION && kvh == 0 && piece == 0 && threadIdx.x == 0 && left_out(p, rows)) atomicOr(p.status, FE_STATUS_LEFT_OUT);
    return;
  }
  const int rows_end = min(rows, row0 + UNIT);
  const Walk<KEYS> walk(p, e.start, row0, rows_end);
  const int pieces = pieces_of(p, walk.count);
  if (piece >= pieces) return;
  const int begin = piece * p.span, end = piece == pieces - 1 ? walk.count : begin + p.span;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int* table = p.block_table + (size_t)entry * p.max_pages;
  unsigned char* ring = smem + warp * (STAGES * STAGE);
  const int steps = (end - begin) * (PORTION ? KEYS / STEP : 1);
  auto key0_of = [&](int i) -> int {
    return PORTION ? walk.tile(begin + i / (KEYS / STEP)) * KEYS + i % (KEYS / STEP) * STEP : walk.tile(begin + i) * KEYS + warp * STEP;
  };
  const int wrow0 = PORTION ? row0 + warp * ROWS : row0;
  // rows past the end take the last row's position; nobody reads them
  const int last = rows_end - 1;
  const int pos_a = e.start + min(wrow0 + g, last) / p.groups, pos_b = e.start + min(wrow0 + g + 8, last) / p.groups;
  const int pos_min = e.start + min(wrow0, last) / p.groups, pos_max = e.start + min(wrow0 + ROWS - 1, last) / p.groups;
  Queries q;
  Sums s;
  WarpRing mine(ring, p, table, kvh, walk.key_lo, walk.key_end, lane);
  auto walk_keys = [&](auto small) {
    s.clear();
    mine.look_up(key0_of(0));
#pragma unroll 1
    for (int i = -1; i < steps; ++i) {
      if (i >= 0) mine.put_scales(i);
      if (i + 1 < steps) mine.ask(i + 1, key0_of(i + 1), i + 2 < steps ? key0_of(i + 2) : walk.key_end);
      cp_async_commit();
      if (i < 0) {
        q.load(p, e, kvh, wrow0, rows_end, lane);
        continue;
      }
      cp_async_wait<1>();
      __syncwarp();
      const int key0 = key0_of(i);
      if (key0 <= pos_max) {
        const bool clear = key0 + STEP - 1 <= pos_min && (p.window <= 0 || pos_max - key0 < p.window);
        take<decltype(small)::value>(q, ring + (i & 1) * STAGE, key0, p, clear, pos_a, pos_b, s, lane);
      }
      __syncwarp();
    }
  };
  walk_keys(std::false_type());
  if (__any_sync(0xffffffffu, mine.least_scale < SMALL_SCALE)) walk_keys(std::true_type());
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    s.l[h] += __shfl_xor_sync(0xffffffffu, s.l[h], 1);
    s.l[h] += __shfl_xor_sync(0xffffffffu, s.l[h], 2);
  }
  float* ws = piece_sums(p, slot, kvh, piece);
  if constexpr (PORTION) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = warp * ROWS + g + 8 * h, row = row0 + r;
      if (row >= rows_end) continue;
      const float inv = s.l[h] == 0.f ? 0.f : 1.f / s.l[h];
#pragma unroll
      for (int n = 0; n < D / 8; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int d = value_column(n, c, t);
          if (pieces == 1) store_row(p, e, kvh, row, d, s.o[n][2 * h + c] * inv);
          else ws[piece_element(p, r, d)] = s.o[n][2 * h + c];
        }
      if (pieces > 1 && t == 0) {
        ws[(size_t)p.ws_rows * D + 2 * r] = s.m[h];
        ws[(size_t)p.ws_rows * D + 2 * r + 1] = s.l[h];
      }
    }
  } else {
    const int n_rows = rows_end - row0;
    __syncthreads();                 // the rings' space takes the warps' sums
    float* acc = reinterpret_cast<float*>(smem);           // [WARPS][16][D]
    float* ml = acc + WARPS * ROWS * D;                    // [WARPS][16][2]
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = g + 8 * h;
      if (r >= n_rows) continue;
      float* to = acc + (warp * ROWS + r) * D;
#pragma unroll
      for (int n = 0; n < D / 8; n += (D % 32 == 0 ? 4 : 1))
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          // in stretches of 32 columns and more, four n-tiles are four neighbouring columns
          if constexpr (D % 32 == 0)
            *reinterpret_cast<float4*>(to + value_column(n, c, t)) = make_float4(s.o[n][2 * h + c], s.o[n + 1][2 * h + c], s.o[n + 2][2 * h + c], s.o[n + 3][2 * h + c]);
          else
            to[value_column(n, c, t)] = s.o[n][2 * h + c];
        }
      if (t == 0) {
        ml[(warp * ROWS + r) * 2] = s.m[h];
        ml[(warp * ROWS + r) * 2 + 1] = s.l[h];
      }
    }
    __syncthreads();
    finish_rows(p, e, kvh, n_rows, pieces, acc, ml, ws);
  }
}

template <typename Kernel>
int launch_blocks(Kernel kernel, const Kv8Attention& p, cudaStream_t stream) {
  const cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)MMA_SMEM);
  if (err != cudaSuccess) return (int)err;
  if (p.spans > 65535) return FE_ERR_TOO_LARGE;
  const dim3 grid((unsigned)p.nkv, (unsigned)p.slots, (unsigned)p.spans);
  if (p.spans == 1) return fe_launch_dependent(kernel, grid, dim3(THREADS), MMA_SMEM, stream, p);
  // Cut entries fill the SMs by count, so no block of theirs is to be placed while the kernel before still holds some of
  // them: as a dependent launch one token behind 32768 keys takes 21.3 to 25.2 us from one count of spans to the next,
  // without 21.4 for all, and a decode step of 16 requests of 4096 tokens through 8 layers 863 and 809.  (48 uncut windows of
  // 15 rows behind a cache write: 85.7 as a dependent launch, 87.3 without.)
  kernel<<<grid, THREADS, MMA_SMEM, stream>>>(p);
  return (int)cudaGetLastError();
}

// Entries with row_lo < rows <= row_hi, at most 16.
int launch_single(Kv8Attention p, cudaStream_t stream) {
  p.slots = p.entries;
  p.ws_rows = (single_rows(p.max_new, p.groups, p.row_hi) + 1) & ~1;
  int rc = 0;
#if FE_HEAD_DIM % 32 == 0
  rc = p.row_hi <= 8 ? launch_blocks(attn_kv8_rows_kernel, p, stream) : launch_blocks(attn_kv8_mma_kernel<false>, p, stream);
#else
  rc = launch_blocks(attn_kv8_mma_kernel<false>, p, stream);
#endif
  return rc || p.spans == 1 ? rc : launch_join<KEYS>(p, stream);
}

#if FE_HEAD_DIM != 64 && FE_HEAD_DIM != 128
int launch_portion(Kv8Attention p, cudaStream_t stream) {
  constexpr int UNIT = ROWS * WARPS;
  p.ws_rows = UNIT;
  const int rc = launch_blocks(attn_kv8_mma_kernel<true>, p, stream);
  return rc || p.spans == 1 ? rc : launch_join_portion<UNIT, KEYS>(p, stream);
}
#endif

}  // namespace

// 32-bit numbers of workspace that a call needs; the three kinds of entries use it one after the other.
FE_EXPORT long long SYM(fe_attention_kv8_workspace_d)(int entries, int max_new, int nkv, int groups, int few_spans, int single_spans,
                                                      int portion_units, int portion_spans) {
#if FE_HEAD_DIM == 64 || FE_HEAD_DIM == 128
  constexpr int UNIT = PORTION_UNIT;
#else
  constexpr int UNIT = ROWS * WARPS;
#endif
  auto single = [&](int spans, int row_hi) -> long long {
    return spans > 1 ? (long long)entries * spans * ((single_rows(max_new, groups, row_hi) + 1) & ~1) : 0;
  };
  long long most = portion_spans > 1 ? (long long)portion_units * portion_spans * UNIT : 0;
  if (single(few_spans, 8) > most) most = single(few_spans, 8);
  if (single(single_spans, ROWS) > most) most = single(single_spans, ROWS);
  return most * nkv * (D + 2);
}

// The entries of a step with at most 8 rows (new tokens x heads per kv head) if few_spans is above zero, those with 9 to 16
// if single_spans is, the others if portion_spans is; `*_span` key tiles of 128 a block, `*_spans` of them for the longest.  The
// portions' row tiles number at most portion_units.  Entries and row tiles that this leaves out set a status bit, unless there
// are fillers, entries whose rows nobody reads.
FE_EXPORT int SYM(fe_attention_kv8_d)(const void* q, long long q_stride, void* out, const void* k, const void* v, const void* ks,
                                      const void* vs, const int* block_table, int max_pages, int page_size, int num_pages,
                                      int nkv, int groups, const int* cu_tokens, const int* starts, int entries, int max_new, int total_tokens,
                                      int window, int keep_first, float scale, int few_span, int few_spans,
                                      int single_span, int single_spans, int portion_units, int portion_span, int portion_spans,
                                      int fillers, float* workspace, int* status,
                                      cudaStream_t stream) {
  if (entries <= 0 || max_new <= 0 || total_tokens <= 0) return 0;
  if (page_size < 1 || nkv < 1 || groups < 1 || window < 0 || keep_first < 0 || keep_first > 0x7fff0000 || max_pages < 0 || num_pages < 0) return FE_ERR_BAD_SHAPE;
  if (portion_spans > 0 && portion_units < 1) return FE_ERR_BAD_SHAPE;
  if (few_spans < 0 || single_spans < 0 || portion_spans < 0 || few_span < 1 || single_span < 1 || portion_span < 1) return FE_ERR_BAD_SHAPE;
  if ((few_spans > 1 || single_spans > 1 || portion_spans > 1) && workspace == nullptr) return FE_ERR_BAD_SHAPE;
  if ((long long)num_pages * nkv > 0x7fffffffLL / page_size) return FE_ERR_TOO_LARGE;       // rows of a cache: 31 bits
  if (entries > 65535 || portion_units > 65535 || nkv > 65535 || (long long)total_tokens * groups > 0x7fffffffLL) return FE_ERR_TOO_LARGE;
  if ((((uintptr_t)k | (uintptr_t)v) & 15) || ((uintptr_t)q & 7) || ((uintptr_t)out & 15) || q_stride % 4) return FE_ERR_BAD_ALIGN;
  Kv8Attention p;
  p.q = (const bf16*)q; p.q_stride = q_stride; p.out = (bf16*)out;
  p.k = (const unsigned char*)k; p.v = (const unsigned char*)v; p.ks = (const unsigned char*)ks; p.vs = (const unsigned char*)vs;
  p.block_table = block_table; p.max_pages = max_pages; p.page_size = page_size; p.num_pages = num_pages;
  p.page_shift = -1;
  for (int s = 0; s < 31; ++s)
    if (page_size == 1 << s) p.page_shift = s;
  p.nkv = nkv; p.groups = groups; p.cu_tokens = cu_tokens; p.starts = starts; p.total_tokens = total_tokens;
  p.entries = entries; p.max_new = max_new; p.slots = 0; p.ws_rows = 0;
  p.window = window; p.keep_first = keep_first; p.scale_log2 = scale * 1.4426950408889634f; p.status = status;
  p.ws = workspace;
  // a plan without anything still finds out whether there are rows
  if (!fillers && few_spans == 0 && single_spans == 0 && portion_spans == 0) few_spans = 1;
  p.kinds = fillers ? KINDS_ALL_TOLD : (few_spans > 0 ? 1 : 0) | (single_spans > 0 ? 2 : 0) | (portion_spans > 0 ? 4 : 0);
  if (few_spans > 0) {
    p.row_lo = 0; p.row_hi = 8; p.span = few_span; p.spans = few_spans;
    const int rc = launch_single(p, stream);
    if (rc) return rc;
  }
  if (single_spans > 0) {
    p.row_lo = 8; p.row_hi = ROWS; p.span = single_span; p.spans = single_spans;
    const int rc = launch_single(p, stream);
    if (rc) return rc;
  }
  if (portion_spans > 0) {
    p.row_lo = ROWS; p.row_hi = 0x7fffffff; p.span = portion_span; p.spans = portion_spans; p.slots = portion_units;
    const int rc = launch_portion(p, stream);
    if (rc) return rc;
  }
  return fe_last_error();
}
