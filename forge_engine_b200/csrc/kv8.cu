// Writing the 8-bit cache and reading it back (layout and rounding: kv8.cuh).
//
// Upstream keeps its pages in the model's type and copies new keys and values into them after the forward
// (src/forge_engine/cache.py:385-416); it has no cache in 8 bits.
//
// Writing takes the finished projection of a step's tokens: q and k normalised per head
// (src/forge_engine/qwen3.py:141-150) and rotated (:345-381), in 32 bits, then
//   b = the largest |x| of a head's vector (a maximum over a group of lanes, on the bits of |x|, so that
//       infinities and NaN win),  e = least with b <= 448 * 2^e,  codes = round(x * 2^-e)
// k and v are quantised from the unrounded 32-bit values: one rounding between the projection and the page.
#include <type_traits>

#include "kv8.cuh"

namespace {

struct Kv8Pages {
  unsigned char* k;
  unsigned char* v;
  unsigned char* ks;
  unsigned char* vs;
  const int* block_table;      // [entries, max_pages]
  int entries, max_pages, page_size, num_pages, nkv, dim;
};

// Row (page * nkv + head) * page_size + slot of (entry, position, head 0), or -1 with a status bit set.
__device__ __forceinline__ long long kv8_row(const Kv8Pages& c, int entry, int pos, int* status, bool tell) {
  const int logical = pos / c.page_size;
  if (pos < 0 || logical >= c.max_pages || entry < 0 || entry >= c.entries) {
    if (tell) atomicOr(status, FE_STATUS_BAD_POSITION);
    return -1;
  }
  const int page = c.block_table[(size_t)entry * c.max_pages + logical];
  if (page < 0 || page >= c.num_pages) {
    if (tell) atomicOr(status, FE_STATUS_BAD_PAGE);
    return -1;
  }
  return (long long)page * c.nkv * c.page_size + (pos - logical * c.page_size);
}

// E consecutive elements (4 or 8)
template <int E, typename T> __device__ __forceinline__ void load_some(const T* src, float* out) {
  if constexpr (E == 8) load8(src, out); else load4(src, out);
}
// E elements as they lie in memory: what is asked for a round ahead waits in as few registers as it can
template <int E, typename T> struct Held {
  static constexpr int WORDS = E * (int)sizeof(T) / 4;
  unsigned w[WORDS];
  __device__ __forceinline__ void load(const T* src) {
    if constexpr (WORDS == 2) {
      const uint2 x = *reinterpret_cast<const uint2*>(src);
      w[0] = x.x; w[1] = x.y;
    } else {
#pragma unroll
      for (int i = 0; i < WORDS; i += 4) {
        const uint4 x = reinterpret_cast<const uint4*>(src)[i / 4];
        w[i] = x.x; w[i + 1] = x.y; w[i + 2] = x.z; w[i + 3] = x.w;
      }
    }
  }
  __device__ __forceinline__ void numbers(float* out) const {
#pragma unroll
    for (int i = 0; i < WORDS; ++i) {
      if constexpr (sizeof(T) == 4) out[i] = __uint_as_float(w[i]);
      else {
        out[2 * i] = __uint_as_float(w[i] << 16);
        out[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    }
  }
};
template <int E> __device__ __forceinline__ void store_some(bf16* dst, const float* v) {
  if constexpr (E == 8) store8(dst, v); else store4(dst, v);
}

// Keys that were normalised or rotated are rounded to four bits behind a 32-bit computation, so an element whose 32-bit
// error spans the middle between two codes could take the wrong one (4,096 tokens of 8 heads: about 5 of 4.2 million).
// The writer converts the two ends of that span, and where they differ anywhere in a head (about one in thirty) the
// head's lanes take it again in 64 bits, from the row as it lies in memory: codes and scale are those of exact arithmetic.
struct Kv8Exact {
  unsigned codes[4];               // of the lane's E elements from ia on, then from ib on
  int e8;
};
// a 64-bit number as a 32-bit one whose last bit says that something is missing: rounding it to fewer bits rounds once
__device__ __forceinline__ float kv8_odd(double x) {
  const float y = __double2float_rz(x);
  return (double)y == x ? y : __int_as_float(__float_as_int(y) | 1);
}
template <typename T, int LANES, int E>
__device__ __forceinline__ Kv8Exact kv8_exact(const T* x, const float* w, const float2* turn, int ia, int ib, bool mine, float eps, int D,
                                           unsigned group) {
  float a[E], b[E];
  Held<E, T> held;
#pragma unroll
  for (int e = 0; e < E; ++e) a[e] = b[e] = 0.f;
  if (mine) {
    held.load(x + ia);
    held.numbers(a);
    held.load(x + ib);
    held.numbers(b);
  }
  double inv = 1.0;
  if (w != nullptr) {
    double ss = 0.0;
#pragma unroll
    for (int e = 0; e < E; ++e) ss = fma((double)a[e], (double)a[e], fma((double)b[e], (double)b[e], ss));
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(group, ss, o);
    inv = rsqrt(ss / D + (double)eps);
  }
  double p[E], r[E];
  unsigned big = 0u;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    p[e] = a[e];
    r[e] = b[e];
    if (w != nullptr && mine) {
      p[e] *= inv * (double)w[ia + e];
      r[e] *= inv * (double)w[ib + e];
    }
    if (turn != nullptr && mine) {
      const double c = turn[e].x, s = turn[e].y, first = p[e] * c - r[e] * s;
      r[e] = r[e] * c + p[e] * s;
      p[e] = first;
    }
    big = max(big, max(__float_as_uint(__double2float_ru(fabs(p[e]))), __float_as_uint(__double2float_ru(fabs(r[e])))));
  }
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) big = max(big, __shfl_xor_sync(group, big, o));
  Kv8Exact out;
  out.e8 = kv8_exponent(big);
  const double down = (double)__int_as_float((127 - out.e8) << 23);
#pragma unroll
  for (int e = 0; e < E; e += 4) {
    out.codes[e / 4] = (unsigned)kv8_codes(kv8_odd(p[e] * down), kv8_odd(p[e + 1] * down)) |
                       (unsigned)kv8_codes(kv8_odd(p[e + 2] * down), kv8_odd(p[e + 3] * down)) << 16;
    out.codes[E / 4 + e / 4] = (unsigned)kv8_codes(kv8_odd(r[e] * down), kv8_odd(r[e + 1] * down)) |
                               (unsigned)kv8_codes(kv8_odd(r[e + 2] * down), kv8_odd(r[e + 3] * down)) << 16;
  }
  return out;
}

template <int E> __device__ __forceinline__ void store_codes(unsigned char* dst, const unsigned* codes) {
  if constexpr (E == 8) *reinterpret_cast<uint2*>(dst) = make_uint2(codes[0], codes[1]);
  else *reinterpret_cast<unsigned*>(dst) = codes[0];
}

constexpr int WRITE_ROUNDS = 64;                 // heads a group of lanes takes one after the other, at most

// A group of LANES lanes (a power of two, at least D / 2E) takes a head's vector; a lane holds E pairs (a[i], b[i])
// that rotate together.  With R rotated dimensions pair i < R/2 is (i, i + R/2); the others pair up
// (R + i', R + (D - R)/2 + i') and stay as they are.  R is a multiple of 2E, so E pairs are two stretches of E elements.
// E = 8 where rows and R allow 16-byte loads of bfloat16, else 4.  Queries are not measured for a scale, values not
// normalised.  4,096 tokens of 32 + 16 heads of 128: 27.2 us, 0.53 of the copy peak, instructions issued in most cycles
// (34.6 with E = 4; 24.2 when keys' codes were those of 32-bit arithmetic: 1.7 for the span's second end, the rest for heads
// taken again; with that inside the loop, where its registers count, 34.6).  64 tokens in 32 bits 5.0, one 3.4, most
// of it the launch and the first loads.  Seven blocks an SM: 27.5 us, eight, with 40 bytes of spills, 28.3, six 28.5.
template <typename T, int LANES, int E>
__global__ void __launch_bounds__(128, 7)
kv8_write_kernel(const T* __restrict__ q, long long q_stride, bf16* __restrict__ q_out, int nq, const T* __restrict__ k,
                 long long k_stride, const T* __restrict__ v, long long v_stride, const float* __restrict__ q_weight,
                 const float* __restrict__ k_weight, float eps, const float2* __restrict__ table, int rot,
                 const int* __restrict__ positions, const int* __restrict__ token_entry, Kv8Pages c, int* status) {
  constexpr int HEADS = 32 / LANES;
  pdl_trigger();
  const int token = blockIdx.x;
  const int lane = threadIdx.x & 31, sub = lane / LANES, l = lane % LANES;
  const int warp = blockIdx.y * (blockDim.x >> 5) + (threadIdx.x >> 5), warps = (blockDim.x >> 5) * gridDim.y;
  const unsigned group = LANES == 32 ? 0xffffffffu : ((1u << LANES % 32) - 1u) << (sub * LANES);
  const int D = c.dim;
  const bool mine = 2 * E * l < D;               // lanes past the vector only take part in the sums
  const int pair = E * l, half = rot >> 1;
  const bool turns = pair < half;
  const int ia = turns ? pair : rot + (pair - half), ib = turns ? pair + half : rot + ((D - rot) >> 1) + (pair - half);
  pdl_wait();
  float cs[E], sn[E];
#pragma unroll
  for (int e = 0; e < E; ++e) { cs[e] = 1.f; sn[e] = 0.f; }
  if (turns && mine) {
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      const float4 both = *reinterpret_cast<const float4*>(table + (size_t)token * half + pair + e);
      cs[e] = both.x; sn[e] = both.y;
      cs[e + 1] = both.z; sn[e + 1] = both.w;
    }
  }
  const int heads = nq + (k == nullptr ? 0 : 2 * c.nkv);
  const T* q_row = q + (size_t)token * q_stride;
  const T* k_row = k + (size_t)token * k_stride;
  const T* v_row = v + (size_t)token * v_stride;
  auto source = [&](int head) -> const T* {
    return head < nq ? q_row + (size_t)head * D : head < nq + c.nkv ? k_row + (size_t)(head - nq) * D : v_row + (size_t)(head - nq - c.nkv) * D;
  };
  Held<E, T> held_a{}, held_b{};
  int head = warp * HEADS + sub;
  auto fetch = [&](int h) {
    if (mine && h < heads) {
      const T* x = source(h);
      held_a.load(x + ia);
      held_b.load(x + ib);
    }
  };
  fetch(head);
  // the first rows are on their way before the place is looked up
  const long long row = k == nullptr ? -1 : kv8_row(c, token_entry[token], positions[token], status, threadIdx.x == 0 && blockIdx.y == 0);
  unsigned long long again = 0ull;               // key heads of this group to take again, by rounds: there are at most WRITE_ROUNDS
  for (; head < heads; head += warps * HEADS) {             // the same for a group's lanes
    const bool is_q = head < nq, is_k = !is_q && head < nq + c.nkv;
    float a[E], b[E];
    held_a.numbers(a);
    held_b.numbers(b);
    fetch(head + warps * HEADS);
    const float* w = is_q ? q_weight : (is_k ? k_weight : nullptr);
    if (w != nullptr) {
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) ss += a[e] * a[e] + b[e] * b[e];
#pragma unroll
      for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(group, ss, o);
      const float inv = rsqrtf(ss / (float)D + eps);
      if (mine) {
        float wa[E], wb[E];
        load_some<E>(w + ia, wa);
        load_some<E>(w + ib, wb);
#pragma unroll
        for (int e = 0; e < E; ++e) { a[e] = a[e] * inv * wa[e]; b[e] = b[e] * inv * wb[e]; }
      }
    }
    if ((is_q || is_k) && turns) {                          // 0 * inf is not 0: what does not turn is left alone
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float x = a[e] * cs[e] - b[e] * sn[e], y = b[e] * cs[e] + a[e] * sn[e];
        a[e] = x;
        b[e] = y;
      }
    }
    if (is_q) {
      if (mine) {
        bf16* dst = q_out + ((size_t)token * nq + head) * D;
        store_some<E>(dst + ia, a);
        store_some<E>(dst + ib, b);
      }
      continue;
    }
    unsigned big = 0u;
#pragma unroll
    for (int e = 0; e < E; ++e)
      big = max(big, max(__float_as_uint(a[e]) & 0x7fffffffu, __float_as_uint(b[e]) & 0x7fffffffu));
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) big = max(big, __shfl_xor_sync(group, big, o));
    if (row < 0) continue;
    const bool finite = big < 0x7f800000u;
    const int e8 = finite ? kv8_exponent(big) : 0;
    const float down = __int_as_float((127 - e8) << 23);
    unsigned codes[E / 2];
    // elements 0 .. E - 1 and E .. 2 E - 1 of the lane, each moved by `by` times the sum of its pair's magnitudes
    auto encode = [&](auto moved, float by, unsigned (&to)[E / 2]) {
#pragma unroll
      for (int e = 0; e < E; e += 4) {
        float x[4], y[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          x[j] = a[e + j] * down;
          y[j] = b[e + j] * down;
          if constexpr (decltype(moved)::value) {
            const float at = (fabsf(x[j]) + fabsf(y[j])) * by;
            x[j] += at;
            y[j] += at;
          }
        }
        to[e / 4] = (unsigned)kv8_codes(x[0], x[1]) | (unsigned)kv8_codes(x[2], x[3]) << 16;
        to[E / 4 + e / 4] = (unsigned)kv8_codes(y[0], y[1]) | (unsigned)kv8_codes(y[2], y[3]) << 16;
      }
    };
    if (is_k && finite && (w != nullptr || rot > 0)) {
      // 32-bit errors in units of 2^-24: sum of squares 13 (two of a term, at most eleven sums) and the mean 2, half of it in
      // the root, the root itself 4 (two ulp), weights 2, relative to an element; a rotation carries that over to
      // a pair's length and adds at most 2 of it; and a pair's magnitudes sum to no less than its length
      constexpr float SPAN = 16.f / 16777216.f;
      unsigned other[E / 2];
      encode(std::true_type(), -SPAN, codes);
      encode(std::true_type(), SPAN, other);
      bool apart = abs((int)(big & 0x7fffffu) - 0x600000) < 32;          // the scale's border
#pragma unroll
      for (int i = 0; i < E / 2; ++i) apart |= mine && codes[i] != other[i];
      if (__any_sync(group, apart)) again |= 1ull << (head - nq) / (warps * HEADS);
    } else if (finite) {
      encode(std::false_type(), 0.f, codes);
    } else {
#pragma unroll
      for (int i = 0; i < E / 2; ++i) codes[i] = 0u;
    }
    if (!mine) continue;
    const int kvh = is_k ? head - nq : head - nq - c.nkv;
    const size_t at = (size_t)row + (size_t)kvh * c.page_size;
    unsigned char* dst = (is_k ? c.k : c.v) + at * D;
    store_codes<E>(dst + ia, codes);
    store_codes<E>(dst + ib, codes + E / 4);
    if (l == 0) (is_k ? c.ks : c.vs)[at] = (unsigned char)(finite ? e8 + KV8_BIAS : KV8_NAN);
  }
  if (again == 0ull) return;
  const int step = warps * HEADS;
  int kvh = warp * HEADS + sub - nq;
  if (kvh < 0) kvh += (-kvh + step - 1) / step * step;
  for (; kvh < c.nkv; kvh += step) {
    if (!(again >> kvh / step & 1ull)) continue;
    const Kv8Exact sure = kv8_exact<T, LANES, E>(k_row + (size_t)kvh * D, k_weight, turns ? table + (size_t)token * half + pair : nullptr, ia, ib,
                                                 mine, eps, D, group);
    const size_t at = (size_t)row + (size_t)kvh * c.page_size;
    if (mine) {
      store_codes<E>(c.k + at * D + ia, sure.codes);
      store_codes<E>(c.k + at * D + ib, sure.codes + E / 4);
    }
    if (l == 0) c.ks[at] = (unsigned char)(sure.e8 + KV8_BIAS);
  }
}

// 16 bytes of output from as many codes, times their scale
__device__ __forceinline__ void kv8_put(bf16* dst, uint2 codes, float scale) {
  float out[8];
  unsigned h[4];
  kv8_halves(codes.x, h[0], h[1]);
  kv8_halves(codes.y, h[2], h[3]);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
    out[2 * i] = f.x * scale;
    out[2 * i + 1] = f.y * scale;
  }
  store8(dst, out);
}
__device__ __forceinline__ void kv8_put(float* dst, unsigned codes, float scale) {
  unsigned h[2];
  kv8_halves(codes, h[0], h[1]);
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&h[0])), b = __half22float2(*reinterpret_cast<const __half2*>(&h[1]));
  *reinterpret_cast<float4*>(dst) = make_float4(a.x * scale, a.y * scale, b.x * scale, b.y * scale);
}

// A warp takes a token: neighbouring lanes write neighbouring 16 bytes of its rows.  32-bit output of several contexts, 4
// heads of 64, 95 MB in all: 21.7 us, 0.67 of the copy peak, warps waiting for their pages, scales and codes (with 16 codes
// a thread, whose 64 bytes of output lay apart, 25.6 us).
template <typename T>
__global__ void __launch_bounds__(256)
kv8_read_kernel(Kv8Pages c, const int* __restrict__ positions, const int* __restrict__ token_entry, T* __restrict__ k_out,
                T* __restrict__ v_out, int tokens, int* status) {
  constexpr int N = 16 / sizeof(T);             // codes a lane takes at a time
  using Codes = std::conditional_t<N == 8, uint2, unsigned>;
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const long long token = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  if (token >= tokens) return;
  const long long row = kv8_row(c, token_entry[token], positions[token], status, lane == 0);
  const int width = c.nkv * c.dim, step = 32 * N, heads_a_step = step / c.dim, rest = step - heads_a_step * c.dim;
  int head = lane * N / c.dim, at = lane * N - head * c.dim;
  T* k_row = k_out + (size_t)token * width;
  T* v_row = v_out + (size_t)token * width;
#pragma unroll 4
  for (int i = lane * N; i < width; i += step) {
    Codes k{}, v{};
    float k_scale = 0.f, v_scale = 0.f;
    if (row >= 0) {
      const size_t place = (size_t)row + (size_t)head * c.page_size;
      k = __ldcs(reinterpret_cast<const Codes*>(c.k + place * c.dim + at));
      v = __ldcs(reinterpret_cast<const Codes*>(c.v + place * c.dim + at));
      k_scale = kv8_scale(c.ks[place]);
      v_scale = kv8_scale(c.vs[place]);
    }
    kv8_put(k_row + i, k, k_scale);
    kv8_put(v_row + i, v, v_scale);
    head += heads_a_step;
    at += rest;
    if (at >= c.dim) { at -= c.dim; ++head; }
  }
}

template <typename T, int E>
int kv8_write_typed(const void* q, long long q_stride, bf16* q_out, int nq, const void* k, long long k_stride, const void* v,
                    long long v_stride, const float* q_weight, const float* k_weight, float eps, const float2* table, int rot,
                    const int* positions, const int* token_entry, const Kv8Pages& c, int tokens, int* status, cudaStream_t stream) {
  int lanes = 1;
  while (lanes * 2 * E < c.dim) lanes *= 2;
  const int heads_a_warp = 32 / lanes, heads = nq + (k == nullptr ? 0 : 2 * c.nkv);
  if (heads == 0) return 0;
  const int rounds = (heads + 4 * heads_a_warp - 1) / (4 * heads_a_warp);      // of a block of four warps over a token's heads
  // few tokens: blocks share a token's heads until the chip has about two blocks an SM
  int share = rounds < (296 + tokens - 1) / tokens ? rounds : (296 + tokens - 1) / tokens;
  if (share < (rounds + WRITE_ROUNDS - 1) / WRITE_ROUNDS) share = (rounds + WRITE_ROUNDS - 1) / WRITE_ROUNDS;
  if (share > 65535) return FE_ERR_TOO_LARGE;
  const dim3 grid((unsigned)tokens, (unsigned)share);
  auto launch = [&](auto kernel) {
    return fe_launch_dependent(kernel, grid, dim3(128), 0, stream, (const T*)q, q_stride, q_out, nq, (const T*)k, k_stride,
                               (const T*)v, v_stride, q_weight, k_weight, eps, table, rot, positions, token_entry, c, status);
  };
  constexpr int LEAST = 8 / E;                  // of heads of 16; 256 take 16 times as many
  switch (lanes / LEAST) {
    case 1: return launch(kv8_write_kernel<T, LEAST, E>);
    case 2: return launch(kv8_write_kernel<T, 2 * LEAST, E>);
    case 4: return launch(kv8_write_kernel<T, 4 * LEAST, E>);
    case 8: return launch(kv8_write_kernel<T, 8 * LEAST, E>);
    default: return launch(kv8_write_kernel<T, 16 * LEAST, E>);
  }
}

int kv8_pages(Kv8Pages* c, const void* k, const void* v, const void* ks, const void* vs, const int* block_table, int entries,
              int max_pages, int page_size, int num_pages, int nkv, int dim) {
  if (dim < 16 || dim > 256 || dim % 16 || page_size < 1 || nkv < 1 || num_pages < 0 || entries < 0 || max_pages < 0)
    return FE_ERR_BAD_SHAPE;
  if (((uintptr_t)k | (uintptr_t)v) & 15) return FE_ERR_BAD_ALIGN;
  c->k = (unsigned char*)k; c->v = (unsigned char*)v; c->ks = (unsigned char*)ks; c->vs = (unsigned char*)vs;
  c->block_table = block_table; c->entries = entries; c->max_pages = max_pages; c->page_size = page_size;
  c->num_pages = num_pages; c->nkv = nkv; c->dim = dim;
  return 0;
}

}  // namespace

// q (nq may be 0), k and v (both may be null: queries only): rows of `dtype`, `*_stride` elements apart, heads side by side.  The norms' weights and the
// table of cosines and sines ([tokens, rot / 2, 2]) may be null (rot 0).
FE_EXPORT int fe_kv8_write(const void* q, long long q_stride, void* q_out, int nq, const void* k, long long k_stride, const void* v,
                           long long v_stride, int dtype, const float* q_weight, const float* k_weight, float eps,
                           const float* table, int rot, const int* positions, const int* token_entry, void* k_cache,
                           void* v_cache, void* k_scale, void* v_scale, const int* block_table, int entries, int max_pages,
                           int page_size, int num_pages, int nkv, int dim, int tokens, int* status, cudaStream_t stream) {
  if (tokens <= 0) return 0;
  Kv8Pages c;
  const int rc = kv8_pages(&c, k_cache, v_cache, k_scale, v_scale, block_table, entries, max_pages, page_size, num_pages, nkv, dim);
  if (rc) return rc;
  if (nq < 0 || rot < 0 || rot > dim || rot % 8 || (rot > 0 && table == nullptr) || (k == nullptr) != (v == nullptr)) return FE_ERR_BAD_SHAPE;
  if (dtype != FE_DTYPE_F32 && dtype != FE_DTYPE_BF16) return FE_ERR_BAD_DTYPE;
  const uintptr_t rows = dtype == FE_DTYPE_F32 ? 15 : 7;
  if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v) & rows || (q_stride | k_stride | v_stride) % 4) return FE_ERR_BAD_ALIGN;
  if (((uintptr_t)q_out & 7) || (((uintptr_t)q_weight | (uintptr_t)k_weight) & 15) || ((uintptr_t)table & 15)) return FE_ERR_BAD_ALIGN;
  // 16-byte loads of eight elements
  const bool wide = rot % 16 == 0 && !((((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)q_out) & 15) || (q_stride | k_stride | v_stride) % 8);
  auto write = [&](auto kind, auto each) {
    using T = decltype(kind);
    return kv8_write_typed<T, decltype(each)::value>(q, q_stride, (bf16*)q_out, nq, k, k_stride, v, v_stride, q_weight, k_weight, eps,
                                                     (const float2*)table, rot, positions, token_entry, c, tokens, status, stream);
  };
  using Eight = std::integral_constant<int, 8>;
  using Four = std::integral_constant<int, 4>;
  const int done = dtype == FE_DTYPE_F32 ? (wide ? write(float(), Eight()) : write(float(), Four())) : (wide ? write(bf16(), Eight()) : write(bf16(), Four()));
  return done ? done : fe_last_error();
}

// k_out, v_out: [tokens, nkv, dim] of `dtype`; a place that is not there gives zeros and a status bit.
FE_EXPORT int fe_kv8_read(const void* k_cache, const void* v_cache, const void* k_scale, const void* v_scale,
                          const int* block_table, int entries, int max_pages, int page_size, int num_pages, int nkv, int dim,
                          const int* positions, const int* token_entry, void* k_out, void* v_out, int dtype, int tokens,
                          int* status, cudaStream_t stream) {
  if (tokens <= 0) return 0;
  Kv8Pages c;
  const int rc = kv8_pages(&c, k_cache, v_cache, k_scale, v_scale, block_table, entries, max_pages, page_size, num_pages, nkv, dim);
  if (rc) return rc;
  if (dtype != FE_DTYPE_F32 && dtype != FE_DTYPE_BF16) return FE_ERR_BAD_DTYPE;
  if (((uintptr_t)k_out | (uintptr_t)v_out) & 15) return FE_ERR_BAD_ALIGN;
  const long long blocks = ((long long)tokens + 7) / 8;
  if (blocks > 0x7fffffffLL) return FE_ERR_TOO_LARGE;
  const dim3 grid((unsigned)blocks);
  const int done = dtype == FE_DTYPE_F32
                       ? fe_launch_dependent(kv8_read_kernel<float>, grid, dim3(256), 0, stream, c, positions, token_entry, (float*)k_out,
                                             (float*)v_out, tokens, status)
                       : fe_launch_dependent(kv8_read_kernel<bf16>, grid, dim3(256), 0, stream, c, positions, token_entry, (bf16*)k_out,
                                             (bf16*)v_out, tokens, status);
  return done ? done : fe_last_error();
}
