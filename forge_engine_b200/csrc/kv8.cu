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
#include <cuda_fp16.h>

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

// A group of LANES lanes (a power of two, at least D / 8) takes a head's vector; a lane holds four pairs
// (a[i], b[i]) that rotate together.  With R rotated dimensions pair i < R/2 is (i, i + R/2); the others
// pair up (R + i', R + (D - R)/2 + i') and stay as they are.  R is a multiple of 8, so four pairs are two
// stretches of four elements.
template <typename T, int LANES>
__global__ void __launch_bounds__(128)
kv8_write_kernel(const T* __restrict__ q, long long q_stride, bf16* __restrict__ q_out, int nq, const T* __restrict__ k,
                 long long k_stride, const T* __restrict__ v, long long v_stride, const float* __restrict__ q_weight,
                 const float* __restrict__ k_weight, float eps, const float2* __restrict__ table, int rot,
                 const int* __restrict__ positions, const int* __restrict__ token_entry, Kv8Pages c, int* status) {
  constexpr int HEADS = 32 / LANES;
  pdl_trigger();
  const int token = blockIdx.x;
  const int lane = threadIdx.x & 31, sub = lane / LANES, l = lane % LANES;
  const int warp = blockIdx.y * (blockDim.x >> 5) + (threadIdx.x >> 5), warps = (blockDim.x >> 5) * gridDim.y;
  const int D = c.dim;
  const bool mine = 8 * l < D;                   // lanes past the vector only take part in the sums
  const int pair = 4 * l, half = rot >> 1;
  const bool turns = pair < half;
  const int ia = turns ? pair : rot + (pair - half), ib = turns ? pair + half : rot + ((D - rot) >> 1) + (pair - half);
  pdl_wait();
  const int pos = positions[token];
  const long long row = k == nullptr ? -1 : kv8_row(c, token_entry[token], pos, status, threadIdx.x == 0 && blockIdx.y == 0);
  float cs[4], sn[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) { cs[e] = 1.f; sn[e] = 0.f; }
  if (turns && mine) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 both = table[(size_t)token * half + pair + e];
      cs[e] = both.x;
      sn[e] = both.y;
    }
  }
  const int heads = nq + (k == nullptr ? 0 : 2 * c.nkv);
  // every lane of a warp makes every round: the sums below are over whole warps
  for (int first = warp * HEADS; first < heads; first += warps * HEADS) {
    const int head = first + sub;
    const bool is_q = head < nq, is_k = !is_q && head < nq + c.nkv;
    const bool on = mine && head < heads && (is_q || row >= 0);
    float a[4] = {0.f, 0.f, 0.f, 0.f}, b[4] = {0.f, 0.f, 0.f, 0.f};
    const int kvh = is_q ? 0 : (is_k ? head - nq : head - nq - c.nkv);
    if (on) {
      const T* x = is_q ? q + (size_t)token * q_stride + (size_t)head * D
                        : (is_k ? k + (size_t)token * k_stride : v + (size_t)token * v_stride) + (size_t)kvh * D;
      load4(x + ia, a);
      load4(x + ib, b);
    }
    const float* w = is_q ? q_weight : (is_k ? k_weight : nullptr);
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) ss += a[e] * a[e] + b[e] * b[e];
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (w != nullptr && on) {
      const float inv = rsqrtf(ss / (float)D + eps);
      float wa[4], wb[4];
      load4(w + ia, wa);
      load4(w + ib, wb);
#pragma unroll
      for (int e = 0; e < 4; ++e) { a[e] = a[e] * inv * wa[e]; b[e] = b[e] * inv * wb[e]; }
    }
    if (is_q || is_k) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x = a[e] * cs[e] - b[e] * sn[e], y = b[e] * cs[e] + a[e] * sn[e];
        if (turns) { a[e] = x; b[e] = y; }        // 0 * inf is not 0: what does not turn is left alone
      }
    }
    unsigned big = 0u;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      big = max(big, max(__float_as_uint(a[e]) & 0x7fffffffu, __float_as_uint(b[e]) & 0x7fffffffu));
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) big = max(big, __shfl_xor_sync(0xffffffffu, big, o));
    if (!on) continue;
    if (is_q) {
      bf16* dst = q_out + ((size_t)token * nq + head) * D;
      store4(dst + ia, a);
      store4(dst + ib, b);
      continue;
    }
    const bool finite = big < 0x7f800000u;
    const int e8 = finite ? kv8_exponent(big) : 0;
    const float down = __int_as_float((127 - e8) << 23);
    unsigned ca = 0u, cb = 0u;
    if (finite) {
      ca = (unsigned)kv8_codes(a[0] * down, a[1] * down) | (unsigned)kv8_codes(a[2] * down, a[3] * down) << 16;
      cb = (unsigned)kv8_codes(b[0] * down, b[1] * down) | (unsigned)kv8_codes(b[2] * down, b[3] * down) << 16;
    }
    const size_t at = (size_t)row + (size_t)kvh * c.page_size;
    unsigned char* dst = (is_k ? c.k : c.v) + at * D;
    *reinterpret_cast<unsigned*>(dst + ia) = ca;
    *reinterpret_cast<unsigned*>(dst + ib) = cb;
    if (l == 0) (is_k ? c.ks : c.vs)[at] = (unsigned char)(finite ? e8 + KV8_BIAS : KV8_NAN);
  }
}

__device__ __forceinline__ void kv8_store16(bf16* dst, const float* v) { store8(dst, v); store8(dst + 8, v + 8); }
__device__ __forceinline__ void kv8_store16(float* dst, const float* v) { store8(dst, v); store8(dst + 8, v + 8); }

// A thread takes 16 codes of a token's key vector and the 16 of its value vector.
template <typename T>
__global__ void __launch_bounds__(256)
kv8_read_kernel(Kv8Pages c, const int* __restrict__ positions, const int* __restrict__ token_entry, T* __restrict__ k_out,
                T* __restrict__ v_out, int tokens, int* status) {
  pdl_trigger();
  pdl_wait();
  const int chunks = c.dim >> 4, per_token = c.nkv * chunks;
  const long long unit = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  const long long token = unit / per_token;
  if (token >= tokens) return;
  const int rest = (int)(unit - token * per_token), head = rest / chunks, chunk = rest - head * chunks;
  const long long row = kv8_row(c, token_entry[token], positions[token], status, rest == 0);
  uint4 raw[2] = {make_uint4(0u, 0u, 0u, 0u), make_uint4(0u, 0u, 0u, 0u)};
  float scale[2] = {0.f, 0.f};
  if (row >= 0) {
    const size_t at = (size_t)row + (size_t)head * c.page_size;
    raw[0] = __ldcs(reinterpret_cast<const uint4*>(c.k + at * c.dim) + chunk);
    raw[1] = __ldcs(reinterpret_cast<const uint4*>(c.v + at * c.dim) + chunk);
    scale[0] = kv8_scale(c.ks[at]);
    scale[1] = kv8_scale(c.vs[at]);
  }
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    const unsigned words[4] = {raw[m].x, raw[m].y, raw[m].z, raw[m].w};
    float out[16];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const unsigned h = kv8_half2((unsigned short)(words[i >> 1] >> (16 * (i & 1))));
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
      out[2 * i] = f.x * scale[m];
      out[2 * i + 1] = f.y * scale[m];
    }
    kv8_store16((m ? v_out : k_out) + (size_t)token * per_token * 16 + (size_t)rest * 16, out);
  }
}

template <typename T>
int kv8_write_typed(const void* q, long long q_stride, bf16* q_out, int nq, const void* k, long long k_stride, const void* v,
                    long long v_stride, const float* q_weight, const float* k_weight, float eps, const float2* table, int rot,
                    const int* positions, const int* token_entry, const Kv8Pages& c, int tokens, int* status, cudaStream_t stream) {
  const int lanes = c.dim <= 16 ? 2 : c.dim <= 32 ? 4 : c.dim <= 64 ? 8 : c.dim <= 128 ? 16 : 32;
  const int heads_a_warp = 32 / lanes, heads = nq + (k == nullptr ? 0 : 2 * c.nkv);
  if (heads == 0) return 0;
  const int rounds = (heads + 4 * heads_a_warp - 1) / (4 * heads_a_warp);      // of a block of four warps over a token's heads
  // few tokens: blocks share a token's heads until the chip has about two blocks an SM
  int share = rounds < (296 + tokens - 1) / tokens ? rounds : (296 + tokens - 1) / tokens;
  const dim3 grid((unsigned)tokens, (unsigned)share);
  auto launch = [&](auto kernel) {
    return fe_launch_dependent(kernel, grid, dim3(128), 0, stream, (const T*)q, q_stride, q_out, nq, (const T*)k, k_stride,
                               (const T*)v, v_stride, q_weight, k_weight, eps, table, rot, positions, token_entry, c, status);
  };
  switch (lanes) {
    case 2: return launch(kv8_write_kernel<T, 2>);
    case 4: return launch(kv8_write_kernel<T, 4>);
    case 8: return launch(kv8_write_kernel<T, 8>);
    case 16: return launch(kv8_write_kernel<T, 16>);
    default: return launch(kv8_write_kernel<T, 32>);
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
  if (((uintptr_t)q_out & 7) || (((uintptr_t)q_weight | (uintptr_t)k_weight) & 15) || ((uintptr_t)table & 7)) return FE_ERR_BAD_ALIGN;
  const int done = dtype == FE_DTYPE_F32
                       ? kv8_write_typed<float>(q, q_stride, (bf16*)q_out, nq, k, k_stride, v, v_stride, q_weight, k_weight, eps,
                                                (const float2*)table, rot, positions, token_entry, c, tokens, status, stream)
                       : kv8_write_typed<bf16>(q, q_stride, (bf16*)q_out, nq, k, k_stride, v, v_stride, q_weight, k_weight, eps,
                                               (const float2*)table, rot, positions, token_entry, c, tokens, status, stream);
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
  const long long blocks = ((long long)tokens * nkv * (dim / 16) + 255) / 256;
  if (blocks > 0x7fffffffLL) return FE_ERR_TOO_LARGE;
  const dim3 grid((unsigned)blocks);
  const int done = dtype == FE_DTYPE_F32
                       ? fe_launch_dependent(kv8_read_kernel<float>, grid, dim3(256), 0, stream, c, positions, token_entry, (float*)k_out,
                                             (float*)v_out, tokens, status)
                       : fe_launch_dependent(kv8_read_kernel<bf16>, grid, dim3(256), 0, stream, c, positions, token_entry, (bf16*)k_out,
                                             (bf16*)v_out, tokens, status);
  return done ? done : fe_last_error();
}
