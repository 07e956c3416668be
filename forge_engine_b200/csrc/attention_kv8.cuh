// What the attention kernels over the 8-bit cache share (attention_kv8.cu, attention_kv8_portion.cu): the call's
// parameters, which key tiles a block walks, where a key lies, and how the pieces of a cut entry are joined.
// Compiled for one head size: -DFE_HEAD_DIM.
#pragma once
#include "kv8.cuh"

#ifndef FE_HEAD_DIM
#error "compile with -DFE_HEAD_DIM=<head size>"
#endif

namespace kv8 {

constexpr int D = FE_HEAD_DIM;
static_assert(D % 16 == 0 && D >= 16 && D <= 256, "head size must be a multiple of 16 up to 256");

struct Kv8Attention {
  const bf16* q;
  long long q_stride;
  bf16* out;               // [tokens, nkv * groups * D]
  const unsigned char *k, *v, *ks, *vs;
  const int* block_table;
  int max_pages, page_size, page_shift, num_pages, nkv, groups;
  const int* cu_tokens;    // [entries + 1]
  const int* starts;       // [entries]
  int total_tokens, window, keep_first;
  float scale_log2;
  int* status;
  int row_lo, row_hi;      // entries with row_lo < rows <= row_hi
  int span, spans;         // a block takes `span` key tiles of a unit; the grid holds `spans` of them
  int units;               // row tiles of the longest entry
  float* ws;               // [entries, nkv, units, spans][rows of a unit x (D + 2)]: see piece_element
};

// The key tiles (of TILE keys) that the rows [row0, row0 + n) of an entry see: first the tiles that hold kept
// first tokens and lie before the window, then the window's.
template <int TILE>
struct Walk {
  int pos_first, pos_last, key_lo, key_end, kept, first, count;
  __device__ __forceinline__ Walk(const Kv8Attention& p, int start, int row0, int rows_end) {
    pos_first = start + row0 / p.groups;
    pos_last = start + (rows_end - 1) / p.groups;
    key_lo = p.window > 0 ? max(0, pos_first - p.window + 1) : 0;
    key_end = pos_last + 1;
    first = key_lo / TILE;
    kept = p.window > 0 ? min((p.keep_first + TILE - 1) / TILE, first) : 0;
    count = kept + (key_end + TILE - 1) / TILE - first;
  }
  __device__ __forceinline__ int tile(int i) const { return i < kept ? i : first + i - kept; }
};

// Pieces of a unit of `count` key tiles; where the grid holds fewer than its spans give, the last takes the rest.
__device__ __forceinline__ int pieces_of(const Kv8Attention& p, int count) { return min(p.spans, (count + p.span - 1) / p.span); }

// Tokens of an entry, held to the tensors the call brought.
struct Entry {
  int tok0, n_new, start;
  __device__ __forceinline__ Entry(const Kv8Attention& p, int entry) {
    tok0 = p.cu_tokens[entry];
    n_new = p.cu_tokens[entry + 1] - tok0;
    start = p.starts[entry];
    if (tok0 < 0 || n_new < 0 || tok0 > p.total_tokens - n_new || start < 0 || start > 0x7fff0000 - n_new) {
      if (threadIdx.x == 0) atomicOr(p.status, FE_STATUS_BAD_POSITION);
      n_new = 0;
    }
  }
};

// The page of a key, or -1 where it is missing; asked for a tile before the key is, so that nothing waits for it.
__device__ __forceinline__ int key_page(const Kv8Attention& p, const int* table, int key, int key_end) {
  const int logical = p.page_shift >= 0 ? key >> p.page_shift : key / p.page_size;
  return key < key_end && logical < p.max_pages ? __ldg(table + logical) : -1;
}

// Row (page, head, slot) of a key in its page; a page that is not there gives row 0 and false.
__device__ __forceinline__ bool key_row(const Kv8Attention& p, int page, int kvh, int key, long long* row) {
  const bool there = page >= 0 && page < p.num_pages;
  const int slot = p.page_shift >= 0 ? key & (p.page_size - 1) : key % p.page_size;
  *row = there ? ((long long)page * p.nkv + kvh) * p.page_size + slot : 0;
  return there;
}

// A key that some row must see and whose page is missing.
__device__ __forceinline__ void tell_missing(const Kv8Attention& p, int key, int key_lo, int key_end) {
  if (key < key_end && (key >= key_lo || key < p.keep_first)) atomicOr(p.status, FE_STATUS_BAD_PAGE);
}

__device__ __forceinline__ void store_row(const Kv8Attention& p, const Entry& e, int kvh, int row, int d, float v) {
  const int token = row / p.groups, g = row - token * p.groups;
  p.out[((size_t)(e.tok0 + token) * p.nkv * p.groups + kvh * p.groups + g) * D + d] = __float2bfloat16_rn(v);
}

// The share of a piece with maximum m and sum l in a join whose largest maximum is `big`.  A piece that saw no
// key has no part; one whose every score was NaN has no maximum, but its sum says so.
__device__ __forceinline__ float piece_share(float m, float l, float big) {
  return m == -INFINITY ? (l == 0.f ? 0.f : 1.f) : exp2f(m - big);
}

// Element (row r of the unit, column d) of a piece's sums: stretches of eight columns, the rows' stretches side by
// side, so that a thread that owns a row stores 32 bytes and its warp 1 KB in a line.  M and l follow the sums.
template <int UNIT> __device__ __forceinline__ size_t piece_element(int r, int d) {
  return ((size_t)(d >> 3) * UNIT + r) * 8 + (d & 7);
}

constexpr int JOIN_WARPS = 4;

// Joins the pieces of a unit's rows, in the order of the keys: a warp a row, a lane D / 32 (at least two)
// neighbouring columns; the lanes work out 32 pieces' shares at a time.
// grid: (units x UNIT / 4, entries, kv heads)
template <int UNIT, int TILE>
__global__ void __launch_bounds__(32 * JOIN_WARPS) attn_kv8_join_kernel(Kv8Attention p) {
  constexpr int COLUMNS = D >= 128 ? 4 : 2, LANES_D = 32 * COLUMNS;
  constexpr int PASSES = (D + LANES_D - 1) / LANES_D;
  pdl_trigger();
  pdl_wait();
  constexpr int BLOCKS = UNIT / JOIN_WARPS;
  const int unit = blockIdx.x / BLOCKS, entry = blockIdx.y, kvh = blockIdx.z, lane = threadIdx.x & 31;
  const Entry e(p, entry);
  const int rows = e.n_new * p.groups, row0 = unit * UNIT;
  if (rows <= p.row_lo || rows > p.row_hi || row0 >= rows) return;
  const int rows_end = min(rows, row0 + UNIT);
  const int r = (blockIdx.x - unit * BLOCKS) * JOIN_WARPS + (threadIdx.x >> 5);
  if (row0 + r >= rows_end) return;
  const Walk<TILE> walk(p, e.start, row0, rows_end);
  const int pieces = pieces_of(p, walk.count);
  if (pieces == 1) return;
  const size_t step = (size_t)UNIT * (D + 2);
  const float* ws = p.ws + (((size_t)entry * p.nkv + kvh) * p.units + unit) * p.spans * step;
  const float* ml = ws + (size_t)UNIT * D + 2 * r;
  float big = -INFINITY;
  for (int s = lane; s < pieces; s += 32) big = fmaxf(big, ml[s * step]);
  big = warp_max(big);
  float den = 0.f, num[PASSES][COLUMNS];
#pragma unroll
  for (int i = 0; i < PASSES; ++i)
#pragma unroll
    for (int c = 0; c < COLUMNS; ++c) num[i][c] = 0.f;
  for (int s0 = 0; s0 < pieces; s0 += 32) {
    float mine = 0.f;
    if (s0 + lane < pieces) {
      const float m = ml[(s0 + lane) * step], l = ml[(s0 + lane) * step + 1];
      mine = piece_share(m, l, big);
      den += l * mine;
    }
    const int here = min(32, pieces - s0);
#pragma unroll 4
    for (int s = 0; s < here; ++s) {
      const float f = __shfl_sync(0xffffffffu, mine, s);
      const float* src = ws + (s0 + s) * step;
#pragma unroll
      for (int i = 0; i < PASSES; ++i) {
        const int d = i * LANES_D + lane * COLUMNS;
        if (D % LANES_D == 0 || d < D) {
#pragma unroll
          for (int c = 0; c < COLUMNS; c += 2) {
            const float2 x = *reinterpret_cast<const float2*>(src + piece_element<UNIT>(r, d + c));
            num[i][c] += x.x * f;
            num[i][c + 1] += x.y * f;
          }
        }
      }
    }
  }
  den = warp_sum(den);
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int d = i * LANES_D + lane * COLUMNS;
    if (D % LANES_D == 0 || d < D) {
#pragma unroll
      for (int c = 0; c < COLUMNS; ++c) store_row(p, e, kvh, row0 + r, d + c, den == 0.f ? 0.f : num[i][c] / den);
    }
  }
}

#if FE_HEAD_DIM == 64 || FE_HEAD_DIM == 128
constexpr int PORTION_UNIT = 256, PORTION_TILE = 128;      // rows of a block and keys of a tile of the tcgen05 kernel
int launch_portion(Kv8Attention p, int entries, int max_new, cudaStream_t stream);
#endif

}  // namespace kv8
