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

constexpr int KINDS_ALL_TOLD = 15;          // of Kv8Attention::kinds: what a launch leaves out is nobody's

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
  int entries, max_new;    // max_new: the most tokens an entry has
  int slots;               // single tokens: entries; portions: row tiles of all of them (see Slot)
  int ws_rows;             // rows of a unit, at most; even
  int kinds;               // bit 0, 1, 2: entries of up to 8, up to 16, more rows are launched (see left_out)
  float* ws;               // [slots, nkv, spans][ws_rows x (D + 2)]: see piece_element
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
    if (tok0 < 0 || n_new < 0 || n_new > p.max_new || tok0 > p.total_tokens - n_new || start < 0 || start > 0x7fff0000 - n_new) {
      if (threadIdx.x == 0) atomicOr(p.status, FE_STATUS_BAD_POSITION);
      n_new = 0;
    }
  }
};

// An entry with rows of a kind that the call's plan has not got would be left as it was: somebody who meets it says so.
__device__ __forceinline__ bool left_out(const Kv8Attention& p, long long rows) {
  return rows > 0 && !(p.kinds >> (rows <= 8 ? 0 : rows <= 16 ? 1 : 2) & 1);
}

// The page of a key, or -1 where it is missing; asked for a tile before the key is, so that nothing waits for it.
__device__ __forceinline__ int key_page(const Kv8Attention& p, const int* table, int key, int key_end) {
  const int logical = p.page_shift >= 0 ? key >> p.page_shift : key / p.page_size;
  return key < key_end && logical < p.max_pages ? __ldg(table + logical) : -1;
}

// Which row tile of which entry a block takes: the tiles of UNIT rows of the entries with more than row_lo rows, one entry
// after another; entry -1 past the last one.  A warp finds it, 32 entries at a time.  Entries that cannot be have one
// tile, whose block says so.  FROM_LAST counts from the last tile, so that the tiles that see most keys come first and what
// the grid has too many comes at its end.
template <int UNIT, bool FROM_LAST> struct Slot {
  int entry, unit, slot;
  static __device__ __forceinline__ long long rows_of(const Kv8Attention& p, int e) {
    return e < p.entries ? ((long long)p.cu_tokens[e + 1] - p.cu_tokens[e]) * p.groups : 0;
  }
  static __device__ __forceinline__ int units(const Kv8Attention& p, long long rows) {
    const bool can_be = rows >= 0 && rows <= (long long)p.total_tokens * p.groups;
    return !can_be ? 1 : rows > p.row_lo ? (int)((rows + UNIT - 1) / UNIT) : 0;
  }
  // every block of the grid finds it, one says it
  static __device__ __forceinline__ void tell(const Kv8Attention& p) {
    if (p.kinds != KINDS_ALL_TOLD && blockIdx.x + blockIdx.y + blockIdx.z == 0) atomicOr(p.status, FE_STATUS_LEFT_OUT);
  }
  __device__ __forceinline__ Slot(const Kv8Attention& p, int index) : entry(-1), unit(0), slot(index) {
    const int lane = threadIdx.x & 31;
    if constexpr (FROM_LAST) {
      int all = 0;
      bool left = false;
      for (int e0 = 0; e0 < p.entries; e0 += 32) {
        const long long rows = rows_of(p, e0 + lane);
        left |= left_out(p, rows);
        all += __reduce_add_sync(0xffffffffu, units(p, rows));
      }
      if (left || all > p.slots) tell(p);
      slot = min(all, p.slots) - 1 - index;          // a grid that is too small takes the first ones
      if (slot < 0) return;
    }
    int before = 0;
    for (int e0 = 0; e0 < p.entries; e0 += 32) {
      const int mine = units(p, rows_of(p, e0 + lane));
      int upto = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int left = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += left;
      }
      const unsigned past = __ballot_sync(0xffffffffu, before + upto > slot);
      if (past != 0u) {
        const int at = __ffs(past) - 1;
        entry = e0 + at;
        unit = slot - before - __shfl_sync(0xffffffffu, upto - mine, at);
        return;
      }
      before += __shfl_sync(0xffffffffu, upto, 31);
    }
  }
};

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

// The root of the share of a piece with maximum m and sum l in a join whose largest maximum is `big`.  A piece that saw no
// key has no part; one whose every score was NaN has no maximum, but its sum says so.  (Where M is that of u = t + b, a sum may
// be 2^64 of its weights and the maxima of keys that count alike 2^128 apart: sums go their way in two halves.)
__device__ __forceinline__ float piece_share_root(float m, float l, float big) {
  return m == -INFINITY ? (l == 0.f ? 0.f : 1.f) : exp2f(0.5f * (m - big));
}

// Element (row r of the unit, column d) of a piece's sums: stretches of eight columns, the rows' stretches side by
// side, so that a thread that owns a row stores 32 bytes and its warp 1 KB in a line.  M and l follow the sums.
__device__ __forceinline__ size_t piece_element(const Kv8Attention& p, int r, int d) {
  return ((size_t)(d >> 3) * p.ws_rows + r) * 8 + (d & 7);
}
__device__ __forceinline__ size_t piece_size(const Kv8Attention& p) { return (size_t)p.ws_rows * (D + 2); }
__device__ __forceinline__ float* piece_sums(const Kv8Attention& p, int slot, int kvh, int piece) {
  return p.ws + (((size_t)slot * p.nkv + kvh) * p.spans + piece) * piece_size(p);
}

// Joins the pieces of a single token's rows.  A row may have a hundred of them: a block a row, its eight warps every
// eighth piece, a lane D / 32 (at least two) neighbouring columns and one piece's share of 32; the warps' sums are
// joined in their order (one warp a row: 13.8 us for 103 pieces).  The grid holds no more rows than an entry can have.
// grid: (entries * rows of an entry, kv heads)
constexpr int JOIN_WARPS = 8;

template <int TILE>
__global__ void __launch_bounds__(32 * JOIN_WARPS) attn_kv8_join_kernel(Kv8Attention p, int rows_most) {
  constexpr int COLUMNS = D >= 128 ? 4 : 2, LANES_D = 32 * COLUMNS;
  constexpr int PASSES = (D + LANES_D - 1) / LANES_D;
  __shared__ float sums[JOIN_WARPS][PASSES * LANES_D], dens[JOIN_WARPS];
  pdl_trigger();
  pdl_wait();
  const int entry = blockIdx.x / rows_most, kvh = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Entry e(p, entry);
  const int rows = e.n_new * p.groups, r = blockIdx.x - entry * rows_most;
  if (rows <= p.row_lo || rows > p.row_hi || r >= rows) return;
  const Walk<TILE> walk(p, e.start, 0, rows);
  const int pieces = pieces_of(p, walk.count);
  if (pieces == 1) return;
  const size_t step = piece_size(p);
  const float* ws = piece_sums(p, entry, kvh, 0);
  const float* ml = ws + (size_t)p.ws_rows * D + 2 * r;
  float big = -INFINITY;
  for (int s = lane; s < pieces; s += 32) big = fmaxf(big, ml[s * step]);
  big = warp_max(big);
  float den = 0.f, num[PASSES][COLUMNS];
#pragma unroll
  for (int i = 0; i < PASSES; ++i)
#pragma unroll
    for (int c = 0; c < COLUMNS; ++c) num[i][c] = 0.f;
  const int mine = (pieces - warp + JOIN_WARPS - 1) / JOIN_WARPS;         // pieces warp, warp + 8, ...
  for (int k0 = 0; k0 < mine; k0 += 32) {
    float share = 0.f;
    if (k0 + lane < mine) {
      const float* at = ml + (size_t)(warp + (k0 + lane) * JOIN_WARPS) * step;
      const float root = piece_share_root(at[0], at[1], big);
      share = root * root;
      den += at[1] * root * root;
    }
    const int here = min(32, mine - k0);
#pragma unroll 8
    for (int k = 0; k < here; ++k) {
      const float f = __shfl_sync(0xffffffffu, share, k);
      const float* src = ws + (size_t)(warp + (k0 + k) * JOIN_WARPS) * step;
#pragma unroll
      for (int i = 0; i < PASSES; ++i) {
        const int d = i * LANES_D + lane * COLUMNS;
        if (D % LANES_D == 0 || d < D) {
#pragma unroll
          for (int c = 0; c < COLUMNS; c += 2) {
            const float2 x = *reinterpret_cast<const float2*>(src + piece_element(p, r, d + c));
            num[i][c] += x.x * f;
            num[i][c + 1] += x.y * f;
          }
        }
      }
    }
  }
  den = warp_sum(den);
#pragma unroll
  for (int i = 0; i < PASSES; ++i)
#pragma unroll
    for (int c = 0; c < COLUMNS; ++c) sums[warp][i * LANES_D + lane * COLUMNS + c] = num[i][c];
  if (lane == 0) dens[warp] = den;
  __syncthreads();
  den = 0.f;
#pragma unroll
  for (int w = 0; w < JOIN_WARPS; ++w) den += dens[w];
  for (int d = threadIdx.x; d < D; d += 32 * JOIN_WARPS) {
    float x = 0.f;
#pragma unroll
    for (int w = 0; w < JOIN_WARPS; ++w) x += sums[w][d];
    store_row(p, e, kvh, r, d, den == 0.f ? 0.f : x / den);
  }
}

// Joins the pieces of a portion's rows, in the order of the keys: a thread takes eight columns of a row, eight lanes eight
// rows, so that a warp reads 256 bytes in a line and its stores fill 64.  Portions have few pieces and many rows.
// grid: (slots * UNIT / rows of a block, kv heads)
constexpr int JOIN_ROWS = D <= 64 ? 32 : D <= 128 ? 16 : 8;         // eight columns of a row a thread
template <int UNIT, int TILE>
__global__ void __launch_bounds__(256) attn_kv8_join_portion_kernel(Kv8Attention p) {
  constexpr int BLOCKS = UNIT / JOIN_ROWS, STRETCHES = D / 8, BATCH = 4;
  pdl_trigger();
  pdl_wait();
  const int slot = blockIdx.x / BLOCKS, kvh = blockIdx.y;
  const Slot<UNIT, false> at(p, slot);
  if (at.entry < 0) return;
  const Entry e(p, at.entry);
  const int rows = e.n_new * p.groups, row0 = at.unit * UNIT, r0 = (blockIdx.x - slot * BLOCKS) * JOIN_ROWS;
  if (rows <= p.row_lo || rows > p.row_hi || row0 < 0 || row0 + r0 >= rows) return;
  const int rows_end = min(rows, row0 + UNIT);
  const Walk<TILE> walk(p, e.start, row0, rows_end);
  const int pieces = pieces_of(p, walk.count);
  if (pieces == 1) return;
  const size_t step = piece_size(p);
  const float* ws = piece_sums(p, slot, kvh, 0);
  const int i = threadIdx.x, r = r0 + (i & 7) + 8 * (i / (8 * STRETCHES)), d = 8 * ((i >> 3) % STRETCHES);
  if (i >= JOIN_ROWS * STRETCHES || row0 + r >= rows_end) return;
  const float* ml = ws + (size_t)p.ws_rows * D + 2 * r;
  float big = -INFINITY, den = 0.f, num[8];
#pragma unroll
  for (int c = 0; c < 8; ++c) num[c] = 0.f;
  for (int s0 = 0; s0 < pieces; s0 += BATCH) {
    float2 of[BATCH];
    float4 a[BATCH], b[BATCH];
    float now = big;
#pragma unroll
    for (int s = 0; s < BATCH; ++s) {
      of[s] = make_float2(-INFINITY, 0.f);
      a[s] = b[s] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (s0 + s < pieces) {
        of[s] = *reinterpret_cast<const float2*>(ml + (s0 + s) * step);
        const float4* src = reinterpret_cast<const float4*>(ws + (s0 + s) * step + piece_element(p, r, d));
        a[s] = src[0];
        b[s] = src[1];
      }
    }
#pragma unroll
    for (int s = 0; s < BATCH; ++s) now = fmaxf(now, of[s].x);
    const float root = big == -INFINITY ? 1.f : exp2f(0.5f * (big - now));         // what is there without a maximum is 0 or NaN
    den = den * root * root;
#pragma unroll
    for (int c = 0; c < 8; ++c) num[c] *= root * root;
    big = now;
#pragma unroll
    for (int s = 0; s < BATCH; ++s) {
      const float root = piece_share_root(of[s].x, of[s].y, big), share = root * root;
      den += of[s].y * root * root;
      num[0] += a[s].x * share; num[1] += a[s].y * share; num[2] += a[s].z * share; num[3] += a[s].w * share;
      num[4] += b[s].x * share; num[5] += b[s].y * share; num[6] += b[s].z * share; num[7] += b[s].w * share;
    }
  }
#pragma unroll
  for (int c = 0; c < 8; ++c) num[c] = den == 0.f ? 0.f : num[c] / den;
  const int row = row0 + r, token = row / p.groups, g = row - token * p.groups;
  bf16* to = p.out + ((size_t)(e.tok0 + token) * p.nkv * p.groups + kvh * p.groups + g) * D + d;
  store4(to, num);
  store4(to + 4, num + 4);
}

// Rows that an entry of a call of single tokens has at most.
inline int single_rows(long long max_new, int groups, int row_hi) { return max_new * groups < row_hi ? (int)(max_new * groups) : row_hi; }

template <int TILE>
inline int launch_join(const Kv8Attention& p, cudaStream_t stream) {
  const int rows = single_rows(p.max_new, p.groups, p.row_hi);
  return fe_launch_dependent(attn_kv8_join_kernel<TILE>, dim3((unsigned)(p.slots * rows), (unsigned)p.nkv), dim3(32 * JOIN_WARPS), 0, stream, p,
                             rows);
}

template <int UNIT, int TILE>
inline int launch_join_portion(const Kv8Attention& p, cudaStream_t stream) {
  return fe_launch_dependent(attn_kv8_join_portion_kernel<UNIT, TILE>, dim3((unsigned)(p.slots * (UNIT / JOIN_ROWS)), (unsigned)p.nkv), dim3(256),
                             0, stream, p);
}

#if FE_HEAD_DIM == 64 || FE_HEAD_DIM == 128
constexpr int PORTION_UNIT = 256, PORTION_TILE = 128;      // rows of a block and keys of a tile of the tcgen05 kernel
int launch_portion(Kv8Attention p, cudaStream_t stream);
#endif

}  // namespace kv8
