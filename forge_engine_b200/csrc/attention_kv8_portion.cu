// Attention of prompt portions over the 8-bit cache on the 5th-generation tensor cores (tcgen05), head sizes 64 and
// 128 (-DFE_HEAD_DIM).  Formulas and layout: attention_kv8.cu, kv8.cuh.
//
//   block = two query tiles of 128 rows (row = token * G + head in group) of one (entry, kv head) and one piece of
//           its keys, in tiles of 128 keys that both query tiles use; one block an SM, 16 warps of 128 registers
//   warps 0-3, 4-7   tile 0 and tile 1.  First its queries, as two e4m3 numbers each: a row times a power of two,
//           rounded, and what the rounding left.  Together they hold bfloat16's 8 bits down to 2^-11 of the row's
//           largest element, and what is smaller to within 2^-18 of it, so the scores are products of 8-bit numbers
//           with the cached codes as they lie in their pages: keys are only copied.  Then softmax, a thread a row:
//           scores from tensor memory times the keys' scales, mask, running maximum (moved only when it grows by more
//           than 2^8), weights back over the scores as bfloat16.  A tile is taken in halves of 64 keys: while a half is
//           in the softmax the tensor core works on the other
//   warps 8-13   copy the keys of a tile, and bring its values: 16-byte pieces of codes into registers a tile ahead,
//           code * 2^b as bfloat16 (exact) into the swizzled tile in shared memory
//   warps 14, 15   issue the products of tile 0 and tile 1: O_x += P_x V with P from tensor memory, then in the weights'
//           place the scores S_x = Q_x K^T (both parts of the queries) of the next tile's half.  A thread that issues
//           products waits for the tensor core most of the time: one for both tiles left the tensor core idle while it
//           waited for weights (5,700 cycles a tile), and a softmax thread that did it held up its row's warp (10,000)
//
// Values are not left as 8-bit numbers, because then the weights would have to be: a weight as two e4m3 numbers costs
// a softmax thread more than the 256 rows' share of converting a value.  Measured with keys converted like the
// values: 7,700 cycles a tile, all of it the staging warps.  20 warps, of 96 and of 120 registers, were slower too.
//
// A tile takes 4,600 to 5,000 cycles (2.6 to 3.2 us), a block about 9 us beside its tiles (row tile, pages, first keys and
// queries one after the other, the last products and stores): 2,048 tokens from the start 69 us, 509 behind 32,259
// keys 435.  The tensor core works in 26 to 38 % of the cycles, the exponentials' unit in 27 to 39 %, instructions issue in
// 49 to 55 %: what bounds a tile is the chain of a softmax warp's half (scores out, maximum, exponentials, weights
// back), of which a scheduler holds two beside the staging warps; registers leave no room for a third.

#include <cuda_fp16.h>

#include "attention_kv8.cuh"

#if FE_HEAD_DIM == 64 || FE_HEAD_DIM == 128
#include "tcgen05.cuh"

using namespace kv8;

namespace {

constexpr int TILE_ROWS = 128, KEYS = PORTION_TILE;
constexpr int SOFTMAX_WARPS = 8, STAGING_WARPS = 6;
constexpr int MMA_WARP = SOFTMAX_WARPS + STAGING_WARPS;      // and the next one; the first also takes and frees tensor memory
constexpr int THREADS = 32 * (MMA_WARP + 2);
constexpr int K_STAGES = 3, V_STAGES = 3, CK_STAGES = 4;
constexpr int HALF = KEYS / 2;                    // keys of a softmax step: a tile is taken in two
constexpr int TMEM_COLS = 512, COL_S = 0, COL_O = 256;     // + 128 x, scores + 64 for the second half
constexpr int CODE_TILE = 128 * 128;              // 128 rows of codes, 128 bytes apart whatever the head size
constexpr int V_BYTES = KEYS * D * 2;
constexpr float RESCALE_STEP = 8.f;               // log2 units
constexpr int CHUNKS = D / 16;                    // 16-byte pieces of a cached vector
constexpr int UNITS = KEYS * CHUNKS / 32;         // a matrix' pieces of a tile, 32 at a time
constexpr int PIECES = (UNITS + STAGING_WARPS - 1) / STAGING_WARPS;       // of them a staging thread takes at most
constexpr size_t SMEM = (size_t)4 * CODE_TILE + (size_t)K_STAGES * CODE_TILE + (size_t)V_STAGES * V_BYTES + CK_STAGES * KEYS * 4 +
                        32 * 8 + 64 + 1024;
static_assert(SMEM > 120 * 1024 && SMEM <= 227 * 1024, "one block an SM: it takes all tensor memory");

__device__ __forceinline__ uint64_t desc_kmajor(const void* tile) { return tc5::umma_desc(tile); }
// The N index runs along a 128-byte row: blocks of 64 N elements `block_bytes` apart, groups of 8 k 1024 bytes apart.
__device__ __forceinline__ uint64_t desc_mnmajor(const void* tile, unsigned block_bytes) {
  uint64_t d = 0;
  d |= (uint64_t)((tc5::smem_u32(tile) & 0x3FFFFu) >> 4);
  d |= (uint64_t)(block_bytes >> 4) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}
__device__ __forceinline__ void mma_ts(unsigned d, unsigned a, uint64_t b, unsigned idesc, unsigned accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
               ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// S += A B of e4m3 numbers, 32 of the contraction
__device__ __forceinline__ void mma_codes(unsigned d, uint64_t a, uint64_t b, unsigned idesc, unsigned accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
               ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// Bounded wait that lets the thread rest: false when the limit was hit or another role has already given up.
constexpr unsigned WAIT_TRIES = 2000000u;
__device__ __forceinline__ bool wait(uint64_t* bar, unsigned parity, volatile int* abort_flag) {
  for (unsigned i = 0; i < WAIT_TRIES; ++i) {
    unsigned ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok) : "r"(tc5::smem_u32(bar)), "r"(parity) : "memory");
    if (ok) return true;
    if ((i & 63u) == 63u && *abort_flag) return false;
  }
  *abort_flag = 1;
  return false;
}
__device__ __forceinline__ void arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(tc5::smem_u32(bar)) : "memory");
}
__device__ __forceinline__ float exp2_fast(float x) {       // the weight is rounded to 8 bits anyway
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(lo), "f"(hi));
  return d;
}
__device__ __forceinline__ void unpair(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ unsigned pack_bf16(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const unsigned*>(&h);
}
__device__ __forceinline__ void tmem_ld32(unsigned addr, unsigned* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st16(unsigned addr, const unsigned (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
      ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// Two half-precision numbers that were codes as bfloat16, times a power of two (`up`, both halves the same).  A code is a half-precision number with 5 bits of exponent; moved down by three bits
// it is the bfloat16 number 2^-112 times as large, never below bfloat16's normal ones.
__device__ __forceinline__ unsigned bf16_of_half(unsigned h, __nv_bfloat162 up) {
  const unsigned r = ((h >> 3) & 0x0fff0fffu) | (h & 0x80008000u);
  const __nv_bfloat162 x = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&r), up);
  return *reinterpret_cast<const unsigned*>(&x);
}

// Where the 16 bytes c of a row of 128 bytes lie (128-byte swizzle).
__device__ __forceinline__ unsigned code_offset(int row, int c) { return (unsigned)(row * 128 + ((c ^ (row & 7)) << 4)); }
// The same for eight bfloat16 elements 8 c .. of a value: blocks of 64 columns.
__device__ __forceinline__ unsigned tile_offset(int row, int c) {
  return (unsigned)((c >> 3) * (128 * 128) + row * 128 + (((c & 7) ^ (row & 7)) << 4));
}

// The key tiles one query tile of the block takes part in.
struct QueryTile {
  bool valid;
  int row0, pos_first, pos_last, lo, end;
  __device__ __forceinline__ QueryTile(const Kv8Attention& p, int start, int first_row, int rows) {
    row0 = first_row;
    valid = first_row < rows;
    const int last = min(rows, first_row + TILE_ROWS) - 1;
    pos_first = start + first_row / p.groups;
    pos_last = start + last / p.groups;
    lo = (p.window > 0 ? max(0, pos_first - p.window + 1) : 0) / KEYS;
    end = pos_last / KEYS + 1;
  }
};

__global__ void __launch_bounds__(THREADS, 1) attn_kv8_portion_kernel(Kv8Attention p) {
  extern __shared__ unsigned char smem_raw[];
  // an offset, not a rounded pointer: the compiler still knows that this is shared memory
  unsigned char* smem = smem_raw + (1024u - (tc5::smem_u32(smem_raw) & 1023u)) % 1024u;
  unsigned char* q_tiles = smem;                              // [2 query tiles][2 parts][128 rows][128 B]
  unsigned char* k_tiles = q_tiles + 4 * CODE_TILE;           // [stages][128 keys][128 B]
  unsigned char* v_tiles = k_tiles + K_STAGES * CODE_TILE;    // [stages][D/64][128 keys][128 B]
  float* k_factor = reinterpret_cast<float*>(v_tiles + V_STAGES * V_BYTES);      // [stages][128 keys] scales
  uint64_t* k_full = reinterpret_cast<uint64_t*>(k_factor + CK_STAGES * KEYS);   // [stages]
  uint64_t* v_full = k_full + K_STAGES;          // [stages]
  // freed[n & 3], event n: for every query tile the tensor core is done with the scores of step n and the value
  // products of step n - 1
  uint64_t* freed = v_full + V_STAGES;           // [4]
  uint64_t* s_full = freed + 4;                  // [2 query tiles][2 halves] scores are there
  uint64_t* p_full = s_full + 4;                 // [2][2] weights are there
  uint64_t* q_full = p_full + 4;                 // [2]
  uint64_t* o_full = q_full + 2;                 // [2]
  unsigned* tmem_slot = reinterpret_cast<unsigned*>(o_full + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  pdl_trigger();
  pdl_wait();
  // blocks start in the order of x, y, z: the row tiles that see most keys first
  const int kvh = blockIdx.x, piece = blockIdx.y;
  const Slot<PORTION_UNIT, true> at(p, blockIdx.z);
  if (at.entry < 0) return;
  const int slot = at.slot;
  const Entry e(p, at.entry);
  const int rows = e.n_new * p.groups, row0 = at.unit * PORTION_UNIT;
  if (rows <= p.row_lo || rows > p.row_hi || row0 < 0 || row0 >= rows) return;
  const Walk<KEYS> walk(p, e.start, row0, min(rows, row0 + PORTION_UNIT));
  const int pieces = pieces_of(p, walk.count);
  if (piece >= pieces) return;
  const int begin = piece * p.span, end = piece == pieces - 1 ? walk.count : begin + p.span, steps = end - begin;
  const QueryTile t0(p, e.start, row0, rows), t1(p, e.start, row0 + TILE_ROWS, rows);
  const int sink_keys = p.window > 0 ? p.keep_first : 0;
  const int sink_tiles = (int)(((long long)sink_keys + KEYS - 1) / KEYS);
  auto active = [&](int x, int i) -> bool {
    const int kt = walk.tile(begin + i);
    return x == 0 ? kt < t0.end && (kt >= t0.lo || kt < sink_tiles) : t1.valid && kt < t1.end && (kt >= t1.lo || kt < sink_tiles);
  };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < K_STAGES; ++s) tc5::mbar_init(k_full + s, STAGING_WARPS);
    for (int s = 0; s < V_STAGES; ++s) tc5::mbar_init(v_full + s, STAGING_WARPS);
    for (int s = 0; s < 4; ++s) tc5::mbar_init(freed + s, t1.valid ? 2 : 1);
    for (int x = 0; x < 4; ++x) { tc5::mbar_init(s_full + x, 1); tc5::mbar_init(p_full + x, 4); }
    for (int x = 0; x < 2; ++x) { tc5::mbar_init(q_full + x, 4); tc5::mbar_init(o_full + x, 1); }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == MMA_WARP) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc5::smem_u32(tmem_slot)), "r"(TMEM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const unsigned tmem = *tmem_slot;

  if (warp >= SOFTMAX_WARPS && warp < MMA_WARP) {
    // ---- staging ----
    const int* table = p.block_table + (size_t)at.entry * p.max_pages;
    // Piece j of this lane is 16 bytes of one of the warp's rows, unit w + 6 j; the lanes of a unit lie so that eight
    // neighbours store their 32 bytes of bfloat16 without meeting in a bank.  A lane looks after one of the warp's
    // rows - its page, its place and its scales - and the others ask it.
    constexpr int UNIT_ROWS = 32 / CHUNKS;
    static_assert(PIECES * UNIT_ROWS <= 32, "a lane a row");
    const int w = warp - SOFTMAX_WARPS;
    const int c = CHUNKS == 8 ? (lane & 3) | ((lane >> 3) & 1) << 2 : lane & 3;
    const int sub = CHUNKS == 8 ? ((lane >> 2) & 1) | (lane >> 4) << 1 : lane >> 2;        // row inside the unit
    const int my_row = lane < PIECES * UNIT_ROWS ? (w + STAGING_WARPS * (lane / UNIT_ROWS)) * UNIT_ROWS + lane % UNIT_ROWS : KEYS;      // KEYS or more: none
    auto mine = [&](int j) -> bool { return UNITS % STAGING_WARPS == 0 || j < PIECES - 1 || w + STAGING_WARPS * j < UNITS; };      // the same for the warp
    struct Row {
      long long at;                   // -1: not there
      int k_scale, v_scale;
    };
    auto look_up = [&](int i) -> int {
      return my_row < KEYS && i < steps ? key_page(p, table, walk.tile(begin + i) * KEYS + my_row, walk.key_end) : -1;
    };
    auto find = [&](int page, int i) -> Row {
      Row r = {-1, KV8_BIAS, KV8_BIAS};
      if (i >= steps || my_row >= KEYS) return r;
      const int key = walk.tile(begin + i) * KEYS + my_row;
      long long at;
      if (key_row(p, page, kvh, key, &at)) {
        r.at = at;
        r.k_scale = __ldg(p.ks + at);
        r.v_scale = __ldg(p.vs + at);
      } else {
        tell_missing(p, key, walk.key_lo, walk.key_end);
      }
      return r;
    };
    auto copy_keys = [&](const Row& row, int i) {
      unsigned char* tile = k_tiles + (i % K_STAGES) * CODE_TILE;
#pragma unroll
      for (int j = 0; j < PIECES; ++j) {
        const long long at = __shfl_sync(0xffffffffu, row.at, j * UNIT_ROWS + sub);
        if (mine(j))
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n"
                     ::"r"(tc5::smem_u32(tile + code_offset((w + STAGING_WARPS * j) * UNIT_ROWS + sub, c))), "l"(p.k + (at < 0 ? 0 : at) * D + 16 * c),
                       "r"(at < 0 ? 0 : 16));
      }
    };
    // a key whose value is not finite counts as not finite itself; missing ones are zero
    auto put_factors = [&](const Row& row, int i) {
      if (my_row < KEYS) k_factor[(i % CK_STAGES) * KEYS + my_row] = kv8_scale(row.v_scale == KV8_NAN ? KV8_NAN : row.k_scale);
    };
    auto fetch_values = [&](uint4 (&raw)[PIECES], const Row& row) {
#pragma unroll
      for (int j = 0; j < PIECES; ++j) {
        const long long at = __shfl_sync(0xffffffffu, row.at, j * UNIT_ROWS + sub);
        raw[j] = make_uint4(0u, 0u, 0u, 0u);
        if (at >= 0) raw[j] = __ldg(reinterpret_cast<const uint4*>(p.v + at * D) + c);
      }
    };
    auto store_values = [&](const uint4 (&raw)[PIECES], int scale, int i) {
      unsigned char* tile = v_tiles + (i % V_STAGES) * V_BYTES;
      const bool large = __any_sync(0xffffffffu, scale - KV8_BIAS > 15);
#pragma unroll
      for (int j = 0; j < PIECES; ++j) {
        // 2^(112 + ex); beyond 2^127 the rest is multiplied separately
        const int ex = __shfl_sync(0xffffffffu, scale, j * UNIT_ROWS + sub) - KV8_BIAS;
        const unsigned bits = (unsigned)(127 + 112 + min(ex, 15)) << 7, twice = bits | bits << 16;
        const __nv_bfloat162 up = *reinterpret_cast<const __nv_bfloat162*>(&twice);
        const unsigned words[4] = {raw[j].x, raw[j].y, raw[j].z, raw[j].w};
        unsigned x[8];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          unsigned lo, hi;
          kv8_halves(words[k], lo, hi);
          x[2 * k] = bf16_of_half(lo, up);
          x[2 * k + 1] = bf16_of_half(hi, up);
        }
        if (large) {
          const __nv_bfloat162 more = __float2bfloat162_rn(__int_as_float((127 + max(ex - 15, 0)) << 23));
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const __nv_bfloat162 y = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&x[k]), more);
            x[k] = *reinterpret_cast<const unsigned*>(&y);
          }
        }
        const unsigned at = tile_offset((w + STAGING_WARPS * j) * UNIT_ROWS + sub, 2 * c);
        if (mine(j)) {
          *reinterpret_cast<uint4*>(tile + at) = make_uint4(x[0], x[1], x[2], x[3]);
          *reinterpret_cast<uint4*>(tile + (at ^ 16u)) = make_uint4(x[4], x[5], x[6], x[7]);
        }
      }
    };
    auto wait_event = [&](int event) -> bool {          // lane 0 waits for the warp
      bool ok = true;
      if (lane == 0) ok = wait(freed + (event & 3), (event >> 2) & 1, abort_flag);
      return __shfl_sync(0xffffffffu, ok, 0);
    };
    auto publish = [&](uint64_t* bar) {                 // what this warp wrote is there for the tensor core
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) arrive(bar);
    };
    // Links of a tile: its rows' pages, three tiles ahead; their places and scales and the keys' codes, two ahead; the
    // values' codes, one ahead; the values as numbers.  The loop starts two steps early instead of in front of itself: code
    // that runs once costs the fetching of its instructions.
    uint4 values[PIECES];
    int page = look_up(0);
    Row now = {-1, KV8_BIAS, KV8_BIAS}, next = now;
#pragma unroll 1
    for (int i = -2; i < steps; ++i) {
      const Row after = find(page, i + 2);
      page = look_up(i + 3);
      if (i >= 0) {
        if (i >= V_STAGES && !wait_event(i - V_STAGES + 1)) break;      // the value products of step i - 3 are done
        store_values(values, now.v_scale == KV8_NAN ? KV8_BIAS : now.v_scale, i);
        publish(v_full + i % V_STAGES);
      }
      if (i >= -1) fetch_values(values, next);
      // the scores of step i - 1 are done, and the weights of step i - 2: nobody waits for an earlier phase of the
      // barriers that are arrived at below
      if (i >= 1 && !wait_event(i - 1)) break;
      if (i + 2 < steps) copy_keys(after, i + 2);
      asm volatile("cp.async.commit_group;\n" ::);
      if (i >= -1 && i + 1 < steps) {
        put_factors(next, i + 1);
        asm volatile("cp.async.wait_group 1;\n" ::: "memory");       // the keys of step i + 1 are here
        publish(k_full + (i + 1) % K_STAGES);
      }
      now = next;
      next = after;
    }
    asm volatile("cp.async.wait_group 0;\n" ::: "memory");
  } else if (warp >= MMA_WARP) {
    // ---- products of query tile x ----
    const int x = warp - MMA_WARP;
    if (lane == 0 && x < (t1.valid ? 2 : 1)) {
      const unsigned idesc_pv = tc5::umma_idesc(D) | (1u << 16);      // values: N-major
      const unsigned idesc_qk = 1u << 4 | (unsigned)(HALF >> 3) << 17 | (unsigned)(TILE_ROWS >> 4) << 24;      // e4m3 by e4m3, 32-bit sums
      const uint64_t q_desc = desc_kmajor(q_tiles + x * 2 * CODE_TILE), k_desc = desc_kmajor(k_tiles), v_desc = desc_mnmajor(v_tiles, KEYS * 128);
      auto scores = [&](int i, int h) {
        const uint64_t kb = k_desc + (uint64_t)((i % K_STAGES) * (CODE_TILE >> 4) + h * (HALF * 128 >> 4));
#pragma unroll
        for (int part = 0; part < 2; ++part)
#pragma unroll
          for (int kk = 0; kk < D / 32; ++kk)
            mma_codes(tmem + COL_S + x * KEYS + h * HALF, q_desc + (uint64_t)(part * (CODE_TILE >> 4) + 2 * kk), kb + (uint64_t)(2 * kk), idesc_qk,
                      (part | kk) != 0 ? 1u : 0u);
      };
      // 16 keys of an N-major tile: 2,048 bytes
      auto products = [&](int i, int h, bool first) {
        const uint64_t vb = v_desc + (uint64_t)((i % V_STAGES) * (V_BYTES >> 4) + h * (HALF * 128 >> 4));
#pragma unroll
        for (int kk = 0; kk < HALF / 16; ++kk)
          mma_ts(tmem + COL_O + x * 128, tmem + COL_S + x * KEYS + h * HALF + kk * 8, vb + (uint64_t)(kk * (2048 >> 4)), idesc_pv,
                 (first && kk == 0) ? 0u : 1u);
      };
      bool ok = wait(q_full + x, 0, abort_flag) && wait(k_full, 0, abort_flag);
      if (ok) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
        for (int h = 0; h < 2; ++h)
          if (active(x, 0)) {
            scores(0, h);
            tc5::umma_commit(s_full + 2 * x + h);
          }
        tc5::umma_commit(freed);
      }
      unsigned count = 0;
      for (int i = 0; i < steps && ok; ++i) {
        const bool more = i + 1 < steps, on = active(x, i), next = more && active(x, i + 1);
        // Both were asked for long ago.  A step without anything of x waits too, so that no event is arrived at before
        // the one four earlier is over.
        ok = wait(v_full + i % V_STAGES, (i / V_STAGES) & 1, abort_flag) &&
             (!more || wait(k_full + (i + 1) % K_STAGES, ((i + 1) / K_STAGES) & 1, abort_flag));
#pragma unroll
        for (int h = 0; h < 2 && ok; ++h) {
          if (on) ok = wait(p_full + 2 * x + h, count & 1, abort_flag);
          if (!ok) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          if (on) products(i, h, count == 0 && h == 0);
          // over the weights that the products read: the tensor core runs them afterwards
          if (next) scores(i + 1, h);
          if (on || next) tc5::umma_commit(s_full + 2 * x + h);
        }
        count += on ? 1u : 0u;
        if (ok && more) tc5::umma_commit(freed + ((i + 1) & 3));
      }
      tc5::umma_commit(o_full + x);
      // a role that gave up: what was issued is over before tensor memory is given back
      for (unsigned n = 0; !ok && n < WAIT_TRIES && !tc5::mbar_try_wait(o_full + x, 0); ++n) {}
    }
    __syncwarp();          // the warp is whole again before barriers and tensor memory
  } else {
    // ---- softmax: a thread a row of query tile x ----
    const int x = warp >> 2;
    const QueryTile& mine = x == 0 ? t0 : t1;
    const int quarter = warp & 3;                      // the quarter of tensor memory this warp may touch
    const int r = quarter * 32 + lane, row = mine.row0 + r;
    const bool row_valid = row < rows;
    const int pos = row_valid ? e.start + row / p.groups : -1;
    const unsigned lane_addr = tmem + ((unsigned)(quarter * 32) << 16);
    const unsigned s_addr = lane_addr + COL_S + x * KEYS, o_addr = lane_addr + COL_O + x * 128;
    const int row_lo = p.window > 0 ? max(0, pos - p.window + 1) : 0;
    const int tile_lo = p.window > 0 ? max(0, mine.pos_last - p.window + 1) : 0;        // first key all rows see
    // The queries of this warp's 32 rows: D / 8 lanes take a row, a lane eight elements of it; four rounds' loads at a
    // time, the next four on their way meanwhile.  In half precision, which holds a scaled row exactly but for what is
    // below 2^-14, under the second part's steps of 2^-9.
    constexpr int Q_LANES = D / 8, Q_ROWS = 32 / Q_LANES, Q_ROUNDS = 32 / Q_ROWS, BATCH = 4;
    float factor = 0.f;
    if (mine.valid) {
      const int c = lane % Q_LANES;
      // the rows of a lane are Q_ROWS apart; past the last one it stays
      int from = mine.row0 + quarter * 32 + lane / Q_LANES;
      const int token_step = Q_ROWS / p.groups, g_step = Q_ROWS - token_step * p.groups;
      int token = min(from, rows - 1) / p.groups, g = min(from, rows - 1) - token * p.groups;
      const bf16* base = p.q + (size_t)e.tok0 * p.q_stride + (size_t)kvh * p.groups * D + 8 * c;
      uint2 held[BATCH][2];
      auto load = [&]() {
#pragma unroll
        for (int n = 0; n < BATCH; ++n) {
          const uint2* src = reinterpret_cast<const uint2*>(base + (size_t)token * p.q_stride + g * D);
          held[n][0] = src[0];                         // rows are multiples of four elements apart
          held[n][1] = src[1];
          from += Q_ROWS;
          if (from < rows) {
            token += token_step;
            g += g_step;
            if (g >= p.groups) { g -= p.groups; ++token; }
          }
        }
      };
      load();
#pragma unroll 1
      for (int n0 = 0; n0 < Q_ROUNDS; n0 += BATCH) {
        unsigned here[BATCH][4];
#pragma unroll
        for (int n = 0; n < BATCH; ++n) { here[n][0] = held[n][0].x; here[n][1] = held[n][0].y; here[n][2] = held[n][1].x; here[n][3] = held[n][1].y; }
        if (n0 + BATCH < Q_ROUNDS) load();
#pragma unroll
        for (int n = 0; n < BATCH; ++n) {
          const int at = quarter * 32 + (n0 + n) * Q_ROWS + lane / Q_LANES;
          unsigned two = 0u;                           // largest |x| of both halves of the words, as bits
#pragma unroll
          for (int k = 0; k < 4; ++k) two = __vmaxu2(two, here[n][k] & 0x7fff7fffu);
          unsigned big = max(two & 0xffff0000u, two << 16);
#pragma unroll
          for (int o = Q_LANES / 2; o > 0; o >>= 1) big = max(big, __shfl_xor_sync(0xffffffffu, big, o));
          const bool finite = big < 0x7f800000u;
          const int ex = finite ? kv8_row_exponent(big) : 0;
          const float down = __int_as_float((127 - ex) << 23);
          unsigned hi[4], lo[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const __half2 v = __floats2half2_rn(__uint_as_float(here[n][k] << 16) * down, __uint_as_float(here[n][k] & 0xffff0000u) * down);
            hi[k] = kv8_codes_of_half2(v);
            const unsigned back = kv8_half2((unsigned short)hi[k]);
            lo[k] = kv8_codes_of_half2(__hsub2(v, *reinterpret_cast<const __half2*>(&back)));
          }
          unsigned char* part = q_tiles + x * 2 * CODE_TILE + code_offset(at, c >> 1) + (c & 1) * 8;
          *reinterpret_cast<uint2*>(part) = make_uint2(__byte_perm(hi[0], hi[1], 0x5410), __byte_perm(hi[2], hi[3], 0x5410));
          *reinterpret_cast<uint2*>(part + CODE_TILE) = make_uint2(__byte_perm(lo[0], lo[1], 0x5410), __byte_perm(lo[2], lo[3], 0x5410));
          // what a score is multiplied by, in log2 units, goes to the lane whose row it is
          const float up = finite ? p.scale_log2 * __int_as_float((127 + ex) << 23) : kv8_scale(KV8_NAN);
          const float got = __shfl_sync(0xffffffffu, up, (lane % Q_ROWS) * Q_LANES);
          if (lane / Q_ROWS == n0 + n) factor = got;
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) arrive(q_full + x);
      // Never zero, because masked scores, minus infinity by then, are multiplied too: products are below 2^90, so what a
      // factor of 2^-126 leaves is nothing.
      if (factor < 0x1p-126f) factor = 0x1p-126f;
    }
    float m = -INFINITY, l = 0.f;
    bool ok = mine.valid;
    unsigned count = 0;                // tiles of this query tile so far
    // s_full[x][h] is arrived at by one commit before the first step, with its scores, and by one in every step that has
    // products or the next step's scores of x, when both are done
    unsigned commits = active(x, 0) ? 1u : 0u;
    for (int i = 0; i < steps && ok; ++i) {
      const bool on = active(x, i), next = i + 1 < steps && active(x, i + 1);
      if (!on) {
        commits += next ? 1u : 0u;
        continue;
      }
      // the keys' barrier too: what it published, their scales, is read here (its next phase but one needs these weights)
      ok = __all_sync(0xffffffffu, wait(k_full + i % K_STAGES, (i / K_STAGES) & 1, abort_flag));
#pragma unroll 1
      for (int h = 0; h < 2 && ok; ++h) {
        ok = __all_sync(0xffffffffu, wait(s_full + 2 * x + h, (commits - 1) & 1, abort_flag));
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const int key0 = walk.tile(begin + i) * KEYS + h * HALF;
        const unsigned s_half = s_addr + h * HALF;
        unsigned raw[HALF];
        tmem_ld32(s_half, raw);
        tmem_ld32(s_half + 32, raw + 32);
        tmem_wait_ld();
        const float4* factors = reinterpret_cast<const float4*>(k_factor + (i % CK_STAGES) * KEYS + h * HALF);
#pragma unroll
        for (int j = 0; j < HALF; j += 4) {
          const float4 f = factors[j / 4];
          float a, b;
          unpair(mul2(pair(__uint_as_float(raw[j]), __uint_as_float(raw[j + 1])), pair(f.x, f.y)), a, b);
          raw[j] = __float_as_uint(a);
          raw[j + 1] = __float_as_uint(b);
          unpair(mul2(pair(__uint_as_float(raw[j + 2]), __uint_as_float(raw[j + 3])), pair(f.z, f.w)), a, b);
          raw[j + 2] = __float_as_uint(a);
          raw[j + 3] = __float_as_uint(b);
        }
        // every key of the half visible to every row of the tile?
        const bool clear = key0 + HALF - 1 <= mine.pos_first && mine.row0 + TILE_ROWS <= rows && key0 >= tile_lo;
        if (!clear) {
          const int j_hi = pos - key0, j_lo = row_lo - key0, j_kept = sink_keys - key0;
          if (p.window > 0) {
#pragma unroll
            for (int j = 0; j < HALF; ++j) raw[j] = (j <= j_hi && (j >= j_lo || j < j_kept)) ? raw[j] : 0xff800000u;
          } else {
#pragma unroll
            for (int j = 0; j < HALF; ++j) raw[j] = j <= j_hi ? raw[j] : 0xff800000u;
          }
        }
        float mx0 = -INFINITY, mx1 = -INFINITY, mx2 = -INFINITY, mx3 = -INFINITY;
#pragma unroll
        for (int j = 0; j < HALF; j += 8) {
          mx0 = max3(mx0, __uint_as_float(raw[j]), __uint_as_float(raw[j + 1]));
          mx1 = max3(mx1, __uint_as_float(raw[j + 2]), __uint_as_float(raw[j + 3]));
          mx2 = max3(mx2, __uint_as_float(raw[j + 4]), __uint_as_float(raw[j + 5]));
          mx3 = max3(mx3, __uint_as_float(raw[j + 6]), __uint_as_float(raw[j + 7]));
        }
        const float mx = fmaxf(fmaxf(mx0, mx1), fmaxf(mx2, mx3)) * factor;       // which is positive
        float corr = 1.f;
        if ((mx > m + RESCALE_STEP || m == -INFINITY) && mx != -INFINITY) {
          corr = m == -INFINITY ? 0.f : exp2f(m - mx);
          m = mx;
        }
        const float neg = m == -INFINITY ? 0.f : -m;
        const uint64_t scale2 = pair(factor, factor), base2 = pair(neg, neg);
        uint64_t sum_a = pair(0.f, 0.f), sum_b = sum_a;
#pragma unroll
        for (int c = 0; c < HALF / 32; ++c) {
          unsigned packed[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            float e0, e1;
            unpair(fma2(pair(__uint_as_float(raw[c * 32 + 2 * j]), __uint_as_float(raw[c * 32 + 2 * j + 1])), scale2, base2), e0, e1);
            e0 = exp2_fast(e0);
            e1 = exp2_fast(e1);
            if (j & 1) sum_b = add2(sum_b, pair(e0, e1));
            else sum_a = add2(sum_a, pair(e0, e1));
            packed[j] = pack_bf16(e0, e1);
          }
          tmem_st16(s_half + c * 16, packed);            // over the scores: this row's are all in registers
        }
        float sum0, sum1;
        unpair(add2(sum_a, sum_b), sum0, sum1);
        l = l * corr + (sum0 + sum1);
        if ((count > 0 || h > 0) && __any_sync(0xffffffffu, corr != 1.f)) {
          // the value products so far have to be done: the first half's of this step, or the second half's of the step
          // before, which the scores of this step's second half came with
          ok = __all_sync(0xffffffffu, wait(s_full + 2 * x + (h ^ 1), (h ? commits : commits - 1) & 1, abort_flag));
          if (!ok) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
          for (int c = 0; c < D; c += 16) {
            float o[16];
            tc5::tmem_ld16(o_addr + c, o);
            unsigned bits[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) bits[j] = __float_as_uint(o[j] * corr);
            tmem_st16(o_addr + c, bits);
          }
        }
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) arrive(p_full + 2 * x + h);
      }
      ++count;
      ++commits;
    }
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");       // of weights of a step that was given up
    if (ok) ok = __all_sync(0xffffffffu, wait(o_full + x, 0, abort_flag));
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (ok) {
      const int ur = x * TILE_ROWS + r;
      const float by = pieces > 1 ? 1.f : l == 0.f ? 0.f : 1.f / l;
      float* ws = piece_sums(p, slot, kvh, piece);
      // a finished warp's 32 rows pass through its queries' place, so that whole rows go out
      unsigned char* rows_here = q_tiles + x * 2 * CODE_TILE + quarter * 32 * D * 2;
#pragma unroll 1
      for (int c = 0; c < D; c += 32) {
        unsigned raw[32];
        tmem_ld32(o_addr + c, raw);
        tmem_wait_ld();
#pragma unroll
        for (int j = 0; j < 32; j += 8) {
          float o[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) o[k] = count == 0 ? 0.f : __uint_as_float(raw[j + k]) * by;      // no key of this piece: nothing was summed
          if (pieces == 1) {
            const int chunk = (c + j) >> 3;
            store8(reinterpret_cast<bf16*>(rows_here + lane * D * 2 + ((chunk ^ (lane & 7)) << 4)), o);
          } else if (row_valid) {
            store8(ws + piece_element(p, ur, c + j), o);
          }
        }
      }
      if (pieces == 1) {
        __syncwarp();
        constexpr int LANES = D / 8, AT_ONCE = 32 / LANES;
        const int chunk = lane % LANES;
#pragma unroll 4
        for (int n = lane / LANES; n < 32; n += AT_ONCE) {
          const int out_row = mine.row0 + quarter * 32 + n;
          if (out_row >= rows) break;
          const int token = out_row / p.groups, g = out_row - token * p.groups;
          *reinterpret_cast<uint4*>(p.out + ((size_t)(e.tok0 + token) * p.nkv * p.groups + kvh * p.groups + g) * D + 8 * chunk) =
              *reinterpret_cast<const uint4*>(rows_here + n * D * 2 + ((chunk ^ (n & 7)) << 4));
        }
      } else if (row_valid) {
        ws[(size_t)p.ws_rows * D + 2 * ur] = m;
        ws[(size_t)p.ws_rows * D + 2 * ur + 1] = l;
      }
    }
  }

  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == MMA_WARP) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
  }
  if (threadIdx.x == 0 && *abort_flag) atomicOr(p.status, FE_STATUS_WAIT_TIMEOUT);
}

}  // namespace

namespace kv8 {

int launch_portion(Kv8Attention p, cudaStream_t stream) {
  if (p.spans > 65535) return FE_ERR_TOO_LARGE;
  p.ws_rows = PORTION_UNIT;
  const cudaError_t err = cudaFuncSetAttribute(attn_kv8_portion_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SMEM);
  if (err != cudaSuccess) return (int)err;
  int rc = fe_launch_dependent(attn_kv8_portion_kernel, dim3((unsigned)p.nkv, (unsigned)p.spans, (unsigned)p.slots), dim3(THREADS), SMEM, stream, p);
  if (rc == 0 && p.spans > 1)
    rc = launch_join_portion<PORTION_UNIT, PORTION_TILE>(p, stream);
  return rc;
}

}  // namespace kv8
#endif
