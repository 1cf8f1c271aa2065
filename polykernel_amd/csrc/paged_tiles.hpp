// paged_tiles.hpp -- what the two paged attention kernels share: their arguments, lane
// helpers, and the loads of tiles of 16 keys from pages into LDS.
#pragma once

#include "attention_decode.hpp"
#include "paged.hpp"

namespace pk {
namespace paged {

using att::bf16x8;
using att::f32x16;
using att::f32x4;
using att::i16x4;

struct AttendArgs {
  Heads q, out;
  Cache cache;
  Batch batch;
  int q_heads, causal, window;
  float c2;  // scale * log2(e)
  FastDiv group;  // query heads per key head
};

// The range of keys that new token i of a sequence sees.
__device__ __forceinline__ void key_range(const AttendArgs &g, const Seq &s, int i, int &lo, int &hi) {
  const int limit = s.kv - s.n + i + 1;
  hi = g.causal ? max(0, limit) : s.kv;
  lo = g.window > 0 && limit > g.window ? limit - g.window : 0;
}

// A wave loads tiles of 16 keys, one of every 64 (a step of 4 waves).
constexpr int PT_KEYS = 16, PT_STEP = 64;

// A value that every lane of the wave holds, in a scalar register.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// Inclusive sum over the lanes of a wave: shifts by 1, 2, 4 and 8 inside rows of 16
// lanes, then the last lane of a row to the next row, and of a half to the other half.
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
  return v;
}

// 16 zero bytes that rows which are not there are read from.
__device__ const uint32_t pd_zeros[4] __attribute__((aligned(16))) = {0, 0, 0, 0};

// An LDS address as the number that m0 takes.
__device__ __forceinline__ uint32_t lds_number(const void *p) {
  return (uint32_t)reinterpret_cast<uintptr_t>((lds_void *)p);
}

#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
// dma_lds16 to a numbered address; resource and address in scalar registers.
template <bool NT>
__device__ __forceinline__ void dma_lds16_to(pk_u32x4 rs, uint32_t lds, uint32_t voff) {
  if constexpr (NT)
    asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dwordx4 %1, %2, 0 offen nt lds" : : "s"(lds), "v"(voff), "s"(rs) : "memory", "m0");
  else
    asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" : : "s"(lds), "v"(voff), "s"(rs) : "memory", "m0");
}
// global_load_lds_dwordx4: lane i copies 16 bytes from its own address to lds + 16 i
// (ordered by vm_wait, as dma_lds16).
__device__ __forceinline__ void dma_lds16_at(const void *src, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(lds), "v"(src) : "memory", "m0");
}
#pragma clang diagnostic pop

// Direct-to-LDS loads of a wave's tiles: tile t holds keys [key0 + 64 t, + 16) of one key
// head, 16-byte chunks swizzled for the fragment reads (att::swz_k, att::swz_v).  Keys from
// `hi` on, keys on pages that are not there and dims behind the head's are zero.
//
// A page size that is a multiple of 16 holds a tile in one page (PAGE16): its address is a
// buffer resource whose length ends the tile, so nothing is computed per lane; 64 tiles'
// pages are looked up at a time, a lane each.  Multiples of 8 have a resource for each half
// of the tile (one token of 2 sequences on up to 46000 keys, 2 heads to 6 of 80, in pages of
// 8: 23 us, by rows 27, in pages of 16 18).  Other sizes look up a page per row, 4 tiles at a
// time, every lane has its own address, and lanes without a row read zeros.
// PAGE: what the page size is a multiple of: 16, 8 or 1.  NT: read once, non-temporal.
template <int DP, int PAGE, bool NT>
struct TileLoader {
  static constexpr bool PAGE16 = PAGE == 16;
  static constexpr int CH = DP / 8, RPI = 1024 / (2 * DP), NI = PT_KEYS / RPI, BYTES = PT_KEYS * DP * 2;
  static constexpr int PARTS = PT_KEYS / PAGE, BATCH = 64 / PARTS;  // look-ups of a tile, tiles of a look-up
  uint32_t kvo[NI], vvo[NI];
  const uint16_t *kbase, *vbase;
  int b, key0, count, hi;
  int kpages, vpages;  // of the batch that the last K and the last V tile is in

  // lane's part of instruction i: row i RPI + lane / CH, chunk by its swizzle
  __device__ __forceinline__ static int row_of(int i) { return i * RPI + (int)(threadIdx.x & 63) / CH; }
  __device__ __forceinline__ static int k_chunk(int i) { return att::swz_k<CH>((threadIdx.x & 63) % CH, row_of(i)); }
  __device__ __forceinline__ static int v_chunk(int i) { return (int)((threadIdx.x & 63) % CH) ^ att::swz_v<DP>(row_of(i)); }

  __device__ __forceinline__ explicit TileLoader(const AttendArgs &g) {
#pragma unroll
    for (int i = 0; i < NI; ++i) {  // chunks behind the head dim lie outside every resource
      kvo[i] = 8 * k_chunk(i) < g.cache.dim ? (uint32_t)(row_of(i) * (int)g.cache.k_row * 2 + 16 * k_chunk(i)) : 0x80000000u;
      vvo[i] = 8 * v_chunk(i) < g.cache.dim ? (uint32_t)(row_of(i) * (int)g.cache.v_row * 2 + 16 * v_chunk(i)) : 0x80000000u;
    }
  }
  __device__ __forceinline__ int look_up(const AttendArgs &g, int t) const {
    const int lane = threadIdx.x & 63;
    const int key = key0 + (t + lane / PARTS) * PT_STEP + lane % PARTS * PAGE;
    return key < hi ? page_of(g.batch, g.cache, b, key) : -1;
  }
  __device__ __forceinline__ void begin(const AttendArgs &g, int b_, int hk, int key0_, int count_, int hi_) {
    b = b_, key0 = key0_, count = count_, hi = hi_;
    kbase = g.cache.k + hk * g.cache.k_head;
    vbase = g.cache.v + hk * g.cache.v_head;
    kpages = vpages = look_up(g, 0);
  }
  // Tiles of K, and of V, in order from 0 to the LDS address `to`; tiles from `count` on load
  // nothing (as many instructions, of no length).
  __device__ __forceinline__ void issue_k(const AttendArgs &g, int t, uint32_t to) {
    if (t % BATCH == 0 && t > 0 && t < count) kpages = look_up(g, t);
    load(g, t, kpages, kbase, g.cache.k_page, g.cache.k_row, kvo, [](int i) { return k_chunk(i); }, to);
  }
  __device__ __forceinline__ void issue_v(const AttendArgs &g, int t, uint32_t to) {
    if (t % BATCH == 0 && t > 0 && t < count) vpages = look_up(g, t);
    load(g, t, vpages, vbase, g.cache.v_page, g.cache.v_row, vvo, [](int i) { return v_chunk(i); }, to);
  }
  // The tile's rows from FROM on, `n` of them from row `row` of a page (none: a resource of no
  // length), to row TO of the tile.  The resource begins where row 0 of the tile would be.
  template <int FROM = 0, int TO = PT_KEYS>
  __device__ __forceinline__ static void load_rows(const AttendArgs &g, int page, int row, int n, const uint16_t *base,
                                                   int64_t page_stride, int64_t row_stride, const uint32_t (&offset)[NI],
                                                   uint32_t to) {
    uint64_t p = reinterpret_cast<uint64_t>(base) + 2 * (uint64_t)(uint32_t)page * (uint64_t)page_stride +
                 (uint32_t)row * (uint32_t)(2 * row_stride);
    if constexpr (FROM > 0) p -= (uint32_t)(2 * FROM * row_stride);
    const pk_u32x4 rs = {(uint32_t)uniform((int)(uint32_t)p), (uint32_t)uniform((int)((uint32_t)(p >> 32) & 0xFFFFu)),
                         (uint32_t)uniform(n > 0 ? ((FROM + n - 1) * (int)row_stride + g.cache.dim) * 2 : 0), 0x00020000u};
#pragma unroll
    for (int i = FROM / RPI; i < TO / RPI; ++i) dma_lds16_to<NT>(rs, (uint32_t)uniform((int)to + i * 1024), offset[i]);
  }
  template <typename Chunk>
  __device__ __forceinline__ void load(const AttendArgs &g, int t, int pages, const uint16_t *base, int64_t page_stride,
                                       int64_t row_stride, const uint32_t (&offset)[NI], Chunk chunk, uint32_t to) {
    const int key = key0 + t * PT_STEP, left = t < count ? hi - key : 0;
    if constexpr (PAGE16) {
      const int page = __builtin_amdgcn_readlane(pages, t % BATCH), n = page < 0 ? 0 : min(PT_KEYS, left);
      const int row = n > 0 ? key - (int)(g.cache.page.div(key) * g.cache.page.d) : 0;
      load_rows(g, n > 0 ? page : 0, row, n, base, page_stride, row_stride, offset, to);
    } else if constexpr (PAGE == 8) {
      const int p0 = __builtin_amdgcn_readlane(pages, t % BATCH * 2), p1 = __builtin_amdgcn_readlane(pages, t % BATCH * 2 + 1);
      const int n0 = p0 < 0 ? 0 : min(8, left), n1 = p1 < 0 ? 0 : min(8, left - 8);
      const int row0 = n0 > 0 ? key - (int)(g.cache.page.div(key) * g.cache.page.d) : 0;
      const int row1 = n1 > 0 ? key + 8 - (int)(g.cache.page.div(key + 8) * g.cache.page.d) : 0;
      load_rows<0, 8>(g, n0 > 0 ? p0 : 0, row0, n0, base, page_stride, row_stride, offset, to);
      load_rows<8, 16>(g, n1 > 0 ? p1 : 0, row1, n1, base, page_stride, row_stride, offset, to);
    } else {
      const uint16_t *src[NI];
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int row = row_of(i), page = __shfl(pages, (t % BATCH) * PARTS + row / PAGE, 64);
        const bool is = row < left && page >= 0 && 8 * chunk(i) < g.cache.dim;
        const int at = is ? key + row - (int)(g.cache.page.div(key + row) * g.cache.page.d) : 0;
        src[i] = is ? base + page * page_stride + at * row_stride + 8 * chunk(i) : reinterpret_cast<const uint16_t *>(pd_zeros);
      }
#pragma unroll
      for (int i = 0; i < NI; ++i) dma_lds16_at(src[i], (uint32_t)uniform((int)to + i * 1024));
    }
  }
  // Which keys of tile t (the last one of K issued) are on pages that are there, a bit each.
  __device__ __forceinline__ uint32_t there(int t) const {
    if constexpr (PAGE16) return __builtin_amdgcn_readlane(kpages, t % BATCH) < 0 ? 0u : 0xFFFFu;
    const uint32_t is = (uint32_t)(__ballot(kpages >= 0) >> (PARTS * (t % BATCH)));
    if constexpr (PAGE == 8) return (is & 1 ? 0xFFu : 0u) | (is & 2 ? 0xFF00u : 0u);
    else return is & 0xFFFFu;
  }
};

// The largest exponent fields seen in the halves of words, and whether one is that of an
// infinity or no number.
__device__ __forceinline__ pk_u16x2 exponents(pk_u16x2 most, uint32_t w) {
  return __builtin_elementwise_max(most, __builtin_bit_cast(pk_u16x2, w & 0x7F807F80u));
}
__device__ __forceinline__ bool not_finite(pk_u16x2 most) { return most.x >= 0x7F80 || most.y >= 0x7F80; }

// A hidden key's value that is no number must not meet its zero weight in a product.  Where
// some rows see such a key and others don't, the products take zero for it (`finite`), and
// the rows that see it get it at the end (`add_not_finite`).
__device__ __forceinline__ uint32_t finite(uint32_t w) {
  const uint32_t lo = (w & 0x7F80u) == 0x7F80u ? 0u : 0xFFFFu, hi = (w & 0x7F800000u) == 0x7F800000u ? 0u : 0xFFFF0000u;
  return w & (lo | hi);
}
// Adds the values of key `key` at `at` that are infinite or no number to four sums.
__device__ __forceinline__ void add_not_finite(const uint16_t *at, f32x4 &sum) {
  const att::u32x2 w = *reinterpret_cast<const att::u32x2 *>(at);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t v = (i & 1 ? w[i >> 1] & 0xFFFF0000u : w[i >> 1] << 16);
    if ((v & 0x7F800000u) == 0x7F800000u) sum[i] += __uint_as_float(v);
  }
}
// The values of key `key` of one head, or null where its page is not there.
__device__ __forceinline__ const uint16_t *value_row(const AttendArgs &g, int b, int hk, int key) {
  const int page = page_of(g.batch, g.cache, b, key);
  if (page < 0) return nullptr;
  return g.cache.v + hk * g.cache.v_head + page * g.cache.v_page +
         (key - (int)(g.cache.page.div(key) * g.cache.page.d)) * g.cache.v_row;
}

}  // namespace paged
}  // namespace pk
