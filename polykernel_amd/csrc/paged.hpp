// paged.hpp -- what the rotary, paged append and paged attention kernels share:
// the arguments as the device sees them, the places of tokens and keys, and the
// argument checks of their entry points.
//
// The new tokens of all sequences lie one behind the other; sequence b owns
// tokens [q_start[b], q_start[b + 1]) and kv_len[b] keys with the new ones, the
// key at position p in row p % page_size of page page_table[b][p / page_size].
// The tables live on the device, where no host check sees them, so every kernel
// brings what it reads from them into range first: token ranges into [0, tokens),
// lengths into [0, table_width * page_size], and a page number outside
// [0, pages) stands for rows that are not there.
#pragma once

#include "pk_common.hpp"

namespace pk {
namespace paged {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// Workgroups of 256 threads along one side of a grid: its threads are a 32-bit number.
constexpr int64_t MOST_BLOCKS = INT64_C(0xFFFFFFFF) / 256;

// n / d for 0 <= n < 2^31 by a multiplication: m = ceil(2^(32 + s) / d), s =
// ceil(log2 d), less 2^32, so that q = (umulhi(n, m) + n) >> s; exact since the
// error n (m' d - 2^(32 + s)) / (d 2^(32 + s)) stays below 1 / d for n < 2^32
// (Granlund and Montgomery 1994); the sum does not overflow for n < 2^31.
struct FastDiv {
  uint32_t d, mul, shift;
  FastDiv() = default;
  explicit FastDiv(uint32_t div) : d(div), mul(0), shift(0) {
    while ((uint64_t(1) << shift) < div) ++shift;
    mul = (uint32_t)(((uint64_t(1) << 32) * ((uint64_t(1) << shift) - div)) / div + 1);
  }
  __device__ __forceinline__ uint32_t div(uint32_t n) const { return (__umulhi(n, mul) + n) >> shift; }
};

// A tensor of heads: element (b, t, h, d) at data + b * batch + t * token + h * head + d.
struct Heads {
  uint16_t *data;
  int64_t batch, token, head;
};

struct Cache {
  uint16_t *k, *v;
  int64_t k_page, k_head, k_row, v_page, v_head, v_row;
  int pages, heads, dim;
  FastDiv page;  // rows per page
};

struct Batch {
  const int32_t *page_table, *q_start, *kv_len;
  int64_t table_stride;
  int sequences, tokens, capacity;  // capacity: table_width * page_size
};

struct Seq {
  int q0, n, kv;  // first new token, new tokens, keys
};

__device__ __forceinline__ Seq sequence(const Batch &g, int b) {
  Seq s;
  if (g.q_start) {
    s.q0 = min(max(g.q_start[b], 0), g.tokens);
    s.n = min(max(g.q_start[b + 1], s.q0), g.tokens) - s.q0;
  } else {
    s.q0 = b;
    s.n = 1;
  }
  s.kv = min(max(g.kv_len[b], 0), g.capacity);
  return s;
}

// The sequence that token t belongs to, by the calling wave (64 entries a step):
// the number of sequences that end at or before t.  -1 behind the last one.
__device__ __forceinline__ int sequence_of(const Batch &g, int t) {
  if (!g.q_start) return t < g.sequences ? t : -1;
  const int lane = threadIdx.x & 63;
  int n = 0;
  for (int b0 = 0; b0 < g.sequences; b0 += 64) {
    const bool before = b0 + lane < g.sequences && g.q_start[b0 + lane + 1] <= t;
    n += __popcll(__ballot(before));
  }
  return n < g.sequences && g.q_start[n] <= t ? n : -1;
}

// The page of position p (0 <= p < capacity) as the table has it, and that number where
// there is such a page, else -1.
__device__ __forceinline__ int page_number(const Batch &g, const Cache &c, int b, int p) {
  return g.page_table[b * g.table_stride + c.page.div(p)];
}
__device__ __forceinline__ int page_or_none(const Cache &c, int page) { return (unsigned)page < (unsigned)c.pages ? page : -1; }
__device__ __forceinline__ int page_of(const Batch &g, const Cache &c, int b, int p) {
  return page_or_none(c, page_number(g, c, b, p));
}

// ---- argument checks -------------------------------------------------------
int check_cache(const char *who, const pk_paged_cache *cache, Cache *out);
int check_batch(const char *who, const pk_paged_batch *batch, const pk_paged_cache *cache, Batch *out);

inline bool strides8(int64_t a, int64_t b, int64_t c = 0) { return ((a | b | c) & 7) == 0; }

}  // namespace paged
}  // namespace pk
