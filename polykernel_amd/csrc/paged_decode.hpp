// paged_decode.hpp -- attention of few new tokens per sequence over a paged cache.
//
// What bounds it: keys and values are read once for the G query heads that share
// them (and the few new tokens), so the time is that of streaming them from HBM.
//
// A row is a (token, query head of the group) pair; 16 MT rows of one sequence and
// key head are one item.  Both products run on the matrix units, transposed: S^T =
// K Q^T (16x16x32, keys x rows) leaves each lane one row and 4 keys of 16, which is
// the B operand of O^T = V^T P^T (16x16x16), its A operand read from V's rows in LDS
// by transposing reads.  So P stays in registers; P is split into two bf16 halves
// (2^-17 relative), which costs nothing under the memory time.
//
// Memory: every wave has a ring of its own of SL tiles of 16 keys in LDS, filled by
// direct-to-LDS loads (16 bytes a lane, chunks swizzled at the source), with no
// barrier in the loop.  A tile of a page size that is a multiple of 16 lies in one
// page: its base address is a buffer resource whose length ends the tile at the last
// key, so rows behind it read as zero and stale pages never reach a product.  Other
// page sizes look up a page per row and point rows that are not there at zeros.
//
// Work: the steps (64 keys of an item, 16 per wave) of all items lie on one line,
// which the workgroups cut into equal parts whatever the sequences' lengths; each
// finds its part from kv_len and q_start alone, so a captured call follows them.  An
// item cut between workgroups leaves its parts in the workspace, and
// paged_decode_merge_kernel adds them in the order of the workgroups.
#pragma once

#include "attention_decode.hpp"
#include "paged.hpp"

namespace pk {
namespace paged {

using att::bf16x8;
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

constexpr int PD_WAVES = 4, PD_THREADS = PD_WAVES * 64, PD_TILE = 16, PD_STEP = PD_WAVES * PD_TILE;

// Bytes of one workgroup's partial state: 16 MT rows of DP sums, and (maximum, sum).
constexpr size_t pd_part_floats(int DP, int MT) { return (size_t)16 * MT * (DP + 2); }

struct DecodeArgs {
  AttendArgs a;
  float *parts;      // two partial states per workgroup
  int least;         // steps per workgroup, where there are enough for all
};

// A value that every lane of the wave holds, in scalar registers.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ int64_t uniform(int64_t v) {
  return (int64_t)((uint64_t)(uint32_t)uniform((int)(uint32_t)v) | (uint64_t)(uint32_t)uniform((int)(v >> 32)) << 32);
}

// The line of steps: what sequence b adds, and a place on it.
struct Line {
  int tiles, steps, klo;  // row tiles, steps of each item, first key of step 0
  int64_t units;
};
template <int ROWS>
__device__ __forceinline__ Line line_of(const AttendArgs &g, const Seq &s) {
  Line l{0, 0, 0, 0};
  if (s.n <= 0) return l;
  int lo, hi, lo2, hi2;
  key_range(g, s, 0, lo, hi);
  key_range(g, s, s.n - 1, lo2, hi2);
  l.klo = lo & ~(PD_TILE - 1);
  l.tiles = (int)(((int64_t)s.n * (int)g.group.d + ROWS - 1) / ROWS);
  l.steps = max(1, (hi2 - l.klo + PD_STEP - 1) / PD_STEP);
  l.units = (int64_t)l.tiles * g.cache.heads * l.steps;
  return l;
}

struct Place {
  int64_t total, first, last;  // of the line; this workgroup's part [first, last)
  int workers;
  int b;                       // sequence of `first`
  int64_t in_seq;              // first, from the sequence's own start
  __device__ __forceinline__ int64_t part(int w) const { return w * total / workers; }
  // the workgroup whose part unit u is in
  __device__ __forceinline__ int worker_of(int64_t u) const { return (int)(((u + 1) * workers - 1) / total); }
};
// Where workgroup w's part begins, found by every wave for itself: lane l adds up the
// sequences [l, l + 1) * ceil(B / 64), and a scan over the lanes gives each its offset.
template <int ROWS>
__device__ __forceinline__ bool find_place(const DecodeArgs &d, int w, Place &p) {
  const AttendArgs &g = d.a;
  const int lane = threadIdx.x & 63, B = g.batch.sequences;
  const int per = (B + 63) / 64;
  int64_t mine = 0;
  for (int i = 0; i < per; ++i) {
    const int b = lane * per + i;
    if (b < B) mine += line_of<ROWS>(g, sequence(g.batch, b)).units;
  }
  int64_t incl = mine;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t up = __shfl_up(incl, o, 64);
    if (lane >= o) incl += up;
  }
  p.total = uniform(__shfl(incl, 63, 64));
  p.workers = (int)min((int64_t)gridDim.x, max((int64_t)1, p.total / d.least));
  if (w >= p.workers || p.total == 0) return false;
  p.first = p.part(w);
  p.last = p.part(w + 1);
  const uint64_t holds = __ballot(p.first >= incl - mine && p.first < incl);
  const int l = __ffsll((unsigned long long)holds) - 1;
  int64_t at = uniform(__shfl(incl - mine, l, 64));
  int b = uniform(l * per);
  for (;; ++b) {
    const int64_t n = line_of<ROWS>(g, sequence(g.batch, b)).units;
    if (p.first < at + n) break;
    at += n;
  }
  p.b = b;
  p.in_seq = p.first - at;
  return true;
}

template <int DP>
struct DecodeShape {
  static constexpr int CH = DP / 8, RPI = 1024 / (2 * DP), NI = PD_TILE / RPI, TB = PD_TILE * DP * 2;
  static constexpr int SL = DP == 64 ? 4 : 2;
  static constexpr int WAVE = 2 * SL * TB;  // ring of a wave
  static constexpr int PS = DP + 4;         // row stride of a state in LDS, floats
  static constexpr int STATE = 16 * PS * 4;  // a wave's 16 rows of sums, then its (maximum, sum) of up to 64 rows
  static_assert(STATE + 64 * 8 <= WAVE, "a wave's state lies in its ring");
};

// 16 zero bytes that rows which are not there are read from.
__device__ const uint32_t pd_zeros[4] __attribute__((aligned(16))) = {0, 0, 0, 0};

#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
// global_load_lds_dwordx4: lane i copies 16 bytes from its own address to lds + 16 i
// (ordered by vm_wait, as dma_lds16).
__device__ __forceinline__ void dma_lds16_at(const void *src, const void *lds) {
  const int m0 = __builtin_amdgcn_readfirstlane((int)(uint32_t)reinterpret_cast<uintptr_t>((lds_void *)lds));
  asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(m0), "v"(src) : "memory", "m0");
}
#pragma clang diagnostic pop

// `n` such that a bit pattern is no number or infinite in either half of a word.
__device__ __forceinline__ bool word_not_finite(uint32_t w) {
  return (w & 0x7F80u) == 0x7F80u || (w & 0x7F800000u) == 0x7F800000u;
}

// A value (low half of w) for the passes over a tile with values that are no numbers: 0
// keeps the finite ones, 1 and 2 hold 2^127 and -2^127 where it is +inf and -inf, both
// for a NaN.
__device__ __forceinline__ uint32_t apart_half(uint32_t w, int pass) {
  const bool finite = (w & 0x7F80u) != 0x7F80u, nan = !finite && (w & 0x7Fu);
  if (pass == 0) return finite ? w & 0xFFFFu : 0u;
  if (pass == 1) return nan || (w & 0xFFFFu) == 0x7F80u ? 0x7F00u : 0u;
  return nan || (w & 0xFFFFu) == 0xFF80u ? 0xFF00u : 0u;
}

template <int DP, int MT, bool PAGE16>
__device__ __forceinline__ void paged_decode_body(const DecodeArgs &d) {
  using S = DecodeShape<DP>;
  constexpr int CH = S::CH, RPI = S::RPI, NI = S::NI, TB = S::TB, SL = S::SL, PS = S::PS;
  constexpr int ROWS = 16 * MT, KS = DP / 32, DB = DP / 16;
  // many query fragments are read from LDS at each tile (the waves share them), few stay in registers
  constexpr bool QLDS = MT * KS > 8;
  __shared__ __attribute__((aligned(1024))) uint8_t ring[PD_WAVES * S::WAVE + (QLDS ? ROWS * DP * 2 : 0)];
  uint8_t *const qs = ring + PD_WAVES * S::WAVE;
  auto ml = [&](int w, int r) __attribute__((always_inline)) {
    return reinterpret_cast<float *>(ring + w * S::WAVE + S::STATE) + 2 * r;
  };
  const AttendArgs &g = d.a;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, grp = lane >> 4;
  const int D = g.cache.dim;
  uint8_t *const mine = ring + wid * S::WAVE;  // K slots, then V slots

  Place at;
  if (!find_place<ROWS>(d, blockIdx.x, at)) return;

  // source offset of instruction i: row i RPI + lane / CH, swizzled chunk; chunks
  // behind the head dim lie outside every resource
  uint32_t kvo[NI], vvo[NI];
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int row = i * RPI + lane / CH, sl = lane % CH;
    const int kc = att::swz_k<CH>(sl, row), vc = sl ^ att::swz_v<DP>(row);
    kvo[i] = 8 * kc < D ? (uint32_t)(row * (int)g.cache.k_row * 2 + 16 * kc) : 0x80000000u;
    vvo[i] = 8 * vc < D ? (uint32_t)(row * (int)g.cache.v_row * 2 + 16 * vc) : 0x80000000u;
  }

  int64_t u = at.first, in_seq = at.in_seq;
  int b = at.b;
  bool first_segment = true;
  while (u < at.last) {
    const Seq s = sequence(g.batch, b);
    const Line ln = line_of<ROWS>(g, s);
    if (in_seq >= ln.units) {
      in_seq = 0;
      ++b;
      continue;
    }
    const int item = (int)(in_seq / ln.steps), st0 = (int)(in_seq - (int64_t)item * ln.steps);
    const int nst = (int)min((int64_t)(ln.steps - st0), at.last - u);
    const int hk = item / ln.tiles, tile = item - hk * ln.tiles;
    const int row0 = tile * ROWS, rows = min(ROWS, s.n * (int)g.group.d - row0);

    // the keys that all rows of the tile see, and those that any does
    int lo_any, hi_all, lo_all, hi_any;
    key_range(g, s, (int)g.group.div(row0), lo_any, hi_all);
    key_range(g, s, (int)g.group.div(row0 + rows - 1), lo_all, hi_any);
    int lo[MT], hi[MT];
    bf16x8 qf[QLDS ? 1 : MT][KS];
    if constexpr (QLDS) {
      for (int x = tid; x < ROWS * CH; x += PD_THREADS) {
        const int r = x / CH, c = x % CH;
        const int i = (int)g.group.div(row0 + min(r, rows - 1)), h = hk * (int)g.group.d + row0 + min(r, rows - 1) - i * (int)g.group.d;
        att::u32x4 v = {0, 0, 0, 0};
        if (8 * c < D) v = *reinterpret_cast<const att::u32x4 *>(g.q.data + (int64_t)(s.q0 + i) * g.q.token + h * g.q.head + 8 * c);
        if (g.c2 < 0.f) v ^= 0x80008000u;
        *reinterpret_cast<att::u32x4 *>(qs + r * DP * 2 + 16 * att::swz_k<CH>(c, r)) = v;
      }
      __syncthreads();
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int r = min(row0 + 16 * m + col, row0 + rows - 1);
      const int i = (int)g.group.div(r), h = hk * (int)g.group.d + r - i * (int)g.group.d;
      key_range(g, s, i, lo[m], hi[m]);
      if constexpr (QLDS) continue;
      const uint16_t *qp = g.q.data + (int64_t)(s.q0 + i) * g.q.token + h * g.q.head + 8 * grp;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        att::u32x4 v = {0, 0, 0, 0};
        if (32 * k + 8 * grp < D) v = *reinterpret_cast<const att::u32x4 *>(qp + 32 * k);
        if (g.c2 < 0.f) v ^= 0x80008000u;
        qf[QLDS ? 0 : m][k] = __builtin_bit_cast(bf16x8, v);
      }
    }
    const float c2 = fabsf(g.c2);

    // ---- the wave's tiles: keys [key0 + 64 t, + 16)
    const int key0 = ln.klo + st0 * PD_STEP + wid * PD_TILE;
    const uint16_t *kbase = g.cache.k + hk * g.cache.k_head, *vbase = g.cache.v + hk * g.cache.v_head;
    // pages looked up 64 tiles (PAGE16) or 4 tiles (a row a lane) at a time
    constexpr int BATCH = PAGE16 ? 64 : 4;
    int pages = -1;
    auto look_up = [&](int t) __attribute__((always_inline)) {
      const int key = PAGE16 ? key0 + (t + lane) * PD_STEP : key0 + (t + (lane >> 4)) * PD_STEP + col;
      pages = key < hi_any ? page_of(g.batch, g.cache, b, key) : -1;
    };
    auto keys_of = [&](int t) __attribute__((always_inline)) { return t < nst ? hi_any - (key0 + t * PD_STEP) : 0; };
    auto issue = [&](int t) __attribute__((always_inline)) {
      if (t % BATCH == 0 && t < nst) look_up(t);
      const int key = key0 + t * PD_STEP;
      uint8_t *ks = mine + (t % SL) * TB, *vs = mine + (SL + t % SL) * TB;
      if constexpr (PAGE16) {
        const int page = __builtin_amdgcn_readlane(pages, t % BATCH), n = page < 0 ? 0 : min(PD_TILE, keys_of(t));
        const int row = n > 0 ? key - (int)(g.cache.page.div(key) * g.cache.page.d) : 0;
        const int64_t pg = n > 0 ? page : 0;
        const pk_u32x4 kr = rsrc_words(kbase + pg * g.cache.k_page + row * g.cache.k_row,
                                       n > 0 ? (uint32_t)(((n - 1) * (int)g.cache.k_row + D) * 2) : 0u);
        const pk_u32x4 vr = rsrc_words(vbase + pg * g.cache.v_page + row * g.cache.v_row,
                                       n > 0 ? (uint32_t)(((n - 1) * (int)g.cache.v_row + D) * 2) : 0u);
#pragma unroll
        for (int i = 0; i < NI; ++i) dma_lds16<true>(kr, ks + i * 1024, kvo[i], 0);
#pragma unroll
        for (int i = 0; i < NI; ++i) dma_lds16<true>(vr, vs + i * 1024, vvo[i], 0);
      } else {
        const int n = keys_of(t);
        const uint16_t *kp[NI], *vp[NI];
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          const int row = i * RPI + lane / CH, sl = lane % CH;
          const int page = __shfl(pages, (t % BATCH) * 16 + row, 64);
          const int kc = att::swz_k<CH>(sl, row), vc = sl ^ att::swz_v<DP>(row);
          const bool there = row < n && page >= 0;
          const int at_row = there ? key + row - (int)(g.cache.page.div(key + row) * g.cache.page.d) : 0;
          const uint16_t *zero = reinterpret_cast<const uint16_t *>(pd_zeros);
          kp[i] = there && 8 * kc < D ? kbase + page * g.cache.k_page + at_row * g.cache.k_row + 8 * kc : zero;
          vp[i] = there && 8 * vc < D ? vbase + page * g.cache.v_page + at_row * g.cache.v_row + 8 * vc : zero;
        }
#pragma unroll
        for (int i = 0; i < NI; ++i) dma_lds16_at(kp[i], ks + i * 1024);
#pragma unroll
        for (int i = 0; i < NI; ++i) dma_lds16_at(vp[i], vs + i * 1024);
      }
    };
    // keys of tile t that are there, a bit each
    auto there_of = [&](int t, int page_word) __attribute__((always_inline)) -> uint32_t {
      if constexpr (PAGE16) return __builtin_amdgcn_readlane(page_word, t % BATCH) < 0 ? 0u : 0xFFFFu;
      else return (uint32_t)(__ballot(page_word >= 0) >> (16 * (t % BATCH))) & 0xFFFFu;
    };

    float m_run[MT], l_run[MT];
    f32x4 acc[MT][DB];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      m_run[m] = -INFINITY;
      l_run[m] = 0.f;
#pragma unroll
      for (int e = 0; e < DB; ++e) acc[m][e] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    // which keys of the next SL tiles are there, 16 bits each: looked up when a tile is issued
    uint64_t there = 0;
#pragma unroll
    for (int t = 0; t < SL; ++t) {
      issue(t);
      there |= (uint64_t)there_of(t, pages) << (16 * t);
    }
#pragma unroll 1
    for (int t = 0; t < nst; ++t) {
      {
        const int o = t % SL;
        const int key = key0 + t * PD_STEP;
        uint8_t *ks = mine + o * TB, *vs = mine + (SL + o) * TB;
        const uint32_t here = (uint32_t)there & 0xFFFFu;
        const bool any = key < hi_any && here != 0;
        const bool masked = key < lo_all || key + PD_TILE > hi_all || here != 0xFFFFu;
        f32x4 sc[MT];
        vm_wait<NI + 2 * NI * (SL - 1)>();
        if (any) {
          bf16x8 kf[KS];
#pragma unroll
          for (int k = 0; k < KS; ++k)
            kf[k] = __builtin_bit_cast(
                bf16x8, *reinterpret_cast<const att::u32x4 *>(ks + col * DP * 2 + 16 * att::swz_k<CH>(4 * k + grp, col)));
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            sc[m] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < KS; ++k) {
              if constexpr (QLDS)
                qf[0][k] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const att::u32x4 *>(
                                                          qs + (16 * m + col) * DP * 2 + 16 * att::swz_k<CH>(4 * k + grp, col)));
              sc[m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[k], qf[QLDS ? 0 : m][k], sc[m], 0, 0, 0);
            }
          }
        }
        vm_wait<2 * NI * (SL - 1)>();
        if (any) {
          uint32_t hid[MT];  // hidden keys of this lane's four
          i16x4 phi[MT], plo[MT];
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            hid[m] = 0;
            if (masked) {
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int kk = 4 * grp + i;
                if (key + kk < lo[m] || key + kk >= hi[m] || !(here >> kk & 1)) {
                  sc[m][i] = -INFINITY;
                  hid[m] |= 1u << i;
                }
              }
            }
            float top = fmaxf(fmaxf(sc[m][0], sc[m][1]), fmaxf(sc[m][2], sc[m][3]));
            top = xor32_max(top);
            float a0, a1;
            att::xor16_pair(top, top, a0, a1);
            top = fmaxf(a0, a1);
            // the maximum in the exponent follows once it is 2^8 behind: sums of p v / p do not depend on it
            if (__any((top - m_run[m]) * c2 > 8.f)) {
              const float m_new = fmaxf(m_run[m], top);
              const float alpha = m_run[m] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m_run[m] - m_new) * c2);
              m_run[m] = m_new;
              l_run[m] *= alpha;
#pragma unroll
              for (int e = 0; e < DB; ++e) acc[m][e] *= alpha;
            }
            const float mc = m_run[m] == -INFINITY ? 0.f : m_run[m] * c2;
            float p[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) p[i] = __builtin_amdgcn_exp2f(fmaf(sc[m][i], c2, -mc));
            l_run[m] += (p[0] + p[1]) + (p[2] + p[3]);
            const uint32_t h0 = pack_bf(p[0], p[1]), h1 = pack_bf(p[2], p[3]);
            phi[m] = __builtin_bit_cast(i16x4, (att::u32x2{h0, h1}));
            plo[m] = __builtin_bit_cast(i16x4, (att::u32x2{pack_bf(p[0] - lo_bf(h0), p[1] - hi_bf(h0)),
                                                           pack_bf(p[2] - lo_bf(h1), p[3] - hi_bf(h1))}));
          }
          // A hidden key's value that is no number must not meet its zero weight: such a tile is
          // multiplied with those values at zero, then with each infinity (a NaN as both signs) at
          // 2^127 and the keys that a row sees at 2^127: sums overflow to what the row sees.
          bool apart = false;
          if (masked) {
            bool odd = false;
#pragma unroll
            for (int i = 0; i < NI; ++i) {
              const att::u32x4 w = *reinterpret_cast<const att::u32x4 *>(vs + i * 1024 + 16 * lane);
#pragma unroll
              for (int e = 0; e < 4; ++e) odd |= word_not_finite(w[e]);
            }
            apart = __any(odd);
          }
#pragma unroll 1
          for (int pass = apart ? 0 : 3;; ++pass) {
            if (pass < 3) {  // the tile as it was is kept in the slot of its keys
#pragma unroll 1
              for (int i = 0; i < NI; ++i) {
                const int x = i * 1024 + 16 * lane;
                att::u32x4 w = *reinterpret_cast<const att::u32x4 *>((pass ? ks : vs) + x);
                if (pass == 0) *reinterpret_cast<att::u32x4 *>(ks + x) = w;
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = apart_half(w[e], pass) | apart_half(w[e] >> 16, pass) << 16;
                *reinterpret_cast<att::u32x4 *>(vs + x) = w;
              }
              if (pass > 0) {
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                  const uint32_t h = hid[m];
                  phi[m] = __builtin_bit_cast(i16x4, (att::u32x2{(h & 1 ? 0u : 0x7F00u) | (h & 2 ? 0u : 0x7F000000u),
                                                                 (h & 4 ? 0u : 0x7F00u) | (h & 8 ? 0u : 0x7F000000u)}));
                  plo[m] = i16x4{0, 0, 0, 0};
                }
              }
            }
#pragma unroll
            for (int e = 0; e < DB; ++e) {
              const int key_r = 4 * grp + (col >> 2), c = 2 * e + (col & 3) / 2;
              const i16x4 vf = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                  (att::lds_i16x4 *)(vs + key_r * DP * 2 + 16 * (c ^ att::swz_v<DP>(key_r)) + 8 * (col & 1)));
#pragma unroll
              for (int m = 0; m < MT; ++m) {
                acc[m][e] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(vf, phi[m], acc[m][e], 0, 0, 0);
                acc[m][e] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(vf, plo[m], acc[m][e], 0, 0, 0);
              }
            }
            if (pass >= 2) break;
          }
        }
        lgkm_wait0();  // the slot's reads are done
        issue(t + SL);
        there = there >> 16 | (uint64_t)there_of(t + SL, pages) << (16 * (SL - 1));
      }
    }
    vm_wait<0>();

    // ---- the waves' states, added in wave order
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      float x0, x1;
      l_run[m] = xor32_sum(l_run[m]);
      att::xor16_pair(l_run[m], l_run[m], x0, x1);
      l_run[m] = x0 + x1;
      if (grp == 0) {
        ml(wid, 16 * m + col)[0] = m_run[m];
        ml(wid, 16 * m + col)[1] = l_run[m];
      }
    }
    const bool whole = nst == ln.steps;
    float *part = d.parts + (size_t)(2 * blockIdx.x + (first_segment ? 0 : 1)) * pd_part_floats(DP, MT);
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      float *so = reinterpret_cast<float *>(mine);
#pragma unroll
      for (int e = 0; e < DB; ++e) *reinterpret_cast<f32x4 *>(so + col * PS + 16 * e + 4 * grp) = acc[m][e];
      __syncthreads();
      for (int x = tid; x < 16 * (DP / 4); x += PD_THREADS) {
        const int rr = x / (DP / 4), dd = 4 * (x % (DP / 4)), r = 16 * m + rr;
        if (r >= rows) continue;
        float M = -INFINITY, L = 0.f;
#pragma unroll
        for (int w = 0; w < PD_WAVES; ++w) M = fmaxf(M, ml(w, r)[0]);
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < PD_WAVES; ++w) {
          const float mw = ml(w, r)[0], f = mw == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((mw - M) * c2);
          L += ml(w, r)[1] * f;
          v += *reinterpret_cast<const f32x4 *>(ring + w * S::WAVE + (rr * PS + dd) * 4) * f;
        }
        if (whole) {
          if (dd >= D) continue;
          const float inv = L == 0.f ? 0.f : 1.f / L;
          const int i = (int)g.group.div(row0 + r), h = hk * (int)g.group.d + row0 + r - i * (int)g.group.d;
          *reinterpret_cast<att::u32x2 *>(g.out.data + (int64_t)(s.q0 + i) * g.out.token + h * g.out.head + dd) =
              att::u32x2{pack_bf(v[0] * inv, v[1] * inv), pack_bf(v[2] * inv, v[3] * inv)};
        } else {
          *reinterpret_cast<f32x4 *>(part + (size_t)r * DP + dd) = v;
          if (dd == 0) {
            part[(size_t)ROWS * DP + 2 * r] = M;
            part[(size_t)ROWS * DP + 2 * r + 1] = L;
          }
        }
      }
      __syncthreads();
    }
    u += nst;
    in_seq += nst;
    first_segment = false;
  }
}

// Adds the parts of the item that is cut where workgroup blockIdx.x's part begins, if no
// earlier workgroup's part begins inside the same item.
template <int DP, int MT>
__device__ __forceinline__ void paged_decode_merge_body(const DecodeArgs &d) {
  constexpr int ROWS = 16 * MT;
  const AttendArgs &g = d.a;
  const int w = blockIdx.x;
  if (w == 0) return;
  Place at;
  if (!find_place<ROWS>(d, w, at)) return;
  const Seq s = sequence(g.batch, at.b);
  const Line ln = line_of<ROWS>(g, s);
  const int item = (int)(at.in_seq / ln.steps), st = (int)(at.in_seq - (int64_t)item * ln.steps);
  const int64_t begin = at.first - st;
  const int w0 = at.worker_of(begin);
  if (st == 0 || w0 != w - 1) return;
  const int w1 = at.worker_of(begin + ln.steps - 1);
  const int hk = item / ln.tiles, tile = item - hk * ln.tiles;
  const int row0 = tile * ROWS, rows = min(ROWS, s.n * (int)g.group.d - row0), D = g.cache.dim;
  const float c2 = fabsf(g.c2);
  const size_t stride = pd_part_floats(DP, MT);
  // the first workgroup's part is its second one unless it began the item
  const float *p0 = d.parts + (size_t)(2 * w0 + (at.part(w0) == begin ? 0 : 1)) * stride;
  auto part = [&](int k) __attribute__((always_inline)) { return k == w0 ? p0 : d.parts + (size_t)(2 * k) * stride; };
  for (int x = threadIdx.x; x < rows * (DP / 4); x += PD_THREADS) {
    const int r = x / (DP / 4), dd = 4 * (x % (DP / 4));
    if (dd >= D) continue;
    float M = -INFINITY, L = 0.f;
    for (int k = w0; k <= w1; ++k) M = fmaxf(M, part(k)[(size_t)ROWS * DP + 2 * r]);
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    for (int k = w0; k <= w1; ++k) {
      const float *p = part(k);
      const float m = p[(size_t)ROWS * DP + 2 * r];
      const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - M) * c2);
      L += p[(size_t)ROWS * DP + 2 * r + 1] * f;
      v += *reinterpret_cast<const f32x4 *>(p + (size_t)r * DP + dd) * f;
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
    const int i = (int)g.group.div(row0 + r), h = hk * (int)g.group.d + row0 + r - i * (int)g.group.d;
    *reinterpret_cast<att::u32x2 *>(g.out.data + (int64_t)(s.q0 + i) * g.out.token + h * g.out.head + dd) =
        att::u32x2{pack_bf(v[0] * inv, v[1] * inv), pack_bf(v[2] * inv, v[3] * inv)};
  }
}

}  // namespace paged
}  // namespace pk
