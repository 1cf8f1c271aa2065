// paged_chunk.hpp -- attention of many new tokens per sequence over a paged cache.
//
// What bounds it: the matrix units and, beside them, the exponentials: 2048 tokens behind
// 6144 keys, 8 heads to 32 of 128, 0.24 TFLOP in 224 to 240 us, 1000 to 1070 TFLOP/s, the
// matrix units at work on half of the cycles.  128 rows (token, query head of the group) of
// one sequence and key head are a workgroup's item, 32 per wave, over steps of 64 keys that
// the four waves share through LDS.  S^T = K Q^T and
// O^T = V^T P^T run on v_mfma_f32_32x32x16_bf16 as in the contiguous flash kernel: a lane
// owns one row and half of the keys, so P never leaves its registers.  P is rounded to
// bf16 once (half a step, 2^-8 of a weight; the second product of a low half would be a
// third of all matrix work), and the fp32 sum is that of the rounded weights, two an
// instruction, so that what all of them lose in common cancels.
//
// Step t + 1's scores are computed while step t's exponentials are, in one run of
// instructions without a branch (two waves of two workgroups on a SIMD fall into step
// otherwise, and both wait for the matrix unit and then both for the exponentials: 313 us).
// At head dim 64, where a step's products are half as long, four workgroups on a CU in 128
// registers do better than that: 24 sequences, 4 of them prompts of 719 to 1531 tokens, on
// the last 1024 keys, 4 heads to 24, 42 us (51 the other way); vector instructions are at
// work on a third of the cycles, since 888 items of nearly one length do not go evenly
// into 256 CUs: at 0.6 us a step, four items of 17 take 41 us and all would take 31.
//
// Four items of one key head at a time run next to each other on one XCD and share its L2; the
// next four items of the line go to the next XCD, so that long sequences are everybody's.  Few
// items are also cut into `splits` runs of keys, whose states paged_chunk_merge_kernel adds in order.
#pragma once

#include "paged_tiles.hpp"

namespace pk {
namespace paged {

constexpr int PC_WAVES = 4, PC_THREADS = PC_WAVES * 64, PC_ROWS = 32 * PC_WAVES, PC_STEP = PT_STEP;

struct ChunkArgs {
  AttendArgs a;
  float *parts;  // splits > 1: [item][split] states
  int items;     // at most
  int splits;
  int above;     // rows of a sequence up to which another kernel takes it
};
constexpr size_t pc_part_floats(int DP) { return (size_t)PC_ROWS * (DP + 2); }

// The runs of keys that an item of so many steps is cut into: at least four steps each.
__device__ __forceinline__ int splits_of(const ChunkArgs &d, int steps) { return min(d.splits, max(1, steps / 4)); }

// An item: 128 rows of one sequence and key head.
struct Item {
  Seq s;
  int b, hk, tile;
  int split;
};
constexpr int PC_RUN = 4;  // items that an XCD takes at a time
constexpr int pc_blocks(int items) { return (items + 8 * PC_RUN - 1) / (8 * PC_RUN) * (8 * PC_RUN); }
// Workgroup i's item and split; false behind the last one.  `order`: place of the item
// on the line of all, for its parts.  `spread`: workgroups i go to XCDs i % 8, else it is the
// i-th of the line; `pairs`: up to 512 of them run at once, two on a CU.
__device__ __forceinline__ bool find_item(const ChunkArgs &d, int splits, int i, bool spread, bool pairs, Item &it, int &order) {
  const AttendArgs &g = d.a;
  const int lane = threadIdx.x & 63, B = g.batch.sequences, per = (B + 63) / 64, G = (int)g.group.d;
  auto tiles_of = [&](const Seq &s) __attribute__((always_inline)) {
    const int64_t rows = (int64_t)s.n * G;
    return rows <= d.above ? 0 : (int)((rows + PC_ROWS - 1) / PC_ROWS);
  };
  int mine = 0;
  Seq last{0, 0, 0};
  for (int k = 0; k < per; ++k) {
    const int b = lane * per + k;
    if (b < B) {
      last = sequence(g.batch, b);
      mine += tiles_of(last) * g.cache.heads;
    }
  }
  const int incl = wave_scan(mine);
  const int total = min(__builtin_amdgcn_readlane(incl, 63), d.items);  // (more only where q_start goes down)
  static_assert(8 * PC_RUN == 32, "the bits of a place");
  const int v = uniform(spread ? (i & ~31) | (i & 7) << 2 | (i >> 3 & 3) : i);
  const int u = v / splits;  // any place of the item's group: groups are whole runs of splits
  if (u >= total) return false;
  const uint64_t beyond = __ballot(u < incl);
  if (beyond == 0) return false;
  const int l = __ffsll((unsigned long long)beyond) - 1;
  int at = __builtin_amdgcn_readlane(incl - mine, l), b = l * per, n;
  for (;; ++b) {
    if (b >= B) return false;
    it.s = B > 64 ? sequence(g.batch, b)
                  : Seq{__builtin_amdgcn_readlane(last.q0, b), __builtin_amdgcn_readlane(last.n, b),
                        __builtin_amdgcn_readlane(last.kv, b)};
    n = tiles_of(it.s);
    if (u < at + n * g.cache.heads) break;
    at += n * g.cache.heads;
  }
  // a sequence's run: splits, of each the tiles from the last one on, which sees the most keys, in
  // runs of four by head; in pairs the workgroups from 256 on take them from the other end, so
  // that long ones share a CU with short
  const int heads = g.cache.heads, all = n * heads, in_seq = v - at * splits;
  if ((unsigned)in_seq >= (unsigned)(all * splits)) return false;
  it.b = uniform(b);
  it.split = uniform(in_seq / all);
  const int x = in_seq - it.split * all;
  const int turn = pairs && total * splits <= 512 ? min(max(256 - (v - x), 0), all) : all;
  int y = x < turn ? x : all - 1 - (x - turn), t = n & ~(PC_RUN - 1), run = PC_RUN;
  if (y < t * heads) {
    t = y / (PC_RUN * heads) * PC_RUN;
    y -= t * heads;
  } else {
    y -= t * heads;
    run = n - t;
  }
  it.hk = uniform(y / run);
  it.tile = uniform(n - 1 - (t + y - it.hk * run));
  order = at + it.hk * n + it.tile;
  return (unsigned)order < (unsigned)d.items;
}

// The item's first key (of a tile) and its steps.
__device__ __forceinline__ int item_steps(const AttendArgs &g, const Item &it, int rows, int &klo, int &hi_all, int &lo_all, int &hi) {
  int lo;
  key_range(g, it.s, (int)g.group.div(it.tile * PC_ROWS), lo, hi_all);
  key_range(g, it.s, (int)g.group.div(it.tile * PC_ROWS + rows - 1), lo_all, hi);
  klo = lo & ~(PT_KEYS - 1);
  return max(1, (hi - klo + PC_STEP - 1) / PC_STEP);
}

// A barrier that waits for this wave's LDS accesses and no loads in flight.
__device__ __forceinline__ void lds_barrier() {
  lgkm_wait0();
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

template <int DP>
struct ChunkShape {
  static constexpr int TB = PC_STEP * DP * 2, SL = 2;  // bytes of a step, slots of a ring
  static constexpr bool PIPE = DP != 64;                     // the next step's scores beside this one's weights
  static constexpr int OS = DP * 2 + 16;                             // row stride of a wave's rows on their way out
  static constexpr int LDS = 2 * SL * TB;
  static_assert(PC_ROWS * OS <= LDS, "the outputs pass through the rings");
};

// DP: dims of a row in LDS; DC: dims that the products take (head dims up to DC).
template <int DP, int DC, int PAGE>
__device__ __forceinline__ void paged_chunk_body(const ChunkArgs &d) {
  using S = ChunkShape<DP>;
  using Tiles = TileLoader<DP, PAGE, false>;
  constexpr bool PAGE16 = PAGE == 16;
  constexpr int CH = DP / 8, TB = S::TB, SL = S::SL, NI = Tiles::NI, DS = DC / 16, DB = DC / 32, RB = DP * 2;
  static_assert(DC <= DP && DC % 32 == 0, "dims");
  constexpr int KO = DS < 8 ? DS : 8, VO = DB < 4 ? DB : 4;  // lane offsets; dims from 128 on lie 256 bytes further
  __shared__ __attribute__((aligned(1024))) uint8_t ring[S::LDS];
  __shared__ __attribute__((aligned(8))) uint16_t there_s[SL][PC_WAVES];
  __shared__ int odd_s;
  const AttendArgs &g = d.a;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wid = uniform(tid >> 6);
  const int col = lane & 31, h = lane >> 5, gi = lane & 15, grp = lane >> 4;
  const int D = g.cache.dim, G = (int)g.group.d;

  Item it;
  int order;
  if (!find_item(d, d.splits, blockIdx.x, true, DP < 256, it, order)) return;
  const Seq s = it.s;
  const int all_rows = s.n * G, row0 = it.tile * PC_ROWS;
  const int rows = min(PC_ROWS, all_rows - row0);
  const int wrow = row0 + 32 * wid, wrows = min(32, all_rows - wrow);  // this wave's (may be none)

  // the item's keys, and those that all of this wave's rows see
  int klo, hi_last, t0, t1;
  const int steps = item_steps(g, it, rows, klo, t0, t1, hi_last), splits = splits_of(d, steps);
  if (it.split >= splits) return;
  const int s0 = (int)((int64_t)steps * it.split / splits), nst = (int)((int64_t)steps * (it.split + 1) / splits) - s0;
  const int kfirst = klo + s0 * PC_STEP;
  Tiles tiles(g);
  tiles.begin(g, it.b, it.hk, kfirst + wid * PT_KEYS, nst, hi_last);
  // PAGE16: a lane per tile, four a step: pages of 16 steps, and of the 16 after them
  auto pages_of = [&](int t) __attribute__((always_inline)) {
    const int key = kfirst + t * PC_STEP + lane * PT_KEYS;
    return t < nst && key < hi_last ? page_number(g.batch, g.cache, it.b, key) : -1;
  };
  int pages = -1, pages_next = -1, v_page = 0, v_row = 0, v_n = 0;
  uint64_t pages_there = 0;  // of `pages`
  if constexpr (PAGE16) {
    pages_next = pages_of(0);
  }
  int lo_all, hi_all, t2, t3;
  key_range(g, s, (int)g.group.div(min(wrow, all_rows - 1)), t2, hi_all);
  key_range(g, s, (int)g.group.div(min(wrow + 31, all_rows - 1)), lo_all, t3);

  // Q^T fragments: row lane % 32, dims 16 ds + 8 h + 0..7
  int lo, hi;
  bf16x8 qf[DS];
  {
    const int my = min(wrow + min(col, max(wrows, 1) - 1), all_rows - 1), i = (int)g.group.div(my);
    key_range(g, s, i, lo, hi);
    const uint16_t *qp = g.q.data + (int64_t)(s.q0 + i) * g.q.token + (it.hk * G + my - i * G) * g.q.head + 8 * h;
#pragma unroll
    for (int ds = 0; ds < DS; ++ds) {
      att::u32x4 v = {0, 0, 0, 0};
      if (16 * ds + 8 * h < D) v = *reinterpret_cast<const att::u32x4 *>(qp + 16 * ds);
      if (g.c2 < 0.f) v ^= 0x80008000u;
      qf[ds] = __builtin_bit_cast(bf16x8, v);
    }
  }
  const float c2 = fabsf(g.c2);

  // The lane's places in a K and a V tile; tile and row offsets are constants of the
  // reads, since every slot of the rings has its own copy of the step.
  uint32_t ko[KO], vo[VO];
#pragma unroll
  for (int ds = 0; ds < KO; ++ds) ko[ds] = (uint32_t)(col * RB + 16 * att::swz_k<CH>(2 * ds + h, col));
#pragma unroll
  for (int e = 0; e < VO; ++e)
    vo[e] = (uint32_t)((4 * h + (gi >> 2)) * RB + 16 * ((4 * e + 2 * (grp & 1) + ((gi & 3) >> 1)) ^ att::swz_v<DP>(gi >> 2)) + 8 * (gi & 1));

  // K of step t and V of step t lie in slot t % 2 of their rings.  Step t's iteration reads K
  // of step t + 1 and V of step t, and loads V of step t + 1 (V of step t - 1 has been read)
  // and K of step t + 2 (K of step t has).
  // Steps of K from 0 on, and a step's V after its K and before the next one's.
  const uint32_t ring_at = lds_number(ring) + wid * Tiles::BYTES;
  uint32_t there_bits[SL];  // PAGE16: tiles of the step in a slot of K that are there, 4 bits
  auto issue_k = [&](int t, int sl) __attribute__((always_inline)) {
    if constexpr (PAGE16) {
      if (t % 16 == 0) {
        pages = page_or_none(g.cache, pages_next);
        pages_there = __ballot(pages >= 0);
        pages_next = pages_of(t + 16);
      }
      const int page = __builtin_amdgcn_readlane(pages, 4 * (t % 16) + wid), key = kfirst + t * PC_STEP + wid * PT_KEYS;
      v_n = t < nst && page >= 0 ? min(PT_KEYS, hi_last - key) : 0;
      v_row = key - (int)(g.cache.page.div(key) * g.cache.page.d);
      v_page = v_n > 0 ? page : 0;
      there_bits[sl] = (uint32_t)(pages_there >> (4 * (t % 16))) & 15u;
      Tiles::load_rows(g, v_page, v_row, v_n, tiles.kbase, g.cache.k_page, g.cache.k_row, tiles.kvo, ring_at + sl * TB);
    } else {
      tiles.issue_k(g, t, ring_at + sl * TB);
      const uint32_t is = tiles.there(t);  // by all lanes
      if (lane == 0) there_s[sl][wid] = (uint16_t)is;
    }
  };
  auto issue_v = [&](int t, int sl) __attribute__((always_inline)) {
    if constexpr (PAGE16)
      Tiles::load_rows(g, v_page, v_row, v_n, tiles.vbase, g.cache.v_page, g.cache.v_row, tiles.vvo, ring_at + (SL + sl) * TB);
    else
      tiles.issue_v(g, t, ring_at + (SL + sl) * TB);
  };

  f32x16 acc[DB], sc[2];
#pragma unroll
  for (int e = 0; e < DB; ++e)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[e][i] = 0.f;
  float m_run = -INFINITY, l_run = 0.f, top = -INFINITY;  // top: row maximum of sc
  bool whole = true;                   // the keys of the step in sc are all on pages that are there
  int odd_first = nst, odd_last = -1;  // steps whose values were not all finite where a row has a hidden key
  if (tid == 0) odd_s = -1;

  // fragment i of the 2 DS of a K tile: head dims 16 (i / 2) + ..., keys 32 (i % 2) + ...
  auto k_fragment = [&](int sl, int i) __attribute__((always_inline)) {
    const int ds = i >> 1;
    return __builtin_bit_cast(bf16x8, *reinterpret_cast<const att::u32x4 *>(ring + sl * TB + ko[ds % KO] + 256 * (ds / KO) +
                                                                            32 * (i & 1) * RB));
  };
  // fragment i of the 4 DB of a V tile: keys 16 (i / DB) + ..., head dims 32 (i % DB) + ...
  auto v_fragment = [&](int sl, int i) __attribute__((always_inline)) {
    const int st = i / DB, e = i % DB;
    i16x4 hv[2];
#pragma unroll
    for (int r = 0; r < 2; ++r)
      hv[r] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (att::lds_i16x4 *)(ring + (SL + sl) * TB + vo[e % VO] + 256 * (e / VO) + (st * 16 + 8 * r) * RB));
    return __builtin_bit_cast(bf16x8, __builtin_shufflevector(hv[0], hv[1], 0, 1, 2, 3, 4, 5, 6, 7));
  };
  // Scores of the step in K slot sl, and beside product i the work of `beside(i)`.  Fragments
  // are read AHEAD products before they are used, and the order of pairs is kept as written.
  constexpr int AHEAD = 4, NA = 2 * DS, NB = 4 * DB;
  auto scores = [&](int sl, f32x16 (&x)[2], auto beside) __attribute__((always_inline)) {
    bf16x8 f[NA];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) f[i] = k_fragment(sl, i);
    x[0] = x[1] = f32x16{};
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < NA; i += 2) {
#pragma unroll
      for (int j = i; j < i + 2; ++j) {
        x[j & 1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f[j], qf[j >> 1], x[j & 1], 0, 0, 0);
        beside(j);
      }
#pragma unroll
      for (int j = i + AHEAD; j < min(NA, i + AHEAD + 2); ++j) f[j] = k_fragment(sl, j);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  auto maximum = [&](const f32x16 (&x)[2]) __attribute__((always_inline)) {
    float m = x[0][0];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int i = 0; i < 16; ++i) m = fmaxf(m, x[kb][i]);
    return xor32_max(m);
  };
  // the keys of the step in K slot sl that are on pages that are there
  auto keys_there = [&](int sl, uint32_t (&there)[2]) __attribute__((always_inline)) {
    if constexpr (PAGE16) {
      const uint32_t f = there_bits[sl];
      whole = f == 15u;
      there[0] = (f & 1 ? 0xFFFFu : 0u) | (f & 2 ? 0xFFFF0000u : 0u);
      there[1] = (f & 4 ? 0xFFFFu : 0u) | (f & 8 ? 0xFFFF0000u : 0u);
    } else {
      const att::u32x2 w = *reinterpret_cast<const att::u32x2 *>(there_s[sl]);
      there[0] = (uint32_t)uniform((int)w[0]);
      there[1] = (uint32_t)uniform((int)w[1]);
      whole = (there[0] & there[1]) == 0xFFFFFFFFu;
    }
  };
  // hides what this wave's rows do not see of step t, whose scores are in sc (K slot sl)
  auto mask = [&](int t, int sl) __attribute__((always_inline)) {
    const int key = kfirst + t * PC_STEP;
    uint32_t there[2];
    keys_there(sl, there);
    if (key < lo_all || key + PC_STEP > hi_all || !whole) {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        // keys [lo, hi) of this half as bits, those on pages that are not there taken out
        const int from = min(max(lo - key - 32 * kb, 0), 32), to = min(max(hi - key - 32 * kb, 0), 32);
        const uint32_t up = to < 32 ? (1u << to) - 1 : ~0u, down = from < 32 ? ~0u << from : 0u;
        const uint32_t seen = (up & down & there[kb]) >> (4 * h);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int on = __builtin_amdgcn_sbfe((int)seen, 8 * (i >> 2) + (i & 3), 1);  // all bits or none
          sc[kb][i] = __uint_as_float(((uint32_t)on & __float_as_uint(sc[kb][i])) | (~(uint32_t)on & 0xFF800000u));
        }
      }
      top = maximum(sc);
    }
  };

  // A wave without rows (`idle`) loads its part and keeps the barriers, and leaves LDS and the matrix
  // units to the others: 24 sequences of 20 rows on 46600 keys take 52 us, 57 with all waves at work.
  auto step = [&](auto slot, int t, auto idle) __attribute__((always_inline)) {
    constexpr int sl = decltype(slot)::value, next = 1 - sl;
    constexpr bool IDLE = decltype(idle)::value;
    vm_wait<0>();  // this wave's part of K of step t + 1 and V of step t has landed
    lds_barrier();  // and every wave's; nobody reads what the next loads overwrite
    uint8_t *const vs = ring + (SL + sl) * TB;
    const int key = kfirst + t * PC_STEP;
    if constexpr (S::PIPE) {
      issue_v(t + 1, next);
    } else {
      issue_k(t + 1, next);
      issue_v(t + 1, next);
      if constexpr (IDLE) {
        uint32_t there[2];
        keys_there(sl, there);
      } else {
        scores(sl, sc, [](int) {});
        top = maximum(sc);
        mask(t, sl);
      }
    }
    // the same for every wave: whether some row of the item has a hidden key in this step
    const bool mixed = key < t1 || key + PC_STEP > t0 || !whole;
    if constexpr (S::PIPE) issue_k(t + 2, sl);

    // the maximum in the exponent follows once it is 2^8 behind
    if (!IDLE && __any((top - m_run) * c2 > 8.f)) {
      const float m_new = fmaxf(m_run, top);
      const float alpha = m_run == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m_run - m_new) * c2);
      m_run = m_new;
      l_run *= alpha;
#pragma unroll
      for (int e = 0; e < DB; ++e) acc[e] *= alpha;
    }
    const float mc = m_run == -INFINITY ? 0.f : m_run * c2;
    f32x16 nx[2];
    att::u32x4 pw[4];
    float sum = 0.f;
    // weights of scores 2 n and 2 n + 1: three quarters beside the next scores, the rest beside the
    // first products with V, which are those of the other weights
    constexpr int EARLY = S::PIPE ? 12 : 16;
    const pk_bf16x2 ones = {(__bf16)1.f, (__bf16)1.f};
    auto weights = [&](int n) __attribute__((always_inline)) {
      const int kb = n >> 3, j = 2 * (n & 7);
      const float p0 = __builtin_amdgcn_exp2f(fmaf(sc[kb][j], c2, -mc));
      const float p1 = __builtin_amdgcn_exp2f(fmaf(sc[kb][j + 1], c2, -mc));
      uint32_t two = pack_bf(p0, p1);
      sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(pk_bf16x2, two), ones, sum, false);
      asm volatile("" : "+v"(two), "+v"(sum));  // here, not where they are used first
      pw[n >> 2][n & 3] = two;
    };
    if constexpr (IDLE) {
    } else if constexpr (S::PIPE) {
      scores(next, nx, [&](int i) __attribute__((always_inline)) {
#pragma unroll
        for (int n = i * EARLY / NA; n < (i + 1) * EARLY / NA; ++n) weights(n);
      });
    } else {
#pragma unroll
      for (int n = 0; n < EARLY; ++n) weights(n);
    }

    if (mixed) {
      pk_u16x2 most = {0, 0};
#pragma unroll 1
      for (int x = 16 * tid; x < TB; x += 16 * PC_THREADS) {
        const att::u32x4 w = *reinterpret_cast<const att::u32x4 *>(vs + x);
#pragma unroll
        for (int e = 0; e < 4; ++e) most = exponents(most, w[e]);
      }
      if (__any(not_finite(most)) && lane == 0) odd_s = t;
      lds_barrier();
      if (uniform(odd_s) == t) {
        odd_first = min(odd_first, t);
        odd_last = t;
#pragma unroll 1
        for (int x = 16 * tid; x < TB; x += 16 * PC_THREADS) {
          att::u32x4 *at = reinterpret_cast<att::u32x4 *>(vs + x), w = *at;
#pragma unroll
          for (int e = 0; e < 4; ++e) w[e] = finite(w[e]);
          *at = w;
        }
        lds_barrier();
      }
    }
    if constexpr (!IDLE) {
      bf16x8 f[NB];
      if constexpr (S::PIPE) top = nx[0][0];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) f[i] = v_fragment(sl, i);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < NB; i += 2) {
#pragma unroll
        for (int j = i; j < i + 2; ++j) {
          acc[j % DB] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f[j], __builtin_bit_cast(bf16x8, pw[j / DB]), acc[j % DB], 0, 0, 0);
          constexpr int ON = 3 * DB;  // products with the early weights
#pragma unroll
          for (int n = EARLY + j * (16 - EARLY) / ON; n < min(16, EARLY + (j + 1) * (16 - EARLY) / ON); ++n) weights(n);
          if constexpr (S::PIPE)
#pragma unroll
            for (int n = j * 32 / NB; n < (j + 1) * 32 / NB; ++n) top = fmaxf(top, nx[n >> 4][n & 15]);
        }
#pragma unroll
        for (int j = i + AHEAD; j < min(NB, i + AHEAD + 2); ++j) f[j] = v_fragment(sl, j);
        __builtin_amdgcn_sched_barrier(0);
      }
      l_run += sum;
    }
    if constexpr (IDLE) {
      uint32_t there[2];
      if constexpr (S::PIPE) keys_there(next, there);
    } else if constexpr (S::PIPE) {
      top = xor32_max(top);
      sc[0] = nx[0];
      sc[1] = nx[1];
      mask(t + 1, next);
    }
  };

  issue_k(0, 0);
  issue_v(0, 0);
  if constexpr (S::PIPE) {
    issue_k(1, 1);
    vm_wait<2 * NI>();
    lds_barrier();
  }
  auto all_steps = [&](auto idle) __attribute__((always_inline)) {
    if constexpr (S::PIPE) {
      if constexpr (decltype(idle)::value) {
        uint32_t there[2];
        keys_there(0, there);
      } else {
        scores(0, sc, [](int) {});
        top = maximum(sc);
        mask(0, 0);
      }
    }
    int t = 0;
#pragma unroll 1
    for (; t + 1 < nst; t += 2) {
      step(std::integral_constant<int, 0>{}, t, idle);
      step(std::integral_constant<int, 1>{}, t + 1, idle);
    }
    if (t < nst) step(std::integral_constant<int, 0>{}, t, idle);
  };
  if (wrows > 0)
    all_steps(std::false_type{});
  else
    all_steps(std::true_type{});
  vm_wait<0>();
  l_run = xor32_sum(l_run);
  for (int k = kfirst + odd_first * PC_STEP; k < min(hi_last, kfirst + (odd_last + 1) * PC_STEP); ++k) {
    const uint16_t *vr = value_row(g, it.b, it.hk, k);
    if (!vr || k < lo || k >= hi) continue;
#pragma unroll
    for (int e = 0; e < DB; ++e)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (32 * e + 8 * j + 4 * h < D) {
          f32x4 x = {acc[e][4 * j], acc[e][4 * j + 1], acc[e][4 * j + 2], acc[e][4 * j + 3]};
          add_not_finite(vr + 32 * e + 8 * j + 4 * h, x);
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[e][4 * j + i] = x[i];
        }
  }

  if (splits > 1) {
    // this split's state of the rows that there are
    if (col >= wrows) return;
    float *part = d.parts + ((size_t)order * d.splits + it.split) * pc_part_floats(DP);
#pragma unroll
    for (int e = 0; e < DB; ++e)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *reinterpret_cast<f32x4 *>(part + (size_t)(((wid * DB + e) * 4 + j) * 64 + lane) * 4) =
            f32x4{acc[e][4 * j], acc[e][4 * j + 1], acc[e][4 * j + 2], acc[e][4 * j + 3]};
    if (h == 0) {
      float *ml = part + (size_t)PC_ROWS * DP + 2 * (32 * wid + col);
      ml[0] = m_run;
      ml[1] = l_run;
    }
    return;
  }
  // rows in bf16 through LDS, so that a store covers whole rows
  lds_barrier();
  uint8_t *const os = ring + wid * 32 * S::OS;
  const float inv = l_run == 0.f ? 0.f : 1.f / l_run;
#pragma unroll
  for (int e = 0; e < DB; ++e)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      *reinterpret_cast<att::u32x2 *>(os + col * S::OS + 2 * (32 * e + 8 * j + 4 * h)) =
          att::u32x2{pack_bf(acc[e][4 * j] * inv, acc[e][4 * j + 1] * inv), pack_bf(acc[e][4 * j + 2] * inv, acc[e][4 * j + 3] * inv)};
  lgkm_wait0();
#pragma unroll
  for (int x = 0; x < 32 * CH / 64; ++x) {
    const int r = (x * 64 + lane) / CH, c = (x * 64 + lane) % CH;
    if (r < wrows && 8 * c < D) {
      const int i = (int)g.group.div(wrow + r);
      *reinterpret_cast<att::u32x4 *>(g.out.data + (int64_t)(s.q0 + i) * g.out.token +
                                      (it.hk * G + wrow + r - i * G) * g.out.head + 8 * c) =
          *reinterpret_cast<const att::u32x4 *>(os + r * S::OS + 16 * c);
    }
  }
}

// Adds the splits of an item in order.  A state holds its sums as the lanes have them (four
// dims of a row; wave, block of 32 dims, run of 8 in it, lane), so that every access is 16
// bytes a lane in a row; a thread takes one of those and reads AT_ONCE splits before it adds them.
constexpr int PC_MERGE = 8;  // workgroups of an item
template <int DP, int DC>
__device__ __forceinline__ void paged_chunk_merge_body(const ChunkArgs &d) {
  constexpr int DB = DC / 32, AT_ONCE = 8;
  const AttendArgs &g = d.a;
  Item it;
  int order;
  if (!find_item(d, 1, blockIdx.x, false, false, it, order)) return;
  const Seq s = it.s;
  const int G = (int)g.group.d, D = g.cache.dim;
  const int row0 = it.tile * PC_ROWS, rows = min(PC_ROWS, s.n * G - row0);
  const float c2 = fabsf(g.c2);
  int t0, t1, t2, t3;
  const int splits = splits_of(d, item_steps(g, it, rows, t0, t1, t2, t3));
  if (splits == 1) return;  // the kernel wrote the rows
  const float *parts = d.parts + (size_t)order * d.splits * pc_part_floats(DP);
  auto weight = [&](float m, float M) __attribute__((always_inline)) {
    return m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - M) * c2);
  };
  for (int x = blockIdx.y * PC_THREADS + threadIdx.x; x < PC_ROWS * DC / 4; x += PC_MERGE * PC_THREADS) {
    const int lane = x & 63, j = x >> 6 & 3, we = x >> 8, w = we / DB, e = we - w * DB;
    const int r = 32 * w + (lane & 31), dd = 32 * e + 8 * j + 4 * (lane >> 5);
    if (r >= rows || dd >= D) continue;
    float M = -INFINITY, L = 0.f;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    for (int k0 = 0; k0 < splits; k0 += AT_ONCE) {
      float m[AT_ONCE], l[AT_ONCE];
      f32x4 o[AT_ONCE];
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i) {
        const float *p = parts + (size_t)min(k0 + i, splits - 1) * pc_part_floats(DP);
        const float2 ml = *reinterpret_cast<const float2 *>(p + (size_t)PC_ROWS * DP + 2 * r);
        o[i] = *reinterpret_cast<const f32x4 *>(p + 4 * x);
        m[i] = k0 + i < splits ? ml.x : -INFINITY;
        l[i] = ml.y;
      }
      float M2 = M;
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i) M2 = fmaxf(M2, m[i]);
      const float a = weight(M, M2);
      L *= a;
      v *= a;
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i) {
        const float f = weight(m[i], M2);
        L += l[i] * f;
        v += o[i] * f;
      }
      M = M2;
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
    const int i = (int)g.group.div(row0 + r);
    *reinterpret_cast<att::u32x2 *>(g.out.data + (int64_t)(s.q0 + i) * g.out.token + (it.hk * G + row0 + r - i * G) * g.out.head + dd) =
        att::u32x2{pack_bf(v[0] * inv, v[1] * inv), pack_bf(v[2] * inv, v[3] * inv)};
  }
}

}  // namespace paged
}  // namespace pk
