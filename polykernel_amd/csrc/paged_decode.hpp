// paged_decode.hpp -- attention of few new tokens per sequence over a paged cache.
//
// What bounds it: keys and values are read once for the G query heads that share
// them (and the few new tokens), so the time is that of streaming them from HBM: 64
// sequences with 281000 keys in all, 8 heads to 32 of 128, 1.15 GB in 190 us, 6.0 TB/s;
// the matrix units work on a tenth of the cycles.  Few short sequences are bound by the
// chain from a page's number to its keys to the sums: 6.7 us for up to 64 keys, 0.85 for
// each 64 more of an item.
//
// A row is a (token, query head of the group) pair; 16 rows of one sequence and key
// head are one item.  Both products run on the matrix units, transposed: S^T =
// K Q^T (16x16x32, keys x rows) leaves each lane one row and 4 keys of 16, which is
// the B operand of O^T = V^T P^T (16x16x16), its A operand read from V's rows in LDS
// by transposing reads.  So P stays in registers; P is split into two bf16 halves
// (2^-17 relative), which costs nothing under the memory time.
//
// Memory: every wave has rings of its own of SL tiles of 16 keys in LDS, filled by
// direct-to-LDS loads (16 bytes a lane, chunks swizzled at the source), with no
// barrier in the loop; a tile's keys make room for those SL tiles on as soon as they
// are read, its values likewise.  Short rings and many workgroups on a CU keep as many
// bytes in flight as long rings and few, and hide each other's beginnings and ends (one
// sequence of 200 keys takes 9.2 us so, 10.3 with rings of four tiles, 10.9 with 16 waves).  A
// tile of a page size that is a multiple of 16 lies in one page: its base address is a
// buffer resource whose length ends the tile at the last key, so rows behind it read as
// zero and stale pages never reach a product.  Page sizes that are no multiple of 8 look
// up a page per row and point rows that are not there at zeros.
//
// Work: the steps (64 keys of an item, 16 per wave) of all items lie on one line,
// which the workgroups cut into equal parts whatever the sequences' lengths; each
// finds its part from kv_len and q_start alone, so a captured call follows them.  An
// item cut between workgroups leaves its parts in the workspace, and
// paged_decode_merge_kernel adds them in the order of the workgroups.
#pragma once

#include "paged_tiles.hpp"

namespace pk {
namespace paged {

constexpr int PD_WAVES = 4, PD_THREADS = PD_WAVES * 64, PD_TILE = PT_KEYS, PD_STEP = PT_STEP, PD_ROWS = 16;

// Bytes of one workgroup's partial state: 16 rows of DP sums, and (maximum, sum).
constexpr size_t pd_part_floats(int DP) { return (size_t)PD_ROWS * (DP + 2); }
constexpr size_t pd_workspace(int DP, int workers) {
  return workers * (2 * pd_part_floats(DP) * sizeof(float) + 32);
}

// Where a workgroup's part begins inside an item: the item's workgroups and rows, for the merge.
struct Cut {
  int first, last, second, q0;  // first < 0: it does not; second: the first's state is its second one
  int hk, row0, rows, unused;
};
struct DecodeArgs {
  AttendArgs a;
  float *parts;  // two partial states per workgroup, then a Cut each
  int most;      // workgroups
  int below;     // rows of a sequence from which on another kernel takes it
  int whole;     // items are not cut: a step of the line is an item
};

// The line of steps: what sequence b adds, and a place on it.  The host has made sure
// that the whole line is below 2^31; a q_start that goes down can make it longer, and
// then the loops over sequences end at the last one.
struct Line {
  int tiles, steps, klo;  // row tiles, steps of each item, first key of step 0
  int unit;               // places of the line that an item takes
  int units;
};
__device__ __forceinline__ Line line_of(const DecodeArgs &d, const Seq &s) {
  const AttendArgs &g = d.a;
  Line l{0, 0, 0, 1, 0};
  if (s.n <= 0 || (int64_t)s.n * (int)g.group.d >= d.below) return l;
  int lo, hi, lo2, hi2;
  key_range(g, s, 0, lo, hi);
  key_range(g, s, s.n - 1, lo2, hi2);
  l.klo = lo & ~(PD_TILE - 1);
  l.tiles = (int)(((int64_t)s.n * (int)g.group.d + PD_ROWS - 1) / PD_ROWS);
  l.steps = max(1, (hi2 - l.klo + PD_STEP - 1) / PD_STEP);
  l.unit = d.whole ? 1 : l.steps;
  l.units = l.tiles * g.cache.heads * l.unit;
  return l;
}

struct Place {
  int total, each, more;  // of the line; workgroups get `each` steps, the first `more` one more
  int workers, first, last;
  int b, in_seq;          // sequence of `first`, and first from that sequence's own start
  Seq mine;               // this lane's sequence, where there are at most 64
  __device__ __forceinline__ int part(int w) const { return w * each + min(w, more); }
  // the workgroup whose part place u is in
  __device__ __forceinline__ int worker_of(int u) const {
    const int wide = more * (each + 1);
    return u < wide ? u / (each + 1) : more + (u - wide) / each;
  }
};
// Sequence b of the batch: from the lane that read it, or from memory.
__device__ __forceinline__ Seq sequence_at(const Batch &g, const Place &p, int b) {
  if (g.sequences > 64) return sequence(g, b);
  return Seq{__builtin_amdgcn_readlane(p.mine.q0, b), __builtin_amdgcn_readlane(p.mine.n, b),
             __builtin_amdgcn_readlane(p.mine.kv, b)};
}
// Where workgroup w's part begins, found by every wave for itself: lane l adds up the
// sequences [l, l + 1) * ceil(B / 64), and a scan over the lanes gives each its offset.
__device__ __forceinline__ bool find_place(const DecodeArgs &d, int w, Place &p) {
  const AttendArgs &g = d.a;
  const int lane = threadIdx.x & 63, B = g.batch.sequences;
  const int per = (B + 63) / 64;
  int mine = 0, longest = 0;
  p.mine = Seq{0, 0, 0};
  for (int i = 0; i < per; ++i) {
    const int b = lane * per + i;
    if (b < B) {
      p.mine = sequence(g.batch, b);
      const Line l = line_of(d, p.mine);
      mine += l.units;
      longest = max(longest, l.unit);
    }
  }
  const int incl = wave_scan(mine);
  p.total = __builtin_amdgcn_readlane(incl, 63);
  // a step per workgroup, where there are so few; two where one item has over 256, whose parts
  // would take longer to add than the steps (1 head of 30000 keys 14.1 against 12.4 us; of 4000
  // 10.6 against 12.0)
  const bool two = !d.whole && __any(longest > 256);
  p.workers = min(d.most, max(1, two ? p.total / 2 : p.total));
  if (w >= p.workers || p.total <= 0) return false;
  p.each = p.total / p.workers;
  p.more = p.total - p.each * p.workers;
  p.first = p.part(w);
  p.last = p.part(w + 1);
  const uint64_t beyond = __ballot(p.first < incl);
  if (beyond == 0) return false;
  const int l = __ffsll((unsigned long long)beyond) - 1;
  int at = __builtin_amdgcn_readlane(incl - mine, l), b = l * per;
  for (;; ++b) {
    if (b >= B) return false;
    const int n = line_of(d, sequence_at(g.batch, p, b)).units;
    if (p.first < at + n) {
      p.b = uniform(b);
      p.in_seq = uniform(p.first - at);
      return (unsigned)p.in_seq < (unsigned)n;
    }
    at += n;
  }
}

template <int DP>
struct DecodeShape {
  static constexpr int NI = TileLoader<DP, 16, true>::NI, TB = TileLoader<DP, 16, true>::BYTES;
  static constexpr int SL = DP == 64 ? 2 : 1;      // tiles of a ring
  static constexpr int PS = DP + 4;                // row stride of a state in LDS, floats
  static constexpr int STATE = PD_ROWS * PS * 4;   // a wave's sums, then (maximum, sum) of its rows
  static constexpr int WAVE = 2 * SL * TB > STATE + 8 * PD_ROWS ? 2 * SL * TB : STATE + 8 * PD_ROWS;  // its rings, later its state
};
constexpr int pd_groups(int DP) { return DP == 256 ? 2 : 4; }  // workgroups on a CU

template <int DP, int PAGE>
__device__ __forceinline__ void paged_decode_body(const DecodeArgs &d) {
  using S = DecodeShape<DP>;
  constexpr int CH = DP / 8, NI = S::NI, TB = S::TB, SL = S::SL, PS = S::PS, KS = DP / 32, DB = DP / 16;
  __shared__ __attribute__((aligned(1024))) uint8_t ring[PD_WAVES * S::WAVE];
  auto ml = [&](int w, int r) __attribute__((always_inline)) {
    return reinterpret_cast<float *>(ring + w * S::WAVE + S::STATE) + 2 * r;
  };
  const AttendArgs &g = d.a;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, grp = lane >> 4;
  const int D = g.cache.dim;
  uint8_t *const mine = ring + wid * S::WAVE;  // K slots, then V slots
  const uint32_t mine_at = lds_number(ring) + wid * S::WAVE;

  auto cut = [&](int w) __attribute__((always_inline)) {
    return reinterpret_cast<Cut *>(d.parts + (size_t)(2 * d.most) * pd_part_floats(DP)) + w;
  };
  Place at;
  if (!find_place(d, blockIdx.x, at)) {
    if (tid == 0 && d.most > 1 && !d.whole) cut(blockIdx.x)->first = -1;
    return;
  }

  TileLoader<DP, PAGE, true> tiles(g);
  int u = at.first, in_seq = at.in_seq, b = at.b;
  bool first_segment = true;
  while (u < at.last && b < g.batch.sequences) {
    const Seq s = sequence_at(g.batch, at, b);
    const Line ln = line_of(d, s);
    if (in_seq >= ln.units) {
      in_seq = 0;
      ++b;
      continue;
    }
    const int item = uniform(in_seq / ln.unit), st0 = uniform(in_seq - item * ln.unit);
    const int took = uniform(min(ln.unit - st0, at.last - u)), nst = d.whole ? ln.steps : took;
    const int hk = uniform(item / ln.tiles), tile = item - hk * ln.tiles;
    const int row0 = tile * PD_ROWS, rows = min(PD_ROWS, s.n * (int)g.group.d - row0);

    // the keys that all rows of the tile see, and those that any does
    int lo_any, hi_all, lo_all, hi_any;
    key_range(g, s, (int)g.group.div(row0), lo_any, hi_all);
    key_range(g, s, (int)g.group.div(row0 + rows - 1), lo_all, hi_any);

    // ---- the wave's tiles: keys [key0 + 64 t, + 16)
    const int key0 = ln.klo + st0 * PD_STEP + wid * PD_TILE;
    tiles.begin(g, b, hk, key0, nst, hi_any);  // before the queries' loads: loads return in order

    int lo, hi;
    bf16x8 qf[KS];
    {
      const int r = min(row0 + col, row0 + rows - 1);
      const int i = (int)g.group.div(r), h = hk * (int)g.group.d + r - i * (int)g.group.d;
      key_range(g, s, i, lo, hi);
      const uint16_t *qp = g.q.data + (int64_t)(s.q0 + i) * g.q.token + h * g.q.head + 8 * grp;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        att::u32x4 v = {0, 0, 0, 0};
        if (32 * k + 8 * grp < D) v = *reinterpret_cast<const att::u32x4 *>(qp + 32 * k);
        if (g.c2 < 0.f) v ^= 0x80008000u;
        qf[k] = __builtin_bit_cast(bf16x8, v);
      }
    }
    const float c2 = fabsf(g.c2);

    auto issue_k = [&](int t) __attribute__((always_inline)) { tiles.issue_k(g, t, mine_at + (t % SL) * TB); };
    auto issue_v = [&](int t) __attribute__((always_inline)) { tiles.issue_v(g, t, mine_at + (SL + t % SL) * TB); };
    float m_run = -INFINITY, l_run = 0.f;
    f32x4 acc[DB];
#pragma unroll
    for (int e = 0; e < DB; ++e) acc[e] = f32x4{0.f, 0.f, 0.f, 0.f};
    // which keys of the next SL tiles are there, 16 bits each: looked up when a tile is issued
    uint64_t there = 0;
#pragma unroll
    for (int t = 0; t < SL; ++t) {
      issue_k(t);
      there |= (uint64_t)tiles.there(t) << (16 * t);
      issue_v(t);
    }
    int odd_first = nst, odd_last = -1;  // tiles whose values were not all finite where a row has a hidden key
#pragma unroll 1
    for (int t = 0; t < nst; ++t) {
      const int key = key0 + t * PD_STEP;
      const uint8_t *ks = mine + (t % SL) * TB;
      uint8_t *vs = mine + (SL + t % SL) * TB;
      const uint32_t here = (uint32_t)there & 0xFFFFu;
      const bool any = key < hi_any && here != 0;
      const bool masked = key < lo_all || key + PD_TILE > hi_all || here != 0xFFFFu;
      f32x4 sc = {0.f, 0.f, 0.f, 0.f};
      vm_wait<NI + 2 * NI * (SL - 1)>();
      if (any) {
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          const att::u32x4 kv = *reinterpret_cast<const att::u32x4 *>(ks + col * DP * 2 + 16 * att::swz_k<CH>(4 * k + grp, col));
          sc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, kv), qf[k], sc, 0, 0, 0);
        }
      }
      lgkm_wait0();  // the slot's keys are read
      issue_k(t + SL);
      there = there >> 16 | (uint64_t)tiles.there(t + SL) << (16 * (SL - 1));
      vm_wait<NI + 2 * NI * (SL - 1)>();
      if (any) {
        if (masked) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int kk = 4 * grp + i;
            if (key + kk < lo || key + kk >= hi || !(here >> kk & 1)) sc[i] = -INFINITY;
          }
        }
        float top = fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3]));
        top = xor32_max(top);
        float a0, a1;
        att::xor16_pair(top, top, a0, a1);
        top = fmaxf(a0, a1);
        // the maximum in the exponent follows once it is 2^8 behind: sums of p v / p do not depend on it
        if (__any((top - m_run) * c2 > 8.f)) {
          const float m_new = fmaxf(m_run, top);
          const float alpha = m_run == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m_run - m_new) * c2);
          m_run = m_new;
          l_run *= alpha;
#pragma unroll
          for (int e = 0; e < DB; ++e) acc[e] *= alpha;
        }
        const float mc = m_run == -INFINITY ? 0.f : m_run * c2;
        float p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = __builtin_amdgcn_exp2f(fmaf(sc[i], c2, -mc));
        l_run += (p[0] + p[1]) + (p[2] + p[3]);
        const uint32_t h0 = pack_bf(p[0], p[1]), h1 = pack_bf(p[2], p[3]);
        const i16x4 phi = __builtin_bit_cast(i16x4, (att::u32x2{h0, h1}));
        const i16x4 plo = __builtin_bit_cast(i16x4, (att::u32x2{pack_bf(p[0] - lo_bf(h0), p[1] - hi_bf(h0)),
                                                                pack_bf(p[2] - lo_bf(h1), p[3] - hi_bf(h1))}));
        if (masked) {
          pk_u16x2 most = {0, 0};
#pragma unroll 1
          for (int i = 0; i < NI; ++i) {
            const att::u32x4 w = *reinterpret_cast<const att::u32x4 *>(vs + i * 1024 + 16 * lane);
#pragma unroll
            for (int e = 0; e < 4; ++e) most = exponents(most, w[e]);
          }
          if (__any(not_finite(most))) {
            odd_first = min(odd_first, t);
            odd_last = t;
#pragma unroll 1
            for (int i = 0; i < NI; ++i) {
              att::u32x4 *at = reinterpret_cast<att::u32x4 *>(vs + i * 1024 + 16 * lane), w = *at;
#pragma unroll
              for (int e = 0; e < 4; ++e) w[e] = finite(w[e]);
              *at = w;
            }
          }
        }
#pragma unroll
        for (int e = 0; e < DB; ++e) {
          const int key_r = 4 * grp + (col >> 2), c = 2 * e + (col & 3) / 2;
          const i16x4 vf = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (att::lds_i16x4 *)(vs + key_r * DP * 2 + 16 * (c ^ att::swz_v<DP>(key_r)) + 8 * (col & 1)));
          acc[e] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(vf, phi, acc[e], 0, 0, 0);
          acc[e] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(vf, plo, acc[e], 0, 0, 0);
        }
      }
      lgkm_wait0();  // its values are read
      issue_v(t + SL);
    }
    vm_wait<0>();
    for (int t = odd_first; t <= odd_last; ++t)
      for (int k = key0 + t * PD_STEP; k < min(hi_any, key0 + t * PD_STEP + PD_TILE); ++k) {
        const uint16_t *vr = value_row(g, b, hk, k);
        if (!vr || k < lo || k >= hi) continue;
#pragma unroll
        for (int e = 0; e < DB; ++e)
          if (16 * e + 4 * grp < D) add_not_finite(vr + 16 * e + 4 * grp, acc[e]);
      }

    // ---- the waves' states, added in wave order
    {
      float x0, x1;
      l_run = xor32_sum(l_run);
      att::xor16_pair(l_run, l_run, x0, x1);
      if (grp == 0) {
        ml(wid, col)[0] = m_run;
        ml(wid, col)[1] = x0 + x1;
      }
      float *so = reinterpret_cast<float *>(mine);
#pragma unroll
      for (int e = 0; e < DB; ++e) *reinterpret_cast<f32x4 *>(so + col * PS + 16 * e + 4 * grp) = acc[e];
    }
    __syncthreads();
    const bool whole = nst == ln.steps;
    float *part = d.parts + (size_t)(2 * blockIdx.x + (first_segment ? 0 : 1)) * pd_part_floats(DP);
    for (int x = tid; x < rows * (DP / 4); x += PD_THREADS) {
      const int r = x / (DP / 4), dd = 4 * (x % (DP / 4));
      if (dd >= D) continue;
      float M = -INFINITY, L = 0.f;
#pragma unroll
      for (int w = 0; w < PD_WAVES; ++w) M = fmaxf(M, ml(w, r)[0]);
      f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < PD_WAVES; ++w) {
        const float mw = ml(w, r)[0], f = mw == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((mw - M) * c2);
        L += ml(w, r)[1] * f;
        v += *reinterpret_cast<const f32x4 *>(ring + w * S::WAVE + (r * PS + dd) * 4) * f;
      }
      if (whole) {
        const float inv = L == 0.f ? 0.f : 1.f / L;
        const int i = (int)g.group.div(row0 + r), h = hk * (int)g.group.d + row0 + r - i * (int)g.group.d;
        *reinterpret_cast<att::u32x2 *>(g.out.data + (int64_t)(s.q0 + i) * g.out.token + h * g.out.head + dd) =
            att::u32x2{pack_bf(v[0] * inv, v[1] * inv), pack_bf(v[2] * inv, v[3] * inv)};
      } else {
        *reinterpret_cast<f32x4 *>(part + (size_t)r * DP + dd) = v;
        if (dd == 0) {
          part[(size_t)PD_ROWS * DP + 2 * r] = M;
          part[(size_t)PD_ROWS * DP + 2 * r + 1] = L;
        }
      }
    }
    __syncthreads();
    if (first_segment && tid == 0 && d.most > 1 && !d.whole) {
      Cut c{-1, 0, 0, s.q0, hk, row0, rows, 0};
      if (st0 > 0) {
        const int begin = at.first - st0;
        c.first = at.worker_of(begin);
        c.last = min(at.worker_of(begin + ln.unit - 1), at.workers - 1);
        c.second = at.part(c.first) != begin;
      }
      *cut(blockIdx.x) = c;
    }
    u += took;
    in_seq += took;
    first_segment = false;
  }
}

// Adds the parts of an item that is cut between workgroups `first` to `last`: the workgroups
// of this launch numbered first + 1 to last share its outputs, 4 dims of a row (a chunk) at a
// time.  A thread reads AT_ONCE parts of a chunk before it adds them; more parts have more
// threads (a power of two up to 32), whose sums meet in LDS.
template <int DP>
__device__ __forceinline__ void paged_decode_merge_body(const DecodeArgs &d) {
  constexpr int AT_ONCE = 4;
  __shared__ float sum[PD_THREADS][6];
  const AttendArgs &g = d.a;
  const int w = blockIdx.x + 1;
  const size_t stride = pd_part_floats(DP);
  const Cut cut = reinterpret_cast<const Cut *>(d.parts + (size_t)(2 * d.most) * stride)[w];
  const int w0 = cut.first, w1 = cut.last, rows = cut.rows, D = g.cache.dim;
  if (w0 < 0 || w0 >= w || w1 < w) return;  // (the latter two only where q_start goes down)
  const float c2 = fabsf(g.c2);
  const float *p0 = d.parts + (size_t)(2 * w0 + cut.second) * stride;
  int groups = 1;
  while (groups < 32 && AT_ONCE * groups < w1 - w0 + 1) groups *= 2;
  const int lanes = PD_THREADS / groups, lane = threadIdx.x & (lanes - 1), grp = threadIdx.x / lanes;
  const int cpr = D / 4, chunks = rows * cpr;
  auto weight = [&](float m, float M) __attribute__((always_inline)) {
    return m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - M) * c2);
  };
  for (int c0 = (w - w0 - 1) * lanes; c0 < chunks; c0 += (w1 - w0) * lanes) {
    const int c = min(c0 + lane, chunks - 1), r = c / cpr, dd = 4 * (c - r * cpr);
    float M = -INFINITY, L = 0.f;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    for (int k0 = w0 + grp; k0 <= w1; k0 += AT_ONCE * groups) {
      float m[AT_ONCE], l[AT_ONCE];
      f32x4 o[AT_ONCE];
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i) {
        const int k = min(k0 + i * groups, w1);
        const float *p = k == w0 ? p0 : d.parts + (size_t)(2 * k) * stride;
        const float2 ml = *reinterpret_cast<const float2 *>(p + (size_t)PD_ROWS * DP + 2 * r);
        o[i] = *reinterpret_cast<const f32x4 *>(p + (size_t)r * DP + dd);
        m[i] = k0 + i * groups <= w1 ? ml.x : -INFINITY;
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
    if (groups > 1) {
      float *x = sum[threadIdx.x];
      x[0] = M, x[1] = L, x[2] = v[0], x[3] = v[1], x[4] = v[2], x[5] = v[3];
      __syncthreads();
      if (grp == 0) {
        for (int k = 1; k < groups; ++k) M = fmaxf(M, sum[k * lanes + lane][0]);
        L = 0.f;
        v = f32x4{0.f, 0.f, 0.f, 0.f};
        for (int k = 0; k < groups; ++k) {
          const float *y = sum[k * lanes + lane];
          const float f = weight(y[0], M);
          L += y[1] * f;
          v += f32x4{y[2], y[3], y[4], y[5]} * f;
        }
      }
      __syncthreads();
    }
    if (grp == 0 && c0 + lane < chunks) {
      const float inv = L == 0.f ? 0.f : 1.f / L;
      const int i = (int)g.group.div(cut.row0 + r), h = cut.hk * (int)g.group.d + cut.row0 + r - i * (int)g.group.d;
      *reinterpret_cast<att::u32x2 *>(g.out.data + (int64_t)(cut.q0 + i) * g.out.token + h * g.out.head + dd) =
          att::u32x2{pack_bf(v[0] * inv, v[1] * inv), pack_bf(v[2] * inv, v[3] * inv)};
    }
  }
}

}  // namespace paged
}  // namespace pk
