// paged_attention.hip -- attention of the new tokens of many sequences over keys and
// values in pages.
//
// Token i of a sequence's n new ones sees keys [lo, hi): hi = kv - n + i + 1 (causal) or
// kv, lo = kv - n + i + 1 - window.  o = sum_j p_j v_j / sum_j p_j, p_j = 2^(c q.k_j - m)
// with c = scale log2(e) and m the running maximum; zero where no key is seen.
#include <algorithm>
#include <cmath>

#include "paged_chunk.hpp"
#include "paged_decode.hpp"

namespace pk {
namespace paged {
namespace {

// Any head dim, stride and alignment: a workgroup per token and query head, its waves
// on KEYS of every 8 KEYS keys, a lane on dims lane, lane + 64, ...; states merged in LDS.
// Bound by the chain from a page's number to the sum over the wave, which KEYS keys go
// through together: a token of 8 sequences on 1000 keys, 2 heads to 8 of 100, 49 us (one key at
// a time and half the waves 199), at head dim 512 246.
constexpr int PG_WAVES = 8, PG_THREADS = PG_WAVES * 64;
template <int N>  // dims per lane
__global__ __launch_bounds__(PG_THREADS) void paged_general_kernel(AttendArgs g) {
  constexpr int KEYS = N <= 4 ? 8 : 32 / N;
  __shared__ float so[PG_WAVES][64 * N], sml[PG_WAVES][2];
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, D = g.cache.dim;
  const int t = blockIdx.x, h = blockIdx.y;
  const int b = sequence_of(g.batch, t);
  if (b < 0) return;
  const Seq s = sequence(g.batch, b);
  int lo, hi;
  key_range(g, s, t - s.q0, lo, hi);
  const int hk = h / (g.q_heads / g.cache.heads);
  const uint16_t *qp = g.q.data + t * g.q.token + h * g.q.head;
  const uint16_t *kp = g.cache.k + hk * g.cache.k_head, *vp = g.cache.v + hk * g.cache.v_head;
  float q[N], acc[N], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    q[i] = lane + 64 * i < D ? bf2f(qp[lane + 64 * i]) : 0.f;
    acc[i] = 0.f;
  }
  for (int j0 = lo + wid * KEYS; j0 < hi; j0 += PG_WAVES * KEYS) {
    const uint16_t *kr[KEYS], *vr[KEYS];  // keys that are not there read the query, and take no part
    bool is[KEYS];
    float sc[KEYS];
#pragma unroll
    for (int u = 0; u < KEYS; ++u) {
      const int j = j0 + u, page = j < hi ? page_of(g.batch, g.cache, b, j) : -1;
      const int row = j - (int)(g.cache.page.div(j) * g.cache.page.d);
      is[u] = page >= 0;
      kr[u] = is[u] ? kp + page * g.cache.k_page + row * g.cache.k_row : qp;
      vr[u] = is[u] ? vp + page * g.cache.v_page + row * g.cache.v_row : qp;
      sc[u] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (lane + 64 * i < D) {
#pragma unroll
        for (int u = 0; u < KEYS; ++u) sc[u] = fmaf(q[i], bf2f(kr[u][lane + 64 * i]), sc[u]);
      }
    float m_new = m;
#pragma unroll
    for (int u = 0; u < KEYS; ++u) {
      const float sum = wave_sum(sc[u]) * g.c2;
      sc[u] = is[u] ? sum : -INFINITY;
      m_new = fmaxf(m_new, sc[u]);
    }
    const float mu = m_new == -INFINITY ? 0.f : m_new;
    const float alpha = __builtin_amdgcn_exp2f(m - mu);
    m = m_new;
    l *= alpha;
#pragma unroll
    for (int u = 0; u < KEYS; ++u) {
      sc[u] = __builtin_amdgcn_exp2f(sc[u] - mu);
      l += sc[u];
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (lane + 64 * i < D) {
        acc[i] *= alpha;
#pragma unroll
        for (int u = 0; u < KEYS; ++u) {
          const float v = bf2f(vr[u][lane + 64 * i]);
          acc[i] = fmaf(sc[u], is[u] ? v : 0.f, acc[i]);
        }
      }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) so[wid][lane + 64 * i] = acc[i];
  if (lane == 0) {
    sml[wid][0] = m;
    sml[wid][1] = l;
  }
  __syncthreads();
  float M = -INFINITY, L = 0.f, w[PG_WAVES];
#pragma unroll
  for (int k = 0; k < PG_WAVES; ++k) M = fmaxf(M, sml[k][0]);
#pragma unroll
  for (int k = 0; k < PG_WAVES; ++k) {
    w[k] = sml[k][0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(sml[k][0] - M);
    L += sml[k][1] * w[k];
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
  uint16_t *op = g.out.data + t * g.out.token + h * g.out.head;
  for (int d = threadIdx.x; d < D; d += PG_THREADS) {
    float o = 0.f;
#pragma unroll
    for (int k = 0; k < PG_WAVES; ++k) o += so[k][d] * w[k];
    op[d] = (uint16_t)f2bf(o * inv);
  }
}

int run_general(const AttendArgs &g, hipStream_t st) {
  const int D = g.cache.dim;
  if (2 * (int64_t)g.batch.tokens > MOST_BLOCKS || g.q_heads > 65535) {
    set_error("launch_paged_attention: %d tokens of %d query heads are not supported", g.batch.tokens, g.q_heads);
    return PK_ERR_UNSUPPORTED;
  }
  const dim3 n(g.batch.tokens, g.q_heads);
  if (D <= 64) paged_general_kernel<1><<<n, PG_THREADS, 0, st>>>(g);
  else if (D <= 128) paged_general_kernel<2><<<n, PG_THREADS, 0, st>>>(g);
  else if (D <= 256) paged_general_kernel<4><<<n, PG_THREADS, 0, st>>>(g);
  else if (D <= 512) paged_general_kernel<8><<<n, PG_THREADS, 0, st>>>(g);
  else paged_general_kernel<16><<<n, PG_THREADS, 0, st>>>(g);
  PK_LAUNCH_CHECK("paged_general_kernel");
  return PK_OK;
}

// ---- the fast kernels (paged_decode.hpp, paged_chunk.hpp) ------------------------
template <int DP, int PAGE>
__global__ __launch_bounds__(PD_THREADS, pd_groups(DP)) void paged_decode_kernel(DecodeArgs d) {
  paged_decode_body<DP, PAGE>(d);
}
template <int DP>
__global__ __launch_bounds__(PD_THREADS) void paged_decode_merge_kernel(DecodeArgs d) {
  paged_decode_merge_body<DP>(d);
}
template <int DP, int DC, int PAGE>
__global__ __launch_bounds__(PC_THREADS, DP == 256 ? 1 : DP == 64 ? 4 : 2) void paged_chunk_kernel(ChunkArgs d) {
  paged_chunk_body<DP, DC, PAGE>(d);
}
template <int DP, int DC>
__global__ __launch_bounds__(PC_THREADS) void paged_chunk_merge_kernel(ChunkArgs d) {
  paged_chunk_merge_body<DP, DC>(d);
}

// How a call runs: head dims padded to `dp` (0: by the general kernel); sequences of up to
// 16 rows (tokens x heads of a group) by the step kernel (workers > 0: at most so many
// workgroups, items cut between them unless `whole`), sequences of more by the chunk kernel
// (splits > 0: `items` items at most, each in up to `splits` runs of keys).  A kernel that
// runs alone takes all sequences.
//
// The step kernel with 32 or 64 rows to an item was slower than the chunk kernel (24
// sequences of 5 tokens on up to 3000 keys, 8 heads to 32, 50 against 48 us; of 8 tokens 49
// and 44; 32 of 6, 8 to 56 heads of 64, 45 and 28; 8 of one token on 8000, 1 to 64, 30 and 20).
struct Choice {
  int dp = 0, workers = 0, whole = 0, splits = 0, items = 0;
  size_t workspace() const {
    if (!dp) return 0;
    const size_t few = workers > 1 && !whole ? pd_workspace(dp, workers) : 0;
    const size_t many = splits > 1 ? (size_t)items * splits * pc_part_floats(dp) * sizeof(float) : 0;
    return std::max(few, many);
  }
};

// Runs of keys of the chunk kernel's items: what a workgroup of the longest item takes among
// those beside it, or, of more than run at once, what a CU takes for all of its own and the end
// of the last, against the states that are written and added (66 KB each at D 128).  `part`:
// an item's steps on average, of the longest's.  `us`: a step of one workgroup alone on a CU;
// `shared`: of each more that runs beside it.
// 8 heads to 32, D 128: 512 tokens on 4096 keys 79 us in one run, 59 in 2 and 50 in 4 (taken);
// 1000 on 1000 27 (taken), 36 and 41; 128 on 16000 296, 157 and 86, 50 in 16 (taken); 24
// sequences of 5 on up to 3000 56, 41, 38 in 3 (taken) and 40.  8 heads to 8: 5 of up to 4000 on
// up to 9000 345 (taken), 390 and 432.
int chunk_splits(int64_t items, int64_t steps, double part, int dp) {
  const int at_once = dp == 64 ? 4 : dp == 128 ? 2 : 1;
  const double us = dp == 64 ? 0.8 : dp == 128 ? 1.2 : 2.3, shared = dp == 64 ? 0.6 : dp == 128 ? 0.97 : 2.3;
  int best = 1;
  double least = 1e30;
  for (int s = 1; s <= 32 && (s == 1 || 4 * s <= steps); ++s) {
    const double groups = (double)items * s, per_cu = groups / 256, longest = (double)((steps + s - 1) / s);
    double time = 3 + (per_cu <= at_once ? std::max(us, shared * std::ceil(per_cu)) * longest
                                         : (shared * part * longest + 1) * per_cu + 0.4 * us * longest);
    if (s > 1) time += 3.5 + 0.02 * dp / 128 * groups;
    if (time < least) {
      least = time;
      best = s;
    }
  }
  return best;
}

Choice choose(int q_heads, const pk_paged_cache &c, const pk_paged_batch &b, int window) {
  Choice r;
  if (c.dim > 256 || c.dim % 8 != 0) return r;
  const int dp = c.dim <= 64 ? 64 : c.dim <= 128 ? 128 : 256;
  const int64_t group = q_heads / c.heads, B = b.sequences;
  int64_t keys = (int64_t)b.table_width * c.page_size;  // of a sequence, at most
  if (b.max_kv > 0) keys = std::min<int64_t>(keys, b.max_kv);
  const int64_t steps = (int64_t)b.table_width * c.page_size / PT_STEP + 2;  // of an item, whatever the hint
  // a hint of fewer tokens than there are on average is none
  const int64_t most = std::max<int64_t>(b.max_q, (b.tokens + B - 1) / B);
  const bool even = (int64_t)b.max_q * B == b.tokens;  // all sequences have the hint's length
  // Short runs of few sequences are the step kernel's up to two items for each: 5 tokens on 1000
  // keys, 8 heads to 32, 11.0 us against 14.0; four sequences of 5 on up to 3000 are not, 22.0 and 19.9.
  const bool brief = B * c.heads * steps <= 512;
  const bool chunks = most * group > (brief ? 2 * PD_ROWS : PD_ROWS);
  bool few = !chunks;
  if (chunks) {
    const int64_t items = (b.tokens * group / PC_ROWS + B) * c.heads;
    // as many as there will be: exactly, or half of the last tiles of sequences
    const int64_t likely = B == 1 || even ? B * ((b.tokens / B * group + PC_ROWS - 1) / PC_ROWS) * c.heads
                                          : (b.tokens * group / PC_ROWS + (B + 1) / 2) * c.heads;
    int64_t reach = keys / PT_STEP + 1;
    // (lengths are taken to be uneven; of one sequence's tokens the first see `most` keys less than the last)
    auto part = [&](int64_t of) { return B > 1 ? 0.6 : 1 - 0.5 * std::min(1.0, (double)most / (PT_STEP * of)); };
    int splits = chunk_splits(likely, reach, part(reach), dp);
    if (window > 0) {  // (no more splits than without, which the workspace is for)
      reach = std::min<int64_t>(reach, (window + PT_KEYS) / PT_STEP + 2);
      splits = std::min(splits, chunk_splits(likely, reach, part(reach), dp));
    }
    if (items * splits > MOST_BLOCKS) return r;
    r.items = (int)items;
    r.splits = splits;
    // Sequences of few rows beside chunks are the step kernel's, unless all are chunks, or the
    // few cost the chunk kernel less than another launch and merge: 30 tokens beside 2 chunks of
    // 500, 8 heads to 32, on up to 1000 keys 61 us with both kernels and 53 with one, 2000 92 and
    // 81, 4000 136 and 134; 60 beside 2048 on 2000 187 and 240; 8 beside 200 on 3000 60 and 50.
    few = !(B == 1 || even || B * c.heads * reach <= 8192);
  }
  if (few) {
    // no more workgroups than the tables can have work for
    const int64_t items = (b.tokens * group / PD_ROWS + B) * c.heads;
    if (items > INT32_MAX / steps) return Choice{};  // a line of 2^31 steps or more: the general kernel
    // Items are left whole, and nothing is merged, where their steps are few, or so many items fill
    // the machine.  8 heads to 32, D 128: 64 sequences of up to 1000 keys 28.5 us whole and 31 cut,
    // of 2000 54 and 56; 128 at D 64 33 and 47; 16 of 500 13.9 and 15.4, of 700 17.4 and 13.9; 1 of
    // 250 9.2 and 9.6, of 350 11.0 and 9.8.  At D 256, 4 heads to 16, 1 of 180 11.1 and 11.3, of 250
    // 12.4 and 11.2.
    const int64_t likely = chunks ? B * c.heads : items;
    const int64_t most_steps = likely >= 512 ? 34 : likely >= 128 ? 8 : dp == 256 ? 3 : 5;
    r.whole = keys <= most_steps * PT_STEP;
    r.workers = (int)std::max<int64_t>(1, std::min<int64_t>(256 * pd_groups(dp), r.whole ? items : items * steps));
  }
  r.dp = dp;
  return r;
}

bool tile_operands(const AttendArgs &g) {
  const Cache &c = g.cache;
  // row offsets within a page, in bytes, and the length of 16 rows are 32-bit numbers
  auto rows = [&](int64_t row) { return row >= c.dim && row < (int64_t(1) << 26) && row * 2 * c.page.d < (int64_t(1) << 32); };
  return aligned16(g.q.data) && aligned16(g.out.data) && aligned16(c.k) && aligned16(c.v) &&
         strides8(g.q.token, g.q.head) && strides8(g.out.token, g.out.head) && strides8(c.k_page, c.k_head, c.k_row) &&
         strides8(c.v_page, c.v_head, c.v_row) && rows(c.k_row) && rows(c.v_row);
}

template <int DP>
int run_decode_as(const DecodeArgs &d, hipStream_t st) {
  const uint32_t page = d.a.cache.page.d;
  if (page % 16 == 0) paged_decode_kernel<DP, 16><<<d.most, PD_THREADS, 0, st>>>(d);
  else if (page % 8 == 0) paged_decode_kernel<DP, 8><<<d.most, PD_THREADS, 0, st>>>(d);
  else paged_decode_kernel<DP, 1><<<d.most, PD_THREADS, 0, st>>>(d);
  PK_LAUNCH_CHECK("paged_decode_kernel");
  if (d.most > 1 && !d.whole) {
    paged_decode_merge_kernel<DP><<<d.most - 1, PD_THREADS, 0, st>>>(d);
    PK_LAUNCH_CHECK("paged_decode_merge_kernel");
  }
  return PK_OK;
}
template <int DP, int DC>
int run_chunk_as(const ChunkArgs &d, hipStream_t st) {
  const unsigned blocks = pc_blocks(d.items * d.splits);
  const uint32_t page = d.a.cache.page.d;
  if (page % 16 == 0) paged_chunk_kernel<DP, DC, 16><<<blocks, PC_THREADS, 0, st>>>(d);
  else if (page % 8 == 0) paged_chunk_kernel<DP, DC, 8><<<blocks, PC_THREADS, 0, st>>>(d);
  else paged_chunk_kernel<DP, DC, 1><<<blocks, PC_THREADS, 0, st>>>(d);
  PK_LAUNCH_CHECK("paged_chunk_kernel");
  if (d.splits > 1) {
    paged_chunk_merge_kernel<DP, DC><<<dim3(d.items, PC_MERGE), PC_THREADS, 0, st>>>(d);
    PK_LAUNCH_CHECK("paged_chunk_merge_kernel");
  }
  return PK_OK;
}
template <int DP>
int run_as(const AttendArgs &g, const Choice &c, float *workspace, hipStream_t st) {
  if (c.workers) {
    const DecodeArgs d{g, workspace, c.workers, c.splits ? PD_ROWS + 1 : INT32_MAX, c.whole};
    if (int rc = run_decode_as<DP>(d, st)) return rc;
  }
  if (c.splits) {
    const ChunkArgs d{g, workspace, c.items, c.splits, c.workers ? PD_ROWS : 0};
    // three quarters of the dims are products enough for head dims up to there
    if constexpr (DP > 64)
      if (g.cache.dim <= DP / 4 * 3) return run_chunk_as<DP, DP / 4 * 3>(d, st);
    return run_chunk_as<DP, DP>(d, st);
  }
  return PK_OK;
}

}  // namespace
}  // namespace paged
}  // namespace pk

using namespace pk;
using namespace pk::paged;

extern "C" {

int pk_paged_attention_plan(int q_heads, const pk_paged_cache *cache, const pk_paged_batch *batch, int window,
                            pk_paged_plan *out) {
  const char *who = "pk_paged_attention_plan";
  Cache c;
  Batch b;
  if (int rc = check_cache(who, cache, &c)) return rc;
  if (int rc = check_batch(who, batch, cache, &b)) return rc;
  PK_CHECK_ARG(out && q_heads > 0 && q_heads % cache->heads == 0 && window >= 0 && batch->sequences > 0, "%s: invalid argument", who);
  const Choice r = choose(q_heads, *cache, *batch, window >= b.capacity ? 0 : window);
  *out = pk_paged_plan{r.dp, r.workers, r.whole, r.splits, r.items};
  return PK_OK;
}

size_t pk_paged_attention_workspace_size(int q_heads, const pk_paged_cache *cache, const pk_paged_batch *batch) {
  if (!cache || !batch || q_heads <= 0 || cache->heads <= 0 || q_heads % cache->heads != 0 || cache->dim <= 0 ||
      cache->page_size <= 0 || batch->tokens <= 0 || batch->sequences <= 0 || batch->table_width < 0)
    return 0;
  return choose(q_heads, *cache, *batch, 0).workspace();  // a window takes no more
}

int launch_paged_attention(const pk_tokens *q, const pk_tokens *out, int q_heads, const pk_paged_cache *cache,
                           const pk_paged_batch *batch, float scale, int causal, int window, void *workspace,
                           size_t workspace_bytes, void *stream) {
  const char *who = "launch_paged_attention";
  AttendArgs g{};
  if (int rc = check_cache(who, cache, &g.cache)) return rc;
  if (int rc = check_batch(who, batch, cache, &g.batch)) return rc;
  PK_CHECK_ARG(q && out, "%s: null q or out", who);
  PK_CHECK_ARG(q_heads > 0 && q_heads % cache->heads == 0, "%s: %d query heads over %d key heads", who, q_heads, cache->heads);
  PK_CHECK_ARG(window >= 0, "%s: window %d", who, window);
  PK_CHECK_ARG((int64_t)batch->tokens * q_heads <= INT32_MAX, "%s: tokens * q_heads = %lld exceeds %d", who,
               (long long)batch->tokens * q_heads, INT32_MAX);
  if (batch->tokens == 0 || batch->sequences == 0) return PK_OK;
  PK_CHECK_ARG(q->data && out->data, "%s: null tensor pointer", who);
  g.q = Heads{q->data, 0, q->token, q->head};
  g.out = Heads{out->data, 0, out->token, out->head};
  g.q_heads = q_heads;
  g.causal = causal != 0;
  g.window = window >= g.batch.capacity ? 0 : window;  // (hides nothing)
  g.c2 = scale * 1.4426950408889634f;
  g.group = FastDiv((uint32_t)(q_heads / cache->heads));
  const Choice c = choose(q_heads, *cache, *batch, g.window);
  // a scale of 0, infinity or no number has no place in the exponents of the fast kernels
  if (!c.dp || !tile_operands(g) || !(std::fabs(g.c2) > 0.f) || std::isinf(g.c2)) return run_general(g, (hipStream_t)stream);
  if (workspace_bytes < c.workspace() || (c.workspace() && (!workspace || !aligned16(workspace)))) {
    set_error("%s: needs a 16-byte aligned workspace of %zu bytes, got %zu", who, c.workspace(), workspace_bytes);
    return PK_ERR_WORKSPACE;
  }
  float *const parts = static_cast<float *>(workspace);
  return c.dp == 64    ? run_as<64>(g, c, parts, (hipStream_t)stream)
         : c.dp == 128 ? run_as<128>(g, c, parts, (hipStream_t)stream)
                       : run_as<256>(g, c, parts, (hipStream_t)stream);
}

}  // extern "C"
