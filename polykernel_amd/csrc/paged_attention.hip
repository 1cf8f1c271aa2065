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
// on every fourth key, a lane on dims lane, lane + 64, ...; states merged in LDS.
constexpr int PG_WAVES = 4, PG_THREADS = PG_WAVES * 64;
template <int N>  // dims per lane
__global__ __launch_bounds__(PG_THREADS) void paged_general_kernel(AttendArgs g) {
  __shared__ float so[PG_WAVES][64 * N], sml[PG_WAVES][2];
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, D = g.cache.dim;
  const int t = blockIdx.x / g.q_heads, h = blockIdx.x % g.q_heads;
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
  for (int j = lo + wid; j < hi; j += PG_WAVES) {
    const int page = page_of(g.batch, g.cache, b, j);
    if (page < 0) continue;
    const int row = j - (int)(g.cache.page.div(j) * g.cache.page.d);
    const uint16_t *kr = kp + page * g.cache.k_page + row * g.cache.k_row;
    const uint16_t *vr = vp + page * g.cache.v_page + row * g.cache.v_row;
    float sc = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (lane + 64 * i < D) sc = fmaf(q[i], bf2f(kr[lane + 64 * i]), sc);
    sc = wave_sum(sc) * g.c2;
    const float m_new = fmaxf(m, sc);
    const float mu = m_new == -INFINITY ? 0.f : m_new;
    const float alpha = __builtin_amdgcn_exp2f(m - mu), p = __builtin_amdgcn_exp2f(sc - mu);
    m = m_new;
    l = fmaf(l, alpha, p);
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (lane + 64 * i < D) acc[i] = fmaf(acc[i], alpha, p * bf2f(vr[lane + 64 * i]));
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
  const int64_t blocks = (int64_t)g.batch.tokens * g.q_heads;
  const unsigned n = (unsigned)blocks;
  const int D = g.cache.dim;
  if (D <= 64) paged_general_kernel<1><<<n, PG_THREADS, 0, st>>>(g);
  else if (D <= 128) paged_general_kernel<2><<<n, PG_THREADS, 0, st>>>(g);
  else if (D <= 256) paged_general_kernel<4><<<n, PG_THREADS, 0, st>>>(g);
  else paged_general_kernel<16><<<n, PG_THREADS, 0, st>>>(g);
  PK_LAUNCH_CHECK("paged_general_kernel");
  return PK_OK;
}

// ---- the fast kernels (paged_decode.hpp, paged_chunk.hpp) ------------------------
template <int DP, int MT, bool PAGE16>
__global__ __launch_bounds__(PD_THREADS, (DecodeShape<DP, MT>::GROUPS)) void paged_decode_kernel(DecodeArgs d) {
  paged_decode_body<DP, MT, PAGE16>(d);
}
template <int DP, int MT>
__global__ __launch_bounds__(PD_THREADS) void paged_decode_merge_kernel(DecodeArgs d) {
  paged_decode_merge_body<DP, MT>(d);
}
template <int DP, int DC, bool PAGE16>
__global__ __launch_bounds__(PC_THREADS, DP == 256 ? 1 : DP == 64 ? 4 : 2) void paged_chunk_kernel(ChunkArgs d) {
  paged_chunk_body<DP, DC, PAGE16>(d);
}
template <int DP, int DC>
__global__ __launch_bounds__(PC_THREADS) void paged_chunk_merge_kernel(ChunkArgs d) {
  paged_chunk_merge_body<DP, DC>(d);
}

constexpr int PD_LEAST = 1;   // steps of a workgroup
// Workgroups of the step kernel on a CU.
constexpr int step_groups(int dp, int mt) {
  return dp == 64    ? mt == 1 ? DecodeShape<64, 1>::GROUPS : mt == 2 ? DecodeShape<64, 2>::GROUPS : DecodeShape<64, 4>::GROUPS
         : dp == 128 ? mt == 1 ? DecodeShape<128, 1>::GROUPS : mt == 2 ? DecodeShape<128, 2>::GROUPS : DecodeShape<128, 4>::GROUPS
         : mt == 1   ? DecodeShape<256, 1>::GROUPS
                     : DecodeShape<256, 2>::GROUPS;
}
constexpr int PD_ROWS = 64;   // rows (tokens x heads of a group) of a sequence up to which it is not a chunk

// How a call runs: head dims padded to `dp` (0: by the general kernel); sequences of up to
// PD_ROWS rows by the decode kernel (mt > 0: 16 mt rows per item, at most `workers`
// workgroups, items cut between them unless `whole`), sequences of more by the chunk kernel
// (splits > 0: `items` items at most, each in `splits` runs of keys).  A kernel that runs
// alone takes all sequences.
struct Choice {
  int dp = 0, mt = 0, workers = 0, whole = 0, splits = 0, items = 0;
  size_t workspace() const {
    if (!dp) return 0;
    const size_t few = mt && workers > 1 && !whole ? pd_workspace(dp, mt, workers) : 0;
    const size_t many = splits > 1 ? (size_t)items * splits * pc_part_floats(dp) * sizeof(float) : 0;
    return std::max(few, many);
  }
};

Choice choose(int q_heads, const pk_paged_cache &c, const pk_paged_batch &b, int window) {
  Choice r;
  if (c.dim > 256 || c.dim % 8 != 0) return r;
  const int dp = c.dim <= 64 ? 64 : c.dim <= 128 ? 128 : 256;
  const int64_t slots = dp == 256 ? 256 : 512;  // chunk workgroups that run at once
  const int64_t group = q_heads / c.heads;
  const int64_t steps = (int64_t)b.table_width * c.page_size / PT_STEP + 2;  // of an item, at most
  // a hint of fewer tokens than there are on average is none
  const int64_t most = std::max<int64_t>(b.max_q, ((int64_t)b.tokens + b.sequences - 1) / b.sequences);
  const bool chunks = most * group > PD_ROWS;
  // Beside chunks the decode kernel takes the others, but not where every sequence is a chunk
  // (there is one, or all have the hint's length), nor where no token reaches further than the
  // chunks' own work goes on (mixed batch of 4 prompts of up to 1531 tokens and 20 single ones, D
  // 64, the last 1024 keys: 54 us and 17 of the decode kernel and its merge, FIGURE with one kernel).
  const int64_t reach = window > 0 ? std::min<int64_t>((window + PT_KEYS) / PT_STEP + 2, steps) : steps;
  const bool few = !chunks || !(b.sequences == 1 || (int64_t)b.max_q * b.sequences == b.tokens || reach <= 32);
  if (chunks) {
    const int64_t items = ((int64_t)b.tokens * group / PC_ROWS + b.sequences) * c.heads;
    const int64_t splits = std::max<int64_t>(1, std::min<int64_t>({slots / items, steps / 8, 32}));
    if (items * splits > INT32_MAX) return r;
    r.items = (int)items;
    r.splits = (int)splits;
  }
  if (few) {
    const int64_t rows = chunks ? group : most * group;
    r.mt = rows <= 16 ? 1 : rows <= 32 || dp == 256 ? 2 : 4;
    // no more workgroups than the tables can have work for
    const int64_t items = ((int64_t)b.tokens * group / (16 * r.mt) + b.sequences) * c.heads;
    if (items > INT32_MAX / steps) return r;  // a line of 2^31 steps or more: the general kernel
    r.whole = steps <= 8;
    r.workers = (int)std::max<int64_t>(1, std::min<int64_t>(256 * step_groups(dp, r.mt), r.whole ? items : items * steps / PD_LEAST));
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

template <int DP, int MT>
int run_decode_as(const DecodeArgs &d, hipStream_t st) {
  if (d.a.cache.page.d % PT_KEYS == 0) paged_decode_kernel<DP, MT, true><<<d.most, PD_THREADS, 0, st>>>(d);
  else paged_decode_kernel<DP, MT, false><<<d.most, PD_THREADS, 0, st>>>(d);
  PK_LAUNCH_CHECK("paged_decode_kernel");
  if (d.most > 1 && !d.whole) {
    paged_decode_merge_kernel<DP, MT><<<d.most - 1, PD_THREADS, 0, st>>>(d);
    PK_LAUNCH_CHECK("paged_decode_merge_kernel");
  }
  return PK_OK;
}
template <int DP, int DC>
int run_chunk_as(const ChunkArgs &d, hipStream_t st) {
  const unsigned blocks = (unsigned)d.items * d.splits;
  if (d.a.cache.page.d % PT_KEYS == 0) paged_chunk_kernel<DP, DC, true><<<blocks, PC_THREADS, 0, st>>>(d);
  else paged_chunk_kernel<DP, DC, false><<<blocks, PC_THREADS, 0, st>>>(d);
  PK_LAUNCH_CHECK("paged_chunk_kernel");
  if (d.splits > 1) {
    paged_chunk_merge_kernel<DP, DC><<<dim3(d.items, PC_MERGE), PC_THREADS, 0, st>>>(d);
    PK_LAUNCH_CHECK("paged_chunk_merge_kernel");
  }
  return PK_OK;
}
template <int DP>
int run_as(const AttendArgs &g, const Choice &c, float *workspace, hipStream_t st) {
  if (c.mt) {
    const DecodeArgs d{g, workspace, c.whole ? 1 : PD_LEAST, c.workers, c.splits ? PD_ROWS + 1 : INT32_MAX, c.whole};
    int rc = PK_OK;
    if (c.mt == 1) rc = run_decode_as<DP, 1>(d, st);
    else if (c.mt == 2 || DP == 256) rc = run_decode_as<DP, 2>(d, st);
    else rc = run_decode_as<DP, DP == 256 ? 2 : 4>(d, st);
    if (rc) return rc;
  }
  if (c.splits) {
    const ChunkArgs d{g, workspace, c.items, c.splits, c.mt ? PD_ROWS : 0};
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
  *out = pk_paged_plan{r.dp, 16 * r.mt, r.workers, r.whole, r.splits, r.items};
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
