// paged_attention.hip -- attention of the new tokens of many sequences over keys and
// values in pages.
//
// Token i of a sequence's n new ones sees keys [lo, hi): hi = kv - n + i + 1 (causal) or
// kv, lo = kv - n + i + 1 - window.  o = sum_j p_j v_j / sum_j p_j, p_j = 2^(c q.k_j - m)
// with c = scale log2(e) and m the running maximum; zero where no key is seen.
#include <algorithm>
#include <cmath>

#include "paged.hpp"

namespace pk {
namespace paged {
namespace {

struct AttendArgs {
  Heads q, out;
  Cache cache;
  Batch batch;
  int q_heads, causal, window;
  float c2;  // scale * log2(e)
};

// The range of keys that new token i of a sequence sees.
__device__ __forceinline__ void key_range(const AttendArgs &g, const Seq &s, int i, int &lo, int &hi) {
  const int limit = s.kv - s.n + i + 1;
  hi = g.causal ? max(0, limit) : s.kv;
  lo = g.window > 0 && limit > g.window ? limit - g.window : 0;
}

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

}  // namespace
}  // namespace paged
}  // namespace pk

using namespace pk;
using namespace pk::paged;

extern "C" {

size_t pk_paged_attention_workspace_size(int q_heads, const pk_paged_cache *cache, const pk_paged_batch *batch) {
  (void)q_heads, (void)cache, (void)batch;
  return 0;
}

int launch_paged_attention(const pk_tokens *q, const pk_tokens *out, int q_heads, const pk_paged_cache *cache,
                           const pk_paged_batch *batch, float scale, int causal, int window, void *workspace,
                           size_t workspace_bytes, void *stream) {
  const char *who = "launch_paged_attention";
  (void)workspace, (void)workspace_bytes;
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
  g.window = window;
  g.c2 = scale * 1.4426950408889634f;
  return run_general(g, (hipStream_t)stream);
}

}  // extern "C"
