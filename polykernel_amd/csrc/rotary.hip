// rotary.hip -- rotation of positions, alone and on the way into a paged cache.
//
// Pair (a, b) of a head at position p: a' = m (a c - b s), b' = m (b c + a s) with
// c, s = cos, sin of 2 pi p t, t the pair's revolutions per position; fp32 products,
// rounded to bf16 once.  p t is formed in fp64 and reduced to a revolution there:
// in fp32 a position of 10^6 would leave the angle off by 0.06.
#include <algorithm>
#include <cmath>

#include "paged.hpp"

namespace pk {
namespace paged {

int check_cache(const char *who, const pk_paged_cache *c, Cache *out) {
  PK_CHECK_ARG(c && ((c->k && c->v) || c->pages == 0), "%s: null cache", who);
  PK_CHECK_ARG(c->pages >= 0 && c->page_size > 0 && c->heads > 0 && c->dim > 0,
               "%s: invalid cache (%d pages of %d rows, %d heads of %d)", who, c->pages, c->page_size, c->heads, c->dim);
  if (c->dim > 1024) {
    set_error("%s: head dim %d > 1024 is not supported", who, c->dim);
    return PK_ERR_UNSUPPORTED;
  }
  *out = Cache{c->k,      c->v,     c->k_page, c->k_head, c->k_row, c->v_page,
               c->v_head, c->v_row, c->pages,  c->heads,  c->dim,   FastDiv((uint32_t)c->page_size)};
  return PK_OK;
}

int check_batch(const char *who, const pk_paged_batch *b, const pk_paged_cache *c, Batch *out) {
  PK_CHECK_ARG(b, "%s: null batch", who);
  PK_CHECK_ARG(b->sequences >= 0 && b->tokens >= 0 && b->table_width >= 0 && b->max_q >= 0,
               "%s: invalid batch (%d sequences, %d tokens, %d pages each)", who, b->sequences, b->tokens, b->table_width);
  PK_CHECK_ARG((b->page_table || b->table_width == 0 || b->sequences == 0) && (b->kv_len || b->sequences == 0),
               "%s: null page_table or kv_len", who);
  PK_CHECK_ARG(b->q_start || b->tokens >= b->sequences,
               "%s: without q_start every sequence has a token (%d tokens, %d sequences)", who, b->tokens, b->sequences);
  PK_CHECK_ARG((int64_t)b->table_width * c->page_size <= INT32_MAX - 1023,
               "%s: %d pages of %d rows: positions are within 1023 of INT32_MAX", who, b->table_width, c->page_size);
  *out = Batch{b->page_table, b->q_start,     b->kv_len,    b->table_stride,
               b->sequences,  b->tokens,      b->table_width * c->page_size};
  return PK_OK;
}

namespace {

constexpr int RO_THREADS = 256, RO_MAX_HALF = 512;

struct Rotation {
  const double *turns;
  int half, interleaved;  // pairs; half 0: no rotation
  float sine, magnitude;  // sine: -1 to turn back
};

// cos and sin (times the magnitude) of every pair at position p, by the workgroup.
__device__ __forceinline__ void angles(const Rotation &r, int p, float2 *cs) {
  for (int i = threadIdx.x; i < r.half; i += RO_THREADS) {
    const double rev = (double)p * r.turns[i];
    float s, c;
    sincospif(2.f * (float)(rev - rint(rev)), &s, &c);
    cs[i] = make_float2(c * r.magnitude, s * r.sine * r.magnitude);
  }
}

// Pieces of a head: a pair, or one dim behind the rotated ones.
__host__ __device__ __forceinline__ int pieces(int half, int D) { return D - half; }
__device__ __forceinline__ void rotate_piece(const Rotation &r, const float2 *cs, const uint16_t *src, uint16_t *dst, int j) {
  if (j < r.half) {
    const int d0 = r.interleaved ? 2 * j : j, d1 = r.interleaved ? d0 + 1 : j + r.half;
    const float a = bf2f(src[d0]), b = bf2f(src[d1]);
    const float c = cs[j].x, s = cs[j].y;
    dst[d0] = (uint16_t)f2bf(fmaf(a, c, -(b * s)));
    dst[d1] = (uint16_t)f2bf(fmaf(b, c, a * s));
  } else {
    dst[j + r.half] = src[j + r.half];
  }
}

struct RotaryArgs {
  Heads x, out;
  const int32_t *positions;
  int64_t position_stride;
  int S, heads;
  FastDiv per_head;
  Rotation rot;
};

// One token per workgroup.
__global__ __launch_bounds__(RO_THREADS) void rotary_kernel(RotaryArgs g) {
  __shared__ float2 cs[RO_MAX_HALF];
  const int b = blockIdx.x / g.S, s = blockIdx.x % g.S;
  angles(g.rot, g.positions[b * g.position_stride + s], cs);
  __syncthreads();
  const uint16_t *src = g.x.data + b * g.x.batch + s * g.x.token;
  uint16_t *dst = g.out.data + b * g.out.batch + s * g.out.token;
  for (int u = threadIdx.x; u < g.heads * (int)g.per_head.d; u += RO_THREADS) {
    const int h = (int)g.per_head.div(u), j = u - h * (int)g.per_head.d;
    rotate_piece(g.rot, cs, src + h * g.x.head, dst + h * g.out.head, j);
  }
}

struct AppendArgs {
  Heads k, v, q, q_out;
  Cache cache;
  Batch batch;
  int q_heads;  // 0: no queries
  FastDiv per_head, per_value;
  Rotation rot;
};

// One new token per workgroup: its query heads, key heads and value heads.
__global__ __launch_bounds__(RO_THREADS) void paged_append_kernel(AppendArgs g) {
  __shared__ float2 cs[RO_MAX_HALF];
  const int t = blockIdx.x;
  const int b = sequence_of(g.batch, t);
  if (b < 0) return;
  const Seq sq = sequence(g.batch, b);
  const int p = sq.kv - sq.n + t - sq.q0;
  angles(g.rot, p, cs);
  const int page = p >= 0 && p < g.batch.capacity ? page_of(g.batch, g.cache, b, p) : -1;
  const int row = page >= 0 ? p - (int)(g.cache.page.div(p) * g.cache.page.d) : 0;
  __syncthreads();
  const int nq = g.q_heads * (int)g.per_head.d;
  const int nk = page >= 0 ? g.cache.heads * (int)g.per_head.d : 0, nv = page >= 0 ? g.cache.heads * (int)g.per_value.d : 0;
  uint16_t *kc = g.cache.k + page * g.cache.k_page + row * g.cache.k_row;
  uint16_t *vc = g.cache.v + page * g.cache.v_page + row * g.cache.v_row;
  for (int u = threadIdx.x; u < nq + nk + nv; u += RO_THREADS) {
    if (u < nq) {
      const int h = (int)g.per_head.div(u), j = u - h * (int)g.per_head.d;
      rotate_piece(g.rot, cs, g.q.data + t * g.q.token + h * g.q.head, g.q_out.data + t * g.q_out.token + h * g.q_out.head, j);
    } else if (u < nq + nk) {
      const int h = (int)g.per_head.div(u - nq), j = u - nq - h * (int)g.per_head.d;
      rotate_piece(g.rot, cs, g.k.data + t * g.k.token + h * g.k.head, kc + h * g.cache.k_head, j);
    } else {
      const int h = (int)g.per_value.div(u - nq - nk), j = u - nq - nk - h * (int)g.per_value.d;
      vc[h * g.cache.v_head + j] = g.v.data[t * g.v.token + h * g.v.head + j];
    }
  }
}

int check_rotary(const char *who, const pk_rotary *r, int D, Rotation *out) {
  PK_CHECK_ARG(r->turns, "%s: null turns", who);
  PK_CHECK_ARG(r->dim > 0 && r->dim % 2 == 0 && r->dim <= D, "%s: %d rotated dims of a head of %d (even, at most all)", who,
               r->dim, D);
  *out = Rotation{r->turns, r->dim / 2, r->interleaved != 0, r->inverse ? -1.f : 1.f, r->magnitude};
  return PK_OK;
}

}  // namespace
}  // namespace paged
}  // namespace pk

using namespace pk;
using namespace pk::paged;

extern "C" {

int pk_rotary_frequencies(int dim, double base, int scaling, double factor, double low, double high, double original,
                          double *turns, double *magnitude) {
  PK_CHECK_ARG(turns && dim > 0 && dim % 2 == 0 && std::isfinite(base) && base > 0,
               "pk_rotary_frequencies: %d dims (even), base %g", dim, base);
  PK_CHECK_ARG(scaling >= PK_ROTARY_NONE && scaling <= PK_ROTARY_RAMP, "pk_rotary_frequencies: unknown scaling %d", scaling);
  PK_CHECK_ARG(scaling == PK_ROTARY_NONE || (std::isfinite(factor) && factor > 0), "pk_rotary_frequencies: factor %g", factor);
  const bool parts = scaling == PK_ROTARY_BANDS || scaling == PK_ROTARY_RAMP;
  PK_CHECK_ARG(!parts || (std::isfinite(original) && original > 0 && low > 0 && std::isfinite(high) && high > low),
               "pk_rotary_frequencies: original length %g, turns %g to %g", original, low, high);
  PK_CHECK_ARG(scaling != PK_ROTARY_BASE || dim > 2, "pk_rotary_frequencies: a stretched base needs more than one pair");
  PK_CHECK_ARG(scaling != PK_ROTARY_RAMP || base != 1, "pk_rotary_frequencies: a ramp needs pairs of different frequencies");
  const double two_pi = 6.283185307179586476925;
  if (scaling == PK_ROTARY_BASE) base *= std::pow(factor, dim / (dim - 2.0));
  double first = 0, last = 1;
  if (scaling == PK_ROTARY_RAMP) {
    auto pair_of = [&](double n) { return dim * std::log(original / (two_pi * n)) / (2 * std::log(base)); };
    first = std::max(std::floor(pair_of(high)), 0.0);
    last = std::min(std::ceil(pair_of(low)), dim - 1.0);
    if (last <= first) last = first + 1e-3;
  }
  for (int i = 0; i < dim / 2; ++i) {
    const double theta = std::pow(base, -2.0 * i / dim);
    double keep = 1;  // weight of theta, the rest on theta / factor
    if (scaling == PK_ROTARY_LINEAR) keep = 0;
    else if (scaling == PK_ROTARY_BANDS) keep = (original * theta / two_pi - low) / (high - low);
    else if (scaling == PK_ROTARY_RAMP) keep = 1 - (i - first) / (last - first);
    keep = std::min(std::max(keep, 0.0), 1.0);
    turns[i] = (keep == 1 ? theta : theta * keep + theta / factor * (1 - keep)) / two_pi;
  }
  if (magnitude) *magnitude = scaling == PK_ROTARY_RAMP ? 0.1 * std::log(factor) + 1 : 1;
  return PK_OK;
}

int launch_rotary(const uint16_t *x, const int64_t *xs, uint16_t *out, const int64_t *os, const int32_t *positions,
                  int64_t position_stride, int B, int S, int H, int D, const pk_rotary *rotary, void *stream) {
  PK_CHECK_ARG(B >= 0 && S >= 0 && H >= 0 && D > 0, "launch_rotary: invalid shape");
  PK_CHECK_ARG(xs && os && rotary, "launch_rotary: null strides or rotary");
  const int64_t tokens = (int64_t)B * S;
  if (D > 1024) {
    set_error("launch_rotary: head dim %d > 1024 is not supported", D);
    return PK_ERR_UNSUPPORTED;
  }
  RotaryArgs g{};
  if (int rc = check_rotary("launch_rotary", rotary, D, &g.rot)) return rc;
  PK_CHECK_ARG(tokens <= INT32_MAX && (int64_t)H * D <= INT32_MAX, "launch_rotary: B * S = %lld or H * D = %lld exceeds %d",
               (long long)tokens, (long long)H * D, INT32_MAX);
  if (tokens == 0 || H == 0) return PK_OK;
  PK_CHECK_ARG(x && out && positions, "launch_rotary: null tensor pointer");
  g.x = Heads{const_cast<uint16_t *>(x), xs[0], xs[1], xs[2]};
  g.out = Heads{out, os[0], os[1], os[2]};
  g.positions = positions;
  g.position_stride = position_stride;
  g.S = S;
  g.heads = H;
  g.per_head = FastDiv((uint32_t)pieces(g.rot.half, D));
  rotary_kernel<<<(unsigned)tokens, RO_THREADS, 0, (hipStream_t)stream>>>(g);
  PK_LAUNCH_CHECK("rotary_kernel");
  return PK_OK;
}

int launch_paged_kv_append(const pk_tokens *k, const pk_tokens *v, const pk_tokens *q, const pk_tokens *q_out, int q_heads,
                           const pk_paged_cache *cache, const pk_paged_batch *batch, const pk_rotary *rotary, void *stream) {
  const char *who = "launch_paged_kv_append";
  AppendArgs g{};
  if (int rc = check_cache(who, cache, &g.cache)) return rc;
  if (int rc = check_batch(who, batch, cache, &g.batch)) return rc;
  PK_CHECK_ARG(k && v, "%s: null k or v", who);
  PK_CHECK_ARG((q != nullptr) == (q_out != nullptr) && (!q || rotary), "%s: q, q_out and rotary come together", who);
  PK_CHECK_ARG(!q || q_heads > 0, "%s: %d query heads", who, q_heads);
  PK_CHECK_ARG(!rotary || !rotary->inverse, "%s: the inverse rotation is not an append", who);
  if (rotary)
    if (int rc = check_rotary(who, rotary, cache->dim, &g.rot)) return rc;
  g.q_heads = q ? q_heads : 0;
  PK_CHECK_ARG(((int64_t)g.q_heads + 2 * (int64_t)cache->heads) * cache->dim <= INT32_MAX, "%s: %d + 2 x %d heads of %d", who,
               g.q_heads, cache->heads, cache->dim);
  if (batch->tokens == 0 || batch->sequences == 0) return PK_OK;
  PK_CHECK_ARG(k->data && v->data && (!q || (q->data && q_out->data)), "%s: null tensor pointer", who);
  g.k = Heads{k->data, 0, k->token, k->head};
  g.v = Heads{v->data, 0, v->token, v->head};
  if (q) {
    g.q = Heads{q->data, 0, q->token, q->head};
    g.q_out = Heads{q_out->data, 0, q_out->token, q_out->head};
  }
  g.per_head = FastDiv((uint32_t)pieces(g.rot.half, cache->dim));
  g.per_value = FastDiv((uint32_t)cache->dim);
  paged_append_kernel<<<(unsigned)batch->tokens, RO_THREADS, 0, (hipStream_t)stream>>>(g);
  PK_LAUNCH_CHECK("paged_append_kernel");
  return PK_OK;
}

}  // extern "C"
