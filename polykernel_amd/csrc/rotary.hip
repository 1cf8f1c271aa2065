// rotary.hip -- rotation of positions, alone and on the way into a paged cache.
//
// Pair (a, b) of a head at position p: a' = m (a c - b s), b' = m (b c + a s) with
// c, s = cos, sin of 2 pi p t, t the pair's revolutions per position; fp32 products,
// rounded to bf16 once.  p t is formed in fp64 and reduced to a revolution there:
// in fp32 a position of 10^6 would leave the angle off by 0.06.
#include <algorithm>
#include <cmath>

#include "attention_kernels.hpp"
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
  PK_CHECK_ARG(b->sequences >= 0 && b->tokens >= 0 && b->table_width >= 0 && b->max_q >= 0 && b->max_kv >= 0,
               "%s: invalid batch (%d sequences, %d tokens, %d pages each)", who, b->sequences, b->tokens, b->table_width);
  PK_CHECK_ARG((b->page_table || b->table_width == 0 || b->sequences == 0) && (b->kv_len || b->sequences == 0),
               "%s: null page_table or kv_len", who);
  PK_CHECK_ARG(b->q_start || b->tokens >= b->sequences,
               "%s: without q_start every sequence has a token (%d tokens, %d sequences)", who, b->tokens, b->sequences);
  // (a wave looks up the pages of 64 tiles, of which the last may lie behind all keys)
  PK_CHECK_ARG((int64_t)b->table_width * c->page_size <= INT32_MAX - 65535,
               "%s: %d pages of %d rows: positions are within 65535 of INT32_MAX", who, b->table_width, c->page_size);
  *out = Batch{b->page_table, b->q_start,     b->kv_len,    b->table_stride,
               b->sequences,  b->tokens,      b->table_width * c->page_size};
  return PK_OK;
}

namespace {

constexpr int RO_THREADS = 256;

struct Rotation {
  const double *turns;
  int half, interleaved;  // pairs; half 0: no rotation
  float sine, magnitude;  // sine: -1 to turn back
};

// Work on a head, in units of V dims (16 bytes, or one where strides, alignment or the
// number of pairs allow no more): the pairs of a unit, or of two units half a rotation
// apart; then a unit behind the rotated dims.
template <int V>
__host__ __device__ __forceinline__ int pieces(int half, int interleaved, int D) {
  const int rotated = V == 1 ? half : interleaved ? 2 * half / V : half / V;
  return rotated + (D - 2 * half) / V;
}
template <int V>
struct Piece {
  att::u32x4 a, b;  // V 8: the units; V 1: a dim in the low half of each first word
};
// Offsets of piece j's two units in its head (the second is the first where there is one).
template <int V>
__device__ __forceinline__ void place(const Rotation &r, int j, int &d0, int &d1, bool &rotated) {
  if constexpr (V == 1) {
    rotated = j < r.half;
    d0 = !rotated ? j + r.half : r.interleaved ? 2 * j : j;
    d1 = !rotated ? d0 : r.interleaved ? d0 + 1 : j + r.half;
  } else {
    const int n = r.interleaved ? 2 * r.half / V : r.half / V;
    rotated = j < n;
    d0 = V * (rotated || r.interleaved ? j : j + n);
    d1 = rotated && !r.interleaved ? d0 + r.half : d0;
  }
}
template <int V>
__device__ __forceinline__ Piece<V> read_piece(const Rotation &r, const uint16_t *src, int j) {
  int d0, d1;
  bool rotated;
  place<V>(r, j, d0, d1, rotated);
  Piece<V> p;
  if constexpr (V == 8) {
    p.a = __builtin_nontemporal_load(reinterpret_cast<const att::u32x4 *>(src + d0));
    if (d1 != d0) p.b = __builtin_nontemporal_load(reinterpret_cast<const att::u32x4 *>(src + d1));
  } else {
    p.a[0] = src[d0];
    if (d1 != d0) p.b[0] = src[d1];
  }
  return p;
}
__device__ __forceinline__ void turn(float2 cs, float a, float b, float &x, float &y) {
  x = fmaf(a, cs.x, -(b * cs.y));
  y = fmaf(b, cs.x, a * cs.y);
}
// cs: the token's cosines and sines, times the magnitude.
template <int V>
__device__ __forceinline__ void write_piece(const Rotation &r, const float2 *cs, Piece<V> p, uint16_t *dst, int j) {
  int d0, d1;
  bool rotated;
  place<V>(r, j, d0, d1, rotated);
  if constexpr (V == 1) {
    if (!rotated) {
      dst[d0] = (uint16_t)p.a[0];
      return;
    }
    float x, y;
    turn(cs[j], bf2f(p.a[0]), bf2f(p.b[0]), x, y);
    dst[d0] = (uint16_t)f2bf(x);
    dst[d1] = (uint16_t)f2bf(y);
  } else {
    if (rotated && r.interleaved) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float x, y;
        turn(cs[4 * j + e], lo_bf(p.a[e]), hi_bf(p.a[e]), x, y);
        p.a[e] = pack_bf(x, y);
      }
    } else if (rotated) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float x0, y0, x1, y1;
        turn(cs[8 * j + 2 * e], lo_bf(p.a[e]), lo_bf(p.b[e]), x0, y0);
        turn(cs[8 * j + 2 * e + 1], hi_bf(p.a[e]), hi_bf(p.b[e]), x1, y1);
        p.a[e] = pack_bf(x0, x1);
        p.b[e] = pack_bf(y0, y1);
      }
      *reinterpret_cast<att::u32x4 *>(dst + d1) = p.b;
    }
    *reinterpret_cast<att::u32x4 *>(dst + d0) = p.a;
  }
}

struct RotateArgs {
  Heads q, q_out;          // what is rotated from tensor to tensor
  Heads k, v;              // append: new keys and values
  Cache cache;
  Batch batch;
  const int32_t *positions;  // rotary: of token (b, s) at b * position_stride + s
  int64_t position_stride;
  int tokens;
  int per_group;             // tokens of a workgroup
  FastDiv of_token, of_head, of_value;  // pieces of a token, of a rotated head, of a value head
  FastDiv of_entry;                     // rotary: tokens of a batch entry
  int q_pieces, k_pieces;
  Rotation rot;
};

// A workgroup takes `per_group` tokens: their positions and places (a wave per token),
// the angles of all pairs, then the pieces of all heads.  What bounds it: the memory, 2 x
// 16 bytes in and out per piece; the first piece of a thread is read before the places
// are known, which hides most of that chain of reads in a call of few tokens.  The gradient
// of 2 x 4096 tokens, 32 heads of 128: 134 MB in 26.5 us, 5.1 TB/s; 8 prompts of up to 4096
// tokens, 32 + 2 x 8 heads, into pages: 548 MB in 113 us, 4.85 TB/s, a copy's rate.  One token:
// 2.3 us, an append for 16 5.5.  Four tokens to a workgroup share its look-ups and angles.
constexpr int RO_TOKENS = 4;
template <int V, bool APPEND>
__global__ __launch_bounds__(RO_THREADS) void rotate_kernel(RotateArgs g) {
  extern __shared__ float2 cs[];  // [per_group][half]
  __shared__ int pos_s[RO_TOKENS], page_s[RO_TOKENS], row_s[RO_TOKENS];
  const int t0 = blockIdx.x * g.per_group, n = min(g.per_group, g.tokens - t0);
  const int tid = threadIdx.x, units = n * (int)g.of_token.d;
  // where piece u comes from, and its number in its head
  struct From {
    const uint16_t *head;
    int token, piece, h, kind;  // kind 0: query, 1: key, 2: value
  };
  auto from = [&](int u) __attribute__((always_inline)) {
    From f;
    f.token = (int)g.of_token.div(u);
    int w = u - f.token * (int)g.of_token.d;
    const int t = t0 + f.token;
    f.kind = !APPEND || w < g.q_pieces ? 0 : w < g.q_pieces + g.k_pieces ? 1 : 2;
    w -= f.kind == 0 ? 0 : f.kind == 1 ? g.q_pieces : g.q_pieces + g.k_pieces;
    const FastDiv &per = f.kind == 2 ? g.of_value : g.of_head;
    f.h = (int)per.div(w);
    f.piece = w - f.h * (int)per.d;
    const Heads &x = f.kind == 0 ? g.q : f.kind == 1 ? g.k : g.v;
    if constexpr (APPEND) {
      f.head = x.data + t * x.token + f.h * x.head;
    } else {
      const int b = (int)g.of_entry.div(t);
      f.head = x.data + b * x.batch + (t - b * (int)g.of_entry.d) * x.token + f.h * x.head;
    }
    return f;
  };
  const Rotation none{nullptr, 0, 0, 0.f, 0.f};
  auto read = [&](const From &f) __attribute__((always_inline)) {
    return read_piece<V>(f.kind == 2 ? none : g.rot, f.head, f.piece);
  };
  From f{};
  Piece<V> p;
  if (tid < units) {
    f = from(tid);
    p = read(f);
  }

  const int wid = tid >> 6;
  if (wid < n) {
    const int t = t0 + wid;
    int pos = 0, page = -1, row = 0;
    if constexpr (APPEND) {
      const int b = sequence_of(g.batch, t);
      if (b >= 0) {
        const Seq s = sequence(g.batch, b);
        pos = s.kv - s.n + t - s.q0;
        page = pos >= 0 && pos < g.batch.capacity ? page_of(g.batch, g.cache, b, pos) : -1;
        row = page >= 0 ? pos - (int)(g.cache.page.div(pos) * g.cache.page.d) : 0;
      } else {
        page = -2;  // behind the last sequence: the query is left alone too
      }
    } else {
      const int b = (int)g.of_entry.div(t);
      pos = g.positions[b * g.position_stride + (t - b * (int)g.of_entry.d)];
    }
    if ((tid & 63) == 0) {
      pos_s[wid] = pos;
      page_s[wid] = page;
      row_s[wid] = row;
    }
  }
  __syncthreads();
  for (int i = tid; i < n * g.rot.half; i += RO_THREADS) {
    const int k = i / g.rot.half;
    const double rev = (double)pos_s[k] * g.rot.turns[i - k * g.rot.half];
    float s, c;
    sincospif(2.f * (float)(rev - rint(rev)), &s, &c);
    cs[i] = make_float2(c * g.rot.magnitude, s * g.rot.sine * g.rot.magnitude);
  }
  __syncthreads();

  for (int u = tid; u < units; u += RO_THREADS) {
    const float2 *token_cs = cs + f.token * g.rot.half;
    const int t = t0 + f.token, page = page_s[f.token], row = row_s[f.token];
    if (f.kind == 0) {
      uint16_t *dst;
      if constexpr (APPEND) {
        dst = g.q_out.data + t * g.q_out.token + f.h * g.q_out.head;
      } else {
        const int b = (int)g.of_entry.div(t);
        dst = g.q_out.data + b * g.q_out.batch + (t - b * (int)g.of_entry.d) * g.q_out.token + f.h * g.q_out.head;
      }
      if (!APPEND || page != -2) write_piece<V>(g.rot, token_cs, p, dst, f.piece);
    } else if (page >= 0) {
      if (f.kind == 1)
        write_piece<V>(g.rot, token_cs, p, g.cache.k + page * g.cache.k_page + f.h * g.cache.k_head + row * g.cache.k_row, f.piece);
      else
        write_piece<V>(none, token_cs, p, g.cache.v + page * g.cache.v_page + f.h * g.cache.v_head + row * g.cache.v_row, f.piece);
    }
    if (u + RO_THREADS < units) {
      f = from(u + RO_THREADS);
      p = read(f);
    }
  }
}

// Fills in the pieces and launches; `wide`: strides and addresses allow 16-byte pieces.
template <bool APPEND>
int run_rotate(RotateArgs g, int q_heads, int kv_heads, int D, bool wide, const char *who, hipStream_t st) {
  wide = wide && D % 8 == 0 && g.rot.half % (g.rot.interleaved ? 4 : 8) == 0;
  const int per_head = wide ? pieces<8>(g.rot.half, g.rot.interleaved, D) : pieces<1>(g.rot.half, g.rot.interleaved, D);
  const int per_value = wide ? D / 8 : D;
  g.q_pieces = q_heads * per_head;
  g.k_pieces = kv_heads * per_head;
  const int total = g.q_pieces + g.k_pieces + kv_heads * per_value;
  g.of_head = FastDiv((uint32_t)per_head);
  g.of_value = FastDiv((uint32_t)per_value);
  g.of_token = FastDiv((uint32_t)total);
  g.per_group = g.tokens >= 4096 && total <= INT32_MAX / (2 * RO_TOKENS) ? RO_TOKENS : 1;
  const int64_t blocks = (g.tokens + (int64_t)g.per_group - 1) / g.per_group;
  if (blocks > MOST_BLOCKS) {
    set_error("%s: %d tokens are not supported", who, g.tokens);
    return PK_ERR_UNSUPPORTED;
  }
  const size_t lds = (size_t)g.per_group * g.rot.half * sizeof(float2);
  if (wide) rotate_kernel<8, APPEND><<<(unsigned)blocks, RO_THREADS, lds, st>>>(g);
  else rotate_kernel<1, APPEND><<<(unsigned)blocks, RO_THREADS, lds, st>>>(g);
  PK_LAUNCH_CHECK("rotate_kernel");
  return PK_OK;
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
  RotateArgs g{};
  if (int rc = check_rotary("launch_rotary", rotary, D, &g.rot)) return rc;
  PK_CHECK_ARG(tokens <= INT32_MAX && (int64_t)H * D <= INT32_MAX - 1023,
               "launch_rotary: B * S = %lld exceeds %d, or H * D = %lld is within 1023 of it", (long long)tokens, INT32_MAX,
               (long long)H * D);
  if (tokens == 0 || H == 0) return PK_OK;
  PK_CHECK_ARG(x && out && positions, "launch_rotary: null tensor pointer");
  g.q = Heads{const_cast<uint16_t *>(x), xs[0], xs[1], xs[2]};
  g.q_out = Heads{out, os[0], os[1], os[2]};
  g.positions = positions;
  g.position_stride = position_stride;
  g.of_entry = FastDiv((uint32_t)S);
  g.tokens = (int)tokens;
  const bool wide = aligned16(x) && aligned16(out) && strides8(xs[0], xs[1], xs[2]) && strides8(os[0], os[1], os[2]);
  return run_rotate<false>(g, H, 0, D, wide, "launch_rotary", (hipStream_t)stream);
}

int launch_paged_kv_append(const pk_tokens *k, const pk_tokens *v, const pk_tokens *q, const pk_tokens *q_out, int q_heads,
                           const pk_paged_cache *cache, const pk_paged_batch *batch, const pk_rotary *rotary, void *stream) {
  const char *who = "launch_paged_kv_append";
  RotateArgs g{};
  if (int rc = check_cache(who, cache, &g.cache)) return rc;
  if (int rc = check_batch(who, batch, cache, &g.batch)) return rc;
  PK_CHECK_ARG(k && v, "%s: null k or v", who);
  PK_CHECK_ARG((q != nullptr) == (q_out != nullptr) && (!q || rotary), "%s: q, q_out and rotary come together", who);
  PK_CHECK_ARG(!q || q_heads > 0, "%s: %d query heads", who, q_heads);
  PK_CHECK_ARG(!rotary || !rotary->inverse, "%s: the inverse rotation is not an append", who);
  if (rotary)
    if (int rc = check_rotary(who, rotary, cache->dim, &g.rot)) return rc;
  if (!q) q_heads = 0;
  PK_CHECK_ARG(((int64_t)q_heads + 2 * (int64_t)cache->heads) * cache->dim <= INT32_MAX - 1023, "%s: %d + 2 x %d heads of %d",
               who, q_heads, cache->heads, cache->dim);
  if (batch->tokens == 0 || batch->sequences == 0) return PK_OK;
  PK_CHECK_ARG(k->data && v->data && (!q || (q->data && q_out->data)), "%s: null tensor pointer", who);
  g.k = Heads{k->data, 0, k->token, k->head};
  g.v = Heads{v->data, 0, v->token, v->head};
  if (q) {
    g.q = Heads{q->data, 0, q->token, q->head};
    g.q_out = Heads{q_out->data, 0, q_out->token, q_out->head};
  }
  g.tokens = batch->tokens;
  bool wide = aligned16(k->data) && aligned16(v->data) && aligned16(cache->k) && aligned16(cache->v) &&
              strides8(k->token, k->head) && strides8(v->token, v->head) &&
              strides8(cache->k_page, cache->k_head, cache->k_row) && strides8(cache->v_page, cache->v_head, cache->v_row);
  if (q) wide = wide && aligned16(q->data) && aligned16(q_out->data) && strides8(q->token, q->head) && strides8(q_out->token, q_out->head);
  return run_rotate<true>(g, q_heads, cache->heads, cache->dim, wide, who, (hipStream_t)stream);
}

}  // extern "C"
