// Position rotation of rows of heads in its layouts, and the rotation on the way into a paged key-value cache:
//   y_a = x_a cos - x_b sin,  y_b = x_b cos + x_a sin  for the pairs (a, b) = (i, i + rot / 2), or (2 i, 2 i + 1), i < rot / 2,
// of each head's first rot dimensions; the others are copied. cos and sin come from tables (row = position), which
// hold any scaling of the angles. The reference rotates whole heads in halves (`_rope_np`, `_rot`:
// webtorch/llm.py:1270-1304; `rope_decode`: webtorch/_core.py:2302-2330) and writes to one contiguous cache (`kv_write`:
// webtorch/_core.py:1504-1540).
//
// A thread takes 4 pairs of a head: two 16-byte loads of fp32 (8-byte ones of fp16), both partners in one
// thread, so that nothing passes between lanes but the sum of a norm, and a tensor may be rotated in place.
//
// Bound: memory for prompts (us a replay: 7001 tokens of 32 heads of 128 fp16, half of each rotated, 116 MB in 23.0, 5.0 TB/s; four prompts of 300 to
// 1500 tokens of 28 / 4 heads into an fp32 cache 37.3, 4.5 TB/s with the zeros of the padded tokens' q), round trips for a batch's
// tokens (64 of 32 / 4 heads appended 4.7, 64 rotated at positions anywhere in 131072 5.7).
#include <math.h>

#include "kv4.h"
#include "paged.h"

namespace miq {

constexpr int kRopeThreads = 256;
// heads of a token a thread takes, where there are enough of them to fill the chip: their loads are all issued first and
// share the tables'
constexpr int kRopeHeads = 4;

// Where the two elements of pair p of a head lie. Pairs of dimensions that are not rotated are neighbours.
template <bool PAIRS> __device__ __forceinline__ void pair_at(int p, int half, int& a, int& b) {
  if (PAIRS || p >= half) {
    a = 2 * p;
    b = 2 * p + 1;
  } else {
    a = p;
    b = p + half;
  }
}

// Vectors at any address that their elements may have: this target's loads and stores take them, at some cost where they cross lines
typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));
typedef _Float16 half4u __attribute__((ext_vector_type(4), aligned(2)));
__device__ __forceinline__ void load4(const float* p, float* v) {
  const float4u t = *reinterpret_cast<const float4u*>(p);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = t[i];
}
__device__ __forceinline__ void load4(const __half* p, float* v) {
  const half4u t = *reinterpret_cast<const half4u*>(p);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = (float)t[i];
}
__device__ __forceinline__ void store4(float* p, const float* v) { *reinterpret_cast<float4u*>(p) = (float4u){v[0], v[1], v[2], v[3]}; }
__device__ __forceinline__ void store4(__half* p, const float* v) {
  *reinterpret_cast<half4u*>(p) = (half4u){(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
}

// The 4 pairs p0 .. p0 + 3 of a head: a[i], b[i]. FAST: rot and HD are multiples of 8, so that the 4 are all rotated or all
// not, and lie in two vectors.
template <typename XT, bool FAST, bool PAIRS>
__device__ __forceinline__ void load_pairs(const XT* x, int p0, int half, int HD, float* a, float* b) {
  if constexpr (FAST) {
    if (PAIRS || p0 >= half) {
      float v[8];
      load4(x + 2 * p0, v);
      load4(x + 2 * p0 + 4, v + 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        a[i] = v[2 * i];
        b[i] = v[2 * i + 1];
      }
    } else {
      load4(x + p0, a);
      load4(x + p0 + half, b);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      int ia, ib;
      pair_at<PAIRS>(p0 + i, half, ia, ib);
      const bool in = 2 * (p0 + i) < HD;
      a[i] = in ? to_f32<XT>(x[ia]) : 0.f;
      b[i] = in ? to_f32<XT>(x[ib]) : 0.f;
    }
  }
}
template <typename XT, bool FAST, bool PAIRS>
__device__ __forceinline__ void store_pairs(XT* x, int p0, int half, int HD, const float* a, const float* b) {
  if constexpr (FAST) {
    if (PAIRS || p0 >= half) {
      const float v[8] = {a[0], b[0], a[1], b[1], a[2], b[2], a[3], b[3]};
      store4(x + 2 * p0, v);
      store4(x + 2 * p0 + 4, v + 4);
    } else {
      store4(x + p0, a);
      store4(x + p0 + half, b);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      int ia, ib;
      pair_at<PAIRS>(p0 + i, half, ia, ib);
      if (2 * (p0 + i) < HD) {
        x[ia] = from_f32<XT>(a[i]);
        x[ib] = from_f32<XT>(b[i]);
      }
    }
  }
}
template <bool FAST> __device__ __forceinline__ void load_angles(const float* cos_t, const float* sin_t, size_t row, int p0, int half, float* c, float* s) {
  if constexpr (FAST) {
    if (p0 < half) {
      load4(cos_t + row * half + p0, c);
      load4(sin_t + row * half + p0, s);
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const bool in = !FAST && p0 + i < half;
    c[i] = in ? cos_t[row * half + p0 + i] : 1.f;
    s[i] = in ? sin_t[row * half + p0 + i] : 0.f;
  }
}
// The pairs p0 .. p0 + 3, those below half (the others are left as they are, infinities and NaN among them).
template <bool FAST> __device__ __forceinline__ void rotate(float* a, float* b, const float* c, const float* s, int p0, int half) {
  if (FAST && p0 >= half) return;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float x = a[i], y = b[i];
    const bool turn = FAST || p0 + i < half;
    a[i] = turn ? fmaf(x, c[i], -(y * s[i])) : x;
    b[i] = turn ? fmaf(y, c[i], x * s[i]) : y;
  }
}

// x and out [T][H] rows of HD, ld values from token to token and lh from head to head. A position outside the tables makes
// zeros.
template <typename XT, bool FAST, bool PAIRS, int U>
__global__ __launch_bounds__(kRopeThreads) void rope_kernel(const XT* x, int64_t ld, int64_t lh, const int32_t* __restrict__ positions,
                                                            const float* __restrict__ cos_t, const float* __restrict__ sin_t, int rows,
                                                            int half, float sign, XT* out, int64_t old, int64_t olh, int T, int H, int HD) {
  const uint32_t per = (HD + 7) / 8, groups = (H + U - 1) / U;  // threads of a head, groups of heads
  const uint32_t id = blockIdx.x * kRopeThreads + threadIdx.x;
  const uint32_t j = id % per, h0 = id / per % groups * U, t = id / per / groups;
  if (t >= (uint32_t)T) return;
  const int p0 = 4 * j;
  float a[U][4], b[U][4], c[4], s[4];
  const XT* xr = x + (int64_t)t * ld + (int64_t)h0 * lh;
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (h0 + u < (uint32_t)H) load_pairs<XT, FAST, PAIRS>(xr + u * lh, p0, half, HD, a[u], b[u]);
  const int pos = positions[t];
  const bool in = pos >= 0 && pos < rows;
  load_angles<FAST>(cos_t, sin_t, in ? (size_t)pos : 0, p0, half, c, s);
#pragma unroll
  for (int i = 0; i < 4; ++i) s[i] *= sign;
  XT* orow = out + (int64_t)t * old + (int64_t)h0 * olh;
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (h0 + u < (uint32_t)H) {
      rotate<FAST>(a[u], b[u], c, s, p0, half);
#pragma unroll
      for (int i = 0; i < 4; ++i) {  // no product: x may hold infinities
        a[u][i] = in ? a[u][i] : 0.f;
        b[u][i] = in ? b[u][i] : 0.f;
      }
      store_pairs<XT, FAST, PAIRS>(orow + u * olh, p0, half, HD, a[u], b[u]);
    }
}

// q|k|v rows of S x T tokens: norm and rotation of the query and key heads, queries to q_out, keys and values to the slots
// of their positions. LG consecutive lanes hold a head's HD / 8 threads (192 dimensions leave 8 of 32 without work).
template <int HD, typename XT, typename CT, bool FAST, bool PAIRS, int U>
__global__ __launch_bounds__(kRopeThreads) void paged_append_kernel(
    const XT* __restrict__ qkv, int64_t ld, const float* __restrict__ qn, const float* __restrict__ kn, float eps,
    const int32_t* __restrict__ positions, const int32_t* __restrict__ pages, int max_pages, const float* __restrict__ cos_t,
    const float* __restrict__ sin_t, int rows, int half, XT* __restrict__ q_out, CT* __restrict__ cache, int num_pages, int pshift,
    int S, int T, int NH, int NKV) {
  constexpr int LG = HD == 64 ? 8 : HD == 128 ? 16 : 32;
  const uint32_t heads = NH + 2 * NKV, groups = (heads + U - 1) / U;
  const uint32_t id = blockIdx.x * kRopeThreads + threadIdx.x;
  const uint32_t j = id % LG, unit = id / LG, h0 = unit % groups * U, tok = unit / groups;
  if (tok >= (uint32_t)S * (uint32_t)T) return;  // whole heads
  const bool mine = HD != 192 || j < HD / 8;
  const int p0 = mine ? 4 * j : 0;
  float a[U][4], b[U][4], c[4], s[4], w[2][8];
  const XT* xr = qkv + (int64_t)tok * ld + (int64_t)h0 * HD;
  // Many tokens: those of a padded batch without a position are not read (four prompts of 300 to 1500 tokens padded to 1500, 41.5 ->
  // 37.3 us); few: the rows are on the way while the position is.
  int pos = 0;
  if constexpr (U > 1) pos = positions[tok];
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (h0 + u < heads && pos >= 0) {
      if (h0 + u < (uint32_t)(NH + NKV))
        load_pairs<XT, FAST, PAIRS>(xr + u * HD, p0, half, HD, a[u], b[u]);
      else  // values: neighbours
        load_pairs<XT, FAST, true>(xr + u * HD, p0, half, HD, a[u], b[u]);
    }
  if constexpr (U == 1) pos = positions[tok];
  bool in = pos >= 0 && (half == 0 || pos < rows) && (pos >> pshift) < max_pages;
  const int page = in ? pages[(int64_t)(tok / (uint32_t)T) * max_pages + (pos >> pshift)] : -1;
  load_angles<FAST>(cos_t, sin_t, in ? (size_t)pos : 0, p0, half, c, s);
  const bool norms = qn || kn;
  if (norms) {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const float* wp = x ? kn : qn;
      if (wp) load_pairs<float, false, PAIRS>(wp, p0, half, HD, w[x], w[x] + 4);
    }
  }
  in = in && (uint32_t)page < (uint32_t)num_pages;
  const int P = 1 << pshift;
  CT* slot = cache + ((int64_t)(in ? page : 0) * 2 * NKV * P + (pos & (P - 1))) * HD;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t h = h0 + u;
    if (h >= heads) break;
    if (h >= (uint32_t)(NH + NKV)) {
      if (in && mine) store_pairs<CT, FAST, true>(slot + (int64_t)(NKV + h - NH - NKV) * P * HD, p0, half, HD, a[u], b[u]);
      continue;
    }
    const bool query = h < (uint32_t)NH;
    if (query ? qn != nullptr : kn != nullptr) {
      float q = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) q = fmaf(a[u][i], a[u][i], fmaf(b[u][i], b[u][i], q));
      if (!mine) q = 0.f;
#pragma unroll
      for (int d = 1; d < LG; d *= 2) q += __shfl_xor(q, d);
      const float r = 1.f / sqrtf(q / (float)HD + eps);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        a[u][i] = a[u][i] * r * (query ? w[0][i] : w[1][i]);
        b[u][i] = b[u][i] * r * (query ? w[0][4 + i] : w[1][4 + i]);
      }
    }
    rotate<FAST>(a[u], b[u], c, s, p0, half);
    if (!mine) continue;
    if (query) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        a[u][i] = in ? a[u][i] : 0.f;
        b[u][i] = in ? b[u][i] : 0.f;
      }
      store_pairs<XT, FAST, PAIRS>(q_out + ((int64_t)tok * NH + h) * HD, p0, half, HD, a[u], b[u]);
    } else if (in) {
      store_pairs<CT, FAST, PAIRS>(slot + (int64_t)(h - NH) * P * HD, p0, half, HD, a[u], b[u]);
    }
  }
}

}  // namespace miq

using namespace miq;

static bool rope_many(int64_t tokens, int heads) { return tokens * heads >= 8192; }

extern "C" int miq_rope(const void* x, int x_dtype, int64_t ld, int64_t lh, const int32_t* positions, const float* cos_tab,
                        const float* sin_tab, int rows, int rot, int pairs, int transpose, void* out, int64_t out_ld, int64_t out_lh,
                        int T, int H, int HD, void* stream) {
  MIQ_REQUIRE(T >= 0 && H >= 0 && H <= (1 << 16) && HD > 0 && HD % 2 == 0 && HD <= 1024 && rot > 0 && rot % 2 == 0 && rot <= HD && rows > 0,
              MIQ_ERR_INVALID, "rope: T=%d H=%d HD=%d rot=%d rows=%d", T, H, HD, rot, rows);
  MIQ_REQUIRE(x_dtype == MIQ_F32 || x_dtype == MIQ_F16, MIQ_ERR_UNSUPPORTED, "rope: x dtype %d", x_dtype);
  if (T == 0 || H == 0) return MIQ_OK;
  MIQ_REQUIRE(x && positions && cos_tab && sin_tab && out, MIQ_ERR_INVALID, "rope: null pointer");
  const size_t size = x_dtype == MIQ_F32 ? 4 : 2;
  int64_t span[2];
  for (int i = 0; i < 2; ++i) {
    const __int128 a = T == 1 ? 0 : i ? out_ld : ld, b = H == 1 ? 0 : i ? out_lh : lh;
    // rows apart: heads within a token, or tokens within a head
    const bool apart = (H == 1 || b >= HD) && (T == 1 || (a >= HD && (H == 1 || a >= (H - 1) * b + HD || b >= (T - 1) * a + HD)));
    const __int128 n = ((T - 1) * a + (H - 1) * b + HD) * size;
    MIQ_REQUIRE(apart && n < (__int128)1 << 48, MIQ_ERR_INVALID, "rope: rows %lld and heads %lld apart overlap (T=%d H=%d HD=%d)",
                (long long)a, (long long)b, T, H, HD);
    span[i] = (int64_t)n;
  }
  const int64_t nx = span[0], no = span[1];
  const bool same = out == x && (T == 1 || out_ld == ld) && (H == 1 || out_lh == lh);
  MIQ_REQUIRE(same || !share_bytes(out, (size_t)no, x, (size_t)nx), MIQ_ERR_INVALID, "rope: out must be x itself or lie apart from it");
  const size_t table = (size_t)rows * (rot / 2) * 4;
  MIQ_REQUIRE(!share_bytes(out, (size_t)no, positions, (size_t)T * 4) && !share_bytes(out, (size_t)no, cos_tab, table) &&
                  !share_bytes(out, (size_t)no, sin_tab, table),
              MIQ_ERR_INVALID, "rope: out must lie apart from the positions and the tables");
  const int U = rope_many(T, H) ? kRopeHeads : 1;
  const int64_t threads = (int64_t)T * ((H + U - 1) / U) * ((HD + 7) / 8);
  MIQ_REQUIRE(threads < (1ll << 32) - kRopeThreads, MIQ_ERR_UNSUPPORTED, "rope: T=%d is past the grid", T);
  const bool fast = rot % 8 == 0 && HD % 8 == 0;
  const dim3 grid((unsigned)((threads + kRopeThreads - 1) / kRopeThreads)), block(kRopeThreads);
  const hipStream_t st = static_cast<hipStream_t>(stream);
#define MIQ_RP(XT, FV, PV, UV)                                                                                                     \
  hipLaunchKernelGGL((rope_kernel<XT, FV, PV, UV>), grid, block, 0, st, static_cast<const XT*>(x), ld, lh, positions, cos_tab, sin_tab, \
                     rows, rot / 2, transpose ? -1.f : 1.f, static_cast<XT*>(out), out_ld, out_lh, T, H, HD)
#define MIQ_RP_U(XT, FV, PV) \
  if (U == 1) { MIQ_RP(XT, FV, PV, 1); } else { MIQ_RP(XT, FV, PV, kRopeHeads); }
#define MIQ_RP_P(XT, FV) \
  if (pairs) { MIQ_RP_U(XT, FV, true) } else { MIQ_RP_U(XT, FV, false) }
#define MIQ_RP_F(XT) \
  if (fast) { MIQ_RP_P(XT, true) } else { MIQ_RP_P(XT, false) }
  if (x_dtype == MIQ_F32) { MIQ_RP_F(float) } else { MIQ_RP_F(__half) }
#undef MIQ_RP_F
#undef MIQ_RP_P
#undef MIQ_RP_U
#undef MIQ_RP
  return check_launch("rope");
}

extern "C" int miq_paged_append(const void* qkv, int x_dtype, int64_t ld, const float* qn, const float* kn, float eps,
                                const int32_t* positions, const int32_t* pages, int max_pages, const float* cos_tab,
                                const float* sin_tab, int rows, int rot, int pairs, void* q_out, void* cache, int cache_dtype,
                                int num_pages, int page, int S, int T, int NH, int NKV, int HD, void* stream) {
  MIQ_REQUIRE(S >= 0 && T >= 0 && NH >= 0 && NH <= (1 << 16) && NKV > 0 && NKV <= (1 << 16) && HD > 0 && num_pages > 0 && max_pages >= 0 &&
                  rot >= 0 && rot % 2 == 0 && rot <= HD && (rot == 0 || rows > 0),
              MIQ_ERR_INVALID, "paged_append: S=%d T=%d NH=%d NKV=%d HD=%d pages=%d of %d rot=%d rows=%d", S, T, NH, NKV, HD, max_pages, num_pages,
              rot, rows);
  MIQ_REQUIRE((x_dtype == MIQ_F32 || x_dtype == MIQ_F16) && (cache_dtype == MIQ_F32 || cache_dtype == MIQ_F16), MIQ_ERR_UNSUPPORTED,
              "paged_append: dtypes %d, %d", x_dtype, cache_dtype);
  if (int rc = check_paged("paged_append", HD, page, num_pages, max_pages)) return rc;
  const int64_t W = (int64_t)(NH + 2 * NKV) * HD, tokens = (int64_t)S * T;
  MIQ_REQUIRE(ld >= W, MIQ_ERR_INVALID, "paged_append: rows %lld apart hold %lld values", (long long)ld, (long long)W);
  if (tokens == 0) return MIQ_OK;
  MIQ_REQUIRE(qkv && positions && (pages || max_pages == 0) && (rot == 0 || (cos_tab && sin_tab)) && (NH == 0 || q_out) && cache, MIQ_ERR_INVALID,
              "paged_append: null pointer");
  MIQ_REQUIRE(aligned(cache, 16), MIQ_ERR_ALIGN, "paged_append: the cache must be 16-byte aligned");
  const int heads = NH + 2 * NKV, U = rope_many(tokens, heads) ? kRopeHeads : 1, lg = HD == 64 ? 8 : HD == 128 ? 16 : 32;
  const int64_t threads = tokens * ((heads + U - 1) / U) * lg;
  MIQ_REQUIRE(tokens < (1ll << 31) && threads < (1ll << 32) - kRopeThreads, MIQ_ERR_UNSUPPORTED, "paged_append: S=%d T=%d is past the grid", S, T);
  const size_t size = x_dtype == MIQ_F32 ? 4 : 2, csize = cache_dtype == MIQ_F32 ? 4 : 2;
  const size_t nx = (size_t)((tokens - 1) * ld + W) * size, nq = (size_t)tokens * NH * HD * size, nc = (size_t)num_pages * 2 * NKV * page * HD * csize;
  MIQ_REQUIRE((!nq || !share_bytes(q_out, nq, qkv, nx)) && !share_bytes(cache, nc, qkv, nx) && (!nq || !share_bytes(cache, nc, q_out, nq)),
              MIQ_ERR_INVALID, "paged_append: qkv, q_out and the cache must lie apart");
  const bool fast = rot % 8 == 0;
  const dim3 grid((unsigned)((threads + kRopeThreads - 1) / kRopeThreads)), block(kRopeThreads);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const int pshift = __builtin_ctz((unsigned)page);
#define MIQ_PA(HDV, XT, CT, FV, PV, UV)                                                                                            \
  hipLaunchKernelGGL((paged_append_kernel<HDV, XT, CT, FV, PV, UV>), grid, block, 0, st, static_cast<const XT*>(qkv), ld, qn, kn, eps, positions, \
                     pages, max_pages, cos_tab, sin_tab, rows, rot / 2, static_cast<XT*>(q_out), static_cast<CT*>(cache), num_pages, pshift, S, T, \
                     NH, NKV)
#define MIQ_PA_U(HDV, XT, CT, FV, PV) \
  if (U == 1) { MIQ_PA(HDV, XT, CT, FV, PV, 1); } else { MIQ_PA(HDV, XT, CT, FV, PV, kRopeHeads); }
#define MIQ_PA_P(HDV, XT, CT, FV) \
  if (pairs) { MIQ_PA_U(HDV, XT, CT, FV, true) } else { MIQ_PA_U(HDV, XT, CT, FV, false) }
#define MIQ_PA_F(HDV, XT, CT) \
  if (fast) { MIQ_PA_P(HDV, XT, CT, true) } else { MIQ_PA_P(HDV, XT, CT, false) }
#define MIQ_PA_C(HDV, XT) \
  if (cache_dtype == MIQ_F32) { MIQ_PA_F(HDV, XT, float) } else { MIQ_PA_F(HDV, XT, __half) }
#define MIQ_PA_X(HDV) \
  if (x_dtype == MIQ_F32) { MIQ_PA_C(HDV, float) } else { MIQ_PA_C(HDV, __half) }
  switch (HD) {
    case 64: MIQ_PA_X(64) break;
    case 128: MIQ_PA_X(128) break;
    case 192: MIQ_PA_X(192) break;
    default: MIQ_PA_X(256)
  }
#undef MIQ_PA_X
#undef MIQ_PA_C
#undef MIQ_PA_F
#undef MIQ_PA_P
#undef MIQ_PA_U
#undef MIQ_PA
  return check_launch("paged_append");
}
