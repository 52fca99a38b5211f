// QK-norm, RoPE and the cache write in one pass over the fused q|k|v rows (`CausalLM._qkv`,
// `_rope_np` and `kv_write` of the reference: webtorch/llm.py:1498-1519, 1270-1304;
// webtorch/_core.py:1504-1540): q_h = rope(x_h / sqrt(mean(x_h^2) + eps) * qn), k likewise, v as it is, k and
// v into an fp32 cache or into the 4-bit one (kv4.h).
//
// A wave takes heads of one token, lane l the dimensions l, l + 64, ..: the mean is a wave sum, a
// group of 32 dimensions is half a wave, and a dimension's rotation partner is another register of the lane
// (HD 128, 256), the lane 32 further (HD 64), or read through LDS. Bound: memory for prompts (4001 tokens into the fp32
// cache: 150 MB in 29.8 us, 5.0 TB/s), the launch and two round trips for a token (2.5 us a replay).
#include <math.h>

#include "kv4.h"

#pragma clang fp contract(off)

namespace miq {

constexpr int kNrWaves = 4;
// One head a wave while that fills the chip's 1024 SIMDs no more than a few times (a token's latency counts), then
// several, whose loads are all issued first and share the rotation's: 4001 tokens of 36 heads of 128 without a norm,
// fp32 cache, 54 us at one head, 30.4 at 2, 29.8 at 4, 30.2 at 8; 700 tokens with norms, 4-bit cache, 19.0 at 4
// heads of q and k, 16.9 at 4 of q or one of k, 16.1 at 2 of q or one of k (each with the 4.5 us of reading back).
constexpr int kNrHeads = 4, kNrHeads4 = 2;
static bool several_heads(int T, int heads) { return (int64_t)T * heads >= 8192; }

template <int CTRL> __device__ __forceinline__ double dpp_d(double v) {
  const int lo = __builtin_amdgcn_update_dpp(0, __double2loint(v), CTRL, 0xF, 0xF, false);
  const int hi = __builtin_amdgcn_update_dpp(0, __double2hiint(v), CTRL, 0xF, 0xF, false);
  return __hiloint2double(hi, lo);
}
__device__ __forceinline__ double lane_at_d(double v, int l) {
  return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(v), l), __builtin_amdgcn_readlane(__double2loint(v), l));
}
__device__ __forceinline__ double other_half(double v) {  // lane l: the value of lane l ^ 32
  return __hiloint2double(__shfl_xor(__double2hiint(v), 32), __shfl_xor(__double2loint(v), 32));
}
__device__ __forceinline__ double wave_sum_d(double v) {
  v += dpp_d<0xB1>(v);
  v += dpp_d<0x4E>(v);
  v += dpp_d<0x141>(v);
  v += dpp_d<0x140>(v);
  return (lane_at_d(v, 0) + lane_at_d(v, 16)) + (lane_at_d(v, 32) + lane_at_d(v, 48));
}

// An fp64 number rounded once to a query's type. fp16: by way of the fp32 number next to it towards zero with its last bit
// set where something is left ("to odd"), so that it is on the same side of every border of fp16 as v is.
template <typename T> __device__ __forceinline__ T from_f64(double v);
template <> __device__ __forceinline__ float from_f64<float>(double v) { return (float)v; }
template <> __device__ __forceinline__ __half from_f64<__half>(double v) {
  const float f = (float)v;
  uint32_t b = __float_as_uint(f) - (fabs((double)f) > fabs(v) ? 1u : 0u);
  if ((double)f != v) b |= 1u;
  return __float2half_rn(__uint_as_float(b));
}

// The rotation partners, HD / 2 dimensions further, of v[i] = dimension lane + 64 i.
template <int HD> __device__ __forceinline__ void partners(const float* v, float* o) {
  if constexpr (HD == 128) {
    o[0] = v[1];
    o[1] = v[0];
  } else if constexpr (HD == 256) {
    o[0] = v[2];
    o[1] = v[3];
    o[2] = v[0];
    o[3] = v[1];
  } else if constexpr (HD == 64) {
    o[0] = __shfl_xor(v[0], 32);
  }
}

// The fp32 cache: every product, quotient and sum rounded where miq_head_rmsnorm and miq_rope_kv
// round theirs, in their order, so that the results are theirs bit for bit. A wave takes U heads of one token,
// all loads first; HDT is the head dimension where a lane's partner is in registers, 0 for any (through LDS).
template <int HDT, int U>
__global__ __launch_bounds__(64 * kNrWaves) void norm_rope_kv_kernel(
    const float* __restrict__ qkv, size_t ld, const float* __restrict__ qn, const float* __restrict__ kn, float eps,
    const int32_t* __restrict__ state, const float* __restrict__ cos_t, const float* __restrict__ sin_t,
    float* __restrict__ q_out, float* __restrict__ kc, float* __restrict__ vc, int T, int NH, int NKV, int HDR, int LMAX) {
  constexpr int N = HDT ? HDT / 64 : 4;
  const int HD = HDT ? HDT : HDR;
  __shared__ float rows[HDT ? 1 : kNrWaves][256];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int heads = NH + 2 * NKV, half = HD / 2, groups = (heads + U - 1) / U;
  const int64_t unit = (int64_t)blockIdx.x * kNrWaves + wave;
  const int t = (int)(unit / groups), h0 = (int)(unit % groups) * U;
  if (t >= T) return;  // whole waves
  const float* row = qkv + (size_t)t * ld;
  float v[U][N], w[2][N], c[N], s[N];
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int i = 0; i < N; ++i)
      v[u][i] = h0 + u < heads && (HDT || lane + 64 * i < HD) ? row[(h0 + u) * HD + lane + 64 * i] : 0.f;
  const int64_t pos = (int64_t)state[0] + t;
  const bool in = pos >= 0 && pos < LMAX;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int d = lane + 64 * i, j = d < half ? d : d - half;
    const bool has = HDT || d < HD;
    w[0][i] = qn && has ? qn[d] : 0.f;
    w[1][i] = kn && has ? kn[d] : 0.f;
    c[i] = in && has ? cos_t[(size_t)pos * half + j] : 0.f;
    s[i] = in && has ? sin_t[(size_t)pos * half + j] : 0.f;
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int h = h0 + u;
    if (h >= heads) break;
    if (h >= NH + NKV) {
      if (in)
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (HDT || lane + 64 * i < HD) vc[((size_t)(h - NH - NKV) * LMAX + pos) * HD + lane + 64 * i] = v[u][i];
      continue;
    }
    if (h < NH ? qn != nullptr : kn != nullptr) {
      float q = 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i) q = q + v[u][i] * v[u][i];
      q = wave_sum(q);
      const float r = sqrtf(q / (float)HD + eps);
#pragma unroll
      for (int i = 0; i < N; ++i) v[u][i] = (v[u][i] / r) * (h < NH ? w[0][i] : w[1][i]);
    }
    float o[N];
    if constexpr (HDT) {
      partners<HDT>(v[u], o);
    } else {
      float* mine = rows[wave];
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
      for (int i = 0; i < N; ++i) mine[lane + 64 * i] = v[u][i];
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int d = lane + 64 * i;
        o[i] = d < HD ? mine[d < half ? d + half : d - half] : 0.f;
      }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int d = lane + 64 * i;
      if (!HDT && d >= HD) break;
      float y = 0.f;  // a position outside the cache: no key, and zeros for its queries
      if (in) y = v[u][i] * c[i] + (d < half ? -o[i] : o[i]) * s[i];
      if (h < NH) q_out[((size_t)t * NH + h) * HD + d] = y;
      else if (in) kc[((size_t)(h - NH) * LMAX + pos) * HD + d] = y;
    }
  }
}

// The 4-bit cache. A key's codes depend on which side of a border its value is, so q and k are computed
// in fp64 (the vector units' fp64 rate is that of fp32) and rounded once. The first waves take 64
// dimensions of the values of the 8 positions that share words (kv4_key; a word that is not wholly new is read
// first), the others U heads of q, or one of k, of one token.
template <int HD, typename XT, int U>
__global__ __launch_bounds__(64 * kNrWaves) void norm_rope_kv4_kernel(
    const XT* __restrict__ qkv, size_t ld, const float* __restrict__ qn, const float* __restrict__ kn, float eps,
    const int32_t* __restrict__ state, const float* __restrict__ cos_t, const float* __restrict__ sin_t,
    XT* __restrict__ q_out, uint8_t* __restrict__ cache, int T, int NH, int NKV, int LMAX, int vblocks) {
  constexpr int N = HD / 64, NG = HD / 32, HALF = HD / 2;
  const int lane = threadIdx.x & 63;
  const int nv = vblocks * NKV * 4 * N, wave = uniform(threadIdx.x >> 6);
  const int64_t unit = (int64_t)blockIdx.x * kNrWaves + wave - nv;
  const int qgroups = (NH + U - 1) / U, groups = qgroups + NKV;
  const int NB = kv4_blocks(LMAX);
  if (unit >= 0) {
    if (unit >= (int64_t)T * groups) return;
    const int t = (int)(unit / groups), group = (int)(unit % groups);
    const int h0 = group < qgroups ? group * U : NH + group - qgroups, end = group < qgroups ? min(NH, h0 + U) : h0 + 1;
    const XT* row = qkv + (size_t)t * ld;
    XT x[U][N];
    float w[2][N], cs[N], sn[N];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < N; ++i) x[u][i] = h0 + u < end ? row[(h0 + u) * HD + lane + 64 * i] : from_f32<XT>(0.f);
    const int64_t pos = (int64_t)state[0] + t;
    const bool in = pos >= 0 && pos < LMAX;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int d = lane + 64 * i, j = d < HALF ? d : d - HALF;
      w[0][i] = qn ? qn[d] : 0.f;
      w[1][i] = kn ? kn[d] : 0.f;
      cs[i] = in ? cos_t[(size_t)pos * HALF + j] : 0.f;
      sn[i] = in ? sin_t[(size_t)pos * HALF + j] : 0.f;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = h0 + u;
      if (h >= end) break;
      if (!in) {  // a position outside the cache: no key, and zeros for its queries
        if (h < NH)
#pragma unroll
          for (int i = 0; i < N; ++i) q_out[((size_t)t * NH + h) * HD + lane + 64 * i] = from_f32<XT>(0.f);
        continue;
      }
      double v[N];
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = (double)to_f32<XT>(x[u][i]);
      if (h < NH ? qn != nullptr : kn != nullptr) {
        double s = 0.0;
#pragma unroll
        for (int i = 0; i < N; ++i) s = fma(v[i], v[i], s);
        const double inv = rsqrt(wave_sum_d(s) * (1.0 / HD) + (double)eps);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = v[i] * inv * (double)(h < NH ? w[0][i] : w[1][i]);
      }
      double y[N];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        double o;  // the rotation partner
        if constexpr (HD % 128 == 0) o = v[(i + N / 2) % N];
        else if constexpr (HD == 64) o = other_half(v[0]);
        else {  // 192: 96 dimensions further, in lane ^ 32 of the register after next or of the next one
          double got[3];
#pragma unroll
          for (int r = 0; r < 3; ++r) got[r] = other_half(v[r]);
          const int k = (i + (lane < 32 ? 1 : 2)) % 3;
          o = k == 0 ? got[0] : k == 1 ? got[1] : got[2];
        }
        const double os = lane + 64 * i < HALF ? -o : o;
        y[i] = fma(os, (double)sn[i], v[i] * (double)cs[i]);
      }
      if (h < NH) {
#pragma unroll
        for (int i = 0; i < N; ++i) q_out[((size_t)t * NH + h) * HD + lane + 64 * i] = from_f64<XT>(y[i]);
        continue;
      }
      const int key = (int)(pos % kKv4Block);
      uint8_t* rec = cache + ((size_t)(h - NH) * NB + (size_t)(pos / kKv4Block)) * kv4_record(HD);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        uint16_t S, Z;
        uint32_t c = kv4_quantize((float)y[i], S, Z) << kv4_shift(lane & 7);
        c |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)c, 0xB1, 0xF, 0xF, false);
        c |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)c, 0x4E, 0xF, 0xF, false);
        c |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)c, 0x141, 0xF, 0xF, false);
        const int grp = 2 * i + (lane >> 5);
        if ((lane & 7) == 0)
          *reinterpret_cast<uint32_t*>(rec + kv4_word((key >> 4) * NG + grp, (lane & 31) >> 3, key & 15)) = c;
        if ((lane & 31) == 0)
          *reinterpret_cast<uint32_t*>(rec + kv4_kmeta(HD) + (key * NG + grp) * 4) = S | ((uint32_t)Z << 16);
      }
    }
    return;
  }
  const int vu = blockIdx.x * kNrWaves + wave, i = vu % N, g = vu / N & 3, kv = vu / (4 * N) % NKV;
  const int64_t pos0 = state[0], first = pos0 > 0 ? pos0 : 0, blk = first / kKv4Block + vu / (4 * N * NKV);
  if (blk >= NB) return;
  const int d = lane + 64 * i, grp = 2 * i + (lane >> 5);
  uint32_t live = 0;
  float x[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int64_t pos = blk * kKv4Block + kv4_key(g, e), t = pos - pos0;
    const bool in = t >= 0 && t < T && pos < LMAX;
    live |= (in ? 15u : 0u) << kv4_shift(e);
    x[e] = in ? to_f32<XT>(qkv[(size_t)t * ld + (size_t)(NH + NKV + kv) * HD + d]) : 0.f;
  }
  if (!live) return;
  uint8_t* rec = cache + ((size_t)kv * NB + (size_t)blk) * kv4_record(HD);
  uint32_t* word = reinterpret_cast<uint32_t*>(rec + kv4_vcodes(HD) + kv4_word(d >> 4, g, d & 15));
  uint16_t* meta = reinterpret_cast<uint16_t*>(rec + kv4_vmeta(HD)) + (grp * 4 + g) * 16;
  uint32_t c = live == 0xFFFFFFFFu ? 0u : *word & ~live;
  uint16_t S[8], Z[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) c |= (kv4_quantize(x[e], S[e], Z[e]) << kv4_shift(e)) & live;
  *word = c;
  if ((lane & 31) == 0)
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if ((live >> kv4_shift(e)) & 1) {
        meta[e] = S[e];
        meta[8 + e] = Z[e];
      }
}

// fp32 rows of the positions [start, start + n): a thread takes one word, of a key 8 dimensions, of the
// values one dimension of 8 positions
__global__ __launch_bounds__(256) void kv4_dequant_kernel(const uint8_t* __restrict__ cache, float* __restrict__ k_out,
                                                          float* __restrict__ v_out, int HD, int NB, int start, int n) {
  const int NT = HD / 16, NG = HD / 32;
  const int x = blockIdx.y * 256 + threadIdx.x;  // word of a block: [n][g][i]
  const int kv = blockIdx.z, blk = start / kKv4Block + blockIdx.x;
  if (x >= NT * 64) return;
  const uint8_t* rec = cache + ((size_t)kv * NB + blk) * kv4_record(HD);
  const int i = x & 15, g = (x >> 4) & 3, wn = x >> 6;
  {
    const int key = 16 * (wn / NG) + i, j = wn % NG, row = blk * kKv4Block + key - start;
    if (k_out && row >= 0 && row < n) {
      const uint32_t w = *reinterpret_cast<const uint32_t*>(rec + kv4_word(wn, g, i));
      const uint32_t m = *reinterpret_cast<const uint32_t*>(rec + kv4_kmeta(HD) + (key * NG + j) * 4);
      const __half S = __ushort_as_half((uint16_t)(m & 0xFFFF)), Z = __ushort_as_half((uint16_t)(m >> 16));
      float* o = k_out + ((size_t)kv * n + row) * HD + 32 * j + 8 * g;
      for (int e = 0; e < 8; ++e)
        o[e] = __half2float(__hfma(S, __ushort_as_half((uint16_t)(0x3C00 | (((w >> kv4_shift(e)) & 15) << 6))), Z));
    }
  }
  if (!v_out) return;
  const uint32_t w = *reinterpret_cast<const uint32_t*>(rec + kv4_vcodes(HD) + kv4_word(wn, g, i));
  const uint16_t* meta = reinterpret_cast<const uint16_t*>(rec + kv4_vmeta(HD)) + ((wn >> 1) * 4 + g) * 16;
  for (int e = 0; e < 8; ++e) {
    const int row = blk * kKv4Block + kv4_key(g, e) - start;
    if (row >= 0 && row < n)
      v_out[((size_t)kv * n + row) * HD + 16 * wn + i] =
          __half2float(__hfma(__ushort_as_half(meta[e]), __ushort_as_half((uint16_t)(0x3C00 | (((w >> kv4_shift(e)) & 15) << 6))),
                              __ushort_as_half(meta[8 + e])));
  }
}

}  // namespace miq

using namespace miq;

extern "C" int miq_kv4_cache_bytes(int NKV, int LMAX, int HD, size_t* bytes) {
  MIQ_REQUIRE(bytes && NKV > 0 && LMAX > 0 && LMAX <= (1 << 30) && HD > 0, MIQ_ERR_INVALID, "kv4_cache_bytes: NKV=%d LMAX=%d HD=%d", NKV,
              LMAX, HD);
  MIQ_REQUIRE(kv4_head(HD), MIQ_ERR_UNSUPPORTED, "kv4_cache_bytes: HD=%d (64, 128, 192 or 256)", HD);
  *bytes = (size_t)NKV * kv4_blocks(LMAX) * kv4_record(HD);
  return MIQ_OK;
}

// a launch has fewer than 2^32 threads
static bool grid_holds(int64_t units) { return units <= (int64_t)kNrWaves * ((1 << 24) - 1); }

static int check_norm_rope(const char* what, const void* qkv, int64_t ld, const int32_t* state, const float* cos_tab,
                           const float* sin_tab, const void* q_out, int T, int NH, int NKV, int HD, int LMAX) {
  MIQ_REQUIRE(T >= 0 && NH > 0 && NKV > 0 && NH % NKV == 0 && NH <= (1 << 16) && HD > 0 && HD % 2 == 0 && HD <= 256 && LMAX > 0 &&
                  LMAX <= (1 << 30),
              MIQ_ERR_INVALID, "%s: T=%d NH=%d NKV=%d HD=%d LMAX=%d", what, T, NH, NKV, HD, LMAX);
  MIQ_REQUIRE(ld >= (int64_t)(NH + 2 * NKV) * HD, MIQ_ERR_INVALID, "%s: rows %lld apart hold %lld values", what, (long long)ld,
              (long long)(NH + 2 * NKV) * HD);
  MIQ_REQUIRE(T == 0 || (qkv && state && cos_tab && sin_tab && q_out), MIQ_ERR_INVALID, "%s: null pointer", what);
  return MIQ_OK;
}

// Whether a range of n bytes at o meets any of T rows of w bytes that lie ld bytes apart from x on.
static bool meets_rows(const void* o, size_t n, const void* x, int T, size_t w, size_t ld) {
  if (!share_bytes(o, n, x, (size_t)(T - 1) * ld + w)) return false;
  const uintptr_t a = reinterpret_cast<uintptr_t>(o), b = reinterpret_cast<uintptr_t>(x);
  return a < b || (a - b) % ld < w || (a - b) % ld + n > ld;  // behind a row: the range reaches the next one
}
// What a wave writes must not be what another still reads: the caches (two of fp32, or one and null) and q_out
// lie apart from each other and from the rows.
static int check_apart(const char* what, const void* qkv, size_t size, int64_t ld, const void* q_out, const void* c0, const void* c1,
                       size_t cache_bytes, int T, int NH, int NKV, int HD) {
  const size_t w = (size_t)(NH + 2 * NKV) * HD * size, q = (size_t)T * NH * HD * size;
  MIQ_REQUIRE(!c1 || !share_bytes(c0, cache_bytes, c1, cache_bytes), MIQ_ERR_INVALID, "%s: the caches overlap", what);
  MIQ_REQUIRE(!meets_rows(q_out, q, qkv, T, w, (size_t)ld * size), MIQ_ERR_INVALID, "%s: q_out must lie apart from qkv", what);
  for (const void* c : {c0, c1})
    MIQ_REQUIRE(!c || (!share_bytes(c, cache_bytes, q_out, q) && !meets_rows(c, cache_bytes, qkv, T, w, (size_t)ld * size)), MIQ_ERR_INVALID,
                "%s: the cache must lie apart from qkv and q_out", what);
  return MIQ_OK;
}

extern "C" int miq_qk_norm_rope_kv(const float* qkv, int64_t ld, const float* qn, const float* kn, float eps,
                                   const int32_t* state, const float* cos_tab, const float* sin_tab, float* q_out,
                                   float* kcache, float* vcache, int T, int NH, int NKV, int HD, int LMAX, void* stream) {
  if (int rc = check_norm_rope("qk_norm_rope_kv", qkv, ld, state, cos_tab, sin_tab, q_out, T, NH, NKV, HD, LMAX)) return rc;
  if (T == 0) return MIQ_OK;
  MIQ_REQUIRE(kcache && vcache, MIQ_ERR_INVALID, "qk_norm_rope_kv: null pointer");
  const int heads = NH + 2 * NKV, U = several_heads(T, heads) ? kNrHeads : 1;
  const int64_t units = (int64_t)T * ((heads + U - 1) / U);
  MIQ_REQUIRE(grid_holds(units), MIQ_ERR_UNSUPPORTED, "qk_norm_rope_kv: T=%d is past the grid", T);
  if (int rc = check_apart("qk_norm_rope_kv", qkv, 4, ld, q_out, kcache, vcache, (size_t)NKV * LMAX * HD * 4, T, NH, NKV, HD)) return rc;
  const dim3 grid((unsigned)((units + kNrWaves - 1) / kNrWaves)), block(64 * kNrWaves);
  const hipStream_t st = static_cast<hipStream_t>(stream);
#define MIQ_NR(HDV, UV)                                                                                                     \
  hipLaunchKernelGGL((norm_rope_kv_kernel<HDV, UV>), grid, block, 0, st, qkv, (size_t)ld, qn, kn, eps, state, cos_tab, sin_tab, q_out, \
                     kcache, vcache, T, NH, NKV, HD, LMAX)
#define MIQ_NR_HD(UV)                     \
  switch (HD) {                           \
    case 64: MIQ_NR(64, UV); break;       \
    case 128: MIQ_NR(128, UV); break;     \
    case 256: MIQ_NR(256, UV); break;     \
    default: MIQ_NR(0, UV);               \
  }
  if (U == 1) { MIQ_NR_HD(1) } else { MIQ_NR_HD(kNrHeads) }
#undef MIQ_NR_HD
#undef MIQ_NR
  return check_launch("qk_norm_rope_kv");
}

extern "C" int miq_qk_norm_rope_kv4(const void* qkv, int x_dtype, int64_t ld, const float* qn, const float* kn, float eps,
                                    const int32_t* state, const float* cos_tab, const float* sin_tab, void* q_out,
                                    void* cache, int T, int NH, int NKV, int HD, int LMAX, void* stream) {
  if (int rc = check_norm_rope("qk_norm_rope_kv4", qkv, ld, state, cos_tab, sin_tab, q_out, T, NH, NKV, HD, LMAX)) return rc;
  MIQ_REQUIRE(x_dtype == MIQ_F32 || x_dtype == MIQ_F16, MIQ_ERR_UNSUPPORTED, "qk_norm_rope_kv4: x dtype %d", x_dtype);
  MIQ_REQUIRE(kv4_head(HD), MIQ_ERR_UNSUPPORTED, "qk_norm_rope_kv4: HD=%d (64, 128, 192 or 256)", HD);
  if (T == 0) return MIQ_OK;
  MIQ_REQUIRE(cache, MIQ_ERR_INVALID, "qk_norm_rope_kv4: null pointer");
  MIQ_REQUIRE(aligned(cache, 16), MIQ_ERR_ALIGN, "qk_norm_rope_kv4: the cache must be 16-byte aligned");
  // T rows lie in at most this many blocks, wherever the first one is
  const int vblocks = (int)(((int64_t)T + kKv4Block - 2) / kKv4Block) + 1;
  const int U = several_heads(T, NH + NKV) ? kNrHeads4 : 1;
  const int64_t units = (int64_t)T * ((NH + U - 1) / U + NKV) + (int64_t)vblocks * NKV * 4 * (HD / 64);
  MIQ_REQUIRE(grid_holds(units), MIQ_ERR_UNSUPPORTED, "qk_norm_rope_kv4: T=%d is past the grid", T);
  if (int rc = check_apart("qk_norm_rope_kv4", qkv, x_dtype == MIQ_F32 ? 4 : 2, ld, q_out, cache, nullptr,
                           (size_t)NKV * kv4_blocks(LMAX) * kv4_record(HD), T, NH, NKV, HD))
    return rc;
  const dim3 grid((unsigned)((units + kNrWaves - 1) / kNrWaves)), block(64 * kNrWaves);
  const hipStream_t st = static_cast<hipStream_t>(stream);
#define MIQ_NR(HDV, XT, UV)                                                                                       \
  hipLaunchKernelGGL((norm_rope_kv4_kernel<HDV, XT, UV>), grid, block, 0, st, static_cast<const XT*>(qkv), (size_t)ld, qn, kn, eps, \
                     state, cos_tab, sin_tab, static_cast<XT*>(q_out), static_cast<uint8_t*>(cache), T, NH, NKV, LMAX, vblocks)
#define MIQ_NR_HD(XT, UV)                   \
  switch (HD) {                             \
    case 64: MIQ_NR(64, XT, UV); break;     \
    case 128: MIQ_NR(128, XT, UV); break;   \
    case 192: MIQ_NR(192, XT, UV); break;   \
    default: MIQ_NR(256, XT, UV);           \
  }
  if (x_dtype == MIQ_F32) {
    if (U == 1) { MIQ_NR_HD(float, 1) } else { MIQ_NR_HD(float, kNrHeads4) }
  } else {
    if (U == 1) { MIQ_NR_HD(__half, 1) } else { MIQ_NR_HD(__half, kNrHeads4) }
  }
#undef MIQ_NR_HD
#undef MIQ_NR
  return check_launch("qk_norm_rope_kv4");
}

extern "C" int miq_kv4_dequant_f32(const void* cache, float* k_out, float* v_out, int NKV, int LMAX, int HD, int start, int n,
                                   void* stream) {
  MIQ_REQUIRE(NKV > 0 && NKV <= 65535 && LMAX > 0 && LMAX <= (1 << 30) && HD > 0 && start >= 0 && n >= 0 && start <= LMAX && n <= LMAX - start,
              MIQ_ERR_INVALID, "kv4_dequant: NKV=%d LMAX=%d HD=%d start=%d n=%d", NKV, LMAX, HD, start, n);
  MIQ_REQUIRE(kv4_head(HD), MIQ_ERR_UNSUPPORTED, "kv4_dequant: HD=%d (64, 128, 192 or 256)", HD);
  if (n == 0 || (!k_out && !v_out)) return MIQ_OK;
  MIQ_REQUIRE(cache, MIQ_ERR_INVALID, "kv4_dequant: null pointer");
  MIQ_REQUIRE(aligned(cache, 16), MIQ_ERR_ALIGN, "kv4_dequant: the cache must be 16-byte aligned");
  const int blocks = (start + n - 1) / kKv4Block - start / kKv4Block + 1;
  MIQ_REQUIRE(blocks < (1 << 24), MIQ_ERR_UNSUPPORTED, "kv4_dequant: n=%d positions are past the grid", n);
  hipLaunchKernelGGL(kv4_dequant_kernel, dim3(blocks, (HD / 16 * 64 + 255) / 256, NKV), dim3(256), 0, static_cast<hipStream_t>(stream),
                     static_cast<const uint8_t*>(cache), k_out, v_out, HD, kv4_blocks(LMAX), start, n);
  return check_launch("kv4_dequant");
}
