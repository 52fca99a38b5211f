// QK-norm, RoPE and the cache write in one pass over the fused q|k|v rows (`CausalLM._qkv`,
// `_rope_np` and `kv_write` of the reference: webtorch/llm.py:1498-1519, 1270-1304;
// webtorch/_core.py:1504-1540): q_h = rope(x_h / sqrt(mean(x_h^2) + eps) * qn), k likewise, v as it is, k and
// v into an fp32 cache or into the 4-bit one (kv4.h).
//
// A wave takes one head of one token, lane l its dimensions l, l + 64, ..: the mean is a wave sum, a
// group of 32 dimensions is half a wave, and a dimension's rotation partner is another register of the lane
// (HD 128, 256), the lane 32 further (HD 64), or read through LDS.
#include <math.h>

#include "kv4.h"

#pragma clang fp contract(off)

namespace miq {

constexpr int kNrWaves = 4;

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

// The fp32 cache: every product, quotient and sum rounded where miq_head_rmsnorm and miq_rope_kv
// round theirs, in their order, so that the results are theirs bit for bit.
__global__ __launch_bounds__(64 * kNrWaves) void norm_rope_kv_kernel(
    const float* __restrict__ qkv, size_t ld, const float* __restrict__ qn, const float* __restrict__ kn, float eps,
    const int32_t* __restrict__ state, const float* __restrict__ cos_t, const float* __restrict__ sin_t,
    float* __restrict__ q_out, float* __restrict__ kc, float* __restrict__ vc, int T, int NH, int NKV, int HD,
    int LMAX) {
  __shared__ float rows[kNrWaves][256];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int heads = NH + 2 * NKV, half = HD / 2;
  const int64_t unit = (int64_t)blockIdx.x * kNrWaves + wave;
  const bool live = unit < (int64_t)T * heads;
  const int t = live ? (int)(unit / heads) : 0, h = live ? (int)(unit % heads) : 0;
  const int64_t pos = (int64_t)state[0] + t;
  const bool in = pos >= 0 && pos < LMAX;
  const float* row = qkv + (size_t)t * ld + (size_t)h * HD;
  float v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = live && lane + 64 * i < HD ? row[lane + 64 * i] : 0.f;
  const float* w = h < NH ? qn : h < NH + NKV ? kn : nullptr;
  if (w) {  // whole waves
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) s = s + v[i] * v[i];
    s = wave_sum(s);
    const float r = sqrtf(s / (float)HD + eps);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (lane + 64 * i < HD) v[i] = (v[i] / r) * w[lane + 64 * i];
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) rows[wave][lane + 64 * i] = v[i];
  __syncthreads();
  if (!live) return;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int d = lane + 64 * i;
    if (d >= HD) break;
    if (h >= NH + NKV) {
      if (in) vc[((size_t)(h - NH - NKV) * LMAX + pos) * HD + d] = v[i];
      continue;
    }
    const int j = d < half ? d : d - half;
    float y = 0.f;
    if (in) {
      const float rv = d < half ? -rows[wave][d + half] : rows[wave][d - half];
      y = v[i] * cos_t[(size_t)pos * half + j] + rv * sin_t[(size_t)pos * half + j];
    }
    if (h < NH) q_out[((size_t)t * NH + h) * HD + d] = y;
    else if (in) kc[((size_t)(h - NH) * LMAX + pos) * HD + d] = y;
  }
}

// The 4-bit cache. A key's codes depend on which side of a border its value is, so q and k are computed
// in fp64 (the vector units' fp64 rate is half the fp32 one, and the pass waits for memory) and rounded once.
// Waves [0, T (NH + NKV)) take a head of q or k; the ones after them 8 values of each dimension, the 8
// positions that share words (kv4_key): a word that is not wholly new is read first.
template <int HD, typename XT>
__global__ __launch_bounds__(64 * kNrWaves) void norm_rope_kv4_kernel(
    const XT* __restrict__ qkv, size_t ld, const float* __restrict__ qn, const float* __restrict__ kn, float eps,
    const int32_t* __restrict__ state, const float* __restrict__ cos_t, const float* __restrict__ sin_t,
    XT* __restrict__ q_out, uint8_t* __restrict__ cache, int T, int NH, int NKV, int LMAX, int vblocks) {
  constexpr int N = HD / 64, NG = HD / 32, HALF = HD / 2;
  const int lane = threadIdx.x & 63;
  const int64_t unit = (int64_t)blockIdx.x * kNrWaves + uniform(threadIdx.x >> 6);
  const int64_t nqk = (int64_t)T * (NH + NKV);
  const int64_t pos0 = state[0];
  const int NB = kv4_blocks(LMAX);
  if (unit < nqk) {
    const int t = (int)(unit / (NH + NKV)), h = (int)(unit % (NH + NKV));
    const int64_t pos = pos0 + t;
    const bool in = pos >= 0 && pos < LMAX;
    const XT* row = qkv + (size_t)t * ld + (size_t)h * HD;
    if (!in) {  // a position outside the cache: no key, and zeros for its queries
      if (h < NH)
#pragma unroll
        for (int i = 0; i < N; ++i) q_out[((size_t)t * NH + h) * HD + lane + 64 * i] = from_f32<XT>(0.f);
      return;
    }
    double v[N];
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (double)to_f32<XT>(row[lane + 64 * i]);
    const float* w = h < NH ? qn : kn;
    if (w) {
      double s = 0.0;
#pragma unroll
      for (int i = 0; i < N; ++i) s += v[i] * v[i];
      const double inv = 1.0 / sqrt(wave_sum_d(s) / HD + (double)eps);
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = v[i] * inv * (double)w[lane + 64 * i];
    }
    float y[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int d = lane + 64 * i, j = d < HALF ? d : d - HALF;
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
      const double c = (double)cos_t[(size_t)pos * HALF + j], s = (double)sin_t[(size_t)pos * HALF + j];
      y[i] = (float)(d < HALF ? v[i] * c - o * s : v[i] * c + o * s);
    }
    if (h < NH) {
#pragma unroll
      for (int i = 0; i < N; ++i) q_out[((size_t)t * NH + h) * HD + lane + 64 * i] = from_f32<XT>(y[i]);
      return;
    }
    const int key = (int)(pos % kKv4Block);
    uint8_t* rec = cache + ((size_t)(h - NH) * NB + (size_t)(pos / kKv4Block)) * kv4_record(HD);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      uint16_t S, Z;
      uint32_t c = kv4_quantize(y[i], S, Z) << kv4_shift(lane & 7);
      c |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)c, 0xB1, 0xF, 0xF, false);
      c |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)c, 0x4E, 0xF, 0xF, false);
      c |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)c, 0x141, 0xF, 0xF, false);
      const int grp = 2 * i + (lane >> 5);
      if ((lane & 7) == 0)
        *reinterpret_cast<uint32_t*>(rec + kv4_word((key >> 4) * NG + grp, (lane & 31) >> 3, key & 15)) = c;
      if ((lane & 31) == 0)
        *reinterpret_cast<uint32_t*>(rec + kv4_kmeta(HD) + (key * NG + grp) * 4) = S | ((uint32_t)Z << 16);
    }
    return;
  }
  const int64_t vu = unit - nqk;
  const int g = (int)(vu & 3), kv = (int)((vu >> 2) % NKV);
  const int64_t first = pos0 > 0 ? pos0 : 0, blk = first / kKv4Block + (vu >> 2) / NKV;
  if ((vu >> 2) / NKV >= vblocks || blk >= NB) return;
  uint32_t live = 0;
  float x[8][N];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int64_t pos = blk * kKv4Block + kv4_key(g, e), t = pos - pos0;
    const bool in = t >= 0 && t < T && pos < LMAX;
    live |= (in ? 15u : 0u) << kv4_shift(e);
#pragma unroll
    for (int i = 0; i < N; ++i)
      x[e][i] = in ? to_f32<XT>(qkv[(size_t)t * ld + (size_t)(NH + NKV + kv) * HD + lane + 64 * i]) : 0.f;
  }
  if (!live) return;
  uint8_t* rec = cache + ((size_t)kv * NB + (size_t)blk) * kv4_record(HD);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int d = lane + 64 * i, grp = 2 * i + (lane >> 5);
    uint32_t* word = reinterpret_cast<uint32_t*>(rec + kv4_vcodes(HD) + kv4_word(d >> 4, g, d & 15));
    uint32_t c = live == 0xFFFFFFFFu ? 0u : *word & ~live;
    uint16_t* meta = reinterpret_cast<uint16_t*>(rec + kv4_vmeta(HD)) + (grp * 4 + g) * 16;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      uint16_t S, Z;
      const uint32_t code = kv4_quantize(x[e][i], S, Z);
      if ((live >> kv4_shift(e)) & 1) {
        c |= code << kv4_shift(e);
        if ((lane & 31) == 0) {
          meta[e] = S;
          meta[8 + e] = Z;
        }
      }
    }
    *word = c;
  }
}

// fp32 rows of the positions [start, start + n): a thread takes one word, of a key 8 dimensions, of the
// values one dimension of 8 positions
__global__ __launch_bounds__(256) void kv4_dequant_kernel(const uint8_t* __restrict__ cache, float* __restrict__ k_out,
                                                          float* __restrict__ v_out, int HD, int NB, int start, int n) {
  const int NT = HD / 16, NG = HD / 32;
  const int x = blockIdx.x * 256 + threadIdx.x;  // word of a block: [n][g][i]
  const int kv = blockIdx.z, blk = start / kKv4Block + blockIdx.y;
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

static int check_norm_rope(const char* what, const void* qkv, int64_t ld, const int32_t* state, const float* cos_tab,
                           const float* sin_tab, const void* q_out, int T, int NH, int NKV, int HD, int LMAX) {
  MIQ_REQUIRE(T >= 0 && NH > 0 && NKV > 0 && NH % NKV == 0 && NH <= (1 << 16) && HD > 0 && HD % 2 == 0 && HD <= 256 && LMAX > 0 &&
                  LMAX <= (1 << 30),
              MIQ_ERR_INVALID, "%s: T=%d NH=%d NKV=%d HD=%d LMAX=%d", what, T, NH, NKV, HD, LMAX);
  MIQ_REQUIRE(ld >= (int64_t)(NH + 2 * NKV) * HD, MIQ_ERR_INVALID, "%s: rows %lld apart hold %lld values", what, (long long)ld,
              (long long)(NH + 2 * NKV) * HD);
  MIQ_REQUIRE((int64_t)T * (NH + 2 * NKV) / kNrWaves < 0x7FFFFFFF - 1, MIQ_ERR_UNSUPPORTED, "%s: T=%d is past the grid", what, T);
  MIQ_REQUIRE(T == 0 || (qkv && state && cos_tab && sin_tab && q_out), MIQ_ERR_INVALID, "%s: null pointer", what);
  return MIQ_OK;
}

extern "C" int miq_qk_norm_rope_kv(const float* qkv, int64_t ld, const float* qn, const float* kn, float eps,
                                   const int32_t* state, const float* cos_tab, const float* sin_tab, float* q_out,
                                   float* kcache, float* vcache, int T, int NH, int NKV, int HD, int LMAX, void* stream) {
  if (int rc = check_norm_rope("qk_norm_rope_kv", qkv, ld, state, cos_tab, sin_tab, q_out, T, NH, NKV, HD, LMAX)) return rc;
  if (T == 0) return MIQ_OK;
  MIQ_REQUIRE(kcache && vcache, MIQ_ERR_INVALID, "qk_norm_rope_kv: null pointer");
  const int64_t units = (int64_t)T * (NH + 2 * NKV);
  hipLaunchKernelGGL(norm_rope_kv_kernel, dim3((unsigned)((units + kNrWaves - 1) / kNrWaves)), dim3(64 * kNrWaves), 0,
                     static_cast<hipStream_t>(stream), qkv, (size_t)ld, qn, kn, eps, state, cos_tab, sin_tab, q_out, kcache,
                     vcache, T, NH, NKV, HD, LMAX);
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
  const int vblocks = (T + kKv4Block - 2) / kKv4Block + 1;
  const int64_t units = (int64_t)T * (NH + NKV) + (int64_t)vblocks * NKV * 4;
  const dim3 grid((unsigned)((units + kNrWaves - 1) / kNrWaves)), block(64 * kNrWaves);
  const hipStream_t st = static_cast<hipStream_t>(stream);
#define MIQ_NR(HDV, XT)                                                                                           \
  hipLaunchKernelGGL((norm_rope_kv4_kernel<HDV, XT>), grid, block, 0, st, static_cast<const XT*>(qkv), (size_t)ld, qn, kn, eps, \
                     state, cos_tab, sin_tab, static_cast<XT*>(q_out), static_cast<uint8_t*>(cache), T, NH, NKV, LMAX, vblocks)
#define MIQ_NR_HD(XT)               \
  switch (HD) {                     \
    case 64: MIQ_NR(64, XT); break; \
    case 128: MIQ_NR(128, XT); break; \
    case 192: MIQ_NR(192, XT); break; \
    default: MIQ_NR(256, XT);       \
  }
  if (x_dtype == MIQ_F32) { MIQ_NR_HD(float) } else { MIQ_NR_HD(__half) }
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
  MIQ_REQUIRE(blocks <= 65535, MIQ_ERR_UNSUPPORTED, "kv4_dequant: n=%d positions are past the grid", n);
  hipLaunchKernelGGL(kv4_dequant_kernel, dim3((HD / 16 * 64 + 255) / 256, blocks, NKV), dim3(256), 0, static_cast<hipStream_t>(stream),
                     static_cast<const uint8_t*>(cache), k_out, v_out, HD, kv4_blocks(LMAX), start, n);
  return check_launch("kv4_dequant");
}
