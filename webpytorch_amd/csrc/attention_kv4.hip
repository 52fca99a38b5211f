// Causal grouped-query attention over the 4-bit cache (kv4.h): row t sits at position pos0 + t (pos0 read
// from the device), and query head h attends to the cache positions 0 .. pos0 + t of kv head
// h / (NH / NKV). scores = (q . k) scale; p = exp(s - max) / sum; out = sum p v.
//
// A kv head's queries are rows r = t rep + hh (rep = NH / NKV heads share its keys and values), 16
// to a tile. A wave multiplies transposed on the fp16 matrix cores: S^T = K Q^T, then O^T = V^T P^T; the
// words of the cache are unpacked in registers, in operand order (kv4.h), and no value moves between lanes
// from the scores to the output. K and V are exact fp16; fp32 rows take q and p as two fp16 numbers each
// (hi + lo: 22 bits; q scaled by a power of two per row), fp16 rows take one (q is exact, p rounded to
// fp16: 2^-12 of a probability). Sums and softmax statistics are fp32. p is held times 2^14, so that its
// lower part stays in fp16's normal range.
#include <math.h>

#include "kv4.h"

namespace miq {

constexpr int kA4Waves = 8;
constexpr int kA4Rows = 16;
constexpr float kA4Unit = 16384.f;  // a probability of 1
constexpr int kA4CtrStride = 32;    // ints between arrival counters: a 128-byte line each
constexpr int kA4MaxSlices = 64;

// the maximum (the sum) over the four lanes c, c + 16, c + 32, c + 48
__device__ __forceinline__ float rows_max(float v) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float rows_sum(float v) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// 2^n of a row: q 2^n has its largest magnitude in [2^13, 2^14); 1 for zero and non-finite rows
__device__ __forceinline__ int row_shift(float mx) {
  const int e = (int)((__float_as_uint(mx) >> 23) & 255);
  return (e == 0 || e == 255) ? 0 : 13 + 127 - e;
}

// the 8 numbers S (1 + c / 16) + Z of a key word: one S and Z
__device__ __forceinline__ half8v unpack_key(uint32_t w, uint32_t meta) {
  const half2v m = as_h2(meta), S = (half2v){m.x, m.x}, Z = (half2v){m.y, m.y};
  return cat4(fma2(kv4_pair<0>(w), S, Z), fma2(kv4_pair<1>(w), S, Z), fma2(kv4_pair<2>(w), S, Z),
              fma2(kv4_pair<3>(w), S, Z));
}
// of a value word: S and Z of its 8 keys in pairs
__device__ __forceinline__ half8v unpack_value(uint32_t w, const uint32_t* S, const uint32_t* Z) {
  return cat4(fma2(kv4_pair<0>(w), as_h2(S[0]), as_h2(Z[0])), fma2(kv4_pair<1>(w), as_h2(S[1]), as_h2(Z[1])),
              fma2(kv4_pair<2>(w), as_h2(S[2]), as_h2(Z[2])), fma2(kv4_pair<3>(w), as_h2(S[3]), as_h2(Z[3])));
}

// Rows that fit a few tiles: the waves of a workgroup share a tile's 16 rows and split its keys, and so do
// the slices (blockIdx.x) of one tile and kv head. A slice's result (maximum, sum, output) goes to the
// workspace; the last slice of a tile to arrive adds them in slice order.
template <int HD, typename XT>
__global__ __launch_bounds__(64 * kA4Waves) void attention_kv4_rows_kernel(
    const XT* __restrict__ q, const uint8_t* __restrict__ cache, const int32_t* __restrict__ state, XT* __restrict__ out,
    int T, int NH, int NKV, int LMAX, float scale, int* __restrict__ counters, float* __restrict__ parts) {
  constexpr int P = sizeof(XT) == 4 ? 2 : 1;  // fp16 numbers per value of q and p
  constexpr int NJ = HD / 32, NT = HD / 16, NW = kA4Waves, QR = kA4Rows;
  extern __shared__ __align__(16) float os[];  // [NW][QR][HD + 4]
  __shared__ float ms[NW][QR], ls[NW][QR];
  __shared__ int last;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), c = lane & 15, g = lane >> 4;
  const int slice = blockIdx.x, tile = blockIdx.y, kv = blockIdx.z, rep = NH / NKV;
  const int R = T * rep, r0 = tile * QR, r = min(r0 + c, R - 1);
  const int t = r / rep, h = kv * rep + r % rep;
  const uint8_t* C = cache + (size_t)kv * kv4_blocks(LMAX) * kv4_record(HD);

  // ---- q as matrix-core operands ----
  half8v qh[P][NJ];
  float back = scale * 1.44269504088896340736f;  // scores in units of log 2
  {
    const XT* qr = q + ((size_t)t * NH + h) * HD + 8 * g;
    float v[NJ][8];
    float mx = 0.f;
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[j][e] = to_f32<XT>(qr[32 * j + e]);
        mx = fmaxf(mx, fabsf(v[j][e]));
      }
    }
    const int n = P == 2 ? row_shift(rows_max(mx)) : 0;
    back = ldexpf(back, -n);
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float x = P == 2 ? ldexpf(v[j][e], n) : v[j][e];
        const _Float16 hi = (_Float16)x;
        qh[0][j][e] = hi;
        if constexpr (P == 2) qh[1][j][e] = (_Float16)(x - (float)hi);
      }
  }

  const int64_t pos0 = state[0];
  const int lim = (int)(pos0 + t < LMAX ? pos0 + t : LMAX - 1);  // this row's last key
  const int tl = (min(r0 + QR, R) - 1) / rep, tf = r0 / rep;
  const int S = (int)max((int64_t)0, min(pos0 + tl, (int64_t)LMAX - 1) + 1);  // keys that any row attends to
  const int first = (int)min(pos0 + tf, (int64_t)LMAX - 1);                   // the smallest last key
  const int nblk = (S + kKv4Block - 1) / kKv4Block;
  // blocks of a slice: at least one a wave
  const int per = max(NW, (nblk + (int)gridDim.x - 1) / (int)gridDim.x);
  const int slices = max(1, (nblk + per - 1) / per);
  if (slice >= slices) return;
  const int b1 = min(nblk, (slice + 1) * per);

  float4v o[NT];
  float m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < NT; ++i) o[i] = (float4v){0.f, 0.f, 0.f, 0.f};
  for (int blk = slice * per + wave; blk < b1; blk += NW) {
    const uint8_t* rec = C + (size_t)blk * kv4_record(HD);
    uint32_t kw[NT], vw[NT], km[2][NJ], vm[NJ][8];
#pragma unroll
    for (int u = 0; u < NT / 4; ++u) {
      *reinterpret_cast<uint4*>(&kw[4 * u]) = *reinterpret_cast<const uint4*>(rec + (u * 64 + lane) * 16);
      *reinterpret_cast<uint4*>(&vw[4 * u]) = *reinterpret_cast<const uint4*>(rec + kv4_vcodes(HD) + (u * 64 + lane) * 16);
    }
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int j = 0; j < NJ; j += 2)
        *reinterpret_cast<uint2*>(&km[b][j]) =
            *reinterpret_cast<const uint2*>(rec + kv4_kmeta(HD) + ((16 * b + c) * NJ + j) * 4);
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int u = 0; u < 2; ++u)
        *reinterpret_cast<uint4*>(&vm[j][4 * u]) =
            *reinterpret_cast<const uint4*>(rec + kv4_vmeta(HD) + (j * 4 + g) * 32 + 16 * u);

    // ---- scores ----
    float4v s[2];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      s[b] = (float4v){0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const half8v k = unpack_key(kw[b * NJ + j], km[b][j]);
#pragma unroll
        for (int p = P - 1; p >= 0; --p) s[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, qh[p][j], s[b], 0, 0, 0);
      }
    }
    const bool masked = blk * kKv4Block + kKv4Block - 1 > first;  // wave-uniform
    float mx = -INFINITY;
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        float v = s[b][x] * back;
        if (masked && blk * kKv4Block + 16 * b + 4 * g + x > lim) v = -INFINITY;
        s[b][x] = v;
        mx = fmaxf(mx, v);
      }
    const float mn = fmaxf(m, rows_max(mx));
    const float ref = mn == -INFINITY ? 0.f : mn;  // no key yet: every probability is 0
    const float alpha = __builtin_amdgcn_exp2f(m - ref);
    m = mn;
    half8v ph[P];
    float ps = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float p = __builtin_amdgcn_exp2f(s[e >> 2][e & 3] - ref) * kA4Unit;
      ps += p;
      const _Float16 hi = (_Float16)p;
      ph[0][e] = hi;
      if constexpr (P == 2) ph[1][e] = (_Float16)(p - (float)hi);
    }
    l = l * alpha + ps;
#pragma unroll
    for (int i = 0; i < NT; ++i) o[i] *= alpha;

    // ---- values ----
    // keys behind the last one hold anything: their S and Z are cleared. A group with a NaN or an
    // infinity (S negative) is cleared too, and makes NaN of exactly the rows that attend to its key.
    if (masked) {
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        const int k = blk * kKv4Block + kv4_key(g, 2 * p);
        const uint32_t keep = (k < S ? 0xFFFFu : 0u) | (k + 1 < S ? 0xFFFF0000u : 0u);
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          vm[j][p] &= keep;
          vm[j][4 + p] &= keep;
        }
      }
    }
    uint32_t odd = 0;
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int p = 0; p < 4; ++p) odd |= vm[j][p];
    const bool bad = __ballot((odd & 0x80008000u) != 0) != 0ull;
    uint32_t hit[NJ];  // keys e of this lane whose group j is bad
    if (bad) {
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        hit[j] = 0;
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          const uint32_t w = vm[j][p];
          const uint32_t keep = ((w >> 15) & 1 ? 0u : 0xFFFFu) | (w >> 31 ? 0u : 0xFFFF0000u);
          hit[j] |= (((w >> 15) & 1) | ((w >> 31) << 1)) << (2 * p);
          vm[j][p] &= keep;
          vm[j][4 + p] &= keep;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const half8v v = unpack_value(vw[i], &vm[i >> 1][0], &vm[i >> 1][4]);
#pragma unroll
      for (int p = P - 1; p >= 0; --p) o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, ph[p], o[i], 0, 0, 0);
    }
    if (bad) {
#pragma unroll
      for (int j = 0; j < NJ; ++j)
        for (int gg = 0; gg < 4; ++gg) {
          const uint32_t hs = (uint32_t)__builtin_amdgcn_readlane((int)hit[j], 16 * gg);
          bool nan = false;
#pragma unroll
          for (int e = 0; e < 8; ++e) nan |= ((hs >> e) & 1) && blk * kKv4Block + kv4_key(gg, e) <= lim;
          if (nan) {
            o[2 * j] += NAN;
            o[2 * j + 1] += NAN;
          }
        }
    }
  }

  // ---- the waves' parts, rescaled to their common maximum ----
  const int nw = max(1, min(NW, b1 - slice * per));  // waves that had keys (wave 0 always takes part)
  const int nr = min(QR, R - r0);
  if (wave < nw) {
    l = rows_sum(l);
    if (g == 0) {
      ms[wave][c] = m;
      ls[wave][c] = l;
    }
    if (c < nr)
#pragma unroll
      for (int i = 0; i < NT; ++i)
        *reinterpret_cast<float4v*>(&os[((size_t)wave * QR + c) * (HD + 4) + 16 * i + 4 * g]) = o[i];
  }
  __syncthreads();
  float* part = slices > 1 ? parts + ((size_t)(kv * gridDim.y + tile) * gridDim.x + slice) * QR * (HD + 4) : nullptr;
  for (int x = threadIdx.x; x < nr * (HD / 4); x += 64 * NW) {
    const int row = x / (HD / 4), d = 4 * (x % (HD / 4));
    float mx = ms[0][row];
    for (int w = 1; w < nw; ++w) mx = fmaxf(mx, ms[w][row]);
    const float ref = mx == -INFINITY ? 0.f : mx;
    float4v a = (float4v){0.f, 0.f, 0.f, 0.f};
    float sum = 0.f;
    for (int w = 0; w < nw; ++w) {
      const float f = __builtin_amdgcn_exp2f(ms[w][row] - ref);
      sum = fmaf(f, ls[w][row], sum);
      const float4v v = *reinterpret_cast<const float4v*>(&os[((size_t)w * QR + row) * (HD + 4) + d]);
#pragma unroll
      for (int e = 0; e < 4; ++e) a[e] = fmaf(f, v[e], a[e]);
    }
    if (slices > 1) {
      uint64_t* o8 = reinterpret_cast<uint64_t*>(part + row * (HD + 4) + d);
#pragma unroll
      for (int e = 0; e < 2; ++e)
        __hip_atomic_store(o8 + e, (uint64_t)__float_as_uint(a[2 * e]) | ((uint64_t)__float_as_uint(a[2 * e + 1]) << 32),
                           __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      if (d == 0)
        __hip_atomic_store(reinterpret_cast<uint64_t*>(part + row * (HD + 4) + HD),
                           (uint64_t)__float_as_uint(mx) | ((uint64_t)__float_as_uint(sum) << 32), __ATOMIC_RELAXED,
                           __HIP_MEMORY_SCOPE_AGENT);
      continue;
    }
    const int rr = r0 + row;
    XT* orow = out + ((size_t)(rr / rep) * NH + kv * rep + rr % rep) * HD + d;
#pragma unroll
    for (int e = 0; e < 4; ++e) orow[e] = from_f32<XT>(sum == 0.f ? 0.f : a[e] / sum);  // a row without keys: zeros
  }
  if (slices == 1) return;

  // ---- the slices' parts, by the last to arrive ----
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  if (threadIdx.x == 0) {
    int* ctr = counters + (kv * gridDim.y + tile) * kA4CtrStride;
    last = __hip_atomic_fetch_add(ctr, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == slices - 1;
    if (last) __hip_atomic_store(ctr, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // re-armed
  }
  __syncthreads();
  if (!last) return;
  const float* p0 = parts + (size_t)(kv * gridDim.y + tile) * gridDim.x * QR * (HD + 4);
  const size_t step = (size_t)QR * (HD + 4);
  for (int x = threadIdx.x; x < nr * (HD / 2); x += 64 * NW) {
    const int row = x / (HD / 2), d = 2 * (x % (HD / 2));
    const float* pr = p0 + row * (HD + 4);
    float mx = -INFINITY, sum = 0.f, a[2] = {0.f, 0.f};
    constexpr int U = 8;
    for (int k0 = 0; k0 < slices; k0 += U) {
      uint64_t st[U], v[U];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const float* ps = pr + (size_t)min(k0 + i, slices - 1) * step;
        st[i] = __hip_atomic_load(reinterpret_cast<const uint64_t*>(ps + HD), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        v[i] = __hip_atomic_load(reinterpret_cast<const uint64_t*>(ps + d), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
      float mn = mx;
#pragma unroll
      for (int i = 0; i < U; ++i) mn = fmaxf(mn, __uint_as_float((uint32_t)st[i]));
      const float ref = mn == -INFINITY ? 0.f : mn;
      const float al = __builtin_amdgcn_exp2f(mx - ref);
      sum *= al;
      a[0] *= al;
      a[1] *= al;
      mx = mn;
#pragma unroll
      for (int i = 0; i < U; ++i)
        if (k0 + i < slices) {
          const float f = __builtin_amdgcn_exp2f(__uint_as_float((uint32_t)st[i]) - ref);
          sum = fmaf(f, __uint_as_float((uint32_t)(st[i] >> 32)), sum);
          a[0] = fmaf(f, __uint_as_float((uint32_t)v[i]), a[0]);
          a[1] = fmaf(f, __uint_as_float((uint32_t)(v[i] >> 32)), a[1]);
        }
    }
    const int rr = r0 + row;
    XT* orow = out + ((size_t)(rr / rep) * NH + kv * rep + rr % rep) * HD + d;
    orow[0] = from_f32<XT>(sum == 0.f ? 0.f : a[0] / sum);
    orow[1] = from_f32<XT>(sum == 0.f ? 0.f : a[1] / sum);
  }
}

// Slices of each tile's keys: as many as give every CU a workgroup, of at least a block a wave of a full cache.
struct Kv4Plan {
  int tiles, slices;
};
static Kv4Plan kv4_plan(int T, int NH, int NKV, int LMAX) {
  Kv4Plan p;
  p.tiles = (int)(((int64_t)T * (NH / NKV) + kA4Rows - 1) / kA4Rows);
  const int64_t wgs = (int64_t)p.tiles * NKV;
  const int most = (kv4_blocks(LMAX) + kA4Waves - 1) / kA4Waves;
  int64_t s = wgs >= kCUs ? 1 : kCUs / wgs;
  if (s > most) s = most;
  if (s > kA4MaxSlices) s = kA4MaxSlices;
  p.slices = (int)s;
  return p;
}

static size_t kv4_part_bytes(const Kv4Plan& p, int NKV, int HD) {
  return p.slices > 1 ? (size_t)p.slices * p.tiles * NKV * kA4Rows * (HD + 4) * 4 : 0;
}

}  // namespace miq

using namespace miq;

static int check_attention_kv4(const char* what, int T, int NH, int NKV, int HD, int LMAX) {
  MIQ_REQUIRE(T >= 0 && NH > 0 && NKV > 0 && NH % NKV == 0 && NH <= (1 << 16) && NKV <= 65535 && HD > 0 && LMAX > 0 && LMAX <= (1 << 30),
              MIQ_ERR_INVALID, "%s: T=%d NH=%d NKV=%d HD=%d LMAX=%d", what, T, NH, NKV, HD, LMAX);
  MIQ_REQUIRE(kv4_head(HD), MIQ_ERR_UNSUPPORTED, "%s: HD=%d (64, 128, 192 or 256)", what, HD);
  MIQ_REQUIRE((int64_t)T * (NH / NKV) <= (int64_t)65535 * kA4Rows, MIQ_ERR_UNSUPPORTED, "%s: T=%d rows of %d heads a kv head are past the grid",
              what, T, NH / NKV);
  return MIQ_OK;
}

extern "C" int miq_attention_kv4_workspace(int T, int NH, int NKV, int HD, int LMAX, size_t* bytes) {
  MIQ_REQUIRE(bytes, MIQ_ERR_INVALID, "attention_kv4_workspace: null pointer");
  if (int rc = check_attention_kv4("attention_kv4_workspace", T, NH, NKV, HD, LMAX)) return rc;
  *bytes = 0;
  if (T == 0) return MIQ_OK;
  const size_t part = kv4_part_bytes(kv4_plan(T, NH, NKV, LMAX), NKV, HD);
  *bytes = part ? kCounterBytes + part : 0;
  return MIQ_OK;
}

extern "C" int miq_attention_kv4(const void* q, int x_dtype, const void* cache, const int32_t* state, void* out, int T,
                                 int NH, int NKV, int HD, int LMAX, float scale, void* workspace, size_t ws_bytes,
                                 void* stream) {
  if (int rc = check_attention_kv4("attention_kv4", T, NH, NKV, HD, LMAX)) return rc;
  MIQ_REQUIRE(x_dtype == MIQ_F32 || x_dtype == MIQ_F16, MIQ_ERR_UNSUPPORTED, "attention_kv4: x dtype %d", x_dtype);
  if (T == 0) return MIQ_OK;
  MIQ_REQUIRE(q && cache && state && out, MIQ_ERR_INVALID, "attention_kv4: null pointer");
  MIQ_REQUIRE(aligned(cache, 16), MIQ_ERR_ALIGN, "attention_kv4: the cache must be 16-byte aligned");
  const Kv4Plan p = kv4_plan(T, NH, NKV, LMAX);
  const size_t part = kv4_part_bytes(p, NKV, HD);
  MIQ_REQUIRE(!part || (workspace && ws_bytes >= kCounterBytes + part), MIQ_ERR_INVALID,
              "attention_kv4: workspace of %zu bytes, %zu needed", workspace ? ws_bytes : (size_t)0, kCounterBytes + part);
  MIQ_REQUIRE(!part || aligned(workspace, 256), MIQ_ERR_ALIGN, "attention_kv4: the workspace must be 256-byte aligned");
  int* counters = static_cast<int*>(workspace);
  float* parts = part ? reinterpret_cast<float*>(static_cast<char*>(workspace) + kCounterBytes) : nullptr;
  const size_t lds = (size_t)kA4Waves * kA4Rows * (HD + 4) * 4;
  if (int rc = require_lds("attention_kv4", lds + 2048)) return rc;
  const dim3 grid((unsigned)p.slices, (unsigned)p.tiles, (unsigned)NKV), block(64 * kA4Waves);
  const hipStream_t st = static_cast<hipStream_t>(stream);
#define MIQ_A4(HDV, XT)                                                                                              \
  hipLaunchKernelGGL((attention_kv4_rows_kernel<HDV, XT>), grid, block, lds, st, static_cast<const XT*>(q),          \
                     static_cast<const uint8_t*>(cache), state, static_cast<XT*>(out), T, NH, NKV, LMAX, scale, counters, parts)
#define MIQ_A4_HD(XT)                 \
  switch (HD) {                       \
    case 64: MIQ_A4(64, XT); break;   \
    case 128: MIQ_A4(128, XT); break; \
    case 192: MIQ_A4(192, XT); break; \
    default: MIQ_A4(256, XT);         \
  }
  if (x_dtype == MIQ_F32) { MIQ_A4_HD(float) } else { MIQ_A4_HD(__half) }
#undef MIQ_A4_HD
#undef MIQ_A4
  return check_launch("attention_kv4");
}
