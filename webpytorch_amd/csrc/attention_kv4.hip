// Causal grouped-query attention over the 4-bit cache (kv4.h): row t sits at position pos0 + t (pos0 read
// from the device), and query head h attends to the cache positions 0 .. pos0 + t of kv head
// h / (NH / NKV). scores = (q . k) scale; p = exp(s - max) / sum; out = sum p v.
//
// A kv head's queries are rows r = t rep + hh (rep = NH / NKV heads share its keys and values), 16
// to a tile. A wave multiplies transposed on the fp16 matrix cores: S^T = K Q^T, then O^T = V^T P^T; the
// words of the cache are unpacked in registers, in operand order (kv4.h), and no value moves between lanes
// from the scores to the output. K and V are exact fp16; p is two fp16 numbers (hi + lo: 22 bits), and so is q of
// fp32 rows (scaled by a power of two per row); q of fp16 rows is exact. Sums and softmax statistics are fp32. p is held
// times 2^11 or more, so that its lower part stays in fp16's normal range. (p of fp16 rows as one number cost the output as
// much again as its own rounding, 2.7e-4 of float64 instead of 2.0e-4, and saved a third of the matrix instructions:
// 6001 rows of 28 / 4 heads of 128 326 us instead of 400.)
//
// Bound and measured (us a pass; the floor is the larger of the bytes at a large copy's 4.8 TB/s and the operations at a
// large fp16 product's 1180 TFLOP/s, twice for fp32 rows and one and a half times for fp16 rows): one token of 32 / 8 heads
// of 128 behind 131000 positions 41 (168 MB, 4.1 TB/s; floor 35: 80 KB in flight a CU); behind 700 positions of 14 / 2
// heads of 64 7.2 (round trips); 2000 fp32 rows of 28 / 4 heads of 128 from an empty cache 81 (floor 49), 6001 fp16 rows
// 400 (floor 328), 77 fp16 tokens of 32 / 8 heads behind 30000 71 and 9 to join 21 slices (floor 48): bound by
// the issue of instructions (2000 rows: a wave and step of 32 keys have 154 vector and 34 matrix instructions; the vector
// units are busy 44 % and the matrix cores 30 % of the time; a third of the vector instructions unpack).
#include <math.h>

#include "kv4.h"

namespace miq {

constexpr int kA4Waves = 8;
constexpr int kA4Rows = 16;
// The reference of the exponentials is raised only when a score passes it by more than 2^4 (a probability, 2^11 at the
// reference, then stays below 2^15), so that the output is seldom rescaled (131000 positions 50 -> 47 us a replay); each
// row by its own scores alone, so that a token's bits do not depend on its neighbours' queries. The unit is as high as
// that and fp16's range allow: two fp16 numbers hold it to 2^-25, so that of 100000 keys that share 0.1 % beside one the sum
// is right to 4e-7 (5e-6 at 2^7; a slack of 2^8 takes the same time).
constexpr float kA4UnitLog2 = 11.f, kA4Slack = 4.f;
constexpr int kA4CtrStride = 32;    // ints between arrival counters: a 128-byte line each
constexpr int kA4MaxSlices = 64;
constexpr int kA4MinSteps = 8;      // key steps of a slice of many rows, at least

// the maximum over the four lanes c, c + 16, c + 32, c + 48
__device__ __forceinline__ float rows_max(float v) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
// 2^n of a row: q 2^n has its largest magnitude in [2^13, 2^14) (less below fp32's normal range); 1 for non-finite rows
__device__ __forceinline__ int row_shift(float mx) {
  const int e = (int)((__float_as_uint(mx) >> 23) & 255);
  return e == 255 ? 0 : 13 + 127 - max(e, 1);
}

// A row's reference: a score s (the matrix cores' sum) has the probability 2^((s - shift) back + neg), a fused product
// and sum. Scores below kA4Far units of log 2 have shift 0 and a whole reference, neg = kA4UnitLog2 - rint(the highest),
// which is exact, so that rescaling is by powers of two. Past it no fp32 number lies near enough to all scores: the
// highest is taken off in the matrix cores' units first, where it leaves an exact 0 for its own key. (A reference
// rounded in units of log 2 is off by its last place, 2^7 at 2^30, and takes the exponentials of every key to 0 or
// to infinity.)
constexpr float kA4Far = 4194304.f, kA4NoKey = 3.402823466e38f;  // 2^22; neg of a row that has met no key
struct Ref {
  float shift, neg;
};
// the exponent that the row's highest score (-inf: none) has now
__device__ __forceinline__ float ref_exponent(const Ref& r, float mx, float back) { return fmaf(mx - r.shift, back, r.neg); }
// Takes mx as the reference where the exponent is past the slack; returns what the row's sums are rescaled by.
__device__ __forceinline__ float ref_raise(Ref& r, float mx, float back) {
  if (!(ref_exponent(r, mx, back) > kA4UnitLog2 + kA4Slack)) return 1.f;
  const float top = mx * back;  // past fp32's range: NaN, as the difference of two such scores is
  const Ref n = fabsf(top) < kA4Far ? Ref{0.f, kA4UnitLog2 - rintf(top)} : Ref{mx, kA4UnitLog2 + (top - top)};
  const float f = __builtin_amdgcn_exp2f(fmaf(r.shift - n.shift, back, n.neg - r.neg));
  r = n;
  return f;
}
// the reference in units of log 2, -inf for none
__device__ __forceinline__ float ref_log2(const Ref& r, float back) {
  return r.neg == kA4NoKey ? -INFINITY : fmaf(r.shift, back, kA4UnitLog2 - r.neg);
}

// the 8 numbers S (1 + c / 16) + Z of a key word: one S and Z
__device__ __forceinline__ half8v unpack_key(uint32_t w, uint32_t meta) {
  const half2v m = as_h2(meta), S = (half2v){m.x, m.x}, Z = (half2v){m.y, m.y};
  return cat4(fma2(kv4_pair<0>(w), S, Z), fma2(kv4_pair<1>(w), S, Z), fma2(kv4_pair<2>(w), S, Z),
              fma2(kv4_pair<3>(w), S, Z));
}
// of a value word: S and Z of its 8 keys in pairs
__device__ __forceinline__ half8v unpack_value(uint32_t w, miq_u32x4 S, miq_u32x4 Z) {
  return cat4(fma2(kv4_pair<0>(w), as_h2(S[0]), as_h2(Z[0])), fma2(kv4_pair<1>(w), as_h2(S[1]), as_h2(Z[1])),
              fma2(kv4_pair<2>(w), as_h2(S[2]), as_h2(Z[2])), fma2(kv4_pair<3>(w), as_h2(S[3]), as_h2(Z[3])));
}

// q of this lane (8 dimensions of every 32) as matrix-core operands: hi, and for fp32 rows lo, of q 2^n with the
// row's largest magnitude in [2^13, 2^14); `back` takes a product to units of log 2 and is positive (the sign
// of the scale goes into q; a scale of 0 makes q 0).
template <int HD, typename XT>
__device__ __forceinline__ void load_q(const XT* qr, float scale, half8v (&qh)[sizeof(XT) == 4 ? 2 : 1][HD / 32], float& back) {
  constexpr int P = sizeof(XT) == 4 ? 2 : 1, NJ = HD / 32;
  float v[NJ][8], mx = 0.f;
#pragma unroll
  for (int j = 0; j < NJ; ++j)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[j][e] = to_f32<XT>(qr[32 * j + e]);
      mx = fmaxf(mx, fabsf(v[j][e]));
    }
  const float sign = scale < 0.f ? -1.f : scale == 0.f ? 0.f : 1.f;
  const int n = P == 2 ? row_shift(rows_max(mx)) : 0;
  back = scale == 0.f ? 1.f : fmaxf(ldexpf(fabsf(scale) * 1.44269504088896340736f, -n), 0x1p-126f);
#pragma unroll
  for (int j = 0; j < NJ; ++j)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float x = sign * (P == 2 ? ldexpf(v[j][e], n) : v[j][e]);
      const _Float16 hi = (_Float16)x;
      qh[0][j][e] = hi;
      if constexpr (P == 2) qh[1][j][e] = (_Float16)(x - (float)hi);
    }
}

// Parts of slices pass through the device-scope coherence point: stores and loads past the XCD's own L2.
__device__ __forceinline__ void put2(float* p, float a, float b) {
  __hip_atomic_store(reinterpret_cast<uint64_t*>(p), (uint64_t)__float_as_uint(a) | ((uint64_t)__float_as_uint(b) << 32), __ATOMIC_RELAXED,
                     __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ uint64_t get2(const float* p) {
  return __hip_atomic_load(reinterpret_cast<const uint64_t*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// Whether this workgroup is the last of the `slices` that stored their parts (the counter is left zero).
__device__ __forceinline__ bool last_slice(int* ctr, int slices, int* last) {
  parts_stored();
  __syncthreads();
  if (threadIdx.x == 0) {
    *last = __hip_atomic_fetch_add(ctr, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == slices - 1;
    if (*last) __hip_atomic_store(ctr, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  return *last;
}
// out rows r0 .. r0 + nr - 1 from the slices' parts ([row][HD + 4]: the output, the maximum and the sum), in
// slice order
template <int HD, typename XT, int THREADS>
__device__ __forceinline__ void join_slices(const float* p0, size_t step, int slices, XT* out, int64_t pos0, int r0, int nr, int rep, int kv,
                                            int NH) {
  for (int x = threadIdx.x; x < nr * (HD / 2); x += THREADS) {
    const int row = x / (HD / 2), d = 2 * (x % (HD / 2));
    const float* pr = p0 + (size_t)row * (HD + 4);
    float mx = -INFINITY, sum = 0.f, a[2] = {0.f, 0.f};
    constexpr int U = 8;
    for (int k0 = 0; k0 < slices; k0 += U) {
      uint64_t st[U], v[U];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const float* ps = pr + (size_t)min(k0 + i, slices - 1) * step;
        st[i] = get2(ps + HD);
        v[i] = get2(ps + d);
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
    const bool none = pos0 + rr / rep < 0;  // a row without keys: zeros
    orow[0] = from_f32<XT>(none ? 0.f : a[0] / sum);
    orow[1] = from_f32<XT>(none ? 0.f : a[1] / sum);
  }
}

// 8 probabilities as matrix-core operands: the nearest fp16 number, and the one nearest to what that leaves (to 2^-25 at
// the least). Both to the nearest: towards zero, all small probabilities shrink alike beside a large one (of 16000 keys that
// share 1 % by a part in 6000). The sum of probabilities is taken of the operands, by the matrix cores.
__device__ __forceinline__ void split_p(const float* p, half8v* ph) {
  typedef float float2v __attribute__((ext_vector_type(2)));
  const float minus = __uint_as_float(opaque(0xBF800000u));  // -1: a difference would take a conversion of hi of its own
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    const half2v hi = __builtin_convertvector((float2v){p[2 * x], p[2 * x + 1]}, half2v);
    ph[0][2 * x] = hi.x;
    ph[0][2 * x + 1] = hi.y;
    ph[1][2 * x] = (_Float16)fmaf((float)hi.x, minus, p[2 * x]);
    ph[1][2 * x + 1] = (_Float16)fmaf((float)hi.y, minus, p[2 * x + 1]);
  }
}
__device__ __forceinline__ half8v ones() { return (half8v){1, 1, 1, 1, 1, 1, 1, 1}; }

// Groups with a NaN or an infinity (S negative) among a lane's 8 keys: their S and Z are cleared; the
// return value has a bit for each such key of the block (all lanes together).
__device__ __forceinline__ uint32_t clear_bad(miq_u32x4& S, miq_u32x4& Z) {
  uint32_t hit = 0;
  const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const uint32_t lo = (S[p] >> 15) & 1, hi = S[p] >> 31, keep = (lo ? 0u : 0xFFFFu) | (hi ? 0u : 0xFFFF0000u);
    hit |= (lo | hi << 1) << kv4_key(g, 2 * p);
    S[p] &= keep;
    Z[p] &= keep;
  }
  hit |= (uint32_t)__shfl_xor((int)hit, 16);
  return hit | (uint32_t)__shfl_xor((int)hit, 32);
}
// bits of the keys k0 .. k0 + 31 that a row attends to, its last key being lim
__device__ __forceinline__ uint32_t attends(int k0, int lim) { return lim < k0 ? 0u : lim - k0 >= 31 ? 0xFFFFFFFFu : (2u << (lim - k0)) - 1u; }
// the halves of a pair of keys k, k + 1 below end
__device__ __forceinline__ uint32_t keep_pair(int k, int end) { return (k < end ? 0xFFFFu : 0u) | (k + 1 < end ? 0xFFFF0000u : 0u); }

// Rows that fit a few tiles: the waves of a workgroup share a tile's 16 rows and split its keys, and so do
// the slices (blockIdx.x) of one tile and kv head. A slice's result (maximum, sum, output) goes to the
// workspace; the last slice of a tile to arrive adds them in slice order. (fp32 rows of 256 dimensions are more than the
// registers hold: 92 of them go through scratch memory, one token of 8 / 2 heads behind 120000 positions 86 us; fp16 39.)
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

  const int64_t pos0 = state[0];
  const int lim = (int)(pos0 + t < LMAX ? pos0 + t : LMAX - 1);  // this row's last key
  const int tl = (min(r0 + QR, R) - 1) / rep, tf = r0 / rep;
  const int S = (int)max((int64_t)0, min(pos0 + tl, (int64_t)LMAX - 1) + 1);  // keys that any row attends to
  const int first = (int)min(pos0 + tf, (int64_t)LMAX - 1);                   // the smallest last key
  const int nblk = (S + kKv4Block - 1) / kKv4Block;
  // blocks of a slice: joining costs 3 us or more, so that up to 3 blocks a wave are one slice (700 positions of 2
  // heads of 64: 8.6 -> 7.5 us), and from 256 blocks on a slice has two a wave (16000 positions: 14.7 -> 12.5 us)
  const int per = nblk <= 3 * NW ? 3 * NW : max(nblk >= 256 ? 2 * NW : NW, (nblk + (int)gridDim.x - 1) / (int)gridDim.x);
  const int slices = max(1, (nblk + per - 1) / per);
  if (slice >= slices) return;
  const int b0 = slice * per, b1 = min(nblk, b0 + per);

  // ---- a block's words: the next one's are loaded while one is multiplied, where the registers hold both ----
  constexpr int NR = HD <= 128 ? 2 : 1;
  struct Raw {
    uint32_t kw[NT], vw[NT], km[2][NJ];
    miq_u32x4 vs[NJ], vz[NJ];
  } raw[NR];
  auto load = [&](Raw& x, int blk) __attribute__((always_inline)) {
    const uint8_t* rec = C + (size_t)blk * kv4_record(HD);
#pragma unroll
    for (int u = 0; u < NT / 4; ++u) *reinterpret_cast<uint4*>(&x.kw[4 * u]) = *reinterpret_cast<const uint4*>(rec + (u * 64 + lane) * 16);
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int j = 0; j < NJ; j += 2)
        *reinterpret_cast<uint2*>(&x.km[b][j]) = *reinterpret_cast<const uint2*>(rec + kv4_kmeta(HD) + ((16 * b + c) * NJ + j) * 4);
#pragma unroll
    for (int u = 0; u < NT / 4; ++u)
      *reinterpret_cast<uint4*>(&x.vw[4 * u]) = *reinterpret_cast<const uint4*>(rec + kv4_vcodes(HD) + (u * 64 + lane) * 16);
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      x.vs[j] = *reinterpret_cast<const miq_u32x4*>(rec + kv4_vmeta(HD) + (j * 4 + g) * 32);
      x.vz[j] = *reinterpret_cast<const miq_u32x4*>(rec + kv4_vmeta(HD) + (j * 4 + g) * 32 + 16);
    }
  };
  const bool work = b0 + wave < b1;  // wave-uniform
  if (work) load(raw[0], b0 + wave);
  half8v qh[P][NJ];
  float back;
  load_q<HD, XT>(q + ((size_t)t * NH + h) * HD + 8 * g, scale, qh, back);

  float4v o[NT];
  float4v l = (float4v){0.f, 0.f, 0.f, 0.f};  // the sum of probabilities, in every row of the product
  Ref ref = {0.f, kA4NoKey};
  bool far = false;  // wave-uniform: a row of the wave has a shift
#pragma unroll
  for (int i = 0; i < NT; ++i) o[i] = (float4v){0.f, 0.f, 0.f, 0.f};
  auto multiply = [&](Raw& w, int blk) __attribute__((always_inline)) {
    auto& kw = w.kw;
    auto& vw = w.vw;
    auto& km = w.km;
    auto& vs = w.vs;
    auto& vz = w.vz;
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
        if (masked && blk * kKv4Block + 16 * b + 4 * g + x > lim) s[b][x] = -INFINITY;
        mx = fmaxf(mx, s[b][x]);
      }
    mx = rows_max(mx);
    if (__ballot(ref_exponent(ref, mx, back) > kA4UnitLog2 + kA4Slack)) {
      const float alpha = ref_raise(ref, mx, back);
      far = __ballot(ref.shift != 0.f) != 0ull;
      l *= alpha;
#pragma unroll
      for (int i = 0; i < NT; ++i) o[i] *= alpha;
    }
    if (far)
#pragma unroll
      for (int b = 0; b < 2; ++b) s[b] -= ref.shift;
    half8v ph[2];
    float p8[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) p8[e] = __builtin_amdgcn_exp2f(fmaf(s[e >> 2][e & 3], back, ref.neg));
    split_p(p8, ph);
#pragma unroll
    for (int p = 1; p >= 0; --p) l = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones(), ph[p], l, 0, 0, 0);

    // ---- values ----
    // keys behind the last one hold anything: their S and Z are cleared. A group with a NaN or an
    // infinity (S negative) is cleared too, and makes NaN of exactly the rows that attend to its key.
    if (masked) {
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        const uint32_t keep = keep_pair(blk * kKv4Block + kv4_key(g, 2 * p), S);
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          vs[j][p] &= keep;
          vz[j][p] &= keep;
        }
      }
    }
    uint32_t odd = 0;
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int p = 0; p < 4; ++p) odd |= vs[j][p];
    const bool bad = __ballot((odd & 0x80008000u) != 0) != 0ull;
    uint32_t hit[NJ] = {};  // keys whose group j is bad
    if (bad)
#pragma unroll
      for (int j = 0; j < NJ; ++j) hit[j] = clear_bad(vs[j], vz[j]);
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const half8v v = unpack_value(vw[i], vs[i >> 1], vz[i >> 1]);
#pragma unroll
      for (int p = 1; p >= 0; --p) o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, ph[p], o[i], 0, 0, 0);
    }
    if (bad)
#pragma unroll
      for (int j = 0; j < NJ; ++j)
        if (hit[j] & attends(blk * kKv4Block, lim)) {
          o[2 * j] += NAN;
          o[2 * j + 1] += NAN;
        }
  };
  if (work) {
    if constexpr (NR == 2) {
      for (int blk = b0 + wave;; blk += 2 * NW) {
        load(raw[1], min(blk + NW, b1 - 1));
        multiply(raw[0], blk);
        if (blk + NW >= b1) break;
        load(raw[0], min(blk + 2 * NW, b1 - 1));
        multiply(raw[1], blk + NW);
        if (blk + 2 * NW >= b1) break;
      }
    } else {
      for (int blk = b0 + wave; blk < b1; blk += NW) {
        if (blk != b0 + wave) load(raw[0], blk);
        multiply(raw[0], blk);
      }
    }
  }

  // ---- the waves' parts, rescaled to their common maximum ----
  const int nw = max(1, min(NW, b1 - b0));  // waves that had keys (wave 0 always takes part)
  const int nr = min(QR, R - r0);
  if (wave < nw) {
    if (g == 0) {
      ms[wave][c] = ref_log2(ref, back);
      ls[wave][c] = l[0];
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
      put2(part + row * (HD + 4) + d, a[0], a[1]);
      put2(part + row * (HD + 4) + d + 2, a[2], a[3]);
      if (d == 0) put2(part + row * (HD + 4) + HD, mx, sum);
      continue;
    }
    const int rr = r0 + row;
    XT* orow = out + ((size_t)(rr / rep) * NH + kv * rep + rr % rep) * HD + d;
#pragma unroll
    for (int e = 0; e < 4; ++e) orow[e] = from_f32<XT>(pos0 + rr / rep < 0 ? 0.f : a[e] / sum);  // a row without keys: zeros
  }
  if (slices == 1) return;

  if (!last_slice(counters + (kv * gridDim.y + tile) * kA4CtrStride, slices, &last)) return;
  join_slices<HD, XT, 64 * NW>(parts + (size_t)(kv * gridDim.y + tile) * gridDim.x * QR * (HD + 4), (size_t)QR * (HD + 4), slices,
                               out, pos0, r0, nr, rep, kv, NH);
}

// Many rows: a workgroup takes 4 x 16 QT of them, every wave its own, and all their keys (or a slice of
// them), 32 at a time (64 for HD 64). The waves unpack the records' words together, once for all rows, into
// operands in LDS, in operand order: each write and read is 16 consecutive bytes a lane. Two buffers, one
// barrier a step: while a step's products run, the next step's words, loaded a step before that, are unpacked.
constexpr int kA4TileWaves = 4;
// blocks of a step and 16-row tiles of a wave: what the registers hold (fp32 rows take twice the operands of q). fp16
// rows of heads of 64 at one tile a wave, which leaves a SIMD four waves instead of two, are faster over short contexts
// (3000 tokens of 14 / 2 heads 56 us instead of 72) and slower over long ones (500 behind 30000 161 instead of 118).
__host__ __device__ constexpr int kv4_step_blocks(int HD, bool f32) { return HD == 64 ? 2 : HD == 128 && !f32 ? 2 : 1; }
__host__ __device__ constexpr int kv4_tile_qt(int HD, bool f32) { return HD <= 128 && !f32 ? 2 : 1; }
__host__ __device__ constexpr int kv4_tile_rows(int HD, bool f32) { return kA4TileWaves * 16 * kv4_tile_qt(HD, f32); }

// Slices of `steps` key steps, of `per` steps each
__device__ __forceinline__ int tile_slices(int steps, int most, int& per) {
  per = max(kA4MinSteps, (steps + most - 1) / most);
  return max(1, (steps + per - 1) / per);
}
// float4s of a slice's part: per 16 rows the lanes' outputs [HD / 16][64] and (maximum, sum) of its rows
__host__ __device__ constexpr int kv4_part_unit(int HD) { return HD * 4 + 8; }

template <int HD, typename XT>
__global__ __launch_bounds__(64 * kA4TileWaves, HD <= 128 && sizeof(XT) == 4 ? 3 : 2) void attention_kv4_tiles_kernel(
    const XT* __restrict__ q, const uint8_t* __restrict__ cache, const int32_t* __restrict__ state, XT* __restrict__ out,
    int T, int NH, int NKV, int LMAX, float scale, float4v* __restrict__ parts) {
  constexpr int P = sizeof(XT) == 4 ? 2 : 1, NJ = HD / 32, NT = HD / 16, QT = kv4_tile_qt(HD, P == 2), NBK = kv4_step_blocks(HD, P == 2);
  constexpr int RW = 16 * QT, QR = kv4_tile_rows(HD, P == 2);
  constexpr int WPW = NBK * NT / kA4TileWaves;      // words of K, and of V, that a lane unpacks per step
  constexpr int NM = WPW % 2 ? WPW : WPW / 2;       // sets of S and Z of those of V (two adjacent tiles share one)
  extern __shared__ __align__(16) half8v ops[];  // [2 of K, 2 of V][NBK NT][64]
  __shared__ uint32_t flags[2][kA4TileWaves], hits[2][NBK][NJ];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), c = lane & 15, g = lane >> 4;
  const int kv = blockIdx.x, tile = (int)gridDim.y - 1 - (int)blockIdx.y, slice = blockIdx.z, rep = NH / NKV;  // long tiles first
  const int R = T * rep, r0 = tile * QR, rw = r0 + wave * RW;
  const uint8_t* C = cache + (size_t)kv * kv4_blocks(LMAX) * kv4_record(HD);

  const int64_t pos0 = state[0];
  const auto last_key = [&](int r) { return (int)min(pos0 + r / rep, (int64_t)LMAX - 1); };  // below 0: none
  const int S = max(0, last_key(min(r0 + QR, R) - 1) + 1);  // keys that any row attends to
  const int steps = (S + kKv4Block * NBK - 1) / (kKv4Block * NBK);
  int per;
  const int slices = tile_slices(steps, gridDim.z, per);
  if (slice >= slices) return;
  const int s0 = slice * per, s1 = min(steps, s0 + per);
  const int nblk = (S + kKv4Block - 1) / kKv4Block;

  // ---- words on their way: numbers n0 .. of a step's K and V words ----
  const int n0 = wave * WPW % NT, bo = wave * WPW / NT;
  uint32_t kw[WPW], km[WPW], vw[WPW];
  miq_u32x4 vs[NM], vz[NM];  // vectors: the loads of arrays of words were merged across S and Z and waited for at once (+1.5 %)
  auto words = [&](const uint8_t* part, uint32_t* w) __attribute__((always_inline)) {
    const uint8_t* at = part + kv4_word(n0, g, c);
    if constexpr (WPW == 2) *reinterpret_cast<uint2*>(w) = *reinterpret_cast<const uint2*>(at);
    else if constexpr (WPW == 4) *reinterpret_cast<uint4*>(w) = *reinterpret_cast<const uint4*>(at);
    else
#pragma unroll
      for (int x = 0; x < WPW; ++x) w[x] = *reinterpret_cast<const uint32_t*>(part + kv4_word(n0 + x, g, c));
  };
  auto fetch_k = [&](int step) __attribute__((always_inline)) {
    const uint8_t* rec = C + (size_t)min(step * NBK + bo, nblk - 1) * kv4_record(HD);
    words(rec, kw);
#pragma unroll
    for (int x = 0; x < WPW; ++x)
      km[x] = *reinterpret_cast<const uint32_t*>(rec + kv4_kmeta(HD) + ((16 * ((n0 + x) / NJ) + c) * NJ + (n0 + x) % NJ) * 4);
  };
  auto fetch_v = [&](int step) __attribute__((always_inline)) {
    const uint8_t* rec = C + (size_t)min(step * NBK + bo, nblk - 1) * kv4_record(HD);
    words(rec + kv4_vcodes(HD), vw);
#pragma unroll
    for (int x = 0; x < NM; ++x) {
      const miq_u32x4* at = reinterpret_cast<const miq_u32x4*>(rec + kv4_vmeta(HD) + ((n0 + x * (WPW / NM)) / 2 * 4 + g) * 32);
      vs[x] = at[0];
      vz[x] = at[1];
    }
  };
  // S and Z of step's values made fit: keys behind the last one hold anything and are cleared; so are groups
  // with a NaN or an infinity, which are noted for the rows
  auto check_v = [&](int step) __attribute__((always_inline)) {
    const int k0 = (step * NBK + bo) * kKv4Block;
    if (k0 + kKv4Block > S) {
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        const uint32_t keep = keep_pair(k0 + kv4_key(g, 2 * p), S);
#pragma unroll
        for (int x = 0; x < NM; ++x) {
          vs[x][p] &= keep;
          vz[x][p] &= keep;
        }
      }
    }
    uint32_t neg = 0;
#pragma unroll
    for (int x = 0; x < NM; ++x)
#pragma unroll
      for (int p = 0; p < 4; ++p) neg |= vs[x][p];
    const bool bad = __ballot((neg & 0x80008000u) != 0) != 0ull;
    uint32_t hit[NM] = {};
    if (bad)
#pragma unroll
      for (int x = 0; x < NM; ++x) hit[x] = clear_bad(vs[x], vz[x]);
    if (lane == 0) {
      flags[step & 1][wave] = bad;
#pragma unroll
      for (int x = 0; x < NM; ++x) hits[step & 1][bo][(n0 + x * (WPW / NM)) / 2] = hit[x];
    }
  };
  auto stage_k = [&](int step) __attribute__((always_inline)) {
    half8v* dst = ops + ((size_t)(step & 1) * NBK * NT + wave * WPW) * 64 + lane;
#pragma unroll
    for (int x = 0; x < WPW; ++x) dst[x * 64] = unpack_key(kw[x], km[x]);
  };
  auto stage_v = [&](int step) __attribute__((always_inline)) {
    half8v* dst = ops + ((size_t)(2 + (step & 1)) * NBK * NT + wave * WPW) * 64 + lane;
#pragma unroll
    for (int x = 0; x < WPW; ++x) dst[x * 64] = unpack_value(vw[x], vs[x * NM / WPW], vz[x * NM / WPW]);
  };

  // ---- q as matrix-core operands; scores in units of log 2, their factor positive ----
  half8v qh[QT][P][NJ];
  float back[QT];
  int lim[QT];
#pragma unroll
  for (int i = 0; i < QT; ++i) {
    const int r = min(rw + 16 * i + c, R - 1);
    lim[i] = last_key(r);
    load_q<HD, XT>(q + ((size_t)(r / rep) * NH + kv * rep + r % rep) * HD + 8 * g, scale, qh[i], back[i]);
  }
  const int first = last_key(min(rw, R - 1));

  float4v o[QT][NT], s[QT][2 * NBK];
  float4v l[QT];  // the sum of probabilities, in every row of the product
  Ref ref[QT];
  bool far = false;  // wave-uniform: a row of the wave has a shift
#pragma unroll
  for (int i = 0; i < QT; ++i) {
    ref[i] = {0.f, kA4NoKey};
    l[i] = (float4v){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int n = 0; n < NT; ++n) o[i][n] = (float4v){0.f, 0.f, 0.f, 0.f};
  }
  auto scores = [&](int step) __attribute__((always_inline)) {
    const half8v* kf = ops + (size_t)(step & 1) * NBK * NT * 64 + lane;
#pragma unroll
    for (int b = 0; b < 2 * NBK; ++b) {
#pragma unroll
      for (int i = 0; i < QT; ++i) s[i][b] = (float4v){0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const half8v k = kf[(b * NJ + j) * 64];
#pragma unroll
        for (int p = P - 1; p >= 0; --p)
#pragma unroll
          for (int i = 0; i < QT; ++i) s[i][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, qh[i][p][j], s[i][b], 0, 0, 0);
      }
    }
  };
  // masks the scores of `step`, raises the references they need and takes the shifts off
  auto refer = [&](int step) __attribute__((always_inline)) {
    const int k0 = step * NBK * kKv4Block;
    if (k0 + NBK * kKv4Block - 1 > first) {  // wave-uniform
#pragma unroll
      for (int i = 0; i < QT; ++i)
#pragma unroll
        for (int b = 0; b < 2 * NBK; ++b)
#pragma unroll
          for (int x = 0; x < 4; ++x)
            if (k0 + 16 * b + 4 * g + x > lim[i]) s[i][b][x] = -INFINITY;
    }
    float mx[QT];
    bool raise = false;
#pragma unroll
    for (int i = 0; i < QT; ++i) {
      mx[i] = -INFINITY;
#pragma unroll
      for (int b = 0; b < 2 * NBK; ++b)
#pragma unroll
        for (int x = 0; x < 4; ++x) mx[i] = fmaxf(mx[i], s[i][b][x]);
      mx[i] = rows_max(mx[i]);
      raise |= ref_exponent(ref[i], mx[i], back[i]) > kA4UnitLog2 + kA4Slack;
    }
    if (__ballot(raise)) {
      bool shifted = false;
#pragma unroll
      for (int i = 0; i < QT; ++i) {
        const float alpha = ref_raise(ref[i], mx[i], back[i]);
        shifted |= ref[i].shift != 0.f;
        l[i] *= alpha;
#pragma unroll
        for (int n = 0; n < NT; ++n) o[i][n] *= alpha;
      }
      far = __ballot(shifted) != 0ull;
    }
    if (far)
#pragma unroll
      for (int i = 0; i < QT; ++i)
#pragma unroll
        for (int b = 0; b < 2 * NBK; ++b) s[i][b] -= ref[i].shift;
  };

  // K runs a step ahead of V: in step t the waves multiply K(t + 1) and V(t), unpack K(t + 2) and V(t + 1), and
  // load the words after those. Words past the slice are loaded (from the last record) and not used.
  if (s0 < s1) {
    fetch_k(s0);
    fetch_v(s0);
    stage_k(s0);
    fetch_k(s0 + 1);
    check_v(s0);
    stage_v(s0);
    fetch_v(s0 + 1);
    __syncthreads();
    scores(s0);
    stage_k(s0 + 1);
    fetch_k(s0 + 2);
    refer(s0);
    __syncthreads();
  }
  if (rw >= R) {  // a wave without rows only unpacks (77 tokens of 4 heads a kv head behind 30000: 81 -> 76.5 us)
    for (int step = s0; step < s1; ++step) {
      check_v(step + 1);
      stage_k(step + 2);
      stage_v(step + 1);
      fetch_k(step + 3);
      fetch_v(step + 2);
      __syncthreads();
    }
    return;
  }
  for (int step = s0; step < s1; ++step) {
    check_v(step + 1);
    const half8v* vf = ops + (size_t)(2 + (step & 1)) * NBK * NT * 64 + lane;
    half8v ph[QT][NBK][2];
#pragma unroll
    for (int i = 0; i < QT; ++i)
#pragma unroll
      for (int b = 0; b < NBK; ++b) {
        float p[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) p[e] = __builtin_amdgcn_exp2f(fmaf(s[i][2 * b + (e >> 2)][e & 3], back[i], ref[i].neg));
        split_p(p, ph[i][b]);
      }
    scores(step + 1);
    stage_k(step + 2);
    stage_v(step + 1);
    fetch_k(step + 3);
    fetch_v(step + 2);
#pragma unroll
    for (int b = 0; b < NBK; ++b)
#pragma unroll
      for (int p = 1; p >= 0; --p)
#pragma unroll
        for (int i = 0; i < QT; ++i) l[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones(), ph[i][b][p], l[i], 0, 0, 0);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int b = 0; b < NBK; ++b) {
        const half8v v = vf[(b * NT + n) * 64];
#pragma unroll
        for (int p = 1; p >= 0; --p)
#pragma unroll
          for (int i = 0; i < QT; ++i) o[i][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, ph[i][b][p], o[i][n], 0, 0, 0);
      }
    const int fb = step & 1;
    if (uniform((int)(flags[fb][0] | flags[fb][1] | flags[fb][2] | flags[fb][3]))) {
#pragma unroll
      for (int b = 0; b < NBK; ++b)
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
          for (int i = 0; i < QT; ++i)
            if (hits[fb][b][j] & attends((step * NBK + b) * kKv4Block, lim[i])) {
              o[i][2 * j] += NAN;
              o[i][2 * j + 1] += NAN;
            }
    }
    if (step + 1 < s1) refer(step + 1);
    __syncthreads();
  }

  // ---- out, or the slice's part ----
#pragma unroll
  for (int i = 0; i < QT; ++i) {
    const float sum = l[i][0];
    const int r = rw + 16 * i + c;
    if (slices > 1) {
      float4v* part = parts + (((size_t)(kv * gridDim.y + tile) * (QR / 16) + wave * QT + i) * gridDim.z + slice) * kv4_part_unit(HD);
#pragma unroll
      for (int n = 0; n < NT; ++n) part[n * 64 + lane] = o[i][n];
      if (g == 0) reinterpret_cast<float2*>(part + NT * 64)[c] = make_float2(ref_log2(ref[i], back[i]), sum);
      continue;
    }
    if (r >= R) continue;
    XT* orow = out + ((size_t)(r / rep) * NH + kv * rep + r % rep) * HD + 4 * g;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) orow[16 * n + e] = from_f32<XT>(lim[i] < 0 ? 0.f : o[i][n][e] / sum);  // a row without keys: zeros
  }
}

// The parts of a tile's slices, added in slice order: a workgroup takes 16 rows, its waves a quarter of the
// dimensions each. (In a launch of its own: one workgroup's last arrival would read all of a tile's parts alone.)
template <int HD, typename XT>
__global__ __launch_bounds__(256) void attention_kv4_join_kernel(const int32_t* __restrict__ state, const float4v* __restrict__ parts,
                                                                 XT* __restrict__ out, int T, int NH, int NKV, int LMAX, int most) {
  constexpr int NT = HD / 16, NW = NT / 4, QR = kv4_tile_rows(HD, sizeof(XT) == 4), STEP = kKv4Block * kv4_step_blocks(HD, sizeof(XT) == 4);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, g = lane >> 4;
  const int kv = blockIdx.y, unit = blockIdx.x, tile = unit / (QR / 16), rep = NH / NKV, R = T * rep, r = unit * 16 + c;
  const int64_t pos0 = state[0];
  const int S = max(0, (int)min(pos0 + (min((tile + 1) * QR, R) - 1) / rep, (int64_t)LMAX - 1) + 1);
  int per;
  const int slices = tile_slices((S + STEP - 1) / STEP, most, per);
  if (slices == 1 || unit * 16 >= R) return;
  const float4v* part = parts + ((size_t)kv * gridDim.x + unit) * most * kv4_part_unit(HD);
  float mx = -INFINITY, sum = 0.f;
  float4v a[NW];
#pragma unroll
  for (int n = 0; n < NW; ++n) a[n] = (float4v){0.f, 0.f, 0.f, 0.f};
  constexpr int U = 4;
  for (int k0 = 0; k0 < slices; k0 += U) {
    float2 st[U];
    float4v v[U][NW];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const float4v* pk = part + (size_t)min(k0 + i, slices - 1) * kv4_part_unit(HD);
      st[i] = reinterpret_cast<const float2*>(pk + NT * 64)[c];
#pragma unroll
      for (int n = 0; n < NW; ++n) v[i][n] = pk[(wave * NW + n) * 64 + lane];
    }
    float mn = mx;
#pragma unroll
    for (int i = 0; i < U; ++i) mn = fmaxf(mn, st[i].x);
    const float ref = mn == -INFINITY ? 0.f : mn, al = __builtin_amdgcn_exp2f(mx - ref);
    mx = mn;
    sum *= al;
#pragma unroll
    for (int n = 0; n < NW; ++n) a[n] *= al;
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (k0 + i < slices) {
        const float f = __builtin_amdgcn_exp2f(st[i].x - ref);
        sum = fmaf(f, st[i].y, sum);
#pragma unroll
        for (int n = 0; n < NW; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) a[n][e] = fmaf(f, v[i][n][e], a[n][e]);
      }
  }
  if (r >= R) return;
  XT* orow = out + ((size_t)(r / rep) * NH + kv * rep + r % rep) * HD + 4 * g;
#pragma unroll
  for (int n = 0; n < NW; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) orow[16 * (wave * NW + n) + e] = from_f32<XT>(pos0 + r / rep < 0 ? 0.f : a[n][e] / sum);
}

// Up to kA4FewRows rows of a kv head go by the rows kernel, and up to kA4SomeRows where the cache is short: it unpacks
// a block for 16 rows where the tiles kernel does for 64 or 128, but starts sooner and needs no second launch
// (us, rows / tiles kernel: 32 / 8 heads of 128, 64 rows, 8000 positions 21 / 28, 60000 65 / 66; 256 rows,
// 0 positions 6.1 / 9.9, 1000 17 / 20, 8000 43 / 42, 60000 214 / 164; 14 / 2 heads of 64, 63 rows, 8000 positions
// 13 / 19, 60000 21 / 38; 252 rows, 8000 14 / 20, 60000 43 / 47; 8 / 2 heads of 256 are the exception, 64 rows, 8000 positions
// 43 / 32, 256 rows 57 / 39). The position is the device's, so the rule goes by LMAX. Each tile's keys are
// split into as many slices as give every CU a workgroup (two of the tiles kernel's), of at least a block a
// wave (8 steps) of a full cache.
constexpr int kA4FewRows = 64, kA4SomeRows = 512;
constexpr int64_t kA4SomeKeys = 1 << 21;  // rows times positions
struct Kv4Plan {
  int tiles, slices, rows;  // rows of a tile
  bool few;
};
static Kv4Plan kv4_plan(int T, int NH, int NKV, int HD, int LMAX, bool f32) {
  Kv4Plan p;
  const int64_t R = (int64_t)T * (NH / NKV);
  p.few = R <= kA4FewRows || (R <= kA4SomeRows && R * LMAX <= kA4SomeKeys);
  p.rows = p.few ? kA4Rows : kv4_tile_rows(HD, f32);
  p.tiles = (int)((R + p.rows - 1) / p.rows);
  const int64_t wgs = (int64_t)p.tiles * NKV;
  const int steps = p.few ? kv4_blocks(LMAX) : (kv4_blocks(LMAX) + kv4_step_blocks(HD, f32) - 1) / kv4_step_blocks(HD, f32);
  const int least = p.few ? kA4Waves : kA4MinSteps;
  const int want = p.few ? kCUs : 2 * kCUs;
  int64_t s = wgs >= want ? 1 : want / wgs;
  if (s > (steps + least - 1) / least) s = (steps + least - 1) / least;
  if (s > kA4MaxSlices) s = kA4MaxSlices;
  p.slices = (int)s;
  return p;
}

static size_t kv4_part_bytes(const Kv4Plan& p, int NKV, int HD) {
  if (p.slices == 1) return 0;
  return (size_t)p.slices * p.tiles * NKV * (p.few ? (size_t)p.rows * (HD + 4) * 4 : (size_t)p.rows / 16 * kv4_part_unit(HD) * 16);
}

}  // namespace miq

using namespace miq;

static int check_attention_kv4(const char* what, int T, int NH, int NKV, int HD, int LMAX) {
  MIQ_REQUIRE(T >= 0 && NH > 0 && NKV > 0 && NH % NKV == 0 && NH <= (1 << 16) && NKV <= 65535 && HD > 0 && LMAX > 0 && LMAX <= (1 << 30),
              MIQ_ERR_INVALID, "%s: T=%d NH=%d NKV=%d HD=%d LMAX=%d", what, T, NH, NKV, HD, LMAX);
  MIQ_REQUIRE(kv4_head(HD), MIQ_ERR_UNSUPPORTED, "%s: HD=%d (64, 128, 192 or 256)", what, HD);
  MIQ_REQUIRE((int64_t)T * (NH / NKV) <= (int64_t)65535 * 16 * kA4TileWaves, MIQ_ERR_UNSUPPORTED, "%s: T=%d rows of %d heads a kv head are past the grid",
              what, T, NH / NKV);
  return MIQ_OK;
}

extern "C" int miq_attention_kv4_workspace(int T, int NH, int NKV, int HD, int LMAX, size_t* bytes) {
  MIQ_REQUIRE(bytes, MIQ_ERR_INVALID, "attention_kv4_workspace: null pointer");
  if (int rc = check_attention_kv4("attention_kv4_workspace", T, NH, NKV, HD, LMAX)) return rc;
  *bytes = 0;
  if (T == 0) return MIQ_OK;
  const size_t a = kv4_part_bytes(kv4_plan(T, NH, NKV, HD, LMAX, true), NKV, HD);
  const size_t b = kv4_part_bytes(kv4_plan(T, NH, NKV, HD, LMAX, false), NKV, HD);
  *bytes = a || b ? kCounterBytes + (a > b ? a : b) : 0;  // of either type of rows
  return MIQ_OK;
}

extern "C" int miq_attention_kv4(const void* q, int x_dtype, const void* cache, const int32_t* state, void* out, int T,
                                 int NH, int NKV, int HD, int LMAX, float scale, void* workspace, size_t ws_bytes,
                                 void* stream) {
  if (int rc = check_attention_kv4("attention_kv4", T, NH, NKV, HD, LMAX)) return rc;
  MIQ_REQUIRE(x_dtype == MIQ_F32 || x_dtype == MIQ_F16, MIQ_ERR_UNSUPPORTED, "attention_kv4: x dtype %d", x_dtype);
  MIQ_REQUIRE(isfinite(scale * 1.44269504088896340736f), MIQ_ERR_INVALID, "attention_kv4: scale=%g", (double)scale);
  if (T == 0) return MIQ_OK;
  MIQ_REQUIRE(q && cache && state && out, MIQ_ERR_INVALID, "attention_kv4: null pointer");
  MIQ_REQUIRE(aligned(cache, 16), MIQ_ERR_ALIGN, "attention_kv4: the cache must be 16-byte aligned");
  const bool f32 = x_dtype == MIQ_F32;
  const Kv4Plan p = kv4_plan(T, NH, NKV, HD, LMAX, f32);
  const size_t part = kv4_part_bytes(p, NKV, HD);
  MIQ_REQUIRE(!part || (workspace && ws_bytes >= kCounterBytes + part), MIQ_ERR_INVALID,
              "attention_kv4: workspace of %zu bytes, %zu needed", workspace ? ws_bytes : (size_t)0, kCounterBytes + part);
  MIQ_REQUIRE(!part || aligned(workspace, 256), MIQ_ERR_ALIGN, "attention_kv4: the workspace must be 256-byte aligned");
  const size_t io = (size_t)T * NH * HD * (f32 ? 4 : 2);  // one tile's rows are written while another's are read
  MIQ_REQUIRE(!share_bytes(out, io, q, io), MIQ_ERR_INVALID, "attention_kv4: out must lie apart from q");
  MIQ_REQUIRE(!share_bytes(out, io, cache, (size_t)NKV * kv4_blocks(LMAX) * kv4_record(HD)), MIQ_ERR_INVALID,
              "attention_kv4: out must lie apart from the cache");
  int* counters = static_cast<int*>(workspace);
  float* parts = part ? reinterpret_cast<float*>(static_cast<char*>(workspace) + kCounterBytes) : nullptr;
  const size_t lds = p.few ? (size_t)kA4Waves * kA4Rows * (HD + 4) * 4
                           : (size_t)4 * kv4_step_blocks(HD, f32) * (HD / 16) * 64 * sizeof(half8v);
  if (int rc = require_lds("attention_kv4", lds + 2048)) return rc;
  const dim3 grid = p.few ? dim3((unsigned)p.slices, (unsigned)p.tiles, (unsigned)NKV) : dim3((unsigned)NKV, (unsigned)p.tiles, (unsigned)p.slices);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  // the join reads what the tiles kernel left in the workspace: another thread's call on the stream waits
  std::unique_lock<std::mutex> whole(stream_lock(st), std::defer_lock);
  if (part) whole.lock();
#define MIQ_A4(HDV, XT)                                                                                              \
  if (p.few) {                                                                                                       \
    hipLaunchKernelGGL((attention_kv4_rows_kernel<HDV, XT>), grid, dim3(64 * kA4Waves), lds, st, static_cast<const XT*>(q), \
                       static_cast<const uint8_t*>(cache), state, static_cast<XT*>(out), T, NH, NKV, LMAX, scale, counters, parts); \
  } else {                                                                                                           \
    hipLaunchKernelGGL((attention_kv4_tiles_kernel<HDV, XT>), grid, dim3(64 * kA4TileWaves), lds, st, static_cast<const XT*>(q), \
                       static_cast<const uint8_t*>(cache), state, static_cast<XT*>(out), T, NH, NKV, LMAX, scale,    \
                       reinterpret_cast<float4v*>(parts));                                                           \
    if (part)                                                                                                        \
      hipLaunchKernelGGL((attention_kv4_join_kernel<HDV, XT>), dim3((unsigned)(p.tiles * (p.rows / 16)), (unsigned)NKV), dim3(256), 0, st, \
                         state, reinterpret_cast<const float4v*>(parts), static_cast<XT*>(out), T, NH, NKV, LMAX, p.slices); \
  }
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
