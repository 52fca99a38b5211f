// Grouped-query attention of a few new tokens of each of many sequences over a paged cache (paged.h): row (s, t) attends to
// the positions 0 .. positions[s][t] of its sequence, query head h to kv head h / (NH / NKV).
// scores = (q . k) scale; p = exp(s - max) / sum; out = sum p v. (`KVCache.attn`, `gqa_attention` of the reference, one
// sequence over a contiguous cache: webtorch/_core.py:1543-1596, 1319-1340.)
//
// A kv head's queries are rows r = t rep + hh, 16 to a tile, NR tiles to a workgroup, whose 8 waves take a block of its keys
// in turn (32 of an fp16 cache, 16 of an fp32 one: 16 KB of keys and values at heads of 128). A wave multiplies
// S^T = K Q^T, then O^T = V^T P^T, on the matrix cores: the rows of K are operands as they lie in memory, the probabilities
// leave the first product in the lanes where the second wants them, and the values, loaded as rows of 16 bytes a lane, become
// operands by 16-bit permutations within the lane (fp16) or as they are (fp32, whose products take 4 keys at a time). No
// key or value passes through LDS; it holds q's operands.
// fp16 caches: K and V are exact, p is two fp16 numbers (22 bits), and so is q of fp32 rows. fp32 caches: fp32 products.
// Sums and softmax statistics are fp32.
//
// The work is split by the lengths, which are the device's: every workgroup adds them up and takes its part of a sequence, the
// parts as long as give the chip about kPaWorkgroups of them, so that long sequences beside short ones fill it too. The last
// part of a sequence and head to arrive adds the parts, in their order.
#include <math.h>

#include "attention_parts.h"
#include "kv4.h"
#include "paged.h"

namespace miq {

constexpr int kPaWaves = 8;
constexpr int kPaWorkgroups = 256;
constexpr int kPaMinSteps = 3;   // blocks a wave of a part, at least: joining costs as much
constexpr int kPaCtrStride = 8;  // ints between arrival counters
constexpr int kPaMaxSplit = 4096;  // sequences x heads x tiles from which they are not split: their counters, 128 KB

template <typename CT> struct PagedKeys;  // keys of a block: 16-key tiles of it
template <> struct PagedKeys<__half> { static constexpr int kBlock = 32, kTiles = 2; };
template <> struct PagedKeys<float> { static constexpr int kBlock = 16, kTiles = 1; };

__host__ __device__ constexpr int pa_planes(bool c16, bool x32) { return c16 && x32 ? 2 : 1; }
// bytes of LDS: the operands of q, then (in their place) the waves' sums of one 16-row tile
__host__ __device__ constexpr size_t pa_lds(int HD, int NR, bool c16, bool x32) {
  const size_t q = (size_t)NR * 16 * HD * (c16 ? 2 * pa_planes(c16, x32) : 4), o = (size_t)kPaWaves * 16 * (HD + 4) * 4;
  return q > o ? q : o;
}

// 16-bit halves of two words: (low, low) or (high, high)
__device__ __forceinline__ uint32_t lows(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x05040100u); }
__device__ __forceinline__ uint32_t highs(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }

template <int HD, int NR, typename CT, typename XT>
__global__ __launch_bounds__(64 * kPaWaves) void paged_attention_kernel(
    const XT* __restrict__ q, const CT* __restrict__ cache, const int32_t* __restrict__ positions, const int32_t* __restrict__ pages,
    XT* __restrict__ out, int S, int T, int NH, int NKV, int tiles, int num_pages, int pshift, int max_pages, float scale, int lshift,
    int target, int* __restrict__ counters, float* __restrict__ parts) {
  constexpr bool C16 = sizeof(CT) == 2;
  constexpr int QP = pa_planes(C16, sizeof(XT) == 4);
  constexpr int KB = PagedKeys<CT>::kBlock, NT = PagedKeys<CT>::kTiles, DL = HD / 16, NW = kPaWaves;
  constexpr int NJ = C16 ? HD / 32 : HD / 16;  // 16-byte loads of a lane per 16 keys
  extern __shared__ __align__(16) char lds[];
  __shared__ float backs[16 * NR], ms[NW][16], ls[NW][16];
  __shared__ int last;
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), c = lane & 15, g = lane >> 4;
  const int rep = NH / NKV, R = T * rep, units = NKV * tiles, unit = blockIdx.x % units, want = blockIdx.x / units;
  const int h = unit % NKV, r0 = unit / NKV * 16 * NR, cap = max_pages << pshift;

  // ---- which sequence, and which part of it: 64 >> lshift sequences at a time, 1 << lshift lanes each ----
  const int lane_s = lane >> lshift, sub = lane & ((1 << lshift) - 1), at_once = 64 >> lshift;
  auto steps_of = [&](int s0) __attribute__((always_inline)) {
    const int s = s0 + lane_s;
    int n = 0;
    if (s < S)
#pragma unroll 4
      for (int t = sub; t < T; t += 1 << lshift) n = max(n, min(positions[(int64_t)s * T + t], cap - 1) + 1);
    for (int d = 1; d < 1 << lshift; d *= 2) n = max(n, __shfl_xor(n, d));
    return (n + KB * NW - 1) / (KB * NW);
  };
  int s = 0, part = 0, nparts = 1, steps = 0;
  {
    int mine = steps_of(0);
    double total = sub == 0 ? mine : 0;
    for (int s0 = at_once; s0 < S; s0 += at_once) {
      const int n = steps_of(s0);
      total += sub == 0 ? n : 0;
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) total += __shfl_xor(total, d);
    // steps of a part: target of them together, and one more for each sequence and head
    const double least = ceil(total * units / target);
    const int per = target <= 0 || least > 1e9 ? 1 << 30 : max(kPaMinSteps, (int)least);
    int before = 0, s0 = 0;
    for (;;) {
      const int n = sub == 0 && s0 + lane_s < S ? max(1, (mine + per - 1) / per) : 0;
      int sum = n;
#pragma unroll
      for (int d = 1; d < 64; d *= 2) {
        const int o = __shfl_up(sum, d);
        sum += lane >= d ? o : 0;
      }
      const uint64_t here = __ballot(n > 0 && want < before + sum);
      if (here) {
        const int l = __builtin_ctzll(here);
        nparts = __builtin_amdgcn_readlane(n, l);
        part = want - before - (__builtin_amdgcn_readlane(sum, l) - nparts);
        s = s0 + (l >> lshift);
        steps = __builtin_amdgcn_readlane(mine, l);
        break;
      }
      before += __builtin_amdgcn_readlane(sum, 63);
      s0 += at_once;
      if (s0 >= S) return;  // no part is left for this workgroup
      mine = steps_of(s0);
    }
  }

  // ---- this workgroup's rows and keys ----
  const int32_t* pos = positions + (int64_t)s * T;
  int lim[NR], first = 0x7FFFFFFF, end = 0;  // a row's last key (-1: none); the smallest of them; keys that any row attends to
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    const int r = r0 + 16 * n + c;
    lim[n] = r < R ? max(-1, min(pos[r / rep], cap - 1)) : -1;
    if (lim[n] >= 0) first = min(first, lim[n]);
    end = max(end, lim[n] + 1);
  }
#pragma unroll
  for (int d = 1; d < 16; d *= 2) {
    first = min(first, __shfl_xor(first, d));
    end = max(end, __shfl_xor(end, d));
  }
  first = uniform(first);
  end = uniform(end);
  const int base = steps / nparts, over = steps % nparts;
  const int b0 = (part * base + min(part, over)) * NW, b1 = min(b0 + (base + (part < over)) * NW, (end + KB - 1) / KB);
  const int32_t* table = pages + (int64_t)s * max_pages;
  const int64_t plane = ((int64_t)NKV << pshift) * HD;  // keys of a page, all heads
  const CT* const mine = cache + ((int64_t)h << pshift) * HD;

  // page of each 16-key tile of the wave's blocks, 64 blocks at a time: lane i the i-th
  int ids[NT];
  auto load_ids = [&](int blk) __attribute__((always_inline)) {
    const int b = blk + NW * lane;
#pragma unroll
    for (int a = 0; a < NT; ++a) {
      const int64_t k = (int64_t)b * KB + 16 * a;
      const int id = b < b1 && k < end ? table[k >> pshift] : -1;
      ids[a] = (uint32_t)id < (uint32_t)num_pages ? id : -1;
    }
  };
  struct Block {
    int id[NT];  // -1: no keys
  };
  miq_u32x4 kr[NT][NJ];
  uint32_t vr[NT][4][C16 ? DL / 2 : DL];
  auto tile_at = [&](int blk, int a, int id) __attribute__((always_inline)) {
    return mine + 2 * plane * (int64_t)max(id, 0) + (int64_t)((blk * KB + 16 * a) & ((1 << pshift) - 1)) * HD;
  };
  auto load_keys = [&](int blk, const Block& b) __attribute__((always_inline)) {
#pragma unroll
    for (int a = 0; a < NT; ++a) {
      const CT* p = tile_at(blk, a, b.id[a]) + c * HD + (C16 ? 8 : 4) * g;
#pragma unroll
      for (int j = 0; j < NJ; ++j) kr[a][j] = *reinterpret_cast<const miq_u32x4*>(p + (C16 ? 32 : 16) * j);
    }
  };
  auto load_values = [&](int blk, const Block& b) __attribute__((always_inline)) {
#pragma unroll
    for (int a = 0; a < NT; ++a) {
      const CT* p = tile_at(blk, a, b.id[a]) + plane + 4 * g * HD + DL * c;
      constexpr int NV = C16 ? DL / 2 : DL;  // words
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (NV % 4 == 0) {
#pragma unroll
          for (int i = 0; i < NV; i += 4) *reinterpret_cast<miq_u32x4*>(&vr[a][e][i]) = *reinterpret_cast<const miq_u32x4*>(p + e * HD + i * (C16 ? 2 : 1));
        } else {
#pragma unroll
          for (int i = 0; i < NV; i += 2) *reinterpret_cast<miq_u32x2*>(&vr[a][e][i]) = *reinterpret_cast<const miq_u32x2*>(p + e * HD + i * (C16 ? 2 : 1));
        }
      }
    }
  };
  auto block_at = [&](int i) __attribute__((always_inline)) {
    Block b;
#pragma unroll
    for (int a = 0; a < NT; ++a) b.id[a] = __builtin_amdgcn_readlane(ids[a], i);
    return b;
  };

  int blk = b0 + wave;
  const bool work = blk < b1;  // wave-uniform
  Block cur;
  if (work) {
    load_ids(blk);
    cur = block_at(0);
    load_keys(blk, cur);
    load_values(blk, cur);
  }

  // ---- q as operands in LDS, LG lanes a row ----
  {
    constexpr int LG = HD == 64 ? 8 : HD == 128 ? 16 : 32;
    const float sign = scale < 0.f ? -1.f : scale == 0.f ? 0.f : 1.f;
    const int ch = tid % LG;
    for (int row = tid / LG; row < 16 * NR; row += 64 * NW / LG) {
      const int r = r0 + row;
      const bool in = r < R && ch < HD / 8;
      float v[8], mx = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = 0.f;
      if (in) {
        const XT* p = q + (((int64_t)s * T + r / rep) * NH + h * rep + r % rep) * HD + 8 * ch;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          v[e] = to_f32<XT>(p[e]);
          mx = fmaxf(mx, fabsf(v[e]));
        }
      }
      int n = 0;
      if constexpr (QP == 2) {
#pragma unroll
        for (int d = 1; d < LG; d *= 2) mx = fmaxf(mx, __shfl_xor(mx, d));
        n = row_shift(mx);
      }
      if (ch == 0) backs[row] = scale == 0.f ? 1.f : fmaxf(ldexpf(fabsf(scale) * 1.44269504088896340736f, -n), 0x1p-126f);
      if (ch < HD / 8) {
        if constexpr (C16) {  // [tile][plane][32 dimensions][g][row][8 dimensions]
          half8v hi, lo;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float x = sign * (QP == 2 ? ldexpf(v[e], n) : v[e]);
            hi[e] = (_Float16)x;
            lo[e] = (_Float16)(x - (float)hi[e]);
          }
          half8v* o = reinterpret_cast<half8v*>(lds) + ((row >> 4) * QP * NJ + (ch >> 2)) * 64 + (ch & 3) * 16 + (row & 15);
          o[0] = hi;
          if constexpr (QP == 2) o[NJ * 64] = lo;
        } else {  // [tile][16 dimensions][g][row][4 dimensions]
#pragma unroll
          for (int i = 0; i < 2; ++i)
            *(reinterpret_cast<float4v*>(lds) + ((row >> 4) * NJ + (2 * ch + i) / 4) * 64 + ((2 * ch + i) & 3) * 16 + (row & 15)) =
                (float4v){sign * v[4 * i], sign * v[4 * i + 1], sign * v[4 * i + 2], sign * v[4 * i + 3]};
        }
      }
    }
  }
  __syncthreads();

  float4v o[NR][DL], l[NR];
  Ref ref[NR];
  float back[NR];
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    ref[n] = Ref{0.f, kA4NoKey};
    back[n] = backs[16 * n + c];
    l[n] = (float4v){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int d = 0; d < DL; ++d) o[n][d] = (float4v){0.f, 0.f, 0.f, 0.f};
  }
  // the operand of values' dimensions DL c + d
  auto value16 = [&](int d) __attribute__((always_inline)) {
    miq_u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t x = vr[i >> 1][2 * (i & 1)][d >> 1], y = vr[i >> 1][2 * (i & 1) + 1][d >> 1];
      w[i] = d & 1 ? highs(x, y) : lows(x, y);
    }
    return __builtin_bit_cast(half8v, w);
  };

  for (int it = 0; work; ++it) {
    const int next = blk + NW;
    const bool more = next < b1;
    // ---- scores: of tile n, lane (g, c) has the keys 4 g .. 4 g + 3 of each 16, row c ----
    float4v sc[NR][NT];
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
      for (int a = 0; a < NT; ++a) sc[n][a] = (float4v){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        if constexpr (C16) {
#pragma unroll
          for (int p = QP - 1; p >= 0; --p) {
            const half8v qv = reinterpret_cast<const half8v*>(lds)[((n * QP + p) * NJ + j) * 64 + lane];
#pragma unroll
            for (int a = 0; a < NT; ++a)
              sc[n][a] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8v, kr[a][j]), qv, sc[n][a], 0, 0, 0);
          }
        } else {
          const float4v qv = reinterpret_cast<const float4v*>(lds)[(n * NJ + j) * 64 + lane], kv = __builtin_bit_cast(float4v, kr[0][j]);
#pragma unroll
          for (int i = 0; i < 4; ++i) sc[n][0] = __builtin_amdgcn_mfma_f32_16x16x4f32(kv[i], qv[i], sc[n][0], 0, 0, 0);
        }
      }
    Block nxt = cur;
    if (more) {
      if (((it + 1) & 63) == 0) load_ids(next);
      nxt = block_at((it + 1) & 63);
      load_keys(next, nxt);
    }
    // ---- what is not attended to ----
    bool gone = false;
#pragma unroll
    for (int a = 0; a < NT; ++a) gone = gone || cur.id[a] < 0;
    const int k0 = blk * KB;
    const bool masked = gone || k0 + KB - 1 > first;  // wave-uniform
    bool odd = false;                                 // a value that is no finite number, in a block that not all rows attend to
    if (masked) {
      bool bad = false;
#pragma unroll
      for (int a = 0; a < NT; ++a)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int k = k0 + 16 * a + 4 * g + e;
          const bool none = cur.id[a] < 0 || k >= end;  // what lies there may be anything
#pragma unroll
          for (int n = 0; n < NR; ++n)
            if (none || k > lim[n]) sc[n][a][e] = -INFINITY;
#pragma unroll
          for (int i = 0; i < (C16 ? DL / 2 : DL); ++i) {
            vr[a][e][i] = none ? 0u : vr[a][e][i];
            const uint32_t v = vr[a][e][i];
            bad = bad || (C16 ? (v & 0x7C00u) == 0x7C00u || (v & 0x7C000000u) == 0x7C000000u : (v & 0x7F800000u) == 0x7F800000u);
          }
        }
      odd = __ballot(bad) != 0ull;
    }
    // ---- probabilities and sums ----
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      float mx = -INFINITY;
#pragma unroll
      for (int a = 0; a < NT; ++a)
#pragma unroll
        for (int e = 0; e < 4; ++e) mx = fmaxf(mx, sc[n][a][e]);
      mx = rows_max(mx);
      if (__ballot(ref_exponent(ref[n], mx, back[n]) > kA4UnitLog2 + kA4Slack)) {
        const float alpha = ref_raise(ref[n], mx, back[n]);
        l[n] *= alpha;
#pragma unroll
        for (int d = 0; d < DL; ++d) o[n][d] *= alpha;
      }
      float p[4 * NT];
#pragma unroll
      for (int e = 0; e < 4 * NT; ++e) p[e] = __builtin_amdgcn_exp2f(fmaf(sc[n][e >> 2][e & 3] - ref[n].shift, back[n], ref[n].neg));
      if constexpr (C16) {
        half8v ph[2];
        split_p(p, ph);
#pragma unroll
        for (int x = 1; x >= 0; --x) l[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones(), ph[x], l[n], 0, 0, 0);
        if (!odd) {
#pragma unroll
          for (int d = 0; d < DL; ++d) {
            const half8v v = value16(d);
#pragma unroll
            for (int x = 1; x >= 0; --x) o[n][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, ph[x], o[n][d], 0, 0, 0);
          }
        } else {  // row by row, with the values that it attends to alone
          for (int x = 0; x < 16; ++x) {
            const int own = __builtin_amdgcn_readlane(lim[n], x);
#pragma unroll
            for (int d = 0; d < DL; ++d) {
              half8v v = value16(d);
#pragma unroll
              for (int e = 0; e < 8; ++e)
                if (k0 + 16 * (e >> 2) + 4 * g + (e & 3) > own) v[e] = (_Float16)0.f;
              float4v t = o[n][d];
#pragma unroll
              for (int y = 1; y >= 0; --y) t = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, ph[y], t, 0, 0, 0);
              if (c == x) o[n][d] = t;
            }
          }
        }
      } else {
        l[n][0] += (p[0] + p[1]) + (p[2] + p[3]);  // of the lane's keys
        if (!odd) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int d = 0; d < DL; ++d) o[n][d] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(vr[0][e][d]), p[e], o[n][d], 0, 0, 0);
        } else {
          for (int x = 0; x < 16; ++x) {
            const int own = __builtin_amdgcn_readlane(lim[n], x);
#pragma unroll
            for (int d = 0; d < DL; ++d) {
              float4v t = o[n][d];
#pragma unroll
              for (int e = 0; e < 4; ++e)
                t = __builtin_amdgcn_mfma_f32_16x16x4f32(k0 + 4 * g + e > own ? 0.f : __uint_as_float(vr[0][e][d]), p[e], t, 0, 0, 0);
              if (c == x) o[n][d] = t;
            }
          }
        }
      }
    }
    if (!more) break;
    load_values(next, nxt);
    cur = nxt;
    blk = next;
  }

  // ---- the waves' sums, rescaled to their common reference, a tile at a time ----
  const int nw = max(1, min(NW, b1 - b0));  // waves that had keys (wave 0 always takes part)
  const int rows = min(16 * NR, R - r0);
  float* const os = reinterpret_cast<float*>(lds);  // [wave][row][HD + 4]
  float* const mypart = nparts > 1 ? parts + ((int64_t)blockIdx.x * 16 * NR) * (HD + 4) : nullptr;
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    const int nr = min(16, rows - 16 * n);
    if (nr <= 0) break;
    __syncthreads();
    if (wave < nw) {
      float sum = l[n][0];
      if constexpr (!C16) {
        sum += __shfl_xor(sum, 16);
        sum += __shfl_xor(sum, 32);
      }
      if (g == 0) {
        ms[wave][c] = ref_log2(ref[n], back[n]);
        ls[wave][c] = sum;
      }
      if (c < nr)
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int d = 0; d < DL; d += 4)
            *reinterpret_cast<float4v*>(&os[((size_t)wave * 16 + c) * (HD + 4) + DL * (4 * g + r) + d]) =
                (float4v){o[n][d][r], o[n][d + 1][r], o[n][d + 2][r], o[n][d + 3][r]};
    }
    __syncthreads();
    for (int x = tid; x < nr * (HD / 4); x += 64 * NW) {
      const int row = x / (HD / 4), d = 4 * (x % (HD / 4));
      float mx = ms[0][row];
      for (int w = 1; w < nw; ++w) mx = fmaxf(mx, ms[w][row]);
      const float rf = mx == -INFINITY ? 0.f : mx;
      float4v a = (float4v){0.f, 0.f, 0.f, 0.f};
      float sum = 0.f;
      for (int w = 0; w < nw; ++w) {
        const float f = __builtin_amdgcn_exp2f(ms[w][row] - rf);
        sum = fmaf(f, ls[w][row], sum);
        const float4v v = *reinterpret_cast<const float4v*>(&os[((size_t)w * 16 + row) * (HD + 4) + d]);
#pragma unroll
        for (int e = 0; e < 4; ++e) a[e] = fmaf(f, v[e], a[e]);
      }
      const int r = 16 * n + row;
      if (mypart) {
        put2(mypart + (int64_t)r * (HD + 4) + d, a[0], a[1]);
        put2(mypart + (int64_t)r * (HD + 4) + d + 2, a[2], a[3]);
        if (d == 0) put2(mypart + (int64_t)r * (HD + 4) + HD, mx, sum);
        continue;
      }
      const int t = (r0 + r) / rep;
      XT* orow = out + (((int64_t)s * T + t) * NH + h * rep + (r0 + r) % rep) * HD + d;
      const bool none = pos[t] < 0 || sum == 0.f;  // nothing to attend to: zeros
#pragma unroll
      for (int e = 0; e < 4; ++e) orow[e] = from_f32<XT>(none ? 0.f : a[e] / sum);
    }
  }
  if (nparts == 1) return;

  if (!last_slice(counters + ((int64_t)s * units + unit) * kPaCtrStride, nparts, &last)) return;
  // this sequence's parts lie `units` workgroups apart
  const float* p0 = parts + ((int64_t)(blockIdx.x - part * units) * 16 * NR) * (HD + 4);
  const int64_t step = (int64_t)units * 16 * NR * (HD + 4);
  for (int x = tid; x < rows * (HD / 2); x += 64 * NW) {
    const int r = x / (HD / 2), d = 2 * (x % (HD / 2));
    const float* pr = p0 + (int64_t)r * (HD + 4);
    float mx = -INFINITY, sum = 0.f, a0 = 0.f, a1 = 0.f;
    constexpr int U = 8;
    for (int k0 = 0; k0 < nparts; k0 += U) {
      uint64_t st[U], v[U];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const float* ps = pr + min(k0 + i, nparts - 1) * step;
        st[i] = get2(ps + HD);
        v[i] = get2(ps + d);
      }
      float mn = mx;
#pragma unroll
      for (int i = 0; i < U; ++i) mn = fmaxf(mn, __uint_as_float((uint32_t)st[i]));
      const float rf = mn == -INFINITY ? 0.f : mn, al = __builtin_amdgcn_exp2f(mx - rf);
      sum *= al;
      a0 *= al;
      a1 *= al;
      mx = mn;
#pragma unroll
      for (int i = 0; i < U; ++i)
        if (k0 + i < nparts) {
          const float f = __builtin_amdgcn_exp2f(__uint_as_float((uint32_t)st[i]) - rf);
          sum = fmaf(f, __uint_as_float((uint32_t)(st[i] >> 32)), sum);
          a0 = fmaf(f, __uint_as_float((uint32_t)v[i]), a0);
          a1 = fmaf(f, __uint_as_float((uint32_t)(v[i] >> 32)), a1);
        }
    }
    const int t = (r0 + r) / rep;
    XT* orow = out + (((int64_t)s * T + t) * NH + h * rep + (r0 + r) % rep) * HD + d;
    const bool none = pos[t] < 0 || sum == 0.f;
    orow[0] = from_f32<XT>(none ? 0.f : a0 / sum);
    orow[1] = from_f32<XT>(none ? 0.f : a1 / sum);
  }
}

// 16-row tiles of a workgroup: as many as the rows fill, of those whose sums the registers hold
static int pa_tiles(int64_t R, int HD) {
  const int most = HD == 64 ? 4 : HD == 128 ? 3 : 2;
  const int64_t n = (R + 15) / 16;
  return n >= most ? most : n == 3 && HD == 64 ? 4 : (int)n;
}
struct PagedPlan {
  int nr, tiles, target;
  int64_t grid, units;
};
static PagedPlan pa_plan(int S, int T, int NH, int NKV, int HD, int64_t cap, bool c16) {
  PagedPlan p;
  const int64_t R = (int64_t)T * (NH / NKV);
  p.nr = pa_tiles(R, HD);
  p.tiles = (int)((R + 16 * p.nr - 1) / (16 * p.nr));
  p.units = (int64_t)NKV * p.tiles;
  const int64_t step = (c16 ? 32 : 16) * kPaWaves * kPaMinSteps, most = (cap + step - 1) / step;  // parts of a full sequence
  const bool split = S * p.units <= kPaMaxSplit && most > 1;
  p.target = split ? kPaWorkgroups : 0;
  p.grid = S * p.units;
  if (split) p.grid = p.grid * most < p.grid + p.target ? p.grid * most : p.grid + p.target;
  return p;
}
static size_t pa_part_bytes(const PagedPlan& p, int HD) { return p.target ? (size_t)p.grid * 16 * p.nr * (HD + 4) * 4 : 0; }

}  // namespace miq

using namespace miq;

static int check_paged_attention(const char* what, int S, int T, int NH, int NKV, int HD, int num_pages, int page, int max_pages, int x_dtype,
                                 int cache_dtype) {
  MIQ_REQUIRE(S >= 0 && T >= 0 && NH > 0 && NKV > 0 && NH % NKV == 0 && NH <= (1 << 16) && HD > 0 && num_pages > 0 && max_pages >= 0, MIQ_ERR_INVALID,
              "%s: S=%d T=%d NH=%d NKV=%d HD=%d pages=%d of %d", what, S, T, NH, NKV, HD, max_pages, num_pages);
  MIQ_REQUIRE((x_dtype == MIQ_F32 || x_dtype == MIQ_F16) && (cache_dtype == MIQ_F32 || cache_dtype == MIQ_F16), MIQ_ERR_UNSUPPORTED,
              "%s: dtypes %d, %d", what, x_dtype, cache_dtype);
  if (int rc = check_paged(what, HD, page, num_pages, max_pages)) return rc;
  const int64_t R = (int64_t)T * (NH / NKV);
  MIQ_REQUIRE(R <= (1 << 30) && (int64_t)S * T <= (1ll << 31) && pa_plan(S, T ? T : 1, NH, NKV, HD, (int64_t)max_pages * page, true).grid < (1 << 22),
              MIQ_ERR_UNSUPPORTED, "%s: S=%d T=%d rows are past the grid", what, S, T);
  return MIQ_OK;
}

extern "C" int miq_paged_attention_workspace(int S, int T, int NH, int NKV, int HD, int page, int max_pages, int cache_dtype, size_t* bytes) {
  MIQ_REQUIRE(bytes, MIQ_ERR_INVALID, "paged_attention_workspace: null pointer");
  if (int rc = check_paged_attention("paged_attention_workspace", S, T, NH, NKV, HD, 1, page, max_pages, MIQ_F32, cache_dtype)) return rc;
  *bytes = 0;
  if (S == 0 || T == 0) return MIQ_OK;
  const size_t part = pa_part_bytes(pa_plan(S, T, NH, NKV, HD, (int64_t)max_pages * page, cache_dtype == MIQ_F16), HD);
  *bytes = part ? kCounterBytes + part : 0;
  return MIQ_OK;
}

extern "C" int miq_paged_attention(const void* q, int x_dtype, const void* cache, int cache_dtype, int num_pages, int page,
                                   const int32_t* positions, const int32_t* pages, int max_pages, void* out, int S, int T, int NH, int NKV,
                                   int HD, float scale, void* workspace, size_t ws_bytes, void* stream) {
  if (int rc = check_paged_attention("paged_attention", S, T, NH, NKV, HD, num_pages, page, max_pages, x_dtype, cache_dtype)) return rc;
  MIQ_REQUIRE(isfinite(scale * 1.44269504088896340736f), MIQ_ERR_INVALID, "paged_attention: scale=%g", (double)scale);
  if (S == 0 || T == 0) return MIQ_OK;
  MIQ_REQUIRE(q && cache && positions && (pages || max_pages == 0) && out, MIQ_ERR_INVALID, "paged_attention: null pointer");
  MIQ_REQUIRE(aligned(cache, 16), MIQ_ERR_ALIGN, "paged_attention: the cache must be 16-byte aligned");
  const bool c16 = cache_dtype == MIQ_F16, x32 = x_dtype == MIQ_F32;
  const PagedPlan p = pa_plan(S, T, NH, NKV, HD, (int64_t)max_pages * page, c16);
  const size_t part = pa_part_bytes(p, HD);
  MIQ_REQUIRE(!part || (workspace && ws_bytes >= kCounterBytes + part), MIQ_ERR_INVALID,
              "paged_attention: workspace of %zu bytes, %zu needed", workspace ? ws_bytes : (size_t)0, kCounterBytes + part);
  MIQ_REQUIRE(!part || aligned(workspace, 256), MIQ_ERR_ALIGN, "paged_attention: the workspace must be 256-byte aligned");
  const size_t io = (size_t)S * T * NH * HD * (x32 ? 4 : 2), nc = (size_t)num_pages * 2 * NKV * page * HD * (c16 ? 2 : 4);
  MIQ_REQUIRE(!share_bytes(out, io, q, io) && !share_bytes(out, io, cache, nc), MIQ_ERR_INVALID,
              "paged_attention: out must lie apart from q and the cache");
  const size_t lds = pa_lds(HD, p.nr, c16, x32);
  if (int rc = require_lds("paged_attention", lds + 4096)) return rc;
  int* counters = static_cast<int*>(workspace);
  float* parts = part ? reinterpret_cast<float*>(static_cast<char*>(workspace) + kCounterBytes) : nullptr;
  int lshift = 0;  // lanes of a sequence, where there are fewer of them than lanes
  while (lshift < 6 && (int64_t)S << (lshift + 1) <= 64) ++lshift;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  // one launch, but it writes to the workspace: not between the launches of another thread's call
  std::unique_lock<std::mutex> whole(stream_lock(st), std::defer_lock);
  if (part) whole.lock();
#define MIQ_PG(HDV, NRV, CT, XT)                                                                                                   \
  hipLaunchKernelGGL((paged_attention_kernel<HDV, NRV, CT, XT>), dim3((unsigned)p.grid), dim3(64 * kPaWaves), lds, st, static_cast<const XT*>(q), \
                     static_cast<const CT*>(cache), positions, pages, static_cast<XT*>(out), S, T, NH, NKV, p.tiles, num_pages,    \
                     __builtin_ctz((unsigned)page), max_pages, scale, lshift, p.target, counters, parts)
#define MIQ_PG_X(HDV, NRV, CT) \
  if (x32) { MIQ_PG(HDV, NRV, CT, float); } else { MIQ_PG(HDV, NRV, CT, __half); }
#define MIQ_PG_C(HDV, NRV) \
  if (c16) { MIQ_PG_X(HDV, NRV, __half) } else { MIQ_PG_X(HDV, NRV, float) }
  switch (HD * 8 + p.nr) {
    case 64 * 8 + 1: MIQ_PG_C(64, 1) break;
    case 64 * 8 + 2: MIQ_PG_C(64, 2) break;
    case 64 * 8 + 4: MIQ_PG_C(64, 4) break;
    case 128 * 8 + 1: MIQ_PG_C(128, 1) break;
    case 128 * 8 + 2: MIQ_PG_C(128, 2) break;
    case 128 * 8 + 3: MIQ_PG_C(128, 3) break;
    case 192 * 8 + 1: MIQ_PG_C(192, 1) break;
    case 192 * 8 + 2: MIQ_PG_C(192, 2) break;
    case 256 * 8 + 1: MIQ_PG_C(256, 1) break;
    case 256 * 8 + 2: MIQ_PG_C(256, 2) break;
    default: return fail(MIQ_ERR_UNSUPPORTED, "paged_attention: no kernel for HD=%d, %d tiles", HD, p.nr);
  }
#undef MIQ_PG_C
#undef MIQ_PG_X
#undef MIQ_PG
  return check_launch("paged_attention");
}
