// Grouped-query attention of a few new tokens of each of many sequences over a paged cache (paged.h): row (s, t) attends to
// the positions 0 .. positions[s][t] of its sequence, query head h to kv head h / (NH / NKV).
// scores = (q . k) scale; p = exp(s - max) / sum; out = sum p v. (`KVCache.attn`, `gqa_attention` of the reference, one
// sequence over a contiguous cache: webtorch/_core.py:1543-1596, 1319-1340.)
//
// A kv head's queries are rows r = t rep + hh, 16 to a tile, NR tiles to a workgroup, whose waves take a block of its keys in
// turn (32 of an fp16 cache, 16 of an fp32 one: 16 KB of keys and values at heads of 128). A wave multiplies
// S^T = K Q^T, then O^T = V^T P^T, on the matrix cores: the rows of K are operands as they lie in memory, the probabilities
// leave the first product in the lanes where the second wants them, and the values, loaded as rows of 16 bytes a lane, become
// operands by 16-bit permutations within the lane (fp16) or as they are (fp32, whose products take 4 keys at a time). No
// key or value passes through LDS; it holds q's operands.
// fp16 caches: K and V are exact, p is two fp16 numbers (22 bits), and so is q of fp32 rows. fp32 caches: fp32 products.
// Sums and softmax statistics are fp32.
//
// The work is split by the lengths, which are the device's: every workgroup adds them up and takes its part of a sequence, the
// parts as long as give the chip the workgroups that it holds, so that long sequences beside short ones fill it too. The last
// part of a sequence and head to arrive adds the parts, in their order. Calls that are not split look for their sequence in the same way.
//
// Bound and measured (us a replay over three states; a large copy moves 5.1 TB/s): memory for long caches, 64 sequences of 50 to 8000 positions,
// 32 / 8 heads of 128, fp16 199 (1.06 GB), one token behind 131000 positions 111 (537 MB); the chain of positions, pages, blocks and joins, and
// code fetched cold, for short ones, one token behind 700 positions of 14 / 2 heads of 64 9.0, behind 120 of 32 / 8 of 128 7.6; the fp32 matrix cores
// where an fp32 cache meets several tiles, 16 sequences of up to 5000, 5 tokens of 28 / 4 heads 70 (174 MB, a block of 16 keys and 48 rows 2.6 us a wave).
// Scratch, which the largest forms spill to (bytes a lane): heads of 128, three tiles, 8 waves, fp32 cache 148 (39 registers), fp16 24; heads of 192,
// one tile, 8 waves, fp32 84; heads of 256, two tiles, fp32 216 (96 registers), fp16 80 to 96.
#pragma once
#include <math.h>

#include "attention_parts.h"
#include "kv4.h"
#include "paged.h"

namespace miq {

// Blocks a wave of a part, at least, and of a sequence that is not split: joining costs as much (us a replay, one token: 700
// positions of 14 / 2 heads of 64 one part 9.3, two 12.7, three 11.6; 8000 of 32 / 8 heads of 128 at least 3 blocks 18.7, 2 17.2, 1 17.2)
constexpr int kPaMinSteps = 2, kPaWhole = 3;
constexpr int kPaCtrStride = 8;  // ints between arrival counters

template <typename CT> struct PagedKeys;  // keys of a block: 16-key tiles of it
template <> struct PagedKeys<__half> { static constexpr int kBlock = 32, kTiles = 2; };
template <> struct PagedKeys<float> { static constexpr int kBlock = 16, kTiles = 1; };

__host__ __device__ constexpr int pa_planes(bool c16, bool x32) { return c16 && x32 ? 2 : 1; }
// bytes of LDS: the operands of q, then (in their place) the waves' sums of one 16-row tile
__host__ __device__ constexpr size_t pa_lds(int HD, int NR, int NW, bool c16, bool x32) {
  const size_t q = (size_t)NR * 16 * HD * (c16 ? 2 * pa_planes(c16, x32) : 4), o = (size_t)NW * 16 * (HD + 4) * 4;
  return q > o ? q : o;
}

// Parts of slices pass by the XCD's own L2 (put2 and get2 of attention_parts.h), 16 bytes at a time
constexpr int kPastL2 = 16;  // sc1
__device__ __forceinline__ void put4(__amdgpu_buffer_rsrc_t r, int at, float4v v) {
  __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(miq_u32x4, v), r, at, 0, kPastL2);
}
__device__ __forceinline__ float4v get4(__amdgpu_buffer_rsrc_t r, int at) {
  return __builtin_bit_cast(float4v, __builtin_amdgcn_raw_buffer_load_b128(r, at, 0, kPastL2));
}

// 16-bit halves of two words: (low, low) or (high, high)
__device__ __forceinline__ uint32_t lows(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x05040100u); }
__device__ __forceinline__ uint32_t highs(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }

// Values (two fp16, one fp32) with infinities and NaN made finite; zeros where `none`
template <bool C16> __device__ __forceinline__ uint32_t finite(uint32_t v, bool none) {
  if constexpr (C16) {
    const half2v top = as_h2(none ? 0u : 0x7BFF7BFFu);  // 65504
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_min(__builtin_elementwise_max(as_h2(v), -top), top));
  } else {
    const float top = none ? 0.f : 3.402823466e38f;
    return __float_as_uint(fminf(fmaxf(__uint_as_float(v), -top), top));
  }
}
// the least and the greatest over a row of 16 lanes
template <int CTRL> __device__ __forceinline__ int dpp_int(int v) { return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xF, 0xF, false); }
__device__ __forceinline__ int row16_min(int v) {
  v = min(v, dpp_int<0xB1>(v));
  v = min(v, dpp_int<0x4E>(v));
  v = min(v, dpp_int<0x141>(v));
  return min(v, dpp_int<0x140>(v));
}
// the sum over lanes 0 .. l
__device__ __forceinline__ int wave_scan(int v) {
  v += dpp_int<0x111>(v);  // row_shr 1, 2, 4, 8
  v += dpp_int<0x112>(v);
  v += dpp_int<0x114>(v);
  v += dpp_int<0x118>(v);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // a row's last lane to the next row: rows 1 and 3
  return v + __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);  // lane 31 to rows 2 and 3
}

template <int HD, int NR, typename CT, typename XT, int NW>
__global__ __launch_bounds__(64 * NW) void paged_attention_kernel(
    const XT* __restrict__ q, const CT* __restrict__ cache, const int32_t* __restrict__ positions, const int32_t* __restrict__ pages,
    XT* __restrict__ out, int S, int T, int NH, int NKV, int tiles, int num_pages, int pshift, int max_pages, float scale, int lshift,
    int target, int fit, int* __restrict__ counters, float* __restrict__ parts) {
  constexpr bool C16 = sizeof(CT) == 2;
  constexpr int QP = pa_planes(C16, sizeof(XT) == 4);
  constexpr int KB = PagedKeys<CT>::kBlock, NT = PagedKeys<CT>::kTiles, DL = HD / 16;
  constexpr int NJ = C16 ? HD / 32 : HD / 16;  // 16-byte loads of a lane per 16 keys
  constexpr int NV = C16 ? DL / 2 : DL;        // words of a key's values in a lane
  extern __shared__ __align__(16) char lds[];
  __shared__ float backs[16 * NR], ms[NW][16], ls[NW][16];
  __shared__ int lims[16 * NR], last;
  __shared__ uint32_t nans[16 * NR][HD / 32];  // dimensions of a row that a value without a number reaches
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), c = lane & 15, g = lane >> 4;
  const int rep = NH / NKV, R = T * rep, units = NKV * tiles, unit = blockIdx.x % units, want = blockIdx.x / units;
  const int h = unit % NKV, r0 = unit / NKV * 16 * NR, cap = max_pages << pshift;

  // ---- which sequence, and which part of it: 64 >> lshift sequences at a time, 1 << lshift lanes each ----
  const int lane_s = lane >> lshift, sub = lane & ((1 << lshift) - 1), at_once = 64 >> lshift;
  auto keys_of = [&](int s0) __attribute__((always_inline)) {  // of sequence s0 + lane_s; steps of them, and parts, count at sub 0
    int n = 0;
    if (s0 + lane_s < S) {
      const int32_t* p = positions + (int64_t)(s0 + lane_s) * T;
#pragma unroll 1
      for (int t = sub; t < T; t += 1 << lshift) n = max(n, min(p[t], cap - 1) + 1);
    }
    if (T > 1)
#pragma unroll 1
      for (int d = 1; d < 1 << lshift; d *= 2) n = max(n, __shfl_xor(n, d));
    return sub == 0 ? n : 0;
  };
  auto steps_of = [&](int n) __attribute__((always_inline)) { return (n + KB * NW - 1) / (KB * NW); };
  int s = 0, part = 0, nparts = 1, len = 0;
  {
    int n = keys_of(0);
    float total = (float)steps_of(n);
#pragma unroll 1
    for (int s0 = at_once; s0 < S; s0 += at_once) total += (float)steps_of(keys_of(s0));
    // steps of a part, so that there are at most `target` of them and one more for each sequence and head (the sum may be off by 1e-6)
    const float least = ceilf(wave_sum(total) * (float)units / (float)target * 1.00001f);
    int per = target <= 0 || least > 1e9f ? 1 << 30 : max(kPaMinSteps, (int)least);
    auto parts_of = [&](int n, int s0) __attribute__((always_inline)) {
      const int steps = steps_of(n);
      return sub == 0 && s0 + lane_s < S ? (steps <= kPaWhole ? 1 : (steps + per - 1) / per) : 0;
    };
    // few sequences: no more parts than fit the chip at once, so that none waits for another's end
    if (fit)
#pragma unroll 1
      for (int i = 0; i < 8; ++i) {
        if (__builtin_amdgcn_readlane(wave_scan(parts_of(n, 0)), 63) * units <= target) break;
        per += max(1, per >> 3);
      }
    int before = 0;
#pragma unroll 1
    for (int s0 = 0;;) {
      const int parts = parts_of(n, s0), sum = wave_scan(parts);
      const uint64_t here = __ballot(parts > 0 && want < before + sum);
      if (here) {
        const int l = __builtin_ctzll(here);
        nparts = __builtin_amdgcn_readlane(parts, l);
        part = want - before - (__builtin_amdgcn_readlane(sum, l) - nparts);
        s = s0 + (l >> lshift);
        len = __builtin_amdgcn_readlane(n, l);
        break;
      }
      before += __builtin_amdgcn_readlane(sum, 63);
      s0 += at_once;
      if (s0 >= S) return;  // no part is left for this workgroup
      n = keys_of(s0);
    }
  }
  const int steps = steps_of(len);

  // ---- this workgroup's rows and keys ----
  const int32_t* pos = positions + (int64_t)s * T;
  // r / rep of this workgroup's rows: within 1 / (2 rep) of the quotient, off by less than that from any whole number
  const int t0 = r0 / rep, m0 = r0 % rep;
  const float each = 1.f / (float)rep;
  auto token = [&](int r) __attribute__((always_inline)) { return t0 + (int)(((float)(m0 + r - r0) + 0.5f) * each); };
  int lim[NR], first = 0x7FFFFFFF, end = 0;  // a row's last key (-1: none); the smallest of them; keys that any row attends to
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    const int r = r0 + 16 * n + c;
    lim[n] = r >= R ? -1 : T == 1 ? len - 1 : max(-1, min(pos[token(r)], cap - 1));
    if (lim[n] >= 0) first = min(first, lim[n]);
    end = max(end, lim[n] + 1);
  }
  first = uniform(row16_min(first));
  end = -uniform(row16_min(-end));
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
  alignas(16) uint32_t vr[NT][4][NV];  // stored to as vectors of 4 words, or 2
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

  // ---- q, LG lanes a row: on its way ahead of the first block, which would hold it up (16 sequences of 5 tokens 72 -> 70 us) ----
  constexpr int LG = HD == 64 ? 8 : HD == 128 ? 16 : 32, QI = (16 * NR * LG + 64 * NW - 1) / (64 * NW);
  const int ch = tid % LG;
  float qv[QI][8];
#pragma unroll
  for (int i = 0; i < QI; ++i) {
    const int row = tid / LG + i * (64 * NW / LG), r = r0 + row;
#pragma unroll
    for (int e = 0; e < 8; ++e) qv[i][e] = 0.f;
    if (row < 16 * NR && r < R && ch < HD / 8) {
      const int t = token(r);
      const XT* p = q + (((int64_t)s * T + t) * NH + h * rep + r - t * rep) * HD + 8 * ch;
#pragma unroll
      for (int e = 0; e < 8; ++e) qv[i][e] = to_f32<XT>(p[e]);
    }
  }

  int blk = b0 + wave;
  const bool work = blk < b1;  // wave-uniform
  Block cur;
  if (work) {
    load_ids(blk);
    cur = block_at(0);
    load_keys(blk, cur);
    load_values(blk, cur);
  }

  // ---- q as operands in LDS ----
  {
    const float sign = scale < 0.f ? -1.f : scale == 0.f ? 0.f : 1.f;
#pragma unroll
    for (int i = 0; i < QI; ++i) {
      const int row = tid / LG + i * (64 * NW / LG), r = r0 + row;
      if (row >= 16 * NR) break;
      float mx = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) mx = fmaxf(mx, fabsf(qv[i][e]));
      int n = 0;
      if constexpr (QP == 2) {
#pragma unroll
        for (int d = 1; d < LG; d *= 2) mx = fmaxf(mx, __shfl_xor(mx, d));
        n = row_shift(mx);
      }
      if (ch < HD / 32) nans[row][ch] = 0;
      if (ch == 0) {
        lims[row] = r >= R ? -1 : T == 1 ? len - 1 : min(pos[token(r)], cap - 1);
        backs[row] = scale == 0.f ? 1.f : fmaxf(ldexpf(fabsf(scale) * 1.44269504088896340736f, -n), 0x1p-126f);
      }
      if (ch < HD / 8) {
        if constexpr (C16) {  // [tile][plane][32 dimensions][g][row][8 dimensions]
          half8v hi, lo;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float x = sign * (QP == 2 ? ldexpf(qv[i][e], n) : qv[i][e]);
            hi[e] = (_Float16)x;
            lo[e] = (_Float16)(x - (float)hi[e]);
          }
          half8v* o = reinterpret_cast<half8v*>(lds) + ((row >> 4) * QP * NJ + (ch >> 2)) * 64 + (ch & 3) * 16 + (row & 15);
          o[0] = hi;
          if constexpr (QP == 2) o[NJ * 64] = lo;
        } else {  // [tile][16 dimensions][g][row][4 dimensions]
#pragma unroll
          for (int k = 0; k < 2; ++k)
            *(reinterpret_cast<float4v*>(lds) + ((row >> 4) * NJ + (2 * ch + k) / 4) * 64 + ((2 * ch + k) & 3) * 16 + (row & 15)) =
                (float4v){sign * qv[i][4 * k], sign * qv[i][4 * k + 1], sign * qv[i][4 * k + 2], sign * qv[i][4 * k + 3]};
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
    // q's operands are read again for every block where the registers do not hold them beside the sums
    if constexpr (NR > 1 || HD > 128) asm volatile("" ::: "memory");
    // ---- scores: of tile n, lane (g, c) has the keys 4 g .. 4 g + 3 of each 16, row c ----
    float4v sc[NR][NT];
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
      for (int a = 0; a < NT; ++a) sc[n][a] = (float4v){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int n = 0; n < NR; ++n) {
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
    if (masked) {
      // Keys behind the last one hold anything: their values become zeros. A value that is no finite number would make NaN of the
      // rows that do not attend to it too: it becomes finite, and the rows that do are marked.
      uint32_t odd = 0;
#pragma unroll
      for (int a = 0; a < NT; ++a)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int k = k0 + 16 * a + 4 * g + e;
          const bool none = cur.id[a] < 0 || k >= end;
#pragma unroll
          for (int n = 0; n < NR; ++n)
            if (none || k > lim[n]) sc[n][a][e] = -INFINITY;
          uint32_t diff = 0;
#pragma unroll
          for (int i = 0; i < NV; ++i) diff |= vr[a][e][i] ^ finite<C16>(vr[a][e][i], false);
          odd |= none ? 0u : diff;
        }
      if (__ballot(odd != 0)) {  // seldom: the words are read again, so that no register is held for it
#pragma unroll 1
        for (int x = 0; x < 4 * NT; ++x) {
          const int k = k0 + 16 * (x >> 2) + 4 * g + (x & 3), id = NT == 2 && x >= 4 ? cur.id[NT - 1] : cur.id[0];
          if (id < 0 || k >= end) continue;
          const uint32_t* w = reinterpret_cast<const uint32_t*>(mine + 2 * plane * id + plane + (int64_t)(k & ((1 << pshift) - 1)) * HD + DL * c);
#pragma unroll 1
          for (int i = 0; i < NV; ++i) {
            const uint32_t diff = w[i] ^ finite<C16>(w[i], false);
            const uint32_t bits = C16 ? (diff & 0xFFFFu ? 1u : 0u) | (diff >> 16 ? 2u : 0u) : diff ? 1u : 0u;
            const int d = DL * c + (C16 ? 2 : 1) * i;
            if (bits)
              for (int row = 0; row < 16 * NR; ++row)
                if (lims[row] >= k) atomicOr(&nans[row][d >> 5], bits << (d & 31));
          }
        }
      }
#pragma unroll
      for (int a = 0; a < NT; ++a)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const bool none = cur.id[a] < 0 || k0 + 16 * a + 4 * g + e >= end;
#pragma unroll
          for (int i = 0; i < NV; ++i) vr[a][e][i] = finite<C16>(vr[a][e][i], none);
        }
    }
    // ---- probabilities and sums ----
    half8v ph[C16 ? NR : 1][2];
    float p[C16 ? 1 : NR][4 * NT];
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
      float* pn = p[C16 ? 0 : n];
#pragma unroll
      for (int e = 0; e < 4 * NT; ++e) pn[e] = __builtin_amdgcn_exp2f(fmaf(sc[n][e >> 2][e & 3] - ref[n].shift, back[n], ref[n].neg));
      if constexpr (C16) {
        split_p(pn, ph[n]);
#pragma unroll
        for (int x = 1; x >= 0; --x) l[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones(), ph[n][x], l[n], 0, 0, 0);
      } else {
        l[n][0] += (pn[0] + pn[1]) + (pn[2] + pn[3]);  // of the lane's keys
      }
    }
    if constexpr (C16) {
#pragma unroll
      for (int d = 0; d < DL; ++d) {
        const half8v v = value16(d);
#pragma unroll
        for (int n = 0; n < NR; ++n)
#pragma unroll
          for (int x = 1; x >= 0; --x) o[n][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, ph[n][x], o[n][d], 0, 0, 0);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int d = 0; d < DL; ++d)
#pragma unroll
          for (int n = 0; n < NR; ++n) o[n][d] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(vr[0][e][d]), p[n][e], o[n][d], 0, 0, 0);
    }
    if (!more) break;
    load_values(next, nxt);
    cur = nxt;
    blk = next;
  }

  // ---- the waves' sums, rescaled to their common reference, a tile at a time ----
  const int rows = min(16 * NR, R - r0);
  float* const os = reinterpret_cast<float*>(lds);  // [wave][row][HD + 4]
  // a part: [row][HD + 4], the sums, the reference and the sum of probabilities
  constexpr int kPart = 16 * NR * (HD + 4) * 4;
  auto part_at = [&](int64_t i) __attribute__((always_inline)) {
    return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<char*>(parts) + i * kPart, 0, kPart, 0x00020000);
  };
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    const int nr = min(16, rows - 16 * n);
    if (nr <= 0) break;
    __syncthreads();
    float sum = l[n][0];  // a wave that had no keys leaves zeros
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
    __syncthreads();
    for (int x = tid; x < nr * (HD / 4); x += 64 * NW) {
      const int row = x / (HD / 4), d = 4 * (x % (HD / 4));
      float m[NW], sums[NW], mx = -INFINITY, sum = 0.f;
      float4v v[NW], a = (float4v){0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        m[w] = ms[w][row];
        sums[w] = ls[w][row];
        v[w] = *reinterpret_cast<const float4v*>(&os[((size_t)w * 16 + row) * (HD + 4) + d]);
      }
#pragma unroll
      for (int w = 0; w < NW; ++w) mx = fmaxf(mx, m[w]);
      const float rf = mx == -INFINITY ? 0.f : mx;
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float f = __builtin_amdgcn_exp2f(m[w] - rf);
        sum = fmaf(f, sums[w], sum);
#pragma unroll
        for (int e = 0; e < 4; ++e) a[e] = fmaf(f, v[w][e], a[e]);
      }
      const int r = 16 * n + row;
      const uint32_t nan = nans[r][d >> 5] >> (d & 31);
#pragma unroll
      for (int e = 0; e < 4; ++e) a[e] = nan >> e & 1 ? NAN : a[e];
      if (nparts > 1) {
        const __amdgpu_buffer_rsrc_t own = part_at(blockIdx.x);
        put4(own, (r * (HD + 4) + d) * 4, a);
        if (d == 0) put4(own, (r * (HD + 4) + HD) * 4, (float4v){mx, sum, 0.f, 0.f});
        continue;
      }
      const int t = token(r0 + r);
      XT* orow = out + (((int64_t)s * T + t) * NH + h * rep + r0 + r - t * rep) * HD + d;
      const bool none = lims[r] < 0 || sum == 0.f;  // nothing to attend to: zeros
#pragma unroll
      for (int e = 0; e < 4; ++e) orow[e] = from_f32<XT>(none ? 0.f : a[e] / sum);
    }
  }
  if (nparts == 1) return;

  if (!last_slice(counters + ((int64_t)s * units + unit) * kPaCtrStride, nparts, &last)) return;
  // this sequence's parts lie `units` workgroups apart
  const int64_t p0 = (int64_t)blockIdx.x - (int64_t)part * units;
  for (int x = tid; x < rows * (HD / 4); x += 64 * NW) {
    const int r = x / (HD / 4), d = 4 * (x % (HD / 4)), at = (r * (HD + 4) + d) * 4, stat = (r * (HD + 4) + HD) * 4;
    float mx = -INFINITY, sum = 0.f;
    float4v a = (float4v){0.f, 0.f, 0.f, 0.f};
    constexpr int U = 8;
    for (int k0 = 0; k0 < nparts; k0 += U) {
      float4v st[U], v[U];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        st[i] = (float4v){-INFINITY, 0.f, 0.f, 0.f};
        v[i] = (float4v){0.f, 0.f, 0.f, 0.f};
        if (k0 + i < nparts) {
          const __amdgpu_buffer_rsrc_t pr = part_at(p0 + (int64_t)(k0 + i) * units);
          st[i] = get4(pr, stat);
          v[i] = get4(pr, at);
        }
      }
      float mn = mx;
#pragma unroll
      for (int i = 0; i < U; ++i) mn = fmaxf(mn, st[i][0]);
      const float rf = mn == -INFINITY ? 0.f : mn, al = __builtin_amdgcn_exp2f(mx - rf);
      sum *= al;
      a *= al;
      mx = mn;
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const float f = __builtin_amdgcn_exp2f(st[i][0] - rf);
        sum = fmaf(f, st[i][1], sum);
#pragma unroll
        for (int e = 0; e < 4; ++e) a[e] = fmaf(f, v[i][e], a[e]);
      }
    }
    const int t = token(r0 + r);
    XT* orow = out + (((int64_t)s * T + t) * NH + h * rep + r0 + r - t * rep) * HD + d;
    const bool none = lims[r] < 0 || sum == 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) orow[e] = from_f32<XT>(none ? 0.f : a[e] / sum);
  }
}

struct PagedCall {
  const void *q, *cache;
  const int32_t *positions, *pages;
  void* out;
  int S, T, NH, NKV, HD, tiles, num_pages, page, max_pages, lshift, target, fit, nr, nw;
  float scale;
  bool x32;
  int* counters;
  float* parts;
  int64_t grid;
  size_t lds;
  hipStream_t st;
};
template <int HD, int NR, int NW, typename CT, typename XT> int launch_paged(const PagedCall& a) {
  hipLaunchKernelGGL((paged_attention_kernel<HD, NR, CT, XT, NW>), dim3((unsigned)a.grid), dim3(64 * NW), a.lds, a.st, static_cast<const XT*>(a.q),
                     static_cast<const CT*>(a.cache), a.positions, a.pages, static_cast<XT*>(a.out), a.S, a.T, a.NH, a.NKV, a.tiles, a.num_pages,
                     __builtin_ctz((unsigned)a.page), a.max_pages, a.scale, a.lshift, a.target, a.fit, a.counters, a.parts);
  return check_launch("paged_attention");
}
template <int HD, int NR, int NW, typename CT> int launch_paged_x(const PagedCall& a) {
  return a.x32 ? launch_paged<HD, NR, NW, CT, float>(a) : launch_paged<HD, NR, NW, CT, __half>(a);
}
template <typename CT> int paged_attention_cache(const PagedCall& a) {
  switch ((a.HD * 8 + a.nr) * 16 + a.nw) {
#define MIQ_PG(HDV, NRV, NWV) case (HDV * 8 + NRV) * 16 + NWV: return launch_paged_x<HDV, NRV, NWV, CT>(a)
    MIQ_PG(64, 1, 8);
    MIQ_PG(64, 2, 8);
    MIQ_PG(64, 4, 8);
    MIQ_PG(64, 1, 4);
    MIQ_PG(64, 2, 4);
    MIQ_PG(64, 4, 4);
    MIQ_PG(128, 1, 8);
    MIQ_PG(128, 2, 8);
    MIQ_PG(128, 3, 8);
    MIQ_PG(128, 1, 4);
    MIQ_PG(128, 2, 4);
    MIQ_PG(128, 3, 4);
    MIQ_PG(192, 1, 8);
    MIQ_PG(192, 1, 4);
    MIQ_PG(192, 2, 4);
    MIQ_PG(256, 1, 4);
    MIQ_PG(256, 2, 4);
#undef MIQ_PG
  }
  return fail(MIQ_ERR_UNSUPPORTED, "paged_attention: no kernel for HD=%d, %d tiles, %d waves", a.HD, a.nr, a.nw);
}
// the two caches' kernels (attention_paged.hip, attention_paged_f32.hip)
int paged_attention_f16(const PagedCall& a);
int paged_attention_f32(const PagedCall& a);

}  // namespace miq
