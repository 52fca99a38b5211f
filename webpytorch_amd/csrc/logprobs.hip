// Log probabilities of given tokens, with the entropy, the rank of the token and the top alternatives, in one
// read of the logits: per row x of V values,
//   lse = log sum exp x;  log p(id) = x[id] - lse;  entropy = lse - sum p x;  rank = #(x > x[id]);
//   alternatives: the k largest, of equal values the lower index first (NaN counts as -inf there).
// The greedy loop of the reference reads the row back to the host and picks there (`_head_argmax`,
// `_pick`: webtorch/llm.py:1309-1336).
//
// A workgroup takes a segment of a row, each of its waves every fourth chunk of 1024 values, which stay in
// registers while the next chunk's loads are in flight; the waves meet once, at the end, so that none waits for
// another in the loop. With the running maximum m and y = (x - m) log2 e, s0 = sum 2^y and s1 = sum 2^y y (fp32)
// give lse = m + ln 2 log2 s0 and entropy = ln 2 (log2 s0 - s1 / s0), in fp64.
//
// Alternatives go by 64-bit keys (the value in an order of integers, then the inverted index), all
// different, so that a result does not depend on any order of arrival. A wave keeps up to 128 keys in LDS; a
// chunk whose maximum is below the wave's k-th best is done with one ballot, otherwise the lanes' values
// above it are appended, and past 64 keys the wave keeps the best k: a key's place is the number of keys above
// it. The first chunk's bound: of 2^n >= k groups of lanes, the least of their maxima.
// Segments of one row meet in the workspace, at the last to arrive.
//
// Bound: memory for many rows (700 fp32 rows of 151936 with 20 alternatives: 425 MB in 95 us, 4.5 TB/s, where a
// large copy moves 4.8), round trips for few (one row 10.7 us: its 38 workgroups read 16 KB each, store their parts, and
// the last to arrive reads them). Measured and not kept: two chunks in flight (100 us), twice the segments (101),
// candidates appended value by value (118 us, one row 13.6: a row's only chunk pays for every line of code it runs).
#include <math.h>

#include "miq_common.h"

namespace miq {

constexpr int kLpThreads = 256, kLpWaves = kLpThreads / 64;
constexpr int kLpPer = 16;             // values of a lane and chunk
constexpr int kLpChunk = 64 * kLpPer;  // of a wave
constexpr int kLpMaxTop = 32;
constexpr int kLpList = 128;           // keys of a wave: at most 64, and 64 appended at a time
constexpr int kLpJoin = 1024;          // keys of all segments of a row
constexpr int kLpCtrStride = 32;       // ints between arrival counters: a 128-byte line each
constexpr float kLog2e = 1.44269504088896340736f;

__device__ __forceinline__ uint64_t lp_key(float v, uint32_t idx) {
  v = v != v ? -INFINITY : v + 0.f;  // -0 as 0
  const uint32_t b = __float_as_uint(v);
  return ((uint64_t)(b & 0x80000000u ? ~b : b | 0x80000000u) << 32) | (0xFFFFFFFFu - idx);
}
__device__ __forceinline__ float lp_value(uint64_t key) {
  const uint32_t b = (uint32_t)(key >> 32);
  return __uint_as_float(b & 0x80000000u ? b & 0x7FFFFFFFu : ~b);
}
__device__ __forceinline__ int lp_index(uint64_t key) { return (int)(0xFFFFFFFFu - (uint32_t)key); }

struct LpSum {
  float m, s0, s1;
};
__device__ __forceinline__ void lp_merge(LpSum& a, float m, float s0, float s1) {
  const float mn = fmaxf(a.m, m);
  if (mn == -INFINITY) {  // nothing yet, but a NaN stays
    a.s0 += s0;
    return;
  }
  const float da = fmaxf((a.m - mn) * kLog2e, -1e4f), db = fmaxf((m - mn) * kLog2e, -1e4f);
  const float fa = __builtin_amdgcn_exp2f(da), fb = __builtin_amdgcn_exp2f(db);
  a.s1 = fa * fmaf(a.s0, da, a.s1) + fb * fmaf(s0, db, s1);
  a.s0 = fa * a.s0 + fb * s0;
  a.m = mn;
}
// over the wave: one exponential a lane, against the wave's maximum
__device__ __forceinline__ void lp_wave(LpSum& a, int& above) {
  const float m = wave_max(a.m);
  if (m == -INFINITY) {
    a.s0 = wave_sum(a.s0);
  } else {
    const float d = fmaxf((a.m - m) * kLog2e, -1e4f), f = __builtin_amdgcn_exp2f(d);
    a.s1 = wave_sum(f * fmaf(a.s0, d, a.s1));
    a.s0 = wave_sum(f * a.s0);
    a.m = m;
  }
  int n = above;
  n += __builtin_amdgcn_update_dpp(0, n, 0xB1, 0xF, 0xF, false);
  n += __builtin_amdgcn_update_dpp(0, n, 0x4E, 0xF, 0xF, false);
  n += __builtin_amdgcn_update_dpp(0, n, 0x141, 0xF, 0xF, false);
  n += __builtin_amdgcn_update_dpp(0, n, 0x140, 0xF, 0xF, false);
  above = (__builtin_amdgcn_readlane(n, 0) + __builtin_amdgcn_readlane(n, 16)) +
          (__builtin_amdgcn_readlane(n, 32) + __builtin_amdgcn_readlane(n, 48));
}
__device__ __forceinline__ uint64_t shfl_xor64(uint64_t v, int s) {
  return ((uint64_t)(uint32_t)__shfl_xor((int)(v >> 32), s) << 32) | (uint32_t)__shfl_xor((int)(uint32_t)v, s);
}

template <typename T> struct LpLoad;
template <> struct LpLoad<float> {
  static constexpr int VEC = 4;
  static __device__ __forceinline__ void get(const float* p, float* v) {
    const float4 t = *reinterpret_cast<const float4*>(p);
    v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
  }
};
template <> struct LpLoad<__half> {
  static constexpr int VEC = 8;
  static __device__ __forceinline__ void get(const __half* p, float* v) { load8(p, v); }
};

// One wave: the k largest of the n <= 128 keys of list, sorted, at its start (zeros where n < k).
__device__ __forceinline__ void lp_keep(uint64_t* list, int n, int k) {
  const int lane = threadIdx.x & 63;
  const uint64_t a = lane < n ? list[lane] : 0, b = lane + 64 < n ? list[lane + 64] : 0;
  if (lane >= n) list[lane] = 0;
  if (lane + 64 >= n) list[lane + 64] = 0;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  int ra = 0, rb = 0;
  for (int j = 0; j < n; j += 8) {
    uint64_t c[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = list[j + i];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      ra += c[i] > a;
      rb += c[i] > b;
    }
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  if (a && ra < k) list[ra] = a;
  if (b && rb < k) list[rb] = b;
  if (lane >= n && lane < k) list[lane] = 0;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
}

template <typename T>
__global__ __launch_bounds__(kLpThreads) void logprobs_kernel(
    const T* __restrict__ logits, size_t ld, const int32_t* __restrict__ ids, int V, int k, float* __restrict__ lp_out,
    float* __restrict__ ent_out, int32_t* __restrict__ rank_out, int32_t* __restrict__ top_ids, float* __restrict__ top_lp,
    const int32_t* __restrict__ state, int out_rows, int* __restrict__ counters, uint64_t* __restrict__ parts) {
  constexpr int VEC = LpLoad<T>::VEC, U = kLpPer / VEC;
  __shared__ __align__(16) uint64_t lists[kLpWaves][kLpList], pool[kLpWaves * kLpChunk / 2];
  float* vals = reinterpret_cast<float*>(pool) + uniform(threadIdx.x >> 6) * kLpChunk;  // a wave's chunk
  uint64_t* join = pool;  // later: the keys of all segments
  static_assert(kLpWaves * kLpChunk / 2 >= kLpJoin, "the join's keys fit");
  __shared__ LpSum sums[kLpWaves];
  __shared__ uint64_t bounds[kLpWaves];
  __shared__ int cnts[kLpWaves], njoin, last;
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const int t = blockIdx.y, seg = blockIdx.x, segs = gridDim.x;
  const T* x = logits + (size_t)t * ld;
  const int id = ids[t];
  const bool given = id >= 0 && id < V;
  uint64_t* list = lists[wave];
  if (tid == 0) njoin = 0;

  // vectors of 16 bytes from the first aligned value on, whole workgroup chunks for each segment (the last
  // may have fewer); the values before and after them are one more value of segment 0's first lanes
  const int mis = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
  const int head = min(V, mis ? VEC - mis : 0), nvec = (V - head) / VEC, ends = V - nvec * VEC;
  constexpr int step = 64 * U;  // vectors of a wave's chunk
  const int per = (nvec + segs - 1) / segs, v0 = min(nvec, seg * per), v1 = min(nvec, v0 + per);
  const T* xv = x + head;

  LpSum a = {-INFINITY, 0.f, 0.f};
  int above = 0, n = 0;
  uint64_t kth = 0;       // keys that are not above it are not among the best k
  float bv = -INFINITY;   // nor values below it
  float nxt[kLpPer];
  auto load = [&](int vb) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int vi = vb + u * 64 + lane;
      if (vi < v1) LpLoad<T>::get(xv + (size_t)vi * VEC, &nxt[u * VEC]);
      else
#pragma unroll
        for (int e = 0; e < VEC; ++e) nxt[u * VEC + e] = -INFINITY;
    }
  };
  load(v0 + wave * step);
  const float xt = given ? to_f32<T>(x[id]) : INFINITY;  // behind the chunk's loads
  bool first = true;
  for (int vb = v0 + wave * step; vb < v1 || first; vb += kLpWaves * step) {
    float v[kLpPer];
#pragma unroll
    for (int e = 0; e < kLpPer; ++e) v[e] = nxt[e];
    const bool ext = first && seg == 0 && tid < ends;
    const int xi = tid < head ? tid : nvec * VEC + tid;
    const float xe = ext ? to_f32<T>(x[xi]) : -INFINITY;
    if (vb + kLpWaves * step < v1) load(vb + kLpWaves * step);

    // ---- sums ----
    float cm = xe;  // the chunk's maximum
#pragma unroll
    for (int e = 0; e < kLpPer; ++e) cm = fmaxf(cm, v[e]);
    const float mx = fmaxf(a.m, cm);
    if (mx > a.m) {
      const float d = fmaxf((a.m - mx) * kLog2e, -1e4f), f = __builtin_amdgcn_exp2f(d);
      a.s1 = f * fmaf(a.s0, d, a.s1);
      a.s0 = f * a.s0;
      a.m = mx;
    }
    auto add = [&](float y) __attribute__((always_inline)) {
      const float d = (y - a.m) * kLog2e;
      const float e = __builtin_amdgcn_exp2f(d);
      a.s0 += e;  // NaN comes in here
      a.s1 = fmaf(e, fmaxf(d, -1e4f), a.s1);
      above += y > xt;
    };
    if (mx > -INFINITY) {
#pragma unroll
      for (int e = 0; e < kLpPer; ++e) add(v[e]);
      if (ext) add(xe);
    } else {  // nothing but -inf and NaN so far
#pragma unroll
      for (int e = 0; e < kLpPer; ++e) a.s0 += v[e] != v[e] ? v[e] : 0.f;
      a.s0 += xe != xe ? xe : 0.f;
    }

    // ---- alternatives ----
    if (k) {
      if (first) {
        float g = cm;
        for (int s = 1; s * k <= 32; s <<= 1) g = fmaxf(g, __shfl_xor(g, s));  // groups of the largest 2^n <= 64 / k lanes
        bv = -wave_max(-g);
      }
      if (__ballot(cm >= bv)) {
        // a bit for each value of the lane that may come in (bit kLpPer: the row's unaligned ends); one of every lane
        // a round, fetched through LDS, so that the code is short: a row's only chunk pays for each line of it
        uint32_t bits = ext && !(xe < bv) ? 1u << kLpPer : 0u;
#pragma unroll
        for (int e = 0; e < kLpPer; ++e)
          if (vb + (e / VEC) * 64 + lane < v1 && !(v[e] < bv)) bits |= 1u << e;
#pragma unroll
        for (int e = 0; e < kLpPer; e += 4)
          *reinterpret_cast<float4*>(&vals[(e * 16 + lane) * 4]) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        while (__ballot(bits != 0)) {
          const int e = __ffs(bits) - 1;
          uint64_t key = 0;
          if (bits) {
            const bool end = e == kLpPer;
            const float y = end ? xe : vals[((e & ~3) * 16 + lane) * 4 + (e & 3)];
            key = lp_key(y, (uint32_t)(end ? xi : head + (vb + (e / VEC) * 64 + lane) * VEC + e % VEC));
            bits &= bits - 1;
          }
          const uint64_t mask = __ballot(key > kth);
          if (key > kth) list[n + __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0))] = key;
          n += __popcll(mask);
          if (n > kLpList - 64) {
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            lp_keep(list, n, k);
            n = k;
            kth = list[k - 1];
            bv = lp_value(kth);
          }
        }
      }
    }
    first = false;
  }

  // ---- the lanes' and the waves' parts ----
  lp_wave(a, above);
  if (k) lp_keep(list, n, k);
  if (lane == 0) {
    sums[wave] = a;
    cnts[wave] = above;
  }
  __syncthreads();
  if (wave == 0 && k) {  // 4 k <= 128 keys
    uint64_t key[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (lane + 64 * i < kLpWaves * k) key[i] = lists[(lane + 64 * i) / k][(lane + 64 * i) % k];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (int i = 0; i < 2; ++i) list[lane + 64 * i] = key[i];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    lp_keep(list, kLpWaves * k, k);
  }
  a = sums[0];
  above = cnts[0];
  for (int w = 1; w < kLpWaves; ++w) {
    lp_merge(a, sums[w].m, sums[w].s0, sums[w].s1);
    above += cnts[w];
  }

  if (segs > 1) {
    // a segment's part: (m, s0), (s1, above), keys
    const size_t words = 2 + (size_t)k;
    uint64_t* part = parts + ((size_t)t * segs + seg) * words;
    auto put = [](uint64_t* p, uint64_t v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
    auto get = [](const uint64_t* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
    if (wave == 0) {  // it alone has the keys, and counts itself in
      if (lane == 0) {
        put(part, (uint64_t)__float_as_uint(a.m) | ((uint64_t)__float_as_uint(a.s0) << 32));
        put(part + 1, (uint64_t)__float_as_uint(a.s1) | ((uint64_t)(uint32_t)above << 32));
      }
      if (lane < k) put(part + 2 + lane, list[lane]);
      parts_stored();
      if (lane == 0) {
        int* ctr = counters + (size_t)t * kLpCtrStride;
        last = __hip_atomic_fetch_add(ctr, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == segs - 1;
        if (last) __hip_atomic_store(ctr, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // re-armed
      }
    }
    __syncthreads();
    if (!last) return;
    const uint64_t* p0 = parts + (size_t)t * segs * words;
    // every load at once: the sums and the k-th key of segment tid, and a share of all keys
    constexpr int KU = kLpJoin / kLpThreads;
    uint64_t w0 = 0, w1 = 0, lb = 0, key[KU];
    const bool mine = tid < segs;
    if (mine) {
      const uint64_t* p = p0 + (size_t)tid * words;
      w0 = get(p);
      w1 = get(p + 1);
      if (k) lb = get(p + 1 + k);
    }
#pragma unroll
    for (int i = 0; i < KU; ++i) {
      const int q = tid + i * kLpThreads;
      key[i] = 0;
      if (q < segs * k) key[i] = get(p0 + (size_t)(q / k) * words + 2 + q % k);
    }
    a = {-INFINITY, 0.f, 0.f};
    above = 0;
    if (mine) {
      a = {__uint_as_float((uint32_t)w0), __uint_as_float((uint32_t)(w0 >> 32)), __uint_as_float((uint32_t)w1)};
      above = (int)(w1 >> 32);
    }
    // no key below the best of the segments' k-th keys is among the row's best k
    lp_wave(a, above);
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
      const uint64_t o = shfl_xor64(lb, s);
      lb = o > lb ? o : lb;
    }
    __syncthreads();  // sums and cnts are read above
    if (lane == 0) {
      sums[wave] = a;
      cnts[wave] = above;
      bounds[wave] = lb;
    }
    __syncthreads();
    a = sums[0];
    above = cnts[0];
    lb = bounds[0];
    for (int w = 1; w < kLpWaves; ++w) {
      lp_merge(a, sums[w].m, sums[w].s0, sums[w].s1);
      above += cnts[w];
      lb = bounds[w] > lb ? bounds[w] : lb;
    }
    if (k) {
#pragma unroll
      for (int i = 0; i < KU; ++i)
        if (key[i] && key[i] >= lb) join[atomicAdd(&njoin, 1)] = key[i];
      __syncthreads();
      const int nj = njoin;
      for (int i = tid; i < nj; i += kLpThreads) {
        const uint64_t me = join[i];
        int place = 0;
#pragma unroll 8
        for (int j = 0; j < nj; ++j) place += join[j] > me;
        if (place < k) lists[0][place] = me;
      }
    }
  }
  __syncthreads();

  // ---- the row's results ----
  int row = t;
  if (state) {  // the token just generated
    row = state[1] - 1;
    if (row < 0) return;
  }
  if (row >= out_rows) return;
  const bool none = a.m == -INFINITY && a.s0 == 0.f;  // every value -inf
  constexpr double kLn2 = 0.69314718055994530942;
  const double lz = log2((double)a.s0) * kLn2;  // lse = m + lz
  auto logp = [&](float y) {
    return none || y == -INFINITY ? (a.s0 != a.s0 ? NAN : -INFINITY) : (float)(((double)y - (double)a.m) - lz);
  };
  if (tid == 0) {
    if (lp_out) lp_out[row] = given ? logp(xt) : 0.f;
    if (ent_out) ent_out[row] = none ? 0.f : (float)(lz - (double)a.s1 / (double)a.s0 * kLn2);
    if (rank_out) rank_out[row] = given ? above : -1;
  }
  if (tid < k) {
    const uint64_t key = lists[0][tid];
    if (top_ids) top_ids[(size_t)row * k + tid] = lp_index(key);
    if (top_lp) top_lp[(size_t)row * k + tid] = logp(lp_value(key));
  }
}

// Segments of a row: as many as give every CU two workgroups, of at least a chunk a wave each, their keys
// within the buffer of the last one, and a thread of it for each.
static int lp_segments(int T, int V, int k) {
  const int most = (V + kLpWaves * kLpChunk - 1) / (kLpWaves * kLpChunk);
  int s = T >= 2 * kCUs ? 1 : (2 * kCUs + T - 1) / T;
  if (s > most) s = most;
  if (s > kLpThreads) s = kLpThreads;
  if (k && s > kLpJoin / k) s = kLpJoin / k;
  return s < 1 ? 1 : s;
}
static size_t lp_part_bytes(int T, int V, int k) {
  const int s = lp_segments(T, V, k);
  return s > 1 ? (size_t)T * s * (2 + k) * 8 : 0;
}

}  // namespace miq

using namespace miq;

static int check_logprobs(const char* what, int T, int V, int k) {
  MIQ_REQUIRE(T >= 0 && V > 0 && V <= (1 << 30) && k >= 0 && k <= V, MIQ_ERR_INVALID, "%s: T=%d V=%d k=%d", what, T, V, k);
  MIQ_REQUIRE(k <= kLpMaxTop, MIQ_ERR_UNSUPPORTED, "%s: k=%d alternatives (at most %d)", what, k, kLpMaxTop);
  MIQ_REQUIRE(T <= 65535, MIQ_ERR_UNSUPPORTED, "%s: T=%d rows (at most 65535)", what, T);
  return MIQ_OK;
}

extern "C" int miq_token_logprobs_workspace(int T, int V, int k, size_t* bytes) {
  MIQ_REQUIRE(bytes, MIQ_ERR_INVALID, "token_logprobs_workspace: null pointer");
  if (int rc = check_logprobs("token_logprobs_workspace", T, V, k)) return rc;
  const size_t part = T ? lp_part_bytes(T, V, k) : 0;
  *bytes = part ? kCounterBytes + part : 0;
  return MIQ_OK;
}

extern "C" int miq_token_logprobs(const void* logits, int x_dtype, int64_t ld, const int32_t* ids, int T, int V, int k,
                                  float* logprobs, float* entropy, int32_t* ranks, int32_t* top_ids, float* top_logprobs,
                                  const int32_t* state, int out_rows, void* workspace, size_t ws_bytes, void* stream) {
  if (int rc = check_logprobs("token_logprobs", T, V, k)) return rc;
  MIQ_REQUIRE(x_dtype == MIQ_F32 || x_dtype == MIQ_F16, MIQ_ERR_UNSUPPORTED, "token_logprobs: logits dtype %d", x_dtype);
  MIQ_REQUIRE(ld >= V && out_rows >= 0 && (!state || T <= 1), MIQ_ERR_INVALID,
              "token_logprobs: rows %lld apart hold V=%d values, out_rows=%d; a state goes with one row (T=%d)", (long long)ld, V,
              out_rows, T);
  if (T == 0) return MIQ_OK;
  MIQ_REQUIRE(logits && ids, MIQ_ERR_INVALID, "token_logprobs: null pointer");
  MIQ_REQUIRE(aligned(logits, x_dtype == MIQ_F32 ? 4 : 2), MIQ_ERR_ALIGN, "token_logprobs: logits must be aligned to their type");
  const int segs = lp_segments(T, V, k);
  const size_t part = lp_part_bytes(T, V, k);
  MIQ_REQUIRE(!part || (workspace && ws_bytes >= kCounterBytes + part), MIQ_ERR_INVALID,
              "token_logprobs: workspace of %zu bytes, %zu needed", workspace ? ws_bytes : (size_t)0, kCounterBytes + part);
  MIQ_REQUIRE(!part || aligned(workspace, 256), MIQ_ERR_ALIGN, "token_logprobs: the workspace must be 256-byte aligned");
  int* counters = static_cast<int*>(workspace);
  uint64_t* parts = part ? reinterpret_cast<uint64_t*>(static_cast<char*>(workspace) + kCounterBytes) : nullptr;
  const dim3 grid((unsigned)segs, (unsigned)T), block(kLpThreads);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  // one launch, but it writes to the workspace: not between the launches of another thread's call
  std::unique_lock<std::mutex> whole(stream_lock(st), std::defer_lock);
  if (part) whole.lock();
  if (x_dtype == MIQ_F32)
    hipLaunchKernelGGL(logprobs_kernel<float>, grid, block, 0, st, static_cast<const float*>(logits), (size_t)ld, ids, V, k,
                       logprobs, entropy, ranks, top_ids, top_logprobs, state, out_rows, counters, parts);
  else
    hipLaunchKernelGGL(logprobs_kernel<__half>, grid, block, 0, st, static_cast<const __half*>(logits), (size_t)ld, ids, V, k,
                       logprobs, entropy, ranks, top_ids, top_logprobs, state, out_rows, counters, parts);
  return check_launch("token_logprobs");
}
