// Log probabilities of given tokens, with the entropy, the rank of the token and the top alternatives, in one
// read of the logits: per row x of V values,
//   lse = log sum exp x;  log p(id) = x[id] - lse;  entropy = lse - sum p x;  rank = #(x > x[id]);
//   alternatives: the k largest, of equal values the lower index first (NaN counts as -inf there).
// The greedy loop of the reference reads the row back to the host and picks there (`_head_argmax`,
// `_pick`: webtorch/llm.py:1309-1336).
//
// A workgroup takes a segment of a row in chunks that stay in registers, and every thread keeps a running
// maximum m with s0 = sum exp(x - m) and s1 = sum exp(x - m) (x - m) (fp32; the threads' sums meet in fp64):
// entropy = log s0 - s1 / s0. Alternatives go by 64-bit keys (the value in an order of integers, then the
// inverted index), all different, so that a result does not depend on the order of arrival: a chunk's
// keys above the segment's k-th best so far are collected in LDS, and a key's place is the number of keys
// above it. The first chunk has no k-th best yet: of 32 groups of threads the least of their largest keys bounds
// it from below. Segments of one row meet in the workspace, at the last to arrive.
#include <math.h>

#include "miq_common.h"

namespace miq {

constexpr int kLpThreads = 256, kLpWaves = kLpThreads / 64;
constexpr int kLpPer = 16;                        // values of a thread and chunk
constexpr int kLpChunk = kLpThreads * kLpPer;
constexpr int kLpMaxTop = 32;
constexpr int kLpGroups = 32;                     // >= kLpMaxTop groups of 8 threads
constexpr int kLpCand = kLpChunk + 2 * kLpMaxTop; // a chunk's keys, its row's unaligned ends, and those kept
constexpr int kLpCtrStride = 32;                  // ints between arrival counters: a 128-byte line each
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

// running maximum and sums
struct LpSum {
  float m, s0, s1;
};
__device__ __forceinline__ void lp_merge(LpSum& a, float m, float s0, float s1) {
  const float mn = fmaxf(a.m, m);
  if (mn == -INFINITY) {  // nothing yet, but a NaN stays
    a.s0 += s0;
    return;
  }
  const float da = fmaxf(a.m - mn, -1e4f), db = fmaxf(m - mn, -1e4f);
  const float fa = __builtin_amdgcn_exp2f(da * kLog2e), fb = __builtin_amdgcn_exp2f(db * kLog2e);
  a.s1 = fa * fmaf(a.s0, da, a.s1) + fb * fmaf(s0, db, s1);
  a.s0 = fa * a.s0 + fb * s0;
  a.m = mn;
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

// The k largest of the n keys in cand, sorted, to best (k <= n): a key's place is the number above it.
__device__ __forceinline__ void lp_select(const uint64_t* cand, int n, int k, uint64_t* best) {
  for (int i = threadIdx.x; i < n; i += kLpThreads) {
    const uint64_t key = cand[i];
    int above = 0;
    for (int j = 0; j < n; ++j) above += cand[j] > key;
    if (above < k) best[above] = key;
  }
}

template <typename T>
__global__ __launch_bounds__(kLpThreads) void logprobs_kernel(
    const T* __restrict__ logits, size_t ld, const int32_t* __restrict__ ids, int V, int k, float* __restrict__ lp_out,
    float* __restrict__ ent_out, int32_t* __restrict__ rank_out, int32_t* __restrict__ top_ids, float* __restrict__ top_lp,
    const int32_t* __restrict__ state, int out_rows, int* __restrict__ counters, uint64_t* __restrict__ parts) {
  constexpr int VEC = LpLoad<T>::VEC, U = kLpPer / VEC;
  __shared__ uint64_t cand[kLpCand], best[kLpMaxTop], gbest[kLpGroups];
  __shared__ LpSum sums[kLpWaves];
  __shared__ int cnts[kLpWaves], ncand, last;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int t = blockIdx.y, seg = blockIdx.x, segs = gridDim.x;
  const T* x = logits + (size_t)t * ld;
  const int id = ids[t];
  const bool given = id >= 0 && id < V;
  const float xt = given ? to_f32<T>(x[id]) : INFINITY;

  // vectors of 16 bytes from the first aligned value on, the same number for each segment (the last may
  // have fewer); the values before and after them are one more value of segment 0's first threads
  const int mis = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
  const int head = min(V, mis ? VEC - mis : 0), nvec = (V - head) / VEC, ends = V - nvec * VEC;
  const int per = (nvec + segs - 1) / segs, v0 = min(nvec, seg * per), v1 = min(nvec, v0 + per);
  const T* xv = x + head;

  LpSum a = {-INFINITY, 0.f, 0.f};
  int above = 0, kept = 0;
  uint64_t bound = 0;  // keys below it are not among the best k
  if (tid == 0) ncand = 0;
  float nxt[kLpPer];
  auto load = [&](int vb) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int vi = vb + u * kLpThreads + tid;
      if (vi < v1) LpLoad<T>::get(xv + (size_t)vi * VEC, &nxt[u * VEC]);
      else
#pragma unroll
        for (int e = 0; e < VEC; ++e) nxt[u * VEC + e] = -INFINITY;
    }
  };
  load(v0);
  bool first = true;
  for (int vb = v0; vb < v1 || first; vb += U * kLpThreads) {
    float v[kLpPer];
#pragma unroll
    for (int e = 0; e < kLpPer; ++e) v[e] = nxt[e];
    const bool ext = first && seg == 0 && tid < ends;
    const int xi = tid < head ? tid : head + nvec * VEC + (tid - head);
    const float xe = ext ? to_f32<T>(x[xi]) : -INFINITY;
    if (vb + U * kLpThreads < v1) load(vb + U * kLpThreads);

    // ---- sums ----
    float cm = xe;  // the chunk's maximum
#pragma unroll
    for (int e = 0; e < kLpPer; ++e) cm = fmaxf(cm, v[e]);
    const float mx = fmaxf(a.m, cm);
    if (mx > a.m) {
      const float d = fmaxf(a.m - mx, -1e4f), f = __builtin_amdgcn_exp2f(d * kLog2e);
      a.s1 = f * fmaf(a.s0, d, a.s1);
      a.s0 = f * a.s0;
      a.m = mx;
    }
    auto add = [&](float y) __attribute__((always_inline)) {
      float d = y - a.m;
      d = d < -1e4f ? -1e4f : d;  // exp is 0 there; a NaN stays
      const float e = __builtin_amdgcn_exp2f(d * kLog2e);
      a.s0 += e;
      a.s1 = fmaf(e, d, a.s1);
      above += y > xt;
    };
    if (mx > -INFINITY) {
#pragma unroll
      for (int e = 0; e < kLpPer; ++e) add(v[e]);
      add(xe);
    } else {  // nothing but -inf and NaN so far
#pragma unroll
      for (int e = 0; e < kLpPer; ++e) a.s0 += v[e] != v[e] ? v[e] : 0.f;
      a.s0 += xe != xe ? xe : 0.f;
    }

    // ---- alternatives ----
    if (k) {
      auto index = [&](int e) __attribute__((always_inline)) {
        return (uint32_t)(head + (vb + (e / VEC) * kLpThreads + tid) * VEC + e % VEC);
      };
      auto valid = [&](int e) __attribute__((always_inline)) { return vb + (e / VEC) * kLpThreads + tid < v1; };
      if (first) {
        uint64_t top = ext ? lp_key(xe, xi) : 0;
#pragma unroll
        for (int e = 0; e < kLpPer; ++e)
          if (valid(e)) {
            const uint64_t key = lp_key(v[e], index(e));
            top = key > top ? key : top;
          }
#pragma unroll
        for (int s = 1; s < 8; s <<= 1) {
          const uint64_t o = ((uint64_t)(uint32_t)__shfl_xor((int)(top >> 32), s) << 32) | (uint32_t)__shfl_xor((int)(uint32_t)top, s);
          top = o > top ? o : top;
        }
        if ((tid & 7) == 0) gbest[tid >> 3] = top;
        __syncthreads();
        bound = gbest[0];
        for (int i = 1; i < kLpGroups; ++i) bound = gbest[i] < bound ? gbest[i] : bound;
      }
      const float bv = bound ? lp_value(bound) : -INFINITY;
      const bool any = !bound || !(cm < bv);
      if (__syncthreads_or(any)) {
        if (any) {
          auto push = [&](float y, uint32_t i) __attribute__((always_inline)) {
            const uint64_t key = lp_key(y, i);
            if (key >= bound) cand[atomicAdd(&ncand, 1)] = key;
          };
          if (ext) push(xe, xi);
#pragma unroll
          for (int e = 0; e < kLpPer; ++e)
            if (valid(e)) push(v[e], index(e));
        }
        __syncthreads();
        const int n = ncand;
        if (n > kept) {  // keys came: the best k of them and of those kept
          const int nk = min(n, k);
          lp_select(cand, n, nk, best);
          __syncthreads();
          if (tid < nk) cand[tid] = best[tid];
          if (tid == 0) ncand = nk;
          kept = nk;
          bound = nk == k ? best[k - 1] + 1 : bound;
          __syncthreads();
        }
      }
    }
    first = false;
  }

  // ---- the threads' sums ----
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) {
    lp_merge(a, __shfl_xor(a.m, s), __shfl_xor(a.s0, s), __shfl_xor(a.s1, s));
    above += __shfl_xor(above, s);
  }
  if (lane == 0) {
    sums[wave] = a;
    cnts[wave] = above;
  }
  __syncthreads();
  a = sums[0];
  above = cnts[0];
  for (int w = 1; w < kLpWaves; ++w) {
    lp_merge(a, sums[w].m, sums[w].s0, sums[w].s1);
    above += cnts[w];
  }

  if (segs > 1) {
    // a segment's part: (m, s0), (s1, above), keys kept, keys
    const size_t step = 3 + (size_t)k;
    uint64_t* part = parts + ((size_t)t * segs + seg) * step;
    auto put = [](uint64_t* p, uint64_t v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
    auto get = [](const uint64_t* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
    if (tid == 0) {
      put(part, (uint64_t)__float_as_uint(a.m) | ((uint64_t)__float_as_uint(a.s0) << 32));
      put(part + 1, (uint64_t)__float_as_uint(a.s1) | ((uint64_t)(uint32_t)above << 32));
      put(part + 2, (uint64_t)kept);
    }
    if (tid < kept) put(part + 3 + tid, cand[tid]);
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (tid == 0) {
      int* ctr = counters + (size_t)t * kLpCtrStride;
      last = __hip_atomic_fetch_add(ctr, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == segs - 1;
      if (last) __hip_atomic_store(ctr, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // re-armed
      ncand = 0;
    }
    __syncthreads();
    if (!last) return;
    const uint64_t* p0 = parts + (size_t)t * segs * step;
    a = {-INFINITY, 0.f, 0.f};
    above = 0;
    // the best of the segments' k-th keys: no key below it is among the row's best k
    uint64_t lb = 0;
    for (int s = tid; s < segs; s += kLpThreads) {
      const uint64_t* p = p0 + (size_t)s * step;
      const uint64_t w0 = get(p), w1 = get(p + 1);
      lp_merge(a, __uint_as_float((uint32_t)w0), __uint_as_float((uint32_t)(w0 >> 32)), __uint_as_float((uint32_t)w1));
      above += (int)(w1 >> 32);
      if (k && (int)get(p + 2) == k) {
        const uint64_t key = get(p + 3 + k - 1);
        lb = key > lb ? key : lb;
      }
    }
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
      lp_merge(a, __shfl_xor(a.m, s), __shfl_xor(a.s0, s), __shfl_xor(a.s1, s));
      above += __shfl_xor(above, s);
      const uint64_t o = ((uint64_t)(uint32_t)__shfl_xor((int)(lb >> 32), s) << 32) | (uint32_t)__shfl_xor((int)(uint32_t)lb, s);
      lb = o > lb ? o : lb;
    }
    if (lane == 0) {
      sums[wave] = a;
      cnts[wave] = above;
      gbest[wave] = lb;
    }
    __syncthreads();
    a = sums[0];
    above = cnts[0];
    lb = gbest[0];
    for (int w = 1; w < kLpWaves; ++w) {
      lp_merge(a, sums[w].m, sums[w].s0, sums[w].s1);
      above += cnts[w];
      lb = gbest[w] > lb ? gbest[w] : lb;
    }
    for (int i = tid; i < segs * k; i += kLpThreads) {
      const int s = i / k, j = i % k;
      const uint64_t* p = p0 + (size_t)s * step;
      if (j >= (int)get(p + 2)) continue;
      const uint64_t key = get(p + 3 + j);
      if (key >= lb) cand[atomicAdd(&ncand, 1)] = key;
    }
    __syncthreads();
    if (k) {
      lp_select(cand, ncand, k, best);
      __syncthreads();
      if (tid < k) cand[tid] = best[tid];
      __syncthreads();
    }
  }

  // ---- the row's results ----
  int row = t;
  if (state) {  // the token just generated
    row = state[1] - 1;
    if (row < 0) return;
  }
  if (row >= out_rows) return;
  const bool none = a.m == -INFINITY && a.s0 == 0.f;  // every value -inf
  const double lz = log((double)a.s0);                // lse = m + lz
  auto logp = [&](float y) { return none || y == -INFINITY ? (a.s0 != a.s0 ? NAN : -INFINITY) : (float)(((double)y - (double)a.m) - lz); };
  if (tid == 0) {
    if (lp_out) lp_out[row] = given ? logp(xt) : 0.f;
    if (ent_out) ent_out[row] = none ? 0.f : (float)(lz - (double)a.s1 / (double)a.s0);
    if (rank_out) rank_out[row] = given ? above : -1;
  }
  if (tid < k) {
    if (top_ids) top_ids[(size_t)row * k + tid] = lp_index(cand[tid]);
    if (top_lp) {
      const int i = lp_index(cand[tid]);
      top_lp[(size_t)row * k + tid] = logp(to_f32<T>(x[i]));
    }
  }
}

// Segments of a row: as many as give every CU four workgroups, of at least a chunk each, their keys within
// the buffer that the last one collects them in.
static int lp_segments(int T, int V, int k) {
  const int most = (V + kLpChunk - 1) / kLpChunk;
  int s = T >= 4 * kCUs ? 1 : (4 * kCUs + T - 1) / T;
  if (s > most) s = most;
  const int cap = kLpCand / (k > 0 ? k : 1);
  if (s > cap) s = cap;
  return s < 1 ? 1 : s;
}
static size_t lp_part_bytes(int T, int V, int k) {
  const int s = lp_segments(T, V, k);
  return s > 1 ? (size_t)T * s * (3 + k) * 8 : 0;
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
  if (x_dtype == MIQ_F32)
    hipLaunchKernelGGL(logprobs_kernel<float>, grid, block, 0, st, static_cast<const float*>(logits), (size_t)ld, ids, V, k,
                       logprobs, entropy, ranks, top_ids, top_logprobs, state, out_rows, counters, parts);
  else
    hipLaunchKernelGGL(logprobs_kernel<__half>, grid, block, 0, st, static_cast<const __half*>(logits), (size_t)ld, ids, V, k,
                       logprobs, entropy, ranks, top_ids, top_logprobs, state, out_rows, counters, parts);
  return check_launch("token_logprobs");
}
