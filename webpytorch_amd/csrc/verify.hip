// Verification of drafted tokens, with the token that follows them: of each sequence s the target's logits rows 0 .. D behind its
// D drafted tokens x_i, the draft's rows 0 .. D - 1 (or none), and random numbers u_0 .. u_D in [0, 1). With p and q the
// softmaxes of the rows over the temperature, x_i is accepted while u_i q_i(x_i) < p_i(x_i). The token behind the n accepted ones
// is drawn from max(p_n - q_n, 0), or from p_n where no draft was refused: the first index whose running sum of weights
// passes u_D times their total. The reference draws on the host, from logits read back (`_pick`: webtorch/llm.py:1309-1336).
//
// Which side of a border between tokens a draw falls on must not depend on rounding: 150000 borders lie in [0, 1), so that
// sums right to 1e-7 would give another token once in a hundred draws. Exponentials and sums are fp64 (to 3e-13; a draw is
// off once in 10^7).
//
// Two launches. Every row's maximum and sum of exponentials, in segments (a row's largest logit where the temperature is 0);
// then a group of workgroups for each sequence, each of which accepts by itself, sums the weights of its chunks, and the last of
// which to arrive finds the chunk, the thread and the index.
#include <math.h>

#include "attention_parts.h"

namespace miq {

constexpr int kVfThreads = 256;
constexpr int kVfLane = 16;                        // consecutive logits a thread
constexpr int kVfChunk = kVfThreads * kVfLane;     // logits of a chunk
constexpr int kVfMaxDrafts = 32;
constexpr int kVfMaxChunks = 1024;                 // sums of a row's chunks in LDS (a longer row's are of several rounds)
constexpr int kVfSegments = 64;                    // segments of a row, at most: a lane each
constexpr int kVfCtrStride = 8;                    // ints between arrival counters

// 2^t, t <= 0: the whole part by ldexp, the rest by the series of 2^f = e^(f ln 2), |f| <= 1 / 2, to the tenth power (off by
// 2.2e-13 at most). NaN stays NaN.
__device__ __forceinline__ double exp2_d(double t) {
  t = t < -1100. ? -1100. : t;
  const double k = rint(t), f = t - k;
  double p = 7.054911620801121e-09;  // (ln 2)^n / n!
  p = fma(p, f, 1.0178086009239696e-07);
  p = fma(p, f, 1.3215486790144305e-06);
  p = fma(p, f, 1.5252733804059838e-05);
  p = fma(p, f, 0.00015403530393381606);
  p = fma(p, f, 0.0013333558146428441);
  p = fma(p, f, 0.009618129107628477);
  p = fma(p, f, 0.055504108664821576);
  p = fma(p, f, 0.2402265069591007);
  p = fma(p, f, 0.6931471805599453);
  p = fma(p, f, 1.0);
  return ldexp(p, (int)k);
}
__device__ __forceinline__ double shfl_xor_d(double v, int d) {
  return __hiloint2double(__shfl_xor(__double2hiint(v), d), __shfl_xor(__double2loint(v), d));
}
__device__ __forceinline__ double shfl_up_d(double v, int d) {
  return __hiloint2double(__shfl_up(__double2hiint(v), d), __shfl_up(__double2loint(v), d));
}

// What is known of a row, or of a part of it: its largest logit with the lowest index of it (-inf, -1: none above -inf) and the
// sum of 2^((x - largest) c), NaN where a logit is NaN or +inf. At temperature 0 there is no sum.
struct RowPart {
  float m;
  int at;
  double s;
};
__device__ __forceinline__ void row_merge(RowPart& a, float m, int at, double s, bool greedy, double c) {
  if (greedy) {
    if (m > a.m || (m == a.m && (uint32_t)at < (uint32_t)a.at)) a = RowPart{m, at, 0.};
    return;
  }
  if (m == -INFINITY && s == 0.) return;
  if (a.m == -INFINITY && a.s == 0.) {
    a = RowPart{m, at, s};
    return;
  }
  const float top = fmaxf(a.m, m);
  const double fa = a.m == top ? 1. : exp2_d(((double)a.m - (double)top) * c), fb = m == top ? 1. : exp2_d(((double)m - (double)top) * c);
  a.s = a.s * fa + s * fb;
  a.m = top;
}
__device__ __forceinline__ void row_merge_wave(RowPart& r, bool greedy, double c) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const float m = __shfl_xor(r.m, d);
    const int at = __shfl_xor(r.at, d);
    row_merge(r, m, at, shfl_xor_d(r.s, d), greedy, c);
  }
}

// kVfLane consecutive logits from i on; -inf behind the row's end
template <typename XT> __device__ __forceinline__ void load_logits(const XT* row, int i, int V, bool vec, float* v) {
  constexpr int N = 16 / sizeof(XT);
  if (vec && i + kVfLane <= V) {
#pragma unroll
    for (int k = 0; k < kVfLane; k += N) {
      const miq_u32x4 w = *reinterpret_cast<const miq_u32x4*>(row + i + k);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        if constexpr (N == 4)
          v[k + e] = __uint_as_float(w[e]);
        else
          v[k + e] = __half2float(__ushort_as_half((unsigned short)(w[e >> 1] >> (16 * (e & 1)))));
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < kVfLane; ++k) v[k] = i + k < V ? to_f32<XT>(row[i + k]) : -INFINITY;
  }
}

struct VerifyArgs {
  const void* logits;      // [S][D + 1] rows
  const void* drafted;     // [S][D] rows, or null
  int64_t ls, lr, ds, dr;  // values from sequence to sequence and from row to row
  const int32_t* ids;      // [S][D]
  const float* uniforms;   // [S][D + 1]
  const float* temps;      // [S] or null
  float temp;
  int32_t* tokens;         // [S][D + 1]
  int32_t* accepted;       // [S]
  int S, D, V, segs, groups, rounds;  // segments of a row, workgroups of a sequence, rounds of 4096 logits a sum
  int lvec, dvec;
  uint64_t* parts;         // [rows][segs][2]
  double* sums;            // [S][kVfMaxChunks]
  int* counters;           // [S]
};
__device__ __forceinline__ float temperature(const VerifyArgs& a, int s) { return a.temps ? a.temps[s] : a.temp; }
// drafts of sequence s: those ahead of the first id below 0 (a wave's 64 lanes call)
__device__ __forceinline__ int drafts_of(const VerifyArgs& a, int s) {
  const int lane = threadIdx.x & 63;
  return __builtin_ctzll(__ballot(lane >= a.D || a.ids[(int64_t)s * a.D + lane] < 0));
}

// Segment blockIdx.x of row blockIdx.y: the S (D + 1) target rows, then the S D draft rows.
template <typename XT>
__global__ __launch_bounds__(kVfThreads) void verify_rows_kernel(VerifyArgs a) {
  __shared__ RowPart waves[kVfThreads / 64];
  const int row = blockIdx.y, seg = blockIdx.x, tid = threadIdx.x, rows = a.S * (a.D + 1);
  const bool target = row < rows;
  const int s = target ? row / (a.D + 1) : (row - rows) / a.D, i = target ? row % (a.D + 1) : (row - rows) % a.D;
  const float temp = temperature(a, s);
  const bool greedy = !(temp > 0.f);
  if (!target && greedy) return;
  if (drafts_of(a, s) < (target ? i : i + 1)) return;  // behind the last draft: not looked at
  const XT* x = target ? static_cast<const XT*>(a.logits) + s * a.ls + i * a.lr : static_cast<const XT*>(a.drafted) + s * a.ds + i * a.dr;
  const bool vec = target ? a.lvec : a.dvec;
  const double c = 1.4426950408889634 / (double)temp;
  const int chunks = (a.V + kVfChunk - 1) / kVfChunk;
  RowPart r = {-INFINITY, -1, 0.};
  for (int ch = seg; ch < chunks; ch += a.segs) {
    float v[kVfLane];
    const int at = ch * kVfChunk + tid * kVfLane;
    load_logits<XT>(x, at, a.V, vec, v);
    if (greedy) {
#pragma unroll
      for (int k = 0; k < kVfLane; ++k)
        if (v[k] > r.m) {
          r.m = v[k];
          r.at = at + k;
        }
      continue;
    }
    float mx = v[0];
    bool bad = false;
#pragma unroll
    for (int k = 0; k < kVfLane; ++k) {
      mx = fmaxf(mx, v[k]);
      bad = bad || !(v[k] < INFINITY);
    }
    if (mx > r.m) {
      r.s *= r.m == -INFINITY ? 0. : exp2_d(((double)r.m - (double)mx) * c);
      r.m = mx;
    }
    if (bad) r.s = NAN;
    if (r.m > -INFINITY) {
#pragma unroll
      for (int k = 0; k < kVfLane; ++k) r.s += exp2_d(((double)v[k] - (double)r.m) * c);
    }
  }
  row_merge_wave(r, greedy, c);
  if ((tid & 63) == 0) waves[tid >> 6] = r;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kVfThreads / 64; ++w) row_merge(r, waves[w].m, waves[w].at, waves[w].s, greedy, c);
    uint64_t* o = a.parts + ((int64_t)row * a.segs + seg) * 2;
    o[0] = (uint64_t)__float_as_uint(r.m) | ((uint64_t)(uint32_t)r.at << 32);
    o[1] = (uint64_t)__double_as_longlong(r.s);
  }
}

// The whole row from its segments, by one wave
__device__ __forceinline__ RowPart row_of(const uint64_t* parts, int segs, bool greedy, double c) {
  const int lane = threadIdx.x & 63;
  RowPart r = {-INFINITY, -1, 0.};
  if (lane < segs) {
    const uint64_t w = parts[2 * lane];
    r = RowPart{__uint_as_float((uint32_t)w), (int)(w >> 32), __longlong_as_double((long long)parts[2 * lane + 1])};
  }
  row_merge_wave(r, greedy, c);
  return r;
}

// Exclusive sum of v over the workgroup's threads, in their order; all is the sum of them all
__device__ __forceinline__ double sums_before(double v, double* waves, double& all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  double x = v;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const double o = shfl_up_d(x, d);
    if (lane >= d) x += o;
  }
  if (lane == 63) waves[wave] = x;
  double before = shfl_up_d(x, 1);
  if (lane == 0) before = 0.;
  __syncthreads();
  double w = 0.;
  all = 0.;
#pragma unroll
  for (int k = 0; k < kVfThreads / 64; ++k) {
    if (k == wave) w = all;
    all += waves[k];
  }
  __syncthreads();
  return w + before;
}

template <typename XT>
__global__ __launch_bounds__(kVfThreads) void verify_token_kernel(VerifyArgs a) {
  __shared__ float tm[kVfMaxDrafts + 1], dm[kVfMaxDrafts];
  __shared__ double ts[kVfMaxDrafts + 1], dsum[kVfMaxDrafts], waves[kVfThreads / 64], list[kVfMaxChunks];
  __shared__ int tat[kVfMaxDrafts + 1], verdict[2], last, found;
  const int s = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, D = a.D;
  const float temp = temperature(a, s);
  const bool greedy = !(temp > 0.f), dist = a.drafted && !greedy;
  const double c = 1.4426950408889634 / (double)temp;
  const int32_t* ids = a.ids + (int64_t)s * D;
  const float* u = a.uniforms + (int64_t)s * (D + 1);
  const int drafts = drafts_of(a, s);
  for (int i = wave; i <= drafts; i += kVfThreads / 64) {
    const RowPart r = row_of(a.parts + ((int64_t)s * (D + 1) + i) * a.segs * 2, a.segs, greedy, c);
    if (lane == 0) {
      tm[i] = r.m;
      ts[i] = r.s;
      tat[i] = r.at;
    }
  }
  if (dist)
    for (int i = wave; i < drafts; i += kVfThreads / 64) {
      const RowPart r = row_of(a.parts + ((int64_t)a.S * (D + 1) + (int64_t)s * D + i) * a.segs * 2, a.segs, false, c);
      if (lane == 0) {
        dm[i] = r.m;
        dsum[i] = r.s;
      }
    }
  __syncthreads();
  const XT* const tl = static_cast<const XT*>(a.logits) + s * a.ls;
  const XT* const dl = dist ? static_cast<const XT*>(a.drafted) + s * a.ds : nullptr;
  if (wave == 0) {  // lane i judges draft i
    bool ok = false;
    if (lane < drafts) {
      const int x = ids[lane];
      if (greedy) {
        ok = x == tat[lane];
      } else if (x < a.V && ts[lane] > 0.) {  // a row without a distribution (NaN, or nothing above -inf) accepts nothing
        const double p = exp2_d(((double)to_f32<XT>(tl[lane * a.lr + x]) - (double)tm[lane]) * c) / ts[lane];
        double q = 1.;
        if (dist) q = dsum[lane] > 0. ? exp2_d(((double)to_f32<XT>(dl[lane * a.dr + x]) - (double)dm[lane]) * c) / dsum[lane] : NAN;
        ok = (double)u[lane] * q < p;
      }
    }
    const uint64_t no = __ballot(!ok);  // lanes from `drafts` on among them
    if (lane == 0) verdict[0] = __builtin_ctzll(no);
  }
  __syncthreads();
  const int n = verdict[0];
  const bool refused = n < drafts;
  const bool law = greedy ? tat[n] >= 0 : ts[n] > 0.;  // the row is a distribution
  auto answer = [&](int token) {  // by one thread
    int32_t* o = a.tokens + (int64_t)s * (D + 1);
    for (int i = 0; i <= D; ++i) o[i] = i < n ? ids[i] : i == n ? token : -1;
    a.accepted[s] = n;
  };
  if (greedy || !law) {
    if (blockIdx.x == 0 && tid == 0) answer(law ? tat[n] : -1);
    return;
  }
  // ---- weights ----
  const XT* const trow = tl + n * a.lr;
  const bool minus = refused && dist && dsum[n] > 0.;   // max(p - q, 0)
  const int without = refused && !dist ? ids[n] : -1;   // p but for the draft
  const XT* const drow = minus ? dl + n * a.dr : nullptr;
  const double tmax = tm[n], ti = 1. / ts[n], dmax = minus ? dm[n] : 0., di = minus ? 1. / dsum[n] : 0.;
  auto weights = [&](int at, double* w) __attribute__((always_inline)) {
    float v[kVfLane];
    load_logits<XT>(trow, at, a.V, a.lvec, v);
#pragma unroll
    for (int k = 0; k < kVfLane; ++k) w[k] = exp2_d(((double)v[k] - tmax) * c) * ti;
    if (minus) {
      load_logits<XT>(drow, at, a.V, a.dvec, v);
#pragma unroll
      for (int k = 0; k < kVfLane; ++k) {
        const double d = w[k] - exp2_d(((double)v[k] - dmax) * c) * di;
        w[k] = d > 0. ? d : 0.;
      }
    }
    if (without >= at && without < at + kVfLane)
#pragma unroll
      for (int k = 0; k < kVfLane; ++k)
        if (at + k == without) w[k] = 0.;
    double sum = 0.;
#pragma unroll
    for (int k = 0; k < kVfLane; ++k) sum += w[k];
    return sum;
  };
  const int span = a.rounds * kVfChunk, chunks = (int)(((int64_t)a.V + span - 1) / span);
  double* const sums = a.sums + (int64_t)s * kVfMaxChunks;
  for (int ch = blockIdx.x; ch < chunks; ch += a.groups) {
    double total = 0.;
    for (int k = 0; k < a.rounds; ++k) {
      const int64_t at = (int64_t)ch * span + k * kVfChunk + tid * kVfLane;
      double w[kVfLane], all;
      const double mine = at < a.V ? weights((int)at, w) : 0.;
      sums_before(mine, waves, all);
      total += all;
    }
    if (tid == 0)
      __hip_atomic_store(reinterpret_cast<uint64_t*>(sums + ch), (uint64_t)__double_as_longlong(total), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  if (a.groups > 1) {
    if (!last_slice(a.counters + s * kVfCtrStride, a.groups, &last)) return;
  } else {
    parts_stored();
    __syncthreads();
  }
  // ---- the last to arrive: the first index whose running sum passes u times the total ----
  for (int ch = tid; ch < chunks; ch += kVfThreads)
    list[ch] = __longlong_as_double((long long)__hip_atomic_load(reinterpret_cast<uint64_t*>(sums + ch), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
  if (tid == 0) found = -1;
  __syncthreads();
  double total = 0.;
  int heavy = -1;  // the last chunk with any weight
  for (int ch = 0; ch < chunks; ++ch) {
    total += list[ch];
    if (list[ch] > 0.) heavy = ch;
  }
  if (heavy < 0) {  // the target leaves nothing beside the draft, or the two are the same
    if (tid == 0) answer(refused && ids[n] < a.V ? ids[n] : -1);
    return;
  }
  const double want = (double)u[D] * total;
  double before = 0.;
  int ch = 0;
  for (; ch < heavy; ++ch) {
    if (before + list[ch] > want) break;
    before += list[ch];
  }
  for (int k = 0; k < a.rounds; ++k) {
    const int64_t at = (int64_t)ch * span + k * kVfChunk + tid * kVfLane;
    double w[kVfLane], all;
    const double mine = at < a.V ? weights((int)at, w) : 0.;
    double run = before + sums_before(mine, waves, all);
    int hit = -1, any = -1;
    if (mine > 0.) {
#pragma unroll
      for (int i = 0; i < kVfLane; ++i) {
        run += w[i];
        if (w[i] > 0.) any = (int)at + i;
        if (w[i] > 0. && run > want && hit < 0) hit = (int)at + i;
      }
    }
    // the first hit; where rounding leaves none, the last index of the chunk with any weight
    if (tid == 0) {
      verdict[0] = 0x7FFFFFFF;
      verdict[1] = -1;
    }
    __syncthreads();
    if (hit >= 0) atomicMin(&verdict[0], hit);
    if (any >= 0) atomicMax(&verdict[1], any);
    __syncthreads();
    const int first = verdict[0];
    if (first != 0x7FFFFFFF) {
      if (tid == 0) answer(first);
      return;
    }
    if (tid == 0 && verdict[1] >= 0) found = verdict[1];
    before += all;
    __syncthreads();
  }
  if (tid == 0) answer(found);
}

struct VerifyPlan {
  int segs, groups, rounds;
  size_t parts, sums;
};
// Segments of a row that give every CU several workgroups; workgroups of a sequence likewise.
static VerifyPlan verify_plan(int S, int D, int V) {
  VerifyPlan p;
  const int chunks = (int)(((int64_t)V + kVfChunk - 1) / kVfChunk);
  const int64_t rows = (int64_t)S * (2 * D + 1);
  int64_t segs = (8 * kCUs + rows - 1) / rows, groups = (4 * kCUs + S - 1) / S;
  p.rounds = (chunks + kVfMaxChunks - 1) / kVfMaxChunks;
  const int spans = (chunks + p.rounds - 1) / p.rounds;
  if (segs > chunks) segs = chunks;
  p.segs = (int)(segs > kVfSegments ? kVfSegments : segs);
  p.groups = (int)(groups > spans ? spans : groups);
  p.parts = (size_t)rows * p.segs * 16;
  p.sums = (size_t)S * kVfMaxChunks * 8;
  return p;
}

}  // namespace miq

using namespace miq;

static int check_verify(const char* what, int S, int D, int V) {
  MIQ_REQUIRE(S >= 0 && D >= 0 && V > 0 && V <= (1 << 30), MIQ_ERR_INVALID, "%s: S=%d D=%d V=%d", what, S, D, V);
  MIQ_REQUIRE(D <= kVfMaxDrafts, MIQ_ERR_UNSUPPORTED, "%s: D=%d drafts (at most %d)", what, D, kVfMaxDrafts);
  MIQ_REQUIRE((int64_t)S * (2 * D + 1) <= 65535, MIQ_ERR_UNSUPPORTED, "%s: S=%d sequences of D=%d drafts (at most 65535 rows)", what, S, D);
  return MIQ_OK;
}

extern "C" int miq_verify_drafts_workspace(int S, int D, int V, size_t* bytes) {
  MIQ_REQUIRE(bytes, MIQ_ERR_INVALID, "verify_drafts_workspace: null pointer");
  if (int rc = check_verify("verify_drafts_workspace", S, D, V)) return rc;
  *bytes = 0;
  if (S == 0) return MIQ_OK;
  const VerifyPlan p = verify_plan(S, D, V);
  *bytes = kCounterBytes + p.parts + p.sums;
  return MIQ_OK;
}

extern "C" int miq_verify_drafts(const void* logits, int x_dtype, int64_t ld_seq, int64_t ld_row, const int32_t* drafts,
                                 const void* draft_logits, int64_t draft_ld_seq, int64_t draft_ld_row, const float* uniforms,
                                 const float* temperatures, float temperature, int32_t* tokens, int32_t* accepted, int S, int D, int V,
                                 void* workspace, size_t ws_bytes, void* stream) {
  if (int rc = check_verify("verify_drafts", S, D, V)) return rc;
  const bool dist = draft_logits && D > 0;
  MIQ_REQUIRE(x_dtype == MIQ_F32 || x_dtype == MIQ_F16, MIQ_ERR_UNSUPPORTED, "verify_drafts: logits dtype %d", x_dtype);
  MIQ_REQUIRE(ld_row >= V && ld_seq >= 0 && (!dist || (draft_ld_row >= V && draft_ld_seq >= 0)), MIQ_ERR_INVALID,
              "verify_drafts: rows %lld and %lld apart hold V=%d values", (long long)ld_row, (long long)draft_ld_row, V);
  MIQ_REQUIRE(temperatures || (temperature >= 0.f && temperature <= 3.4e38f), MIQ_ERR_INVALID, "verify_drafts: temperature=%g", (double)temperature);
  if (S == 0) return MIQ_OK;
  MIQ_REQUIRE(logits && (drafts || D == 0) && uniforms && tokens && accepted, MIQ_ERR_INVALID, "verify_drafts: null pointer");
  const int size = x_dtype == MIQ_F32 ? 4 : 2;
  MIQ_REQUIRE(aligned(logits, size) && (!dist || aligned(draft_logits, size)), MIQ_ERR_ALIGN, "verify_drafts: logits must be aligned to their type");
  const VerifyPlan p = verify_plan(S, D, V);
  const size_t need = kCounterBytes + p.parts + p.sums;
  MIQ_REQUIRE(workspace && ws_bytes >= need, MIQ_ERR_INVALID, "verify_drafts: workspace of %zu bytes, %zu needed", workspace ? ws_bytes : (size_t)0,
              need);
  MIQ_REQUIRE(aligned(workspace, 256), MIQ_ERR_ALIGN, "verify_drafts: the workspace must be 256-byte aligned");
  VerifyArgs a;
  a.logits = logits;
  a.drafted = dist ? draft_logits : nullptr;
  a.ls = ld_seq;
  a.lr = ld_row;
  a.ds = draft_ld_seq;
  a.dr = draft_ld_row;
  a.ids = drafts;
  a.uniforms = uniforms;
  a.temps = temperatures;
  a.temp = temperature;
  a.tokens = tokens;
  a.accepted = accepted;
  a.S = S;
  a.D = D;
  a.V = V;
  a.segs = p.segs;
  a.groups = p.groups;
  a.rounds = p.rounds;
  a.lvec = aligned(logits, 16) && ld_seq * size % 16 == 0 && ld_row * size % 16 == 0;
  a.dvec = dist && aligned(draft_logits, 16) && draft_ld_seq * size % 16 == 0 && draft_ld_row * size % 16 == 0;
  a.counters = static_cast<int*>(workspace);
  a.parts = reinterpret_cast<uint64_t*>(static_cast<char*>(workspace) + kCounterBytes);
  a.sums = reinterpret_cast<double*>(static_cast<char*>(workspace) + kCounterBytes + p.parts);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  // the second launch reads what the first left in the workspace: another thread's call on the stream waits
  std::unique_lock<std::mutex> whole(stream_lock(st));
  const dim3 rows((unsigned)p.segs, (unsigned)(S * (dist ? 2 * D + 1 : D + 1))), group((unsigned)p.groups, (unsigned)S), block(kVfThreads);
  if (x_dtype == MIQ_F32) {
    hipLaunchKernelGGL(verify_rows_kernel<float>, rows, block, 0, st, a);
    hipLaunchKernelGGL(verify_token_kernel<float>, group, block, 0, st, a);
  } else {
    hipLaunchKernelGGL(verify_rows_kernel<__half>, rows, block, 0, st, a);
    hipLaunchKernelGGL(verify_token_kernel<__half>, group, block, 0, st, a);
  }
  return check_launch("verify_drafts");
}
