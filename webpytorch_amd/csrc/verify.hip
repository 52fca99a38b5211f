// Verification of drafted tokens, with the token that follows them: of each sequence s the target's logits rows 0 .. D behind its
// D drafted tokens x_i, the draft's rows 0 .. D - 1 (or none), and random numbers u_0 .. u_D in [0, 1). With p and q the
// softmaxes of the rows over the temperature, x_i is accepted while u_i q_i(x_i) < p_i(x_i). The token behind the n accepted ones
// is drawn from max(p_n - q_n, 0), or from p_n where no draft was refused: the first index whose running sum of weights
// passes u_D times their total. The reference draws on the host, from logits read back (`_pick`: webtorch/llm.py:1309-1336).
//
// Which side of a border between tokens a draw falls on must not depend on rounding: 150000 borders lie in [0, 1), so that
// sums right to 1e-7 would give another token once in a hundred draws. Exponentials and sums are fp64 (to 2e-13; a draw is
// off once in 10^7), and a temperature given for all sequences stays the fp64 number that it is: fp32's next to 0.8 gives another token in 5000 draws.
//
// Two launches. Every row's maximum and sum of exponentials, in segments (a row's largest logit where the temperature is 0), where the
// last segment of a sequence to arrive judges its drafts; then a group of workgroups for each sequence sums the weights of its
// chunks, and the last of them to arrive finds the chunk, the thread and the index.
//
// Bound and measured (us a replay): 64 sequences of 4 drafts, V 128256, fp32 93: the rows 65 (295 MB, 4.5 TB/s) and the draw 26 (66 MB of them
// again, fp64 issue); one sequence, V 151936, 21: the chain logits, part, counter, judgement and then weights, sum, counter, chunk.
#include <math.h>

#include "attention_parts.h"
#include "kv4.h"

namespace miq {

constexpr int kVfThreads = 256;
constexpr int kVfLane = 16, kVfLaneW = 8;          // logits of a chunk a thread: of a row's sums, and of the weights
constexpr int kVfChunk = kVfThreads * kVfLane, kVfChunkW = kVfThreads * kVfLaneW;
constexpr int kVfMaxDrafts = 32;
constexpr int kVfMaxChunks = 1024;                 // sums of a row's weights (a longer row's are of several chunks each)
constexpr int kVfSegments = 64;                    // segments of a row, at most: a lane each
constexpr int kVfCtrStride = 8;                    // ints between the counters of sequences

// 2^(i / 256) in LDS
constexpr int kVfPowers = 256;
__device__ __forceinline__ void fill_powers(double* tab) {
  tab[threadIdx.x] = exp2((double)threadIdx.x / kVfPowers);
  __syncthreads();
}
// c of a temperature: at most 1e300, where the logits nearest to the largest (2^-149 below) are past every border, and 0 c is 0
__device__ __forceinline__ double power_unit(double temperature) { return fmin(kVfPowers * 1.4426950408889634 / temperature, 1e300); }
// High word of -899 kVfPowers. Powers are no lower than 2^-899 (-inf among them), which no sum sees. The border is drawn on the exponent: of the
// fp32 logits, m less 623 temperatures rounds to m itself where the temperature is small. Exponents are 0 or negative, so that
// their high words, as unsigned numbers, ascend as they descend: the least of two words bounds one, at the cost of an fp32 maximum.
constexpr uint32_t kVfDeepest = 0xC10C1800u;
// 2^((x - m) c / 256), x <= m, added to `sum`, 1 for m itself: whole multiples of 1 / 256 by the table and the exponent, the rest, |f| <= 1 / 512, by the
// series of e^(f ln 2) to the third power (1.4e-13). 10 fp64 operations (a table of 32 takes 12, the series of |f| <= 1 / 2 alone 19),
// which with the loads' latency bound the kernel of the rows (64 sequences of 4 drafts, V 128256: fp16 61 us, fp32 65, where its bytes take 58).
// ZERO: nothing for what is as low as the border, so that no draw falls on it.
template <bool ZERO = false> __device__ __forceinline__ double power_plus(float x, double m, double c, const double* tab, double sum) {
  const double far = ((double)x - m) * c, magic = 6755399441055744.;  // 1.5 2^52: the whole part in the low word
  const uint32_t high = (uint32_t)__double2hiint(far);
  const double y = __hiloint2double((int)min(high, kVfDeepest), __double2loint(far));
  const double up = y + magic, f = y - (up - magic);
  const int k = __double2loint(up);
  double p = 3.308302680541371e-09;  // (ln 2 / 256)^n / n!
  p = fma(p, f, 3.665565596910106e-06);
  p = fma(p, f, 0.0027076061740622863);
  p = fma(p, f, 1.0);
  const double t = tab[k & (kVfPowers - 1)], power = __hiloint2double(__double2hiint(t) + ((k >> 8) << 20), __double2loint(t));
  return fma(ZERO && high >= kVfDeepest ? 0. : power, p, sum);
}
template <int CTRL, int ROWS = 0xF> __device__ __forceinline__ double dpp_double(double v) {  // 0 where no lane is the source
  return __hiloint2double(__builtin_amdgcn_update_dpp(0, __double2hiint(v), CTRL, ROWS, 0xF, false),
                          __builtin_amdgcn_update_dpp(0, __double2loint(v), CTRL, ROWS, 0xF, false));
}
__device__ __forceinline__ double lane_double(double v, int l) {
  return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(v), l), __builtin_amdgcn_readlane(__double2loint(v), l));
}
// the sum over lanes 0 .. l, in a fixed order
__device__ __forceinline__ double scan_double(double v) {
  v += dpp_double<0x111>(v);  // row_shr 1, 2, 4, 8
  v += dpp_double<0x112>(v);
  v += dpp_double<0x114>(v);
  v += dpp_double<0x118>(v);
  v += dpp_double<0x142, 0xA>(v);  // a row's last lane to the next row: rows 1 and 3
  return v + dpp_double<0x143, 0xC>(v);  // lane 31 to rows 2 and 3
}

// What is known of a row, or of a part of it: its largest logit with the lowest index of it (-inf, -1: none above -inf) and the
// sum of 2^((x - largest) c / 256), NaN where a logit is NaN or +inf. At temperature 0 there is no sum, otherwise no index.
struct RowPart {
  float m;
  int at;
  double s;
};
// of the parts that the lanes of a wave hold
__device__ __forceinline__ RowPart row_of_lanes(RowPart r, bool greedy, double c, const double* tab) {
  const float top = wave_max(r.m);
  if (greedy) {
    uint32_t at = r.m == top && r.m > -INFINITY ? (uint32_t)r.at : 0xFFFFFFFFu;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) at = min(at, (uint32_t)__shfl_xor((int)at, d));
    return RowPart{top, (int)at, 0.};
  }
  const double s = r.m > -INFINITY ? r.s * power_plus(r.m, top, c, tab, 0.) : r.s;  // 0 or NaN
  return RowPart{top, -1, lane_double(scan_double(s), 63)};
}

// A thread's N logits of a chunk of N kVfThreads from i0 on. In order: N consecutive ones; otherwise vectors of consecutive threads. Rows
// may start at any value: this target's 16-byte loads do. -inf behind the row's end
template <typename XT, int N> __device__ __forceinline__ int logit_at(int e, bool in_order) {  // offset of value e in the chunk
  constexpr int W = 16 / sizeof(XT);
  const int tid = threadIdx.x;
  return in_order ? N * tid + e : (e / W * kVfThreads + tid) * W + e % W;
}
// as they lie in memory, so that the next chunk's take few registers on their way
typedef uint32_t UnalignedVector __attribute__((ext_vector_type(4), aligned(2)));
template <typename XT, int N> struct Logits {
  static constexpr int W = 16 / sizeof(XT);
  uint32_t raw[N * sizeof(XT) / 4];
  __device__ __forceinline__ void load(const XT* row, int64_t i0, int V, bool in_order) {
    if (i0 + N * kVfThreads <= V) {
#pragma unroll
      for (int k = 0; k < N; k += W) {
        const UnalignedVector w = *reinterpret_cast<const UnalignedVector*>(row + i0 + logit_at<XT, N>(k, in_order));
#pragma unroll
        for (int e = 0; e < 4; ++e) raw[k / W * 4 + e] = w[e];
      }
    } else {
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const int64_t i = i0 + logit_at<XT, N>(k, in_order);
        if constexpr (W == 4) {
          raw[k] = i < V ? __float_as_uint(row[i]) : 0xFF800000u;
        } else {
          const uint32_t h = i < V ? (uint32_t)__half_as_ushort(row[i]) : 0xFC00u;
          raw[k / 2] = k & 1 ? raw[k / 2] | h << 16 : h;
        }
      }
    }
  }
  __device__ __forceinline__ float operator[](int k) const {
    if constexpr (W == 4)
      return __uint_as_float(raw[k]);
    else
      return __half2float(__ushort_as_half((unsigned short)(raw[k >> 1] >> (16 * (k & 1)))));
  }
};

// What a sequence's judgement leaves for its draw
struct Verdict {
  int n, token;                 // drafts accepted; the token, or kVfDraw
  int refused, without;         // draft n was refused; the token that p lacks (-1: none)
  float tmax, dmax;             // of the target's row n, and of the draft's
  double ti, di;                // 1 / sums; di 0: nothing is taken off p
};
constexpr int kVfDraw = -2;

struct VerifyArgs {
  const void* logits;      // [S][D + 1] rows
  const void* drafted;     // [S][D] rows, or null
  int64_t ls, lr, ds, dr;  // values from sequence to sequence and from row to row
  const int32_t* ids;      // [S][D]
  const float* uniforms;   // [S][D + 1]
  const float* temps;      // [S] or null
  double temp;
  int32_t* tokens;         // [S][D + 1]
  int32_t* accepted;       // [S]
  int S, D, V, segs, groups, rounds;  // segments of a row, workgroups of a sequence, chunks a sum of weights
  uint64_t* parts;         // [rows][segs][2]
  double* sums;            // [S][kVfMaxChunks]
  Verdict* verdicts;       // [S]
  int* counters;           // [S][kVfCtrStride]: parts of rows, groups of weights
};
// 0 for what is no finite number above 0
__device__ __forceinline__ double temperature(const VerifyArgs& a, int s) {
  const double t = a.temps ? (double)a.temps[s] : a.temp;
  return t > 0. && t < INFINITY ? t : 0.;
}
// by a wave, whose lane i has draft i: one store (with the marks by ballots, where LDS atomics and one thread in a loop were, the draw behind 4 drafts
// 12.6 -> 7.8 us)
__device__ __forceinline__ void answer(const VerifyArgs& a, int s, int n, int token, int id) {
  const int lane = threadIdx.x & 63;
  if (lane <= a.D) a.tokens[(int64_t)s * (a.D + 1) + lane] = lane < n ? id : lane == n ? token : -1;
  if (lane == 0) a.accepted[s] = n;
}

// Segment blockIdx.x of row blockIdx.y: the S (D + 1) target rows, then the S D draft rows. The last segment of a sequence's rows to
// arrive judges its drafts.
template <typename XT>
__global__ __launch_bounds__(kVfThreads) void verify_rows_kernel(VerifyArgs a) {
  __shared__ RowPart waves[kVfThreads / 64], trow[kVfMaxDrafts + 1], drow[kVfMaxDrafts];
  __shared__ double tab[kVfPowers];
  __shared__ int last;
  const int row = blockIdx.y, seg = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, rows = a.S * (a.D + 1), D = a.D;
  const bool target = row < rows;
  const int s = target ? row / (D + 1) : (row - rows) / D, i = target ? row % (D + 1) : (row - rows) % D;
  const double temp = temperature(a, s);
  const bool greedy = !(temp > 0.), dist = a.drafted && !greedy;
  if (!target && greedy) return;
  const XT* const tl = static_cast<const XT*>(a.logits) + s * a.ls;
  const XT* const dl = static_cast<const XT*>(a.drafted) + s * a.ds;
  const XT* x = target ? tl + i * a.lr : dl + i * a.dr;
  const int chunks = (int)(((int64_t)a.V + kVfChunk - 1) / kVfChunk);
  Logits<XT, kVfLane> next;
  next.load(x, (int64_t)seg * kVfChunk, a.V, false);
  // lane i has draft i, its logits and its random number: for the judgement, on the way from here on
  const int id = lane < D ? a.ids[(int64_t)s * D + lane] : -1;
  const int drafts = __builtin_ctzll(__ballot(id < 0));  // those ahead of the first id below 0
  if (drafts < (target ? i : i + 1)) return;  // behind the last draft: not looked at
  const bool inside = lane < drafts && id < a.V;
  const float tx = inside ? to_f32<XT>(tl[lane * a.lr + id]) : 0.f, dx = inside && dist ? to_f32<XT>(dl[lane * a.dr + id]) : 0.f;
  const float ux = lane < drafts ? a.uniforms[(int64_t)s * (D + 1) + lane] : 0.f;
  const double c = power_unit(temp);
  fill_powers(tab);
  RowPart r = {-INFINITY, -1, 0.};
  double top = 0.;
  for (int ch = seg; ch < chunks; ch += a.segs) {
    const Logits<XT, kVfLane> v = next;
    if (ch + a.segs < chunks) next.load(x, (int64_t)(ch + a.segs) * kVfChunk, a.V, false);
    if (greedy) {
#pragma unroll
      for (int k = 0; k < kVfLane; ++k)
        if (v[k] > r.m) {
          r.m = v[k];
          r.at = ch * kVfChunk + logit_at<XT, kVfLane>(k, false);
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
      r.s = r.m == -INFINITY ? r.s : r.s * power_plus(r.m, mx, c, tab, 0.);
      r.m = mx;
      top = mx;
    }
    if (bad) r.s = NAN;
    if (r.m > -INFINITY) {
#pragma unroll
      for (int k = 0; k < kVfLane; ++k) r.s = power_plus(v[k], top, c, tab, r.s);
    }
  }
  r = row_of_lanes(r, greedy, c, tab);
  if (lane == 0) waves[wave] = r;
  __syncthreads();
  if (wave == 0) {
    r = row_of_lanes(tid < kVfThreads / 64 ? waves[tid] : RowPart{-INFINITY, -1, 0.}, greedy, c, tab);
    if (tid == 0) {
      uint64_t* o = a.parts + ((int64_t)row * a.segs + seg) * 2;
      __hip_atomic_store(o, (uint64_t)__float_as_uint(r.m) | ((uint64_t)(uint32_t)r.at << 32), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      __hip_atomic_store(o + 1, (uint64_t)__double_as_longlong(r.s), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }
  const int all = drafts + 1 + (dist ? drafts : 0);  // rows that are looked at
  if (!last_slice(a.counters + s * kVfCtrStride, all * a.segs, &last)) return;

  // ---- the judgement: lane i of wave 0 has draft i ----
  constexpr int U = 4;  // the target's rows, then the draft's: a wave U at a time, a lane a segment
  for (int k0 = wave * U; k0 < all; k0 += kVfThreads / 64 * U) {
    uint64_t w[U][2];
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int k = min(k0 + j, all - 1);
      const int64_t at = k <= drafts ? (int64_t)s * (D + 1) + k : rows + (int64_t)s * D + k - drafts - 1;
      uint64_t* p = a.parts + (at * a.segs + min(lane, a.segs - 1)) * 2;
      w[j][0] = __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      w[j][1] = __hip_atomic_load(p + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
#pragma unroll
    for (int j = 0; j < U; ++j) {
      RowPart one = {-INFINITY, -1, 0.};
      if (lane < a.segs) one = RowPart{__uint_as_float((uint32_t)w[j][0]), (int)(w[j][0] >> 32), __longlong_as_double((long long)w[j][1])};
      one = row_of_lanes(one, greedy, c, tab);
      const int k = k0 + j;
      if (lane == 0 && k < all) (k <= drafts ? trow[k] : drow[k - drafts - 1]) = one;
    }
  }
  __syncthreads();
  if (wave != 0) return;
  bool ok = false;
  if (lane < drafts) {
    if (greedy) {
      ok = id == trow[lane].at;
    } else if (inside && trow[lane].s > 0.) {  // a row without a distribution (NaN, or nothing above -inf) accepts nothing
      // down to fp64's least numbers, where both sides are small
      const double p = exp2(((double)tx - (double)trow[lane].m) * c / kVfPowers) / trow[lane].s;
      double q = 1.;
      if (dist) q = drow[lane].s > 0. ? exp2(((double)dx - (double)drow[lane].m) * c / kVfPowers) / drow[lane].s : (double)NAN;
      ok = (double)ux * q < p;
    }
  }
  const int n = __builtin_ctzll(__ballot(!ok));  // lanes from `drafts` on say no
  const int refusal = __builtin_amdgcn_readlane(id, n);
  const bool refused = n < drafts, law = greedy ? trow[n].at >= 0 : trow[n].s > 0.;  // law: the row is a distribution
  Verdict v = {n, greedy || !law ? (law ? trow[n].at : -1) : kVfDraw, refused, refused && !dist ? refusal : -1, trow[n].m, 0.f,
               1. / trow[n].s, 0.};
  if (refused && dist && drow[n].s > 0.) {  // max(p - q, 0)
    v.dmax = drow[n].m;
    v.di = 1. / drow[n].s;
  }
  if (lane == 0) a.verdicts[s] = v;
  if (v.token != kVfDraw) answer(a, s, n, v.token, id);
}

// Exclusive sum of v over the workgroup's threads, in their order; all is the sum of them all
__device__ __forceinline__ double sums_before(double v, double* waves, double& all) {
  const int wave = threadIdx.x >> 6;
  const double x = scan_double(v);
  if ((threadIdx.x & 63) == 63) waves[wave] = x;
  __syncthreads();
  double w = 0.;
  all = 0.;
#pragma unroll
  for (int k = 0; k < kVfThreads / 64; ++k) {
    if (k == wave) w = all;
    all += waves[k];
  }
  __syncthreads();
  return w + (x - v);
}

// The first of the threads' `hit` and the last of their `any` that are not -1 (they ascend with the threads); -1 where there is none
__device__ __forceinline__ void first_and_last(int hit, int any, int (*marks)[kVfThreads / 64], int& first, int& last) {
  const uint64_t h = __ballot(hit >= 0), y = __ballot(any >= 0);
  first = h ? __builtin_amdgcn_readlane(hit, __builtin_ctzll(h)) : -1;
  last = y ? __builtin_amdgcn_readlane(any, 63 - __builtin_clzll(y)) : -1;
  if ((threadIdx.x & 63) == 0) {
    marks[0][threadIdx.x >> 6] = first;
    marks[1][threadIdx.x >> 6] = last;
  }
  __syncthreads();
  first = last = -1;
#pragma unroll
  for (int w = 0; w < kVfThreads / 64; ++w) {
    if (first < 0) first = marks[0][w];
    if (marks[1][w] >= 0) last = marks[1][w];
  }
}

template <typename XT>
__global__ __launch_bounds__(kVfThreads) void verify_token_kernel(VerifyArgs a) {
  __shared__ double waves[kVfThreads / 64], tab[kVfPowers], found_before;
  __shared__ int marks[2][kVfThreads / 64], last;
  const int s = blockIdx.y, tid = threadIdx.x, wave = tid >> 6, D = a.D;
  const Verdict j = a.verdicts[s];
  const int id = tid < D ? a.ids[(int64_t)s * D + tid] : -1;  // for the answer
  const double c = power_unit(temperature(a, s)), ulast = a.uniforms[(int64_t)s * (D + 1) + D];
  fill_powers(tab);
  if (j.token != kVfDraw) return;
  const bool minus = j.di > 0.;
  const XT* const trow = static_cast<const XT*>(a.logits) + s * a.ls + j.n * a.lr;
  const XT* const drow = minus ? static_cast<const XT*>(a.drafted) + s * a.ds + j.n * a.dr : nullptr;
  const double tmax = j.tmax, dmax = j.dmax;
  struct Chunk {
    Logits<XT, kVfLaneW> t, d;
  };
  auto load = [&](Chunk& x, int64_t i0, bool in_order) __attribute__((always_inline)) {
    x.t.load(trow, i0, a.V, in_order);
    if (minus) x.d.load(drow, i0, a.V, in_order);
  };
  auto weights = [&](const Chunk& x, int64_t i0, bool in_order, double* w) __attribute__((always_inline)) {
    const Logits<XT, kVfLaneW>&v = x.t, &q = x.d;
#pragma unroll
    for (int k = 0; k < kVfLaneW; ++k) w[k] = power_plus<true>(v[k], tmax, c, tab, 0.) * j.ti;
    if (minus) {
#pragma unroll
      for (int k = 0; k < kVfLaneW; ++k) w[k] = fmax(w[k] - power_plus<true>(q[k], dmax, c, tab, 0.) * j.di, 0.);
    }
    if (j.without >= i0 && j.without < i0 + kVfChunkW)
#pragma unroll
      for (int k = 0; k < kVfLaneW; ++k)
        if (i0 + logit_at<XT, kVfLaneW>(k, in_order) == j.without) w[k] = 0.;
    double sum = 0.;
#pragma unroll
    for (int k = 0; k < kVfLaneW; ++k) sum += w[k];
    return sum;
  };
  const int span = a.rounds * kVfChunkW, chunks = (int)(((int64_t)a.V + span - 1) / span);
  double* const sums = a.sums + (int64_t)s * kVfMaxChunks;
  // this workgroup's chunks, span after span of them: the next one is loaded while one is added up
  auto start = [&](int ch, int k) __attribute__((always_inline)) { return (int64_t)ch * span + k * kVfChunkW; };
  Chunk next;
  load(next, start(blockIdx.x, 0), false);
  for (int ch = blockIdx.x; ch < chunks; ch += a.groups) {
    double mine = 0., all;
    for (int k = 0; k < a.rounds; ++k) {
      const Chunk x = next;
      if (k + 1 < a.rounds)
        load(next, start(ch, k + 1), false);
      else if (ch + a.groups < chunks)
        load(next, start(ch + a.groups, 0), false);
      double w[kVfLaneW];
      mine += weights(x, start(ch, k), false, w);
    }
    sums_before(mine, waves, all);
    if (tid == 0)
      __hip_atomic_store(reinterpret_cast<uint64_t*>(sums + ch), (uint64_t)__double_as_longlong(all), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  if (a.groups > 1) {
    if (!last_slice(a.counters + s * kVfCtrStride + 1, a.groups, &last)) return;
  } else {
    parts_stored();
    __syncthreads();
  }
  // ---- the last to arrive: the first index whose running sum passes u times the total ----
  // the chunk: each thread has some of them, in order
  constexpr int kEach = kVfMaxChunks / kVfThreads;
  double part[kEach], mine = 0., total;
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const int ch = tid * kEach + k;
    part[k] = ch < chunks ? __longlong_as_double((long long)__hip_atomic_load(reinterpret_cast<uint64_t*>(sums + ch), __ATOMIC_RELAXED,
                                                                              __HIP_MEMORY_SCOPE_AGENT))
                          : 0.;
    mine += part[k];
  }
  double run = sums_before(mine, waves, total);
  const double want = ulast * total;
  int hit = -1, heavy = -1;  // the first chunk past it; the last with any weight
  double at_hit = 0., at_heavy = 0.;
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    if (part[k] > 0.) {
      heavy = tid * kEach + k;
      at_heavy = run;
      if (hit < 0 && run + part[k] > want) {
        hit = heavy;
        at_hit = run;
      }
    }
    run += part[k];
  }
  int first, rest;
  first_and_last(hit, heavy, marks, first, rest);
  const int ch = first >= 0 ? first : rest;
  if (ch < 0) {  // the target leaves nothing beside the draft, or the two are the same
    const int draft = j.refused ? a.ids[(int64_t)s * D + j.n] : -1;
    if (wave == 0) answer(a, s, j.n, draft < a.V ? draft : -1, id);
    return;
  }
  if (hit == ch)
    found_before = at_hit;
  else if (heavy == ch && first < 0)
    found_before = at_heavy;
  __syncthreads();
  double before = found_before;
  int fallback = -1;
  for (int k = 0; k < a.rounds; ++k) {
    const int64_t i0 = (int64_t)ch * span + k * kVfChunkW;
    double w[kVfLaneW], all;
    Chunk x;
    load(x, i0, true);
    const double mine = weights(x, i0, true, w);
    double run = before + sums_before(mine, waves, all);
    int hit = -1, any = -1;
#pragma unroll
    for (int i = 0; i < kVfLaneW; ++i) {
      run += w[i];
      if (w[i] > 0.) {
        any = (int)i0 + kVfLaneW * tid + i;
        if (run > want && hit < 0) hit = any;
      }
    }
    // the first hit; where rounding leaves none, the last index of the chunk with any weight
    first_and_last(hit, any, marks, first, rest);
    if (rest >= 0) fallback = rest;
    if (first >= 0 || k == a.rounds - 1) {
      if (wave == 0) answer(a, s, j.n, first >= 0 ? first : fallback, id);
      return;
    }
    before += all;
  }
}

struct VerifyPlan {
  int segs, groups, rounds;
  size_t parts, sums, verdicts;
};
// Segments of a row: four workgroups a CU run at once, one after another takes as long as its chunks and some 4 more (start and sums).
// (24 sequences of 6 looked-up drafts, fp16, V 32003: 7 segments, 1176 workgroups, 20.4 us; 4, which fit at once, 17.8, and 14.8 since rows
// of odd length are read by vectors.) Workgroups of a sequence's
// weights: likewise at once.
static VerifyPlan verify_plan(int S, int D, int V, bool dist) {
  VerifyPlan p;
  const int chunks = (int)(((int64_t)V + kVfChunk - 1) / kVfChunk), most = chunks < kVfSegments ? chunks : kVfSegments;
  const int64_t rows = (int64_t)S * (dist ? 2 * D + 1 : D + 1);
  p.segs = 1;
  int64_t best = INT64_MAX;
  for (int s = 1; s <= most; ++s) {
    const int64_t cost = (rows * s + 4 * kCUs - 1) / (4 * kCUs) * ((chunks + s - 1) / s + 4);
    if (cost < best) {
      best = cost;
      p.segs = s;
    }
  }
  const int wchunks = (int)(((int64_t)V + kVfChunkW - 1) / kVfChunkW);
  p.rounds = (wchunks + kVfMaxChunks - 1) / kVfMaxChunks;
  const int spans = (wchunks + p.rounds - 1) / p.rounds, groups = (4 * kCUs + S - 1) / S;
  p.groups = groups > spans ? spans : groups;
  p.parts = (size_t)rows * p.segs * 16;
  p.sums = (size_t)S * kVfMaxChunks * 8;
  p.verdicts = (size_t)S * sizeof(Verdict);
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
  const VerifyPlan p = verify_plan(S, D, V, true), q = verify_plan(S, D, V, false);  // with and without draft rows
  *bytes = kCounterBytes + (p.parts > q.parts ? p.parts : q.parts) + p.sums + p.verdicts;
  return MIQ_OK;
}

extern "C" int miq_verify_drafts(const void* logits, int x_dtype, int64_t ld_seq, int64_t ld_row, const int32_t* drafts,
                                 const void* draft_logits, int64_t draft_ld_seq, int64_t draft_ld_row, const float* uniforms,
                                 const float* temperatures, double temperature, int32_t* tokens, int32_t* accepted, int S, int D, int V,
                                 void* workspace, size_t ws_bytes, void* stream) {
  if (int rc = check_verify("verify_drafts", S, D, V)) return rc;
  const bool dist = draft_logits && D > 0;
  MIQ_REQUIRE(x_dtype == MIQ_F32 || x_dtype == MIQ_F16, MIQ_ERR_UNSUPPORTED, "verify_drafts: logits dtype %d", x_dtype);
  MIQ_REQUIRE(ld_row >= V && ld_seq >= 0 && (!dist || (draft_ld_row >= V && draft_ld_seq >= 0)), MIQ_ERR_INVALID,
              "verify_drafts: rows %lld and %lld apart hold V=%d values", (long long)ld_row, (long long)draft_ld_row, V);
  MIQ_REQUIRE(temperatures || (temperature >= 0. && temperature < INFINITY), MIQ_ERR_INVALID, "verify_drafts: temperature=%g", temperature);
  if (S == 0) return MIQ_OK;
  MIQ_REQUIRE(logits && (drafts || D == 0) && uniforms && tokens && accepted, MIQ_ERR_INVALID, "verify_drafts: null pointer");
  const int size = x_dtype == MIQ_F32 ? 4 : 2;
  MIQ_REQUIRE(aligned(logits, size) && (!dist || aligned(draft_logits, size)), MIQ_ERR_ALIGN, "verify_drafts: logits must be aligned to their type");
  const VerifyPlan p = verify_plan(S, D, V, dist);
  const size_t need = kCounterBytes + p.parts + p.sums + p.verdicts;
  MIQ_REQUIRE(workspace && ws_bytes >= need, MIQ_ERR_INVALID, "verify_drafts: workspace of %zu bytes, %zu needed", workspace ? ws_bytes : (size_t)0,
              need);
  MIQ_REQUIRE(aligned(workspace, 256), MIQ_ERR_ALIGN, "verify_drafts: the workspace must be 256-byte aligned");
  // the answers are written while other sequences are read
  const auto span = [&](int64_t ls, int64_t lr, int rows) { return (((__int128)(S - 1) * ls + (__int128)(rows - 1) * (rows > 1 ? lr : 0) + V) * size); };
  const __int128 nx = span(S > 1 ? ld_seq : 0, ld_row, D + 1), nd = dist ? span(S > 1 ? draft_ld_seq : 0, draft_ld_row, D) : 0, most = (__int128)1 << 48;
  MIQ_REQUIRE(nx < most && nd < most, MIQ_ERR_INVALID, "verify_drafts: sequences %lld and %lld, rows %lld and %lld apart pass the address space",
              (long long)ld_seq, (long long)draft_ld_seq, (long long)ld_row, (long long)draft_ld_row);
  const size_t na = (size_t)S * 4, nt = na * (D + 1);
  const auto apart = [&](const void* p, size_t n) { return !p || n == 0 || (!share_bytes(tokens, nt, p, n) && !share_bytes(accepted, na, p, n)); };
  MIQ_REQUIRE(apart(logits, (size_t)nx) && apart(dist ? draft_logits : nullptr, (size_t)nd) && apart(drafts, na * D) && apart(uniforms, nt) &&
                  apart(temperatures, na) && apart(workspace, need) && !share_bytes(tokens, nt, accepted, na),
              MIQ_ERR_INVALID, "verify_drafts: tokens and accepted must lie apart from each other, the inputs and the workspace");
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
  a.counters = static_cast<int*>(workspace);
  a.parts = reinterpret_cast<uint64_t*>(static_cast<char*>(workspace) + kCounterBytes);
  a.sums = reinterpret_cast<double*>(static_cast<char*>(workspace) + kCounterBytes + p.parts);
  a.verdicts = reinterpret_cast<Verdict*>(static_cast<char*>(workspace) + kCounterBytes + p.parts + p.sums);
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
