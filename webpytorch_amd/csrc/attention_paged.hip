// miq_paged_attention: the plan of a call, and the kernels (attention_paged.h) of fp16 caches.
#include "attention_paged.h"

namespace miq {

constexpr int kPaMaxSplit = 4096;  // sequences x heads x tiles from which they are not split: their counters, 128 KB

// 16-row tiles of a workgroup: as many as the rows fill, of those whose sums the registers hold
static int pa_tiles(int64_t R, int HD) {
  const int most = HD == 64 ? 4 : HD == 128 ? 3 : 2;
  const int64_t n = (R + 15) / 16;
  return n >= most ? most : n == 3 && HD == 64 ? 4 : (int)n;
}
struct PagedPlan {
  int nr, nw, tiles, target, fit;
  int64_t grid, units;
};
// Workgroups of 8 waves, one a CU (two waves a SIMD fill the registers). From kPaMany sequences x heads x tiles on, of 4 waves, so that one
// workgroup starts while another ends (fp16 cache, one token, 256 sequences of 10 to 500 positions 98 -> 74 us; 64 of up to 8000 196 -> 200);
// of 4 also where the sums take most of the registers (heads of 256, wide heads of several tiles).
// A CU holds two or three workgroups of 4 waves at heads of 64 with one or two tiles and at heads of 128 with one tile of an fp16 cache. The other
// kernels take accumulation registers beside the vector ones in this form and keep one wave a SIMD; their 8-wave form, where they have one, keeps two. From kPaMany on
// both forms of those are not compared; as they run: 64 sequences of 50 to 8000, 32 / 8 heads of 128, fp32 cache 405 us (2.1 GB, 5.2 TB/s: memory), fp16
// cache and 5 tokens 242 (1.07 GB, 4.4 TB/s).
// The parts: where sequences, heads and tiles are at most half of the CUs, no more parts than there are CUs (320 parts on 256 CUs took
// twice the time of 256: 16 sequences of 300 to 5000, 5 tokens, fp32 90 -> 75 us); otherwise kPaParts of them, which ends evenly
// (64 sequences of up to 8000, us at 256 / 512 / 1024 / 2048 parts: 223 / 212 / 200 / 196, but 256 short ones 74 / 74 / 74 / 82).
constexpr int kPaMany = 512, kPaParts = 1024;
static PagedPlan pa_plan(int S, int T, int NH, int NKV, int HD, int64_t cap, bool c16) {
  PagedPlan p;
  const int64_t R = (int64_t)T * (NH / NKV);
  p.nr = pa_tiles(R, HD);
  p.tiles = (int)((R + 16 * p.nr - 1) / (16 * p.nr));
  p.units = (int64_t)NKV * p.tiles;
  const bool wide = HD == 256 || (HD == 192 && p.nr == 2);
  p.nw = wide || S * p.units >= kPaMany ? 4 : 8;
  const int64_t step = (c16 ? 32 : 16) * p.nw, most = cap <= kPaWhole * step ? 1 : (cap + kPaMinSteps * step - 1) / (kPaMinSteps * step);
  const bool split = S * p.units <= kPaMaxSplit && most > 1;  // most: parts of a full sequence
  p.fit = split && S <= 64 && S * p.units * 2 <= kCUs;
  p.target = !split ? 0 : p.fit ? kCUs : kPaParts;
  p.grid = S * p.units;
  if (split) p.grid = p.grid * most < p.grid + p.target ? p.grid * most : p.grid + p.target;
  return p;
}
static size_t pa_part_bytes(const PagedPlan& p, int HD) { return p.target ? (size_t)p.grid * 16 * p.nr * (HD + 4) * 4 : 0; }

int paged_attention_f16(const PagedCall& a) { return paged_attention_cache<__half>(a); }

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
  const size_t lds = pa_lds(HD, p.nr, p.nw, c16, x32);
  if (int rc = require_lds("paged_attention", lds + 4096)) return rc;
  int* counters = static_cast<int*>(workspace);
  float* parts = part ? reinterpret_cast<float*>(static_cast<char*>(workspace) + kCounterBytes) : nullptr;
  int lshift = 0;  // lanes of a sequence, where there are fewer of them than lanes
  while (lshift < 6 && (int64_t)S << (lshift + 1) <= 64) ++lshift;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  // one launch, but it writes to the workspace: not between the launches of another thread's call
  std::unique_lock<std::mutex> whole(stream_lock(st), std::defer_lock);
  if (part) whole.lock();
  const PagedCall call = {q,      cache, positions, pages, out, S,   T,        NH,    NKV,    HD,  p.tiles, num_pages, page, max_pages,
                          lshift, p.target, p.fit, p.nr, p.nw, scale, x32, counters, parts, p.grid, lds, st};
  return c16 ? paged_attention_f16(call) : paged_attention_f32(call);
}
