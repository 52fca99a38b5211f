// The 4-bit key-value cache (layout in include/miq.h): per kv head, records of 40 HD bytes for 32
// positions. A group of 32 consecutive dimensions of one position shares two fp16 numbers S and Z, and
// a code c stands for fp16(S (1 + c / 16) + Z). In that form a code needs no conversion: OR-ed into bits
// 6..9 of 1.0 it is the fp16 number 1 + c / 16, and one packed fma makes two values of it.
//
// The record's order is that of the matrix-core operands (v_mfma_f32_16x16x32_f16, whose lane (i, g) =
// (lane % 16, lane / 16) holds 8 consecutive k of row i): a word is one lane's 8 codes, the lanes' words
// lie 16 bytes a lane, so that a wave reads 1 KB at a time and unpacks operands with no exchange. For
// S^T = K Q^T a key word holds 8 dimensions of one key; for O^T = V^T P^T a value word holds one dimension
// of the 8 keys whose scores that lane has in the two 16-key tiles of S^T.
#pragma once
#include "miq_common.h"

namespace miq {

constexpr int kKv4Block = 32;        // positions of a record
constexpr float kKv4Max = 16384.f;   // larger magnitudes saturate: S and Z stay finite in fp16
constexpr uint16_t kKv4Bad = 0xFE00; // S of a group with a NaN or an infinity: a NaN, and the only S with a sign

__host__ __device__ constexpr size_t kv4_record(int HD) { return (size_t)40 * HD; }
__host__ __device__ inline int kv4_blocks(int LMAX) { return (LMAX + kKv4Block - 1) / kKv4Block; }
// bytes from a record's start to its parts
__host__ __device__ constexpr int kv4_vcodes(int HD) { return 16 * HD; }
__host__ __device__ constexpr int kv4_kmeta(int HD) { return 32 * HD; }
__host__ __device__ constexpr int kv4_vmeta(int HD) { return 36 * HD; }
// byte of word n of lane (i, g) among the codes
__host__ __device__ constexpr int kv4_word(int n, int g, int i) { return (((n >> 2) * 64 + g * 16 + i) * 4 + (n & 3)) * 4; }
// bit of code e of a word: pairs (2 p, 2 p + 1) in the two halves
__host__ __device__ constexpr int kv4_shift(int e) { return 4 * (e >> 1) + 16 * (e & 1); }
// position within its block of key e of lane group g
__host__ __device__ constexpr int kv4_key(int g, int e) { return 16 * (e >> 2) + 4 * g + (e & 3); }

// whether two ranges of bytes share any
inline bool share_bytes(const void* a, size_t na, const void* b, size_t nb) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return x < y + nb && y < x + na;
}

inline bool kv4_head(int HD) { return HD == 64 || HD == 128 || HD == 192 || HD == 256; }

// The fp16 numbers 1 + c / 16 of code pair p of a word.
template <int P> __device__ __forceinline__ half2v kv4_pair(uint32_t w) {
  const uint32_t s = P == 0 ? w << 6 : P == 1 ? w << 2 : P == 2 ? w >> 2 : w >> 6;
  return as_h2(and_or(s, 0x03C003C0u, 0x3C003C00u));
}
__device__ __forceinline__ half2v fma2(half2v a, half2v b, half2v c) { return __builtin_elementwise_fma(a, b, c); }

// (maximum) over each half wave of 32 lanes
__device__ __forceinline__ float half_wave_max(float v) {
  v = fmaxf(v, dpp_move<0xB1>(v));
  v = fmaxf(v, dpp_move<0x4E>(v));
  v = fmaxf(v, dpp_move<0x141>(v));
  v = fmaxf(v, dpp_move<0x140>(v));
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}

// Code, S and Z of one value of a group held by the 32 lanes of a half wave, one value each. Every
// operation is a single IEEE fp32 operation, so that the codes are the same wherever the rule is computed.
// The bound |lo| / 128 keeps a step (S / 16) from falling below an fp16 ulp of the values, where it could
// not help, and keeps S (1 + c / 16) + Z exact in fp32.
__device__ __forceinline__ uint32_t kv4_quantize(float x, uint16_t& S, uint16_t& Z) {
#pragma clang fp contract(off)
  const uint64_t odd = __ballot(!(fabsf(x) < INFINITY));
  const bool bad = (uint32_t)((threadIdx.x & 32) ? odd >> 32 : odd) != 0;
  x = fminf(fmaxf(x, -kKv4Max), kKv4Max);
  const float hi = half_wave_max(x), lo = -half_wave_max(-x);
  const __half s = __float2half_rn(fmaxf((hi - lo) * 16.f / 15.f, fabsf(lo) * (1.f / 128.f)));
  const float sf = __half2float(s);
  const __half z = __float2half_rn(lo - sf);
  S = bad ? kKv4Bad : __half_as_ushort(s);
  Z = bad ? kKv4Bad : __half_as_ushort(z);
  const float c = fminf(fmaxf(rintf((x - __half2float(z)) / sf * 16.f) - 16.f, 0.f), 15.f);
  return !bad && sf > 0.f ? (uint32_t)c : 0u;  // no branch: calls on several groups overlap
}

}  // namespace miq
