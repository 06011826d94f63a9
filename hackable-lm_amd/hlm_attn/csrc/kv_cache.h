// The 8-bit key/value cache and the arguments of the kernels over it.
//
// One layer's cache of B sequences, Hkv heads of D values and S slots (token
// positions, a multiple of 64).  A row x (one token's key or value of one kv
// head) is held as whole numbers c = -127 .. 127, stored as the bytes c + 128,
// and one fp32 scale:
//     a = max |x_d|,   scale = a / 127,   c_d = 127 x_d / a  (nearest, ties to even),
// so x_d ~ c_d scale with an error of at most half a scale.  A row whose a is
// below 2^-119 is held as zeros (its scale would leave the normal fp32 range);
// one that holds an infinity or a NaN gets the scale NaN and reads as NaN.
//
//   keys    k  bytes (B, Hkv, S / 16, D / 16, 16, 16): [token / 16][dim / 16][token % 16][dim % 16]
//   values  v  bytes (B, Hkv, S / 64, D / 16, 4, 16, 16): blocks of 64 tokens,
//              [dim / 16][token / 4 % 4][dim % 16][4 (token / 16) + token % 4]
//   k_scale, v_scale  fp32 (B, Hkv, S)
//
// A 64-token block of one head is 64 D contiguous bytes of either, in the order
// in which the attention's matrix operands want them (cached_attn.hip): the
// products contract q.k over D and p.v over tokens, and each load instruction of
// 16 bytes a lane reads 1 KB as it lies, without a pass through LDS.
//
// Token t of sequence b lies at position starts[b] + t (`start` for all
// sequences where starts is null).  Tokens t >= counts[b], and positions
// outside 0 .. S - 1, are padding: they are not written, read as zeros, and
// their queries' output rows are zeros.
#pragma once

#include "attn_common.h"

namespace hlm {

constexpr int kCacheBlock = 64;  // tokens of a block
// The byte of (token, dim) within a head's keys or values.
template <int D>
__device__ __forceinline__ int64_t key_byte(int token, int d) {
  return (int64_t)(token >> 4) * (16 * D) + (d >> 4) * 256 + (token & 15) * 16 + (d & 15);
}
template <int D>
__device__ __forceinline__ int64_t value_byte(int token, int d) {
  return (int64_t)(token >> 6) * (64 * D) + (d >> 4) * 1024 + (token >> 2 & 3) * 256 + (d & 15) * 16 +
         (token >> 4 & 3) * 4 + (token & 3);
}
constexpr float kCacheTiny = 1.504632769052528e-36f;  // 2^-119

// x op'ed over 8 neighbouring lanes, for all of them, without LDS (DPP: the
// other of a pair, the other pair of a quad, the mirrored quad).
template <int CTRL, class T>
__device__ __forceinline__ T dpp(T x) {
  return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}
template <class T, class Op>
__device__ __forceinline__ T over_8_lanes(T x, Op op) {
  x = op(x, dpp<0xb1>(x));      // quad_perm 1 0 3 2
  x = op(x, dpp<0x4e>(x));      // quad_perm 2 3 0 1
  return op(x, dpp<0x141>(x));  // row_half_mirror
}
struct Max {
  __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); }
  __device__ __forceinline__ int operator()(int a, int b) const { return max(a, b); }
};

struct KvCache {
  uint8_t* k;
  uint8_t* v;
  float* ks;
  float* vs;
  int slots;
};

// The new tokens' places.
struct CacheSpan {
  const int* starts;
  const int* counts;  // null: T each
  int start;
  int T;
};

// The position of token t of sequence b, or -1 for padding.
__device__ __forceinline__ int64_t span_start(const CacheSpan& s, int b) { return s.starts ? s.starts[b] : s.start; }
__device__ __forceinline__ int span_count(const CacheSpan& s, int b) {  // 0 .. T
  return s.counts ? max(0, min(s.counts[b], s.T)) : s.T;
}
__device__ __forceinline__ int cache_position(int64_t start, int count, int t, int slots) {
  const int64_t p = start + t;
  return t < count && p >= 0 && p < slots ? (int)p : -1;
}

struct CacheIoArgs {
  KvCache cache;
  CacheSpan span;
  const bf16* k;  // write: inputs (B, T, Hkv, D), unit D stride
  const bf16* v;
  int64_t sk[3], sv[3];
  bf16* k_out;  // read: outputs (B, T, Hkv, D), contiguous
  bf16* v_out;
  int B, Hkv;
  int blocks;  // 64-token blocks that T tokens can touch
};

struct CachedAttnArgs {
  const bf16* q;
  int64_t sq[3];
  bf16* o;  // (B, T, H, D), contiguous
  KvCache own, prefix;  // prefix of one sequence; prefix.slots 0: none
  CacheSpan span;
  int B, H, Hkv, G;
  int P;       // prefix tokens
  int window;  // >= 1
  float scale_part;  // scale log2(e) = scale_part 2^scale_exp, scale_part in 0.5 .. 1
  int scale_exp;
  FastDiv div_G, div_T;
  int variant, prefix_variant;  // of the kernel, by its rows (-1: no prefix, -2: with the own keys)
  // Splits of the keys: own_splits workgroups share a sequence's keys (for one
  // tile of its rows), prefix_splits the prefix's.
  int own_splits, prefix_splits, own_tiles, prefix_tiles, prefix_items;
  float* part_o;   // (splits, B T H, D), unnormalised
  float* part_ml;  // (splits, B T H, 2): running maximum in log2 units and sum
};

}  // namespace hlm
