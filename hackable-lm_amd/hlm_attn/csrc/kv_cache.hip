// Writing tokens into the 8-bit cache of kv_cache.h and reading them back.
//
// Per row x of D values: a = max |x_d|, c_d = 127 x_d / a to the nearest.  The
// kernels form it as x_d r with r = 127 / a rounded up, x r exact (a fused
// multiply-add).  That gives the same whole number: with x and a of 8
// significant bits, 127 x / a lies on a half-integer or keeps off it by 1 / 510
// of x's own power of two, far more than the 2^-23 by which x r is off.  It lies
// on one, 254 x = (2 k + 1) a, only if 127 divides 2 k + 1 or a's significand:
// at 63.5 (x = a / 2), which r from above takes to 64 like ties to even, or
// where that significand is 254, r a power of two and x r exact.
//
// Memory-bound: 4 D bytes in and 2 (D + 4) out per token and head to write, the
// reverse to read.  On an MI355X: 8 sequences of 1024 to 2048 tokens, 12 heads of
// 64, written in 16.5 us (57.8 MB, 3.5 TB/s), read in 11.9 (70.4 MB with the
// padding's zeros, 5.9 TB/s); 4 x 4096 tokens of 12 heads of 128 read in 24.9 us
// (6.1 TB/s).  One token of 16 sequences: 4.1 and 3.4 us, a launch and one trip to
// memory.
#include "kv_cache.h"

namespace hlm {
namespace {

// From this many tokens on, whole blocks; below, rows.  64 sequences of 12 heads
// of 64, one to 64 tokens each: rows 4.1 (1), 5.8 (8), 9.2 (16), 23.6 us (64),
// blocks 5.3, 7.2, 8.0, 10.8.
constexpr int kBlockTokens = 16;

// One row of D values over D / 8 lanes, 8 values each: dwords whose last byte is
// the code, and the row's scale.
template <int D>
__device__ __forceinline__ void encode8(const bf16x8& x, unsigned u[8], float& scale) {
  typedef __attribute__((ext_vector_type(8))) unsigned short u16x8;
  const u16x8 bits = __builtin_bit_cast(u16x8, x);
  int top = 0;  // as bits, so that a NaN is the largest
#pragma unroll
  for (int e = 0; e < 8; ++e) top = max(top, (int)(bits[e] & 0x7fff));
  top = over_8_lanes(top, Max());
  if constexpr (D == 128) top = max(top, dpp<0x140>(top));  // row_mirror
  const float a = __builtin_bit_cast(float, top << 16);
  const bool finite = top < 0x7f80, tiny = a < kCacheTiny;
  float r = tiny || !finite ? 0.f : 127.f / a;
  if (fmaf(r, a, -127.f) < 0.f && r > 0.f) r = __builtin_bit_cast(float, __builtin_bit_cast(int, r) + 1);
  scale = !finite ? __builtin_nanf("") : tiny ? 0.f : a / 127.f;
  // x r + 1.5 2^23 + 128: the sum's last bits are the whole number + 128
#pragma unroll
  for (int e = 0; e < 8; ++e)
    u[e] = __builtin_bit_cast(unsigned, fmaf(finite ? (float)x[e] : 0.f, r, 12582912.f + 128.f));
}

// The last bytes of four dwords as one.
__device__ __forceinline__ unsigned last_bytes(unsigned a, unsigned b, unsigned c, unsigned d) {
  return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, 0x0c0c0400u), __builtin_amdgcn_perm(b, a, 0x0c0c0400u), 0x05040100u);
}

// One row to D / 8 lanes; a workgroup takes 2048 / D rows of k or of v
// (blockIdx.y).
template <int D>
__global__ __launch_bounds__(256) void cache_write_rows_kernel(CacheIoArgs p) {
  constexpr int LPR = D / 8;
  const bool is_v = blockIdx.y != 0;
  const int64_t row = (int64_t)blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
  const int c = threadIdx.x % LPR;
  if (row >= (int64_t)p.B * p.span.T * p.Hkv) return;
  const int h = (int)(row % p.Hkv);
  const int64_t bt = row / p.Hkv;
  const int t = (int)(bt % p.span.T), b = (int)(bt / p.span.T);
  const int pos = cache_position(span_start(p.span, b), span_count(p.span, b), t, p.cache.slots);
  if (pos < 0) return;
  const int64_t* s = is_v ? p.sv : p.sk;
  const bf16x8 x = *reinterpret_cast<const bf16x8*>((is_v ? p.v : p.k) + b * s[0] + t * s[1] + h * s[2] + 8 * c);
  unsigned u[8];
  float scale;
  encode8<D>(x, u, scale);
  const int64_t head = ((int64_t)b * p.Hkv + h) * p.cache.slots;
  if (c == 0) (is_v ? p.cache.vs : p.cache.ks)[head + pos] = scale;
  if (!is_v) {
    *reinterpret_cast<uint2*>(p.cache.k + head * D + key_byte<D>(pos, 8 * c)) =
        make_uint2(last_bytes(u[0], u[1], u[2], u[3]), last_bytes(u[4], u[5], u[6], u[7]));
  } else {
    uint8_t* to = p.cache.v + head * D + value_byte<D>(pos, 8 * c);
#pragma unroll
    for (int e = 0; e < 8; ++e) to[16 * e] = (uint8_t)u[e];
  }
}

template <int D>
__global__ __launch_bounds__(256) void cache_read_rows_kernel(CacheIoArgs p) {
  constexpr int LPR = D / 8;
  const bool is_v = blockIdx.y != 0;
  const int64_t row = (int64_t)blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
  const int c = threadIdx.x % LPR;
  if (row >= (int64_t)p.B * p.span.T * p.Hkv) return;
  const int h = (int)(row % p.Hkv);
  const int64_t bt = row / p.Hkv;
  const int t = (int)(bt % p.span.T), b = (int)(bt / p.span.T);
  const int pos = cache_position(span_start(p.span, b), span_count(p.span, b), t, p.cache.slots);
  bf16x8 x = {};
  if (pos >= 0) {
    const int64_t head = ((int64_t)b * p.Hkv + h) * p.cache.slots;
    const float scale = (is_v ? p.cache.vs : p.cache.ks)[head + pos];
    uint8_t code[8];
    if (!is_v) {
      *reinterpret_cast<uint2*>(code) = *reinterpret_cast<const uint2*>(p.cache.k + head * D + key_byte<D>(pos, 8 * c));
    } else {
      const uint8_t* from = p.cache.v + head * D + value_byte<D>(pos, 8 * c);
#pragma unroll
      for (int e = 0; e < 8; ++e) code[e] = from[16 * e];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = (bf16)((float)((int)code[e] - 128) * scale);
  }
  *reinterpret_cast<bf16x8*>((is_v ? p.v_out : p.k_out) + row * D + 8 * c) = x;
}

// Many tokens: one workgroup per (sequence, head, 64-token block), whose image
// is put together in LDS and moves as 16 contiguous bytes a thread.  Half of the
// threads take the keys, half the values; a thread holds 8 dims of 4 consecutive
// tokens.  The image's 256-byte pieces are 272 bytes apart in LDS, so that the
// lanes of a store fall on different banks (two to a bank at most).  bf16 rows
// pass by the caches' retention (8 sequences of up to 2048 tokens written and read
// back: 30.4 -> 28.3 us; 4 x 4096 of 12 heads of 128 read: 28.4 -> 25.4); codes do
// not (1.4 us more for the former with their loads past them too).
template <int D>
struct Block {
  int64_t head;  // this head's first slot
  int b, h, count;
  int64_t start, first;  // of the sequence; the block's first position
  int lo, hi;            // its tokens lo .. hi - 1 are real

  __device__ __forceinline__ explicit Block(const CacheIoArgs& p) {
    const int id = blockIdx.x, bn = id / p.Hkv;
    h = id - bn * p.Hkv;
    b = bn / p.blocks;
    start = span_start(p.span, b);
    count = span_count(p.span, b);
    first = ((start >> 6) + (bn - b * p.blocks)) * kCacheBlock;
    head = ((int64_t)b * p.Hkv + h) * p.cache.slots;
    lo = hi = 0;
    if (first < 0 || first >= p.cache.slots) return;
    lo = (int)max((int64_t)0, start - first);
    hi = (int)min((int64_t)kCacheBlock, start + count - first);
  }
};

constexpr int kPiece = 272;  // bytes of LDS for 256
// The LDS byte of byte i of a block.
__device__ __forceinline__ int piece_byte(int i) { return (i >> 8) * kPiece + (i & 255); }

// Bytes j of four dwords as one dword.
template <int J>
__device__ __forceinline__ unsigned gather_bytes(unsigned a, unsigned b, unsigned c, unsigned d) {
  constexpr unsigned sel = (4 + J) << 8 | J;
  return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, sel), __builtin_amdgcn_perm(b, a, sel), 0x05040100u);
}

template <int D>
__global__ __launch_bounds__(4 * D) void cache_write_blocks_kernel(CacheIoArgs p) {
  constexpr int LPR = D / 8;
  __shared__ __align__(16) uint8_t image[2][D / 4 * kPiece];
  const Block<D> blk(p);
  if (blk.lo >= blk.hi) return;
  const bool is_v = threadIdx.x >= 2 * D;
  const int u = threadIdx.x % (2 * D), c = u % LPR, quad = u / LPR;
  const int64_t* s = is_v ? p.sv : p.sk;
  const bf16* from = (is_v ? p.v : p.k) + blk.b * s[0] + (blk.first - blk.start) * s[1] + blk.h * s[2] + 8 * c;
  bf16x8 x[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int i = 4 * quad + j;
    x[j] = bf16x8{};
    if (i >= blk.lo && i < blk.hi) x[j] = __builtin_nontemporal_load(reinterpret_cast<const bf16x8*>(from + i * s[1]));
  }
  unsigned u4[4][8];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int i = 4 * quad + j;
    float scale;
    encode8<D>(x[j], u4[j], scale);
    if (c == 0 && i >= blk.lo && i < blk.hi) (is_v ? p.cache.vs : p.cache.ks)[blk.head + blk.first + i] = scale;
  }
  if (!is_v) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const unsigned* w = u4[j];
      *reinterpret_cast<uint2*>(image[0] + piece_byte((int)key_byte<D>(4 * quad + j, 8 * c))) =
          make_uint2(last_bytes(w[0], w[1], w[2], w[3]), last_bytes(w[4], w[5], w[6], w[7]));
    }
  } else {
    uint8_t* to = image[1] + piece_byte((int)value_byte<D>(4 * quad, 8 * c));
#pragma unroll
    for (int e = 0; e < 8; ++e)
      *reinterpret_cast<unsigned*>(to + 16 * e) = last_bytes(u4[0][e], u4[1][e], u4[2][e], u4[3][e]);
  }
  __syncthreads();
  const int64_t base = (blk.head + blk.first) * D;
  const bool full = blk.lo == 0 && blk.hi == kCacheBlock;
  const int byte = 16 * threadIdx.x;  // of 64 D
  const u32x4 kw = *reinterpret_cast<const u32x4*>(image[0] + piece_byte(byte));
  const u32x4 vw = *reinterpret_cast<const u32x4*>(image[1] + piece_byte(byte));
  // 16 bytes of keys are one token's
  const int token = (byte / (16 * D)) * 16 + (byte / 16) % 16;
  if (full || (token >= blk.lo && token < blk.hi)) *reinterpret_cast<u32x4*>(p.cache.k + base + byte) = kw;
  if (full) {
    *reinterpret_cast<u32x4*>(p.cache.v + base + byte) = vw;
  } else {  // 16 bytes of values are tokens 16 t + 4 g + i, byte 4 t + i; four at a time where all are real
    const int g = byte / 256 % 4;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int i = 16 * t + 4 * g;
      uint8_t* to = p.cache.v + base + byte + 4 * t;
      if (i >= blk.lo && i + 4 <= blk.hi) {
        *reinterpret_cast<unsigned*>(to) = vw[t];
      } else {  // others' bytes are left alone, not rewritten: a call on another stream may own them
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (i + k >= blk.lo && i + k < blk.hi) to[k] = (uint8_t)(vw[t] >> (8 * k));
      }
    }
  }
}

// Eight codes times a scale.
__device__ __forceinline__ bf16x8 decode8(unsigned lo, unsigned hi, float scale) {
  bf16x8 x;
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = (bf16)((float)((int)(((e < 4 ? lo : hi) >> (8 * (e % 4))) & 0xff) - 128) * scale);
  return x;
}

template <int D>
__global__ __launch_bounds__(4 * D) void cache_read_blocks_kernel(CacheIoArgs p) {
  constexpr int LPR = D / 8;
  __shared__ __align__(16) uint8_t image[2][D / 4 * kPiece];
  const Block<D> blk(p);
  const bool is_v = threadIdx.x >= 2 * D;
  const int u = threadIdx.x % (2 * D), c = u % LPR, quad = u / LPR;
  const bool any = blk.lo < blk.hi;
  uint2 kc[4];
  float scale[4];
  if (any) {  // a block with a real token lies in the cache, all of it
    const int64_t base = (blk.head + blk.first) * D;
    const int byte = 16 * threadIdx.x;
    const u32x4 kw = *reinterpret_cast<const u32x4*>(p.cache.k + base + byte);
    const u32x4 vw = *reinterpret_cast<const u32x4*>(p.cache.v + base + byte);
    const f32x4 sc = *reinterpret_cast<const f32x4*>((is_v ? p.cache.vs : p.cache.ks) + blk.head + blk.first + 4 * quad);
    *reinterpret_cast<u32x4*>(image[0] + piece_byte(byte)) = kw;
    *reinterpret_cast<u32x4*>(image[1] + piece_byte(byte)) = vw;
#pragma unroll
    for (int j = 0; j < 4; ++j) scale[j] = sc[j];
  }
  __syncthreads();
  if (any && !is_v) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      kc[j] = *reinterpret_cast<const uint2*>(image[0] + piece_byte((int)key_byte<D>(4 * quad + j, 8 * c)));
  }
  if (any && is_v) {
    const uint8_t* from = image[1] + piece_byte((int)value_byte<D>(4 * quad, 8 * c));
    unsigned w[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = *reinterpret_cast<const unsigned*>(from + 16 * e);
    kc[0] = make_uint2(gather_bytes<0>(w[0], w[1], w[2], w[3]), gather_bytes<0>(w[4], w[5], w[6], w[7]));
    kc[1] = make_uint2(gather_bytes<1>(w[0], w[1], w[2], w[3]), gather_bytes<1>(w[4], w[5], w[6], w[7]));
    kc[2] = make_uint2(gather_bytes<2>(w[0], w[1], w[2], w[3]), gather_bytes<2>(w[4], w[5], w[6], w[7]));
    kc[3] = make_uint2(gather_bytes<3>(w[0], w[1], w[2], w[3]), gather_bytes<3>(w[4], w[5], w[6], w[7]));
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int i = 4 * quad + j;
    const int64_t t = blk.first - blk.start + i;
    if (t < 0 || t >= p.span.T) continue;
    bf16x8 x = {};
    if (i >= blk.lo && i < blk.hi) x = decode8(kc[j].x, kc[j].y, scale[j]);
    __builtin_nontemporal_store(x, reinterpret_cast<bf16x8*>((is_v ? p.v_out : p.k_out) + (((int64_t)blk.b * p.span.T + t) * p.Hkv + blk.h) * D + 8 * c));
  }
}

}  // namespace

template <int D>
hipError_t launch_cache_io(CacheIoArgs& p, bool write, hipStream_t stream) {
  const int64_t rows = (int64_t)p.B * p.span.T * p.Hkv;
  p.blocks = (p.span.T + 2 * kCacheBlock - 2) / kCacheBlock;
  if (p.span.T >= kBlockTokens) {
    const dim3 grid((unsigned)((int64_t)p.B * p.Hkv * p.blocks)), block(4 * D);
    if (write)
      hipLaunchKernelGGL((cache_write_blocks_kernel<D>), grid, block, 0, stream, p);
    else
      hipLaunchKernelGGL((cache_read_blocks_kernel<D>), grid, block, 0, stream, p);
    return hipGetLastError();
  }
  const dim3 grid((unsigned)((rows + 2048 / D - 1) / (2048 / D)), 2);
  if (write)
    hipLaunchKernelGGL((cache_write_rows_kernel<D>), grid, dim3(256), 0, stream, p);
  else
    hipLaunchKernelGGL((cache_read_rows_kernel<D>), grid, dim3(256), 0, stream, p);
  return hipGetLastError();
}
template hipError_t launch_cache_io<64>(CacheIoArgs&, bool, hipStream_t);
template hipError_t launch_cache_io<128>(CacheIoArgs&, bool, hipStream_t);

}  // namespace hlm
