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
// reverse to read.
#include "kv_cache.h"

namespace hlm {
namespace {

// One row of D values over D / 8 lanes, 8 values each: the codes as two dwords
// and the row's scale.
template <int D>
__device__ __forceinline__ void encode8(const bf16x8& x, unsigned code[2], float& scale) {
  typedef __attribute__((ext_vector_type(8))) unsigned short u16x8;
  const u16x8 bits = __builtin_bit_cast(u16x8, x);
  int top = 0;  // as bits, so that a NaN is the largest
#pragma unroll
  for (int e = 0; e < 8; ++e) top = max(top, (int)(bits[e] & 0x7fff));
#pragma unroll
  for (int m = D / 16; m >= 1; m >>= 1) top = max(top, __shfl_xor(top, m));
  const float a = __builtin_bit_cast(float, top << 16);
  const bool finite = top < 0x7f80, tiny = a < kCacheTiny;
  float r = tiny || !finite ? 0.f : 127.f / a;
  if (fmaf(r, a, -127.f) < 0.f && r > 0.f) r = __builtin_bit_cast(float, __builtin_bit_cast(int, r) + 1);
  scale = !finite ? __builtin_nanf("") : tiny ? 0.f : a / 127.f;
  // x r + 1.5 2^23 + 128: the sum's last bits are the whole number + 128
  unsigned u[8];
#pragma unroll
  for (int e = 0; e < 8; ++e)
    u[e] = __builtin_bit_cast(unsigned, fmaf(finite ? (float)x[e] : 0.f, r, 12582912.f + 128.f)) & 0xff;
#pragma unroll
  for (int i = 0; i < 2; ++i) code[i] = u[4 * i] | u[4 * i + 1] << 8 | u[4 * i + 2] << 16 | u[4 * i + 3] << 24;
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
  unsigned code[2];
  float scale;
  encode8<D>(x, code, scale);
  const int64_t head = ((int64_t)b * p.Hkv + h) * p.cache.slots;
  if (c == 0) (is_v ? p.cache.vs : p.cache.ks)[head + pos] = scale;
  if (!is_v) {
    *reinterpret_cast<uint2*>(p.cache.k + (head + pos) * D + 8 * c) = make_uint2(code[0], code[1]);
  } else {
    uint8_t* to = p.cache.v + (head + (pos & ~63)) * D + (pos & 63) + (8 * c) * 64;
#pragma unroll
    for (int e = 0; e < 8; ++e) to[64 * e] = (uint8_t)(code[e / 4] >> (8 * (e % 4)));
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
      *reinterpret_cast<uint2*>(code) = *reinterpret_cast<const uint2*>(p.cache.k + (head + pos) * D + 8 * c);
    } else {
      const uint8_t* from = p.cache.v + (head + (pos & ~63)) * D + (pos & 63) + (8 * c) * 64;
#pragma unroll
      for (int e = 0; e < 8; ++e) code[e] = from[64 * e];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = (bf16)((float)((int)code[e] - 128) * scale);
  }
  *reinterpret_cast<bf16x8*>((is_v ? p.v_out : p.k_out) + row * D + 8 * c) = x;
}

}  // namespace

template <int D>
hipError_t launch_cache_io(const CacheIoArgs& p, bool write, hipStream_t stream) {
  const int64_t rows = (int64_t)p.B * p.span.T * p.Hkv;
  const dim3 grid((unsigned)((rows + 2048 / D - 1) / (2048 / D)), 2);
  if (write)
    hipLaunchKernelGGL((cache_write_rows_kernel<D>), grid, dim3(256), 0, stream, p);
  else
    hipLaunchKernelGGL((cache_read_rows_kernel<D>), grid, dim3(256), 0, stream, p);
  return hipGetLastError();
}
template hipError_t launch_cache_io<64>(const CacheIoArgs&, bool, hipStream_t);
template hipError_t launch_cache_io<128>(const CacheIoArgs&, bool, hipStream_t);

}  // namespace hlm
