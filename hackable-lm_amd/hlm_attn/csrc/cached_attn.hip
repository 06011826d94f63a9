// Attention of new tokens over the 8-bit cache of kv_cache.h, with an optional
// prefix that all sequences share.
//
// Query row r of sequence b at position p sees keys j = max(0, p - W + 1) .. p
// of the sequence (with a prefix of P tokens, positions 0 .. P - 1 are the
// prefix's and the sequence's own follow):
//   o = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),   s_j = scale q.k_j.
// With k_j = kc_j ks_j and v_j = vc_j vs_j (whole numbers and scales),
//   s_j = scale ks_j (q.kc_j),   sum_j p_j v_j = sum_j (p_j vs_j) vc_j,
// so the matrix products run on the whole numbers, which fp16 holds exactly,
// and the scales multiply fp32 scores and probabilities.
//
// One workgroup takes 16 NT rows (the query heads of one kv head, of one or
// more tokens; for the prefix, of all sequences) and a share of their keys in
// blocks of 64; its four waves take the share's blocks in turn and their sums
// are joined in LDS, those of several workgroups by the combine kernel.
//
// Layouts (v_mfma_f32_16x16x32_f16, lane l, n = l % 16, g = l / 16):
//   A (16 x 32): row n, k = 8 g + e;  B (32 x 16): k = 8 g + e, column n;
//   C (16 x 16): column n, rows 4 g + i.
// Scores are formed transposed, keys by rows: tile t's row 4 g' + i is the
// block's key 16 g' + 4 t + i, so lane (n, g) ends up with the scores of query
// row n and the 16 consecutive keys 16 g .. 16 g + 15 in its 4 tiles.  Rounded
// to fp16 they are the B operand of o^T = v^T p^T as they are, if its k slot
// 8 g + e is key 16 g + 8 h + e in half h; lane (n, g) then needs the values of
// dim n and the same 16 keys, 16 contiguous bytes of the transposed block.
// A score's maximum, sum and rescaling stay in the lane, but for the maximum
// over the four g.
//
// Numerics.  q is scaled by a power of two to at most 2 per row and then held
// in fp16 (exact but for values 2^-14 of the row's largest and below, whose
// error is 2^-25 of it); whole numbers are exact; products and sums are fp32.
// p_j vs_j is rounded to fp16 relative to the largest vs so far, 2^12 at
// p = 1: 11 bits for p above 2^-26, and no weight above 2^-37 is lost.
#include <utility>

#include "kv_cache.h"

namespace hlm {
namespace {

typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;

constexpr float kWeightTop = 4096.f;  // a probability of 1 as fp16
// The running maximum is moved only when a score passes it by 2^3: weights
// reach 2^15, within fp16, and the sums stay where they are meanwhile.
constexpr float kSlack = 3.f;

__device__ __forceinline__ f32x4 mfma16(f16x8 a, f16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// Lane 16 g + J of each group of 16, for all of the group (DPP row_newbcast).
template <int J>
__device__ __forceinline__ float row_lane(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x150 + J, 0xf, 0xf, true));
}

// f(0), .. f(N - 1) with compile-time arguments.
template <class F, int... E>
__device__ __forceinline__ void each_of(F f, std::integer_sequence<int, E...>) {
  (f(std::integral_constant<int, E>{}), ...);
}
template <int N, class F>
__device__ __forceinline__ void each(F f) {
  each_of(f, std::make_integer_sequence<int, N>{});
}

__device__ __forceinline__ float max_over_groups(float x) {
  x = fmaxf(x, __shfl_xor(x, 16));
  return fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float sum_over_groups(float x) {
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}

// Four codes (bytes c + 128) as fp16 whole numbers: 0x6400 | byte is 1024 + byte.
__device__ __forceinline__ void decode4(unsigned b, f16x2& lo, f16x2& hi) {
  const f16x2 off = {(_Float16)-1152.f, (_Float16)-1152.f};
  lo = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, b, 0x04010400u)) + off;
  hi = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, b, 0x04030402u)) + off;
}
__device__ __forceinline__ f16x8 decode8(unsigned b0, unsigned b1) {
  f16x2 a, b, c, d;
  decode4(b0, a, b);
  decode4(b1, c, d);
  return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// The keys of one workgroup: a head's rows of a cache, and which rows see them.
struct Keys {
  const uint8_t* k;
  const uint8_t* v;
  const float* ks;
  const float* vs;
};

// A query row: where it lies in q (null: padding or past the end) and which
// keys lo .. hi of the segment it sees.
struct Row {
  const bf16* q;
  int lo, hi;
};

template <bool PREFIX>
__device__ __forceinline__ Row row_of(const CachedAttnArgs& p, int unit, int r, int64_t& out) {
  int bt, b, t, h;
  const int rt = fast_div(r, p.div_G), g = r - rt * p.G;
  if constexpr (PREFIX) {
    bt = rt;
    b = fast_div(bt, p.div_T);
    t = bt - b * p.span.T;
    h = unit;
  } else {
    b = unit / p.Hkv;
    h = unit - b * p.Hkv;
    t = rt;
    bt = b * p.span.T + t;
  }
  const int head = h * p.G + g;
  out = (int64_t)bt * p.H + head;
  const int pos = cache_position(span_start(p.span, b), span_count(p.span, b), t, p.own.slots);
  Row row{nullptr, 0x7fffffff, -1};
  if (pos < 0) return row;
  row.q = p.q + b * p.sq[0] + t * p.sq[1] + head * p.sq[2];
  const int64_t from = (int64_t)pos - p.window + 1;
  if constexpr (PREFIX) {
    const int64_t lo = from + p.P;
    row.hi = p.P - 1;
    row.lo = (int)min((int64_t)p.P, max((int64_t)0, lo));
  } else {
    row.hi = pos;
    row.lo = (int)max((int64_t)0, from);
  }
  return row;
}

template <int D, int NT, bool PREFIX>
__device__ __forceinline__ void attend(const CachedAttnArgs& p, int unit, int tile, int split, int n_splits, int slot,
                                       bool partial, float* lds) {
  constexpr int C = D / 64, DT = D / 16, ROWS = 16 * NT, LD = D + 4;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, g = lane >> 4;
  const int n_rows = PREFIX ? p.B * p.span.T * p.G : p.span.T * p.G;
  Keys s;
  {
    const KvCache& c = PREFIX ? p.prefix : p.own;
    const int64_t head = (int64_t)unit * c.slots;
    s = {c.k + head * D, c.v + head * D, c.ks + head, c.vs + head};
  }

  // This lane's query rows: their keys, and q in fp16.
  int lo[NT], hi[NT], first = 0x7fffffff, last = -1, inner_first = -1, inner_last = 0x7fffffff;
  f16x8 q[NT][C][2];
  float rs[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int r = tile * ROWS + 16 * nt + n;
    int64_t out;
    Row row{nullptr, 0x7fffffff, -1};
    if (r < n_rows) row = row_of<PREFIX>(p, unit, r, out);
    lo[nt] = row.lo;
    hi[nt] = row.hi;
    if (row.hi >= row.lo) {
      first = min(first, row.lo);
      last = max(last, row.hi);
      inner_first = max(inner_first, row.lo);
      inner_last = min(inner_last, row.hi);
    }
    typedef __attribute__((ext_vector_type(8))) unsigned short u16x8;
    bf16x8 x[C][2];
    int top = 0;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        x[c][h] = bf16x8{};
        if (row.q != nullptr) x[c][h] = *reinterpret_cast<const bf16x8*>(row.q + 64 * c + 16 * g + 8 * h);
        const u16x8 bits = __builtin_bit_cast(u16x8, x[c][h]);
#pragma unroll
        for (int e = 0; e < 8; ++e) top = max(top, (int)(bits[e] & 0x7fff));
      }
    top = max(top, __shfl_xor(top, 16));
    top = max(top, __shfl_xor(top, 32));
    const int ex = min(126, max(-120, (top >> 7) - 127));
    const float down = __builtin_bit_cast(float, (127 - ex) << 23);
    // kept positive and finite: a score of -infinity times it stays what it is
    rs[nt] = fminf(3e38f, fmaxf(1e-37f, p.scale_log2 * __builtin_bit_cast(float, (127 + ex) << 23)));
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 8; ++e) q[nt][c][h][e] = (_Float16)((float)x[c][h][e] * down);
  }
#pragma unroll
  for (int m = 1; m < 16; m <<= 1) {
    first = min(first, __shfl_xor(first, m));
    last = max(last, __shfl_xor(last, m));
    inner_first = max(inner_first, __shfl_xor(inner_first, m));
    inner_last = min(inner_last, __shfl_xor(inner_last, m));
  }
  first = __builtin_amdgcn_readfirstlane(first);
  last = __builtin_amdgcn_readfirstlane(last);
  inner_first = __builtin_amdgcn_readfirstlane(inner_first);
  inner_last = __builtin_amdgcn_readfirstlane(inner_last);

  // This workgroup's blocks begin .. end - 1, shared out evenly.
  int begin = 0, end = 0;
  if (last >= first) {
    const int b0 = first >> 6, blocks = (last >> 6) - b0 + 1;
    const int per = (blocks + n_splits - 1) / n_splits;
    begin = b0 + min(blocks, split * per);
    end = b0 + min(blocks, split * per + per);
  }

  float mt[NT], l[NT], vtop = 0.f;  // running maximum of (q.kc) ks, sum, largest value scale
  f32x4 o[NT][DT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    mt[nt] = -__builtin_inff();
    l[nt] = 0.f;
#pragma unroll
    for (int d = 0; d < DT; ++d) o[nt][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  u32x4 kr[4][C], vr[DT];
  float ksl = 0.f, vsl = 0.f;
  const int key_row = 16 * (n >> 2) + (n & 3);  // + 4 t: this lane's key of tile t as an A row
  auto load_k = [&](int blk) {
    const uint8_t* at = s.k + (int64_t)blk * (64 * D) + key_row * D + 16 * g;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int c = 0; c < C; ++c) kr[t][c] = *reinterpret_cast<const u32x4*>(at + 4 * t * D + 64 * c);
    ksl = s.ks[blk * 64 + lane];
  };
  auto load_v = [&](int blk) {
    const uint8_t* at = s.v + (int64_t)blk * (64 * D) + n * 64 + 16 * g;
#pragma unroll
    for (int d = 0; d < DT; ++d) vr[d] = *reinterpret_cast<const u32x4*>(at + 16 * 64 * d);
    vsl = s.vs[blk * 64 + lane];
  };

  int blk = begin + wave;
  if (blk < end) {
    load_k(blk);
    load_v(blk);
  }
  for (; blk < end; blk += 4) {
    const bool more = blk + 4 < end;
    const int k0 = blk * 64;
    const bool whole = k0 >= inner_first && k0 + 63 <= inner_last;  // every row sees every key
    // scores of all rows
    f32x4 sc[NT][4];
    {
      const float ks = ksl;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        f16x8 kf[C][2];
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int h = 0; h < 2; ++h) kf[c][h] = decode8(kr[t][c][2 * h], kr[t][c][2 * h + 1]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          f32x4 acc{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int c = 0; c < C; ++c)
#pragma unroll
            for (int h = 0; h < 2; ++h) acc = mfma16(kf[c][h], q[nt][c][h], acc);
          sc[nt][t] = acc;
        }
      }
      if (more) load_k(blk + 4);
      each<16>([&](auto e) {
        const float f = row_lane<e>(ks);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) sc[nt][e / 4][e % 4] *= f;
      });
    }
    if (!whole) {  // selected, not added: masked slots may hold any scale
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int key = k0 + 16 * g + 4 * t + i;
            if (key < lo[nt] || key > hi[nt]) sc[nt][t][i] = -__builtin_inff();
          }
    }
    // the values' scales relative to the largest so far
    float vs = vsl;
    if (!whole && (k0 + lane < first || k0 + lane > last)) vs = 0.f;
    float top = vs;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) top = fmaxf(top, __shfl_xor(top, m));
    top = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, top)));
    if (top > vtop) {
      const float f = vtop / top;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int d = 0; d < DT; ++d) o[nt][d] *= f;
      vtop = top;
    }
    vs = vtop > 0.f ? vs * (kWeightTop / vtop) : 0.f * vs;
    // probabilities
    f16x8 w[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float mx = sc[nt][0][0];
#pragma unroll
      for (int e = 1; e < 16; ++e) mx = fmaxf(mx, sc[nt][e / 4][e % 4]);
      if (__any((mx - mt[nt]) * rs[nt] > kSlack)) {
        const float m = fmaxf(mt[nt], max_over_groups(mx));
        const float alpha = m > mt[nt] ? __builtin_amdgcn_exp2f((mt[nt] - m) * rs[nt]) : 1.f;
        mt[nt] = m;
        l[nt] *= alpha;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[nt][d] *= alpha;
      }
      const float off = mt[nt] == -__builtin_inff() ? 0.f : -mt[nt] * rs[nt];
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float pe = __builtin_amdgcn_exp2f(fmaf(sc[nt][e / 4][e % 4], rs[nt], off));
        l[nt] += pe;
        sc[nt][e / 4][e % 4] = pe;
      }
    }
    each<16>([&](auto e) {
      const float f = row_lane<e>(vs);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float pe = sc[nt][e / 4][e % 4];
        w[nt][e / 8][e % 8] = (_Float16)(pe == 0.f ? 0.f : pe * f);
      }
    });
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      const f16x8 v0 = decode8(vr[d][0], vr[d][1]), v1 = decode8(vr[d][2], vr[d][3]);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        o[nt][d] = mfma16(v0, w[nt][0], o[nt][d]);
        o[nt][d] = mfma16(v1, w[nt][1], o[nt][d]);
      }
    }
    if (more) load_v(blk + 4);
  }

  // Join the four waves: maxima and sums, then o relative to the common maximum.
  float* ml = lds;                   // (4, ROWS, 2)
  float* sums = lds + 4 * ROWS * 2;  // (4, ROWS, LD)
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    l[nt] = sum_over_groups(l[nt]);
    if (g == 0) {
      float* at = ml + (wave * ROWS + 16 * nt + n) * 2;
      at[0] = mt[nt] == -__builtin_inff() ? mt[nt] : mt[nt] * rs[nt];
      at[1] = l[nt];
    }
  }
  __syncthreads();
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int r = 16 * nt + n;
    float m = ml[r * 2];
#pragma unroll
    for (int w = 1; w < 4; ++w) m = fmaxf(m, ml[(w * ROWS + r) * 2]);
    const float mine = ml[(wave * ROWS + r) * 2];
    const float f = mine == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(mine - m) * (vtop / kWeightTop);
#pragma unroll
    for (int d = 0; d < DT; ++d)
      *reinterpret_cast<f32x4*>(sums + (wave * ROWS + r) * LD + 16 * d + 4 * g) = o[nt][d] * f;
  }
  __syncthreads();
  constexpr int U = D / 8;
  for (int i = threadIdx.x; i < ROWS * U; i += kThreads) {
    const int rl = i / U, u = i % U, r = tile * ROWS + rl;
    if (r >= n_rows) continue;
    int64_t out;
    const Row row = row_of<PREFIX>(p, unit, r, out);
    const bool real = row.hi >= row.lo;
    float m = ml[rl * 2];
#pragma unroll
    for (int w = 1; w < 4; ++w) m = fmaxf(m, ml[(w * ROWS + rl) * 2]);
    float sum = 0.f, x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float mw = ml[(w * ROWS + rl) * 2], lw = ml[(w * ROWS + rl) * 2 + 1];
      sum += mw == -__builtin_inff() ? 0.f * lw : __builtin_amdgcn_exp2f(mw - m) * lw;
      const f32x4 a = *reinterpret_cast<const f32x4*>(sums + (w * ROWS + rl) * LD + 8 * u);
      const f32x4 b = *reinterpret_cast<const f32x4*>(sums + (w * ROWS + rl) * LD + 8 * u + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[e] += a[e];
        x[4 + e] += b[e];
      }
    }
    if (!partial) {
      bf16x8 y = {};
      if (real) {
        const float inv = 1.f / sum;
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = (bf16)(x[e] * inv);
      }
      *reinterpret_cast<bf16x8*>(p.o + out * D + 8 * u) = y;
    } else {
      const int64_t at = (int64_t)slot * ((int64_t)p.B * p.span.T * p.H) + out;
      const bool has = real && end > begin;
      if (u == 0) {
        p.part_ml[2 * at] = has ? m : -__builtin_inff();
        p.part_ml[2 * at + 1] = has ? sum : 0.f;
      }
      if (has) {
        *reinterpret_cast<f32x4*>(p.part_o + at * D + 8 * u) = f32x4{x[0], x[1], x[2], x[3]};
        *reinterpret_cast<f32x4*>(p.part_o + at * D + 8 * u + 4) = f32x4{x[4], x[5], x[6], x[7]};
      }
    }
  }
}

template <int D, int NT>
constexpr int attend_lds_floats() {
  return 4 * 16 * NT * (2 + D + 4);
}

// Workgroups in order: the prefix's items (tile slowest), then the sequences'.
template <int D, int NT, int NTP>
__global__ __launch_bounds__(kThreads) void cached_attn_kernel(CachedAttnArgs p) {
  __shared__ __align__(16) float lds[attend_lds_floats<D, (NTP > NT ? NTP : NT)>()];
  int id = blockIdx.x;
  const bool partial = p.own_splits + p.prefix_splits > 1;
  if constexpr (NTP > 0) {
    if (id < p.prefix_items) {
      const int per = p.prefix_splits * p.Hkv, tile = id / per, rest = id - tile * per, split = rest / p.Hkv;
      attend<D, NTP, true>(p, rest - split * p.Hkv, tile, split, p.prefix_splits, split, partial, lds);
      return;
    }
    id -= p.prefix_items;
  }
  const int units = p.B * p.Hkv, st = id / units, unit = id - st * units;
  const int split = st / p.own_tiles, tile = st - split * p.own_tiles;
  attend<D, NT, false>(p, unit, p.own_tiles - 1 - tile, split, p.own_splits, p.prefix_splits + split, partial, lds);
}

// Joins the splits: o = sum_s 2^(m_s - m) o_s / sum_s 2^(m_s - m) l_s, in the
// order of s.  D / 4 lanes to a row.
template <int D>
__global__ __launch_bounds__(kThreads) void cached_combine_kernel(CachedAttnArgs p) {
  constexpr int LPR = D / 4;
  const int64_t rows = (int64_t)p.B * p.span.T * p.H;
  const int64_t row = (int64_t)blockIdx.x * (kThreads / LPR) + threadIdx.x / LPR;
  const int c = threadIdx.x % LPR, n = p.own_splits + p.prefix_splits;
  if (row >= rows) return;
  float m = -__builtin_inff();
  for (int s = 0; s < n; ++s) m = fmaxf(m, p.part_ml[2 * (s * rows + row)]);
  float sum = 0.f;
  bool any = false;
  f32x4 x{0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < n; ++s) {
    const float ms = p.part_ml[2 * (s * rows + row)], ls = p.part_ml[2 * (s * rows + row) + 1];
    if (ls == 0.f) continue;  // no key of this split
    any = true;
    const float f = ms == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(ms - m);
    sum += f * ls;
    x += *reinterpret_cast<const f32x4*>(p.part_o + (s * rows + row) * D + 4 * c) * f;
  }
  bf16x4 y = {};
  if (any) {
    const float inv = 1.f / sum;
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = (bf16)(x[e] * inv);
  }
  *reinterpret_cast<bf16x4*>(p.o + row * D + 4 * c) = y;
}

template <int D, int NT, int NTP>
hipError_t launch(const CachedAttnArgs& p, hipStream_t stream) {
  const int64_t items = (int64_t)p.prefix_items + (int64_t)p.B * p.Hkv * p.own_tiles * p.own_splits;
  hipLaunchKernelGGL((cached_attn_kernel<D, NT, NTP>), dim3((unsigned)items), dim3(kThreads), 0, stream, p);
  hipError_t err = hipGetLastError();
  if (err != hipSuccess || p.own_splits + p.prefix_splits == 1) return err;
  const int64_t rows = (int64_t)p.B * p.span.T * p.H, per = kThreads / (D / 4);
  hipLaunchKernelGGL((cached_combine_kernel<D>), dim3((unsigned)((rows + per - 1) / per)), dim3(kThreads), 0, stream, p);
  return hipGetLastError();
}

// 16-row tiles of a workgroup for n rows.
template <int D>
int tiles_of(int64_t rows) {
  return rows <= 16 ? 1 : rows <= 32 || D == 128 ? 2 : 4;
}

}  // namespace

// Row tiles, splits and work items of a problem.  `keys` bounds the own keys
// that a sequence holds; the plan only decides how the work is shared out.
template <int D>
int64_t plan_cached_attn(CachedAttnArgs& p, int64_t keys) {
  const int64_t own_rows = (int64_t)p.span.T * p.G, prefix_rows = own_rows * p.B;
  const int nt = tiles_of<D>(own_rows), ntp = tiles_of<D>(prefix_rows);
  p.own_tiles = (int)((own_rows + 16 * nt - 1) / (16 * nt));
  const int64_t target = 1024;
  const auto splits = [&](int64_t items, int64_t most_keys) {
    const int64_t blocks = (most_keys + 63) / 64;
    return (int)std::max<int64_t>(1, std::min((target + items - 1) / items, (blocks + 3) / 4));
  };
  const int64_t tokens = (16 * nt + p.G - 1) / p.G + 1, reach = (int64_t)p.window + tokens + 63;
  p.own_splits = splits((int64_t)p.B * p.Hkv * p.own_tiles, std::min(keys, reach));
  p.prefix_tiles = p.prefix_splits = 0;
  p.prefix_items = 0;
  if (p.P > 0) {
    p.prefix_tiles = (int)((prefix_rows + 16 * ntp - 1) / (16 * ntp));
    p.prefix_splits = splits((int64_t)p.Hkv * p.prefix_tiles, p.P);
  }
  return (int64_t)p.Hkv * p.prefix_tiles * p.prefix_splits + (int64_t)p.B * p.Hkv * p.own_tiles * p.own_splits;
}

template <int D>
hipError_t launch_cached_attn(CachedAttnArgs& p, hipStream_t stream) {
  p.prefix_items = p.Hkv * p.prefix_tiles * p.prefix_splits;
  const int64_t own_rows = (int64_t)p.span.T * p.G;
  const int nt = tiles_of<D>(own_rows), ntp = p.P > 0 ? tiles_of<D>(own_rows * p.B) : 0;
  switch (8 * nt + ntp) {
    case 8 * 1 + 0: return launch<D, 1, 0>(p, stream);
    case 8 * 2 + 0: return launch<D, 2, 0>(p, stream);
    case 8 * 1 + 1: return launch<D, 1, 1>(p, stream);
    case 8 * 1 + 2: return launch<D, 1, 2>(p, stream);
    case 8 * 2 + 2: return launch<D, 2, 2>(p, stream);
  }
  if constexpr (D == 64) switch (8 * nt + ntp) {
      case 8 * 4 + 0: return launch<D, 4, 0>(p, stream);
      case 8 * 1 + 4: return launch<D, 1, 4>(p, stream);
      case 8 * 2 + 4: return launch<D, 2, 4>(p, stream);
      case 8 * 4 + 4: return launch<D, 4, 4>(p, stream);
    }
  return hipErrorInvalidValue;
}

template int64_t plan_cached_attn<64>(CachedAttnArgs&, int64_t);
template int64_t plan_cached_attn<128>(CachedAttnArgs&, int64_t);
template hipError_t launch_cached_attn<64>(CachedAttnArgs&, hipStream_t);
template hipError_t launch_cached_attn<128>(CachedAttnArgs&, hipStream_t);

}  // namespace hlm
