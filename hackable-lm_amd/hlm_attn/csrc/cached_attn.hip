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
// A unit's rows are the query heads of one kv head, of one or more tokens; for
// the prefix, of all sequences, so that its keys are read once (a short one's
// are taken by each sequence together with its own: plan_cached_attn).  Few rows
// (attend_split): a workgroup takes 16 and a share of their keys in blocks of
// 64, which its four waves take in turn; their sums are joined in LDS.  More
// (attend_tile): 64 or 128 rows, shared out to the waves, and each block's
// operands shared by them in LDS.  The sums of several workgroups over the same
// rows' keys are joined by the combine kernel.
//
// Single tokens are bound by memory: 64 sequences of up to 2048 tokens, 12
// heads of 64, 110.6 MB in 24.6 us (4.5 TB/s; a copy on this MI355X 4.8); 16384
// keys of 16 heads of 128, 69 MB in 14.8 us and a join of 16 splits in 3.9.  Many
// rows are bound by the softmax's vector instructions, about 13 a score, of which
// the exponential takes four slots: 2 x 500 tokens over 1500 and 2500, 12 heads of
// 64, 23.3 + 4.6 us (each kernel alone).  A single token over a window of 512 takes
// 5.3 us, most of it three trips to memory (places, keys, rows of q with them) and
// the launch.
//
// Layouts (v_mfma_f32_16x16x32_f16, lane l, n = l % 16, g = l / 16):
//   A (16 x 32): row n, k = 8 g + e;  B (32 x 16): k = 8 g + e, column n;
//   C (16 x 16): column n, rows 4 g + i.
// Scores are formed transposed, keys by rows: tile t is the block's keys
// 16 t .. 16 t + 15, so lane (n, g) ends up with the scores of query row n and
// the 16 keys 16 t + 4 g + i.  Rounded to fp16 they are the B operand of
// o^T = v^T p^T as they are, if its k slot 8 g + e is key 16 (2 h + e / 4) + 4 g
// + e % 4 in half h; the A operand's lane (n, g) then needs dim n of the same 16
// keys, which is how the cache keeps the values.
// A score's maximum, sum and rescaling stay in the lane, but for the maximum
// over the four g.
//
// Numerics.  q is scaled by a power of two to at most 2 per row and then held
// in fp16 (exact but for values 2^-14 of the row's largest and below, whose
// error is 2^-25 of it); whole numbers are exact; products and sums are fp32.
// p_j vs_j is rounded to fp16 relative to the largest vs that the wave's rows have
// seen so far, 2^11 at p = 1, or to 2^8 times the row's own largest p_j vs_j if that
// is less (a key of little weight may have a value far above the others): 11 bits
// for weights above 2^-25 of it, and none above 2^-36 is lost.
// Nothing passes fp32 while keys are at most 2^118 (q.kc ks with q at 4, D = 128),
// scale |q| and scale |q.k| at most 2^126 (log2 units) and values at most 2^100
// (sums of 2^24 keys at up to 2^3).
#include <cmath>
#include <utility>

#include "kv_cache.h"

namespace hlm {
namespace {

typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;

constexpr float kWeightTop = 2048.f;  // a probability of 1 as fp16
// The running maximum is moved only when a score passes it by 2^3, and what weights
// are relative to then or when a value scale passes the smallest by 2: weights
// reach 2^15, within fp16, and the sums stay where they are meanwhile.
constexpr float kSlack = 3.f;
// What weights are relative to stays within this of the row's largest weight:
// keys that get 2^-8 of the row's attention, beside one that takes it all with a
// value as much smaller, still leave it where it is for all rows of a wave.
constexpr float kWeightRoom = 256.f;
constexpr float kSmallest = 1.17549435e-38f;  // 2^-126

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

// x op'ed over the 16 lanes of each group, and over lane n of the four groups
// (swaps of 16 and 32 lanes).  Both give every lane the result.
template <class T, class Op>
__device__ __forceinline__ T over_lanes(T x, Op op) {
  x = over_8_lanes(x, op);
  return op(x, dpp<0x140>(x));  // row_mirror
}
template <class T, class Op>
__device__ __forceinline__ T over_groups(T x, Op op) {
  const unsigned a = __builtin_bit_cast(unsigned, x);
  const auto p = __builtin_amdgcn_permlane16_swap(a, a, false, false);
  x = op(__builtin_bit_cast(T, (unsigned)p[0]), __builtin_bit_cast(T, (unsigned)p[1]));
  const unsigned b = __builtin_bit_cast(unsigned, x);
  const auto q = __builtin_amdgcn_permlane32_swap(b, b, false, false);
  return op(__builtin_bit_cast(T, (unsigned)q[0]), __builtin_bit_cast(T, (unsigned)q[1]));
}
struct Min {
  __device__ __forceinline__ float operator()(float a, float b) const { return fminf(a, b); }
  __device__ __forceinline__ int operator()(int a, int b) const { return min(a, b); }
};
struct Sum {
  __device__ __forceinline__ float operator()(float a, float b) const { return a + b; }
};
// A value that all lanes hold, as a scalar.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ float uniform(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, x)));
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

// A query row: its sequence, token and head, and its number in o.
struct Row {
  int b, t, head;
  int64_t out;
};

// The keys that a workgroup takes: a sequence's own, the prefix's for the rows of
// all sequences, or the prefix's followed by the sequence's own (from the
// prefix's next whole block on).
enum Segment { kOwn, kPrefix, kBoth };

template <Segment SEG>
__device__ __forceinline__ Row row_of(const CachedAttnArgs& p, int unit, int r) {
  Row row;
  const int rt = fast_div(r, p.div_G), g = r - rt * p.G;
  int bt, h;
  if constexpr (SEG == kPrefix) {
    bt = rt;
    row.b = fast_div(bt, p.div_T);
    row.t = bt - row.b * p.span.T;
    h = unit;
  } else {
    row.b = unit / p.Hkv;
    h = unit - row.b * p.Hkv;
    row.t = rt;
    bt = row.b * p.span.T + row.t;
  }
  row.head = h * p.G + g;
  row.out = (int64_t)bt * p.H + row.head;
  return row;
}

// The first own key in kBoth's count of keys.
__device__ __forceinline__ int own_key(const CachedAttnArgs& p) { return (p.P + kCacheBlock - 1) / kCacheBlock * kCacheBlock; }

// The segment's keys lo .. hi that the row sees (hi < lo: none).
template <Segment SEG>
__device__ __forceinline__ void keys_seen(const CachedAttnArgs& p, const Row& row, int& lo, int& hi) {
  lo = 0;
  hi = -1;
  const int pos = cache_position(span_start(p.span, row.b), span_count(p.span, row.b), row.t, p.own.slots);
  if (pos < 0) return;
  const int64_t from = (int64_t)pos - p.window + 1;
  const int in_prefix = (int)min((int64_t)p.P, max((int64_t)0, from + p.P)), in_own = (int)max((int64_t)0, from);
  if constexpr (SEG == kPrefix) {
    hi = p.P - 1;
    lo = in_prefix;
  } else if constexpr (SEG == kOwn) {
    hi = pos;
    lo = in_own;
  } else {
    hi = own_key(p) + pos;
    lo = in_prefix < p.P ? in_prefix : own_key(p) + in_own;
  }
}

// Lane 16 g + 4 t + i holds the scales of the block's key 16 t + 4 g + i, so
// that row_lane<4 t + i> hands a group those of its own keys.
__device__ __forceinline__ int lane_key(int lane) { return 16 * (lane >> 2 & 3) + 4 * (lane >> 4) + (lane & 3); }

// What one wave holds of its 16 NT query rows.
template <int D, int NT>
struct Rows {
  static constexpr int C = D / 64, DT = D / 16;
  int lo[NT], hi[NT];  // the keys that this lane's rows see
  int first, last;     // all keys that some row of the wave sees
  int inner_first, inner_last;  // the keys that every row sees
  f16x8 q[NT][C][2];
  // The power of two in scale log2(e) and q's: a row's scores (q.kc) ks times it are
  // in log2 units, exactly, so that the largest one's probability is 1 however large
  // it is.  The rest of scale log2(e), 0.5 .. 1, is in ks.
  float rs[NT];
  float mt[NT], l[NT];      // running maximum of (q.kc) ks, sum
  // The value scale that each row's weights are relative to (0: none yet), and a
  // weight p vs that the row has seen, its largest when they were last looked at.
  // The scales' smallest and largest, for the wave, and the largest's inverse:
  // mostly they are the same.
  float ref[NT], heavy[NT], vlow, vhigh, per_vhigh;
  f32x4 o[NT][DT];          // o^T: dims 16 d + 4 g + i of row n

  // The rows r0 .. of a unit.  Queries are loaded before the places are known
  // (of padding rows too, whose results nothing uses): both come from memory.
  template <Segment SEG>
  __device__ __forceinline__ void begin(const CachedAttnArgs& p, int unit, int r0, int n_rows, int lane, bf16x8 x[NT][C][2]) {
    const int n = lane & 15, g = lane >> 4;
    Row row[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = r0 + 16 * nt + n;
      row[nt] = row_of<SEG>(p, unit, min(r, n_rows - 1));
      const bf16* at = p.q + row[nt].b * p.sq[0] + row[nt].t * p.sq[1] + row[nt].head * p.sq[2] + 16 * g;
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int h = 0; h < 2; ++h) x[nt][c][h] = *reinterpret_cast<const bf16x8*>(at + 64 * c + 8 * h);
    }
    first = inner_last = 0x7fffffff;
    last = inner_first = -1;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      keys_seen<SEG>(p, row[nt], lo[nt], hi[nt]);
      if (r0 + 16 * nt + n >= n_rows || hi[nt] < lo[nt]) {
        lo[nt] = 0;
        hi[nt] = -1;
      }
      if (hi[nt] >= lo[nt]) {
        first = min(first, lo[nt]);
        last = max(last, hi[nt]);
        inner_first = max(inner_first, lo[nt]);
        inner_last = min(inner_last, hi[nt]);
      }
    }
    first = uniform(over_lanes(first, Min()));
    last = uniform(over_lanes(last, Max()));
    inner_first = uniform(over_lanes(inner_first, Max()));
    inner_last = uniform(over_lanes(inner_last, Min()));
  }

  __device__ __forceinline__ void take_q(const CachedAttnArgs& p, const bf16x8 x[NT][C][2]) {
    typedef __attribute__((ext_vector_type(8))) unsigned short u16x8;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      int top = 0;
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const u16x8 bits = __builtin_bit_cast(u16x8, x[nt][c][h]);
#pragma unroll
          for (int e = 0; e < 8; ++e) top = max(top, (int)(bits[e] & 0x7fff));
        }
      top = over_groups(top, Max());
      const int ex = min(126, max(-120, (top >> 7) - 127));
      // rs is kept positive and finite: a score of -infinity times it stays what it is.
      // What is missing at 2^-126 makes q smaller (127 - ex + rest is 1 at least).
      const int e = ex + p.scale_exp, rest = min(0, e + 126);
      const float down = __builtin_bit_cast(float, (127 - ex + rest) << 23);
      rs[nt] = __builtin_bit_cast(float, (127 + min(127, max(-126, e))) << 23);
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 8; ++e) q[nt][c][h][e] = (_Float16)((float)x[nt][c][h][e] * down);
      mt[nt] = -__builtin_inff();
      l[nt] = ref[nt] = heavy[nt] = 0.f;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[nt][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    vlow = vhigh = per_vhigh = 0.f;
  }

  // Scores sc of block k0 .. k0 + 63 (before the keys' scales; ks, vs: those of
  // key k0 + lane_key(lane), ks with p.scale_part) into weights w, updating the
  // rows' statistics.  Keys of the block behind `end` are nobody's.
  __device__ __forceinline__ void weigh(f32x4 sc[NT][4], float ks, float vs, int k0, int end, int lane, f16x8 w[NT][2]) {
    const int g = lane >> 4;
    const bool whole = k0 >= inner_first && k0 + 63 <= min(inner_last, end);  // every row sees every key
    each<16>([&](auto e) {
      const float f = row_lane<e>(ks);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) sc[nt][e / 4][e % 4] *= f;
    });
    if (!whole) {  // selected, not added: masked slots may hold any scale
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const unsigned from = k0 + 4 * g - lo[nt], seen = max(0, min(hi[nt], end) - lo[nt] + 1);  // lo = 0 where hi < lo
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (from + (16 * (e / 4) + e % 4) >= seen) sc[nt][e / 4][e % 4] = -__builtin_inff();
      }
      if (k0 + lane_key(lane) < first || k0 + lane_key(lane) > min(last, end)) vs = 0.f;
    }
    bool light = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float mx = sc[nt][0][0];
#pragma unroll
      for (int e = 1; e < 16; ++e) mx = fmaxf(mx, sc[nt][e / 4][e % 4]);
      if (__any((mx - mt[nt]) * rs[nt] > kSlack)) {
        const float m = fmaxf(mt[nt], over_groups(mx, Max()));
        const float alpha = m > mt[nt] ? __builtin_amdgcn_exp2f((mt[nt] - m) * rs[nt]) : 1.f;
        mt[nt] = m;
        l[nt] *= alpha;
        heavy[nt] *= alpha;
        light |= ref[nt] > kWeightRoom * heavy[nt];
#pragma unroll
        for (int d = 0; d < DT; ++d) o[nt][d] *= alpha;
      }
      const float off = mt[nt] == -__builtin_inff() ? 0.f : -mt[nt] * rs[nt];
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float pe = __builtin_amdgcn_exp2f(fmaf(sc[nt][e / 4][e % 4], rs[nt], off));
        sum[e % 4] += pe;
        sc[nt][e / 4][e % 4] = pe;
      }
      l[nt] += (sum[0] + sum[1]) + (sum[2] + sum[3]);
    }
    if (__any(light || vs > 2.f * vlow)) settle(sc, vs);
    if (whole && vlow == vhigh) {
      const float rel = vs * per_vhigh * kWeightTop;  // 1 / vhigh <= 2^126: kWeightTop times it may be beyond fp32
      each<16>([&](auto e) {
        const float f = row_lane<e>(rel);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) w[nt][e / 8][e % 8] = (_Float16)(sc[nt][e / 4][e % 4] * f);
      });
    } else {  // a masked key's scale may be anything
      float per[NT];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) per[nt] = __builtin_amdgcn_rcpf(fmaxf(ref[nt], kSmallest));  // 0 while all scales were
      each<16>([&](auto e) {
        const float f = row_lane<e>(vs);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float pe = sc[nt][e / 4][e % 4];
          w[nt][e / 8][e % 8] = (_Float16)(pe == 0.f ? 0.f : f * per[nt] * kWeightTop * pe);
        }
      });
    }
  }

  // Sets what the rows' weights are relative to, by the block's probabilities p and
  // value scales vs (0 for keys that no row sees): the largest scale, or kWeightRoom
  // times the row's largest weight if that is less (so a row keeps clear of scales
  // that only others see; its own p is 0 there).  A weight is then at most 2^3
  // kWeightTop, in later blocks 2^4, since they come here if a scale passes 2 ref;
  // and o, in its old units at most as large as in the new ones, cannot pass fp32.
  __device__ __forceinline__ void settle(const f32x4 p[NT][4], float vs) {
    float low = __builtin_inff(), high = 0.f;
    const float scale = over_groups(over_lanes(vs, Max()), Max());
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float weight = 0.f;
      each<16>([&](auto e) { weight = fmaxf(weight, p[nt][e / 4][e % 4] * row_lane<e>(vs)); });  // a NaN is passed over
      heavy[nt] = fmaxf(heavy[nt], over_groups(weight, Max()));
      const float to = fmaxf(kSmallest, fminf(fmaxf(ref[nt], scale), kWeightRoom * heavy[nt]));
      if (ref[nt] > 0.f && to != ref[nt]) {  // before the first weight o is zero
        const float f = fminf(3e38f, ref[nt] / to);
#pragma unroll
        for (int d = 0; d < DT; ++d) o[nt][d] *= f;
      }
      ref[nt] = to;
      if (hi[nt] >= lo[nt]) {
        low = fminf(low, ref[nt]);
        high = fmaxf(high, ref[nt]);
      }
    }
    vlow = uniform(over_lanes(low, Min()));
    vhigh = uniform(over_lanes(high, Max()));
    per_vhigh = vhigh > 0.f ? 1.f / vhigh : 0.f;
  }

  // The maximum in log2 units.
  __device__ __forceinline__ float top2(int nt) const { return mt[nt] == -__builtin_inff() ? mt[nt] : mt[nt] * rs[nt]; }
};

// Where block blk of a unit's keys lies (keys: k, ks; values: v, vs), and the
// last key that belongs to somebody as far as the block goes.
template <int D, Segment SEG>
struct Blocks {
  Keys a, b;
  int split, last;  // a's blocks are those before split, b's the others

  static __device__ __forceinline__ Keys of(const KvCache& c, int unit) {
    const int64_t head = (int64_t)unit * c.slots;
    return {c.k + head * D, c.v + head * D, c.ks + head, c.vs + head};
  }
  __device__ __forceinline__ Blocks(const CachedAttnArgs& p, int unit) : split(own_key(p) / kCacheBlock), last(p.P - 1) {
    if constexpr (SEG != kBoth) {
      a = of(SEG == kPrefix ? p.prefix : p.own, unit);
    } else {
      a = of(p.prefix, unit % p.Hkv);
      b = of(p.own, unit);
    }
  }
  __device__ __forceinline__ Keys at(int blk) const {
    const bool own = SEG == kBoth && blk >= split;
    const Keys& s = own ? b : a;
    const int n = own ? blk - split : blk;
    return {s.k + (int64_t)n * (64 * D), s.v + (int64_t)n * (64 * D), s.ks + 64 * n, s.vs + 64 * n};
  }
  __device__ __forceinline__ int end(int blk) const { return SEG == kBoth && blk < split ? last : 0x7fffffff; }
};

// This workgroup's blocks begin .. end - 1 of the keys first .. last, shared
// out evenly.
__device__ __forceinline__ void share(int first, int last, int split, int n_splits, int& begin, int& end) {
  begin = end = 0;
  if (last < first) return;
  const int b0 = first >> 6, blocks = (last >> 6) - b0 + 1, per = (blocks + n_splits - 1) / n_splits;
  begin = b0 + min(blocks, split * per);
  end = b0 + min(blocks, split * per + per);
}

// 16 rows, the keys shared by the four waves.
template <int D, Segment SEG>
__device__ __forceinline__ void attend_split(const CachedAttnArgs& p, int unit, int tile, int split, int n_splits, int slot,
                                             bool partial, float* lds) {
  constexpr int C = D / 64, DT = D / 16, ROWS = 16, LD = D + 4, NW = 4;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, g = lane >> 4;
  const int n_rows = SEG == kPrefix ? p.B * p.span.T * p.G : p.span.T * p.G;
  const Blocks<D, SEG> keys(p, unit);
  Rows<D, 1> rows;
  bf16x8 x_q[1][C][2];
  rows.template begin<SEG>(p, unit, tile * ROWS, n_rows, lane, x_q);
  int begin, end;
  share(rows.first, rows.last, split, n_splits, begin, end);

  // Past the caches' retention, for own keys and values are read once (26.5 against
  // 29.4 us for 64 sequences of up to 2048 tokens, 12 heads of 64).  A prefix's in
  // the joint pass are read by every sequence, and no slower so: 24 tokens over a
  // prefix of 60, 6 heads of 64, 6.7 us with either kind of load, 60 over 100 7.4 and 7.1.
  u32x4 kr[4][C], vr[DT];
  float ksl = 0.f, vsl = 0.f;
  auto load_k = [&](int blk) {
    const Keys s = keys.at(blk);
    const u32x4* at = reinterpret_cast<const u32x4*>(s.k) + lane;
    ksl = s.ks[lane_key(lane)];
    vsl = s.vs[lane_key(lane)];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int c = 0; c < C; ++c) kr[t][c] = __builtin_nontemporal_load(at + (t * C + c) * 64);
  };
  auto load_v = [&](int blk) {
    const u32x4* at = reinterpret_cast<const u32x4*>(keys.at(blk).v) + lane;
#pragma unroll
    for (int d = 0; d < DT; ++d) vr[d] = __builtin_nontemporal_load(at + 64 * d);
  };

  int blk = begin + wave;
  if (blk < end) {
    load_k(blk);
    load_v(blk);
  }
  rows.take_q(p, x_q);
  for (; blk < end; blk += NW) {
    const bool more = blk + NW < end;
    f32x4 sc[1][4];
    f16x8 w[1][2];
    const float ks = ksl * p.scale_part, vs = vsl;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      f16x8 kf[C][2];
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int h = 0; h < 2; ++h) kf[c][h] = decode8(kr[t][c][2 * h], kr[t][c][2 * h + 1]);
      sc[0][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int h = 0; h < 2; ++h) sc[0][t] = mfma16(kf[c][h], rows.q[0][c][h], sc[0][t]);
    }
    if (more) load_k(blk + NW);
    rows.weigh(sc, ks, vs, blk * 64, keys.end(blk), lane, w);
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      const f16x8 v0 = decode8(vr[d][0], vr[d][1]), v1 = decode8(vr[d][2], vr[d][3]);
      rows.o[0][d] = mfma16(v0, w[0][0], rows.o[0][d]);
      rows.o[0][d] = mfma16(v1, w[0][1], rows.o[0][d]);
    }
    if (more) load_v(blk + NW);
  }

  // Join the waves: maxima and sums, then o relative to the common maximum.
  float* ml = lds;                        // (NW, ROWS, 2)
  int* real = reinterpret_cast<int*>(lds + NW * ROWS * 2);  // (ROWS)
  float* sums = lds + NW * ROWS * 2 + ROWS;                 // (NW, ROWS, LD)
  const float mine = rows.top2(0), l = over_groups(rows.l[0], Sum());
  if (g == 0) {
    float* at = ml + (wave * ROWS + n) * 2;
    at[0] = mine;
    at[1] = l;
    if (wave == 0) real[n] = rows.hi[0] >= rows.lo[0];
  }
  __syncthreads();
  float top = ml[n * 2];
#pragma unroll
  for (int w = 1; w < NW; ++w) top = fmaxf(top, ml[(w * ROWS + n) * 2]);
  const float f = mine == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(mine - top) / kWeightTop;
#pragma unroll
  for (int d = 0; d < DT; ++d)
    *reinterpret_cast<f32x4*>(sums + (wave * ROWS + n) * LD + 16 * d + 4 * g) = rows.o[0][d] * f * rows.ref[0];
  __syncthreads();
  constexpr int U = D / 4;
  for (int i = threadIdx.x; i < ROWS * U; i += 64 * NW) {
    const int rl = i / U, u = i % U, r = tile * ROWS + rl;
    if (r >= n_rows) continue;
    const int64_t out = row_of<SEG>(p, unit, r).out;
    float m = ml[rl * 2];
#pragma unroll
    for (int w = 1; w < NW; ++w) m = fmaxf(m, ml[(w * ROWS + rl) * 2]);
    float sum = 0.f;
    f32x4 x{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float mw = ml[(w * ROWS + rl) * 2], lw = ml[(w * ROWS + rl) * 2 + 1];
      sum += mw == -__builtin_inff() ? 0.f * lw : __builtin_amdgcn_exp2f(mw - m) * lw;
      x += *reinterpret_cast<const f32x4*>(sums + (w * ROWS + rl) * LD + 4 * u);
    }
    if (!partial) {
      bf16x4 y = {};
      if (real[rl]) {
        const float inv = 1.f / sum;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = (bf16)(x[e] * inv);
      }
      *reinterpret_cast<bf16x4*>(p.o + out * D + 4 * u) = y;
    } else {
      const int64_t at = (int64_t)slot * ((int64_t)p.B * p.span.T * p.H) + out;
      const bool has = real[rl] && end > begin;
      if (u == 0) {
        p.part_ml[2 * at] = has ? m : -__builtin_inff();
        p.part_ml[2 * at + 1] = has ? sum : 0.f;
      }
      if (has) *reinterpret_cast<f32x4*>(p.part_o + at * D + 4 * u) = x;
    }
  }
}

// 64 NT rows, 16 NT to a wave.  Each wave turns a quarter of a block's codes
// into fp16 operands in LDS, in the order in which the lanes read them (1 KB to
// an operand, one block ahead, no conflicts), and multiplies all of the block.
template <int D, int NT, Segment SEG>
__device__ __forceinline__ void attend_tile(const CachedAttnArgs& p, int unit, int tile, int split, int n_splits, int slot,
                                            bool partial, float* lds) {
  constexpr int C = D / 64, DT = D / 16, VD = DT / 4, ROWS = 64 * NT, KF = 8 * C, F = KF + 2 * DT;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, g = lane >> 4;
  const int n_rows = SEG == kPrefix ? p.B * p.span.T * p.G : p.span.T * p.G;
  const Blocks<D, SEG> keys(p, unit);
  Rows<D, NT> rows;
  bf16x8 x_q[NT][C][2];
  const int r0 = tile * ROWS + wave * 16 * NT;
  rows.template begin<SEG>(p, unit, r0, n_rows, lane, x_q);
  int* range = reinterpret_cast<int*>(lds);
  if (lane == 0) {
    range[wave] = rows.first;
    range[4 + wave] = rows.last;
  }
  __syncthreads();
  int first = range[0], last = range[4];
#pragma unroll
  for (int w = 1; w < 4; ++w) {
    first = min(first, range[w]);
    last = max(last, range[4 + w]);
  }
  first = uniform(first);
  last = uniform(last);
  int begin, end;
  share(first, last, split, n_splits, begin, end);
  __syncthreads();  // range is read: the operands may overwrite it

  f16x8* ops = reinterpret_cast<f16x8*>(lds);  // (2, F, 64)
  u32x4 kr[C], vr[VD];
  float ks_next = 0.f, vs_next = 0.f;
  auto load = [&](int blk) {
    const Keys s = keys.at(blk);
    const u32x4* k = reinterpret_cast<const u32x4*>(s.k) + C * 64 * wave + lane;
    const u32x4* v = reinterpret_cast<const u32x4*>(s.v) + VD * 64 * wave + lane;
#pragma unroll
    for (int c = 0; c < C; ++c) kr[c] = k[64 * c];
#pragma unroll
    for (int d = 0; d < VD; ++d) vr[d] = v[64 * d];
  };
  auto load_scales = [&](int blk) {
    const Keys s = keys.at(blk);
    ks_next = s.ks[lane_key(lane)];
    vs_next = s.vs[lane_key(lane)];
  };
  auto store = [&](int buf) {
    f16x8* to = ops + buf * (F * 64) + lane;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int h = 0; h < 2; ++h) to[((wave * C + c) * 2 + h) * 64] = decode8(kr[c][2 * h], kr[c][2 * h + 1]);
#pragma unroll
    for (int d = 0; d < VD; ++d)
#pragma unroll
      for (int h = 0; h < 2; ++h) to[(KF + (wave * VD + d) * 2 + h) * 64] = decode8(vr[d][2 * h], vr[d][2 * h + 1]);
  };
  if (begin < end) {
    load(begin);
    load_scales(begin);
  }
  rows.take_q(p, x_q);
  if (begin < end) {
    store(0);
    if (begin + 1 < end) load(begin + 1);
  }
  __syncthreads();
  for (int blk = begin; blk < end; ++blk) {
    const int buf = (blk - begin) & 1;
    const float ks = ks_next * p.scale_part, vs = vs_next;
    if (blk + 1 < end) {
      store(buf ^ 1);
      load_scales(blk + 1);
      if (blk + 2 < end) load(blk + 2);
    }
    if (blk * 64 <= rows.last && blk * 64 + 63 >= rows.first) {
      const f16x8* at = ops + buf * (F * 64) + lane;
      f32x4 sc[NT][4];
      f16x8 w[NT][2];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) sc[nt][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const f16x8 kf = at[((t * C + c) * 2 + h) * 64];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) sc[nt][t] = mfma16(kf, rows.q[nt][c][h], sc[nt][t]);
          }
      }
      // Small tiles have the registers to read the values while the weights are
      // worked out (500 tokens over 1500 and 2500: 27.2 against 28.8 us).
      f16x8 vf[DT][2];
      if constexpr (NT == 1) {
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int h = 0; h < 2; ++h) vf[d][h] = at[(KF + d * 2 + h) * 64];
        __builtin_amdgcn_sched_barrier(0);
      }
      rows.weigh(sc, ks, vs, blk * 64, keys.end(blk), lane, w);
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if constexpr (NT > 1) vf[d][h] = at[(KF + d * 2 + h) * 64];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) rows.o[nt][d] = mfma16(vf[d][h], w[nt][h], rows.o[nt][d]);
        }
    }
    __syncthreads();
  }

#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const float l = over_groups(rows.l[nt], Sum());
    const int r = r0 + 16 * nt + n;
    if (r >= n_rows) continue;
    const int64_t out = row_of<SEG>(p, unit, r).out;
    const bool real = rows.hi[nt] >= rows.lo[nt];
    if (!partial) {
      const float f = real ? 1.f / (l * kWeightTop) : 0.f;
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        bf16x4 y = {};
        if (real)
#pragma unroll
          for (int i = 0; i < 4; ++i) y[i] = (bf16)(rows.o[nt][d][i] * f * rows.ref[nt]);
        *reinterpret_cast<bf16x4*>(p.o + out * D + 16 * d + 4 * g) = y;
      }
    } else {
      const int64_t at = (int64_t)slot * ((int64_t)p.B * p.span.T * p.H) + out;
      const bool has = real && end > begin;
      if (g == 0) {
        p.part_ml[2 * at] = has ? rows.top2(nt) : -__builtin_inff();
        p.part_ml[2 * at + 1] = has ? l : 0.f;
      }
      // past the caches' retention: 500 tokens over 1500 and 2500 28.4 -> 27.1 us
      // (the few rows of attend_split: 16384 keys of 16 heads 18.3 -> 18.6, so not there)
      if (has)
#pragma unroll
        for (int d = 0; d < DT; ++d)
          __builtin_nontemporal_store(rows.o[nt][d] / kWeightTop * rows.ref[nt],
                                      reinterpret_cast<f32x4*>(p.part_o + at * D + 16 * d + 4 * g));
    }
  }
}

// Rows of a workgroup by variant: 0: 16, the waves share the keys; 1 and 2: 64
// and 128, the waves share the rows.
constexpr int tile_rows(int variant) { return variant == 0 ? 16 : 64 * variant; }
template <int D>
constexpr int lds_floats(int variant) {
  return variant < 0 ? 0 : variant == 0 ? 16 * (1 + 4 * (2 + D + 4)) : 2 * (8 * (D / 64) + 2 * (D / 16)) * 64 * 4;
}

template <int D, int V, Segment SEG>
__device__ __forceinline__ void attend(const CachedAttnArgs& p, int unit, int tile, int split, int n_splits, int slot,
                                       bool partial, float* lds) {
  if constexpr (V == 0)
    attend_split<D, SEG>(p, unit, tile, split, n_splits, slot, partial, lds);
  else
    attend_tile<D, V, SEG>(p, unit, tile, split, n_splits, slot, partial, lds);
}

// Workgroups in order: the prefix's items (tile slowest), then the sequences'.
// V, VP: variants of the own keys and of the prefix (-1: none; kJoint: the
// sequences' items take the prefix's keys as well).
// The 16- and 64-row kernels at head dim 64 are held to 128 registers, four waves a
// SIMD: left alone the compiler takes up to 133, three (300 x 1 token over 512, 12
// heads, 46.5 us with three and 42.1 with four; 512 x 1 over 300, 57.3 and 53.4;
// alike where a CU has up to three workgroups).  None spills.
constexpr int kJoint = -2;
template <int D, int V, int VP>
__global__ __launch_bounds__(kThreads, D == 64 && V < 2 && VP < 2 ? 4 : 1) void cached_attn_kernel(CachedAttnArgs p) {
  constexpr int own_lds = lds_floats<D>(V), prefix_lds = lds_floats<D>(VP);
  __shared__ __align__(16) float lds[prefix_lds > own_lds ? prefix_lds : own_lds];
  int id = blockIdx.x;
  const bool partial = p.own_splits + p.prefix_splits > 1;
  if constexpr (VP >= 0) {
    if (id < p.prefix_items) {
      const int per = p.prefix_splits * p.Hkv, tile = id / per, rest = id - tile * per, split = rest / p.Hkv;
      attend<D, VP, kPrefix>(p, rest - split * p.Hkv, tile, split, p.prefix_splits, split, partial, lds);
      return;
    }
    id -= p.prefix_items;
  }
  const int units = p.B * p.Hkv, st = id / units, unit = id - st * units;
  const int split = st / p.own_tiles, tile = st - split * p.own_tiles;
  attend<D, V, VP == kJoint ? kBoth : kOwn>(p, unit, p.own_tiles - 1 - tile, split, p.own_splits, p.prefix_splits + split, partial, lds);
}

// Joins the splits: o = sum_s 2^(m_s - m) o_s / sum_s 2^(m_s - m) l_s.  D / 4
// lanes take a split's row, GROUPS such teams share a row's splits (in the
// order s = team, team + GROUPS, ..), and are added in the order of the teams.
template <int D, int GROUPS>
__global__ __launch_bounds__(kThreads) void cached_combine_kernel(CachedAttnArgs p) {
  constexpr int LPR = D / 4, PER = kThreads / (LPR * GROUPS);
  __shared__ float sums[PER][GROUPS][D + 4];
  const int64_t rows = (int64_t)p.B * p.span.T * p.H;
  const int c = threadIdx.x % LPR, team = threadIdx.x / LPR % GROUPS, rl = threadIdx.x / (LPR * GROUPS);
  const int64_t row = (int64_t)blockIdx.x * PER + rl;
  const int n = p.own_splits + p.prefix_splits;
  const bool live = row < rows;
  const float2* ml = reinterpret_cast<const float2*>(p.part_ml) + (live ? row : 0);
  const float* po = p.part_o + (live ? row : 0) * D + 4 * c;
  // each team over its own splits, relative to its own maximum
  float m = -__builtin_inff(), sum = 0.f;
  f32x4 x{0.f, 0.f, 0.f, 0.f};
  for (int s0 = team; s0 < n; s0 += 4 * GROUPS) {
    float2 a[4];
    f32x4 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t s = min(s0 + i * GROUPS, n - 1);
      a[i] = ml[s * rows];
      v[i] = *reinterpret_cast<const f32x4*>(po + s * rows * D);
      if (s0 + i * GROUPS >= n) a[i] = make_float2(-__builtin_inff(), 0.f);
    }
    float top = m;
#pragma unroll
    for (int i = 0; i < 4; ++i) top = fmaxf(top, a[i].x);
    const float f = m == top ? 1.f : m == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(m - top);
    x *= f;
    sum *= f;
    m = top;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float w = a[i].x == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(a[i].x - m);
      sum += w * a[i].y;
      // a split without keys (sum 0) wrote no row: what lies there may be anything
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] += a[i].y == 0.f ? 0.f : w * v[i][e];
    }
  }
  if constexpr (GROUPS > 1) {
    float* to = sums[rl][team];
    *reinterpret_cast<f32x4*>(to + 4 * c) = x;
    if (c == 0) {
      to[D] = m;
      to[D + 1] = sum;
    }
    __syncthreads();
    if (team != 0) return;
    float top = -__builtin_inff();
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) top = fmaxf(top, sums[rl][g][D]);
    x = f32x4{0.f, 0.f, 0.f, 0.f};
    sum = 0.f;
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
      const float mg = sums[rl][g][D], w = mg == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(mg - top);
      sum += w * sums[rl][g][D + 1];
      x += *reinterpret_cast<const f32x4*>(&sums[rl][g][4 * c]) * w;
    }
  }
  if (!live) return;
  bf16x4 y = {};
  if (sum != 0.f) {  // NaN passes
    const float inv = 1.f / sum;
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = (bf16)(x[e] * inv);
  }
  *reinterpret_cast<bf16x4*>(p.o + row * D + 4 * c) = y;
}

template <int D, int GROUPS>
hipError_t combine(const CachedAttnArgs& p, hipStream_t stream) {
  const int64_t rows = (int64_t)p.B * p.span.T * p.H, per = kThreads / (D / 4) / GROUPS;
  hipLaunchKernelGGL((cached_combine_kernel<D, GROUPS>), dim3((unsigned)((rows + per - 1) / per)), dim3(kThreads), 0, stream, p);
  return hipGetLastError();
}

template <int D, int V, int VP>
hipError_t launch(const CachedAttnArgs& p, hipStream_t stream) {
  const int64_t items = (int64_t)p.prefix_items + (int64_t)p.B * p.Hkv * p.own_tiles * p.own_splits;
  hipLaunchKernelGGL((cached_attn_kernel<D, V, VP>), dim3((unsigned)items), dim3(kThreads), 0, stream, p);
  hipError_t err = hipGetLastError();
  if (err != hipSuccess || p.own_splits + p.prefix_splits == 1) return err;
  // Four splits to a team, whose loads are in flight together; with many rows
  // the chip is full without teams.
  const int n = p.own_splits + p.prefix_splits;
  if (n <= 4 || (int64_t)p.B * p.span.T * p.H >= 16384) return combine<D, 1>(p, stream);
  return n <= 16 ? combine<D, 4>(p, stream) : combine<D, 8>(p, stream);
}

// How `rows` query rows of each of `units` (head, keys) pairs are cut into tiles
// and their keys, `blocks` of 64, into splits: the choice with the least time
// by a model in microseconds, fitted on an MI355X.
//  * Variant 0 reads keys at 4.8 TB/s on all 256 CUs, on a share x of them at
//    x (2 - x) of that, and takes 0.8 (head dim 64) or 1.4 for each round of its
//    four waves.
//  * Variants 1 and 2 take 1.0 or 1.15 for a block (1.15, 1.65 at head dim 128)
//    while a CU has one or two workgroups, then 0.5 or 0.85 (0.8, 1.3) a
//    workgroup: the larger tile costs less a row, the smaller spreads better.
//  * Partial sums cost 3.0 for the second kernel (the prefix's are joined with
//    the own ones in any case) and are written and read at 4.5 TB/s.
// `others` workgroups run beside these; `most` is the largest variant.
struct Split {
  int variant, tiles, splits;
  double us;
};

constexpr double kJoinUs = 3.0;

template <int D>
Split choose(int64_t rows, int64_t units, int64_t blocks, int64_t all_rows, bool joined, int64_t others, int most = 2) {
  Split best{0, 1, 1, 1e300};
  const double row_us = (D + 2) * 8 / 4.5e6;
  for (int v = rows <= 16 ? 0 : 1; v <= (rows <= 16 ? 0 : rows <= 64 ? 1 : most); ++v) {
    const int64_t tiles = (rows + tile_rows(v) - 1) / tile_rows(v), items = units * tiles;
    for (int n : {1, 2, 3, 4, 5, 6, 8, 10, 12, 16, 20, 24, 32, 48, 64}) {
      if (n > blocks && n > 1) break;
      const double per = (double)((blocks + n - 1) / n), wg = (double)(items * n), q = std::ceil((wg + others) / 256);
      double t;
      if (v == 0) {
        const double bytes = (double)items * blocks * (128 * (D + 4));
        const double share = std::min(1.0, wg / 256);
        const double rounds = std::ceil(per / 4) * std::max(1.0, q / (D == 64 ? 4 : 2));
        t = std::max(rounds * (D == 64 ? 0.8 : 1.4), bytes / (4.8e6 * share * (2 - share)));
      } else {
        const double one = D == 64 ? (v == 1 ? 1.0 : 1.15) : (v == 1 ? 1.15 : 1.65);
        const double more = D == 64 ? (v == 1 ? 0.5 : 0.85) : (v == 1 ? 0.8 : 1.3);
        t = per * std::max(one, more * q);
      }
      if (n > 1 || joined) t += (joined ? 0.0 : kJoinUs) + n * (double)all_rows * row_us;
      if (t < 0.97 * best.us) best = {v, (int)tiles, n, t};  // a later choice needs to be clearly better
    }
  }
  return best;
}

}  // namespace

// Variants, tiles, splits and work items of a problem.  `keys` bounds the own
// keys that a sequence holds; the plan only decides how the work is shared out.
template <int D>
int64_t plan_cached_attn(CachedAttnArgs& p, int64_t keys) {
  const int64_t rows = (int64_t)p.span.T * p.G, units = (int64_t)p.B * p.Hkv, all = (int64_t)p.B * p.span.T * p.H;
  const int64_t reach = std::min(keys, (int64_t)p.window + p.span.T + 64);
  Split own = choose<D>(rows, units, (reach + 63) / 64, all, p.P > 0, 0);
  p.prefix_variant = -1;
  p.prefix_tiles = p.prefix_splits = 0;
  if (p.P > 0) {
    const int64_t seen = std::min<int64_t>(p.P, p.window);  // own tokens stand behind the prefix
    // Beside own tiles of 16 rows the model has the prefix's 128-row ones ahead in one
    // shape of 2500, where they are not: 6 x 12 tokens over 11351, 16 heads of 64,
    // 26.4 us with them and 26.5 with 64 rows; 23 tokens over 24516, 32 heads of 128 in
    // 8 groups, 51.6 and 47.0; 202 x 2 over 476 in one group, 32.3 and 27.9.
    Split pre = choose<D>(rows * p.B, p.Hkv, (seen + 63) / 64 + 1, all, true, units * own.tiles * own.splits, own.variant == 0 ? 1 : 2);
    // one kernel for both: 128-row tiles of a sequence's rows need them of the prefix's
    if (pre.variant < own.variant) pre.variant = own.variant, pre.tiles = (int)((rows * p.B + 127) / 128);
    // Or each sequence's rows over both: the prefix is read once per sequence, mostly
    // from the caches, but there is no join, or a smaller one.  Few rows go there at
    // par, tiles up to where the model has it 15% above, from some 200 measured shapes:
    // 24 x 1 token over a prefix of 60, 6 heads of 64, 5.9 against 8.3 us (over 800,
    // 10.3 and 9.4); 32 x 64 tokens over 50, 12 heads of 64 in 4 groups, 10.1 and 15.8
    // (over 1500, 34.3 and 34.1); 4 x 37 over 1000 in a window of 512, 10.4 and 11.5.
    const int64_t total = std::min(keys + p.P + 63, (int64_t)p.window + p.span.T + 64 + 63);
    const Split both = choose<D>(rows, units, (total + 63) / 64, all, false, 0);
    if (both.us < (both.variant > 0 ? 1.15 : 1.0) * (std::max(own.us, pre.us) + kJoinUs)) {
      own = both;
      p.prefix_variant = kJoint;
    } else {
      p.prefix_variant = pre.variant;
      p.prefix_tiles = pre.tiles;
      p.prefix_splits = pre.splits;
    }
  }
  p.variant = own.variant;
  p.own_tiles = own.tiles;
  p.own_splits = own.splits;
  const int64_t prefix_items = (int64_t)p.Hkv * p.prefix_tiles * p.prefix_splits;
  p.prefix_items = (int)prefix_items;
  return prefix_items + units * p.own_tiles * p.own_splits;
}

template <int D>
hipError_t launch_cached_attn(const CachedAttnArgs& p, hipStream_t stream) {
  if (p.prefix_variant == kJoint) {
    if (p.variant == 0) return launch<D, 0, kJoint>(p, stream);
    return p.variant == 1 ? launch<D, 1, kJoint>(p, stream) : launch<D, 2, kJoint>(p, stream);
  }
  switch (4 * p.variant + p.prefix_variant) {
    case 4 * 0 - 1: return launch<D, 0, -1>(p, stream);
    case 4 * 1 - 1: return launch<D, 1, -1>(p, stream);
    case 4 * 2 - 1: return launch<D, 2, -1>(p, stream);
    case 4 * 0 + 0: return launch<D, 0, 0>(p, stream);
    case 4 * 0 + 1: return launch<D, 0, 1>(p, stream);
    case 4 * 1 + 1: return launch<D, 1, 1>(p, stream);
    case 4 * 1 + 2: return launch<D, 1, 2>(p, stream);
    case 4 * 2 + 2: return launch<D, 2, 2>(p, stream);
  }
  return hipErrorInvalidValue;
}

template int64_t plan_cached_attn<64>(CachedAttnArgs&, int64_t);
template int64_t plan_cached_attn<128>(CachedAttnArgs&, int64_t);
template hipError_t launch_cached_attn<64>(const CachedAttnArgs&, hipStream_t);
template hipError_t launch_cached_attn<128>(const CachedAttnArgs&, hipStream_t);

}  // namespace hlm
