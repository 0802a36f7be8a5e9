// ctmi_kv_attend: attention over the 8-bit block cache.
//
//   s_ij = (q_i . c_j) * key_scale(block of j) * scale,   o_i = sum_j softmax_j(s_ij) w_j,
//   w_j = value code * value_scale(block of j)
//
// computed in one pass over the keys with a running maximum and sum.  A wavefront takes RT
// tiles of 16 query rows (the queries of one kv head: tokens x the heads that share it) and
// walks the keys 64 at a time:
//
//   S^T = K Q^T   4 key tiles x head_dim / 32 products 16x16x32; the codes become bf16 / f16
//                 in registers (exact), the scales multiply the fp32 scores
//   O^T = V^T P^T head_dim / 16 tiles x 2 products, P as one f16 or several bf16 numbers
//
// Both operands that come from memory are what the lanes already hold: a product's result has
// its rows (keys) in lane group j = lane / 16 and its columns (query rows) in lane % 16, and
// the second product wants keys in groups j, too.  Taking key (r / 4) * 16 + t * 4 + r % 4 as
// row r of key tile t gives group j the 16 neighbouring keys 16 j ... 16 j + 15: P needs no
// exchange, and with tokens innermost in the value blocks a lane's V operand is one 16-byte
// load.  The next step's keys are requested when this step's are used up, and so are the
// values.
//
// With few rows (a decode step) the four wavefronts of a workgroup share them, split the keys
// and meet in LDS at the end; with many they take rows of their own and share the keys through
// LDS.  A long axis is cut into chunks for several workgroups, whose unnormalised sums, maxima
// and weights meet in a second, small kernel.
//
// Measured on one MI355X, 32 heads over 8 of 128 dimensions: one token for each of 64 requests
// of up to 4096, 83 us, 5.4 TB/s (memory bounds it); 6 of up to 32768, 77 us, 5.0 TB/s, and 5 us
// for the parts; 2 prompts of 2000 over 4000 keys 259 us, 0.69 PFLOP/s, vector units 55 % and
// matrix cores 31 % busy: the softmax between the products bounds it.
#include <type_traits>

#include "kv_blocks.h"

namespace ctmi {
namespace {

constexpr int kAttendWaves = 4;
constexpr int kStep = 64;  // keys per step of a wavefront
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLeastVs = 0x1p-90f, kMostVs = 0x1p90f;  // scales of values that are taken as they are

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

struct AttendArgs {
  const uint16_t* q;
  int64_t q_token_stride, q_head_stride;
  uint16_t* out;
  const uint8_t *key, *value;
  const float *key_scale, *value_scale;
  const int32_t *table, *lens, *start;
  float *part_o, *part_ml;  // [chunk][token][head][dim], [chunk][token][head][2]
  int64_t table_stride;
  int32_t num_blocks, kv_heads, block_size, q_heads, width, tokens, requests;
  int32_t tiles, units, chunks, chunk_keys;  // of the grid: tiles of a request, or units of all and no tiles
  uint32_t sixteenths, magic;         // block_size / 16 and ceil(2^32 / that) (0: it is 1)
  float scale;                        // times log2(e)
  int32_t clear;                      // rows of no request become zeros
};

struct Request {
  int q0, queries, len;
};

__device__ __forceinline__ Request request_of(const AttendArgs& a, int r) {
  Request o;
  int q1;
  if (a.start) {
    o.q0 = min(max(a.start[r], 0), a.tokens);
    q1 = min(max(a.start[r + 1], o.q0), a.tokens);
  } else {
    o.q0 = r;
    q1 = r + 1;
  }
  o.queries = q1 - o.q0;
  o.len = min(max(a.lens[r], 0), a.width * a.block_size);
  return o;
}

// keys the rows of a tile may see, the first and the last row's
__device__ __forceinline__ int last_key(const Request& rq, int row, int share) {
  return max(rq.len - rq.queries + row / share + 1, 0);
}

// 4 codes -> 4 numbers in the operand's type, exact
template <typename T, bool FP8>
__device__ __forceinline__ void widen4(uint32_t w, uint32_t* o) {
  if constexpr (FP8) {
    if constexpr (T::id == CTMI_BF16) {
      o[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false));
      o[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true));
    } else {
      o[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false));
      o[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true));
    }
  } else {
    if constexpr (T::id == CTMI_BF16) {
      // integers of 8 bits are whole bf16 numbers: the upper halves of their fp32 forms
      const uint32_t f0 = f2u((float)(int8_t)w), f1 = f2u((float)(int8_t)(w >> 8));
      const uint32_t f2 = f2u((float)(int8_t)(w >> 16)), f3 = f2u((float)(int8_t)(w >> 24));
      o[0] = __builtin_amdgcn_perm(f1, f0, 0x07060302u);
      o[1] = __builtin_amdgcn_perm(f3, f2, 0x07060302u);
    } else {
      // 0x64uu is 1024 + u; with u = code + 128, less 1152
      const uint32_t u = w ^ 0x80808080u;
      const f16x2 off = {(_Float16)1152.0f, (_Float16)1152.0f};
      const f16x2 a = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - off;
      const f16x2 b = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - off;
      o[0] = __builtin_bit_cast(uint32_t, a);
      o[1] = __builtin_bit_cast(uint32_t, b);
    }
  }
}

struct Operand {
  uint32_t w[4];
};
struct Operands {  // of 16 elements
  Operand half[2];
};

template <typename T, bool FP8>
__device__ __forceinline__ Operand widen8(uint32_t lo, uint32_t hi) {
  Operand o;
  widen4<T, FP8>(lo, o.w);
  widen4<T, FP8>(hi, o.w + 2);
  return o;
}

template <typename T>
__device__ __forceinline__ f32x4 product(const Operand& a, const Operand& b, f32x4 c) {
  if constexpr (T::id == CTMI_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// over the four lane groups (lanes that differ in bits 4 and 5)
__device__ __forceinline__ float groups_max(float v) {
  v = fmaxf(v, wave_shfl_xor(v, 16));
  return fmaxf(v, wave_shfl_xor(v, 32));
}
__device__ __forceinline__ float groups_sum(float v) {
  v += wave_shfl_xor(v, 16);
  return v + wave_shfl_xor(v, 32);
}

// bytes of w that hold an e4m3 NaN (0x7F or 0xFF), as 0xFF each
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) {
  return (((w & 0x7F7F7F7Fu) + 0x01010101u) >> 7 & 0x01010101u) * 0xFFu;
}

// half `u` of 16 elements that are codes, or operands already
template <typename T, bool FP8>
__device__ __forceinline__ Operand operand(const Vec<uint32_t, 4>& codes, int u) {
  return widen8<T, FP8>(codes.v[2 * u], codes.v[2 * u + 1]);
}
template <typename T, bool FP8>
__device__ __forceinline__ Operand operand(const Operands& ready, int u) {
  return ready.half[u];
}

// What a weight of the softmax is held in for the second product: this many bf16 numbers that add
// up to it (three are all 24 bits of fp32, two 16 of them), or one f16 number (11 bits).
enum class Weights { kHalf = 1, kPair = 2, kTriple = 3 };

// The rows of a wavefront and what they have gathered: RT tiles of 16, row `first` + 16 t + c
// in lanes with lane % 16 == c.  UNIFORM: a step lies in one block, so its scales are one
// number, and `sum` is the row's in all its lanes; otherwise each lane group has a part of it.
//
// `top` is the largest of score + log2(scale of the values), by which weight times scale is taken
// from one exponential, as 2^7 at the top: what f16 loses at its lower end is then 2^-32 of the
// largest product a key has, whatever the scales are.  `sum` has the weights alone, in the same
// unit: with scales of 2^-90 at least it stays below 2^127.
template <typename T, bool FP8, int D, int RT, Weights W, bool UNIFORM>
struct AttendRows {
  static constexpr int CH = D / 64;  // 16-byte pieces of a key per lane
  static constexpr int DT = D / 16;  // tiles of the output's dimensions
  static constexpr bool HALF = W == Weights::kHalf;
  static constexpr int PARTS = (int)W;  // operands a weight takes
  using V = std::conditional_t<HALF, F16, BF16>;

  Operand q[RT][CH][2];  // dimensions ch * 64 + j * 16 + half * 8 + 0 ... 7
  f32x4 o[RT][DT];       // dimension d * 16 + j * 4 + i
  float top[RT], sum[RT];
  float most_vs;                           // the largest scale of values so far
  int ends[RT], seen_by_all, seen_by_any;  // keys seen: by each row, by the first and the last

  __device__ __forceinline__ void begin(const AttendArgs& a, const Request& rq, int first, int rows, int kv, int share) {
    const int c = lane_id() & 15, j = lane_id() >> 4;
    seen_by_any = first < rows ? last_key(rq, min(first + RT * 16, rows) - 1, share) : 0;
    seen_by_all = first < rows ? last_key(rq, first, share) : 0;
    most_vs = 0.0f;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const int row = first + t * 16 + c;
      ends[t] = row < rows ? last_key(rq, row, share) : 0;
      const uint16_t* p = a.q + (int64_t)(rq.q0 + row / share) * a.q_token_stride + (int64_t)(kv * share + row % share) * a.q_head_stride;
#pragma unroll
      for (int ch = 0; ch < CH; ++ch)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          q[t][ch][h] = Operand{};
          if (row < rows) q[t][ch][h] = *(const Operand*)(p + ch * 64 + j * 16 + h * 8);
        }
      top[t] = -INFINITY, sum[t] = 0.0f;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[t][d] = f32x4{0, 0, 0, 0};
    }
  }

  // the queries are there: not to be waited for behind the loads of a step
  __device__ __forceinline__ void arrived() {
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int ch = 0; ch < CH; ++ch)
#pragma unroll
        for (int i = 0; i < 8; ++i) asm volatile("" : "+v"(q[t][ch][i / 4].w[i % 4]));
  }

  // the weights of two keys as operands
  template <bool INFINITE>
  static __device__ __forceinline__ void split(uint32_t* parts, float w0, float w1) {
    if constexpr (HALF) {
      typedef float f32x2 __attribute__((ext_vector_type(2)));
      parts[0] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{w0, w1}), f16x2));
    } else {
#pragma unroll
      for (int n = 0; n < PARTS; ++n) {
        parts[n] = pack_bf16x2(w0, w1);
        if (n + 1 < PARTS) {
          // (nothing is left of an infinity)
          w0 = INFINITE && fabsf(w0) == INFINITY ? 0.0f : w0 - u2f(parts[n] << 16);
          w1 = INFINITE && fabsf(w1) == INFINITY ? 0.0f : w1 - u2f(parts[n] & 0xFFFF0000u);
        }
      }
    }
  }

  // 64 keys from kb on.  key(t, ch): 16 bytes of this lane's row of key tile t; value(d): the
  // codes of its 16 keys in dimension d * 16 + c.  ks, vs: the scales of those keys' block (ks
  // with the softmax's); valid: whether there is one.  keys_done() comes when the last key is used.
  template <typename Key, typename Value, typename Done>
  __device__ __forceinline__ void step(int kb, float ks, float vs, bool valid, Key key, Value value, Done keys_done) {
    const int at16 = kb + (lane_id() >> 4) * 16;  // first of this lane's 16 keys
    // a step that every row sees whole, of blocks that are all there, needs no masks
    const bool whole = kb + kStep <= seen_by_all && __all(valid && ks >= 0.0f);
    // e4m3 values at keys that no row sees: whatever is there, their weight is 0 and must stay so
    const int seen = valid ? min(max(seen_by_any - at16, 0), 16) : 0;
    auto clean = [&](Vec<uint32_t, 4> v, bool nans) {
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const int n = min(max(seen - w * 4, 0), 4);
        v.v[w] &= n == 4 ? 0xFFFFFFFFu : (1u << (8 * n)) - 1u;
        if (nans) v.v[w] &= ~nan_bytes(v.v[w]);
      }
      return v;
    };
    if constexpr (FP8) {
      if (!whole) {
        // a NaN value at a key that some rows see and others do not: 0 * NaN would reach them
        // all.  It is left out of the sums and counted by a product of its own.
        uint32_t any = 0;
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          const Vec<uint32_t, 4> v = clean(value(d), false);
#pragma unroll
          for (int w = 0; w < 4; ++w) any |= nan_bytes(v.v[w]);
        }
        if (__any(any != 0)) mark_nans(at16, valid, [&](int d) { return clean(value(d), false); });
      }
    }

    // the wavefront that multiplies goes before the one that weighs: the matrix cores wait for
    // neither (2 x 2000 of 4000: 266 us without, 253 with)
    f32x4 s[RT][4];
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
#pragma unroll
      for (int t = 0; t < RT; ++t) s[t][kt] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int ch = 0; ch < CH; ++ch) {
        const auto w = key(kt, ch);
        const Operand k0 = operand<T, FP8>(w, 0), k1 = operand<T, FP8>(w, 1);
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          s[t][kt] = product<T>(k0, q[t][ch][0], s[t][kt]);
          s[t][kt] = product<T>(k1, q[t][ch][1], s[t][kt]);
        }
      }
    }
    __builtin_amdgcn_s_setprio(0);
    keys_done();

    float unit = ks;  // what a score is still to be multiplied by
    if (!whole) {
      unit = 1.0f;
#pragma unroll
      for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int kt = 0; kt < 4; ++kt)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[t][kt][i] = !valid || at16 + kt * 4 + i >= ends[t] ? -INFINITY : s[t][kt][i] * ks;
    }
    // plain: scales as they should be, and where the sum is of rounded numbers (below) none of
    // them so small beside others that f16 would have lost what a weight adds to the sum
    most_vs = fmaxf(most_vs, vs);
    const bool plain = __all(vs >= kLeastVs && vs <= kMostVs && (!(HALF && UNIFORM) || vs * 256.0f >= most_vs));
    float log_vs = __builtin_amdgcn_logf(vs), by_vs = __builtin_amdgcn_rcpf(vs), times = 1.0f;
    if (!plain) {  // vs = 2^log_vs times
      const float size = fabsf(vs);
      const bool ordinary = size >= kLeastVs && size <= kMostVs;
      log_vs = ordinary ? __builtin_amdgcn_logf(size) : size > kMostVs ? 90.0f : -90.0f;
      times = ordinary ? copysignf(1.0f, vs) : vs * (size > kMostVs ? kLeastVs : kMostVs);
    }
    Operand w[RT][2][PARTS];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      float m = s[t][0][0];
#pragma unroll
      for (int kt = 0; kt < 4; ++kt)
#pragma unroll
        for (int i = 0; i < 4; ++i) m = fmaxf(m, s[t][kt][i]);
      m = fmaf(m, unit, log_vs);
      // weights may exceed the top's by 2^8 before the sums are brought to a new one: the operands
      // keep their precision there, and the lanes of a row need not be asked for their maximum in
      // most steps
      if (__any(m > top[t] + 8.0f)) {
        const float now = fmaxf(top[t], groups_max(m));
        const float shrink = top[t] == -INFINITY ? 0.0f : exp2_fast(top[t] - now);
        top[t] = now;
        sum[t] *= shrink;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[t][d] *= shrink;
      }
      const float base = (top[t] == -INFINITY ? 0.0f : top[t]) - 7.0f, less = base - log_vs;
      float part = 0.0f;
      if (plain) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float w0 = exp2_fast(fmaf(s[t][u * 2 + e / 2][(e % 2) * 2], unit, -less));
            const float w1 = exp2_fast(fmaf(s[t][u * 2 + e / 2][(e % 2) * 2 + 1], unit, -less));
            if constexpr (!UNIFORM) part += w0 + w1;
            uint32_t parts[PARTS];
            split<false>(parts, w0, w1);
#pragma unroll
            for (int n = 0; n < PARTS; ++n) w[t][u][n].w[e] = parts[n];
          }
        if constexpr (UNIFORM) {
          // all weights carry the same scale: their sum is two products with ones
          constexpr uint32_t one = HALF ? 0x3C003C00u : 0x3F803F80u;
          const Operand ones = {{one, one, one, one}};
          f32x4 all = {0, 0, 0, 0};
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int n = 0; n < PARTS; ++n) all = product<V>(ones, w[t][u][n], all);
          part = all[0];
        }
        sum[t] = fmaf(part, by_vs, sum[t]);
      } else {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float weight[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const float score = s[t][u * 2 + e / 2][(e % 2) * 2 + i];
              part += exp2_fast(fmaf(score, unit, -base));
              // a key that a row does not see does not touch it, whatever the scale of its block
              weight[i] = score == -INFINITY ? 0.0f : exp2_fast(fmaf(score, unit, -less)) * times;
            }
            uint32_t parts[PARTS];
            split<true>(parts, weight[0], weight[1]);
#pragma unroll
            for (int n = 0; n < PARTS; ++n) w[t][u][n].w[e] = parts[n];
          }
        sum[t] += UNIFORM ? groups_sum(part) : part;
      }
    }
    // (two loops: a branch for each d would leave each load of a value alone with its wait)
    __builtin_amdgcn_s_setprio(1);
    if constexpr (FP8) {
      if (whole) gather(w, value);
      else gather(w, [&](int d) { return clean(value(d), true); });
    } else {
      gather(w, value);
    }
    __builtin_amdgcn_s_setprio(0);
  }

  template <typename Value>
  __device__ __forceinline__ void gather(const Operand (*w)[2][PARTS], Value value) {
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      const auto codes = value(d);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const Operand v = operand<V, FP8>(codes, u);
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
          for (int n = 0; n < PARTS; ++n) o[t][d] = product<V>(v, w[t][u][n], o[t][d]);
      }
    }
  }

  template <typename Value>
  __device__ __forceinline__ void mark_nans(int at16, bool valid, Value value) {
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      const Vec<uint32_t, 4> w = value(d);
      uint32_t mark[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) mark[i] = nan_bytes(w.v[i]) & 0x38383838u;  // 1.0 as e4m3
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        f32x4 hit = {0, 0, 0, 0};
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          Operand p;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int key = at16 + u * 8 + e * 2;
            p.w[e] = (valid && key < ends[t] ? 0x3F80u : 0u) | (valid && key + 1 < ends[t] ? 0x3F800000u : 0u);
          }
          hit = product<BF16>(widen8<BF16, true>(mark[2 * u], mark[2 * u + 1]), p, hit);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (hit[i] > 0.0f) o[t][d][i] = NAN;
      }
    }
  }

  __device__ __forceinline__ void finish() {
#pragma unroll
    for (int t = 0; t < RT; ++t)
      if constexpr (!UNIFORM) sum[t] = groups_sum(sum[t]);
  }
};

// What a workgroup works on, from its number.  A request has a.tiles workgroups, or, where its
// queries are not known (a.tiles is 0), one for its first tile, and for the further ones those from
// start[r] * share / ROWS on: that leaves room for all of each request before it, and for one
// more at times.  Whose a number is, the wavefront finds with 64 requests at a glance.
// FIRST: first tiles come first (of a decode step there are no others), else last, as the rows
// that see most do not lie in them.
template <int ROWS, bool FIRST>
struct AttendUnit {
  static constexpr int kNone = 0x7FFFFFFF / ROWS;  // a tile behind those of any request
  int kv, chunk, tile, r;
  __device__ __forceinline__ AttendUnit(const AttendArgs& a, int share) {
    int id = blockIdx.x;
    kv = id % a.kv_heads;
    id /= a.kv_heads;
    chunk = id % a.chunks;
    id /= a.chunks;
    if (a.tiles) {
      r = id % a.requests;
      tile = a.tiles - 1 - id / a.requests;  // the rows that see most come first
      return;
    }
    const int unit = FIRST ? id : a.units - 1 - id;
    r = unit, tile = 0;
    if (unit < a.requests) return;
    const int further = unit - a.requests;
    auto first_of = [&](int q) { return (int)((uint32_t)min(max(a.start[q], 0), a.tokens) * (uint32_t)share / ROWS); };
    int n = a.requests;
    r = 0;
    while (n > 1) {
      const int step = (n + kWave - 1) / kWave, at = lane_id() * step;
      const uint64_t begun = __ballot(at < n && first_of(r + min(at, n - 1)) <= further);
      const int skip = max(__builtin_popcountll(begun) - 1, 0) * step;
      r += skip, n = min(step, n - skip);
    }
    tile = further - first_of(r) + 1;
    if (tile < 1) tile = kNone;
  }
  __device__ __forceinline__ int next(const AttendArgs& a, int now) const { return a.tiles ? now + a.tiles : kNone; }
};

// the block of 16 keys from `key` on, and where in it they start
__device__ __forceinline__ int look_up(const AttendArgs& a, int r, int key, int* at, uint32_t nothing = 0) {
  const uint32_t u = (uint32_t)key >> 4;
  const uint32_t index = a.magic ? __umulhi(u, a.magic) : u;
  *at = (int)(u - index * a.sixteenths) * 16;
  return (a.table + (int64_t)r * a.table_stride + min((int)index, a.width - 1))[nothing];
}
__device__ __forceinline__ bool in_pool(const AttendArgs& a, int block) { return (uint32_t)block < (uint32_t)a.num_blocks; }
__device__ __forceinline__ int64_t cell_of(const AttendArgs& a, int block, int kv) {
  return (int64_t)(in_pool(a, block) ? block : 0) * a.kv_heads + kv;
}

// Rows before the first request's and behind the last one's, which become zeros if they are to, a
// share by each workgroup when it is done.  Where they are is asked for when it begins: at the end
// the answer would be waited for (0.5 us).
struct Rest {
  int before, behind;
  __device__ __forceinline__ explicit Rest(const AttendArgs& a) : before(0), behind(a.tokens) {
    if (a.clear) before = a.start[0], behind = a.start[a.requests];
  }
  __device__ __forceinline__ void arrived() { asm volatile("" : "+s"(before), "+s"(behind)); }
  __device__ __forceinline__ void clear(const AttendArgs& a, int dim) {
    if (__builtin_expect(before <= 0 && behind >= a.tokens, 1)) return;
    before = min(max(before, 0), a.tokens), behind = min(max(behind, before), a.tokens);
    const int64_t pieces = (int64_t)a.q_heads * dim / 8, first = before * pieces;
    const int64_t all = (before + a.tokens - behind) * pieces, skip = (behind - before) * pieces;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < all; i += (int64_t)gridDim.x * blockDim.x)
      ((Vec<uint32_t, 4>*)a.out)[i < first ? i : i + skip] = Vec<uint32_t, 4>{};
  }
};

// few rows: the wavefronts of a workgroup share them and split the keys; keys and values go
// from memory into the registers they are multiplied from
template <typename T, bool FP8, int D, int RT>
__global__ __launch_bounds__(kAttendWaves* kWave, D == 256 || RT == 2 ? 1 : 2) void kv_attend_split_kernel(AttendArgs a) {
  using Rows = AttendRows<T, FP8, D, RT, Weights::kTriple, false>;
  constexpr int ROWS = RT * 16, CH = Rows::CH, DT = Rows::DT;
  const int lane = lane_id(), wave = threadIdx.x / kWave, c = lane & 15, j = lane >> 4;
  const int share = a.q_heads / a.kv_heads;
  const AttendUnit<ROWS, true> unit(a, share);
  Rest rest(a);
  const int kv = unit.kv, chunk = unit.chunk, r = unit.r;
  const Request rq = request_of(a, r);
  rest.arrived();
  const int rows = rq.queries * share;
  const int64_t bytes = (int64_t)a.block_size * D;  // of a block's head
  __shared__ float meet_top[kAttendWaves][ROWS], meet_sum[kAttendWaves][ROWS];
  __shared__ float meet_o[kAttendWaves][16][D + 4];

  for (int tile = unit.tile; tile * ROWS < rows; tile = unit.next(a, tile)) {
    const int first = tile * ROWS, tile_end = last_key(rq, min(first + ROWS, rows) - 1, share);
    const int pieces = min(max((tile_end + a.chunk_keys - 1) / a.chunk_keys, 1), a.chunks);
    if (chunk >= pieces) continue;
    Rows w;
    w.begin(a, rq, first, rows, kv, share);
    const int key0 = chunk * a.chunk_keys + wave * kStep;
    int key1 = a.num_blocks ? tile_end : 0;
    if (chunk < pieces - 1) key1 = min(key1, (chunk + 1) * a.chunk_keys);

    constexpr int STRIDE = kAttendWaves * kStep;
    Vec<uint32_t, 4> kw[4][CH], vw[DT];
    float ks = 0.0f, vs = 0.0f;
    int bk, ak, bv, av;  // block and position: of the keys this lane multiplies, of those it gets
    // (not there: all lanes read the pool's first block, the same few lines for every wavefront)
    auto load_keys = [&](int block, int at, bool there) {
      const uint8_t* p = a.key + (there ? cell_of(a, block, kv) * bytes + (at + (c & 3)) * D + j * 16 : 0);
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int ch = 0; ch < CH; ++ch) kw[t][ch] = ldg_nt<uint32_t, 4>((const uint32_t*)(p + t * 4 * D + ch * 64));
    };
    auto load_scales = [&](int block) {
      ks = a.key_scale[cell_of(a, block, kv)];
      vs = a.value_scale[cell_of(a, block, kv)];
    };
    auto load_values = [&](int block, int at, bool there) {
      const uint8_t* p = a.value + (there ? cell_of(a, block, kv) * bytes + c * a.block_size + at : 0);
#pragma unroll
      for (int d = 0; d < DT; ++d) vw[d] = ldg_nt<uint32_t, 4>((const uint32_t*)(p + d * 16 * a.block_size));
    };
    // What a step multiplies is asked for one step before it, where its blocks lie two steps
    // before: no address waits for a load that others were asked for ahead of.  Behind the last
    // step the loads stay, but read nothing new: a branch around them, or around the loop, would
    // make each wait in it one for all of them (6 requests of up to 32768: 91 us so, 81 now; with
    // the last step read again 83).
    if (key0 < key1) {
      const int last = key0 + (key1 - 1 - key0) / STRIDE * STRIDE;
      bk = look_up(a, r, key0 + (c >> 2) * 16, &ak);
      bv = look_up(a, r, key0 + j * 16, &av);
      const int second = min(key0 + STRIDE, last);
      load_keys(bk, ak, true);
      bk = look_up(a, r, second + (c >> 2) * 16, &ak);
      load_scales(bv);
      load_values(bv, av, true);
      int bs = bv;  // block of the scales
      bv = look_up(a, r, second + j * 16, &av);
      for (int kb = key0; kb < key1; kb += STRIDE) {
        const bool valid = in_pool(a, bs);
        const float ks_now = ks * a.scale, vs_now = vs;
        const int later = min(kb + 2 * STRIDE, last);
        const bool more = kb < last;
        w.step(kb, ks_now, vs_now, valid, [&](int t, int ch) { return kw[t][ch]; }, [&](int d) { return vw[d]; },
               [&] {
                 load_keys(bk, ak, more);
                 bk = look_up(a, r, later + (c >> 2) * 16, &ak);
               });
        load_scales(bv);
        load_values(bv, av, more);
        bs = bv;
        bv = look_up(a, r, later + j * 16, &av);
      }
    }
    w.finish();

    // the wavefronts bring their sums to the common maximum and add them in LDS
    if (j == 0) {
#pragma unroll
      for (int t = 0; t < RT; ++t) meet_top[wave][t * 16 + c] = w.top[t], meet_sum[wave][t * 16 + c] = w.sum[t];
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      float all = -INFINITY;
#pragma unroll
      for (int i = 0; i < kAttendWaves; ++i) all = fmaxf(all, meet_top[i][t * 16 + c]);
      const float mine = w.top[t] == -INFINITY ? 0.0f : exp2_fast(w.top[t] - all);
#pragma unroll
      for (int d = 0; d < DT; ++d) *(f32x4*)&meet_o[wave][c][d * 16 + j * 4] = w.o[t][d] * mine;
      __syncthreads();
      // 16 threads a row, 4 numbers at a time
      const int row_in = threadIdx.x / 16, piece = threadIdx.x % 16, row = first + t * 16 + row_in;
      float row_top = -INFINITY, row_sum = 0.0f;
#pragma unroll
      for (int i = 0; i < kAttendWaves; ++i) row_top = fmaxf(row_top, meet_top[i][t * 16 + row_in]);
#pragma unroll
      for (int i = 0; i < kAttendWaves; ++i) {
        const float m = meet_top[i][t * 16 + row_in];
        row_sum += meet_sum[i][t * 16 + row_in] * (m == -INFINITY ? 1.0f : exp2_fast(m - row_top));
      }
      if (row < rows) {
        const int64_t cell = (int64_t)(rq.q0 + row / share) * a.q_heads + kv * share + row % share;
#pragma unroll
        for (int x = 0; x < D / 64; ++x) {
          f32x4 v = {0, 0, 0, 0};
#pragma unroll
          for (int i = 0; i < kAttendWaves; ++i) v += *(const f32x4*)&meet_o[i][row_in][x * 64 + piece * 4];
          if (pieces == 1) {
            const float by = row_sum == 0.0f ? 0.0f : 1.0f / row_sum;
            Vec<uint16_t, 4> h;
#pragma unroll
            for (int e = 0; e < 4; ++e) h.v[e] = T::from_f32(row_sum == 0.0f ? 0.0f : v[e] * by);
            stg(a.out + cell * D + x * 64 + piece * 4, h);
          } else {
            const int64_t at = (int64_t)chunk * a.tokens * a.q_heads + cell;
            *(f32x4*)(a.part_o + at * D + x * 64 + piece * 4) = v;
            if (x == 0 && piece == 0) a.part_ml[at * 2] = row_top, a.part_ml[at * 2 + 1] = row_sum;
          }
        }
      }
      __syncthreads();
    }
  }
  rest.clear(a, D);
}

// many rows: each wavefront has its own, and the workgroup reads the keys and values once,
// 64 keys ahead, into LDS.  A lane's operand is 16 bytes of a row of its own: read from memory
// directly that is one cache line a lane, and the lines a cycle are what bound the kernel
// (measured at 2 x 2000 queries over 4000 keys: 455 us).  Pieces of a row are swapped in LDS
// by some bits of the row's number, so that the rows that are read together lie in different
// banks.
//
// WIDE: blocks are whole steps of 64 keys, so a step lies in one of them: its number, its
// addresses and scales are the wavefront's and cost no vector instruction.
template <typename T, bool FP8, int D, int RT, Weights W, bool WIDE>
__global__ __launch_bounds__(kAttendWaves* kWave, D == 256 ? 1 : 2) void kv_attend_rows_kernel(AttendArgs a) {
  using Rows = AttendRows<T, FP8, D, RT, W, WIDE>;
  constexpr int ROWS = kAttendWaves * RT * 16, PIECES = D / 64;  // 16-byte pieces a thread loads of either
  constexpr int KP = D / 16;                                     // pieces of a key
  constexpr int KEYS = kAttendWaves * kWave / KP;                // keys per round of loads
  const int lane = lane_id(), wave = threadIdx.x / kWave, c = lane & 15, j = lane >> 4;
  const int share = a.q_heads / a.kv_heads;
  const AttendUnit<ROWS, false> unit(a, share);
  Rest rest(a);
  const int kv = unit.kv, chunk = unit.chunk, r = unit.r;
  const Request rq = request_of(a, r);
  rest.arrived();
  const int rows = rq.queries * share;
  const int64_t bytes = (int64_t)a.block_size * D;
  // e4m3 codes stay codes in LDS: one instruction makes two elements of them.  int8 codes take
  // more and are widened on the way in, once for the workgroup (269 against 316 us for the two
  // prompts above; e4m3 266 against 259 that way).  Places count 16 bytes.
  constexpr int PER = FP8 ? 1 : 2;
  __shared__ Vec<uint32_t, 4> keys[2][kStep * KP * PER], values[2][D * 4 * PER];
  auto key_place = [](int key, int piece) {
    return key * KP * PER + (piece ^ (((key & 3) | ((key >> 4) & 1) << 2) & (KP * PER - 1)));
  };
  auto value_place = [](int d, int piece) { return d * 4 * PER + (piece ^ (FP8 ? (d >> 2) & 3 : d & 7)); };
  auto take = [](const Vec<uint32_t, 4>* at, auto place) {  // 16 elements, place(i): their i-th 16 bytes
    if constexpr (FP8) {
      return at[place(0)];
    } else {
      return Operands{{__builtin_bit_cast(Operand, at[place(0)]), __builtin_bit_cast(Operand, at[place(1)])}};
    }
  };

  for (int tile = unit.tile; tile * ROWS < rows; tile = unit.next(a, tile)) {
    const int row0 = tile * ROWS, tile_end = last_key(rq, min(row0 + ROWS, rows) - 1, share);
    const int pieces = min(max((tile_end + a.chunk_keys - 1) / a.chunk_keys, 1), a.chunks);
    if (chunk >= pieces) continue;
    const int first = row0 + wave * RT * 16;
    Rows w;
    w.begin(a, rq, first, rows, kv, share);
    const int key0 = chunk * a.chunk_keys;
    int key1 = a.num_blocks ? tile_end : 0;
    if (chunk < pieces - 1) key1 = min(key1, key0 + a.chunk_keys);

    Vec<uint32_t, 4> kr[PIECES], vr[PIECES];
    float ks = 0.0f, vs = 0.0f;
    int bk[PIECES], ak[PIECES], bv, av, bs_next = 0;  // blocks of the step to load; bs_next: of this lane's 16 keys
    const int my_key = threadIdx.x / KP, my_piece = threadIdx.x % KP, my_group = threadIdx.x % 4, my_d = threadIdx.x / 4;
    uint32_t nothing = 0;  // which only the lanes know: what is read with it stays theirs until found()
    asm volatile("" : "+v"(nothing));
    auto find = [&](int kb) {
      if constexpr (WIDE) {
        bv = look_up(a, r, __builtin_amdgcn_readfirstlane(kb), &av, nothing);
        av = __builtin_amdgcn_readfirstlane(av);
      } else {
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
          const int key = kb + my_key + p * KEYS;
          bk[p] = look_up(a, r, key, &ak[p]);
          ak[p] += key & 15;
        }
        bv = look_up(a, r, kb + my_group * 16, &av);
      }
    };
    // What find and load ask for is first looked at when a step is over: a number made uniform or
    // multiplied where it is asked for would hold the step up until it is there, with all that
    // was asked for before it (blocks of 16: 277 us so, 258 now; 64 dimensions 181 and 165).
    auto found = [&] {
      if constexpr (WIDE) bv = __builtin_amdgcn_readfirstlane(bv);
    };
    const uint32_t key_at = threadIdx.x * 16, value_at = my_d * a.block_size + my_group * 16, value_step = 64 * a.block_size;
    auto load = [&] {
      if constexpr (WIDE) {
        const int64_t cell = cell_of(a, bv, kv);
        const uint8_t *k = a.key + cell * bytes + av * D, *v = a.value + cell * bytes + av;
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
          kr[p] = ldg<uint32_t, 4>((const uint32_t*)(k + (key_at + p * kAttendWaves * kWave * 16)));
          vr[p] = ldg<uint32_t, 4>((const uint32_t*)(v + (value_at + p * value_step)));
        }
        bs_next = bv;
        ks = a.key_scale[cell];
        vs = a.value_scale[cell];
      } else {
#pragma unroll
        for (int p = 0; p < PIECES; ++p)
          kr[p] = ldg<uint32_t, 4>((const uint32_t*)(a.key + cell_of(a, bk[p], kv) * bytes + ak[p] * D + my_piece * 16));
        const uint8_t* v = a.value + cell_of(a, bv, kv) * bytes + value_at - my_group * 16 + av;
#pragma unroll
        for (int p = 0; p < PIECES; ++p) vr[p] = ldg<uint32_t, 4>((const uint32_t*)(v + p * value_step));
        bs_next = __shfl(bv, j, kWave);  // lane j's group is j
        ks = a.key_scale[cell_of(a, bs_next, kv)];
        vs = a.value_scale[cell_of(a, bs_next, kv)];
      }
    };
    auto store = [&](int half) {
#pragma unroll
      for (int p = 0; p < PIECES; ++p) {
        const int key = my_key + p * KEYS, d = my_d + p * 64;
        if constexpr (FP8) {
          keys[half][key_place(key, my_piece)] = kr[p];
          values[half][value_place(d, my_group)] = vr[p];
        } else {
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            using Bits = Vec<uint32_t, 4>;
            keys[half][key_place(key, my_piece * 2 + u)] = __builtin_bit_cast(Bits, operand<T, FP8>(kr[p], u));
            values[half][value_place(d, my_group * 2 + u)] = __builtin_bit_cast(Bits, operand<typename Rows::V, FP8>(vr[p], u));
          }
        }
      }
    };
    __syncthreads();  // the tile before may still be read
    if (key0 < key1) {
      find(key0);
      found();
      load();
      find(key0 + kStep);
      store(0);
      found();
    }
    __syncthreads();
    w.arrived();
    int half = 0;
    for (int kb = key0; kb < key1; kb += kStep, half ^= 1) {
      const float ks_now = ks * a.scale, vs_now = vs;
      const bool valid = in_pool(a, bs_next);
      load();  // behind the last step, too: the table's last block, or the pool's first
      find(kb + 2 * kStep);
      if (kb < w.seen_by_any)
        w.step(kb, ks_now, vs_now, valid,
               [&](int t, int ch) {
                 const int key = (c >> 2) * 16 + t * 4 + (c & 3);
                 return take(keys[half], [&](int i) { return key_place(key, (ch * 4 + j) * PER + i); });
               },
               [&](int d) { return take(values[half], [&](int i) { return value_place(d * 16 + c, j * PER + i); }); },
               [] {});
      store(half ^ 1);
      found();
      __syncthreads();
    }
    w.finish();
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const int row = first + t * 16 + c;
      if (row >= rows) continue;
      const int64_t cell = (int64_t)(rq.q0 + row / share) * a.q_heads + kv * share + row % share;
      if (pieces == 1) {
        const float by = w.sum[t] == 0.0f ? 0.0f : 1.0f / w.sum[t];
#pragma unroll
        for (int d = 0; d < Rows::DT; ++d) {
          Vec<uint16_t, 4> h;
#pragma unroll
          for (int e = 0; e < 4; ++e) h.v[e] = T::from_f32(w.sum[t] == 0.0f ? 0.0f : w.o[t][d][e] * by);
          stg(a.out + cell * D + d * 16 + j * 4, h);
        }
      } else {
        const int64_t at = (int64_t)chunk * a.tokens * a.q_heads + cell;
#pragma unroll
        for (int d = 0; d < Rows::DT; ++d) *(f32x4*)(a.part_o + at * D + d * 16 + j * 4) = w.o[t][d];
        if (j == 0) a.part_ml[at * 2] = w.top[t], a.part_ml[at * 2 + 1] = w.sum[t];
      }
    }
  }
  rest.clear(a, D);
}

// brings the chunks of a row together: one wavefront per token and head
template <typename T, int D>
__global__ __launch_bounds__(kAttendWaves* kWave) void kv_attend_join_kernel(AttendArgs a, int tile_rows, int max_query) {
  constexpr int PER = D / kWave;
  const int lane = lane_id();
  const int64_t id = (int64_t)blockIdx.x * kAttendWaves + threadIdx.x / kWave;
  const int head = (int)(id % a.q_heads);
  const int64_t rest = id / a.q_heads;
  const int r = (int)(rest / max_query), share = a.q_heads / a.kv_heads;
  if (r >= a.requests) return;
  const Request rq = request_of(a, r);
  const int rows = rq.queries * share;
  for (int i = (int)(rest % max_query); i < rq.queries; i += max_query) {
    const int row0 = (i * share + head % share) / tile_rows * tile_rows;
    const int tile_end = last_key(rq, min(row0 + tile_rows, rows) - 1, share);
    const int pieces = min(max((tile_end + a.chunk_keys - 1) / a.chunk_keys, 1), a.chunks);
    if (pieces == 1) continue;
    const int64_t cell = (int64_t)(rq.q0 + i) * a.q_heads + head, step = (int64_t)a.tokens * a.q_heads;
    // lane p holds the weight of chunk p; 64 at a time
    float top = -INFINITY;
    for (int p = lane; p < pieces; p += kWave) top = fmaxf(top, a.part_ml[(p * step + cell) * 2]);
#pragma unroll
    for (int m = 1; m < kWave; m *= 2) top = fmaxf(top, wave_shfl_xor(top, m));
    float sum = 0.0f, o[PER] = {};
    for (int p0 = 0; p0 < pieces; p0 += kWave) {
      float w = 0.0f, part = 0.0f;
      if (p0 + lane < pieces) {
        const int64_t at = ((p0 + lane) * step + cell) * 2;
        const float m = a.part_ml[at];
        w = m == -INFINITY ? 0.0f : exp2_fast(m - top);
        part = a.part_ml[at + 1] * (m == -INFINITY ? 1.0f : w);  // a chunk without a maximum: 0, or NaN
      }
#pragma unroll
      for (int m = 1; m < kWave; m *= 2) part += wave_shfl_xor(part, m);
      sum += part;
      const int n = min(pieces - p0, kWave);
      for (int p = 0; p < n; p += 8) {
        Vec<float, PER> v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e)  // the last ones again, with no weight, behind the last
          v[e] = ldg<float, PER>(a.part_o + ((p0 + min(p + e, n - 1)) * step + cell) * D + lane * PER);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float by = p + e < n ? __shfl(w, p + e, kWave) : 0.0f;
#pragma unroll
          for (int x = 0; x < PER; ++x) o[x] = by == 0.0f ? o[x] : fmaf(by, v[e].v[x], o[x]);
        }
      }
    }
    const float by = sum == 0.0f ? 0.0f : 1.0f / sum;
    Vec<uint16_t, PER> h;
#pragma unroll
    for (int e = 0; e < PER; ++e) h.v[e] = T::from_f32(sum == 0.0f ? 0.0f : o[e] * by);
    stg(a.out + cell * D + lane * PER, h);
  }
}

// Weights where rows are many and products the bound: bf16 outputs take one f16 number (2^-11 of
// the weight, a quarter of half an output's step, at the price of one bf16 number; two numbers would
// take 295 for 246 us at 2 x 2000 queries over 4000 keys), f16 outputs two bf16 numbers (2^-16).
// Where rows are few memory is the bound and weights keep all their bits.
template <typename T>
constexpr Weights kRows = T::id == CTMI_F16 ? Weights::kPair : Weights::kHalf;

// the launch: which kernel, how many tiles of rows and chunks of keys a request gets
struct Launch {
  bool split_keys;
  int row_tiles, tile_rows;
  int64_t tiles, units, chunks, chunk_keys;
  int64_t most_chunks;   // of any shorter max_seq, too
  int64_t join_queries;  // a wavefront of the joining kernel has every so manyth query of a request
};

// A max_query above the tokens is one that the caller does not know.  No more tokens than requests
// are then taken for a decode step, others for prompts, of which any may have all tokens (64
// requests of 2500 keys, a token each: 58 us, as with hints; laid out for prompts 84).
Launch plan_launch(int64_t tokens, int64_t requests, int32_t q_heads, int32_t kv_heads, int32_t head_dim,
                   int64_t max_query, int64_t max_seq) {
  constexpr int64_t kMost = 1 << 23;  // workgroups: a request of more tiles has each walk some
  Launch l;
  const bool known = max_query <= tokens;
  const int64_t mean = cdiv(tokens, requests), share = q_heads / kv_heads;
  const int64_t rows = (known ? max_query : mean == 1 ? 1 : tokens) * share;
  // Up to 64 rows a request share their keys' operands with nobody worth the trip through LDS.
  // 4 requests of 1500 keys, split against rows: 32 rows 16.0 and 17.7 us, 64 rows 19.7 and 19.3, 128
  // rows 26.4 and 23.7.  At 64 rows 16 requests of 500 keys 15.8 and 23.5, 32 of 2000 70 and 67, 64
  // of 4000 240 and 157.
  l.split_keys = rows <= 64;
  l.row_tiles = head_dim == 256 || rows <= 16 ? 1 : 2;
  l.tile_rows = (l.split_keys ? 1 : kAttendWaves) * l.row_tiles * 16;
  l.tiles = cdiv(rows, l.tile_rows);
  // As many workgroups as are resident at once (two per compute unit; one, where registers
  // leave room for one), in one go: with 512 of them 64 x 4096 takes 81 to 88 us, with 768 121 and
  // with 1024 to 2048 89 to 98; 4 requests of 16 queries over 1500 keys 18 us with 192, with 384,
  // one and a half times what is resident, 25.
  constexpr int64_t kFloor = 256;
  const int64_t resident = head_dim == 256 || (l.split_keys && l.row_tiles == 2) ? 256 : 512;
  const int64_t units = requests * kv_heads * l.tiles;
  int64_t chunks = resident / (units < resident ? units : resident);
  // a chunk's sums leave and come back in fp32: not for more rows than the keys they stand for
  if (!l.split_keys && units >= resident / 2) chunks = 1;
  // Bringing parts together is a launch, and costs what 1024 keys do (32 requests, 1000 keys:
  // one workgroup each 17 us, two 21; 2000 keys 26 and 33; one request, 2000 keys: 16, eight 11)
  if (l.split_keys && max_seq * (chunks - 1) <= 1024 * chunks) chunks = 1;
  int64_t keys = cdiv(cdiv(max_seq, chunks), 256) * 256;
  if (keys < kFloor) keys = kFloor;
  l.chunk_keys = chunks == 1 && !l.split_keys ? 1 << 30 : keys;
  // Requests of very different lengths: the long ones are cut further.  With 4096, 8192, 16384 and
  // no limit, one request of 60000 keys beside 63 of 1000: 73, 104, 151 and 454 us; 64 of between 300
  // and 32768 300, 369, 344 and 453; 6 of 20000 50.8, 48.2, 47.6 and 47.3.
  constexpr int64_t kLongest = 8192;
  if (l.split_keys && l.chunk_keys > kLongest) l.chunk_keys = kLongest;
  l.chunks = cdiv(max_seq, l.chunk_keys);
  l.most_chunks = cdiv(max_seq, kFloor) < chunks ? cdiv(max_seq, kFloor) : chunks;
  if (l.split_keys && cdiv(max_seq, kLongest) > l.most_chunks) l.most_chunks = cdiv(max_seq, kLongest);
  const int64_t most = kMost / (requests * l.chunks * kv_heads);
  if (l.tiles > most) l.tiles = most < 1 ? 1 : most;
  l.units = requests * l.tiles;
  if (!known) l.tiles = 0, l.units = requests + tokens * share / l.tile_rows;
  l.join_queries = known ? max_query : mean;
  if (l.join_queries > kMost / (requests * q_heads)) l.join_queries = kMost / (requests * q_heads) < 1 ? 1 : kMost / (requests * q_heads);
  return l;
}

}  // namespace
}  // namespace ctmi

using namespace ctmi;

extern "C" int64_t ctmi_kv_attend_tmp_bytes(int64_t tokens, int64_t requests, int32_t q_heads,
                                            int32_t kv_heads, int32_t head_dim, int64_t max_query,
                                            int64_t max_seq) {
  if (tokens < 1 || requests < 1 || q_heads < 1 || kv_heads < 1 || max_query < 1 || max_seq < 1) return 0;
  if (max_seq > 1ll << 30) max_seq = 1ll << 30;
  const Launch l = plan_launch(tokens, requests, q_heads, kv_heads, head_dim, max_query, max_seq);
  return l.most_chunks > 1 ? l.most_chunks * tokens * q_heads * (head_dim + 2) * 4 : 0;
}

static int attend(bool clear, const void* q, int32_t dtype, int64_t q_token_stride, int64_t q_head_stride, void* out,
                  int64_t tokens, int32_t q_heads, const ctmi_kv_blocks* blocks, const int32_t* block_table,
                  int64_t table_stride, int64_t width, const int32_t* seq_lens, const int32_t* query_start,
                  int64_t requests, float scale, int64_t max_query, int64_t max_seq, void* tmp, int64_t tmp_bytes,
                  void* stream) {
  CTMI_REQUIRE(dtype == CTMI_BF16 || dtype == CTMI_F16, CTMI_ERR_UNSUPPORTED,
               "queries must be bfloat16 or float16");
  const int rc = check_kv_blocks(blocks);
  if (rc != CTMI_OK) return rc;
  CTMI_REQUIRE(q_heads >= 1 && q_heads % blocks->kv_heads == 0, CTMI_ERR_VALUE,
               "%d query heads are no multiple of %d key heads", q_heads, blocks->kv_heads);
  CTMI_REQUIRE(tokens >= 0 && requests >= 0 && width >= 0 && table_stride >= width, CTMI_ERR_VALUE,
               "bad sizes: %lld tokens, %lld requests, %lld table columns, stride %lld", (long long)tokens,
               (long long)requests, (long long)width, (long long)table_stride);
  CTMI_REQUIRE(tokens < (1ll << 30) / q_heads && requests < (1ll << 30) &&
                   width < (1ll << 30) / blocks->block_size,
               CTMI_ERR_UNSUPPORTED, "tokens x heads, requests and positions must stay below 2^30");
  CTMI_REQUIRE(query_start != nullptr || tokens == requests, CTMI_ERR_VALUE,
               "without query_start every request has one token: got %lld tokens for %lld requests",
               (long long)tokens, (long long)requests);
  CTMI_REQUIRE(max_query >= 1 && max_seq >= 1, CTMI_ERR_VALUE, "max_query and max_seq must be at least 1");
  if (tokens == 0 || requests == 0) return CTMI_OK;
  CTMI_REQUIRE(q && out && seq_lens && (width == 0 || block_table), CTMI_ERR_VALUE, "NULL tensor");
  CTMI_REQUIRE(q_token_stride % 8 == 0 && q_head_stride % 8 == 0 && ((uintptr_t)q | (uintptr_t)out) % 16 == 0,
               CTMI_ERR_VALUE, "queries must be 16-byte aligned, token by token and head by head");
  const int32_t dim = blocks->head_dim;
  if (query_start == nullptr && max_query > tokens) max_query = 1;  // known after all; the same launch
  if (max_seq > width * blocks->block_size) max_seq = width * blocks->block_size > 0 ? width * blocks->block_size : 1;
  const Launch l = plan_launch(tokens, requests, q_heads, blocks->kv_heads, dim, max_query, max_seq);
  const int64_t cells = l.chunks > 1 ? l.chunks * tokens * q_heads : 0;
  CTMI_REQUIRE(tmp_bytes >= cells * (dim + 2) * 4 && (cells == 0 || (tmp != nullptr && (uintptr_t)tmp % 16 == 0)),
               CTMI_ERR_VALUE, "tmp needs %lld bytes at a 16-byte boundary, has %lld", (long long)(cells * (dim + 2) * 4),
               (long long)tmp_bytes);
  const int64_t grid = l.units * l.chunks * blocks->kv_heads;
  const int64_t join = cdiv(requests * l.join_queries * q_heads, (int64_t)kAttendWaves);
  CTMI_REQUIRE(grid < (1ll << 24) && (cells == 0 || join < (1ll << 24)), CTMI_ERR_UNSUPPORTED, "too many requests and heads for one launch");
  const uint32_t sixteenths = blocks->block_size / 16;
  AttendArgs a{(const uint16_t*)q, q_token_stride, q_head_stride, (uint16_t*)out,
               (const uint8_t*)blocks->key, (const uint8_t*)blocks->value, blocks->key_scale,
               blocks->value_scale, block_table, seq_lens, query_start, (float*)tmp,
               (float*)tmp + cells * dim, table_stride, (int32_t)blocks->num_blocks, blocks->kv_heads,
               blocks->block_size, q_heads, (int32_t)width, (int32_t)tokens, (int32_t)requests,
               (int32_t)l.tiles, (int32_t)l.units, (int32_t)l.chunks, (int32_t)l.chunk_keys, sixteenths,
               sixteenths == 1 ? 0u : (uint32_t)(((1ull << 32) + sixteenths - 1) / sixteenths),
               scale * kLog2e, clear && query_start != nullptr};
  const hipStream_t s = (hipStream_t)stream;
  const dim3 blocks_of((unsigned)grid), threads(kAttendWaves * kWave);
  const bool fp8 = blocks->code_dtype == CTMI_F8E4M3;
#define BY_TILE(T, F, D)                                                                                           \
  do {                                                                                                             \
    constexpr int RT2 = D == 256 ? 1 : 2;                                                                          \
    if (!l.split_keys && a.block_size % kStep == 0)                                                                \
      kv_attend_rows_kernel<T, F, D, RT2, kRows<T>, true><<<blocks_of, threads, 0, s>>>(a);               \
    else if (!l.split_keys)                                                                                        \
      kv_attend_rows_kernel<T, F, D, RT2, kRows<T>, false><<<blocks_of, threads, 0, s>>>(a);              \
    else if (RT2 == 1 || l.row_tiles == 1) kv_attend_split_kernel<T, F, D, 1><<<blocks_of, threads, 0, s>>>(a);    \
    else kv_attend_split_kernel<T, F, D, RT2><<<blocks_of, threads, 0, s>>>(a);                                    \
    if (cells) kv_attend_join_kernel<T, D><<<dim3((unsigned)join), threads, 0, s>>>(a, l.tile_rows, (int)l.join_queries); \
  } while (0)
#define BY_CODE(T, D) do { if (fp8) BY_TILE(T, true, D); else BY_TILE(T, false, D); } while (0)
#define BY_DIM(T) do { if (dim == 64) BY_CODE(T, 64); else if (dim == 128) BY_CODE(T, 128); else BY_CODE(T, 256); } while (0)
  if (dtype == CTMI_BF16) BY_DIM(BF16);
  else BY_DIM(F16);
#undef BY_DIM
#undef BY_CODE
#undef BY_TILE
  return check_launch("kv_attend");
}

extern "C" int ctmi_kv_attend(const void* q, int32_t dtype, int64_t q_token_stride, int64_t q_head_stride,
                              void* out, int64_t tokens, int32_t q_heads, const ctmi_kv_blocks* blocks,
                              const int32_t* block_table, int64_t table_stride, int64_t width,
                              const int32_t* seq_lens, const int32_t* query_start, int64_t requests,
                              float scale, int64_t max_query, int64_t max_seq, void* tmp,
                              int64_t tmp_bytes, void* stream) {
  return attend(false, q, dtype, q_token_stride, q_head_stride, out, tokens, q_heads, blocks, block_table,
                table_stride, width, seq_lens, query_start, requests, scale, max_query, max_seq, tmp, tmp_bytes, stream);
}

extern "C" int ctmi_kv_attend_padded(const void* q, int32_t dtype, int64_t q_token_stride, int64_t q_head_stride,
                                     void* out, int64_t tokens, int32_t q_heads, const ctmi_kv_blocks* blocks,
                                     const int32_t* block_table, int64_t table_stride, int64_t width,
                                     const int32_t* seq_lens, const int32_t* query_start, int64_t requests,
                                     float scale, int64_t max_query, int64_t max_seq, void* tmp,
                                     int64_t tmp_bytes, void* stream) {
  CTMI_REQUIRE(requests >= 1 || tokens < 1, CTMI_ERR_VALUE, "no request to take the rows of %lld tokens", (long long)tokens);
  return attend(true, q, dtype, q_token_stride, q_head_stride, out, tokens, q_heads, blocks, block_table,
                table_stride, width, seq_lens, query_start, requests, scale, max_query, max_seq, tmp, tmp_bytes, stream);
}
