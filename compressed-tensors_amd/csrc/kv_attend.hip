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
//   O^T = V^T P^T head_dim / 16 tiles x 2 products, P as bf16
//
// Both operands that come from memory are what the lanes already hold: a product's result has
// its rows (keys) in lane group j = lane / 16 and its columns (query rows) in lane % 16, and
// the second product wants keys in groups j, too.  Taking key (r / 4) * 16 + t * 4 + r % 4 as
// row r of key tile t gives group j the 16 neighbouring keys 16 j ... 16 j + 15: P needs no
// exchange, and with tokens innermost in the value blocks a lane's V operand is one 16-byte
// load.  No LDS in the loop; keys and values go from memory into operand registers, the next
// step's keys are requested when this step's are used up, and so are the values.
//
// KS: the four wavefronts of a workgroup share the rows and split the keys (few rows: a
// decode step) and meet in LDS at the end; otherwise they take rows of their own.  A long
// axis is cut into chunks for several workgroups, whose unnormalised sums, maxima and
// weights meet in a second, small kernel.
#include "kv_blocks.h"

namespace ctmi {
namespace {

constexpr int kAttendWaves = 4;
constexpr int kStep = 64;  // keys per step of a wavefront
constexpr float kLog2e = 1.4426950408889634f;

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
  int32_t tiles, chunks, chunk_keys;  // of the grid
  uint32_t sixteenths, magic;         // block_size / 16 and ceil(2^32 / that) (0: it is 1)
  float scale;                        // times log2(e)
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

template <typename T, bool FP8, int D, int RT, bool KS, bool SPLIT>
__global__ __launch_bounds__(kAttendWaves* kWave) void kv_attend_kernel(AttendArgs a) {
  constexpr int CH = D / 64;   // 16-byte pieces of a key per lane
  constexpr int DT = D / 16;   // tiles of the output's dimensions
  constexpr int ROWS = (KS ? 1 : kAttendWaves) * RT * 16;  // of a workgroup
  const int lane = lane_id(), wave = threadIdx.x / kWave, c = lane & 15, j = lane >> 4;
  const int share = a.q_heads / a.kv_heads;
  int id = blockIdx.x;
  const int kv = id % a.kv_heads;
  id /= a.kv_heads;
  const int chunk = id % a.chunks;
  id /= a.chunks;
  const int tile0 = a.tiles - 1 - id % a.tiles;  // the rows that see most come first
  const int r = id / a.tiles;
  const Request rq = request_of(a, r);
  const int rows = rq.queries * share;
  const int64_t bytes = (int64_t)a.block_size * D;  // of a block's head

  for (int tile = tile0; tile * ROWS < rows; tile += a.tiles) {
    const int row0 = tile * ROWS, tile_end = last_key(rq, min(row0 + ROWS, rows) - 1, share);
    const int pieces = min(max((tile_end + a.chunk_keys - 1) / a.chunk_keys, 1), a.chunks);
    if (chunk >= pieces) continue;
    const int first = row0 + (KS ? 0 : wave * RT * 16);  // this wavefront's rows
    const int key0 = chunk * a.chunk_keys;
    int key1 = first < rows ? last_key(rq, min(first + RT * 16, rows) - 1, share) : 0;
    const int seen_by_any = key1, seen_by_all = first < rows ? last_key(rq, first, share) : 0;
    if (chunk < pieces - 1) key1 = min(key1, key0 + a.chunk_keys);
    if (a.num_blocks == 0) key1 = 0;

    // queries: column c of the products, dimensions ch * 64 + j * 16 + half * 8 + 0 ... 7
    Operand q[RT][CH][2];
    int ends[RT];
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
    }

    f32x4 o[RT][DT];
    float top[RT], sum[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      top[t] = -INFINITY, sum[t] = 0.0f;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[t][d] = f32x4{0, 0, 0, 0};
    }

    const int stride = KS ? kAttendWaves * kStep : kStep;
    const int begin = key0 + (KS ? wave * kStep : 0);
    // which block holds 16 keys, and where in it they start
    auto look_up = [&](int key, int* at) {
      const uint32_t u = (uint32_t)key >> 4;
      const uint32_t index = a.magic ? __umulhi(u, a.magic) : u;
      *at = (int)(u - index * a.sixteenths) * 16;
      return a.table[(int64_t)r * a.table_stride + min((int)index, a.width - 1)];
    };
    Vec<uint32_t, 4> kw[4][CH], vw[DT];
    float ks = 0.0f, vs = 0.0f;
    int bk, ak, bv, av;  // block and position: of the keys this lane multiplies, of those it gets
    auto load_keys = [&](int block, int at) {
      block = (uint32_t)block < (uint32_t)a.num_blocks ? block : 0;
      const uint8_t* p = a.key + ((int64_t)block * a.kv_heads + kv) * bytes + (at + (c & 3)) * D + j * 16;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int ch = 0; ch < CH; ++ch) kw[t][ch] = ldg_nt<uint32_t, 4>((const uint32_t*)(p + t * 4 * D + ch * 64));
    };
    auto load_scales = [&](int block) {
      block = (uint32_t)block < (uint32_t)a.num_blocks ? block : 0;
      ks = a.key_scale[(int64_t)block * a.kv_heads + kv];
      vs = a.value_scale[(int64_t)block * a.kv_heads + kv];
    };
    auto load_values = [&](int block, int at) {
      block = (uint32_t)block < (uint32_t)a.num_blocks ? block : 0;
      const uint8_t* p = a.value + ((int64_t)block * a.kv_heads + kv) * bytes + c * a.block_size + at;
#pragma unroll
      for (int d = 0; d < DT; ++d) vw[d] = ldg_nt<uint32_t, 4>((const uint32_t*)(p + d * 16 * a.block_size));
    };
    if (begin < key1) {
      bk = look_up(begin + (c >> 2) * 16, &ak);
      bv = look_up(begin + j * 16, &av);
      load_keys(bk, ak);
      load_scales(bv);
      load_values(bv, av);
    }
    for (int kb = begin; kb < key1; kb += stride) {
      const bool more = kb + stride < key1;
      const bool valid = (uint32_t)bv < (uint32_t)a.num_blocks;
      const float ks_now = ks * a.scale, vs_now = vs;
      const int at16 = kb + j * 16;  // first of this lane's 16 keys
      int bk1 = 0, ak1 = 0, bv1 = 0, av1 = 0;
      if (more) {
        bk1 = look_up(kb + stride + (c >> 2) * 16, &ak1);
        bv1 = look_up(kb + stride + j * 16, &av1);
      }
      f32x4 s[RT][4];
#pragma unroll
      for (int kt = 0; kt < 4; ++kt) {
#pragma unroll
        for (int t = 0; t < RT; ++t) s[t][kt] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int ch = 0; ch < CH; ++ch) {
          const Operand k0 = widen8<T, FP8>(kw[kt][ch].v[0], kw[kt][ch].v[1]);
          const Operand k1 = widen8<T, FP8>(kw[kt][ch].v[2], kw[kt][ch].v[3]);
#pragma unroll
          for (int t = 0; t < RT; ++t) {
            s[t][kt] = product<T>(k0, q[t][ch][0], s[t][kt]);
            s[t][kt] = product<T>(k1, q[t][ch][1], s[t][kt]);
          }
        }
      }
      if (more) {
        load_keys(bk1, ak1);
        load_scales(bv1);
      }
      // a step that every row sees whole skips all of this
      const bool whole = kb + kStep <= seen_by_all && __all(valid);
      if (!whole) {
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
          for (int kt = 0; kt < 4; ++kt)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (!valid || at16 + kt * 4 + i >= ends[t]) s[t][kt][i] = -INFINITY;
              else s[t][kt][i] *= ks_now;
        // values at keys that no row sees: whatever is there, its weight is 0 and must stay so
        const int seen = valid ? min(max(seen_by_any - at16, 0), 16) : 0;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const int n = min(max(seen - w * 4, 0), 4);
          const uint32_t keep = n == 4 ? 0xFFFFFFFFu : (1u << (8 * n)) - 1u;
#pragma unroll
          for (int d = 0; d < DT; ++d) vw[d].v[w] &= keep;
        }
        if constexpr (FP8) {
          // a NaN value at a key that some rows see and others do not: 0 * NaN would reach
          // them all.  Take it out and count it by a product of its own.
          uint32_t any = 0;
#pragma unroll
          for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int w = 0; w < 4; ++w) any |= nan_bytes(vw[d].v[w]);
          if (__any(any != 0)) {
#pragma unroll
            for (int d = 0; d < DT; ++d) {
              uint32_t mark[4];
#pragma unroll
              for (int w = 0; w < 4; ++w) {
                const uint32_t n = nan_bytes(vw[d].v[w]);
                vw[d].v[w] &= ~n;
                mark[w] = n & 0x38383838u;  // 1.0 as e4m3
              }
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
        }
      } else {
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
          for (int kt = 0; kt < 4; ++kt)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[t][kt][i] *= ks_now;
      }

      Operand hi[RT][2], lo[RT][2];
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        float m = s[t][0][0];
#pragma unroll
        for (int kt = 0; kt < 4; ++kt)
#pragma unroll
          for (int i = 0; i < 4; ++i) m = fmaxf(m, s[t][kt][i]);
        m = groups_max(m);
        // weights may exceed 1 by 2^8 before the sums are brought to a new maximum: fp32 and
        // bf16 keep their relative precision there
        if (__any(m > top[t] + 8.0f)) {
          const float now = fmaxf(top[t], m);
          const float shrink = top[t] == -INFINITY ? 0.0f : exp2_fast(top[t] - now);
          top[t] = now;
          sum[t] *= shrink;
#pragma unroll
          for (int d = 0; d < DT; ++d) o[t][d] *= shrink;
        }
        const float base = top[t] == -INFINITY ? 0.0f : top[t];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float p0 = exp2_fast(s[t][u * 2 + e / 2][(e % 2) * 2] - base);
            const float p1 = exp2_fast(s[t][u * 2 + e / 2][(e % 2) * 2 + 1] - base);
            sum[t] += p0 + p1;
            // a hidden key's weight is 0 whatever its block's scale
            const float w0 = p0 == 0.0f ? 0.0f : p0 * vs_now, w1 = p1 == 0.0f ? 0.0f : p1 * vs_now;
            hi[t][u].w[e] = pack_bf16x2(w0, w1);
            if constexpr (SPLIT)
              lo[t][u].w[e] = pack_bf16x2(w0 - u2f(hi[t][u].w[e] << 16), w1 - u2f(hi[t][u].w[e] & 0xFFFF0000u));
          }
      }
#pragma unroll
      for (int d = 0; d < DT; ++d) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const Operand v = widen8<BF16, FP8>(vw[d].v[2 * u], vw[d].v[2 * u + 1]);
#pragma unroll
          for (int t = 0; t < RT; ++t) {
            o[t][d] = product<BF16>(v, hi[t][u], o[t][d]);
            if constexpr (SPLIT) o[t][d] = product<BF16>(v, lo[t][u], o[t][d]);
          }
        }
      }
      if (more) load_values(bv1, av1);
      bv = bv1;
    }
#pragma unroll
    for (int t = 0; t < RT; ++t) sum[t] = groups_sum(sum[t]);

    if constexpr (KS) {
      // the wavefronts bring their sums to the common maximum and add them in LDS
      __shared__ float meet_top[kAttendWaves][RT * 16], meet_sum[kAttendWaves][RT * 16];
      __shared__ float meet_o[kAttendWaves][16][D + 4];
      if (j == 0) {
#pragma unroll
        for (int t = 0; t < RT; ++t) meet_top[wave][t * 16 + c] = top[t], meet_sum[wave][t * 16 + c] = sum[t];
      }
      __syncthreads();
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        float all = -INFINITY, total = 0.0f;
#pragma unroll
        for (int w = 0; w < kAttendWaves; ++w) all = fmaxf(all, meet_top[w][t * 16 + c]);
#pragma unroll
        for (int w = 0; w < kAttendWaves; ++w) {
          const float m = meet_top[w][t * 16 + c];
          if (m != -INFINITY) total += meet_sum[w][t * 16 + c] * exp2_fast(m - all);
        }
        const float mine = top[t] == -INFINITY ? 0.0f : exp2_fast(top[t] - all);
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          const f32x4 v = o[t][d] * mine;
          *(f32x4*)&meet_o[wave][c][d * 16 + j * 4] = v;
        }
        __syncthreads();
        // 16 rows x D: 16 threads a row, 4 numbers at a time; the row's maximum and sum come
        // from a lane that has them (lane % 16 is the row there)
        const int row_in = threadIdx.x / 16, piece = threadIdx.x % 16;
        float row_all = -INFINITY, row_total = 0.0f;
#pragma unroll
        for (int w = 0; w < kAttendWaves; ++w) row_all = fmaxf(row_all, meet_top[w][t * 16 + row_in]);
#pragma unroll
        for (int w = 0; w < kAttendWaves; ++w) {
          const float m = meet_top[w][t * 16 + row_in];
          if (m != -INFINITY) row_total += meet_sum[w][t * 16 + row_in] * exp2_fast(m - row_all);
        }
        const int row = first + t * 16 + row_in;
        if (row < rows) {
          const int64_t cell = (int64_t)(rq.q0 + row / share) * a.q_heads + kv * share + row % share;
#pragma unroll
          for (int x = 0; x < D / 64; ++x) {
            f32x4 v = {0, 0, 0, 0};
#pragma unroll
            for (int w = 0; w < kAttendWaves; ++w) v += *(const f32x4*)&meet_o[w][row_in][x * 64 + piece * 4];
            if (pieces == 1) {
              const float by = row_total == 0.0f ? 0.0f : 1.0f / row_total;
              Vec<uint16_t, 4> h;
#pragma unroll
              for (int e = 0; e < 4; ++e) h.v[e] = T::from_f32(row_total == 0.0f ? 0.0f : v[e] * by);
              stg(a.out + cell * D + x * 64 + piece * 4, h);
            } else {
              const int64_t at = (int64_t)chunk * a.tokens * a.q_heads + cell;
              *(f32x4*)(a.part_o + at * D + x * 64 + piece * 4) = v;
              if (x == 0 && piece == 0) a.part_ml[at * 2] = row_all, a.part_ml[at * 2 + 1] = row_total;
            }
          }
        }
        __syncthreads();
        (void)total;
      }
    } else {
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        const int row = first + t * 16 + c;
        if (row >= rows) continue;
        const int64_t cell = (int64_t)(rq.q0 + row / share) * a.q_heads + kv * share + row % share;
        if (pieces == 1) {
          const float by = sum[t] == 0.0f ? 0.0f : 1.0f / sum[t];
#pragma unroll
          for (int d = 0; d < DT; ++d) {
            Vec<uint16_t, 4> h;
#pragma unroll
            for (int e = 0; e < 4; ++e) h.v[e] = T::from_f32(sum[t] == 0.0f ? 0.0f : o[t][d][e] * by);
            stg(a.out + cell * D + d * 16 + j * 4, h);
          }
        } else {
          const int64_t at = (int64_t)chunk * a.tokens * a.q_heads + cell;
#pragma unroll
          for (int d = 0; d < DT; ++d) *(f32x4*)(a.part_o + at * D + d * 16 + j * 4) = o[t][d];
          if (j == 0) a.part_ml[at * 2] = top[t], a.part_ml[at * 2 + 1] = sum[t];
        }
      }
    }
  }
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
    float top = -INFINITY, sum = 0.0f, o[PER] = {};
    for (int p = 0; p < pieces; ++p) top = fmaxf(top, a.part_ml[(p * step + cell) * 2]);
    for (int p = 0; p < pieces; ++p) {
      const int64_t at = p * step + cell;
      const float m = a.part_ml[at * 2];
      if (m == -INFINITY) {
        sum += a.part_ml[at * 2 + 1];  // 0, or NaN where every score was
        continue;
      }
      const float w = exp2_fast(m - top);
      sum += w * a.part_ml[at * 2 + 1];
#pragma unroll
      for (int e = 0; e < PER; ++e) o[e] += w * a.part_o[at * D + lane * PER + e];
    }
    const float by = sum == 0.0f ? 0.0f : 1.0f / sum;
    Vec<uint16_t, PER> h;
#pragma unroll
    for (int e = 0; e < PER; ++e) h.v[e] = T::from_f32(sum == 0.0f ? 0.0f : o[e] * by);
    stg(a.out + cell * D + lane * PER, h);
  }
}

// the launch: which kernel, how many tiles of rows and chunks of keys a request gets
struct Launch {
  bool split_keys;
  int row_tiles, tile_rows;
  int64_t tiles, chunks, chunk_keys;
};

Launch plan_launch(int64_t requests, int32_t q_heads, int32_t kv_heads, int32_t head_dim, int64_t max_query,
                   int64_t max_seq) {
  Launch l;
  const int64_t rows = max_query * (q_heads / kv_heads);
  l.split_keys = rows <= 64;
  l.row_tiles = head_dim == 256 || rows <= 16 ? 1 : 2;
  l.tile_rows = (l.split_keys ? 1 : kAttendWaves) * l.row_tiles * 16;
  l.tiles = cdiv(rows, l.tile_rows);
  const int64_t units = requests * kv_heads * l.tiles, wanted = 1024;
  const int64_t floor_keys = l.split_keys ? 512 : 1024, cap = 8192;
  int64_t keys = cdiv(cdiv(max_seq * units, wanted), 256) * 256;
  if (keys < floor_keys) keys = floor_keys;
  if (keys > cap) keys = cap;
  l.chunk_keys = keys;
  l.chunks = cdiv(max_seq, keys);
  if (!l.split_keys && units >= wanted / 2) l.chunks = 1, l.chunk_keys = 1 << 30;
  return l;
}

}  // namespace
}  // namespace ctmi

using namespace ctmi;

extern "C" int64_t ctmi_kv_attend_tmp_bytes(int64_t tokens, int64_t requests, int32_t q_heads,
                                            int32_t kv_heads, int32_t head_dim, int64_t max_query,
                                            int64_t max_seq) {
  if (tokens < 1 || requests < 1 || q_heads < 1 || kv_heads < 1 || max_query < 1 || max_seq < 1) return 0;
  const Launch l = plan_launch(requests, q_heads, kv_heads, head_dim, max_query, max_seq);
  return l.chunks > 1 ? l.chunks * tokens * q_heads * (head_dim + 2) * 4 : 0;
}

extern "C" int ctmi_kv_attend(const void* q, int32_t dtype, int64_t q_token_stride, int64_t q_head_stride,
                              void* out, int64_t tokens, int32_t q_heads, const ctmi_kv_blocks* blocks,
                              const int32_t* block_table, int64_t table_stride, int64_t width,
                              const int32_t* seq_lens, const int32_t* query_start, int64_t requests,
                              float scale, int64_t max_query, int64_t max_seq, void* tmp,
                              int64_t tmp_bytes, void* stream) {
  CTMI_REQUIRE(dtype == CTMI_BF16 || dtype == CTMI_F16, CTMI_ERR_UNSUPPORTED,
               "queries must be bfloat16 or float16");
  const int rc = check_kv_blocks(blocks);
  if (rc != CTMI_OK) return rc;
  CTMI_REQUIRE(q_heads >= 1 && q_heads % blocks->kv_heads == 0, CTMI_ERR_VALUE,
               "%d query heads are no multiple of %d key heads", q_heads, blocks->kv_heads);
  CTMI_REQUIRE(tokens >= 0 && requests >= 0 && width >= 0 && table_stride >= width, CTMI_ERR_VALUE,
               "bad sizes: %lld tokens, %lld requests, %lld table columns, stride %lld", (long long)tokens,
               (long long)requests, (long long)width, (long long)table_stride);
  CTMI_REQUIRE(tokens < (1ll << 31) / q_heads && requests < (1ll << 31) &&
                   width < (1ll << 30) / blocks->block_size,
               CTMI_ERR_UNSUPPORTED, "tokens x heads and requests must stay below 2^31, positions below 2^30");
  CTMI_REQUIRE(query_start != nullptr || tokens == requests, CTMI_ERR_VALUE,
               "without query_start every request has one token: got %lld tokens for %lld requests",
               (long long)tokens, (long long)requests);
  CTMI_REQUIRE(max_query >= 1 && max_seq >= 1, CTMI_ERR_VALUE, "max_query and max_seq must be at least 1");
  if (tokens == 0 || requests == 0) return CTMI_OK;
  CTMI_REQUIRE(q && out && seq_lens && (width == 0 || block_table), CTMI_ERR_VALUE, "NULL tensor");
  CTMI_REQUIRE(q_token_stride % 8 == 0 && q_head_stride % 8 == 0 && ((uintptr_t)q | (uintptr_t)out) % 16 == 0,
               CTMI_ERR_VALUE, "queries must be 16-byte aligned, token by token and head by head");
  const int32_t dim = blocks->head_dim;
  if (max_query > tokens) max_query = tokens;
  if (max_seq > width * blocks->block_size) max_seq = width * blocks->block_size > 0 ? width * blocks->block_size : 1;
  const Launch l = plan_launch(requests, q_heads, blocks->kv_heads, dim, max_query, max_seq);
  const int64_t cells = l.chunks > 1 ? l.chunks * tokens * q_heads : 0;
  CTMI_REQUIRE(tmp_bytes >= cells * (dim + 2) * 4 && (cells == 0 || (tmp != nullptr && (uintptr_t)tmp % 16 == 0)),
               CTMI_ERR_VALUE, "tmp needs %lld bytes at a 16-byte boundary, has %lld", (long long)(cells * (dim + 2) * 4),
               (long long)tmp_bytes);
  const int64_t grid = requests * l.tiles * l.chunks * blocks->kv_heads;
  const int64_t join = cdiv(requests * max_query * q_heads, (int64_t)kAttendWaves);
  CTMI_REQUIRE(grid < (1ll << 31) && (cells == 0 || join < (1ll << 31)), CTMI_ERR_UNSUPPORTED, "too many requests and queries for one launch");
  const uint32_t sixteenths = blocks->block_size / 16;
  AttendArgs a{(const uint16_t*)q, q_token_stride, q_head_stride, (uint16_t*)out,
               (const uint8_t*)blocks->key, (const uint8_t*)blocks->value, blocks->key_scale,
               blocks->value_scale, block_table, seq_lens, query_start, (float*)tmp,
               (float*)tmp + cells * dim, table_stride, (int32_t)blocks->num_blocks, blocks->kv_heads,
               blocks->block_size, q_heads, (int32_t)width, (int32_t)tokens, (int32_t)requests,
               (int32_t)l.tiles, (int32_t)l.chunks, (int32_t)l.chunk_keys, sixteenths,
               sixteenths == 1 ? 0u : (uint32_t)(((1ull << 32) + sixteenths - 1) / sixteenths),
               scale * kLog2e};
  const hipStream_t s = (hipStream_t)stream;
  const dim3 blocks_of((unsigned)grid), threads(kAttendWaves * kWave);
  const bool fp8 = blocks->code_dtype == CTMI_F8E4M3;
  // bf16 outputs of long prompts take the weights as one bf16 number (2^-8, half a step of the
  // output's type); elsewhere they are two, which costs nothing while memory is the bound
#define LAUNCH(T, F, D, RT, KS) kv_attend_kernel<T, F, D, RT, KS, KS || T::id == CTMI_F16><<<blocks_of, threads, 0, s>>>(a)
#define BY_TILE(T, F, D)                                          \
  do {                                                            \
    if (l.split_keys) {                                           \
      if (D == 256 || l.row_tiles == 1) LAUNCH(T, F, D, 1, true); \
      else LAUNCH(T, F, D, (D == 256 ? 1 : 2), true);             \
    } else {                                                      \
      LAUNCH(T, F, D, (D == 256 ? 1 : 2), false);                 \
    }                                                             \
    if (cells) kv_attend_join_kernel<T, D><<<dim3((unsigned)join), threads, 0, s>>>(a, l.tile_rows, (int)max_query); \
  } while (0)
#define BY_CODE(T, D) do { if (fp8) BY_TILE(T, true, D); else BY_TILE(T, false, D); } while (0)
#define BY_DIM(T) do { if (dim == 64) BY_CODE(T, 64); else if (dim == 128) BY_CODE(T, 128); else BY_CODE(T, 256); } while (0)
  if (dtype == CTMI_BF16) BY_DIM(BF16);
  else BY_DIM(F16);
#undef BY_DIM
#undef BY_CODE
#undef BY_TILE
#undef LAUNCH
  return check_launch("kv_attend");
}
