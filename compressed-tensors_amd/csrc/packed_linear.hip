// ctmi_packed_linear: products of a few rows with a 4-bit packed weight.
//
//   y[m, n] = sum_g s[n, g] (sum_{k in g} x[m, k] u[n, k] - z[n, g] X[m, g]) + b[n]
//
// with u the stored codes 0 ... 15, z the zero point as stored (8 for a symmetric weight) and
// X[m, g] the sum of x over a group.  The bound is the weight's read, half a byte per element,
// and next to it the vector instructions that turn codes into operands.  A byte holding 0 ... 15
// is, read as e4m3, that many times 2^-9 (subnormal and first binade are one linear range), so
// v_cvt_scalef32_pk_{bf16,f16}_fp8 with a scale of 2^9 makes two exact operands of two codes:
// 7 instructions for the 8 codes of a word.  The zero point is taken off the sums instead of
// the codes; X is one more product, with ones.  Codes and zero points are whole numbers, sums
// and scales stay in fp32, and nothing is rounded before the output.
//
// Should a sum not be finite (an infinity or NaN in x, or an overflow that the codes less their
// zero points would not have), the wavefront does its share again with those operands: inf * 0
// and inf - inf are then what the formula makes of them.
//
// Layout: 16x16x32 products, x as rows (MT tiles of 16), the weight as columns (NT tiles).  Lane
// (c, j) = (lane % 16, lane / 16) reads 16 bytes - 32 codes - of weight row c per 128 columns,
// and owns the row's scale and zero point, which is also the output column it accumulates.
// The wavefronts of a workgroup, and workgroups along grid z, split k; sums meet in LDS and,
// for a split over workgroups, in a second kernel.
//
// Measured on one MI355X (groups of 128): 1 x 4096 x 4096 5.6 us, of which the bytes are 1.7;
// 16 x 28672 x 4096 20 us, 3.2 TB/s, with the vector units 27 % busy - 5.6 us of ramp are in
// it, whatever the size; 64 x 4096 x 14336 21 us and 4.8 us for the sum of its parts.
#include <type_traits>

#include "ctmi_device.h"
#include "ctmi_host.h"

namespace ctmi {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int kStepK = 128;  // columns per step of a wavefront

struct LinearArgs {
  const uint16_t* x;
  int64_t x_stride;
  const uint32_t* packed;
  const void* scale;
  const uint32_t* zero;
  const uint16_t* bias;
  uint16_t* out;
  float* part;  // [split][m][n], or NULL
  int32_t m, n, k, group, groups, words;
  int32_t wave_k;   // columns a wavefront takes
  int32_t aligned;  // whole 8s of columns, weight rows at 16-byte boundaries
};

struct Operand {
  uint32_t w[4];
};

template <typename T>
__device__ __forceinline__ f32x4 product(const Operand& a, const Operand& b, f32x4 c) {
  if constexpr (T::id == CTMI_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// the codes of a word as operands: nibbles to bytes in their order, two bytes to two numbers
template <typename T>
__device__ __forceinline__ Operand codes_of(uint32_t w) {
  const uint32_t even = w & 0x0F0F0F0Fu, odd = (w >> 4) & 0x0F0F0F0Fu;
  const uint32_t lo = __builtin_amdgcn_perm(odd, even, 0x05010400u), hi = __builtin_amdgcn_perm(odd, even, 0x07030602u);
  Operand o;
  if constexpr (T::id == CTMI_BF16) {
    o.w[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 512.0f, false));
    o.w[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 512.0f, true));
    o.w[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 512.0f, false));
    o.w[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 512.0f, true));
  } else {
    o.w[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 512.0f, false));
    o.w[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 512.0f, true));
    o.w[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 512.0f, false));
    o.w[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 512.0f, true));
  }
  return o;
}

// ... less the zero point (whole numbers up to 15 in magnitude: exact in either type)
template <typename T>
__device__ __forceinline__ Operand signed_codes_of(uint32_t w, float zero) {
  Operand o;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float a = (float)((w >> (8 * e)) & 15) - zero, b = (float)((w >> (8 * e + 4)) & 15) - zero;
    o.w[e] = (uint32_t)T::from_f32(a) | ((uint32_t)T::from_f32(b) << 16);
  }
  return o;
}

// The four lane groups hold words 4 j + t; afterwards w[t] is word 4 t + j: 32 neighbouring
// columns per product.
__device__ __forceinline__ void transpose4(const u32x4& from, uint32_t* w) {
  typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int t = 0; t < 4; t += 2) {
    const u32x2 r = __builtin_amdgcn_permlane16_swap(from[t], from[t + 1], false, false);
    w[t] = r[0], w[t + 1] = r[1];
  }
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const u32x2 r = __builtin_amdgcn_permlane32_swap(w[t], w[t + 2], false, false);
    w[t] = r[0], w[t + 2] = r[1];
  }
}

// Loads through a buffer descriptor: an offset behind its end (kNowhere) reads nothing and
// gives 0, so a wavefront can "load" a step that does not exist without a branch.
constexpr uint32_t kNowhere = 0x80000000u;
struct Buffer {
  __amdgpu_buffer_rsrc_t r;
  // (a descriptor whose numbers the compiler has put into lanes is looked at lane by lane, in a
  // loop around each load)
  static __device__ __forceinline__ void* uniform(const void* p) {
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)p);
    const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)((uintptr_t)p >> 32));
    return (void*)((uintptr_t)hi << 32 | lo);
  }
  __device__ __forceinline__ Buffer(const void* base, uint32_t bytes)
      : r(__builtin_amdgcn_make_buffer_rsrc(uniform(base), 0, __builtin_amdgcn_readfirstlane((int)bytes), 0x00027000)) {}
  __device__ __forceinline__ Vec<uint32_t, 4> load16(uint32_t at) const {
    return __builtin_bit_cast(Vec<uint32_t, 4>, __builtin_amdgcn_raw_buffer_load_b128(r, (int)at, 0, 0));
  }
  __device__ __forceinline__ uint32_t load4(uint32_t at) const { return __builtin_amdgcn_raw_buffer_load_b32(r, (int)at, 0, 0); }
  __device__ __forceinline__ uint16_t load2(uint32_t at) const { return __builtin_amdgcn_raw_buffer_load_b16(r, (int)at, 0, 0); }
};

// SMALL: groups that are no multiple of 128 columns, so a scale holds for one product of 32
// columns only.  WIDE: scales are fp32, else of x's type.  XL: loads of 4 rows of x each, as
// many as there are rows (one for a decoding request or four).
//
// A wavefront keeps two steps requested: a slot is loaded again as soon as its step is
// multiplied.  The slots are registers by name, the loads stand in no branch (behind the last
// step they read nothing): a load that may not have been issued, or a copy of a register that
// is still to arrive, would make the wait for one step a wait for all.  The loop holds the two
// steps and nothing is unrolled beyond them: a wavefront runs few steps, and code it has to
// fetch for each of them costs more than the steps do.
//
// What a compute unit's loads cost is the places they touch: lanes next to each other in one
// line are looked up together, others one by one.  So x comes in rows of 256 bytes, 16 lanes
// each, and reaches the operands' layout through the wavefront's own 4 KB of LDS per 16 rows
// (pieces of a row swapped by the row's number: no bank is hit twice); and one load brings the
// scales of all NT x 16 weight rows, one lane each, from where the lanes that use them take
// them.  With operands loaded where they are used, 16 x 28672 x 4096 took 26 us, 7 of them for
// x and 4 for scales.
template <typename T, int MT, int NT, int XL, bool SMALL, bool WIDE>
struct LinearWave {
  static constexpr int PARTS = SMALL ? 4 : 1;  // groups in a step
  struct Step {
    u32x4 w[NT];  // (one value: a number of it carried from step to step by itself is copied there)
    // scale of weight row `lane` (as it is stored: widened where it is asked for, it would be used
    // there), zero points of rows 8 (lane % 8) on
    std::conditional_t<WIDE, uint32_t, uint16_t> s[PARTS];
    uint32_t z[PARTS];
    Vec<uint32_t, 4> x[XL];       // rows 4 i + lane / 16, columns (lane % 16) * 8 on
  };

  const LinearArgs& a;
  int lane, c, j;
  // where there are no zero points the buffer is empty, reads 0, and every zero point is 8
  uint32_t z_none;
  Buffer w_buf, s_buf, z_buf, x_buf;  // of the workgroup's rows; rows behind the last read as 0
  uint32_t w_at, s_at, z_at, x_at, w_tile, x_four;
  Vec<uint32_t, 4>* mine;  // of LDS
  f32x4 y[NT][MT];

  __device__ __forceinline__ LinearWave(const LinearArgs& args, int n0, int m0, Vec<uint32_t, 4>* lds)
      : a(args),
        w_buf(a.packed + (int64_t)n0 * a.words, (uint32_t)min(NT * 16, a.n - n0) * (uint32_t)a.words * 4u),
        s_buf((const uint8_t*)a.scale + (int64_t)n0 * a.groups * (WIDE ? 4 : 2),
              (uint32_t)min(NT * 16, a.n - n0) * (uint32_t)a.groups * (WIDE ? 4 : 2)),
        z_buf(a.zero + (int64_t)(n0 >> 3) * a.groups, a.zero ? (uint32_t)((min(NT * 16, a.n - n0) + 7) >> 3) * (uint32_t)a.groups * 4u : 0u),
        x_buf(a.x + m0 * a.x_stride, ((uint32_t)(min(MT * 16, a.m - m0) - 1) * (uint32_t)a.x_stride + (uint32_t)a.k) * 2u),
        mine(lds) {
    lane = lane_id(), c = lane & 15, j = lane >> 4;
    z_none = a.zero ? 0u : 8u;
    w_at = (uint32_t)c * (uint32_t)a.words * 4u + j * 16;
    w_tile = (uint32_t)a.words * 64u;
    s_at = (uint32_t)(lane % (NT * 16)) * (uint32_t)a.groups * (WIDE ? 4 : 2);  // n0 is a multiple of 16
    z_at = (uint32_t)(lane & 7) * (uint32_t)a.groups * 4u;
    x_at = (uint32_t)j * (uint32_t)a.x_stride * 2u + c * 16;
    x_four = (uint32_t)a.x_stride * 8u;
#pragma unroll
    for (int i = XL; i < MT * 4; ++i) mine[i * 64 + lane] = Vec<uint32_t, 4>{};
    clear();
  }

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) y[t][mt] = f32x4{0, 0, 0, 0};
  }

  // the group of the next columns, and how many of it are left, as steps are loaded one after
  // the other
  struct Groups {
    int g, left;
  };
  __device__ __forceinline__ Groups groups_at(int kb) const {
    const int g = kb / a.group;
    return Groups{g, (g + 1) * a.group - kb};
  }
  __device__ __forceinline__ void load_scales(Step& st, Groups& at, bool there) const {
#pragma unroll
    for (int i = 0; i < PARTS; ++i) {
      const uint32_t g = min(at.g, a.groups - 1);
      if constexpr (WIDE) st.s[i] = s_buf.load4(there ? s_at + g * 4u : kNowhere);
      else st.s[i] = s_buf.load2(there ? s_at + g * 2u : kNowhere);
      st.z[i] = z_buf.load4(there ? z_at + g * 4u : kNowhere);
      at.left -= SMALL ? 32 : kStepK;
      const int over = (int)((uint32_t)(at.left - 1) >> 31);  // no branch here either
      at.left += -over & a.group, at.g += over;
    }
  }

  __device__ __forceinline__ void load(Step& st, int kb, bool there, Groups& at) const {
    // (behind the row's end x is 0 and the codes are the next row's: they do not count)
    const uint32_t wk = there ? w_at + (uint32_t)kb / 2u : kNowhere, xk = (int)there & (int)(kb + c * 8 < a.k) ? x_at + (uint32_t)kb * 2u : kNowhere;
#pragma unroll
    for (int t = 0; t < NT; ++t) st.w[t] = __builtin_bit_cast(u32x4, w_buf.load16(wk + t * w_tile));
    load_scales(st, at, there);
#pragma unroll
    for (int i = 0; i < XL; ++i) st.x[i] = x_buf.load16(xk + i * x_four);
  }

  // a step of rows that need not start at 16-byte boundaries, element by element
  __device__ __forceinline__ void load_guarded(Step& st, int kb) const {
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        st.w[t][i] = w_buf.load4(kb / 8 + j * 4 + i < a.words ? w_at + kb / 2 + t * w_tile + i * 4 : kNowhere);
    Groups at = groups_at(kb);
    load_scales(st, at, true);
#pragma unroll
    for (int i = 0; i < XL; ++i) {
      const int first = kb + c * 8;
      const uint32_t at = x_at + kb * 2 + i * x_four;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        st.x[i].v[e] = x_buf.load2(first + 2 * e < a.k ? at + 4 * e : kNowhere) |
                       (uint32_t)x_buf.load2(first + 2 * e + 1 < a.k ? at + 4 * e + 2 : kNowhere) << 16;
    }
  }

  template <bool SIGNED>
  __device__ __forceinline__ void step(Step& st) {
    const Operand ones = T::id == CTMI_BF16 ? Operand{{0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u}}
                                            : Operand{{0x3C003C00u, 0x3C003C00u, 0x3C003C00u, 0x3C003C00u}};
#pragma unroll
    for (int i = 0; i < XL; ++i) mine[(i * 4 + j) * 16 + (c ^ ((i * 4 + j) & 15))] = st.x[i];
    Operand x[MT][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int t = 0; t < 4; ++t) x[mt][t] = __builtin_bit_cast(Operand, mine[(mt * 16 + c) * 16 + ((t * 4 + j) ^ c)]);
    auto add = [&](f32x4 sum, const Operand& v) { return product<T>(v, ones, sum); };
    auto scale_zero = [&](int nt, int part, float& s, float& z) {
      const uint32_t raw = __shfl((uint32_t)st.s[part], nt * 16 + c, kWave), zeros = __shfl(st.z[part], nt * 2 + (c >> 3), kWave);
      s = WIDE ? u2f(raw) : T::to_f32((uint16_t)raw);
      z = (float)(((zeros >> (4 * (c & 7))) & 15u) | z_none);
    };
    auto take = [&](int nt, int mt, float s, float z, const f32x4& acc, const f32x4& sum) {
#pragma unroll
      for (int i = 0; i < 4; ++i) y[nt][mt][i] = fmaf(s, SIGNED ? acc[i] : fmaf(-z, sum[i], acc[i]), y[nt][mt][i]);
    };
    uint32_t codes[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) transpose4(st.w[nt], codes[nt]);
    f32x4 sums[MT];
    if constexpr (SMALL) {
#pragma unroll
      for (int t = 0; t < 4; ++t) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) sums[mt] = add(f32x4{0, 0, 0, 0}, x[mt][t]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float s, z;
          scale_zero(nt, t, s, z);
          const Operand w = SIGNED ? signed_codes_of<T>(codes[nt][t], z) : codes_of<T>(codes[nt][t]);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) take(nt, mt, s, z, product<T>(x[mt][t], w, f32x4{0, 0, 0, 0}), sums[mt]);
        }
        // (the scales of all parts and tiles together would not leave registers for the rest)
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        sums[mt] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int t = 0; t < 4; ++t) sums[mt] = add(sums[mt], x[mt][t]);
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float s, z;
        scale_zero(nt, 0, s, z);
        f32x4 acc[MT];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) acc[mt] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const Operand w = SIGNED ? signed_codes_of<T>(codes[nt][t], z) : codes_of<T>(codes[nt][t]);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) acc[mt] = product<T>(x[mt][t], w, acc[mt]);
        }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) take(nt, mt, s, z, acc[mt], sums[mt]);
      }
    }
  }

  // columns k0 ... k1 - 1; returns where it stopped: nothing is done, and all left to
  // run_signed, if the rows of the weight do not start at 16-byte boundaries
  __device__ __forceinline__ int run(int k0, int k1) {
    const int end = a.aligned ? k1 : k0;
    if (k0 < end) {
      Step one, two;
      Groups at = groups_at(k0);
      load(one, k0, true, at);
      load(two, k0 + kStepK, k0 + kStepK < end, at);
#pragma unroll 1
      for (int kb = k0; kb < end; kb += 2 * kStepK) {
        step<false>(one);
        load(one, kb + 2 * kStepK, kb + 2 * kStepK < end, at);
        __builtin_amdgcn_sched_barrier(0);
        step<false>(two);
        load(two, kb + 3 * kStepK, kb + 3 * kStepK < end, at);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    return end;
  }

  __device__ __forceinline__ void run_signed(int k0, int k1) {
#pragma unroll 1
    for (int kb = k0; kb < k1; kb += kStepK) {
      Step st;
      load_guarded(st, kb);
      step<true>(st);
    }
  }
};

template <typename T, int MT, int NT, int XL, bool SMALL, bool WIDE, int WAVES, int PER_SIMD>
__global__ __launch_bounds__(WAVES* kWave, PER_SIMD) void packed_linear_kernel(LinearArgs a) {
  constexpr int TM = MT * 16, TN = NT * 16;
  // each wavefront's x, TM rows of 256 bytes; at the end [wave][TM][TN] sums
  extern __shared__ Vec<uint32_t, 4> lds[];
  float* meet = (float*)lds;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), waves = blockDim.x / kWave;
  const int n0 = blockIdx.x * TN;
  LinearWave<T, MT, NT, XL, SMALL, WIDE> w(a, n0, blockIdx.y * TM, lds + wave * TM * 16);
  const int64_t begin = ((int64_t)blockIdx.z * waves + wave) * a.wave_k;
  const int k0 = (int)(begin < a.k ? begin : a.k), k1 = (int)(begin + a.wave_k < a.k ? begin + a.wave_k : a.k);
  int redo = w.run((int)k0, k1);
  bool bad = false;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int i = 0; i < 4; ++i) bad |= !(fabsf(w.y[nt][mt][i]) <= 3.4028235e38f);
  if (__any(bad)) w.clear(), redo = (int)k0;
  w.run_signed(redo, k1);
  __syncthreads();  // sums take the place of x
  const int m0 = blockIdx.y * TM, rows = min(TM, a.m - m0);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = mt * 16 + w.j * 4 + i;
        if (r < rows) meet[(wave * TM + r) * TN + nt * 16 + w.c] = w.y[nt][mt][i];
      }
  __syncthreads();
  for (int at = threadIdx.x; at < rows * TN; at += blockDim.x) {
    const int r = at / TN, n = n0 + at % TN;
    float v = 0.0f;
    for (int i = 0; i < waves; ++i) v += meet[i * TM * TN + at];
    if (n < a.n) {
      const int64_t cell = (int64_t)(m0 + r) * a.n + n;
      if (a.part) a.part[(int64_t)blockIdx.z * a.m * a.n + cell] = v;
      else a.out[cell] = T::from_f32(v + (a.bias ? T::to_f32(a.bias[n]) : 0.0f));
    }
  }
}

// More than 16 rows: 8 wavefronts, 4 beside each other along n (NT tiles each) and 2 along k.
// A compute unit then needs each element of x once: the 4 load a step of it together, two steps
// ahead, into LDS.  (Each wavefront with x of its own, which is 4 times as much from the second
// level cache, took 34 us for 64 x 4096 x 14336.)
template <typename T, int MT, int NT, bool SMALL, bool WIDE>
struct LinearShared {
  static constexpr int PARTS = SMALL ? 4 : 1, ACROSS = 4, ALONG = 2;
  struct Step {
    u32x4 w[NT];
    std::conditional_t<WIDE, uint32_t, uint16_t> s[PARTS];
    uint32_t z[PARTS];
  };
  const LinearArgs& a;
  int lane, c, j;
  uint32_t z_none;
  Buffer w_buf, s_buf, z_buf, x_buf;
  uint32_t w_at, s_at, z_at, x_at, w_tile, x_four;
  int across;
  f32x4 y[NT][MT];

  // n0: the wavefront's first column; one behind the last has empty buffers
  __device__ __forceinline__ LinearShared(const LinearArgs& args, int n0, int m0, int wn)
      : a(args),
        w_buf(a.packed + (int64_t)min(n0, a.n - 1) * a.words, (uint32_t)max(min(NT * 16, a.n - n0), 0) * (uint32_t)a.words * 4u),
        s_buf((const uint8_t*)a.scale + (int64_t)min(n0, a.n - 1) * a.groups * (WIDE ? 4 : 2),
              (uint32_t)max(min(NT * 16, a.n - n0), 0) * (uint32_t)a.groups * (WIDE ? 4 : 2)),
        z_buf(a.zero + (int64_t)(min(n0, a.n - 1) >> 3) * a.groups,
              a.zero ? (uint32_t)((max(min(NT * 16, a.n - n0), 0) + 7) >> 3) * (uint32_t)a.groups * 4u : 0u),
        x_buf(a.x + m0 * a.x_stride, ((uint32_t)(min(MT * 16, a.m - m0) - 1) * (uint32_t)a.x_stride + (uint32_t)a.k) * 2u),
        across(wn) {
    lane = lane_id(), c = lane & 15, j = lane >> 4;
    z_none = a.zero ? 0u : 8u;
    w_at = (uint32_t)c * (uint32_t)a.words * 4u + j * 16;
    w_tile = (uint32_t)a.words * 64u;
    s_at = (uint32_t)(lane % (NT * 16)) * (uint32_t)a.groups * (WIDE ? 4 : 2);
    z_at = (uint32_t)(lane & 7) * (uint32_t)a.groups * 4u;
    x_at = (uint32_t)(across * MT * 4 + j) * (uint32_t)a.x_stride * 2u + c * 16;
    x_four = (uint32_t)a.x_stride * 8u;
    clear();
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) y[t][mt] = f32x4{0, 0, 0, 0};
  }
  struct Groups {
    int g, left;
  };
  __device__ __forceinline__ Groups groups_at(int kb) const {
    const int g = kb / a.group;
    return Groups{g, (g + 1) * a.group - kb};
  }
  __device__ __forceinline__ void load(Step& st, int kb, bool there, Groups& at) const {
    const uint32_t wk = there ? w_at + (uint32_t)kb / 2u : kNowhere;
#pragma unroll
    for (int t = 0; t < NT; ++t) st.w[t] = __builtin_bit_cast(u32x4, w_buf.load16(wk + t * w_tile));
#pragma unroll
    for (int i = 0; i < PARTS; ++i) {
      const uint32_t g = min(at.g, a.groups - 1);
      if constexpr (WIDE) st.s[i] = s_buf.load4(there ? s_at + g * 4u : kNowhere);
      else st.s[i] = s_buf.load2(there ? s_at + g * 2u : kNowhere);
      st.z[i] = z_buf.load4(there ? z_at + g * 4u : kNowhere);
      at.left -= SMALL ? 32 : kStepK;
      const int over = (int)((uint32_t)(at.left - 1) >> 31);
      at.left += -over & a.group, at.g += over;
    }
  }
  __device__ __forceinline__ void load_rows(Vec<uint32_t, 4>* x, int kb, bool there) const {
    const uint32_t xk = (int)there & (int)(kb + c * 8 < a.k) ? x_at + (uint32_t)kb * 2u : kNowhere;
#pragma unroll
    for (int i = 0; i < MT; ++i) x[i] = x_buf.load16(xk + i * x_four);
  }
  __device__ __forceinline__ void store_rows(const Vec<uint32_t, 4>* x, Vec<uint32_t, 4>* lds) const {
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const int r = across * MT * 4 + i * 4 + j;
      lds[r * 16 + (c ^ (r & 15))] = x[i];
    }
  }

  // x(mt, t): the operand of rows 16 mt ..., columns 32 t ... of the step
  template <bool SIGNED, typename X>
  __device__ __forceinline__ void step(Step& st, X x) {
    const Operand ones = T::id == CTMI_BF16 ? Operand{{0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u}}
                                            : Operand{{0x3C003C00u, 0x3C003C00u, 0x3C003C00u, 0x3C003C00u}};
    uint32_t codes[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) transpose4(st.w[nt], codes[nt]);
    f32x4 acc[NT][MT], sums[MT];
    float s[NT], z[NT];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      if (SMALL || t == 0) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) sums[mt] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const uint32_t raw = __shfl((uint32_t)st.s[t], nt * 16 + c, kWave), zeros = __shfl(st.z[t], nt * 2 + (c >> 3), kWave);
          s[nt] = WIDE ? u2f(raw) : T::to_f32((uint16_t)raw);
          z[nt] = (float)(((zeros >> (4 * (c & 7))) & 15u) | z_none);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) acc[nt][mt] = f32x4{0, 0, 0, 0};
        }
      }
      Operand w[NT];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) w[nt] = SIGNED ? signed_codes_of<T>(codes[nt][t], z[nt]) : codes_of<T>(codes[nt][t]);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const Operand v = x(mt, t);
        if constexpr (!SIGNED) sums[mt] = product<T>(v, ones, sums[mt]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) acc[nt][mt] = product<T>(v, w[nt], acc[nt][mt]);
      }
      if (SMALL || t == 3) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              y[nt][mt][i] = fmaf(s[nt], SIGNED ? acc[nt][mt][i] : fmaf(-z[nt], sums[mt][i], acc[nt][mt][i]), y[nt][mt][i]);
      }
    }
  }

  // columns k0 ... k0 + wave_k - 1, as far as there are any; the 4 wavefronts that share x, and
  // with them the workgroup, go through the same steps
  __device__ __forceinline__ void run(int k0, int k1, Vec<uint32_t, 4>* lds) {
    constexpr int TILE = MT * 16 * 16;
    Step one, two;
    Vec<uint32_t, 4> rows[MT];
    Groups at = groups_at(min(k0, a.k - 1));
    load_rows(rows, k0, k0 < k1);
    load(one, k0, k0 < k1, at);
    __builtin_amdgcn_sched_barrier(0);
    store_rows(rows, lds);
    load_rows(rows, k0 + kStepK, k0 + kStepK < k1);
    load(two, k0 + kStepK, k0 + kStepK < k1, at);
    __builtin_amdgcn_sched_barrier(0);
    __syncthreads();
    auto from = [&](const Vec<uint32_t, 4>* tile) {
      return [tile, this](int mt, int t) { return __builtin_bit_cast(Operand, tile[(mt * 16 + c) * 16 + ((t * 4 + j) ^ c)]); };
    };
#pragma unroll 1
    for (int kb = k0; kb < k0 + a.wave_k; kb += 2 * kStepK) {
      step<false>(one, from(lds));
      __builtin_amdgcn_sched_barrier(0);
      store_rows(rows, lds + TILE);
      load_rows(rows, kb + 2 * kStepK, kb + 2 * kStepK < k1);
      load(one, kb + 2 * kStepK, kb + 2 * kStepK < k1, at);
      __builtin_amdgcn_sched_barrier(0);
      __syncthreads();
      step<false>(two, from(lds + TILE));
      __builtin_amdgcn_sched_barrier(0);
      store_rows(rows, lds);
      load_rows(rows, kb + 3 * kStepK, kb + 3 * kStepK < k1);
      load(two, kb + 3 * kStepK, kb + 3 * kStepK < k1, at);
      __builtin_amdgcn_sched_barrier(0);
      __syncthreads();
    }
  }

  // the same by one wavefront alone, x from where it lies
  __device__ __forceinline__ void run_signed(int k0, int k1) {
    clear();
#pragma unroll 1
    for (int kb = k0; kb < k1; kb += kStepK) {
      Step st;
      Groups at = groups_at(kb);
      load(st, kb, true, at);
      step<true>(st, [&](int mt, int t) {
        const int k = kb + t * 32 + j * 8;
        return __builtin_bit_cast(Operand, x_buf.load16(k < a.k ? (uint32_t)(mt * 16 + c) * (uint32_t)a.x_stride * 2u + k * 2u : kNowhere));
      });
    }
  }
};

template <typename T, int MT, int NT, bool SMALL, bool WIDE>
__global__ __launch_bounds__(8 * kWave, 2) void packed_linear_shared_kernel(LinearArgs a) {
  using Wave = LinearShared<T, MT, NT, SMALL, WIDE>;
  constexpr int TM = MT * 16, TN = Wave::ACROSS * NT * 16;
  extern __shared__ Vec<uint32_t, 4> lds[];  // x: two steps for each half of k; then sums [TM][TN]
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), across = wave % Wave::ACROSS, along = wave / Wave::ACROSS;
  const int n0 = blockIdx.x * TN, m0 = blockIdx.y * TM;
  Wave w(a, n0 + across * NT * 16, m0, across);
  const int64_t begin = ((int64_t)blockIdx.z * Wave::ALONG + along) * a.wave_k;
  const int k0 = (int)(begin < a.k ? begin : a.k), k1 = (int)(begin + a.wave_k < a.k ? begin + a.wave_k : a.k);
  w.run(k0, k1, lds + along * 2 * MT * 16 * 16);
  bool bad = false;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int i = 0; i < 4; ++i) bad |= !(fabsf(w.y[nt][mt][i]) <= 3.4028235e38f);
  if (__any(bad)) w.run_signed(k0, k1);
  float* meet = (float*)lds;
  const int rows = min(TM, a.m - m0);
#pragma unroll
  for (int half = 1; half >= 0; --half) {
    if (along == half) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float* at = &meet[(mt * 16 + w.j * 4 + i) * TN + across * NT * 16 + nt * 16 + w.c];
            *at = half == 1 ? w.y[nt][mt][i] : *at + w.y[nt][mt][i];
          }
    }
    __syncthreads();
  }
  for (int at = threadIdx.x; at < rows * TN; at += 8 * kWave) {
    const int r = at / TN, n = n0 + at % TN;
    if (n < a.n) {
      const int64_t cell = (int64_t)(m0 + r) * a.n + n;
      if (a.part) a.part[(int64_t)blockIdx.z * a.m * a.n + cell] = meet[at];
      else a.out[cell] = T::from_f32(meet[at] + (a.bias ? T::to_f32(a.bias[n]) : 0.0f));
    }
  }
}

template <typename T>
__global__ __launch_bounds__(256) void packed_linear_join_kernel(LinearArgs a, int splits) {
  const int64_t cells = (int64_t)a.m * a.n;
  for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < cells; at += (int64_t)gridDim.x * 256) {
    float v = 0.0f;
    for (int i = 0; i < splits; ++i) v += a.part[i * cells + at];
    a.out[at] = T::from_f32(v + (a.bias ? T::to_f32(a.bias[at % a.n]) : 0.0f));
  }
}

struct LinearLaunch {
  int mt, nt, waves;
  int64_t splits, wave_k;
};

// More than 16 rows go to the shared kernel where rows of weight and x are whole 16-byte pieces;
// otherwise they are taken 16 at a time.
LinearLaunch plan_linear(int64_t m, int64_t n, int64_t k) {
  LinearLaunch l;
  const int64_t tiles = cdiv(n, 16);
  l.splits = 1;
  if (m <= 16 || k % 32 != 0) {
    l.mt = 1;
    // Wide enough to fill the device, a wavefront takes more tiles: x and its sums serve more columns.
    // Of k 4096, one row (16 rows), 1, 2 and 4 tiles: 4096 columns 6.2, 7.2, 11.0 us (7.2, 8.4, 12.3);
    // 8192 9.1, 7.8, 11.2 (11.0, 8.8, 12.7); 16384 14.8, 11.6, 11.8 (18.0, 13.6, 13.8); 28672 23.8, 19.0,
    // 16.2 (28.1, 22.5, 20.0).
    l.nt = tiles >= 1024 ? 4 : tiles >= 512 ? 2 : 1;
    l.waves = l.nt == 4 ? 4 : 8;
    l.wave_k = cdiv(cdiv(k, l.waves), kStepK) * kStepK;
  } else {
    l.mt = m <= 32 ? 2 : 4;
    l.nt = 2;
    l.waves = 8;
    // one workgroup per compute unit; a split's sums leave and come back in fp32, so no more
    // of them than it takes, of 256 columns at least.  Not above 16: 64 x 1024 x 14336 takes 23.2,
    // 19.9 and 22.2 us with up to 8, 16 and 32, 32 x 1024 x 14336 17.7, 16.0 and 17.8 (of 28672
    // columns 34.1, 26.1 and 24.8).
    const int64_t units = cdiv(tiles, 8) * cdiv(m, l.mt * 16);
    if (units < 256) l.splits = 256 / units;
    if (l.splits > k / 512) l.splits = k / 512 > 0 ? k / 512 : 1;
    if (l.splits > 16) l.splits = 16;
    l.wave_k = cdiv(cdiv(k, 2 * l.splits), 2 * kStepK) * 2 * kStepK;
    l.splits = cdiv(k, 2 * l.wave_k);
  }
  return l;
}

}  // namespace
}  // namespace ctmi

using namespace ctmi;

extern "C" int64_t ctmi_packed_linear_tmp_bytes(int64_t m, int64_t n, int64_t k, int64_t group) {
  if (m < 1 || n < 1 || k < 1) return 0;
  const LinearLaunch l = plan_linear(m, n, k);
  return l.splits > 1 ? l.splits * m * n * 4 : 0;
}

extern "C" int ctmi_packed_linear(const void* x, int32_t x_dtype, int64_t x_stride, const int32_t* packed,
                                  const void* scale, int32_t scale_dtype, const int32_t* zero_point,
                                  const void* bias, void* out, int64_t m, int64_t n, int64_t k,
                                  int64_t group, void* tmp, int64_t tmp_bytes, void* stream) {
  CTMI_REQUIRE(x_dtype == CTMI_BF16 || x_dtype == CTMI_F16, CTMI_ERR_UNSUPPORTED,
               "activations must be bfloat16 or float16");
  CTMI_REQUIRE(scale_dtype == CTMI_F32 || scale_dtype == x_dtype, CTMI_ERR_UNSUPPORTED,
               "scales must be float32 or of x's type, got dtype %d", scale_dtype);
  CTMI_REQUIRE(m >= 0 && n >= 0 && k >= 1, CTMI_ERR_VALUE, "bad sizes [%lld, %lld] x [%lld, %lld]",
               (long long)m, (long long)k, (long long)n, (long long)k);
  CTMI_REQUIRE(m < (1ll << 31) && n < (1ll << 31) && k <= (1ll << 24), CTMI_ERR_UNSUPPORTED,
               "sizes must stay below 2^31 (columns: 2^24)");
  CTMI_REQUIRE(group == k || (group >= 32 && group % 32 == 0 && k % group == 0), CTMI_ERR_UNSUPPORTED,
               "groups of %lld do not fit %lld columns: a multiple of 32 that divides them, or one group",
               (long long)group, (long long)k);
  CTMI_REQUIRE(x_stride >= k || m <= 1, CTMI_ERR_VALUE, "x_stride %lld is less than %lld columns",
               (long long)x_stride, (long long)k);
  if (m == 0 || n == 0) return CTMI_OK;
  CTMI_REQUIRE(x && packed && scale && out, CTMI_ERR_VALUE, "NULL tensor");
  CTMI_REQUIRE(((uintptr_t)x % 16 == 0) && (x_stride % 8 == 0 || m == 1), CTMI_ERR_VALUE,
               "rows of x must start at 16-byte boundaries");
  CTMI_REQUIRE(x_stride < (1ll << 24) || m == 1, CTMI_ERR_UNSUPPORTED, "rows of x more than 2^24 elements apart");
  const LinearLaunch l = plan_linear(m, n, k);
  const int64_t need = l.splits > 1 ? l.splits * m * n * 4 : 0;
  CTMI_REQUIRE(tmp_bytes >= need && (need == 0 || (tmp != nullptr && (uintptr_t)tmp % 16 == 0)), CTMI_ERR_VALUE,
               "tmp needs %lld bytes at a 16-byte boundary, has %lld", (long long)need, (long long)tmp_bytes);
  const int64_t tm = l.mt * 16, tn = l.nt * 16 * (l.mt == 1 ? 1 : 4);
  CTMI_REQUIRE(cdiv(m, tm) < (1 << 16), CTMI_ERR_UNSUPPORTED, "too many rows: %lld", (long long)m);
  const bool aligned = k % 32 == 0 && (uintptr_t)packed % 16 == 0;
  CTMI_REQUIRE(aligned || l.mt == 1, CTMI_ERR_VALUE, "weight_packed must be 16-byte aligned for more than 16 rows");
  LinearArgs a{(const uint16_t*)x, x_stride, (const uint32_t*)packed, scale, (const uint32_t*)zero_point,
               (const uint16_t*)bias, (uint16_t*)out, need ? (float*)tmp : nullptr, (int32_t)m, (int32_t)n,
               (int32_t)k, (int32_t)group, (int32_t)(k / group), (int32_t)cdiv(k, 8), (int32_t)l.wave_k, aligned};
  const dim3 grid((unsigned)cdiv(n, tn), (unsigned)cdiv(m, tm), (unsigned)l.splits), threads(l.waves * kWave);
  const size_t lds = l.mt == 1 ? (size_t)l.waves * 16 * (tn * 4 > 256 ? tn * 4 : 256) : (size_t)l.mt * 16 * 256 * 4;
  const hipStream_t s = (hipStream_t)stream;
  const bool small = group % kStepK != 0 && group != k;
#define BY_SCALE(KERNEL, ...)                                                       \
  do {                                                                              \
    if (scale_dtype == CTMI_F32) KERNEL(__VA_ARGS__, true);                         \
    else KERNEL(__VA_ARGS__, false);                                                \
  } while (0)
#define BY_GROUP(KERNEL, ...)                                                       \
  do {                                                                              \
    if (small) BY_SCALE(KERNEL, __VA_ARGS__, true);                                 \
    else BY_SCALE(KERNEL, __VA_ARGS__, false);                                      \
  } while (0)
#define FEW(T, NT, XL, W, P, SMALL, WIDE) packed_linear_kernel<T, 1, NT, XL, SMALL, WIDE, W, P><<<grid, threads, lds, s>>>(a)
#define MANY(T, MT, SMALL, WIDE) packed_linear_shared_kernel<T, MT, 2, SMALL, WIDE><<<grid, threads, lds, s>>>(a)
#define BY_SIZE(T)                                  \
  do {                                              \
    if (l.mt == 4) BY_GROUP(MANY, T, 4);            \
    else if (l.mt == 2) BY_GROUP(MANY, T, 2);       \
    else if (m > 4) {                               \
      if (l.nt == 4) BY_GROUP(FEW, T, 4, 4, 4, 3);  \
      else if (l.nt == 2) BY_GROUP(FEW, T, 2, 4, 8, 4); \
      else BY_GROUP(FEW, T, 1, 4, 8, 4);            \
    } else {                                        \
      if (l.nt == 4) BY_GROUP(FEW, T, 4, 1, 4, 3);  \
      else if (l.nt == 2) BY_GROUP(FEW, T, 2, 1, 8, 4); \
      else BY_GROUP(FEW, T, 1, 1, 8, 4);            \
    }                                               \
    if (need) packed_linear_join_kernel<T><<<dim3((unsigned)(cdiv(m * n, 256) < 2048 ? cdiv(m * n, 256) : 2048)), dim3(256), 0, s>>>(a, (int)l.splits); \
  } while (0)
  if (x_dtype == CTMI_BF16) BY_SIZE(BF16);
  else BY_SIZE(F16);
#undef BY_SIZE
#undef MANY
#undef FEW
#undef BY_GROUP
#undef BY_SCALE
  return check_launch("packed_linear");
}
