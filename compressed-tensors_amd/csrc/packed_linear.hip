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
#include "ctmi_device.h"
#include "ctmi_host.h"

namespace ctmi {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
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
  int32_t scale_dtype, wave_k;  // columns a wavefront takes
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

// the codes of a word as operands, in the order 0 2 4 6 1 3 5 7
template <typename T>
__device__ __forceinline__ Operand codes_of(uint32_t w) {
  const uint32_t even = w & 0x0F0F0F0Fu, odd = (w >> 4) & 0x0F0F0F0Fu;
  Operand o;
  if constexpr (T::id == CTMI_BF16) {
    o.w[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(even, 512.0f, false));
    o.w[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(even, 512.0f, true));
    o.w[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(odd, 512.0f, false));
    o.w[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(odd, 512.0f, true));
  } else {
    o.w[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(even, 512.0f, false));
    o.w[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(even, 512.0f, true));
    o.w[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(odd, 512.0f, false));
    o.w[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(odd, 512.0f, true));
  }
  return o;
}

// ... less the zero point (whole numbers up to 15 in magnitude: exact in either type)
template <typename T>
__device__ __forceinline__ Operand signed_codes_of(uint32_t w, float zero) {
  Operand o;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int at = (e % 2) * 16 + (e / 2) * 4;  // 0 2, 4 6, 1 3, 5 7
    const float a = (float)((w >> at) & 15) - zero, b = (float)((w >> (at + 8)) & 15) - zero;
    o.w[e] = (uint32_t)T::from_f32(a) | ((uint32_t)T::from_f32(b) << 16);
  }
  return o;
}

// 8 neighbouring elements of x in that order
__device__ __forceinline__ Operand reorder(const Vec<uint32_t, 4>& x) {
  return Operand{{__builtin_amdgcn_perm(x.v[1], x.v[0], 0x05040100u), __builtin_amdgcn_perm(x.v[3], x.v[2], 0x05040100u),
                  __builtin_amdgcn_perm(x.v[1], x.v[0], 0x07060302u), __builtin_amdgcn_perm(x.v[3], x.v[2], 0x07060302u)}};
}

// The four lane groups hold words 4 j + t; afterwards w[t] is word 4 t + j: 32 neighbouring
// columns per product.
__device__ __forceinline__ void transpose4(uint32_t* w) {
  typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int t = 0; t < 4; t += 2) {
    const u32x2 r = __builtin_amdgcn_permlane16_swap(w[t], w[t + 1], false, false);
    w[t] = r[0], w[t + 1] = r[1];
  }
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const u32x2 r = __builtin_amdgcn_permlane32_swap(w[t], w[t + 2], false, false);
    w[t] = r[0], w[t + 2] = r[1];
  }
}

// SMALL: groups that are no multiple of 128 columns, so a scale holds for one product of 32
// columns only.  PF steps are requested before the ones in hand are multiplied.
template <typename T, int MT, int NT, bool SMALL>
struct LinearWave {
  static constexpr int PF = SMALL ? (NT == 1 ? 2 : 1) : (NT == 1 ? 4 : NT == 2 ? 2 : 1);
  static constexpr int SC = SMALL ? 4 : 1;  // scales per step

  const LinearArgs& a;
  int lane, c, j, m0;
  int row[NT];  // weight row of each tile, within the weight
  f32x4 y[NT][MT];

  struct Step {
    uint32_t w[NT][4];
    float s[NT][SC], z[NT][SC];
  };

  __device__ __forceinline__ void load(Step& st, int kb) {
    const bool whole = kb + kStepK <= a.k && a.words % 4 == 0;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const uint32_t* p = a.packed + (int64_t)row[t] * a.words;
      const int w0 = kb / 8 + j * 4;
      if (whole && ((uintptr_t)a.packed & 15) == 0) {
        const Vec<uint32_t, 4> v = ldg_nt<uint32_t, 4>(p + w0);
#pragma unroll
        for (int i = 0; i < 4; ++i) st.w[t][i] = v.v[i];
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) st.w[t][i] = w0 + i < a.words ? p[w0 + i] : 0u;
      }
#pragma unroll
      for (int i = 0; i < SC; ++i) {
        const int g = min((kb + i * 32) / a.group, a.groups - 1);
        st.s[t][i] = load_f32(a.scale, a.scale_dtype, (int64_t)row[t] * a.groups + g);
        st.z[t][i] = a.zero ? (float)((a.zero[(int64_t)(row[t] >> 3) * a.groups + g] >> (4 * (row[t] & 7))) & 15u) : 8.0f;
      }
    }
  }

  template <bool SIGNED>
  __device__ __forceinline__ void step(Step& st, int kb) {
    const Operand ones = T::id == CTMI_BF16 ? Operand{{0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u}}
                                            : Operand{{0x3C003C00u, 0x3C003C00u, 0x3C003C00u, 0x3C003C00u}};
    Operand x[MT][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const int m = m0 + mt * 16 + c;
      const uint16_t* p = a.x + (int64_t)m * a.x_stride;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int at = kb + (SMALL ? t * 32 + j * 8 : j * 32 + t * 8);
        Vec<uint32_t, 4> v = {};
        if (m < a.m) {
          if (at + 8 <= a.k) {
            v = ldg<uint32_t, 4>((const uint32_t*)(p + at));
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (at + e < a.k) v.v[e / 2] |= (uint32_t)p[at + e] << (16 * (e % 2));
          }
        }
        x[mt][t] = reorder(v);
      }
    }
    f32x4 sums[MT];
    if constexpr (!SIGNED && !SMALL) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        sums[mt] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int t = 0; t < 4; ++t) sums[mt] = product<T>(x[mt][t], ones, sums[mt]);
      }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      if constexpr (SMALL) transpose4(st.w[nt]);
      f32x4 acc[MT];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) acc[mt] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int at = SMALL ? t : 0;
        Operand w;
        if constexpr (SIGNED) w = signed_codes_of<T>(st.w[nt][t], st.z[nt][at]);
        else w = codes_of<T>(st.w[nt][t]);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          acc[mt] = product<T>(x[mt][t], w, acc[mt]);
          if constexpr (SMALL) {
            if constexpr (!SIGNED) sums[mt] = product<T>(x[mt][t], ones, f32x4{0, 0, 0, 0});
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float v = SIGNED ? acc[mt][i] : fmaf(-st.z[nt][at], sums[mt][i], acc[mt][i]);
              y[nt][mt][i] = fmaf(st.s[nt][at], v, y[nt][mt][i]);
            }
            acc[mt] = f32x4{0, 0, 0, 0};
          }
        }
      }
      if constexpr (!SMALL) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float v = SIGNED ? acc[mt][i] : fmaf(-st.z[nt][0], sums[mt][i], acc[mt][i]);
            y[nt][mt][i] = fmaf(st.s[nt][0], v, y[nt][mt][i]);
          }
      }
    }
  }

  template <bool SIGNED>
  __device__ __forceinline__ void run(int k0, int k1) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) y[nt][mt] = f32x4{0, 0, 0, 0};
    Step now[PF];
#pragma unroll
    for (int p = 0; p < PF; ++p)
      if (k0 + p * kStepK < k1) load(now[p], k0 + p * kStepK);
    for (int kb = k0; kb < k1; kb += PF * kStepK) {
      Step next[PF];
#pragma unroll
      for (int p = 0; p < PF; ++p) {
        const int at = kb + (PF + p) * kStepK;
        if (at < k1) load(next[p], at);
      }
#pragma unroll
      for (int p = 0; p < PF; ++p)
        if (kb + p * kStepK < k1) step<SIGNED>(now[p], kb + p * kStepK);
#pragma unroll
      for (int p = 0; p < PF; ++p) now[p] = next[p];
    }
  }
};

template <typename T, int MT, int NT, bool SMALL, int WAVES>
__global__ __launch_bounds__(WAVES* kWave) void packed_linear_kernel(LinearArgs a) {
  constexpr int TM = MT * 16, TN = NT * 16;
  extern __shared__ float meet[];  // [wave][TM][TN]
  const int wave = threadIdx.x / kWave, waves = blockDim.x / kWave;
  const int n0 = blockIdx.x * TN;
  LinearWave<T, MT, NT, SMALL> w{a};
  w.lane = lane_id(), w.c = w.lane & 15, w.j = w.lane >> 4, w.m0 = blockIdx.y * TM;
#pragma unroll
  for (int t = 0; t < NT; ++t) w.row[t] = min(n0 + t * 16 + w.c, a.n - 1);
  const int64_t k0 = ((int64_t)blockIdx.z * waves + wave) * a.wave_k;
  const int k1 = (int)(k0 + a.wave_k < a.k ? k0 + a.wave_k : a.k);
  if (k0 < k1) {
    w.template run<false>((int)k0, k1);
    bool bad = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int i = 0; i < 4; ++i) bad |= !(fabsf(w.y[nt][mt][i]) <= 3.4028235e38f);
    if (__any(bad)) w.template run<true>((int)k0, k1);
  } else {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) w.y[nt][mt] = f32x4{0, 0, 0, 0};
  }
  const int rows = min(TM, a.m - w.m0);
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
      const int64_t cell = (int64_t)(w.m0 + r) * a.n + n;
      if (a.part) a.part[(int64_t)blockIdx.z * a.m * a.n + cell] = v;
      else a.out[cell] = T::from_f32(v + (a.bias ? T::to_f32(a.bias[n]) : 0.0f));
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

LinearLaunch plan_linear(int64_t m, int64_t n, int64_t k) {
  LinearLaunch l;
  l.mt = m <= 16 ? 1 : m <= 32 ? 2 : 4;
  const int64_t tiles = cdiv(n, 16), m_blocks = cdiv(m, l.mt * 16);
  l.splits = 1;
  if (l.mt == 1) {
    l.nt = tiles >= 1024 ? 4 : tiles >= 512 ? 2 : 1;
    l.waves = 8;
    if (k > 8 * 512 && tiles <= 512) l.waves = 16;
  } else {
    l.nt = 4;
    l.waves = 4;
    const int64_t units = cdiv(n, 64) * m_blocks;
    while (units * l.splits < 256 && k / (l.waves * l.splits * 2) >= 256 && l.splits < 16) l.splits *= 2;
  }
  l.wave_k = cdiv(cdiv(k, l.waves * l.splits), kStepK) * kStepK;
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
  CTMI_REQUIRE(scale_dtype == CTMI_F32 || scale_dtype == CTMI_F16 || scale_dtype == CTMI_BF16,
               CTMI_ERR_UNSUPPORTED, "unsupported scale dtype %d", scale_dtype);
  CTMI_REQUIRE(m >= 0 && n >= 0 && k >= 1, CTMI_ERR_VALUE, "bad sizes [%lld, %lld] x [%lld, %lld]",
               (long long)m, (long long)k, (long long)n, (long long)k);
  CTMI_REQUIRE(m < (1ll << 31) && n < (1ll << 31) && k < (1ll << 31), CTMI_ERR_UNSUPPORTED,
               "sizes must stay below 2^31");
  CTMI_REQUIRE(group == k || (group >= 32 && group % 32 == 0 && k % group == 0), CTMI_ERR_UNSUPPORTED,
               "groups of %lld do not fit %lld columns: a multiple of 32 that divides them, or one group",
               (long long)group, (long long)k);
  CTMI_REQUIRE(x_stride >= k || m <= 1, CTMI_ERR_VALUE, "x_stride %lld is less than %lld columns",
               (long long)x_stride, (long long)k);
  if (m == 0 || n == 0) return CTMI_OK;
  CTMI_REQUIRE(x && packed && scale && out, CTMI_ERR_VALUE, "NULL tensor");
  CTMI_REQUIRE(((uintptr_t)x % 16 == 0) && (x_stride % 8 == 0 || m == 1), CTMI_ERR_VALUE,
               "rows of x must start at 16-byte boundaries");
  const LinearLaunch l = plan_linear(m, n, k);
  const int64_t need = l.splits > 1 ? l.splits * m * n * 4 : 0;
  CTMI_REQUIRE(tmp_bytes >= need && (need == 0 || (tmp != nullptr && (uintptr_t)tmp % 16 == 0)), CTMI_ERR_VALUE,
               "tmp needs %lld bytes at a 16-byte boundary, has %lld", (long long)need, (long long)tmp_bytes);
  const int64_t tm = l.mt * 16, tn = l.nt * 16;
  CTMI_REQUIRE(cdiv(m, tm) < (1 << 16), CTMI_ERR_UNSUPPORTED, "too many rows: %lld", (long long)m);
  LinearArgs a{(const uint16_t*)x, x_stride, (const uint32_t*)packed, scale, (const uint32_t*)zero_point,
               (const uint16_t*)bias, (uint16_t*)out, need ? (float*)tmp : nullptr, (int32_t)m, (int32_t)n,
               (int32_t)k, (int32_t)group, (int32_t)(k / group), (int32_t)cdiv(k, 8), scale_dtype,
               (int32_t)l.wave_k};
  const dim3 grid((unsigned)cdiv(n, tn), (unsigned)cdiv(m, tm), (unsigned)l.splits), threads(l.waves * kWave);
  const size_t lds = (size_t)l.waves * tm * tn * sizeof(float);
  const hipStream_t s = (hipStream_t)stream;
  const bool small = group % kStepK != 0 && group != k;
#define LAUNCH(T, MT, NT, W) do { if (small) packed_linear_kernel<T, MT, NT, true, W><<<grid, threads, lds, s>>>(a); \
                                  else packed_linear_kernel<T, MT, NT, false, W><<<grid, threads, lds, s>>>(a); } while (0)
#define BY_SIZE(T)                                  \
  do {                                              \
    if (l.mt == 4) LAUNCH(T, 4, 4, 4);              \
    else if (l.mt == 2) LAUNCH(T, 2, 4, 4);         \
    else if (l.nt == 4) LAUNCH(T, 1, 4, 8);         \
    else if (l.nt == 2) LAUNCH(T, 1, 2, 16);        \
    else LAUNCH(T, 1, 1, 16);                       \
    if (need) packed_linear_join_kernel<T><<<dim3((unsigned)(cdiv(m * n, 256) < 2048 ? cdiv(m * n, 256) : 2048)), dim3(256), 0, s>>>(a, (int)l.splits); \
  } while (0)
  if (x_dtype == CTMI_BF16) BY_SIZE(BF16);
  else BY_SIZE(F16);
#undef BY_SIZE
#undef LAUNCH
  return check_launch("packed_linear");
}
