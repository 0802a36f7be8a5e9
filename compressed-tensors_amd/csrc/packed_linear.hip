// ctmi_packed_linear: products of a few rows with a 4-bit packed weight.
//
// One wavefront per output column; a lane takes every 64th word (8 codes) of the row.
#include "ctmi_device.h"
#include "ctmi_host.h"

namespace ctmi {
namespace {

struct LinearArgs {
  const uint16_t* x;
  int64_t x_stride;
  const uint32_t* packed;
  const void* scale;
  const uint32_t* zero;
  const uint16_t* bias;
  uint16_t* out;
  int64_t m, n, k, group;
  int32_t scale_dtype;
};

template <typename T>
__global__ __launch_bounds__(kWave) void packed_linear_kernel(LinearArgs a) {
  constexpr int ROWS = 4;
  const int64_t n = blockIdx.x, m0 = (int64_t)blockIdx.y * ROWS, words = (a.k + 7) / 8, groups = a.k / a.group;
  const int lane = lane_id();
  float sum[ROWS] = {};
  for (int64_t w = lane; w < words; w += kWave) {
    const uint32_t word = a.packed[n * words + w];
    const int64_t g = w * 8 / a.group;
    const float scale = load_f32(a.scale, a.scale_dtype, n * groups + g);
    int zero = 8;
    if (a.zero) zero = (a.zero[(n / 8) * groups + g] >> (4 * (n % 8))) & 15;
    for (int i = 0; i < 8 && w * 8 + i < a.k; ++i) {
      const float v = (float)((int)((word >> (4 * i)) & 15) - zero) * scale;
      for (int j = 0; j < ROWS; ++j)
        if (m0 + j < a.m) sum[j] = fmaf(v, T::to_f32(a.x[(m0 + j) * a.x_stride + w * 8 + i]), sum[j]);
    }
  }
  for (int j = 0; j < ROWS; ++j) {
    float s = sum[j];
    for (int d = 1; d < kWave; d *= 2) s += wave_shfl_xor(s, d);
    if (lane == 0 && m0 + j < a.m)
      a.out[(m0 + j) * a.n + n] = T::from_f32(s + (a.bias ? T::to_f32(a.bias[n]) : 0.0f));
  }
}

}  // namespace
}  // namespace ctmi

using namespace ctmi;

extern "C" int64_t ctmi_packed_linear_tmp_bytes(int64_t m, int64_t n, int64_t k, int64_t group) { return 0; }

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
  CTMI_REQUIRE(tmp_bytes >= ctmi_packed_linear_tmp_bytes(m, n, k, group), CTMI_ERR_VALUE,
               "tmp holds %lld bytes, too few", (long long)tmp_bytes);
  LinearArgs a{(const uint16_t*)x, x_stride, (const uint32_t*)packed, scale, (const uint32_t*)zero_point,
               (const uint16_t*)bias, (uint16_t*)out, m, n, k, group, scale_dtype};
  CTMI_REQUIRE(cdiv(m, 4) < (1 << 16), CTMI_ERR_UNSUPPORTED, "too many rows: %lld", (long long)m);
  const dim3 grid((unsigned)n, (unsigned)cdiv(m, 4));
  if (x_dtype == CTMI_BF16) packed_linear_kernel<BF16><<<grid, dim3(kWave), 0, (hipStream_t)stream>>>(a);
  else packed_linear_kernel<F16><<<grid, dim3(kWave), 0, (hipStream_t)stream>>>(a);
  return check_launch("packed_linear");
}
