// ctmi_kv_append: new keys and values into the 8-bit block cache.
//
// A workgroup owns one block, head and side (keys or values): the scale of a block is one
// number, so whoever finds the largest new value also rewrites the older codes where the
// scale grew and encodes the new ones.  The grid has a workgroup per token; the one whose
// token starts a run of slots in a block does the whole run, the others leave at once.
#include "kv_blocks.h"

namespace ctmi {
namespace {

constexpr int kAppendThreads = 256;
constexpr float kScaleFloor = 1.1920928955078125e-07f;  // eps of fp32, as calculate_qparams clamps

struct AppendArgs {
  const uint16_t* x[2];           // keys, values
  int64_t token_stride[2], head_stride[2];
  const int64_t* slots;
  int64_t tokens;
  uint8_t* codes[2];
  float* scales[2];
  int64_t pool;                   // slots in the pool
  int32_t kv_heads, head_dim, block_size, dynamic;
};

template <bool FP8>
__device__ __forceinline__ uint8_t encode(float v) {  // v = x / scale
  if constexpr (FP8) {
    return f32_to_f8e4m3(v != v ? v : fminf(fmaxf(v, -448.0f), 448.0f));
  } else {
    return (uint8_t)(int8_t)f32_to_int(rintf(v != v ? v : fminf(fmaxf(v, -128.0f), 127.0f)));
  }
}

template <bool FP8>
__device__ __forceinline__ float decode(uint8_t c) {
  return FP8 ? f8e4m3_to_f32(c) : (float)(int8_t)c;
}

template <typename T, bool FP8>
__global__ __launch_bounds__(kAppendThreads) void kv_append_kernel(AppendArgs a) {
  const int64_t t = blockIdx.x;
  const int head = blockIdx.y, side = blockIdx.z, bs = a.block_size, d = a.head_dim;
  const int64_t slot = a.slots[t];
  if (slot < 0 || slot >= a.pool) return;
  const int64_t block = slot / bs;
  const int at = (int)(slot - block * bs);
  if (t > 0 && at > 0 && a.slots[t - 1] == slot - 1) return;  // inside a run another workgroup does
  int n = 1;
  while (n < bs - at && t + n < a.tokens && a.slots[t + n] == slot + n) ++n;

  const uint16_t* x = a.x[side] + t * a.token_stride[side] + head * a.head_stride[side];
  const int64_t stride = a.token_stride[side];
  uint8_t* codes = a.codes[side] + (block * a.kv_heads + head) * (int64_t)bs * d;
  float* scale = a.scales[side] + block * a.kv_heads + head;
  // place of element e of the token at position p
  const int step_p = side ? 1 : d, step_e = side ? bs : 1;

  float now = *scale;
  if (a.dynamic) {
    float peak = 0.0f;
    for (int i = threadIdx.x; i < n * d; i += kAppendThreads) {
      const float v = fabsf(T::to_f32(x[(i / d) * stride + i % d]));
      peak = fmaxf(peak, v <= 3.4028235e38f ? v : 0.0f);
    }
    __shared__ float peaks[kAppendThreads / kWave];
#pragma unroll
    for (int m = 1; m < kWave; m *= 2) peak = fmaxf(peak, wave_shfl_xor(peak, m));
    if (lane_id() == 0) peaks[threadIdx.x / kWave] = peak;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kAppendThreads / kWave; ++w) peak = fmaxf(peak, peaks[w]);
    const float was = now, fits = fmaxf(peak / (FP8 ? 448.0f : 127.5f), kScaleFloor);
    now = at == 0 ? fits : fmaxf(was, fits);
    if (at > 0 && now != was) {
      const float ratio = was / now;
      for (int i = threadIdx.x; i < at * d; i += kAppendThreads) {
        uint8_t* c = codes + (i / d) * step_p + (i % d) * step_e;
        *c = encode<FP8>(decode<FP8>(*c) * ratio);
      }
    }
    if (threadIdx.x == 0) *scale = now;
  }
  for (int i = threadIdx.x; i < n * d; i += kAppendThreads) {
    const float v = T::to_f32(x[(i / d) * stride + i % d]);
    codes[(at + i / d) * step_p + (i % d) * step_e] = encode<FP8>(v / now);
  }
}

}  // namespace
}  // namespace ctmi

using namespace ctmi;

extern "C" int ctmi_kv_append(const void* key, const void* value, int32_t dtype, int64_t key_token_stride,
                              int64_t key_head_stride, int64_t value_token_stride,
                              int64_t value_head_stride, const int64_t* slots, int64_t tokens,
                              const ctmi_kv_blocks* blocks, int32_t dynamic, void* stream) {
  CTMI_REQUIRE(dtype == CTMI_BF16 || dtype == CTMI_F16, CTMI_ERR_UNSUPPORTED,
               "keys and values must be bfloat16 or float16");
  const int rc = check_kv_blocks(blocks);
  if (rc != CTMI_OK) return rc;
  CTMI_REQUIRE(tokens >= 0 && tokens < (1ll << 31), CTMI_ERR_VALUE, "bad token count %lld", (long long)tokens);
  CTMI_REQUIRE(blocks->kv_heads < (1 << 16), CTMI_ERR_UNSUPPORTED, "at most 65535 heads");
  if (tokens == 0 || blocks->num_blocks == 0) return CTMI_OK;
  CTMI_REQUIRE(key && value && slots, CTMI_ERR_VALUE, "NULL tensor");
  AppendArgs a{{(const uint16_t*)key, (const uint16_t*)value},
               {key_token_stride, value_token_stride},
               {key_head_stride, value_head_stride},
               slots, tokens,
               {(uint8_t*)blocks->key, (uint8_t*)blocks->value},
               {blocks->key_scale, blocks->value_scale},
               blocks->num_blocks * blocks->block_size,
               blocks->kv_heads, blocks->head_dim, blocks->block_size, dynamic};
  const dim3 grid((unsigned)tokens, (unsigned)blocks->kv_heads, 2), threads(kAppendThreads);
  const hipStream_t s = (hipStream_t)stream;
  const bool fp8 = blocks->code_dtype == CTMI_F8E4M3;
  if (dtype == CTMI_BF16) {
    if (fp8) kv_append_kernel<BF16, true><<<grid, threads, 0, s>>>(a);
    else kv_append_kernel<BF16, false><<<grid, threads, 0, s>>>(a);
  } else {
    if (fp8) kv_append_kernel<F16, true><<<grid, threads, 0, s>>>(a);
    else kv_append_kernel<F16, false><<<grid, threads, 0, s>>>(a);
  }
  return check_launch("kv_append");
}
