// ctmi_kv_attend: attention over the 8-bit block cache.
//
// One wavefront per query and head walks its keys once with a running maximum and sum; a
// lane owns head_dim / 64 of the dimensions.
#include "kv_blocks.h"

namespace ctmi {
namespace {

struct AttendArgs {
  const uint16_t* q;
  int64_t q_token_stride, q_head_stride;
  uint16_t* out;
  const uint8_t *key, *value;
  const float *key_scale, *value_scale;
  int64_t num_blocks;
  int32_t kv_heads, head_dim, block_size, q_heads;
  const int32_t *table, *lens, *start;
  int64_t table_stride, width, tokens, requests;
  float scale;
};

template <bool FP8>
__device__ __forceinline__ float decode(uint8_t c) {
  return FP8 ? f8e4m3_to_f32(c) : (float)(int8_t)c;
}

template <typename T, bool FP8, int D>
__global__ __launch_bounds__(kWave) void kv_attend_kernel(AttendArgs a) {
  constexpr int PER = D / kWave;
  const int64_t r = blockIdx.x;
  const int head = blockIdx.y, lane = lane_id();
  const int kv = head / (a.q_heads / a.kv_heads), bs = a.block_size;
  const int64_t q0 = a.start ? min(max((int64_t)a.start[r], (int64_t)0), a.tokens) : r;
  const int64_t q1 = a.start ? min(max((int64_t)a.start[r + 1], q0), a.tokens) : r + 1;
  const int64_t len = min(max((int64_t)a.lens[r], (int64_t)0), a.width * bs);
  for (int64_t t = q0 + blockIdx.z; t < q1; t += gridDim.z) {
    float q[PER], o[PER] = {}, top = -INFINITY, sum = 0.0f;
    for (int e = 0; e < PER; ++e)
      q[e] = T::to_f32(a.q[t * a.q_token_stride + head * a.q_head_stride + e * kWave + lane]);
    const int64_t end = len - (q1 - q0) + (t - q0) + 1;  // keys this query sees
    for (int64_t j = 0; j < end; ++j) {
      const int64_t block = a.table[r * a.table_stride + j / bs];
      if (block < 0 || block >= a.num_blocks) continue;
      const int64_t cell = block * a.kv_heads + kv;
      const int at = (int)(j % bs);
      float s = 0.0f;
      for (int e = 0; e < PER; ++e) s += q[e] * decode<FP8>(a.key[(cell * bs + at) * D + e * kWave + lane]);
      for (int m = 1; m < kWave; m *= 2) s += wave_shfl_xor(s, m);
      s *= a.key_scale[cell] * a.scale;
      const float now = fmaxf(top, s);
      const float shrink = top == -INFINITY ? 0.0f : expf(top - now);
      const float p = s == -INFINITY ? 0.0f : expf(s - now);
      sum = sum * shrink + p;
      const float pv = p * a.value_scale[cell];
      for (int e = 0; e < PER; ++e)
        o[e] = o[e] * shrink + pv * decode<FP8>(a.value[(cell * D + e * kWave + lane) * bs + at]);
      top = now;
    }
    for (int e = 0; e < PER; ++e)
      a.out[(t * a.q_heads + head) * D + e * kWave + lane] = T::from_f32(sum == 0.0f ? 0.0f : o[e] / sum);
  }
}

}  // namespace
}  // namespace ctmi

using namespace ctmi;

extern "C" int64_t ctmi_kv_attend_tmp_bytes(int64_t tokens, int64_t requests, int32_t q_heads,
                                            int32_t kv_heads, int32_t head_dim, int64_t max_query,
                                            int64_t max_seq) {
  return 0;
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
  CTMI_REQUIRE(tokens < (1ll << 31) && requests < (1ll << 31) && q_heads < (1 << 16) &&
                   width * blocks->block_size < (1ll << 31),
               CTMI_ERR_UNSUPPORTED, "tokens, requests and positions must stay below 2^31, heads below 65536");
  CTMI_REQUIRE(query_start != nullptr || tokens == requests, CTMI_ERR_VALUE,
               "without query_start every request has one token: got %lld tokens for %lld requests",
               (long long)tokens, (long long)requests);
  CTMI_REQUIRE(max_query >= 1 && max_seq >= 1, CTMI_ERR_VALUE, "max_query and max_seq must be at least 1");
  if (tokens == 0 || requests == 0) return CTMI_OK;
  CTMI_REQUIRE(q && out && seq_lens && (width == 0 || block_table), CTMI_ERR_VALUE, "NULL tensor");
  CTMI_REQUIRE(q_token_stride % 8 == 0 && q_head_stride % 8 == 0 && ((uintptr_t)q | (uintptr_t)out) % 16 == 0,
               CTMI_ERR_VALUE, "queries must be 16-byte aligned, token by token and head by head");
  CTMI_REQUIRE(tmp_bytes >= ctmi_kv_attend_tmp_bytes(tokens, requests, q_heads, blocks->kv_heads,
                                                     blocks->head_dim, max_query, max_seq),
               CTMI_ERR_VALUE, "tmp holds %lld bytes, too few", (long long)tmp_bytes);
  AttendArgs a{(const uint16_t*)q, q_token_stride, q_head_stride, (uint16_t*)out,
               (const uint8_t*)blocks->key, (const uint8_t*)blocks->value, blocks->key_scale,
               blocks->value_scale, blocks->num_blocks, blocks->kv_heads, blocks->head_dim,
               blocks->block_size, q_heads, block_table, seq_lens, query_start, table_stride, width,
               tokens, requests, scale};
  const int64_t z = max_query < 65535 ? max_query : 65535;
  const dim3 grid((unsigned)requests, (unsigned)q_heads, (unsigned)z);
  const hipStream_t s = (hipStream_t)stream;
  const bool fp8 = blocks->code_dtype == CTMI_F8E4M3;
#define LAUNCH(T, F, D) kv_attend_kernel<T, F, D><<<grid, dim3(kWave), 0, s>>>(a)
#define BY_CODE(T, D) do { if (fp8) LAUNCH(T, true, D); else LAUNCH(T, false, D); } while (0)
#define BY_DIM(T) do { if (blocks->head_dim == 64) BY_CODE(T, 64); else if (blocks->head_dim == 128) BY_CODE(T, 128); else BY_CODE(T, 256); } while (0)
  if (dtype == CTMI_BF16) BY_DIM(BF16);
  else BY_DIM(F16);
#undef BY_DIM
#undef BY_CODE
#undef LAUNCH
  return check_launch("kv_attend");
}
