// ctmi_kv_append: new keys and values into the 8-bit block cache.
//
// A workgroup owns one block, head and side (keys or values): the scale of a block is one
// number, so whoever finds the largest new value also rewrites the older codes where the
// scale grew and encodes the new ones.  The workgroup whose window of tokens holds the first
// of a run of slots in a block does the whole run; the rest of the run is skipped.
//
// x / scale has to be the correctly rounded quotient (the codes are defined by it).  The
// compiler's division is about 16 instructions an element; here it is a product with the
// correctly rounded reciprocal and two corrections by the exact remainder, 5 instructions,
// whose result is the same for finite x and scales within 2^+-100.  A run that holds anything
// else, or values beyond 2^16 scales (which scales given by the caller allow), divides.
//
// Measured on one MI355X, 8 heads of 128: 3 prompts of 4001 tokens (67 MB) 21 us, 3.2 TB/s, with
// the vector units 57 % busy and wavefronts waiting 27 % of their time: neither alone bounds it;
// one token for each of 48 requests 5.5 us.
//
// Keys: a thread encodes 4 neighbouring dimensions of a token and stores a word.  Values lie
// transposed, tokens innermost: a thread takes 4 dimensions of the 4 tokens that share a word
// and stores 4 words; lanes next to each other take the next words, so that a row's tokens
// leave as whole pieces without a trip through LDS.
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
  int32_t pool;                   // slots in the pool
  uint32_t magic;                 // ceil(2^32 / (block_size / 16)), 0 where that is 1
  int32_t kv_heads, block_size, dynamic, window;
};

template <bool FP8>
__device__ __forceinline__ uint8_t encode(float v) {  // v = x / scale
  if constexpr (FP8) {
    return f32_to_f8e4m3(v != v ? v : fminf(fmaxf(v, -448.0f), 448.0f));
  } else {
    return (uint8_t)(int8_t)f32_to_int(rintf(v != v ? v : fminf(fmaxf(v, -128.0f), 127.0f)));
  }
}

// four quotients, finite -> four codes
template <bool FP8>
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
  constexpr float lo = FP8 ? -448.0f : -128.0f, hi = FP8 ? 448.0f : 127.0f;
  a = __builtin_amdgcn_fmed3f(a, lo, hi), b = __builtin_amdgcn_fmed3f(b, lo, hi);
  c = __builtin_amdgcn_fmed3f(c, lo, hi), d = __builtin_amdgcn_fmed3f(d, lo, hi);
  if constexpr (FP8) {
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false), true);
  } else {
    // 1.5 * 2^23 + v holds the rounded integer (nearest even) in its low bits
    const uint32_t u0 = f2u(a + 12582912.0f), u1 = f2u(b + 12582912.0f);
    const uint32_t u2 = f2u(c + 12582912.0f), u3 = f2u(d + 12582912.0f);
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(u3, u2, 0x0C0C0400u), __builtin_amdgcn_perm(u1, u0, 0x0C0C0400u), 0x05040100u);
  }
}

// x / s, correctly rounded, for finite x and s within 2^+-100; r = 1 / s.  The remainders are taken
// as q s - x: of x = -0 that is +0, and -0 less +0 r stays -0 (x - q s would make it +0).
struct Divisor {
  float s, r;
  __device__ __forceinline__ float operator()(float x) const {
    const float q = x * r, q1 = fmaf(fmaf(q, s, -x), -r, q);
    return fmaf(fmaf(q1, s, -x), -r, q1);
  }
};

template <typename T, bool FP8>
__device__ __forceinline__ uint32_t encode4(const Vec<uint16_t, 4>& x, const Divisor& by) {
  return encode4<FP8>(by(T::to_f32(x.v[0])), by(T::to_f32(x.v[1])), by(T::to_f32(x.v[2])), by(T::to_f32(x.v[3])));
}

// the codes of a word, those of its `count` first positions times ratio (at most 1)
template <bool FP8>
__device__ __forceinline__ uint32_t rescale4(uint32_t w, float ratio, int count) {
  uint32_t o;
  if constexpr (FP8) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    o = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(b[0] * ratio, b[1] * ratio,
                                                  __builtin_amdgcn_cvt_pk_fp8_f32(a[0] * ratio, a[1] * ratio, 0, false), true);
  } else {
    o = encode4<false>((float)(int8_t)w * ratio, (float)(int8_t)(w >> 8) * ratio, (float)(int8_t)(w >> 16) * ratio,
                       (float)(int8_t)(w >> 24) * ratio);
  }
  const uint32_t mask = count >= 4 ? 0xFFFFFFFFu : (1u << (8 * count)) - 1u;
  return (o & mask) | (w & ~mask);
}

// The run of tokens t ... t + n - 1, positions at ... of a block, whose scale is `was`; returns what
// it is afterwards.  peaks: LDS that no wavefront still reads for the run before.
template <typename T, bool FP8, int D, int side>
__device__ __forceinline__ float append_run(const AppendArgs& a, int64_t t, int n, int at, int head, int stride, float was,
                                            uint8_t* codes, float* scale, uint32_t* peaks) {
  constexpr int CH = D / 4;  // pieces of 4 dimensions
  // What a thread loads for the maximum and keeps for the codes: 8 pieces, those of 8 tokens
  // (keys) or of the 4 tokens of 2 words (values).  That is 64 tokens of 128 dimensions; the
  // rest of a longer run is read twice.
  constexpr int KEEP = 8;
  const int bs = a.block_size, lane = lane_id();
  const uint16_t* x = a.x[side] + t * a.token_stride[side] + head * a.head_stride[side];
  // keys: piece i is 4 dimensions of token i / CH.  Values: item i is 4 dimensions of the 4
  // tokens of a word, of which those outside the run are read as its nearest; words of a row
  // of the block are lanes next to each other
  const int word0 = at / 4, words = (at + n + 3) / 4 - word0, items = side == 0 ? n * CH : words * CH;
  const uint32_t magic = 0xFFFFFFFFu / (uint32_t)words + 1;  // i / words for the i there are (words > 1)
  auto row_of = [&](int i) { return words == 1 ? i : (int)__umulhi((uint32_t)i, magic); };
  auto key_piece = [&](int i) { return ldg<uint16_t, 4>(x + (uint32_t)((i / CH) * stride + (i % CH) * 4)); };
  auto first_token = [&](int i) { return (word0 + i - row_of(i) * words) * 4 - at; };
  auto value_piece = [&](int i, int e) {
    return ldg<uint16_t, 4>(x + (uint32_t)(min(max(first_token(i) + e, 0), n - 1) * stride + row_of(i) * 4));
  };
  // magnitudes order like the unsigned integers of their bits, infinities and NaNs above all
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  u16x2 most = {0, 0};
  auto look = [&](const Vec<uint16_t, 4>& v) {
    const Vec<uint32_t, 2> w = __builtin_bit_cast(Vec<uint32_t, 2>, v);
#pragma unroll
    for (int e = 0; e < 2; ++e) most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, w.v[e] & 0x7FFF7FFFu));
  };
  Vec<uint16_t, 4> kept[KEEP];
#pragma unroll
  for (int p = 0; p < KEEP; ++p) {
    // behind the last one the last: loads that stand in no branch
    const int i = min((int)threadIdx.x + (side == 0 ? p : p / 4) * kAppendThreads, items - 1);
    kept[p] = side == 0 ? key_piece(i) : value_piece(i, p % 4);
  }
#pragma unroll
  for (int p = 0; p < KEEP; ++p) look(kept[p]);
  if (side == 0) {
#pragma unroll 1
    for (int i = threadIdx.x + KEEP * kAppendThreads; i < items; i += kAppendThreads) look(key_piece(i));
  } else {
#pragma unroll 1
    for (int i = threadIdx.x + KEEP / 4 * kAppendThreads; i < items; i += kAppendThreads)
      for (int e = 0; e < 4; ++e) look(value_piece(i, e));
  }
  // (the other half of peaks may still be read for the run before)
  uint32_t high = most[0] > most[1] ? most[0] : most[1];
#pragma unroll
  for (int m = 1; m < kWave; m *= 2) high = max(high, (uint32_t)wave_shfl_xor((int)high, m));
  if (lane == 0) peaks[threadIdx.x / kWave] = high;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kAppendThreads / kWave; ++w) high = max(high, peaks[w]);
  constexpr uint32_t kInfinity = T::id == CTMI_BF16 ? 0x7F80u : 0x7C00u;
  const bool strange = high >= kInfinity;
  if (strange) {  // the largest that is finite, element by element
    high = 0;
#pragma unroll 1
    for (int i = threadIdx.x; i < n * D; i += kAppendThreads) {
      const uint32_t m = x[(i / D) * stride + i % D] & 0x7FFFu;
      high = m < kInfinity ? max(high, m) : high;
    }
#pragma unroll
    for (int m = 1; m < kWave; m *= 2) high = max(high, (uint32_t)wave_shfl_xor((int)high, m));
    __syncthreads();
    if (lane == 0) peaks[threadIdx.x / kWave] = high;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kAppendThreads / kWave; ++w) high = max(high, peaks[w]);
  }
  const float peak = T::to_f32((uint16_t)high);

  float now = was;
  if (a.dynamic) {
    const float fits = fmaxf(peak / (FP8 ? 448.0f : 127.5f), kScaleFloor);
    now = at == 0 ? fits : fmaxf(was, fits);
    if (at > 0 && now != was) {
      const float ratio = was / now;
      if (side == 0) {
        uint32_t* w = (uint32_t*)codes;
#pragma unroll 1
        for (int i = threadIdx.x; i < at * (D / 4); i += kAppendThreads) w[i] = rescale4<FP8>(w[i], ratio, 4);
      } else {
        const int old = (at + 3) / 4;
#pragma unroll 1
        for (int i = threadIdx.x; i < old * D; i += kAppendThreads) {
          uint32_t* w = (uint32_t*)(codes + (i / old) * bs) + i % old;
          *w = rescale4<FP8>(*w, ratio, at - (i % old) * 4);
        }
      }
      __syncthreads();  // words that old and new codes share are rewritten before the new ones come
    }
    if (threadIdx.x == 0) *scale = now;
  }

  if (strange || !(now > 0x1p-100f && now < 0x1p100f && peak <= now * 65536.0f)) {
#pragma unroll 1
    for (int i = threadIdx.x; i < n * D; i += kAppendThreads) {
      const int token = i / D, d = i % D;
      codes[side == 0 ? (at + token) * D + d : d * bs + at + token] = encode<FP8>(T::to_f32(x[token * stride + d]) / now);
    }
    return now;
  }
  const Divisor by{now, 1.0f / now};
  if (side == 0) {
#pragma unroll
    for (int p = 0; p < KEEP; ++p) {
      const int i = threadIdx.x + p * kAppendThreads;
      if (i < items) *(uint32_t*)(codes + at * D + i * 4) = encode4<T, FP8>(kept[p], by);
    }
#pragma unroll 1
    for (int i = threadIdx.x + KEEP * kAppendThreads; i < items; i += kAppendThreads)
      *(uint32_t*)(codes + at * D + i * 4) = encode4<T, FP8>(key_piece(i), by);
  } else {
#pragma unroll 1
    for (int i = threadIdx.x, turn = 0; i < items; i += kAppendThreads, ++turn) {
      uint32_t o[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        o[e] = encode4<T, FP8>(turn == 0 ? kept[e] : turn == 1 ? kept[4 + e] : value_piece(i, e), by);
      const int first = first_token(i);
      uint8_t* row = codes + (row_of(i) * 4) * bs + at + first;
      if (first >= 0 && first + 4 <= n) {
        // 4 tokens x 4 dimensions of bytes, transposed
        const uint32_t a01 = __builtin_amdgcn_perm(o[1], o[0], 0x05010400u), b01 = __builtin_amdgcn_perm(o[1], o[0], 0x07030602u);
        const uint32_t a23 = __builtin_amdgcn_perm(o[3], o[2], 0x05010400u), b23 = __builtin_amdgcn_perm(o[3], o[2], 0x07030602u);
        *(uint32_t*)row = __builtin_amdgcn_perm(a23, a01, 0x05040100u);
        *(uint32_t*)(row + bs) = __builtin_amdgcn_perm(a23, a01, 0x07060302u);
        *(uint32_t*)(row + 2 * bs) = __builtin_amdgcn_perm(b23, b01, 0x05040100u);
        *(uint32_t*)(row + 3 * bs) = __builtin_amdgcn_perm(b23, b01, 0x07060302u);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (first + e >= 0 && first + e < n) {
#pragma unroll
            for (int d = 0; d < 4; ++d) row[d * bs + e] = (uint8_t)(o[e] >> (8 * d));
          }
      }
    }
  }
  return now;
}

constexpr uint32_t kNoSlot = 0x80000000u;

// the slot of the first token from `from` on that has one, and which token that is; 512 at a time,
// as the rest of a padded batch has none
__device__ __forceinline__ uint32_t next_slot(const AppendArgs& a, int64_t from, int64_t* token) {
  constexpr int FAR = 8;
  uint32_t slot = kNoSlot;
  for (; from < a.tokens && slot == kNoSlot; from += FAR * kWave) {
    int64_t there[FAR];
#pragma unroll
    for (int f = 0; f < FAR; ++f) {
      const int64_t at = from + f * kWave + lane_id();
      there[f] = at < a.tokens ? a.slots[at] : -1;
    }
#pragma unroll
    for (int f = 0; f < FAR; ++f) {
      const uint64_t any = __ballot((uint64_t)there[f] < (uint64_t)a.pool);
      if (any && slot == kNoSlot) {
        slot = __builtin_amdgcn_readlane((uint32_t)there[f], __builtin_ctzll(any));
        *token = from + f * kWave + __builtin_ctzll(any);
      }
    }
  }
  return slot;
}

template <typename T, bool FP8, int D, int side>
__device__ __forceinline__ void append_window(const AppendArgs& a) {
  const int head = blockIdx.y, bs = a.block_size, lane = lane_id();
  const int stride = (int)a.token_stride[side];
  const int64_t t0 = (int64_t)blockIdx.x * a.window;
  __shared__ uint32_t peaks[2][kAppendThreads / kWave];

  // lane i holds the slot of token t0 - 1 + i: one look at them tells which tokens of the
  // window begin a run and, for all but the longest, how far it goes
  const int64_t mine = t0 - 1 + lane;
  const int64_t wide = mine >= 0 && mine < a.tokens ? a.slots[mine] : -1;
  const bool valid = (uint64_t)wide < (uint64_t)a.pool;
  const uint32_t slot_here = valid ? (uint32_t)wide : kNoSlot;
  const uint32_t slot_before = __shfl_up(slot_here, 1, kWave);
  const uint32_t block_here = a.magic ? __umulhi(slot_here >> 4, a.magic) : slot_here >> 4;
  const int at_here = (int)(slot_here - block_here * (uint32_t)bs);
  // the token before lies before it in the same block: it goes on with that one's run, or has a
  // later one of the block
  const bool later = valid && slot_before < slot_here && slot_before >= slot_here - (uint32_t)at_here && lane > 0;
  const bool goes_on = later && slot_before == slot_here - 1;
  const uint64_t follows = __ballot(goes_on), valids = __ballot(valid);
  // behind whose predecessor the block may have another run
  const uint64_t chained = __ballot((later && !goes_on) || (!valid && slot_before != kNoSlot && mine < a.tokens));
  auto same_block = [&](uint32_t slot, uint32_t before) {
    const uint32_t block = a.magic ? __umulhi(slot >> 4, a.magic) : slot >> 4;
    return before < slot && before >= block * (uint32_t)bs;
  };
  bool begins = valid && !later && lane > 0 && lane <= a.window;
  // (behind tokens that are skipped it lies further back)
  if (__builtin_expect(__any(begins && slot_before == kNoSlot), 0)) {
    const uint64_t before_me = valids & ((1ull << lane) - 1);
    const uint32_t last_before = __shfl(slot_here, before_me ? 63 - __builtin_clzll(before_me) : 0, kWave);
    if (before_me && same_block(slot_here, last_before)) begins = false;
    const int first_valid = __builtin_ctzll(valids);
    for (int64_t base = t0 - 2; first_valid > 0 && base >= 0; base -= kWave) {
      const int64_t there = base - lane >= 0 ? a.slots[base - lane] : -1;
      const uint64_t any = __ballot((uint64_t)there < (uint64_t)a.pool);
      if (any) {
        const uint32_t slot = __builtin_amdgcn_readlane((uint32_t)there, __builtin_ctzll(any));
        if (lane == first_valid && same_block(slot_here, slot)) begins = false;
        break;
      }
    }
  }
  uint64_t left = __ballot(begins);
  int lead = 0, at = 0;  // the run's first token (one behind what was looked at: kWave), its position
  int64_t t = 0, block = 0;
  float was = 0.0f;
  bool same = false;  // the block is that of the run before
  for (int parity = 0; same || left; parity ^= 1) {
    if (!same) {
      lead = __builtin_ctzll(left);
      left &= left - 1;
      t = t0 - 1 + lead;
      block = (int64_t)__builtin_amdgcn_readlane(block_here, lead);
      at = __builtin_amdgcn_readlane(at_here, lead);
      was = a.scales[side][block * a.kv_heads + head];
    }
    const uint64_t behind = lead >= 63 ? 0 : ~(follows >> (lead + 1));  // 0 bits: tokens of the run
    int n = 1 + (lead >= 63 ? 0 : __builtin_ctzll(behind | 1ull << (63 - lead)));
    if (lead + n >= kWave) {  // it may go on behind what was looked at
      const int64_t slot = block * bs + at;
      for (const int most = bs - at; n < most;) {
        const int i = n + lane;
        const uint64_t other = __ballot(!(i < most && t + i < a.tokens && a.slots[t + i] == slot + i));
        if (other) {
          n += __builtin_ctzll(other);
          break;
        }
        n += kWave;
      }
    }
    const int64_t cell = block * a.kv_heads + head;
    was = append_run<T, FP8, D, side>(a, t, n, at, head, stride, was, a.codes[side] + cell * bs * D, a.scales[side] + cell, peaks[parity]);

    // the block's next run: of the nearest token behind that has a slot
    same = false;
    if (at + n < bs && (lead + n >= kWave || (chained >> (lead + n) & 1))) {
      const uint64_t ahead = lead + n < kWave ? valids >> (lead + n) : 0;
      uint32_t next;
      if (ahead) {
        lead += n + __builtin_ctzll(ahead);
        t = t0 - 1 + lead;
        next = __builtin_amdgcn_readlane(slot_here, lead);
      } else {
        next = next_slot(a, t + n > t0 - 1 + kWave ? t + n : t0 - 1 + kWave, &t);
        lead = kWave;
      }
      if (next != kNoSlot && same_block(next, (uint32_t)(block * bs) + at + n - 1)) {
        at = (int)(next - (uint32_t)(block * bs));
        same = true;
        __syncthreads();  // the run before has written its codes
      }
    }
  }
}

template <typename T, bool FP8, int D>
__global__ __launch_bounds__(kAppendThreads) void kv_append_kernel(AppendArgs a) {
  if (blockIdx.z == 0) append_window<T, FP8, D, 0>(a);
  else append_window<T, FP8, D, 1>(a);
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
  CTMI_REQUIRE((key_token_stride | key_head_stride | value_token_stride | value_head_stride) % 8 == 0 &&
                   ((uintptr_t)key | (uintptr_t)value) % 16 == 0,
               CTMI_ERR_VALUE, "keys and values must be 16-byte aligned, token by token and head by head");
  CTMI_REQUIRE(key_token_stride >= 0 && key_token_stride < (1 << 22) && value_token_stride >= 0 &&
                   value_token_stride < (1 << 22),
               CTMI_ERR_UNSUPPORTED, "tokens more than 2^22 elements apart");
  CTMI_REQUIRE(blocks->num_blocks * blocks->block_size < (1ll << 31), CTMI_ERR_UNSUPPORTED,
               "a pool must have fewer than 2^31 slots");
  const uint32_t sixteenths = blocks->block_size / 16;
  AppendArgs a{{(const uint16_t*)key, (const uint16_t*)value},
               {key_token_stride, value_token_stride},
               {key_head_stride, value_head_stride},
               slots, tokens,
               {(uint8_t*)blocks->key, (uint8_t*)blocks->value},
               {blocks->key_scale, blocks->value_scale},
               (int32_t)(blocks->num_blocks * blocks->block_size),
               sixteenths == 1 ? 0u : (uint32_t)(((1ull << 32) + sixteenths - 1) / sixteenths),
               blocks->kv_heads, blocks->block_size, dynamic, 1};
  // a workgroup for each token of a decoding batch; of a prompt most tokens are inside a run,
  // and workgroups that only leave cost more than looking through 32 tokens does
  a.window = tokens <= 1024 ? 1 : tokens < 32 * 256 ? (int32_t)(tokens / 256) : 32;
  const dim3 grid((unsigned)cdiv(tokens, a.window), (unsigned)blocks->kv_heads, 2), threads(kAppendThreads);
  const hipStream_t s = (hipStream_t)stream;
  const bool fp8 = blocks->code_dtype == CTMI_F8E4M3;
#define LAUNCH(T, F, D) kv_append_kernel<T, F, D><<<grid, threads, 0, s>>>(a)
#define BY_CODE(T, D) do { if (fp8) LAUNCH(T, true, D); else LAUNCH(T, false, D); } while (0)
#define BY_DIM(T) do { if (blocks->head_dim == 64) BY_CODE(T, 64); else if (blocks->head_dim == 128) BY_CODE(T, 128); else BY_CODE(T, 256); } while (0)
  if (dtype == CTMI_BF16) BY_DIM(BF16);
  else BY_DIM(F16);
#undef BY_DIM
#undef BY_CODE
#undef LAUNCH
  return check_launch("kv_append");
}
