// ctmi_kv_plan: block tables, slots and the free list of one serving step.
//
// Integer bookkeeping over a few thousand numbers, so a launch's latency is all there is to
// it.  One launch does it: every workgroup computes the three running sums over the requests
// (new tokens, blocks to take, blocks given back) for itself in LDS - at most 4096 requests,
// 16 a thread -, then fills its share of the outputs.  Workgroups never wait for each other
// and no output is read back, which is why inputs and outputs may not overlap.
// Measured on one MI355X: 24 requests 6 us, 1000 requests (3.8 MB in and out) 10 us.
#include "ctmi_device.h"
#include "ctmi_host.h"

namespace ctmi {
namespace {

constexpr int kPlanThreads = 256;
constexpr int64_t kPlanMaxRequests = 4096;

struct PlanArgs {
  const int32_t *lens, *add, *table, *free, *num_free;
  int64_t width, capacity, slot_count;
  int32_t requests, block_size;
  int32_t *lens_out, *start;
  int64_t* slots;
  int32_t *table_out, *free_out, *num_free_out, *status;
};

// the last index i of the rising a[0 ... n] (a[0] == 0) with a[i] <= v, for v < a[n]
__device__ __forceinline__ int last_at_most(const int32_t* a, int n, int32_t v) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a[mid] <= v) lo = mid;
    else hi = mid;
  }
  return lo;
}

// exclusive running sums of two numbers per thread over the workgroup, in place; *all_ = the sums
__device__ __forceinline__ void scan256(uint64_t& a, uint64_t& b, uint64_t (*sums)[2], uint64_t* all_a, uint64_t* all_b) {
  const int lane = lane_id(), wave = threadIdx.x / kWave;
  uint64_t up_a = a, up_b = b;
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) {
    const uint64_t o_a = __shfl_up(up_a, d, kWave), o_b = __shfl_up(up_b, d, kWave);
    if (lane >= d) up_a += o_a, up_b += o_b;
  }
  if (lane == kWave - 1) sums[wave][0] = up_a, sums[wave][1] = up_b;
  __syncthreads();
  a = up_a - a, b = up_b - b;
  *all_a = *all_b = 0;
#pragma unroll
  for (int w = 0; w < kPlanThreads / kWave; ++w) {
    if (w < wave) a += sums[w][0], b += sums[w][1];
    *all_a += sums[w][0], *all_b += sums[w][1];
  }
}

// A request in 32 bits: lengths are below 2^31, so is what a length and an addition need in
// blocks, and every sum over the requests once they all fit their rows (requests x width is).
struct PlanRequest {
  uint32_t len, add, held, need;  // tokens, and blocks before and after
  bool ends, fits;
  __device__ __forceinline__ PlanRequest(const PlanArgs& a, int r) {
    const int32_t l = a.lens[r], n = a.add[r];
    const uint32_t bs = a.block_size;
    len = (uint32_t)l, ends = n < 0, add = ends ? 0u : (uint32_t)n;
    held = len / bs + (len % bs != 0);
    const uint32_t after = len + add;
    need = after / bs + (after % bs != 0);
    fits = l >= 0 && after <= 0x7FFFFFFFu && need <= (uint32_t)a.width && held <= (uint32_t)a.width;
  }
};

__global__ __launch_bounds__(kPlanThreads) void kv_plan_kernel(PlanArgs a) {
  extern __shared__ int32_t lds[];  // start, want, back: requests + 1 each
  __shared__ uint64_t sums[kPlanThreads / kWave][2];
  const int n = a.requests;
  int32_t *start = lds, *want = lds + n + 1, *back = lds + 2 * (n + 1);
  const int32_t had = a.num_free[0];

  const int per = (n + kPlanThreads - 1) / kPlanThreads;
  const int r0 = min(n, (int)threadIdx.x * per), r1 = min(n, r0 + per);
  uint64_t tokens = 0, blocks = 0;  // blocks: those to take, and above 2^32 those that come back
  bool misfit = false;
  for (int r = r0; r < r1; ++r) {
    const PlanRequest q(a, r);
    misfit |= !q.fits;
    tokens += q.add;
    blocks += q.ends ? (uint64_t)q.held << 32 : (uint64_t)(q.need - q.held);
  }
  uint64_t all_tokens, all_blocks;
  scan256(tokens, blocks, sums, &all_tokens, &all_blocks);
  misfit = __syncthreads_or(misfit);
  const int64_t all_wants = (uint32_t)all_blocks, all_backs = all_blocks >> 32;

  int64_t status = 0;
  if (misfit) status = -1;
  else if (all_tokens > (uint64_t)a.slot_count) status = -2;
  else if (had < 0 || had > a.capacity || had + all_backs > a.capacity) status = -3;
  else if (all_wants > had + all_backs) status = all_wants - had - all_backs;
  const bool ok = status == 0;

  if (ok) {
    uint32_t t = (uint32_t)tokens, w = (uint32_t)blocks, b = (uint32_t)(blocks >> 32);
    for (int r = r0; r < r1; ++r) {
      const PlanRequest q(a, r);
      start[r] = (int32_t)t, want[r] = (int32_t)w, back[r] = (int32_t)b;
      t += q.add;
      if (q.ends) b += q.held;
      else w += q.need - q.held;
    }
    if (threadIdx.x == 0) start[n] = (int32_t)all_tokens, want[n] = (int32_t)all_wants, back[n] = (int32_t)all_backs;
  }
  __syncthreads();

  const uint32_t width = (uint32_t)a.width;
  const int32_t top = had + (int32_t)all_backs;  // height of the stack before the pops
  // entry p of the stack: the free list, above it what ended requests give back
  auto stack = [&](int32_t p) -> int32_t {
    if (p < had) return a.free[p];
    const int r = last_at_most(back, n, p - had);
    return a.table[(uint32_t)r * width + (uint32_t)(p - had - back[r])];
  };
  // block `column` of request r, old or newly taken
  auto block_of = [&](int r, uint32_t column, uint32_t held) -> int32_t {
    return column < held ? a.table[(uint32_t)r * width + column] : stack(top - 1 - (int32_t)((uint32_t)want[r] + column - held));
  };

  const uint32_t first = blockIdx.x * kPlanThreads + threadIdx.x, step = gridDim.x * kPlanThreads;
  for (uint32_t i = first; i < (uint32_t)a.slot_count; i += step) {
    int64_t slot = -1;
    if (ok && i < all_tokens) {
      const int r = last_at_most(start, n, (int32_t)i);
      const PlanRequest q(a, r);
      const uint32_t place = q.len + (i - (uint32_t)start[r]), bs = a.block_size, column = place / bs;
      const int64_t block = block_of(r, column, q.held);
      if (block >= 0) slot = block * bs + (place - column * bs);
    }
    a.slots[i] = slot;
  }
  for (uint32_t i = first; i < (uint32_t)n * width; i += step) {
    int32_t v = a.table[i];
    if (ok) {
      const uint32_t r = i / width, column = i - r * width;
      const PlanRequest q(a, (int)r);
      if (q.ends) v = -1;
      else if (column >= q.held && column < q.need) v = block_of((int)r, column, q.held);
    }
    a.table_out[i] = v;
  }
  const int32_t left = ok ? top - (int32_t)all_wants : had;
  for (uint32_t i = first; i < (uint32_t)a.capacity; i += step)
    a.free_out[i] = !ok ? a.free[i] : (int32_t)i < left ? stack((int32_t)i) : -1;
  for (uint32_t i = first; i <= (uint32_t)n; i += step) {
    a.start[i] = ok ? start[i] : 0;
    if (i < (uint32_t)n) {
      const int32_t len = a.lens[i], add = a.add[i];
      a.lens_out[i] = !ok ? len : add < 0 ? 0 : len + add;
    }
  }
  if (first == 0) {
    a.num_free_out[0] = left;
    a.status[0] = (int32_t)status;
  }
}

}  // namespace
}  // namespace ctmi

using namespace ctmi;

extern "C" int ctmi_kv_plan(const int32_t* seq_lens, const int32_t* new_tokens, const int32_t* block_table,
                            const int32_t* free_blocks, const int32_t* num_free, int64_t requests,
                            int64_t width, int64_t free_capacity, int64_t slot_count, int32_t block_size,
                            int32_t* seq_lens_out, int32_t* query_start, int64_t* slots,
                            int32_t* table_out, int32_t* free_out, int32_t* num_free_out,
                            int32_t* status, void* stream) {
  CTMI_REQUIRE(requests >= 0 && width >= 1 && free_capacity >= 0 && slot_count >= 0, CTMI_ERR_VALUE,
               "bad sizes: %lld requests, %lld table columns, %lld free blocks, %lld slots",
               (long long)requests, (long long)width, (long long)free_capacity, (long long)slot_count);
  CTMI_REQUIRE(requests <= kPlanMaxRequests, CTMI_ERR_UNSUPPORTED, "at most %lld requests per call, got %lld",
               (long long)kPlanMaxRequests, (long long)requests);
  CTMI_REQUIRE(width < (1ll << 31) && (requests == 0 || width < (1ll << 31) / requests) &&
                   free_capacity < (1ll << 31) && slot_count < (1ll << 31),
               CTMI_ERR_UNSUPPORTED, "table entries, free blocks and slots must each stay below 2^31");
  CTMI_REQUIRE(block_size >= 1, CTMI_ERR_VALUE, "block_size must be at least 1, got %d", block_size);
  CTMI_REQUIRE(num_free && query_start && num_free_out && status &&
                   (requests == 0 || (seq_lens && new_tokens && block_table && seq_lens_out && table_out)) &&
                   (free_capacity == 0 || (free_blocks && free_out)) && (slot_count == 0 || slots),
               CTMI_ERR_VALUE, "NULL tensor");
  PlanArgs a{seq_lens, new_tokens, block_table, free_blocks, num_free, width, free_capacity, slot_count,
             (int32_t)requests, block_size, seq_lens_out, query_start, slots, table_out, free_out,
             num_free_out, status};
  // An output is a chain of dependent loads, so a thread has one, if the grid allows (1000
  // requests 7.9 us, with eight a thread 14.3).  Each workgroup repeats the scan: of many requests
  // one workgroup per compute unit does (4096 requests, 64 blocks each: 17 us, 41 with four times
  // as many), of fewer up to four (1000 requests, 256 blocks each and 10^5 tokens: 10.0, one 13.3).
  const int64_t most = slot_count > requests * width ? slot_count : requests * width;
  int64_t grid = cdiv(most > free_capacity ? most : free_capacity, (int64_t)kPlanThreads);
  const int64_t cap = requests > 1024 ? 256 : 1024;
  if (grid < 1) grid = 1;
  if (grid > cap) grid = cap;
  const size_t lds = (size_t)(requests + 1) * 3 * sizeof(int32_t);
  kv_plan_kernel<<<dim3((unsigned)grid), dim3(kPlanThreads), lds, (hipStream_t)stream>>>(a);
  return check_launch("kv_plan");
}
