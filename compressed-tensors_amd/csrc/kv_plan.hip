// ctmi_kv_plan: block tables, slots and the free list of one serving step.
//
// Integer bookkeeping over a few thousand numbers, so a launch's latency is all there is to
// it.  One launch does it: every workgroup computes the three running sums over the requests
// (new tokens, blocks to take, blocks given back) for itself in LDS - at most 4096 requests,
// 16 a thread -, then fills its share of the outputs.  Workgroups never wait for each other
// and no output is read back, which is why inputs and outputs may not overlap.
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

// exclusive running sum of one number per thread over the workgroup; *total = the sum
__device__ __forceinline__ int64_t scan256(int64_t v, int64_t* wave_sums, int64_t* total) {
  const int lane = lane_id(), wave = threadIdx.x / kWave;
  int64_t up = v;
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) {
    const int64_t o = __shfl_up(up, d, kWave);
    if (lane >= d) up += o;
  }
  __syncthreads();  // wave_sums may still be read from the call before
  if (lane == kWave - 1) wave_sums[wave] = up;
  __syncthreads();
  int64_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kPlanThreads / kWave; ++w) {
    if (w < wave) before += wave_sums[w];
    all += wave_sums[w];
  }
  *total = all;
  return before + up - v;
}

__global__ __launch_bounds__(kPlanThreads) void kv_plan_kernel(PlanArgs a) {
  extern __shared__ int32_t lds[];  // start, want, back: requests + 1 each
  __shared__ int64_t wave_sums[kPlanThreads / kWave];
  const int n = a.requests;
  int32_t *start = lds, *want = lds + n + 1, *back = lds + 2 * (n + 1);
  const int64_t bs = a.block_size;

  const int per = (n + kPlanThreads - 1) / kPlanThreads;
  const int r0 = min(n, (int)threadIdx.x * per), r1 = min(n, r0 + per);
  int64_t tokens = 0, wants = 0, backs = 0;
  int misfit = 0;
  for (int r = r0; r < r1; ++r) {
    const int64_t len = a.lens[r], add = a.add[r];
    const int64_t held = (len + bs - 1) / bs;
    misfit |= len < 0 || held > a.width;
    if (add < 0) {
      backs += held;
    } else {
      const int64_t need = (len + add + bs - 1) / bs;
      misfit |= need > a.width;
      tokens += add;
      wants += need - held;
    }
  }
  misfit = __syncthreads_or(misfit);
  int64_t all_tokens, all_wants, all_backs;
  int64_t t = scan256(tokens, wave_sums, &all_tokens);
  int64_t w = scan256(wants, wave_sums, &all_wants);
  int64_t b = scan256(backs, wave_sums, &all_backs);

  const int64_t had = a.num_free[0];
  int64_t status = 0;
  if (misfit) status = -1;
  else if (all_tokens > a.slot_count) status = -2;
  else if (had < 0 || had > a.capacity || had + all_backs > a.capacity) status = -3;
  else if (all_wants > had + all_backs) status = all_wants - had - all_backs;
  const bool ok = status == 0;

  if (ok) {  // every sum fits 32 bits: tokens <= slot_count, blocks <= capacity
    for (int r = r0; r < r1; ++r) {
      const int64_t len = a.lens[r], add = a.add[r], held = (len + bs - 1) / bs;
      start[r] = (int32_t)t, want[r] = (int32_t)w, back[r] = (int32_t)b;
      if (add < 0) b += held;
      else t += add, w += (len + add + bs - 1) / bs - held;
    }
    if (threadIdx.x == 0) start[n] = (int32_t)all_tokens, want[n] = (int32_t)all_wants, back[n] = (int32_t)all_backs;
  }
  __syncthreads();

  const int64_t top = had + all_backs;  // height of the stack before the pops
  // entry p of the stack: the free list, above it what ended requests give back
  auto stack = [&](int64_t p) -> int32_t {
    if (p < had) return a.free[p];
    const int r = last_at_most(back, n, (int32_t)(p - had));
    return a.table[(int64_t)r * a.width + (p - had - back[r])];
  };
  // block `column` of request r, old or newly taken
  auto block_of = [&](int r, int64_t column, int64_t held) -> int32_t {
    return column < held ? a.table[(int64_t)r * a.width + column] : stack(top - 1 - (want[r] + column - held));
  };

  const int64_t first = (int64_t)blockIdx.x * kPlanThreads + threadIdx.x, step = (int64_t)gridDim.x * kPlanThreads;
  for (int64_t i = first; i < a.slot_count; i += step) {
    int64_t slot = -1;
    if (ok && i < all_tokens) {
      const int r = last_at_most(start, n, (int32_t)i);
      const int64_t len = a.lens[r], place = len + (i - start[r]);
      const int64_t block = block_of(r, place / bs, (len + bs - 1) / bs);
      if (block >= 0) slot = block * bs + place % bs;
    }
    a.slots[i] = slot;
  }
  for (int64_t i = first; i < (int64_t)n * a.width; i += step) {
    const int r = (int)(i / a.width);
    const int64_t column = i - (int64_t)r * a.width;
    int32_t v = a.table[i];
    if (ok) {
      const int64_t len = a.lens[r], add = a.add[r], held = (len + bs - 1) / bs;
      if (add < 0) v = -1;
      else if (column >= held && column < (len + add + bs - 1) / bs) v = block_of(r, column, held);
    }
    a.table_out[i] = v;
  }
  const int64_t left = ok ? top - all_wants : had;
  for (int64_t i = first; i < a.capacity; i += step)
    a.free_out[i] = !ok ? a.free[i] : i < left ? stack(i) : -1;
  for (int64_t i = first; i <= n; i += step) {
    a.start[i] = ok ? start[i] : 0;
    if (i < n) {
      const int32_t len = a.lens[i], add = a.add[i];
      a.lens_out[i] = !ok ? len : add < 0 ? 0 : len + add;
    }
  }
  if (first == 0) {
    a.num_free_out[0] = (int32_t)left;
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
  CTMI_REQUIRE(width < (1ll << 31) && free_capacity < (1ll << 31) && slot_count < (1ll << 31), CTMI_ERR_UNSUPPORTED,
               "table columns, free blocks and slots must each stay below 2^31");
  CTMI_REQUIRE(block_size >= 1, CTMI_ERR_VALUE, "block_size must be at least 1, got %d", block_size);
  CTMI_REQUIRE(num_free && query_start && num_free_out && status &&
                   (requests == 0 || (seq_lens && new_tokens && block_table && seq_lens_out && table_out)) &&
                   (free_capacity == 0 || (free_blocks && free_out)) && (slot_count == 0 || slots),
               CTMI_ERR_VALUE, "NULL tensor");
  PlanArgs a{seq_lens, new_tokens, block_table, free_blocks, num_free, width, free_capacity, slot_count,
             (int32_t)requests, block_size, seq_lens_out, query_start, slots, table_out, free_out,
             num_free_out, status};
  // eight outputs a thread: fewer workgroups repeat the scan less, more of them hide its
  // latency no better
  const int64_t most = slot_count > requests * width ? slot_count : requests * width;
  int64_t grid = cdiv(most > free_capacity ? most : free_capacity, (int64_t)kPlanThreads * 8);
  if (grid < 1) grid = 1;
  if (grid > 1024) grid = 1024;
  const size_t lds = (size_t)(requests + 1) * 3 * sizeof(int32_t);
  kv_plan_kernel<<<dim3((unsigned)grid), dim3(kPlanThreads), lds, (hipStream_t)stream>>>(a);
  return check_launch("kv_plan");
}
