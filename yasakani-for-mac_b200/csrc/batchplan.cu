// Blocks, slots and positions of one step of a batch, from the request lengths alone.
//
// The cache is paged: a request's own rows (those after the shared prefix) lie in blocks of
// block_size places, named in order by its row of the block tables; unused block numbers
// lie on a stack (the pool). For request i with length len (rows in the cache, the prefix
// counted), P the prefix length, bs the block size and new its new tokens of this step:
//   rows = max(len - P, 0), held = ceil(rows / bs)
//   new < 0: the request has ended. Its held blocks go onto the stack, its length becomes 0.
//   new > 0: it is served if the blocks of rows + new fit its table row, and the blocks and
//     tokens of it and of all such requests before it fit the stack (with what the ended
//     requests gave back) and the step; else it waits (no tokens, its length stays). Its
//     missing blocks are taken from the top of the stack, requests in order.
// Every served request's token t gets its position P + rows + t, its request, and the slot
// (block * bs + place) its K/V row goes to. The served requests are a prefix of those that
// fit their tables, so sums over all that fit give the served ones' places: no second pass.
//
// What bounds it: latency at a decode step (a few KB move); at a large prompt step the 16
// bytes written per token. So one launch: every CTA forms the same three prefix sums (blocks
// given back, blocks needed, tokens) over the whole batch (at most 4096 requests, from L2)
// in shared memory, then takes its share of the tokens and of the blocks given back, and no
// CTA waits for another. A token finds its request by a binary search in shared memory; the
// token in a fresh block's first place writes the table entry (a fresh block always starts
// with a new token). Nothing that any CTA reads is written in the launch: the lengths and the
// stack's count go to other arrays, fresh table entries are never read, and the stack is
// written only above its old count, read only below it (blocks given back in this step and
// taken in it are read from the ended request's table row).
#include <algorithm>

#include "common.cuh"

namespace yskn {

constexpr int PLAN_THREADS = 512;
constexpr int PLAN_WARPS = PLAN_THREADS / 32;

struct PlanParams {
  const int32_t* lens;
  const int32_t* new_lens;
  int32_t* tables;  // [batch][table_stride]
  int64_t table_stride;
  int table_width;
  int32_t* pool;
  int pool_capacity;
  const int32_t* free_count;
  int batch, block_size, prefix_len, max_tokens;
  int32_t* lens_out;
  int32_t* free_out;
  int32_t* starts;     // [batch + 1]
  int64_t* slots;      // [max_tokens]
  int32_t* positions;  // [max_tokens]
  int32_t* requests;   // [max_tokens]
  unsigned* err;
};

struct Sum3 {
  long long back, need, tokens;
};
__device__ __forceinline__ Sum3 operator+(Sum3 a, Sum3 b) {
  return {a.back + b.back, a.need + b.need, a.tokens + b.tokens};
}

struct PlanRequest {
  int len, rows, held, fresh, n, back;  // n: new tokens if its table row can hold them, else 0
  bool ended, too_long;
};

__device__ __forceinline__ PlanRequest plan_request(const PlanParams& p, int i) {
  PlanRequest r{};
  const int len = __ldg(p.lens + i), n = __ldg(p.new_lens + i);
  const unsigned bs = p.block_size;
  r.len = len;
  r.rows = len > p.prefix_len ? len - p.prefix_len : 0;
  r.held = (int)((unsigned)r.rows / bs + ((unsigned)r.rows % bs != 0));
  r.ended = n < 0;
  r.too_long = r.held > p.table_width;
  if (r.ended) r.back = min(r.held, p.table_width);
  if (n > 0 && r.rows <= INT32_MAX - n) {
    const unsigned end = (unsigned)(r.rows + n);
    const int total = (int)(end / bs + (end % bs != 0));
    if (total <= p.table_width) {
      r.n = n;
      r.fresh = total - r.held;
    }
  }
  return r;
}

// Last index i in [0, n) with a[i] <= v (a ascending, a[0] <= v).
__device__ __forceinline__ int last_at_most(const int* a, int n, int v) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a[mid] <= v) lo = mid;
    else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(PLAN_THREADS) batch_plan_kernel(const __grid_constant__ PlanParams p) {
  extern __shared__ int s_plan[];
  const int B = p.batch;
  int* s_start = s_plan;               // [B + 1] tokens, then first token, of each request
  int* s_back = s_start + B + 1;       // [B + 1] blocks given back, then those before each request
  int* s_need = s_back + B + 1;        // [B] fresh blocks, then those taken before each request
  int* s_rows = s_need + B;            // [B]
  __shared__ Sum3 s_warp[PLAN_WARPS];
  __shared__ Sum3 s_served;            // sums over the served requests
  __shared__ int s_any_long;
  pdl_begin();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int count = __ldg(p.free_count);
  if (tid == 0) s_served = {0, 0, 0}, s_any_long = 0;
  __syncthreads();
  for (int i = tid; i < B; i += PLAN_THREADS) {
    const PlanRequest r = plan_request(p, i);
    s_start[i] = r.n;
    s_back[i] = r.back;
    s_need[i] = r.fresh;
    s_rows[i] = r.rows;
    if (r.too_long) s_any_long = 1;
    if (blockIdx.x == 0) p.lens_out[i] = r.ended ? 0 : r.len;  // served ones below
  }
  __syncthreads();
  const int per = (B + PLAN_THREADS - 1) / PLAN_THREADS;
  const int i0 = min(B, tid * per), i1 = min(B, i0 + per);
  Sum3 mine{0, 0, 0};
  for (int i = i0; i < i1; ++i) mine = mine + Sum3{s_back[i], s_need[i], s_start[i]};
  Sum3 incl = mine;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const Sum3 o{__shfl_up_sync(0xffffffffu, incl.back, off), __shfl_up_sync(0xffffffffu, incl.need, off),
                 __shfl_up_sync(0xffffffffu, incl.tokens, off)};
    if (lane >= off) incl = incl + o;
  }
  if (lane == 31) s_warp[warp] = incl;
  __syncthreads();
  Sum3 before{incl.back - mine.back, incl.need - mine.need, incl.tokens - mine.tokens};
  long long back_total = 0;
  for (int w = 0; w < PLAN_WARPS; ++w) {
    const Sum3 o = s_warp[w];
    if (w < warp) before = before + o;
    back_total += o.back;
  }
  const int free0 = min(max(count, 0), p.pool_capacity);
  const long long have = free0 + back_total;
  // Served requests: both sums only grow, so the last served one's end is their total.
  Sum3 run = before, end{0, 0, 0};
  for (int i = i0; i < i1; ++i) {
    const int n = s_start[i];
    const Sum3 next = run + Sum3{s_back[i], s_need[i], n};
    const bool served = n > 0 && next.need <= have && next.tokens <= p.max_tokens;
    if (served) end = next;
    s_back[i] = (int)run.back;
    s_need[i] = (int)min(run.need, (long long)INT32_MAX);
    s_start[i] = (int)min(run.tokens, (long long)INT32_MAX);  // cut at the served total below
    if (served && blockIdx.x == 0)
      p.lens_out[i] = (int)min((long long)max(__ldg(p.lens + i), p.prefix_len) + n, (long long)INT32_MAX);
    run = next;
  }
  if (end.tokens > 0) {
    atomicMax(reinterpret_cast<unsigned long long*>(&s_served.need), (unsigned long long)end.need);
    atomicMax(reinterpret_cast<unsigned long long*>(&s_served.tokens), (unsigned long long)end.tokens);
  }
  __syncthreads();
  const int total = (int)s_served.tokens;
  const int left = (int)min(have - s_served.need, (long long)INT32_MAX);
  for (int i = tid; i <= B; i += PLAN_THREADS) {
    const int st = i < B ? min(s_start[i], total) : total;
    s_start[i] = st;
    if (i == B) s_back[B] = (int)back_total;
    if (blockIdx.x == 0) p.starts[i] = st;
  }
  if (blockIdx.x == 0 && tid == 0) {
    *p.free_out = left;
    if (s_any_long || count != free0 || have > p.pool_capacity) raise_device_error(p.err, DERR_RANGE);
  }
  __syncthreads();

  // Block number at place v of the stack with what came back on top.
  auto stack_at = [&](int v) -> int {
    if (v < free0) return __ldg(p.pool + v);
    const int k = v - free0;
    const int g = last_at_most(s_back, B, k);  // requests that give nothing share a start with the next one
    return p.tables[(int64_t)g * p.table_stride + (k - s_back[g])];
  };
  const int first = blockIdx.x * PLAN_THREADS + tid, step = gridDim.x * PLAN_THREADS;
  for (int v = free0 + first; v < min(left, p.pool_capacity); v += step) p.pool[v] = stack_at(v);
  for (int t = first; t < p.max_tokens; t += step) {
    if (t >= total) {
      p.slots[t] = -1;
      p.positions[t] = -1;
      p.requests[t] = -1;
      continue;
    }
    const int i = last_at_most(s_start, B, t);
    const int rows = s_rows[i], row = rows + (t - s_start[i]);
    const unsigned bs = p.block_size;
    const int held = (int)((unsigned)rows / bs + ((unsigned)rows % bs != 0));
    const int b = (int)((unsigned)row / bs), place = row - b * (int)bs;
    int32_t* entry = p.tables + (int64_t)i * p.table_stride + b;
    int block;
    if (b < held) {
      block = *entry;
    } else {
      block = stack_at((int)(have - 1 - s_need[i]) - (b - held));
      if (place == 0) *entry = block;
    }
    p.slots[t] = (int64_t)block * p.block_size + place;
    p.positions[t] = p.prefix_len + row;
    p.requests[t] = i;
  }
}

}  // namespace yskn

using namespace yskn;

extern "C" YSKN_B200_API int yskn_b200_batch_plan(const yskn_b200_batch_plan_args* args, void* stream) {
  if (!args) return fail(YSKN_EINVAL, "batch_plan: null argument");
  const yskn_b200_batch_plan_args& a = *args;
  if (!a.lens || !a.new_lens || !a.block_tables || !a.pool || !a.free || !a.lens_out || !a.free_out || !a.starts ||
      (a.max_tokens > 0 && (!a.slots || !a.positions || !a.requests)))
    return fail(YSKN_EINVAL, "batch_plan: null argument");
  if (a.batch < 1 || a.batch > YSKN_PLAN_MAX_BATCH || a.block_size < 1 || a.prefix_len < 0 || a.table_width < 1 ||
      (a.batch > 1 && a.table_stride < a.table_width) || a.pool_capacity < 1 || a.max_tokens < 0)
    return fail(YSKN_EINVAL, "batch_plan: batch outside 1..4096, or a size or stride out of range");
  if (a.lens_out == a.lens || a.free_out == a.free)
    return fail(YSKN_EINVAL, "batch_plan: the new lengths and the new count need arrays of their own");
  PlanParams p{a.lens, a.new_lens, a.block_tables, a.table_stride, a.table_width, a.pool, a.pool_capacity, a.free,
               a.batch, a.block_size, a.prefix_len, a.max_tokens, a.lens_out, a.free_out, a.starts, a.slots,
               a.positions, a.requests, device_error_word()};
  const size_t smem = (4 * (size_t)a.batch + 2) * sizeof(int);
  static SmemOptIn opt_in;
  if (cudaError_t e = opt_in(batch_plan_kernel, (4 * YSKN_PLAN_MAX_BATCH + 2) * sizeof(int)))
    return cuda_fail(e, "batch_plan_kernel attributes");
  // Four tokens a thread, at most two CTAs an SM: more only repeat the prefix sums.
  const int grid = (int)std::min<int64_t>(ceil_div(std::max(a.max_tokens, 1), 4 * PLAN_THREADS), 296);
  return cuda_fail(launch_pdl(batch_plan_kernel, grid, PLAN_THREADS, smem, reinterpret_cast<cudaStream_t>(stream), p),
                   "batch_plan_kernel");
}
