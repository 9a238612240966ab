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
// CTA waits for another. A warp's tokens are adjacent: it finds the first one's request by a
// search of 32 probes a round and walks on from there; the token in a fresh block's first place
// writes the table entry (a fresh block always starts with a new token). Nothing that any CTA reads is written in the launch: the lengths and the
// stack's count go to other arrays, fresh table entries are never read, and the stack is
// written only above its old count, read only below it (blocks given back in this step and
// taken in it are read from the ended request's table row).
#include <algorithm>

#include "common.cuh"

namespace yskn {

constexpr int PLAN_THREADS = 512;
constexpr int PLAN_WARPS = PLAN_THREADS / 32;
constexpr int PLAN_PER = YSKN_PLAN_MAX_BATCH / PLAN_THREADS;  // requests of a thread, at most
// A thread's requests are adjacent: a place in 8 left free keeps its stores off each other's banks.
__host__ __device__ constexpr int plan_at(int i) { return i + (i >> 3); }

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
  int warp_tokens;  // adjacent tokens of a warp, a multiple of 32
  int32_t* lens_out;
  int32_t* free_out;
  int32_t* starts;     // [batch + 1]
  int64_t* slots;      // [max_tokens]
  int32_t* positions;  // [max_tokens]
  int32_t* requests;   // [max_tokens]
  unsigned* err;
};

// Sums that stop at 2^31 - 1, which no array holds.
struct Sum3 {
  unsigned back, need, tokens;
};
__device__ __forceinline__ unsigned plan_sum(unsigned a, unsigned b) { return min(a + b, (unsigned)INT32_MAX); }
__device__ __forceinline__ Sum3 operator+(Sum3 a, Sum3 b) {
  return {plan_sum(a.back, b.back), plan_sum(a.need, b.need), plan_sum(a.tokens, b.tokens)};
}

struct PlanRequest {
  int len, rows, held, fresh, n, back;  // n: new tokens if its table row can hold them, else 0
  bool ended, too_long;
};

// From r.len and the new tokens in r.n.
__device__ __forceinline__ void plan_request(const PlanParams& p, PlanRequest& r) {
  const unsigned bs = p.block_size;
  const int n = r.n;
  r.n = 0;
  r.rows = r.len > p.prefix_len ? r.len - p.prefix_len : 0;
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
}

// Last index i in [lo, hi) with a[plan_at(i)] <= v (ascending, the first <= v).
__device__ __forceinline__ int last_at_most(const int* a, int lo, int hi, int v) {
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a[plan_at(mid)] <= v) lo = mid;
    else hi = mid;
  }
  return lo;
}
// The same for a whole warp's v: 32 probes a round.
__device__ __forceinline__ int warp_last_at_most(const int* a, int n, int v) {
  const int lane = threadIdx.x & 31;
  int lo = 0;
  while (n > 1) {
    const int step = (n + 31) >> 5, at = lane * step;
    const unsigned below = __ballot_sync(0xffffffffu, at < n && a[plan_at(lo + min(at, n - 1))] <= v);
    const int k = __popc(below) - 1;
    lo += k * step;
    n = min(step, n - k * step);
  }
  return lo;
}

__global__ void __launch_bounds__(PLAN_THREADS, 2) batch_plan_kernel(const __grid_constant__ PlanParams p) {
  extern __shared__ int s_plan[];
  const int B = p.batch;
  const int room = plan_at(B) + 1;
  int* s_start = s_plan;         // [B + 1] first token of each request
  int* s_back = s_start + room;  // [B + 1] blocks given back before each request
  int* s_need = s_back + room;   // [B] fresh blocks taken before each request
  int* s_rows = s_need + room;   // [B]
  __shared__ Sum3 s_warp[PLAN_WARPS];
  __shared__ uint2 s_served[PLAN_WARPS];  // need and tokens up to each warp's last served request
  __shared__ int s_any_long;
  pdl_begin();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int count = __ldg(p.free_count);
  if (tid == 0) s_any_long = 0;
  const int per = (B + PLAN_THREADS - 1) / PLAN_THREADS, i0 = tid * per;
  PlanRequest r[PLAN_PER];
#pragma unroll
  for (int k = 0; k < PLAN_PER; ++k) {
    r[k] = PlanRequest{};
    if (k < per && i0 + k < B) r[k].len = __ldg(p.lens + i0 + k), r[k].n = __ldg(p.new_lens + i0 + k);
  }
  Sum3 mine{0, 0, 0};
  bool too_long = false;
#pragma unroll
  for (int k = 0; k < PLAN_PER; ++k) {
    if (k >= per) break;
    plan_request(p, r[k]);
    mine = mine + Sum3{(unsigned)r[k].back, (unsigned)r[k].fresh, (unsigned)r[k].n};
    too_long |= r[k].too_long;
  }
  Sum3 incl = mine;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const Sum3 o{__shfl_up_sync(0xffffffffu, incl.back, off), __shfl_up_sync(0xffffffffu, incl.need, off),
                 __shfl_up_sync(0xffffffffu, incl.tokens, off)};
    if (lane >= off) incl = incl + o;
  }
  if (lane == 31) s_warp[warp] = incl;
  __syncthreads();
  if (too_long) s_any_long = 1;
  // a thread's own part taken off again: exact unless a sum has stopped, and then nothing fits
  Sum3 before{incl.back - mine.back, incl.need - mine.need, incl.tokens - mine.tokens};
  unsigned back_total = 0;
#pragma unroll
  for (int w = 0; w < PLAN_WARPS; ++w) {
    const Sum3 o = s_warp[w];
    if (w < warp) before = before + o;
    back_total = plan_sum(back_total, o.back);
  }
  const int free0 = min(max(count, 0), p.pool_capacity);
  const unsigned have = plan_sum(free0, back_total);
  // Served requests: both sums only grow, so the last served one's end is their total.
  Sum3 run = before, end{0, 0, 0};
#pragma unroll
  for (int k = 0; k < PLAN_PER; ++k) {
    const int i = i0 + k;
    if (k >= per || i >= B) break;
    const Sum3 next = run + Sum3{(unsigned)r[k].back, (unsigned)r[k].fresh, (unsigned)r[k].n};
    const bool served = r[k].n > 0 && next.need <= have && next.tokens <= (unsigned)p.max_tokens;
    if (served) end = next;
    s_back[plan_at(i)] = (int)run.back;
    s_need[plan_at(i)] = (int)run.need;
    s_rows[plan_at(i)] = r[k].rows;
    s_start[plan_at(i)] = (int)run.tokens;  // cut at the served total below
    if (blockIdx.x == 0)
      p.lens_out[i] = r[k].ended ? 0
                      : served   ? (int)min((long long)max(r[k].len, p.prefix_len) + r[k].n, (long long)INT32_MAX)
                                 : r[k].len;
    run = next;
  }
  const unsigned warp_need = __reduce_max_sync(0xffffffffu, end.need);
  const unsigned warp_tokens = __reduce_max_sync(0xffffffffu, end.tokens);
  if (lane == 0) s_served[warp] = make_uint2(warp_need, warp_tokens);
  __syncthreads();
  unsigned taken = 0, tokens = 0;
#pragma unroll
  for (int w = 0; w < PLAN_WARPS; ++w) taken = max(taken, s_served[w].x), tokens = max(tokens, s_served[w].y);
  const int total = (int)tokens, left = (int)(have - taken);
  for (int i = tid; i <= B; i += PLAN_THREADS) {
    const int st = i < B ? min(s_start[plan_at(i)], total) : total;
    s_start[plan_at(i)] = st;
    if (i == B) s_back[plan_at(B)] = (int)back_total;
    if (blockIdx.x == 0) p.starts[i] = st;
  }
  if (blockIdx.x == 0 && tid == 0) {
    *p.free_out = left;
    if (s_any_long || count != free0 || have > (unsigned)p.pool_capacity) raise_device_error(p.err, DERR_RANGE);
  }
  __syncthreads();

  // Block number at place v of the stack with what came back on top; the givers lie in [lo, hi).
  auto stack_at = [&](int v, int lo, int hi) -> int {
    if (v < free0) return __ldg(p.pool + v);
    const int k = v - free0;
    const int g = last_at_most(s_back, lo, hi, k);  // requests that give nothing share a start with the next one
    return p.tables[(int64_t)g * p.table_stride + (k - s_back[plan_at(g)])];
  };
  const int first = blockIdx.x * PLAN_THREADS + tid, step = gridDim.x * PLAN_THREADS;
  for (int v = free0 + first; v < min(left, p.pool_capacity); v += step) p.pool[v] = stack_at(v, 0, B);
  const unsigned bs = p.block_size;
  // A warp's tokens are adjacent, 32 at a time: their requests lie at or after the last ones', and
  // the givers of the blocks they take (the stack's places fall from token to token) at or before.
  const int t_first = (blockIdx.x * PLAN_WARPS + warp) * p.warp_tokens;
  const int t_end = min(t_first + p.warp_tokens, p.max_tokens);
  int lo = -1, g_hi = -1;
  for (int t0 = t_first; t0 < t_end; t0 += 32) {
    const int t = t0 + lane;
    if (t0 >= total) {
      if (t < t_end) p.slots[t] = -1, p.positions[t] = -1, p.requests[t] = -1;
      continue;
    }
    const int last = min(t0 + 31, total - 1), mine = min(t, last);
    if (lo < 0) lo = warp_last_at_most(s_start, B, t0);
    int hi = lo;  // the last token's request
    for (unsigned more = ~0u; more == ~0u; hi += __popc(more))
      more = __ballot_sync(0xffffffffu, hi + 1 + lane < B && s_start[plan_at(min(hi + 1 + lane, B))] <= last);
    const int i = last_at_most(s_start, lo, hi + 1, mine);
    lo = hi;
    const int rows = s_rows[plan_at(i)], row = rows + (mine - s_start[plan_at(i)]);
    const int held = (int)((unsigned)rows / bs + ((unsigned)rows % bs != 0));
    const int b = (int)((unsigned)row / bs), place = row - b * (int)bs;
    const bool fresh = b >= held;
    const int v = (int)(have - 1 - s_need[plan_at(i)]) - (b - held);  // place of a fresh block in the stack
    const int v_hi = __reduce_max_sync(0xffffffffu, fresh ? v - free0 : -1);
    int g_lo = 0;
    if (v_hi >= 0) {  // some come from ended requests
      const int v_lo = __reduce_min_sync(0xffffffffu, fresh ? max(v - free0, 0) : INT32_MAX);
      if (g_hi < 0) g_hi = warp_last_at_most(s_back, B, v_hi);
      g_lo = g_hi;
      for (unsigned more = ~0u; more == ~0u; g_lo -= __popc(more))
        more = __ballot_sync(0xffffffffu, g_lo - lane >= 0 && s_back[plan_at(max(g_lo - lane, 0))] > v_lo);
    }
    int32_t* entry = p.tables + (int64_t)i * p.table_stride + b;
    if (t <= last) {
      int block;
      if (fresh) {
        block = stack_at(v, g_lo, g_hi + 1);
        if (place == 0) *entry = block;
      } else {
        block = *entry;
      }
      p.slots[t] = (int64_t)block * p.block_size + place;
      p.positions[t] = p.prefix_len + row;
      p.requests[t] = i;
    } else if (t < t_end) {
      p.slots[t] = -1, p.positions[t] = -1, p.requests[t] = -1;
    }
    if (v_hi >= 0) g_hi = g_lo;
    __syncwarp();
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
  if (a.max_tokens > 1 << 30)  // the last warp's places stay below 2^31
    return fail(YSKN_EINVAL, "batch_plan: more than 2^30 tokens");
  if (a.lens_out == a.lens || a.free_out == a.free)
    return fail(YSKN_EINVAL, "batch_plan: the new lengths and the new count need arrays of their own");
  PlanParams p{a.lens, a.new_lens, a.block_tables, a.table_stride, a.table_width, a.pool, a.pool_capacity, a.free,
               a.batch, a.block_size, a.prefix_len, a.max_tokens, 0, a.lens_out, a.free_out, a.starts, a.slots,
               a.positions, a.requests, device_error_word()};
  const size_t smem = 4 * (size_t)(plan_at(a.batch) + 1) * sizeof(int);
  static SmemOptIn opt_in;
  if (cudaError_t e = opt_in(batch_plan_kernel, 4 * (plan_at(YSKN_PLAN_MAX_BATCH) + 1) * sizeof(int)))
    return cuda_fail(e, "batch_plan_kernel attributes");
  // A warp's tokens: at most two CTAs an SM (more only repeat the prefix sums), 32 or more a warp.
  p.warp_tokens = (int)(ceil_div(ceil_div(std::max(a.max_tokens, 1), 2 * 148 * PLAN_WARPS), 32) * 32);
  const int grid = (int)ceil_div(std::max(a.max_tokens, 1), (int64_t)p.warp_tokens * PLAN_WARPS);
  return cuda_fail(launch_pdl(batch_plan_kernel, grid, PLAN_THREADS, smem, reinterpret_cast<cudaStream_t>(stream), p),
                   "batch_plan_kernel");
}
