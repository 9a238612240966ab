// Which rows each request of a batch keeps and whose it continues: lengths, block tables, the pool of
// unused blocks, and the list of blocks that have to be copied.
//
// Request i becomes the first k_i = min(keep_i, len of s_i) rows of request s_i, c_i blocks of own rows
// (those after the shared prefix). Of the requests with source j, the heir of j is the one of the
// largest k (the lowest of several): it goes on in j's first c blocks. The others need c fresh
// blocks each and a copy of j's. The heir has at least as many blocks of j as any of them, so what is
// copied is never among the blocks that go back to the pool and may be written by the same copies.
// Blocks given back go on top of the stack, fresh ones come from its top, as in batchplan.cu: the places
// of all are sums over the requests before.
//
// What bounds it: latency; for many long requests the tables' bytes. One launch: every CTA forms the
// heirs (atomic maxima of (k, i) in shared memory: no two are equal, so the order changes nothing) and the
// sums over the whole batch, then its warps take pieces of 64 entries of the new tables, and of the
// pool's and the list's ends. Nothing that any CTA reads is written: the stack is read below its old count
// and written above it, the tables and lengths go to other arrays. 64 requests that keep fewer rows 3.5 us in a captured
// graph, 1024 of which a third continue others 6.6 (with a division for each request's blocks, where a shift does, 7.2);
// calls by themselves, which the host bounds, 6.3 and 8.5.
#include <algorithm>

#include "common.cuh"

namespace yskn {

constexpr int EDIT_THREADS = 512;
constexpr int EDIT_WARPS = EDIT_THREADS / 32;
constexpr int EDIT_PER = YSKN_PLAN_MAX_BATCH / EDIT_THREADS;  // requests of a thread, at most
// Table entries of a warp at a time. 128, 64, 32: 1024 requests of up to 63 own blocks 7.2, 6.6, 7.0 us, 256 of up to
// 250 6.6, 5.3, 4.8, 4096 of up to 63 20.2, 21.5, 20.8.
constexpr int EDIT_PIECE = 64;

struct EditParams {
  const int32_t *lens, *keep, *source;
  const int32_t* tables;
  int64_t table_stride;
  int32_t* tables_out;
  int64_t out_stride;
  int32_t* pool;
  const int32_t* free_count;
  int32_t *lens_out, *free_out;
  int32_t* copies;
  int64_t copies_stride;
  int32_t* n_copies;
  int batch, prefix_len, table_width, pool_capacity, max_copies;
  unsigned block_size;
  int block_shift;  // of a power of two, else -1
  unsigned* err;
};

// Sums that stop at 2^31 - 1, which no array holds.
__device__ __forceinline__ unsigned edit_sum(unsigned a, unsigned b) { return min(a + b, (unsigned)INT32_MAX); }
// Blocks of a request's own rows, and as many as its table has.
__device__ __forceinline__ int edit_asked(const EditParams& p, int len) {
  const unsigned rows = len > p.prefix_len ? len - p.prefix_len : 0;
  return p.block_shift >= 0 ? (int)((rows + (p.block_size - 1)) >> p.block_shift)
                            : (int)(rows / p.block_size + (rows % p.block_size != 0));
}
__device__ __forceinline__ int edit_blocks(const EditParams& p, int len) {
  return min(edit_asked(p, len), p.table_width);
}
// Last index i of n with a[i] <= v (ascending, the first <= v).
__device__ __forceinline__ int edit_last(const int* a, int n, int v) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a[mid] <= v) lo = mid;
    else hi = mid;
  }
  return lo;
}

template <bool FORK>
__global__ void __launch_bounds__(EDIT_THREADS) batch_edit_kernel(const __grid_constant__ EditParams p) {
  extern __shared__ __align__(16) uint8_t s_edit[];
  const int B = p.batch;
  unsigned long long* s_heir = reinterpret_cast<unsigned long long*>(s_edit);  // [B] (k + 1, ~i) of each one's heir
  int* s_back = reinterpret_cast<int*>(s_edit + (FORK ? 8 * (size_t)B : 0));   // [B] blocks given back before
  int* s_stay = s_back + B;                                                    // [B] blocks that stay
  int* s_need = s_stay + B;                                                    // [B] fresh blocks before
  int* s_kept = s_need + B;                                                    // [B] blocks of the new one
  int* s_from = s_kept + B;  // [B] source; ~source for one that gets copies; B: nothing
  __shared__ uint2 s_warp[EDIT_WARPS];
  __shared__ unsigned s_served[EDIT_WARPS];
  __shared__ int s_wrong;
  pdl_begin();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (B + EDIT_THREADS - 1) / EDIT_THREADS, i0 = min(B, tid * per), i1 = min(B, i0 + per);
  const int count = __ldg(p.free_count);
  if (tid == 0) s_wrong = 0;
  int len[EDIT_PER], source[EDIT_PER], held[EDIT_PER];  // the new length; where it comes from; blocks so far
  if (FORK)
    for (int i = tid; i < B; i += EDIT_THREADS) s_heir[i] = 0;
  __syncthreads();
  bool wrong = false;
#pragma unroll
  for (int k = 0; k < EDIT_PER; ++k) {
    const int i = i0 + k;
    len[k] = 0, source[k] = -1;
    if (k >= per || i >= i1) continue;
    const int j = FORK ? __ldg(p.source + i) : i;
    wrong |= j >= B;
    if (j < 0 || j >= B) continue;
    source[k] = j;
    len[k] = max(min(__ldg(p.keep + i), __ldg(p.lens + j)), 0);
    if (FORK) atomicMax(s_heir + j, (unsigned long long)(len[k] + 1ll) << 32 | ~(unsigned)i);
  }
  __syncthreads();
  uint2 mine = make_uint2(0, 0);  // blocks given back, fresh ones
#pragma unroll
  for (int k = 0; k < EDIT_PER; ++k) {
    const int i = i0 + k;
    if (k >= per || i >= i1) continue;
    const int kept = edit_blocks(p, len[k]), asked = edit_asked(p, __ldg(p.lens + i));
    held[k] = min(asked, p.table_width);
    int stay = kept, need = 0;
    if (FORK) {
      const unsigned long long heir = s_heir[i];
      stay = heir ? edit_blocks(p, (int)((heir >> 32) - 1)) : 0;
      if (source[k] >= 0 && (unsigned)s_heir[source[k]] != ~(unsigned)i) need = kept;
    }
    wrong |= asked > p.table_width;
    s_stay[i] = stay;
    s_kept[i] = kept;
    s_from[i] = source[k] < 0 ? B : need ? ~source[k] : source[k];
    mine.x = edit_sum(mine.x, held[k] - stay);
    mine.y = edit_sum(mine.y, need);
  }
  uint2 incl = mine;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const unsigned x = __shfl_up_sync(0xffffffffu, incl.x, off), y = __shfl_up_sync(0xffffffffu, incl.y, off);
    if (lane >= off) incl.x = edit_sum(incl.x, x), incl.y = edit_sum(incl.y, y);
  }
  if (lane == 31) s_warp[warp] = incl;
  __syncthreads();
  if (wrong) s_wrong = 1;
  // a thread's own part taken off again: exact unless a sum has stopped, and then nothing fits
  uint2 run = make_uint2(incl.x - mine.x, incl.y - mine.y);
  unsigned back_total = 0;
#pragma unroll
  for (int w = 0; w < EDIT_WARPS; ++w) {
    const uint2 o = s_warp[w];
    if (w < warp) run.x = edit_sum(run.x, o.x), run.y = edit_sum(run.y, o.y);
    back_total = edit_sum(back_total, o.x);
  }
  const int free0 = min(max(count, 0), p.pool_capacity);
  const unsigned have = edit_sum(free0, back_total), room = FORK ? min(have, (unsigned)p.max_copies) : have;
  unsigned served = 0;  // fresh blocks up to the last served request: the sums only grow
#pragma unroll
  for (int k = 0; k < EDIT_PER; ++k) {
    const int i = i0 + k;
    if (k >= per || i >= i1) continue;
    const int kept = s_kept[i], from = s_from[i];
    const unsigned need = FORK && from < 0 ? kept : 0, after = edit_sum(run.y, need);
    s_back[i] = (int)run.x;
    s_need[i] = (int)run.y;
    if (after <= room) served = max(served, after);
    else if (need > 0) s_from[i] = B, len[k] = 0;  // it ends
    run.x = edit_sum(run.x, held[k] - s_stay[i]);
    run.y = after;
    if (blockIdx.x == 0) p.lens_out[i] = len[k];
  }
  served = __reduce_max_sync(0xffffffffu, served);
  if (lane == 0) s_served[warp] = served;
  __syncthreads();
  unsigned taken = 0;
#pragma unroll
  for (int w = 0; w < EDIT_WARPS; ++w) taken = max(taken, s_served[w]);
  const int left = (int)(have - taken);
  if (blockIdx.x == 0 && tid == 0) {
    *p.free_out = left;
    if (FORK) *p.n_copies = (int)taken;
    if (s_wrong || count != free0 || have > (unsigned)p.pool_capacity) raise_device_error(p.err, DERR_RANGE);
  }

  // Block number at place v of the stack with what came back on top.
  auto stack_at = [&](int v) -> int {
    if (v < free0) return __ldg(p.pool + v);
    const int k = v - free0, g = edit_last(s_back, B, k);  // one that gives nothing shares a start with the next
    return __ldg(p.tables + (int64_t)g * p.table_stride + min(s_stay[g] + (k - s_back[g]), p.table_width - 1));
  };
  const int first = blockIdx.x * EDIT_THREADS + tid, step = gridDim.x * EDIT_THREADS;
  for (int v = free0 + first; v < min(left, p.pool_capacity); v += step) p.pool[v] = stack_at(v);
  if constexpr (FORK) {
    for (int e = (int)taken + first; e < p.max_copies; e += step) {
      p.copies[e] = p.copies[e + p.copies_stride] = -1;
      p.copies[e + 2 * p.copies_stride] = 0;
    }
    const int pieces = (p.table_width + EDIT_PIECE - 1) / EDIT_PIECE;
    const int64_t units = (int64_t)B * pieces;
    for (int64_t u = blockIdx.x * EDIT_WARPS + warp; u < units; u += gridDim.x * EDIT_WARPS) {
      const int i = (int)(u / pieces), b0 = (int)(u - (int64_t)i * pieces) * EDIT_PIECE;
      const int kept = s_kept[i], from = s_from[i];
      if (from == B || b0 >= kept) continue;
      const bool copy = from < 0;
      const int j = copy ? ~from : from;
      const int32_t* in = p.tables + (int64_t)j * p.table_stride;
      int32_t* out = p.tables_out + (int64_t)i * p.out_stride;
      int own = 0;
      if (copy) own = min(__ldg(p.keep + i), __ldg(p.lens + j)) - p.prefix_len;  // own rows of the new one
      for (int b = b0 + lane; b < min(b0 + EDIT_PIECE, kept); b += 32) {
        int block = __ldg(in + b);
        if (copy) {
          const int e = s_need[i] + b, fresh = stack_at((int)have - 1 - e);
          p.copies[e] = block;
          p.copies[e + p.copies_stride] = fresh;
          p.copies[e + 2 * p.copies_stride] = (int)min((int64_t)p.block_size, own - (int64_t)b * p.block_size);
          block = fresh;
        }
        out[b] = block;
      }
    }
  }
}

}  // namespace yskn

using namespace yskn;

extern "C" YSKN_B200_API int yskn_b200_batch_edit(const yskn_b200_batch_edit_args* args, void* stream) {
  if (!args) return fail(YSKN_EINVAL, "batch_edit: null argument");
  const yskn_b200_batch_edit_args& a = *args;
  const bool fork = a.source != nullptr;
  if (!a.lens || !a.keep || !a.block_tables || !a.pool || !a.free || !a.lens_out || !a.free_out ||
      (fork && (!a.tables_out || !a.copies || !a.n_copies)))
    return fail(YSKN_EINVAL, "batch_edit: null argument");
  if (a.batch < 1 || a.batch > YSKN_PLAN_MAX_BATCH || a.block_size < 1 || a.prefix_len < 0 || a.table_width < 1 ||
      (a.batch > 1 && a.table_stride < a.table_width) || a.pool_capacity < 1)
    return fail(YSKN_EINVAL, "batch_edit: batch outside 1..4096, or a size or stride out of range");
  if (fork && (a.max_copies < 1 || a.copies_stride < a.max_copies ||
               (a.batch > 1 && a.tables_out_stride < a.table_width)))
    return fail(YSKN_EINVAL, "batch_edit: an empty list of copies, or a stride below its width");
  // Every CTA reads the lengths, sources and count, the first one writes: dense arrays by all their bytes. (Tables may be
  // interleaved.)
  const int64_t row = 4ll * a.batch;
  const Span in[] = {{a.lens, row}, {a.keep, row}, {a.source, row}, {a.free, 4}};
  const Span out[] = {{a.lens_out, row}, {a.free_out, 4}, {a.pool, 4ll * a.pool_capacity}, {fork ? a.n_copies : nullptr, 4}};
  bool meet = fork && a.tables_out == a.block_tables;
  for (int i = 0; i < 4; ++i) {
    for (const Span& s : in) meet = meet || out[i].meets(s);
    for (int j = 0; j < i; ++j) meet = meet || out[i].meets(out[j]);
  }
  if (meet) return fail(YSKN_EINVAL, "batch_edit: the new lengths, counts, tables and the pool need arrays of their own");
  EditParams p{};
  p.lens = a.lens, p.keep = a.keep, p.source = a.source;
  p.tables = a.block_tables, p.table_stride = a.table_stride;
  p.tables_out = a.tables_out, p.out_stride = a.tables_out_stride;
  p.pool = a.pool, p.free_count = a.free, p.lens_out = a.lens_out, p.free_out = a.free_out;
  p.copies = a.copies, p.copies_stride = a.copies_stride, p.n_copies = a.n_copies;
  p.batch = a.batch, p.prefix_len = a.prefix_len, p.table_width = a.table_width;
  p.pool_capacity = a.pool_capacity, p.max_copies = a.max_copies;
  p.block_size = a.block_size, p.block_shift = -1;
  for (int x = 0; x < 31; ++x)
    if (a.block_size == 1 << x) p.block_shift = x;
  p.err = device_error_word();
  const size_t smem = (size_t)a.batch * (fork ? 28 : 20);
  // Every CTA repeats the sums: as many as the tables' pieces keep busy, one an SM at most.
  const int64_t units = fork ? a.batch * ceil_div(a.table_width, EDIT_PIECE) : ceil_div(a.batch, 8);
  const unsigned grid = (unsigned)std::min<int64_t>(ceil_div(units, EDIT_WARPS), 148);
  auto run = [&](auto kernel, SmemOptIn& opt_in) {
    if (cudaError_t e = opt_in(kernel, YSKN_PLAN_MAX_BATCH * 28)) return cuda_fail(e, "batch_edit_kernel attributes");
    return cuda_fail(launch_pdl(kernel, grid, EDIT_THREADS, smem, reinterpret_cast<cudaStream_t>(stream), p),
                     "batch_edit_kernel");
  };
  static SmemOptIn opt_fork, opt_keep;
  return fork ? run(batch_edit_kernel<true>, opt_fork) : run(batch_edit_kernel<false>, opt_keep);
}
