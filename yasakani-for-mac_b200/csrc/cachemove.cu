// Rows moved inside the layers' paged 16-bit caches: whole blocks copied for requests that continue
// others, and the rows of accepted paths made adjacent. All layers' K and V caches in one launch.
//
// What bounds both: bytes, each read once and written once; for short paths, latency.
// cache_copy: a warp copies a piece, 4 KB of one head of one block of one cache (8 rows of 256 channels, 8 16-byte
// loads a lane before the first store). Many more CTAs than the SMs hold, each a few pieces, so that the SMs keep
// busy whatever rows the blocks hold: 256 copies of 1 to 64 rows in 16 caches 88 us (6.4 TB/s; whole blocks 6.7), as
// many CTAs as are resident 96, and one CTA a head of a block with the next one's loads ahead of its stores 104 to 117.
// cache_compact: a warp takes one head of one request's path in three caches: the path and the blocks are looked up
// once, and three rows in each cache are under way at once (64 paths of 6 nodes in 32 caches 7.2 us, 64 of 12 in 64
// caches 35; in four caches, with three CTAs an SM, 8.0 and 40; in two, with six, 7.4 and 37; in one 11.4 and 50).
// Row base + path[k] goes to base + k, and path[k] >= k, in ascending order: a row that is written (k) was a source
// only for smaller k (path[k'] = k means k' <= k), so that a warp that loads a run of rows before it stores them, run
// after run, never reads a row that it has overwritten.
#include <algorithm>

#include "paged.cuh"

namespace yskn {

constexpr int MOVE_THREADS = 128;
constexpr int MOVE_WARPS = MOVE_THREADS / 32;
constexpr int COPY_LOADS = 8;   // 16-byte loads of a lane under way
constexpr int COPY_CTAS = 80;   // of an SM's share of a long list, most of them waiting
constexpr int MOVE_RUN = 3;     // rows of a path that a lane moves at once
constexpr int MOVE_CACHES = 3;  // in so many caches

struct MoveCaches {
  uint16_t* base[YSKN_MAX_CACHES];
  CacheStrides stride;
  int n_caches, n_blocks, block_size, n_kvh, units;  // units: 16-byte units of a head's row, a power of two
  int unit_shift;
};

struct CopyParams {
  MoveCaches c;
  const int32_t* copies;
  int64_t copies_stride;
  const int32_t* count;
  int max_copies;
  unsigned* err;
};

__global__ void __launch_bounds__(MOVE_THREADS) cache_copy_kernel(const __grid_constant__ CopyParams p) {
  pdl_begin();
  const MoveCaches& c = p.c;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int n = p.count ? min(max(__ldg(p.count), 0), p.max_copies) : p.max_copies;
  const int at_once = 32 >> c.unit_shift, sub = lane >> c.unit_shift, unit = lane & (c.units - 1);
  const int step = at_once * COPY_LOADS, steps = (c.block_size + step - 1) / step;  // rows of a piece; pieces of a head
  const int per = c.n_caches * c.n_kvh * steps;                                     // and of an entry
  const int64_t pieces = (int64_t)n * per;
  for (int64_t u = (int64_t)blockIdx.x * MOVE_WARPS + warp; u < pieces; u += (int64_t)gridDim.x * MOVE_WARPS) {
    const int e = (int)(u / per), rest = (int)(u - (int64_t)e * per), head = rest / steps;
    const int first = (rest - head * steps) * step, cache = head / c.n_kvh, h = head - cache * c.n_kvh;
    const int from = __ldg(p.copies + e), to = __ldg(p.copies + e + p.copies_stride);
    const int rows = __ldg(p.copies + e + 2 * p.copies_stride);
    if (rows <= first) continue;
    if (from < 0 || from >= c.n_blocks || to < 0 || to >= c.n_blocks || rows > c.block_size) {
      if (lane == 0) raise_device_error(p.err, DERR_RANGE);
      continue;
    }
    uint16_t* base = c.base[cache] + h * c.stride.head + (first + sub) * c.stride.token + unit * 8;
    const uint16_t* src = base + from * c.stride.block;
    uint16_t* dst = base + to * c.stride.block;
    const int64_t by = at_once * c.stride.token;
    uint4 v[COPY_LOADS];
#pragma unroll
    for (int x = 0; x < COPY_LOADS; ++x)
      if (first + x * at_once + sub < rows) v[x] = __ldcs(reinterpret_cast<const uint4*>(src + x * by));
#pragma unroll
    for (int x = 0; x < COPY_LOADS; ++x)
      if (first + x * at_once + sub < rows) __stcs(reinterpret_cast<uint4*>(dst + x * by), v[x]);
  }
}

struct CompactParams {
  MoveCaches c;
  const int32_t* tables;
  int64_t table_stride;
  const int32_t *lens, *starts, *path;
  int64_t path_stride;
  int batch, table_width, prefix_len, path_width;
  unsigned* err;
};

__global__ void __launch_bounds__(MOVE_THREADS, 5) cache_compact_kernel(const __grid_constant__ CompactParams p) {
  pdl_begin();
  const MoveCaches& c = p.c;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int groups = (c.n_caches + MOVE_CACHES - 1) / MOVE_CACHES, per = groups * c.n_kvh;  // units of a request
  const int at_once = 32 >> c.unit_shift, sub = lane >> c.unit_shift, unit = lane & (c.units - 1);
  const int64_t units = (int64_t)p.batch * per;
  for (int64_t u = (int64_t)blockIdx.x * MOVE_WARPS + warp; u < units; u += (int64_t)gridDim.x * MOVE_WARPS) {
    const int r = (int)(u / per), rest = (int)(u - (int64_t)r * per);
    const int group = rest / c.n_kvh, h = rest - group * c.n_kvh;
    const int cache0 = group * MOVE_CACHES, caches = min(MOVE_CACHES, c.n_caches - cache0);
    const int s0 = __ldg(p.starts + r), n = (int)((unsigned)__ldg(p.starts + r + 1) - (unsigned)s0);
    const int len = __ldg(p.lens + r);
    const int32_t* table = p.tables + (int64_t)r * p.table_stride;
    const int32_t* path = p.path + (int64_t)r * p.path_stride;
    // Lane l: node k0 + l of the path, for the run from k0 on; the first asked for beside the lengths.
    auto nodes = [&](int k0) {
      return lane < min(at_once * MOVE_RUN, p.path_width - k0) ? __ldg(path + k0 + lane) : -1;
    };
    int node = nodes(0);
    const long long base = (long long)len - n - p.prefix_len;  // own row of the first new one
    if (n == 0) continue;
    // the same in all lanes; a block of this lane's outside the caches
    bool wrong = n < 0 || base < 0 || (base + n - 1) / c.block_size >= p.table_width, lost = false;
    // This lane's element of own row `row`, or -1.
    auto place = [&](long long row) -> int64_t {
      const int b = (int)((unsigned)row / (unsigned)c.block_size), block = __ldg(table + b);
      if (block < 0 || block >= c.n_blocks) {
        lost = true;
        return -1;
      }
      return block * c.stride.block + (row - (int64_t)b * c.block_size) * c.stride.token + h * c.stride.head + unit * 8;
    };
    int before = -1;  // the node before this run's first
    for (int k0 = 0; !wrong && k0 < p.path_width; k0 += at_once * MOVE_RUN) {
      const int run = min(at_once * MOVE_RUN, p.path_width - k0);  // how many of them are in order:
      int prior = __shfl_up_sync(0xffffffffu, node, 1);
      if (lane == 0) prior = before;
      const unsigned ends = __ballot_sync(0xffffffffu, lane >= run || node < 0);
      const unsigned bad = __ballot_sync(0xffffffffu, lane < run && node >= 0 && (node <= prior || node >= n));
      const int stop = min(ends ? __ffs(ends) - 1 : 32, bad ? __ffs(bad) - 1 : 32);
      if (bad && __ffs(bad) - 1 == stop) wrong = true;
      uint4 v[MOVE_CACHES][MOVE_RUN];
      int64_t from[MOVE_RUN], to[MOVE_RUN];
#pragma unroll
      for (int x = 0; x < MOVE_RUN; ++x) {
        const int k = x * at_once + sub, source = __shfl_sync(0xffffffffu, node, k & 31);
        to[x] = -1;
        if (k < stop && source != k0 + k) {
          from[x] = place(base + source), to[x] = place(base + k0 + k);
          if (from[x] < 0) to[x] = -1;
        }
      }
#pragma unroll
      for (int y = 0; y < MOVE_CACHES; ++y)
#pragma unroll
        for (int x = 0; x < MOVE_RUN; ++x)
          if (y < caches && to[x] >= 0) v[y][x] = *reinterpret_cast<const uint4*>(c.base[cache0 + y] + from[x]);
      __syncwarp();
#pragma unroll
      for (int y = 0; y < MOVE_CACHES; ++y)
#pragma unroll
        for (int x = 0; x < MOVE_RUN; ++x)
          if (y < caches && to[x] >= 0) *reinterpret_cast<uint4*>(c.base[cache0 + y] + to[x]) = v[y][x];
      __syncwarp();
      if (stop < run) break;
      before = __shfl_sync(0xffffffffu, node, run - 1);
      node = nodes(k0 + run);
    }
    if (__any_sync(0xffffffffu, wrong || lost) && lane == 0) raise_device_error(p.err, DERR_RANGE);
  }
}

// The caches of a call; nullptr on success, else what is wrong.
static const char* move_caches(MoveCaches& c, void* const* caches, int n_caches, int64_t block, int64_t token,
                               int64_t head_stride, int n_blocks, int block_size, int n_kvh, int head) {
  if (!caches) return "null argument";
  if (n_caches < 1 || n_caches > YSKN_MAX_CACHES || n_blocks < 1 || block_size < 1 || n_kvh < 1)
    return "1..256 caches, and no empty shape";
  if (head != 64 && head != 128 && head != 256) return "heads of 64, 128 or 256 channels";
  if (n_kvh == 1) head_stride = 0;  // strides that nothing steps over may be anything
  if (n_blocks == 1) block = 0;
  if (block_size == 1) token = 0;
  if ((block | token | head_stride) % 8) return "strides are multiples of 16 bytes";
  for (int i = 0; i < n_caches; ++i) {
    if (!caches[i]) return "null cache";
    if (!aligned16(caches[i])) return "pointers are multiples of 16 bytes";
    c.base[i] = reinterpret_cast<uint16_t*>(caches[i]);
  }
  c.stride = {block, token, head_stride};
  c.n_caches = n_caches, c.n_blocks = n_blocks, c.block_size = block_size, c.n_kvh = n_kvh;
  c.units = head / 8;
  c.unit_shift = head == 64 ? 3 : head == 128 ? 4 : 5;
  return nullptr;
}

}  // namespace yskn

using namespace yskn;

extern "C" YSKN_B200_API int yskn_b200_cache_copy(const yskn_b200_cache_copy_args* args, void* stream) {
  if (!args) return fail(YSKN_EINVAL, "cache_copy: null argument");
  const yskn_b200_cache_copy_args& a = *args;
  CopyParams p{};
  if (const char* what = move_caches(p.c, a.caches, a.n_caches, a.block_stride, a.token_stride, a.head_stride,
                                     a.n_blocks, a.block_size, a.n_kvh, a.head))
    return fail(YSKN_EINVAL, std::string("cache_copy: ") + what);
  if (!a.copies || a.max_copies < 1 || a.copies_stride < a.max_copies)
    return fail(YSKN_EINVAL, "cache_copy: no list of copies, or a stride below its width");
  const int at_once = COPY_LOADS * (32 >> p.c.unit_shift);  // rows of a piece
  const int64_t pieces = (int64_t)a.n_caches * a.n_kvh * ceil_div(a.block_size, at_once);  // of an entry
  if (pieces > INT32_MAX) return fail(YSKN_EINVAL, "cache_copy: more rows, heads and caches than 2^31 pieces");
  p.copies = a.copies, p.copies_stride = a.copies_stride, p.count = a.count, p.max_copies = a.max_copies;
  p.err = device_error_word();
  const int64_t ctas = ceil_div(a.max_copies * pieces, MOVE_WARPS);
  const unsigned grid = (unsigned)std::min<int64_t>(ctas, 148 * COPY_CTAS);
  return cuda_fail(launch_pdl(cache_copy_kernel, grid, MOVE_THREADS, 0, reinterpret_cast<cudaStream_t>(stream), p),
                   "cache_copy_kernel");
}

extern "C" YSKN_B200_API int yskn_b200_cache_compact(const yskn_b200_cache_compact_args* args, void* stream) {
  if (!args) return fail(YSKN_EINVAL, "cache_compact: null argument");
  const yskn_b200_cache_compact_args& a = *args;
  CompactParams p{};
  if (const char* what = move_caches(p.c, a.caches, a.n_caches, a.block_stride, a.token_stride, a.head_stride,
                                     a.n_blocks, a.block_size, a.n_kvh, a.head))
    return fail(YSKN_EINVAL, std::string("cache_compact: ") + what);
  if (!a.block_tables || !a.lens || !a.starts || !a.path) return fail(YSKN_EINVAL, "cache_compact: null argument");
  if (a.batch < 1 || a.table_width < 1 || a.prefix_len < 0 || a.path_width < 1 ||
      (a.batch > 1 && (a.table_stride < a.table_width || a.path_stride < a.path_width)) ||
      (int64_t)a.n_caches * a.n_kvh > INT32_MAX / 2)
    return fail(YSKN_EINVAL, "cache_compact: empty shape, or a stride below its width");
  p.tables = a.block_tables, p.table_stride = a.table_stride, p.lens = a.lens, p.starts = a.starts;
  p.path = a.path, p.path_stride = a.path_stride;
  p.batch = a.batch, p.table_width = a.table_width, p.prefix_len = a.prefix_len, p.path_width = a.path_width;
  p.err = device_error_word();
  const int64_t units = ceil_div((int64_t)a.batch * ceil_div(a.n_caches, MOVE_CACHES) * a.n_kvh, MOVE_WARPS);
  const unsigned grid = (unsigned)std::min<int64_t>(units, 148 * 16);
  return cuda_fail(launch_pdl(cache_compact_kernel, grid, MOVE_THREADS, 0, reinterpret_cast<cudaStream_t>(stream), p),
                   "cache_compact_kernel");
}
