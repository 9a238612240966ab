// Attention of trees of drafted tokens over a paged 16-bit cache: each request's new rows beside the rows
// that its tokens share (the batch's prefix and the request's own cached ones), with the output gate.
//
// New token t of request i (its n new rows are the last of its len rows) sees the len - n rows before them and,
// of the new ones, those whose bit is set in its mask (and that are not behind it). Per query head, in binary32:
//   s_j = scale * <q, k_j>, out = sum_j exp(s_j - max s) v_j / sum_j exp(s_j - max s)
//   out *= 1 / (1 + exp(-gate))  (with a gate), rounded once. A token that sees nothing gives 0.
// The softmax is joined from parts, each with its maximum m, l = sum exp(s - m) and o = sum exp(s - m) v:
//   the rows before the new ones  seen alike by all tokens of a request, so without a mask: the tensor cores
//                                 (tree_attention_kernel). n G query rows of a KV head share them.
//   the new rows                  a handful that a node sees (its ancestors), each node its own: binary32
//                                 multiplications, one visible row after another (tree_join_kernel). A new row that a
//                                 token does not see is not touched for it, whatever it holds.
//
// tree_attention_kernel: persistent, clusters of two CTAs (a pair of SMs) of 12 warps each, with the roles and the
// ring of prefixattn.cu, which says what they do and why a pair: 256 rows with tcgen05.mma.cta_group::2, each CTA its
// 128 rows of Q, S, P and O and half of each K and V tile. What is different:
//   items     up to 256 query rows (a row is a token and one of the G query heads of a KV head; whole tokens) against a
//             row of key tiles (128 cache rows): the prefix's, for tokens of the batch, whichever request they belong
//             to; or one request's own, for its tokens. Where a request fills a good part of its items, these take the
//             prefix's tiles before their own and there are no prefix items (every CTA decides this alike from the
//             units that either way takes). An item counts one unit more than it has tiles, and pair c takes units
//             [c per, (c + 1) per) of all items in order; its part of an item is a segment.
//   the list  a warp lists the pair's segments in shared memory, a lane a request, up to 16 at once, for all roles:
//             each of them looking its segments up by itself cost a chain of loads a segment.
//   results   each segment's m, l and o go to the workspace in binary32, o as [D / 4][rows][4], so that the 32 rows of
//             a warp's store are adjacent. (Rows finished in place, a thread its row's channels and gate one after
//             another, held the softmax warps up for 10 us a segment.)
// What bounds it: K and V once, where items have many tiles (1.97 us a tile and pair from memory, 4.9 TB/s: what the
// ring holds does not cover the memory's latency; the tensor cores need 1.1); results, 1 KB a row and segment both
// ways, where they have few (a segment of one tile and 252 rows 4.9 us, without its stores 2.8); set-up, 8 us.
// Everything is summed in a fixed order: the same call gives the same bits.
// Rounded to 16 bits: the weights over the rows before the new ones, as the tensor cores take them (the type of V; 32-bit
// ones would be tf32, at half the rate, with V widened on the way), and the result. m, l, o, the joins and the new rows'
// weights are binary32, l the sum of the unrounded weights. Error against 64 bits 0.0021 to 0.0023 of the norm in bf16,
// where the result's rounding alone gives 0.0017, 0.00028 and 0.00021 in f16.
// us in a captured graph, and with a mask on prefix_attention's kernel instead: one request of 60 nodes and 2000 rows
// 18.5, 29.7; of 32 nodes and 8000 rows 22, 43.7; 8 of 60 nodes and up to 8000 rows 58, 100; 64 of 16 nodes and up to
// 1000 rows 62, 119; 32 of 32 nodes behind 4096 rows with up to 4096 of their own 146, 151. Calls one after another, each
// on inputs of its own, take 20 for the first and, at the clocks of a long run, 170 to 176 for the last. (One CTA with 128
// rows instead of the pair, whose ring holds 1.25 tiles instead of 2.5: 25, 37, 72, 67 and 180, where the pair then took
// 25, 24, 60, 69 and 156, with a slower join and an item's rows not halved between the CTAs.)
// Every mbarrier wait is bounded; after a timeout the softmax warps go through their remaining tiles without waiting,
// so that the halves' named barriers still match, and both CTAs meet before either leaves.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "attention.cuh"

namespace yskn {

constexpr int TA_ROWS = 128;    // query rows of a CTA, TMEM lanes
constexpr int TA_KEYS = 128;    // cache rows per tile
constexpr int TA_SLOT = 16384;  // bytes per ring slot
constexpr int TA_THREADS = 384;
constexpr int TA_MAX_PAIRS = 74;
constexpr int TA_MAX_SLOTS = 12;
// An item's fixed cost in tiles. 0, 1, 2, 3: 32 requests behind 4096 rows 170, 156, 152, 152 us, 64 of 8 nodes behind
// them 90, 83, 87, 91, one of 32 nodes and 8000 rows 25, 24, 24, 27.
constexpr int TA_COST = 1;
constexpr int TA_LIST = 16;  // segments listed at once
constexpr unsigned TA_MANY = 1u << 30;

template <int D>
struct TaShape {
  static constexpr int CHUNKS = D / 64;                     // 64-channel columns of a head
  static constexpr int SLOTS = D <= 128 ? 1 : D / 128;      // ring slots of a K or a V tile (one CTA's half)
  static constexpr int K_CHUNKS = CHUNKS / SLOTS;           // K slot: 64 rows of so many columns
  static constexpr int V_ROWS = TA_KEYS / SLOTS;            // V slot: so many rows
  static constexpr int V_CHUNKS = D <= 128 ? 1 : D / 128;   // of so many columns (D = 64: half a column)
  static constexpr int V_LINE = D == 64 ? 64 : 128;         // bytes of a V row in a column, the swizzle's span
  static constexpr int RING = D == 256 ? 10 : TA_MAX_SLOTS;
  static constexpr int Q_BYTES = CHUNKS * TA_ROWS * 128;
  static constexpr int SMEM = Q_BYTES + RING * TA_SLOT + 3072 /*TaShared*/;
  static constexpr int S_COL = D < 128 ? 128 : D;  // TMEM columns: O at 0, S tiles at S_COL and S_COL + 128
};

// The workspace: sizes from the host's bounds alone. Rows of results: those of the prefix items' places, 256 each, then
// those of the own items', own_rows each; a place more for each cut, of which there is one a pair at most.
struct TaWork {
  int64_t base, ml, o, bytes;  // byte offsets
  int own_rows;                // of an own item's place
  int64_t own_items;           // own items that there is room for
  int pre_items;
};
inline TaWork ta_work(int tokens, int batch, int max_new, int prefix_len, int n_qh, int n_kvh, int head) {
  auto up = [](int64_t v) { return (v + 255) / 256 * 256; };
  const int G = n_qh / n_kvh, tpc = TA_ROWS / G, tpi = 2 * tpc;  // tokens per CTA and per item
  TaWork w{};
  w.own_rows = G * std::min(tpi, max_new);
  // sum of ceil(n_i / tpi) over requests with n_i > 0: at most one more than n_i / tpi each
  w.own_items = (std::min(batch, tokens) + (int64_t)tokens / tpi) * n_kvh;
  w.pre_items = prefix_len > 0 ? (int)(ceil_div(tokens, tpi) * n_kvh) : 0;
  const int64_t cuts = (prefix_len > 0 ? TA_MAX_PAIRS * 2 * TA_ROWS : 0) + (int64_t)TA_MAX_PAIRS * w.own_rows;
  const int64_t rows = (int64_t)w.pre_items * 2 * TA_ROWS + w.own_items * w.own_rows + cuts;
  w.base = 256;
  w.ml = w.base + up((int64_t)batch * 8);
  w.o = w.ml + up(rows * 8);
  w.bytes = w.o + up(rows * head * 4);
  return w;
}

struct TreeAttnParams {
  const uint16_t *q, *k_cache, *v_cache;
  int64_t q_row, q_head;
  CacheStrides cache;
  const void* gate;  // of the queries' type, or f32
  int64_t gate_row, gate_head;
  bool gate_f32;
  const int32_t *prefix_blocks, *tables;
  int64_t table_stride;
  const int32_t *lens, *starts;
  const uint32_t* mask;
  int64_t mask_stride;
  int mask_words;
  int n_blocks, block_shift, prefix_len;  // blocks of 1 << block_shift rows
  int own_limit;                          // rows that a table row can name
  int batch, tokens, max_new, n_kvh, G;
  int tpc, tpi;                 // tokens per CTA and per item
  unsigned g_magic, tpi_magic;  // ceil(2^32 / d): quotients of numbers below 2^32 / d
  int pre_items, pre_tiles;     // prefix items, if there are any, and their tiles
  float c;                      // scale log2 e
  uint32_t negate_q;            // c is negative: the tensor cores take -Q, and |c|
  // for the join: units of a pair, whether there are prefix items (0: none; -1: nothing is computed), their units,
  // their places' rows
  int4* how;
  int2* base;  // [batch] own items, and units of all items, before each request's own
  float2* ml;  // (m, l) of each row of results
  float* o;
  int own_rows;
  long long own_items;  // more of them (starts that do not ascend), or 2^30 units, is an error: nothing is computed
  uint16_t* out;        // [tokens][n_qh][D]
  unsigned* err;
};

__device__ __forceinline__ int ta_quotient(int n, unsigned magic) {
  return magic ? (int)__umulhi((unsigned)n, magic) : n;
}

// Request i: its first token, its tokens (0 if there are none, or not what the host bounded), and its own rows before
// them.
struct TaRequest {
  int s0, n, own;
};
__device__ __forceinline__ TaRequest ta_request(const TreeAttnParams& p, int i) {
  TaRequest r;
  r.s0 = __ldg(p.starts + i);
  const int n = (int)((unsigned)__ldg(p.starts + i + 1) - (unsigned)r.s0);  // whatever the two are
  const int64_t own = (int64_t)__ldg(p.lens + i) - n - p.prefix_len;
  const bool wrong = n < 0 || n > p.max_new || r.s0 < 0 || r.s0 > p.tokens - n || own < 0;
  r.n = wrong ? 0 : n;
  r.own = wrong ? 0 : (int)min(own, (int64_t)p.own_limit);
  return r;
}
__device__ __forceinline__ int ta_items(const TreeAttnParams& p, const TaRequest& r) {  // of a KV head
  return r.n <= p.tpi ? r.n > 0 : ta_quotient(r.n + p.tpi - 1, p.tpi_magic);
}
__device__ __forceinline__ int ta_tiles(const TreeAttnParams& p, const TaRequest& r, bool alone) {
  return ((r.own + TA_KEYS - 1) / TA_KEYS) + (alone ? p.pre_tiles : 0);
}
__host__ __device__ __forceinline__ int ta_units(int tiles) { return tiles > 0 ? tiles + TA_COST : 0; }
__device__ __forceinline__ unsigned ta_sum(unsigned a, unsigned b) { return min(a + b, TA_MANY); }
__device__ __forceinline__ unsigned ta_times(unsigned a, unsigned b) {
  return (unsigned)min((unsigned long long)a * b, (unsigned long long)TA_MANY);
}

struct TaSegment {
  int row0;             // its first row of results
  int kvh, tok0, ntok;  // KV head, first token and whole tokens
  int req;              // own items: the request; -1: a prefix item
  int key0, key1;       // key tiles [key0, key1)
  int pre;              // the item's first tiles that are the prefix's
  int own;              // own rows
  // The item's tokens are halved between the CTAs: the first one of a CTA, and how many.
  __device__ int first_of(int rank) const { return rank ? (ntok + 1) >> 1 : 0; }
  __device__ int tokens_of(int rank) const { return rank ? ntok >> 1 : (ntok + 1) >> 1; }
  // Rows of tile kt.
  __device__ int rows_of(const TreeAttnParams& p, int kt) const {
    return min(TA_KEYS, kt < pre ? p.prefix_len - kt * TA_KEYS : own - (kt - pre) * TA_KEYS);
  }
};

// Shared memory beside Q and the ring. "First": only the first CTA's copy is used.
struct TaShared {
  uint64_t full[TA_MAX_SLOTS];     // ring place landed in both CTAs (first)
  uint64_t empty[TA_MAX_SLOTS];    // ring place read
  uint64_t q_full, q_empty;        // Q landed in both CTAs (first), read
  uint64_t s_full[2], pv_done[2];  // by tile parity: S written, P V done
  uint64_t p_full[2];              // P written by both CTAs (first)
  uint64_t o_free;                 // O read by both CTAs (first)
  uint64_t drained, tail_full, tail_done;
  int2 tail_at;
  uint32_t tmem_slot;
  int abort_word;
  int n_segments, more;  // listed; whether others follow
  // the pair's units, where the list is at, and the request that it is at with its first unit and own item
  int unit, unit_end, req, req_unit, req_item;
  int alone, per, pre_units;  // no prefix items; units of a pair; units of all prefix items
  union {
    uint4 sum[TA_THREADS / 32];
    float half[2][2][TA_ROWS];  // tile parity, half, row: what a row's halves exchange
  };
  TaSegment list[TA_LIST];
};
static_assert(sizeof(TaShared) <= 3072, "shared memory beside the ring");

// The next segments of the pair's units into the list (both CTAs list the same); warp 2, a lane an item of the prefix
// or a request at a time.
__device__ __forceinline__ void ta_list(const TreeAttnParams& p, TaShared& sh, int lane) {
  const int end = sh.unit_end, per = sh.per, pre_units = sh.pre_units, pair = blockIdx.x >> 1;
  const bool alone = sh.alone;
  int unit = sh.unit, n = 0;
  auto put = [&](int at, int u0, int u1, TaSegment s) {  // units [u0, u1) of an item
    s.key0 = max(u0 - TA_COST, 0), s.key1 = u1 - TA_COST;
    sh.list[at] = s;
  };
  const int pre_each = ta_units(p.pre_tiles), pre_q = max(p.pre_items / p.n_kvh, 1), pre_end = min(end, pre_units);
  while (unit < pre_end && n < TA_LIST) {
    const int item = unit / pre_each + lane;
    const int64_t b = (int64_t)item * pre_each;
    const int lo = (int)max((int64_t)unit, b), hi = (int)min((int64_t)pre_end, b + pre_each);
    const bool has = lo < hi && hi - b > TA_COST;
    const unsigned who = __ballot_sync(0xffffffffu, has);
    const int at = n + __popc(who & ((1u << lane) - 1));
    if (has && at < TA_LIST) {
      const int kvh = item / pre_q, q = item - kvh * pre_q;
      put(at, (int)(lo - b), (int)(hi - b),
          TaSegment{(item + pair) * 2 * TA_ROWS, kvh, q * p.tpi, min(p.tpi, p.tokens - q * p.tpi), -1, 0, 0,
                    p.pre_tiles, 0});
    }
    n = min(n + __popc(who), TA_LIST);
    unit = max(unit, (int)__reduce_max_sync(0xffffffffu, lo < hi && at < TA_LIST ? hi : 0));
  }
  // Rows of results of the prefix items' places, and the first pair that has own units.
  const int pre_rows = pre_units > 0 ? (p.pre_items + (pre_units + per - 1) / per) * 2 * TA_ROWS : 0;
  const int first_own = pre_units / per;
  int req = sh.req, req_unit = sh.req_unit, req_item = sh.req_item;
  while (unit < end && n < TA_LIST && req < p.batch) {
    TaRequest r{0, 0, 0};
    if (req + lane < p.batch) r = ta_request(p, req + lane);
    const int q = ta_items(p, r), each = ta_units(ta_tiles(p, r, alone)), all = q * p.n_kvh;
    int u1 = each * all, it1 = all;  // the ends of the request's units and own items
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int a = __shfl_up_sync(0xffffffffu, u1, off), c = __shfl_up_sync(0xffffffffu, it1, off);
      if (lane >= off) u1 += a, it1 += c;
    }
    u1 += req_unit, it1 += req_item;
    const int u0 = u1 - each * all, it0 = it1 - all, lo = max(unit, u0), hi = min(end, u1);
    // its items [x0, x1) that have tiles in this pair's part
    int x0 = 0, x1 = 0;
    if (lo < hi) {
      x0 = (lo - u0) / each, x1 = (hi - u0 + each - 1) / each;
      if (hi - u0 - (x1 - 1) * each <= TA_COST) --x1;  // no tile of the last one
    }
    const int count = max(x1 - x0, 0);
    int at = count;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int a = __shfl_up_sync(0xffffffffu, at, off);
      if (lane >= off) at += a;
    }
    const int total = __shfl_sync(0xffffffffu, at, 31);
    at += n - count;
    for (int x = x0; x < x1 && at + x - x0 < TA_LIST; ++x) {
      const int kvh = x / q, qt = x - kvh * q, b = u0 + x * each;
      put(at + x - x0, max(lo, b) - b, min(hi, b + each) - b,
          TaSegment{pre_rows + (it0 + x + pair - first_own) * p.own_rows, kvh, r.s0 + qt * p.tpi,
                    min(p.tpi, r.n - qt * p.tpi), req + lane, 0, 0, alone ? p.pre_tiles : 0, r.own});
    }
    if (n + total >= TA_LIST) {  // full: on from the last one's end, in its request
      const int left = TA_LIST - at;  // of the lane's: so many are listed
      const unsigned who = __ballot_sync(0xffffffffu, left > 0 && left <= count);
      const int by = __ffs(who) - 1;
      unit = __shfl_sync(0xffffffffu, min(hi, u0 + (x0 + left) * each), by);
      req_unit = __shfl_sync(0xffffffffu, u0, by), req_item = __shfl_sync(0xffffffffu, it0, by);
      req += by;
      n = TA_LIST;
    } else {
      unit = max(unit, (int)__reduce_max_sync(0xffffffffu, lo < hi ? hi : 0));
      req_unit = __shfl_sync(0xffffffffu, u1, 31), req_item = __shfl_sync(0xffffffffu, it1, 31);
      req += 32;
      n += total;
    }
  }
  __syncwarp();
  if (lane == 0) {
    sh.unit = unit, sh.req = req, sh.req_unit = req_unit, sh.req_item = req_item;
    sh.n_segments = n;
    sh.more = n == TA_LIST && unit < end;
  }
}

// Both warps of a row quarter.
__device__ __forceinline__ void ta_quarter_sync(int quarter) {
  asm volatile("bar.sync %0, 64;" ::"r"(1 + quarter) : "memory");
}

template <int D, int DT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(TA_THREADS, 1)
    tree_attention_kernel(const __grid_constant__ CUtensorMap map_q_pre, const __grid_constant__ CUtensorMap map_q_own,
                          const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                          const __grid_constant__ TreeAttnParams p) {
  using Shape = TaShape<D>;
  constexpr int RING = Shape::RING, SLOTS = Shape::SLOTS, VR = Shape::V_ROWS;
  extern __shared__ __align__(1024) uint8_t smem[];  // swizzled tiles start on 1024 bytes
  uint8_t* sQ = smem;                                // [D / 64][128 rows][128 B]
  uint8_t* ring = smem + Shape::Q_BYTES;             // [RING][16 KB]
  TaShared& sh = *reinterpret_cast<TaShared*>(ring + RING * TA_SLOT);
  volatile int* abort_flag = &sh.abort_word;
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);  // known to be the same in all lanes
  const int rank = blockIdx.x & 1, pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

  if (tid == 0) {
    for (int s = 0; s < RING; ++s) mbar_init(&sh.full[s], 2), mbar_init(&sh.empty[s], 1);
    mbar_init(&sh.q_full, 2), mbar_init(&sh.q_empty, 1);
    for (int b = 0; b < 2; ++b) mbar_init(&sh.s_full[b], 1), mbar_init(&sh.p_full[b], 16), mbar_init(&sh.pv_done[b], 1);
    mbar_init(&sh.o_free, 16), mbar_init(&sh.drained, 1);
    mbar_init(&sh.tail_full, 1), mbar_init(&sh.tail_done, 1);
    sh.abort_word = 0;
    mbar_init_fence();
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 3) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem_slot)),
                 "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
  if (warp == 2 && lane < 4) {
    const CUtensorMap* map = lane == 0 ? &map_q_pre : lane == 1 ? &map_q_own : lane == 2 ? &map_k : &map_v;
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // both CTAs' barriers are set up
  tc_fence_after();
  pdl_begin();

  // Units of all requests and where this pair begins. A thread's requests are adjacent.
  {
    const int per_thread = (p.batch + TA_THREADS - 1) / TA_THREADS;
    const int i0 = min(p.batch, tid * per_thread), i1 = min(p.batch, i0 + per_thread);
    unsigned items = 0, units[2] = {0, 0};  // beside prefix items, and alone
    for (int i = i0; i < i1; ++i) {
      const TaRequest r = ta_request(p, i);
      const unsigned all = ta_times(ta_items(p, r), p.n_kvh);
      items = ta_sum(items, all);
      for (int x = 0; x < 2; ++x) units[x] = ta_sum(units[x], ta_times(all, ta_units(ta_tiles(p, r, x))));
      if (blockIdx.x == 0) {
        const int64_t rows = (int64_t)__ldg(p.lens + i) - p.prefix_len;  // own ones, the new among them
        if (__ldg(p.starts + i + 1) != r.s0 + r.n || (r.n > 0 && rows > p.own_limit))
          raise_device_error(p.err, DERR_RANGE);
      }
    }
    unsigned ui[2] = {units[0], units[1]}, it = items;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const unsigned a = __shfl_up_sync(0xffffffffu, ui[0], off), b = __shfl_up_sync(0xffffffffu, ui[1], off);
      const unsigned c = __shfl_up_sync(0xffffffffu, it, off);
      if (lane >= off) ui[0] = ta_sum(ui[0], a), ui[1] = ta_sum(ui[1], b), it = ta_sum(it, c);
    }
    if (lane == 31) sh.sum[warp] = make_uint4(ui[0], ui[1], it, 0);
    __syncthreads();
    unsigned before[2] = {0, 0}, total[2] = {0, 0}, items_before = 0, total_items = 0;
    for (int w = 0; w < TA_THREADS / 32; ++w) {
      const uint4 o = sh.sum[w];
      if (w < warp) {
        before[0] = ta_sum(before[0], o.x), before[1] = ta_sum(before[1], o.y);
        items_before = ta_sum(items_before, o.z);
      }
      total[0] = ta_sum(total[0], o.x), total[1] = ta_sum(total[1], o.y), total_items = ta_sum(total_items, o.z);
    }
    // Alone, if that is at most an eighth more: the prefix items' results have to be stored and joined too.
    const unsigned pre_all = (unsigned)p.pre_items * ta_units(p.pre_tiles);  // below 2^30: the host looked
    const bool alone =
        pre_all == 0 || (total[1] < TA_MANY && 8ull * total[1] <= 9ull * (pre_all + (unsigned long long)total[0]));
    const unsigned pre = alone ? 0 : pre_all, own = alone ? total[1] : total[0];
    const bool sound = total_items <= (unsigned long long)p.own_items && own < TA_MANY && pre + own < TA_MANY;
    const int all = sound ? (int)(pre + own) : 0, per = max((all + pairs - 1) / pairs, 1);
    const int t0 = min(all, pair * per), t1 = min(all, t0 + per);
    if (tid == 0) {
      sh.unit = t0, sh.unit_end = t1, sh.alone = alone, sh.per = per, sh.pre_units = sound ? (int)pre : 0;
      if (t0 < (int)pre) sh.req = 0, sh.req_unit = (int)pre, sh.req_item = 0;
      if (t0 >= all) sh.req = p.batch, sh.req_unit = sh.req_item = 0;
      if (blockIdx.x == 0) {
        *p.how = make_int4(per, sound ? (int)pre : -1, alone, 0);
        if (!sound) raise_device_error(p.err, DERR_RANGE);
      }
    }
    // the first own unit of this pair lies in one thread's requests
    unsigned u = pre + (alone ? ta_sum(before[1], ui[1] - units[1]) : ta_sum(before[0], ui[0] - units[0]));
    unsigned item = ta_sum(items_before, it - items);
    const unsigned mine_end = u + (alone ? units[1] : units[0]);
    const bool mine = t0 >= (int)pre && t0 < all && (unsigned)t0 >= u && (unsigned)t0 < mine_end;
    if (sound && (mine || blockIdx.x == 0)) {
      for (int i = i0; i < i1; ++i) {
        const TaRequest r = ta_request(p, i);
        const unsigned n = (unsigned)ta_items(p, r) * p.n_kvh, next = u + n * ta_units(ta_tiles(p, r, alone));
        if (mine && (unsigned)t0 >= u && (unsigned)t0 < next) sh.req = i, sh.req_unit = (int)u, sh.req_item = (int)item;
        if (blockIdx.x == 0) p.base[i] = make_int2((int)item, (int)u);
        u = next;
        item += n;
      }
    }
  }
  __syncthreads();
  const uint32_t tmem = sh.tmem_slot;

  // Where each role is, over all lists.
  int s_at = 0;                             // warps 0, 1: the ring's place
  uint32_t turn = warp == 0 ? 1 : 0;        // and the parity of its last reading (first round: already free) or filling
  uint32_t tails = 0;                       // warp 0: slots that warp 3 has had to clear
  int g = 0, n_seg = 0;                     // tiles and segments so far
  bool ok = true;
  const bool leader = warp == 1 && rank == 0 && elect_one();
  for (;;) {
    if (warp == 2) ta_list(p, sh, lane);
    __syncthreads();
    const int n_list = sh.n_segments;
    const bool more = sh.more;
    if (warp == 0) {
      // ---- K and V through the ring, in the order in which the MMAs use them: this CTA's half of
      // each tile's K rows, and of V's channels
      const int shift = p.block_shift, pages = TA_KEYS >> shift;
      const int box_k = min(1 << shift, TA_KEYS / 2), box_v = min(1 << shift, VR);
      const uint32_t full0 = first_cta(&sh.full[0]);
      const int v_chunk = D == 64 ? 0 : rank * Shape::V_CHUNKS, v_x = D == 64 ? rank * 32 : 0;
      for (int i = 0; ok && i < n_list; ++i) {
        const TaSegment seg = sh.list[i];
        auto block_of = [&](int kt) {  // lane l: the block of page l of tile kt
          int b = 0;
          if (kt < seg.key1 && lane < pages && (lane << shift) < seg.rows_of(p, kt)) {
            b = __ldg(kt < seg.pre ? p.prefix_blocks + kt * pages + lane
                                   : p.tables + (int64_t)seg.req * p.table_stride + (kt - seg.pre) * pages + lane);
            if ((unsigned)b >= (unsigned)p.n_blocks) raise_device_error(p.err, DERR_RANGE);  // the copy gives zeros
          }
          return b;
        };
        // The next place of the ring, once both CTAs' part of it has been read.
        auto claim = [&]() {
          ok = __all_sync(0xffffffffu, mbar_wait(&sh.empty[s_at], turn, abort_flag));
          return ring + s_at * TA_SLOT;
        };
        auto advance = [&]() {
          if (++s_at == RING) s_at = 0, turn ^= 1;
        };
        // Rows key0 .. key0 + n * box - 1 of the tile, `chunks` columns from `chunk` on, as
        // [column][ROWS rows][line] at `to`: one box, or one per block and column.
        auto copy = [&](uint8_t* to, const CUtensorMap* map, uint32_t bar, int key0, int n, int box, int rows, int x,
                        int chunk, int chunks, int line, int block) {
          const int key = key0 + lane * box;
          const int b = __shfl_sync(0xffffffffu, block, (key >> shift) & 31);
          if (lane < n) {
            const int y = key & ((1 << shift) - 1);
            if (box == rows) pair_load_5d(to, map, bar, x, y, chunk, seg.kvh, b);
            else
              for (int d = 0; d < chunks; ++d)
                pair_load_5d(to + (d * rows + lane * box) * line, map, bar, x, y, chunk + d, seg.kvh, b);
          }
        };
        auto put_k = [&](int kt, int block) {
          const int nk = min(max(seg.rows_of(p, kt) - rank * (TA_KEYS / 2), 0), TA_KEYS / 2);
          const int n = (nk + box_k - 1) / box_k;
          for (int d = 0; ok && d < SLOTS; ++d) {
            uint8_t* to = claim();
            if (!ok) break;
            const uint32_t bar = full0 + 8 * s_at;
            if (lane == 0) expect_first(bar, (uint32_t)(n * box_k * 128 * Shape::K_CHUNKS));
            __syncwarp();
            copy(to, &map_k, bar, rank * (TA_KEYS / 2), n, box_k, TA_KEYS / 2, 0, d * Shape::K_CHUNKS, Shape::K_CHUNKS,
                 128, block);
            advance();
          }
        };
        auto put_v = [&](int kt, int block) {
          const int nk = seg.rows_of(p, kt);
          for (int v = 0; ok && v * VR < nk; ++v) {
            const int rows = min(VR, nk - v * VR), n = (rows + box_v - 1) / box_v;
            uint8_t* to = claim();
            if (!ok) break;
            uint32_t bar = full0 + 8 * s_at;
            const uint32_t bytes = (uint32_t)(n * box_v) * Shape::V_LINE * Shape::V_CHUNKS;
            if (rows & 15) {  // lands on this CTA's barrier; warp 3 clears the end and then arrives
              if (tails > 0) ok = __all_sync(0xffffffffu, mbar_wait(&sh.tail_done, (tails - 1) & 1, abort_flag));
              if (!ok) break;
              ++tails;
              if (lane == 0) {
                sh.tail_at = make_int2(s_at, rows);
                mbar_expect_tx(&sh.tail_full, bytes);
              }
              bar = smem_u32(&sh.tail_full);  // of this CTA, as a cluster address
              asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(bar) : "r"(smem_u32(&sh.tail_full)), "r"(rank));
            } else if (lane == 0) {
              expect_first(bar, bytes);
            }
            __syncwarp();
            copy(to, &map_v, bar, v * VR, n, box_v, VR, v_x, v_chunk, Shape::V_CHUNKS, Shape::V_LINE, block);
            advance();
          }
        };
        int cur = block_of(seg.key0), nxt = block_of(seg.key0 + 1);
        put_k(seg.key0, cur);
        for (int kt = seg.key0; ok && kt < seg.key1; ++kt) {
          const int after = block_of(kt + 2);
          if (kt + 1 < seg.key1) put_k(kt + 1, nxt);
          if (ok) put_v(kt, cur);
          cur = nxt;
          nxt = after;
        }
      }
      if (!more) {
        if (ok && tails > 0) ok = __all_sync(0xffffffffu, mbar_wait(&sh.tail_done, (tails - 1) & 1, abort_flag));
        if (!ok) {  // a copy lands within microseconds: let those that this warp started do so
          const long long t0 = clock64();
          while (clock64() - t0 < TC_WAIT_LIMIT / 1000) {
          }
        }
      }
    } else if (warp == 1) {
      // ---- MMAs: one thread of the first CTA
      if (leader) {
        const uint32_t id_qk = pair_idesc(DT, TA_KEYS, 0, p.negate_q), id_pv = pair_idesc(DT, D, 1, 0);
        // descriptors: Q, and K or V at the ring's first place; the high words hold no address
        const uint32_t a_lo = (uint32_t)sw128_desc(smem_u32(sQ)), b_lo = (uint32_t)sw128_desc(smem_u32(ring));
        const uint32_t k_hi = (uint32_t)(sw128_desc(0) >> 32), v_hi = (uint32_t)(mn_desc<Shape::V_LINE>(0, 0) >> 32);
        const uint32_t v_lo = (uint32_t)mn_desc<Shape::V_LINE>(smem_u32(ring), VR * Shape::V_LINE);
        auto advance = [&]() {
          umma2_commit(&sh.empty[s_at]);
          if (++s_at == RING) s_at = 0, turn ^= 1;
        };
        auto qk = [&](int tile) {  // S of the pair's tile number `tile`
          const uint32_t d = tmem + Shape::S_COL + (tile & 1) * TA_KEYS;
#pragma unroll
          for (int v = 0; v < SLOTS; ++v) {
            ok = ok && mbar_wait(&sh.full[s_at], turn, abort_flag);
            if (!ok) return;
            tc_fence_after();
#pragma unroll
            for (int ch = 0; ch < Shape::K_CHUNKS; ++ch) {
              const uint32_t a = a_lo + (v * Shape::K_CHUNKS + ch) * (TA_ROWS * 128 >> 4);
              const uint32_t b = b_lo + s_at * (TA_SLOT >> 4) + ch * (TA_KEYS / 2 * 128 >> 4);
#pragma unroll
              for (int k = 0; k < 4; ++k) umma2_ss(d, a + 2 * k, b + 2 * k, k_hi, id_qk, v > 0 || ch > 0 || k > 0);
            }
            advance();
          }
          umma2_commit(&sh.s_full[tile & 1]);
        };
        auto pv = [&](int nk, uint32_t pt, bool first) {
#pragma unroll
          for (int v = 0; v < SLOTS; ++v) {
            const int rows = nk - v * VR;
            if (rows <= 0) break;
            ok = ok && mbar_wait(&sh.full[s_at], turn, abort_flag);
            if (!ok) return;
            tc_fence_after();
            const uint32_t b = v_lo + s_at * (TA_SLOT >> 4);
#pragma unroll
            for (int k = 0; k < VR / 16; ++k)
              if (k * 16 < rows)
                umma2_ts(tmem, pt + (v * VR + k * 16) / 2, b + (16 * Shape::V_LINE >> 4) * k, v_hi, id_pv,
                         !first || v > 0 || k > 0);
            advance();
          }
        };
        for (int i = 0; ok && i < n_list; ++i, ++n_seg) {
          const TaSegment seg = sh.list[i];
          ok = mbar_wait(&sh.q_full, n_seg & 1, abort_flag);
          const int n = seg.key1 - seg.key0;
          if (ok) qk(g);
          for (int j = 0; ok && j < n; ++j, ++g) {
            if (j + 1 < n) qk(g + 1);
            if (ok && j == max(0, n - 2)) umma2_commit(&sh.q_empty);  // after the segment's last S
            if (j == 0 && n_seg > 0) ok = ok && mbar_wait(&sh.o_free, (n_seg - 1) & 1, abort_flag);
            ok = ok && mbar_wait(&sh.p_full[g & 1], (g >> 1) & 1, abort_flag);
            if (!ok) break;
            tc_fence_after();
            pv(seg.rows_of(p, seg.key0 + j), tmem + Shape::S_COL + (g & 1) * TA_KEYS, j == 0);
            if (ok) umma2_commit(&sh.pv_done[g & 1]);
          }
        }
        if (!more) {  // every MMA of the pair has completed before its TMEM is freed
          umma2_commit(&sh.drained);
          const long long t0 = clock64();
          while (!mbar_try_wait(&sh.drained, 0) && clock64() - t0 < TC_WAIT_LIMIT) {
          }
        }
      }
      __syncwarp();
    } else if (warp == 2) {
      // ---- Q: this CTA's tokens of each segment
      if (lane == 0) {
        const uint32_t bar = first_cta(&sh.q_full);
        for (int i = 0; i < n_list; ++i, ++n_seg) {
          const TaSegment seg = sh.list[i];
          if (n_seg > 0 && !(ok = ok && mbar_wait(&sh.q_empty, (n_seg - 1) & 1, abort_flag))) break;
          const bool prefix = seg.req < 0, any = seg.tokens_of(rank) > 0;
          const int box = prefix ? p.tpc : min(p.tpc, p.max_new);
          expect_first(bar, any ? (uint32_t)(box * p.G * 128 * Shape::CHUNKS) : 0u);
          if (any)
            for (int d = 0; d < Shape::CHUNKS; ++d)
              pair_load_3d(sQ + d * TA_ROWS * 128, prefix ? &map_q_pre : &map_q_own, bar, d * 64, seg.kvh * p.G,
                           seg.tok0 + seg.first_of(rank));
        }
        if (!ok) {
          const long long t0 = clock64();
          while (clock64() - t0 < TC_WAIT_LIMIT / 1000) {
          }
        }
      }
      __syncwarp();
    } else if (warp == 3) {
      // ---- V rows past the last one, up to the end of the 16-row step, to zero, in the slots that warp 0 names:
      // one for each segment that ends inside a step
      const uint32_t full0 = first_cta(&sh.full[0]);
      for (int i = 0; i < n_list; ++i) {
        const TaSegment seg = sh.list[i];
        for (int kt = seg.key0; ok && kt < seg.key1; ++kt) {
          if (!(seg.rows_of(p, kt) & 15)) continue;
          ok = __all_sync(0xffffffffu, mbar_wait(&sh.tail_full, tails & 1, abort_flag));
          if (!ok) break;
          ++tails;
          const int2 t = sh.tail_at;  // ring place, rows to keep
          constexpr int UNITS = Shape::V_LINE / 16;  // 16-byte units of a row
          const int units = (16 - (t.y & 15)) * UNITS;
          uint8_t* base = ring + t.x * TA_SLOT + t.y * Shape::V_LINE;
          for (int x = lane; x < units * Shape::V_CHUNKS; x += 32) {
            const int ch = x / units, y = x - ch * units;
            *reinterpret_cast<uint4*>(base + ch * VR * Shape::V_LINE + y * 16) = make_uint4(0, 0, 0, 0);
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) {
            release_first(full0 + 8 * t.x);
            mbar_arrive(&sh.tail_done);
          }
        }
      }
    } else {
      // ---- softmax, a row's column halves in two threads, then the segment's result
      const int quarter = warp & 3, half = (warp - 4) >> 2, row = quarter * 32 + lane;
      const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
      const uint32_t p_full0 = first_cta(&sh.p_full[0]), o_free0 = first_cta(&sh.o_free);
      const float c = fabsf(p.c);
      for (int i = 0; i < n_list; ++i) {
        const TaSegment seg = sh.list[i];
        const bool valid = row < seg.tokens_of(rank) * p.G;
        const bool live = __any_sync(0xffffffffu, valid);  // a warp without rows only keeps the barriers going
        float m = -INFINITY, l = 0.0f;
        for (int kt = seg.key0; kt < seg.key1; ++kt, ++g) {
          const int b = g & 1;
          mbar_wait(&sh.s_full[b], (g >> 1) & 1, abort_flag);
          __syncwarp();
          if (live) {
            tc_fence_after();
            const uint32_t at = tmem + lanes + Shape::S_COL + b * TA_KEYS;
            uint32_t s[2][32];
            tmem_ld32(at + half * 64, s[0]);
            tmem_ld32(at + half * 64 + 32, s[1]);
            tmem_ld_wait32(s[0]);
            tmem_ld_wait32(s[1]);
            const int see = seg.rows_of(p, kt) - half * 64;
            if (see < 64) {
#pragma unroll
              for (int x = 0; x < 64; ++x)
                if (x >= see) s[x >> 5][x & 31] = 0xff800000u;  // -inf
            }
            auto val = [&](int x) { return __uint_as_float(s[x >> 5][x & 31]); };
            float t[4] = {val(0), val(1), val(2), val(3)};
#pragma unroll
            for (int x = 4; x < 60; x += 8)
#pragma unroll
              for (int y = 0; y < 4; ++y) t[y] = max3(t[y], val(x + 2 * y), val(x + 2 * y + 1));
            t[0] = max3(t[0], val(60), val(61));
            t[1] = max3(t[1], val(62), val(63));
            const float mine = fmaxf(max3(t[0], t[1], t[2]), t[3]);
            sh.half[b][half][row] = mine;
            ta_quarter_sync(quarter);  // also: both halves have read S, so P may take its place
            const float top = __fmul_rn(fmaxf(mine, sh.half[b][half ^ 1][row]), c);
            if (m == -INFINITY) m = top;  // nothing before: o and l are zero
            const bool grown = top > m + 8.0f;
            if (__any_sync(0xffffffffu, grown)) {
              // o is complete up to the tile before; then scale it
              mbar_wait(&sh.pv_done[b ^ 1], ((g - 1) >> 1) & 1, abort_flag);
              __syncwarp();
              tc_fence_after();
              const float f = grown ? exp2_approx(m - top) : 1.0f;
#pragma unroll 1
              for (int x = half * (D / 2); x < (half + 1) * (D / 2); x += 32) {  // rolled: rare code, else spills
                uint32_t o[32];
                tmem_ld32(tmem + lanes + x, o);
                tmem_ld_wait();
#pragma unroll
                for (int y = 0; y < 32; ++y) o[y] = __float_as_uint(__uint_as_float(o[y]) * f);
                tmem_st32(tmem + lanes + x, o);
              }
              l *= f;
              if (grown) m = top;
            }
            const float base = m == -INFINITY ? 0.0f : -m;
            const float2 c2 = make_float2(c, c), b2 = make_float2(base, base);
            float2 sum[2] = {{0.0f, 0.0f}, {0.0f, 0.0f}};
            uint32_t w[32];
#pragma unroll
            for (int x = 0; x < 32; ++x) {
              const float2 e = fma2(make_float2(val(2 * x), val(2 * x + 1)), c2, b2);
              const float2 a = make_float2(exp2_approx(e.x), exp2_approx(e.y));
              sum[x & 1] = add2(sum[x & 1], a);
              w[x] = Elem<DT>::pack(a.x, a.y);
            }
            tmem_st32(at + half * 32, w);
            sum[0] = add2(sum[0], sum[1]);
            l += sum[0].x + sum[0].y;
            tmem_st_wait();
            tc_fence_before();
          }
          __syncwarp();
          if (lane == 0) arrive_first(p_full0 + 8 * b);
        }
        mbar_wait(&sh.pv_done[(g - 1) & 1], ((g - 1) >> 1) & 1, abort_flag);
        __syncwarp();
        if (live) {
          tc_fence_after();
          ta_quarter_sync(quarter);  // the tiles' exchanges have been read
          sh.half[0][half][row] = l;
          ta_quarter_sync(quarter);
          l += sh.half[0][half ^ 1][row];
          const int rows = seg.req < 0 ? 2 * TA_ROWS : p.own_rows;
          const int at = seg.first_of(rank) * p.G + row;  // of the place
          float4* o = reinterpret_cast<float4*>(p.o + (int64_t)seg.row0 * D) + at;
          for (int x = half * (D / 2); x < (half + 1) * (D / 2); x += 32) {
            uint32_t v[32];
            tmem_ld32(tmem + lanes + x, v);
            tmem_ld_wait32(v);
            if (valid) {
#pragma unroll
              for (int y = 0; y < 32; y += 4)
                o[(x + y) / 4 * rows] = make_float4(__uint_as_float(v[y]), __uint_as_float(v[y + 1]),
                                                    __uint_as_float(v[y + 2]), __uint_as_float(v[y + 3]));
            }
          }
          if (valid && half == 0) p.ml[seg.row0 + at] = make_float2(m, l);
          tc_fence_before();
          ta_quarter_sync(quarter);  // the halves' sums have been read
        }
        __syncwarp();
        if (lane == 0) arrive_first(o_free0);
      }
    }
    __syncthreads();  // the list has been read
    if (!more) break;
  }
  tc_fence_before();
  __syncthreads();
  if (tid == 0 && *abort_flag) raise_device_error(p.err, DERR_TIMEOUT);
  __syncwarp();
  cluster_sync();  // neither CTA's memory is used any more
  if (warp == 3) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
  }
}

// Four channels of the output gate, as they are stored, and as f32: apart, so that other loads are under way too.
__device__ __forceinline__ uint4 ta_gate_load(const TreeAttnParams& p, int64_t at) {
  if (p.gate_f32) return __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const float*>(p.gate) + at));
  const uint2 g = __ldg(reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(p.gate) + at));
  return make_uint4(g.x, g.y, 0, 0);
}
// Four 16-bit values as f32.
template <int DT>
__device__ __forceinline__ float4 ta_four(uint2 v) {
  return make_float4(Elem<DT>::to_float((uint16_t)v.x), Elem<DT>::to_float((uint16_t)(v.x >> 16)),
                     Elem<DT>::to_float((uint16_t)v.y), Elem<DT>::to_float((uint16_t)(v.y >> 16)));
}

// Joins a row's segments with the new rows that it sees, divides, gates and rounds. A CTA takes 8 rows (a row is a
// token and one of the G query heads of a KV head), 4 warps with a quarter of the channels each: lane (r, qd) row r,
// every fourth 16-byte unit of the quarter from qd on. The new rows first: a few visible ones of each row at a time,
// keys and values asked for together, the scores of the quarters added up through shared memory. Then the row's
// segments. What bounds it is the chain of dependent loads (the token's request, its table, its rows; the segments),
// and instructions where there are many rows (64 requests of 16 nodes: 17 of 62 us, of which new rows 8). Where there
// are few rows, which then have many segments (SPLIT), four more warps take the segments beside those for the new rows,
// which do not wait for the first kernel. By one group, by two, by four (a CTA an SM then): one request of 60 nodes and 2000 rows 24, 20,
// 25 us; of 32 nodes and 8000 rows 33, 23, 22; 16 of 16 nodes and 1500 rows, more rows than the rule's, 27, 30, 30.
// (A warp for all heads of a token, whose lanes share the keys and values: fewer instructions, but 200 registers, and
// 64 requests 89 us where this takes 69.)
// Its new rows' work grows with what a node sees, and each query head reads it again: a tree's few ancestors, not a long
// chain (us behind 2000 rows, a chain of 8, 16, 32, 60, 128: 14.5, 18, 29, 45, 105, prefix_attention 23, 24, 28, 34, 33).
// It reads the call's inputs before pdl_begin(), and the first group of SPLIT never waits: it starts only once every CTA
// of tree_attention_kernel has passed its own pdl_begin(), so that what came before the call is done and in memory; the
// first kernel's results, and all writes, come after the wait. Nothing may be launched between the two.
// Per cent of the largest shared memory, a hint: the join needs few KB of it, and the rest caches the rows that a
// token's heads share. Without it the join runs with what the first kernel has asked for, all of it: one request of 60
// nodes 20.2 us, with 15 to 65 per cent 18.5; 64 of 16 nodes 64.1, with up to 35 per cent 61.9.
constexpr int TJ_CARVE = 35;
// CTAs an SM of one group. 4, 5, 6, 7: 64 requests of 16 nodes 65, 62, 63, 69 us, 32 of 32 behind 4096 rows 149, 146,
// 149, 152.
constexpr int TJ_RESIDENT = 5;

template <int D, int DT, bool SPLIT>
__global__ void __launch_bounds__(SPLIT ? 256 : 128, SPLIT ? 2 : TJ_RESIDENT)
    tree_join_kernel(const __grid_constant__ TreeAttnParams p) {
  constexpr int NJ = D / 64;            // 16-byte units (4 channels) of a lane
  constexpr int ONCE = SPLIT ? 4 : 2;   // new rows, or segments, asked for at once: what registers hold
  __shared__ __align__(16) float s_part[2][4][8][4];  // a warp's part of each score
  __shared__ bool s_sound;
  __shared__ float s_state[4][2 + 4 * NJ][32];  // what the second group has
  const int lane = threadIdx.x & 31, group = threadIdx.x >> 7, part = threadIdx.x >> 5 & 3;
  const int r = lane & 7, qd = lane >> 3;
  const int idx = blockIdx.x * 8 + r, kvh = blockIdx.y, t = ta_quotient(idx, p.g_magic), gh = idx - t * p.G;
  const int h = kvh * p.G + gh, unit0 = part * (D / 16) + qd;  // of 4 channels; then every fourth
  const bool live = t < p.tokens;
  uint2 qv[NJ];
  uint32_t bits = 0;
  if (group == 0) {  // what does not depend on the request
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      qv[j] = make_uint2(0, 0);
      if (live) qv[j] = __ldg(reinterpret_cast<const uint2*>(p.q + t * p.q_row + h * p.q_head + 4 * (unit0 + 4 * j)));
    }
    if (live) bits = __ldg(p.mask + t * p.mask_stride);
  }
  // The request of the CTA's first token (the last whose first token is at or before it), 32 probes a round; then the
  // row's.
  int req = 0;
  {
    const int first = ta_quotient(blockIdx.x * 8, p.g_magic);
    int n = p.batch;
    while (n > 1) {
      const int step = (n + 31) >> 5, at = lane * step;
      const unsigned below = __ballot_sync(0xffffffffu, at < n && __ldg(p.starts + req + min(at, n - 1)) <= first);
      const int k = below ? 31 - __clz(below) : 0;
      req += k * step;
      n = min(step, n - k * step);
    }
    if (req + 1 < p.batch && __ldg(p.starts + req + 1) <= t) {
      int hi = p.batch;
      while (hi - req > 1) {
        const int mid = (req + hi) >> 1;
        if (__ldg(p.starts + mid) <= t) req = mid;
        else hi = mid;
      }
    }
  }
  const TaRequest rq = ta_request(p, req);
  const int self = t - rq.s0;  // of the request's new rows
  const bool valid = live && self >= 0 && self < rq.n;

  float m = -INFINITY, l = 0.0f;
  float2 o[NJ][2];
#pragma unroll
  for (int j = 0; j < NJ; ++j) o[j][0] = o[j][1] = make_float2(0.0f, 0.0f);
  auto scale_by = [&](float f) {
#pragma unroll
    for (int j = 0; j < NJ; ++j)
      o[j][0].x *= f, o[j][0].y *= f, o[j][1].x *= f, o[j][1].y *= f;
  };
  uint4 gate[NJ];
  if (group == 0) {
    // ---- the new rows that the token sees
    const int32_t* table = p.tables + (int64_t)req * p.table_stride;
    const int last = valid ? min(self >> 5, p.mask_words - 1) : -1, named = p.own_limit - rq.own;
    int word = 0;
    auto cut = [&]() {  // to the new rows up to itself, of those that the table names
      const int upto = min(self + 1, named) - 32 * word;
      if (upto < 32) bits = upto > 0 ? bits & ((1u << upto) - 1) : 0;
    };
    if (last < 0) bits = 0;
    cut();
    auto skip_empty = [&]() {
      while (bits == 0 && word < last) {
        bits = __ldg(p.mask + t * p.mask_stride + ++word);
        cut();
      }
    };
    skip_empty();
    for (int buffer = 0; __any_sync(0xffffffffu, bits != 0); buffer ^= 1) {  // the same in the four warps
      uint2 k[ONCE][NJ], v[ONCE][NJ];
      bool sees[ONCE];
#pragma unroll
      for (int x = 0; x < ONCE; ++x) {
        sees[x] = bits != 0;
        int64_t at = -1;
        if (sees[x]) {
          const int row = rq.own + 32 * word + __ffs(bits) - 1, block = __ldg(table + (row >> p.block_shift));
          bits &= bits - 1;
          skip_empty();
          if ((unsigned)block < (unsigned)p.n_blocks)
            at = block * p.cache.block + (row & ((1 << p.block_shift) - 1)) * p.cache.token + kvh * p.cache.head +
                 4 * unit0;
          else
            raise_device_error(p.err, DERR_RANGE);  // it is zeros
        }
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          k[x][j] = v[x][j] = make_uint2(0, 0);
          if (at >= 0) {
            k[x][j] = *reinterpret_cast<const uint2*>(p.k_cache + at + 16 * j);
            v[x][j] = *reinterpret_cast<const uint2*>(p.v_cache + at + 16 * j);
          }
        }
      }
      float mine = 0.0f;  // of new row qd
#pragma unroll
      for (int x = 0; x < ONCE; ++x) {
        float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          const float4 a = ta_four<DT>(qv[j]), b = ta_four<DT>(k[x][j]);
          sum = fma2(make_float2(a.x, a.y), make_float2(b.x, b.y), sum);
          sum = fma2(make_float2(a.z, a.w), make_float2(b.z, b.w), sum);
        }
        float one = sum.x + sum.y;
        one += __shfl_xor_sync(0xffffffffu, one, 8);
        one += __shfl_xor_sync(0xffffffffu, one, 16);
        if (qd == x) mine = one;
      }
      s_part[buffer][part][r][qd] = mine;
      asm volatile("bar.sync 1, 128;" ::: "memory");
      float z[ONCE], top = m;
      {
        float4 y = *reinterpret_cast<const float4*>(s_part[buffer][0][r]);
#pragma unroll
        for (int w = 1; w < 4; ++w) {
          const float4 d = *reinterpret_cast<const float4*>(s_part[buffer][w][r]);
          y.x += d.x, y.y += d.y, y.z += d.z, y.w += d.w;
        }
        z[0] = y.x * p.c, z[1] = y.y * p.c;
        if constexpr (ONCE == 4) z[2] = y.z * p.c, z[3] = y.w * p.c;
      }
#pragma unroll
      for (int x = 0; x < ONCE; ++x)
        if (sees[x]) top = fmaxf(top, z[x]);
      const float base = top == -INFINITY ? 0.0f : top, keep = m == -INFINITY ? 0.0f : exp2_approx(m - base);
      if (m != -INFINITY) {  // (before, l and o are zero, or NaN that has to stay)
        l *= keep;
        scale_by(keep);
      }
      m = top;
#pragma unroll
      for (int x = 0; x < ONCE; ++x)
        if (sees[x]) {
          const float a = exp2_approx(z[x] - base);
          const float2 a2 = make_float2(a, a);
          l += a;
#pragma unroll
          for (int j = 0; j < NJ; ++j) {
            const float4 b = ta_four<DT>(v[x][j]);
            o[j][0] = fma2(a2, make_float2(b.x, b.y), o[j][0]);
            o[j][1] = fma2(a2, make_float2(b.z, b.w), o[j][1]);
          }
        }
    }
    // (before them its registers cost more than its latency here: 64 requests of 16 nodes 66.5 us instead of 64.1)
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      gate[j] = make_uint4(0, 0, 0, 0);
      if (p.gate && live) gate[j] = ta_gate_load(p, t * p.gate_row + h * p.gate_head + 4 * (unit0 + 4 * j));
    }
  }
  bool sound = true;
  if (!SPLIT || group > 0) {
    pdl_begin();  // the first kernel's results
    // ---- the row's segments: n_pre of its prefix item, then those of its own
    const int4 how = *p.how;
    const int2 base = valid ? p.base[req] : make_int2(0, 0);
    const int per = how.x, pre_units = max(how.y, 0);
    const bool alone = how.z;
    sound = how.y >= 0;
    int n_pre = 0, n = 0, pre_in = 0, own_in = 0;
    int64_t pre_row = 0, own_row = 0;
    if (valid && sound) {
      if (pre_units > 0) {
        const int each = ta_units(p.pre_tiles), qt = ta_quotient(t, p.tpi_magic);
        const int item = kvh * (p.pre_items / p.n_kvh) + qt, b = item * each + TA_COST, c0 = b / per;
        n_pre = (b + p.pre_tiles - 1) / per - c0 + 1;
        pre_row = (int64_t)(item + c0) * 2 * TA_ROWS;
        pre_in = (t - qt * p.tpi) * p.G + gh;
      }
      const int tiles = ta_tiles(p, rq, alone);
      n = n_pre;
      if (tiles > 0) {
        const int each = ta_units(tiles), qt = ta_quotient(self, p.tpi_magic);
        const int item = kvh * ta_items(p, rq) + qt;
        const int b = base.y + item * each + TA_COST, c0 = b / per;
        const int pre_rows = pre_units > 0 ? (p.pre_items + (pre_units + per - 1) / per) * 2 * TA_ROWS : 0;
        n += (b + tiles - 1) / per - c0 + 1;
        own_row = pre_rows + (int64_t)(base.x + item + c0 - pre_units / per) * p.own_rows;
        own_in = (self - qt * p.tpi) * p.G + gh;
      }
    }
    const int most = (int)__reduce_max_sync(0xffffffffu, n);
    for (int x0 = 0; x0 < most; x0 += ONCE) {
      float2 ml[ONCE];
      float4 y[ONCE][NJ];
      float now = m;
#pragma unroll
      for (int u = 0; u < ONCE; ++u) {
        const int x = x0 + u;
        const bool pre = x < n_pre;
        const int rows = pre ? 2 * TA_ROWS : p.own_rows, in = pre ? pre_in : own_in;
        const int64_t row = pre ? pre_row + (int64_t)x * rows : own_row + (int64_t)(x - n_pre) * rows;
        ml[u] = make_float2(-INFINITY, 0.0f);
        if (x < n) ml[u] = p.ml[row + in];
        const float4* from = reinterpret_cast<const float4*>(p.o) + row * (D / 4) + in;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          y[u][j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          if (x < n) y[u][j] = from[(unit0 + 4 * j) * rows];
        }
      }
#pragma unroll
      for (int u = 0; u < ONCE; ++u) now = fmaxf(now, ml[u].x);
      if (m != -INFINITY) {  // (before, l and o are zero, or NaN that has to stay)
        const float keep = exp2_approx(m - now);
        l *= keep;
        scale_by(keep);
      }
      m = now;
#pragma unroll
      for (int u = 0; u < ONCE; ++u) {
        const float w = ml[u].x == -INFINITY ? 0.0f : exp2_approx(ml[u].x - now);
        const float2 w2 = make_float2(w, w);
        l = fmaf(ml[u].y, w, l);
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          o[j][0] = fma2(w2, make_float2(y[u][j].x, y[u][j].y), o[j][0]);
          o[j][1] = fma2(w2, make_float2(y[u][j].z, y[u][j].w), o[j][1]);
        }
      }
    }
    if constexpr (SPLIT) {
      if (threadIdx.x == 128) s_sound = sound;
      float(&mine)[2 + 4 * NJ][32] = s_state[part];
      mine[0][lane] = m, mine[1][lane] = l;
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        mine[2 + 4 * j][lane] = o[j][0].x, mine[3 + 4 * j][lane] = o[j][0].y;
        mine[4 + 4 * j][lane] = o[j][1].x, mine[5 + 4 * j][lane] = o[j][1].y;
      }
    }
  }
  if constexpr (SPLIT) {
    __syncthreads();
    if (group > 0 || !live) return;
    const float(&other)[2 + 4 * NJ][32] = s_state[part];
    const float top = other[0][lane], now = fmaxf(m, top);
    const float keep = exp2_approx(m - now), w = top == -INFINITY ? 0.0f : exp2_approx(top - now);
    if (m != -INFINITY) {
      l *= keep;
      scale_by(keep);
    }
    l = fmaf(other[1][lane], w, l);
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      o[j][0].x = fmaf(other[2 + 4 * j][lane], w, o[j][0].x), o[j][0].y = fmaf(other[3 + 4 * j][lane], w, o[j][0].y);
      o[j][1].x = fmaf(other[4 + 4 * j][lane], w, o[j][1].x), o[j][1].y = fmaf(other[5 + 4 * j][lane], w, o[j][1].y);
    }
    sound = s_sound;
  }
  if (!live) return;
  const float inv = !valid || !sound || l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    float z[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (inv != 0.0f) {
      z[0] = o[j][0].x * inv, z[1] = o[j][0].y * inv, z[2] = o[j][1].x * inv, z[3] = o[j][1].y * inv;
      if (p.gate) {
        const float4 g =
            p.gate_f32 ? make_float4(__uint_as_float(gate[j].x), __uint_as_float(gate[j].y),
                                     __uint_as_float(gate[j].z), __uint_as_float(gate[j].w))
                       : ta_four<DT>(make_uint2(gate[j].x, gate[j].y));
        z[0] = gated(z[0], g.x), z[1] = gated(z[1], g.y), z[2] = gated(z[2], g.z), z[3] = gated(z[3], g.w);
      }
    }
    *reinterpret_cast<uint2*>(p.out + ((int64_t)t * p.n_kvh * p.G + h) * D + 4 * (unit0 + 4 * j)) =
        make_uint2(Elem<DT>::pack(z[0], z[1]), Elem<DT>::pack(z[2], z[3]));
  }
}

template <int D, int DT>
static int launch_tree_attention(const CUtensorMap (&maps)[4], const TreeAttnParams& p, int ctas, cudaStream_t st) {
  static SmemOptIn opt_in;
  if (cudaError_t e = opt_in(tree_attention_kernel<D, DT>, TaShape<D>::SMEM))
    return cuda_fail(e, "tree_attention_kernel attributes");
  if (cudaError_t e = launch_pdl(tree_attention_kernel<D, DT>, ctas, TA_THREADS, TaShape<D>::SMEM, st, maps[0],
                                 maps[1], maps[2], maps[3], p))
    return cuda_fail(e, "tree_attention_kernel");
  const dim3 grid((unsigned)ceil_div((int64_t)p.tokens * p.G, 8), p.n_kvh);
  auto join = [&](auto split) {  // a second group where the rows alone do not fill the SMs
    constexpr bool SPLIT = decltype(split)::value;
    static SmemOptIn carve{cudaFuncAttributePreferredSharedMemoryCarveout};
    if (cudaError_t e = carve(tree_join_kernel<D, DT, SPLIT>, TJ_CARVE))
      return cuda_fail(e, "tree_join_kernel attributes");
    return cuda_fail(launch_pdl(tree_join_kernel<D, DT, SPLIT>, grid, SPLIT ? 256 : 128, 0, st, p), "tree_join_kernel");
  };
  return (int64_t)grid.x * grid.y <= 2 * 148 ? join(std::true_type{}) : join(std::false_type{});
}

}  // namespace yskn

using namespace yskn;

extern "C" YSKN_B200_API int yskn_b200_tree_attention(const yskn_b200_tree_attention_args* args, void* stream) {
  if (!args || !args->mask) return fail(YSKN_EINVAL, "tree_attention: null argument");
  if (args->mask_words < 1 || (args->attn.tokens > 1 && args->mask_stride < args->mask_words))
    return fail(YSKN_EINVAL, "tree_attention: no mask words, or a stride below them");
  yskn_b200_prefix_attention_args a = args->attn;
  if (const char* what = attention_refusal(a)) return fail(YSKN_EINVAL, std::string("tree_attention: ") + what);
  const int head = a.head, n_qh = a.n_qh, n_kvh = a.n_kvh, block_size = a.block_size, dtype = a.dtype;
  const int G = n_qh / n_kvh, tpc = TA_ROWS / G;
  // the workspace is what prefix_attention asks for, by the caller's max_new; a request cannot have more tokens than
  // the call, or than mask bits
  if (a.work_bytes < yskn_b200_prefix_attention_work_bytes(a.tokens, a.batch, a.max_new, n_qh, n_kvh, head))
    return fail(YSKN_EINVAL, "tree_attention: workspace too small");
  a.max_new = (int)std::min<int64_t>({(int64_t)a.max_new, (int64_t)a.tokens, 32ll * args->mask_words});
  const TaWork w = ta_work(a.tokens, a.batch, a.max_new, a.prefix_len, n_qh, n_kvh, head);
  TreeAttnParams p{};
  p.pre_tiles = (int)ceil_div(a.prefix_len, TA_KEYS);
  if ((int64_t)w.pre_items * ta_units(p.pre_tiles) >= (int64_t)TA_MANY || (w.o - w.ml) / 8 > INT32_MAX ||
      (int64_t)a.tokens * n_qh * head > INT32_MAX || a.tokens >= 1 << 24 || n_kvh > 65535 || a.work_bytes < w.bytes)
    return fail(YSKN_EINVAL, "tree_attention: too much work");
  p.q = reinterpret_cast<const uint16_t*>(a.q), p.q_row = a.q_row, p.q_head = a.q_head;
  p.k_cache = reinterpret_cast<const uint16_t*>(a.k_cache), p.v_cache = reinterpret_cast<const uint16_t*>(a.v_cache);
  p.cache = {a.block_stride, a.token_stride, a.head_stride};
  p.gate = a.gate, p.gate_f32 = a.gate_dtype == YSKN_DT_F32;
  p.gate_row = a.gate_row, p.gate_head = a.gate_head;
  p.prefix_blocks = a.prefix_blocks;
  p.tables = a.block_tables, p.table_stride = a.table_stride;
  p.lens = a.lens, p.starts = a.starts;
  p.mask = args->mask, p.mask_stride = args->mask_stride, p.mask_words = args->mask_words;
  p.n_blocks = a.n_blocks, p.prefix_len = a.prefix_len;
  p.block_shift = block_size == 16 ? 4 : block_size == 32 ? 5 : block_size == 64 ? 6 : 7;
  p.own_limit = (int)std::min<int64_t>((int64_t)a.table_width * block_size, INT32_MAX - TA_KEYS);
  p.batch = a.batch, p.tokens = a.tokens, p.max_new = a.max_new, p.n_kvh = n_kvh, p.G = G, p.tpc = tpc, p.tpi = 2 * tpc;
  int dev = 0, sms = 2 * TA_MAX_PAIRS;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const int grid = 2 * std::min(sms / 2, TA_MAX_PAIRS);
  auto magic = [](int d) { return d == 1 ? 0u : (unsigned)(((1ull << 32) + d - 1) / d); };
  p.g_magic = magic(G), p.tpi_magic = magic(p.tpi);
  p.pre_items = w.pre_items;
  // a scale of zero keeps its meaning (equal weights) with a factor that leaves -inf alone
  p.negate_q = a.scale < 0.0f;
  p.c = std::max(std::fabs(a.scale) * 1.4426950408889634f, 1e-30f) * (p.negate_q ? -1.0f : 1.0f);
  uint8_t* work = reinterpret_cast<uint8_t*>(a.work);
  p.how = reinterpret_cast<int4*>(work);
  p.base = reinterpret_cast<int2*>(work + w.base);
  p.ml = reinterpret_cast<float2*>(work + w.ml), p.o = reinterpret_cast<float*>(work + w.o);
  p.own_rows = w.own_rows, p.own_items = w.own_items;
  p.out = reinterpret_cast<uint16_t*>(a.out), p.err = device_error_word();
  // The cache's 64-channel columns are an axis of their own, so that one box holds several columns of its rows in the
  // order of the ring's slots; where a slot takes several boxes (blocks shorter than it), a box is one column.
  const int slots = head <= 128 ? 1 : head / 128, v_rows = TA_KEYS / slots;
  const int64_t q_dims[3] = {head, n_qh, a.tokens}, q_strides[2] = {a.q_head, a.q_row};
  const int64_t c_dims[5] = {64, block_size, head / 64, n_kvh, a.n_blocks};
  const int64_t c_strides[4] = {a.token_stride, 64, a.head_stride, a.block_stride};
  const int box_pre[3] = {64, G, tpc}, box_own[3] = {64, G, std::min(tpc, a.max_new)};
  const int box_k[5] = {64, std::min(block_size, TA_KEYS / 2), block_size < TA_KEYS / 2 ? 1 : head / 64 / slots, 1, 1};
  const int box_v[5] = {head == 64 ? 32 : 64, std::min(block_size, v_rows),
                        block_size < v_rows || head <= 128 ? 1 : head / 128, 1, 1};
  CUtensorMap maps[4] = {};
  if (int rc = paged_map("tree_attention", &maps[0], a.q, dtype, 3, q_dims, q_strides, box_pre)) return rc;
  if (int rc = paged_map("tree_attention", &maps[1], a.q, dtype, 3, q_dims, q_strides, box_own)) return rc;
  if (int rc = paged_map("tree_attention", &maps[2], a.k_cache, dtype, 5, c_dims, c_strides, box_k)) return rc;
  if (int rc = paged_map("tree_attention", &maps[3], a.v_cache, dtype, 5, c_dims, c_strides, box_v)) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  auto run = [&](auto d) {
    constexpr int N = decltype(d)::value;
    return dtype == YSKN_DT_BF16 ? launch_tree_attention<N, YSKN_DT_BF16>(maps, p, grid, st)
                                 : launch_tree_attention<N, YSKN_DT_F16>(maps, p, grid, st);
  };
  if (head == 64) return run(std::integral_constant<int, 64>{});
  if (head == 128) return run(std::integral_constant<int, 128>{});
  return run(std::integral_constant<int, 256>{});
}
