// Attention of a batch's new tokens over a prefix that all its requests share and each
// request's own rows, both in blocks of a paged 16-bit cache, with the output gate.
//
// Token t of request i (its n tokens are the last of its len rows, the prefix's P counted)
// sees the first lim = max(0, len - n + t + 1) rows of the sequence: rows below P in the
// prefix's blocks, the others in the request's. Per query head, in binary32:
//   s_j = scale * <q, k_j>, out = sum_j exp(s_j - max s) v_j / sum_j exp(s_j - max s)
//   out *= 1 / (1 + exp(-gate))  (with a gate), rounded once. A token that sees nothing gives 0.
// Rows that no token of the call sees are not read into any sum, whatever the cache holds there: the
// prefix's tiles end at the longest length, an own item's at its last token. (A row that some token of
// an item sees has weight zero for the others, and so has to hold a number for them.)
//
// The softmax over all rows is the join of softmaxes over parts: with a part's maximum m,
// l = sum exp(s - m) and o = sum exp(s - m) v, parts join as sum exp(m - M) o / sum
// exp(m - M) l, M the largest m. So the work is cut into items:
//   prefix items  256 query rows (a row is a token and one of the G query heads of a KV head;
//                 2 * floor(128 / G) whole tokens of the batch, whichever request they belong
//                 to) against the P prefix rows: the prefix is read once per 256 rows, not once
//                 per request;
//   own items     up to 256 rows of one request against that request's own rows; thin ones, where
//                 every request of the call has at most 8 rows a KV head (G max_new <= 8).
// Where requests have many tokens each (prompt chunks), 256 rows of one request read the prefix as
// well as 256 rows of several do: then an own item takes the prefix's tiles before its own and
// there are no prefix items, so that most rows are finished in one place. Every CTA decides this
// alike from the units that either way takes (below).
// Items are cut along their key tiles (128 rows of the cache; 16 for thin ones) so that every pair of
// SMs (a warp, for thin ones, in the SMs that the prefix items leave) gets the same share: an item
// counts a fixed cost in units and one per tile, and pair c takes units [c per, (c + 1) per) of all
// items in order. A piece of an item is a segment; its unnormalised (m, l, o) goes to the workspace in
// binary32, at place item + c, which no two segments share, and prefix_combine_kernel joins a row's
// segments, divides, gates and rounds; a segment that holds all that its rows see finishes them
// itself. Everything is summed in a fixed order: the same call gives the same bits. The lengths stay
// on the device: every CTA forms the prefix sum of the requests' units itself.
//
// prefix_attention_kernel: persistent, clusters of two CTAs (a pair of SMs), 12 warps each. The
// pair works on 256 rows with tcgen05.mma.cta_group::2: each CTA holds its 128 rows of Q, S, P and
// O, and half of each K tile (64 of its 128 rows) and V tile (half of the channels). With one
// SM per 128 rows, the operands' reads (128 KB of Q and K and 64 KB of V per tile) and the copies'
// writes (128 KB) alone need 2560 clocks of shared memory per tile, against 2048 of the tensor
// cores at D = 256, and twice the L2 traffic; halved K and V bring it to 1536. In each CTA:
//   warp 0  brings 16 KB slots of K and V (64 K rows of 128 channels; 64 V rows of 128 channels or
//           128 of 64 or 32) through a ring with TMA, each box within one block. The copies of
//           both CTAs count on the first CTA's barriers;
//   warp 1  (one thread of the first CTA) issues S = Q K^T (256 x 128, K = D) into one of two
//           TMEM tiles, then O += P V (256 x D, K = 128) with P read from TMEM, S of the next tile
//           before P V of this one, so that the tensor cores run while the softmax does;
//   warp 2  brings Q (TMA; a box is the G heads of whole tokens);
//   warp 3  clears the V rows past a segment's last visible row (below);
//   warps 4..11  two threads per row, one for each half of S's columns (and of O's): S from
//           TMEM, the running maximum, P = 2^(s c - m) (c = scale log2 e) rounded to the cache's
//           type over S's place, the row sum in binary32 of the unrounded weights. The maximum in
//           use may lag: o and l are rescaled only when a row's maximum has grown by more than
//           2^8, so that a weight is at most 256 and o is seldom touched; the join uses the
//           maximum in use, which cancels. (Two groups that take whole tiles in turn, so that one's
//           exponentials run beside the other's loads, measured 134 against 110 us at 64 requests
//           behind 32k rows: with two S tiles it is a tile's latency that counts. A share of the
//           exponentials as polynomials on the FMA pipe: 119 to 123 against 117 us.)
// A tile's rows past the last visible one: their scores are set to -inf before the maximum, P V
// runs over the 16-row steps that hold a visible row, and warp 3 clears the rest of the last
// step's V rows in shared memory (a zero weight does not silence a NaN).
// Every mbarrier wait is bounded as in gemm.cu; after a timeout the softmax warps go through
// their remaining tiles without waiting, so that the halves' named barriers still match, and
// both CTAs meet before either leaves.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "attention.cuh"

namespace yskn {

constexpr int PA_ROWS = 128;    // query rows of a CTA, TMEM lanes
constexpr int PA_KEYS = 128;    // cache rows per tile
constexpr int PA_SLOT = 16384;  // bytes per ring slot
constexpr int PA_THREADS = 384;
constexpr int PA_MAX_PAIRS = 74;
constexpr int PA_MAX_SLOTS = 12;
constexpr int PA_WHOLE_TILES = 1;  // tiles up to which few items are not cut
constexpr int PA_ITEM_COST = 3;    // an item's fixed cost (Q, the last P V's wait, its result) in tiles
// Thin items. Cost, least and time per tile as they served 64 requests best (us behind 32k rows, and
// without a prefix): costs of 1, 3, 5: 100 and 50, 93 and 46, 81 and 41; times of 10, 14, 18 and 22:
// 93, 89, 81, 97. A least of 2 rather than 4: two requests 13.7, not 14.8; of 1: 8 requests 17.2, not 15.7.
// All that at heads of 256 and 6 query heads a KV head. The time per tile at others, us behind 32k rows with 18, 22
// and 28: heads of 128 with 2, 4, 8 query heads 43, 46, 57, then 41, 45, 56, then 41, 43, 54; heads of 64 36, 36, 51,
// then 34, 34, 50, then 33, 33, 48; heads of 256 64, 66, 81, then 64, 65, 100, then 68, 69, 96: one number for all
// costs the smaller heads up to 7 %, a larger one the large heads a fifth.
constexpr int PA_THIN_ROWS = 8;       // rows of a thin item, at most
constexpr int PA_THIN_SHIFT = 4;      // its tiles: 16 rows of the cache
constexpr int PA_THIN_COST = 5;       // its fixed cost in such tiles
constexpr int PA_THIN_LEAST = 2;      // units of a warp, at least
constexpr int PA_THIN_WHOLE = 6;      // tiles up to which few thin items are not cut
constexpr int PA_THIN_PER_TILE = 18;  // thin tiles (two CTAs) in the time of a pair's tile of 128
constexpr int PA_THIN_WARPS = 12;     // warps of a CTA: each takes thin items by itself
constexpr int PA_THIN_STAGE = 16384;  // bytes on the way to one of them
constexpr int PA_MAX_THIN = 2 * PA_MAX_PAIRS * PA_THIN_WARPS;

template <int D>
struct PaShape {
  static constexpr int CHUNKS = D / 64;                     // 64-channel columns of a head
  static constexpr int SLOTS = D <= 128 ? 1 : D / 128;      // ring slots of a K or a V tile (one CTA's half)
  static constexpr int K_CHUNKS = CHUNKS / SLOTS;           // K slot: 64 rows of so many columns
  static constexpr int V_ROWS = PA_KEYS / SLOTS;            // V slot: so many rows
  static constexpr int V_CHUNKS = D <= 128 ? 1 : D / 128;   // of so many columns (D = 64: half a column)
  static constexpr int V_LINE = D == 64 ? 64 : 128;         // bytes of a V row in a column, the swizzle's span
  static constexpr int RING = D == 256 ? 10 : PA_MAX_SLOTS;
  static constexpr int Q_BYTES = CHUNKS * PA_ROWS * 128;
  static constexpr int SMEM = Q_BYTES + RING * PA_SLOT + 3072 /*PaShared*/;
  static constexpr int S_COL = D < 128 ? 128 : D;  // TMEM columns: O at 0, S tiles at S_COL and S_COL + 128
};

// The workspace: sizes from the host's bounds alone, so that both sides agree.
struct PaWork {
  int64_t base, pre_ml, pre_o, own_ml, own_o, bytes;  // byte offsets
  int own_half, own_rows;                                   // rows of a CTA and of the pair in an own item's place
  int64_t own_items;                                        // own items that there is room for
};
inline PaWork pa_work(int tokens, int batch, int max_new, int n_qh, int n_kvh, int head) {
  auto up = [](int64_t v) { return (v + 255) / 256 * 256; };
  max_new = std::min(max_new, tokens);  // a request cannot have more
  const int G = n_qh / n_kvh, tpc = PA_ROWS / G, tpi = 2 * tpc;  // tokens per CTA and per item
  const int64_t pre_items = ceil_div(tokens, tpi) * n_kvh;
  // sum of ceil(n_i / tpi) over requests with n_i > 0: at most one more than n_i / tpi each
  const int64_t own_items = (std::min(batch, tokens) + (int64_t)tokens / tpi) * n_kvh;
  const int64_t pre = pre_items + PA_MAX_PAIRS;
  const int64_t own = own_items + ((int64_t)G * max_new <= PA_THIN_ROWS ? PA_MAX_THIN : PA_MAX_PAIRS);
  PaWork w{};
  w.own_half = G * std::min(tpc, max_new);
  w.own_rows = max_new > tpc ? 2 * w.own_half : w.own_half;
  w.own_items = own_items;
  w.base = 256;
  w.pre_ml = w.base + up((int64_t)batch * 8);
  w.pre_o = w.pre_ml + up(pre * 2 * PA_ROWS * 8);
  w.own_ml = w.pre_o + up(pre * 2 * PA_ROWS * head * 4);
  w.own_o = w.own_ml + up(own * w.own_rows * 8);
  w.bytes = w.own_o + up(own * w.own_rows * head * 4);
  // Smaller calls fit too: those of few rows a KV head have more places, if smaller ones.
  if (G <= PA_THIN_ROWS) {
    const int64_t thin = (own_items + PA_MAX_THIN) * G * std::min(max_new, PA_THIN_ROWS / G);
    w.bytes = std::max(w.bytes, w.own_ml + up(thin * 8) + up(thin * head * 4));
  }
  return w;
}

struct PrefixAttnParams {
  const void* gate;  // of the queries' type, or f32
  int64_t gate_row, gate_head;
  bool gate_f32;
  const int32_t* prefix_blocks;
  const int32_t* tables;
  int64_t table_stride;
  const int32_t *lens, *starts;
  int n_blocks, block_shift, prefix_len;  // blocks of 1 << block_shift rows
  int own_limit;  // rows that a table row can name
  int batch, tokens, max_new, n_kvh, G;
  int tpc, tpi;  // tokens per CTA and per item
  unsigned g_magic, tpi_magic;  // ceil(2^32 / d): quotients of numbers below 2^32 / d
  int pre_qtiles, shared_items;  // prefix items, if there are any
  // Own items: thin ones (below) or not, the rows of a tile as a power of two, and an item's fixed
  // cost in tiles.
  bool thin;
  int tile_shift, item_cost;
  const uint16_t *q, *k_cache, *v_cache;  // thin items read them by address
  int64_t q_row, q_head;
  CacheStrides cache;
  bool whole;  // items are not cut: no join
  int join_span, join_split;  // 16-channel parts of a row that a warp of the join takes; warps for one part
  float c;     // |scale| log2 e
  uint32_t negate_q;
  int4* work_per;  // for the join: units per pair of prefix items and of own ones, prefix tiles (-1: alone), own units
  int2* work_base;        // [batch] own items, and units of all items, before each request's own
  // per place: (m, l) of each row; o as [D / 4][rows][4], so that a warp's rows are adjacent
  float2 *pre_ml, *own_ml;
  float *pre_o, *own_o;
  int own_half, own_rows;
  unsigned many_per_head;  // PA_MANY / n_kvh
  long long own_items;  // more of them (starts that do not ascend), or 2^30 own units, is an error: nothing is computed
  uint16_t* out;  // [tokens][n_qh][D]
  unsigned* err;
};

// n / d by its magic number (0 for d = 1).
__device__ __forceinline__ int pa_quotient(int n, unsigned magic) {
  return magic ? (int)__umulhi((unsigned)n, magic) : n;
}

// The last request whose first token is at or before t (requests without tokens share a
// start with the next one), or the batch if t is past the last token. One token for each
// request is the common case: looked at first.
__device__ __forceinline__ int request_of(const int32_t* starts, int batch, int t) {
  if (t < batch && __ldg(starts + t) == t && __ldg(starts + t + 1) == t + 1) return t;
  if (t >= __ldg(starts + batch)) return batch;
  int lo = 0, hi = batch;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(starts + mid) <= t) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Request i: its first token, its tokens (0 if there are none, or not what the host bounded)
// and its length.
struct PaRequest {
  int s0, n, len;
};
__device__ __forceinline__ PaRequest pa_request(const PrefixAttnParams& p, int i) {
  PaRequest r;
  r.s0 = __ldg(p.starts + i);
  const int n = (int)((unsigned)__ldg(p.starts + i + 1) - (unsigned)r.s0);  // whatever the two are
  r.len = __ldg(p.lens + i);
  r.n = n < 0 || n > p.max_new || r.s0 < 0 || r.s0 > p.tokens - n ? 0 : n;
  return r;
}
// Own rows that the last of the request's first `upto` tokens sees.
__device__ __forceinline__ int pa_visible(const PrefixAttnParams& p, const PaRequest& r, int upto) {
  return min(max(r.len - r.n + upto - p.prefix_len, 0), p.own_limit);
}
// Rows of the prefix that it sees.
__device__ __forceinline__ int pa_visible_prefix(const PrefixAttnParams& p, const PaRequest& r, int upto) {
  return min(max(r.len - r.n + upto, 0), p.prefix_len);
}
// Units of an item of so many tiles (0: nothing to do): unit u is tile u - cost; or the whole
// item is one unit.
__host__ __device__ __forceinline__ int pa_units(int tiles, bool whole, int cost) {
  return tiles <= 0 ? 0 : whole ? 1 : tiles + cost;
}
__device__ __forceinline__ int pa_qtiles(const PrefixAttnParams& p, const PaRequest& r) {
  return r.n <= p.tpi ? r.n > 0 : pa_quotient(r.n + p.tpi - 1, p.tpi_magic);
}
// Tiles of a request's item `qt`: own ones, after the prefix's where there are no prefix items.
__device__ __forceinline__ int pa_tiles(const PrefixAttnParams& p, const PaRequest& r, int qt, bool alone) {
  const int upto = min(r.n, (qt + 1) * p.tpi), up = (1 << p.tile_shift) - 1;
  const int own = (pa_visible(p, r, upto) + up) >> p.tile_shift;
  return alone ? own + ((pa_visible_prefix(p, r, upto) + up) >> p.tile_shift) : own;
}
// Units of a request's items of one KV head; sums of units stop at PA_MANY, which is an error.
constexpr unsigned PA_MANY = 1u << 30;
__device__ __forceinline__ unsigned pa_sum(unsigned a, unsigned b) { return min(a + b, PA_MANY); }
__device__ __forceinline__ unsigned pa_own_units(const PrefixAttnParams& p, const PaRequest& r, int nq, bool alone) {
  unsigned u = 0;
  for (int q = 0; q < nq; ++q) u = pa_sum(u, pa_units(pa_tiles(p, r, q, alone), p.whole, p.item_cost));
  return u;
}

struct PaSegment {
  bool prefix, whole;   // prefix item; all that its rows see
  int kvh, tok0, ntok;  // KV head, first token and whole tokens
  int req;              // own items: the request
  int pre;              // the item's first tiles that are the prefix's
  int key0, key1;       // key tiles [key0, key1)
  int keys;             // own rows that any of its tokens sees
  int first;            // rows of the sequence that token tok0 sees, one more for each token (prefix
                        // items: as if its last token saw what the longest request does)
  int64_t place;        // of its partial result
  // Rows of the prefix that any of its tokens sees.
  __device__ int pre_keys(const PrefixAttnParams& p) const { return min(first + ntok - 1, p.prefix_len); }
  // Rows of tile kt that the rows on its axis leave it.
  __device__ int rows_of(const PrefixAttnParams& p, int kt) const {
    return min(PA_KEYS, kt < pre ? pre_keys(p) - kt * PA_KEYS : keys - (kt - pre) * PA_KEYS);
  }
};

// Where a pair's units begin, found by each of its CTAs.
struct PaStart {
  int who;           // this pair, or this warp of those that take thin items
  bool thin;         // the latter
  bool sound;        // false: more items than there is room for, nothing is computed
  int left;          // its units
  int alone;         // no prefix items: each request's items take the prefix too
  int pre_seen;      // rows of the prefix that any token of the call sees
  int pre_item, u0;  // prefix item and unit in it
  int req, item;     // own items: request and the items before it
  int skip;          // units of the request before this pair's first
};

// The pair's segments in order; every lane of a warp walks alike.
struct PaWalk {
  const PrefixAttnParams& p;
  const bool alone;
  const int who, pre_seen;
  int left, pre_item, u0, req, item, kvh, qt;
  PaRequest r;
  int nq;
  bool loaded;
  __device__ PaWalk(const PrefixAttnParams& p_, const PaStart& s)
      : p(p_), alone(s.alone), who(s.who), pre_seen(s.pre_seen), left(s.left), pre_item(s.pre_item), u0(s.u0), req(s.req), item(s.item),
        kvh(0), qt(0), r{}, nq(0), loaded(false) {
    if (s.skip > 0) {
      load();
      const int head = (int)pa_own_units(p, r, nq, alone);
      kvh = s.skip / head;
      int skip = s.skip - kvh * head;
      for (;; ++qt) {
        const int u = pa_units(pa_tiles(p, r, qt, alone), p.whole, p.item_cost);
        if (skip < u) break;
        skip -= u;
      }
      u0 = skip;
    }
  }
  __device__ void load() {
    r = pa_request(p, req);
    nq = pa_qtiles(p, r);
    loaded = true;
  }
  // The next segment; false past the last.
  __device__ bool next(PaSegment& s) {
    while (left > 0 && !alone && pre_item < p.shared_items) {
      s.prefix = true;
      s.kvh = p.pre_qtiles == 1 ? pre_item : pre_item / p.pre_qtiles;
      s.tok0 = (pre_item - s.kvh * p.pre_qtiles) * p.tpi;
      s.ntok = min(p.tpi, p.tokens - s.tok0);
      s.req = 0;
      s.pre = (pre_seen + PA_KEYS - 1) / PA_KEYS;
      s.keys = 0;
      s.first = pre_seen - s.ntok + 1;
      ++pre_item;
      if (take(s, s.pre, pre_item - 1)) return true;
    }
    while (left > 0 && req < p.batch) {
      if (!loaded) load();
      for (; kvh < p.n_kvh; ++kvh, qt = 0)
        while (qt < nq) {
          const int q = qt++, kt = pa_tiles(p, r, q, alone);
          if (kt == 0) continue;
          s.prefix = false;
          s.kvh = kvh;
          s.tok0 = r.s0 + q * p.tpi;
          s.ntok = min(p.tpi, r.n - q * p.tpi);
          s.req = req;
          s.keys = pa_visible(p, r, q * p.tpi + s.ntok);
          s.pre = kt - ((s.keys + (1 << p.tile_shift) - 1) >> p.tile_shift);
          s.first = r.len - r.n + q * p.tpi + 1;
          if (take(s, kt, item + kvh * nq + q)) return true;
          if (left <= 0) return false;
        }
      item += p.n_kvh * nq;
      ++req;
      kvh = qt = 0;
      loaded = false;
    }
    return false;
  }
  // This pair's part of an item; false if it holds no tile.
  __device__ bool take(PaSegment& s, int tiles, int it) {
    const int cost = s.prefix ? PA_ITEM_COST : p.item_cost;
    const int n = p.whole ? 1 : min(tiles + cost - u0, left);
    s.key0 = p.whole ? 0 : max(u0 - cost, 0);
    s.key1 = p.whole ? tiles : max(u0 + n - cost, 0);
    s.whole = !s.prefix && s.key0 == 0 && s.key1 == tiles && alone;
    s.place = (int64_t)it + who;
    left -= n;
    u0 = 0;
    return s.key0 < s.key1;
  }
};

// Four of the output gate's channels from element `at` on, as they are stored, and as f32: apart, so
// that several loads are under way before the first is waited for.
__device__ __forceinline__ uint4 gate_load(const PrefixAttnParams& p, int64_t at) {
  if (p.gate_f32) return __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const float*>(p.gate) + at));
  const uint2 g = __ldg(reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(p.gate) + at));
  return make_uint4(g.x, g.y, 0, 0);
}
template <int DT>
__device__ __forceinline__ float4 gate_value(const PrefixAttnParams& p, uint4 g) {
  if (p.gate_f32)
    return make_float4(__uint_as_float(g.x), __uint_as_float(g.y), __uint_as_float(g.z), __uint_as_float(g.w));
  return make_float4(Elem<DT>::to_float((uint16_t)g.x), Elem<DT>::to_float((uint16_t)(g.x >> 16)),
                     Elem<DT>::to_float((uint16_t)g.y), Elem<DT>::to_float((uint16_t)(g.y >> 16)));
}
// Both warps of a row quarter.
__device__ __forceinline__ void quarter_sync(int quarter) {
  asm volatile("bar.sync %0, 64;" ::"r"(1 + quarter) : "memory");
}

// Where no join visits every row: zeros for this CTA's share of the tokens that no item holds (all, where
// nothing is computed). One warp; each lane looks at a token.
template <int D>
__device__ __forceinline__ void zero_unheld(const PrefixAttnParams& p, bool sound, int lane) {
  for (int t0 = blockIdx.x * 32; t0 < p.tokens; t0 += gridDim.x * 32) {
    const int t = t0 + lane;
    bool bare = t < p.tokens;
    if (bare && sound) {
      const int i = request_of(p.starts, p.batch, t);
      const PaRequest r = i < p.batch ? pa_request(p, i) : PaRequest{};
      bare = t < r.s0 || t >= r.s0 + r.n || pa_tiles(p, r, pa_quotient(t - r.s0, p.tpi_magic), true) == 0;
    }
    for (unsigned left = __ballot_sync(0xffffffffu, bare); left; left &= left - 1) {
      uint4* row = reinterpret_cast<uint4*>(p.out + (int64_t)(t0 + __ffs(left) - 1) * p.n_kvh * p.G * D);
      for (int x = lane; x < p.n_kvh * p.G * D / 8; x += 32) row[x] = make_uint4(0, 0, 0, 0);
    }
  }
}

// ---- thin items: up to 8 rows (one token of up to 8 query heads a KV head, or a few of fewer)
// against the request's own rows. 256 rows of MMA for 6 are 2048 clocks a tile for work that the
// memory bounds, and an item's Q, S, P, O pass through one after another (64 requests of up to 1024
// own rows, no prefix: 74 us for 142 MB; thin 41, of which the join is 7). Here each warp takes a run of
// 16-row slices by itself, with warp-level MMAs (m16n8k16): no barrier. What bounds it: bytes, so
// the copies run a ring of 8 chunks (16 rows of 64 channels of K or V) ahead, across items, 192 KB an SM
// (in steady state 6.6 TB/s; the rest is the start, a warp's last slices and the join).
//   S = Q K^T   A: Q, rows 0..7 (8..15 zero); B: K, of a lane (g, t) the 16-byte units t and t + 4 of
//               row g in a chunk: steps of 16 channels in an order that Q's registers share;
//   O^T = V^T P^T  B: P^T, which is S as it left the first MMA (row g, keys 2t, 2t + 1, 2t + 8 and
//               2t + 9); A: V^T, of a lane unit g of those four rows: word w's two channels of two
//               rows by one byte permutation each, rows g and g + 8 of MMA w.
// (Eight warps on one item, joined in shared memory at its end: 71 us where one each takes 54, both with
// the copies of that step; the MMAs are 5 % of it.)
// A chunk's rows are 128 bytes; 8 lanes bring one (lanes that fetch just what they need later,
// 64 or 32 bytes of a line a request, had the L2 answer 1.3 sectors a request: 54 us, not 47). The
// 16-byte unit c of row r lies at c ^ (4 (r2 ^ r0) + 2 r1), r's low bits, where both reads find their
// 8 lanes on 8 different units.
template <int DT>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  if constexpr (DT == YSKN_DT_BF16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, "
        "%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, "
        "%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 16 bytes into shared memory, or zeros.
__device__ __forceinline__ void copy16(uint32_t to, const uint16_t* from, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ uint4 stage_load(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(at)
               : "memory");
  return v;
}

// The rows that this warp's copies are at. Each segment that it comes to goes into the warp's queue in
// shared memory, from which the arithmetic takes it: at most LEAD + 2 slices later.
constexpr int PA_THIN_QUEUE = 8;
struct ThinCursor {
  const PrefixAttnParams& p;
  PaWalk walk;
  PaSegment seg;
  PaSegment* queue;
  int found;  // segments put into it
  int kt;
  bool live;
  int block;  // of slice kt: asked for one slice ahead
  const uint16_t *k, *v;  // the slice that is being copied, and how many of its rows there are
  int rows;
  __device__ ThinCursor(const PrefixAttnParams& p_, const PaStart& s, PaSegment* queue_)
      : p(p_), walk(p_, s), queue(queue_), found(0), kt(0), live(true), block(0), k(nullptr), v(nullptr), rows(0) {
    seg.key1 = 0;
    advance();
  }
  __device__ void advance() {
    if (++kt >= seg.key1 && live) {
      live = walk.next(seg);  // a segment holds a slice
      kt = seg.key0;
      if (live) {
        if ((threadIdx.x & 31) == 0) queue[found % PA_THIN_QUEUE] = seg;
        __syncwarp();
        ++found;
      }
    }
    if (live) {
      const int at = (kt < seg.pre ? kt : kt - seg.pre) << PA_THIN_SHIFT >> p.block_shift;
      block = __ldg(kt < seg.pre ? p.prefix_blocks + at : p.tables + (int64_t)seg.req * p.table_stride + at);
    }
  }
  // To the next slice's rows.
  __device__ void next() {
    rows = 0;
    k = p.k_cache, v = p.v_cache;
    if (!live) return;
    const int at = (kt < seg.pre ? kt : kt - seg.pre) << PA_THIN_SHIFT;
    if ((unsigned)block < (unsigned)p.n_blocks) {
      rows = min(1 << PA_THIN_SHIFT, (kt < seg.pre ? seg.pre_keys(p) : seg.keys) - at);
      const int64_t from = block * p.cache.block + (at & ((1 << p.block_shift) - 1)) * p.cache.token +
                           seg.kvh * p.cache.head;
      k += from, v += from;
    } else {
      raise_device_error(p.err, DERR_RANGE);  // the copies give zeros
    }
    advance();
  }
};

template <int D, int DT>
__device__ __forceinline__ void thin_items(const PrefixAttnParams& p, const PaStart& start, uint8_t* smem, int warp,
                                           int lane) {
  constexpr int C = D / 64, CHUNKS = 2 * C;  // chunks of a slice's K; of K and V
  constexpr int LEAD = 8 / CHUNKS;           // slices on the way
  static_assert(PaShape<D>::Q_BYTES + PaShape<D>::RING * PA_SLOT >=
                    PA_THIN_WARPS * (PA_THIN_STAGE + PA_THIN_QUEUE * (int)sizeof(PaSegment)) &&
                    LEAD + 2 < PA_THIN_QUEUE,
                "the warps' rings and queues");
  const uint32_t mine = smem_u32(smem + warp * PA_THIN_STAGE);
  const int g = lane >> 2, t = lane & 3;
  const float c = p.negate_q ? -p.c : p.c;
  const int64_t tok = p.cache.token;
  PaSegment* queue = reinterpret_cast<PaSegment*>(smem + PA_THIN_WARPS * PA_THIN_STAGE) + warp * PA_THIN_QUEUE;
  ThinCursor from(p, start, queue);
  // Chunk x of the slice that the cursor is at, into place `at` of the ring.
  const int row0 = lane >> 3, unit = lane & 7;
  const uint32_t put = row0 * 128 + (unit ^ ((row0 & 1) << 2) ^ (row0 & 2)) * 16;
  auto copy = [&](int x, uint32_t at) {
    const uint16_t* src = (x < C ? from.k + 64 * x : from.v + 64 * (x - C)) + row0 * tok + 8 * unit;
#pragma unroll
    for (int u = 0; u < 4; ++u) {  // rows 4 u + row0
      const bool valid = 4 * u + row0 < from.rows;
      copy16(at + u * 512 + (put ^ ((u & 1) << 6)), valid ? src + 4 * u * tok : p.k_cache, valid);
    }
  };
  // where this lane reads: rows g and g + 8 of K, units t and t + 4; rows 2t, 2t + 1, 2t + 8 and
  // 2t + 9 of V, unit g
  const uint32_t get_k = g * 128 + (t ^ (((g >> 2 ^ g) & 1) << 2) ^ (g & 2)) * 16;
  const uint32_t get_v = 2 * t * 128 + (g ^ ((t >> 1) << 2) ^ ((t & 1) << 1)) * 16;
  auto commit = [] { asm volatile("cp.async.commit_group;" ::: "memory"); };
  const int tl = pa_quotient(g, p.g_magic);  // row g's token
  uint4 q[2 * C];
  auto load_q = [&](const PaSegment& seg) {
    const int h = seg.kvh * p.G + g - tl * p.G;
#pragma unroll
    for (int x = 0; x < 2 * C; ++x) {
      q[x] = make_uint4(0, 0, 0, 0);
      if (g < seg.ntok * p.G)
        q[x] = __ldg(reinterpret_cast<const uint4*>(p.q + (seg.tok0 + tl) * p.q_row + h * p.q_head + 32 * x + 8 * t));
    }
  };
  if (from.found > 0) load_q(queue[0]);  // ahead of the copies, behind which it would wait for microseconds
#pragma unroll 1
  for (int i = 0; i < LEAD; ++i) {
    from.next();
#pragma unroll
    for (int x = 0; x < CHUNKS; ++x) copy(x, mine + (i * CHUNKS + x) * 2048), commit();
  }
  int turn = 0;  // the slice's place in the ring
  for (int taken = 0; taken < from.found;) {
    const PaSegment& seg = queue[taken % PA_THIN_QUEUE];
    const int n_rows = seg.ntok * p.G, sees = seg.first + tl;  // rows of the sequence that row g sees
    float o[C][4][4];
#pragma unroll
    for (int x = 0; x < C * 16; ++x) o[x / 16][x / 4 % 4][x % 4] = 0.0f;
    float m = -INFINITY, l = 0.0f;
#pragma unroll 1
    for (int kt = seg.key0, end = seg.key1; kt < end; ++kt) {
      from.next();
      const uint32_t at = mine + turn * (CHUNKS * 2048);
      float s[4][4];  // 8 keys; even and odd steps apart
#pragma unroll
      for (int x = 0; x < 16; ++x) s[x / 4][x % 4] = 0.0f;
#pragma unroll
      for (int x = 0; x < C; ++x) {
        asm volatile("cp.async.wait_group 7;" ::: "memory");
        __syncwarp();
        uint4 k[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) k[u] = stage_load(at + x * 2048 + (u >> 1) * 1024 + (get_k ^ ((u & 1) << 6)));
        __syncwarp();
        copy(x, at + x * 2048), commit();
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const uint4 a = q[2 * x + (u & 1)];
          mma16816<DT>(s[u >> 1], a.x, 0, a.y, 0, k[u].x, k[u].y);
          mma16816<DT>(s[2 + (u >> 1)], a.z, 0, a.w, 0, k[u].z, k[u].w);
        }
      }
      // row g, keys 2t, 2t + 1, 2t + 8, 2t + 9
      const bool pre = kt < seg.pre;
      const int first = (pre ? kt : kt - seg.pre) << PA_THIN_SHIFT;
      const int seen = min((pre ? p.prefix_len : seg.keys) - first, sees - first - (pre ? 0 : p.prefix_len)) - 2 * t;
      float z[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        z[x] = (s[x >> 1][x & 1] + s[2 + (x >> 1)][x & 1]) * c;
        if ((x & 1) + 8 * (x >> 1) >= seen) z[x] = -INFINITY;
      }
      float top = fmaxf(fmaxf(z[0], z[1]), fmaxf(z[2], z[3]));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const bool grown = top > m + 8.0f;  // the maximum may lag by 2^8
      if (__any_sync(0xffffffffu, grown)) {
        const float f = grown ? exp2_approx(m - top) : 1.0f;
        const float f0 = __shfl_sync(0xffffffffu, f, 8 * t), f1 = __shfl_sync(0xffffffffu, f, 8 * t + 4);
#pragma unroll
        for (int x = 0; x < C * 4; ++x) {
          float(&y)[4] = o[x / 4][x % 4];
          y[0] *= f0, y[1] *= f1, y[2] *= f0, y[3] *= f1;
        }
        l *= f;
        if (grown) m = top;
      }
      const float base = m == -INFINITY ? 0.0f : m;
#pragma unroll
      for (int x = 0; x < 4; ++x) z[x] = exp2_approx(z[x] - base);
      l += (z[0] + z[1]) + (z[2] + z[3]);
      const uint32_t b0 = Elem<DT>::pack(z[0], z[1]), b1 = Elem<DT>::pack(z[2], z[3]);
#pragma unroll
      for (int x = 0; x < C; ++x) {
        asm volatile("cp.async.wait_group 7;" ::: "memory");
        __syncwarp();
        uint32_t v[4][4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const uint4 y =
              stage_load(at + (C + x) * 2048 + (u >> 1) * 1024 + (u & 1) * 128 + (get_v ^ ((u & 1) << 6)));
          v[u][0] = y.x, v[u][1] = y.y, v[u][2] = y.z, v[u][3] = y.w;
        }
        __syncwarp();
        copy(C + x, at + (C + x) * 2048), commit();
#pragma unroll
        for (int w = 0; w < 4; ++w)
          mma16816<DT>(o[x][w], __byte_perm(v[0][w], v[1][w], 0x5410), __byte_perm(v[0][w], v[1][w], 0x7632),
                       __byte_perm(v[2][w], v[3][w], 0x5410), __byte_perm(v[2][w], v[3][w], 0x7632), b0, b1);
      }
      if (++turn == LEAD) turn = 0;
    }
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    if (seg.whole) {
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
      for (int y = 0; y < 2; ++y) {  // row 2t + y: channels 64 x + 8 g + 0..7
        const int row = 2 * t + y, rt = pa_quotient(row, p.g_magic), rh = seg.kvh * p.G + row - rt * p.G;
        const float f = __shfl_sync(0xffffffffu, inv, 8 * t + 4 * y);
        if (row >= n_rows) continue;
        const int64_t tk = seg.tok0 + rt;
        uint16_t* out = p.out + (tk * p.n_kvh * p.G + rh) * D + 8 * g;
        const int64_t gate = tk * p.gate_row + rh * p.gate_head + 8 * g;
#pragma unroll
        for (int x = 0; x < C; ++x) {
          float e[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) e[k] = o[x][k / 2][y + 2 * (k % 2)] * f;
          if (p.gate) {
            const float4 a = gate_value<DT>(p, gate_load(p, gate + 64 * x));
            const float4 d = gate_value<DT>(p, gate_load(p, gate + 64 * x + 4));
            const float gs[8] = {a.x, a.y, a.z, a.w, d.x, d.y, d.z, d.w};
#pragma unroll
            for (int k = 0; k < 8; ++k) e[k] = f == 0.0f ? 0.0f : gated(e[k], gs[k]);
          }
          *reinterpret_cast<uint4*>(out + 64 * x) = make_uint4(Elem<DT>::pack(e[0], e[1]), Elem<DT>::pack(e[2], e[3]),
                                                               Elem<DT>::pack(e[4], e[5]), Elem<DT>::pack(e[6], e[7]));
        }
      }
    } else {
      const int64_t at = seg.place * p.own_rows;
      if (t == 0 && g < n_rows) p.own_ml[at + g] = make_float2(m, l);
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        if (2 * t + y >= n_rows) continue;
        float4* to = reinterpret_cast<float4*>(p.own_o + at * D) + 2 * g * p.own_rows + 2 * t + y;
#pragma unroll
        for (int x = 0; x < C; ++x) {
          to[16 * x * p.own_rows] = make_float4(o[x][0][y], o[x][0][2 + y], o[x][1][y], o[x][1][2 + y]);
          to[(16 * x + 1) * p.own_rows] = make_float4(o[x][2][y], o[x][2][2 + y], o[x][3][y], o[x][3][2 + y]);
        }
      }
    }
    if (++taken < from.found) load_q(queue[taken % PA_THIN_QUEUE]);
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

// Shared memory beside Q and the ring. "First": only the first CTA's copy is used.
struct PaShared {
  uint64_t full[PA_MAX_SLOTS];   // ring place landed in both CTAs (first)
  uint64_t empty[PA_MAX_SLOTS];  // ring place read
  uint64_t q_full, q_empty;      // Q landed in both CTAs (first), read
  uint64_t s_full[2], pv_done[2];  // by tile parity: S written, P V done
  uint64_t p_full[2];              // P written by both CTAs (first)
  uint64_t o_free;                 // O read by both CTAs (first)
  uint64_t drained, tail_full, tail_done;
  int2 tail_at;
  uint32_t tmem_slot;
  int abort_word;
  PaStart start[PA_THIN_WARPS];  // of the pair's walk (all alike), or of each warp's
  uint4 sum[PA_THREADS / 32];
  float half[2][2][PA_ROWS];  // tile parity, half, row: what a row's halves exchange
};
static_assert(sizeof(PaShared) <= 3072, "shared memory beside the ring");

template <int D, int DT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(PA_THREADS, 1)
    prefix_attention_kernel(const __grid_constant__ CUtensorMap map_q_pre, const __grid_constant__ CUtensorMap map_q_own,
                            const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                            const __grid_constant__ PrefixAttnParams p) {
  using Shape = PaShape<D>;
  constexpr int RING = Shape::RING, SLOTS = Shape::SLOTS, VR = Shape::V_ROWS;
  extern __shared__ __align__(1024) uint8_t smem[];  // swizzled tiles start on 1024 bytes
  uint8_t* sQ = smem;                     // [D / 64][128 rows][128 B]
  uint8_t* ring = smem + Shape::Q_BYTES;  // [RING][16 KB]
  PaShared& sh = *reinterpret_cast<PaShared*>(ring + RING * PA_SLOT);
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
  if (warp == 2 && lane < 4 && (!p.thin || p.shared_items > 0)) {
    const CUtensorMap* map = lane == 0 ? &map_q_pre : lane == 1 ? &map_q_own : lane == 2 ? &map_k : &map_v;
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // both CTAs' barriers are set up
  tc_fence_after();
  pdl_begin();

  // Unit counts of all requests and where this pair begins. A thread's requests are adjacent.
  {
    const int per = p.batch <= PA_THREADS ? 1 : (p.batch + PA_THREADS - 1) / PA_THREADS;
    const int i0 = min(p.batch, tid * per), i1 = min(p.batch, i0 + per);
    unsigned items = 0, units_of[2] = {0, 0}, seen = 0;  // beside prefix items, and alone; of the prefix
    for (int i = i0; i < i1; ++i) {
      const PaRequest r = pa_request(p, i);
      const int nq = pa_qtiles(p, r);
      auto times = [&](unsigned n) { return n > p.many_per_head ? PA_MANY : n * p.n_kvh; };
      units_of[0] = pa_sum(units_of[0], times(pa_own_units(p, r, nq, false)));
      units_of[1] = pa_sum(units_of[1], times(pa_own_units(p, r, nq, true)));
      items = pa_sum(items, times(nq));
      if (r.n > 0) seen = max(seen, (unsigned)pa_visible_prefix(p, r, r.n));
      if (blockIdx.x == 0 && (__ldg(p.starts + i + 1) != r.s0 + r.n ||
                              (r.n > 0 && r.len > p.prefix_len && r.len - p.prefix_len > p.own_limit)))
        raise_device_error(p.err, DERR_RANGE);
    }
    unsigned ui[2] = {units_of[0], units_of[1]}, it = items;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const unsigned a = __shfl_up_sync(0xffffffffu, ui[0], off), b = __shfl_up_sync(0xffffffffu, ui[1], off);
      const unsigned c = __shfl_up_sync(0xffffffffu, it, off);
      if (lane >= off) ui[0] = pa_sum(ui[0], a), ui[1] = pa_sum(ui[1], b), it = pa_sum(it, c);
    }
    seen = __reduce_max_sync(0xffffffffu, seen);
    if (lane == 31) sh.sum[warp] = make_uint4(ui[0], ui[1], it, seen);
    __syncthreads();
    unsigned before_of[2] = {0, 0}, total_of[2] = {0, 0}, items_before = 0, total_items = 0;
    const int used = per == 1 ? p.batch : PA_THREADS;  // threads with requests
    for (int w = 0; w * 32 < used; ++w) {
      const uint4 o = sh.sum[w];
      seen = max(seen, o.w);
      if (w < warp) {
        before_of[0] = pa_sum(before_of[0], o.x);
        before_of[1] = pa_sum(before_of[1], o.y);
        items_before = pa_sum(items_before, o.z);
      }
      total_of[0] = pa_sum(total_of[0], o.x);
      total_of[1] = pa_sum(total_of[1], o.y);
      total_items = pa_sum(total_items, o.z);
    }
    // Alone, if that is at most an eighth more: about what the join of two results per row costs
    // (16 prompt chunks: 960 us with prefix items, 850 alone, at the step that added it).
    const int pre_tiles = (int)(seen + PA_KEYS - 1) / PA_KEYS, pre_units = pa_units(pre_tiles, false, PA_ITEM_COST);
    const int pre_all = p.shared_items * pre_units;  // below 2^30: the host looked
    const unsigned long long pre_time = (unsigned long long)pre_all * (p.thin ? PA_THIN_PER_TILE : 1);
    const bool alone = p.whole || p.shared_items == 0 ||
                       (total_of[1] < PA_MANY && 8ull * total_of[1] <= 9ull * (pre_time + total_of[0]));
    const unsigned units = alone ? units_of[1] : units_of[0], total = alone ? total_of[1] : total_of[0];
    const unsigned before =
        alone ? pa_sum(before_of[1], ui[1] - units_of[1]) : pa_sum(before_of[0], ui[0] - units_of[0]);
    items_before = pa_sum(items_before, it - items);
    const bool sound = total_items <= (unsigned)p.own_items && total < PA_MANY;
    const int pre_items = alone ? 0 : p.shared_items, pre = alone || !sound ? 0 : pre_all;
    const int own = sound ? (int)total : 0;
    // Without thin items, the pairs share prefix units and then own ones as one line. With them, the
    // first pairs take the prefix items, as many as their part of the time, and each warp of the
    // other pairs a share of the thin ones.
    int tc = pairs, share_pre, share_own;
    if (!p.thin) {
      const int all = pre + own;
      share_pre = pairs == PA_MAX_PAIRS ? (all + PA_MAX_PAIRS - 1) / PA_MAX_PAIRS : (all + pairs - 1) / pairs;
      share_own = share_pre;
    } else {
      if (pre == 0) tc = 0;
      else if (own > 0)
        tc = min(max((int)((float)pairs * (float)pre_time / ((float)pre_time + (float)own) + 0.5f), 1), pairs - 1);
      const int warps = 2 * PA_THIN_WARPS * (pairs - tc);
      share_pre = tc > 0 ? (pre + tc - 1) / tc : 0;
      share_own = warps > 0 && own > 0 ? max((own + warps - 1) / warps, p.whole ? 1 : PA_THIN_LEAST) : 0;
    }
    const bool thin = pair >= tc;  // this pair's CTAs
    // a CTA's first thin warp, and from each to its next (neighbours are on different SMs: where there
    // are few units, every SM has some)
    const int ctas = 2 * (pairs - tc), who0 = thin ? blockIdx.x - 2 * tc : pair;
    if (tid < PA_THIN_WARPS) {
      const int who = who0 + (thin ? tid * ctas : 0), share = thin ? share_own : share_pre;
      const int all = thin ? own : p.thin ? pre : pre + own, t0 = min(all, who * share);
      PaStart s{who,       thin, sound, min(all, t0 + share) - t0,        alone, (int)seen,
                pre_items, 0,    p.thin && !thin ? p.batch : 0, 0,     0};
      if (!thin && t0 < pre) {
        s.pre_item = t0 / pre_units;
        s.u0 = t0 - s.pre_item * pre_units;
      }
      sh.start[tid] = s;
      if (blockIdx.x == 0 && tid == 0) {
        *p.work_per = make_int4(share_pre, share_own, alone ? -1 : pre_tiles, own);
        if (!sound) raise_device_error(p.err, DERR_RANGE);
      }
    }
    __syncthreads();
    // the walks that begin inside this thread's requests: walk x begins at own unit first + x step
    const int step = ctas * share_own;
    const int walks = thin ? PA_THIN_WARPS : p.thin ? 0 : 1, first = who0 * share_own - (p.thin ? 0 : pre);
    const int last = first + (walks - 1) * step;
    if (sound && (blockIdx.x == 0 || (units > 0 && last >= (int)before && first < (int)(before + units)))) {
      int b = (int)before, item = (int)items_before;
      for (int i = i0; i < i1; ++i) {
        int u = (int)units, n = (int)items;
        if (per > 1) {
          const PaRequest r = pa_request(p, i);
          n = pa_qtiles(p, r);
          u = (int)pa_own_units(p, r, n, alone) * p.n_kvh;
          n *= p.n_kvh;
        }
        for (int x = 0; x < walks; ++x) {
          const int at = first + x * step;
          if (at >= b && at < b + u) {
            PaStart& s = sh.start[thin ? x : 0];
            s.req = i, s.item = item, s.skip = at - b;
          }
        }
        if (blockIdx.x == 0) p.work_base[i] = make_int2(item, p.thin ? b : pre + b);
        b += u;
        item += n;
      }
    }
  }
  __syncthreads();
  const uint32_t tmem = sh.tmem_slot;
  if (sh.start[0].thin) {
    if (p.whole && warp == PA_THIN_WARPS - 1) zero_unheld<D>(p, sh.start[0].sound, lane);
    thin_items<D, DT>(p, sh.start[warp], smem, warp, lane);
  } else {
    PaWalk walk(p, sh.start[0]);
    PaSegment seg;

    if (warp == 0) {
      // ---- K and V through the ring, in the order in which the MMAs use them: this CTA's half of
      // each tile's K rows, and of V's channels
      int s = 0;          // the ring's place
      uint32_t turn = 1;  // parity of a place's last reading (first round: already free)
      uint32_t tails = 0;
      bool ok = true;
      const int shift = p.block_shift, pages = PA_KEYS >> shift;
      const int box_k = min(1 << shift, PA_KEYS / 2), box_v = min(1 << shift, VR);
      const uint32_t full0 = first_cta(&sh.full[0]);
      const int v_chunk = D == 64 ? 0 : rank * Shape::V_CHUNKS, v_x = D == 64 ? rank * 32 : 0;
      while (ok && walk.next(seg)) {
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
          ok = __all_sync(0xffffffffu, mbar_wait(&sh.empty[s], turn, abort_flag));
          return ring + s * PA_SLOT;
        };
        auto advance = [&]() {
          if (++s == RING) s = 0, turn ^= 1;
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
          const int nk = min(max(seg.rows_of(p, kt) - rank * (PA_KEYS / 2), 0), PA_KEYS / 2);
          const int n = (nk + box_k - 1) / box_k;
          for (int d = 0; ok && d < SLOTS; ++d) {
            uint8_t* to = claim();
            if (!ok) break;
            const uint32_t bar = full0 + 8 * s;
            if (lane == 0) expect_first(bar, (uint32_t)(n * box_k * 128 * Shape::K_CHUNKS));
            __syncwarp();
            copy(to, &map_k, bar, rank * (PA_KEYS / 2), n, box_k, PA_KEYS / 2, 0, d * Shape::K_CHUNKS, Shape::K_CHUNKS,
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
            uint32_t bar = full0 + 8 * s;
            const uint32_t bytes = (uint32_t)(n * box_v) * Shape::V_LINE * Shape::V_CHUNKS;
            if (rows & 15) {  // lands on this CTA's barrier; warp 3 clears the end and then arrives
              if (tails > 0) ok = __all_sync(0xffffffffu, mbar_wait(&sh.tail_done, (tails - 1) & 1, abort_flag));
              if (!ok) break;
              ++tails;
              if (lane == 0) {
                sh.tail_at = make_int2(s, rows);
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
      if (ok && tails > 0) ok = __all_sync(0xffffffffu, mbar_wait(&sh.tail_done, (tails - 1) & 1, abort_flag));
      if (ok && lane == 0) {
        sh.tail_at = make_int2(0, 0);  // no more of them
        mbar_arrive(&sh.tail_full);
      }
      if (!ok) {  // a copy lands within microseconds: let those that this warp started do so
        const long long t0 = clock64();
        while (clock64() - t0 < TC_WAIT_LIMIT / 1000) {
        }
      }
    } else if (warp == 1) {
      // ---- MMAs: one thread of the first CTA
      if (rank == 0 && elect_one()) {
        const uint32_t id_qk = pair_idesc(DT, PA_KEYS, 0, p.negate_q), id_pv = pair_idesc(DT, D, 1, 0);
        int s = 0, g = 0, n_seg = 0;  // ring place, tiles issued, segments
        uint32_t turn = 0;
        bool ok = true;
        // descriptors: Q, and K or V at the ring's first place; the high words hold no address
        const uint32_t a_lo = (uint32_t)sw128_desc(smem_u32(sQ)), b_lo = (uint32_t)sw128_desc(smem_u32(ring));
        const uint32_t k_hi = (uint32_t)(sw128_desc(0) >> 32), v_hi = (uint32_t)(mn_desc<Shape::V_LINE>(0, 0) >> 32);
        const uint32_t v_lo = (uint32_t)mn_desc<Shape::V_LINE>(smem_u32(ring), VR * Shape::V_LINE);
        auto advance = [&]() {
          umma2_commit(&sh.empty[s]);
          if (++s == RING) s = 0, turn ^= 1;
        };
        auto qk = [&](int tile) {  // S of the pair's tile number `tile`
          const uint32_t d = tmem + Shape::S_COL + (tile & 1) * PA_KEYS;
#pragma unroll
          for (int v = 0; v < SLOTS; ++v) {
            ok = ok && mbar_wait(&sh.full[s], turn, abort_flag);
            if (!ok) return;
            tc_fence_after();
#pragma unroll
            for (int ch = 0; ch < Shape::K_CHUNKS; ++ch) {
              const uint32_t a = a_lo + (v * Shape::K_CHUNKS + ch) * (PA_ROWS * 128 >> 4);
              const uint32_t b = b_lo + s * (PA_SLOT >> 4) + ch * (PA_KEYS / 2 * 128 >> 4);
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
            ok = ok && mbar_wait(&sh.full[s], turn, abort_flag);
            if (!ok) return;
            tc_fence_after();
            const uint32_t b = v_lo + s * (PA_SLOT >> 4);
#pragma unroll
            for (int k = 0; k < VR / 16; ++k)
              if (k * 16 < rows)
                umma2_ts(tmem, pt + (v * VR + k * 16) / 2, b + (16 * Shape::V_LINE >> 4) * k, v_hi, id_pv,
                         !first || v > 0 || k > 0);
            advance();
          }
        };
        for (; ok && walk.next(seg); ++n_seg) {
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
            const int nk = seg.rows_of(p, seg.key0 + j);
            pv(nk, tmem + Shape::S_COL + (g & 1) * PA_KEYS, j == 0);
            if (ok) umma2_commit(&sh.pv_done[g & 1]);
          }
        }
        // every MMA of the pair has completed before its TMEM is freed
        umma2_commit(&sh.drained);
        const long long t0 = clock64();
        while (!mbar_try_wait(&sh.drained, 0) && clock64() - t0 < TC_WAIT_LIMIT) {
        }
      }
    } else if (warp == 2) {
      // ---- Q: this CTA's tokens of each item
      if (lane == 0) {
        const uint32_t bar = first_cta(&sh.q_full);
        int n_seg = 0;
        bool ok = true;
        for (; walk.next(seg); ++n_seg) {
          if (n_seg > 0 && !(ok = mbar_wait(&sh.q_empty, (n_seg - 1) & 1, abort_flag))) break;
          const int box = seg.prefix ? p.tpc : min(p.tpc, p.max_new);
          const bool any = seg.ntok > rank * p.tpc;
          expect_first(bar, any ? (uint32_t)(box * p.G * 128 * Shape::CHUNKS) : 0u);
          if (any)
            for (int d = 0; d < Shape::CHUNKS; ++d)
              pair_load_3d(sQ + d * PA_ROWS * 128, seg.prefix ? &map_q_pre : &map_q_own, bar, d * 64, seg.kvh * p.G,
                           seg.tok0 + rank * p.tpc);
        }
        if (!ok) {
          const long long t0 = clock64();
          while (clock64() - t0 < TC_WAIT_LIMIT / 1000) {
          }
        }
      }
    } else if (warp == 3) {
      if (walk.alone) zero_unheld<D>(p, sh.start[0].sound, lane);
      // ---- V rows past the last visible one, up to the end of the 16-row step, to zero, in the
      // slots that warp 0 names: once for each segment that ends inside a step
      const uint32_t full0 = first_cta(&sh.full[0]);
      for (uint32_t n = 0;; ++n) {
        if (!__all_sync(0xffffffffu, mbar_wait(&sh.tail_full, n & 1, abort_flag))) break;
        const int2 t = sh.tail_at;  // ring place, rows to keep
        if (t.y == 0) break;
        constexpr int UNITS = Shape::V_LINE / 16;  // 16-byte units of a row
        const int units = (16 - (t.y & 15)) * UNITS;
        uint8_t* base = ring + t.x * PA_SLOT + t.y * Shape::V_LINE;
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
    } else {
      // ---- softmax, a row's column halves in two threads, then the segment's result
      const int quarter = warp & 3, half = (warp - 4) >> 2, row = quarter * 32 + lane;
      const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
      const uint32_t p_full0 = first_cta(&sh.p_full[0]), o_free0 = first_cta(&sh.o_free);
      const float c = p.c;
      int g = 0;
      while (walk.next(seg)) {
        const int row_tok = pa_quotient(row, p.g_magic), tl = rank * p.tpc + row_tok;  // token of the item
        const bool valid = row_tok < p.tpc && tl < seg.ntok;
        int lim = 0;  // rows of the sequence that the row sees
        if (valid) {
          if (seg.prefix) {
            const int i = request_of(p.starts, p.batch, seg.tok0 + tl);
            if (i < p.batch) {
              const PaRequest r = pa_request(p, i);
              lim = max(r.len - r.n + (seg.tok0 + tl - r.s0) + 1, 0);
            }
          } else {
            lim = max(seg.first + tl, 0);
          }
        }
        const bool live = __any_sync(0xffffffffu, valid);  // a warp without rows only keeps the barriers going
        // on either axis, and the least of the warp's rows
        const int lim_pre = min(lim, p.prefix_len), lim_own = min(max(lim - p.prefix_len, 0), seg.keys);
        const int least_pre = __reduce_min_sync(0xffffffffu, valid ? lim_pre : INT32_MAX);
        const int least_own = __reduce_min_sync(0xffffffffu, valid ? lim_own : INT32_MAX);
        float m = -INFINITY, l = 0.0f;
        for (int kt = seg.key0; kt < seg.key1; ++kt, ++g) {
          const int b = g & 1;
          mbar_wait(&sh.s_full[b], (g >> 1) & 1, abort_flag);
          __syncwarp();
          if (live) {
            tc_fence_after();
            const uint32_t at = tmem + lanes + Shape::S_COL + b * PA_KEYS;
            uint32_t s[2][32];
            tmem_ld32(at + half * 64, s[0]);
            tmem_ld32(at + half * 64 + 32, s[1]);
            tmem_ld_wait32(s[0]);
            tmem_ld_wait32(s[1]);
            const bool pre = kt < seg.pre;
            const int from = (pre ? kt : kt - seg.pre) * PA_KEYS;  // the tile's first row on its axis
            if ((pre ? least_pre : least_own) < from + PA_KEYS) {
              const int see = (pre ? lim_pre : lim_own) - from - half * 64;
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
            quarter_sync(quarter);  // also: both halves have read S, so P may take its place
            const float top = __fmul_rn(fmaxf(mine, sh.half[b][half ^ 1][row]), c);
            if (m == -INFINITY) m = top;  // nothing seen before: o and l are zero
            const bool grown = top > m + 8.0f;
            if (__any_sync(0xffffffffu, grown)) {
              // o is complete up to the tile before; then scale it
              mbar_wait(&sh.pv_done[b ^ 1], ((g - 1) >> 1) & 1, abort_flag);
              __syncwarp();
              tc_fence_after();
              const float f = grown ? exp2_approx(m - top) : 1.0f;
              // (Rolled: unrolled it is rare code that costs 800 bytes of spilled registers at D = 256.)
#pragma unroll 1
              for (int x = half * (D / 2); x < (half + 1) * (D / 2); x += 32) {
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
          quarter_sync(quarter);  // the tiles' exchanges have been read
          sh.half[0][half][row] = l;
          quarter_sync(quarter);
          l += sh.half[0][half ^ 1][row];
          if (seg.whole) {
            const int h = seg.kvh * p.G + row - row_tok * p.G;
            const int64_t t = seg.tok0 + tl;
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            uint16_t* out = p.out + (t * p.n_kvh * p.G + h) * D;
            const int64_t gate = t * p.gate_row + h * p.gate_head;
            for (int x = half * (D / 2); x < (half + 1) * (D / 2); x += 32) {
              uint32_t v[32];
              tmem_ld32(tmem + lanes + x, v);
              tmem_ld_wait32(v);
              if (valid) {
#pragma unroll
                for (int y0 = 0; y0 < 32; y0 += 16) {
                  uint4 g[4];
                  if (p.gate) {
#pragma unroll
                    for (int y = 0; y < 4; ++y) g[y] = gate_load(p, gate + x + y0 + 4 * y);
                  }
#pragma unroll
                  for (int y = 0; y < 16; y += 8) {
                    float z[8];
#pragma unroll
                    for (int k = 0; k < 8; ++k) z[k] = __uint_as_float(v[y0 + y + k]) * inv;
                    if (p.gate) {
                      const float4 a = gate_value<DT>(p, g[y / 4]), d = gate_value<DT>(p, g[y / 4 + 1]);
                      const float gs[8] = {a.x, a.y, a.z, a.w, d.x, d.y, d.z, d.w};
#pragma unroll
                      for (int k = 0; k < 8; ++k) z[k] = inv == 0.0f ? 0.0f : gated(z[k], gs[k]);
                    }
                    *reinterpret_cast<uint4*>(out + x + y0 + y) =
                        make_uint4(Elem<DT>::pack(z[0], z[1]), Elem<DT>::pack(z[2], z[3]), Elem<DT>::pack(z[4], z[5]),
                                   Elem<DT>::pack(z[6], z[7]));
                  }
                }
              }
            }
          } else {
            const int rows = seg.prefix ? 2 * PA_ROWS : p.own_rows;
            const int at = rank * (seg.prefix ? PA_ROWS : p.own_half) + row;  // of the place
            float4* o = reinterpret_cast<float4*>((seg.prefix ? p.pre_o : p.own_o) + seg.place * rows * D) + at;
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
            if (valid && half == 0)
              ((seg.prefix ? p.pre_ml : p.own_ml) + seg.place * rows)[at] = make_float2(m, l);
          }
          tc_fence_before();
          quarter_sync(quarter);  // the halves' sums have been read
        }
        __syncwarp();
        if (lane == 0) arrive_first(o_free0);
      }
    }
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

// Joins the segments of each row. A warp takes 8 rows (in the order of the prefix items' rows) of a
// KV head and 16 channels: lane (r, q) row r, the channels 4 q .. 4 q + 3, so that a load of the warp
// is 4 runs of 128 adjacent bytes and a store 8 runs of 32. What bounds it is the chain of
// dependent loads (lengths, places, partial results), so as many segments as a row has in most
// calls are asked for at once, and a thread has few channels (16 of them and 4 segments at once: 17 us
// of the 93 of 64 requests behind 32k rows, 10 so; 12 segments at once 12, 4 13).
struct RowSum {
  float4 o;
  float den, top;
};
// Every stride-th segment of a row from `first` on: x < n_pre of its prefix item, the others of its own
// (own_ml and own_o are where segment 0 would be). BATCH: segments asked for at once.
template <int D, int BATCH>
__device__ __forceinline__ RowSum join_segments(const float2* pre_ml, const float4* pre_o, const float2* own_ml,
                                                const float4* own_o, int own_step, int n_pre, int n, int first,
                                                int stride) {
  RowSum s{make_float4(0.0f, 0.0f, 0.0f, 0.0f), 0.0f, -INFINITY};
#pragma unroll 1
  for (int x0 = first; x0 < n; x0 += BATCH * stride) {
    float2 ml[BATCH];
    float4 y[BATCH];
    float now = s.top;
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
      ml[u] = make_float2(-INFINITY, 0.0f), y[u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      const int x = x0 + u * stride;
      if (x < n) {
        const bool pre = x < n_pre;
        const int64_t at = (int64_t)x * (pre ? 2 * PA_ROWS : own_step);
        ml[u] = (pre ? pre_ml : own_ml)[at];
        y[u] = (pre ? pre_o : own_o)[at * (D / 4)];
      }
    }
#pragma unroll
    for (int u = 0; u < BATCH; ++u) now = fmaxf(now, ml[u].x);
    const float keep = s.top == -INFINITY ? 0.0f : exp2_approx(s.top - now);
    s.top = now;
    s.den *= keep, s.o.x *= keep, s.o.y *= keep, s.o.z *= keep, s.o.w *= keep;
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
      const float w = ml[u].x == -INFINITY ? 0.0f : exp2_approx(ml[u].x - now);
      s.den = fmaf(ml[u].y, w, s.den);
      s.o.x = fmaf(y[u].x, w, s.o.x), s.o.y = fmaf(y[u].y, w, s.o.y);
      s.o.z = fmaf(y[u].z, w, s.o.z), s.o.w = fmaf(y[u].w, w, s.o.w);
    }
  }
  return s;
}
// A row's four channels 4 ch .. 4 ch + 3: divided, gated, rounded.
template <int D, int DT>
__device__ __forceinline__ void join_store(const PrefixAttnParams& p, int t, int h, int ch, const RowSum& s,
                                           uint4 gate) {
  const float inv = s.den == 0.0f ? 0.0f : 1.0f / s.den;
  float v[4] = {s.o.x * inv, s.o.y * inv, s.o.z * inv, s.o.w * inv};
  if (p.gate && inv != 0.0f) {
    const float4 g = gate_value<DT>(p, gate);
    v[0] = gated(v[0], g.x), v[1] = gated(v[1], g.y), v[2] = gated(v[2], g.z), v[3] = gated(v[3], g.w);
  }
  *reinterpret_cast<uint2*>(p.out + ((int64_t)t * p.n_kvh * p.G + h) * D + ch * 4) =
      make_uint2(Elem<DT>::pack(v[0], v[1]), Elem<DT>::pack(v[2], v[3]));
}
__device__ __forceinline__ uint4 join_gate(const PrefixAttnParams& p, int t, int h, int ch) {
  return p.gate ? gate_load(p, t * p.gate_row + h * p.gate_head + ch * 4) : make_uint4(0, 0, 0, 0);
}
// b / per, a pair's or a warp's number: small, so that one correction makes the quotient in binary32
// right.
__device__ __forceinline__ int pair_of(int b, int per) {
  int q = (int)((float)b * (1.0f / (float)per));
  q -= q * per > b;
  return q + ((q + 1) * per <= b);
}

// Without prefix items only the items that a pair's share cuts are left to join: the warps take
// their rows, 8 rows and 64 channels each, by the pair that the cut ends at. (16 prompt chunks, whose rows
// were looked at one by one before: the join 45 us, 24 so, with flushed caches.)
template <int D, int DT>
__device__ __forceinline__ void join_cut_items(const PrefixAttnParams& p, int per, int units, int warp, int lane) {
  const int groups = (p.own_rows + 7) / 8, each = groups * (D / 64), cuts = (units + per - 1) / per - 1;
  const int warps = gridDim.x * gridDim.y * 8;
  for (int w = (blockIdx.y * gridDim.x + blockIdx.x) * 8 + warp; w < cuts * each; w += warps) {
    const int c = 1 + w / each, rest = w % each, unit = c * per;
    int lo = 0, hi = p.batch;  // the last request whose units begin at or before this one
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (p.work_base[mid].y <= unit) lo = mid;
      else hi = mid;
    }
    const int2 base = p.work_base[lo];
    const PaRequest r = pa_request(p, lo);
    const int nq = pa_qtiles(p, r), head = (int)pa_own_units(p, r, nq, true);
    int u = unit - base.y, kvh = 0, qt = 0, kt = 0;
    if (head <= 0) continue;
    kvh = u / head, u -= kvh * head;
    for (; qt < nq; ++qt) {
      kt = pa_tiles(p, r, qt, true);
      const int n = pa_units(kt, false, p.item_cost);
      if (u < n) break;
      u -= n;
    }
    if (kvh >= p.n_kvh || qt >= nq) continue;
    const int b = unit - u + p.item_cost, c0 = pair_of(b, per), n = pair_of(b + kt - 1, per) - c0 + 1;
    if (n < 2 || c0 != c - 1) continue;  // not cut here, or first cut before
    const int row = rest / (D / 64) * 8 + (lane & 7), rank = row >= p.own_half, in = row - rank * p.own_half;
    const int tl = rank * p.tpc + pa_quotient(in, p.g_magic), h = kvh * p.G + in - pa_quotient(in, p.g_magic) * p.G;
    if (row >= p.own_rows || tl >= min(p.tpi, r.n - qt * p.tpi)) continue;
    const int t = r.s0 + qt * p.tpi + tl;
    const int64_t at = (int64_t)(base.x + kvh * nq + qt + c0) * p.own_rows;
    int ch = rest % (D / 64) * 16 + (lane >> 3);
    const float2* ml = p.own_ml + at + row;
    const float4* o = reinterpret_cast<const float4*>(p.own_o) + at * (D / 4) + row;
    if (n == 2) {  // the common case: eight channels asked for at once
      const float2 m0 = ml[0], m1 = ml[p.own_rows];
      const float top = fmaxf(m0.x, m1.x);
      const float w0 = m0.x == -INFINITY ? 0.0f : exp2_approx(m0.x - top);
      const float w1 = m1.x == -INFINITY ? 0.0f : exp2_approx(m1.x - top);
      const int step = p.own_rows * (D / 4);
      const float4* from = o + ch * p.own_rows;
#pragma unroll 1
      for (int j = 0; j < 4; j += 2, ch += 8, from += 8 * p.own_rows) {
        const float4 y0 = from[0], y1 = from[step], y2 = from[4 * p.own_rows], y3 = from[4 * p.own_rows + step];
        const uint4 g0 = join_gate(p, t, h, ch), g1 = join_gate(p, t, h, ch + 4);
        RowSum s{make_float4(fmaf(y1.x, w1, y0.x * w0), fmaf(y1.y, w1, y0.y * w0), fmaf(y1.z, w1, y0.z * w0),
                             fmaf(y1.w, w1, y0.w * w0)),
                 fmaf(m1.y, w1, m0.y * w0), top};
        join_store<D, DT>(p, t, h, ch, s, g0);
        s.o = make_float4(fmaf(y3.x, w1, y2.x * w0), fmaf(y3.y, w1, y2.y * w0), fmaf(y3.z, w1, y2.z * w0),
                          fmaf(y3.w, w1, y2.w * w0));
        join_store<D, DT>(p, t, h, ch + 4, s, g1);
      }
      continue;
    }
#pragma unroll 1
    for (int j = 0; j < 4; ++j, ch += 4) {
      const uint4 gate = join_gate(p, t, h, ch);
      join_store<D, DT>(p, t, h, ch, join_segments<D, 4>(ml, o, ml, o + ch * p.own_rows, p.own_rows, 0, n, 0, 1), gate);
    }
  }
}

template <int D, int DT>
__global__ void __launch_bounds__(256) prefix_combine_kernel(const __grid_constant__ PrefixAttnParams p) {
  __shared__ float joined[8][6][32];
  const int parts = D / 16 / p.join_span, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int split = p.join_split, part = warp & (split - 1);
  const int unit = (blockIdx.x * 8 + warp) / split, idx = unit / parts * 8 + (lane & 7);
  const int kvh = blockIdx.y, t = pa_quotient(idx, p.g_magic), gh = idx - t * p.G, h = kvh * p.G + gh;
  int ch = (unit % parts) * p.join_span * 4 + (lane >> 3);  // of 4 channels; then every 4th, join_span in all
  bool live = t < p.tokens;
  pdl_begin();
  const int4 how = *p.work_per;
  const bool alone = how.z < 0;
  // one token for each request is the common case: its request's numbers are asked for at once
  int i = t;
  PaRequest r{-1, 0, 0};
  int2 base{};
  if (t < p.batch) r = pa_request(p, t), base = p.work_base[t];
  if (alone && !p.thin) {
    if (how.y > 0) join_cut_items<D, DT>(p, how.y, how.w, warp, lane);
    return;
  }
  if (live && (r.s0 != t || r.n != 1)) {
    i = request_of(p.starts, p.batch, t);
    r = i < p.batch ? pa_request(p, i) : PaRequest{-1, 0, 0};
    if (i < p.batch) base = p.work_base[i];
  }
  // segments of the row: n_pre of its prefix item, n_own of its own, from their first places on
  int n_pre = 0, n_own = 0;
  const float4 *pre_o = nullptr, *own_o = nullptr;
  const float2 *pre_ml = nullptr, *own_ml = nullptr;
  if (live && (how.x | how.y) > 0 && t >= r.s0 && t < r.s0 + r.n) {
    const int nq = pa_qtiles(p, r), own_qt = nq > 1 ? pa_quotient(t - r.s0, p.tpi_magic) : 0;
    const int kt = pa_tiles(p, r, own_qt, alone);
    if (kt > 0 && how.y > 0) {
      int b = base.y + p.item_cost;
      if (kvh > 0) b += kvh * (int)pa_own_units(p, r, nq, alone);
      for (int q = 0; q < own_qt; ++q) b += pa_units(pa_tiles(p, r, q, alone), false, p.item_cost);
      const int c0 = pair_of(b, how.y), tl = t - r.s0 - own_qt * p.tpi, rank = tl >= p.tpc;
      n_own = pair_of(b + kt - 1, how.y) - c0 + 1;
      const int64_t at = (int64_t)(base.x + kvh * nq + own_qt + c0) * p.own_rows;
      const int row = rank * p.own_half + (tl - rank * p.tpc) * p.G + gh;
      own_ml = p.own_ml + at + row;
      own_o = reinterpret_cast<const float4*>(p.own_o) + at * (D / 4) + ch * p.own_rows + row;
    }
    if (n_own == 1 && alone) live = false;  // finished where it was computed
    if (!alone && how.x > 0) {
      const int qt = pa_quotient(t, p.tpi_magic), it = kvh * p.pre_qtiles + qt, tl = t - qt * p.tpi, rank = tl >= p.tpc;
      const int b = it * pa_units(how.z, false, PA_ITEM_COST) + PA_ITEM_COST, c0 = pair_of(b, how.x);
      n_pre = pair_of(b + how.z - 1, how.x) - c0 + 1;
      const int64_t at = (int64_t)(it + c0) * (2 * PA_ROWS);
      const int row = rank * PA_ROWS + (tl - rank * p.tpc) * p.G + gh;
      pre_ml = p.pre_ml + at + row;
      pre_o = reinterpret_cast<const float4*>(p.pre_o) + at * (D / 4) + ch * (2 * PA_ROWS) + row;
    }
  }
  const int n = live ? n_pre + n_own : 0;
  own_ml -= (int64_t)n_pre * p.own_rows, own_o -= (int64_t)n_pre * p.own_rows * (D / 4);
  if (split == 1 && !live) return;
#pragma unroll 1
  for (int j = 0; j < p.join_span; ++j, ch += 4, pre_o += 4 * 2 * PA_ROWS, own_o += 4 * p.own_rows) {
    const uint4 gate = live ? join_gate(p, t, h, ch) : make_uint4(0, 0, 0, 0);
    RowSum s = join_segments<D, 8>(pre_ml, pre_o, own_ml, own_o, p.own_rows, n_pre, n, part, split);
    if (split > 1) {  // the parts of the row's segments, in order
      float(&mine)[6][32] = joined[warp];
      mine[0][lane] = s.top, mine[1][lane] = s.den;
      mine[2][lane] = s.o.x, mine[3][lane] = s.o.y, mine[4][lane] = s.o.z, mine[5][lane] = s.o.w;
      __syncthreads();
      if (part > 0 || !live) return;
      for (int x = 1; x < split; ++x) {
        const float(&other)[6][32] = joined[warp + x];
        const float most = other[0][lane], now = fmaxf(s.top, most);
        const float keep = s.top == -INFINITY ? 0.0f : exp2_approx(s.top - now);
        const float w = most == -INFINITY ? 0.0f : exp2_approx(most - now);
        s.top = now;
        s.den = s.den * keep + other[1][lane] * w;
        s.o.x = s.o.x * keep + other[2][lane] * w, s.o.y = s.o.y * keep + other[3][lane] * w;
        s.o.z = s.o.z * keep + other[4][lane] * w, s.o.w = s.o.w * keep + other[5][lane] * w;
      }
    }
    join_store<D, DT>(p, t, h, ch, s, gate);
  }
}

template <int D, int DT>
static int launch_prefix_attention(const CUtensorMap (&maps)[4], const PrefixAttnParams& p, int grid, cudaStream_t st) {
  static SmemOptIn opt_in;
  if (cudaError_t e = opt_in(prefix_attention_kernel<D, DT>, PaShape<D>::SMEM))
    return cuda_fail(e, "prefix_attention_kernel attributes");
  if (cudaError_t e = launch_pdl(prefix_attention_kernel<D, DT>, grid, PA_THREADS, PaShape<D>::SMEM, st, maps[0],
                                 maps[1], maps[2], maps[3], p))
    return cuda_fail(e, "prefix_attention_kernel");
  if (p.whole) return YSKN_OK;
  const int64_t warps = ceil_div((int64_t)p.tokens * p.G, 8) * (D / 16 / p.join_span) * p.join_split;
  return cuda_fail(launch_pdl(prefix_combine_kernel<D, DT>, dim3((unsigned)ceil_div(warps, 8), p.n_kvh), 256, 0, st, p),
                   "prefix_combine_kernel");
}

}  // namespace yskn

using namespace yskn;

extern "C" YSKN_B200_API int64_t yskn_b200_prefix_attention_work_bytes(int tokens, int batch, int max_new, int n_qh,
                                                                      int n_kvh, int head) {
  if (tokens < 1 || batch < 1 || max_new < 1 || n_qh < 1 || n_kvh < 1 || n_qh % n_kvh || n_qh / n_kvh > PA_ROWS ||
      (head != 64 && head != 128 && head != 256))
    return -1;
  return pa_work(tokens, batch, max_new, n_qh, n_kvh, head).bytes;
}

extern "C" YSKN_B200_API int yskn_b200_prefix_attention(const yskn_b200_prefix_attention_args* args, void* stream) {
  if (!args) return fail(YSKN_EINVAL, "prefix_attention: null argument");
  yskn_b200_prefix_attention_args a = *args;
  if (const char* what = attention_refusal(a)) return fail(YSKN_EINVAL, std::string("prefix_attention: ") + what);
  const int head = a.head, n_qh = a.n_qh, n_kvh = a.n_kvh, block_size = a.block_size, dtype = a.dtype;
  a.max_new = std::min(a.max_new, a.tokens);  // as pa_work does
  const PaWork w = pa_work(a.tokens, a.batch, a.max_new, n_qh, n_kvh, head);
  if (a.work_bytes < w.bytes) return fail(YSKN_EINVAL, "prefix_attention: workspace too small");
  const int G = n_qh / n_kvh, tpc = PA_ROWS / G;
  int dev = 0, sms = 2 * PA_MAX_PAIRS;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const int pairs = std::min(sms / 2, PA_MAX_PAIRS);
  PrefixAttnParams p{};
  p.q = reinterpret_cast<const uint16_t*>(a.q), p.q_row = a.q_row, p.q_head = a.q_head;
  p.k_cache = reinterpret_cast<const uint16_t*>(a.k_cache), p.v_cache = reinterpret_cast<const uint16_t*>(a.v_cache);
  p.cache = {a.block_stride, a.token_stride, a.head_stride};
  p.gate = a.gate, p.gate_f32 = a.gate_dtype == YSKN_DT_F32;
  p.gate_row = a.gate_row, p.gate_head = a.gate_head;
  p.prefix_blocks = a.prefix_blocks;
  p.tables = a.block_tables, p.table_stride = a.table_stride;
  p.lens = a.lens, p.starts = a.starts;
  p.n_blocks = a.n_blocks, p.prefix_len = a.prefix_len;
  p.block_shift = block_size == 16 ? 4 : block_size == 32 ? 5 : block_size == 64 ? 6 : 7;
  p.own_limit = (int)std::min<int64_t>((int64_t)a.table_width * block_size, INT32_MAX - PA_KEYS);
  p.batch = a.batch, p.tokens = a.tokens, p.max_new = a.max_new, p.n_kvh = n_kvh, p.G = G;
  p.tpc = tpc, p.tpi = 2 * tpc;
  auto magic = [](int d) { return d == 1 ? 0u : (unsigned)(((1ull << 32) + d - 1) / d); };
  p.g_magic = magic(G), p.tpi_magic = magic(p.tpi);
  const int pre_tiles = (int)ceil_div(a.prefix_len, PA_KEYS);  // at most: where a request sees the whole prefix
  p.pre_qtiles = (int)ceil_div(a.tokens, 2 * tpc);
  const int64_t items = (int64_t)p.pre_qtiles * n_kvh;
  if (items * pa_units(pre_tiles, false, PA_ITEM_COST) >= (int64_t)PA_MANY ||
      (int64_t)a.tokens * n_qh * head > INT32_MAX || a.tokens >= 1 << 24 || n_kvh > 65535)
    return fail(YSKN_EINVAL, "prefix_attention: too much work");
  p.shared_items = a.prefix_len > 0 ? (int)items : 0;
  // Few items of few tiles: each by one pair of SMs (a thin one by one warp) from end to end, which is
  // quicker than the second launch that joins its parts. Two requests, us whole and cut: of two
  // tokens and one tile 15.5, 19.2, of two tiles 17.3, 14.8; thin with up to 32 and 64 rows 10.3, 14.4
  // and 12.1, 16.1, with 128 15.7, 13.8 (12.2 since a warp's least is 2 units).
  p.thin = (int64_t)G * a.max_new <= PA_THIN_ROWS && pairs > 1;
  p.tile_shift = p.thin ? PA_THIN_SHIFT : 7;
  p.item_cost = p.thin ? PA_THIN_COST : PA_ITEM_COST;
  const int64_t most_tiles = ceil_div(a.prefix_len, 1 << p.tile_shift) + ceil_div(p.own_limit, 1 << p.tile_shift);
  p.whole = p.thin ? w.own_items <= 2 * PA_THIN_WARPS * pairs && most_tiles <= PA_THIN_WHOLE
                   : w.own_items <= pairs && most_tiles <= PA_WHOLE_TILES;
  p.many_per_head = PA_MANY / (unsigned)n_kvh;
  // A warp of the join takes 16 channels of 8 rows; or more, where that makes twice the warps that the
  // SMs hold (128 requests of 8 tokens: 162 us with 16 channels, 141 so; 16 prompt chunks, where most
  // warps find nothing to do, 835, 740).
  const int64_t join_rows = ceil_div((int64_t)a.tokens * G, 8) * n_kvh;
  p.join_span = 1;
  while (p.join_span < head / 16 && join_rows * (head / 16 / p.join_span) > 2 * 148 * 24) p.join_span *= 2;
  // Few: several warps share a row's segments (42 requests of one KV head behind 32k rows: 44.5 us by one
  // warp, 28 by eight).
  p.join_split = 1;
  while (p.join_split < 8 && join_rows * (head / 16) * 2 * p.join_split <= 148 * 24) p.join_split *= 2;
  // a scale of zero keeps its meaning (equal weights) with a factor that leaves -inf alone
  p.c = std::max(std::fabs(a.scale) * 1.4426950408889634f, 1e-30f);
  p.negate_q = a.scale < 0.0f;
  uint8_t* work = reinterpret_cast<uint8_t*>(a.work);
  p.work_per = reinterpret_cast<int4*>(work);
  p.work_base = reinterpret_cast<int2*>(work + w.base);
  p.pre_ml = reinterpret_cast<float2*>(work + w.pre_ml), p.pre_o = reinterpret_cast<float*>(work + w.pre_o);
  p.own_ml = reinterpret_cast<float2*>(work + w.own_ml), p.own_o = reinterpret_cast<float*>(work + w.own_o);
  p.own_half = w.own_half, p.own_rows = w.own_rows, p.own_items = w.own_items;
  p.out = reinterpret_cast<uint16_t*>(a.out), p.err = device_error_word();
  // The cache's 64-channel columns are an axis of their own, so that one box holds several columns
  // of its rows in the order of the ring's slots; where a slot takes several boxes (blocks
  // shorter than it), a box is one column.
  const int slots = head <= 128 ? 1 : head / 128, v_rows = PA_KEYS / slots;
  const int64_t q_dims[3] = {head, n_qh, a.tokens}, q_strides[2] = {a.q_head, a.q_row};
  const int64_t c_dims[5] = {64, block_size, head / 64, n_kvh, a.n_blocks};
  const int64_t c_strides[4] = {a.token_stride, 64, a.head_stride, a.block_stride};
  const int box_pre[3] = {64, G, tpc}, box_own[3] = {64, G, std::min(tpc, a.max_new)};
  const int box_k[5] = {64, std::min(block_size, PA_KEYS / 2), block_size < PA_KEYS / 2 ? 1 : head / 64 / slots, 1, 1};
  const int box_v[5] = {head == 64 ? 32 : 64, std::min(block_size, v_rows),
                        block_size < v_rows || head <= 128 ? 1 : head / 128, 1, 1};
  CUtensorMap maps[4] = {};
  if (!p.thin || p.shared_items > 0) {  // thin items need no map
    if (int rc = paged_map("prefix_attention", &maps[0], a.q, dtype, 3, q_dims, q_strides, box_pre)) return rc;
    if (int rc = paged_map("prefix_attention", &maps[2], a.k_cache, dtype, 5, c_dims, c_strides, box_k)) return rc;
    if (int rc = paged_map("prefix_attention", &maps[3], a.v_cache, dtype, 5, c_dims, c_strides, box_v)) return rc;
    maps[1] = maps[0];
    if (!p.thin)
      if (int rc = paged_map("prefix_attention", &maps[1], a.q, dtype, 3, q_dims, q_strides, box_own)) return rc;
  }
  const int grid = 2 * pairs;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  auto run = [&](auto d) {
    constexpr int D = decltype(d)::value;
    return dtype == YSKN_DT_BF16 ? launch_prefix_attention<D, YSKN_DT_BF16>(maps, p, grid, st)
                                 : launch_prefix_attention<D, YSKN_DT_F16>(maps, p, grid, st);
  };
  if (head == 64) return run(std::integral_constant<int, 64>{});
  if (head == 128) return run(std::integral_constant<int, 128>{});
  return run(std::integral_constant<int, 256>{});
}
