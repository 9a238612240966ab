// Log probabilities of given tokens, the entropy and the most likely tokens of rows of logits.
//
// Per row, with M the largest logit and R the sum of exp(x - M) over all tokens but one of logit M:
//   log p(t) = (x_t - M) - log(1 + R)
//   entropy  = log(1 + R) - E / (1 + R),  E = sum of exp(x - M) (x - M)
// The maximum's own 1 stays out of R, so that a row that is nearly sure (R far below 1) keeps R's
// digits: log(1 + R) is log1p, and nothing is subtracted. States (M, R, E) of two parts join as
//   M = max, f = exp(m - M) of the lesser part, R = R_greater + f (R_lesser + 1),
//   E = E_greater + f (E_lesser + (R_lesser + 1) (m - M)).
//
// What bounds it: one read of the logits (4 bytes each); for few rows, the chain of latencies. A
// cluster of 1 to 8 CTAs takes a row, one part each; the parts are joined through distributed shared
// memory, so that there is one launch, no workspace and no counter that a second call could meet.
// A warp streams its own run of the part in slices, 8 or 10 16-byte loads a lane for the next slice under way
// while it works on one: its maximum and its sums. (512 rows of 151936, without the largest tokens: 67 us with three
// CTAs an SM that load and work in turn, 52.5 with two that load 8 ahead; half the slice, four CTAs, 49.9, but with
// the largest tokens 74 against 60, and 12.2 against 9.0 for one row.)
// A logit is a key: its bits in an order of unsigned numbers, above the complement of its number, so that keys are all
// different and equal logits go by the lowest number. A bound holds most keys off that cannot be among the n_top
// largest: n_top of the 32 groups of 8 lanes have a logit that reaches it. (The 8 largest of 151936 normal ones: 9 of the
// 10240 in the warps' first slices reach it, 30 in all.) What reaches it goes to the warp's buffer in shared memory; in the end each key of
// the CTA's buffers counts the keys above it, which is its place. Rows whose largest come late fill a buffer: then 32
// keys are sorted (bitonic, in registers) and merged into a list of the warp's 32 largest, whose n_top-th is a bound
// too. (All keys through such lists: 93 us for 512 rows, and the chain of shuffles made one row wait 13.)
// The passing logits are read again, from the cache, by a rolled loop: 32 copies of its code for the slice's registers
// took 62 us for 512 rows instead of 59.8, and one row, where each CTA runs the code once and waits for it, 10.6
// instead of 9.0.
// Measured on the device: one row of 151936 with 20 largest 7.9 us (without them 4.7), 33 rows of 50257 7.5, 256 rows
// of 151936 with 8 largest 29.8 (5.2 TB/s), 512 rows 56.1 (5.5 TB/s, without the largest 50.4; two CTAs of 512 on every
// SM and a half).
#include <algorithm>
#include <type_traits>

#include "common.cuh"

namespace yskn {

constexpr int LP_WARPS = 8, LP_THREADS = LP_WARPS * 32;
// 16-byte loads of a lane in a slice, one of the two: a slice is 32 times as many 16-byte groups.
constexpr int LP_FEW = 8, LP_MANY = 10;
constexpr int LP_RESIDENT = 2;           // CTAs of an SM
constexpr int LP_MAX_CLUSTER = 8;
constexpr int LP_LEAST_PART = 7500;      // logits of a CTA where a row has several, at least
constexpr float LP_LOG2E = 1.44269504088896340736f;

struct LogprobsParams {
  const float* logits;
  int64_t logits_stride;
  const int32_t* tokens;
  int64_t token_stride;
  float *logprobs, *entropy, *top_logprobs;
  int32_t* top_ids;
  int vocab, n_tokens, n_top, cluster;
};

struct LpState {
  float m, rest, e;  // the part's maximum (-inf: nothing above it), R and E
};

// Two binary32 operations in one instruction.
__device__ __forceinline__ float2 lp_add2(float2 a, float2 b) {
  float2 y;
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 d, a, b;\n\t"
      "mov.b64 {%0, %1}, d;\n\t}"
      : "=f"(y.x), "=f"(y.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return y;
}
__device__ __forceinline__ float2 lp_mul2(float2 a, float2 b) {
  float2 y;
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmul.rn.f32x2 d, a, b;\n\t"
      "mov.b64 {%0, %1}, d;\n\t}"
      : "=f"(y.x), "=f"(y.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return y;
}
__device__ __forceinline__ float2 lp_fma2(float2 a, float2 b, float2 c) {
  float2 y;
  asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(y.x), "=f"(y.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return y;
}
__device__ __forceinline__ float lp_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float lp_exp(float d) { return lp_exp2(d * LP_LOG2E); }  // d <= 0, -inf included
// Bits whose order as an unsigned number is the logits' order; -0 counts as 0.
__device__ __forceinline__ uint32_t lp_ordered(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float lp_value(uint32_t o) {
  return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o);
}
__device__ __forceinline__ uint64_t lp_key(float x, int id) {
  return (uint64_t)lp_ordered(x) << 32 | (uint32_t)~(uint32_t)id;
}
__device__ __forceinline__ LpState lp_join(LpState a, LpState b) {
  const bool more = b.m > a.m;
  const LpState hi = more ? b : a, lo = more ? a : b;
  if (lo.m == -INFINITY) return LpState{hi.m, hi.rest + lo.rest, hi.e};  // lo.rest is 0, or NaN that has to stay
  const float d = lo.m - hi.m, f = lp_exp(d), w = lo.rest + 1.0f;
  // (f of 0: d may be the type's lowest number, and its product with w infinite)
  return LpState{hi.m, fmaf(f, w, hi.rest), f == 0.0f ? hi.e : fmaf(f, fmaf(w, d, lo.e), hi.e)};
}

// Sorted by lanes: ascending, and a bitonic sequence into descending order.
__device__ __forceinline__ uint64_t lp_exchange(uint64_t v, int by, bool keep_max) {
  const uint64_t o = __shfl_xor_sync(0xffffffffu, v, by);
  return (v > o) == keep_max ? v : o;
}
__device__ __forceinline__ uint64_t lp_sort_up(uint64_t v, int lane) {
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
    for (int by = size >> 1; by > 0; by >>= 1) v = lp_exchange(v, by, ((lane & by) != 0) == ((lane & size) == 0));
  return v;
}
__device__ __forceinline__ uint64_t lp_bitonic_down(uint64_t v, int lane) {
#pragma unroll
  for (int by = 16; by > 0; by >>= 1) v = lp_exchange(v, by, (lane & by) == 0);
  return v;
}
// The 32 largest of a list (descending) and 32 others (ascending), descending.
__device__ __forceinline__ uint64_t lp_merge(uint64_t list, uint64_t up, int lane) {
  return lp_bitonic_down(list > up ? list : up, lane);
}

__device__ __forceinline__ uint4 lp_shared_u32x4(const uint32_t* p) {
  uint4 y;
  asm volatile("ld.volatile.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(y.x), "=r"(y.y), "=r"(y.z), "=r"(y.w)
               : "r"((uint32_t)__cvta_generic_to_shared(p))
               : "memory");
  return y;
}

// ---- the cluster
__device__ __forceinline__ void lp_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t lp_remote(const void* p, int rank) {
  uint32_t a;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
  return a;
}
__device__ __forceinline__ void lp_put_u64(uint32_t a, uint64_t v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(a), "l"(v) : "memory");
}
__device__ __forceinline__ void lp_put_f32(uint32_t a, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(a), "f"(v) : "memory");
}

// Up to so many largest the bound is the groups' n_top-th largest logit; for more, where that is nearly the groups'
// least, the least of the warps' ceil(n_top / 8)-th largest lane maxima. us by groups, by warps: 512 rows with 8
// largest 56.1, 57.7, with one 52.9, 57.7; 64 rows with 20 14.5, 15.9, one row 7.9, 8.2; 300 rows with 32 71, 56.5.
constexpr int LP_BINNED = 24;
constexpr int LP_BUFFER = 160;  // keys: up to 31 that are left, and 128 that may join them

// A warp's largest keys: `list` descending over the lanes, `bound` the least that may still enter, `held` keys in
// its buffer.
struct LpTop {
  uint64_t list, bound;
  int held;
};
// The buffer's keys into the list, 32 at a time, while there are at least `least`. (Called, not inlined: a copy of
// it at each place made the kernel wait for instructions.)
__device__ __noinline__ LpTop lp_flush(LpTop t, uint64_t* buffer, int least, int n_top) {
  const int lane = threadIdx.x & 31;
  __syncwarp();
  while (t.held >= least) {
    const int at = max(t.held - 32, 0) + lane;  // the last ones
    const uint64_t v = at < t.held ? buffer[at] : 0;
    t.held = max(t.held - 32, 0);
    t.list = lp_merge(t.list, lp_sort_up(v, lane), lane);
  }
  __syncwarp();
  const uint64_t last = __shfl_sync(0xffffffffu, t.list, n_top - 1);
  t.bound = last > t.bound ? last : t.bound;
  return t;
}

struct LpShared {
  uint64_t buffer[LP_WARPS][LP_BUFFER];
  alignas(16) uint32_t bound[32];  // of each 8 lanes the largest so far, or each warp's m-th largest lane maximum
  int held[LP_WARPS];  // keys in each buffer; in the end all of the warp's
  alignas(16) uint64_t keys[LP_WARPS * 64 + 1];  // to be ranked
  uint64_t list[YSKN_MAX_TOP];   // this CTA's largest
  LpState state[LP_WARPS];
  // in the cluster's first CTA: what the others have put there, and the row's largest
  LpState parts[LP_MAX_CLUSTER];
  uint64_t lists[LP_MAX_CLUSTER * YSKN_MAX_TOP];
  uint64_t row_list[YSKN_MAX_TOP];
  // the first tokens and their logits, asked for ahead of the row
  int id[LP_THREADS];
  float logit[LP_THREADS];
};

// The largest n_top of n different keys in shared memory (a 0 behind them), in order, into `list`, which holds zeros;
// all threads.
__device__ __forceinline__ void lp_rank(const uint64_t* keys, int n, uint64_t* list, int n_top, int tid) {
  for (int i = tid; i < n; i += LP_THREADS) {
    const uint64_t key = keys[i];
    int above = 0;
#pragma unroll 4
    for (int j = 0; j < n; j += 2) {
      const ulonglong2 y = *reinterpret_cast<const ulonglong2*>(keys + j);
      above += (y.x > key) + (y.y > key);
    }
    if (above < n_top) list[above] = key;
  }
}
// The same of n (1..8) lists of `width` (up to 32) descending keys, zeros at their ends.
__device__ __forceinline__ void lp_rank_lists(const uint64_t* keys, int n, int width, uint64_t* list, int n_top,
                                              int tid) {
  if (tid >= n * width) return;
  const uint64_t key = keys[tid];
  if (key == 0) return;
  int above[LP_MAX_CLUSTER] = {};
#pragma unroll
  for (int step = 32; step > 0; step >>= 1)
#pragma unroll
    for (int l = 0; l < LP_MAX_CLUSTER; ++l) {
      const int at = above[l] + step;
      if (l < n && at <= width && keys[l * width + at - 1] > key) above[l] = at;
    }
  int place = 0;
#pragma unroll
  for (int l = 0; l < LP_MAX_CLUSTER; ++l) place += above[l];
  if (place < n_top) list[place] = key;
}
// n (1..8) states in shared memory, joined; a whole warp.
__device__ __forceinline__ LpState lp_whole(const LpState* state, int n, int lane) {
  LpState t = lane < n ? state[lane] : LpState{-INFINITY, 0.0f, 0.0f};
#pragma unroll
  for (int by = 4; by > 0; by >>= 1)
    t = lp_join(t, LpState{__shfl_down_sync(0xffffffffu, t.m, by), __shfl_down_sync(0xffffffffu, t.rest, by),
                           __shfl_down_sync(0xffffffffu, t.e, by)});
  t.m = __shfl_sync(0xffffffffu, t.m, 0);
  t.rest = __shfl_sync(0xffffffffu, t.rest, 0);
  t.e = __shfl_sync(0xffffffffu, t.e, 0);
  return t;
}

template <bool TOP, int LOADS>
__global__ void __launch_bounds__(LP_THREADS, LP_RESIDENT)
    token_logprobs_kernel(const __grid_constant__ LogprobsParams p) {
  constexpr int SLICE = LOADS * 32;
  __shared__ LpShared sh;
  pdl_begin();
  if (p.cluster > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");  // this CTA has begun
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.x / p.cluster, rank = blockIdx.x - row * p.cluster;
  const float* x = p.logits + row * p.logits_stride;
  // The row's whole 16-byte groups, of which this part has [g0, g1) and this warp [w0, w1): all warps some, where
  // there are 8, so that each has a part of the bound. Up to three logits before and after them (lanes 0..2 and
  // 3..5) are a slice of their own of the first part's first warp.
  const int head = min((int)(-(reinterpret_cast<uintptr_t>(x) >> 2) & 3), p.vocab);
  const int n_groups = (p.vocab - head) >> 2, tail = p.vocab - head - 4 * n_groups;
  const float4* groups = reinterpret_cast<const float4*>(x + head);
  const int per = (n_groups + p.cluster - 1) / p.cluster;
  const int g0 = min(rank * per, n_groups), g1 = min(g0 + per, n_groups);
  const int w0 = g0 + (int)((int64_t)(g1 - g0) * warp / LP_WARPS);
  const int w1 = g0 + (int)((int64_t)(g1 - g0) * (warp + 1) / LP_WARPS);
  bool edges = warp == 0 && rank == 0 && head + tail > 0;

  LpState s{-INFINITY, 0.0f, 0.0f};  // m: of the warp; rest and e: of the lane
  const uint64_t lowest = (uint64_t)lp_ordered(-INFINITY) << 32 | 0xffffffffu;  // only logits above -inf pass
  LpTop top{0, lowest, 0};
  uint32_t so_far = 0;  // the lane's largest
  bool raise = true;    // the bound may be lower than it could
  uint64_t* buffer = sh.buffer[warp];
  if (TOP && lane == 0) sh.held[warp] = 0;
  const float4 nothing = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
  float4 next[LOADS];  // on their way while a slice is worked on
  auto load = [&](int g) {
#pragma unroll
    for (int u = 0; u < LOADS; ++u) {
      const int at = g + u * 32 + lane;
      next[u] = at < w1 ? __ldcs(groups + at) : nothing;
    }
  };
  load(w0);
  if (rank == 0 && tid < p.n_tokens) {  // behind the row, their two loads would be its last 1.2 us
    const int id = p.tokens[row * p.token_stride + tid];
    sh.id[tid] = id;
    if ((unsigned)id < (unsigned)p.vocab)
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"((uint32_t)__cvta_generic_to_shared(sh.logit + tid)),
                   "l"(__cvta_generic_to_global(x + id))
                   : "memory");
  }
  for (int g = w0;; g += SLICE) {  // once at least, since the warps meet in it
    float2 v[LOADS][2];
#pragma unroll
    for (int u = 0; u < LOADS; ++u) {
      v[u][0] = make_float2(next[u].x, next[u].y);
      v[u][1] = make_float2(next[u].z, next[u].w);
    }
    uint32_t first_id = head + 4 * (g + lane), in_group = 4;
    const bool more = g + SLICE < w1;
    load(g + SLICE);  // nothing, past the end
    if (g >= w1 && edges) {
      const int at = lane < 3 ? lane : p.vocab - tail + lane - 3;
      if (lane < 3 ? lane < head : lane - 3 < tail) v[0][0].x = x[at];
      first_id = at, in_group = 1;
      edges = false;
    }
    float most4[LOADS], mine = -INFINITY;
#pragma unroll
    for (int u = 0; u < LOADS; ++u) {
      most4[u] = fmaxf(fmaxf(v[u][0].x, v[u][0].y), fmaxf(v[u][1].x, v[u][1].y));
      mine = fmaxf(mine, most4[u]);
    }
    if constexpr (TOP) {
      so_far = max(so_far, mine == mine ? lp_ordered(mine) : 0u);  // (a NaN is no one's bound)
      if (raise) {
        uint32_t least;
        if (p.n_top <= LP_BINNED) {
          uint32_t most = so_far;
#pragma unroll
          for (int by = 1; by < 8; by <<= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, by));
          if ((lane & 7) == 0) *reinterpret_cast<volatile uint32_t*>(sh.bound + warp * 4 + (lane >> 3)) = most;
          if (g == w0) __syncthreads();  // later older numbers of the other warps serve as well: they only grow
          const uint32_t own = *reinterpret_cast<volatile uint32_t*>(sh.bound + lane);
          int reach = 0;
#pragma unroll
          for (int j = 0; j < 32; j += 4) {
            const uint4 y = lp_shared_u32x4(sh.bound + j);
            reach += (y.x >= own) + (y.y >= own) + (y.z >= own) + (y.w >= own);
          }
          least = __reduce_max_sync(0xffffffffu, reach >= p.n_top ? own : 0u);
        } else {
          uint32_t o = so_far, mth = 0;
          for (int i = 0; i < p.n_top; i += LP_WARPS) {  // the largest goes, one lane of it
            mth = __reduce_max_sync(0xffffffffu, o);
            if (lane == __ffs(__ballot_sync(0xffffffffu, o == mth)) - 1) o = 0;
          }
          if (lane == 0) *reinterpret_cast<volatile uint32_t*>(sh.bound + warp) = mth;
          if (g == w0) __syncthreads();
          least = lane < LP_WARPS ? *reinterpret_cast<volatile uint32_t*>(sh.bound + lane) : 0xffffffffu;
          least = __reduce_min_sync(0xffffffffu, least);
        }
        const uint64_t below = ((uint64_t)least << 32) - 1;
        top.bound = below + 1 > top.bound ? below : top.bound;
      }
      // What passes (keys from bound + 1 on) is above `edge`, or equal to it and of a number up to edge_id.
      float edge = lp_value((uint32_t)((top.bound + 1) >> 32));
      raise = __any_sync(0xffffffffu, mine >= edge);  // for the next slice: this one's may change it
      if (raise) {
        uint32_t edge_id = ~(uint32_t)(top.bound + 1), hits = 0;  // this lane's groups that pass
#pragma unroll
        for (int u = 0; u < LOADS; ++u) hits |= most4[u] >= edge ? 1u << u : 0u;
        do {  // once, mostly, for one or two lanes: each takes places by itself
          if (hits) {
            // (read again: a loop over registers would have to be unrolled, and its code fetched)
            const uint32_t id = first_id + (__ffs(hits) - 1) * 128;
            hits &= hits - 1;
            float y[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) y[c] = c < in_group ? x[id + c] : -INFINITY;
#pragma unroll
            for (int c = 0; c < 4; ++c)
              if (y[c] > edge || (y[c] == edge && id + c <= edge_id))
                buffer[atomicAdd(sh.held + warp, 1)] = lp_key(y[c], id + c);
          }
          __syncwarp();
          top.held = *reinterpret_cast<volatile int*>(sh.held + warp);
          if (top.held >= 32) {
            top = lp_flush(top, buffer, 32, p.n_top);
            if (lane == 0) *reinterpret_cast<volatile int*>(sh.held + warp) = top.held;
            __syncwarp();
            edge = lp_value((uint32_t)((top.bound + 1) >> 32));
            edge_id = ~(uint32_t)(top.bound + 1);
          }
        } while (__any_sync(0xffffffffu, hits != 0));
      }
    }
    const uint32_t most = __reduce_max_sync(0xffffffffu, lp_ordered(mine));
    const float now = fmaxf(s.m, lp_value(most));
    // Sums, relative to the largest yet; a new one is left out once, by the first lane that has it.
    if (now > s.m) {
      const unsigned who = __ballot_sync(0xffffffffu, lp_ordered(mine) == most);
      if (s.m != -INFINITY) {
        const float d = s.m - now, f = lp_exp(d), w = s.rest + (lane == 0 ? 1.0f : 0.0f);  // the old one counts now
        s.e = f == 0.0f ? 0.0f : f * fmaf(w, d, s.e);
        s.rest = f * w;
      }
      s.m = now;
      bool out = lane == __ffs(who) - 1;
      auto leave = [&](float& y) {
        const bool it = out && y == now;
        y = it ? -INFINITY : y;
        out = out && !it;
      };
#pragma unroll
      for (int u = 0; u < LOADS; ++u) leave(v[u][0].x), leave(v[u][0].y), leave(v[u][1].x), leave(v[u][1].y);
    }
    const float base = now == -INFINITY ? 0.0f : -now;
    const float2 base2 = make_float2(base, base), log2e = make_float2(LP_LOG2E, LP_LOG2E);
    float2 rest = make_float2(s.rest, 0.0f), e = make_float2(s.e, 0.0f);
#pragma unroll
    for (int u = 0; u < LOADS; ++u)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float2 d = lp_add2(v[u][c], base2), z = lp_mul2(d, log2e);
        const float2 w = make_float2(lp_exp2(z.x), lp_exp2(z.y));
        rest = lp_add2(rest, w);
        e = lp_fma2(w, make_float2(fmaxf(d.x, -1e30f), fmaxf(d.y, -1e30f)), e);  // -inf: 0 times a number
      }
    s.rest = rest.x + rest.y, s.e = e.x + e.y;
    if (!more && !edges) break;
  }
#pragma unroll
  for (int by = 16; by > 0; by >>= 1) {
    s.rest += __shfl_xor_sync(0xffffffffu, s.rest, by);
    s.e += __shfl_xor_sync(0xffffffffu, s.e, by);
  }
  if (lane == 0) sh.state[warp] = s;
  // What the CTA holds, joined: the warps' buffers, and their lists where a buffer has been full.
  const int listed = TOP ? __popc(__ballot_sync(0xffffffffu, top.list != 0)) : 0;
  if (TOP && lane == 0) sh.held[warp] = top.held + listed;
  __syncthreads();
  if constexpr (TOP) {
    int at = 0, n = 0;
#pragma unroll
    for (int w = 0; w < LP_WARPS; ++w) {
      if (w == warp) at = n;
      n += sh.held[w];
    }
    if (lane < listed) sh.keys[at + lane] = top.list;
    if (lane < top.held) sh.keys[at + listed + lane] = buffer[lane];
    if (tid == 0) sh.keys[n] = 0;
    if (tid < YSKN_MAX_TOP) sh.list[tid] = sh.row_list[tid] = 0;
    __syncthreads();
    lp_rank(sh.keys, n, sh.list, p.n_top, tid);
  }
  LpState t = lp_whole(sh.state, LP_WARPS, lane);
  if (p.cluster > 1) {
    if (TOP) __syncthreads();  // the list is whole
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // the first CTA has begun
    if (tid == 0) {
      const uint32_t to = lp_remote(sh.parts + rank, 0);
      lp_put_f32(to, t.m), lp_put_f32(to + 4, t.rest), lp_put_f32(to + 8, t.e);
    }
    if (TOP && tid < p.n_top) lp_put_u64(lp_remote(sh.lists + rank * p.n_top + tid, 0), sh.list[tid]);
    lp_cluster_sync();
    if (rank != 0) return;
    if (TOP) lp_rank_lists(sh.lists, p.cluster, p.n_top, sh.row_list, p.n_top, tid);
    t = lp_whole(sh.parts, p.cluster, lane);
  }
  if (TOP) __syncthreads();
  const bool none = t.m == -INFINITY && t.rest == 0.0f, bad = !(t.m < INFINITY) || !(t.rest < INFINITY);
  const float log_sum = log1pf(t.rest), nan = __int_as_float(0x7fc00000);
  asm volatile("cp.async.wait_all;" ::: "memory");  // each thread its own
  for (int j = tid; j < p.n_tokens; j += LP_THREADS) {
    const int id = j < LP_THREADS ? sh.id[j] : p.tokens[row * p.token_stride + j];
    float y = -INFINITY;
    if ((unsigned)id < (unsigned)p.vocab && !none) y = ((j < LP_THREADS ? sh.logit[j] : x[id]) - t.m) - log_sum;
    p.logprobs[(int64_t)row * p.n_tokens + j] = bad ? nan : y;
  }
  if (tid == 0 && p.entropy) p.entropy[row] = bad ? nan : none ? 0.0f : log_sum - t.e / (1.0f + t.rest);
  if (TOP && tid < p.n_top) {
    const uint64_t key = p.cluster > 1 ? sh.row_list[tid] : sh.list[tid];
    const int64_t at = (int64_t)row * p.n_top + tid;
    const bool any = key != 0 && !bad;
    p.top_logprobs[at] = bad ? nan : any ? (lp_value((uint32_t)(key >> 32)) - t.m) - log_sum : -INFINITY;
    p.top_ids[at] = any ? (int)~(uint32_t)key : -1;
  }
}

}  // namespace yskn

using namespace yskn;

extern "C" YSKN_B200_API int yskn_b200_token_logprobs(const yskn_b200_token_logprobs_args* args, void* stream) {
  if (!args) return fail(YSKN_EINVAL, "token_logprobs: null argument");
  const yskn_b200_token_logprobs_args& a = *args;
  if (!a.logits || a.rows < 1 || a.vocab < 1 || a.vocab > INT32_MAX - 65536 ||
      (a.rows > 1 && a.logits_stride < a.vocab))
    return fail(YSKN_EINVAL, "token_logprobs: null logits, empty shape, or a stride below the vocabulary");
  if (a.rows > INT32_MAX / LP_MAX_CLUSTER) return fail(YSKN_EINVAL, "token_logprobs: too many rows");
  if (a.n_tokens < 0 || (a.n_tokens > 0 && (!a.tokens || !a.logprobs || (a.rows > 1 && a.token_stride < a.n_tokens))))
    return fail(YSKN_EINVAL, "token_logprobs: tokens need an output and a stride of their number");
  if (a.n_top < 0 || a.n_top > YSKN_MAX_TOP || (a.n_top > 0 && (!a.top_logprobs || !a.top_ids)))
    return fail(YSKN_EINVAL, "token_logprobs: 0..32 top tokens, with both outputs");
  LogprobsParams p{a.logits, a.logits_stride, a.tokens, a.token_stride, a.logprobs, a.entropy, a.top_logprobs,
                   a.top_ids, a.vocab, a.n_tokens, a.n_top, 1};
  // CTAs of a row: as many as the SMs hold at once, with a slice for every warp of each. us at 151936 logits, 8
  // largest, with 1, 2, 4, 8: 64 rows (20 largest) 24.6, 18.6, 15.9, 25; 128 rows 21.7, 20.4, 25, 37; 256 rows 31.9,
  // 40, 49, 71; one row with 20 largest 22, 16.6, 11.5, 9.0; 33 rows of 50257 with 1, 2, 4, 8: 11.8, 9.6, 7.8, 10.2.
  while (p.cluster < LP_MAX_CLUSTER && (int64_t)a.rows * p.cluster * 2 <= 148 * LP_RESIDENT &&
         a.vocab / (p.cluster * 2) >= LP_LEAST_PART)
    p.cluster *= 2;
  // The slice whose last one of a warp's run is emptiest by fewest groups, the larger of two alike. us with 8, 10 loads
  // where 10 leave no more empty: one row of 151936 with 20 largest 9.0, 8.2, 256 rows 31.8, 30.9, 512 rows 60.0, 57.9;
  // where 8 leave less: 33 rows of 50257 7.8, 8.4, 512 rows of 32000 19.6, 20.9, of 2000 9.4, 10.0. (11 spill.)
  const int run = (int)ceil_div(ceil_div(a.vocab / 4, p.cluster), LP_WARPS);
  const bool many = ceil_div(run, LP_MANY * 32) * LP_MANY <= ceil_div(run, LP_FEW * 32) * LP_FEW;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = (unsigned)(a.rows * p.cluster);
  cfg.blockDim = LP_THREADS;
  cfg.stream = reinterpret_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)p.cluster, attr[1].val.clusterDim.y = 1, attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  auto launch = [&](auto loads) {
    constexpr int LOADS = decltype(loads)::value;
    return cuda_fail(a.n_top > 0 ? cudaLaunchKernelEx(&cfg, token_logprobs_kernel<true, LOADS>, p)
                                 : cudaLaunchKernelEx(&cfg, token_logprobs_kernel<false, LOADS>, p),
                     "token_logprobs_kernel");
  };
  return many ? launch(std::integral_constant<int, LP_MANY>{}) : launch(std::integral_constant<int, LP_FEW>{});
}
