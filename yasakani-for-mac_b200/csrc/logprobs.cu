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
// A warp streams slices of 4096 bytes (8 16-byte loads a lane under way at once) by itself: its
// maximum, its sums, and its list of the 32 largest in registers, one a lane, sorted. A logit is a
// key: its bits in an order of unsigned numbers, above the complement of its number, so that keys are
// all different and equal logits go by the lowest number. What exceeds the list's n_top-th key goes to a
// buffer in shared memory; 32 of them are sorted (bitonic, in registers) and merged into the
// list at once, since one at a time costs as long a chain of shuffles each. The first slice has no
// such key: the n_top-th largest of its lanes' maxima serves, which at least n_top logits reach.
#include <algorithm>

#include "common.cuh"

namespace yskn {

constexpr int LP_WARPS = 8, LP_THREADS = LP_WARPS * 32;
constexpr int LP_LOADS = 8;                         // 16-byte loads of a lane in a slice
constexpr int LP_SLICE = LP_LOADS * 32;             // 16-byte groups of a warp's slice
constexpr int LP_MAX_CLUSTER = 8;
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

__device__ __forceinline__ float lp_exp(float d) {  // d <= 0, -inf included
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(d * LP_LOG2E));
  return y;
}
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

// ---- the cluster
__device__ __forceinline__ void lp_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t lp_remote(const void* p, int rank) {
  uint32_t a;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
  return a;
}
__device__ __forceinline__ uint64_t lp_remote_u64(uint32_t a) {
  uint64_t v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ float lp_remote_f32(uint32_t a) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}

struct LpShared {
  uint64_t buffer[LP_WARPS][64];
  uint64_t list[LP_WARPS][32];   // each warp's, then each CTA's of the cluster
  LpState state[LP_WARPS];
  uint64_t part_list[32];        // this CTA's, for rank 0
  LpState part;
};

// n (1..8) lists and states in shared memory into the first; all threads.
__device__ __forceinline__ void lp_merge_all(LpShared& sh, int n, bool top, int warp, int lane) {
  for (int step = 4; step > 0; step >>= 1) {
    __syncthreads();
    if (warp < step && warp + step < n) {
      if (top) {
        const uint64_t up = sh.list[warp + step][31 - lane];  // descending, so this is ascending
        sh.list[warp][lane] = lp_merge(sh.list[warp][lane], up, lane);
      }
      if (lane == 0) sh.state[warp] = lp_join(sh.state[warp], sh.state[warp + step]);
    }
  }
  __syncthreads();
}

template <bool TOP>
__global__ void __launch_bounds__(LP_THREADS, 3) token_logprobs_kernel(const __grid_constant__ LogprobsParams p) {
  __shared__ LpShared sh;
  pdl_begin();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.x / p.cluster, rank = blockIdx.x - row * p.cluster;
  const float* x = p.logits + row * p.logits_stride;
  // The row as 16-byte groups: `skew` logits before it fill its first group up. Groups of this part.
  const int skew = (int)(reinterpret_cast<uintptr_t>(x) >> 2 & 3), end = skew + p.vocab;
  const float4* groups = reinterpret_cast<const float4*>(x - skew);
  const int n_groups = (end + 3) >> 2, per = (n_groups + p.cluster - 1) / p.cluster;
  const int g0 = min(rank * per, n_groups), g1 = min(g0 + per, n_groups);

  LpState s{-INFINITY, 0.0f, 0.0f};  // m: of the warp; rest and e: of the lane
  const uint64_t lowest = (uint64_t)lp_ordered(-INFINITY) << 32 | 0xffffffffu;  // only logits above -inf pass
  uint64_t list = 0, bound = lowest;
  int held = 0;  // keys in the warp's buffer
  bool fresh = true;
  uint64_t* buffer = sh.buffer[warp];
  auto flush = [&]() {  // the buffer's first 32 into the list
    __syncwarp();
    const uint64_t v = lane < held ? buffer[lane] : 0, rest = lane + 32 < held ? buffer[lane + 32] : 0;
    __syncwarp();
    buffer[lane] = rest;
    held = max(held - 32, 0);
    list = lp_merge(list, lp_sort_up(v, lane), lane);
    const uint64_t last = __shfl_sync(0xffffffffu, list, p.n_top - 1);
    bound = last > bound ? last : bound;
  };
  for (int g = g0 + warp * LP_SLICE; g < g1; g += LP_WARPS * LP_SLICE) {
    float v[LP_LOADS][4];
#pragma unroll
    for (int u = 0; u < LP_LOADS; ++u) {
      const int at = g + u * 32 + lane, i = 4 * at;
      float4 y = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
      if (at < g1) {
        if (i >= skew && i + 4 <= end) {
          y = __ldcs(groups + at);
        } else {  // the row's first and last group, of which only its own logits are read
          const float* z = x - skew + i;
          if (i >= skew && i < end) y.x = z[0];
          if (i + 1 >= skew && i + 1 < end) y.y = z[1];
          if (i + 2 >= skew && i + 2 < end) y.z = z[2];
          if (i + 3 >= skew && i + 3 < end) y.w = z[3];
        }
      }
      v[u][0] = y.x, v[u][1] = y.y, v[u][2] = y.z, v[u][3] = y.w;
    }
    float top4[LP_LOADS], mine = -INFINITY;
#pragma unroll
    for (int u = 0; u < LP_LOADS; ++u) {
      top4[u] = fmaxf(fmaxf(v[u][0], v[u][1]), fmaxf(v[u][2], v[u][3]));
      mine = fmaxf(mine, top4[u]);
    }
    const uint32_t most = __reduce_max_sync(0xffffffffu, lp_ordered(mine));
    const float now = fmaxf(s.m, lp_value(most));
    // Sums, relative to the largest yet; a new one is left out once, by the first lane that has it.
    if (now > s.m) {
      const unsigned who = __ballot_sync(0xffffffffu, lp_ordered(mine) == most);
      bool skip = lane == __ffs(who) - 1;
      if (s.m != -INFINITY) {
        const float d = s.m - now, f = lp_exp(d), w = s.rest + (lane == 0 ? 1.0f : 0.0f);  // the old one counts now
        s.e = f == 0.0f ? 0.0f : f * fmaf(w, d, s.e);
        s.rest = f * w;
      }
      s.m = now;
#pragma unroll
      for (int u = 0; u < LP_LOADS; ++u)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const float d = v[u][c] - now;
          const bool out = skip && v[u][c] == now;
          const float w = out ? 0.0f : lp_exp(d);
          skip = skip && !out;
          s.rest += w;
          s.e = fmaf(w, fmaxf(d, -1e30f), s.e);
        }
    } else {
      const float base = now == -INFINITY ? 0.0f : now;
      float rest[2] = {s.rest, 0.0f}, e[2] = {s.e, 0.0f};
#pragma unroll
      for (int u = 0; u < LP_LOADS; ++u)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const float d = v[u][c] - base, w = lp_exp(d);
          rest[c & 1] += w;
          e[c & 1] = fmaf(w, fmaxf(d, -1e30f), e[c & 1]);
        }
      s.rest = rest[0] + rest[1], s.e = e[0] + e[1];
    }
    if constexpr (TOP) {
      if (fresh) {  // at least n_top of the slice's logits reach the n_top-th of the lanes' maxima
        uint32_t o = lp_ordered(mine);
        o = mine == mine ? o : 0;  // a NaN is no one's bound
#pragma unroll
        for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
          for (int by = size >> 1; by > 0; by >>= 1) {
            const uint32_t other = __shfl_xor_sync(0xffffffffu, o, by);
            o = (o > other) == (((lane & by) == 0) == ((lane & size) == 0)) ? o : other;
          }
        // descending in lanes now
        const uint64_t least = ((uint64_t)__shfl_sync(0xffffffffu, o, p.n_top - 1) << 32) - 1;
        bound = least + 1 > bound ? least : bound;
        fresh = false;
      }
#pragma unroll
      for (int u = 0; u < LP_LOADS; ++u) {
        float edge = lp_value((uint32_t)((bound + 1) >> 32));  // what passes is at least this
        if (!__any_sync(0xffffffffu, top4[u] >= edge)) continue;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int id = 4 * (g + u * 32 + lane) + c - skew;
          const uint64_t key = lp_key(v[u][c], id);
          const bool pass = v[u][c] >= edge && key > bound;
          const unsigned who = __ballot_sync(0xffffffffu, pass);
          if (who == 0) continue;
          if (pass) buffer[held + __popc(who & ((1u << lane) - 1))] = key;
          held += __popc(who);
          if (held >= 32) {
            flush();
            edge = lp_value((uint32_t)((bound + 1) >> 32));
          }
        }
      }
    }
  }
  if constexpr (TOP) {
    if (held > 0) flush();
    sh.list[warp][lane] = list;
  }
#pragma unroll
  for (int by = 16; by > 0; by >>= 1) {
    s.rest += __shfl_xor_sync(0xffffffffu, s.rest, by);
    s.e += __shfl_xor_sync(0xffffffffu, s.e, by);
  }
  if (lane == 0) sh.state[warp] = s;
  lp_merge_all(sh, LP_WARPS, TOP, warp, lane);
  if (p.cluster > 1) {
    if (warp == 0) {
      if (TOP) sh.part_list[lane] = sh.list[0][lane];
      if (lane == 0) sh.part = sh.state[0];
    }
    lp_cluster_sync();
    if (rank == 0) {
      if (warp < p.cluster) {
        const uint32_t from = lp_remote(&sh.part, warp);
        if (lane == 0)
          sh.state[warp] = LpState{lp_remote_f32(from), lp_remote_f32(from + 4), lp_remote_f32(from + 8)};
        if (TOP) sh.list[warp][lane] = lp_remote_u64(lp_remote(&sh.part_list[lane], warp));
      }
      lp_merge_all(sh, p.cluster, TOP, warp, lane);
    }
    lp_cluster_sync();  // the others' memory has been read
    if (rank != 0) return;
  }
  const LpState t = sh.state[0];
  const bool none = t.m == -INFINITY && t.rest == 0.0f, bad = !(t.m < INFINITY) || !(t.rest < INFINITY);
  const float log_sum = log1pf(t.rest), nan = __int_as_float(0x7fc00000);
  for (int j = tid; j < p.n_tokens; j += LP_THREADS) {
    const int id = p.tokens[row * p.token_stride + j];
    float y = -INFINITY;
    if ((unsigned)id < (unsigned)p.vocab && !none) y = (x[id] - t.m) - log_sum;
    p.logprobs[(int64_t)row * p.n_tokens + j] = bad ? nan : y;
  }
  if (tid == 0 && p.entropy) p.entropy[row] = bad ? nan : none ? 0.0f : log_sum - t.e / (1.0f + t.rest);
  if (TOP && tid < p.n_top) {
    const uint64_t key = sh.list[0][tid];
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
  // CTAs of a row: as many as keep about four on each SM, with a slice for every warp of each.
  while (p.cluster < LP_MAX_CLUSTER && (int64_t)a.rows * p.cluster * 2 <= 4 * 148 &&
         a.vocab / (p.cluster * 2) >= LP_WARPS * LP_SLICE * 4 / 2)
    p.cluster *= 2;
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
  return cuda_fail(a.n_top > 0 ? cudaLaunchKernelEx(&cfg, token_logprobs_kernel<true>, p)
                               : cudaLaunchKernelEx(&cfg, token_logprobs_kernel<false>, p),
                   "token_logprobs_kernel");
}
