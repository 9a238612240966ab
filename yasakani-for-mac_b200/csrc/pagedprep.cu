// Query and key heads of a batch's new tokens normalised and rotated, and the new key and
// value rows into the paged cache, in one pass.
//
// Per token t and head, with x the projection row (f32, bf16 or f16) in binary32:
//   queries and keys: y = x * rsqrt(mean(x^2) + eps) * (1 + w) (without w: y = x), then for
//   each pair i < R / 2 of the rotated channels, with the angle a = float(position) * freq[i]
//   (a binary32 product, as the decode path's rotation; position from the pair's axis):
//     (y[i], y[i + R/2]) <- (y[i] cos a - y[i + R/2] sin a, y[i + R/2] cos a + y[i] sin a)
//   values: y = x. Every result is rounded once, to the cache's type.
// Queries go to a dense array, keys and values to the cache place that the token's slot
// names; a token with a negative slot (a padded place of the batch) writes no cache row, and
// zeros as its query.
//
// What bounds it: bytes (each row read once and written once; 48 KB a token at 24 + 4 + 4
// heads of 256 from f32). So one warp holds one head row in registers, lane l the channels
// V l .. V l + V - 1 (V = D / 32): 16-byte accesses, the sum of squares by shuffles, and a
// pair's other half R / 2 channels away is V-aligned in another lane, one shuffle per
// channel. A warp takes up to PP_RUN heads of one token where there are many rows (one where
// there are few), each row requested two rows ahead, and computes the token's R / 2 cosines and
// sines once, one pair a lane, while its first rows arrive. No block-wide step. The cosine and
// sine are the portable ones of the decode path's rotation (binary64 reduction).
#include <algorithm>

#include "paged.cuh"
#include "pmath.cuh"

namespace yskn {

constexpr int PP_WARPS = 8;
constexpr int PP_MAX_PAIRS = YSKN_MAX_PAIRS;
constexpr int PP_RUN = 8;         // heads of a warp's run, at most
constexpr int PP_FULL = 148 * 16;  // warps that keep the SMs busy: runs get longer beyond that

struct PagedPrepParams {
  const void *q, *k, *v;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;  // strides in elements
  const int64_t* slots;
  const int32_t* positions;  // [axes][position_stride]
  int64_t position_stride;
  const float* inv_freq;  // [rot / 2]
  const uint16_t *q_norm, *k_norm;  // bf16 [D] or nullptr
  float eps;
  int tokens, n_qh, n_kvh, rot;
  int run;  // heads of one token that a warp takes
  uint16_t* query;  // [tokens][n_qh][D]
  uint16_t *k_cache, *v_cache;
  CacheStrides cache;
  int block_size;
  int64_t n_slots;
  unsigned* err;
  uint8_t axis[PP_MAX_PAIRS];
};

// V consecutive channels from 16-byte aligned (or V-element aligned) memory, as f32.
template <int SRC, int V>
__device__ __forceinline__ void load_row(const void* base, int64_t at, float (&x)[V]) {
  if constexpr (SRC == YSKN_DT_F32) {
    const float* p = reinterpret_cast<const float*>(base) + at;
    if constexpr (V == 2) {
      const float2 a = __ldg(reinterpret_cast<const float2*>(p));
      x[0] = a.x, x[1] = a.y;
    } else {
#pragma unroll
      for (int j = 0; j < V; j += 4) {
        const float4 a = __ldg(reinterpret_cast<const float4*>(p + j));
        x[j] = a.x, x[j + 1] = a.y, x[j + 2] = a.z, x[j + 3] = a.w;
      }
    }
  } else {
    const uint16_t* p = reinterpret_cast<const uint16_t*>(base) + at;
    uint32_t w[V / 2];
    if constexpr (V == 2) w[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
    else if constexpr (V == 4) {
      const uint2 a = __ldg(reinterpret_cast<const uint2*>(p));
      w[0] = a.x, w[1] = a.y;
    } else {
      const uint4 a = __ldg(reinterpret_cast<const uint4*>(p));
      w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w;
    }
#pragma unroll
    for (int j = 0; j < V / 2; ++j) {
      x[2 * j] = Elem<SRC>::to_float((uint16_t)w[j]);
      x[2 * j + 1] = Elem<SRC>::to_float((uint16_t)(w[j] >> 16));
    }
  }
}

template <int DT, int V>
__device__ __forceinline__ void store_row(uint16_t* p, const float (&x)[V]) {
  uint32_t w[V / 2];
#pragma unroll
  for (int j = 0; j < V / 2; ++j) w[j] = Elem<DT>::pack(x[2 * j], x[2 * j + 1]);
  if constexpr (V == 2) *reinterpret_cast<uint32_t*>(p) = w[0];
  else if constexpr (V == 4) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  else *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

template <int SRC, int DT, int V>
__global__ void __launch_bounds__(PP_WARPS * 32) paged_prep_kernel(const __grid_constant__ PagedPrepParams p) {
  constexpr int D = 32 * V;
  __shared__ float2 s_turn[PP_WARPS][PP_MAX_PAIRS];  // (cosine, sine) of the warp's token
  pdl_begin();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int heads = p.n_qh + 2 * p.n_kvh;  // query heads, then key heads, then value heads
  const int runs = (heads + p.run - 1) / p.run;
  const int64_t item = (int64_t)blockIdx.x * PP_WARPS + warp;
  if (item >= (int64_t)p.tokens * runs) return;
  const int t = (int)(item / runs), h0 = (int)(item - (int64_t)t * runs) * p.run, h1 = min(heads, h0 + p.run);
  auto load = [&](int h, float (&x)[V]) {
    if (h < p.n_qh) load_row<SRC, V>(p.q, t * p.q_row + h * p.q_head + lane * V, x);
    else if (h < p.n_qh + p.n_kvh) load_row<SRC, V>(p.k, t * p.k_row + (h - p.n_qh) * p.k_head + lane * V, x);
    else load_row<SRC, V>(p.v, t * p.v_row + (h - p.n_qh - p.n_kvh) * p.v_head + lane * V, x);
  };
  float x[V], next[V];
  load(h0, x);
  if (h0 + 1 < h1) load(h0 + 1, next);
  const int64_t slot = __ldg(p.slots + t);
  const int half = p.rot >> 1;
  for (int i = lane; i < half; i += 32) {
    const float pos = (float)__ldg(p.positions + p.axis[i] * p.position_stride + t);
    float sn, cs;
    if (!pm_sincos(__fmul_rn(pos, __ldg(p.inv_freq + i)), &cs, &sn)) raise_device_error(p.err, DERR_RANGE);
    s_turn[warp][i] = make_float2(cs, sn);
  }
  __syncwarp();
  const int lanes = half / V;  // lanes of each half of the rotated channels
  const bool low = lane < lanes, rotated = lane < 2 * lanes;
  const int other = rotated ? (low ? lane + lanes : lane - lanes) : lane;
  const int i0 = rotated ? (low ? lane : lane - lanes) * V : 0;
  const int64_t block = slot >= 0 ? slot / p.block_size : 0, place = slot - block * p.block_size;
  const int64_t to = block * p.cache.block + place * p.cache.token + lane * V;
  if (slot >= p.n_slots && lane == 0) raise_device_error(p.err, DERR_RANGE);
  for (int h = h0; h < h1; ++h) {
    float after[V];
    if (h + 2 < h1) load(h + 2, after);
    const bool query = h < p.n_qh, value = h >= p.n_qh + p.n_kvh;
    if (!value) {
      const uint16_t* w = query ? p.q_norm : p.k_norm;
      if (w) {
        float wt[V];
        load_row<YSKN_DT_BF16, V>(w, lane * V, wt);
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < V; ++j) sum = fmaf(x[j], x[j], sum);
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
        const float inv = rsqrtf(sum * (1.0f / D) + p.eps);
#pragma unroll
        for (int j = 0; j < V; ++j) x[j] = x[j] * inv * (1.0f + wt[j]);
      }
      if (half) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float o = __shfl_sync(0xffffffffu, x[j], other);
          const float2 turn = s_turn[warp][i0 + j];
          if (rotated) x[j] = low ? fmaf(x[j], turn.x, -(o * turn.y)) : fmaf(x[j], turn.x, o * turn.y);
        }
      }
    }
    if (query) {
      if (slot < 0) {
#pragma unroll
        for (int j = 0; j < V; ++j) x[j] = 0.0f;
      }
      store_row<DT, V>(p.query + ((int64_t)t * p.n_qh + h) * D + lane * V, x);
    } else if (slot >= 0 && slot < p.n_slots) {
      const int kvh = value ? h - p.n_qh - p.n_kvh : h - p.n_qh;
      store_row<DT, V>((value ? p.v_cache : p.k_cache) + to + kvh * p.cache.head, x);
    }
#pragma unroll
    for (int j = 0; j < V; ++j) x[j] = next[j], next[j] = after[j];
  }
}

template <int SRC, int DT>
static cudaError_t launch_paged_prep(const PagedPrepParams& p, int head, unsigned grid, cudaStream_t st) {
  switch (head) {
    case 64: return launch_pdl(paged_prep_kernel<SRC, DT, 2>, grid, PP_WARPS * 32, 0, st, p);
    case 128: return launch_pdl(paged_prep_kernel<SRC, DT, 4>, grid, PP_WARPS * 32, 0, st, p);
    default: return launch_pdl(paged_prep_kernel<SRC, DT, 8>, grid, PP_WARPS * 32, 0, st, p);
  }
}

}  // namespace yskn

using namespace yskn;

extern "C" YSKN_B200_API int yskn_b200_paged_prep(const yskn_b200_paged_prep_args* args, void* stream) {
  if (!args) return fail(YSKN_EINVAL, "paged_prep: null argument");
  yskn_b200_paged_prep_args a = *args;
  if (!a.q || !a.k || !a.v || !a.slots || !a.query || !a.k_cache || !a.v_cache ||
      (a.rot > 0 && (!a.positions || !a.inv_freq)))
    return fail(YSKN_EINVAL, "paged_prep: null argument");
  if (a.head != 64 && a.head != 128 && a.head != 256)
    return fail(YSKN_EINVAL, "paged_prep: heads of 64, 128 or 256 channels");
  if (!is_16bit(a.dtype) || (a.source != YSKN_DT_F32 && a.source != a.dtype))
    return fail(YSKN_EINVAL, "paged_prep: the cache is f16 or bf16, the projections f32 or of the cache's type");
  if (a.tokens < 1 || a.n_qh < 1 || a.n_kvh < 1 || a.rot < 0 || a.rot > a.head || a.rot % 16 || a.n_blocks < 1 ||
      a.block_size < 1)
    return fail(YSKN_EINVAL, "paged_prep: empty shape, or rotated channels not a multiple of 16 up to the head's");
  for (int i = 0; i < a.rot / 2; ++i)
    if (a.axes[i] >= a.n_axes || a.axes[i] > 2)
      return fail(YSKN_EINVAL, "paged_prep: a pair's axis is 0, 1 or 2, and one of the positions'");
  if (a.tokens == 1) a.q_row = a.k_row = a.v_row = 0;  // strides that nothing steps over may be anything
  if (a.n_qh == 1) a.q_head = 0;
  if (a.n_kvh == 1) a.k_head = a.v_head = a.head_stride = 0;
  if (a.block_size == 1) a.token_stride = 0;
  if (a.n_blocks == 1) a.block_stride = 0;
  const int64_t unit = a.source == YSKN_DT_F32 ? 4 : 8;  // elements of 16 bytes
  if (!aligned16(a.q) || !aligned16(a.k) || !aligned16(a.v) || !aligned16(a.query) || !aligned16(a.k_cache) ||
      !aligned16(a.v_cache) || (a.q_row | a.q_head | a.k_row | a.k_head | a.v_row | a.v_head) % unit ||
      (a.block_stride | a.token_stride | a.head_stride) % 8 || !aligned16(a.q_norm) || !aligned16(a.k_norm))
    return fail(YSKN_EINVAL, "paged_prep: pointers and strides are multiples of 16 bytes");
  PagedPrepParams p{};
  p.q = a.q, p.k = a.k, p.v = a.v;
  p.q_row = a.q_row, p.q_head = a.q_head, p.k_row = a.k_row, p.k_head = a.k_head, p.v_row = a.v_row, p.v_head = a.v_head;
  p.slots = a.slots, p.positions = a.positions, p.position_stride = a.position_stride, p.inv_freq = a.inv_freq;
  p.q_norm = a.q_norm, p.k_norm = a.k_norm, p.eps = a.eps;
  p.tokens = a.tokens, p.n_qh = a.n_qh, p.n_kvh = a.n_kvh, p.rot = a.rot;
  p.query = reinterpret_cast<uint16_t*>(a.query);
  p.k_cache = reinterpret_cast<uint16_t*>(a.k_cache), p.v_cache = reinterpret_cast<uint16_t*>(a.v_cache);
  p.cache = {a.block_stride, a.token_stride, a.head_stride};
  p.block_size = a.block_size, p.n_slots = (int64_t)a.n_blocks * a.block_size;
  p.err = device_error_word();
  for (int i = 0; i < a.rot / 2; ++i) p.axis[i] = a.axes[i];
  const int heads = a.n_qh + 2 * a.n_kvh;
  p.run = (int)std::min<int64_t>(PP_RUN, std::max<int64_t>(1, (int64_t)a.tokens * heads / PP_FULL));
  const int64_t grid = ceil_div(a.tokens * ceil_div(heads, p.run), PP_WARPS);
  if (grid > (int64_t)INT32_MAX) return fail(YSKN_EINVAL, "paged_prep: too many rows");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (a.dtype == YSKN_DT_BF16)
    e = a.source == YSKN_DT_F32 ? launch_paged_prep<YSKN_DT_F32, YSKN_DT_BF16>(p, a.head, (unsigned)grid, st)
                                : launch_paged_prep<YSKN_DT_BF16, YSKN_DT_BF16>(p, a.head, (unsigned)grid, st);
  else
    e = a.source == YSKN_DT_F32 ? launch_paged_prep<YSKN_DT_F32, YSKN_DT_F16>(p, a.head, (unsigned)grid, st)
                                : launch_paged_prep<YSKN_DT_F16, YSKN_DT_F16>(p, a.head, (unsigned)grid, st);
  return cuda_fail(e, "paged_prep_kernel");
}
