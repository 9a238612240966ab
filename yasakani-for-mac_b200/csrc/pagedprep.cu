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
// W l .. W l + W - 1 of each 32 W (W = 4, or 2 where D = 64): every access of the warp is one
// run of adjacent bytes, the sum of squares comes by shuffles, and a pair's other half, R / 2 (a
// multiple of W) channels away, by one shuffle per channel (two where pairs straddle the runs).
// A warp takes up to PP_RUN heads of one token where there are many rows (one where there are
// few: chosen with the launch), each row requested while the one before is worked on (two rows
// ahead leaves room for fewer warps: 86 us for 8192 tokens, not 78; runs of 4: 84); the cosines and
// sines of its channels are computed once, one pair a lane, while its first rows arrive, and stay in
// registers. No block-wide step.
#include <algorithm>

#include "paged.cuh"

namespace yskn {

constexpr int PP_WARPS = 8;
constexpr int PP_MAX_PAIRS = YSKN_MAX_PAIRS;
constexpr int PP_RUN = 16;           // heads of a warp's run, at most
constexpr int PP_SETUP = 3;          // a warp's set-up in the time of a head
constexpr int PP_RESIDENT = 148 * 4;  // CTAs at a time

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

// Cosine and sine of a binary32 angle: reduced by its nearest multiple of pi / 2 in binary64 (two
// parts of pi / 2), then on [-pi / 4, pi / 4] polynomials that interpolate (sin r - r) / r^3 and
// (cos r - 1 + r^2 / 2) / r^4 at the Chebyshev nodes in r^2, in binary32: within 1e-7 (a unit of
// 1; the most in 200 million angles of all sizes was 9.4e-8). (With the decode path's portable function, binary64 throughout: 81 us for 8192 tokens,
// not 78.)
// False for an angle past 2^30, whose multiple is not held.
__device__ __forceinline__ bool turn_of(float angle, float2* turn) {
  const double v = (double)angle;
  const int n = __double2int_rn(v * 0.63661977236758134308);
  const double r64 = fma((double)n, -6.12323399573676603587e-17, fma((double)n, -1.57079632679489661923, v));
  const float r = (float)r64, t = r * r;
  const float s = fmaf(r * t, fmaf(t, fmaf(t, -1.958789088e-4f, 8.332748271e-3f), -1.666666466e-1f), r);
  const float u = fmaf(t, fmaf(t, 2.454794208e-5f, -1.388830304e-3f), 4.166666466e-2f);
  const float c = fmaf(t * t, u, fmaf(t, -0.5f, 1.0f));
  const float x = n & 1 ? s : c, y = n & 1 ? c : s;  // cosine and sine up to their signs
  *turn = make_float2((n + 1) & 2 ? -x : x, n & 2 ? -y : y);
  return fabsf(angle) < 1073741824.0f;
}

// W channels from W-element aligned memory, as f32.
template <int SRC, int W>
__device__ __forceinline__ void load_part(const void* base, int64_t at, float* x) {
  if constexpr (SRC == YSKN_DT_F32) {
    const float* p = reinterpret_cast<const float*>(base) + at;
    if constexpr (W == 2) {
      const float2 a = __ldg(reinterpret_cast<const float2*>(p));
      x[0] = a.x, x[1] = a.y;
    } else {
      const float4 a = __ldg(reinterpret_cast<const float4*>(p));
      x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
    }
  } else {
    const uint16_t* p = reinterpret_cast<const uint16_t*>(base) + at;
    uint32_t w[W / 2];
    if constexpr (W == 2) {
      w[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
    } else {
      const uint2 a = __ldg(reinterpret_cast<const uint2*>(p));
      w[0] = a.x, w[1] = a.y;
    }
#pragma unroll
    for (int j = 0; j < W / 2; ++j) {
      x[2 * j] = Elem<SRC>::to_float((uint16_t)w[j]);
      x[2 * j + 1] = Elem<SRC>::to_float((uint16_t)(w[j] >> 16));
    }
  }
}

template <int DT, int W>
__device__ __forceinline__ void store_part(uint16_t* p, const float* x) {
  if constexpr (W == 2) *reinterpret_cast<uint32_t*>(p) = Elem<DT>::pack(x[0], x[1]);
  else *reinterpret_cast<uint2*>(p) = make_uint2(Elem<DT>::pack(x[0], x[1]), Elem<DT>::pack(x[2], x[3]));
}

template <int SRC, int DT, int D>
__global__ void __launch_bounds__(PP_WARPS * 32, 4) paged_prep_kernel(const __grid_constant__ PagedPrepParams p) {
  constexpr int W = D == 64 ? 2 : 4, RUN = 32 * W, C = D / RUN;  // a lane's channels: W of each of C runs
  __shared__ float2 s_turn[PP_WARPS][PP_MAX_PAIRS];  // (cosine, sine) of the warp's token
  pdl_begin();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int heads = p.n_qh + 2 * p.n_kvh;  // query heads, then key heads, then value heads
  const int t = blockIdx.x * PP_WARPS + warp;
  if (t >= p.tokens) return;
  const int h0 = blockIdx.y * p.run, h1 = min(heads, h0 + p.run);
  auto load = [&](int h, float (&x)[C][W]) {
    const void* src;
    int64_t at;
    if (h < p.n_qh) src = p.q, at = t * p.q_row + h * p.q_head;
    else if (h < p.n_qh + p.n_kvh) src = p.k, at = t * p.k_row + (h - p.n_qh) * p.k_head;
    else src = p.v, at = t * p.v_row + (h - p.n_qh - p.n_kvh) * p.v_head;
#pragma unroll
    for (int c = 0; c < C; ++c) load_part<SRC, W>(src, at + c * RUN + lane * W, x[c]);
  };
  float x[C][W];
  load(h0, x);
  const int64_t slot = __ldg(p.slots + t);
  const int half = p.rot >> 1;
  for (int i = lane; i < half; i += 32) {
    const float pos = (float)__ldg(p.positions + p.axis[i] * p.position_stride + t);
    if (!turn_of(__fmul_rn(pos, __ldg(p.inv_freq + i)), &s_turn[warp][i])) raise_device_error(p.err, DERR_RANGE);
  }
  __syncwarp();
  // The turns of this lane's channels, the sine negated in a pair's first half: y = x cos + other sin;
  // (1, 0) for channels that are not rotated. `from`: the lane that holds the other half, `far`
  // whether it holds it in its other run.
  float cs[C][W], sn[C][W];
  int from[C];
  bool far[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int ch = c * RUN + lane * W;
    const bool rotated = ch < p.rot, low = ch < half;
    const int other = rotated ? (low ? ch + half : ch - half) : ch;
    from[c] = other % RUN / W;
    far[c] = other / RUN != c;
#pragma unroll
    for (int j = 0; j < W; ++j) {
      const float2 turn = rotated ? s_turn[warp][(low ? ch : ch - half) + j] : make_float2(1.0f, 0.0f);
      cs[c][j] = turn.x;
      sn[c][j] = low ? -turn.y : turn.y;
    }
  }
  int64_t block, place;  // a 64-bit division takes longer than the rest of the set-up
  if ((uint64_t)slot <= UINT32_MAX) block = (uint32_t)slot / (uint32_t)p.block_size;
  else block = slot >= 0 ? slot / p.block_size : 0;
  place = slot - block * p.block_size;
  const int64_t to = block * p.cache.block + place * p.cache.token + lane * W;
  if (slot >= p.n_slots && lane == 0) raise_device_error(p.err, DERR_RANGE);
  const uint16_t* w_of = nullptr;  // what `scale` holds 1 + w of
  float scale[C][W];
  for (int h = h0; h < h1; ++h) {
    float after[C][W];
    if (h + 1 < h1) load(h + 1, after);
    const bool query = h < p.n_qh, value = h >= p.n_qh + p.n_kvh;
    if (!value) {
      const uint16_t* w = query ? p.q_norm : p.k_norm;
      if (w) {
        if (w != w_of) {
          w_of = w;
#pragma unroll
          for (int c = 0; c < C; ++c) {
            load_part<YSKN_DT_BF16, W>(w, c * RUN + lane * W, scale[c]);
#pragma unroll
            for (int j = 0; j < W; ++j) scale[c][j] += 1.0f;
          }
        }
        float sum = 0.0f;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int j = 0; j < W; ++j) sum = fmaf(x[c][j], x[c][j], sum);
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
        const float inv = rsqrtf(sum * (1.0f / D) + p.eps);
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int j = 0; j < W; ++j) x[c][j] = x[c][j] * inv * scale[c][j];
      }
      if (half) {
        if (C == 1 || p.rot <= RUN) {  // pairs within the first run
#pragma unroll
          for (int j = 0; j < W; ++j) {
            const float o = __shfl_sync(0xffffffffu, x[0][j], from[0]);
            x[0][j] = fmaf(x[0][j], cs[0][j], o * sn[0][j]);
          }
        } else {
#pragma unroll
          for (int j = 0; j < W; ++j) {
            float o[C];
#pragma unroll
            for (int c = 0; c < C; ++c) {
              const float near_one = __shfl_sync(0xffffffffu, x[c][j], from[c]);
              const float far_one = __shfl_sync(0xffffffffu, x[C - 1 - c][j], from[c]);
              o[c] = far[c] ? far_one : near_one;
            }
#pragma unroll
            for (int c = 0; c < C; ++c) x[c][j] = fmaf(x[c][j], cs[c][j], o[c] * sn[c][j]);
          }
        }
      }
    }
    if (query) {
      if (slot < 0) {
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int j = 0; j < W; ++j) x[c][j] = 0.0f;
      }
#pragma unroll
      for (int c = 0; c < C; ++c)
        store_part<DT, W>(p.query + ((int64_t)t * p.n_qh + h) * D + c * RUN + lane * W, x[c]);
    } else if (slot >= 0 && slot < p.n_slots) {
      uint16_t* row = (value ? p.v_cache + (h - p.n_qh - p.n_kvh) * p.cache.head
                             : p.k_cache + (h - p.n_qh) * p.cache.head) + to;
#pragma unroll
      for (int c = 0; c < C; ++c) store_part<DT, W>(row + c * RUN, x[c]);
    }
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int j = 0; j < W; ++j) x[c][j] = after[c][j];
  }
}

template <int SRC, int DT>
static cudaError_t launch_paged_prep(const PagedPrepParams& p, int head, dim3 grid, cudaStream_t st) {
  switch (head) {
    case 64: return launch_pdl(paged_prep_kernel<SRC, DT, 64>, grid, PP_WARPS * 32, 0, st, p);
    case 128: return launch_pdl(paged_prep_kernel<SRC, DT, 128>, grid, PP_WARPS * 32, 0, st, p);
    default: return launch_pdl(paged_prep_kernel<SRC, DT, 256>, grid, PP_WARPS * 32, 0, st, p);
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
  // The run that takes the least time in whole rounds of resident CTAs (300 tokens of 30 heads of 128: 8.7 us
  // with runs that just fill the SMs, 6.0 so; 1037 tokens 11.8, 10.6; 3000 of 32 heads of 256 31.1, 29.7).
  int64_t least = INT64_MAX;
  for (int run = 1; run <= std::min(PP_RUN, heads); ++run) {
    const int64_t time = ceil_div(ceil_div(a.tokens, PP_WARPS) * ceil_div(heads, run), PP_RESIDENT) * (PP_SETUP + run);
    if (time < least) least = time, p.run = run;
  }
  const int64_t runs = ceil_div(heads, std::max(p.run, 1));
  if (heads < 0 || runs > 65535) return fail(YSKN_EINVAL, "paged_prep: too many heads");
  const dim3 grid((unsigned)ceil_div(a.tokens, PP_WARPS), (unsigned)runs);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (a.dtype == YSKN_DT_BF16)
    e = a.source == YSKN_DT_F32 ? launch_paged_prep<YSKN_DT_F32, YSKN_DT_BF16>(p, a.head, grid, st)
                                : launch_paged_prep<YSKN_DT_BF16, YSKN_DT_BF16>(p, a.head, grid, st);
  else
    e = a.source == YSKN_DT_F32 ? launch_paged_prep<YSKN_DT_F32, YSKN_DT_F16>(p, a.head, grid, st)
                                : launch_paged_prep<YSKN_DT_F16, YSKN_DT_F16>(p, a.head, grid, st);
  return cuda_fail(e, "paged_prep_kernel");
}
