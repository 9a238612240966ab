// Attention of a batch's new tokens over a prefix that all its requests share and each
// request's own rows, both in blocks of a paged 16-bit cache, with the output gate.
//
// Token t of request i (its n tokens are the last of its len rows, the prefix's P counted)
// sees the first lim = max(0, len - n + t + 1) rows of the sequence: rows below P in the
// prefix's blocks, the others in the request's. Per query head, in binary32:
//   s_j = scale * <q, k_j>, out = sum_j exp(s_j - max s) v_j / sum_j exp(s_j - max s)
//   out *= 1 / (1 + exp(-gate))  (with a gate), rounded once. A token that sees nothing gives 0.
// Rows at or past lim are not read into any sum, whatever the cache holds there.
#include <algorithm>

#include "paged.cuh"

namespace yskn {

struct PrefixAttnParams {
  const uint16_t *q, *gate;
  int64_t q_row, q_head, gate_row, gate_head;
  const uint16_t *k_cache, *v_cache;
  CacheStrides cache;
  int n_blocks, block_size;
  const int32_t* prefix_blocks;
  int prefix_len;
  const int32_t* tables;
  int64_t table_stride;
  int table_width;
  const int32_t *lens, *starts;
  int batch, tokens, max_new, n_qh, n_kvh;
  float scale;
  uint16_t* out;  // [tokens][n_qh][D]
  unsigned* err;
};

// The last request whose first token is at or before t (requests without tokens share a
// start with the next one), or the batch if t is past the last token.
__device__ __forceinline__ int request_of(const int32_t* starts, int batch, int t) {
  if (t >= __ldg(starts + batch)) return batch;
  int lo = 0, hi = batch;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(starts + mid) <= t) lo = mid;
    else hi = mid;
  }
  return lo;
}

// One warp per (token, query head); lane l holds channels V l .. V l + V - 1.
template <int DT, int V>
__global__ void __launch_bounds__(256) prefix_attention_kernel(const __grid_constant__ PrefixAttnParams p) {
  constexpr int D = 32 * V;
  pdl_begin();
  const int lane = threadIdx.x & 31;
  const int64_t item = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (item >= (int64_t)p.tokens * p.n_qh) return;
  const int t = (int)(item / p.n_qh), h = (int)(item - (int64_t)t * p.n_qh), kvh = h / (p.n_qh / p.n_kvh);
  const int i = request_of(p.starts, p.batch, t);
  int lim = 0;
  if (i < p.batch) {
    const int s0 = __ldg(p.starts + i), n = __ldg(p.starts + i + 1) - s0;
    lim = max(0, __ldg(p.lens + i) - n + (t - s0) + 1);
    if (n > p.max_new) {
      if (lane == 0) raise_device_error(p.err, DERR_RANGE);
      lim = 0;
    }
    lim = min((int64_t)lim, (int64_t)p.prefix_len + (int64_t)p.table_width * p.block_size);
  }
  float q[V], o[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    q[j] = Elem<DT>::to_float(p.q[t * p.q_row + h * p.q_head + lane * V + j]) * p.scale;
    o[j] = 0.0f;
  }
  float top = -INFINITY, den = 0.0f;
  for (int r = 0; r < lim; ++r) {
    const bool shared = r < p.prefix_len;
    const int at = shared ? r : r - p.prefix_len;
    const int block = shared ? __ldg(p.prefix_blocks + at / p.block_size)
                             : __ldg(p.tables + i * p.table_stride + at / p.block_size);
    if ((unsigned)block >= (unsigned)p.n_blocks) {
      if (lane == 0) raise_device_error(p.err, DERR_RANGE);
      continue;
    }
    const int64_t row = block * p.cache.block + (at % p.block_size) * p.cache.token + kvh * p.cache.head + lane * V;
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < V; ++j) s = fmaf(q[j], Elem<DT>::to_float(p.k_cache[row + j]), s);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    const float next = fmaxf(top, s), keep = top == -INFINITY ? 0.0f : expf(top - next), w = expf(s - next);
    den = fmaf(den, keep, w);
#pragma unroll
    for (int j = 0; j < V; ++j) o[j] = fmaf(o[j], keep, w * Elem<DT>::to_float(p.v_cache[row + j]));
    top = next;
  }
#pragma unroll
  for (int j = 0; j < V; ++j) {
    float y = den > 0.0f || den != den ? o[j] / den : 0.0f;
    if (p.gate) y = y / (1.0f + expf(-Elem<DT>::to_float(p.gate[t * p.gate_row + h * p.gate_head + lane * V + j])));
    p.out[((int64_t)t * p.n_qh + h) * D + lane * V + j] = Elem<DT>::from_float(y);
  }
}

template <int DT>
static cudaError_t launch_prefix_attention(const PrefixAttnParams& p, int head, cudaStream_t st) {
  const unsigned grid = (unsigned)ceil_div((int64_t)p.tokens * p.n_qh, 8);
  switch (head) {
    case 64: return launch_pdl(prefix_attention_kernel<DT, 2>, grid, 256, 0, st, p);
    case 128: return launch_pdl(prefix_attention_kernel<DT, 4>, grid, 256, 0, st, p);
    default: return launch_pdl(prefix_attention_kernel<DT, 8>, grid, 256, 0, st, p);
  }
}

}  // namespace yskn

using namespace yskn;

extern "C" YSKN_B200_API int64_t yskn_b200_prefix_attention_work_bytes(int tokens, int batch, int max_new, int n_qh,
                                                                      int n_kvh, int head) {
  if (tokens < 1 || batch < 1 || max_new < 1 || n_qh < 1 || n_kvh < 1 || n_qh % n_kvh ||
      (head != 64 && head != 128 && head != 256))
    return -1;
  return 256;
}

extern "C" YSKN_B200_API int yskn_b200_prefix_attention(
    const void* d_q, int64_t q_row, int64_t q_head, const void* d_gate, int64_t gate_row, int64_t gate_head,
    const void* d_k_cache, const void* d_v_cache, int64_t block_stride, int64_t token_stride, int64_t head_stride,
    int n_blocks, int block_size, const int32_t* d_prefix_blocks, int prefix_len, const int32_t* d_block_tables,
    int table_width, int64_t table_stride, const int32_t* d_lens, const int32_t* d_starts, int batch, int tokens,
    int max_new, int n_qh, int n_kvh, int head, int dtype, float scale, void* d_work, void* d_out, void* stream) {
  if (!d_q || !d_k_cache || !d_v_cache || !d_block_tables || !d_lens || !d_starts || !d_work || !d_out ||
      (prefix_len > 0 && !d_prefix_blocks))
    return fail(YSKN_EINVAL, "prefix_attention: null argument");
  if (head != 64 && head != 128 && head != 256)
    return fail(YSKN_EINVAL, "prefix_attention: heads of 64, 128 or 256 channels");
  if (!is_16bit(dtype)) return fail(YSKN_EINVAL, "prefix_attention: queries and cache are f16 or bf16");
  if (tokens < 1 || batch < 1 || max_new < 1 || n_kvh < 1 || n_qh < 1 || n_qh % n_kvh || n_qh / n_kvh > 128 ||
      prefix_len < 0 || table_width < 1 || (batch > 1 && table_stride < table_width) || n_blocks < 1)
    return fail(YSKN_EINVAL, "prefix_attention: empty shape, heads not a multiple, or a stride below its width");
  if (block_size != 16 && block_size != 32 && block_size != 64 && block_size != 128)
    return fail(YSKN_EINVAL, "prefix_attention: blocks of 16, 32, 64 or 128 rows");
  if (tokens == 1) q_row = gate_row = 0;  // strides that nothing steps over may be anything
  if (n_qh == 1) q_head = gate_head = 0;
  if (n_kvh == 1) head_stride = 0;
  if (n_blocks == 1) block_stride = 0;
  if (!aligned16(d_q) || !aligned16(d_gate) || !aligned16(d_k_cache) || !aligned16(d_v_cache) || !aligned16(d_work) ||
      !aligned16(d_out) || (q_row | q_head | block_stride | token_stride | head_stride) % 8 ||
      (d_gate && (gate_row | gate_head) % 8))
    return fail(YSKN_EINVAL, "prefix_attention: pointers and strides are multiples of 16 bytes");
  PrefixAttnParams p{};
  p.q = reinterpret_cast<const uint16_t*>(d_q), p.gate = reinterpret_cast<const uint16_t*>(d_gate);
  p.q_row = q_row, p.q_head = q_head, p.gate_row = gate_row, p.gate_head = gate_head;
  p.k_cache = reinterpret_cast<const uint16_t*>(d_k_cache), p.v_cache = reinterpret_cast<const uint16_t*>(d_v_cache);
  p.cache = {block_stride, token_stride, head_stride};
  p.n_blocks = n_blocks, p.block_size = block_size;
  p.prefix_blocks = d_prefix_blocks, p.prefix_len = prefix_len;
  p.tables = d_block_tables, p.table_stride = table_stride, p.table_width = table_width;
  p.lens = d_lens, p.starts = d_starts, p.batch = batch, p.tokens = tokens, p.max_new = max_new;
  p.n_qh = n_qh, p.n_kvh = n_kvh, p.scale = scale;
  p.out = reinterpret_cast<uint16_t*>(d_out), p.err = device_error_word();
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return cuda_fail(dtype == YSKN_DT_BF16 ? launch_prefix_attention<YSKN_DT_BF16>(p, head, st)
                                         : launch_prefix_attention<YSKN_DT_F16>(p, head, st),
                   "prefix_attention_kernel");
}
