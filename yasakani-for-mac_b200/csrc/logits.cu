// Penalties for repeated tokens, biases and a grammar mask on the head's logits, before the
// selection (head.cu).
//
// Per row, with c the token's count in the history after the prompt and seen its presence in
// the whole history, in binary32, each step rounded:
//   x = seen ? (x > 0 ? x / repetition : x * repetition) : x
//   x = x - frequency * c - (c > 0 ? presence : 0)
//   x = x + bias of the token's last entry in the row's list
//   x = the mask's bit of the token is set ? x : -inf
// A row whose mask allows nothing becomes -inf throughout, and the selection then answers
// that no token is eligible. Entries of the history and of the bias list outside the
// vocabulary (padding) count for nothing.
//
// What bounds it: bytes, 8 per logit (read, write) and the history. The counts are the only
// state, so a CTA takes one chunk of one row's vocabulary: it counts the history's tokens of
// its chunk in shared memory (integer atomics: the order cannot change a result), then
// streams the chunk once.
// A count word: bit 31 for a token of the prompt, the low bits the count after it, so that
// a token is seen if the word is not zero. The bias list comes last, on the written chunk:
// the word of each listed token is reused to find its last entry (an atomic maximum of
// entry numbers), which alone adds, so that lists with repeated tokens give one result.
#include <algorithm>

#include "common.cuh"

namespace yskn {

constexpr int LA_THREADS = 512;
constexpr int LA_MAX_CHUNK = 24576;  // count words: 96 KB of shared memory, two CTAs an SM
constexpr uint32_t LA_PROMPT = 0x80000000u;

struct LogitsParams {
  const float* logits;
  int64_t logits_stride;
  int rows, vocab;
  const int32_t* history;  // [rows][history_stride] or nullptr
  int64_t history_stride;
  int history_width;
  const int32_t* history_lens;
  const int32_t* prompt_lens;  // or nullptr: 0
  const float *repetition, *presence, *frequency;  // [rows] or nullptr
  const int32_t* bias_ids;  // [rows][n_bias] or nullptr
  const float* bias;
  int n_bias;
  const uint32_t* mask;  // [rows][mask_stride] or nullptr
  int64_t mask_stride;
  float* out;
  int64_t out_stride;
  int chunk;  // a multiple of 32
  unsigned* err;
};

__device__ __forceinline__ bool la_allowed(const uint32_t* mask, int i) {
  return !mask || ((__ldg(mask + (i >> 5)) >> (i & 31)) & 1u);
}

__device__ __forceinline__ float la_penalised(float x, uint32_t word, float rep, float pres, float freq) {
  if (word) {
    x = x > 0.0f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
    const uint32_t c = word & ~LA_PROMPT;
    if (c) x = __fsub_rn(__fsub_rn(x, __fmul_rn(freq, (float)c)), pres);
  }
  return x;
}

__global__ void __launch_bounds__(LA_THREADS) logits_adjust_kernel(const __grid_constant__ LogitsParams p) {
  extern __shared__ uint32_t s_count[];
  pdl_begin();
  const int tid = threadIdx.x, m = blockIdx.y;
  const int lo = blockIdx.x * p.chunk, n = min(p.chunk, p.vocab - lo);
  const bool counted = p.history != nullptr;
  float rep = 1.0f, pres = 0.0f, freq = 0.0f;
  if (counted) {
    if (p.repetition) rep = __ldg(p.repetition + m);
    if (p.presence) pres = __ldg(p.presence + m);
    if (p.frequency) freq = __ldg(p.frequency + m);
    for (int i = tid; i < n; i += LA_THREADS) s_count[i] = 0u;
    __syncthreads();
    int len = __ldg(p.history_lens + m);
    const int prompt = p.prompt_lens ? __ldg(p.prompt_lens + m) : 0;
    if (len > p.history_width) {
      len = p.history_width;
      if (tid == 0) raise_device_error(p.err, DERR_RANGE);
    }
    const int32_t* hist = p.history + m * p.history_stride;
    for (int j = tid; j < len; j += LA_THREADS) {
      const unsigned at = (unsigned)__ldg(hist + j) - (unsigned)lo;
      if (at < (unsigned)n) {
        if (j >= prompt) atomicAdd(s_count + at, 1u);
        else atomicOr(s_count + at, LA_PROMPT);
      }
    }
    __syncthreads();
  }
  const float* in = p.logits + m * p.logits_stride + lo;
  float* out = p.out + m * p.out_stride + lo;
  const uint32_t* mask = p.mask ? p.mask + m * p.mask_stride : nullptr;
  for (int i = tid; i < n; i += LA_THREADS) {
    float x = in[i];
    if (counted) x = la_penalised(x, s_count[i], rep, pres, freq);
    out[i] = la_allowed(mask, lo + i) ? x : -INFINITY;
  }
  if (p.n_bias) {
    __syncthreads();
    const int32_t* ids = p.bias_ids + (int64_t)m * p.n_bias;
    const float* bias = p.bias + (int64_t)m * p.n_bias;
    for (int j = tid; j < p.n_bias; j += LA_THREADS) {
      const unsigned at = (unsigned)__ldg(ids + j) - (unsigned)lo;
      if (at < (unsigned)n) s_count[at] = 0u;
    }
    __syncthreads();
    for (int j = tid; j < p.n_bias; j += LA_THREADS) {
      const unsigned at = (unsigned)__ldg(ids + j) - (unsigned)lo;
      if (at < (unsigned)n) atomicMax(s_count + at, (uint32_t)j + 1u);
    }
    __syncthreads();
    for (int j = tid; j < p.n_bias; j += LA_THREADS) {
      const unsigned at = (unsigned)__ldg(ids + j) - (unsigned)lo;
      if (at < (unsigned)n && s_count[at] == (uint32_t)j + 1u && la_allowed(mask, lo + (int)at))
        out[at] = __fadd_rn(out[at], __ldg(bias + j));
    }
  }
}

}  // namespace yskn

using namespace yskn;

extern "C" YSKN_B200_API int yskn_b200_logits_adjust(
    const float* d_logits, int64_t logits_stride, int rows, int vocab, const int32_t* d_history,
    int64_t history_stride, int history_width, const int32_t* d_history_lens, const int32_t* d_prompt_lens,
    const float* d_repetition, const float* d_presence, const float* d_frequency, const int32_t* d_bias_ids,
    const float* d_bias, int n_bias, const uint32_t* d_mask, int64_t mask_stride, float* d_out, int64_t out_stride,
    void* stream) {
  if (!d_logits || !d_out || rows < 1 || vocab < 1 || vocab > INT32_MAX - LA_MAX_CHUNK ||
      (rows > 1 && (logits_stride < vocab || out_stride < vocab)))
    return fail(YSKN_EINVAL, "logits_adjust: null logits or output, empty shape, or a stride below the vocabulary");
  if (rows > 65535) return fail(YSKN_EINVAL, "logits_adjust: more than 65535 rows");
  if (d_history && (!d_history_lens || history_width < 0 || (rows > 1 && history_stride < history_width)))
    return fail(YSKN_EINVAL, "logits_adjust: a history needs its lengths and a stride of its width");
  if (!d_history && (d_prompt_lens || d_repetition || d_presence || d_frequency))
    return fail(YSKN_EINVAL, "logits_adjust: penalties without a history");
  if (n_bias < 0 || (n_bias > 0 && (!d_bias_ids || !d_bias)))
    return fail(YSKN_EINVAL, "logits_adjust: a bias list needs its ids and values");
  if (d_mask && rows > 1 && mask_stride < ceil_div(vocab, 32))
    return fail(YSKN_EINVAL, "logits_adjust: mask rows shorter than the vocabulary");
  LogitsParams p{d_logits, logits_stride, rows, vocab, d_history, history_stride, history_width, d_history_lens,
                 d_prompt_lens, d_repetition, d_presence, d_frequency, d_bias_ids, d_bias, n_bias, d_mask, mask_stride,
                 d_out, out_stride, 0, device_error_word()};
  // Chunks for two waves of CTAs, at least 1024 logits each; every chunk reads the history.
  const int64_t want = ceil_div((int64_t)rows * vocab, 4 * 148);
  p.chunk = (int)std::min<int64_t>(LA_MAX_CHUNK, std::max<int64_t>(1024, ceil_div(want, 32) * 32));
  const size_t smem = d_history || n_bias ? (size_t)std::min(p.chunk, vocab) * sizeof(uint32_t) : 0;
  static SmemOptIn opt_in;
  if (cudaError_t e = opt_in(logits_adjust_kernel, LA_MAX_CHUNK * sizeof(uint32_t)))
    return cuda_fail(e, "logits_adjust_kernel attributes");
  return cuda_fail(launch_pdl(logits_adjust_kernel, dim3((unsigned)ceil_div(vocab, p.chunk), rows), LA_THREADS, smem,
                              reinterpret_cast<cudaStream_t>(stream), p),
                   "logits_adjust_kernel");
}
