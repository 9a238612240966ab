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
// A token's count: the top bit for a token of the prompt, the others the count after it, so that
// a token is seen if it is not zero. Histories shorter than 32768 are counted in 16 bits (two
// counts a word), longer ones in 32: half the shared memory is twice the CTAs an SM, and one
// CTA's counting then overlaps another's streaming. The bias list comes last, on the written
// chunk: the count words of the listed tokens are reused to find each token's last entry (an
// atomic maximum of entry numbers), which alone adds, so that lists with repeated tokens give
// one result.
// The chunk is streamed in 16-byte accesses. A row may start at any 4-byte boundary (an odd
// vocabulary): input and output are then equally far from one, the chunk begins with up to
// three single logits, and the counts are shifted with it. Where the two are unequally far,
// each access is one logit.
#include <algorithm>

#include "common.cuh"

namespace yskn {

constexpr int LA_THREADS = 256;
constexpr int LA_MAX_CHUNK = 24576;  // counts of 2 bytes: 48 KB of shared memory, four CTAs an SM
constexpr int LA_NARROW = 32768;     // histories below this are counted in 16 bits

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

__device__ __forceinline__ float la_penalised(float x, bool seen, uint32_t c, float rep, float pres, float freq) {
  if (seen) {
    x = x > 0.0f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
    if (c) x = __fsub_rn(__fsub_rn(x, __fmul_rn(freq, (float)c)), pres);
  }
  return x;
}

template <typename Count>
__global__ void __launch_bounds__(LA_THREADS) logits_adjust_kernel(const __grid_constant__ LogitsParams p) {
  constexpr int PER_WORD = 4 / sizeof(Count);
  constexpr uint32_t PROMPT = 1u << (8 * sizeof(Count) - 1), ALL = PROMPT | (PROMPT - 1);
  extern __shared__ __align__(16) uint32_t s_count[];
  pdl_begin();
  const int tid = threadIdx.x, m = blockIdx.y;
  const int lo = blockIdx.x * p.chunk, n = min(p.chunk, p.vocab - lo);
  const float* in = p.logits + m * p.logits_stride + lo;
  float* out = p.out + m * p.out_stride + lo;
  // single logits before the first 16-byte boundary; counts are kept from place `shift` on, so
  // that they meet the boundary too
  const int shift = (int)((reinterpret_cast<uintptr_t>(in) >> 2) & 3), head = min(n, (4 - shift) & 3);
  const bool wide = ((reinterpret_cast<uintptr_t>(out) >> 2) & 3) == (unsigned)shift;
  const bool counted = p.history != nullptr;
  auto place = [&](unsigned at) { return (at + shift) / PER_WORD; };
  auto bits = [&](unsigned at) { return ((at + shift) % PER_WORD) * 8 * (unsigned)sizeof(Count); };
  float rep = 1.0f, pres = 0.0f, freq = 0.0f;
  if (counted) {
    if (p.repetition) rep = __ldg(p.repetition + m);
    if (p.presence) pres = __ldg(p.presence + m);
    if (p.frequency) freq = __ldg(p.frequency + m);
    int len = __ldg(p.history_lens + m);
    const int prompt = p.prompt_lens ? __ldg(p.prompt_lens + m) : 0;
    for (int i = tid; i < (n + 3 + 4 * PER_WORD - 1) / (4 * PER_WORD); i += LA_THREADS)
      reinterpret_cast<uint4*>(s_count)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    if (len > p.history_width) {
      len = p.history_width;
      if (tid == 0) raise_device_error(p.err, DERR_RANGE);
    }
    const int32_t* hist = p.history + m * p.history_stride;
    constexpr int BATCH = 8;
    for (int j0 = tid; j0 < len; j0 += BATCH * LA_THREADS) {
      int id[BATCH];
#pragma unroll
      for (int u = 0; u < BATCH; ++u) {
        const int j = j0 + u * LA_THREADS;
        id[u] = j < len ? __ldg(hist + j) : -1;
      }
#pragma unroll
      for (int u = 0; u < BATCH; ++u) {
        const unsigned at = (unsigned)id[u] - (unsigned)lo;
        if (id[u] >= 0 && at < (unsigned)n) {
          if (j0 + u * LA_THREADS >= prompt) atomicAdd(s_count + place(at), 1u << bits(at));
          else atomicOr(s_count + place(at), PROMPT << bits(at));
        }
      }
    }
    __syncthreads();
  }
  const uint32_t* mask = p.mask ? p.mask + m * p.mask_stride : nullptr;
  auto allowed = [&](int i) { return !mask || ((__ldg(mask + (i >> 5)) >> (i & 31)) & 1u); };
  auto adjusted = [&](float x, uint32_t count) {
    return la_penalised(x, count != 0, count & (PROMPT - 1), rep, pres, freq);
  };
  auto single = [&](int i) {
    float x = in[i];
    if (counted) x = adjusted(x, (s_count[place(i)] >> bits(i)) & ALL);
    out[i] = allowed(lo + i) ? x : -INFINITY;
  };
  if (wide) {
    if (tid < head) single(tid);
    const int quads = (n - head) / 4;
    constexpr int BATCH = 4;
    for (int q0 = tid; q0 < quads; q0 += BATCH * LA_THREADS) {
      float4 x[BATCH];
      uint32_t ok[BATCH];
#pragma unroll
      for (int u = 0; u < BATCH; ++u) {
        const int q = q0 + u * LA_THREADS, i = head + 4 * q;
        if (q >= quads) break;
        x[u] = *reinterpret_cast<const float4*>(in + i);
        ok[u] = 15u;
        if (mask) {  // four bits, from two words where they straddle
          const int at = lo + i, w = at >> 5, s = at & 31;
          const uint32_t a = __ldg(mask + w), b = s > 28 ? __ldg(mask + w + 1) : 0u;
          ok[u] = __funnelshift_r(a, b, s);
        }
      }
#pragma unroll
      for (int u = 0; u < BATCH; ++u) {
        const int q = q0 + u * LA_THREADS, i = head + 4 * q;
        if (q >= quads) break;
        float v[4] = {x[u].x, x[u].y, x[u].z, x[u].w};
        if (counted) {
          uint32_t w[4 / PER_WORD];
          if constexpr (PER_WORD == 2) {
            const uint2 c = *reinterpret_cast<const uint2*>(s_count + place(i));
            w[0] = c.x, w[1] = c.y;
          } else {
            const uint4 c = *reinterpret_cast<const uint4*>(s_count + place(i));
            w[0] = c.x, w[1] = c.y, w[2] = c.z, w[3] = c.w;
          }
          uint32_t any = 0;
#pragma unroll
          for (int k = 0; k < 4 / PER_WORD; ++k) any |= w[k];
          if (any) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              v[k] = adjusted(v[k], (w[k / PER_WORD] >> (k % PER_WORD * 8 * sizeof(Count))) & ALL);
          }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (!((ok[u] >> k) & 1u)) v[k] = -INFINITY;
        *reinterpret_cast<float4*>(out + i) = make_float4(v[0], v[1], v[2], v[3]);
      }
    }
    for (int i = head + 4 * quads + tid; i < n; i += LA_THREADS) single(i);
  } else {
    for (int i = tid; i < n; i += LA_THREADS) single(i);
  }
  if (p.n_bias) {
    // a word for each listed token: here tokens whose counts share a word share an entry number,
    // so the last entry is sought among the tokens of a word's first place, then of its second
    __syncthreads();
    const int32_t* ids = p.bias_ids + (int64_t)m * p.n_bias;
    const float* bias = p.bias + (int64_t)m * p.n_bias;
    for (int turn = 0; turn < PER_WORD; ++turn) {
      auto mine = [&](int j, unsigned& at) {
        at = (unsigned)__ldg(ids + j) - (unsigned)lo;
        return at < (unsigned)n && (at + shift) % PER_WORD == (unsigned)turn;
      };
      unsigned at;
      for (int j = tid; j < p.n_bias; j += LA_THREADS)
        if (mine(j, at)) s_count[place(at)] = 0u;
      __syncthreads();
      for (int j = tid; j < p.n_bias; j += LA_THREADS)
        if (mine(j, at)) atomicMax(s_count + place(at), (uint32_t)j + 1u);
      __syncthreads();
      for (int j = tid; j < p.n_bias; j += LA_THREADS)
        if (mine(j, at) && s_count[place(at)] == (uint32_t)j + 1u && allowed(lo + (int)at))
          out[at] = __fadd_rn(out[at], __ldg(bias + j));
      __syncthreads();
    }
  }
}

}  // namespace yskn

using namespace yskn;

extern "C" YSKN_B200_API int yskn_b200_logits_adjust(const yskn_b200_logits_adjust_args* args, void* stream) {
  if (!args) return fail(YSKN_EINVAL, "logits_adjust: null argument");
  const yskn_b200_logits_adjust_args& a = *args;
  if (!a.logits || !a.out || a.rows < 1 || a.vocab < 1 || a.vocab > INT32_MAX - LA_MAX_CHUNK ||
      (a.rows > 1 && (a.logits_stride < a.vocab || a.out_stride < a.vocab)))
    return fail(YSKN_EINVAL, "logits_adjust: null logits or output, empty shape, or a stride below the vocabulary");
  if (a.rows > 65535) return fail(YSKN_EINVAL, "logits_adjust: more than 65535 rows");
  if (a.history && (!a.history_lens || a.history_width < 0 || (a.rows > 1 && a.history_stride < a.history_width)))
    return fail(YSKN_EINVAL, "logits_adjust: a history needs its lengths and a stride of its width");
  if (!a.history && (a.prompt_lens || a.repetition || a.presence || a.frequency))
    return fail(YSKN_EINVAL, "logits_adjust: penalties without a history");
  if (a.n_bias < 0 || (a.n_bias > 0 && (!a.bias_ids || !a.bias)))
    return fail(YSKN_EINVAL, "logits_adjust: a bias list needs its ids and values");
  if (a.mask && a.rows > 1 && a.mask_stride < ceil_div(a.vocab, 32))
    return fail(YSKN_EINVAL, "logits_adjust: mask rows shorter than the vocabulary");
  LogitsParams p{a.logits, a.logits_stride, a.rows, a.vocab, a.history, a.history_stride, a.history_width,
                 a.history_lens, a.prompt_lens, a.repetition, a.presence, a.frequency, a.bias_ids, a.bias, a.n_bias,
                 a.mask, a.mask_stride, a.out, a.out_stride, 0, device_error_word()};
  // Chunks for four CTAs an SM, of at least 1024 logits; every chunk reads the history.
  const bool narrow = a.history_width < LA_NARROW;
  const int64_t want = ceil_div((int64_t)a.rows * a.vocab, 4 * 148);
  p.chunk = (int)std::min<int64_t>(LA_MAX_CHUNK, std::max<int64_t>(1024, ceil_div(want, 32) * 32));
  const size_t count = narrow ? 2 : 4;
  const size_t smem = a.history || a.n_bias ? ((size_t)std::min(p.chunk, a.vocab) + 8) / 8 * 8 * count + 16 : 0;
  auto run = [&](auto kernel, SmemOptIn& opt_in) {
    if (cudaError_t e = opt_in(kernel, (int)((LA_MAX_CHUNK + 8) * count + 16)))
      return cuda_fail(e, "logits_adjust_kernel attributes");
    return cuda_fail(launch_pdl(kernel, dim3((unsigned)ceil_div(a.vocab, p.chunk), a.rows), LA_THREADS, smem,
                                reinterpret_cast<cudaStream_t>(stream), p),
                     "logits_adjust_kernel");
  };
  static SmemOptIn opt_narrow, opt_wide;
  return narrow ? run(logits_adjust_kernel<uint16_t>, opt_narrow) : run(logits_adjust_kernel<uint32_t>, opt_wide);
}
