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
// What bounds it: bytes, 8 per logit (read, write) and the history. A piece of work is one chunk
// of one row's vocabulary: the history's tokens of the chunk are counted in shared memory (integer
// atomics: the order cannot change a result), then the chunk is streamed once. A persistent
// CTA per SM has two count buffers: 16 warps count the next chunk's history, and add the biases of
// the one before, while 16 warps stream the present one, so that the memory does not wait for
// the counting. (Of 256 rows of 151936 with up to 16384 tokens of history: one logit a thread
// 255 us; 16-byte accesses, counting and streaming in turn in four CTAs an SM 114; this way
// 82. Streaming a plain copy and adjusting the history's logits afterwards took 141: two
// million scattered 4-byte updates.) Some of nearly every 128 neighbouring tokens are in a
// long history, so the penalties run for nearly every warp: no division among them (Penalties).
// A token's count: the top bit for a token of the prompt, the others the count after it, so that
// a token is seen if it is not zero. Histories shorter than 32768 are counted in 16 bits (two
// counts a word), longer ones in 32: a chunk may be as large as its counts allow, because every
// chunk of a row reads the row's history. The bias list comes last, on the written chunk: the
// count words of the listed tokens are reused to find each token's last entry (an atomic maximum
// of entry numbers), which alone adds, so that lists with repeated tokens give one result.
// The chunk is streamed in 16-byte accesses. A row may start at any 4-byte boundary (an odd
// vocabulary): input and output are then equally far from one, the chunk begins with up to
// three single logits, and the counts are shifted with it. Where the two are unequally far,
// each access is one logit.
#include <algorithm>

#include "common.cuh"

namespace yskn {

constexpr int LA_STREAMERS = 512, LA_COUNTERS = 512, LA_THREADS = LA_STREAMERS + LA_COUNTERS;
constexpr int LA_BUFFER = 98304;  // bytes of counts of a chunk, at most (two buffers)
constexpr int LA_NARROW = 32768;  // histories below this are counted in 16 bits
constexpr int LA_MIN_CHUNK = 1024;

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
  int chunk, chunks;  // logits of a chunk (a multiple of 32), chunks of a row
  int buffer;         // bytes of a count buffer
  unsigned* err;
};

// Named barriers, by a chunk's parity: its counts are there (LA_FULL + b), it has been streamed
// (LA_DONE + b); the counting warps alone.
enum { LA_FULL = 1, LA_DONE = 3, LA_COUNT = 5 };
__device__ __forceinline__ void bar_sync(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
__device__ __forceinline__ void bar_arrive(int id, int threads) {
  asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

struct LogitsItem {
  int m, lo, n;  // row, first logit, logits
  const float* in;
  float* out;
  const uint32_t* mask;
  int shift;  // logits of `in` past a 16-byte boundary: the counts start at this place
  __device__ LogitsItem(const LogitsParams& p, int item)
      : m(item / p.chunks), lo((item - m * p.chunks) * p.chunk), n(min(p.chunk, p.vocab - lo)),
        in(p.logits + m * p.logits_stride + lo), out(p.out + m * p.out_stride + lo),
        mask(p.mask ? p.mask + m * p.mask_stride : nullptr),
        shift((int)((reinterpret_cast<uintptr_t>(in) >> 2) & 3)) {}
  __device__ bool allowed(int at) const {
    return !mask || ((__ldg(mask + ((lo + at) >> 5)) >> ((lo + at) & 31)) & 1u);
  }
};

template <typename Count>
struct LogitsCount {
  static constexpr int PER_WORD = 4 / sizeof(Count), BITS = 8 * sizeof(Count);
  static constexpr uint32_t PROMPT = 1u << (BITS - 1), ALL = PROMPT | (PROMPT - 1);
};

// The quotient by the repetition penalty is the binary64 product with its binary64 reciprocal, rounded:
// off by 2^-52 of itself before that, and a quotient of two 24-bit numbers that is normal in binary32
// lies 2^-49 of itself or more from where binary32's rounding turns, so this is the division's result;
// infinities, overflow and penalties of any size included. A subnormal quotient half way between two
// numbers may fall on the other one. (256 rows of 151936: 82 us; the division where binary32's
// product and one Newton step do not hold, as a rare branch, 98.)
struct Penalties {
  float rep, pres, freq;
  double inv;
  __device__ void repeated(float r) {
    rep = r;
    inv = 1.0 / (double)r;
  }
  __device__ float operator()(float x, uint32_t count, uint32_t prompt) const {
    float y = x > 0.0f ? (float)((double)x * inv) : __fmul_rn(x, rep);
    const float c = (float)(count & (prompt - 1));
    y = c > 0.0f ? __fsub_rn(__fsub_rn(y, __fmul_rn(freq, c)), pres) : y;
    return count ? y : x;
  }
};

// Streams a chunk: ready() is called once, when the first logits are on their way.
template <typename Count, typename Ready>
__device__ __forceinline__ void la_stream(const LogitsItem& it, const uint32_t* counts, const Penalties& pen, bool counted,
                                          Ready ready) {
  using L = LogitsCount<Count>;
  constexpr int W = 4 / L::PER_WORD;  // words of a quad's counts
  const int st = threadIdx.x, n = it.n, head = min(n, (4 - it.shift) & 3);
  auto single = [&](int i) {
    float x = it.in[i];
    if (counted) {
      const int at = i + it.shift;
      x = pen(x, (counts[at / L::PER_WORD] >> (at % L::PER_WORD * L::BITS)) & L::ALL, L::PROMPT);
    }
    it.out[i] = it.allowed(i) ? x : -INFINITY;
  };
  if (((reinterpret_cast<uintptr_t>(it.out) >> 2) & 3) != (unsigned)it.shift) {
    ready();
    for (int i = st; i < n; i += LA_STREAMERS) single(i);
    return;
  }
  const int quads = (n - head) / 4, first = it.lo + head;
  const float4* in = reinterpret_cast<const float4*>(it.in + head);
  float4* out = reinterpret_cast<float4*>(it.out + head);
  const uint32_t* qcounts = counts + (head + it.shift) / L::PER_WORD;
  const bool straddles = (first & 3) != 0;  // a quad's four mask bits may lie in two words
  constexpr int BATCH = 4;
  bool waiting = true;
  for (int q0 = st; q0 - st < quads; q0 += BATCH * LA_STREAMERS) {
    float4 x[BATCH];
    uint32_t ok[BATCH];
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
      const int q = q0 + u * LA_STREAMERS;
      if (q < quads) x[u] = in[q];
    }
    if (it.mask) {
#pragma unroll
      for (int u = 0; u < BATCH; ++u) {
        const int at = first + 4 * min(q0 + u * LA_STREAMERS, quads - 1), w = at >> 5, s = at & 31;
        const uint32_t a = __ldg(it.mask + w);
        ok[u] = __funnelshift_r(a, straddles && s > 28 ? __ldg(it.mask + w + 1) : 0u, s);
      }
    }
    if (waiting) {
      waiting = false;
      ready();
    }
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
      const int q = q0 + u * LA_STREAMERS;
      if (q >= quads) break;
      float v[4] = {x[u].x, x[u].y, x[u].z, x[u].w};
      if (counted) {
        uint32_t w[W], any = 0;
#pragma unroll
        for (int z = 0; z < W; z += 2) {
          const uint2 c = *reinterpret_cast<const uint2*>(qcounts + q * W + z);
          w[z] = c.x, w[z + 1] = c.y;
          any |= c.x | c.y;
        }
        if (any) {
#pragma unroll
          for (int z = 0; z < 4; ++z)
            v[z] = pen(v[z], (w[z / L::PER_WORD] >> (z % L::PER_WORD * L::BITS)) & L::ALL, L::PROMPT);
        }
      }
      if (it.mask) {
#pragma unroll
        for (int z = 0; z < 4; ++z)
          if (!((ok[u] >> z) & 1u)) v[z] = -INFINITY;
      }
      out[q] = make_float4(v[0], v[1], v[2], v[3]);
    }
  }
  if (waiting) ready();
  if (st < head) single(st);
  for (int i = head + 4 * quads + st; i < n; i += LA_STREAMERS) single(i);
}

template <typename Count>
__global__ void __launch_bounds__(LA_THREADS) logits_adjust_kernel(const __grid_constant__ LogitsParams p) {
  using L = LogitsCount<Count>;
  extern __shared__ __align__(16) uint8_t s_buffers[];
  pdl_begin();
  const int items = p.rows * p.chunks, step = gridDim.x;
  const bool counted = p.history != nullptr, paired = counted || p.n_bias;
  auto counts_of = [&](int k) { return reinterpret_cast<uint32_t*>(s_buffers + (k & 1) * p.buffer); };

  if (threadIdx.x < LA_STREAMERS) {
    int k = 0;
    for (int item = blockIdx.x; item < items; item += step, ++k) {
      const LogitsItem it(p, item);
      Penalties pen{1.0f, 0.0f, 0.0f, 1.0};
      if (p.repetition) pen.repeated(__ldg(p.repetition + it.m));
      if (p.presence) pen.pres = __ldg(p.presence + it.m);
      if (p.frequency) pen.freq = __ldg(p.frequency + it.m);
      la_stream<Count>(it, counts_of(k), pen, counted, [&]() {
        if (paired) bar_sync(LA_FULL + (k & 1), LA_THREADS);
      });
      if (paired) {
        __threadfence_block();
        bar_arrive(LA_DONE + (k & 1), LA_THREADS);
      }
    }
    return;
  }
  if (!paired) return;

  const int ct = threadIdx.x - LA_STREAMERS;
  const int mine = (items - (int)blockIdx.x + step - 1) / step;  // this CTA's chunks
  for (int k = 0; k < mine + 2; ++k) {
    uint32_t* counts = counts_of(k);
    if (k >= 2) {  // the chunk two before has been streamed: its biases, then its buffer is free
      bar_sync(LA_DONE + (k & 1), LA_THREADS);
      if (p.n_bias) {
        // Where two counts share a word, their tokens share an entry number: the last entry is sought
        // among the tokens of the words' first places, then of their second.
        const LogitsItem it(p, (int)blockIdx.x + (k - 2) * step);
        const int32_t* ids = p.bias_ids + (int64_t)it.m * p.n_bias;
        const float* bias = p.bias + (int64_t)it.m * p.n_bias;
        for (int turn = 0; turn < L::PER_WORD; ++turn) {
          auto word_of = [&](int j, int& at) -> uint32_t* {
            const int id = __ldg(ids + j);
            if (id < it.lo || id - it.lo >= it.n) return nullptr;
            at = id - it.lo;
            const int c = at + it.shift;
            return c % L::PER_WORD == turn ? counts + c / L::PER_WORD : nullptr;
          };
          int at;
          for (int j = ct; j < p.n_bias; j += LA_COUNTERS)
            if (uint32_t* w = word_of(j, at)) *w = 0u;
          bar_sync(LA_COUNT, LA_COUNTERS);
          for (int j = ct; j < p.n_bias; j += LA_COUNTERS)
            if (uint32_t* w = word_of(j, at)) atomicMax(w, (uint32_t)j + 1u);
          bar_sync(LA_COUNT, LA_COUNTERS);
          for (int j = ct; j < p.n_bias; j += LA_COUNTERS) {
            uint32_t* w = word_of(j, at);
            if (w && *w == (uint32_t)j + 1u && it.allowed(at)) it.out[at] = __fadd_rn(it.out[at], __ldg(bias + j));
          }
          bar_sync(LA_COUNT, LA_COUNTERS);
        }
      }
    }
    if (k >= mine) continue;
    const LogitsItem it(p, (int)blockIdx.x + k * step);
    if (counted) {
      int len = __ldg(p.history_lens + it.m);
      const int prompt = p.prompt_lens ? __ldg(p.prompt_lens + it.m) : 0;
      for (int i = ct; i < p.buffer / 16; i += LA_COUNTERS) reinterpret_cast<uint4*>(counts)[i] = make_uint4(0, 0, 0, 0);
      bar_sync(LA_COUNT, LA_COUNTERS);
      if (len > p.history_width) {
        len = p.history_width;
        if (ct == 0) raise_device_error(p.err, DERR_RANGE);
      }
      const int32_t* hist = p.history + it.m * p.history_stride;
      constexpr int BATCH = 8;
      for (int j0 = ct; j0 < len; j0 += BATCH * LA_COUNTERS) {
        int id[BATCH];
#pragma unroll
        for (int u = 0; u < BATCH; ++u) {
          const int j = j0 + u * LA_COUNTERS;
          id[u] = j < len ? __ldg(hist + j) : -1;
        }
#pragma unroll
        for (int u = 0; u < BATCH; ++u) {
          if (id[u] < it.lo || id[u] - it.lo >= it.n) continue;
          const int at = id[u] - it.lo + it.shift;
          uint32_t* w = counts + at / L::PER_WORD;
          const int bit = at % L::PER_WORD * L::BITS;
          if (j0 + u * LA_COUNTERS >= prompt) atomicAdd(w, 1u << bit);
          else atomicOr(w, L::PROMPT << bit);
        }
      }
      __threadfence_block();
    }
    bar_arrive(LA_FULL + (k & 1), LA_THREADS);
  }
}

}  // namespace yskn

using namespace yskn;

extern "C" YSKN_B200_API int yskn_b200_logits_adjust(const yskn_b200_logits_adjust_args* args, void* stream) {
  if (!args) return fail(YSKN_EINVAL, "logits_adjust: null argument");
  const yskn_b200_logits_adjust_args& a = *args;
  if (!a.logits || !a.out || a.rows < 1 || a.vocab < 1 || a.vocab > INT32_MAX - LA_BUFFER ||
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
                 a.mask, a.mask_stride, a.out, a.out_stride, 0, 0, 0, device_error_word()};
  // The fewest chunks a row that the counts allow read the history the fewest times, but the last
  // round of chunks over the SMs should be full too: of the counts of chunks that fill one to six
  // rounds, and the fewest, the one with the least time (a chunk's logits, a fixed part and a
  // share of the history's width, over the rounds).
  const bool narrow = a.history_width < LA_NARROW;
  const int count = narrow ? 2 : 4, most = LA_BUFFER / count - 32, sms = 148;
  const int fewest = (int)ceil_div(a.vocab, most), limit = std::max(fewest, a.vocab / LA_MIN_CHUNK);
  int64_t best = INT64_MAX;
  for (int rounds = 0; rounds <= 6; ++rounds) {
    const int n = std::min(limit, std::max(fewest, (int)((int64_t)rounds * sms / a.rows)));
    const int chunk = ((a.vocab + n - 1) / n + 31) / 32 * 32, chunks = (a.vocab + chunk - 1) / chunk;
    const int64_t time = ((int64_t)a.rows * chunks + sms - 1) / sms * (chunk + 512 + a.history_width / 16);
    if (time < best) best = time, p.chunk = chunk;
  }
  p.chunks = (int)ceil_div(a.vocab, p.chunk);
  p.buffer = (int)ceil_div((int64_t)(p.chunk + 3) * count, 16) * 16;
  if ((int64_t)a.rows * p.chunks > INT32_MAX / 2) return fail(YSKN_EINVAL, "logits_adjust: too many logits");
  const size_t smem = a.history || a.n_bias ? 2 * (size_t)p.buffer : 0;
  const unsigned grid = (unsigned)std::min<int64_t>((int64_t)a.rows * p.chunks, sms);
  auto run = [&](auto kernel, SmemOptIn& opt_in) {
    if (cudaError_t e = opt_in(kernel, 2 * LA_BUFFER)) return cuda_fail(e, "logits_adjust_kernel attributes");
    return cuda_fail(launch_pdl(kernel, grid, LA_THREADS, smem, reinterpret_cast<cudaStream_t>(stream), p),
                     "logits_adjust_kernel");
  };
  static SmemOptIn opt_narrow, opt_wide;
  return narrow ? run(logits_adjust_kernel<uint16_t>, opt_narrow) : run(logits_adjust_kernel<uint32_t>, opt_wide);
}
