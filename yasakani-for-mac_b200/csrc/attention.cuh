// Shared pieces of the attention kernels over the paged cache (prefixattn.cu, treeattn.cu): operand descriptors,
// packed and approximate arithmetic, the gate, tensor maps and the calls' refusals.
#pragma once
#include <string>

#include "paged.cuh"
#include "tcgen05.cuh"

namespace yskn {

constexpr int ATTENTION_MAX_GROUP = 128;  // query heads of a KV head, at most

// B operand whose N runs along the swizzled rows (V: rows are keys, MMA K), in columns of LINE
// bytes `stride` bytes apart, 8-key groups 8 LINE bytes apart. Swizzle span 128 or 64 bytes.
template <int LINE>
__device__ __forceinline__ uint64_t mn_desc(uint32_t saddr, uint32_t stride) {
  return (uint64_t)((saddr >> 4) & 0x3fff) | ((uint64_t)(stride >> 4) << 16) | ((uint64_t)(8 * LINE >> 4) << 32) |
         (1ull << 46) | ((LINE == 128 ? 2ull : 4ull) << 61);
}
// ---- pairs of SMs (clusters of two CTAs) that work on 256 rows with tcgen05.mma.cta_group::2
// kind::f16 with f32 accumulators, M = 256: type of both operands, N, B's major axis, A's sign.
__device__ __forceinline__ uint32_t pair_idesc(int dt, int n, uint32_t b_mn, uint32_t negate_a) {
  const uint32_t t = dt == YSKN_DT_BF16 ? 1u : 0u;
  return (1u << 4) | (t << 7) | (t << 10) | (negate_a << 13) | (b_mn << 16) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(256 >> 4) << 24);
}
// A and B by the low words of their descriptors (the high words are the same throughout), which
// leaves one 32-bit addition per operand and step to the issuing thread.
__device__ __forceinline__ void umma2_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t hi, uint32_t idesc,
                                         uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tsetp.ne.b32 p, %5, 0;\n\t"
      "mov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], a, b, %4, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(hi), "r"(idesc), "r"(accumulate));
}
__device__ __forceinline__ void umma2_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t hi, uint32_t idesc,
                                         uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b64 b, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], b, %4, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(hi), "r"(idesc), "r"(accumulate));
}
// Arrives on the barrier at this place in both CTAs once the MMAs issued so far are done.
__device__ __forceinline__ void umma2_commit(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"((uint16_t)3)
      : "memory");
}

// ---- the pair: addresses and barriers of its first CTA
__device__ __forceinline__ uint32_t first_cta(const void* p) {
  uint32_t a;
  asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(smem_u32(p)));
  return a;
}
// What these two announce is in TMEM or comes by TMA, so that they order no memory of their own
// (cluster-scope release and acquire here cost hundreds of clocks each: 16 prompt chunks 1439 us, now 986).
__device__ __forceinline__ void arrive_first(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void expect_first(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cluster.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// After stores to this CTA's shared memory that the first CTA's MMAs read.
__device__ __forceinline__ void release_first(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// TMA into this CTA's shared memory, counted on a barrier of the pair's first CTA.
__device__ __forceinline__ void pair_load_3d(void* dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, "
      "%5}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z)
      : "memory");
}
__device__ __forceinline__ void pair_load_5d(void* dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z,
                                             int w, int v) {
  asm volatile(
      "cp.async.bulk.tensor.5d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, "
      "%5, %6, %7}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z), "r"(w), "r"(v)
      : "memory");
}

// One lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
  return one != 0;
}
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
// Two binary32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 y;
  asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(y.x), "=f"(y.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return y;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 y;
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 d, a, b;\n\t"
      "mov.b64 {%0, %1}, d;\n\t}"
      : "=f"(y.x), "=f"(y.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return y;
}
// The gate's factor. (A row that sees nothing is zero whatever its gate holds.)
__device__ __forceinline__ float gated(float x, float gate) {
  return __fdividef(x, 1.0f + exp2_approx(-1.44269504f * gate));
}
// ------------------------------------------------------------------ host side
// 16-bit tensor of 3 to 5 axes with swizzled boxes of 64 channels (128-byte lines) or 32 (64). Strides in elements.
inline int paged_map(const char* name, CUtensorMap* map, const void* base, int dt, int rank, const int64_t* dims,
                     const int64_t* strides, const int* box) {
  EncodeTiled fn = encode_fn();
  if (!fn) return fail(YSKN_ECUDA, "cuTensorMapEncodeTiled is not available");
  cuuint64_t d[5], s[4];
  cuuint32_t b[5], one[5] = {1, 1, 1, 1, 1};
  for (int i = 0; i < rank; ++i) d[i] = (cuuint64_t)dims[i], b[i] = (cuuint32_t)box[i];
  for (int i = 0; i + 1 < rank; ++i) s[i] = (cuuint64_t)(dims[i + 1] == 1 ? dims[0] : strides[i]) * 2;
  const CUresult r = fn(map, dt == YSKN_DT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                        rank, const_cast<void*>(base), d, s, b, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        box[0] == 32 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(YSKN_EINVAL, std::string(name) + ": strides that a tensor map cannot hold");
  return YSKN_OK;
}

// What is wrong with a call's arguments, or nullptr; strides that nothing steps over are set to 0.
inline const char* attention_refusal(yskn_b200_prefix_attention_args& a) {
  if (!a.q || !a.k_cache || !a.v_cache || !a.block_tables || !a.lens || !a.starts || !a.work || !a.out ||
      (a.prefix_len > 0 && !a.prefix_blocks))
    return "null argument";
  const int head = a.head, n_qh = a.n_qh, n_kvh = a.n_kvh, block_size = a.block_size, dtype = a.dtype;
  if (head != 64 && head != 128 && head != 256)
    return "heads of 64, 128 or 256 channels";
  if (!is_16bit(dtype) || (a.gate && a.gate_dtype != dtype && a.gate_dtype != YSKN_DT_F32))
    return "queries and cache are f16 or bf16, the gate of their type or f32";
  if (a.tokens < 1 || a.batch < 1 || a.max_new < 1 || n_kvh < 1 || n_qh < 1 || n_qh % n_kvh ||
      n_qh / n_kvh > ATTENTION_MAX_GROUP || a.prefix_len < 0 || a.table_width < 1 ||
      (a.batch > 1 && a.table_stride < a.table_width) || a.n_blocks < 1)
    return "empty shape, heads not a multiple, or a stride below its width";
  if (block_size != 16 && block_size != 32 && block_size != 64 && block_size != 128)
    return "blocks of 16, 32, 64 or 128 rows";
  if (a.tokens == 1) a.q_row = a.gate_row = 0;  // strides that nothing steps over may be anything
  if (n_qh == 1) a.q_head = a.gate_head = 0;
  if (n_kvh == 1) a.head_stride = 0;
  if (a.n_blocks == 1) a.block_stride = 0;
  if (!aligned16(a.q) || !aligned16(a.gate) || !aligned16(a.k_cache) || !aligned16(a.v_cache) || !aligned16(a.work) ||
      !aligned16(a.out) || (a.q_row | a.q_head | a.block_stride | a.token_stride | a.head_stride) % 8 ||
      (a.gate && (a.gate_row | a.gate_head) % (a.gate_dtype == YSKN_DT_F32 ? 4 : 8)))
    return "pointers and strides are multiples of 16 bytes";
  return nullptr;
}

}  // namespace yskn
