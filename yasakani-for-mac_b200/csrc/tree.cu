// A step's trees of drafted tokens: what each node sees and where it stands, and, after the step, the
// path that the model's own choices take.
//
// tree_plan: for node j of a request, with parent(j) < j, the bits of j, parent(j), parent(parent(j)),
// ... and their number less one, its depth; its position is the request's length before the step
// plus the depth. tree_accept: path = 0, then in index order every node whose parent is the path's
// last one and whose token is the model's choice after that one.
//
// What bounds both: latency, a chain as long as the tree is deep (a few KB move). A warp takes a
// node (tree_plan) or a request (tree_accept). What the chain reads is loaded before it, 64 nodes in
// two registers a lane, and followed by shuffles; only parents past the 64th node are followed
// through the cache. A lane holds one word of the node's bits. Both calls, in a captured chain: a tree of 60 nodes
// 3.6 us, 256 of up to 64 nodes 6.0.
#include "common.cuh"

namespace yskn {

constexpr int TREE_WARPS = 8;

struct TreePlanParams {
  const int32_t *parents, *requests, *starts, *lens;
  uint32_t* mask;
  int64_t mask_stride;
  int32_t* positions;
  int tokens, batch, words;
  unsigned* err;
};

__global__ void __launch_bounds__(TREE_WARPS * 32) tree_plan_kernel(const __grid_constant__ TreePlanParams p) {
  pdl_begin();
  const int lane = threadIdx.x & 31, t = blockIdx.x * TREE_WARPS + (threadIdx.x >> 5);
  if (t >= p.tokens) return;
  const int r = __ldg(p.requests + t);
  uint32_t word = 0;
  int position = -1;
  bool wrong = r >= p.batch;
  if (r >= 0 && r < p.batch) {
    const int s0 = __ldg(p.starts + r), s1 = __ldg(p.starts + r + 1), len = __ldg(p.lens + r);
    const int j = t - s0;
    if (s0 >= 0 && s0 <= t && t < s1 && s1 <= p.tokens) {
      const int32_t* parents = p.parents + s0;
      const int low = lane <= j ? __ldg(parents + lane) : -1, high = lane + 32 <= j ? __ldg(parents + lane + 32) : -1;
      int depth = -1;
      for (int at = j; at >= 0;) {  // falls: ends after at most j rounds
        ++depth;
        if (at >> 5 == lane) word |= 1u << (at & 31);
        const int a = __shfl_sync(0xffffffffu, low, at & 31), b = __shfl_sync(0xffffffffu, high, at & 31);
        int up = at < 32 ? a : at < 64 ? b : __ldg(parents + at);
        if (up >= at) wrong = true, up = -1;
        at = up;
      }
      wrong = wrong || j >> 5 >= p.words;
      position = (int)min((long long)len - (s1 - s0) + depth, (long long)INT32_MAX);
    } else {
      wrong = true;
    }
  }
  if (lane < p.words) p.mask[t * p.mask_stride + lane] = word;
  if (lane == 0) {
    p.positions[t] = position;
    if (wrong) raise_device_error(p.err, DERR_RANGE);
  }
}

struct TreeAcceptParams {
  const int32_t *tokens, *parents, *choice, *starts, *lens;
  int32_t* path;
  int64_t path_stride;
  int32_t *accepted, *lens_out, *next;
  int batch, n_tokens, path_width;
  unsigned* err;
};

__global__ void __launch_bounds__(TREE_WARPS * 32) tree_accept_kernel(const __grid_constant__ TreeAcceptParams p) {
  pdl_begin();
  const int lane = threadIdx.x & 31, r = blockIdx.x * TREE_WARPS + (threadIdx.x >> 5);
  if (r >= p.batch) return;
  const int s0 = __ldg(p.starts + r), s1 = __ldg(p.starts + r + 1), len = p.lens[r];
  const bool sound = s0 >= 0 && s0 <= s1 && s1 <= p.n_tokens;
  const int n = sound ? s1 - s0 : 0;
  int32_t* path = p.path + r * p.path_stride;
  int last = 0, count = n > 0, next = -1;
  for (int j0 = 0; j0 < n; j0 += 32) {
    const int j = j0 + lane, at = s0 + min(j, n - 1);
    const int parent = __ldg(p.parents + at), token = __ldg(p.tokens + at), choice = __ldg(p.choice + at);
    if (j0 == 0) {
      next = __shfl_sync(0xffffffffu, choice, 0);
      if (lane == 0) path[0] = 0;
    }
    for (;;) {
      const unsigned who =
          __ballot_sync(0xffffffffu, j < n && j > last && parent == last && token == next && next >= 0);
      if (who == 0 || count >= p.path_width) break;
      const int first = __ffs(who) - 1;
      last = j0 + first;
      next = __shfl_sync(0xffffffffu, choice, first);
      if (lane == 0) path[count] = last;
      ++count;
    }
  }
  for (int k = count + lane; k < p.path_width; k += 32) path[k] = -1;
  if (lane == 0) {
    p.accepted[r] = count;
    p.lens_out[r] = max(len - (n - count), 0);
    p.next[r] = next;
    if (!sound) raise_device_error(p.err, DERR_RANGE);
  }
}

}  // namespace yskn

using namespace yskn;

extern "C" YSKN_B200_API int yskn_b200_tree_plan(const yskn_b200_tree_plan_args* args, void* stream) {
  if (!args) return fail(YSKN_EINVAL, "tree_plan: null argument");
  const yskn_b200_tree_plan_args& a = *args;
  if (!a.parents || !a.requests || !a.starts || !a.lens || !a.mask || !a.positions)
    return fail(YSKN_EINVAL, "tree_plan: null argument");
  if (a.tokens < 1 || a.tokens > 1 << 30 || a.batch < 1 || a.mask_words < 1 || a.mask_words > YSKN_TREE_MAX_WORDS ||
      (a.tokens > 1 && a.mask_stride < a.mask_words))
    return fail(YSKN_EINVAL, "tree_plan: empty shape, 1..32 mask words, or a stride below them");
  // Each warp reads its tree's parents and its request's lengths: not where others have written.
  const Span parents{a.parents, 4ll * a.tokens}, starts{a.starts, 4ll * a.batch + 4}, lens{a.lens, 4ll * a.batch};
  const Span positions{a.positions, 4ll * a.tokens};
  for (const Span& in : {parents, starts, lens})
    if (positions.meets(in) || rows_meet(a.mask, a.tokens, 4 * a.mask_stride, 4ll * a.mask_words, in))
      return fail(YSKN_EINVAL, "tree_plan: the masks and positions need arrays of their own");
  TreePlanParams p{a.parents, a.requests, a.starts,  a.lens,  a.mask,       a.mask_stride,
                   a.positions, a.tokens, a.batch, a.mask_words, device_error_word()};
  return cuda_fail(launch_pdl(tree_plan_kernel, (unsigned)ceil_div(a.tokens, TREE_WARPS), TREE_WARPS * 32, 0,
                              reinterpret_cast<cudaStream_t>(stream), p),
                   "tree_plan_kernel");
}

extern "C" YSKN_B200_API int yskn_b200_tree_accept(const yskn_b200_tree_accept_args* args, void* stream) {
  if (!args) return fail(YSKN_EINVAL, "tree_accept: null argument");
  const yskn_b200_tree_accept_args& a = *args;
  if (!a.tokens || !a.parents || !a.choice || !a.starts || !a.lens || !a.path || !a.accepted || !a.lens_out || !a.next)
    return fail(YSKN_EINVAL, "tree_accept: null argument");
  if (a.batch < 1 || a.batch > 1 << 30 || a.n_tokens < 1 || a.n_tokens > 1 << 30 || a.path_width < 1 ||
      (a.batch > 1 && a.path_stride < a.path_width))
    return fail(YSKN_EINVAL, "tree_accept: empty shape, or a stride below the path's width");
  // Other warps read these; its request's length a warp reads alone, so that a result may take that one's place.
  const int64_t row = 4ll * a.batch, nodes = 4ll * a.n_tokens;
  const Span in[] = {{a.tokens, nodes}, {a.parents, nodes}, {a.choice, nodes}, {a.starts, row + 4}, {a.lens, row}};
  bool meet = false;
  for (const Span& s : in) {
    for (const int32_t* out : {a.accepted, a.lens_out, a.next})
      meet = meet || (out != a.lens && Span{out, row}.meets(s));
    meet = meet || rows_meet(a.path, a.batch, 4 * a.path_stride, 4ll * a.path_width, s);
  }
  if (meet) return fail(YSKN_EINVAL, "tree_accept: paths, counts and lengths need arrays of their own");
  TreeAcceptParams p{a.tokens,   a.parents,  a.choice, a.starts, a.lens,     a.path,       a.path_stride,
                     a.accepted, a.lens_out, a.next,   a.batch,  a.n_tokens, a.path_width, device_error_word()};
  return cuda_fail(launch_pdl(tree_accept_kernel, (unsigned)ceil_div(a.batch, TREE_WARPS), TREE_WARPS * 32, 0,
                              reinterpret_cast<cudaStream_t>(stream), p),
                   "tree_accept_kernel");
}
