"""The operators for drafted trees at the ends of what they take: rows past 2^31 elements, two streams at once, captured
calls replayed on other inputs. All of them give the same bits as the plain call, which the other tests hold against
64-bit formulas."""
import pytest

pytestmark = pytest.mark.gpu

D, HQ, HK, BS = 128, 8, 2, 64
FAR = 2 ** 30  # elements from block to block


class Batch:
    """Three requests of 9, 0 and 40 nodes with 100, 20 and 61 rows before them, behind nothing."""

    def __init__(self, cuda, seed, caches=None, new=(9, 0, 40), own=(100, 20, 61)):
        import torch
        import yskn_b200 as Y
        g = torch.Generator(device=cuda)
        g.manual_seed(seed)
        i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=cuda)  # noqa: E731
        T = sum(new)
        rnd = lambda *s: torch.randn(s, generator=g, device=cuda).bfloat16()  # noqa: E731
        self.caches = [torch.empty(6, BS, HK, D, dtype=torch.bfloat16, device=cuda) for _ in range(2)]
        for c in self.caches:
            c.copy_(rnd(*c.shape))
        if caches is not None:
            for far, c in zip(caches, self.caches):
                far.copy_(c)
            self.caches = caches
        self.q = rnd(T, HQ, D)
        self.tables, self.starts = i32([[5, 2], [3, 1], [0, 4]]), i32([0, new[0], new[0] + new[1], T])
        self.lens = i32([a + b for a, b in zip(new, own)])
        self.requests = i32([0] * new[0] + [1] * new[1] + [2] * new[2])
        self.parents = torch.cat([torch.arange(n, dtype=torch.int32, device=cuda).sub(1).div(2, rounding_mode="floor")
                                  for n in new if n]).int()
        self.mask, self.positions = torch.zeros(T, 2, dtype=torch.int32, device=cuda), i32([0] * T)
        self.work = torch.empty(Y.prefix_attention_work_bytes(T, 3, 40, HQ, HK, D), dtype=torch.uint8, device=cuda)
        self.out = torch.zeros_like(self.q)
        self.tokens, self.choice = (torch.randint(0, 2, (T,), generator=g, device=cuda).int() for _ in range(2))
        self.path = torch.zeros(3, 8, dtype=torch.int32, device=cuda)
        self.accepted, self.keep, self.next = i32([0] * 3), i32([0] * 3), i32([0] * 3)
        self.pool, self.free, self.lens2, self.free2 = i32([0] * 6), i32([0]), i32([0] * 3), i32([0])
        self.logits = torch.randn(T, 5000, generator=g, device=cuda)
        self.logprob, self.entropy = torch.zeros(T, 1, device=cuda), torch.zeros(T, device=cuda)
        self.top, self.ids = torch.zeros(T, 6, device=cuda), torch.zeros(T, 6, dtype=torch.int32, device=cuda)
        self.set = Y.CacheSet(self.caches)

    def run(self):
        import yskn_b200 as Y
        Y.tree_plan(self.parents, self.requests, self.starts, self.lens, self.mask, self.positions)
        Y.tree_attention(self.q, *self.caches, self.tables, self.lens, self.starts, 40, self.mask, self.work, self.out)
        Y.token_logprobs(self.logits, self.choice.unsqueeze(1), self.logprob, self.entropy, self.top, self.ids)
        Y.tree_accept(self.tokens, self.parents, self.choice, self.starts, self.lens, self.path, self.accepted,
                      self.keep, self.next)
        Y.cache_compact(self.set, self.tables, self.lens, self.starts, self.path)
        Y.batch_edit(self.lens, self.keep, self.tables, self.pool, self.free, BS, self.lens2, self.free2)

    def results(self):
        return [t.clone() for t in (self.mask, self.positions, self.out, self.logprob, self.entropy, self.top, self.ids,
                                    self.path, self.accepted, self.keep, self.next, self.lens2, self.free2, self.pool,
                                    *self.caches)]


def equal(a, b):
    import torch
    assert len(a) == len(b) and all(torch.equal(x, y) for x, y in zip(a, b)), [torch.equal(x, y) for x, y in zip(a, b)]


def test_blocks_past_2_31_elements(cuda):
    import torch
    import yskn_b200 as Y
    buffer = torch.empty(5 * FAR + 2 ** 20, dtype=torch.bfloat16, device=cuda)
    far = [torch.as_strided(buffer, (6, BS, HK, D), (FAR, HK * D, D, 1), at) for at in (0, 2 ** 16)]
    plain, at = Batch(cuda, 1), Batch(cuda, 1, far)
    plain.run(), at.run()
    assert Y.status() == 0 and int(plain.accepted.sum()) > 2
    equal(plain.results(), at.results())
    copies = torch.tensor([[5, 3], [1, 4], [64, 33]], dtype=torch.int32, device=cuda)
    Y.cache_copy(plain.set, copies)
    Y.cache_copy(at.set, copies)
    assert Y.status() == 0
    equal(plain.results(), at.results())


def test_logits_past_2_31_elements(cuda):
    import torch
    import yskn_b200 as Y
    buffer = torch.empty(2 * FAR + 2 ** 20, device=cuda)
    got = []
    for far in (False, True):
        b = Batch(cuda, 2)
        logits = b.logits[:3]
        if far:
            logits = torch.as_strided(buffer, (3, 5000), (FAR, 1))
            logits.copy_(b.logits[:3])
        Y.token_logprobs(logits, b.choice[:3].unsqueeze(1), b.logprob[:3], b.entropy[:3], b.top[:3], b.ids[:3])
        got.append(b.results())
    assert Y.status() == 0
    equal(*got)


def test_two_streams_at_once(cuda):
    import torch
    import yskn_b200 as Y
    alone = []
    for seed in range(4):
        b = Batch(cuda, seed)
        b.run()
        alone.append(b.results())
    for _ in range(5):
        batches, streams = [Batch(cuda, seed) for seed in range(4)], [torch.cuda.Stream(cuda) for _ in range(4)]
        torch.cuda.synchronize()
        for b, s in zip(batches, streams):
            with torch.cuda.stream(s):
                b.run()
        torch.cuda.synchronize()
        for b, r in zip(batches, alone):
            equal(b.results(), r)
    assert Y.status() == 0


def test_captured_calls_on_other_inputs(cuda):
    """Two graphs of two batches; then the first on a third one's inputs: other lengths, nodes and numbers."""
    import torch
    import yskn_b200 as Y
    inputs = ("q", "tables", "starts", "lens", "requests", "parents", "tokens", "choice", "logits", "pool", "free")
    batches, graphs = [Batch(cuda, seed) for seed in (5, 6)], []
    stream = torch.cuda.Stream(cuda)
    for b in batches:
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            b.run()
        graphs.append(g)
    other = Batch(cuda, 7, new=(17, 31, 1), own=(0, 97, 127))
    for k in inputs:
        getattr(batches[0], k).copy_(getattr(other, k))
    for a, b in zip(batches[0].caches, other.caches):
        a.copy_(b)
    second = Batch(cuda, 6)
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        for g in graphs:
            g.replay()
    torch.cuda.synchronize()
    other.run(), second.run()
    assert Y.status() == 0
    equal(batches[0].results(), other.results())
    equal(batches[1].results(), second.results())


def test_the_largest_tree_and_many_requests(cuda):
    import test_gpu_tree_attention as attention
    attention.run(cuda, new=(1024, 3), ctx=(33, 200), n_qh=4, n_kvh=2, D=64, seed=3)
    attention.run(cuda, new=[1] * 1500, ctx=[i % 5 for i in range(1500)], P=40, n_qh=2, n_kvh=1, D=64, seed=4)


def test_starts_that_do_not_ascend(cuda):
    """Reported, and all numbers finite. The request whose own starts are sound keeps its result, though with other
    parts to join: with u = 2^-8 and weights that sum to one, each of two results is off by at most u (weights) + u (its
    rounding) + u / 5 (sums of 109 rows, exponentials) of the largest |v|."""
    import torch
    import yskn_b200 as Y
    b = Batch(cuda, 8)
    Y.tree_plan(b.parents, b.requests, b.starts, b.lens, b.mask, b.positions)

    def attend():
        Y.tree_attention(b.q, *b.caches, b.tables, b.lens, b.starts, 40, b.mask, b.work, b.out)
        return Y.status()

    assert attend() == 0
    want, off = b.out.clone(), 2 * 2.2 * 2.0 ** -8 * float(b.caches[1].abs().max())
    for starts in ([0, 9, 5, 49], [-3, 9, 9, 49], [0, 9, 9, 50], [9, 0, 0, 2 ** 31 - 1]):
        b.starts.copy_(torch.tensor(starts, dtype=torch.int32))
        assert attend() == Y.EINVAL and bool(b.out.float().isfinite().all())
        if starts == [0, 9, 9, 50]:
            assert float((b.out[:9].float() - want[:9].float()).abs().max()) <= off and bool((b.out[9:] == 0).all())
