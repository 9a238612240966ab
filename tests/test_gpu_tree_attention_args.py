"""Attention of drafted trees (yskn_b200_tree_attention) over its arguments: scales of either sign and zero, masks and
largest requests wider than the trees, gates in f32 with strides and of any size, starts that overlap. Few rows are
joined by two groups of warps a CTA, many by one; both are taken.

Tolerance as in test_gpu_tree_attention.py, whose run() takes the scale into it. A gate's factor 1 / (1 + exp(-g)), one
approximate exponential, sum and quotient in binary32, is off by at most 2^-20 of itself."""
import pytest

import test_gpu_tree_attention as A

pytestmark = pytest.mark.gpu

FEW, MANY = dict(new=(20, 7, 1), n_qh=6, n_kvh=2), dict(new=(40, 33, 64), n_qh=24, n_kvh=2)


@pytest.mark.parametrize("scale", [-0.1, 0.0, 1.0, -1.0])
@pytest.mark.parametrize("size", [FEW, MANY])
@pytest.mark.parametrize("D,dtype", [(64, "bf16"), (128, "f16"), (256, "bf16")])
def test_scales(cuda, scale, size, D, dtype):
    """The new rows alone; and scores of theirs beside those of the rows before them, which the tensor cores take with
    -Q and |scale|."""
    A.run(cuda, ctx=(0, 0, 0), D=D, dtype=dtype, scale=scale, seed=D, **size)
    A.run(cuda, ctx=(300, 16, 5), D=D, dtype=dtype, scale=scale, seed=D, P=130, gate=True, **size)


@pytest.mark.parametrize("more", [1, 2, 31])
@pytest.mark.parametrize("size", [FEW, MANY])
def test_masks_wider_than_the_trees(cuda, more, size):
    A.run(cuda, ctx=(70, 0, 200), words=-(-max(size["new"]) // 32) + more, seed=more, **size)


@pytest.mark.parametrize("max_new", [20, 21, 41, 42, 43, 85, 86, 1000])
def test_largest_requests_that_are_not_there(cuda, max_new):
    """The bound of a request's tokens at, below and above what an item holds (42 tokens a CTA, 84 an item, where 3 query
    heads share a KV head), and above the call's tokens."""
    A.run(cuda, ctx=(70, 0, 200), max_new=max_new, seed=max_new, P=33, **FEW)
    if max_new >= 43:
        A.run(cuda, new=(43,), ctx=(600,), max_new=max_new, words=4, seed=max_new, n_qh=6, n_kvh=2)


class Case:
    """Three requests of 9, 2 and 40 nodes (stars: node 0 and itself) behind P shared rows and 70, 0 and 130 own."""

    def __init__(self, cuda, D, hq, hk, P, seed=0):
        import torch
        import yskn_b200 as Y
        g = torch.Generator(device=cuda)
        g.manual_seed(seed)
        i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=cuda)  # noqa: E731
        self.new, own, bs = (9, 2, 40), (70, 0, 130), 64
        T, pre = sum(self.new), -(-P // bs)
        rnd = lambda *s: torch.randn(s, generator=g, device=cuda).bfloat16()  # noqa: E731
        self.q, self.kc, self.vc = rnd(T, hq, D), rnd(pre + 9, bs, hk, D), rnd(pre + 9, bs, hk, D)
        self.tables, self.prefix = i32([[8, 0, 1], [2, 3, 4], [5, 6, 7]]), torch.arange(9, 9 + pre, device=cuda).int()
        self.P, self.lens = P, i32([P + a + b for a, b in zip(self.new, own)])
        self.starts = i32([0, 9, 11, T])
        self.mask = i32([[0, 0]] * T)
        t = 0
        for n in self.new:
            for j in range(n):
                for k in {0, j}:
                    self.mask[t, k // 32] |= (1 << k % 32) - (1 << 32 if k % 32 == 31 else 0)
                t += 1
        self.work = torch.empty(Y.prefix_attention_work_bytes(T, 3, 40, hq, hk, D), dtype=torch.uint8, device=cuda)
        flat = lambda c, b: c[b.long()].reshape(-1, hk, D)  # noqa: E731
        self.want, self.bound = [], []
        for i, n in enumerate(self.new):
            k, v = (torch.cat([flat(c, self.prefix)[:P], flat(c, self.tables[i])[:own[i] + n]]).double()
                    .repeat_interleave(hq // hk, 1) for c in (self.kc, self.vc))
            for j in range(n):
                at = list(range(P + own[i])) + sorted({P + own[i], P + own[i] + j})
                qd = self.q[sum(self.new[:i]) + j].double()
                s = torch.einsum("hd,lhd->hl", qd, k[at]) * D ** -0.5
                w = torch.softmax(s, -1)
                y, a = (torch.einsum("hl,lhd->hd", w, x) for x in (v[at], v[at].abs()))
                e = 2.0 ** -22 * D ** 0.5 * torch.einsum("hd,lhd->hl", qd.abs(), k[at].abs()).amax(-1)[:, None]
                self.want.append(y)
                self.bound.append((2.0 ** -8 + 2 * e + 2.0 ** -23 * len(at) + 2.0 ** -21) * a)
        self.want, self.bound = torch.stack(self.want), torch.stack(self.bound)

    def run(self, gate=None, **change):
        import torch
        import yskn_b200 as Y
        out = torch.full_like(self.q, 3.0)
        args = dict(dict(starts=self.starts, lens=self.lens, work=self.work), **change)
        Y.tree_attention(self.q, self.kc, self.vc, self.tables, max_new=40, mask=self.mask, out=out, gate=gate,
                         prefix_blocks=self.prefix, prefix_len=self.P, **args)
        torch.cuda.synchronize()
        return out


SHAPES = [(64, 4, 2, 0), (128, 6, 2, 100), (256, 24, 4, 200)]


@pytest.mark.parametrize("D,hq,hk,P", SHAPES)
def test_gates_in_f32_with_strides(cuda, D, hq, hk, P):
    """As the serving loop has them: the second half of each head's projection."""
    import torch
    import yskn_b200 as Y
    c = Case(cuda, D, hq, hk, P)
    gate = (torch.randn((len(c.q), hq, 2 * D), device=cuda) * 2)[:, :, D:]
    out = c.run(gate)
    sg = torch.sigmoid(gate.double())
    y = c.want * sg
    tol = c.bound * sg + 2.0 ** -20 * y.abs() + 2.0 ** -8 * y.abs() + 2.0 ** -25
    assert Y.status() == 0 and bool(((out.double() - y).abs() <= tol).all())


@pytest.mark.parametrize("D,hq,hk,P", SHAPES)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_gates_of_any_size(cuda, D, hq, hk, P, dtype):
    """Infinite and large gates: all of the output or none of it."""
    import torch
    import yskn_b200 as Y
    c = Case(cuda, D, hq, hk, P)
    gate = torch.zeros((len(c.q), hq, D), device=cuda)
    for i, x in enumerate((float("inf"), 3e38, 200.0, 89.0, -float("inf"), -3e38, -200.0, -89.0)):
        gate[:, :, i::8] = x
    out, bare = c.run(gate.to({"bf16": torch.bfloat16, "f32": torch.float32}[dtype])), c.run()
    assert Y.status() == 0
    assert bool(((bare.double() - c.want).abs() <= c.bound + 2.0 ** -8 * c.want.abs() + 2.0 ** -25).all())
    for i in range(8):
        if i < 4:
            assert torch.equal(out[:, :, i::8], bare[:, :, i::8])
        else:
            assert bool((out[:, :, i::8].abs() <= 2.0 ** -25).all())


@pytest.mark.parametrize("D,hq,hk,P", SHAPES)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_tokens_that_see_nothing_give_zeros_whatever_their_gate_holds(cuda, D, hq, hk, P, dtype):
    """Of requests without rows before their new ones, the nodes whose bits are all clear."""
    import torch
    import yskn_b200 as Y
    c = Case(cuda, D, hq, hk, 0)
    c.mask[9:11] = 0
    gate = torch.randn((len(c.q), hq, D), device=cuda).to({"bf16": torch.bfloat16, "f32": torch.float32}[dtype])
    gate[9] = float("nan")
    gate[10] = -float("inf")
    out = c.run(gate)
    assert Y.status() == 0 and bool((out[9:11] == 0).all()) and not bool(out.isnan().any())


@pytest.mark.parametrize("P", [0, 130])
def test_requests_that_overlap_stay_inside_the_workspace(cuda, P):
    """Starts that go back again name 12 items of 16 tokens a KV head, where six requests of 64 tokens in all have 10
    places: nothing is computed, every row is zero, and the status says so."""
    import torch
    import yskn_b200 as Y
    T, B, G, hk, D, bs = 64, 6, 16, 2, 64, 16
    g = torch.Generator(device=cuda)
    g.manual_seed(1)
    rnd = lambda *s: torch.randn(s, generator=g, device=cuda).bfloat16()  # noqa: E731
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=cuda)  # noqa: E731
    q, kc, vc = rnd(T, G * hk, D), rnd(60, bs, hk, D), rnd(60, bs, hk, D)
    n = Y.prefix_attention_work_bytes(T, B, T, G * hk, hk, D)
    buffer = torch.full((n + 4096,), 91, dtype=torch.uint8, device=cuda)
    out, mask = torch.full_like(q, 3.0), torch.full((T, 2), -1, dtype=torch.int32, device=cuda)
    tables, prefix = torch.arange(48, device=cuda).int().view(B, 8), torch.arange(48, 57, device=cuda).int()
    args = (q, kc, vc, tables, i32([P + 100] * B))

    def attend(starts):
        Y.tree_attention(*args, i32(starts), T, mask, buffer[:n], out, prefix_blocks=prefix, prefix_len=P)
        torch.cuda.synchronize()
        assert bool((buffer[n:] == 91).all())
        return Y.status()

    assert attend([0, 64, 0, 64, 0, 64, 0]) == Y.EINVAL and bool((out == 0).all())
    assert attend([0, 64, 64, 64, 64, 64, 64]) == 0 and bool(out.float().isfinite().all()) and bool((out != 0).any())
