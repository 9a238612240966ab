"""Attention of drafted trees (yskn_b200_tree_attention) against the formula in 64 bits.

Tolerance, as for yskn_b200_prefix_attention: with w the softmax weights over what the token sees and A = sum w |v|, the
weights rounded to the cache's type (half a step u: bf16 2^-8, f16 2^-11; f16 weights below 2^-14 of the largest lose at
most 2^-24 each) give u A; scores are binary32 sums of D products, e = 2^-22 D scale sum |q k|, which moves the quotient
by 2 e A; sums over n rows 2^-23 n A; exponentials 2^-21 A; the result is rounded once, u |out|."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
HALF_STEP = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}


def tree(rng, n, kind="random"):
    """Parents of n nodes."""
    if kind == "chain":
        return list(range(-1, n - 1))
    if kind == "star":
        return [-1] + [0] * (n - 1)
    if kind == "apart":
        return [-1] * n
    return [-1] + [int(rng.integers(max(0, (j - 1) // 4), (j - 1) // 2 + 1)) for j in range(1, n)]


def bits_of(parents):
    seen = []
    for j, p in enumerate(parents):
        seen.append((seen[p] if p >= 0 else set()) | {j})
    return seen


def run(cuda, new=(5, 1), ctx=(40, 0), P=0, n_qh=6, n_kvh=2, D=128, dtype="bf16", block=16, gate=False, kind="random",
        sees=None, words=None, seed=0, max_new=None, pad=0, stream=None, fill=float("nan"), scale=None):
    """ctx: each request's own rows before its new ones; sees: per request a list of sets of new rows, else its
    tree's."""
    import torch
    import yskn_b200 as Y
    dt = {"bf16": torch.bfloat16, "f16": torch.float16}[dtype]
    g = torch.Generator(device=cuda)
    g.manual_seed(seed)
    rng = np.random.default_rng(seed)
    B, T = len(new), sum(new) + pad
    if sees is None:
        sees = [bits_of(tree(rng, n, kind)) if n else [] for n in new]
    pre, held = -(-P // block), [-(-(c + n) // block) for c, n in zip(ctx, new)]
    n_blocks = pre + sum(held) + 2
    caches = [torch.full((n_blocks, n_kvh, block, D), fill, dtype=dt, device=cuda).transpose(1, 2) for _ in range(2)]
    numbers = torch.randperm(n_blocks, generator=g, device=cuda).to(torch.int32)
    width = max(held + [1]) + 1
    tables = torch.full((B, width + 1), 2 ** 30, dtype=torch.int32, device=cuda)[:, :width]
    at = pre
    for i in range(B):
        tables[i, :held[i]] = numbers[at:at + held[i]]
        at += held[i]

    def put(cache, blocks, n):
        x = torch.randn((n, n_kvh, D), generator=g, device=cuda).to(dt)
        j = torch.arange(n, device=cuda)
        cache[blocks.long()[j // block], j % block] = x
        return x

    shared = [put(c, numbers[:pre], P) for c in caches]
    rows = [[torch.cat([s, put(c, tables[i], ctx[i] + new[i])]) for s, c in zip(shared, caches)] for i in range(B)]
    q = (torch.randn((T, n_qh, D), generator=g, device=cuda) * 1.5).to(dt)
    gt = (torch.randn((T, n_qh, D), generator=g, device=cuda) * 2).to(dt) if gate else None
    starts = np.concatenate([[0], np.cumsum(new)])
    words = max(1, -(-max(new) // 32)) if words is None else words
    mask = np.zeros((T, words + 1), np.uint32)  # a stride of its own; the word behind is all ones
    mask[:, words] = 0xffffffff
    for i in range(B):
        for t, s in enumerate(sees[i]):
            for j in s:
                mask[starts[i] + t, j // 32] |= np.uint32(1 << (j % 32))
    i32 = lambda a: torch.tensor(list(map(int, a)), dtype=torch.int32, device=cuda)  # noqa: E731
    d_mask = torch.from_numpy(mask.view(np.int32)).to(cuda)[:, :words]
    max_new = max(max(new), 1) if max_new is None else max_new
    work = torch.full((Y.prefix_attention_work_bytes(T, B, max_new, n_qh, n_kvh, D),), 255, dtype=torch.uint8,
                      device=cuda)
    out = torch.full((T, n_qh, D), 3.0, dtype=dt, device=cuda)
    lens, d_starts = i32([P + c + n for c, n in zip(ctx, new)]), i32(starts)
    torch.cuda.synchronize()
    Y.tree_attention(q, *caches, tables, lens, d_starts, max_new, d_mask, work, out,
                     prefix_blocks=numbers[:pre].clone(), prefix_len=P, gate=gt, scale=scale, stream=stream)
    torch.cuda.synchronize()
    assert Y.status() == 0
    G, sc, u = n_qh // n_kvh, D ** -0.5 if scale is None else scale, HALF_STEP[dtype]
    for i in range(B):
        before = P + ctx[i]
        for t in range(new[i]):
            tok = int(starts[i]) + t
            at = list(range(before)) + [before + j for j in sorted(sees[i][t]) if j <= t]
            if not at:
                assert bool((out[tok] == 0).all())
                continue
            k, v = (r[at].double().repeat_interleave(G, 1) for r in rows[i])
            qd = q[tok].double()
            s = torch.einsum("hd,lhd->hl", qd, k) * sc
            w = torch.softmax(s, -1)
            y, A = torch.einsum("hl,lhd->hd", w, v), torch.einsum("hl,lhd->hd", w, v.abs())
            e = 2.0 ** -22 * D * abs(sc) * torch.einsum("hd,lhd->hl", qd.abs(), k.abs()).amax(-1)[:, None]
            tol = (u + 2 * e + 2.0 ** -23 * len(at) + 2.0 ** -21) * A
            if dtype == "f16":
                tol = tol + 2.0 ** -24 * (v.abs().sum(0) / torch.exp(s - s.amax(-1, keepdim=True)).sum(-1)[:, None])
            if gate:
                sg = torch.sigmoid(gt[tok].double())
                y, tol = y * sg, tol * sg + 2.0 ** -20 * (y * sg).abs()
            tol = tol + u * y.abs() + 2.0 ** -25
            d = (out[tok].double() - y).abs()
            assert bool((d <= tol).all()), (i, t, float((d - tol).max()), float(d.max()))
    if pad:
        assert bool((out[T - pad:] == 0).all())
    return out


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("ctx", [0, 1, 15, 16, 63, 64, 100, 127, 128, 129, 700])
def test_where_the_new_rows_begin(cuda, ctx, D):
    run(cuda, new=(20, 7), ctx=(ctx, 30), D=D, seed=ctx + D)


@pytest.mark.parametrize("new", [1, 2, 8, 31, 32, 33, 63, 64, 65, 97, 128, 130, 200])
def test_tree_sizes(cuda, new):
    run(cuda, new=(new, 3), ctx=(70, 200), seed=new)


@pytest.mark.parametrize("kind", ["chain", "star", "apart"])
@pytest.mark.parametrize("P", [0, 1, 128, 517])
def test_shapes_of_trees_behind_a_prefix(cuda, kind, P):
    run(cuda, new=(40, 9, 1), ctx=(100, 0, 3), P=P, kind=kind, seed=P, gate=True)


@pytest.mark.parametrize("n_qh,n_kvh", [(1, 1), (2, 1), (4, 2), (8, 1), (16, 2), (24, 4), (128, 1)])
@pytest.mark.parametrize("new", [1, 2, 5])
def test_heads(cuda, n_qh, n_kvh, new):
    """Few rows a KV head take the thin items: at most 8."""
    run(cuda, new=(new, 1, new), ctx=(150, 9, 0), n_qh=n_qh, n_kvh=n_kvh, D=64, seed=n_qh + new)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("ctx", [0, 3, 14, 16, 30, 100])
def test_thin_items(cuda, D, ctx):
    run(cuda, new=(4, 2, 3), ctx=(ctx, 5, 0), n_qh=4, n_kvh=2, D=D, P=33, seed=ctx, kind="star", dtype="f16")
    run(cuda, new=(8, 8, 1), ctx=(ctx, 5, 0), n_qh=2, n_kvh=2, D=D, seed=ctx, kind="apart")


@pytest.mark.parametrize("block", [16, 32, 64, 128])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_blocks_and_types(cuda, block, dtype):
    run(cuda, new=(33, 12), ctx=(130, 61), P=40, block=block, dtype=dtype, seed=block, D=256)


def test_masks_that_are_no_trees(cuda):
    """Rows that see nothing, not themselves, or rows after themselves (which are cut off)."""
    rng = np.random.default_rng(5)
    sees = [[set() if t % 3 == 0 else {int(j) for j in np.flatnonzero(rng.random(50) < 0.3)} for t in range(50)],
            [set(), {0}, set()]]
    for ctx in ((0, 0), (77, 0), (128, 5)):
        run(cuda, new=(50, 3), ctx=ctx, sees=sees, seed=ctx[0])
        run(cuda, new=(3, 3), ctx=ctx, sees=[sees[0][:3], sees[1]], n_qh=2, n_kvh=2, seed=ctx[0])  # thin
    run(cuda, new=(6,), ctx=(0,), sees=[[set()] * 6])


def test_many_requests_and_long_contexts(cuda):
    run(cuda, new=(16,) * 40, ctx=tuple(7 * i for i in range(40)), P=300, D=64, seed=3)
    run(cuda, new=(60,), ctx=(9000,), n_qh=12, n_kvh=2, seed=4)
    run(cuda, new=(0, 5, 0), ctx=(4, 600, 0), seed=5, pad=3)


def test_a_chains_mask_is_the_plain_order(cuda):
    """Every earlier row's bit set: what prefix_attention gives, whose error is bounded like this one's: each half a step
    of the result and of the weights, and little else."""
    import torch
    import yskn_b200 as Y
    B, n, ctx, D, hq, hk, bs = 3, 21, 150, 128, 6, 2, 64
    g = torch.Generator(device=cuda)
    g.manual_seed(1)
    rnd = lambda *s: torch.randn(s, generator=g, device=cuda).bfloat16()  # noqa: E731
    q, kc, vc = rnd(B * n, hq, D), rnd(12, bs, hk, D), rnd(12, bs, hk, D)
    tables = torch.arange(9, dtype=torch.int32, device=cuda).view(3, 3)
    lens = torch.full((B,), ctx + n, dtype=torch.int32, device=cuda)
    starts = torch.arange(0, B * n + 1, n, dtype=torch.int32, device=cuda)
    work = torch.empty(Y.prefix_attention_work_bytes(B * n, B, n, hq, hk, D), dtype=torch.uint8, device=cuda)
    a, b = torch.empty_like(q), torch.empty_like(q)
    Y.prefix_attention(q, kc, vc, tables, lens, starts, n, work, a)
    Y.tree_attention(q, kc, vc, tables, lens, starts, n, torch.full((B * n, 1), -1, dtype=torch.int32, device=cuda),
                     work, b)
    torch.cuda.synchronize()
    most = vc.float().abs().max()  # a weighted mean of values: A is at most this
    assert bool(((a.float() - b.float()).abs() <= 2 * (2.0 ** -8 * (a.float().abs() + most) + 2.0 ** -10 * most)).all())


@pytest.mark.parametrize("hq,hk,n,ctx", [(6, 2, 20, 50), (2, 2, 4, 50), (24, 4, 40, 0), (8, 1, 33, 200)])
def test_hidden_rows_may_hold_anything(cuda, hq, hk, n, ctx):
    """Keys and values of infinities and NaN in new rows that a token does not see change no bit of its result."""
    import torch
    import yskn_b200 as Y
    D, bs = 64, 16
    g = torch.Generator(device=cuda)
    g.manual_seed(n)
    rnd = lambda *s: torch.randn(s, generator=g, device=cuda).bfloat16()  # noqa: E731
    blocks = -(-(ctx + n) // bs)
    q, kc, vc = rnd(n, hq, D), rnd(blocks, bs, hk, D), rnd(blocks, bs, hk, D)
    tables = torch.arange(blocks, dtype=torch.int32, device=cuda).view(1, blocks)
    lens = torch.tensor([ctx + n], dtype=torch.int32, device=cuda)
    starts = torch.tensor([0, n], dtype=torch.int32, device=cuda)
    mask = torch.zeros((n, 2), dtype=torch.int64, device=cuda)  # a star, all of whose nodes see node 0 and themselves
    for t in range(n):
        mask[t, 0] |= 1
        mask[t, t // 32] |= 1 << t % 32
    mask = torch.where(mask >= 2 ** 31, mask - 2 ** 32, mask).to(torch.int32)
    work = torch.empty(Y.prefix_attention_work_bytes(n, 1, n, hq, hk, D), dtype=torch.uint8, device=cuda)
    outs, hidden = [], [n - 2, 1]
    for bad in (None, float("nan"), float("inf"), -float("inf")):
        k2, v2 = kc.clone(), vc.clone()
        if bad is not None:
            for j in hidden:
                row = ctx + j
                k2[row // bs, row % bs] = bad
                v2[row // bs, row % bs] = bad
        out = torch.empty_like(q)
        Y.tree_attention(q, k2, v2, tables, lens, starts, n, mask, work, out)
        torch.cuda.synchronize()
        outs.append(out)
    others = [t for t in range(n) if t not in hidden]
    assert all(torch.equal(outs[0][others], o[others]) for o in outs[1:])
    assert all(bool(o[hidden].isnan().any()) for o in outs[1:3])  # those that see it, see it
    assert Y.status() == 0


def test_what_the_device_refuses(cuda):
    """More new tokens than mask bits, and new rows inside the prefix: reported, no result."""
    import torch
    import yskn_b200 as Y
    D, hq, hk, bs = 64, 4, 2, 16
    rnd = lambda *s: torch.randn(s, device=cuda).bfloat16()  # noqa: E731
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=cuda)  # noqa: E731
    for new, lens, P in (((40, 2), (50, 20), 0), ((4, 2), (18, 30), 16)):
        T = sum(new)
        q, kc, vc = rnd(T, hq, D), rnd(12, bs, hk, D), rnd(12, bs, hk, D)
        out = torch.full_like(q, 3.0)
        work = torch.empty(Y.prefix_attention_work_bytes(T, 2, max(new), hq, hk, D), dtype=torch.uint8, device=cuda)
        Y.tree_attention(q, kc, vc, i32([[0, 1, 2, 3], [4, 5, 6, 7]]), i32(lens), i32([0, new[0], T]), max(new),
                         torch.full((T, 1), -1, dtype=torch.int32, device=cuda), work, out,
                         prefix_blocks=i32([8]), prefix_len=P)
        assert Y.status() == Y.EINVAL
        assert bool((out[:new[0]] == 0).all()) and bool(out[new[0]:].float().isfinite().all())


def test_another_stream(cuda):
    import torch
    run(cuda, new=(20, 7), ctx=(130, 30), seed=9, stream=torch.cuda.Stream(cuda))
