"""Attention of a batch over a shared prefix (yskn_b200_prefix_attention) against the formula in
64 bits.

Tolerance. With w the softmax weights and A = sum w |v|: the weights are rounded to p bits
(bf16 8, f16 11) before they meet the values, at most 2^-p A in the sum (f16 weights below
2^-14 of the largest lose at most 2^-24 each: 2^-24 sum |v|); scores are binary32 sums of D products, off by at most
e = 2^-22 D scale sum |q k| (a unit for each addition, twice for truncating adders), which moves
the quotient by at most 2 e A; the sums over n rows by 2^-23 n' A with n' the longest chain of
additions (n at most); exponentials by 2^-21. The result is rounded once: 2^-p |out|."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
P_BITS = {"bf16": 8, "f16": 11}


def run(cuda, new=(1, 1), own=(5, 40), P=100, n_qh=6, n_kvh=2, D=128, dtype="bf16", block=16, gate=False,
        paired=False, head_major=True, pad_tokens=0, lens=None, seed=0, stream=None, scale=None, spread=1.0,
        fill=float("nan"), max_new=None, check=True, gate_f32=False):
    """own: each request's own rows with its new ones; lens overrides P + own."""
    import torch
    import yskn_b200 as Y
    dt = {"bf16": torch.bfloat16, "f16": torch.float16}[dtype]
    g = torch.Generator(device=cuda)
    g.manual_seed(seed)
    B, T = len(new), sum(new) + pad_tokens
    lens = [P + o for o in own] if lens is None else lens
    pre = -(-P // block)
    held = [-(-max(n - P, 0) // block) for n in lens]
    n_blocks = pre + sum(held) + 2
    shape = (n_blocks, n_kvh, block, D) if head_major else (n_blocks, block, n_kvh, D)
    # rows that no request owns hold `fill`
    caches = [torch.full(shape, fill, dtype=dt, device=cuda) for _ in range(2)]
    kc, vc = (c.transpose(1, 2) if head_major else c for c in caches)
    numbers = torch.randperm(n_blocks, generator=g, device=cuda).to(torch.int32)
    width = max(held + [1]) + 2
    tables = torch.full((B, width + 1), 2 ** 30, dtype=torch.int32, device=cuda)[:, :width]  # unused: not a block
    at = pre
    rows = {}
    for i in range(B):
        tables[i, :held[i]] = numbers[at:at + held[i]]
        at += held[i]
    prefix_blocks = numbers[:pre].clone()

    def put(cache, blocks, n):
        x = (torch.randn((n, n_kvh, D), generator=g, device=cuda) * spread).to(dt)
        j = torch.arange(n, device=cuda)
        cache[blocks.long()[j // block], j % block] = x
        return x

    pk, pv = put(kc, prefix_blocks, P), put(vc, prefix_blocks, P)
    for i in range(B):
        n = max(lens[i] - P, 0)
        rows[i] = [torch.cat([a, put(c, tables[i], n)]) for a, c in ((pk, kc), (pv, vc))]
    q = (torch.randn((T, n_qh, D * (2 if paired else 1)), generator=g, device=cuda) * 1.5).to(dt)[:, :, :D]
    gt = (torch.randn((T, n_qh, 2 * D), generator=g, device=cuda) * 2).to(torch.float32 if gate_f32 else dt)[:, :, D:] if gate else None
    starts = np.concatenate([[0], np.cumsum(new)])
    i32 = lambda a: torch.tensor(list(map(int, a)), dtype=torch.int32, device=cuda)  # noqa: E731
    max_new = max(max(new), 1) if max_new is None else max_new
    work = torch.full((Y.prefix_attention_work_bytes(T, B, max_new, n_qh, n_kvh, D),), 255, dtype=torch.uint8,
                      device=cuda)
    out = torch.full((T, n_qh, D), 3.0, dtype=dt, device=cuda)
    d_lens, d_starts = i32(lens), i32(starts)
    torch.cuda.synchronize()
    Y.prefix_attention(q, kc, vc, tables, d_lens, d_starts, max_new, work, out, prefix_blocks=prefix_blocks,
                       prefix_len=P, gate=gt, scale=scale, stream=stream)
    torch.cuda.synchronize()
    if not check:
        return out
    assert Y.status() == 0
    G, sc, u = n_qh // n_kvh, D ** -0.5 if scale is None else scale, 2.0 ** -P_BITS[dtype]
    for i in range(B):
        for t in range(new[i]):
            lim = max(0, lens[i] - new[i] + t + 1)
            tok = int(starts[i]) + t
            if lim == 0:
                assert bool((out[tok] == 0).all())
                continue
            k, v = (r[:lim].double().repeat_interleave(G, 1) for r in rows[i])  # [lim][n_qh][D]
            qd = q[tok].double()
            s = torch.einsum("hd,lhd->hl", qd, k) * sc
            w = torch.softmax(s, -1)
            y, A = torch.einsum("hl,lhd->hd", w, v), torch.einsum("hl,lhd->hd", w, v.abs())
            e = 2.0 ** -22 * D * abs(sc) * torch.einsum("hd,lhd->hl", qd.abs(), k.abs()).amax(-1)[:, None]
            tol = (u + 2 * e + 2.0 ** -23 * lim + 2.0 ** -21) * A
            if dtype == "f16":
                # weights relative to the row's largest; a stale maximum scales them up, never down
                tol = tol + 2.0 ** -24 * (v.abs().sum(0) / torch.exp(s - s.amax(-1, keepdim=True)).sum(-1)[:, None])
            if gate:
                sg = torch.sigmoid(gt[tok].double())
                y, tol = y * sg, tol * sg + 2.0 ** -20 * (y * sg).abs()
            tol = tol + u * y.abs() + 2.0 ** -25
            d = (out[tok].double() - y).abs()
            assert bool((d <= tol).all()), (i, t, float((d - tol).max()), float(d.max()))
    if pad_tokens:
        assert bool((out[T - pad_tokens:] == 0).all())
    return out


@pytest.mark.parametrize("P", [0, 1, 15, 16, 127, 128, 129, 1000, 5000])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_prefix_lengths(cuda, P, D):
    run(cuda, P=P, D=D, new=(1, 1, 1), own=(1, 17, 300), seed=P + D)


@pytest.mark.parametrize("own", [1, 2, 16, 63, 64, 65, 127, 128, 129, 600])
def test_own_lengths(cuda, own):
    run(cuda, own=(own, 3), P=64, seed=own)


@pytest.mark.parametrize("block", [16, 32, 64, 128])
@pytest.mark.parametrize("head_major", [True, False])
def test_block_sizes_and_orders(cuda, block, head_major):
    run(cuda, P=333, new=(2, 1, 5), own=(200, 64, 131), block=block, head_major=head_major, D=256, seed=block)


@pytest.mark.parametrize("n_qh,n_kvh", [(1, 1), (4, 4), (24, 4), (5, 1), (16, 2), (128, 1), (14, 2), (60, 3)])
def test_head_groups(cuda, n_qh, n_kvh):
    run(cuda, n_qh=n_qh, n_kvh=n_kvh, new=(1, 3, 1), own=(9, 140, 1), P=200, seed=n_qh)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("gate,paired", [(True, False), (False, True), (True, True)])
@pytest.mark.parametrize("D", [64, 256])
def test_types_gates_and_strides(cuda, dtype, gate, paired, D):
    run(cuda, dtype=dtype, gate=gate, paired=paired, D=D, new=(1, 4), own=(50, 200), P=150, seed=3)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("new,own,P", [((1, 4), (50, 200), 150), ((1, 1), (9, 60), 0), ((130,), (130,), 300)])
def test_gates_in_f32(cuda, dtype, new, own, P):
    run(cuda, dtype=dtype, gate=True, gate_f32=True, D=256, new=new, own=own, P=P, seed=14)


@pytest.mark.parametrize("new,own", [((130, 1, 47), (300, 1, 47)), ((300,), (300,)), ((33, 64, 2), (500, 64, 128)),
                                     ((8,) * 19, tuple(range(8, 160, 8)))])
@pytest.mark.parametrize("D", [128, 256])
def test_prompt_chunks_are_causal(cuda, new, own, D):
    run(cuda, new=new, own=own, P=70, D=D, seed=len(new))


def test_batches_larger_than_a_tile(cuda):
    run(cuda, new=(1,) * 70, own=tuple(1 + 5 * i % 211 for i in range(70)), n_qh=24, n_kvh=4, D=256, P=700, gate=True,
        seed=1)
    run(cuda, new=(1,) * 300, own=tuple(1 + i % 7 for i in range(300)), n_qh=4, n_kvh=1, D=64, P=40, seed=2)


def test_requests_that_see_nothing_or_little(cuda):
    """Empty, idle and short requests: a length of zero, below the prefix, below their tokens."""
    run(cuda, new=(1, 0, 1, 3, 2, 0, 2), lens=[0, 0, 30, 2, 101, 120, 1], P=100, seed=4)
    run(cuda, new=(2, 3), lens=[0, 0], P=0, seed=5)
    run(cuda, new=(0, 4, 0, 0, 1, 0), lens=[0, 104, 0, 500, 260, 0], P=100, pad_tokens=5, seed=6)


@pytest.mark.parametrize("n_qh,n_kvh,D", [(24, 4, 256), (6, 2, 128), (3, 3, 64)])
def test_few_items_of_few_tiles(cuda, n_qh, n_kvh, D):
    """Items that one pair of SMs finishes from end to end, empty and idle requests among them."""
    kw = dict(n_qh=n_qh, n_kvh=n_kvh, D=D, block=16, gate=True)
    run(cuda, new=(1, 0, 2, 1), lens=[30, 0, 2, 0], P=0, pad_tokens=3, seed=15, **kw)
    run(cuda, new=(1, 1), own=(1, 90), P=100, pad_tokens=1, seed=16, **kw)
    run(cuda, new=(1, 3, 1), lens=[0, 50, 101], P=100, seed=17, **kw)
    run(cuda, new=(90, 1), own=(90, 120), P=0, seed=18, **kw)


@pytest.mark.parametrize("G,n", [(1, 8), (2, 4), (3, 2), (4, 2), (8, 1), (5, 2), (9, 1)])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_few_rows_a_head(cuda, G, n, D):
    """Up to 8 rows a KV head (and just over), own rows from one slice to many, each count of tokens."""
    kw = dict(n_qh=2 * G, n_kvh=2, D=D, gate=True)
    run(cuda, new=(n, 1, max(1, n - 1), n, n), own=(n, 700, n + 15, 2100, n + 16), P=130, seed=21, **kw)
    run(cuda, new=(n, 1, n), own=(n + 40, 1, 555), P=0, dtype="f16", block=64, head_major=False, seed=22, **kw)


def test_many_short_requests(cuda):
    """More requests than threads of a CTA, and than warps of all of them."""
    run(cuda, new=(1,) * 500, own=tuple(1 + i % 40 for i in range(500)), n_qh=8, n_kvh=2, D=64, P=20, seed=23)
    run(cuda, new=(1,) * 1000, own=tuple(1 + i % 5 for i in range(1000)), n_qh=6, n_kvh=3, D=64, P=0, seed=24)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_items_cut_in_many_places(cuda, D):
    """Long own rows of few requests, idle and empty ones and padding among them; without a prefix, and
    with one that each request's items take themselves."""
    kw = dict(n_qh=10, n_kvh=2, D=D, gate=True, block=128)
    run(cuda, new=(3, 0, 2, 4, 0), lens=[5000, 0, 2, 3000, 7], P=0, pad_tokens=40, seed=25, **kw)
    run(cuda, new=(60, 0, 2, 55), lens=[2000, 0, 0, 900], P=0, pad_tokens=3, seed=26, **kw)
    run(cuda, new=(130, 0, 70), lens=[900, 300, 230], P=160, pad_tokens=3, seed=27, **kw)


def test_padded_tokens_give_zeros(cuda):
    run(cuda, new=(1, 1), own=(5, 40), pad_tokens=200, seed=7)
    run(cuda, new=(0, 0), own=(5, 40), pad_tokens=3, seed=8)


@pytest.mark.parametrize("fill", [float("inf"), float("-inf"), 3e38, 0.0])
def test_rows_outside_hold_anything(cuda, fill):
    """NaN (the other tests' fill), infinities and huge values in every row that no token sees."""
    import torch
    a = run(cuda, P=77, own=(9, 150), fill=fill, D=256, seed=9)
    assert torch.equal(a, run(cuda, P=77, own=(9, 150), D=256, seed=9))


def test_rising_and_large_scores(cuda):
    run(cuda, P=900, own=(300, 7), spread=6.0, scale=1.0 / 16, D=256, seed=10)
    run(cuda, P=900, own=(300, 7), spread=6.0, scale=1.0 / 16, D=256, dtype="f16", seed=10)
    run(cuda, P=300, own=(30, 7), scale=-0.1, seed=11)
    run(cuda, P=300, own=(30, 7), scale=0.0, seed=12)


def test_same_result_twice_and_on_another_stream(cuda):
    import torch
    kw = dict(new=(1, 9, 1), own=(400, 129, 1), P=2000, D=256, n_qh=24, n_kvh=4, gate=True, seed=13)
    a = run(cuda, **kw)
    assert torch.equal(a, run(cuda, **kw)) and torch.equal(a, run(cuda, stream=torch.cuda.Stream(), **kw))


def test_long_cache(cuda):
    """Blocks past 2^31 elements into the cache."""
    import torch
    import yskn_b200 as Y
    D, block, n_blocks = 256, 128, 70000  # 70000 * 128 * 256 > 2^31 elements
    kc = torch.zeros((n_blocks, block, 1, D), dtype=torch.bfloat16, device=cuda)
    vc = torch.zeros((n_blocks, block, 1, D), dtype=torch.bfloat16, device=cuda)
    kc[-1].normal_()
    vc[-1].normal_()
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device=cuda)  # noqa: E731
    q = torch.randn((1, 2, D), device=cuda).to(torch.bfloat16)
    out = torch.empty_like(q)
    work = torch.empty(Y.prefix_attention_work_bytes(1, 1, 1, 2, 1, D), dtype=torch.uint8, device=cuda)
    Y.prefix_attention(q, kc, vc, i32(n_blocks - 1)[None], i32(100), i32(0, 1), 1, work, out)
    w = torch.softmax(torch.einsum("hd,ld->hl", q[0].double(), kc[-1, :100, 0].double()) / 16, -1)
    y, A = w @ vc[-1, :100, 0].double(), w @ vc[-1, :100, 0].double().abs()
    assert Y.status() == 0
    assert bool(((out[0].double() - y).abs() <= 2.0 ** -8 * y.abs() + (2.0 ** -8 + 1e-2) * A).all())


def test_blocks_outside_the_cache_are_reported(cuda):
    import torch
    import yskn_b200 as Y
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device=cuda)  # noqa: E731
    c = torch.ones((4, 16, 1, 64), dtype=torch.bfloat16, device=cuda)
    q = torch.ones((1, 1, 64), dtype=torch.bfloat16, device=cuda)
    work = torch.empty(Y.prefix_attention_work_bytes(1, 1, 1, 1, 1, 64), dtype=torch.uint8, device=cuda)
    for bad in (4, -1, 2 ** 30):
        Y.prefix_attention(q, c, c, i32(0, bad)[None], i32(20), i32(0, 1), 1, work, torch.empty_like(q))
        assert Y.status() == Y.EINVAL
    Y.prefix_attention(q, c, c, i32(0, 9)[None], i32(16), i32(0, 1), 1, work, torch.empty_like(q))
    assert Y.status() == 0  # an entry past the length is not looked at


def test_more_tokens_than_promised_are_reported(cuda):
    import yskn_b200 as Y
    run(cuda, new=(3, 200), own=(20, 200), max_new=1, check=False)
    assert Y.status() == Y.EINVAL
    run(cuda, new=(3, 2), own=(20, 20), seed=1)


def call(cuda, new, lens, P, fill, n_qh=6, n_kvh=2, D=128, block=16, gate=None, seed=0):
    """A bf16 call without a wrapper around it: q, the rows of each request ([len][n_kvh][D] K and V), out and
    the starts. Cache rows that no token sees hold `fill`, those of the prefix too."""
    import torch
    import yskn_b200 as Y
    g = torch.Generator(device=cuda)
    g.manual_seed(seed)
    B, T, pre = len(new), sum(new), -(-P // block)
    seen = [n if k else 0 for n, k in zip(lens, new)]
    held = [-(-max(n - P, 0) // block) for n in lens]
    n_blocks = pre + sum(held) + 1
    kc, vc = (torch.full((n_blocks, block, n_kvh, D), fill, dtype=torch.bfloat16, device=cuda) for _ in range(2))
    numbers = torch.randperm(n_blocks, generator=g, device=cuda).to(torch.int32)
    tables = torch.full((B, max(held + [1])), -1, dtype=torch.int32, device=cuda)

    def put(cache, blocks, n):
        x = torch.randn((n, n_kvh, D), generator=g, device=cuda).to(torch.bfloat16)
        j = torch.arange(n, device=cuda)
        cache[blocks.long()[j // block], j % block] = x
        return x

    prefix, at, rows = [put(c, numbers, min(P, max(seen + [0]))) for c in (kc, vc)], pre, []
    for i in range(B):
        tables[i, :held[i]] = numbers[at:at + held[i]]
        at += held[i]
        rows.append([torch.cat([a, put(c, tables[i], max(seen[i] - P, 0))]) for a, c in zip(prefix, (kc, vc))])
    q = (torch.randn((T, n_qh, D), generator=g, device=cuda) * 1.5).to(torch.bfloat16)
    starts = np.concatenate([[0], np.cumsum(new)]).tolist()
    i32 = lambda a: torch.tensor(list(map(int, a)), dtype=torch.int32, device=cuda)  # noqa: E731
    work = torch.full((Y.prefix_attention_work_bytes(T, B, max(new), n_qh, n_kvh, D),), 255, dtype=torch.uint8,
                      device=cuda)
    out = torch.full((T, n_qh, D), 3.0, dtype=torch.bfloat16, device=cuda)
    Y.prefix_attention(q, kc, vc, tables, i32(lens), i32(starts), max(new), work, out, prefix_blocks=numbers[:pre],
                       prefix_len=P, gate=gate)
    return q, rows, out, starts


def near(q, rows, out, starts, new, lens):
    """The bound at the top of the file, for bf16 without a gate."""
    import torch
    n_qh, D, u = q.shape[1], q.shape[2], 2.0 ** -8
    for i, (k, v) in enumerate(rows):
        for t in range(new[i]):
            lim, tok = max(0, lens[i] - new[i] + t + 1), starts[i] + t
            if lim == 0:
                assert bool((out[tok] == 0).all()), (i, t)
                continue
            kd, vd = (x[:lim].double().repeat_interleave(n_qh // x.shape[1], 1) for x in (k, v))
            qd = q[tok].double()
            w = torch.softmax(torch.einsum("hd,lhd->hl", qd, kd) * D ** -0.5, -1)
            y, A = torch.einsum("hl,lhd->hd", w, vd), torch.einsum("hl,lhd->hd", w, vd.abs())
            e = 2.0 ** -22 * D ** 0.5 * torch.einsum("hd,lhd->hl", qd.abs(), kd.abs()).amax(-1)[:, None]
            tol = (u + 2 * e + 2.0 ** -23 * lim + 2.0 ** -21) * A + u * y.abs() + 2.0 ** -25
            assert bool(((out[tok].double() - y).abs() <= tol).all()), (i, t)


UNSEEN = [  # new tokens, lengths and prefix: requests that end inside the prefix
    ((1, 1, 1), (30, 100, 1), 200),  # few rows a head: each request by itself
    ((1,) * 40, tuple(300 + 7 * i for i in range(40)), 5000),  # beside prefix items
    ((4,) * 40, tuple(300 + 7 * i for i in range(40)), 5000),  # many rows, prefix items
    ((150, 0, 90), (330, 900, 140), 700),  # each request by itself, an idle one sees no row
    ((2, 3), (1, 0), 100),  # tokens that see nothing
]


@pytest.mark.parametrize("fill", [float("nan"), float("inf")])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("case", range(len(UNSEEN)))
def test_prefix_rows_that_no_token_sees_hold_anything(cuda, case, D, fill):
    import torch
    import yskn_b200 as Y
    new, lens, P = UNSEEN[case]
    q, rows, out, starts = call(cuda, new, lens, P, fill, D=D, seed=case)
    assert Y.status() == 0
    near(q, rows, out, starts, new, lens)
    assert torch.equal(out, call(cuda, new, lens, P, 0.0, D=D, seed=case)[2])


@pytest.mark.parametrize("n", [1, 20])
def test_lengths_past_a_table_row_are_reported(cuda, n):
    import torch
    import yskn_b200 as Y
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device=cuda)  # noqa: E731
    c = torch.ones((6, 16, 1, 64), dtype=torch.bfloat16, device=cuda)
    q = torch.ones((2 * n, 1, 64), dtype=torch.bfloat16, device=cuda)
    tables, prefix = i32(0, 1, 2, 3).view(2, 2), i32(4, 5)
    work = torch.empty(Y.prefix_attention_work_bytes(2 * n, 3, n, 1, 1, 64), dtype=torch.uint8, device=cuda)

    def status(lens, starts, P):
        Y.prefix_attention(q, c, c, tables, i32(*lens), i32(*starts), n, work, torch.empty_like(q),
                           prefix_blocks=prefix, prefix_len=P)
        return Y.status()

    for P in (0, 20):  # a table row names 32 rows after the prefix
        assert status((P + 32, P + 30), (0, n, 2 * n), P) == 0
        assert status((P + 30, P + 33), (0, n, 2 * n), P) == Y.EINVAL
        assert status((P + 33, P + 30), (0, n, 2 * n), P) == Y.EINVAL
        assert status((2 ** 31 - 1, P + 32), (0, n, 2 * n), P) == Y.EINVAL
        assert status((P + 32, P + 33), (0, n, n), P) == 0  # one without tokens is not read


@pytest.mark.parametrize("G", [1, 2, 4, 6, 8])
@pytest.mark.parametrize("max_new", [2 ** 31 - 1, 2 ** 30, 357913942])
def test_no_bound_on_the_new_tokens(cuda, G, max_new):
    """max_new far above the tokens there are, whose product with G passes 32 bits."""
    run(cuda, new=(1, 50, 2), own=(30, 300, 2), P=200, n_qh=2 * G, n_kvh=2, max_new=max_new, seed=28)
    run(cuda, new=(1, 1), own=(30, 300), P=200, n_qh=2 * G, n_kvh=2, max_new=max_new, seed=28)


@pytest.mark.parametrize("P", [0, 40, 3000])
@pytest.mark.parametrize("n_qh,D", [(6, 64), (40, 128)])  # few rows a KV head, and many
@pytest.mark.parametrize("width", [1, 60])  # of few tiles, and of many
def test_starts_that_do_not_ascend_are_reported(cuda, P, n_qh, D, width):
    """More requests with tokens than there are tokens: nothing is computed, every row is zero."""
    import torch
    import yskn_b200 as Y
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=cuda)  # noqa: E731
    T, B = 2, 60
    c = torch.ones((8, 16, 2, D), dtype=torch.bfloat16, device=cuda)
    q = torch.ones((T, n_qh, D), dtype=torch.bfloat16, device=cuda)
    tables = (torch.arange(B * width, device=cuda) % 8).to(torch.int32).view(B, width)
    work = torch.full((Y.prefix_attention_work_bytes(T, B, 1, n_qh, 2, D),), 255, dtype=torch.uint8, device=cuda)
    for _ in range(2):
        out = torch.full((T, n_qh, D), 3.0, dtype=torch.bfloat16, device=cuda)
        Y.prefix_attention(q, c, c, tables, i32([P + 16 * width] * B), i32([0, 1] * (B // 2) + [0]), 1, work, out,
                           prefix_blocks=i32([0] * -(-max(P, 1) // 16)), prefix_len=P)
        assert Y.status() == Y.EINVAL
        assert bool((out == 0).all())


NOTHING = [  # new tokens, lengths and prefix: some tokens see nothing
    ((1, 1, 1), (30, 0, 1), 40),  # items that are not cut
    ((1, 2, 1), (3000, 1, 0), 0),  # cut ones
    ((2,) * 40, tuple([1, 300] * 20), 5000),  # few rows a head, beside prefix items
    ((4,) * 40, tuple([2, 300, 0, 90] * 10), 5000),  # prefix items
    ((150, 90), (330, 60), 700),  # many rows, each request by itself
    ((20, 9), (4, 15), 0),
]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("case", range(len(NOTHING)))
def test_tokens_that_see_nothing_give_zeros_whatever_their_gate_holds(cuda, case, dtype):
    import torch
    import yskn_b200 as Y
    new, lens, P = NOTHING[case]
    g = torch.randn((sum(new), 6, 128), device=cuda).to({"bf16": torch.bfloat16, "f32": torch.float32}[dtype])
    blind = torch.tensor([n - k + t + 1 <= 0 for n, k in zip(lens, new) for t in range(k)], device=cuda)
    g[blind] = float("nan")
    out = call(cuda, new, lens, P, float("nan"), gate=g, seed=case)[2]
    assert Y.status() == 0 and bool(blind.any())
    assert bool((out[blind] == 0).all()) and not bool(out[~blind].isnan().any())


@pytest.mark.parametrize("own", [12, 15, 16, 17, 63, 64, 65, 127, 128, 129, 191, 192, 193, 255, 256, 257, 600])
@pytest.mark.parametrize("P", [0, 64, 130])
def test_own_lengths_of_many_rows_a_head(cuda, own, P):
    """A tile's edges where items are 256 rows of the tensor cores."""
    for D in (64, 128, 256):
        run(cuda, new=(12, 3), own=(own, 3), P=P, D=D, seed=own)


def test_long_cache_of_many_rows_a_head(cuda):
    """Blocks past 2^31 elements into the cache, prefix and own ones, by the tensor maps."""
    import torch
    import yskn_b200 as Y
    D, block, n_blocks, T, P = 256, 128, 70000, 12, 200
    g = torch.Generator(device=cuda)
    g.manual_seed(29)
    kc, vc = (torch.zeros((n_blocks, block, 1, D), dtype=torch.bfloat16, device=cuda) for _ in range(2))
    for c in (kc, vc):
        c[-3:].normal_(generator=g)
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device=cuda)  # noqa: E731
    q = torch.randn((T, 2, D), generator=g, device=cuda).to(torch.bfloat16)
    out = torch.empty_like(q)
    work = torch.empty(Y.prefix_attention_work_bytes(T, 1, T, 2, 1, D), dtype=torch.uint8, device=cuda)
    Y.prefix_attention(q, kc, vc, i32(n_blocks - 1)[None], i32(P + 100), i32(0, T), T, work, out,
                       prefix_blocks=i32(n_blocks - 3, n_blocks - 2), prefix_len=P)
    assert Y.status() == 0
    rows = [torch.cat([c[-3:-1].reshape(-1, 1, D)[:P], c[-1, :100]]) for c in (kc, vc)]
    near(q, [rows], out, [0, T], (T,), (P + 100,))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("new,lens,P", [((1, 1), (60, 150), 40), ((20, 5), (60, 150), 40), ((4,) * 30, (900,) * 30, 800)])
def test_gates_of_any_size(cuda, new, lens, P, dtype):
    """Infinite and large gates: all of the output or none of it."""
    import torch
    import yskn_b200 as Y
    g = torch.zeros((sum(new), 6, 128), device=cuda)
    for i, x in enumerate((float("inf"), 3e38, 200.0, 89.0, -float("inf"), -3e38, -200.0, -89.0)):
        g[:, :, i::8] = x
    g = g.to({"bf16": torch.bfloat16, "f32": torch.float32}[dtype])
    q, rows, out, starts = call(cuda, new, lens, P, float("nan"), gate=g, seed=30)
    bare = call(cuda, new, lens, P, float("nan"), seed=30)[2]
    assert Y.status() == 0
    for i in range(8):
        if i < 4:
            assert torch.equal(out[:, :, i::8], bare[:, :, i::8])
        else:
            assert bool((out[:, :, i::8].abs() <= 2.0 ** -25).all())


@pytest.mark.parametrize("P", [0, 3000])
@pytest.mark.parametrize("n_qh", [6, 40])
@pytest.mark.parametrize("starts", [(0, 2 ** 31 - 1, -2 ** 31, 1), (2 ** 31 - 1, -2 ** 31, 0, 2), (-2 ** 31, 2 ** 31 - 1, 0, 0),
                                    (3, 4, 4, 3), (-1, 0, 0, 0), (2 ** 31 - 2, 2 ** 31 - 1, -2 ** 31, 0)])
def test_starts_of_any_value_are_reported(cuda, P, n_qh, starts):
    """Tokens that the call does not have, and differences that pass 32 bits."""
    import torch
    import yskn_b200 as Y
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=cuda)  # noqa: E731
    c = torch.ones((8, 16, 2, 64), dtype=torch.bfloat16, device=cuda)
    q = torch.ones((2, n_qh, 64), dtype=torch.bfloat16, device=cuda)
    out = torch.full((2, n_qh, 64), 3.0, dtype=torch.bfloat16, device=cuda)
    work = torch.full((Y.prefix_attention_work_bytes(2, 3, 1, n_qh, 2, 64),), 255, dtype=torch.uint8, device=cuda)
    Y.prefix_attention(q, c, c, i32([[0, 1, 2, 3]] * 3), i32([P + 60] * 3), i32(starts), 1, work, out,
                       prefix_blocks=i32([5] * 188), prefix_len=P)
    assert Y.status() == Y.EINVAL
    assert bool(torch.isin(out, torch.tensor([0.0, 1.0], dtype=torch.bfloat16, device=cuda)).all())
