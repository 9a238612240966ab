"""Blocks copied and accepted rows made adjacent in the layers' caches (yskn_b200_cache_copy, yskn_b200_cache_compact):
every element of every cache equal to a copy made row by row, what is not moved unchanged."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def make(cuda, n, n_blocks, block, heads, D, head_major, gen):
    import torch
    shape = (n_blocks, heads, block, D + 8) if head_major else (n_blocks, block, heads, D + 8)  # rows with a stride
    out = []
    for _ in range(n):
        c = torch.randint(-2 ** 15, 2 ** 15, shape, generator=gen, device=cuda, dtype=torch.int16)
        out.append(c[..., :D].transpose(1, 2) if head_major else c[..., :D])
    return out


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("block", [1, 16, 64, 100, 128])
@pytest.mark.parametrize("head_major", [True, False])
def test_copies(cuda, D, block, head_major):
    import torch
    import yskn_b200 as Y
    gen = torch.Generator(device=cuda)
    gen.manual_seed(D + block)
    rng = np.random.default_rng(D + block)
    n, heads = 23, 3
    caches = make(cuda, 5, 60, block, heads, D, head_major, gen)
    whole = [c.clone() for c in caches]
    numbers = rng.permutation(60)
    source, target = numbers[rng.integers(0, 20, n)], numbers[20:20 + n]
    rows = rng.integers(0, block + 1, n)
    copies = torch.from_numpy(np.stack([source, target, rows]).astype(np.int32)).to(cuda)
    for count in (0, 7, n):
        Y.cache_copy(Y.CacheSet(caches), copies, torch.tensor([count], dtype=torch.int32, device=cuda))
        for c, w in zip(caches, whole):
            for e in range(count):
                w[target[e], :rows[e]] = w[source[e], :rows[e]]
            assert torch.equal(c, w)
    assert Y.status() == 0


def test_a_whole_list_and_many_caches(cuda):
    import torch
    import yskn_b200 as Y
    gen = torch.Generator(device=cuda)
    gen.manual_seed(1)
    caches = make(cuda, 256, 10, 16, 1, 64, True, gen)
    whole = [c.clone() for c in caches]
    copies = torch.tensor([[0, 0, -1, 3], [5, 6, -1, 7], [16, 3, 0, 9]], dtype=torch.int32, device=cuda)
    side = torch.cuda.Stream(cuda)
    torch.cuda.synchronize()
    Y.cache_copy(Y.CacheSet(caches), copies, stream=side)
    torch.cuda.synchronize()
    for c, w in zip(caches, whole):
        w[5], w[6, :3], w[7, :9] = w[0], w[0, :3], w[3, :9]
        assert torch.equal(c, w)
    assert Y.status() == 0


def test_copies_that_the_device_refuses(cuda):
    import torch
    import yskn_b200 as Y
    gen = torch.Generator(device=cuda)
    gen.manual_seed(2)
    caches = make(cuda, 2, 6, 16, 2, 64, True, gen)
    whole = [c.clone() for c in caches]
    for bad in ((6, 0, 4), (-1, 0, 4), (0, 6, 4), (0, -3, 4), (0, 1, 17), (2 ** 30, 2 ** 30, 1)):
        copies = torch.tensor([[bad[0], 2], [bad[1], 3], [bad[2], 5]], dtype=torch.int32, device=cuda)
        Y.cache_copy(Y.CacheSet(caches), copies)
        assert Y.status() == Y.EINVAL
        for c, w in zip(caches, whole):
            w[3, :5] = w[2, :5]
            assert torch.equal(c, w)
    # a count outside the list is cut to it
    for count in (-4, 9):
        Y.cache_copy(Y.CacheSet(caches), torch.tensor([[2], [4], [1]], dtype=torch.int32, device=cuda),
                     torch.tensor([count], dtype=torch.int32, device=cuda))
        for c, w in zip(caches, whole):
            if count > 0:
                w[4, :1] = w[2, :1]
            assert torch.equal(c, w)
    assert Y.status() == 0


def compact(cuda, D=64, block=16, P=0, head_major=True, new=(9, 0, 30), ctx=(10, 3, 50), paths=None, width=12, n=4,
            heads=2, seed=0, bad_block=None, lens=None, stream=None, status=0):
    import torch
    import yskn_b200 as Y
    gen = torch.Generator(device=cuda)
    gen.manual_seed(seed)
    rng = np.random.default_rng(seed)
    held = [-(-(c + m) // block) for c, m in zip(ctx, new)]
    n_blocks = sum(held) + 2
    caches = make(cuda, n, n_blocks, block, heads, D, head_major, gen)
    whole = [c.clone() for c in caches]
    numbers = rng.permutation(n_blocks)
    tables = np.full((len(new), max(held) + 1), -1, np.int32)
    at = 0
    for i in range(len(new)):
        tables[i, :held[i]] = numbers[at:at + held[i]]
        at += held[i]
    if paths is None:
        paths = []
        for m in new:
            k = int(rng.integers(1, min(m, width) + 1)) if m else 0
            paths.append(sorted(int(x) for x in rng.choice(m, k, replace=False)) if m else [])
    path = np.full((len(new), width + 1), 5, np.int32)
    path[:, :width] = -1
    for i, p in enumerate(paths):
        path[i, :min(len(p), width)] = p[:width]
    if bad_block is not None:
        tables[bad_block] = n_blocks
    t = lambda a: torch.from_numpy(np.array(a, np.int32)).to(cuda)  # noqa: E731
    starts = np.concatenate([[0], np.cumsum(new)])
    d_lens = t([P + c + m for c, m in zip(ctx, new)]) if lens is None else t(lens)
    args = Y.CacheSet(caches), t(tables), d_lens, t(starts), t(path)[:, :width]
    torch.cuda.synchronize()
    Y.cache_compact(*args, prefix_len=P, stream=stream)
    torch.cuda.synchronize()
    assert Y.status() == status
    return caches, whole, tables, paths


def expect(whole, tables, paths, ctx, block, n_blocks):
    import torch
    for w in whole:
        for i, p in enumerate(paths):
            old = [w[tables[i, (ctx[i] + j) // block], (ctx[i] + j) % block].clone() if
                   0 <= tables[i, (ctx[i] + j) // block] < n_blocks else None for j in p]
            for k, row in enumerate(old):
                b = tables[i, (ctx[i] + k) // block]
                if row is not None and 0 <= b < n_blocks:
                    w[b, (ctx[i] + k) % block] = row
    torch.cuda.synchronize()
    return whole


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("block", [1, 7, 16, 64])
@pytest.mark.parametrize("P", [0, 100])
def test_paths(cuda, D, block, P):
    import torch
    for head_major in (True, False):
        for seed in range(3):
            ctx = (10, 3, 50)
            caches, whole, tables, paths = compact(cuda, D=D, block=block, P=P, head_major=head_major, ctx=ctx,
                                                   seed=seed)
            for c, w in zip(caches, expect(whole, tables, paths, ctx, block, len(whole[0]))):
                assert torch.equal(c, w)


def test_rows_that_are_sources_and_places_at_once(cuda):
    """Long paths whose every row moves by a little: each row is read before it is overwritten."""
    import torch
    for D in (64, 128, 256):
        for paths in ([list(range(1, 90)), list(range(90)), [0] + list(range(2, 91))],
                      [list(range(10, 90)), [89], list(range(0, 90, 2))]):
            ctx = (5, 0, 33)
            caches, whole, tables, paths = compact(cuda, D=D, new=(91, 90, 91), ctx=ctx, paths=paths, width=90, n=2,
                                                   seed=D)
            for c, w in zip(caches, expect(whole, tables, paths, ctx, 16, len(whole[0]))):
                assert torch.equal(c, w)


def test_paths_that_the_device_refuses(cuda):
    import torch
    import yskn_b200 as Y
    for paths, good in (([[0, 2, 2]], [[0, 2]]), ([[3, 1]], [[3]]), ([[0, 4, 9, 10]], [[0, 4]]),
                        ([[0, 3, 2 ** 30]], [[0, 3]])):
        caches, whole, tables, _ = compact(cuda, new=(9,), ctx=(10,), paths=paths, status=Y.EINVAL)
        for c, w in zip(caches, expect(whole, tables, good, (10,), 16, len(whole[0]))):
            assert torch.equal(c, w)
    # a block outside the caches: its rows are left alone
    caches, whole, tables, paths = compact(cuda, new=(9,), ctx=(10,), paths=[[1, 2, 7, 8]], bad_block=(0, 1),
                                           status=Y.EINVAL)
    for c, w in zip(caches, expect(whole, tables, paths, (10,), 16, len(whole[0]))):
        assert torch.equal(c, w)
    # lengths that do not hold the new rows, or that the table does not name
    for lens in ((5,), (2 ** 31 - 1,), (0,)):
        caches, whole, _, _ = compact(cuda, new=(9,), ctx=(10,), paths=[[0, 2]], lens=lens, status=Y.EINVAL)
        assert all(torch.equal(c, w) for c, w in zip(caches, whole))


def test_another_stream(cuda):
    import torch
    ctx = (10, 3, 50)
    caches, whole, tables, paths = compact(cuda, ctx=ctx, stream=torch.cuda.Stream(cuda))
    for c, w in zip(caches, expect(whole, tables, paths, ctx, 16, len(whole[0]))):
        assert torch.equal(c, w)
