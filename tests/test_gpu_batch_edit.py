"""Kept rows and forked requests (yskn_b200_batch_edit) against a one-request-at-a-time restatement in Python integers:
all outputs equal, what the call does not own unchanged."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def restated(lens, keep, source, tables, pool, free, bs, P, out_tables, max_copies):
    B, width = tables.shape
    blocks = lambda n: -(-max(n - P, 0) // bs)  # noqa: E731
    own = list(range(B)) if source is None else [int(j) for j in source]
    new = [min(max(int(keep[i]), 0), int(lens[j])) if j >= 0 else 0 for i, j in enumerate(own)]
    heir = {}
    for i, j in enumerate(own):
        if j >= 0 and (j not in heir or new[i] > new[heir[j]]):
            heir[j] = i
    stack = [int(b) for b in pool[:free]]
    for j in range(B):
        stays = blocks(new[heir[j]]) if j in heir else 0
        stack += [int(b) for b in tables[j, stays:blocks(int(lens[j]))]]
    have, copies, waits, asked = len(stack), [], False, 0
    out = out_tables.copy()
    for i, j in enumerate(own):
        if j < 0:
            continue
        n = blocks(new[i])
        if heir[j] == i:
            out[i, :n] = tables[j, :n]
            continue
        asked += n
        waits = waits or asked > min(have, max_copies)
        if waits and n:
            new[i] = 0
            continue
        for b in range(n):
            out[i, b] = stack.pop()
            copies.append((int(tables[j, b]), int(out[i, b]), min(bs, new[i] - P - b * bs)))
    pool = pool.copy()
    pool[free:len(stack)] = stack[free:]
    return new, len(stack), out, pool, copies


def case(rng, B, max_rows, bs, P, fork, ended=0.1, room=1.0, spare=0):
    rows = rng.integers(0, max_rows + 1, B)
    lens = np.where(rows > 0, P + rows, np.where(rng.random(B) < 0.5, 0, P))
    source = None
    if fork is not None:
        source = np.where(rng.random(B) < fork, rng.integers(0, B, B), np.arange(B))
        source[rng.random(B) < ended] = -1
    of = np.arange(B) if source is None else np.maximum(source, 0)
    keep = np.maximum(lens[of] - rng.integers(-3, 2 * bs, B), -1)
    held = -(-np.maximum(lens - P, 0) // bs)
    width = int(max(1, held.max())) + spare
    free = int(room * B * 2)
    numbers = rng.permutation(int(held.sum()) + free + 3)
    tables = np.full((B, width), -7, np.int32)
    at = 0
    for i in range(B):
        tables[i, :held[i]] = numbers[at:at + held[i]]
        at += held[i]
    pool = np.full(int(held.sum()) + free + 1, -9, np.int32)
    pool[:free] = numbers[at:at + free]
    return lens.astype(np.int32), keep.astype(np.int32), source, tables, pool, free, bs, P


def run(cuda, c, max_copies=10000, stream=None, status=0):
    import torch
    import yskn_b200 as Y
    lens, keep, source, tables, pool, free, bs, P = c
    B, width = tables.shape
    t = lambda a: torch.from_numpy(np.array(a, np.int32)).to(cuda)  # noqa: E731
    wide = torch.full((B, width + 3), -5, dtype=torch.int32, device=cuda)
    wide[:, :width].copy_(t(tables))
    out = torch.full((B, width + 2), -6, dtype=torch.int32, device=cuda)
    copies = torch.full((3, max_copies + 4), -77, dtype=torch.int32, device=cuda)
    d_pool, lens_out, free_out, n = t(pool), t([-77] * B), t([-77]), t([-77])
    fork = {} if source is None else dict(source=t(source), tables_out=out[:, :width], copies=copies[:, :max_copies],
                                          n_copies=n)
    args = t(lens), t(keep), wide[:, :width], d_pool, t([free]), bs, lens_out, free_out
    torch.cuda.synchronize()
    Y.batch_edit(*args, prefix_len=P, stream=stream, **fork)
    torch.cuda.synchronize()
    assert Y.status() == status
    want = restated(lens, keep, source, tables, pool, free, bs, P, np.full((B, width), -6, np.int32), max_copies)
    assert lens_out.cpu().tolist() == want[0]
    assert int(free_out) == want[1]
    assert np.array_equal(d_pool.cpu().numpy(), want[3])
    assert np.array_equal(wide[:, :width].cpu().numpy(), tables) and (wide[:, width:] == -5).all()
    if source is not None:
        assert np.array_equal(out[:, :width].cpu().numpy(), want[2]) and (out[:, width:] == -6).all()
        got = copies.cpu().numpy()
        assert (got[:, max_copies:] == -77).all()
        assert int(n) == len(want[4])
        assert [tuple(map(int, e)) for e in got[:, :len(want[4])].T] == want[4]
        assert (got[:2, len(want[4]):max_copies] == -1).all() and (got[2, len(want[4]):max_copies] == 0).all()
    return want


@pytest.mark.parametrize("B", [1, 2, 31, 33, 511, 513, 2000, 4096])
@pytest.mark.parametrize("fork", [None, 0.0, 0.4, 1.0])
def test_batches(cuda, B, fork):
    run(cuda, case(np.random.default_rng(B), B, 90, 16, 40, fork))


@pytest.mark.parametrize("bs", [1, 5, 16, 64, 128])
@pytest.mark.parametrize("P", [0, 1, 1000])
def test_blocks_and_prefixes(cuda, bs, P):
    for fork in (None, 0.5):
        run(cuda, case(np.random.default_rng(bs + P), 60, 700, bs, P, fork, spare=2))


@pytest.mark.parametrize("room", [0.0, 0.3, 0.7])
def test_pools_that_are_too_small(cuda, room):
    """Most requests continue the two longest ones: more blocks than the others give back."""
    for seed in range(5):
        c = case(np.random.default_rng(seed), 200, 300, 16, 20, 0.6, ended=0.0, room=room)
        longest = np.argsort(c[0])[-2:]
        c[2][:] = np.where(np.arange(200) % 5 < 4, longest[np.arange(200) % 2], c[2])
        c[1][:] = c[0][c[2]] - np.arange(200) % 3
        want = run(cuda, c)
        assert any(w == 0 and k > 20 for w, k in zip(want[0], c[1]))


def test_a_short_list_of_copies(cuda):
    c = case(np.random.default_rng(3), 100, 100, 16, 0, 0.6)
    for n in (1, 2, 40, 100):
        run(cuda, c, max_copies=n)


def test_beams_of_one_and_exchanged_requests(cuda):
    rng = np.random.default_rng(4)
    c = list(case(rng, 64, 500, 32, 100, 0.0, ended=0.0, room=20.0))
    c[0][9] = 100 + 490
    c[2] = np.full(64, 9)  # all continue request 9
    held = -(-np.maximum(c[0] - 100, 0) // 32)
    numbers = rng.permutation(5000)
    width = int(held.max())
    c[3] = np.full((64, width), -7, np.int32)
    at = 0
    for i in range(64):
        c[3][i, :held[i]] = numbers[at:at + held[i]]
        at += held[i]
    c[5] = 1100
    c[4] = np.full(int(held.sum()) + 1100, -9, np.int32)
    c[4][:1100] = numbers[at:at + 1100]
    run(cuda, tuple(c))
    c[2] = np.arange(64)[::-1].copy()  # every request another's: tables move, nothing is copied
    c[1] = c[0][::-1].copy()
    assert run(cuda, tuple(c))[4] == []


def test_long_tables(cuda):
    run(cuda, case(np.random.default_rng(5), 3, 70000, 16, 0, 1.0, ended=0.0, room=3000.0))


def test_what_the_device_refuses(cuda):
    import torch
    import yskn_b200 as Y
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device=cuda)  # noqa: E731

    def call(lens=(20, 5), keep=(20, 5), source=(0, 1), free=2, width=2):
        outs = dict(lens_out=i32(-7, -7), free_out=i32(-7))
        Y.batch_edit(i32(*lens), i32(*keep), i32(*range(2 * width)).view(2, width), i32(8, 9, 10, -1, -1, -1, -1),
                     i32(free), 16, **outs, source=i32(*source),
                     tables_out=torch.zeros(2, width, dtype=torch.int32, device=cuda),
                     copies=torch.zeros(3, 5, dtype=torch.int32, device=cuda), n_copies=i32(0))
        return Y.status(), outs["lens_out"].tolist()

    assert call() == (0, [20, 5])
    assert call(source=(0, 2)) == (Y.EINVAL, [20, 0])
    assert call(lens=(50, 5))[0] == Y.EINVAL  # more rows than its table row names
    assert call(free=-1)[0] == Y.EINVAL and call(free=8)[0] == Y.EINVAL
    assert call(free=7, lens=(20, 5), keep=(1, 5))[0] == Y.EINVAL  # more than the pool holds
    assert call(lens=(2 ** 31 - 1, 5), keep=(2 ** 31 - 1, 5))[0] == Y.EINVAL
    assert call(lens=(-5, 5), keep=(3, 5)) == (0, [0, 5])


def test_another_stream_and_a_graph(cuda):
    import torch
    import yskn_b200 as Y
    c = case(np.random.default_rng(6), 50, 100, 16, 20, 0.5)
    run(cuda, c, stream=torch.cuda.Stream(cuda))
    lens, keep, source, tables, pool, free, bs, P = c
    t = lambda a: torch.from_numpy(np.array(a, np.int32)).to(cuda)  # noqa: E731
    d = [t(lens), t(np.zeros_like(keep)), t(tables), t(pool), t([free])]
    lo, fo, out, n = t(lens), t([0]), t(np.full_like(tables, -6)), t([0])
    cp = torch.zeros(3, 500, dtype=torch.int32, device=cuda)
    src = t(source)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        Y.batch_edit(*d, bs, lo, fo, source=src, tables_out=out, copies=cp, n_copies=n, prefix_len=P)
    d[1].copy_(t(keep))
    d[3].copy_(t(pool))
    g.replay()
    torch.cuda.synchronize()
    want = restated(lens, keep, source, tables, pool, free, bs, P, np.full_like(tables, -6), 500)
    assert lo.cpu().tolist() == want[0] and int(n) == len(want[4]) and np.array_equal(out.cpu().numpy(), want[2])
