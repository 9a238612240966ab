"""Ancestor bits and positions of drafted trees (yskn_b200_tree_plan) and accepted paths (yskn_b200_tree_accept) against
one-node-at-a-time restatements in Python integers."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def draw_trees(rng, counts, kind="random"):
    out = []
    for n in counts:
        if kind == "chain":
            out.append(list(range(-1, n - 1)))
        elif kind == "forest":
            out.append([int(rng.integers(-1, j)) if j else -1 for j in range(n)])
        else:
            out.append([-1][:n] + [int(rng.integers((j - 1) // 4, (j - 1) // 2 + 1)) for j in range(1, n)])
    return out


def plan(cuda, trees, before, words, pad=0, requests=None, parents=None, stream=None):
    import torch
    import yskn_b200 as Y
    counts = [len(t) for t in trees]
    T, B = sum(counts) + pad, len(trees)
    i32 = lambda a: torch.tensor(list(map(int, a)), dtype=torch.int32, device=cuda)  # noqa: E731
    starts = np.concatenate([[0], np.cumsum(counts)])
    req = [i for i, n in enumerate(counts) for _ in range(n)] + [-1] * pad if requests is None else requests
    par = [p for t in trees for p in t] + [7] * pad if parents is None else parents
    mask = torch.full((T, words + 2), 77, dtype=torch.int32, device=cuda)
    pos = torch.full((T,), 77, dtype=torch.int32, device=cuda)
    args = [i32(par), i32(req), i32(starts), i32([b + n for b, n in zip(before, counts)])]
    torch.cuda.synchronize()
    Y.tree_plan(*args, mask[:, :words], pos, stream=stream)
    torch.cuda.synchronize()
    m = mask.cpu().numpy()
    assert (m[:, words:] == 77).all()
    return m[:, :words].view(np.uint32), pos.cpu().numpy(), Y.status()


@pytest.mark.parametrize("counts", [[1], [0, 3, 0], [32, 33], [64, 65, 1], [100, 7, 128, 0, 31], [1024, 5]])
@pytest.mark.parametrize("kind", ["random", "chain", "forest"])
def test_plan(cuda, counts, kind):
    rng = np.random.default_rng(sum(counts))
    trees = draw_trees(rng, counts, kind)
    before = rng.integers(0, 1000, len(counts))
    words = max(1, -(-max(counts) // 32))
    mask, pos, status = plan(cuda, trees, before, words, pad=3)
    assert status == 0
    t = 0
    for parents, b in zip(trees, before):
        seen = []
        for j, p in enumerate(parents):
            seen.append((seen[p] if p >= 0 else 0) | 1 << j)
            assert sum(int(w) << 32 * k for k, w in enumerate(mask[t])) == seen[j]
            assert pos[t] == b + bin(seen[j]).count("1") - 1
            t += 1
    assert (mask[t:] == 0).all() and (pos[t:] == -1).all()


def test_plan_of_what_does_not_fit(cuda):
    """Parents at or behind their node are taken for none, nodes past the mask have no bits: both reported."""
    import yskn_b200 as Y
    mask, pos, status = plan(cuda, [[-1, 1, 0, 9, 2]], [10], 1)
    assert status == Y.EINVAL
    assert mask[:, 0].tolist() == [1, 2, 5, 8, 21] and pos.tolist() == [10, 10, 11, 10, 12]
    mask, pos, status = plan(cuda, draw_trees(None, [40], "chain"), [0], 1)
    assert status == Y.EINVAL and mask[:, 0].tolist() == [(1 << min(j + 1, 32)) - 1 for j in range(40)]
    assert pos.tolist() == list(range(40))
    for req in ([0, 0, 1], [0, 1, 1], [2, 0, 0], [0, 0, 5]):  # tokens that are not their request's
        status = plan(cuda, [[-1, 0], [-1]], [4, 4], 1, requests=req)[2]
        assert status == (0 if req == [0, 0, 1] else Y.EINVAL)
    assert plan(cuda, [[-1]], [2 ** 31 - 2], 1)[1].tolist() == [2 ** 31 - 2]


def accept(cuda, trees, tokens, choice, lens, width, starts=None, in_place=False, stream=None):
    import torch
    import yskn_b200 as Y
    i32 = lambda a: torch.tensor(list(map(int, a)), dtype=torch.int32, device=cuda)  # noqa: E731
    starts = np.concatenate([[0], np.cumsum([len(t) for t in trees])]) if starts is None else starts
    B = len(trees)
    path = torch.full((B, width + 1), 77, dtype=torch.int32, device=cuda)
    outs = [torch.full((B,), 77, dtype=torch.int32, device=cuda) for _ in range(3)]
    d_lens = i32(lens)
    if in_place:
        outs[1] = d_lens
    args = [i32(tokens), i32([p for t in trees for p in t]), i32(choice), i32(starts)]
    torch.cuda.synchronize()
    Y.tree_accept(*args, d_lens, path[:, :width], *outs, stream=stream)
    torch.cuda.synchronize()
    assert (path[:, width] == 77).all()
    return [path[:, :width].cpu().tolist()] + [o.cpu().tolist() for o in outs] + [Y.status()]


def restated(trees, tokens, choice, lens, width):
    paths, accepted, out, nxt, s = [], [], [], [], 0
    for parents, n_rows in zip(trees, lens):
        n, path = len(parents), []
        if n:
            path = [0]
            while len(path) < width:
                c = choice[s + path[-1]]
                follows = [j for j in range(path[-1] + 1, n)
                           if parents[j] == path[-1] and tokens[s + j] == c and c >= 0]
                if not follows:
                    break
                path.append(follows[0])
        paths.append(path + [-1] * (width - len(path)))
        accepted.append(len(path))
        out.append(n_rows - n + len(path))
        nxt.append(choice[s + path[-1]] if path else -1)
        s += n
    return [paths, accepted, out, nxt, 0]


@pytest.mark.parametrize("counts", [[1], [0, 3, 0], [32, 33], [64, 65, 1], [100, 7, 128, 0, 31] * 5, [500]])
@pytest.mark.parametrize("kind", ["random", "chain", "forest"])
@pytest.mark.parametrize("width", [1, 4, 200])
def test_accept(cuda, counts, kind, width):
    rng = np.random.default_rng(sum(counts) + width)
    trees = draw_trees(rng, counts, kind)
    T, starts = sum(counts), np.concatenate([[0], np.cumsum(counts)])
    tokens, choice = rng.integers(0, 3, T), rng.integers(-1, 3, T)  # siblings with equal tokens among them
    if kind == "chain":
        choice = np.where(rng.random(T) < 0.97, np.roll(tokens, -1), choice)
    lens = [int(rng.integers(0, 900)) + n for n in counts]
    want = restated(trees, tokens.tolist(), choice.tolist(), lens, width)
    assert accept(cuda, trees, tokens, choice, lens, width) == want
    assert accept(cuda, trees, tokens, choice, lens, width, in_place=True) == want
    assert len(starts) == len(counts) + 1


def test_accept_of_what_does_not_fit(cuda):
    import yskn_b200 as Y
    trees = [[-1, 0], [-1]]
    for starts in ([0, 2, 9], [-1, 2, 3], [0, 3, 2]):
        got = accept(cuda, trees, [1, 1, 1], [1, 1, 1], [5, 5], 3, starts=starts)
        assert got[4] == Y.EINVAL
        for i in range(2):
            if not 0 <= starts[i] <= starts[i + 1] <= 3:
                assert got[0][i] == [-1] * 3 and got[1][i] == 0 and got[2][i] == 5 and got[3][i] == -1
    # a negative choice is no padding node's token
    assert accept(cuda, [[-1, 0]], [4, -1], [-1, -1], [5], 3)[:4] == [[[0, -1, -1]], [1], [4], [-1]]


def test_streams_and_a_graph(cuda):
    import torch
    import yskn_b200 as Y
    rng = np.random.default_rng(1)
    trees = draw_trees(rng, [20, 30])
    tokens, choice = rng.integers(0, 2, 50), rng.integers(0, 2, 50)
    side = torch.cuda.Stream(cuda)
    a = accept(cuda, trees, tokens, choice, [30, 40], 6)
    assert accept(cuda, trees, tokens, choice, [30, 40], 6, stream=side) == a
    m, p, _ = plan(cuda, trees, [5, 9], 1)
    m2, p2, _ = plan(cuda, trees, [5, 9], 1, stream=side)
    assert (m == m2).all() and (p == p2).all()
    i32 = lambda v: torch.tensor(list(map(int, v)), dtype=torch.int32, device=cuda)  # noqa: E731
    par, req, st, ln = i32([x for t in trees for x in t]), i32([0] * 20 + [1] * 30), i32([0, 20, 50]), i32([25, 39])
    mask, pos = torch.zeros(50, 1, dtype=torch.int32, device=cuda), i32([0] * 50)
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        Y.tree_plan(par, req, st, ln, mask, pos)
    ln.copy_(i32([35, 49]))
    g.replay()
    torch.cuda.synchronize()
    assert (mask.cpu().numpy().view(np.uint32) == m).all() and (pos.cpu().numpy() == p + 10).all()
