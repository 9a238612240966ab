"""Drafted trees, forked requests and log probabilities in the serving loop (yskn_b200/batch.py): two attention layers,
a 4096-row head, against the same loop one token at a time.

Tolerance of the logits as in the loop's own test: the L2 norm of the difference over that of the logits, at most 20
roundings of 2^-8 in two layers. A row that is missing, or another node's in its place, differs by more than that: the
tests compare against such a cache too."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

VOCAB = 4096
TOL = 20 * 2.0 ** -8


def _stack(cuda, **kw):
    from yskn_b200 import batch
    return batch.BatchStack(cuda, layers=2, vocab=VOCAB, seed=5, block_size=16, **kw)


def _prefix(cuda, n):
    import torch
    return ((torch.arange(n, device=cuda) * 977 + 13) % VOCAB).to(torch.int32)


def _prompt(i, n):
    return [(131 * i + 29 * j + 7) % VOCAB for j in range(n)]


def _close(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


def _started(cuda, sizes, P=75, **kw):
    """A loop whose requests have run their prompts and said one token."""
    st = _stack(cuda, batch=len(sizes), max_tokens=96, capacity=64, n_blocks=40, nodes=40, **kw)
    if P:
        st.fill_prefix(_prefix(cuda, P))
    for i, n in enumerate(sizes):
        st.say(i, _prompt(i, n))
    st.new.copy_(st.said)
    st.step(sum(sizes), max(sizes))
    return st


def _choices(monkeypatch, forced):
    """The selection answers forced[row] for those rows of a verification: the model's own choice is as good as a coin's
    where two logits are about equal, and other orders of sums move them by 0.2 here."""
    import yskn_b200 as Y
    select = Y.head_select

    def chosen(logits, token=None, **kw):
        select(logits, token=token, **kw)
        for row, t in forced.items():
            token[row] = t

    monkeypatch.setattr(Y, "head_select", chosen)


@pytest.mark.parametrize("P", [0, 75])
def test_verified_trees_equal_steps(cuda, P, monkeypatch):
    import torch
    import yskn_b200 as Y
    sizes, right = [3, 19, 14], [4, 1, 0]
    one = _started(cuda, sizes, P)
    logits = [one.blogits.clone()]
    for _ in range(6):
        one.new.fill_(1)
        one.step(3, 1)
        logits.append(one.blogits.clone())
    text = one.text.tolist()

    st = _started(cuda, sizes, P)
    # the true continuation's first 4, 1 and 0 tokens, each among others that are not the model's
    forced, nodes = {}, []
    for i, n in enumerate(sizes):
        tokens, parents, path = [], [], [0]
        for t in text[i][n + 1:n + 1 + right[i]]:  # two wrong ones, the right one, and the right one under a wrong one
            tokens += [(t + 1) % VOCAB, (t + 2) % VOCAB, t]
            parents += [path[-1]] * 3
            path.append(len(tokens))
            tokens.append(t)
            parents.append(len(tokens) - 2)
        tokens.append((text[i][n + 1 + right[i]] + 5) % VOCAB)  # where the draft goes wrong
        parents.append(path[-1])
        st.draft(i, tokens, parents)
        st.new[i] = 1 + len(tokens)
        first = int(st.new[:i].sum())
        forced.update({first + node: text[i][n + 1 + k] for k, node in enumerate(path)})
        nodes.append([first + node for node in path])
    before = st.free.item()
    _choices(monkeypatch, forced)
    st.verify(int(st.new.sum()))
    monkeypatch.undo()
    assert Y.status() == 0
    assert st.accepted.tolist() == [1 + r for r in right]
    assert st.said.tolist() == [n + 2 + r for n, r in zip(sizes, right)]
    assert st.lens.tolist() == [P + n + 1 + r for n, r in zip(sizes, right)]
    held = [-(-(n + 1 + r) // 16) - -(-n // 16) for n, r in zip(sizes, right)]
    assert st.free.item() == before - sum(held)
    for i, n in enumerate(sizes):
        assert st.text[i, :n + 2 + right[i]].tolist() == text[i][:n + 2 + right[i]]
        # every node on the path has the logits of the step that its token was said in, and they leave room for what
        # was chosen there
        for k, node in enumerate(nodes[i]):
            row, step = st.tlogits[node], logits[1 + k][i]
            assert _close(row, step) <= TOL, (i, k)
            assert row.max() - row[text[i][n + 1 + k]] <= 2 * (row - step).abs().max()
    # and the cache is as those steps left it
    st.new.fill_(1)
    st.step(3, 1)
    for i in range(3):
        assert _close(st.blogits[i], logits[2 + right[i]][i]) <= TOL, i
    assert Y.status() == 0


def test_wrong_rows_in_the_cache_would_show(cuda, monkeypatch):
    """The tolerance tells a cache with the path's rows left where they were from a packed one."""
    import yskn_b200 as Y
    far = []
    for packed in (True, False):
        st = _started(cuda, [9], 40)
        st.draft(0, [1, 2, 3, 4], [0, 0, 0, 3])
        st.new.fill_(5)
        _choices(monkeypatch, {0: 3, 3: 4, 4: 5})
        if not packed:
            monkeypatch.setattr(Y, "cache_compact", lambda *a, **k: None)
        st.verify(5)
        monkeypatch.undo()
        assert st.accepted.tolist() == [3] and st.text[0, 10:13].tolist() == [3, 4, 5]
        st.new.fill_(1)
        st.step(1, 1)
        far.append(st.blogits[0].clone())
    assert _close(far[1], far[0]) > TOL


def test_verify_beside_waiting_and_idle_requests(cuda):
    import torch
    import yskn_b200 as Y
    st = _started(cuda, [3, 19, 14, 5])
    said, lens = st.said.tolist(), st.lens.tolist()
    st.draft(1, [5, 6, 7], [0, 1, 0])
    st.draft(3, [9], [0])
    st.new.copy_(torch.tensor([0, 4, -1, 2], dtype=torch.int32))
    st.verify(30)  # padded places behind the trees
    assert Y.status() == 0
    acc = st.accepted.tolist()
    assert acc[0] == acc[2] == 0 and 1 <= acc[1] <= 3 and 1 <= acc[3] <= 2
    assert st.said.tolist() == [said[i] + acc[i] for i in range(4)]
    assert st.lens.tolist() == [lens[0], lens[1] + acc[1], 0, lens[3] + acc[3]]
    text = st.text.clone()
    st.new.zero_()
    st.verify(8)
    assert torch.equal(st.text, text) and Y.status() == 0


def test_a_full_text_takes_no_more(cuda):
    import torch
    import yskn_b200 as Y
    st = _stack(cuda, batch=1, max_tokens=64, capacity=16, n_blocks=8, nodes=8)
    st.say(0, _prompt(0, 14))
    st.new.fill_(14)
    st.step(14, 14)
    st.draft(0, [1], [0])
    st.new.fill_(2)
    st.verify(2)
    assert st.said.item() == min(15 + st.accepted.item(), 16) and st.lens.item() == 14 + st.accepted.item()
    st.draft(0, [1, 2], [0, 1])
    st.new.fill_(3)
    st.verify(3)  # its rows do not fit its table: it waits
    assert st.said.item() == 16 and st.lens.item() <= 16 and Y.status() == 0
    with pytest.raises(Y.YsknError):
        st.draft(0, [1] * 8, [0] * 8)
    with pytest.raises(Y.YsknError):
        st.draft(0, [1, 2], [0, 2])
    with pytest.raises(Y.YsknError):
        _stack(cuda, batch=1, max_tokens=4, capacity=16, n_blocks=4).draft(0, [1], [0])
    assert torch.cuda.is_available()


def test_forked_requests_go_on_alike(cuda):
    import torch
    import yskn_b200 as Y
    sizes = [3, 19, 14, 5, 1]
    one, st = _started(cuda, sizes, logprobs=4), _started(cuda, sizes, logprobs=4)
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device=cuda)  # noqa: E731
    source = [1, 1, -1, 1, 0]
    st.presence[1] = 0.5
    one.presence[1] = 0.5
    st.fork(i32(*source))
    assert Y.status() == 0
    assert st.said.tolist() == [20, 20, 0, 20, 4] and st.lens.tolist() == [94, 94, 0, 94, 78]
    assert st.presence.tolist() == [0.5, 0.5, 0.0, 0.5, 0.0]
    assert st.free.item() == 40 - 5 - 2 * 3 - 1
    used = [st.tables[i, :-(-max(st.lens[i].item() - 75, 0) // 16)].tolist() for i in range(5)]
    flat = [b for t in used for b in t]
    assert len(set(flat)) == len(flat) and not set(flat) & set(st.prefix_blocks.tolist())
    for _ in range(14):  # past a block's end
        one.new.fill_(1)
        one.step(5, 1)
        st.new.copy_(i32(1, 1, 0, 1, 1))
        st.step(5, 1)
        for i, j in enumerate(source):
            if j >= 0:
                assert _close(st.blogits[i], one.blogits[j]) <= TOL, (i, j)
        assert torch.equal(st.text[0], st.text[1]) and torch.equal(st.text[0], st.text[3])
        # the chosen token's log probability, the entropy, and the likeliest tokens
        logp = torch.log_softmax(st.blogits.double(), -1)
        chosen = logp.gather(1, st.btoken.long().unsqueeze(1))
        assert torch.allclose(st.logprob.double(), chosen, rtol=0, atol=1e-5)
        assert torch.equal(st.top_ids[:, 0], st.btoken) and torch.equal(st.top_logprobs[:, :1], st.logprob)
        assert torch.allclose(st.entropy.double(), -(logp.exp() * logp).sum(-1), rtol=0, atol=1e-4)
    assert Y.status() == 0


def test_a_fork_that_the_pool_does_not_hold_runs_again(cuda):
    import torch
    import yskn_b200 as Y
    st = _stack(cuda, batch=2, max_tokens=64, capacity=32, n_blocks=4, nodes=4)
    st.fill_prefix(_prefix(cuda, 16))
    st.say(0, _prompt(0, 20))
    st.new.copy_(torch.tensor([20, 0], dtype=torch.int32))
    st.step(20, 20)
    assert st.free.item() == 1
    st.fork(torch.tensor([0, 0], dtype=torch.int32, device=cuda))
    assert st.lens.tolist() == [36, 0] and st.said.tolist() == [21, 21] and st.free.item() == 1
    assert torch.equal(st.text[0], st.text[1]) and Y.status() == 0
    st.new.copy_(torch.tensor([-1, 21], dtype=torch.int32))
    st.step(42, 21)
    assert st.lens.tolist() == [0, 37] and st.said.tolist() == [21, 22] and Y.status() == 0


def test_graphs_and_streams(cuda):
    """A verification and a fork, captured and replayed, on a stream of their own: as eager ones."""
    import torch
    import yskn_b200 as Y

    def run(kind):
        st = _started(cuda, [3, 19, 14], logprobs=2)
        for i in range(3):
            st.draft(i, [(11 * i + j) % VOCAB for j in range(5)], [0, 0, 1, 2, 1])
        st.new.fill_(6)
        source = torch.tensor([1, 1, 2], dtype=torch.int32, device=cuda)
        torch.cuda.synchronize()
        stream = torch.cuda.Stream(cuda) if kind else None
        if kind == "graph":
            with torch.cuda.stream(stream):
                copy = [t.clone() for t in (st.lens, st.free, st.text, st.said, st.pool, st.tables)]
                pages = [c.clone() for c in st.caches.caches]
                st.verify(18, stream)  # warm; then everything back
                for t, c in zip((st.lens, st.free, st.text, st.said, st.pool, st.tables), copy):
                    t.copy_(c)
                for t, c in zip(st.caches.caches, pages):
                    t.copy_(c)
                torch.cuda.synchronize()
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g, stream=stream):
                    st.verify(18, stream)
                    st.fork(source, stream)
                for _ in range(2):
                    g.replay()
        else:
            for _ in range(2):
                st.verify(18, stream)
                st.fork(source, stream)
        torch.cuda.synchronize()
        assert Y.status() == 0
        return [t.clone() for t in (st.text, st.said, st.lens, st.free, st.tlogits[:18], st.node_logprob[:18])]

    eager = run(None)
    for kind in ("stream", "graph"):
        for a, b in zip(eager, run(kind)):
            assert torch.equal(a, b), kind
    assert np.isfinite(eager[4].cpu().numpy()).all()


def test_a_fork_of_a_request_that_is_not_there_ends(cuda):
    import torch
    import yskn_b200 as Y
    st = _started(cuda, [3, 19, 14])
    st.fork(torch.tensor([1, 3, 2 ** 31 - 1], dtype=torch.int32, device=cuda))
    torch.cuda.synchronize()
    assert Y.status() == Y.EINVAL and Y.status() == 0
    assert st.lens.tolist() == [94, 0, 0] and st.said.tolist() == [20, 0, 0] and st.free.item() == 40 - 5 - 2
    st.new.copy_(torch.tensor([1, 0, 0], dtype=torch.int32))
    st.step(3, 1)
    assert st.lens.tolist() == [95, 0, 0] and st.said.tolist() == [21, 0, 0] and Y.status() == 0


def test_calls_that_do_not_fit_the_loop(cuda):
    import yskn_b200 as Y
    st = _started(cuda, [3, 5])
    for request in (-1, 2):
        with pytest.raises(Y.YsknError):
            st.draft(request, [1], [0])
    for n in (0, 97):
        with pytest.raises(Y.YsknError):
            st.verify(n)
    with pytest.raises(Y.YsknError):
        _stack(cuda, batch=1, max_tokens=4, capacity=16, n_blocks=4).verify(1)


def test_a_tree_of_more_nodes_than_the_loop_has_is_an_error(cuda):
    import torch
    import yskn_b200 as Y
    st = _stack(cuda, batch=2, max_tokens=64, capacity=64, n_blocks=16, nodes=3)
    for i in range(2):
        st.say(i, _prompt(i, 5))
    st.new.copy_(st.said)
    st.step(10, 5)
    st.draft(1, [3, 4], [0, 0])
    st.new.copy_(torch.tensor([7, 3], dtype=torch.int32))
    st.verify(10)
    torch.cuda.synchronize()
    assert Y.status() == Y.EINVAL and Y.status() == 0
    assert 1 <= st.said[1].item() - 6 <= 3 and st.lens[1].item() == st.said[1].item() - 1
