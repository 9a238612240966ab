"""Verified trees of requests that are behind their text, at its end, or under controls (yskn_b200/batch.py): what the
loop one token at a time would have done, nothing lost.

Everything here is whole numbers held equal, but for the adjusted logits: the unadjusted ones have the same bits in a
second loop (same calls, same inputs), to which the formula is applied in 64 bits; the call rounds each of its four steps
once, and a quotient by the repetition, so that with u = 2^-24 the result is off by at most 4 u times the largest
intermediate value."""
import numpy as np
import pytest

from test_gpu_batch_tree import VOCAB, _choices, _prompt, _stack, _started

pytestmark = pytest.mark.gpu


def _i32(cuda, *a):
    import torch
    return torch.tensor(a, dtype=torch.int32, device=cuda)


def _pages(st, request):
    """All layers' rows of the request's own blocks, as long as its length says."""
    import torch
    own = max(st.lens[request].item() - st.prefix_len, 0)
    blocks = st.tables[request, :-(-own // st.block_size)].long()
    return [c[blocks].reshape(-1, *c.shape[2:])[:own].clone() for c in st.caches.caches] + [torch.tensor(own)]


def test_a_fork_that_the_pool_does_not_hold_waits_in_verify(cuda):
    """Its copy has no rows (length 0) and its whole text: the last token alone, at the text's beginning, is no answer."""
    import torch
    import yskn_b200 as Y
    from test_gpu_batch_tree import _prefix
    st = _stack(cuda, batch=3, max_tokens=64, capacity=48, n_blocks=5, nodes=4)
    st.fill_prefix(_prefix(cuda, 16))
    st.say(0, _prompt(0, 20))
    st.say(2, _prompt(2, 3))
    st.new.copy_(st.said)
    st.step(23, 20)
    assert st.free.item() == 1  # too few for the copy, enough for a token or two
    st.fork(_i32(cuda, 0, 0, 2))
    assert st.lens.tolist() == [36, 0, 19] and st.said.tolist() == [21, 21, 4]
    text = st.text.clone()
    for i in range(3):
        st.draft(i, [5, 6], [0, 1])
    st.new.copy_(_i32(cuda, 3, 3, 3))
    st.verify(9)
    acc = st.accepted.tolist()
    assert Y.status() == 0 and acc[1] == 0 and min(acc[0], acc[2]) >= 1
    assert st.lens.tolist() == [36 + acc[0], 0, 19 + acc[2]] and st.said.tolist() == [21 + acc[0], 21, 4 + acc[2]]
    assert torch.equal(st.text[1], text[1]) and st.free.item() == 1


@pytest.mark.parametrize("P", [0, 75])
def test_requests_that_are_behind_their_text_wait(cuda, P):
    """Nothing run, some of a prompt run, nothing said, all run: none of them has one token left; the one that has goes
    on, and an ending one ends."""
    import torch
    import yskn_b200 as Y
    st = _started(cuda, [3, 19, 14, 5, 7, 2], P)
    st.say(0, _prompt(9, 12))      # a longer prompt: 3 of 12 run
    st.said[1] = 19                # all run
    st.new.copy_(_i32(cuda, 0, 0, -1, 0, 0, -1))
    st.step(6, 1)                  # requests 2 and 5 end
    st.say(2, _prompt(8, 10))      # nothing run
    st.said[5] = 0                 # nothing said
    text, said, lens, free = st.text.clone(), st.said.tolist(), st.lens.tolist(), st.free.item()
    pages = [_pages(st, i) for i in (0, 1, 3)]
    for i in range(6):
        st.draft(i, [5, 6], [0, 0])
    st.new.copy_(_i32(cuda, 3, 3, 1, 3, -1, 3))
    st.verify(18)
    acc = st.accepted.tolist()
    assert Y.status() == 0 and acc[:3] == [0, 0, 0] and acc[3] >= 1 and acc[4:] == [0, 0]
    said[3] += acc[3]
    own = [P + n if n else 0 for n in (3, 19, 0, 5 + acc[3], 0, 0)]
    assert st.said.tolist() == said and st.lens.tolist() == own
    assert all(torch.equal(st.text[i], text[i]) for i in (0, 1, 2, 4, 5))
    assert torch.equal(st.text[3, :6], text[3, :6])
    for i, before in zip((0, 1), pages):
        assert all(torch.equal(a, b) for a, b in zip(before, _pages(st, i)))
    assert all(torch.equal(a[:5], b[:5]) for a, b in zip(pages[2][:-1], _pages(st, 3)[:-1]))
    held = lambda n: -(-n // 16)  # noqa: E731
    assert st.free.item() == free + held(7) - held(5 + acc[3]) + held(5)
    # and those behind are served by step, which runs what they said
    st.new.copy_(_i32(cuda, 9, 0, 10, 0, 0, 0))
    st.step(19, 10)
    assert Y.status() == 0 and st.said.tolist()[:3] == [13, 19, 11] and st.lens.tolist()[:3] == [P + 12, P + 19, P + 10]


def test_a_captured_fork_and_verify_keep_a_request_that_did_not_fit(cuda):
    """Nobody on the host sees the length between the two."""
    import torch
    import yskn_b200 as Y
    got = []
    for captured in (False, True):
        st = _stack(cuda, batch=2, max_tokens=64, capacity=48, n_blocks=5, nodes=4)
        st.say(0, _prompt(0, 40))
        st.new.copy_(_i32(cuda, 40, 0))
        st.step(40, 40)
        st.draft(0, [5, 6], [0, 1])
        st.draft(1, [5, 6], [0, 1])
        st.new.fill_(3)
        source, stream = _i32(cuda, 0, 0), torch.cuda.Stream(cuda)
        torch.cuda.synchronize()
        if captured:
            warm = _stack(cuda, batch=2, max_tokens=64, capacity=48, n_blocks=5, nodes=4)
            warm.say(0, [1])
            warm.new.fill_(1)
            warm.step(2, 1)
            warm.fork(source, stream)
            warm.verify(6, stream)
            torch.cuda.synchronize()
            assert Y.status() == 0
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                st.fork(source, stream)
                st.verify(6, stream)
            g.replay()
        else:
            st.fork(source, stream)
            st.verify(6, stream)
        torch.cuda.synchronize()
        assert Y.status() == 0
        assert st.lens[1].item() == 0 and st.said[1].item() == 41 and st.accepted[1].item() == 0
        assert torch.equal(st.text[1, :41], st.text[0, :41]) and not bool(st.text[1, 41:].any())
        got.append([st.text.clone(), st.said.clone(), st.lens.clone(), st.free.clone()])
    assert all(torch.equal(a, b) for a, b in zip(*got))


@pytest.mark.parametrize("capacity,said", [(20, 18), (20, 19), (20, 20), (20, 14), (33, 30), (31, 29)])
def test_paths_end_where_the_text_does(cuda, capacity, said, monkeypatch):
    """A chain of 7 right drafts near the end of a text whose last block has more rows than it has tokens."""
    import yskn_b200 as Y
    st = _stack(cuda, batch=2, max_tokens=64, capacity=capacity, n_blocks=12, nodes=8)
    rows = 16 * -(-capacity // 16)
    st.say(0, _prompt(0, said - 1))
    st.say(1, _prompt(1, 3))
    st.new.copy_(st.said)
    st.step(said + 2, said - 1)
    assert st.said.tolist() == [said, 4]
    n = min(8, rows - said + 1)  # what the table holds
    chain = [100 + j for j in range(n - 1)]
    st.draft(0, chain, list(range(n - 1)))
    st.draft(1, [100, 101], [0, 1])
    st.new.copy_(_i32(cuda, n, 3))
    # the model's choice after node j is node j + 1's token; after the last one 777
    _choices(monkeypatch, {**{j: t for j, t in enumerate(chain + [777])}, n: 100, n + 1: 101, n + 2: 55})
    st.verify(n + 3)
    monkeypatch.undo()
    took = min(n, capacity - said + 1)  # rows up to the text's last token
    text = _prompt(0, said - 1) + st.text[0, said - 1:said].tolist() + chain + [777]
    assert Y.status() == 0
    assert st.accepted.tolist() == [took, 3]
    assert st.path[0].tolist() == list(range(took)) + [-1] * (8 - took)
    assert st.next[0].item() == (chain + [777])[took - 1]
    assert st.said.tolist() == [min(said + took, capacity), 7] and st.lens.tolist() == [said - 1 + took, 6]
    assert st.text[0, :st.said[0].item()].tolist() == text[:min(said + took, capacity)]
    assert st.text[1, 4:7].tolist() == [100, 101, 55]
    assert st.free.item() == 12 - -(-(said - 1 + took) // 16) - 1
    # the text full: verify leaves it alone from here on
    before = st.text.clone()
    for _ in range(3):
        lens = st.lens[0].item()
        st.new.copy_(_i32(cuda, 1, 0))
        st.verify(1)
        assert Y.status() == 0 and st.said[0].item() <= capacity and st.lens[0].item() <= capacity
        if lens == capacity:
            assert st.accepted.tolist() == [0, 0] and st.lens[0].item() == capacity
            assert (st.text[0] == before[0]).all()


def _controls(st, cuda, seed):
    """A penalty or two for each request, and masks that allow half the tokens (all of request 2's)."""
    import torch
    rng = np.random.default_rng(seed)
    B = st.batch
    st.repetition.copy_(torch.tensor([1.0, 1.7, 1.3, 0.8][:B]))
    st.presence.copy_(torch.tensor([0.0, 0.5, -0.25, 1.5][:B]))
    st.frequency.copy_(torch.tensor([0.0, 0.25, 0.75, -0.5][:B]))
    mask = rng.integers(0, 2 ** 32, (B, VOCAB // 32), dtype=np.uint32)
    if B > 2:
        mask[2] = 0xffffffff
    st.mask.copy_(torch.from_numpy(mask.view(np.int32)))
    return (mask[:, np.arange(VOCAB) // 32] >> (np.arange(VOCAB) % 32).astype(np.uint32)) & 1 == 1


@pytest.mark.parametrize("P", [0, 75])
def test_controls_of_every_node(cuda, P):
    """Each node's logits under its request's controls, by the request's text and what the node's ancestors say (its own
    token among them; often one that the text has, or an ancestor)."""
    import torch
    import yskn_b200 as Y
    sizes = [3, 19, 14, 5]
    trees = [([7, 7, 9], [0, 1, 1]), (_prompt(1, 6) + [7, 7], [0, 0, 1, 3, 4, 4, 6, 7]), ([], []),
             ([50, 50, 50, 51], [0, 1, 2, 3])]
    T = sum(1 + len(t) for t, _ in trees)
    loops = []
    for controlled in (False, True):
        st = _started(cuda, sizes, P)
        for i, (tokens, parents) in enumerate(trees):
            st.draft(i, tokens, parents)
            st.new[i] = 1 + len(tokens)
        allowed = _controls(st, cuda, 3) if controlled else None
        text = [st.text[i, :st.said[i].item()].tolist() for i in range(4)]
        st.verify(T + 2)  # and two places that hold no token
        assert Y.status() == 0
        loops.append((st, text))
    (plain, text), (st, _) = loops
    raw, got, t = plain.tlogits[:T].double().cpu().numpy(), st.tlogits[:T].cpu().numpy(), 0
    u = 2.0 ** -24
    for i, (tokens, parents) in enumerate(trees):
        said = [[]]
        for tok, p in zip(tokens, parents):
            said.append(said[p] + [tok])
        r, pres, freq = (x[i].item() for x in (st.repetition, st.presence, st.frequency))
        for path in said:
            history, x = text[i] + path, raw[t].copy()
            seen, count = np.zeros(VOCAB, bool), np.zeros(VOCAB)
            seen[history] = True
            np.add.at(count, history[sizes[i]:], 1)  # behind the prompt
            x = np.where(seen, np.where(x > 0, x / r, x * r), x)
            most = np.maximum(np.abs(raw[t]), np.abs(x))
            x = x - freq * count
            most = np.maximum(most, np.abs(freq * count) + np.abs(x))
            x = x - np.where(count > 0, pres, 0.0)
            most = np.maximum(most, np.abs(x) + abs(pres))
            assert np.array_equal(np.isneginf(got[t]), ~allowed[i]), (i, path)
            ok = allowed[i]
            assert (np.abs(got[t][ok] - x[ok]) <= 4 * u * most[ok]).all(), (i, path)
            assert st.choice[t].item() == int(got[t].argmax())  # of the adjusted ones, the first of equal ones
            t += 1
    for i in range(4):  # no token that the mask forbids has been said
        assert all(allowed[i][tok] for tok in st.text[i, sizes[i] + 1:st.said[i].item()].tolist())


@pytest.mark.parametrize("seed", [1, 2])
def test_one_node_alone_is_a_step_under_controls(cuda, seed):
    """Without drafts: the choice of verify is that of step, whose penalties and masks it has."""
    import yskn_b200 as Y
    sizes, P = [3, 19, 14, 5], 75
    one, st = _started(cuda, sizes, P, logprobs=3), _started(cuda, sizes, P, logprobs=3)
    for s in (one, st):
        allowed = _controls(s, cuda, seed)
        s.new.fill_(1)
    one.step(4, 1)
    st.verify(4)
    assert Y.status() == 0 and st.accepted.tolist() == [1] * 4
    a, b = one.blogits.cpu().numpy(), st.tlogits[:4].cpu().numpy()
    assert np.array_equal(np.isneginf(a), np.isneginf(b)) and np.array_equal(np.isneginf(a), ~allowed)
    for i in range(4):
        ok, chose = allowed[i], int(b[i].argmax())
        off = 2 * np.abs(a[i][ok] - b[i][ok]).max()  # the two orders of sums
        assert off < 1.0 and a[i].max() - a[i][chose] <= off and st.next[i].item() == chose
        assert st.text[i, sizes[i] + 1].item() == chose and ok[chose]
    # the log probability is that of the adjusted logits, as in step
    lse = np.log(np.exp(b.astype(np.float64)).sum(1))
    want = b[np.arange(4), st.choice[:4].tolist()] - lse
    assert np.abs(st.node_logprob[:4, 0].cpu().numpy() - want).max() <= 1e-5
