"""The serving loop over the batch operators (yskn_b200/batch.py): two attention layers, a
4096-row head, requests behind a shared prefix against each request alone, whose own text
then begins with the prefix.

Tolerance of the logits, as the L2 norm of the difference over that of the logits. The two ways
sum an attention row in a different order, so a value rounded to bf16 may fall on the neighbouring
one: at most 2^-8 of it. Each layer rounds at most nine times what depends on it (attention output,
residual twice, gate, up, silu, product, and the new rows of K and V of the layer after it), the
last norm's residual once: 20 neighbours in all for two layers, each counted in full: 20 * 2^-8. A
request that misses the prefix or another request's row in its place differs by more than 1/2."""
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


def test_shared_prefix_equals_requests_alone(cuda):
    import torch
    import yskn_b200 as Y
    P, sizes = 75, [1, 19, 33, 6]
    st = _stack(cuda, batch=4, max_tokens=64, capacity=48, n_blocks=24)
    prefix = _prefix(cuda, P)
    st.fill_prefix(prefix)  # in two parts
    for i, n in enumerate(sizes):
        st.say(i, _prompt(i, n))
    st.new.copy_(st.said)
    st.step(64, max(sizes))
    first = st.blogits.clone()
    assert st.said.tolist() == [n + 1 for n in sizes]
    assert st.lens.tolist() == [P + n for n in sizes]
    st.new.fill_(1)
    st.step(4, 1)
    assert Y.status() == 0
    text = st.text.tolist()
    assert all(0 <= t < VOCAB for i, n in enumerate(sizes) for t in text[i][:n + 2])

    alone = _stack(cuda, batch=1, max_tokens=128, capacity=160, n_blocks=10)
    for i, n in enumerate(sizes):
        whole = prefix.tolist() + text[i][:n]
        for row, said in ((first[i], whole), (st.blogits[i], whole + text[i][n:n + 1])):
            alone.say(0, said)
            alone.new.fill_(len(said))
            alone.step(len(said), len(said))
            assert _close(row, alone.blogits[0]) <= TOL, (i, len(said))
            alone.new.fill_(-1)  # ends it: its blocks go back
            alone.step(1, 1)
            assert alone.lens.tolist() == [0] and alone.free.tolist() == [10]
    # without the prefix the answer is another one
    alone.say(0, text[0][:1])
    alone.new.fill_(1)
    alone.step(1, 1)
    assert _close(first[0], alone.blogits[0]) > 0.5


def test_waiting_ending_and_controls(cuda):
    import torch
    import yskn_b200 as Y
    # blocks for the prefix (2) and for two of the three requests (2 each)
    st = _stack(cuda, batch=3, max_tokens=64, capacity=32, n_blocks=6)
    st.fill_prefix(_prefix(cuda, 32))
    for i in range(3):
        st.say(i, _prompt(i, 20))
    st.mask[1].zero_()
    st.mask[1, 3] = 1 << 9  # only token 105
    st.new.copy_(st.said)
    st.step(60, 20)
    assert st.lens.tolist() == [52, 52, 0] and st.free.tolist() == [0]
    assert st.said.tolist() == [21, 21, 20]
    assert st.text[1, 20].item() == 3 * 32 + 9
    st.new.copy_(torch.tensor([-1, 1, 20], dtype=torch.int32))
    st.step(60, 20)  # the first ends; the third takes its blocks
    assert st.lens.tolist() == [0, 53, 52] and st.free.tolist() == [0]
    assert st.said.tolist() == [21, 22, 21]
    assert Y.status() == 0


def test_graph_equals_eager(cuda):
    import torch
    import yskn_b200 as Y

    def run(use_graph):
        st = _stack(cuda, batch=5, max_tokens=64, capacity=32, n_blocks=24)
        stream = torch.cuda.Stream(cuda)
        with torch.cuda.stream(stream):
            st.fill_prefix(_prefix(cuda, 70), stream)
            for i in range(5):
                st.say(i, _prompt(i, 3 + i))
            st.presence.fill_(0.25)
            st.new.copy_(st.said)
            st.step(25, 7, stream)
            st.new.fill_(1)
            st.step(5, 1, stream)
            torch.cuda.synchronize()
            if use_graph:
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=stream):
                    st.step(5, 1, stream)
                step = graph.replay
            else:
                step = lambda: st.step(5, 1, stream)  # noqa: E731
            for _ in range(14):  # past a block's end for each request
                step()
            torch.cuda.synchronize()
        assert Y.status(stream) == 0
        return st.text.clone(), st.lens.clone(), st.blogits.clone()

    for a, b in zip(run(False), run(True)):
        assert torch.equal(a, b)


def test_a_stream_that_is_not_the_current_one(cuda):
    """All of a step runs on the stream it is given: the same steps, held up there, give the same."""
    import torch
    import yskn_b200 as Y

    def run(stream):
        st = _stack(cuda, batch=5, max_tokens=64, capacity=32, n_blocks=24)
        here = torch.cuda.current_stream(cuda)

        def late():
            if stream is not None:  # after the inputs, and well after what the current stream does next
                stream.wait_stream(here)
                with torch.cuda.stream(stream):
                    torch.cuda._sleep(4000000)

        prefix = _prefix(cuda, 70)
        late()
        st.fill_prefix(prefix, stream)
        if stream is not None:
            here.wait_stream(stream)
        for i in range(5):
            st.say(i, _prompt(i, 3 + i))
        st.presence.fill_(0.25)
        st.new.copy_(st.said)
        late()
        st.step(25, 7, stream)
        if stream is not None:
            here.wait_stream(stream)
        st.new.fill_(1)
        for _ in range(6):
            late()
            st.step(5, 1, stream)
        torch.cuda.synchronize()
        assert Y.status() == 0
        return st.text.clone(), st.lens.clone(), st.said.clone(), st.blogits.clone()

    for a, b in zip(run(None), run(torch.cuda.Stream(cuda))):
        assert torch.equal(a, b)


@pytest.mark.parametrize("max_tokens", [2, 5, 16])
def test_small_steps_of_a_small_loop(cuda, max_tokens):
    """A step of one token for each request in a loop made for few tokens a step."""
    import yskn_b200 as Y
    st = _stack(cuda, batch=2, max_tokens=max_tokens, capacity=32, n_blocks=12)
    st.fill_prefix(_prefix(cuda, 21))
    for i in range(2):
        st.say(i, _prompt(i, 1))
    for n in range(3):
        st.new.fill_(1)
        st.step(2, 1)
        assert st.lens.tolist() == [22 + n] * 2 and st.said.tolist() == [2 + n] * 2
    assert Y.status() == 0


def test_a_prefix_larger_than_the_pool_is_refused(cuda):
    import yskn_b200 as Y
    st = _stack(cuda, batch=2, max_tokens=64, capacity=32, n_blocks=4)
    with pytest.raises(Y.YsknError) as e:
        st.fill_prefix(_prefix(cuda, 65))
    assert e.value.code == Y.EINVAL and st.prefix_len == 0 and st.free.tolist() == [4]
    st.fill_prefix(_prefix(cuda, 64))
    assert st.prefix_len == 64 and st.free.tolist() == [0] and Y.status() == 0
