"""Blocks, slots and positions of a batch's step (yskn_b200_batch_plan) against a
one-request-at-a-time restatement in Python integers: all outputs equal, arrays that the call
does not own unchanged."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def restated(lens, new, tables, pool, free, bs, P, T):
    """The rules of the call, one request after another."""
    tables, pool = tables.copy(), list(pool)
    B, width = tables.shape
    stack = pool[:free]
    held = [-(-max(int(n) - P, 0) // bs) for n in lens]
    for i in range(B):
        if new[i] < 0:
            stack += [int(b) for b in tables[i, :held[i]]]
    have, tokens, waits = len(stack), 0, False
    lens_out, starts, slots, positions, requests = list(map(int, lens)), [0], [], [], []
    for i in range(B):
        rows, n = max(int(lens[i]) - P, 0), int(new[i])
        if n < 0:
            lens_out[i] = 0
        total = -(-(rows + max(n, 0)) // bs)
        if n > 0 and total <= width:
            fresh = total - held[i]
            waits = waits or fresh > len(stack) or tokens + n > T
            if not waits:
                for b in range(held[i], total):
                    tables[i, b] = stack.pop()
                for t in range(rows, rows + n):
                    slots.append(int(tables[i, t // bs]) * bs + t % bs)
                    positions.append(P + t)
                    requests.append(i)
                tokens += n
                lens_out[i] = max(int(lens[i]), P) + n
        starts.append(tokens)
    pad = [-1] * (T - tokens)
    for v in range(free, len(stack)):  # what came back and was not taken
        pool[v] = stack[v]
    return lens_out, len(stack), starts, slots + pad, positions + pad, requests + pad, tables, pool


def case(rng, B, max_new, max_rows, bs, P, ended, room, T=None, spare=0, idle=0.1):
    rows = rng.integers(0, max_rows + 1, B)
    new = rng.integers(1, max_new + 1, B)
    new[rng.random(B) < idle] = 0
    new[rng.random(B) < ended] = -1
    lens = np.where(rows > 0, P + rows, np.where(rng.random(B) < 0.5, 0, P))
    held = -(-rows // bs)
    total = -(-(rows + np.maximum(new, 0)) // bs)
    width = int(max(1, total.max())) + spare
    need = int((total - held).sum())
    free = max(0, int(need * room))
    numbers = rng.permutation(int(held.sum()) + free + 3)
    tables = np.full((B, width), -7, np.int32)
    at = 0
    for i in range(B):
        tables[i, :held[i]] = numbers[at:at + held[i]]
        at += held[i]
    pool = np.full(int(held.sum()) + free + 1, -9, np.int32)
    pool[:free] = numbers[at:at + free]
    T = int(np.maximum(new, 0).sum()) + 3 if T is None else T
    return lens.astype(np.int32), new.astype(np.int32), tables, pool, free, bs, P, T


def run(cuda, c, stream=None):
    import torch
    import yskn_b200 as Y
    lens, new, tables, pool, free, bs, P, T = c
    t = lambda a: torch.from_numpy(np.array(a, np.int32)).to(cuda)  # noqa: E731
    wide = torch.full((len(lens), tables.shape[1] + 3), -5, dtype=torch.int32, device=cuda)  # rows with a stride
    view = wide[:, :tables.shape[1]]
    view.copy_(t(tables))
    d_pool, d_lens, d_free = t(pool), t(lens), t([free])
    i32 = lambda n: torch.full((n,), -77, dtype=torch.int32, device=cuda)  # noqa: E731
    out = [i32(len(lens)), i32(1), i32(len(lens) + 1), torch.full((T,), -77, dtype=torch.int64, device=cuda), i32(T),
           i32(T)]
    torch.cuda.synchronize()
    Y.batch_plan(d_lens, t(new), view, d_pool, d_free, bs, *out, prefix_len=P, stream=stream)
    torch.cuda.synchronize()
    assert Y.status() == 0
    got = [o.cpu().numpy() for o in out] + [view.cpu().numpy(), d_pool.cpu().numpy()]
    exp = restated(*c)
    for name, a, b in zip(("lens", "free", "starts", "slots", "positions", "requests", "tables", "pool"), got, exp):
        assert np.array_equal(a, np.array(b).reshape(a.shape)), name
    assert np.array_equal(d_lens.cpu().numpy(), lens) and int(d_free) == free
    assert bool((wide[:, tables.shape[1]:] == -5).all())
    return got


@pytest.mark.parametrize("B,max_new,max_rows,bs,P,ended,room", [
    (1, 1, 0, 16, 0, 0, 1), (1, 1, 40, 16, 100, 0, 1), (2, 1, 16, 16, 16, 0, 1), (33, 1, 64, 16, 31, 0.2, 1),
    (256, 1, 300, 64, 4096, 0.05, 1), (7, 700, 50, 128, 5, 0.3, 1), (512, 9, 100, 32, 0, 0.5, 0.4),
    (513, 40, 90, 16, 17, 0.1, 0.7), (4096, 30, 200, 16, 1000, 0.1, 0.9), (1000, 3, 20, 1, 9, 0.2, 0.8),
    (40, 50, 60, 7, 3, 0.2, 0.5)])
def test_plans(cuda, B, max_new, max_rows, bs, P, ended, room):
    run(cuda, case(np.random.default_rng(B + max_new), B, max_new, max_rows, bs, P, ended, room))


def test_step_too_small_for_all_tokens(cuda):
    run(cuda, case(np.random.default_rng(1), 64, 20, 100, 16, 8, 0.1, 1, T=211))
    run(cuda, case(np.random.default_rng(2), 64, 20, 100, 16, 8, 0.1, 1, T=1))
    run(cuda, case(np.random.default_rng(3), 64, 20, 100, 16, 8, 0.1, 1, T=0))


def test_request_too_long_for_its_table_waits_alone(cuda):
    c = list(case(np.random.default_rng(4), 20, 30, 100, 16, 8, 0, 1, idle=0))
    c[1][7] = 100000  # more than its table row holds: the others are served
    got = run(cuda, c)
    assert got[2][8] == got[2][7] and got[2][-1] > got[2][8]


def test_empty_pool_lives_on_what_ended_requests_give_back(cuda):
    c = list(case(np.random.default_rng(5), 200, 20, 100, 16, 8, 0.4, 0, idle=0))
    assert c[4] == 0
    assert run(cuda, c)[2][-1] > 0


def test_all_idle_and_all_ended(cuda):
    c = list(case(np.random.default_rng(6), 90, 3, 100, 16, 8, 0, 1, idle=0))
    c[1][:] = 0
    run(cuda, c)
    c[1][:] = -1
    run(cuda, c)


def test_other_stream_and_same_result_twice(cuda):
    import torch
    c = case(np.random.default_rng(7), 300, 50, 100, 16, 8, 0.2, 0.8)
    a, b = run(cuda, c), run(cuda, c, stream=torch.cuda.Stream())
    assert all(np.array_equal(x, y) for x, y in zip(a, b))


def test_steps_hand_every_block_to_one_place(cuda):
    """Forty steps with arrivals and ends: no block is held twice or lost."""
    import torch
    import yskn_b200 as Y
    rng = np.random.default_rng(8)
    B, bs, P, cap, width = 30, 16, 50, 200, 12
    i32 = lambda n, v=0: torch.full((n,), v, dtype=torch.int32, device=cuda)  # noqa: E731
    lens, lens2, free, free2 = i32(B), i32(B), i32(1, cap), i32(1)
    pool = torch.randperm(cap, device=cuda).to(torch.int32)
    tables, starts = torch.full((B, width), -1, dtype=torch.int32, device=cuda), i32(B + 1)
    T = 400
    slots, positions, requests = torch.empty(T, dtype=torch.int64, device=cuda), i32(T), i32(T)
    for step in range(40):
        new = rng.integers(0, 30, B).astype(np.int32)
        new[rng.random(B) < 0.2] = -1
        Y.batch_plan(lens, torch.from_numpy(new).to(cuda), tables, pool, free, bs, lens2, free2, starts, slots,
                     positions, requests, prefix_len=P)
        lens, lens2, free, free2 = lens2, lens, free2, free
        ln, nf = lens.cpu().numpy(), int(free)
        held = [int(b) for i in range(B) for b in tables[i, :-(-max(ln[i] - P, 0) // bs)].tolist()]
        assert sorted(held + pool[:nf].tolist()) == list(range(cap)), step
    assert Y.status() == 0


def test_lengths_past_the_table_are_reported(cuda):
    import torch
    import yskn_b200 as Y
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)  # noqa: E731
    out = [i32([0, 0]), i32([0]), i32([0, 0, 0]), torch.zeros(4, dtype=torch.int64, device=cuda), i32([0] * 4),
           i32([0] * 4)]
    Y.batch_plan(i32([100, 5]), i32([-1, 1]), i32([[1, 2], [3, 4]]), i32([7, 8, 9, 0]), i32([3]), 16, *out)
    assert Y.status() == Y.EINVAL
    assert Y.status() == 0
