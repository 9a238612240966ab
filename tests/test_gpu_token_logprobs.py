"""Log probabilities, entropy and most likely tokens (yskn_b200_token_logprobs) against 64-bit sums.

Tolerance. With M the largest logit, d = x - M (rounded: 2^-24 |d|), w = exp(d): the product with log2 e and the
hardware exponential leave a relative error of at most h = 2^-23 |d| + 2^-22 in a weight, so that R = sum w (all but one
maximum) is off by at most sum h w + a R, a = 2^-23 times the longest chain of additions n (a lane's share of the row
and the joins; V / 256 + 64), and log1p(R) by that over 1 + R, and its own 2^-22 of the result. A log probability adds
the rounding of d and of one subtraction. The entropy log1p(R) - E / (1 + R), E = sum w d, likewise:
E off by sum (h + 2^-23) w |d| + a |E|, the quotient by 2^-22 of itself and its part of R's error."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def expected(x, ids):
    """x float64 [V] (finite or -inf, something above -inf): (log p, its bound, entropy, its bound)."""
    top = x.max()
    first = int(x.argmax())
    d = x - top
    fin = np.where(np.isinf(d), 0.0, d)
    w = np.exp(d)
    w[first] = 0.0
    R, E = w.sum(), (w * fin).sum()
    h = 2.0 ** -23 * -fin + 2.0 ** -22
    a = 2.0 ** -23 * (len(x) / 256 + 64)
    dR = (h * w).sum() + a * R
    L = np.log1p(R)
    dL = dR / (1 + R) + 2.0 ** -22 * L + 1e-44
    H = L - E / (1 + R)
    dE = ((h + 2.0 ** -23) * w * -fin).sum() + a * -E
    dH = dL + dE / (1 + R) + -E / (1 + R) * (dR / (1 + R) + 2.0 ** -22) + 2.0 ** -24 * H
    lp = d[ids] - L
    tol = dL + 2.0 ** -24 * -fin[ids] + 2.0 ** -23 * np.where(np.isinf(lp), 0.0, -lp)
    return lp, tol, H, dH


def order(x, k):
    """The k largest above -inf, equal ones by number."""
    by = np.lexsort((np.arange(len(x)), -(x + 0.0)))
    return [int(i) for i in by[:k] if x[i] > -np.inf]


def call(cuda, x, tokens=None, k=0, entropy=True, stride=None, offset=0, stream=None):
    """x float32 numpy [M][V], in rows of `stride` logits that begin `offset` logits behind 16 bytes."""
    import torch
    import yskn_b200 as Y
    M, V = x.shape
    stride = V if stride is None else stride
    flat = torch.full((M * stride + offset + 8,), float("nan"), device=cuda)
    view = flat[offset:offset + M * stride].view(M, stride)[:, :V]
    view.copy_(torch.from_numpy(x))
    f = lambda *s: torch.full(s, 7.0, device=cuda)  # noqa: E731
    t = None if tokens is None else torch.from_numpy(np.asarray(tokens, np.int32)).to(cuda)
    lp = None if t is None else f(*t.shape)
    H = f(M) if entropy else None
    tops, ids = (f(M, k), torch.full((M, k), 7, dtype=torch.int32, device=cuda)) if k else (None, None)
    torch.cuda.synchronize()
    Y.token_logprobs(view, t, lp, H, tops, ids, stream=stream)
    torch.cuda.synchronize()
    assert Y.status() == 0
    return [None if o is None else o.cpu().numpy() for o in (lp, H, tops, ids)]


def check(cuda, x, tokens, k, **kw):
    lp, H, tops, ids = call(cuda, x, tokens, k, **kw)
    for m in range(len(x)):
        row = x[m].astype(np.float64)
        want, tol, h, dh = expected(row, np.asarray(tokens[m]))
        both = np.isinf(want) & np.isinf(lp[m])
        assert (both | (np.abs(lp[m] - want) <= tol)).all(), (m, lp[m], want, tol)
        assert abs(H[m] - h) <= dh, (m, H[m], h, dh)
        best = order(x[m], k)
        assert ids[m].tolist() == best + [-1] * (k - len(best)), m
        want, tol, _, _ = expected(row, np.asarray(best, int))
        assert (np.abs(tops[m, :len(best)] - want) <= tol).all() and (tops[m, len(best):] == -np.inf).all()


def rows(seed, M, V, scale=3.0):
    return (np.random.default_rng(seed).standard_normal((M, V)) * scale).astype(np.float32)


@pytest.mark.parametrize("V", [1, 2, 3, 5, 31, 33, 1023, 1024, 1025, 4099, 8191, 50257, 151936])
@pytest.mark.parametrize("M", [1, 3, 40])
def test_sizes(cuda, V, M):
    x = rows(V + M, M, V)
    tokens = np.random.default_rng(V).integers(0, V, (M, 5))
    tokens[:, 0] = x.argmax(1)
    check(cuda, x, tokens, min(20, 32))


@pytest.mark.parametrize("M", [80, 150, 320, 700])
def test_many_rows(cuda, M):
    x = rows(M, M, 20011)
    check(cuda, x, x.argmax(1)[:, None], 8)


@pytest.mark.parametrize("offset", [0, 1, 2, 3])
@pytest.mark.parametrize("V,stride", [(5, 5), (5, 9), (1021, 1022), (20001, 20003)])
def test_rows_at_any_boundary_between_numbers_that_are_not_theirs(cuda, offset, V, stride):
    x = rows(V + offset, 3, V)
    check(cuda, x, [[0, V - 1]] * 3, 4, offset=offset, stride=stride)


@pytest.mark.parametrize("k", [1, 2, 7, 31, 32])
def test_ties_go_to_the_lowest_number(cuda, k):
    rng = np.random.default_rng(k)
    x = np.stack([np.zeros(9000, np.float32), rng.integers(-2, 2, 9000).astype(np.float32),
                  np.repeat(rows(k, 1, 90)[0], 100)])
    x[1, ::7] = -0.0
    check(cuda, x, [[3], [5], [8999]], k)


def test_orders_that_fill_the_lists(cuda):
    """Ever larger logits, ever smaller ones, and the largest in one lane's places."""
    up = np.linspace(-20, 20, 70000, dtype=np.float32)
    lane = rows(3, 1, 70000)[0]
    lane[5 * 128:6 * 128] += 40
    lane[7::128] += 30
    check(cuda, np.stack([up, up[::-1], lane]), [[0, 69999]] * 3, 32)


def test_sure_rows_keep_their_small_numbers(cuda):
    x = rows(1, 4, 30000, 0.5)
    for m, gap in enumerate((18.0, 25.0, 60.0, 200.0)):
        x[m, 777 * (m + 1)] = gap
    lp, H, _, _ = call(cuda, x, [[777 * (m + 1)] for m in range(4)])
    for m in range(4):
        want, tol, h, dh = expected(x[m].astype(np.float64), np.array([777 * (m + 1)]))
        assert want[0] < 0 and abs(lp[m, 0] - want[0]) <= max(tol[0], 2.0 ** -126) and tol[0] < 1e-3 * -want[0] + 2e-38
        assert abs(H[m] - h) <= max(dh, 2.0 ** -126)


def test_masked_rows(cuda):
    x = rows(5, 6, 10007)
    x[0, 1:] = -np.inf           # one token left
    x[1, :9000] = -np.inf
    x[2, ::2] = -np.inf
    x[3, :] = np.finfo(np.float32).min  # the type's lowest value, throughout
    x[4, 5:] = np.finfo(np.float32).min
    x[5] = -np.inf
    x[5, 10006] = np.finfo(np.float32).min
    check(cuda, x, [[0, 1], [9000, 2], [1, 0], [9, 8], [4, 7], [10006, 1]], 6)


def test_rows_without_a_distribution(cuda):
    x = rows(6, 5, 9001)
    x[0] = -np.inf
    x[1, 8000] = np.nan
    x[2, 17] = np.inf
    x[3] = np.nan
    x[4, ::3] = np.inf
    lp, H, tops, ids = call(cuda, x, [[5, 17]] * 5, 3)
    assert (lp[0] == -np.inf).all() and H[0] == 0 and (tops[0] == -np.inf).all()
    for o in (lp, H, tops):
        assert np.isnan(o[1:]).all()
    assert (ids == -1).all()
    for V in (1, 3, 100):  # the same in a few logits
        lp, H, tops, ids = call(cuda, np.full((1, V), np.nan, np.float32), [[0]], 1)
        assert np.isnan(lp).all() and np.isnan(H).all() and np.isnan(tops).all() and (ids == -1).all()


def test_extreme_finite_logits(cuda):
    big = np.finfo(np.float32).max
    x = np.zeros((2, 5000), np.float32)
    x[0, 9], x[0, 10] = big, -big
    x[1] = -big
    x[1, 4999] = big
    lp, H, tops, ids = call(cuda, x, [[9, 0], [4999, 0]], 2)
    assert lp[0, 0] == 0 and lp[1, 0] == 0 and H[0] == 0 and H[1] == 0
    assert lp[0, 1] == -big and lp[1, 1] == -np.inf  # -2 big passes the type
    assert ids.tolist() == [[9, 0], [4999, 0]]


def test_padding_and_what_is_left_out(cuda):
    import torch
    import yskn_b200 as Y
    x = rows(7, 3, 4000)
    lp, H, tops, ids = call(cuda, x, [[-1, 4000, 2 ** 31 - 1, 5]] * 3, 0, entropy=False)
    assert (lp[:, :3] == -np.inf).all() and np.isfinite(lp[:, 3]).all() and H is None and ids is None
    assert np.isfinite(call(cuda, x)[1]).all()
    d = torch.from_numpy(x).to(cuda)
    wide = torch.arange(12, dtype=torch.int32, device=cuda).view(3, 4)
    out = torch.empty(3, 2, device=cuda)
    Y.token_logprobs(d, wide[:, 1:3], out)  # rows of tokens with a stride
    assert np.array_equal(out.cpu().numpy(), call(cuda, x, wide[:, 1:3].cpu().numpy())[0])


def test_same_bits_each_time_on_another_stream_and_in_a_graph(cuda):
    import torch
    import yskn_b200 as Y
    x = torch.from_numpy(rows(8, 9, 151936)).to(cuda)
    t = x.argmax(1, keepdim=True).to(torch.int32)
    z = lambda *s: torch.zeros(s, device=cuda)  # noqa: E731
    outs = lambda: [z(9, 1), z(9), z(9, 20), z(9, 20).int()]  # noqa: E731
    a, b, c = outs(), outs(), outs()
    Y.token_logprobs(x, t, *a)
    side = torch.cuda.Stream(cuda)
    side.wait_stream(torch.cuda.current_stream())
    Y.token_logprobs(x, t, *b, stream=side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        Y.token_logprobs(x, t, *c)
    g.replay()
    torch.cuda.synchronize()
    for p, q, r in zip(a, b, c):
        assert torch.equal(p, q) and torch.equal(p, r)
    assert (a[3][:, 0] == t[:, 0]).all()


@pytest.mark.parametrize("k", [1, 8, 20, 23, 24, 25])
def test_largest_in_few_places(cuda, k):
    """Both bounds where they hold off least: the largest in one lane's places, in eight lanes', in one warp's run, at
    the row's ends, few logits above -inf, and rows of two numbers; in one part and in several."""
    rng = np.random.default_rng(k)
    for V, M in ((50257, 6), (151936, 6), (9001, 300)):
        x = rows(k, M, V)
        x[0, 4 * 17::1024] += 30
        x[1, (np.arange(V) // 4 % 32) < 8] += 25
        x[2, V // 3:V // 3 + 900] += 25
        x[3, :7] += 40
        x[3, -9:] += 40
        keep = rng.choice(V, k + 1, replace=False)
        x[4] = np.where(np.isin(np.arange(V), keep), x[4], -np.inf)
        x[5] = np.where(rng.random(V) < 0.3, np.float32(2.5), np.float32(-1.0))
        if M > 6:
            x[6:] = np.sort(x[6:], axis=1)
        check(cuda, x[:7] if M > 6 else x, [[0, V - 1]] * min(M, 7), k)
        if M > 6:  # one CTA a row, and all rows' numbers
            _, _, _, ids = call(cuda, x, [[0]] * M, k)
            assert [i.tolist() for i in ids] == [order(r.astype(np.float64), k) for r in x]
