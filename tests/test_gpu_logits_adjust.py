"""Penalties, biases and masks on logits (yskn_b200_logits_adjust) against the formula in 64 bits.

Tolerance: at most five binary32 roundings (quotient, product, two differences, one sum), each
of a value no larger than |x| max(r, 1 / r) + f c + p + |b|: 5 * 2^-24 of that sum."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def run(cuda, M=3, V=1000, L=50, n_bias=0, mask=False, pad=0, repeat_bias=False, prompts=True, penalties=True,
        in_place=False, seed=0, logits=None, stream=None, hot=None, lens=None):
    import torch
    import yskn_b200 as Y
    rng = np.random.default_rng(seed)
    x = (rng.standard_normal((M, V)) * 3).astype(np.float32) if logits is None else logits
    hist = rng.integers(-2, V + 3, (M, max(L, 1))).astype(np.int32)  # ids outside are padding
    if hot is not None:
        hist[:] = hot
    lens = rng.integers(0, L + 1, M).astype(np.int32) if lens is None else np.full(M, lens, np.int32)
    if M > 1:
        lens[0] = 0
    prompt = (lens * rng.random(M)).astype(np.int32)
    rep, pres, freq = (rng.uniform(*r, M).astype(np.float32) for r in ((0.7, 1.8), (-0.5, 1.0), (0.0, 0.7)))
    ids = bias = words = None
    if n_bias:
        ids = rng.integers(-1, V + 2, (M, n_bias)).astype(np.int32)
        if not repeat_bias:
            ids = np.stack([rng.permutation(V + 2)[:n_bias] - 1 for _ in range(M)]).astype(np.int32)
        bias = (rng.standard_normal((M, n_bias)) * 5).astype(np.float32)
    if mask:
        words = rng.integers(0, 2 ** 32, (M, -(-V // 32)), dtype=np.uint64).astype(np.uint32)
        words[M // 2] = 0  # a row that allows nothing
    dev = lambda a: None if a is None else torch.from_numpy(a).to(cuda)  # noqa: E731
    wide = torch.full((M, V + pad), 55.0, device=cuda)
    d_x = wide[:, :V]
    d_x.copy_(dev(x))
    out = d_x if in_place else torch.full((M, V + pad), 66.0, device=cuda)[:, :V]
    kw = dict(history=dev(hist), history_lens=dev(lens), prompt_lens=dev(prompt) if prompts else None,
              repetition=dev(rep), presence=dev(pres), frequency=dev(freq)) if penalties else {}
    torch.cuda.synchronize()
    Y.logits_adjust(d_x, out, bias_ids=dev(ids), bias=dev(bias),
                    mask=None if words is None else dev(words.view(np.int32)), stream=stream, **kw)
    torch.cuda.synchronize()
    assert Y.status() == 0
    got = out.cpu().numpy()
    exp, size = x.astype(np.float64), np.abs(x.astype(np.float64))
    for m in range(M):
        if penalties:
            h = hist[m, :lens[m]]
            inside = (h >= 0) & (h < V)
            seen = np.bincount(h[inside], minlength=V) > 0
            late = inside & (np.arange(lens[m]) >= (prompt[m] if prompts else 0))
            c = np.bincount(h[late], minlength=V)
            r = np.float64(rep[m])
            exp[m] = np.where(seen, np.where(exp[m] > 0, exp[m] / r, exp[m] * r), exp[m])
            exp[m] -= np.where(c > 0, c * np.float64(freq[m]) + np.float64(pres[m]), 0.0)
            size[m] = size[m] * max(r, 1 / r) + c * abs(np.float64(freq[m])) + abs(np.float64(pres[m]))
        if n_bias:
            last = {int(t): b for t, b in zip(ids[m], bias[m]) if 0 <= t < V}
            for t, b in last.items():
                exp[m, t] += np.float64(b)
                size[m, t] += abs(np.float64(b))
        if mask:
            t = np.arange(V)
            exp[m] = np.where((words[m, t >> 5] >> (t & 31).astype(np.uint32)) & 1, exp[m], -np.inf)
    same = (got == exp) | (np.isnan(got) & np.isnan(exp))
    with np.errstate(invalid="ignore"):
        assert np.all(same | (np.abs(got - exp) <= 5 * 2.0 ** -24 * size))
    if pad:
        assert bool((wide[:, V:] == 55.0).all())
    return out


@pytest.mark.parametrize("V", [1, 31, 32, 33, 1000, 1024, 1025, 50257, 151936])
@pytest.mark.parametrize("M", [1, 3])
def test_vocabularies(cuda, M, V):
    run(cuda, M=M, V=V, L=200, n_bias=min(V, 7), mask=True, seed=V + M)


@pytest.mark.parametrize("L", [0, 1, 511, 513, 20000])
def test_histories(cuda, L):
    run(cuda, M=4, V=5000, L=L, seed=L)


@pytest.mark.parametrize("M", [40, 300])
def test_many_rows(cuda, M):
    run(cuda, M=M, V=30001, L=300, n_bias=5, mask=True, seed=M)


def test_each_step_alone(cuda):
    run(cuda, penalties=False, n_bias=9, seed=1)
    run(cuda, penalties=False, mask=True, seed=2)
    run(cuda, penalties=False, seed=3)
    run(cuda, prompts=False, seed=4)


def test_the_last_of_repeated_biases_counts(cuda):
    import torch
    a = run(cuda, M=5, V=40, n_bias=300, repeat_bias=True, mask=True, seed=5)
    assert torch.equal(a, run(cuda, M=5, V=40, n_bias=300, repeat_bias=True, mask=True, seed=5))


def test_one_token_repeated(cuda):
    run(cuda, M=2, V=3000, L=9000, hot=77, lens=9000, seed=6)


@pytest.mark.parametrize("pad", [1, 3, 64])
def test_strides_and_in_place(cuda, pad):
    run(cuda, M=5, V=2049, pad=pad, n_bias=11, mask=True, seed=7)
    run(cuda, M=5, V=2049, pad=pad, n_bias=11, mask=True, in_place=True, seed=7)


def test_infinities_and_nan_pass_through(cuda):
    x = np.random.default_rng(8).standard_normal((3, 500)).astype(np.float32)
    x[:, ::7] = np.inf
    x[:, 1::7] = -np.inf
    x[:, 2::7] = np.nan
    x[:, 3::7] = -3.4028235e38
    with np.errstate(over="ignore", invalid="ignore"):
        import torch
        import yskn_b200 as Y
        d = torch.from_numpy(x).to(cuda)
        out = torch.empty_like(d)
        mask = torch.full((3, 16), -1, dtype=torch.int32, device=cuda)
        mask[:, 3] = 0
        Y.logits_adjust(d, out, mask=mask)
        exp = x.copy()
        exp[:, 96:128] = -np.inf  # masked places are -inf whatever was there
        assert np.array_equal(out.cpu().numpy(), exp, equal_nan=True)


def test_selection_after_it(cuda):
    """A row that allows nothing answers no token; the others the best allowed one."""
    import torch
    import yskn_b200 as Y
    out = run(cuda, M=3, V=2000, mask=True, seed=9)
    token = torch.empty(3, dtype=torch.int32, device=cuda)
    Y.head_select(out.contiguous(), token=token)
    got, ref = token.tolist(), out.argmax(1).tolist()
    assert got[1] == 2 ** 31 - 1 and got[0] == ref[0] and got[2] == ref[2]


def test_other_stream(cuda):
    import torch
    assert torch.equal(run(cuda, M=9, V=7777, L=800, mask=True, n_bias=4, seed=10),
                       run(cuda, M=9, V=7777, L=800, mask=True, n_bias=4, seed=10, stream=torch.cuda.Stream()))


def test_history_longer_than_its_width_is_reported(cuda):
    import torch
    import yskn_b200 as Y
    x = torch.zeros((1, 100), device=cuda)
    Y.logits_adjust(x, torch.empty_like(x), history=torch.zeros((1, 4), dtype=torch.int32, device=cuda),
                    history_lens=torch.tensor([5], dtype=torch.int32, device=cuda),
                    presence=torch.ones(1, device=cuda))
    assert Y.status() == Y.EINVAL


@pytest.mark.parametrize("rep", [0.5, 1.0, 1.3, 3.0, 1e-39, 1e-45, 1e-30, 2.0 ** -126, 2.0 ** 127, 3e38, 0.0, -0.7, np.inf])
@pytest.mark.parametrize("wide", [False, True])
def test_penalties_of_every_size_round_as_the_division(cuda, rep, wide):
    """Infinities, NaN, the largest, the subnormal and bit patterns at random: binary32's quotient and
    product, bit for bit (each step is rounded once, so nothing may differ)."""
    import torch
    import yskn_b200 as Y
    rng = np.random.default_rng(11)
    V = 4099
    x = rng.integers(0, 2 ** 32, V, dtype=np.uint64).astype(np.uint32).view(np.float32)
    x[:12] = [3e38, -3e38, 3.4028235e38, np.inf, -np.inf, np.nan, 0.0, -0.0, 1e-45, 1.1754944e-38, -1e-39, 1.0]
    x[12:1000] = rng.standard_normal(988).astype(np.float32) * 4
    rep = np.float32(rep)
    L = 40000 if wide else V  # counts of 32 bits, or of 16
    hist = np.resize(np.arange(V, dtype=np.int32), (1, L))
    dev = lambda a: torch.from_numpy(a).to(cuda)  # noqa: E731
    out = torch.empty((1, V), device=cuda)
    Y.logits_adjust(dev(x[None]), out, history=dev(hist), history_lens=dev(np.array([L], np.int32)),
                    prompt_lens=dev(np.array([L], np.int32)), repetition=dev(np.array([rep])))
    with np.errstate(all="ignore"):
        exp = np.where(x > 0, x / rep, x * rep)
    got = out.cpu().numpy()[0]
    assert Y.status() == 0
    assert np.array_equal(np.isnan(got), np.isnan(exp))
    bits = ~np.isnan(exp)
    assert np.array_equal(got.view(np.uint32)[bits], exp.view(np.uint32)[bits])


def test_a_history_of_no_entries(cuda):
    """Nothing has been said yet: penalties and all, the logits stay as they are."""
    import torch
    import yskn_b200 as Y
    x = torch.randn((3, 777), device=cuda)
    out, ones = torch.empty_like(x), torch.ones(3, device=cuda)
    none = torch.zeros(3, dtype=torch.int32, device=cuda)
    Y.logits_adjust(x, out, history=torch.zeros((3, 0), dtype=torch.int32, device=cuda), history_lens=none,
                    prompt_lens=none, repetition=2 * ones, presence=ones, frequency=ones)
    assert Y.status() == 0 and torch.equal(out, x)
    Y.logits_adjust(x, out, history=torch.zeros((3, 0), dtype=torch.int32, device=cuda), history_lens=none + 1,
                    presence=ones)
    assert Y.status() == Y.EINVAL and torch.equal(out, x)
