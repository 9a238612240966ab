"""Head norms, rotation and cache rows (yskn_b200_paged_prep) against the formula in 64 bits.

Tolerance. The result is rounded once to p bits (bf16 8, f16 11): half a step, at most
2^-p |y|. In binary32 before that: the mean, the inverse root and the products, under 8
roundings with D / 32 + 5 additions of positive squares, and sine and cosine to 2 units, so at
most 64 * 2^-24 of |a| + |b|, the pair's magnitudes. f16 subnormal steps add 2^-25."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
P_BITS = {"bf16": 8, "f16": 11}


def run(cuda, T=5, n_qh=6, n_kvh=2, D=128, rot=64, n_axes=1, source="f32", dtype="bf16", norm=True, paired=False,
        block=16, head_major=True, seed=0, scale=1.0, stream=None, position=40000, one_dim=False):
    import torch
    import yskn_b200 as Y
    types = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
    g = torch.Generator(device=cuda)
    g.manual_seed(seed)
    rnd = lambda *s: torch.randn(s, generator=g, device=cuda)  # noqa: E731
    q = (rnd(T, n_qh, D * (2 if paired else 1)) * scale).to(types[source])[:, :, :D]
    k, v = (rnd(T, n_kvh, D) * scale).to(types[source]), rnd(T, n_kvh, D).to(types[source])
    n_blocks = -(-T // block) + 2
    slots = torch.randperm(n_blocks * block, generator=g, device=cuda)[:T]
    if T > 2:
        slots[1] = -1
    shape = (n_blocks, n_kvh, block, D) if head_major else (n_blocks, block, n_kvh, D)
    caches = [torch.full(shape, 7.0, dtype=types[dtype], device=cuda) for _ in range(2)]
    views = [c.transpose(1, 2) if head_major else c for c in caches]
    positions = torch.randint(0, position, (n_axes, T), generator=g, device=cuda, dtype=torch.int32)
    axes = [(i // 3) % n_axes for i in range(rot // 2)]
    freq = torch.tensor([1e7 ** (-2.0 * i / max(rot, 1)) for i in range(rot // 2)], dtype=torch.float32, device=cuda)
    qn, kn = ((rnd(D) * 0.3).to(torch.bfloat16) for _ in range(2)) if norm else (None, None)
    query = torch.full((T, n_qh, D), 9.0, dtype=types[dtype], device=cuda)
    torch.cuda.synchronize()
    Y.paged_prep(q, k, v, slots, positions[0] if one_dim else positions, query, views[0], views[1],
                 inv_freq=freq if rot else None, axes=None if one_dim else axes, q_norm=qn, k_norm=kn, eps=1e-6,
                 stream=stream)
    torch.cuda.synchronize()
    assert Y.status() == 0

    def expected(x, w):
        x = x.double()
        if w is not None:
            x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * (1 + w.double())
        y, mag = x.clone(), x.abs()
        for i, a in enumerate(axes):
            ang = (positions[a].float() * freq[i]).double()[:, None]
            lo, hi = x[..., i], x[..., i + rot // 2]
            y[..., i] = lo * ang.cos() - hi * ang.sin()
            y[..., i + rot // 2] = hi * ang.cos() + lo * ang.sin()
            mag[..., i] = mag[..., i + rot // 2] = lo.abs() + hi.abs()
        return y, mag

    def near(got, exp, mag):
        tol = 2.0 ** -P_BITS[dtype] * exp.abs() + 64 * 2.0 ** -24 * mag + 2.0 ** -25
        assert bool(((got.double() - exp).abs() <= tol).all()), float(((got.double() - exp).abs() - tol).max())

    real = slots >= 0
    y, mag = expected(q, qn)
    near(query[real], y[real], mag[real])
    assert bool((query[~real] == 0).all())
    at = slots[real]
    for view, rows in ((views[0], expected(k, kn)), (views[1], (v.double(), v.double().abs()))):
        near(view[at // block, at % block], rows[0][real], rows[1][real])
        left = torch.ones(view.shape[:2], dtype=torch.bool, device=cuda)
        left[at // block, at % block] = False
        assert bool((view[left] == 7.0).all())  # no other place is written
    return query, caches


@pytest.mark.parametrize("T", [1, 2, 3, 17, 130])
@pytest.mark.parametrize("D,rot", [(256, 64), (256, 256), (256, 96), (128, 128), (128, 32), (64, 64), (64, 16),
                                   (64, 0)])
def test_sizes(cuda, T, D, rot):
    run(cuda, T=T, D=D, rot=rot, seed=T + D)


@pytest.mark.parametrize("source,dtype", [("f32", "bf16"), ("f32", "f16"), ("bf16", "bf16"), ("f16", "f16")])
@pytest.mark.parametrize("paired", [False, True])
def test_types(cuda, source, dtype, paired):
    run(cuda, T=21, D=256, source=source, dtype=dtype, paired=paired, n_axes=3, seed=3)


@pytest.mark.parametrize("n_qh,n_kvh", [(1, 1), (24, 4), (7, 7), (9, 3), (128, 1)])
def test_head_counts(cuda, n_qh, n_kvh):
    run(cuda, T=6, n_qh=n_qh, n_kvh=n_kvh, seed=4)


@pytest.mark.parametrize("block,head_major", [(16, False), (128, True), (1, True), (10, False)])
def test_cache_orders(cuda, block, head_major):
    run(cuda, T=40, block=block, head_major=head_major, seed=5)


def test_without_norm_and_one_axis_positions(cuda):
    run(cuda, T=9, norm=False, seed=6)
    run(cuda, T=9, one_dim=True, seed=6)


def test_far_positions_and_small_and_large_values(cuda):
    run(cuda, T=60, D=256, rot=64, position=2 ** 24, seed=7)
    run(cuda, T=6, scale=1e-4, seed=8)
    run(cuda, T=6, scale=1e15, seed=9)


def test_other_stream_and_same_result_twice(cuda):
    import torch
    a, b = run(cuda, T=50, seed=10), run(cuda, T=50, seed=10, stream=torch.cuda.Stream())
    assert torch.equal(a[0], b[0]) and all(torch.equal(x, y) for x, y in zip(a[1], b[1]))


def test_a_zero_row_stays_zero(cuda):
    import torch
    import yskn_b200 as Y
    z = lambda *s: torch.zeros(s, device=cuda)  # noqa: E731
    c = [torch.ones((1, 16, 1, 64), dtype=torch.bfloat16, device=cuda) for _ in range(2)]
    query = torch.ones((1, 1, 64), dtype=torch.bfloat16, device=cuda)
    w = torch.zeros(64, dtype=torch.bfloat16, device=cuda)
    Y.paged_prep(z(1, 1, 64), z(1, 1, 64), z(1, 1, 64), torch.zeros(1, dtype=torch.int64, device=cuda),
                 torch.ones((1, 1), dtype=torch.int32, device=cuda), query, c[0], c[1],
                 inv_freq=torch.ones(16, device=cuda), q_norm=w, k_norm=w)
    torch.cuda.synchronize()
    assert bool((query == 0).all()) and bool((c[0][0, 0] == 0).all()) and bool((c[1][0, 1:] == 1).all())


def test_a_slot_past_the_cache_is_reported_and_not_written(cuda):
    import torch
    import yskn_b200 as Y
    x = torch.randn((2, 1, 64), device=cuda)
    c = [torch.zeros((2, 16, 1, 64), dtype=torch.bfloat16, device=cuda) for _ in range(2)]
    Y.paged_prep(x, x, x, torch.tensor([32, 2 ** 40], device=cuda), None, torch.empty_like(x, dtype=torch.bfloat16),
                 c[0], c[1])
    assert Y.status() == Y.EINVAL
    assert all(bool((t == 0).all()) for t in c)
