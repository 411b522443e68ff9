"""Paged attention where scores lie far apart, against the plain 64-bit form.

A key that takes nearly all of a row's weight and whose value is zero leaves
the output to keys with weights of e^-gap, all of one sign here so that
nothing averages out.  Such an output is off by the error of the ratio of two
weights, which is the difference of the errors of two scores.  u = 2^-24:
 - the high score, gap plus a little, comes out of at most 12 roundings (parts
   of q, scale, product, difference) and of a chain of c MMAs that each cut up to
   2e-8 = u/3 of the sum: (gap + 1)(12 + c/3) u, which covers the weights' own
   exponentials and sums (a few u) by the + 1.  c is 2, 3 or 6 products (f16,
   bf16, f32 pages) of head_dim/16 steps.
 - weights below 2^-23 of the largest one are held to 2^-46 of it with f16
   pages: 2^(gap log2(e) - 46) of themselves.
"""
import numpy as np
import pytest

from test_gpu_paged import Cache, attend, near, queries, reference

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def peaked(torch, kv, lengths, hd, gap, sink, spread, seed):
    """Keys of scores near 0 but for key `sink`, `gap` above them, with value 0."""
    c = Cache(torch, kv, lengths, 2, hd, 16, seed=seed)
    c.k.mul_(spread)
    c.v.abs_()
    c.view(c.k)[..., 0] = 0
    for s, n in enumerate(lengths):
        if sink < n:
            key = torch.zeros(hd, device="cuda")
            key[0] = gap * hd ** 0.5 / 8
            c.set(c.k, s, sink, key.to(c.k.dtype))
            c.set(c.v, s, sink, 0)
    return c


def peaked_queries(torch, n, heads, hd, seed):
    q = queries(torch, n, heads, hd, seed)
    q.view(n, heads, hd)[..., 0] = 8
    return q


@pytest.mark.parametrize("kv,parts", [("f32", 6), ("f16", 2), ("bf16", 3)])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("gap", [10, 14, 17, 20])
@pytest.mark.parametrize("rows", [None, [70, 60]])
@pytest.mark.parametrize("sink,spread", [(0, 0.0), (37, 0.1)])
def test_values_of_small_weights(cuda, kv, parts, hd, gap, rows, sink, spread):
    lengths = [2000, 60]
    c = peaked(cuda, kv, lengths, hd, gap, sink, spread, seed=gap)
    n = [1, 1] if rows is None else rows
    q = peaked_queries(cuda, sum(n), 8, hd, gap)
    got = attend(cuda, c, q, 8, rows).double().cpu().numpy()
    want = reference(c, q, n, 8)
    tol = (gap + 1) * (12 + parts * hd / 16 / 3) * U + (2.0 ** (gap * np.log2(np.e) - 46) if kv == "f16" else 0)
    off, size = np.linalg.norm(got - want, axis=1), np.linalg.norm(want, axis=1)
    assert (off <= tol * size).all(), (off / size).max() / tol
    assert (np.abs(got - want).max(1) <= 4 * tol * np.abs(want).max(1)).all()


@pytest.mark.parametrize("kv", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("factor", [1e5, 1e7, 1e9, 1e15, 1e25])
@pytest.mark.parametrize("rows", [None, [150]])
def test_scores_of_any_size(cuda, kv, factor, rows):
    """So far apart that one key takes the whole weight: the output is its value
    (two of a row's scores nearer than their error, 1e-6 of them, would be a rare draw)."""
    c = Cache(cuda, kv, [150], 2, 64, 16, seed=31)
    n = [1] if rows is None else rows
    q = queries(cuda, sum(n), 4, 64, 12) * factor
    near(attend(cuda, c, q, 4, rows), reference(c, q, n, 4))


@pytest.mark.parametrize("kv,q0,k0", [("f32", 1e19, -2.2e19), ("bf16", 1e19, -2.2e19), ("f16", 3.36e33, -65504.0)])
@pytest.mark.parametrize("rows", [None, [40]])
@pytest.mark.parametrize("length", [50, 1500])
def test_scores_near_the_lowest_f32(cuda, kv, q0, k0, rows, length):
    """-2.2e38, times log2(e) -3.2e38: finite, and the same for every key, whose values are averaged."""
    c = Cache(cuda, kv, [length], 2, 64, 16, seed=32)
    c.k.zero_()
    c.view(c.k)[..., 0] = k0
    n = [1] if rows is None else rows
    q = cuda.zeros(sum(n), 4 * 64, device="cuda")
    q.view(-1, 4, 64)[..., 0] = q0
    near(attend(cuda, c, q, 4, rows, scale=1.0), reference(c, q, n, 4, scale=1.0))
