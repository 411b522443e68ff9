"""Attention over 8-bit pages where scales or scores lie far apart, against the 64-bit reference.

Tolerances (u = 2^-24): a score x (in powers of two) is rounded to f32 and its
difference to the reference of its row again, so a weight is off by at most
(2 |x| u + 2^-22) ln 2 of itself, and the output, of values of one sign, by twice the
largest of these.  Elsewhere as in test_gpu_paged.
"""
import numpy as np
import pytest

from test_gpu_paged import NORM_TOL, U, attend, queries, reference
from test_gpu_q8_pages import Q8Cache

pytestmark = pytest.mark.gpu


def negative(torch, lengths, kvh, hd, magnitude, seed):
    """Keys of elements -magnitude, values above zero."""
    c = Q8Cache(torch, lengths, kvh, hd, 16, seed=seed)
    k, scale = c.parts(c.k)
    k.fill_(-127)
    scale.fill_(magnitude / 127)
    c.parts(c.v)[0].abs_()
    return c


def seen_values(c):
    """[position][KV head][head_dim] of the first sequence's values."""
    j = np.arange(int(c.lengths[0]))
    return c.host(c.v)[c.table[0, j // c.page], :, j % c.page]


def fine_rows(got, want, tol):
    got = got.double().cpu().numpy()
    assert np.isfinite(got).all()
    off, size = np.linalg.norm(got - want, axis=1), np.linalg.norm(want, axis=1)
    assert (off <= tol * np.maximum(size, 1e-30)).all(), (off / np.maximum(size, 1e-30)).max()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("size,magnitude", [(1.0, 1e33), (1.0, 1e35), (1e-20, 1e36), (1e6, 1e30)])
@pytest.mark.parametrize("rows,length", [(None, 50), (None, 2000), ([40], 50), ([300], 2000)])
def test_scores_far_below_zero(cuda, hd, size, magnitude, rows, length):
    """Every score finite, and the same for every key: the values are averaged."""
    c = negative(cuda, [length], 2, hd, magnitude, 3)
    n = [1] if rows is None else rows
    q = queries(cuda, sum(n), 4, hd, 7).abs() * size
    got = attend(cuda, c, q, 4, rows)
    # (not by the scores in 64 bits: sums of the same products in another order differ by more than the weights bear)
    v = seen_values(c)
    want = np.stack([np.repeat(v[:length - n[0] + 1 + i].mean(0), 2, 0).reshape(-1) for i in range(n[0])])
    # (sums of up to 2000 values of one sign in f32, over at least 32 lanes)
    fine_rows(got, want, NORM_TOL)
    assert int(c.status) == 0


@pytest.mark.parametrize("rows", [None, [60]])
@pytest.mark.parametrize("window,sinks", [(0, 0), (20, 3)])
def test_the_nearest_of_scores_far_below_zero(cuda, rows, window, sinks):
    """One key's score lies above the others', all of them finite and far below zero."""
    c = negative(cuda, [90], 2, 64, 1e35, 4)
    c.parts(c.k)[1][int(c.table[0, 80 // 16]), :, 80 % 16] = 5e34 / 127
    c.parts(c.k)[1][int(c.table[0, 40 // 16]), :, 40 % 16] = 9e34 / 127
    n = [1] if rows is None else rows
    q = queries(cuda, sum(n), 4, 64, 7).abs()
    got, v, want = attend(cuda, c, q, 4, rows, window, sinks), seen_values(c), []
    for p in range(90 - n[0], 90):
        seen = [j for j in range(p + 1) if not window or p - j < window or j < sinks]
        best = [80] if 80 in seen else [40] if 40 in seen else seen
        want.append(np.repeat(v[best].mean(0), 2, 0).reshape(-1))
    fine_rows(got, np.stack(want), NORM_TOL)


@pytest.mark.parametrize("sign", [-1, 1])
@pytest.mark.parametrize("heads", [4, 12])
@pytest.mark.parametrize("rows", [None, [200]])
def test_tiny_queries_and_huge_keys(cuda, rows, heads, sign):
    """Scores of 30 to 36 of either sign from elements of 1e-32 and 1e33."""
    c = negative(cuda, [200], 2, 64, 0.0, 5)
    g = cuda.Generator().manual_seed(2)
    k, scale = c.parts(c.k)
    k.fill_(127 * sign)
    scale.copy_((30 + 6 * cuda.rand(scale.shape, generator=g)) / (64 * 127 * 0.125) * 1e32)
    n = [1] if rows is None else rows
    q = cuda.full((sum(n), heads * 64), 1e-32, device="cuda")
    fine_rows(attend(cuda, c, q, heads, rows), reference(c, q, n, heads), 2 * (2 * 36 * np.log2(np.e) * U + 2.0 ** -22) * np.log(2))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("ratio", [2.0 ** 10, 2.0 ** 20, 2.0 ** 36, 2.0 ** 60, 2.0 ** 120])
@pytest.mark.parametrize("length,window,sinks", [(100, 0, 0), (300, 25, 0), (300, 25, 4), (1500, 0, 0)])
def test_large_values_that_a_row_does_not_see(cuda, hd, ratio, length, window, sinks):
    """Values `ratio` times the others', later than a row or behind its window, in the
    tiles of what it sees: each row is held to its own size."""
    c = Q8Cache(cuda, [length], 2, hd, 16, seed=8)
    c.parts(c.v)[0].abs_()
    scale = c.parts(c.v)[1]
    for at in (70, length - 31):
        scale[int(c.table[0, at // 16]), :, at % 16] *= ratio
    q = queries(cuda, length, 4, hd, 9)
    got, want = attend(cuda, c, q, 4, [length], window, sinks), reference(c, q, [length], 4, window, sinks)
    fine_rows(got, want, NORM_TOL)
    # the last row alone, as one of many
    one = attend(cuda, c, q[-1:], 4, None, window, sinks)
    fine_rows(one, want[-1:], NORM_TOL)


@pytest.mark.parametrize("rows", [[100], [40, 3]])
def test_rows_of_zeros_beside_large_values(cuda, rows):
    """Scales of 0 are nothing that a larger one could hide."""
    c = Q8Cache(cuda, [100, 60][:len(rows)], 2, 64, 16, seed=9)
    scale = c.parts(c.v)[1]
    for s, n in enumerate(c.lengths):
        for at in range(0, int(n), 3):
            scale[int(c.table[s, at // 16]), :, at % 16] = 0
        scale[int(c.table[s, (int(n) - 1) // 16]), :, (int(n) - 1) % 16] = 1e20
    q = queries(cuda, sum(rows), 4, 64, 10)
    fine_rows(attend(cuda, c, q, 4, rows), reference(c, q, rows, 4), NORM_TOL)


@pytest.mark.parametrize("hd", [48, 64, 128])
@pytest.mark.parametrize("ratio", [2.0 ** 12, 2.0 ** 30, 2.0 ** 45, 2.0 ** 60])
@pytest.mark.parametrize("rows,heads", [(None, 4), (None, 12), ([90], 4)])
@pytest.mark.parametrize("length", [100, 1500])
def test_large_values_of_no_weight(cuda, hd, ratio, rows, heads, length):
    """Values `ratio` times the others', of keys that every row sees with a weight of
    e^-40 or less: beside them in their tiles, and with up to 2^60 e^-40 = 5 of the others' size in all."""
    c = Q8Cache(cuda, [length], 2, hd, 16, seed=11)
    c.parts(c.v)[0].abs_()
    k, k_scale = c.parts(c.k)
    k[..., 0] = 0
    v_scale = c.parts(c.v)[1]
    for at in range(0, length - 90 if rows else length, 45):
        to = int(c.table[0, at // 16]), slice(None), at % 16
        k[to] = 0
        k[to[0], :, to[2], 0] = -127
        k_scale[to] = 40 * hd ** 0.5 / 8 / 127
        v_scale[to] *= ratio
    n = [1] if rows is None else rows
    q = queries(cuda, sum(n), heads, hd, 9)
    q.view(-1, heads, hd)[..., 0] = 8
    got, want = attend(cuda, c, q, heads, rows), reference(c, q, n, heads)
    # (scores to 40 log2(e) = 58, of both signs)
    fine_rows(got, want, 2 * (2 * 58 * U + 2.0 ** -22) * np.log(2))


@pytest.mark.parametrize("spread", [2.0, 4.0, 8.0])
@pytest.mark.parametrize("rows", [None, [120, 7, 33]])
@pytest.mark.parametrize("window,sinks", [(0, 0), (30, 4)])
def test_values_of_all_sizes(cuda, spread, rows, window, sinks):
    """Scales that are spread by e^(8 N): each row and head is held to its own size."""
    c = Q8Cache(cuda, [150, 64, 700], 2, 64, 16, seed=13)
    g = cuda.Generator().manual_seed(6)
    scale = c.parts(c.v)[1]
    scale.mul_(cuda.exp(spread * cuda.randn(scale.shape, generator=g)).cuda())
    c.parts(c.v)[0].abs_()
    n = [1, 1, 1] if rows is None else rows
    q = queries(cuda, sum(n), 6, 64, 12)
    got, want = attend(cuda, c, q, 6, rows, window, sinks), reference(c, q, n, 6, window, sinks)
    fine_rows(got.reshape(-1, 64), want.reshape(-1, 64), NORM_TOL)
