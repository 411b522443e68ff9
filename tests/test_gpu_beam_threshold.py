"""Selection where the threshold that a row's warps share moves all the time.

Each of a row's warps takes every fourth chunk of 512 logits and raises the common
threshold while the others read it.  With logits that rise, in steps or through
every warp's own chunks apart, it moves with every chunk of every warp; the result is
that of a sort, and the same bits each time.
"""
import numpy as np
import pytest

from test_gpu_beam import select

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("out", [1, 5, 32, 33, 64])
@pytest.mark.parametrize("shape", ["rising", "rising by chunk", "one warp above the others", "rising and falling"])
def test_thresholds_that_move(cuda, shape, out):
    vocab, rows = 40 * 2048 + 77, 64
    t = np.arange(vocab, dtype=np.float32)
    chunk = t.astype(np.int64) // 512
    x = {"rising": t * 1e-3, "rising by chunk": chunk.astype(np.float32) * 0.5,
         "one warp above the others": chunk * 0.25 + 50.0 * (chunk % 4 == 2),
         "rising and falling": np.where(chunk % 2 == 0, t, vocab - t) * 1e-3}[shape].astype(np.float32)
    logits = cuda.from_numpy(x).cuda().repeat(rows, 1)
    scores = cuda.zeros(rows, device="cuda")
    order = np.argsort(-x, kind="stable")[:out]
    top = x.max()
    lse = top + np.log(np.exp(x.astype(np.float64) - top).sum())
    first = select(cuda, logits, scores, 1, out)
    assert (first[2] == order).all() and (first[1] == np.arange(rows)[:, None]).all()
    assert np.abs(first[0] - (x[order].astype(np.float64) - lse)).max() <= 4e-6 + 2.0 ** -23 * abs(top - lse)
    for _ in range(20):
        again = select(cuda, logits, scores, 1, out)
        assert all(np.array_equal(a, b) for a, b in zip(first, again))
