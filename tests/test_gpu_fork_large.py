"""Forks of pages of which one KV head's slots take 4 GB and more: counts of bytes that pass 32 bits.

The pools are not initialised as a whole: only the slots that are looked at are written first.
"""
import numpy as np
import pytest

import static_lm as S
from test_gpu_beam import fork

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv,heads,slots,used", [
    ("f32", 2, 1 << 23, 5),              # 2^32 bytes from one head to the next
    ("f16", 2, 1 << 24, 9),
    ("f32", 1, (1 << 23) + 16, (1 << 23) + 1),  # more than 2^32 bytes of used slots
])
def test_fork_of_large_pages(cuda, kv, heads, slots, used):
    hd, dt = 128, {"f32": cuda.float32, "f16": cuda.float16}[kv]
    k, v = (cuda.empty(2, heads, slots, hd, dtype=dt, device="cuda") for _ in range(2))
    g = cuda.Generator().manual_seed(used)
    for pool in (k, v):
        # the used slots' first and last ones and those around 2^32 / 16 pieces; the slots behind them keep what they have
        for at in (0, used - 5):
            pool[0, :, at:at + 5] = cuda.randn(heads, 5, hd, generator=g).to(dt).cuda()
            pool[1, :, at:at + 5] = 0
        pool[:, :, used:used + 4] = 7
    pages = [S.KvPages(k=k.data_ptr(), v=v.data_ptr(), num_pages=2, page_size=slots, num_kv_heads=heads, head_dim=hd,
                       dtype=S.KV_DTYPES[kv])]
    got = fork(cuda, pages, np.array([[0]], np.int32), [used], [0, 0], [-1, 1])
    assert got[0].tolist() == [[0], [1]] and got[1].tolist() == [used, used] and got[2].tolist() == [0, 1]
    for pool in (k, v):
        for at in (0, used - 5):
            assert cuda.equal(pool[1, :, at:at + 5], pool[0, :, at:at + 5])
            assert (pool[1, :, at:at + 5] != 0).any(-1).all()
        assert (pool[1, :, used:used + 4] == 7).all()
    del k, v, pool
    cuda.cuda.empty_cache()
