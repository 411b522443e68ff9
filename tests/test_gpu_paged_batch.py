"""Paged attention over batches whose rows are no sequence's."""
import numpy as np
import pytest

import static_lm as S
from test_gpu_paged import Cache, queries

pytestmark = pytest.mark.gpu


def call(torch, c, q, heads, start, num_rows, max_kv_len, out):
    start_d = torch.tensor(start, dtype=torch.int32).cuda()
    batch = S.PagedBatch(row_start=start_d.data_ptr(), kv_len=c.len_d.data_ptr(), page_table=c.table_d.data_ptr(),
                         table_stride=c.table.shape[1], num_seqs=len(start) - 1, num_rows=num_rows, max_kv_len=max_kv_len)
    args = S.PagedAttentionArgs(q=q.data_ptr(), out=out.data_ptr(), ldq=q.stride(0), ldo=out.stride(0), num_heads=heads)
    size = S.paged_attention_scratch_bytes(c.pages, batch, args)
    scratch = torch.full((size + 16,), 0xFF, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    S.paged_attention(c.pages, batch, args, scratch.data_ptr(), size, torch.cuda.current_stream().cuda_stream)
    copy = out.clone()
    torch.cuda.synchronize()
    return copy


@pytest.mark.parametrize("kv", ["f32", "f16", "bf16"])
def test_a_padded_batch_without_a_request_is_zero(cuda, kv):
    """Planned with splits: every CTA of the join waits for the zeros."""
    c = Cache(cuda, kv, [2000, 9], 2, 64, 16, seed=3)
    q = queries(cuda, 15, 4, 64, 3)
    for at in (0, 6, 15):
        for _ in range(10):
            out = cuda.full((15, 256), 7.0, device="cuda")
            assert (call(cuda, c, q, 4, [at, at, at], 15, 2000, out) == 0).all()
    assert int(c.status) == 0
