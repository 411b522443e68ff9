"""Paged attention and append over batches whose rows are no sequence's, or not all in the call."""
import numpy as np
import pytest

import static_lm as S
from static_lm._lib import SlmError
from test_gpu_paged import Cache, append_reference, near, queries, reference, rope_table, run_append

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


@pytest.mark.parametrize("kv", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("length", [70, 2000])  # one CTA a tile, and keys split over CTAs
def test_rows_past_the_call_are_flagged_and_the_others_keep_their_positions(cuda, kv, length):
    c = Cache(cuda, kv, [length, 9], 2, 64, 16, seed=4)
    q = queries(cuda, 14, 4, 64, 4)
    want = reference(c, q[2:], [5, 7], 4)
    out = cuda.full((11, 256), 7.0, device="cuda")  # the second sequence's last three rows are not there
    call(cuda, c, q, 4, [2, 7, 14], 11, length, out)
    assert (out[:2] == 0).all()
    near(out[2:], want[:9])
    assert int(c.status) == 8
    with pytest.raises(SlmError):
        S.paged_check(c.pages)
    assert int(c.status) == 0


def test_append_of_rows_past_the_call(cuda):
    c = Cache(cuda, "f32", [30, 9], 2, 64, 16, seed=5)
    x = queries(cuda, 14, 4 + 4, 64, 5)
    cos, sin = rope_table(30, 64)
    want, _, _, _ = append_reference(c, x[2:], [5, 7], 4, cos, sin, 64, False, None, None, 0)
    cos, sin = cuda.from_numpy(cos).cuda(), cuda.from_numpy(sin).cuda()
    start = cuda.tensor([2, 7, 14], dtype=cuda.int32).cuda()
    out = cuda.full((11, 256), 7.0, device="cuda")
    S.paged_append(c.pages, S.PagedBatch(row_start=start.data_ptr(), kv_len=c.len_d.data_ptr(), page_table=c.table_d.data_ptr(),
                                         table_stride=c.table.shape[1], num_seqs=2, num_rows=11, max_kv_len=30),
                   S.PagedAppendArgs(q=x.data_ptr(), k=x.data_ptr() + 4 * 256, v=x.data_ptr() + 4 * 384, q_out=out.data_ptr(),
                                     ldq=512, ldk=512, ldv=512, ldq_out=256, num_heads=4, rope_cos=cos.data_ptr(),
                                     rope_sin=sin.data_ptr(), rope_rows=30, rotary_dim=64))
    got = out.double().cpu().numpy()
    assert (got[:2] == 0).all()
    assert np.abs(got[2:] - want[:9].reshape(9, 256)).max() <= 6 * 2.0 ** -24 * np.abs(want).max()
    assert int(c.status) == 8


@pytest.mark.parametrize("start", [[0, 6, 4, 9], [-2, 3, 5, 9]])
def test_row_starts_that_fall_or_are_negative_are_flagged(cuda, start):
    c = Cache(cuda, "f16", [40, 30, 20], 2, 64, 16, seed=6)
    q = queries(cuda, 9, 4, 64, 6)
    out = cuda.full((10, 256), 7.0, device="cuda")
    call(cuda, c, q, 4, start, 9, 40, out)
    assert int(c.status) == 8 and (out[9] == 7.0).all()


@pytest.mark.parametrize("table,length,rope,bits", [
    ([-1, -1], 5, 9, 1),  # a page that is not held
    ([90, 0], 1, 9, 1),   # an id past the pool
    ([0, 1], 9, 9, 2),    # a position past the table
    ([0, 1], 8, 7, 2),    # one past the rope table
    ([0, 1], 8, 9, 0),
])
def test_append_flags_what_it_met_and_nothing_else(cuda, table, length, rope, bits):
    c = Cache(cuda, "f32", [length], 1, 64, 4, seed=7)
    c.table = np.array([table], np.int32)
    c.table_d = cuda.from_numpy(c.table).cuda()
    run_append(cuda, c, queries(cuda, 1, 2 + 2, 64, 7), None, 2, *rope_table(rope, 64), 64)
    assert int(c.status) == bits
