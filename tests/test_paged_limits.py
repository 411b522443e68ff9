"""How many positions a page table may cover, without a GPU: a call without rows
checks its arguments and launches nothing."""
import pytest

import static_lm as S
from static_lm._lib import SlmError

A = 1 << 20  # an aligned address that nothing reads
MOST = 2 ** 31 - 1 - 65536


@pytest.mark.parametrize("page,stride,ok", [(1, MOST, True), (1, MOST + 1, False), (16, MOST // 16, True),
                                            (16, MOST // 16 + 1, False), (1, 2 ** 31 - 1, False), (1 << 20, 2047, True),
                                            (1 << 20, 2048, False)])
def test_positions_of_a_table(page, stride, ok):
    pages = S.KvPages(k=A, v=A, num_pages=4, page_size=page, num_kv_heads=1, head_dim=8, dtype=S.KV_F16)
    batch = S.PagedBatch(row_start=A, kv_len=A, page_table=A, table_stride=stride, num_seqs=1, num_rows=0, max_kv_len=64)
    for call in (lambda: S.paged_append(pages, batch, S.PagedAppendArgs(k=A, v=A, ldk=8, ldv=8)),
                 lambda: S.paged_attention(pages, batch, S.PagedAttentionArgs(q=A, out=A + 64, ldq=8, ldo=8, num_heads=1))):
        if ok:
            call()
        else:
            with pytest.raises(SlmError) as e:
                call()
            assert e.value.code == 4
