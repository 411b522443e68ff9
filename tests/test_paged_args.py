"""Refusals of the paged key/value cache entry points, without a GPU: every
check here fails before any CUDA call."""
import pytest

import static_lm as S
from static_lm._lib import SlmError

A = 1 << 20  # an aligned address that no check reads


def pages(**k):
    d = dict(k=A, v=A, num_pages=4, page_size=16, num_kv_heads=2, head_dim=64, dtype=S.KV_F16)
    return S.KvPages(**{**d, **k})


def batch(**k):
    d = dict(row_start=A, kv_len=A, page_table=A, table_stride=4, num_seqs=2, num_rows=3, max_kv_len=64)
    return S.PagedBatch(**{**d, **k})


def append_args(**k):
    d = dict(q=A, k=A, v=A, q_out=A + 4096, ldq=256, ldk=128, ldv=128, ldq_out=256, num_heads=4, rope_cos=A,
             rope_sin=A, rope_rows=64, rotary_dim=64)
    return S.PagedAppendArgs(**{**d, **k})


def attention_args(**k):
    d = dict(q=A, out=A + 4096, ldq=256, ldo=256, num_heads=4)
    return S.PagedAttentionArgs(**{**d, **k})


INVALID, OVERLAP, SHAPE = 1, 3, 4

BAD_PAGES = [
    (dict(k=None), INVALID), (dict(v=None), INVALID), (dict(k=A + 8), INVALID), (dict(dtype=7), INVALID),
    (dict(num_pages=0), SHAPE), (dict(page_size=0), SHAPE), (dict(num_kv_heads=0), SHAPE),
    (dict(head_dim=0), SHAPE), (dict(head_dim=60), SHAPE), (dict(head_dim=136), SHAPE),
    (dict(page_stride=2 * 16 * 64 - 8), SHAPE), (dict(page_stride=2 * 16 * 64 + 4), INVALID),
    (dict(status=A + 2), INVALID), (dict(num_pages=1 << 31), SHAPE),
]
BAD_BATCH = [
    (dict(kv_len=None), INVALID), (dict(page_table=None), INVALID), (dict(table_stride=0), SHAPE),
    (dict(num_seqs=0), SHAPE), (dict(row_start=None), SHAPE), (dict(table_stride=1 << 28), SHAPE),
    (dict(num_rows=1 << 31), SHAPE),
]


@pytest.mark.parametrize("change,code", BAD_PAGES)
def test_pages_are_checked(change, code):
    for call in (lambda: S.paged_append(pages(**change), batch(), append_args()),
                 lambda: S.paged_attention(pages(**change), batch(), attention_args(), A, 1 << 30)):
        with pytest.raises(SlmError) as e:
            call()
        assert e.value.code == code


@pytest.mark.parametrize("change,code", BAD_BATCH)
def test_batches_are_checked(change, code):
    for call in (lambda: S.paged_append(pages(), batch(**change), append_args()),
                 lambda: S.paged_attention(pages(), batch(**change), attention_args(), A, 1 << 30)):
        with pytest.raises(SlmError) as e:
            call()
        assert e.value.code == code


@pytest.mark.parametrize("change,code", [
    (dict(k=None), INVALID), (dict(v=None), INVALID), (dict(q=None), INVALID), (dict(q_out=None), INVALID),
    (dict(num_heads=3), SHAPE), (dict(ldq=255), SHAPE), (dict(ldk=127), SHAPE), (dict(ldv=127), SHAPE),
    (dict(ldq_out=255), SHAPE), (dict(rotary_dim=12), SHAPE), (dict(rotary_dim=72), SHAPE),
    (dict(rope_cos=None), INVALID), (dict(rope_sin=None), INVALID), (dict(rope_style=2), INVALID),
    (dict(q_norm=A, norm_eps=-1.0), INVALID), (dict(k_norm=A, norm_eps=float("nan")), INVALID),
    (dict(q_out=A, ldq_out=320), OVERLAP),
])
def test_append_arguments_are_checked(change, code):
    with pytest.raises(SlmError) as e:
        S.paged_append(pages(), batch(), append_args(**change))
    assert e.value.code == code


@pytest.mark.parametrize("change,code", [
    (dict(q=None), INVALID), (dict(out=None), INVALID), (dict(num_heads=0), SHAPE), (dict(num_heads=5), SHAPE),
    (dict(ldq=255), SHAPE), (dict(ldo=255), SHAPE), (dict(scale=-0.5), INVALID),
    (dict(scale=float("inf")), INVALID), (dict(scale=float("nan")), INVALID), (dict(out=A), OVERLAP),
])
def test_attention_arguments_are_checked(change, code):
    with pytest.raises(SlmError) as e:
        S.paged_attention(pages(), batch(), attention_args(**change), A, 1 << 30)
    assert e.value.code == code


def test_no_rows_is_no_work():
    S.paged_append(pages(), batch(num_rows=0), append_args())
    S.paged_attention(pages(), batch(num_rows=0), attention_args())


def test_check_needs_a_status_word():
    with pytest.raises(SlmError) as e:
        S.paged_check(pages())
    assert e.value.code == INVALID


def test_null_descriptors():
    from static_lm._lib import lib
    for rc in (lib().dll.slm_paged_append(None, batch(), append_args(), None),
               lib().dll.slm_paged_append(pages(), None, append_args(), None),
               lib().dll.slm_paged_append(pages(), batch(), None, None),
               lib().dll.slm_paged_attention(pages(), batch(), None, None, 0, None)):
        assert rc == INVALID


def test_page_types_have_names():
    assert S.KV_DTYPES == {"f32": S.KV_F32, "f16": S.KV_F16, "bf16": S.KV_BF16}
    assert len(set(S.KV_DTYPES.values())) == 3
