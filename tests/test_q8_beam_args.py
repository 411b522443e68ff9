"""Refusals of 8-bit pages, reading back, forking and beam selection, without a
GPU: every check here fails before any CUDA call."""
import random

import pytest

import static_lm as S
from static_lm._lib import SlmError, lib
from test_paged_args import A, INVALID, OVERLAP, SHAPE, append_args, attention_args, batch, pages

CAPACITY = 5


def code(call):
    with pytest.raises(SlmError) as e:
        call()
    return e.value.code


def q8(**k):
    return pages(**{**dict(dtype=S.KV_Q8), **k})


def read_args(**k):
    return S.PagedReadArgs(**{**dict(k_out=A, v_out=A + 4096, ldk=128, ldv=128, out_dtype=S.KV_F16), **k})


def fork_args(**k):
    d = dict(parent=A, kv_len=A, page_table=A, spare=A, kv_len_out=A + 4096, page_table_out=A + 8192, taken=A, table_stride=4,
             num_seqs=2, num_new=3)
    return S.PagedForkArgs(**{**d, **k})


def beam_args(**k):
    d = dict(logits=A, ld=1000, scores=A, num_groups=2, beams=3, vocab=1000, num_out=4, out_scores=A + 4096, out_rows=A + 8192,
             out_tokens=A + 16384)
    return S.BeamSelectArgs(**{**d, **k})


@pytest.mark.parametrize("change,want", [
    (dict(head_dim=24), SHAPE), (dict(head_dim=8), SHAPE), (dict(head_dim=144), SHAPE), (dict(k=A + 8), INVALID),
    (dict(page_stride=2 * 16 * 68 - 16), SHAPE), (dict(page_stride=2 * 16 * 68 + 8), INVALID),
])
def test_8_bit_pages_are_checked(change, want):
    for call in (lambda: S.paged_append(q8(**change), batch(), append_args()),
                 lambda: S.paged_attention(q8(**change), batch(), attention_args(), A, 1 << 30),
                 lambda: S.paged_read(q8(**change), batch(), read_args()),
                 lambda: S.paged_fork([q8(**change)], fork_args())):
        assert code(call) == want


def test_page_bytes():
    assert S.paged_page_bytes(q8()) == 2 * 16 * 68
    assert S.paged_page_bytes(q8(page_size=7, num_kv_heads=3, k=None, v=None)) == 1440  # 3 * 7 * 68 = 1428
    assert S.paged_page_bytes(pages()) == 2 * 16 * 64 * 2
    assert S.paged_page_bytes(pages(dtype=S.KV_F32, page_stride=1 << 20)) == 2 * 16 * 64 * 4
    assert S.paged_page_bytes(q8(head_dim=24)) == S.paged_page_bytes(pages(dtype=9)) == 0
    assert lib().slm_paged_page_bytes(None) == 0


@pytest.mark.parametrize("change,want", [
    (dict(k_out=None, v_out=None), INVALID), (dict(ldk=127), SHAPE), (dict(ldv=127), SHAPE), (dict(out_dtype=S.KV_Q8), INVALID),
    (dict(out_dtype=-1), INVALID), (dict(k_out=A + 1), INVALID), (dict(v_out=A + 2, out_dtype=S.KV_F32), INVALID),
    (dict(v_out=A), OVERLAP),
])
def test_read_arguments_are_checked(change, want):
    assert code(lambda: S.paged_read(q8(), batch(), read_args(**change))) == want


@pytest.mark.parametrize("change,want", [
    (dict(parent=None), INVALID), (dict(kv_len=None), INVALID), (dict(page_table=None), INVALID),
    (dict(kv_len_out=None), INVALID), (dict(page_table_out=None), INVALID), (dict(table_stride=0), SHAPE),
    (dict(table_stride=1 << 28), SHAPE), (dict(num_seqs=0), SHAPE), (dict(num_new=65537), SHAPE),
    (dict(page_table_out=A), OVERLAP), (dict(kv_len_out=A), OVERLAP),
])
def test_fork_arguments_are_checked(change, want):
    assert code(lambda: S.paged_fork([q8(), q8()], fork_args(**change))) == want


@pytest.mark.parametrize("change", [dict(page_size=32), dict(num_pages=5), dict(dtype=S.KV_F16), dict(page_stride=4096),
                                    dict(num_kv_heads=1), dict(head_dim=32)])
def test_layers_have_one_shape(change):
    assert code(lambda: S.paged_fork([q8(), q8(**change)], fork_args())) == SHAPE


@pytest.mark.parametrize("name", ["parent", "kv_len", "page_table", "spare", "kv_len_out", "page_table_out", "taken"])
def test_fork_pointers_are_aligned(name):
    assert code(lambda: S.paged_fork([q8()], fork_args(**{name: A + 2}))) == INVALID


@pytest.mark.parametrize("name", ["logits", "scores", "ended", "out_scores", "out_rows", "out_tokens"])
def test_beam_pointers_are_aligned(name):
    assert code(lambda: S.beam_select(beam_args(**{name: A + 2}), A, 1 << 40)) == INVALID


def test_fork_pages_have_a_largest_size():
    # (one layer's keys of a page: 32 GB and more)
    for change in (dict(dtype=S.KV_F32, page_size=1 << 19, num_kv_heads=128, head_dim=128), dict(page_size=1 << 20, num_kv_heads=256, head_dim=128)):
        assert code(lambda: S.paged_fork([q8(num_pages=1, page_stride=0, **change)], fork_args(table_stride=8))) == SHAPE


def test_no_layers_and_no_sequences():
    assert code(lambda: S.paged_fork([], fork_args())) == INVALID
    S.paged_fork([q8()], fork_args(num_new=0))
    S.paged_read(q8(), batch(num_rows=0), read_args())


@pytest.mark.parametrize("change,want", [
    (dict(logits=None), INVALID), (dict(scores=None), INVALID), (dict(out_scores=None), INVALID), (dict(out_rows=None), INVALID),
    (dict(out_tokens=None), INVALID), (dict(beams=0), SHAPE), (dict(beams=257), SHAPE), (dict(num_out=0), SHAPE),
    (dict(num_out=65), SHAPE), (dict(vocab=0), SHAPE), (dict(vocab=(1 << 30) + 1, ld=1 << 31), SHAPE), (dict(ld=999), SHAPE),
    (dict(num_groups=1 << 24), SHAPE), (dict(out_rows=A + 16384), OVERLAP), (dict(out_scores=A), OVERLAP),
])
def test_beam_arguments_are_checked(change, want):
    assert code(lambda: S.beam_select(beam_args(**change), A, 1 << 40)) == want


def test_beam_scratch_is_checked():
    size = S.beam_select_scratch_bytes(beam_args())
    assert size > 0
    assert code(lambda: S.beam_select(beam_args(), A, size - 1)) == CAPACITY
    assert code(lambda: S.beam_select(beam_args(), 0, size)) == INVALID
    assert code(lambda: S.beam_select(beam_args(), A + 8, size)) == INVALID
    S.beam_select(beam_args(num_groups=0), 0, 0)


def test_null_descriptors():
    for rc in (lib().dll.slm_paged_read(q8(), batch(), None, None), lib().dll.slm_paged_read(None, batch(), read_args(), None),
               lib().dll.slm_paged_fork(None, 1, fork_args(), None), lib().dll.slm_paged_fork(q8(), 1, None, None),
               lib().dll.slm_beam_select(None, None, 0, None)):
        assert rc == INVALID
    assert lib().slm_beam_select_scratch_bytes(None) == 0


def test_smaller_selections_need_no_more_scratch():
    rng = random.Random(3)
    most = lambda hi: max(1, min(hi, int(2 ** rng.uniform(0, hi.bit_length()))))  # noqa: E731
    for _ in range(3000):
        big = dict(num_groups=most(2048), beams=most(64), vocab=most(1 << 20), num_out=most(64))
        less = {k: most(v) if rng.random() < 0.6 else v for k, v in big.items()}
        size = lambda d: S.beam_select_scratch_bytes(beam_args(**d, ld=1 << 20))  # noqa: E731
        assert size(less) <= size(big), (big, less)


@pytest.mark.parametrize("decode", [True, False])
def test_smaller_calls_over_8_bit_pages_need_no_more_scratch(decode):
    rng = random.Random(6)
    most = lambda hi: max(1, min(hi, int(2 ** rng.uniform(0, hi.bit_length()))))  # noqa: E731

    def size(shape, rows, seqs, keys, window):
        heads, kv_heads, hd = shape
        args = S.PagedAttentionArgs(q=A, out=A + 4096, ldq=heads * hd, ldo=heads * hd, num_heads=heads, window=window, sinks=4)
        return S.paged_attention_scratch_bytes(
            q8(num_kv_heads=kv_heads, head_dim=hd, num_pages=1 << 20),
            batch(row_start=None if decode else A, num_seqs=rows if decode else seqs, num_rows=rows, max_kv_len=keys,
                  table_stride=1 << 14), args)

    for _ in range(300):
        shape = rng.choice([(9, 3, 64), (6, 6, 48), (32, 8, 128), (12, 2, 80), (16, 1, 64), (64, 1, 128), (26, 2, 64)])
        window = most(4096) if rng.random() < 0.4 else 0
        keys, rows = most(1 << 17), most(512 if decode else 16384)
        seqs = most(min(rows, 300))
        whole = size(shape, rows, seqs, keys, window)
        for _ in range(40):
            assert size(shape, most(rows), most(seqs), most(keys), window) <= whole
