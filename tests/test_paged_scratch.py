"""The scratch of a serving loop's largest call serves every smaller one.  The
size is worked out on the host: no GPU."""
import random

import pytest

import static_lm as S

A = 1 << 20  # an aligned address that nothing reads

SHAPES = [(9, 3, 64), (6, 6, 48), (32, 8, 128), (12, 2, 80), (16, 1, 64), (10, 2, 112), (7, 1, 8), (64, 1, 128), (26, 2, 64)]


def size(shape, kv, rows, seqs, keys, window=0, sinks=0, page=16):
    """seqs None: one new row per sequence."""
    heads, kv_heads, hd = shape
    pages = S.KvPages(k=A, v=A, num_pages=1 << 20, page_size=page, num_kv_heads=kv_heads, head_dim=hd, dtype=S.KV_DTYPES[kv])
    batch = S.PagedBatch(row_start=None if seqs is None else A, kv_len=A, page_table=A, table_stride=1 << 14,
                         num_seqs=rows if seqs is None else seqs, num_rows=rows, max_kv_len=keys)
    args = S.PagedAttentionArgs(q=A, out=A + 4096, ldq=heads * hd, ldo=heads * hd, num_heads=heads, window=window, sinks=sinks)
    return S.paged_attention_scratch_bytes(pages, batch, args)


def spread(rng, hi):
    return min(hi, int(2 ** rng.uniform(0, hi.bit_length())))


@pytest.mark.parametrize("kv", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("decode", [True, False])
def test_smaller_calls_need_no_more(kv, decode):
    rng = random.Random(5)
    for _ in range(400):
        shape = rng.choice(SHAPES)
        window, sinks = (spread(rng, 4096), rng.choice([0, 4, 300])) if rng.random() < 0.4 else (0, 0)
        keys, rows = spread(rng, 1 << 17), spread(rng, 512 if decode else 16384)
        seqs = None if decode else spread(rng, min(rows, 300))
        whole = size(shape, kv, rows, seqs, keys, window, sinks)
        for _ in range(60):
            fewer = spread(rng, rows)
            few = None if decode else min(spread(rng, seqs), seqs)
            less = keys if rng.random() < 0.5 else spread(rng, keys)
            assert size(shape, kv, fewer, few, less, window, sinks) <= whole, (shape, rows, seqs, keys, window, fewer, few, less)


@pytest.mark.parametrize("shape,kv,large,small", [
    # many sequences are not split, fewer are
    ((32, 8, 128), "f16", (256, None, 2048), (22, None, 2048)),
    ((9, 3, 64), "f32", (128, None, 2049), (64, None, 2049)),
    ((32, 8, 128), "f16", (4096, 1, 8192), (287, 1, 8192)),
    ((9, 3, 64), "bf16", (256, 8, 2048), (64, 1, 512)),
])
def test_calls_that_are_split_where_a_larger_one_is_not(shape, kv, large, small):
    assert 0 < size(shape, kv, *small) <= size(shape, kv, *large)


def test_the_size_stays_small():
    """Long prompts and large batches of short sequences: a few megabytes, whatever their number."""
    assert size((32, 8, 128), "f16", 100000, 50, 8192) <= 16 << 20
    assert size((32, 8, 128), "f16", 10000, None, 2000) <= 16 << 20
    assert size((9, 3, 64), "f32", 100, 100, 1) == size((9, 3, 64), "f32", 100, None, 1) == 0
