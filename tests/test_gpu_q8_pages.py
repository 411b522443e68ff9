"""8-bit pages of the paged cache against a plain 64-bit implementation.

Tolerances, set from the arithmetic (u = 2^-24, the rounding of f32):
 - a value that is stored: y' = y + e with |e| <= tol of the append (its rotation
   and norm), max|y'| within tol of max|y|.  q is y' 127/max|y'| rounded, off by
   1/2 and by the roundings of the quotient and the product, 127 * 2.1u at most;
   q scale, with one more rounding of the scale, is off y' by
   max|y'| / 127 (1/2 + 127 * 3.1u).  Together (max|y| + tol) (1/254 + 4u) + tol.
   Without a norm every step is a single rounding in the order of the formula:
   bytes and scales are then equal to those of numpy's f32.
 - attention: as for f16 pages, whose bytes and f16 parts it shares: the score and
   the weight each take the scale with one rounding more.
"""
import numpy as np
import pytest

import static_lm as S
from static_lm._lib import SlmError
from test_gpu_paged import (DECODES, MAX_TOL, ROWS, U, Cache, append_reference, attend, near, queries, reference, rope_table,
                            run_append, torch_type)

pytestmark = pytest.mark.gpu


class Q8Cache(Cache):
    """Pools of bytes; host() and view() give the values they stand for, bytes() and scales() the parts."""

    def __init__(self, torch, lengths, kv_heads, hd, page, seed=0, spare=2, stride_extra=0, table_extra=0, spread=0.0):
        super().__init__(torch, "f16", lengths, kv_heads, hd, page, seed, spare, 0, 0.0, table_extra)
        n = kv_heads * page
        dense = -(-n * (hd + 4) // 16) * 16
        self.stride = dense + stride_extra
        g = torch.Generator().manual_seed(seed)
        pools = []
        for _ in range(2):
            p = torch.randint(0, 256, (self.num_pages, self.stride), dtype=torch.uint8, generator=g)
            q, scale = self.parts(p)
            q.copy_(torch.randint(-127, 128, q.shape, generator=g))
            # values of about N(0, 1) size; spread: rows of unlike sizes
            scale.copy_(torch.exp(spread * torch.randn(scale.shape, generator=g)) / 74)
            pools.append(p.cuda())
        self.k, self.v = pools
        self.pages = S.KvPages(k=self.k.data_ptr(), v=self.v.data_ptr(), page_stride=self.stride if stride_extra else 0,
                               num_pages=self.num_pages, page_size=page, num_kv_heads=kv_heads, head_dim=hd, dtype=S.KV_Q8,
                               status=self.status.data_ptr())
        assert S.paged_page_bytes(self.pages) == dense

    def parts(self, pool):
        n = self.kv_heads * self.page
        return (pool[:, :n * self.hd].view(self.torch.int8).view(-1, self.kv_heads, self.page, self.hd),
                pool[:, n * self.hd:n * (self.hd + 4)].view(self.torch.float32).view(-1, self.kv_heads, self.page))

    def view(self, pool):
        q, scale = self.parts(pool)
        return q.double() * scale[..., None].double()


def make(torch, kv, *args, **more):
    return Q8Cache(torch, *args, **more) if kv == "q8" else Cache(torch, kv, *args, **more)


# ------------------------------------------------------------------- store

APPENDS = [  # heads, kv_heads, hd, page, lengths, rows, rd, halves, norm, offset
    (9, 3, 64, 16, [1], None, 64, False, False, 0),
    (32, 8, 128, 16, [5, 40, 17], None, 128, True, True, 0),
    (6, 6, 48, 24, [30, 7, 100], [12, 7, 1], 48, False, True, 0),
    (4, 4, 16, 1, [9, 2], [3, 2], 16, True, False, 0),
    (12, 2, 80, 7, [33, 64], [33, 0], 32, True, True, 0),
    (20, 4, 96, 16, [21], [21], 96, False, False, 0),
    (9, 3, 64, 16, [50, 3], [20, 3], 16, False, True, 1),   # columns off 16-byte boundaries
    (2, 1, 112, 16, [18], [5], 0, False, False, 3),         # no rotation
    (8, 8, 32, 5, [70], [70], 32, True, False, 0),
]


@pytest.mark.parametrize("case", range(len(APPENDS)))
def test_append(cuda, case):
    heads, kvh, hd, page, lengths, rows, rd, halves, norm, offset = APPENDS[case]
    c = Q8Cache(cuda, lengths, kvh, hd, page, seed=case, stride_extra=32 if case % 2 else 0)
    n = [1] * len(lengths) if rows is None else rows
    x = queries(cuda, sum(n), heads + 2 * kvh, hd, case, pad=offset)
    cos, sin = rope_table(max(lengths), rd)
    g = cuda.Generator().manual_seed(case)
    qn = (1 + 0.3 * cuda.randn(hd, generator=g)).cuda() if norm else None
    kn = (1 + 0.3 * cuda.randn(hd, generator=g)).cuda() if norm else None
    want_q, want_k, want_v, where = append_reference(c, x[:, offset:], n, heads, cos, sin, rd, halves, qn, kn, 1e-5)
    keep = c.k.clone(), c.v.clone()
    got = run_append(cuda, c, x, rows, heads, cos, sin, rd, halves, qn, kn, offset=offset)
    big = 3 * float(np.abs(want_q).max()) + 3 * float(np.abs(want_k).max())
    tol = ((hd / 8 + 10) * U if norm else 0) * big + 3 * U * big
    assert np.abs(got.double().cpu().numpy().reshape(want_q.shape) - want_q).max() <= tol
    touched = np.zeros((c.num_pages, c.page), bool)
    for pool, want, e in ((c.k, want_k, tol), (c.v, want_v, 0.0)):
        values, q = c.host(pool), c.parts(pool)[0].cpu().numpy()
        for r, at in enumerate(where):
            touched[at] = True
            top = np.abs(want[r]).max(-1, keepdims=True)
            assert (np.abs(values[at[0], :, at[1]] - want[r]) <= (top + e) * (1 / 254 + 4 * U) + e).all()
            assert (np.abs(q[at[0], :, at[1]].astype(int)).max(-1) == 127).all()
    # only the rows' slots changed, bit for bit
    for pool, old in ((c.k, keep[0]), (c.v, keep[1])):
        for a, b in zip(c.parts(pool), c.parts(old)):
            same = (a == b).reshape(c.num_pages, kvh, c.page, -1).all(-1).all(1).cpu().numpy()
            assert same[~touched].all()
        n_used = kvh * c.page * (hd + 4)
        assert cuda.equal(pool[:, n_used:], old[:, n_used:])
    assert int(c.status) == 0


def quantised(x):
    """numpy's f32, step by step."""
    top = np.abs(x).max(-1, keepdims=True)
    with np.errstate(all="ignore"):
        up = np.where(top >= np.float32(2.0 ** -100), np.float32(127) / top, np.float32(0)).astype(np.float32)
        scale = np.where(top >= np.float32(2.0 ** -100), top / np.float32(127), np.float32(0)).astype(np.float32)
    return np.rint(x * up).astype(np.int8), scale[..., 0]


@pytest.mark.parametrize("halves", [False, True])
def test_append_without_a_norm_gives_the_formulas_bytes(cuda, halves):
    heads, kvh, hd, n = 4, 2, 64, 130
    c = Q8Cache(cuda, [n], kvh, hd, 8, seed=3)
    x = queries(cuda, n, heads + 2 * kvh, hd, 4)
    x[7, heads * hd:] *= 1e-30       # near f32's smallest normal scales
    x[8, heads * hd:] *= 1e30
    x[9, heads * hd:] *= 2.0 ** -110  # stored as zeros
    x[10, heads * hd:] = 0
    cos, sin = rope_table(n, hd)
    run_append(cuda, c, x, [n], heads, cos, sin, hd, halves=halves)
    k, v = (t.cpu().numpy().reshape(n, kvh, hd) for t in x[:, heads * hd:].split(kvh * hd, 1))
    a, b = (k[..., :hd // 2], k[..., hd // 2:]) if halves else (k[..., 0::2], k[..., 1::2])
    cc, ss = cos[:n, None], sin[:n, None]
    lo, hi = a * cc - b * ss, a * ss + b * cc
    k = np.concatenate([lo, hi], -1) if halves else np.stack([lo, hi], -1).reshape(n, kvh, hd)
    page, slot = c.table[0, np.arange(n) // 8], np.arange(n) % 8
    for pool, want in ((c.k, k), (c.v, v)):
        q, scale = (t.cpu().numpy()[page, :, slot] for t in c.parts(pool))
        want_q, want_scale = quantised(want.astype(np.float32))
        assert np.array_equal(q, want_q) and np.array_equal(scale, want_scale)
    assert (c.parts(c.v)[1].cpu().numpy()[page[9:11], :, slot[9:11]] == 0).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_a_row_that_is_not_finite_reads_back_as_nan(cuda, bad):
    c = Q8Cache(cuda, [3], 2, 16, 4, seed=1)
    x = queries(cuda, 3, 2, 16, 1)
    x[1, 5] = bad
    args = S.PagedAppendArgs(k=x.data_ptr(), v=x.data_ptr(), ldk=32, ldv=32)
    S.paged_append(c.pages, c.batch([3]), args, cuda.cuda.current_stream().cuda_stream)
    cuda.cuda.synchronize()
    got = c.host(c.k)[int(c.table[0, 0])]  # [head][slot][hd]
    assert np.isnan(got[0, 1]).all() and np.isfinite(got[1, :3]).all() and np.isfinite(got[0, [0, 2]]).all()


def test_append_rows_outside_sequences_and_bad_pages(cuda):
    hd, heads, kvh, page = 64, 2, 1, 4
    x = queries(cuda, 8, heads + 2 * kvh, hd, 7)
    for table, length, rope, bit in (([-1, -1], 5, 9, 1), ([99, 0], 1, 9, 1), ([0, 1], 9, 9, 2), ([0, 1], 8, 7, 2)):
        c = Q8Cache(cuda, [length], kvh, hd, page, seed=2)
        c.table = np.array([table], np.int32)
        c.table_d = cuda.from_numpy(c.table).cuda()
        old = c.k.clone()
        run_append(cuda, c, x[:1], None, heads, *rope_table(rope, hd), hd)
        assert int(c.status) & bit and cuda.equal(c.k, old)
        with pytest.raises(SlmError):
            S.paged_check(c.pages)


# --------------------------------------------------------------- read back

READS = [  # kv, kv_heads, hd, page, lengths, rows
    ("q8", 3, 64, 16, [1], None),
    ("q8", 8, 128, 16, [50, 1, 17], [50, 0, 3]),
    ("q8", 2, 80, 7, [33, 64], [33, 60]),
    ("q8", 1, 16, 1, [9], [9]),
    ("f32", 3, 48, 24, [30, 7], [12, 7]),
    ("f16", 4, 8, 16, [100], [100]),
    ("bf16", 2, 120, 5, [21, 3], None),
]


def read(torch, c, rows, dt, ld=None, offset=0, stream=None, parts=(True, True)):
    w = c.kv_heads * c.hd
    ld = ld or w
    batch = c.batch(rows)
    out = [torch.full((max(batch.num_rows, 1), ld), 7.0, dtype=torch_type(torch, dt), device="cuda") for _ in range(2)]
    ptr = [o.data_ptr() + offset * o.element_size() if p else None for o, p in zip(out, parts)]
    args = S.PagedReadArgs(k_out=ptr[0], v_out=ptr[1], ldk=ld, ldv=ld, out_dtype=S.KV_DTYPES[dt])
    torch.cuda.synchronize()
    S.paged_read(c.pages, batch, args, stream.cuda_stream if stream else torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    for o, p in zip(out, parts):
        assert (o[:, :offset] == 7.0).all() and (o[:, offset + w:] == 7.0).all()
        assert p or (o == 7.0).all()
    return [o[:batch.num_rows, offset:offset + w] for o in out]


def read_reference(torch, c, rows, dt):
    """The slots of the batch's rows, through f32 as the kernel's product is."""
    out = []
    for pool in (c.k, c.v):
        if isinstance(c, Q8Cache):
            q, scale = c.parts(pool)
            values = q.float() * scale[..., None]
        else:
            values = c.view(pool).float()
        rows_out = []
        for s, length in enumerate(c.lengths):
            for i in range(rows[s]):
                p = int(length) - rows[s] + i
                page = int(c.table[s, p // c.page]) if p >= 0 else -1
                rows_out.append(values[page, :, p % c.page].reshape(-1) if page >= 0 else values.new_zeros(c.kv_heads * c.hd))
        out.append(torch.stack(rows_out).to(torch_type(torch, dt)))
    return out


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("case", range(len(READS)))
def test_read(cuda, case, dt):
    kv, kvh, hd, page, lengths, rows = READS[case]
    c = make(cuda, kv, lengths, kvh, hd, page, seed=case)
    n = [1] * len(lengths) if rows is None else rows
    want = read_reference(cuda, c, n, dt)
    for ld, offset in ((None, 0), (kvh * hd + 8, 8), (kvh * hd + 5, 1)):
        got = read(cuda, c, rows, dt, ld, offset)
        assert all(cuda.equal(a, b) for a, b in zip(got, want))
    assert cuda.equal(read(cuda, c, rows, dt, parts=(True, False))[0], want[0])
    assert cuda.equal(read(cuda, c, rows, dt, parts=(False, True), stream=cuda.cuda.Stream())[1], want[1])
    assert int(c.status) == 0


def test_read_of_what_is_not_there_is_zero(cuda):
    c = Q8Cache(cuda, [40, 0, 2], 2, 64, 16, seed=4)
    rows = [40, 1, 4]  # a row of an empty sequence, two before position 0
    c.table[0, 1] = -1
    c.table_d = cuda.from_numpy(c.table).cuda()
    want = read_reference(cuda, c, rows, "f32")
    got = read(cuda, c, rows, "f32")
    assert all(cuda.equal(a, b) for a, b in zip(got, want)) and int(c.status) == 0
    assert (got[0][16:32] == 0).all() and (got[0][40:43] == 0).all() and (got[1][43:] != 0).any()
    c.table[0, 0] = c.num_pages
    c.table_d = cuda.from_numpy(c.table).cuda()
    assert (read(cuda, c, rows, "f32")[0][:32] == 0).all() and int(c.status) == 1
    c.status.zero_()
    c.len_d = cuda.tensor([100, 0, 2], dtype=cuda.int32).cuda()  # past the table's 48 positions
    read(cuda, c, rows, "f32")
    assert int(c.status) == 2
    # places of a padded batch that are no sequence's
    c = Q8Cache(cuda, [9, 5], 2, 64, 16, seed=4)
    c.batch([2, 3])
    start = cuda.tensor([1, 3, 6], dtype=cuda.int32).cuda()
    out = cuda.full((2, 9, 128), 7.0, device="cuda")
    batch = S.PagedBatch(row_start=start.data_ptr(), kv_len=c.len_d.data_ptr(), page_table=c.table_d.data_ptr(),
                         table_stride=c.table.shape[1], num_seqs=2, num_rows=9, max_kv_len=9)
    S.paged_read(c.pages, batch, S.PagedReadArgs(k_out=out[0].data_ptr(), v_out=out[1].data_ptr(), ldk=128, ldv=128,
                                                 out_dtype=S.KV_F32), cuda.cuda.current_stream().cuda_stream)
    want = read_reference(cuda, c, [2, 3], "f32")
    assert cuda.equal(out[0, 1:6], want[0]) and cuda.equal(out[1, 1:6], want[1])
    assert (out[:, :1] == 0).all() and (out[:, 6:] == 0).all()


# --------------------------------------------------------------- attention

Q8_DECODES = [d for d in DECODES if d[3] % 16 == 0]
Q8_ROWS = [r for r in ROWS if r[3] % 16 == 0]


@pytest.mark.parametrize("case", range(len(Q8_DECODES)))
def test_decode(cuda, case):
    _, heads, kvh, hd, page, lengths, window, sinks = Q8_DECODES[case]
    c = Q8Cache(cuda, lengths, kvh, hd, page, seed=case, stride_extra=16 * (case % 3), spread=0.3 * (case % 2))
    q = queries(cuda, len(lengths), heads, hd, case)
    got = attend(cuda, c, q, heads, None, window, sinks)
    near(got, reference(c, q, [1] * len(lengths), heads, window, sinks))
    assert cuda.equal(got, attend(cuda, c, q, heads, None, window, sinks)), "not the same bits again"
    assert int(c.status) == 0


@pytest.mark.parametrize("case", range(len(Q8_ROWS)))
def test_rows(cuda, case):
    _, heads, kvh, hd, page, lengths, rows, window, sinks = Q8_ROWS[case]
    c = Q8Cache(cuda, lengths, kvh, hd, page, seed=50 + case, stride_extra=16 * (case % 3), spread=0.3 * (case % 2))
    q = queries(cuda, sum(rows), heads, hd, case)
    got = attend(cuda, c, q, heads, rows, window, sinks)
    near(got, reference(c, q, rows, heads, window, sinks))
    assert cuda.equal(got, attend(cuda, c, q, heads, rows, window, sinks)), "not the same bits again"
    assert int(c.status) == 0


@pytest.mark.parametrize("rows", [None, [3, 2, 70]])
def test_rows_that_see_nothing_are_zero(cuda, rows):
    c = Q8Cache(cuda, [0, 1, 40], 2, 64, 8, seed=9)
    n = [1, 1, 1] if rows is None else rows
    q = queries(cuda, sum(n), 4, 64, 3)
    got, want = attend(cuda, c, q, 4, rows), reference(c, q, n, 4)
    near(got, want)
    assert (got.cpu().numpy()[np.abs(want).max(1) == 0] == 0).all()


@pytest.mark.parametrize("length", [70, 2000])  # one CTA a tile, and keys split over CTAs
def test_rows_of_no_sequence_are_zero(cuda, length):
    c = Q8Cache(cuda, [length, 9], 2, 64, 16, seed=10)
    q = queries(cuda, 3 + 8 + 4, 4, 64, 3)
    want = reference(c, q[3:11], [5, 3], 4)
    c.batch([5, 3])
    start = cuda.tensor([3, 8, 11], dtype=cuda.int32).cuda()
    out = cuda.full((15, 256), 7.0, device="cuda")
    batch = S.PagedBatch(row_start=start.data_ptr(), kv_len=c.len_d.data_ptr(), page_table=c.table_d.data_ptr(),
                         table_stride=c.table.shape[1], num_seqs=2, num_rows=15, max_kv_len=length)
    args = S.PagedAttentionArgs(q=q.data_ptr(), out=out.data_ptr(), ldq=256, ldo=256, num_heads=4)
    size = S.paged_attention_scratch_bytes(c.pages, batch, args)
    scratch = cuda.full((size + 16,), 0xFF, dtype=cuda.uint8, device="cuda")
    cuda.cuda.synchronize()
    S.paged_attention(c.pages, batch, args, scratch.data_ptr(), size)
    cuda.cuda.synchronize()
    near(out[3:11], want)
    assert (out[:3] == 0).all() and (out[11:] == 0).all() and int(c.status) == 0


def seen_by_none_is_nan(c, n, window, sinks):
    """Scales of NaN, and bytes of anything, in every slot that no row sees."""
    for pool in (c.k, c.v):
        q, scale = c.parts(pool)
        keep_q, keep_s = q.clone(), scale.clone()
        q.fill_(-128), scale.fill_(float("nan"))
        for s, length in enumerate(c.lengths):
            for j in range(int(length)):
                if j >= int(length) - n[s] - window + 1 or j < sinks:
                    at = int(c.table[s, j // c.page]), slice(None), j % c.page
                    q[at], scale[at] = keep_q[at], keep_s[at]


@pytest.mark.parametrize("rows", [None, [9, 60]])
def test_slots_not_seen_do_not_matter(cuda, rows):
    n = [1, 1] if rows is None else rows
    c = Q8Cache(cuda, [21, 150], 2, 64, 16, seed=11)
    q = queries(cuda, sum(n), 4, 64, 5)
    want = reference(c, q, n, 4, 50, 3)
    seen_by_none_is_nan(c, n, 50, 3)
    near(attend(cuda, c, q, 4, rows, 50, 3), want)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_what_is_not_finite_reaches_the_rows_that_see_it_and_no_others(cuda, hd, bad):
    """In the middle of a tile, for keys and for values, with rows before it, in its window and past its window."""
    c = Q8Cache(cuda, [90, 30], 2, hd, 16, seed=23)
    c.parts(c.v)[1][int(c.table[0, 40 // 16]), 1, 40 % 16] = bad
    c.parts(c.k)[1][int(c.table[1, 20 // 16]), 0, 20 % 16] = float("nan")
    q = queries(cuda, 120, 4, hd, 7)
    for rows, window, sinks in (([90, 30], 20, 2), (None, 0, 0)):
        n = 120 if rows else 2
        got = attend(cuda, c, q[:n], 4, rows, window, sinks).double().cpu().numpy()
        with np.errstate(all="ignore"):
            want = reference(c, q[:n], rows or [1, 1], 4, window, sinks)
        # the bytes of a value whose scale is infinite may be 0: NaN there, as in the reference
        assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(np.isinf(got), np.isinf(want))
        fine = np.isfinite(want)
        assert (~fine).any()
        assert np.abs(got[fine] - want[fine]).max(initial=0) <= MAX_TOL * np.abs(want[fine]).max(initial=1)
        assert np.array_equal(got[np.isinf(want)], want[np.isinf(want)])


@pytest.mark.parametrize("rows", [None, [40, 2]])
def test_pages_not_held_are_not_seen(cuda, rows):
    c = Q8Cache(cuda, [100, 37], 2, 64, 16, seed=13)
    c.table[0, 1] = c.table[0, 2] = c.table[1, 0] = -1
    c.table_d = cuda.from_numpy(c.table).cuda()
    n = [1, 1] if rows is None else rows
    q = queries(cuda, sum(n), 4, 64, 6)
    near(attend(cuda, c, q, 4, rows), reference(c, q, n, 4))
    assert int(c.status) == 0
    c.table[:] = -1
    c.table_d = cuda.from_numpy(c.table).cuda()
    assert (attend(cuda, c, q, 4, rows) == 0).all()


@pytest.mark.parametrize("rows", [None, [5, 30]])
def test_bad_page_ids_are_flagged_and_not_read(cuda, rows):
    c = Q8Cache(cuda, [40, 30], 1, 64, 16, seed=14)
    n = [1, 1] if rows is None else rows
    q = queries(cuda, sum(n), 2, 64, 6)
    real = c.table.copy()
    c.table[0, 0] = -1
    want = reference(c, q, n, 2)
    c.table = real
    c.table[0, 0] = c.num_pages
    c.table_d = cuda.from_numpy(c.table).cuda()
    near(attend(cuda, c, q, 2, rows), want)
    assert int(c.status) == 1
    c = Q8Cache(cuda, [40, 30], 1, 64, 16, seed=14)  # a length past the table: what the table holds is seen
    c.len_d = cuda.tensor([40, 3000], dtype=cuda.int32).cuda()
    attend(cuda, c, q, 2, rows, max_kv_len=3000)
    assert int(c.status) == 2


def test_row_strides_and_odd_alignment(cuda):
    c = Q8Cache(cuda, [90, 200], 2, 64, 16, seed=15, stride_extra=48)
    for rows in (None, [60, 150]):
        n = [1, 1] if rows is None else rows
        wide = queries(cuda, sum(n), 6, 64, 8, pad=13)
        q = wide[:, 5:5 + 6 * 64]
        near(attend(cuda, c, q, 6, rows, ldq=wide.stride(0), ldo=6 * 64 + 3), reference(c, q.contiguous(), n, 6))


@pytest.mark.parametrize("factor", [1e-30, 1e-6, 1e6, 1e30])
@pytest.mark.parametrize("rows", [None, [40]])
def test_queries_and_scales_of_any_size(cuda, rows, factor):
    """The scores scale with q and with the keys, the output with the values."""
    n = [1] if rows is None else rows
    c = Q8Cache(cuda, [90], 2, 64, 16, seed=18)
    q = queries(cuda, sum(n), 4, 64, 9)
    scale = float(np.float32(0.125 / factor))
    near(attend(cuda, c, q * factor, 4, rows, scale=scale), reference(c, q * factor, n, 4, scale=scale))
    for pool in (c.k, c.v):
        c.parts(pool)[1].mul_(factor)
    near(attend(cuda, c, q, 4, rows, scale=scale), reference(c, q, n, 4, scale=scale))


@pytest.mark.parametrize("rows", [None, [50]])
def test_values_of_unlike_sizes(cuda, rows):
    """Scales that differ by up to e^12 between the rows of a tile, for keys whose
    scores stay of one size and for values: what the largest leaves of the others."""
    n = [1] if rows is None else rows
    c = Q8Cache(cuda, [700], 2, 64, 16, seed=19)
    g = cuda.Generator().manual_seed(5)
    q8, scale = c.parts(c.v)
    scale.mul_(cuda.exp(3 * cuda.randn(scale.shape, generator=g)).cuda())
    q = queries(cuda, sum(n), 4, 64, 9)
    near(attend(cuda, c, q, 4, rows), reference(c, q, n, 4))
    scale.zero_()
    assert (attend(cuda, c, q, 4, rows) == 0).all()


def test_offsets_past_32_bits(cuda):
    """Pages further apart than 2^31 bytes."""
    c = Q8Cache(cuda, [20], 2, 64, 16, seed=18, spare=0)
    far = (1 << 31) + 4096
    pools = [cuda.zeros(far * (c.num_pages - 1) + c.stride, dtype=cuda.uint8, device="cuda") for _ in range(2)]
    for to, pool in zip(pools, (c.k, c.v)):
        for i in range(c.num_pages):
            to[i * far:i * far + c.stride] = pool[i]
    q, x = queries(cuda, 20, 4, 64, 3), queries(cuda, 20, 2 + 2, 64, 4)
    want = [attend(cuda, c, q[:1], 4), attend(cuda, c, q, 4, [20]), *read(cuda, c, [20], "f32")]
    c.pages.k, c.pages.v, c.pages.page_stride = pools[0].data_ptr(), pools[1].data_ptr(), far
    got = [attend(cuda, c, q[:1], 4), attend(cuda, c, q, 4, [20]), *read(cuda, c, [20], "f32")]
    assert all(cuda.equal(a, b) for a, b in zip(got, want))
    args = S.PagedAppendArgs(k=x.data_ptr(), v=x.data_ptr() + 4 * 128, ldk=256, ldv=256)
    S.paged_append(c.pages, c.batch([20]), args, cuda.cuda.current_stream().cuda_stream)
    k, v = read(cuda, c, [20], "f32")
    cuda.cuda.synchronize()
    for got, want in ((k, x[:, :128]), (v, x[:, 128:])):
        got, want = got.view(20, 2, 64), want.view(20, 2, 64)
        assert ((got - want).abs() <= want.abs().amax(-1, keepdim=True) * (1 / 254 + 5 * U)).all()


@pytest.mark.parametrize("rows", [None, [33, 1, 20]])
def test_another_stream_and_graph_replay(cuda, rows):
    """Append, read back and attention captured once, replayed after the lengths and the data changed."""
    heads, kvh, hd = 8, 2, 64
    c = Q8Cache(cuda, [120, 60, 90], kvh, hd, 16, seed=19)
    n = [1] * 3 if rows is None else rows
    x = queries(cuda, sum(n), heads + 2 * kvh, hd, 5)
    cos, sin = (cuda.from_numpy(t).cuda() for t in rope_table(130, hd))
    ld, w = x.stride(0), heads * hd
    q, out = cuda.zeros(sum(n), w, device="cuda"), cuda.zeros(sum(n), w, device="cuda")
    back = cuda.zeros(2, sum(n), kvh * hd, device="cuda")
    batch = c.batch(rows)
    append = S.PagedAppendArgs(q=x.data_ptr(), k=x.data_ptr() + 4 * w, v=x.data_ptr() + 4 * (w + kvh * hd), q_out=q.data_ptr(),
                               ldq=ld, ldk=ld, ldv=ld, ldq_out=w, num_heads=heads, rope_cos=cos.data_ptr(),
                               rope_sin=sin.data_ptr(), rope_rows=130, rotary_dim=hd)
    args = S.PagedAttentionArgs(q=q.data_ptr(), out=out.data_ptr(), ldq=w, ldo=w, num_heads=heads)
    reading = S.PagedReadArgs(k_out=back[0].data_ptr(), v_out=back[1].data_ptr(), ldk=kvh * hd, ldv=kvh * hd, out_dtype=S.KV_F32)
    size = S.paged_attention_scratch_bytes(c.pages, batch, args)
    scratch = cuda.empty(size + 16, dtype=cuda.uint8, device="cuda")

    def step(stream):
        S.paged_append(c.pages, batch, append, stream)
        S.paged_read(c.pages, batch, reading, stream)
        S.paged_attention(c.pages, batch, args, scratch.data_ptr(), size, stream)

    side, graph = cuda.cuda.Stream(), cuda.cuda.CUDAGraph()
    cuda.cuda.synchronize()
    step(side.cuda_stream)
    cuda.cuda.synchronize()
    near(out, reference(c, q, n, heads))
    with cuda.cuda.graph(graph, stream=side):
        step(cuda.cuda.current_stream().cuda_stream)
    for lengths in ([120, 60, 90], [64, 57, 77]):
        c.lengths = np.array(lengths, np.int32)
        c.len_d.copy_(cuda.from_numpy(c.lengths))
        x.copy_(queries(cuda, sum(n), heads + 2 * kvh, hd, 6))
        graph.replay()
        cuda.cuda.synchronize()
        near(out, reference(c, q, n, heads))
        assert all(cuda.equal(a, b) for a, b in zip(back, read_reference(cuda, c, n, "f32")))
    assert int(c.status) == 0


def test_wrong_length_hint_changes_nothing(cuda):
    for rows in (None, [50, 3]):
        c = Q8Cache(cuda, [900, 400], 2, 64, 16, seed=21)
        n = [1, 1] if rows is None else rows
        q = queries(cuda, sum(n), 4, 64, 5)
        want = reference(c, q, n, 4)
        for hint in (0, 1, 100, 900, 5000):
            near(attend(cuda, c, q, 4, rows, max_kv_len=hint), want)


def test_two_calls_at_once(cuda):
    """On two streams, with a scratch each: what each gives alone."""
    work = []
    for seed, (lengths, rows) in enumerate((([900, 33, 1500], None), ([700, 40], [300, 40]))):
        c = Q8Cache(cuda, lengths, 2, 64, 16, seed=30 + seed)
        q = queries(cuda, len(lengths) if rows is None else sum(rows), 8, 64, seed)
        want = attend(cuda, c, q, 8, rows).clone()
        out = cuda.zeros_like(want)
        batch = c.batch(rows)
        args = S.PagedAttentionArgs(q=q.data_ptr(), out=out.data_ptr(), ldq=512, ldo=512, num_heads=8)
        size = S.paged_attention_scratch_bytes(c.pages, batch, args)
        scratch = cuda.empty(size + 16, dtype=cuda.uint8, device="cuda")
        work.append((c, batch, args, scratch, size, cuda.cuda.Stream(), out, want, q))
    cuda.cuda.synchronize()
    for _ in range(20):
        for c, batch, args, scratch, size, stream, out, want, q in work:
            S.paged_attention(c.pages, batch, args, scratch.data_ptr(), size, stream.cuda_stream)
    cuda.cuda.synchronize()
    for *_, out, want, q in work:
        assert cuda.equal(out, want)


@pytest.mark.parametrize("shape", [(9, 3, 64), (8, 1, 128)])
def test_long_prompts(cuda, shape):
    """Several row blocks and key tiles, both streams of a block, blocks that end in either."""
    heads, kvh, hd = shape
    lengths, rows = [700, 129, 260], [650, 129, 3]
    c = Q8Cache(cuda, lengths, kvh, hd, 16, seed=40, spread=0.2)
    q = 2 * queries(cuda, sum(rows), heads, hd, 3)
    for window, sinks in ((0, 0), (300, 5)):
        near(attend(cuda, c, q, heads, rows, window, sinks), reference(c, q, rows, heads, window, sinks))


def peaked(torch, lengths, hd, gap, sink, spread, seed):
    """Keys of scores near 0 but for key `sink`, `gap` above them, with value 0."""
    c = Q8Cache(torch, lengths, 2, hd, 16, seed=seed)
    k, k_scale = c.parts(c.k)
    v, _ = c.parts(c.v)
    k[..., 0] = 0
    k_scale.mul_(spread)
    v.abs_()
    for s, n in enumerate(lengths):
        if sink < n:
            at = int(c.table[s, sink // 16]), slice(None), sink % 16
            k[at], v[at] = 0, 0
            k[at[0], :, at[2], 0] = 127
            k_scale[at] = gap * hd ** 0.5 / 8 / 127
    return c


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("gap", [10, 14, 17, 20])
@pytest.mark.parametrize("rows", [None, [70, 60]])
@pytest.mark.parametrize("sink,spread", [(0, 0.0), (37, 0.1)])
def test_values_of_small_weights(cuda, hd, gap, rows, sink, spread):
    """As with f16 pages (see its tolerance), with two more roundings, the scales', and
    weights that are halved at most by a value's scale relative to a power of two."""
    lengths = [2000, 60]
    c = peaked(cuda, lengths, hd, gap, sink, spread, seed=gap)
    n = [1, 1] if rows is None else rows
    q = queries(cuda, sum(n), 8, hd, gap)
    q.view(-1, 8, hd)[..., 0] = 8
    got = attend(cuda, c, q, 8, rows).double().cpu().numpy()
    want = reference(c, q, n, 8)
    tol = (gap + 1) * (14 + 2 * hd / 16 / 3) * U + 2.0 ** (gap * np.log2(np.e) - 45)
    off, size = np.linalg.norm(got - want, axis=1), np.linalg.norm(want, axis=1)
    assert (off <= tol * size).all(), (off / size).max() / tol
    assert (np.abs(got - want).max(1) <= 4 * tol * np.abs(want).max(1)).all()


@pytest.mark.parametrize("factor", [1e5, 1e7, 1e9, 1e15, 1e25])
@pytest.mark.parametrize("rows", [None, [150]])
def test_scores_of_any_size(cuda, factor, rows):
    """So far apart that one key takes the whole weight: the output is its value."""
    c = Q8Cache(cuda, [150], 2, 64, 16, seed=31)
    n = [1] if rows is None else rows
    q = queries(cuda, sum(n), 4, 64, 12) * factor
    near(attend(cuda, c, q, 4, rows), reference(c, q, n, 4))


@pytest.mark.parametrize("rows", [None, [40]])
@pytest.mark.parametrize("length", [50, 1500])
def test_scores_near_the_lowest_f32(cuda, rows, length):
    """-2.2e38, times log2(e) -3.2e38: finite, and the same for every key, whose values are averaged."""
    c = Q8Cache(cuda, [length], 2, 64, 16, seed=32)
    k, scale = c.parts(c.k)
    k.zero_()
    k[..., 0] = -127
    scale.fill_(2.2e19 / 127)
    n = [1] if rows is None else rows
    q = cuda.zeros(sum(n), 4 * 64, device="cuda")
    q.view(-1, 4, 64)[..., 0] = 1e19
    near(attend(cuda, c, q, 4, rows, scale=1.0), reference(c, q, n, 4, scale=1.0))
