"""The paged key/value cache against a plain 64-bit implementation.

Tolerances, set from the arithmetic (u = 2^-24, the rounding of f32):
 - a rotated element is two products and a sum, 3u(|a| + |b|); with the norm
   before it the mean of head_dim squares and the two products add at most
   (head_dim/8 + 10)u relative.  Stored in f16 / bf16 it moves by at most half
   a unit in the last place more: 2^-11 / 2^-8 of the value (2^-25 in f16's
   subnormals).
 - attention: a score is a dot product of head_dim terms, off by about
   sqrt(head_dim) u sum|q k| scale, which is the relative error of its weight;
   with q and k of N(0, 1) that is about 1e-6 of the output, which is held to
   5e-6 in the 2-norm and to 2e-4 of the largest value element by element.
"""
import numpy as np
import pytest

import static_lm as S
from static_lm._lib import SlmError

pytestmark = pytest.mark.gpu

NORM_TOL, MAX_TOL = 5e-6, 2e-4
U = 2.0 ** -24


def torch_type(torch, kv):
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[kv]


class Cache:
    """A pool with sequences of the given lengths in pages dealt out in a shuffled order."""

    def __init__(self, torch, kv, lengths, kv_heads, hd, page, seed=0, spare=2, stride_extra=0, fill=None, table_extra=0):
        self.torch, self.kv, self.page, self.kv_heads, self.hd = torch, kv, page, kv_heads, hd
        rng = np.random.default_rng(seed)
        need = [-(-n // page) for n in lengths]
        self.num_pages = sum(need) + spare
        ids = rng.permutation(self.num_pages)
        self.table = np.full((len(lengths), max(max(need), 1) + table_extra), -1, np.int32)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = ids[at:at + n]
            at += n
        self.lengths = np.array(lengths, np.int32)
        dense = kv_heads * page * hd
        self.stride = dense + stride_extra
        g = torch.Generator().manual_seed(seed)
        dt = torch_type(torch, kv)

        def pool():
            if fill is not None:
                return torch.full((self.num_pages * self.stride,), fill, dtype=dt, device="cuda")
            return torch.randn(self.num_pages * self.stride, generator=g).to(dt).cuda()

        self.k, self.v = pool(), pool()
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.table_d = torch.from_numpy(self.table).cuda()
        self.len_d = torch.from_numpy(self.lengths).cuda()
        self.pages = S.KvPages(k=self.k.data_ptr(), v=self.v.data_ptr(), page_stride=self.stride if stride_extra else 0,
                               num_pages=self.num_pages, page_size=page, num_kv_heads=kv_heads, head_dim=hd,
                               dtype=S.KV_DTYPES[kv], status=self.status.data_ptr())

    def view(self, pool):
        """[page][head][slot][hd] of a flat pool."""
        d = self.kv_heads * self.page * self.hd
        return pool.view(self.num_pages, self.stride)[:, :d].view(self.num_pages, self.kv_heads, self.page, self.hd)

    def host(self, pool):
        return self.view(pool).double().cpu().numpy()

    def set(self, pool, seq, key, value):
        self.view(pool)[int(self.table[seq, key // self.page]), :, key % self.page] = value

    def batch(self, rows=None, max_kv_len=None):
        t = self.torch
        n = len(self.lengths)
        if rows is None:
            self.start_d, total, start = None, n, None
        else:
            start = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
            self.start_d = t.from_numpy(start).cuda()
            total = int(start[-1])
        return S.PagedBatch(row_start=None if rows is None else self.start_d.data_ptr(), kv_len=self.len_d.data_ptr(),
                            page_table=self.table_d.data_ptr(), table_stride=self.table.shape[1], num_seqs=n,
                            num_rows=total, max_kv_len=int(max(self.lengths)) if max_kv_len is None else max_kv_len)


def reference(c, q, rows, heads, window=0, sinks=0, scale=None):
    """Row by row in 64 bits; q [rows][heads*hd]."""
    k, v = c.host(c.k), c.host(c.v)
    hd, group = c.hd, heads // c.kv_heads
    scale = 1 / np.sqrt(hd) if scale is None else scale
    q = q.double().cpu().numpy().reshape(-1, heads, hd)
    out = np.zeros_like(q)
    r = 0
    for s, length in enumerate(c.lengths):
        for i in range(rows[s]):
            p = int(length) - rows[s] + i
            j = np.arange(p + 1) if p >= 0 else np.zeros(0, int)
            if window:
                j = j[(p - j < window) | (j < sinks)]
            page = c.table[s, j // c.page] if j.size else j
            j, page = j[page >= 0], page[page >= 0]
            if j.size:
                kk, vv = k[page, :, j % c.page], v[page, :, j % c.page]  # [n][kvh][hd]
                for h in range(heads):
                    x = kk[:, h // group] @ q[r, h] * scale
                    w = np.exp(x - x.max())
                    out[r, h] = w / w.sum() @ vv[:, h // group]
            r += 1
    return out.reshape(r, heads * hd)


def attend(torch, c, q, heads, rows=None, window=0, sinks=0, scale=0.0, ldq=None, ldo=None, stream=None, max_kv_len=None):
    n, w = q.shape[0], heads * c.hd
    ldo = ldo or w
    out = torch.full((max(n, 1), ldo), 7.0, device="cuda")
    batch = c.batch(rows, max_kv_len)
    args = S.PagedAttentionArgs(q=q.data_ptr(), out=out.data_ptr(), ldq=ldq or q.stride(0), ldo=ldo, num_heads=heads,
                                scale=scale, window=window, sinks=sinks)
    size = S.paged_attention_scratch_bytes(c.pages, batch, args)
    # not zeros: the scratch's contents are of no account
    scratch = torch.full((size + 16,), 0xFF, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    S.paged_attention(c.pages, batch, args, scratch.data_ptr(), size,
                      stream.cuda_stream if stream else torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert (scratch[size:] == 0xFF).all(), "wrote past the scratch"
    assert (out[:, w:] == 7.0).all(), "wrote between the rows"
    return out[:n, :w]


def near(got, want, vmax=None):
    got = got.double().cpu().numpy()
    assert np.isfinite(got).all()
    norm = np.linalg.norm(want)
    assert np.linalg.norm(got - want) <= NORM_TOL * max(norm, 1e-30), np.linalg.norm(got - want) / norm
    assert np.abs(got - want).max() <= MAX_TOL * max(np.abs(want).max(), 1e-30)


def queries(torch, n, heads, hd, seed, pad=0):
    g = torch.Generator().manual_seed(1000 + seed)
    return torch.randn(n, heads * hd + pad, generator=g).cuda()


# ------------------------------------------------------------------ append


def append_reference(c, x, rows, heads, cos, sin, rd, halves, qn, kn, eps):
    """Rotated q [rows][heads][hd] and the (page, slot, k, v) of every row."""
    hd = c.hd
    x = x.double().cpu().numpy().reshape(-1, heads + 2 * c.kv_heads, hd)
    q, k, v = x[:, :heads].copy(), x[:, heads:heads + c.kv_heads].copy(), x[:, heads + c.kv_heads:]
    for t, w in ((q, qn), (k, kn)):
        if w is not None:
            t *= 1 / np.sqrt((t * t).mean(-1, keepdims=True) + eps) * w.double().cpu().numpy()
    r, where = 0, []
    for s, length in enumerate(c.lengths):
        for i in range(rows[s]):
            p = int(length) - rows[s] + i
            if p >= 0 and rd:
                cc, ss = cos[p].astype(np.float64), sin[p].astype(np.float64)
                for t in (q, k):
                    a = t[r, :, :rd // 2].copy() if halves else t[r, :, 0:rd:2].copy()
                    b = t[r, :, rd // 2:rd].copy() if halves else t[r, :, 1:rd:2].copy()
                    lo, hi = a * cc - b * ss, a * ss + b * cc
                    if halves:
                        t[r, :, :rd // 2], t[r, :, rd // 2:rd] = lo, hi
                    else:
                        t[r, :, 0:rd:2], t[r, :, 1:rd:2] = lo, hi
            if p < 0:
                q[r] = 0
            where.append((int(c.table[s, p // c.page]), p % c.page) if p >= 0 else None)
            r += 1
    return q, k, v, where


def run_append(torch, c, x, rows, heads, cos, sin, rd, halves=False, qn=None, kn=None, eps=1e-5, in_place=False,
               offset=0, stream=None):
    """x [rows][ld] holds q, k, v side by side from column `offset` on."""
    hd, ld = c.hd, x.stride(0)
    n = x.shape[0]
    base = x.data_ptr() + 4 * offset
    out = x if in_place else torch.full((n, heads * hd + offset), 7.0, device="cuda")
    cd, sd = torch.from_numpy(cos).cuda(), torch.from_numpy(sin).cuda()
    args = S.PagedAppendArgs(
        q=base, k=base + 4 * heads * hd, v=base + 4 * (heads + c.kv_heads) * hd,
        q_out=base if in_place else out.data_ptr() + 4 * offset, ldq=ld, ldk=ld, ldv=ld, ldq_out=out.stride(0),
        num_heads=heads, q_norm=None if qn is None else qn.data_ptr(), k_norm=None if kn is None else kn.data_ptr(),
        norm_eps=eps, rope_cos=cd.data_ptr(), rope_sin=sd.data_ptr(), rope_rows=cos.shape[0], rotary_dim=rd,
        rope_style=S.ROPE_HALVES if halves else S.ROPE_PAIRS)
    batch = c.batch(rows)
    torch.cuda.synchronize()
    S.paged_append(c.pages, batch, args, stream.cuda_stream if stream else torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    return out[:, offset:offset + heads * hd]


def rope_table(rows, rd):
    a = np.arange(rows)[:, None] * 10000.0 ** (-np.arange(0, max(rd, 2), 2) / max(rd, 2))[None, :]
    return np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)


APPENDS = [  # kv, heads, kv_heads, hd, page, lengths, rows, rd, halves, norm, offset
    ("f32", 9, 3, 64, 16, [1], None, 64, False, False, 0),
    ("f16", 32, 8, 128, 16, [5, 40, 17], None, 128, True, True, 0),
    ("bf16", 6, 6, 48, 24, [30, 7, 100], [12, 7, 1], 48, False, True, 0),
    ("f16", 4, 4, 8, 1, [9, 2], [3, 2], 8, True, False, 0),
    ("f32", 12, 2, 80, 7, [33, 64], [33, 0], 32, True, True, 0),
    ("bf16", 20, 4, 96, 16, [21], [21], 96, False, False, 0),
    ("f16", 9, 3, 64, 16, [50, 3], [20, 3], 16, False, True, 1),   # columns off 16-byte boundaries
    ("f32", 2, 1, 120, 16, [18], [5], 0, False, False, 3),         # no rotation
]


@pytest.mark.parametrize("case", range(len(APPENDS)))
def test_append(cuda, case):
    kv, heads, kvh, hd, page, lengths, rows, rd, halves, norm, offset = APPENDS[case]
    c = Cache(cuda, kv, lengths, kvh, hd, page, seed=case, stride_extra=16 if case % 2 else 0)
    n = [1] * len(lengths) if rows is None else rows
    x = queries(cuda, sum(n), heads + 2 * kvh, hd, case, pad=offset)
    cos, sin = rope_table(max(lengths), rd)
    g = cuda.Generator().manual_seed(case)
    qn = (1 + 0.3 * cuda.randn(hd, generator=g)).cuda() if norm else None
    kn = (1 + 0.3 * cuda.randn(hd, generator=g)).cuda() if norm else None
    xq = x[:, offset:] if offset else x
    want_q, want_k, want_v, where = append_reference(c, xq, n, heads, cos, sin, rd, halves, qn, kn, 1e-5)
    before_k, before_v = c.host(c.k), c.host(c.v)
    keep = c.k.clone(), c.v.clone()
    got = run_append(cuda, c, x, rows, heads, cos, sin, rd, halves, qn, kn, offset=offset)
    big = 3 * float(np.abs(want_q).max()) + 3 * float(np.abs(want_k).max())
    tol = ((hd / 8 + 10) * U if norm else 0) * big + 3 * U * big
    assert np.abs(got.double().cpu().numpy().reshape(want_q.shape) - want_q).max() <= tol
    step = {"f32": 0.0, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[kv]
    for r, at in enumerate(where):
        before_k[at[0], :, at[1]], before_v[at[0], :, at[1]] = want_k[r], want_v[r]
    for pool, want in ((c.k, before_k), (c.v, before_v)):
        d = np.abs(c.host(pool) - want)
        assert (d <= tol + step * np.abs(want) * (1 + 2.0 ** -6) + (2.0 ** -25 if step else 0)).all()
    # only the rows' slots changed, bit for bit
    touched = np.zeros((c.num_pages, c.page), bool)
    for at in where:
        touched[at] = True
    for pool, old in ((c.k, keep[0]), (c.v, keep[1])):
        same = (c.view(pool) == c.view(old)).all(-1).all(1).cpu().numpy()
        assert same[~touched].all()
    assert int(c.status) == 0


def test_append_pairs_are_the_bits_of_apply_rope_cached(cuda):
    from static_lm._lib import lib
    hd, heads, kvh, n = 64, 4, 2, 19
    c = Cache(cuda, "f32", [n], kvh, hd, 8, seed=3)
    x = queries(cuda, n, heads + 2 * kvh, hd, 4)
    cos, sin = S.rope_tables(n, hd)
    got = run_append(cuda, c, x, [n], heads, cos.reshape(n, -1), sin.reshape(n, -1), hd)
    cd, sd = cuda.from_numpy(cos).cuda(), cuda.from_numpy(sin).cuda()
    y = x.clone()
    for r in range(n):
        lib().slm_apply_rope_cached(y[r].data_ptr(), (heads + kvh) * hd, cd[r * hd // 2:].data_ptr(),
                                    sd[r * hd // 2:].data_ptr(), hd, None)
    cuda.cuda.synchronize()
    assert cuda.equal(got, y[:, :heads * hd])
    for r in range(n):
        page, slot = c.table[0, r // 8], r % 8
        assert cuda.equal(c.view(c.k)[int(page), :, slot].reshape(-1), y[r, heads * hd:(heads + kvh) * hd])
        assert cuda.equal(c.view(c.v)[int(page), :, slot].reshape(-1), x[r, (heads + kvh) * hd:])


def test_append_in_place_on_another_stream(cuda):
    hd, heads, kvh = 128, 8, 2
    c = Cache(cuda, "f16", [37, 12], kvh, hd, 16, seed=5)
    x = queries(cuda, 16, heads + 2 * kvh, hd, 6)
    cos, sin = rope_table(37, hd)
    want = run_append(cuda, c, x, [5, 11], heads, cos, sin, hd, halves=True).clone()
    pools = c.k.clone(), c.v.clone()
    c.k.zero_(), c.v.zero_()
    side = cuda.cuda.Stream()
    y = x.clone()
    run_append(cuda, c, y, [5, 11], heads, cos, sin, hd, halves=True, in_place=True, stream=side)
    assert cuda.equal(y[:, :heads * hd], want) and cuda.equal(y[:, heads * hd:], x[:, heads * hd:])
    for got, old in ((c.k, pools[0]), (c.v, pools[1])):
        a, b = c.view(got), c.view(old)
        for s, (first, length) in enumerate(((32, 37), (1, 12))):
            for p in range(first, length):
                at = int(c.table[s, p // 16]), slice(None), p % 16
                assert cuda.equal(a[at], b[at])


def test_append_without_queries_and_to_the_type_limits(cuda):
    c = Cache(cuda, "f16", [3], 1, 8, 4, seed=1)
    x = cuda.tensor([[65504.0, 65520.0, -1e9, 6e-8, 2e-8, float("inf"), float("nan"), 0.0]] * 3).cuda()
    args = S.PagedAppendArgs(k=x.data_ptr(), v=x.data_ptr(), ldk=8, ldv=8)
    S.paged_append(c.pages, c.batch([3]), args, cuda.cuda.current_stream().cuda_stream)
    cuda.cuda.synchronize()
    for p in range(3):
        got = c.view(c.k)[int(c.table[0, 0]), 0, p]
        want = x[0].half()
        assert cuda.equal(got.isnan(), want.isnan()) and cuda.equal(got[:6], want[:6]) and got[7] == 0


def test_append_rows_outside_sequences_and_bad_pages(cuda):
    hd, heads, kvh, page = 64, 2, 1, 4
    c = Cache(cuda, "f32", [2, 0, 9], kvh, hd, page, seed=2, table_extra=1)
    rows = [4, 1, 3]  # two rows before position 0, one of an empty sequence
    x = queries(cuda, 8, heads + 2 * kvh, hd, 7)
    cos, sin = rope_table(9, hd)
    old = c.k.clone()
    got = run_append(cuda, c, x, rows, heads, cos, sin, hd)
    assert (got[:2] == 0).all() and (got[4] == 0).all() and (got[2:4] != 0).any() and (got[5:] != 0).any()
    assert int(c.status) == 0
    changed = (c.view(c.k) != c.view(old)).any(-1).any(1).sum()
    assert int(changed) == 5
    # a page that is not held, an id past the pool, a position past the table, one past the rope table
    for table, length, rope, bit in (([-1, -1], 5, 9, 1), ([c.num_pages, 0], 1, 9, 1), ([0, 1], 9, 9, 2), ([0, 1], 8, 7, 2)):
        c2 = Cache(cuda, "f32", [length], kvh, hd, page, seed=2)
        c2.table = np.array([table], np.int32)
        c2.table_d = cuda.from_numpy(c2.table).cuda()
        c2.pages.num_pages = c2.num_pages = min(c2.num_pages, c.num_pages)
        old = c2.k.clone()
        got = run_append(cuda, c2, x[:1], None, heads, *rope_table(rope, hd), hd)
        assert int(c2.status) & bit and cuda.equal(c2.k, old)
        with pytest.raises(SlmError) as e:
            S.paged_check(c2.pages)
        assert e.value.code == 7
        S.paged_check(c2.pages)  # read once, then clear


# --------------------------------------------------------------- attention

DECODES = [  # kv, heads, kv_heads, hd, page, lengths, window, sinks
    ("f32", 6, 6, 48, 16, [77], 0, 0),
    ("f32", 9, 3, 64, 16, [1, 2, 63, 64, 65, 300], 0, 0),
    ("f16", 32, 8, 128, 16, [1000, 1, 517], 0, 0),
    ("bf16", 8, 2, 128, 32, [2049, 31, 33], 0, 0),
    ("f16", 32, 8, 128, 16, [4, 5, 1024, 1025, 1500], 1024, 4),
    ("bf16", 12, 2, 80, 24, [100, 700], 33, 1),
    ("f32", 20, 4, 96, 7, [500, 8], 1, 0),
    ("f16", 16, 1, 64, 64, [333, 1200], 100, 37),
    ("f32", 32, 1, 128, 16, [129], 0, 0),
    ("f16", 5, 1, 8, 1, [50, 3], 0, 0),
    ("bf16", 7, 7, 32, 8, [257] * 3, 64, 200),
    ("f16", 10, 2, 112, 16, [640], 0, 0),
    ("f32", 48, 8, 128, 16, [3000, 100], 0, 0),
    ("bf16", 26, 2, 64, 16, [90, 1], 0, 0),
]


@pytest.mark.parametrize("case", range(len(DECODES)))
def test_decode(cuda, case):
    kv, heads, kvh, hd, page, lengths, window, sinks = DECODES[case]
    c = Cache(cuda, kv, lengths, kvh, hd, page, seed=case)
    q = queries(cuda, len(lengths), heads, hd, case)
    got = attend(cuda, c, q, heads, None, window, sinks)
    near(got, reference(c, q, [1] * len(lengths), heads, window, sinks))
    assert cuda.equal(got, attend(cuda, c, q, heads, None, window, sinks)), "not the same bits again"
    assert int(c.status) == 0


ROWS = [  # kv, heads, kv_heads, hd, page, lengths, rows, window, sinks
    ("f16", 9, 3, 64, 16, [200], [200], 0, 0),
    ("bf16", 9, 3, 64, 16, [129, 1, 300], [129, 1, 40], 0, 0),
    ("f32", 9, 3, 64, 16, [150, 64], [150, 3], 0, 0),
    ("f16", 32, 8, 128, 16, [300, 33], [260, 33], 0, 0),
    ("bf16", 8, 2, 128, 32, [500, 90], [17, 90], 0, 0),
    ("f32", 8, 2, 128, 16, [280], [130], 0, 0),
    ("f16", 8, 2, 128, 16, [600], [300], 100, 4),
    ("f32", 6, 6, 48, 24, [190, 20], [100, 20], 33, 2),
    ("bf16", 12, 2, 80, 7, [100, 70, 5], [3, 0, 5], 1, 0),
    ("f16", 16, 1, 64, 64, [333], [222], 64, 37),
    ("f32", 20, 4, 96, 16, [140], [70], 0, 0),
    ("f16", 4, 4, 8, 1, [65, 40], [65, 2], 0, 0),
    ("bf16", 5, 1, 120, 16, [260], [131], 128, 0),
    ("f16", 32, 1, 32, 16, [70], [30], 0, 0),
    ("f16", 2, 1, 64, 16, [2000, 900], [2, 4], 0, 0),
    ("f32", 2, 1, 128, 16, [1500], [5], 700, 3),
    ("bf16", 3, 3, 64, 16, [1030, 5], [129, 2], 256, 130),
]


@pytest.mark.parametrize("case", range(len(ROWS)))
def test_rows(cuda, case):
    kv, heads, kvh, hd, page, lengths, rows, window, sinks = ROWS[case]
    c = Cache(cuda, kv, lengths, kvh, hd, page, seed=50 + case)
    q = queries(cuda, sum(rows), heads, hd, case)
    got = attend(cuda, c, q, heads, rows, window, sinks)
    near(got, reference(c, q, rows, heads, window, sinks))
    assert cuda.equal(got, attend(cuda, c, q, heads, rows, window, sinks)), "not the same bits again"
    assert int(c.status) == 0


@pytest.mark.parametrize("kv", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [None, [3, 2, 70]])
def test_rows_that_see_nothing_are_zero(cuda, kv, rows):
    lengths = [0, 1, 40]
    c = Cache(cuda, kv, lengths, 2, 64, 8, seed=9)
    n = [1, 1, 1] if rows is None else rows
    q = queries(cuda, sum(n), 4, 64, 3)
    got = attend(cuda, c, q, 4, rows)
    want = reference(c, q, n, 4)
    near(got, want)
    assert (got.cpu().numpy()[np.abs(want).max(1) == 0] == 0).all()


@pytest.mark.parametrize("kv", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("length", [70, 2000])  # one CTA a tile, and keys split over CTAs
def test_rows_of_no_sequence_are_zero(cuda, kv, length):
    """Places of a padded batch before the first sequence's rows and after the last's."""
    c = Cache(cuda, kv, [length, 9], 2, 64, 16, seed=10)
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
    assert (out[:3] == 0).all() and (out[11:] == 0).all()
    cos, sin = (cuda.from_numpy(t).cuda() for t in rope_table(length, 64))
    x = queries(cuda, 15, 4 + 4, 64, 4)
    q_out = cuda.full((15, 256), 7.0, device="cuda")
    S.paged_append(c.pages, batch, S.PagedAppendArgs(
        q=x.data_ptr(), k=x.data_ptr() + 4 * 256, v=x.data_ptr() + 4 * 384, q_out=q_out.data_ptr(), ldq=512, ldk=512, ldv=512,
        ldq_out=256, num_heads=4, rope_cos=cos.data_ptr(), rope_sin=sin.data_ptr(), rope_rows=length, rotary_dim=64))
    cuda.cuda.synchronize()
    assert (q_out[:3] == 0).all() and (q_out[11:] == 0).all() and (q_out[3:11].abs().sum(1) > 0).all()
    assert int(c.status) == 0


@pytest.mark.parametrize("kv", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [None, [9, 60]])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_slots_not_seen_do_not_matter(cuda, kv, rows, bad):
    lengths = [21, 150]
    c = Cache(cuda, kv, lengths, 2, 64, 16, seed=11, fill=bad)
    good = Cache(cuda, kv, lengths, 2, 64, 16, seed=11)
    window, sinks = 50, 3
    n = [1, 1] if rows is None else rows
    for s, length in enumerate(lengths):
        first = length - n[s]
        for j in range(length):
            if j >= first - window + 1 or j < sinks:  # seen by some row
                for bad_pool, pool in ((c.k, good.k), (c.v, good.v)):
                    c.set(bad_pool, s, j, good.view(pool)[int(good.table[s, j // 16]), :, j % 16])
    q = queries(cuda, sum(n), 4, 64, 5)
    got = attend(cuda, c, q, 4, rows, window, sinks)
    near(got, reference(good, q, n, 4, window, sinks))


@pytest.mark.parametrize("kv", ["f32", "f16"])
@pytest.mark.parametrize("rows", [None, [40, 2]])
def test_pages_not_held_are_not_seen(cuda, kv, rows):
    c = Cache(cuda, kv, [100, 37], 2, 64, 16, seed=13)
    c.table[0, 1] = c.table[0, 2] = c.table[1, 0] = -1
    c.table_d = cuda.from_numpy(c.table).cuda()
    n = [1, 1] if rows is None else rows
    q = queries(cuda, sum(n), 4, 64, 6)
    near(attend(cuda, c, q, 4, rows), reference(c, q, n, 4))
    assert int(c.status) == 0
    # every page gone: zero
    c.table[:] = -1
    c.table_d = cuda.from_numpy(c.table).cuda()
    assert (attend(cuda, c, q, 4, rows) == 0).all()


@pytest.mark.parametrize("rows", [None, [5, 30]])
def test_bad_page_ids_are_flagged_and_not_read(cuda, rows):
    c = Cache(cuda, "f16", [40, 30], 1, 64, 16, seed=14)
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
    with pytest.raises(SlmError):
        S.paged_check(c.pages)
    # a length past the table: what the table holds is seen
    c = Cache(cuda, "f16", [40, 30], 1, 64, 16, seed=14)
    c.len_d = cuda.tensor([40, 3000], dtype=cuda.int32).cuda()
    attend(cuda, c, q, 2, rows, max_kv_len=3000)
    assert int(c.status) == 2


def test_row_strides_and_odd_alignment(cuda):
    c = Cache(cuda, "f16", [90, 200], 2, 64, 16, seed=15, stride_extra=40)
    for rows in (None, [60, 150]):
        n = [1, 1] if rows is None else rows
        wide = queries(cuda, sum(n), 6, 64, 8, pad=13)
        q = wide[:, 5:5 + 6 * 64]
        got = attend(cuda, c, q, 6, rows, ldq=wide.stride(0), ldo=6 * 64 + 3)
        near(got, reference(c, q.contiguous(), n, 6))


def test_large_scores_and_scale(cuda):
    c = Cache(cuda, "f32", [300], 2, 64, 16, seed=16)
    for rows in (None, [200]):
        n = [1] if rows is None else rows
        q = queries(cuda, sum(n), 4, 64, 9)
        near(attend(cuda, c, q, 4, rows, scale=0.5), reference(c, q, n, 4, scale=np.float32(0.5)))
        # scores far apart: one key takes all the weight, large negative ones none
        q = q * 1000
        got = attend(cuda, c, q, 4, rows).double().cpu().numpy()
        want = reference(c, q, n, 4)
        assert np.abs(got - want).max() <= 0.05 * np.abs(want).max() and np.isfinite(got).all()


@pytest.mark.parametrize("factor", [1e-30, 1e-6, 1e6, 1e30])
@pytest.mark.parametrize("rows", [None, [40]])
def test_queries_of_any_size(cuda, rows, factor):
    """The scores scale with q; 1/factor as the scale gives the same weights."""
    for kv in ("f32", "f16", "bf16"):
        c = Cache(cuda, kv, [90], 2, 64, 16, seed=18)
        n = [1] if rows is None else rows
        q = queries(cuda, sum(n), 4, 64, 9)
        big = q * factor
        scale = float(np.float32(0.125 / factor))
        near(attend(cuda, c, big, 4, rows, scale=scale), reference(c, big, n, 4, scale=scale))


def test_nan_in_a_seen_slot_reaches_its_rows(cuda):
    for kv in ("f32", "f16", "bf16"):
        c = Cache(cuda, kv, [20, 40], 1, 64, 16, seed=17)
        c.set(c.k, 1, 3, float("nan"))
        q = queries(cuda, 2, 2, 64, 4)
        got = attend(cuda, c, q, 2)
        assert got[1].isnan().all() and got[0].isfinite().all()


@pytest.mark.parametrize("kv", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_what_is_not_finite_reaches_the_rows_that_see_it_and_no_others(cuda, kv, hd, bad):
    """In the middle of a tile, for keys and for values, with rows before it, in
    its window and past its window."""
    c = Cache(cuda, kv, [90, 30], 2, hd, 16, seed=23)
    c.view(c.v)[int(c.table[0, 40 // 16]), 1, 40 % 16, 5] = bad
    c.view(c.k)[int(c.table[1, 20 // 16]), 0, 20 % 16] = float("nan")
    q = queries(cuda, 120, 4, hd, 7)
    got = attend(cuda, c, q, 4, [90, 30], window=20, sinks=2).double().cpu().numpy().reshape(120, 4, hd)
    with np.errstate(all="ignore"):
        want = reference(c, q, [90, 30], 4, window=20, sinks=2).reshape(120, 4, hd)
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(np.isinf(got), np.isinf(want))
    fine = np.isfinite(want)
    assert fine.mean() > 0.9 and (~fine).any()
    assert np.abs(got[fine] - want[fine]).max() <= MAX_TOL * np.abs(want[fine]).max()
    assert np.array_equal(got[np.isinf(want)], want[np.isinf(want)])
    # one new row each
    got = attend(cuda, c, q[:2], 4).double().cpu().numpy().reshape(2, 4, hd)
    with np.errstate(all="ignore"):
        want = reference(c, q[:2], [1, 1], 4).reshape(2, 4, hd)
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(got[np.isinf(want)], want[np.isinf(want)])
    fine = np.isfinite(want)
    assert np.abs(got[fine] - want[fine]).max() <= MAX_TOL * np.abs(want[fine]).max()


def test_offsets_past_32_bits(cuda):
    """Pages further apart than 2^31 elements."""
    stride = (1 << 31) // 2 + 2 * 16 * 64
    c = Cache(cuda, "f16", [40], 2, 64, 16, seed=18, spare=0, stride_extra=stride - 2 * 16 * 64, fill=0.0)
    assert c.num_pages == 3
    cuda.manual_seed(1)
    for pool in (c.k, c.v):
        c.view(pool).copy_(cuda.randn(3, 2, 16, 64, device="cuda"))
    x = queries(cuda, 40, 4 + 4, 64, 2)
    cos, sin = rope_table(40, 64)
    run_append(cuda, c, x, [40], 4, cos, sin, 64)
    _, want_k, want_v, where = append_reference(c, x, [40], 4, cos, sin, 64, False, None, None, 0)
    for r, (page, slot) in enumerate(where):
        got = c.view(c.k)[page, :, slot].double().cpu().numpy()
        assert np.abs(got - want_k[r]).max() <= 2.0 ** -10 * np.abs(want_k[r]).max()
    q = queries(cuda, 40, 4, 64, 3)
    small = Cache(cuda, "f16", [40], 2, 64, 16, seed=18, spare=0)
    for a, b in ((small.k, c.k), (small.v, c.v)):
        small.view(a).copy_(c.view(b))
    near(attend(cuda, c, q[:1], 4), reference(small, q[:1], [1], 4))
    near(attend(cuda, c, q, 4, [40]), reference(small, q, [40], 4))


@pytest.mark.parametrize("rows", [None, [33, 1, 20]])
def test_another_stream_and_graph_replay(cuda, rows):
    """Captured once, replayed after the lengths, the tables and the data changed."""
    c = Cache(cuda, "bf16", [120, 60, 90], 2, 64, 16, seed=19)
    n = [1] * 3 if rows is None else rows
    q = queries(cuda, sum(n), 8, 64, 5)
    side = cuda.cuda.Stream()
    got = attend(cuda, c, q, 8, rows, stream=side)
    near(got, reference(c, q, n, 8))
    out = cuda.zeros_like(q)
    batch = c.batch(rows)
    args = S.PagedAttentionArgs(q=q.data_ptr(), out=out.data_ptr(), ldq=512, ldo=512, num_heads=8)
    size = S.paged_attention_scratch_bytes(c.pages, batch, args)
    scratch = cuda.empty(size + 16, dtype=cuda.uint8, device="cuda")
    graph = cuda.cuda.CUDAGraph()
    with cuda.cuda.graph(graph, stream=side):
        S.paged_attention(c.pages, batch, args, scratch.data_ptr(), size, cuda.cuda.current_stream().cuda_stream)
    graph.replay()
    cuda.cuda.synchronize()
    assert cuda.equal(out, got)
    c.lengths = np.array([64, 57, 77], np.int32)
    c.len_d.copy_(cuda.from_numpy(c.lengths))
    c.k.copy_(c.k.flip(0))
    graph.replay()
    cuda.cuda.synchronize()
    near(out, reference(c, q, n, 8))


def test_scratch_too_small_is_refused(cuda):
    c = Cache(cuda, "f16", [8192], 1, 128, 16, seed=20)
    q = queries(cuda, 1, 8, 128, 5)
    out = cuda.zeros_like(q)
    batch = c.batch(None)
    args = S.PagedAttentionArgs(q=q.data_ptr(), out=out.data_ptr(), ldq=1024, ldo=1024, num_heads=8)
    size = S.paged_attention_scratch_bytes(c.pages, batch, args)
    assert size > 0
    scratch = cuda.empty(size, dtype=cuda.uint8, device="cuda")
    for ptr, n in ((scratch.data_ptr(), size - 1), (0, size), (scratch.data_ptr() + 8, size)):
        with pytest.raises(SlmError) as e:
            S.paged_attention(c.pages, batch, args, ptr, n)
        assert e.value.code in (1, 5)


def test_wrong_length_hint_changes_nothing(cuda):
    """max_kv_len sizes the grid and the scratch; the lengths on the device decide."""
    for rows in (None, [50, 3]):
        c = Cache(cuda, "f16", [900, 400], 2, 64, 16, seed=21)
        n = [1, 1] if rows is None else rows
        q = queries(cuda, sum(n), 4, 64, 5)
        want = reference(c, q, n, 4)
        for hint in (0, 1, 100, 900, 5000):
            near(attend(cuda, c, q, 4, rows, max_kv_len=hint), want)
