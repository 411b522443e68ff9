"""Beam selection and the forking of page tables against plain implementations.

Selection: a candidate's sum hangs on log sum exp, whose terms e^(x - m) are off
by 2u(|x - m|) (difference and product), the exponential's 2^-22 and the sums'
roundings, at most 40u of f32 additions in a row before 64 bits take over (u =
2^-24): with |x - m| e^(x - m) <= 0.37 below 3e-6 together, and the result's own
rounding u |sum|.  Tokens of one row are in the order of their logits whatever
the sum; the inputs' sums of different rows lie further apart than 1e-5 where
they are compared (checked in the reference), or are equal bit for bit.
"""
import numpy as np
import pytest

import static_lm as S

pytestmark = pytest.mark.gpu

TOL, GAP = 4e-6, 1e-5


def select_reference(logits, scores, beams, out, ended=None, end_token=0):
    """[groups][out] sums, rows and tokens, in 64 bits; and the least gap that the order hangs on."""
    groups = len(scores) // beams
    x = logits.astype(np.float64)
    x[np.isnan(x)] = -np.inf
    found, gap = [], np.inf
    for g in range(groups):
        cand = []
        for r in range(g * beams, (g + 1) * beams):
            if not np.isfinite(scores[r]):
                continue
            if ended is not None and ended[r]:
                cand.append((-float(scores[r]), r, 0.0, end_token))
                continue
            top = x[r].max()
            if not np.isfinite(top):
                continue
            lse = top + np.log(np.exp(x[r] - top).sum())
            # as many of the row as can be among the best, ties by the lower token
            order = np.argsort(-x[r], kind="stable")[:out + 1]
            cand += [(-(float(scores[r]) + (x[r, t] - lse)), r, -x[r, t], int(t)) for t in order if x[r, t] > -np.inf]
        cand.sort()
        for a, b in zip(cand[:out], cand[1:out + 1]):
            if a[1] != b[1] and a[0] != b[0]:
                gap = min(gap, b[0] - a[0])
        cand = [(-c, r, t) for c, r, _, t in cand[:out]]
        found.append(cand + [(-np.inf, -1, -1)] * (out - len(cand)))
    found = np.array(found)
    return found[..., 0], found[..., 1].astype(int), found[..., 2].astype(int), gap


def select(torch, logits, scores, beams, out, ended=None, end_token=0, vocab=None, stream=None, in_place=False, fill=0xFF):
    groups = scores.numel() // beams
    o = [torch.full((groups, out), 7, dtype=t, device="cuda") for t in (torch.float32, torch.int32, torch.int32)]
    args = S.BeamSelectArgs(logits=logits.data_ptr(), ld=logits.stride(0), scores=scores.data_ptr(),
                            ended=None if ended is None else ended.data_ptr(), num_groups=groups, beams=beams,
                            vocab=vocab or logits.shape[1], num_out=out, end_token=end_token,
                            out_scores=(scores if in_place else o[0]).data_ptr(), out_rows=o[1].data_ptr(),
                            out_tokens=o[2].data_ptr())
    size = S.beam_select_scratch_bytes(args)
    scratch = torch.full((size + 16,), fill, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    S.beam_select(args, scratch.data_ptr(), size, stream.cuda_stream if stream else torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert (scratch[size:] == fill).all(), "wrote past the scratch"
    if in_place:
        o[0] = scores.view(groups, out)
    return [t.cpu().numpy() for t in o]


def check(got, want):
    scores, rows, tokens, gap = want
    assert gap > GAP, "the inputs do not decide the order"
    assert np.array_equal(got[1], rows) and np.array_equal(got[2], tokens)
    inf = np.isinf(scores)
    assert np.array_equal(np.isinf(got[0]), inf) and (got[0][inf] == -np.inf).all()
    assert (np.abs(got[0][~inf] - scores[~inf]) <= TOL + 2.0 ** -23 * np.abs(scores[~inf])).all()


SELECTS = [  # groups, beams, vocab, out, pad
    (1, 1, 1, 1, 0),
    (1, 4, 49152, 4, 0),
    (3, 2, 17, 8, 0),
    (2, 3, 5, 20, 3),          # fewer candidates than places
    (5, 5, 4097, 10, 0),       # rows off 16-byte boundaries
    (2, 8, 4096, 16, 4),
    (1, 16, 131072, 32, 0),
    (40, 4, 20001, 8, 3),
    (1, 1, 300000, 64, 0),
    (1, 70, 1000, 64, 0),      # many rows in a group
    (300, 2, 700, 3, 0),
    (1, 256, 40, 5, 0),
]


def inputs(torch, groups, beams, vocab, pad, seed):
    g = torch.Generator().manual_seed(seed)
    wide = 3 * torch.randn(groups * beams, vocab + pad, generator=g)
    return wide, -20 + 1.5 * torch.randn(groups * beams, generator=g)


@pytest.mark.parametrize("case", range(len(SELECTS)))
def test_select(cuda, case):
    groups, beams, vocab, out, pad = SELECTS[case]
    wide, scores = inputs(cuda, groups, beams, vocab, pad, case)
    want = select_reference(wide[:, :vocab].numpy(), scores.numpy(), beams, out)
    logits = wide.cuda()
    got = select(cuda, logits, scores.cuda(), beams, out, vocab=vocab)
    check(got, want)
    again = select(cuda, logits, scores.cuda(), beams, out, vocab=vocab, fill=0)
    assert all(np.array_equal(a, b) for a, b in zip(got, again)), "not the same bits again"


@pytest.mark.parametrize("shape", ["rising", "falling", "equal", "two values", "steps", "few", "peak", "zeros of both signs"])
@pytest.mark.parametrize("out", [1, 4, 64])
def test_orders_of_the_logits(cuda, shape, out):
    """Long runs that pass the threshold, ties by the hundred, and rows with hardly a candidate."""
    vocab, beams = 50001, 2
    t = np.arange(vocab, dtype=np.float32)
    x = np.stack([{"rising": t * 1e-3, "falling": -t * 1e-3, "equal": 0 * t, "two values": np.float32(t % 97 == 5),
                   "steps": t // 1000, "few": np.where(t % 9999 == 1, t, -np.inf), "peak": np.where(t == 44444, 90, 0 * t),
                   "zeros of both signs": np.where(t % 2 == 0, -0.0, 0.0)}[shape]] * beams).astype(np.float32)
    scores = np.array([-3.0, -3.25], np.float32)
    got = select(cuda, cuda.from_numpy(x).cuda(), cuda.from_numpy(scores).cuda(), beams, out)
    want = select_reference(x, scores, beams, out)
    check(got, want)


def test_ties_between_rows_go_to_the_lower_row(cuda):
    g = cuda.Generator().manual_seed(4)
    one = cuda.randn(1, 30000, generator=g)
    x = one.repeat(6, 1)
    scores = cuda.full((6,), -1.5)
    got = select(cuda, x.cuda(), scores.cuda(), 3, 7)
    want = select_reference(x.numpy(), scores.numpy(), 3, 7)
    check(got, want)
    assert got[1].tolist() == [[0, 1, 2, 0, 1, 2, 0], [3, 4, 5, 3, 4, 5, 3]]


@pytest.mark.parametrize("groups,beams,vocab,out", [(1, 1, 131072, 40), (1, 2, 49152, 8), (2, 64, 20000, 8), (1, 200, 9000, 33)])
def test_sums_that_are_equal_go_by_row_and_logit(cuda, groups, beams, vocab, out):
    """Scores beside which no log probability shows: every sum of a row is equal, wherever its tokens lie."""
    torch = cuda
    rng = np.random.default_rng(21)
    x = rng.standard_normal((groups * beams, vocab)).astype(np.float32)
    for row in x[::beams]:  # a group's first row has fewer tokens
        row[np.argsort(-row)[out // 2:]] = -np.inf
    scores = np.full(groups * beams, -1e20, np.float32)
    want = select_reference(x, scores, beams, out)
    got = select(torch, torch.tensor(x, device="cuda"), torch.tensor(scores, device="cuda"), beams, out)
    assert np.array_equal(got[1], want[1]) and np.array_equal(got[2], want[2])
    assert np.array_equal(got[0], want[0].astype(np.float32))


def test_beams_that_ended_or_are_not_used(cuda):
    beams, vocab = 4, 5000
    wide, scores = inputs(cuda, 4, beams, vocab, 0, 11)
    ended = cuda.zeros(16, dtype=cuda.int32)
    ended[1] = 1
    ended[4:8] = 1                           # every beam of the group
    scores[9:12] = -float("inf")             # the first step: one beam
    scores[12:16] = cuda.tensor([float("nan"), float("inf"), -float("inf"), -2.0])
    ended[14] = 1                            # ended and not used
    wide[1] = float("nan")                   # not read
    want = select_reference(wide.numpy(), scores.numpy(), beams, 6, ended.numpy(), 77)
    got = select(cuda, wide.cuda(), scores.cuda(), beams, 6, ended.cuda(), 77)
    check(got, want)
    assert (got[2][1] == [77] * 4 + [-1] * 2).all() and (got[1][1, 4:] == -1).all()
    assert (got[1][2] == 8).all() and (got[1][3] == 15).all()


def test_logits_that_are_not_finite(cuda):
    beams, vocab = 3, 9000
    wide, scores = inputs(cuda, 3, beams, vocab, 0, 12)
    nan, inf = float("nan"), float("inf")
    wide[0, ::7] = nan
    wide[1, 1:] = -inf        # one candidate, of probability one
    wide[2, 100:8000] = -inf
    wide[3, 4000] = inf       # no candidates
    wide[4] = -inf
    wide[5] = nan
    wide[6] = 3e38            # the largest there are
    wide[7] = -3e38
    wide[8, ::2] = 3e38
    want = select_reference(np.where(np.isnan(wide.numpy()), -np.inf, wide.numpy()), scores.numpy(), beams, 10)
    got = select(cuda, wide.cuda(), scores.cuda(), beams, 10)
    assert (got[1][1] == -1).all() and (got[2][1] == -1).all()
    check(got, want)


def test_scores_in_place_on_another_stream(cuda):
    wide, scores = inputs(cuda, 6, 4, 3001, 3, 13)
    want = select_reference(wide[:, :3001].numpy(), scores.numpy(), 4, 4)
    check(select(cuda, wide.cuda(), scores.cuda(), 4, 4, vocab=3001, stream=cuda.cuda.Stream(), in_place=True), want)


# -------------------------------------------------------------------- fork


def pools(torch, kv, layers, num_pages, kvh, page, hd, seed):
    """[page][layer][k, v][bytes] and its descriptors."""
    g = torch.Generator().manual_seed(seed)
    el = {"f32": 4, "f16": 2, "bf16": 2, "q8": 1}[kv]
    one = -(-kvh * page * (hd + 4) // 16) * 16 if kv == "q8" else kvh * page * hd * el
    pool = torch.randint(0, 256, (num_pages, layers, 2, one), dtype=torch.uint8, generator=g).cuda()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    code = S.KV_Q8 if kv == "q8" else S.KV_DTYPES[kv]
    pages = [S.KvPages(k=pool[0, i, 0].data_ptr(), v=pool[0, i, 1].data_ptr(), page_stride=layers * 2 * one // el,
                       num_pages=num_pages, page_size=page, num_kv_heads=kvh, head_dim=hd, dtype=code,
                       status=status.data_ptr()) for i in range(layers)]
    return pool, pages, status


def slots(pool, kv, kvh, page, hd):
    """Views [page][layer][2][kv_head][slot][bytes] of the elements, and of the scales."""
    el = {"f32": 4, "f16": 2, "bf16": 2, "q8": 1}[kv]
    n = kvh * page * hd * el
    shape = (*pool.shape[:3], kvh, page)
    views = [pool[..., :n].view(*shape, hd * el)]
    if kv == "q8":
        views.append(pool[..., n:n + kvh * page * 4].view(*shape, 4))
    return views


def fork_reference(table, kv_len, parent, spare, num_pages, page, views):
    """Tables, lengths, taken; copies the slots in the views."""
    stride, seen = table.shape[1], set()
    out = np.full((len(parent), stride), -1, np.int32)
    lens, taken = np.zeros(len(parent), np.int32), np.zeros(len(parent), np.int32)
    for i, p in enumerate(parent):
        if p < 0 or p >= len(kv_len):
            continue
        n = lens[i] = max(kv_len[p], 0)
        t, used = n // page, n % page
        first = p not in seen
        seen.add(p)
        out[i] = table[p] if first else np.where(np.arange(stride) < t, table[p], -1)
        if t >= stride:
            continue
        ok = spare is not None and 0 <= spare[i] < num_pages
        if used == 0 and (not first or table[p, t] < 0):
            out[i, t] = spare[i] if ok else -1
            taken[i] = ok
        if used and not first and 0 <= table[p, t] < num_pages:
            out[i, t] = spare[i] if ok else -1
            taken[i] = ok
            if ok:
                for v in views:
                    v[spare[i], :, :, :, :used] = v[table[p, t], :, :, :, :used]
    return out, lens, taken


def fork(torch, pages, table, kv_len, parent, spare, want_taken=True, stream=None):
    dev = [None if a is None else torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda() for a in (parent, kv_len, table, spare)]
    n, stride = len(parent), table.shape[1]
    out = [torch.full(s, 99, dtype=torch.int32, device="cuda") for s in ((n, stride), (n,), (n,))]
    args = S.PagedForkArgs(parent=dev[0].data_ptr(), kv_len=dev[1].data_ptr(), page_table=dev[2].data_ptr(),
                           spare=None if spare is None else dev[3].data_ptr(), page_table_out=out[0].data_ptr(),
                           kv_len_out=out[1].data_ptr(), taken=out[2].data_ptr() if want_taken else None, table_stride=stride,
                           num_seqs=len(kv_len), num_new=n)
    torch.cuda.synchronize()
    S.paged_fork(pages, args, stream.cuda_stream if stream else torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    return [t.cpu().numpy() for t in out]


FORKS = [  # kv, layers, kv_heads, hd, page, lengths, parents
    ("f16", 1, 2, 64, 16, [5], [0, 0, 0]),
    ("q8", 3, 3, 64, 16, [40, 33, 32], [0, 0, 1, 1, 2, 2]),
    ("q8", 2, 1, 16, 7, [6, 7, 8, 13], [3, 3, 2, 2, 1, 1, 0, 0]),
    ("f32", 65, 1, 8, 4, [9, 3], [1, 0, 1, 0]),          # more layers than a launch takes
    ("bf16", 130, 2, 32, 5, [12, 4, 9], [2, -1, 2, 2, 0]),
    ("q8", 4, 8, 128, 32, [100, 64, 1, 31], [0, 2, 0, 2, 0, 2, 3, 3]),
    ("f16", 2, 4, 48, 24, [1, 0], [1, 1, 0, 0]),
    ("f32", 2, 2, 128, 1, [3, 2], [0, 1, 0, 1]),
    ("bf16", 1, 1, 64, 16, [17] * 300, list(range(299, -1, -1)) + [0, 299, 150] * 20),
]


@pytest.mark.parametrize("case", range(len(FORKS)))
def test_fork(cuda, case):
    kv, layers, kvh, hd, page, lengths, parent = FORKS[case]
    need = [-(-n // page) for n in lengths]
    stride = max(need) + 1
    num_pages = sum(need) + len(parent) + 2
    ids = np.random.default_rng(case).permutation(num_pages).astype(np.int32)
    table, at = np.full((len(lengths), stride), -1, np.int32), 0
    for s, k in enumerate(need):
        table[s, :k] = ids[at:at + k]
        at += k
    spare = ids[at:at + len(parent)]
    pool, pages, status = pools(cuda, kv, layers, num_pages, kvh, page, hd, case)
    want_pool = pool.clone()
    want = fork_reference(table, lengths, parent, spare, num_pages, page, slots(want_pool, kv, kvh, page, hd))
    got = fork(cuda, pages, table, lengths, parent, spare, stream=cuda.cuda.Stream() if case % 2 else None)
    for a, b in zip(got, want):
        assert np.array_equal(a, b)
    assert cuda.equal(pool, want_pool) and int(status) == 0
    # again over its own result: the same copies
    assert np.array_equal(fork(cuda, pages, table, lengths, parent, spare, want_taken=False)[0], want[0])
    assert cuda.equal(pool, want_pool)


def test_fork_keeps_pages_held_ahead_and_lacks_what_is_not_held(cuda):
    pool, pages, status = pools(cuda, "f16", 1, 12, 1, 4, 8, 1)
    # 0: pages held past its length; 1: full, and none held for the next position; 2: its last page given back
    table = np.array([[0, 1, 2, -1], [3, 4, -1, -1], [5, -1, -1, -1], [-1, -1, -1, -1]], np.int32)
    lengths, parent, spare = [6, 8, 6, 0], [0, 0, 1, 1, 2, 2, 3], [6, 7, 8, 9, 10, 11, 6]
    want = fork_reference(table, lengths, parent, spare, 12, 4, slots(pool.clone(), "f16", 1, 4, 8))
    got = fork(cuda, pages, table, lengths, parent, spare)
    assert all(np.array_equal(a, b) for a, b in zip(got, want)) and int(status) == 0
    assert got[0].tolist()[:4] == [[0, 1, 2, -1], [0, 7, -1, -1], [3, 4, 8, -1], [3, 4, 9, -1]]
    assert got[2].tolist() == [0, 1, 1, 1, 0, 0, 1]


def test_fork_flags_what_it_cannot_do(cuda):
    for table, length, parent, spare, bit in (
            ([[0, 1]], 6, [0, 0], [4, -1], 1),       # no page to copy into
            ([[0, 1]], 6, [0, 0], None, 1),
            ([[0, 1]], 6, [0, 0], [4, 12], 1),       # an id past the pool
            ([[0, 12]], 6, [0, 0], [4, 5], 1),       # the parent's
            ([[0, 1]], 6, [0, 1], [4, 5], 8),        # a parent past the sequences
            ([[0, 1]], 9, [0, 0], [4, 5], 2),        # a length past the table
            ([[0, 1]], 8, [0, 0], None, 0),          # the table's end: nothing to give
            ([[0, -1]], 4, [0, 0], None, 0),         # a page is not needed yet
            ([[0, -1]], 4, [0, 0], [-1, -1], 0)):
        pool, pages, status = pools(cuda, "q8", 2, 12, 1, 4, 16, 1)
        keep = pool.clone()
        want = fork_reference(np.array(table, np.int32), [length], parent, spare, 12, 4, [])
        got = fork(cuda, pages, np.array(table, np.int32), [length], parent, spare)
        assert int(status) == bit and cuda.equal(pool, keep)
        assert all(np.array_equal(a, b) for a, b in zip(got, want))


def test_select_and_fork_captured_and_replayed(cuda):
    """A step of a search on the device: the rows that were selected are the parents."""
    groups, beams, vocab, kvh, page, hd = 3, 4, 2500, 2, 8, 32
    n, stride = groups * beams, 6
    pool, pages, status = pools(cuda, "q8", 3, n * stride + n, kvh, page, hd, 2)
    table = np.arange(n * stride, dtype=np.int32).reshape(n, stride)
    spare = np.arange(n * stride, n * stride + n, dtype=np.int32)
    lengths = np.repeat([13, 40, 7], beams).astype(np.int32)
    dev = {k: cuda.from_numpy(v).cuda() for k, v in (("table", table), ("spare", spare), ("len", lengths))}
    logits, scores = (t.cuda() for t in inputs(cuda, groups, beams, vocab, 0, 21))
    rows, tokens, new_len, taken = (cuda.zeros(n, dtype=cuda.int32, device="cuda") for _ in range(4))
    new_scores, new_table = cuda.zeros(n, device="cuda"), cuda.zeros(n, stride, dtype=cuda.int32, device="cuda")
    pick = S.BeamSelectArgs(logits=logits.data_ptr(), ld=vocab, scores=scores.data_ptr(), num_groups=groups, beams=beams,
                            vocab=vocab, num_out=beams, out_scores=new_scores.data_ptr(), out_rows=rows.data_ptr(),
                            out_tokens=tokens.data_ptr())
    go = S.PagedForkArgs(parent=rows.data_ptr(), kv_len=dev["len"].data_ptr(), page_table=dev["table"].data_ptr(),
                         spare=dev["spare"].data_ptr(), kv_len_out=new_len.data_ptr(), page_table_out=new_table.data_ptr(),
                         taken=taken.data_ptr(), table_stride=stride, num_seqs=n, num_new=n)
    size = S.beam_select_scratch_bytes(pick)
    scratch = cuda.empty(size, dtype=cuda.uint8, device="cuda")
    graph = cuda.cuda.CUDAGraph()
    with cuda.cuda.graph(graph):
        stream = cuda.cuda.current_stream().cuda_stream
        S.beam_select(pick, scratch.data_ptr(), size, stream)
        S.paged_fork(pages, go, stream)
    for seed in (21, 22, 23):
        x, s = inputs(cuda, groups, beams, vocab, 0, seed)
        logits.copy_(x), scores.copy_(s)
        want_pool = pool.clone()
        graph.replay()
        cuda.cuda.synchronize()
        want = select_reference(x.numpy(), s.numpy(), beams, beams)
        check([t.cpu().numpy().reshape(groups, beams) for t in (new_scores, rows, tokens)], want)
        tables = fork_reference(table, lengths, want[1].reshape(-1), spare, pool.shape[0], page, slots(want_pool, "q8", kvh, page, hd))
        assert all(np.array_equal(a.cpu().numpy(), b) for a, b in zip((new_table, new_len, taken), tables))
        assert cuda.equal(pool, want_pool) and int(status) == 0


def test_fork_of_pages_far_apart(cuda):
    """Pages further apart than 2^31 bytes."""
    kvh, page, hd = 2, 16, 64
    far, one = (1 << 31) + 4096, kvh * page * (hd + 4)
    pool = cuda.zeros(2 * far + 2 * one, dtype=cuda.uint8, device="cuda")
    g = cuda.Generator().manual_seed(1)
    pool[:2 * one] = cuda.randint(0, 256, (2 * one,), dtype=cuda.uint8, generator=g).cuda()
    pages = [S.KvPages(k=pool.data_ptr(), v=pool.data_ptr() + one, page_stride=far, num_pages=3, page_size=page,
                       num_kv_heads=kvh, head_dim=hd, dtype=S.KV_Q8)]
    got = fork(cuda, pages, np.array([[0]], np.int32), [11], [0, 0, 0], [1, 1, 2])
    assert got[0].tolist() == [[0], [1], [2]] and got[2].tolist() == [0, 1, 1]
    for first in (far, 2 * far):
        for base in (0, one):
            a, b = pool[base:base + one], pool[first + base:first + base + one]
            x, y = (t[:kvh * page * hd].view(kvh, page, hd) for t in (a, b))
            assert cuda.equal(x[:, :11], y[:, :11]) and (y[:, 11:] == 0).all()
            x, y = (t[kvh * page * hd:].view(kvh, page, 4) for t in (a, b))
            assert cuda.equal(x[:, :11], y[:, :11]) and (y[:, 11:] == 0).all()


def test_two_selections_at_once(cuda):
    """On two streams, with a scratch each."""
    work = []
    for seed, (groups, beams, vocab, out) in enumerate(((5, 4, 30000, 8), (2, 3, 50000, 6))):
        wide, scores = inputs(cuda, groups, beams, vocab, 0, 30 + seed)
        logits, scores = wide.cuda(), scores.cuda()
        want = select(cuda, logits, scores, beams, out)
        o = [cuda.zeros(groups, out, dtype=t, device="cuda") for t in (cuda.float32, cuda.int32, cuda.int32)]
        args = S.BeamSelectArgs(logits=logits.data_ptr(), ld=vocab, scores=scores.data_ptr(), num_groups=groups, beams=beams,
                                vocab=vocab, num_out=out, out_scores=o[0].data_ptr(), out_rows=o[1].data_ptr(),
                                out_tokens=o[2].data_ptr())
        size = S.beam_select_scratch_bytes(args)
        work.append((args, cuda.empty(size, dtype=cuda.uint8, device="cuda"), size, cuda.cuda.Stream(), o, want, logits, scores))
    cuda.cuda.synchronize()
    for _ in range(20):
        for args, scratch, size, stream, *_ in work:
            S.beam_select(args, scratch.data_ptr(), size, stream.cuda_stream)
    cuda.cuda.synchronize()
    for *_, o, want, logits, scores in work:
        assert all(np.array_equal(t.cpu().numpy(), w) for t, w in zip(o, want))
