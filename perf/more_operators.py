"""8-bit pages of the paged key/value cache and beam search over it, as cases to measure.

store    new keys and values into 8-bit pages (per-head RMSNorm of q and k
         optional, rotary positions, quantisation on the way), and the same
         rows read back as f16
decode   attention of one new token per sequence over 8-bit pages
rows     attention of several new rows per sequence (a prompt, or a chunk of
         one behind an earlier context) over 8-bit pages
select   the best continuations of every group of beams over the vocabulary
fork     the page tables of the beams that go on, full pages shared, partly
         filled ones copied where a beam has several successors

An 8-bit page holds, for every (KV head, slot), head_dim signed bytes q and one
f32 scale: value = q scale, scale = max |x| / 127, q = x 127 / max |x| rounded
to the nearest (ties to even).  The bytes come first, [kv_head][slot][head_dim],
then the scales, [kv_head][slot]; pages lie a multiple of 16 bytes apart.
"""
import math
import os
import sys

import torch

own = False

F16, BF16, F32, Q8 = "f16", "bf16", "f32", "q8"
DTYPES = {F16: torch.float16, BF16: torch.bfloat16, F32: torch.float32}
EPS = 1e-5
THETA = 10000.0


def paged(name, op, seqs, heads, kv_heads, head_dim, page, ctx, new=(1, 1), window=0, sinks=0, norm=False, halves=False):
    """ctx: shortest and longest length of a sequence, its new rows included; new: fewest and most new rows."""
    return {"name": name, "op": op, "seqs": seqs, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "page": page,
            "ctx_min": ctx[0], "ctx_max": ctx[1], "new_min": new[0], "new_max": new[1], "window": window, "sinks": sinks,
            "norm": norm, "halves": halves}


def select(name, groups, beams, vocab, out, ended=0, banned=0):
    """ended: how many beams of each group have ended; banned: so many tokens of every row are at -infinity."""
    return {"name": name, "op": "select", "groups": groups, "beams": beams, "vocab": vocab, "out": out, "ended": ended,
            "banned": banned}


def fork(name, groups, beams, parents, layers, kv_heads, head_dim, kv, page, ctx):
    """parents: how many different beams of each group go on."""
    return {"name": name, "op": "fork", "groups": groups, "beams": beams, "parents": parents, "layers": layers,
            "kv_heads": kv_heads, "head_dim": head_dim, "kv": kv, "page": page, "ctx_min": ctx[0], "ctx_max": ctx[1]}


def listed():
    return [
        # one user's next token on the 8B shape, normed queries and keys: the smallest call
        paged("store-1", "store", 1, 32, 8, 128, 16, (2048, 2048), norm=True, halves=True),
        # eight prompts of 4096 tokens on the 135M shape
        paged("store-prompts", "store", 8, 9, 3, 64, 16, (4096, 4096), (4096, 4096)),
        # a first token of the 15M shape over a short context: latency
        paged("decode-1x77", "decode", 1, 6, 6, 48, 16, (77, 77)),
        # the 135M shape at 64 sequences of 2048 positions
        paged("decode-64x2048", "decode", 64, 9, 3, 64, 16, (2049, 2049)),
        # one long sequence on the 8B shape: the length has to be split
        paged("decode-1x8192", "decode", 1, 32, 8, 128, 16, (8192, 8192)),
        # a serving batch of unlike lengths on the 8B shape
        paged("decode-64-ragged", "decode", 64, 32, 8, 128, 32, (500, 8192)),
        # eight prompts of 4096 tokens on the 135M shape
        paged("rows-8x4096", "rows", 8, 9, 3, 64, 16, (4096, 4096), (4096, 4096)),
        # chunks of unlike lengths behind unlike contexts on the 8B shape
        paged("rows-chunks", "rows", 16, 32, 8, 128, 16, (600, 8192), (1, 512)),
        # one user's four beams, the 135M shape's vocabulary
        select("select-1x4", 1, 4, 49152, 4),
        # 64 users of four beams, a large vocabulary, twice as many candidates as beams
        select("select-64x4", 64, 4, 131072, 8, banned=5),
        # one user's four beams on the 15M shape
        fork("fork-1x4", 1, 4, 3, 6, 6, 48, F32, 16, (70, 70)),
        # 64 users of four beams on the 135M shape
        fork("fork-64x4", 64, 4, 2, 30, 3, 64, F16, 32, (200, 1000)),
    ]


SHAPES = [(9, 3, 64), (9, 3, 64), (6, 6, 48), (4, 4, 64), (32, 8, 128), (32, 8, 128), (12, 2, 80), (20, 4, 96),
          (16, 1, 64), (8, 8, 32)]


def draw(rng):
    def spread(lo, hi):
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))

    while True:
        op = rng.choice(["store", "decode", "rows", "select", "fork"])
        if op == "select":
            groups, beams, vocab = spread(1, 128), spread(1, 16), spread(257, 131072)
            out = spread(1, min(32, 2 * beams + 1))
            c = select("", groups, beams, vocab, out, rng.choice([0, 0, rng.randrange(beams)]), rng.choice([0, 3, 40]))
            ok = groups * beams * vocab <= 32e6
        elif op == "fork":
            heads, kv_heads, head_dim = rng.choice(SHAPES)
            groups, beams = spread(1, 128), spread(1, 16)
            hi = spread(1, 2000)
            c = fork("", groups, beams, rng.randint(1, beams), spread(1, 32), kv_heads, head_dim, rng.choice([F16, BF16, F32]),
                     rng.choice([8, 16, 16, 24, 32]), (rng.choice([hi, max(1, hi // 3)]), hi))
            el = 4 if c["kv"] == F32 else 2
            pages = groups * (-(-hi // c["page"]) + 2 * beams)
            ok = pages * c["layers"] * 2 * el * kv_heads * c["page"] * head_dim <= 2e9 and work(c)["bytes"] <= 90e6
        else:
            heads, kv_heads, head_dim = rng.choice(SHAPES)
            page = rng.choice([8, 16, 16, 24, 32, 64])
            seqs = spread(1, 32 if op == "rows" else 128)
            hi = spread(2, 8192)
            lo = rng.choice([hi, max(1, hi // rng.randint(2, 9))])
            new = (1, 1)
            if op != "decode":
                most = rng.choice([lo, spread(1, lo)])
                new = (rng.choice([most, 1]), most)
                if op == "store" and rng.random() < 0.3:
                    new = (1, 1)
            window, sinks = 0, 0
            if op != "store" and rng.random() < 0.5:
                window, sinks = spread(1, 2048), rng.choice([0, 1, 4, 16, 37])
            c = paged("", op, seqs, heads, kv_heads, head_dim, page, (lo, hi), new, window, sinks,
                      op == "store" and rng.random() < 0.5, op == "store" and rng.random() < 0.5)
            w, rows = work(c), _rows(c)
            if op == "store":
                ok = sum(rows) <= 32768 and w["bytes"] <= 210e6 and seqs * hi * kv_heads * head_dim <= 270e6
            elif op == "decode":
                ok = w["bytes"] <= 590e6 and seqs * hi * kv_heads * head_dim <= 540e6
            else:
                ok = w["flops"] <= 1.2e11 and seqs * max(rows) * heads * hi <= 2.1e9
        if ok:
            del c["name"]
            return c


# ------------------------------------------------------------------ lengths


def _spread(n, lo, hi, step):
    """n whole numbers spread over [lo, hi], the same for every seed; both ends are among them where n allows."""
    v = [lo + int((hi - lo + 1) * ((i * step) % 1.0)) for i in range(n)]
    v[-1] = hi
    return v


def _lengths(c):
    return _spread(c["seqs"] if "seqs" in c else c["groups"], c["ctx_min"], c["ctx_max"], 0.6180339887)


def _rows(c):
    return [min(r, n) for r, n in zip(_spread(c["seqs"], c["new_min"], c["new_max"], 0.7548776662), _lengths(c))]


def _seen(p, window, sinks):
    """Keys visible to a row at position p."""
    if not window or p + 1 <= window:
        return p + 1
    return window + min(sinks, p + 1 - window)


def work(c):
    if c["op"] == "select":
        rows = c["groups"] * (c["beams"] - c["ended"])  # the logits of a beam that has ended are not needed
        return {"bytes": 4 * rows * c["vocab"] + 12 * c["groups"] * c["out"], "flops": 4 * rows * c["vocab"]}
    if c["op"] == "fork":
        el, lengths = (4 if c["kv"] == F32 else 2), _lengths(c)
        one = 2 * el * c["layers"] * c["kv_heads"] * c["head_dim"]  # a position's keys and values
        copied = (c["beams"] - c["parents"]) * sum(n % c["page"] for n in lengths)
        table = 4 * c["groups"] * c["beams"] * _table_width(c)
        return {"bytes": 2 * one * copied + 2 * table, "flops": 0}
    heads, kv_heads, hd = c["heads"], c["kv_heads"], c["head_dim"]
    lengths, rows = _lengths(c), _rows(c)
    n, held = sum(rows), kv_heads * (hd + 4)  # bytes of a position's keys
    if c["op"] == "store":
        # q, k, v in, q out, the pages written and read, k and v out as f16, the tables of angles
        return {"bytes": n * (4 * hd * (2 * heads + 2 * kv_heads) + 4 * held + 4 * kv_heads * hd + 4 * hd),
                "flops": n * hd * ((heads + kv_heads) * (3 + (4 if c["norm"] else 0)) + 6 * kv_heads)}
    pairs, keys = 0, 0
    for length, r in zip(lengths, rows):
        first, w = length - r, c["window"]
        if not w:
            pairs += r * first + r * (r + 1) // 2
            keys += length
        else:
            pairs += sum(_seen(p, w, c["sinks"]) for p in range(first, length))
            low = max(0, first - w + 1)
            keys += length - low + min(c["sinks"], low)
    return {"bytes": 8 * n * heads * hd + 2 * keys * held, "flops": 4 * pairs * heads * hd}


# ------------------------------------------------------------------- inputs


def _page_bytes(c):
    return -(-c["kv_heads"] * c["page"] * (c["head_dim"] + 4) // 16) * 16


def _parts(c, pool):
    """The bytes [page][kv_head][slot][head_dim] and the scales [page][kv_head][slot] of a pool of 8-bit pages."""
    n = c["kv_heads"] * c["page"]
    return (pool[:, :n * c["head_dim"]].view(torch.int8).view(-1, c["kv_heads"], c["page"], c["head_dim"]),
            pool[:, n * c["head_dim"]:n * (c["head_dim"] + 4)].view(torch.float32).view(-1, c["kv_heads"], c["page"]))


def _quantised(x):
    """x [.., head_dim] as bytes and scales."""
    top = x.abs().amax(-1)
    up = torch.where(top > 0, 127.0 / top, 0.0)
    return torch.round(x * up[..., None]).to(torch.int8), top / 127.0


def _pool(c, pages, g):
    pool = torch.zeros(pages, _page_bytes(c), dtype=torch.uint8, device="cuda")
    q, scale = _parts(c, pool)
    step = max(1, (1 << 26) // (q[0].numel()))
    for i in range(0, pages, step):
        q[i:i + step], scale[i:i + step] = _quantised(torch.randn(q[i:i + step].shape, generator=g, device="cuda"))
    return pool


def _table_width(c):
    return -(-max(_lengths(c)) // c["page"]) + 1


def _prepare_select(c, g):
    rows = c["groups"] * c["beams"]
    logits = torch.empty(rows, c["vocab"], device="cuda").normal_(0.0, 3.0, generator=g)
    if c["banned"]:
        logits.scatter_(1, torch.randint(c["vocab"], (rows, c["banned"]), generator=g, device="cuda"), -math.inf)
    # the sums of beams that are some steps old lie near each other
    scores = -20.0 + 1.5 * torch.randn(rows, generator=g, device="cuda")
    ended = torch.zeros(c["groups"], c["beams"], dtype=torch.int32, device="cuda")
    if c["ended"]:
        which = torch.rand(c["groups"], c["beams"], generator=g, device="cuda").argsort(1)[:, :c["ended"]]
        ended.scatter_(1, which, 1)
    out = lambda t: torch.zeros(c["groups"], c["out"], dtype=t, device="cuda")  # noqa: E731
    return {"logits": logits, "scores": scores, "ended": ended.view(-1), "out_scores": out(torch.float32),
            "out_rows": out(torch.int32), "out_tokens": out(torch.int32)}


def _prepare_fork(c, g):
    groups, beams, page, dev = c["groups"], c["beams"], c["page"], "cuda"
    n, width, lengths = groups * beams, _table_width(c), torch.tensor(_lengths(c), device=dev)
    full = lengths // page  # pages of a group that its beams share; each has a last page and a spare one of its own
    pages = int(full.sum()) + 2 * n
    ids = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    at = torch.arange(width, device=dev)
    shared = torch.where(at < full[:, None], ids[((full.cumsum(0) - full)[:, None] + at).clamp(max=pages - 1)], -1)
    table = shared.repeat_interleave(beams, 0)
    mine = ids[int(full.sum()):]
    table.scatter_(1, full.repeat_interleave(beams)[:, None], mine[:n, None])
    # `parents` beams of each group go on, every one of them at least once
    alive = torch.rand(groups, beams, generator=g, device=dev).argsort(1)[:, :c["parents"]]
    pick = torch.randint(c["parents"], (groups, beams), generator=g, device=dev)
    pick[:, :c["parents"]] = torch.arange(c["parents"], device=dev)
    pick = pick.gather(1, torch.rand(groups, beams, generator=g, device=dev).argsort(1))
    parent = alive.gather(1, pick) + beams * torch.arange(groups, device=dev)[:, None]
    pool = torch.empty(pages, c["layers"], 2, c["kv_heads"], page, c["head_dim"], dtype=DTYPES[c["kv"]], device=dev)
    pool.normal_(generator=g)
    return {"pool": pool, "table": table.contiguous(), "kv_len": lengths.repeat_interleave(beams).to(torch.int32),
            "parent": parent.reshape(-1).to(torch.int32), "spare": mine[n:].contiguous(),
            "table_out": torch.zeros(n, width, dtype=torch.int32, device=dev),
            "len_out": torch.zeros(n, dtype=torch.int32, device=dev), "taken": torch.zeros(n, dtype=torch.int32, device=dev)}


def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(1000003 * (seed + 1))
    if c["op"] in ("select", "fork"):
        return {"case": dict(c), **(_prepare_select if c["op"] == "select" else _prepare_fork)(c, g)}
    dev = "cuda"
    heads, kv_heads, hd, page = c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    lengths, rows = _lengths(c), _rows(c)
    n, longest = sum(rows), max(lengths)
    per_seq = -(-longest // page)
    need = [-(-length // page) for length in lengths]
    pages = sum(need) + 3
    # pages in no order, as a pool that has been in use hands them out
    ids = torch.randperm(pages, generator=g, device=dev, dtype=torch.int64).to(torch.int32)
    need_t = torch.tensor(need, device=dev)
    at = torch.arange(per_seq, device=dev)[None, :]
    start = (need_t.cumsum(0) - need_t)[:, None]
    table = torch.where(at < need_t[:, None], ids[torch.clamp(start + at, max=pages - 1)], -1).to(torch.int32)
    rand = lambda *shape: torch.randn(*shape, generator=g, device=dev)  # noqa: E731
    s = {"case": dict(c), "table": table.contiguous(), "pages": pages, "longest": longest,
         "kv_len": torch.tensor(lengths, dtype=torch.int32, device=dev),
         "row_start": torch.tensor([0] + rows, device=dev).cumsum(0).to(torch.int32),
         "k_pool": _pool(c, pages, g), "v_pool": _pool(c, pages, g)}
    if c["op"] == "store":
        # one projection's output: q, k and v of a row side by side
        s["qkv"] = rand(n, (heads + 2 * kv_heads) * hd)
        s["q_out"] = torch.zeros(n, heads * hd, device=dev)
        s["k_out"], s["v_out"] = (torch.zeros(n, kv_heads * hd, dtype=torch.float16, device=dev) for _ in range(2))
        angle = torch.arange(longest, dtype=torch.float64)[:, None] * THETA ** (
            -torch.arange(0, hd, 2, dtype=torch.float64) / hd)[None, :]
        s["cos"], s["sin"] = angle.cos().float().to(dev), angle.sin().float().to(dev)
        s["q_norm"], s["k_norm"] = 1 + 0.1 * rand(hd), 1 + 0.1 * rand(hd)
    else:
        s["q"] = 1.5 * rand(n, heads * hd)
        s["out"] = torch.zeros(n, heads * hd, device=dev)
    return s


# ---------------------------------------------------------------- plain form


def _place(s):
    """Sequence and position of every row."""
    start = s["row_start"].long()
    row = torch.arange(int(sum(_rows(s["case"]))), device=start.device)
    seq = torch.searchsorted(start, row, right=True) - 1
    pos = s["kv_len"].long()[seq] - start[seq + 1] + row
    return seq, pos


def _plain_store(s):
    c = s["case"]
    heads, kv_heads, hd, page = c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    seq, pos = _place(s)
    x = s["qkv"].view(len(seq), heads + 2 * kv_heads, hd)
    q, k, v = x.split([heads, kv_heads, kv_heads], 1)
    if c["norm"]:
        q = q * torch.rsqrt((q * q).mean(-1, keepdim=True) + EPS) * s["q_norm"]
        k = k * torch.rsqrt((k * k).mean(-1, keepdim=True) + EPS) * s["k_norm"]
    cos, sin = s["cos"][pos][:, None, :], s["sin"][pos][:, None, :]

    def turn(t):
        if c["halves"]:
            a, b = t[..., :hd // 2], t[..., hd // 2:]
            return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
        a, b = t[..., 0::2], t[..., 1::2]
        return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)

    s["q_out"].copy_(turn(q).reshape(len(seq), heads * hd))
    at, slot = s["table"][seq, pos // page].long(), pos % page
    for x, pool, out in ((turn(k), "k_pool", "k_out"), (v, "v_pool", "v_out")):
        held, scale = _parts(c, s[pool])
        held[at, :, slot], scale[at, :, slot] = _quantised(x)
        s[out].copy_((held[at, :, slot].float() * scale[at, :, slot][..., None]).reshape(len(seq), kv_heads * hd))
    return {"q": s["q_out"], "k": s["k_out"], "v": s["v_out"]}


def _plain_attention(s):
    c = s["case"]
    heads, kv_heads, hd = c["heads"], c["kv_heads"], c["head_dim"]
    group, seqs = heads // kv_heads, c["seqs"]
    seq, pos = _place(s)
    start = s["row_start"].long()
    most = max(_rows(c))
    col = torch.arange(len(seq), device=seq.device) - start[seq]
    q = torch.zeros(seqs, most, heads * hd, device=seq.device)
    q[seq, col] = s["q"]
    q = q.view(seqs, most, kv_heads, group, hd).permute(0, 2, 3, 1, 4).reshape(seqs, kv_heads, group * most, hd)
    table = s["table"].long().clamp(min=0)

    def gather(pool):
        held, scale = _parts(c, pool)
        x = held[table].permute(0, 2, 1, 3, 4).reshape(seqs, kv_heads, -1, hd).float()
        return x.mul_(scale[table].permute(0, 2, 1, 3).reshape(seqs, kv_heads, -1, 1))

    at = torch.full((seqs, most), -1, device=seq.device, dtype=torch.long)
    at[seq, col] = pos
    j = torch.arange(table.shape[1] * c["page"], device=seq.device)
    seen = j <= at[..., None]
    if c["window"]:
        seen &= (at[..., None] - j < c["window"]) | (j < c["sinks"])
    p = (q @ gather(s["k_pool"]).transpose(-1, -2)).mul_(1.0 / math.sqrt(hd)).view(seqs, kv_heads, group, most, -1)
    p.masked_fill_(~seen[:, None, None], -math.inf)
    top = p.amax(-1, keepdim=True).clamp_(min=torch.finfo(torch.float32).min)
    p = p.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = p.view(seqs, kv_heads, group * most, -1) @ gather(s["v_pool"])
    out = out.view(seqs, kv_heads, group, most, hd) / torch.where(total == 0, 1.0, total)
    out = out.permute(0, 3, 1, 2, 4).reshape(seqs, most, heads * hd)
    s["out"].copy_(out[seq, col])
    return {"out": s["out"]}


def _plain_select(s):
    """In 64 bits: which of two candidates of different beams is the better one hangs on the last bits of their sums."""
    c = s["case"]
    groups, beams, vocab = c["groups"], c["beams"], c["vocab"]
    x = s["logits"].double()
    top = x.amax(1, keepdim=True)
    total = top + (x - top).exp_().sum(1, keepdim=True).log_()
    x = x.sub_(total).add_(s["scores"].double()[:, None])
    # a beam that has ended proposes its end once more, at its own score
    last = torch.full_like(x, -math.inf)
    last[:, 0] = s["scores"].double()
    x = torch.where(s["ended"][:, None] != 0, last, x).view(groups, beams * vocab)
    best, at = torch.sort(x, dim=1, descending=True, stable=True)
    best, at = best[:, :c["out"]], at[:, :c["out"]]
    found = best > -math.inf
    row = at // vocab + beams * torch.arange(groups, device=at.device)[:, None]
    s["out_scores"].copy_(best)
    s["out_rows"].copy_(torch.where(found, row, -1))
    s["out_tokens"].copy_(torch.where(found, at % vocab, -1))
    return {"scores": s["out_scores"], "rows": s["out_rows"], "tokens": s["out_tokens"]}


def _plain_fork(s):
    c = s["case"]
    page, pool = c["page"], s["pool"]
    parent, n = s["parent"].long(), s["parent"].numel()
    length = s["kv_len"].long()[parent]
    tail, used = length // page, length % page
    i = torch.arange(n, device=parent.device)
    first = ~((parent[:, None] == parent[None, :]) & (i[None, :] < i[:, None])).any(1)
    j = torch.arange(s["table"].shape[1], device=parent.device)
    old = s["table"][parent]
    table = torch.where(first[:, None] | (j < tail[:, None]), old, -1)
    here = table.gather(1, tail[:, None])[:, 0]
    taken = here < 0
    table.scatter_(1, tail[:, None], torch.where(taken, s["spare"], here)[:, None])
    which = torch.nonzero(taken & (used > 0))[:, 0]
    slot = torch.arange(page, device=parent.device)
    keep = (slot[None, :] < used[which][:, None])[:, None, None, None, :, None]
    source, to = old.gather(1, tail[:, None])[which, 0].long(), s["spare"][which].long()
    pool[to] = torch.where(keep, pool[source], pool[to])
    s["table_out"].copy_(table)
    s["len_out"].copy_(length)
    s["taken"].copy_(taken)
    return {"table": s["table_out"], "kv_len": s["len_out"], "taken": s["taken"], "pool": pool}


PLAIN = {"store": _plain_store, "decode": _plain_attention, "rows": _plain_attention, "select": _plain_select,
         "fork": _plain_fork}


# --------------------------------------------------------- the framework's


def _package():
    path = os.path.join(os.getcwd(), "static-lm_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import static_lm
    return static_lm


def _plan(s):
    """The calls of one pass: the descriptors of this state's buffers and the scratch, as a program with fixed buffers keeps them."""
    S, c = _package(), s["case"]
    if c["op"] == "select":
        args = S.BeamSelectArgs(logits=s["logits"].data_ptr(), ld=c["vocab"], scores=s["scores"].data_ptr(),
                                ended=s["ended"].data_ptr(), num_groups=c["groups"], beams=c["beams"], vocab=c["vocab"],
                                num_out=c["out"], end_token=0, out_scores=s["out_scores"].data_ptr(),
                                out_rows=s["out_rows"].data_ptr(), out_tokens=s["out_tokens"].data_ptr())
        size = S.beam_select_scratch_bytes(args)
        s["scratch"] = torch.empty(max(size, 16), dtype=torch.uint8, device="cuda")
        return [(S.beam_select, (args, s["scratch"].data_ptr(), size))]
    if c["op"] == "fork":
        pool, layers = s["pool"], c["layers"]
        pages = [S.KvPages(k=pool[0, i, 0].data_ptr(), v=pool[0, i, 1].data_ptr(), page_stride=pool.stride(0),
                           num_pages=pool.shape[0], page_size=c["page"], num_kv_heads=c["kv_heads"], head_dim=c["head_dim"],
                           dtype=S.KV_DTYPES[c["kv"]]) for i in range(layers)]
        args = S.PagedForkArgs(parent=s["parent"].data_ptr(), kv_len=s["kv_len"].data_ptr(), page_table=s["table"].data_ptr(),
                               spare=s["spare"].data_ptr(), kv_len_out=s["len_out"].data_ptr(),
                               page_table_out=s["table_out"].data_ptr(), taken=s["taken"].data_ptr(),
                               table_stride=s["table"].shape[1], num_seqs=s["kv_len"].numel(), num_new=s["parent"].numel())
        return [(S.paged_fork, ((S.KvPages * layers)(*pages), args))]
    heads, kv_heads, hd = c["heads"], c["kv_heads"], c["head_dim"]
    n = sum(_rows(c))
    pages = S.KvPages(k=s["k_pool"].data_ptr(), v=s["v_pool"].data_ptr(), num_pages=s["pages"], page_size=c["page"],
                      num_kv_heads=kv_heads, head_dim=hd, dtype=S.KV_Q8)
    batch = S.PagedBatch(row_start=None if max(_rows(c)) == 1 else s["row_start"].data_ptr(),
                         kv_len=s["kv_len"].data_ptr(), page_table=s["table"].data_ptr(),
                         table_stride=s["table"].shape[1], num_seqs=c["seqs"], num_rows=n, max_kv_len=s["longest"])
    if c["op"] == "store":
        base, width = s["qkv"].data_ptr(), (heads + 2 * kv_heads) * hd
        args = S.PagedAppendArgs(
            q=base, k=base + 4 * heads * hd, v=base + 4 * (heads + kv_heads) * hd, q_out=s["q_out"].data_ptr(),
            ldq=width, ldk=width, ldv=width, ldq_out=heads * hd, num_heads=heads,
            q_norm=s["q_norm"].data_ptr() if c["norm"] else None,
            k_norm=s["k_norm"].data_ptr() if c["norm"] else None, norm_eps=EPS, rope_cos=s["cos"].data_ptr(),
            rope_sin=s["sin"].data_ptr(), rope_rows=s["longest"], rotary_dim=hd,
            rope_style=S.ROPE_HALVES if c["halves"] else S.ROPE_PAIRS)
        back = S.PagedReadArgs(k_out=s["k_out"].data_ptr(), v_out=s["v_out"].data_ptr(), ldk=kv_heads * hd, ldv=kv_heads * hd,
                               out_dtype=S.KV_F16)
        return [(S.paged_append, (pages, batch, args)), (S.paged_read, (pages, batch, back))]
    args = S.PagedAttentionArgs(q=s["q"].data_ptr(), out=s["out"].data_ptr(), ldq=heads * hd, ldo=heads * hd,
                                num_heads=heads, scale=1.0 / math.sqrt(hd), window=c["window"], sinks=c["sinks"])
    size = S.paged_attention_scratch_bytes(pages, batch, args)
    s["scratch"] = torch.empty(max(size, 16), dtype=torch.uint8, device="cuda")
    return [(S.paged_attention, (pages, batch, args, s["scratch"].data_ptr(), size))]


def run(s):
    if not own:
        return PLAIN[s["case"]["op"]](s)
    if "plan" not in s:
        s["plan"] = _plan(s)
    stream = torch.cuda.current_stream().cuda_stream
    for call, args in s["plan"]:
        call(*args, stream=stream)
    op = s["case"]["op"]
    if op == "store":
        return {"q": s["q_out"], "k": s["k_out"], "v": s["v_out"]}
    if op == "select":
        return {"scores": s["out_scores"], "rows": s["out_rows"], "tokens": s["out_tokens"]}
    if op == "fork":
        return {"table": s["table_out"], "kv_len": s["len_out"], "taken": s["taken"], "pool": s["pool"]}
    return {"out": s["out"]}


# -------------------------------------------------------------- in 64 bits


def exact(c, seed):
    """The definition, sequence by sequence, in 64 bits."""
    s = prepare(c, seed)
    d = torch.float64
    if c["op"] == "select":
        found = []
        for i in range(c["groups"]):
            lists = []
            for b in range(i * c["beams"], (i + 1) * c["beams"]):
                if s["ended"][b]:
                    lists.append(s["scores"][b:b + 1].to(d))
                else:
                    lists.append(torch.topk(s["scores"][b].to(d) + torch.log_softmax(s["logits"][b].to(d), 0),
                                            min(c["out"], c["vocab"])).values)
            best = torch.cat(lists).sort(descending=True).values[:c["out"]]
            found.append(torch.cat([best, best.new_full((c["out"] - len(best),), -math.inf)]))
        return {"scores": torch.stack(found), "rows": None, "tokens": None}
    if c["op"] == "fork":
        old, pool = s["pool"].clone(), s["pool"]
        table, length, spare = s["table"].tolist(), s["kv_len"].tolist(), s["spare"].tolist()
        kept = set()
        for i, p in enumerate(s["parent"].tolist()):
            t, used = divmod(length[p], c["page"])
            if p in kept and used:
                pool[spare[i], :, :, :, :used] = old[table[p][t], :, :, :, :used]
            kept.add(p)
        return {"table": None, "kv_len": None, "taken": None, "pool": pool}
    heads, kv_heads, hd, page = c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    lengths, rows = _lengths(c), _rows(c)
    if c["op"] == "store":
        found, first = {"q": [], "k": [], "v": []}, 0
        for length, r in zip(lengths, rows):
            x = s["qkv"][first:first + r].to(d).view(r, -1, hd)
            q, k, v = x[:, :heads], x[:, heads:heads + kv_heads], x[:, heads + kv_heads:]
            if c["norm"]:
                q = q / (q.square().sum(-1, keepdim=True) / hd + EPS).sqrt() * s["q_norm"].to(d)
                k = k / (k.square().sum(-1, keepdim=True) / hd + EPS).sqrt() * s["k_norm"].to(d)
            at = torch.arange(length - r, length, device="cuda")
            turn = torch.complex(s["cos"][at].to(d), s["sin"][at].to(d))[:, None, :]
            for name, t in (("q", q), ("k", k), ("v", v)):
                if name != "v":
                    if c["halves"]:
                        z = torch.complex(t[..., :hd // 2].contiguous(), t[..., hd // 2:].contiguous()) * turn
                        t = torch.cat([z.real, z.imag], -1)
                    else:
                        z = torch.view_as_complex(t.reshape(r, -1, hd // 2, 2).contiguous()) * turn
                        t = torch.view_as_real(z).reshape(r, -1, hd)
                if name != "q":
                    step = t.abs().max(-1, keepdim=True).values / 127
                    t = (t / step).round() * step
                found[name].append(t.reshape(r, -1))
            first += r
        return {name: torch.cat(t) for name, t in found.items()}
    group = heads // kv_heads
    out = torch.zeros(sum(rows), heads, hd, dtype=d, device="cuda")
    pools = [_parts(c, s["k_pool"]), _parts(c, s["v_pool"])]
    first = 0
    for i, (length, r) in enumerate(zip(lengths, rows)):
        where = s["table"][i].long()[:-(-length // page)]
        k, v = ((b[where].to(d) * e[where][..., None].to(d)).transpose(0, 1).reshape(kv_heads, -1, hd)[:, :length]
                for b, e in pools)
        p = torch.arange(length - r, length, device="cuda")[:, None]
        j = torch.arange(length, device="cuda")[None, :]
        hidden = j > p
        if c["window"]:
            hidden = hidden | ((j <= p - c["window"]) & (j >= c["sinks"]))
        for h in range(heads):
            logits = s["q"][first:first + r].to(d).view(r, heads, hd)[:, h] @ k[h // group].T / math.sqrt(hd)
            logits[hidden] = -math.inf
            out[first:first + r, h] = torch.softmax(logits, -1) @ v[h // group]
        first += r
    return {"out": out.reshape(sum(rows), heads * hd)}
