"""The paged key/value cache operators, as cases to measure.

append   per-head RMSNorm of q and k (optional), rotary positions, and the new
         keys and values into the pages of their sequences
decode   attention of one new token per sequence over its pages
rows     attention of several new rows per sequence (a prompt, or a chunk of
         one behind an earlier context) over its pages

A key j is visible to a row at position p when j <= p and, with a window,
p - j < window or j < sinks.  Pages hold [kv_head][slot][head_dim]; activations
are f32; the pages are f32, f16 or bf16.
"""
import math
import os
import sys

import torch

own = False

F16, BF16, F32 = "f16", "bf16", "f32"
DTYPES = {F16: torch.float16, BF16: torch.bfloat16, F32: torch.float32}
EPS = 1e-5
THETA = 10000.0


def case(name, op, seqs, heads, kv_heads, head_dim, kv, page, ctx, new=(1, 1), window=0, sinks=0, norm=False,
         halves=False):
    """ctx: shortest and longest length of a sequence, its new rows included; new: fewest and most new rows."""
    return {"name": name, "op": op, "seqs": seqs, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "kv": kv,
            "page": page, "ctx_min": ctx[0], "ctx_max": ctx[1], "new_min": new[0], "new_max": new[1],
            "window": window, "sinks": sinks, "norm": norm, "halves": halves}


def listed():
    return [
        # one user's next token on the 135M shape, f32 pages: the smallest call
        case("append-1", "append", 1, 9, 3, 64, F32, 16, (2048, 2048)),
        # a decode step of 64 sequences on the 8B shape, normed queries and keys
        case("append-64", "append", 64, 32, 8, 128, F16, 16, (50, 700), norm=True, halves=True),
        # eight prompts of 4096 tokens on the 135M shape
        case("append-prompts", "append", 8, 9, 3, 64, F16, 16, (4096, 4096), (4096, 4096)),
        # a first token of the 15M shape over a short context: latency
        case("decode-1x77", "decode", 1, 6, 6, 48, F32, 16, (77, 77)),
        # the 135M shape at 64 sequences of 2048 positions, f32 pages
        case("decode-64x2048", "decode", 64, 9, 3, 64, F32, 16, (2049, 2049)),
        # one long sequence on the 8B shape: the length has to be split
        case("decode-1x8192", "decode", 1, 32, 8, 128, F16, 16, (8192, 8192)),
        # a serving batch of unlike lengths on the 8B shape
        case("decode-64-ragged", "decode", 64, 32, 8, 128, BF16, 32, (500, 8192)),
        # long sequences that keep a window and their first tokens
        case("decode-128-window", "decode", 128, 32, 8, 128, F16, 16, (600, 8192), window=1024, sinks=4),
        # eight prompts of 4096 tokens on the 135M shape
        case("rows-8x4096", "rows", 8, 9, 3, 64, F16, 16, (4096, 4096), (4096, 4096)),
        # one prompt on the 8B shape
        case("rows-1x4096", "rows", 1, 32, 8, 128, BF16, 16, (4096, 4096), (4096, 4096)),
        # a long prompt with a window and sinks on the 8B shape
        case("rows-8192-window", "rows", 1, 32, 8, 128, F16, 16, (8192, 8192), (8192, 8192), window=1024, sinks=4),
        # chunks of unlike lengths behind unlike contexts, f32 pages
        case("rows-chunks", "rows", 16, 9, 3, 64, F32, 16, (600, 2048), (1, 512)),
    ]


SHAPES = [(9, 3, 64), (9, 3, 64), (6, 6, 48), (4, 4, 64), (32, 8, 128), (32, 8, 128), (12, 2, 80), (20, 4, 96),
          (16, 1, 64), (8, 8, 32)]


def draw(rng):
    def spread(lo, hi):
        v = min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))
        return v + 1 if v == 3072 else v

    while True:
        op = rng.choice(["append", "decode", "rows"])
        heads, kv_heads, head_dim = rng.choice(SHAPES)
        kv, page = rng.choice([F16, BF16, F32]), rng.choice([8, 16, 16, 24, 32, 64])
        seqs = spread(1, 32 if op == "rows" else 128)
        hi = spread(2, 8192)
        lo = rng.choice([hi, max(1, hi // rng.randint(2, 9))])
        new = (1, 1)
        if op != "decode":
            most = rng.choice([lo, spread(1, lo)])
            new = (rng.choice([most, 1]), most)
            if op == "append" and rng.random() < 0.3:
                new = (1, 1)
        window, sinks = 0, 0
        if op != "append" and rng.random() < 0.5:
            window, sinks = spread(1, 2048), rng.choice([0, 1, 4, 16, 37])
        c = case("", op, seqs, heads, kv_heads, head_dim, kv, page, (lo, hi), new, window, sinks,
                 op == "append" and rng.random() < 0.5, op == "append" and rng.random() < 0.5)
        del c["name"]
        w = work(c)
        rows, most = sum(_rows(c)), max(_rows(c))
        if op == "append" and rows <= 32768 and w["bytes"] <= 234e6:
            return c
        if op == "decode" and w["bytes"] <= 1.1e9 and seqs * hi * kv_heads * head_dim <= 540e6:
            return c
        if op == "rows" and w["flops"] <= 1.3e11 and seqs * most * heads * hi <= 2.2e9:
            return c


# ------------------------------------------------------------------ lengths


def _spread(n, lo, hi, step):
    """n whole numbers spread over [lo, hi], the same for every seed; both ends are among them where n allows."""
    v = [lo + int((hi - lo + 1) * ((i * step) % 1.0)) for i in range(n)]
    v[-1] = hi
    return v


def _lengths(c):
    return _spread(c["seqs"], c["ctx_min"], c["ctx_max"], 0.6180339887)


def _rows(c):
    return [min(r, n) for r, n in zip(_spread(c["seqs"], c["new_min"], c["new_max"], 0.7548776662), _lengths(c))]


def _seen(p, window, sinks):
    """Keys visible to a row at position p."""
    if not window or p + 1 <= window:
        return p + 1
    return window + min(sinks, p + 1 - window)


def work(c):
    heads, kv_heads, hd = c["heads"], c["kv_heads"], c["head_dim"]
    el = 4 if c["kv"] == F32 else 2
    lengths, rows = _lengths(c), _rows(c)
    n = sum(rows)
    if c["op"] == "append":
        width = heads + 2 * kv_heads
        return {"bytes": n * hd * (4 * width + 4 * heads + 2 * el * kv_heads) + 4 * n * hd,
                "flops": n * hd * (heads + kv_heads) * (3 + (4 if c["norm"] else 0))}
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
    return {"bytes": 8 * n * heads * hd + 2 * el * keys * kv_heads * hd, "flops": 4 * pairs * heads * hd}


# ------------------------------------------------------------------- inputs


def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(1000003 * (seed + 1))
    dev, dt = "cuda", DTYPES[c["kv"]]
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
         "k_pool": torch.empty(pages, kv_heads, page, hd, device=dev, dtype=dt).normal_(generator=g),
         "v_pool": torch.empty(pages, kv_heads, page, hd, device=dev, dtype=dt).normal_(generator=g)}
    if c["op"] == "append":
        # one projection's output: q, k and v of a row side by side
        s["qkv"] = rand(n, (heads + 2 * kv_heads) * hd)
        s["q_out"] = torch.zeros(n, heads * hd, device=dev)
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


def _plain_append(s):
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
    s["k_pool"][at, :, slot] = turn(k).to(s["k_pool"].dtype)
    s["v_pool"][at, :, slot] = v.to(s["v_pool"].dtype)
    return {"q": s["q_out"], "k_pool": s["k_pool"], "v_pool": s["v_pool"]}


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
        return pool[table].permute(0, 2, 1, 3, 4).reshape(seqs, kv_heads, -1, hd).float()

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


# --------------------------------------------------------- the framework's


def _package():
    path = os.path.join(os.getcwd(), "static-lm_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import static_lm
    return static_lm


def _plan(s):
    """The descriptors of this state's buffers and the scratch, as a program with fixed buffers keeps them."""
    S, c = _package(), s["case"]
    heads, kv_heads, hd = c["heads"], c["kv_heads"], c["head_dim"]
    n = sum(_rows(c))
    pages = S.KvPages(k=s["k_pool"].data_ptr(), v=s["v_pool"].data_ptr(), num_pages=s["pages"], page_size=c["page"],
                      num_kv_heads=kv_heads, head_dim=hd, dtype=S.KV_DTYPES[c["kv"]])
    batch = S.PagedBatch(row_start=None if c["op"] == "decode" else s["row_start"].data_ptr(),
                         kv_len=s["kv_len"].data_ptr(), page_table=s["table"].data_ptr(),
                         table_stride=s["table"].shape[1], num_seqs=c["seqs"], num_rows=n, max_kv_len=s["longest"])
    if c["op"] == "append":
        base, width = s["qkv"].data_ptr(), (heads + 2 * kv_heads) * hd
        args = S.PagedAppendArgs(
            q=base, k=base + 4 * heads * hd, v=base + 4 * (heads + kv_heads) * hd, q_out=s["q_out"].data_ptr(),
            ldq=width, ldk=width, ldv=width, ldq_out=heads * hd, num_heads=heads,
            q_norm=s["q_norm"].data_ptr() if c["norm"] else None,
            k_norm=s["k_norm"].data_ptr() if c["norm"] else None, norm_eps=EPS, rope_cos=s["cos"].data_ptr(),
            rope_sin=s["sin"].data_ptr(), rope_rows=s["longest"], rotary_dim=hd,
            rope_style=S.ROPE_HALVES if c["halves"] else S.ROPE_PAIRS)
        return S.paged_append, (pages, batch, args)
    args = S.PagedAttentionArgs(q=s["q"].data_ptr(), out=s["out"].data_ptr(), ldq=heads * hd, ldo=heads * hd,
                                num_heads=heads, scale=1.0 / math.sqrt(hd), window=c["window"], sinks=c["sinks"])
    size = S.paged_attention_scratch_bytes(pages, batch, args)
    s["scratch"] = torch.empty(max(size, 16), dtype=torch.uint8, device="cuda")
    return S.paged_attention, (pages, batch, args, s["scratch"].data_ptr(), size)


def run(s):
    if not own:
        return _plain_append(s) if s["case"]["op"] == "append" else _plain_attention(s)
    if "plan" not in s:
        s["plan"] = _plan(s)
    call, args = s["plan"]
    call(*args, stream=torch.cuda.current_stream().cuda_stream)
    if s["case"]["op"] == "append":
        return {"q": s["q_out"], "k_pool": s["k_pool"], "v_pool": s["v_pool"]}
    return {"out": s["out"]}


# -------------------------------------------------------------- in 64 bits


def exact(c, seed):
    """The definition, row by row of the table of sequences, in 64 bits."""
    s = prepare(c, seed)
    heads, kv_heads, hd, page = c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    lengths, rows = _lengths(c), _rows(c)
    d = torch.float64
    if c["op"] == "append":
        keys, values = s["k_pool"].to(d), s["v_pool"].to(d)
        q_all = torch.zeros(sum(rows), heads, hd, dtype=d, device="cuda")
        first = 0
        for i, (length, r) in enumerate(zip(lengths, rows)):
            x = s["qkv"][first:first + r].to(d).view(r, -1, hd)
            q, k, v = x[:, :heads], x[:, heads:heads + kv_heads], x[:, heads + kv_heads:]
            if c["norm"]:
                q = q / (q.square().sum(-1, keepdim=True) / hd + EPS).sqrt() * s["q_norm"].to(d)
                k = k / (k.square().sum(-1, keepdim=True) / hd + EPS).sqrt() * s["k_norm"].to(d)
            at = torch.arange(length - r, length, device="cuda")
            turn = torch.complex(s["cos"][at].to(d), s["sin"][at].to(d))[:, None, :]
            for t, store in ((q, q_all), (k, None)):
                if c["halves"]:
                    z = torch.complex(t[..., :hd // 2].contiguous(), t[..., hd // 2:].contiguous()) * turn
                    t = torch.cat([z.real, z.imag], -1)
                else:
                    z = torch.view_as_complex(t.reshape(r, -1, hd // 2, 2).contiguous()) * turn
                    t = torch.view_as_real(z).reshape(r, -1, hd)
                if store is not None:
                    store[first:first + r] = t
                else:
                    k = t
            where = s["table"][i].long()[at // page]
            keys[where, :, at % page] = k
            values[where, :, at % page] = v
            first += r
        return {"q": q_all.reshape(sum(rows), -1), "k_pool": keys, "v_pool": values}
    group = heads // kv_heads
    out = torch.zeros(sum(rows), heads, hd, dtype=d, device="cuda")
    first = 0
    for i, (length, r) in enumerate(zip(lengths, rows)):
        where = s["table"][i].long()[:-(-length // page)]
        k = s["k_pool"][where].transpose(0, 1).reshape(kv_heads, -1, hd)[:, :length]
        v = s["v_pool"][where].transpose(0, 1).reshape(kv_heads, -1, hd)[:, :length]
        p = torch.arange(length - r, length, device="cuda")[:, None]
        j = torch.arange(length, device="cuda")[None, :]
        hidden = j > p
        if c["window"]:
            hidden = hidden | ((j <= p - c["window"]) & (j >= c["sinks"]))
        for h in range(heads):
            logits = s["q"][first:first + r].to(d).view(r, heads, hd)[:, h] @ k[h // group].to(d).T / math.sqrt(hd)
            logits[hidden] = -math.inf
            out[first:first + r, h] = torch.softmax(logits, -1) @ v[h // group].to(d)
        first += r
    return {"out": out.reshape(sum(rows), heads * hd)}
