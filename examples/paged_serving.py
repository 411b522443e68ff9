#!/usr/bin/env python3
"""Serving requests of unlike lengths from one pool of key/value pages.

Requests join and leave while others run.  A step takes either the prompts
that are waiting, in chunks (several new rows per sequence), or one new token
of every running request (one row per sequence); both write their keys and
values with paged_append and read the pages with paged_attention.  Pages come
from a free list and go back when a request ends, or, for a model with an
attention window, as soon as no later row sees them.

  python examples/paged_serving.py [--model cfg1] [--requests 6] [--tokens 24]
                                   [--pages f32|f16|bf16] [--window W --sinks S]
"""
from __future__ import annotations

import argparse
import ctypes as C
import os
import sys
import time

import numpy as np
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "static-lm_b200"))
import static_lm as S  # noqa: E402
from static_lm import synth  # noqa: E402

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def dequantize_rows(blocks: np.ndarray, rows, cols: int) -> np.ndarray:
    """Rows of a BlockQ4_0 matrix as f32 (18 bytes per 32 weights)."""
    b = blocks.reshape(-1, cols // 32, 18)[np.asarray(rows)]
    d = b[..., :2].copy().view(np.float16).astype(np.float32)
    q = np.concatenate([b[..., 2:] & 15, b[..., 2:] >> 4], -1).astype(np.float32) - 8
    return (d * q).reshape(len(rows), cols)


class Request:
    def __init__(self, prompt, n_out):
        self.prompt, self.n_out = list(prompt), n_out
        self.done = 0  # prompt tokens whose keys are in the pages
        self.length = 0  # positions in the pages
        self.out: list[int] = []
        self.pages: dict[int, int] = {}  # page of the sequence -> page of the pool


class PagedServer:
    def __init__(self, cfg, weights, num_pages=64, page_size=16, kv="f32", window=0, sinks=0, max_rows=256, chunk=64):
        self.cfg, self.w, self.page, self.window, self.sinks, self.chunk = cfg, weights, page_size, window, sinks, chunk
        self.hd = cfg.dim // cfg.num_heads
        self.kv_dim = self.hd * cfg.num_kv_heads
        self.max_rows, self.per_seq = max_rows, -(-cfg.max_seq_len // page_size)
        q = lambda blocks, rows, cols: S.QMatrix(blocks, rows, cols)  # noqa: E731
        d, h, k = cfg.dim, cfg.hidden_dim, self.kv_dim
        self.layers = []
        for lw in weights.layers:
            self.layers.append(dict(qkv=q(np.concatenate([lw["wq"], lw["wk"], lw["wv"]]), d + 2 * k, d), wo=q(lw["wo"], d, d),
                                    gate=q(lw["w_gate"], h, d), up=q(lw["w_up"], h, d), down=q(lw["w_down"], d, h),
                                    norm1=torch.from_numpy(lw["rms_att_weight"]).cuda(),
                                    norm2=torch.from_numpy(lw["rms_ffn_weight"]).cuda()))
        head = weights.lm_head if weights.lm_head is not None else weights.token_embd
        self.head = q(head, weights.vocab, d)
        self.norm = torch.from_numpy(np.asarray(weights.output_norm, np.float32)).cuda()
        cos, sin = S.rope_tables(cfg.max_seq_len, self.hd)
        self.cos, self.sin = torch.from_numpy(cos).cuda(), torch.from_numpy(sin).cuda()
        # every layer's keys and values of a page lie together: page_stride spans the layers
        n, one = len(self.layers), cfg.num_kv_heads * page_size * self.hd
        self.pool = torch.zeros(num_pages, n, 2, one, dtype=TORCH[kv], device="cuda")
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.pages = [S.KvPages(k=self.pool[0, i, 0].data_ptr(), v=self.pool[0, i, 1].data_ptr(),
                                page_stride=n * 2 * one, num_pages=num_pages, page_size=page_size,
                                num_kv_heads=cfg.num_kv_heads, head_dim=self.hd, dtype=S.KV_DTYPES[kv],
                                status=self.status.data_ptr()) for i in range(n)]
        self.free = list(range(num_pages))[::-1]
        buf = lambda cols: torch.zeros(max_rows, cols, device="cuda")  # noqa: E731
        self.x, self.xb, self.qkv, self.att, self.y = buf(d), buf(d), buf(d + 2 * k), buf(d), buf(d)
        self.g, self.u = buf(h), buf(h)
        self.logits = buf(weights.vocab)
        self.next = torch.zeros(max_rows, dtype=torch.int32, device="cuda")
        self.requests: list[Request] = []
        self.stream = torch.cuda.current_stream().cuda_stream
        # the scratch of the largest call of this loop, in either form, serves all of them
        batch = lambda start: S.PagedBatch(row_start=start, kv_len=1, page_table=1, table_stride=self.per_seq,  # noqa: E731
                                           num_seqs=max_rows, num_rows=max_rows, max_kv_len=cfg.max_seq_len)
        size = max(S.paged_attention_scratch_bytes(self.pages[0], batch(start), self._attention_args()) for start in (None, 1))
        self.scratch = torch.empty(size + 16, dtype=torch.uint8, device="cuda")

    def _attention_args(self):
        return S.PagedAttentionArgs(q=self.qkv.data_ptr(), out=self.att.data_ptr(), ldq=self.qkv.stride(0), ldo=self.cfg.dim,
                                    num_heads=self.cfg.num_heads, scale=1.0 / np.sqrt(np.float32(self.hd)),
                                    window=self.window, sinks=self.sinks)

    # -------------------------------------------------------------- pages
    def _hold(self, r: Request, length: int):
        """Pages for positions below `length`; those no later row sees go back."""
        if self.window:
            first = (r.length - self.window + 1) // self.page  # the first page the next row's window touches
            for i in [i for i in r.pages if i < first and i * self.page >= self.sinks]:
                self.free.append(r.pages.pop(i))
        for i in range(r.length // self.page, -(-length // self.page)):
            if i not in r.pages:
                if not self.free:
                    raise S.SlmError(5, "out of pages")
                r.pages[i] = self.free.pop()

    def _batch(self, seqs, rows):
        table = np.full((len(seqs), self.per_seq), -1, np.int32)
        for s, r in enumerate(seqs):
            for i, page in r.pages.items():
                table[s, i] = page
        lengths = np.array([r.length + n for r, n in zip(seqs, rows)], np.int32)
        start = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        self.dev = [torch.from_numpy(a).cuda() for a in (table, lengths, start)]
        one = all(n == 1 for n in rows)
        return S.PagedBatch(row_start=None if one else self.dev[2].data_ptr(), kv_len=self.dev[1].data_ptr(),
                            page_table=self.dev[0].data_ptr(), table_stride=self.per_seq, num_seqs=len(seqs),
                            num_rows=int(start[-1]), max_kv_len=int(lengths.max()))

    # ------------------------------------------------------------ forward
    def _gemm(self, w, src, dst, n):
        S.lib().slm_gemm_q4_0_f32_noalloc(w.h, src.data_ptr(), dst.data_ptr(), n, w.rows, w.cols, self.stream)

    def _call(self, name, inputs, out, n, *more):
        ptrs = (C.c_void_p * len(inputs))(*[t.data_ptr() for t in inputs])
        getattr(S.lib(), name)(C.cast(ptrs, C.POINTER(C.c_void_p)), out.data_ptr(), n, *more, self.stream)

    def _norm(self, src, w, dst, n):
        for i in range(n):
            self._call("slm_exec_rmsnorm", [src[i], w], dst[i], self.cfg.dim, self.cfg.rms_eps)

    def _forward(self, tokens, batch):
        n, d, k = len(tokens), self.cfg.dim, self.kv_dim
        self.x[:n] = torch.from_numpy(dequantize_rows(self.w.token_embd, tokens, d)).cuda()
        base = self.qkv.data_ptr()
        append = S.PagedAppendArgs(q=base, k=base + 4 * d, v=base + 4 * (d + k), q_out=base, ldq=d + 2 * k, ldk=d + 2 * k,
                                   ldv=d + 2 * k, ldq_out=d + 2 * k, num_heads=self.cfg.num_heads,
                                   rope_cos=self.cos.data_ptr(), rope_sin=self.sin.data_ptr(),
                                   rope_rows=self.cfg.max_seq_len, rotary_dim=self.hd, rope_style=S.ROPE_PAIRS)
        attention = self._attention_args()
        for w, pages in zip(self.layers, self.pages):
            self._norm(self.x, w["norm1"], self.xb, n)
            self._gemm(w["qkv"], self.xb, self.qkv, n)
            S.paged_append(pages, batch, append, self.stream)
            S.paged_attention(pages, batch, attention, self.scratch.data_ptr(), self.scratch.numel() - 16, self.stream)
            self._gemm(w["wo"], self.att, self.y, n)
            self._call("slm_exec_residual_add", [self.x, self.y], self.x, n * d)
            self._norm(self.x, w["norm2"], self.xb, n)
            self._gemm(w["gate"], self.xb, self.g, n)
            self._gemm(w["up"], self.xb, self.u, n)
            self._call("slm_exec_swiglu", [self.g, self.u], self.g, n * self.cfg.hidden_dim)
            self._gemm(w["down"], self.g, self.y, n)
            self._call("slm_exec_residual_add", [self.x, self.y], self.x, n * d)

    def _sample(self, rows):
        """Greedy next tokens of the given activation rows."""
        for i, row in enumerate(rows):
            self._norm(self.x[row:], self.norm, self.xb[i:], 1)
        self._gemm(self.head, self.xb, self.logits, len(rows))
        for i in range(len(rows)):
            S.lib().slm_sample_argmax(self.logits[i].data_ptr(), self.w.vocab, self.next[i:].data_ptr(), self.stream)
        return self.next[:len(rows)].tolist()

    # -------------------------------------------------------------- steps
    def submit(self, prompt, n_out) -> Request:
        if not prompt or n_out < 1:
            raise S.SlmError(1, "a request has a prompt and asks for a token at least")
        if len(prompt) + n_out > self.cfg.max_seq_len:
            raise S.SlmError(2, "prompt and output exceed max_seq_len")
        self.requests.append(Request(prompt, n_out))
        return self.requests[-1]

    def step(self) -> bool:
        """One forward pass; False when no request is left."""
        waiting = [r for r in self.requests if r.done < len(r.prompt)]
        room, seqs, rows = self.max_rows, [], []
        if waiting:
            for r in waiting:
                n = min(self.chunk, len(r.prompt) - r.done, room)
                if n:
                    seqs.append(r), rows.append(n)
                    room -= n
        else:
            seqs = self.requests[:self.max_rows]
            rows = [1] * len(seqs)
        if not seqs:
            return False
        tokens = []
        for r, n in zip(seqs, rows):
            self._hold(r, r.length + n)
            tokens += r.prompt[r.done:r.done + n] if r.done < len(r.prompt) else [r.out[-1]]
        self._forward(tokens, self._batch(seqs, rows))
        ends, last = np.cumsum(rows) - 1, []
        for r, n, end in zip(seqs, rows, ends):
            r.length += n
            r.done = min(len(r.prompt), r.done + n)
            if r.done == len(r.prompt):
                last.append((r, int(end)))
        if last:
            for (r, _), tok in zip(last, self._sample([end for _, end in last])):
                r.out.append(tok)
                if len(r.out) == r.n_out:
                    self.free += r.pages.values()
                    r.pages.clear()
                    self.requests.remove(r)
        S.paged_check(self.pages[0], self.stream)
        return True

    def run(self):
        while self.step():
            pass


def main(argv=None):
    p = argparse.ArgumentParser()
    p.add_argument("--model", default="cfg1", choices=sorted(synth.CONFIGS))
    p.add_argument("--requests", type=int, default=6)
    p.add_argument("--tokens", type=int, default=24)
    p.add_argument("--pages", default="f32", choices=sorted(TORCH))
    p.add_argument("--window", type=int, default=0)
    p.add_argument("--sinks", type=int, default=0)
    a = p.parse_args(argv)
    cfg, layers, vocab = synth.config(a.model)
    w = synth.synth_model(cfg, layers, vocab, seed=1)
    server = PagedServer(cfg, w, num_pages=256, kv=a.pages, window=a.window, sinks=a.sinks)
    rng = np.random.default_rng(0)
    made = []
    t = time.time()
    for i in range(a.requests):
        made.append(server.submit([int(x) for x in rng.integers(0, vocab, int(rng.integers(1, 100)))], a.tokens))
        server.step()  # the others go on while this one arrives
    server.run()
    print(f"{a.requests} requests, {sum(len(r.out) for r in made)} tokens in {time.time() - t:.2f} s; "
          f"{len(server.free)} of {server.pool.shape[0]} pages free")
    for r in made:
        print(len(r.prompt), "->", r.out)
    return server, made


if __name__ == "__main__":
    main()
