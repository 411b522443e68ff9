#!/usr/bin/env python3
"""Beam search over the paged cache.

Every prompt is one sequence until its first new token; then its beams share
the prompt's pages.  A step is a decode pass over all beams of all prompts,
beam_select over their logits, and paged_fork, which makes the page tables of
the beams that go on: full pages are shared, and where a beam has several
successors all but one get a copy of its last page.  The selected rows are the
parents, so that nothing but the bookkeeping of free pages is the host's.

  python examples/beam_search.py [--model cfg1] [--prompts 3] [--beams 4] [--tokens 16]
                                 [--pages f32|f16|bf16|q8] [--end TOKEN]
"""
from __future__ import annotations

import argparse
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from paged_serving import PAGES, PagedServer  # noqa: E402

import static_lm as S  # noqa: E402
from static_lm import synth  # noqa: E402


class BeamSearch:
    def __init__(self, server: PagedServer, beams: int, end_token: int = -1, share: bool = True):
        """share False: every beam gets pages of its own and a copy of all of its parent's."""
        self.s, self.beams, self.end, self.share = server, beams, end_token, share

    def _positions(self, prompts):
        """The prompts into the pages; the logits of their last tokens, the tables and the lengths."""
        s, made, logits = self.s, [], []
        for prompt in prompts:
            r = s.submit(prompt, 1)
            while r.done < len(prompt) - 1:  # all chunks but the last one's last row
                n = min(s.chunk, len(prompt) - 1 - r.done)
                s._hold(r, r.length + n)
                s._forward(prompt[r.done:r.done + n], s._batch([r], [n]))
                r.length += n
                r.done += n
            s._hold(r, r.length + 1)
            s._forward(prompt[-1:], s._batch([r], [1]))
            r.length += 1
            s.requests.remove(r)
            logits.append(self._logits(1).clone())
            made.append(r)
        return made, torch.cat(logits)

    def _logits(self, n):
        s = self.s
        for i in range(n):
            s._norm(s.x[i:], s.norm, s.xb[i:], 1)
        s._gemm(s.head, s.xb, s.logits, n)
        return s.logits[:n]

    def run(self, prompts, n_out):
        """[prompt][beam] of (score, tokens), best first; every page is given back, also by a search that fails."""
        s = self.s
        free, requests = list(s.free), list(s.requests)
        try:
            return self._run(prompts, n_out)
        finally:
            s.free, s.requests = free, requests

    def _run(self, prompts, n_out):
        s, beams = self.s, self.beams
        groups, n = len(prompts), len(prompts) * self.beams
        if n > s.max_rows:
            raise S.SlmError(2, "more beams than rows")
        if max(map(len, prompts)) + n_out > s.cfg.max_seq_len:
            raise S.SlmError(2, "prompt and output exceed max_seq_len")
        made, first = self._positions(prompts)
        dev = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()  # noqa: E731
        table = np.full((n, s.per_seq), -1, np.int32)
        for i, r in enumerate(made):
            for j, page in r.pages.items():
                table[i * beams, j] = page
        # two of each: a step reads one and writes the other
        tables = [dev(table), torch.empty(n, s.per_seq, dtype=torch.int32, device="cuda")]
        lengths = [dev(np.repeat([r.length for r in made], beams)), torch.empty(n, dtype=torch.int32, device="cuda")]
        logits = torch.zeros(n, first.shape[1], device="cuda")
        logits[::beams] = first
        scores = torch.full((n,), -float("inf"), device="cuda")
        scores[::beams] = 0.0  # one beam of each prompt to begin with
        parent, tokens, taken = (torch.zeros(n, dtype=torch.int32, device="cuda") for _ in range(3))
        ended = torch.zeros(n, dtype=torch.int32, device="cuda")
        stream = torch.cuda.current_stream().cuda_stream
        pick = S.BeamSelectArgs(logits=logits.data_ptr(), ld=logits.stride(0), scores=scores.data_ptr(), ended=ended.data_ptr(),
                                num_groups=groups, beams=beams, vocab=logits.shape[1], num_out=beams, end_token=self.end,
                                out_scores=scores.data_ptr(), out_rows=parent.data_ptr(), out_tokens=tokens.data_ptr())
        size = S.beam_select_scratch_bytes(pick)
        scratch = torch.empty(size, dtype=torch.uint8, device="cuda")
        history = np.zeros((n, 0), np.int64)
        longest = max(r.length for r in made) + n_out
        for step in range(n_out):
            S.beam_select(pick, scratch.data_ptr(), size, stream)
            old, new = tables[step & 1], tables[1 - (step & 1)]
            len_old, len_new = lengths[step & 1], lengths[1 - (step & 1)]
            self._fork(old, len_old, parent, new, len_new, taken, stream)
            rows, toks = parent.cpu().numpy(), tokens.cpu().numpy()
            alive = rows >= 0
            history = np.concatenate([history[np.where(alive, rows, 0)], toks[:, None]], 1)
            ended.copy_(torch.where(parent >= 0, ended[parent.clamp(min=0).long()], 0) | (tokens == self.end).int())
            if step + 1 == n_out or bool(ended.all()):
                break
            len_new += (parent >= 0).int()  # the tokens' own positions
            batch = S.PagedBatch(kv_len=len_new.data_ptr(), page_table=new.data_ptr(), table_stride=s.per_seq, num_seqs=n,
                                 num_rows=n, max_kv_len=longest)
            s._forward(np.maximum(toks, 0), batch)
            logits.copy_(self._logits(n))
            S.paged_check(s.pages[0], stream)
        result = []
        for g in range(groups):
            found = [(float(scores[i]), [int(t) for t in history[i]]) for i in range(g * beams, (g + 1) * beams) if scores[i] > -np.inf]
            result.append(found)
        return result

    def _held(self, table):
        return [int(p) for p in np.unique(table.cpu().numpy()) if 0 <= p < self.s.pool.shape[0]]

    def _take(self, count):
        s = self.s
        if len(s.free) < count:
            raise S.SlmError(5, "out of pages")
        return [s.free.pop() for _ in range(count)]

    def _fork(self, old, len_old, parent, new, len_new, taken, stream):
        s, n = self.s, parent.numel()
        if self.share:
            spare = self._take(n)
            spare_d = torch.tensor(spare, dtype=torch.int32, device="cuda")
            S.paged_fork(s.pages, S.PagedForkArgs(
                parent=parent.data_ptr(), kv_len=len_old.data_ptr(), page_table=old.data_ptr(), spare=spare_d.data_ptr(),
                kv_len_out=len_new.data_ptr(), page_table_out=new.data_ptr(), taken=taken.data_ptr(), table_stride=s.per_seq,
                num_seqs=n, num_new=n), stream)
            s.free += [p for p, t in zip(spare, taken.tolist()) if not t]
        else:
            rows, table, lengths = parent.tolist(), old.tolist(), len_old.tolist()
            out = np.full((n, s.per_seq), -1, np.int32)
            for i, p in enumerate(rows):
                if p < 0:
                    continue
                count = lengths[p] // s.page + 1  # the next position's page too
                mine = self._take(count)
                for j, page in enumerate(mine):
                    out[i, j] = page
                    if table[p][j] >= 0:
                        s.pool[page] = s.pool[table[p][j]]
            new.copy_(torch.from_numpy(out))
            len_new.copy_(torch.tensor([lengths[p] if p >= 0 else 0 for p in rows], dtype=torch.int32))
        # pages that no beam holds any more
        s.free += sorted(set(self._held(old)) - set(self._held(new)))


def main(argv=None):
    p = argparse.ArgumentParser()
    p.add_argument("--model", default="cfg1", choices=sorted(synth.CONFIGS))
    p.add_argument("--prompts", type=int, default=3)
    p.add_argument("--beams", type=int, default=4)
    p.add_argument("--tokens", type=int, default=16)
    p.add_argument("--pages", default="q8", choices=sorted(PAGES))
    p.add_argument("--end", type=int, default=-1)
    a = p.parse_args(argv)
    cfg, layers, vocab = synth.config(a.model)
    server = PagedServer(cfg, synth.synth_model(cfg, layers, vocab, seed=1), num_pages=512, kv=a.pages)
    rng = np.random.default_rng(0)
    prompts = [[int(x) for x in rng.integers(0, vocab, int(rng.integers(1, 100)))] for _ in range(a.prompts)]
    found = BeamSearch(server, a.beams, a.end).run(prompts, a.tokens)
    for prompt, beams in zip(prompts, found):
        print(len(prompt), "->")
        for score, tokens in beams:
            print("  %9.4f" % score, tokens)
    print(f"{len(server.free)} of {server.pool.shape[0]} pages free")
    return server, found


if __name__ == "__main__":
    main()
