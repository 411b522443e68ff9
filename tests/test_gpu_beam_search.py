"""The beam search example: 8-bit (and other) pages, attention, selection and forking together.

A search whose beams share pages and one whose beams have pages and copies of
their own run the same kernels over the same numbers in other places, so that
tokens and scores are the same bits.  One beam is the greedy server's request.
"""
import importlib.util
import os

import numpy as np
import pytest

from static_lm import synth

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def example(name):
    spec = importlib.util.spec_from_file_location(name, os.path.join(ROOT, "examples", name + ".py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def model():
    cfg, layers, vocab = synth.config("cfg1")
    return cfg, synth.synth_model(cfg, layers, vocab, seed=1), vocab


def prompts_of(vocab):
    rng = np.random.default_rng(5)
    return [[int(t) for t in rng.integers(0, vocab, n)] for n in (15, 1, 64, 90)]


@pytest.mark.parametrize("kv,page,beams", [("q8", 8, 4), ("q8", 7, 3), ("f32", 16, 4), ("f16", 8, 5), ("bf16", 1, 2)])
def test_shared_pages_give_what_copies_give(cuda, kv, page, beams):
    cfg, w, vocab = model()
    m, prompts = example("beam_search"), prompts_of(vocab)
    found = []
    for share in (True, False):
        server = m.PagedServer(cfg, w, num_pages=4000 if page == 1 else 800, page_size=page, kv=kv)
        found.append(m.BeamSearch(server, beams, share=share).run(prompts, 11))
        assert sorted(server.free) == list(range(server.pool.shape[0])) and not server.requests
    assert found[0] == found[1]
    for group in found[0]:
        assert len(group) == beams and all(len(t) == 11 for _, t in group)
        scores = [s for s, _ in group]
        assert scores == sorted(scores, reverse=True) and len({tuple(t) for _, t in group}) == beams


def test_one_beam_is_greedy(cuda):
    cfg, w, vocab = model()
    m, prompts = example("beam_search"), prompts_of(vocab)
    server = m.PagedServer(cfg, w, num_pages=400, page_size=8, kv="f32")
    found = m.BeamSearch(server, 1).run(prompts, 10)
    made = [server.submit(p, 10) for p in prompts]
    server.run()
    assert [g[0][1] for g in found] == [r.out for r in made]


def test_ended_beams_keep_their_score(cuda):
    """The end is a token that some beam takes: from there on it repeats it, and its score stays."""
    cfg, w, vocab = model()
    m, prompts = example("beam_search"), prompts_of(vocab)[:2]
    server = m.PagedServer(cfg, w, num_pages=400, page_size=8, kv="q8")
    free = m.BeamSearch(server, 4).run(prompts, 4)
    end = free[0][0][1][0]  # the first token of the best continuation
    short = m.BeamSearch(server, 4, end_token=end).run(prompts[:1], 2)[0]
    longer = m.BeamSearch(server, 4, end_token=end).run(prompts[:1], 8)[0]
    ended = [(s, t) for s, t in short if t[0] == end]
    assert ended and all(t[1:] == [end] for _, t in ended)
    assert all((s, t + [end] * 6) in longer for s, t in ended)


def test_8_bit_pages_serve(cuda):
    cfg, w, vocab = model()
    server = example("paged_serving").PagedServer(cfg, w, num_pages=32, kv="q8")
    made = [server.submit([1 + i] * (5 + 9 * i), 6) for i in range(3)]
    server.run()
    assert all(len(r.out) == 6 and all(0 <= t < vocab for t in r.out) for r in made)
    assert len(server.free) == 32
