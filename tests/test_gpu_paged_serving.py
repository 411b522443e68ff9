"""The paged serving example against the model driver on contiguous caches."""
import importlib.util
import os

import numpy as np
import pytest

import static_lm as S
from static_lm import synth

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def example():
    spec = importlib.util.spec_from_file_location("paged_serving", os.path.join(ROOT, "examples", "paged_serving.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def model():
    cfg, layers, vocab = synth.config("cfg1")
    return cfg, synth.synth_model(cfg, layers, vocab, seed=1), vocab


def test_requests_that_share_pages_get_the_models_tokens(cuda):
    cfg, w, vocab = model()
    rng = np.random.default_rng(3)
    prompts = [[int(t) for t in rng.integers(0, vocab, n)] for n in (16, 1, 70, 33)]
    server = example().PagedServer(cfg, w, num_pages=40, page_size=8, kv="f32")
    made = []
    for p in prompts:
        made.append(server.submit(p, 12))
        server.step()
    server.run()
    assert len(server.free) == 40 and not server.requests
    m = S.Model(cfg, w, max_sequences=1, max_rows=128)
    for p, r in zip(prompts, made):
        assert r.out == m.generate(p, 12)


@pytest.mark.parametrize("kv", ["f16", "bf16"])
def test_sixteen_bit_pages_serve(cuda, kv):
    cfg, w, vocab = model()
    server = example().PagedServer(cfg, w, num_pages=32, kv=kv)
    made = [server.submit([1 + i] * (5 + 9 * i), 6) for i in range(3)]
    server.run()
    assert all(len(r.out) == 6 and all(0 <= t < vocab for t in r.out) for r in made)


def test_window_gives_pages_back(cuda):
    cfg, w, vocab = model()
    server = example().PagedServer(cfg, w, num_pages=12, page_size=8, window=24, sinks=4, chunk=16)
    r = server.submit(list(range(1, 121)), 40)  # 160 positions: twenty pages without the window
    server.run()
    assert len(r.out) == 40 and len(server.free) == 12


def test_long_prompts_and_few_long_requests(cuda):
    """Calls that are split over more CTAs than the loop's largest: the last
    chunk of a prompt near max_seq_len, and a handful of long sequences.  (Which
    tokens come is not compared: Q8_0 activations turn differences of 1e-7 into
    some 1e-2 of a logit, and over so many positions some logits lie that near.)"""
    cfg, w, vocab = model()
    rng = np.random.default_rng(5)
    server = example().PagedServer(cfg, w, num_pages=256)
    made = [server.submit([int(t) for t in rng.integers(0, vocab, n)], 8)
            for n in (cfg.max_seq_len - 8, 430, 433, 410, 417, 440)]
    server.run()
    assert all(len(r.out) == 8 and all(0 <= t < vocab for t in r.out) for r in made)
    assert len(server.free) == 256


@pytest.mark.parametrize("prompt,n_out,code", [([], 4, 1), ([5], 0, 1), ([5], -1, 1), ([5] * 500, 13, 2)])
def test_requests_that_could_not_end_are_refused(cuda, prompt, n_out, code):
    cfg, w, vocab = model()
    server = example().PagedServer(cfg, w, num_pages=4)
    with pytest.raises(S.SlmError) as e:
        server.submit(prompt, n_out)
    assert e.value.code == code and not server.step()
