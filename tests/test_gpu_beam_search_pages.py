"""The beam search example gives every page back, whatever ends it, and no page of others."""
import pytest

from static_lm import SlmError
from test_gpu_beam_search import example, model, prompts_of

pytestmark = pytest.mark.gpu


def server_of(m, pages):
    cfg, w, vocab = model()
    server = m.PagedServer(cfg, w, num_pages=pages, page_size=8, kv="q8")
    live = server.submit([1, 2, 3] * 10, 40)  # another request, half way
    server.step(), server.step()
    return server, live, prompts_of(vocab)


def whole(server, live):
    assert server.requests == [live]
    assert sorted(server.free + list(live.pages.values())) == list(range(server.pool.shape[0]))


def test_a_search_for_no_tokens_takes_no_pages(cuda, monkeypatch):
    m = example("beam_search")
    server, live, prompts = server_of(m, 200)
    # what memory that is not initialised may hold: the id of a page that is another's
    held, empty = next(iter(live.pages.values())), cuda.empty
    monkeypatch.setattr(cuda, "empty", lambda *a, **k: empty(*a, **k).fill_(held) if k.get("dtype") == cuda.int32 else empty(*a, **k))
    found = m.BeamSearch(server, 4).run(prompts[:2], 0)
    assert found == [[(0.0, [])]] * 2
    whole(server, live)


@pytest.mark.parametrize("pages", [6, 20, 32, 40])
def test_a_search_that_runs_out_of_pages_gives_them_back(cuda, pages):
    m = example("beam_search")
    server, live, prompts = server_of(m, pages)
    with pytest.raises(SlmError) as e:
        m.BeamSearch(server, 4).run(prompts, 30)
    assert e.value.code == 5
    whole(server, live)


def test_a_refused_search_gives_its_pages_back(cuda):
    m = example("beam_search")
    server, live, prompts = server_of(m, 200)
    with pytest.raises(SlmError):
        m.BeamSearch(server, 65).run(prompts[:1], 3)  # more than a selection's 64 places
    whole(server, live)
    m.BeamSearch(server, 3).run(prompts, 9)
    whole(server, live)
    server.run()
    assert len(live.out) == 40 and sorted(server.free) == list(range(200))
