"""Pages that BatchGenerator sets aside for several continuations of a prompt, without a GPU: its steps on the restated books
(oracle/beams.py, oracle/paged.py) of a cache that has just as many."""
import numpy as np
import pytest
import torch

from oracle import beams as oracle
from oracle import paged as opaged
from sejong_b200.generate import Sampling
from sejong_b200.serve import BatchGenerator

EOS, VOCAB = 256, 257


class Booked(BatchGenerator):
    """The host's side of the steps; logits are drawn from the texts."""

    def __init__(self, batch, context, page, pages=None, seed=0):
        self.batch, self.context, self.page, self.seed = batch, context, page, seed
        self.width = -(-context // page)
        self.pages = pages or self.default_pages()
        self.logits, self.ids = torch.zeros(batch, VOCAB), torch.zeros(context, dtype=torch.int32)
        self.shared_graph, self.spare = self, True
        self._clear()

    def _clear(self):
        self.slots, self.finished, self.reserved = [None] * self.batch, set(), 0
        self.cached, self.table = [0] * self.batch, np.full((self.batch, self.width), -1)
        self.shares, self.free, self.least = [0] * self.pages, list(range(self.pages)), self.pages
        self.texts = [[] for _ in range(self.batch)]

    def _device_error(self):
        self.spent = self.pages - self.least
        return 0

    def _check_shared(self):
        pass

    def _write_shared(self, parents, added, ids=(), groups=()):
        self.step = list(parents), dict(added), list(ids)

    def _fork_and_plan(self, rows):
        parents, added, _ = self.step
        self.cached, self.table, shares, self.free, copies, _, status = oracle.fork(parents, self.page, self.cached, self.table,
                                                                                    self.shares, self.free)
        assert status == 0, f"of the fork {status}"
        self.shares = [int(s) for s in shares]
        want = [added.get(b, 0) for b in range(self.batch)]
        self.table, self.cached, _, _, _, summary = opaged.plan(self.cached, want, self.page, self.free, self.table, rows)
        assert summary[2] == 0, f"status {summary[2]}"
        self.free = self.free[:summary[3]]
        self.least = min(self.least, len(self.free))
        self.texts = [list(self.texts[p]) if p >= 0 else [] for p in parents]

    def _prompt(self, n, file):
        slot, = self.step[1]
        self.texts[slot] = self.ids[:n].tolist()
        self._show([slot])

    def _head(self, first, rows, out):
        pass

    def replay(self):
        self._fork_and_plan(self.batch)
        live = [b for b in range(self.batch) if self.step[1].get(b)]
        for b, token in zip(live, self.step[2]):
            self.texts[b].append(token)
        for b in live:
            assert len(self.texts[b]) == self.cached[b]
        self._show(live)

    def _show(self, slots):
        for r, b in enumerate(slots):
            rng = np.random.default_rng([self.seed, len(self.texts[b]), *self.texts[b][-8:]])
            self.logits[r] = torch.from_numpy(rng.standard_normal(VOCAB) * 2).float()
            self.logits[r, EOS] -= 3

    def _select(self, rows, scores, beams, keep):
        x = self.logits[:rows].double().numpy().reshape(-1, beams, VOCAB)
        return [a.tolist() for a in oracle.select(x, np.array(scores, dtype=np.float64).reshape(-1, beams), keep)]


SHAPES = [(4, 32, 8), (3, 20, 1), (5, 30, 16), (8, 24, 4), (2, 17, 32), (6, 40, 3)]


@pytest.mark.parametrize("batch,context,page", SHAPES)
def test_samples_get_by_with_what_is_set_aside(batch, context, page):
    """Prompts of every length to one below the context, and texts that fit, fill the context, or start again."""
    for n in range(0, context - 1, 3):
        for most in (1, 2, context - n - 1, context):
            gen = Booked(batch, context, page, pages=10 ** 4, seed=n)
            pages = gen._reserve([EOS] + [65] * n, most, batch, False)
            gen = Booked(batch, context, page, pages=pages, seed=n)
            done = gen.generate([bytes([65]) * n], Sampling(max_bytes=most, temperature=1.0, seed=n), samples=batch)[0]
            assert all(d.ended or len(d.text) == most for d in done)


@pytest.mark.parametrize("batch,context,page", SHAPES)
def test_beams_get_by_with_what_is_set_aside(batch, context, page):
    for n in range(0, context - 1, 3):
        for most in {1, 2, 7, context - n - 1}:
            if n + 1 + most > context:
                continue
            gen = Booked(batch, context, page, pages=10 ** 4, seed=n)
            pages = gen._reserve([EOS] + [65] * n, most, batch, True)
            gen = Booked(batch, context, page, pages=pages, seed=n)
            assert gen.beam_search([bytes([65]) * n], beams=batch, max_bytes=most)[0]


@pytest.mark.parametrize("batch,context,page", SHAPES)
def test_a_default_cache_holds_a_whole_batch_of_continuations(batch, context, page):
    gen = Booked(batch, context, page)
    for n in range(0, context - 1):
        for most in (1, context - n - 1, 5 * context):
            assert gen._reserve([EOS] + [65] * n, most, batch, False) <= gen.pages
            if n + 1 + most <= context:
                assert gen._reserve([EOS] + [65] * n, most, batch, True) <= gen.pages


def test_several_prompts_get_by_with_few_pages():
    """More prompts than the cache has room for at once."""
    prompts = [bytes([65 + i]) * (1 + 4 * i) for i in range(6)]
    for page in (1, 3, 8):
        need = max(Booked(6, 40, page, 10 ** 4)._reserve([EOS] + list(p), 12, 3, True) for p in prompts)
        for pages in (need, need + 7, 2 * need):
            assert all(Booked(6, 40, page, pages).beam_search(prompts, beams=3, max_bytes=12))
            found = Booked(6, 40, page, pages).generate(prompts, Sampling(max_bytes=12, temperature=1.0), samples=3)
            assert all(d.ended or len(d.text) == 12 for done in found for d in done)


def test_a_cache_of_more_pages_than_can_be_shared_is_refused_at_once():
    gen = Booked(2, 32, 8, pages=(1 << 18) + 1)

    def staged(*args):
        raise AssertionError("a step was staged")

    gen._write_shared = staged
    with pytest.raises(ValueError, match="262144 pages"):
        gen.generate([b"a"], Sampling(max_bytes=3), samples=2)
    with pytest.raises(ValueError, match="262144 pages"):
        gen.beam_search([b"a"], beams=2, max_bytes=3)
    gen = Booked(2, 32, 8, pages=1 << 18)
    assert gen.beam_search([b"a"], beams=2, max_bytes=1)[0]
