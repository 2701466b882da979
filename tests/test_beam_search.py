"""The host's side of a beam search (BatchGenerator.beam_search) on scripted models, without a GPU: the steps' kernels are
replaced by lists of tokens and the 64-bit selection (oracle/beams.py)."""
import math

import numpy as np
import pytest

from oracle import beams as oracle
from sejong_b200.serve import BatchGenerator

EOS, VOCAB = 256, 257


class Scripted(BatchGenerator):
    """model(drawn bytes): {token: probability}; the rest has none."""

    def __init__(self, model, batch=8, context=64, page=8):
        self.model, self.batch, self.context, self.page = model, batch, context, page
        self.width = -(-context // page)
        self.pages = batch * self.width + batch - 1
        self.texts, self.rows, self.steps = [None] * batch, [], 0
        self.slots, self.finished, self.reserved = [None] * batch, set(), 0

    def _share(self):
        pass

    def _clear(self):
        self.slots, self.finished, self.reserved = [None] * self.batch, set(), 0

    def _device_error(self):
        return 0

    def _start_shared(self, slot, tokens, pending):
        self.prompt = len(tokens)
        self.finished.discard(slot)
        self.texts[slot] = list(tokens)
        self.rows = [list(tokens)]

    def _step_shared(self, parents, live, ids, common):
        self.steps += 1
        self.finished.clear()
        texts = [list(self.texts[p]) if p >= 0 and self.texts[p] is not None else None for p in parents]
        for b, token in zip(live, ids):
            texts[b].append(token)
        self.texts, self.rows = texts, [texts[b] for b in live]

    def _select(self, rows, scores, beams, keep):
        x = np.full((rows, VOCAB), -np.inf)
        for r in range(rows):
            for token, p in self.model(tuple(self.rows[r][self.prompt:])).items():
                x[r, token] = math.log(p)
        return [a.tolist() for a in oracle.select(x.reshape(-1, beams, VOCAB),
                                                  np.array(scores, dtype=np.float64).reshape(-1, beams), keep)]


def search_to_the_end(model, beams, most, penalty):
    """The same search that never stops early: (ranked, text, ended) of the best `beams`."""
    live, found = [((), 0.0)], []
    for _ in range(most):
        order = []
        for i, (drawn, score) in enumerate(live):
            order += [(-(score + math.log(p)), i, token) for token, p in model(drawn).items()]
        order, new = sorted(order)[:2 * beams], []
        for at, (total, i, token) in enumerate(order):
            if len(new) == beams:
                break
            drawn = live[i][0]
            if token == EOS:
                if at < beams:
                    found.append((-total / (len(drawn) + 1) ** penalty, drawn, True))
                continue
            new.append((drawn + (token,), -total))
        live = new
    found += [(score / len(drawn) ** penalty, drawn, False) for drawn, score in live]
    return sorted(found, key=lambda h: -h[0])[:beams]


def overtaking(drawn):
    """Two beams that probably end at once, and rarely go on to a long text without doubt."""
    if not drawn:
        return {97: 0.5, 98: 0.45, 99: 0.05}
    if len(drawn) == 1:
        return {EOS: 0.6, 120: 0.4}
    return {120: 0.999, EOS: 0.001}


def test_a_beam_that_overtakes_ended_ones_is_found():
    gen = Scripted(overtaking)
    best = gen.beam_search([b""], beams=2, max_bytes=20)[0][0]
    assert best.text == b"a" + b"x" * 19 and not best.ended
    assert best.ranked == pytest.approx((math.log(0.5 * 0.4) + 18 * math.log(0.999)) / 20)


def test_a_search_ends_when_no_beam_can_overtake():
    gen = Scripted(overtaking)  # without a penalty a longer text is worth no more
    found = gen.beam_search([b""], beams=2, max_bytes=20, length_penalty=0.0)[0]
    assert [(h.text, h.ended) for h in found] == [(b"a", True), (b"b", True)]
    assert gen.steps == 1


def random_model(seed, tokens=5):
    def model(drawn):
        rng = np.random.default_rng([seed, *drawn])
        p = rng.dirichlet(np.full(tokens + 1, 0.4))
        return {t: float(v) for t, v in zip([*range(97, 97 + tokens), EOS], p) if v > 1e-12}
    return model


@pytest.mark.parametrize("penalty", [0.0, 0.5, 1.0, 2.0, -1.0])
@pytest.mark.parametrize("beams", [1, 2, 4])
def test_stopping_early_loses_nothing(beams, penalty):
    for seed in range(12):
        model = random_model(seed)
        found = Scripted(model).beam_search([b"p"], beams=beams, max_bytes=9, length_penalty=penalty)[0]
        want = search_to_the_end(model, beams, 9, penalty)
        assert [(h.text, h.ended) for h in found] == [(bytes(d), e) for _, d, e in want]
        assert [h.ranked for h in found] == pytest.approx([r for r, _, _ in want])


@pytest.mark.parametrize("penalty", [float("nan"), float("inf"), -float("inf"), 51, 1e6])
def test_length_penalties_that_rank_nothing_are_refused(penalty):
    """By NaN no text is worth more than another, by infinities none or all, and 20 ** 1e6 is no number."""
    with pytest.raises(ValueError, match="length penalty"):
        Scripted(overtaking).beam_search([b"a"], beams=2, max_bytes=20, length_penalty=penalty)


def test_the_largest_length_penalties_rank():
    for penalty in (-50, 50):
        found = Scripted(overtaking).beam_search([b""], beams=2, max_bytes=20, length_penalty=penalty)[0]
        assert all(math.isfinite(h.ranked) for h in found) and found[0].ended == (penalty < 0)
