"""Several continuations of one prompt (BatchGenerator.generate with samples, beam_search) against the FP64 model at the
bf16-cast weights.  Log probabilities are off by a few hundredths (test_gpu_serve.py), bounded by 0.1 a byte."""
import io
import json
import os

import numpy as np
import pytest
import torch

from oracle import model as omodel
from oracle import scores as oscores
from sejong_b200 import model as pm

pytestmark = pytest.mark.gpu


def logits(params, c, tokens):
    oc = omodel.ModelConfig(width=c.width, layers=c.layers, heads=c.heads, ffn_width=c.ffn_width, kv_heads=c.kv_heads,
                            rope_theta=c.rope_theta, norm_epsilon=c.norm_epsilon, seed=c.seed, init_std=c.init_std)
    p = {k: torch.tensor(v, dtype=torch.float64) for k, v in omodel.compute_cast(params, "bf16").items()}
    ids = torch.as_tensor(np.asarray(tokens, dtype=np.int64))
    with torch.no_grad():
        return (omodel.hidden(p, oc, ids, len(tokens)) @ p["output"]).numpy()[:, :257]


@pytest.fixture(scope="module")
def made():
    c = pm.with_(pm.with_(pm.config_c1(), layers=2), init_std=0.08)
    return c, pm.initialize(c)


@pytest.fixture(params=["rule", "always"])
def sharing(request, monkeypatch):
    if request.param == "always":
        monkeypatch.setenv("SJ_ATTN_SHARE", "always")


def generator(made, **kw):
    from sejong_b200.serve import BatchGenerator
    c, params = made
    return BatchGenerator(c, params, device=0, **{**dict(context=96, batch=8, page=8), **kw})


def logp_of(made, prompt, drawn):
    """The FP64 log probabilities of drawn bytes after EOS and the prompt."""
    c, params = made
    seq = [256] + list(prompt) + list(drawn)
    rows = logits(params, c, seq[:-1])[len(prompt):]
    return oscores.scores(rows, np.array(drawn), 0)[0]


def check_clean(gen):
    torch.cuda.synchronize()
    assert gen.free_count.item() == gen.pages and (gen.shares == 0).all() and gen.reserved == 0
    assert gen.slots == [None] * gen.batch


def test_samples_follow_the_fp64_model(made, sharing):
    from sejong_b200.generate import Sampling
    gen = generator(made)
    prompts = [b"ab", b"some words that fill more than a page", b"", b"another prompt of this batch, the last"]
    options = [Sampling(max_bytes=n, temperature=1.0, seed=7 + n) for n in (9, 14, 5, 11)]
    found = gen.generate(prompts, options, top=2, samples=3)
    check_clean(gen)
    for prompt, o, done in zip(prompts, options, found):
        assert len(done) == 3 and len({d.text for d in done}) > 1
        for d in done:
            drawn = list(d.text) + ([256] if d.ended else [])
            assert len(drawn) == o.max_bytes or d.ended
            assert np.abs(np.array(d.scores.logp) - logp_of(made, prompt, drawn)).max() < 0.1
            assert all(len(a) == 2 for a in d.scores.alternatives)


def test_greedy_samples_are_alike_and_equal_single_requests(made, sharing):
    """Without randomness every sample is the same; a byte may differ from a single request's only where two logits lie
    within the noise."""
    from sejong_b200.generate import Sampling
    gen = generator(made)
    o = Sampling(max_bytes=12, temperature=0.0)
    alone = gen.generate([b"a prompt of twenty bytes"], o)[0]
    found = gen.generate([b"a prompt of twenty bytes"], o, samples=8)[0]
    assert len({d.text for d in found}) == 1
    c, params = made
    seq = [256] + list(b"a prompt of twenty bytes")
    for byte in found[0].text:
        ref = logits(params, c, seq)[-1]
        assert ref[byte] >= ref.max() - 0.05 * np.abs(ref).max()
        seq.append(byte)
    assert alone == gen.generate([b"a prompt of twenty bytes"], o)[0]  # and sharing leaves the other way as it was


def test_samples_of_a_full_context_start_again(made):
    from sejong_b200.generate import Sampling
    gen = generator(made, context=32, page=8, batch=4, pages=40)
    found = gen.generate([b"0123456789012345678901234"], Sampling(max_bytes=20, temperature=0.9, seed=5), samples=4)[0]
    assert all(len(d.text) == 20 or d.ended for d in found)
    check_clean(gen)


@pytest.mark.parametrize("page", [8, 64])
def test_a_whole_batch_of_continuations_on_a_default_cache(made, page):
    """Samples that start again from a full context, and beams that fill it, of prompts shorter and longer than a page."""
    from sejong_b200.generate import Sampling
    gen = generator(made, context=32, page=page, batch=4)
    for prompt in (b"ab", b"0123456789012345678901234"):
        found = gen.generate([prompt], Sampling(max_bytes=33, temperature=0.9, seed=5), samples=4)[0]
        assert all(len(d.text) == 33 or d.ended for d in found)
        check_clean(gen)
        found = gen.beam_search([prompt], beams=4, max_bytes=31 - len(prompt))[0]
        assert found and all(len(h.text) == 31 - len(prompt) or h.ended for h in found)
        check_clean(gen)


def test_more_prompts_than_blocks_and_few_pages(made, sharing):
    from sejong_b200.generate import Sampling
    gen = generator(made, batch=5, page=4, pages=50)
    prompts = [bytes([65 + i]) * (3 + 5 * i) for i in range(7)]
    found = gen.generate(prompts, Sampling(max_bytes=6, temperature=0.8, seed=1), top=0, samples=2)
    for prompt, done in zip(prompts, found):
        for d in done:
            drawn = list(d.text) + ([256] if d.ended else [])
            assert np.abs(np.array(d.scores.logp) - logp_of(made, prompt, drawn)).max() < 0.1
    check_clean(gen)


def reference_beams(made, prompt, beams, most):
    """A beam search on the FP64 model: (ranked, text) of the best."""
    c, params = made
    live, ended = [([], 0.0)], []
    for _ in range(most):
        rows = []
        for drawn, score in live:
            x = logits(params, c, [256] + list(prompt) + drawn)[-1]
            rows.append(score + oscores.statistics(x[None])[2][0])
        order = np.argsort(-np.concatenate(rows), kind="stable")[:2 * beams]
        new = []
        for at, i in enumerate(order):
            p, t = divmod(int(i), 257)
            if len(new) == beams:
                break
            if t == 256:
                if at < beams:
                    ended.append((rows[p][t] / (len(live[p][0]) + 1), live[p][0]))
                continue
            new.append((live[p][0] + [t], rows[p][t]))
        live = new
    return max(ended + [(s / len(d), d) for d, s in live])


@pytest.mark.parametrize("beams", [1, 3, 8])
def test_beam_search(made, sharing, beams):
    gen = generator(made)
    prompts, most = [b"", b"a prompt that is longer than one page", b"xy"], 7
    found = gen.beam_search(prompts, beams=beams, max_bytes=most)
    check_clean(gen)
    for prompt, hyps in zip(prompts, found):
        assert 1 <= len(hyps) <= beams and [h.ranked for h in hyps] == sorted([h.ranked for h in hyps], reverse=True)
        assert len({(h.text, h.ended) for h in hyps}) == len(hyps)
        for h in hyps:
            drawn = list(h.text) + ([256] if h.ended else [])
            assert len(h.text) == most or h.ended
            assert abs(h.score - logp_of(made, prompt, drawn).sum()) < 0.1 * len(drawn)
            assert h.ranked == pytest.approx(h.score / len(drawn))
        best, _ = reference_beams(made, prompt, beams, most)
        assert hyps[0].ranked > best - 0.2


def test_calls_that_are_refused(made):
    from sejong_b200.generate import Sampling
    gen = generator(made, context=32, page=8, pages=12, batch=4)
    for bad in (dict(samples=0), dict(samples=5)):
        with pytest.raises(ValueError):
            gen.generate([b"a"], Sampling(max_bytes=3), **bad)
    with pytest.raises(ValueError, match="pages"):
        gen.generate([b"a" * 20], Sampling(max_bytes=12), samples=4)
    with pytest.raises(ValueError, match="fills the context"):
        gen.generate([b"a" * 40], Sampling(max_bytes=2), samples=2)
    with pytest.raises(ValueError, match="beams"):
        gen.beam_search([b"a"], beams=5)
    with pytest.raises(ValueError, match="fit the context"):
        gen.beam_search([b"a" * 30], beams=2, max_bytes=10)
    with pytest.raises(ValueError, match="max_bytes"):
        gen.beam_search([b"a"], beams=2, max_bytes=0)
    assert gen.beam_search([], beams=2) == [] and gen.generate([], Sampling(), samples=2) == []


def test_a_call_that_is_broken_off_leaves_an_empty_cache(made, monkeypatch):
    from sejong_b200.generate import Sampling
    gen = generator(made)
    want = gen.generate([b"one", b"two"], Sampling(max_bytes=6, temperature=0.7, seed=2), samples=3)
    count = [0]
    check = gen._check_shared

    def failing():
        count[0] += 1
        if count[0] == 4:
            raise KeyboardInterrupt
        check()

    monkeypatch.setattr(gen, "_check_shared", failing)
    with pytest.raises(KeyboardInterrupt):
        gen.generate([b"one", b"two"], Sampling(max_bytes=6, temperature=0.7, seed=2), samples=3)
    monkeypatch.undo()
    check_clean(gen)
    assert gen.generate([b"one", b"two"], Sampling(max_bytes=6, temperature=0.7, seed=2), samples=3) == want


def test_a_step_whose_fork_fails_is_an_error(made):
    gen = generator(made)
    gen.beam_search([b"warm"], beams=2, max_bytes=2)
    free = gen._write_shared

    def broken(parents, *rest):
        free([99] * gen.batch, *rest)

    gen._write_shared = broken
    with pytest.raises(RuntimeError, match="of the fork 4"):
        gen.beam_search([b"warm"], beams=2, max_bytes=2)
    gen._write_shared = free
    check_clean(gen)


def test_command(tmp_path, made):
    from sejong_b200 import checkpoint, cli
    c, params = made
    where = os.path.join(str(tmp_path), "model")
    checkpoint.save(where, c, params, 0)
    prompts = os.path.join(str(tmp_path), "prompts.txt")
    with open(prompts, "wb") as fh:
        fh.write(b"first line\nsecond\n")
    out = io.StringIO()
    cli.generate_batch(where, prompts, 5, 0.8, 0, 0.95, 3, 6, 16, None, 1, out=out, samples=3)
    records = [json.loads(x) for x in out.getvalue().splitlines()]
    assert [len(r["samples"]) for r in records] == [3, 3] and "scores" in records[0]["samples"][0]
    out = io.StringIO()
    cli.generate_batch(where, prompts, 5, 0.8, 0, 0.95, 3, 6, 16, None, None, out=out, beams=2)
    records = [json.loads(x) for x in out.getvalue().splitlines()]
    assert [r["prompt"] for r in records] == ["first line", "second"]
    assert [len(r["beams"]) for r in records] == [2, 2] and records[0]["beams"][0]["score"] < 0
