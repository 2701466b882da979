"""Batched generation, scoring and differentiable scores on the GPU (sejong_b200/serve.py, scores.py) against the
FP64 model: the dense byte model at the bf16-cast weights, as for the single-sequence generator.

Greedy bytes have to be within 5% of the largest FP64 logit (the bf16 bar of the path, as in
test_gpu_generate.py); log probabilities and entropies of logits that are off by at most 2e-2 of their norm over
257 entries are off by a few hundredths, bounded here by 0.1."""
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


def _model():
    return pm.with_(pm.config_c1(), layers=2)


def _oracle_logits(params, c, tokens):
    oc = omodel.ModelConfig(width=c.width, layers=c.layers, heads=c.heads, ffn_width=c.ffn_width, kv_heads=c.kv_heads,
                            rope_theta=c.rope_theta, norm_epsilon=c.norm_epsilon, seed=c.seed, init_std=c.init_std)
    p = {k: torch.tensor(v, dtype=torch.float64) for k, v in omodel.compute_cast(params, "bf16").items()}
    ids = torch.as_tensor(np.asarray(tokens, dtype=np.int64))
    with torch.no_grad():
        return (omodel.hidden(p, oc, ids, len(tokens)) @ p["output"]).numpy()[:, :257]


@pytest.fixture(scope="module")
def made():
    # weights four times the usual size: logits of some units, so that greedy choices and scores mean something
    c = pm.with_(_model(), init_std=0.08)
    return c, pm.initialize(c)


def _follow(params, c, prompt, done, top, context):
    """Every drawn byte against the FP64 model given the bytes before it."""
    seq = [256] + list(prompt)
    drawn = list(done.text) + ([256] if done.ended else [])
    assert len(done.scores.logp) == len(done.scores.entropy) == len(done.scores.alternatives) == len(drawn)
    for i, byte in enumerate(drawn):
        ref = _oracle_logits(params, c, seq[-context:])[-1]
        assert ref[byte] >= ref.max() - 0.05 * np.abs(ref).max(), (i, byte, int(ref.argmax()))
        logp, entropy, _, _, _ = oscores.scores(ref[None], np.array([byte]), top)
        assert abs(done.scores.logp[i] - logp[0]) < 0.1
        assert abs(done.scores.entropy[i] - entropy[0]) < 0.1
        best = done.scores.alternatives[i]
        assert len(best) == top and [p for _, p in best] == sorted([p for _, p in best], reverse=True)
        if top:
            assert best[0][0] == byte and abs(best[0][1] - done.scores.logp[i]) < 1e-6  # greedy: the best itself
        seq.append(byte)


def test_greedy_batch_follows_the_fp64_model(made):
    """More requests than slots, fewer pages than they would like, prompts from empty to long: all follow the model."""
    from sejong_b200.generate import Sampling
    from sejong_b200.serve import BatchGenerator
    c, params = made
    gen = BatchGenerator(c, params, device=0, context=256, batch=3, page=7, pages=60)
    rng = np.random.default_rng(0)
    prompts = [bytes(rng.integers(0, 256, n).astype(np.uint8)) for n in (5, 0, 200, 31, 64, 1)]
    options = [Sampling(max_bytes=n, temperature=0.0) for n in (9, 12, 8, 1, 10, 15)]
    done = gen.generate(prompts, options, top=3)
    for prompt, option, result in zip(prompts, options, done):
        assert result.ended or len(result.text) == option.max_bytes
        _follow(params, c, prompt, result, 3, 256)
    # every page came back
    gen._write({}, [])
    gen._commit_and_plan(0)
    torch.cuda.synchronize()
    assert gen.free_count.item() == 60 and sorted(gen.free.tolist()) == list(range(60))
    assert (gen.lengths == 0).all() and gen.reserved == 0


def test_requests_do_not_touch_each_other(made):
    """The same request alone and among others, in the same generator: the same bytes and scores, bit for bit (its rows
    are computed by the same kernels on the same values)."""
    from sejong_b200.generate import Sampling
    from sejong_b200.serve import BatchGenerator
    c, params = made
    gen = BatchGenerator(c, params, device=0, context=128, batch=4, page=16)
    one = Sampling(max_bytes=20, temperature=0.9, seed=7)
    alone = gen.generate([b"a prompt"], one, top=2)[0]
    others = [Sampling(max_bytes=n, temperature=1.0, seed=n) for n in (30, 5, 11)]
    among = gen.generate([b"x" * 40, b"a prompt", b"", b"zz"], [others[0], one, others[1], others[2]], top=2)[1]
    assert alone.text == among.text and alone.ended == among.ended
    assert alone.scores == among.scores


def test_full_context_restarts_from_its_tail(made):
    from sejong_b200.generate import Sampling
    from sejong_b200.serve import BatchGenerator
    c, params = made
    gen = BatchGenerator(c, params, device=0, context=32, batch=2, page=8)
    prompts = [b"0123456789" * 2, b"short"]
    done = gen.generate(prompts, Sampling(max_bytes=16, temperature=0.0), top=1)
    for prompt, result in zip(prompts, done):
        assert result.ended or len(result.text) == 16
        _follow(params, c, prompt, result, 1, 32)


def test_score_of_a_text(made):
    from sejong_b200.serve import BatchGenerator
    c, params = made
    gen = BatchGenerator(c, params, device=0, context=300, batch=2, page=16)
    rng = np.random.default_rng(5)
    for n in (1, 77, 300):
        text = bytes(rng.integers(0, 256, n).astype(np.uint8))
        got = gen.score(text, top=5)
        ref = _oracle_logits(params, c, [256] + list(text)[:-1])
        logp, entropy, _, _, best = oscores.scores(ref, np.frombuffer(text, dtype=np.uint8).astype(np.int64), 5)
        np.testing.assert_allclose(got.logp, logp, atol=0.1)
        np.testing.assert_allclose(got.entropy, entropy, atol=0.1)
        np.testing.assert_allclose([[p for _, p in row] for row in got.alternatives], best, atol=0.1)
    assert gen.score(b"").logp == []
    with pytest.raises(ValueError, match="longer than the context"):
        gen.score(b"x" * 301)


@pytest.mark.parametrize("kind,factor", [("linear", 4.0), ("base", 4.0), ("ramp", 4.0)])
def test_scaled_positions_serve_a_longer_context(made, kind, factor):
    """The generator's tables are the scaled ones for prompts and decode steps alike: a decoded byte's scores equal
    those of the whole text in one pass."""
    from sejong_b200.generate import Sampling
    from sejong_b200.serve import BatchGenerator, RopeScaling
    c, params = made
    gen = BatchGenerator(c, params, device=0, context=128, batch=2, page=16,
                         rope_scaling=RopeScaling(kind, factor, original=32))
    prompt = b"positions past the trained ones, "
    done = gen.generate([prompt], Sampling(max_bytes=24, temperature=0.0), top=0)[0]
    whole = gen.score(prompt + done.text)
    n = len(done.text)
    # two bf16 evaluations of the same row
    np.testing.assert_allclose(done.scores.logp[:n], whole.logp[len(prompt):], atol=0.1)
    plain = BatchGenerator(c, params, device=0, context=128, batch=2, page=16).score(prompt + done.text)
    assert np.abs(np.array(plain.logp) - np.array(whole.logp)).max() > 1e-3


def test_generate_refuses(made):
    from sejong_b200.generate import Sampling
    from sejong_b200.serve import BatchGenerator
    c, params = made
    gen = BatchGenerator(c, params, device=0, context=64, batch=2, page=16, pages=2)
    with pytest.raises(ValueError, match="pages"):
        gen.generate([b"x" * 40], Sampling(max_bytes=4))
    with pytest.raises(ValueError, match="Sampling"):
        gen.generate([b"x"], [Sampling(), Sampling()])
    with pytest.raises(ValueError, match="top"):
        gen.generate([b"x"], Sampling(max_bytes=1), top=33)
    with pytest.raises(ValueError, match="max_bytes"):
        gen.generate([b"x"], Sampling(max_bytes=0))
    assert len(gen.generate([b"still works"], Sampling(max_bytes=3, temperature=1.0))[0].text) <= 3


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_differentiable_scores(dtype):
    """Through torch autograd, with a strided view of logits, against autograd of the formula in 64 bits."""
    from sejong_b200.scores import token_scores
    gen = torch.Generator().manual_seed(0)
    base = torch.randn(50, 264, generator=gen).to(dtype).cuda().requires_grad_()
    target = torch.randint(0, 257, (50,), generator=gen).cuda()
    a, b = torch.randn(50, generator=gen).cuda(), torch.randn(50, generator=gen).cuda()
    got = token_scores(base[:, :257], target, top=4)
    (got.logp * a + got.entropy * b).sum().backward()
    x = base.detach().double()[:, :257].requires_grad_()
    logp = torch.log_softmax(x, 1)
    entropy = -(logp.exp() * logp).sum(1)
    picked = logp.gather(1, target[:, None])[:, 0]
    (picked * a.double() + entropy * b.double()).sum().backward()
    torch.testing.assert_close(got.logp.double(), picked.detach(), rtol=0, atol=2e-5)
    torch.testing.assert_close(got.entropy.double(), entropy.detach(), rtol=0, atol=2e-5)
    grad = base.grad.double()
    assert (grad[:, 257:] == 0).all()
    bound = 1e-5 if dtype == torch.float32 else 2.0 ** -8
    assert (grad[:, :257] - x.grad).norm() <= bound * x.grad.norm()
    assert torch.equal(got.top_id.long(), logp.topk(4, 1).indices) or dtype == torch.bfloat16


def test_commands(tmp_path, made):
    from sejong_b200 import checkpoint, cli
    c, params = made
    c = pm.with_(c, context=128)
    where = os.path.join(str(tmp_path), "model")
    checkpoint.save(where, c, params, 0)
    prompts = os.path.join(str(tmp_path), "prompts.txt")
    with open(prompts, "wb") as fh:
        fh.write(b"first line\nsecond\n")
    out = io.StringIO()
    cli.generate_batch(where, prompts, 6, 0.8, 0, 0.95, 3, 2, 16, None, 2, out=out)
    records = [json.loads(x) for x in out.getvalue().splitlines()]
    assert [r["prompt"] for r in records] == ["first line", "second"]
    assert all(len(r["scores"]["alternatives"][0]) == 2 for r in records)
    out = io.StringIO()
    cli.score(where, prompts, 1, out=out)
    record = json.loads(out.getvalue())
    assert record["bytes"] == 18 and len(record["logp"]) == 18 and record["bits_per_byte"] > 0


# ---------------------------------------------------------------- calls that fail
def _all_pages_free(gen):
    gen._write({}, [])
    gen._commit_and_plan(0)
    torch.cuda.synchronize()
    assert gen.free_count.item() == gen.pages and sorted(gen.free.tolist()) == list(range(gen.pages))
    assert (gen.lengths == 0).all() and gen.reserved == 0 and gen.slots == [None] * gen.batch


@pytest.mark.parametrize("bad", [dict(top_p=0.0), dict(top_p=1.5), dict(temperature=-1.0),
                                 dict(temperature=float("nan"))])
def test_generate_checks_the_options_before_it_takes_a_request(made, bad):
    from sejong_b200.generate import Sampling
    from sejong_b200.serve import BatchGenerator
    c, params = made
    gen = BatchGenerator(c, params, device=0, context=64, batch=2, page=16)
    good = Sampling(max_bytes=5, temperature=0.9, seed=3)
    want = gen.generate([b"good", b"ones"], good, top=1)
    with pytest.raises(ValueError, match="temperature"):
        gen.generate([b"first", b"bad"], [good, Sampling(max_bytes=5, **bad)], top=1)
    _all_pages_free(gen)
    assert gen.generate([b"good", b"ones"], good, top=1) == want


@pytest.mark.parametrize("at", ["first draw", "later draw", "between the host's write and the step", "step"])
def test_generate_after_a_call_that_was_broken_off(made, monkeypatch, at):
    """Whatever a call that raised has left behind, the next one starts from an empty cache."""
    from sejong_b200.generate import Sampling
    from sejong_b200.serve import BatchGenerator
    c, params = made
    gen = BatchGenerator(c, params, device=0, context=64, batch=2, page=16)
    good = Sampling(max_bytes=8, temperature=0.9, seed=3)
    want = gen.generate([b"good", b"ones", b"more"], good, top=1)
    name, calls = {"first draw": ("_draw", 1), "later draw": ("_draw", 6), "step": ("_step", 2),
                   "between the host's write and the step": ("_commit_and_plan", 2)}[at]
    whole, count = getattr(gen, name), [0]

    def broken(*args):
        count[0] += 1
        if count[0] == calls:
            raise KeyboardInterrupt
        return whole(*args)

    with monkeypatch.context() as m:
        m.setattr(gen, name, broken)
        with pytest.raises(KeyboardInterrupt):
            gen.generate([b"a", b"b", b"c", b"d"], Sampling(max_bytes=30, temperature=1.0), top=0)
    assert count[0] == calls
    # one request: had it the old ones beside it, their completions would go past its results
    assert gen.generate([b"good"], good, top=1) == want[:1]
    assert gen.generate([b"good", b"ones", b"more"], good, top=1) == want
    _all_pages_free(gen)


def test_generate_reports_a_step_that_could_not_be_planned(made):
    """A cache whose free pages are gone: an error, not bytes of a step that never ran; the next call is whole again."""
    from sejong_b200.generate import Sampling
    from sejong_b200.serve import BatchGenerator
    c, params = made
    gen = BatchGenerator(c, params, device=0, context=64, batch=2, page=4)
    good = Sampling(max_bytes=8, temperature=0.9, seed=3)
    want = gen.generate([b"good", b"ones"], good)
    _all_pages_free(gen)  # those of finished requests as well, which the next commit would return
    gen.free_count.zero_()  # no page for a prompt
    with pytest.raises(RuntimeError, match="status 2"):
        gen.generate([b"good", b"ones"], good)
    assert gen.generate([b"good", b"ones"], good) == want
    start = gen._start

    def last_pages(*args):  # pages for the prompt, none for the step that needs one more
        start(*args)
        gen.free_count.fill_(2)  # what the step's commit takes off for the prompt's two pages

    gen._start = last_pages
    with pytest.raises(RuntimeError, match="status 2"):
        gen.generate([b"seven b"], Sampling(max_bytes=8, temperature=0.0))
    del gen._start
    assert gen.generate([b"good", b"ones"], good) == want


def test_differentiable_scores_refuse_a_second_derivative():
    """The gradient kernel's result has no derivative of its own: asking for one is an error, not a term left out.  The
    first derivative can be part of a graph."""
    from sejong_b200.scores import token_scores
    x = torch.randn(5, 257, device="cuda", requires_grad=True)
    target = torch.arange(5, device="cuda")
    got = token_scores(x, target)
    plain, = torch.autograd.grad(got.logp.sum() + got.entropy.sum(), x, retain_graph=True)
    g, = torch.autograd.grad(got.logp.sum() + got.entropy.sum(), x, create_graph=True)
    assert torch.equal(g, plain)
    for again in (g, torch.autograd.grad(got.logp.sum() + (x * x).sum(), x, create_graph=True)[0]):
        with pytest.raises(RuntimeError, match="token_scores has no derivative"):
            again.sum().backward()
    # a gradient that comes back with a graph of its own, and logits without one
    scale, logits = torch.ones((), device="cuda", requires_grad=True), x.detach().requires_grad_()
    g, = torch.autograd.grad(token_scores(logits, target).logp.sum() * scale, logits, create_graph=True)
    with pytest.raises(RuntimeError, match="token_scores has no derivative"):
        torch.autograd.grad(g.sum(), scale)


@pytest.mark.parametrize("strides", [(1, 1), (0, 1), (7, 1), (3, 2), (2 ** 32 + 264, 1), (2 ** 31 + 8, 1)])
@pytest.mark.parametrize("rows", [1, 3])
def test_differentiable_scores_of_any_row_stride(rows, strides):
    """Rows that overlap, one row of any stride, strides past 32 bits: the values of a contiguous copy."""
    from sejong_b200.scores import token_scores
    vocab = 257
    base = torch.empty((rows - 1) * strides[0] + (vocab - 1) * strides[1] + 1, dtype=torch.bfloat16, device="cuda")
    x = base.as_strided((rows, vocab), strides)
    gen = torch.Generator(device="cuda").manual_seed(1)
    for r in range(rows):
        x[r] = torch.randn(vocab, generator=gen, device="cuda").bfloat16()
    target = torch.arange(rows, device="cuda")
    want_x = x.clone(memory_format=torch.contiguous_format).view(-1).view(rows, vocab).requires_grad_()
    x = x.detach().requires_grad_()
    got, want = token_scores(x, target, top=3), token_scores(want_x, target, top=3)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    g, = torch.autograd.grad(got.logp.sum() + got.entropy.sum(), x)
    w, = torch.autograd.grad(want.logp.sum() + want.entropy.sum(), want_x)
    assert torch.equal(g, w)
    ref = torch.log_softmax(x.detach().double(), 1)
    torch.testing.assert_close(got.logp.double(), ref.gather(1, target[:, None])[:, 0], rtol=0, atol=2e-5)


def test_differentiable_scores_select_the_device_of_the_logits(monkeypatch):
    """Forward and backward are launched with the logits' GPU current, whichever is outside."""
    from sejong_b200 import scores
    inside, seen, device = [], [], torch.cuda.device

    class Recorded(device):
        def __enter__(self):
            inside.append(self.idx)
            return super().__enter__()

        def __exit__(self, *args):
            inside.pop()
            return super().__exit__(*args)

    launch = scores.call
    monkeypatch.setattr(torch.cuda, "device", Recorded)
    monkeypatch.setattr(scores, "call", lambda name, *args: (seen.append((name, list(inside))), launch(name, *args))[1])
    x = torch.randn(4, 257, device="cuda:0", requires_grad=True)
    scores.token_scores(x, torch.arange(4, device="cuda:0")).logp.sum().backward()
    assert seen == [("sj_token_scores", [0]), ("sj_token_scores_bwd", [0])]


def test_a_generator_can_be_used_on_another_stream_than_it_was_made_on(made, monkeypatch):
    """What the constructor has launched is done when it returns: a call on another stream does not wait for it."""
    from sejong_b200 import serve
    c, params = made
    launch = serve.call

    def slow(name, *args):
        launch(name, *args)
        if name == "sj_rope_table":
            torch.cuda._sleep(200_000_000)  # a tenth of a second

    # a new pinned buffer waits for the GPU, one of an earlier generator does not
    serve.BatchGenerator(c, params, device=0, context=64, batch=2, page=16)
    monkeypatch.setattr(serve, "call", slow)
    gen = serve.BatchGenerator(c, params, device=0, context=64, batch=2, page=16)
    assert torch.cuda.current_stream().query()
    monkeypatch.setattr(serve, "call", launch)
    want = gen.score(b"some text")
    other = torch.cuda.Stream()
    with torch.cuda.stream(other):
        assert gen.score(b"some text") == want
