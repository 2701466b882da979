"""Refusals of the paged-serving and token-score entry points (checked before anything is launched, so they
need no GPU) and the restatements' own properties."""
import numpy as np
import pytest
import torch

from oracle import paged as opaged
from oracle import scores as oscores


@pytest.fixture(scope="module")
def lib():
    from sejong_b200 import _lib, build
    build.build()
    return _lib.load()


def refused(name, args, code):
    from sejong_b200._lib import SejongError, call
    with pytest.raises(SejongError) as e:
        call(name, *args)
    assert e.value.code == code, str(e.value)
    assert name in str(e.value)


SHAPE, CAPACITY, ARGUMENT, UNSUPPORTED = 1, 2, 6, 7
A = 1 << 20  # an address that passes the checks of alignment; nothing is launched


def change(args, **kw):
    names = list(args)
    assert set(kw) <= set(names), kw
    return [kw.get(n, args[n]) for n in names]


PLAN = dict(cached=A, added=A, batch=4, page=16, free=A, count=A, table=A, ld_table=8, lengths=A, request=A, position=A,
            slot=A, rows=8, summary=A, stream=0)


@pytest.mark.parametrize("kw,code", [(dict(batch=0), SHAPE), (dict(batch=4097), SHAPE), (dict(page=0), SHAPE),
                                     (dict(ld_table=0), SHAPE), (dict(rows=-1), SHAPE), (dict(rows=(1 << 19) + 1), SHAPE),
                                     (dict(cached=0), ARGUMENT), (dict(free=0), ARGUMENT), (dict(slot=0), ARGUMENT),
                                     (dict(summary=0), ARGUMENT)])
def test_plan_refusals(lib, kw, code):
    refused("sj_paged_plan", change(PLAN, **kw), code)


COMMIT = dict(cached=A, lengths=A, release=0, batch=4, page=16, table=A, ld_table=8, free=A, count=A, pages=10, summary=A,
              stream=0)


@pytest.mark.parametrize("kw,code", [(dict(batch=0), SHAPE), (dict(batch=5000), SHAPE), (dict(pages=0), SHAPE),
                                     (dict(cached=0), ARGUMENT), (dict(free=0), ARGUMENT)])
def test_commit_refusals(lib, kw, code):
    refused("sj_paged_commit", change(COMMIT, **kw), code)


ROPE = dict(table=A, t=16, rope_dim=64, offset=0, theta=1e4, scaling=0, factor=1.0, original=2048, fast=32.0, slow=1.0,
            stream=0)


@pytest.mark.parametrize("kw,code", [(dict(t=0), SHAPE), (dict(rope_dim=7), SHAPE), (dict(offset=-1), SHAPE),
                                     (dict(offset=2 ** 31 - 2), SHAPE), (dict(table=0), ARGUMENT), (dict(theta=0.0), ARGUMENT),
                                     (dict(theta=float("nan")), ARGUMENT), (dict(scaling=4), ARGUMENT),
                                     (dict(scaling=1, factor=0.5), ARGUMENT), (dict(scaling=3, factor=2.0, original=0), ARGUMENT),
                                     (dict(scaling=3, factor=2.0, fast=1.0, slow=1.0), ARGUMENT)])
def test_rope_table_refusals(lib, kw, code):
    refused("sj_rope_table_scaled", change(ROPE, **kw), code)


CACHE = dict(pages=8, page=16, page_stride=2048, head_stride=1024, token_stride=64)
APPEND = dict(qkv=A, ld=512, position=A, slot=A, rows=3, hq=4, hk=2, dim=64, rope=A, rope_len=100, rope_dim=64, half=0, q=A,
              ldq=256, k=A, v=A, **CACHE, stream=0)


@pytest.mark.parametrize("kw,code", [
    (dict(dim=96), UNSUPPORTED), (dict(rows=-1), SHAPE), (dict(hk=0), SHAPE), (dict(rope_dim=24), SHAPE),
    (dict(rope_dim=80), SHAPE), (dict(rope_len=0), SHAPE), (dict(ld=504), SHAPE), (dict(ldq=248), SHAPE),
    (dict(pages=0), SHAPE), (dict(pages=1 << 28), SHAPE), (dict(page_stride=1 << 34), SHAPE),
    (dict(token_stride=60), ARGUMENT), (dict(head_stride=-64), ARGUMENT), (dict(k=A + 8), ARGUMENT), (dict(v=0), ARGUMENT),
    (dict(qkv=0), ARGUMENT), (dict(qkv=A + 2), ARGUMENT), (dict(ld=515), ARGUMENT), (dict(rope=0), ARGUMENT),
    (dict(q=0), ARGUMENT)])
def test_append_refusals(lib, kw, code):
    refused("sj_paged_append", change(APPEND, **kw), code)


ATTEND = dict(q=A, ldq=256, k=A, v=A, **CACHE, table=A, ld_table=8, requests=3, request=0, position=A, rows=3, hq=4, hk=2,
              dim=64, window=0, o=A, ldo=256, lse=0, work=A, size=1 << 30, stream=0)


@pytest.mark.parametrize("kw,code", [
    (dict(dim=32), UNSUPPORTED), (dict(rows=-1), SHAPE), (dict(hq=5), SHAPE), (dict(hk=0), SHAPE), (dict(window=-1), SHAPE),
    (dict(rows=4), SHAPE), (dict(ld_table=0), SHAPE), (dict(ldq=248), SHAPE), (dict(ldo=128), SHAPE),
    (dict(page=0), SHAPE), (dict(page_stride=2050), ARGUMENT), (dict(k=A + 4), ARGUMENT), (dict(q=0), ARGUMENT),
    (dict(o=A + 2), ARGUMENT), (dict(ldo=260), ARGUMENT), (dict(table=0), ARGUMENT), (dict(position=0), ARGUMENT),
    (dict(work=0), CAPACITY), (dict(size=0), CAPACITY)])
def test_attention_refusals(lib, kw, code):
    refused("sj_attn_paged", change(ATTEND, **kw), code)


SCORES = dict(logits=A, dtype=0, ld=100, target=A, rows=3, vocab=100, top=5, logp=A, entropy=A, lse=A, top_id=A, top_logp=A,
              work=A, size=1 << 30, stream=0)


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=2), UNSUPPORTED), (dict(rows=-1), SHAPE), (dict(vocab=0), SHAPE), (dict(ld=99), SHAPE), (dict(top=33), SHAPE),
    (dict(top=-1), SHAPE), (dict(vocab=4, top=5), SHAPE), (dict(logits=0), ARGUMENT), (dict(logits=A + 2), ARGUMENT),
    (dict(dtype=4, logits=A + 1), ARGUMENT), (dict(target=0), ARGUMENT), (dict(top_id=0), ARGUMENT),
    (dict(top_logp=0), ARGUMENT), (dict(work=0), CAPACITY), (dict(size=0), CAPACITY)])
def test_score_refusals(lib, kw, code):
    refused("sj_token_scores", change(SCORES, **kw), code)


GRADIENT = dict(logits=A, dtype=0, ld=100, target=A, rows=3, vocab=100, lse=A, entropy=A, d_logp=A, d_entropy=A, d=2 * A,
                ldd=100, stream=0)


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=1), UNSUPPORTED), (dict(rows=-1), SHAPE), (dict(vocab=0), SHAPE), (dict(ld=99), SHAPE), (dict(ldd=99), SHAPE),
    (dict(logits=0), ARGUMENT), (dict(d=0), ARGUMENT), (dict(d=A + 1), ARGUMENT), (dict(lse=0), ARGUMENT),
    (dict(d_logp=0, d_entropy=0), ARGUMENT), (dict(target=0), ARGUMENT), (dict(entropy=0), ARGUMENT),
    (dict(d=A, ldd=104), ARGUMENT)])
def test_gradient_refusals(lib, kw, code):
    refused("sj_token_scores_bwd", change(GRADIENT, **kw), code)


def test_no_rows_is_no_work(lib):
    from sejong_b200._lib import call
    call("sj_paged_append", *change(APPEND, rows=0, qkv=0, position=0, slot=0))
    call("sj_attn_paged", *change(ATTEND, rows=0, q=0, o=0, table=0, position=0))
    call("sj_token_scores", *change(SCORES, rows=0, logits=0))
    call("sj_token_scores_bwd", *change(GRADIENT, rows=0, logits=0))


def test_restated_attention_equals_one_softmax_over_contiguous_keys():
    g = torch.Generator().manual_seed(0)
    q = torch.randn(2, 4, 64, generator=g, dtype=torch.float64)
    k, v = (torch.randn(5, 2, 8, 64, generator=g, dtype=torch.float64) for _ in range(2))
    table = torch.tensor([[3, 0, 4], [1, 2, 0]])
    o, lse, _, _ = opaged.attention(q, k, v, table, [0, 1], [18, 11], 8)
    for r, n in ((0, 19), (1, 12)):
        for h in range(4):
            keys = torch.cat([k[i, h // 2] for i in table[r]])[:n]
            vals = torch.cat([v[i, h // 2] for i in table[r]])[:n]
            s = keys @ q[r, h] / 8.0
            torch.testing.assert_close(o[r, h], torch.softmax(s, 0) @ vals)
            torch.testing.assert_close(lse[r, h], torch.logsumexp(s, 0))


def test_restated_gradient_against_differences():
    rng = np.random.default_rng(1)
    x, target = rng.standard_normal((3, 11)), np.array([2, -1, 10])
    a, b = rng.standard_normal(3), rng.standard_normal(3)

    def value(y):
        logp, entropy, *_ = oscores.scores(y, target, 0)
        return (a * logp + b * entropy).sum()

    g = oscores.gradient(x, target, a, b)
    for i in range(3):
        for j in range(11):
            e = np.zeros_like(x)
            e[i, j] = 1e-5
            assert abs((value(x + e) - value(x - e)) / 2e-5 - g[i, j]) < 1e-8


def test_restated_scaled_tables():
    """A factor of 1 changes nothing but the ramp's table keeps its amplitude of 1; linear interpolation is a
    position divided by the factor; the changed base divides the lowest frequency by the factor."""
    plain = opaged.rope_table(100, 64, 10000.0)
    for kind in ("linear", "base", "ramp"):
        np.testing.assert_allclose(opaged.rope_table(100, 64, 10000.0, scaling=kind, factor=1.0, original=64), plain, atol=1e-12)
    np.testing.assert_allclose(opaged.rope_table(400, 64, 10000.0, scaling="linear", factor=4.0)[::4], plain, atol=1e-10)
    f, _ = opaged.frequencies(64, 10000.0, scaling="base", factor=8.0)
    f0, _ = opaged.frequencies(64, 10000.0)
    assert abs(f[-1] * 8 / f0[-1] - 1) < 1e-12 and f[0] == f0[0]


# ---------------------------------------------------------------- the Python layer's own refusals
def test_batch_generator_refuses_models_it_does_not_serve():
    from sejong_b200 import model as pm
    from sejong_b200.serve import BatchGenerator, RopeScaling
    with pytest.raises(ValueError, match="dense"):
        BatchGenerator(pm.small_hierarchy())
    with pytest.raises(ValueError, match="dense"):
        BatchGenerator(pm.with_(pm.config_c5(), hierarchy=None))
    for kw in (dict(batch=0), dict(batch=5000), dict(page=0)):
        with pytest.raises(ValueError, match="batch"):
            BatchGenerator(pm.config_c1(), **kw)
    with pytest.raises(ValueError, match="rope scaling"):
        RopeScaling("cubic", 2.0).code()


def test_token_scores_refuses(lib):
    from sejong_b200.scores import token_scores
    x, t = torch.zeros(3, 5), torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="rows"):
        token_scores(x, t[:2])
    with pytest.raises(ValueError, match="rows"):
        token_scores(x[0], t)
    with pytest.raises(ValueError, match="float32 or bfloat16"):
        token_scores(x.half(), t)
    with pytest.raises(ValueError, match="GPU"):
        token_scores(x, t)


@pytest.mark.parametrize("vocab", [2 ** 31 - 1, 2 ** 31 - 2000, 2 ** 31 - 16383])
def test_scores_refuse_columns_that_32_bits_do_not_count(lib, vocab):
    for dtype in (0, 4):
        refused("sj_token_scores", change(SCORES, dtype=dtype, ld=vocab, vocab=vocab), SHAPE)
        refused("sj_token_scores_bwd", change(GRADIENT, dtype=dtype, ld=vocab, vocab=vocab, ldd=vocab), SHAPE)
        refused("sj_token_scores_bwd", change(GRADIENT, dtype=dtype, ldd=vocab), SHAPE)


def test_plan_takes_fewer_than_2_to_the_19_rows(lib):
    refused("sj_paged_plan", change(PLAN, rows=1 << 19), SHAPE)
