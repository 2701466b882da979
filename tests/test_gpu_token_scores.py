"""Token scores and their gradient against the 64-bit restatement (oracle/scores.py).

Bounds, from the arithmetic.  With d = x - max and s = sum e^d >= 1: d is rounded once (2^-24 |d|), an f32
exponential is off by at most a few 2^-23, and a sum of n of them in 32 bits in lanes, warps and parts adds at
most a few times 2^-20 for the sizes here, so log s is off by at most 2^-19 and a log probability by 2^-19 +
2^-22 |value|; the entropy is log s - sum e d / s, both parts >= 0, so off by 2^-19 (1 + its parts).  The
gradient's p is off by 2^-20 + 2^-23 |log p| of itself.  bf16 gradients are rounded once (8 significant bits: 2^-8).
"""
import ctypes

import numpy as np
import pytest
import torch

from oracle import scores as oracle

pytestmark = pytest.mark.gpu

DEV = "cuda"
F32, BF16 = 0, 4


@pytest.fixture(scope="module", autouse=True)
def lib():
    from sejong_b200 import _lib
    lib = _lib.load()
    _lib.call("sj_device_init", 0)
    return lib


@pytest.fixture(autouse=True)
def no_device_error(lib):
    yield
    assert device_error() == 0


def device_error():
    from sejong_b200._lib import call
    code = ctypes.c_int(0)
    call("sj_device_error", ctypes.byref(code), 1, stream())
    return code.value


def ptr(t):
    return 0 if t is None else t.data_ptr()


def stream():
    return torch.cuda.current_stream().cuda_stream


def run_scores(x, target, vocab, top, calls=1, optional=True):
    from sejong_b200 import _lib
    rows, ld = x.shape[0], x.stride(0)
    out = [torch.full((rows,), 9.0, device=DEV) for _ in range(3)]
    ids = torch.full((rows, top), -9, dtype=torch.int32, device=DEV)
    best = torch.full((rows, top), 9.0, device=DEV)
    size = _lib.load().sj_token_scores_workspace(rows, vocab, top)
    work = torch.zeros(max(size, 1), dtype=torch.uint8, device=DEV)
    got = []
    for _ in range(calls):
        _lib.call("sj_token_scores", ptr(x), F32 if x.dtype == torch.float32 else BF16, ld, ptr(target), rows, vocab, top,
                  *[ptr(t) if optional else 0 for t in out], ptr(ids), ptr(best), ptr(work), size, stream())
        got.append([t.cpu().numpy().copy() for t in (*out, ids, best)])
    for again in got[1:]:
        for a, b in zip(got[0], again):
            np.testing.assert_array_equal(a, b)
    return got[0]


def check_scores(x, target, vocab, top):
    got = run_scores(x, target, vocab, top, calls=2)
    exact = x[:, :vocab].double().cpu().numpy()
    want = oracle.scores(exact, target.cpu().numpy(), top)
    np.testing.assert_array_equal(got[3], want[3])
    d = np.where(np.isneginf(exact), 0.0, exact - np.maximum(exact.max(1, keepdims=True), -1e300))
    deep = np.abs(d).max(1)
    for g, w, extra in ((got[0], want[0], 0), (got[1], want[1], 1 + deep), (got[2], want[2], 0), (got[4], want[4], 0)):
        finite = np.isfinite(w)
        np.testing.assert_array_equal(np.isfinite(g), finite)
        np.testing.assert_array_equal(g[~finite], w[~finite])
        extra = np.broadcast_to(np.asarray(extra, dtype=np.float64).reshape(-1, *[1] * (w.ndim - 1)), w.shape)
        bound = 2.0 ** -19 * (1 + extra) + 2.0 ** -22 * np.abs(np.where(finite, w, 0.0))
        assert (np.abs(np.where(finite, g, 0.0) - np.where(finite, w, 0.0)) <= bound).all()


def logits(rows, vocab, ld, kind, seed, scale=3.0):
    gen = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, ld, generator=gen) * scale).to(kind)
    x[:, vocab:] = float("nan")  # the padding is not read
    target = torch.randint(-1, vocab, (rows,), generator=gen, dtype=torch.int32)
    return x.to(DEV), target.to(DEV)


@pytest.mark.parametrize("rows,vocab,ld,top", [
    (1, 1, 1, 1), (3, 2, 2, 2), (7, 31, 33, 0), (5, 32, 32, 32), (64, 257, 264, 5), (1000, 257, 264, 20), (33, 257, 257, 32),
    (9, 1000, 1001, 20), (17, 4096, 4096, 20), (4, 8191, 8200, 32), (3, 16385, 16385, 20), (2, 50001, 50008, 20),
    (300, 5003, 5008, 7), (1, 131072, 131072, 32), (2, 262147, 262147, 5)])
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
def test_scores_match_the_restatement(rows, vocab, ld, top, kind):
    check_scores(*logits(rows, vocab, ld, kind, rows + vocab), vocab, top)


@pytest.mark.parametrize("vocab", [257, 5000, 40000])
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
def test_scores_of_ties_and_orders(vocab, kind):
    """Equal logits, rising and falling rows, few distinct values, signed zeros: the lowest index first."""
    step = torch.arange(vocab, dtype=torch.float32)
    rows = [torch.zeros(vocab), torch.full((vocab,), -7.5), step / vocab, -step / vocab, (step % 3), (step % 32 == 31) * 4.0,
            torch.where(step % 2 == 0, 0.0, -0.0), (step // 64) % 5, -(step - vocab // 2).abs() / 100]
    x = torch.stack(rows).to(kind).to(DEV)
    target = torch.arange(len(rows), dtype=torch.int32, device=DEV)
    for top in (1, 5, 32):
        check_scores(x, target, vocab, top)


@pytest.mark.parametrize("vocab", [512, 513, 1024, 1025, 2047, 2048, 2049, 4095, 4096, 4097])
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
def test_scores_around_the_widths_of_the_kernels(vocab, kind):
    """Random rows, equal ones, few distinct values, all but a few forbidden, the best at either end."""
    x, target = logits(9, vocab, vocab + 3, kind, vocab)
    step = torch.arange(vocab, device=DEV)
    x[1, :vocab] = 2.0
    x[2, :vocab] = (step % 5).to(kind)
    x[3, :vocab] = torch.where(step % 31 == 7, x[3, :vocab], torch.tensor(-float("inf"), dtype=kind, device=DEV))
    x[4, vocab - 1], x[4, 0] = 30.0, 30.0
    x[5, :vocab] = torch.where(step >= vocab - 40, 40.0, 0.0).to(kind)
    target[:6] = vocab - 1
    for top in (0, 1, 8, 9):
        check_scores(x, target, vocab, top)


@pytest.mark.parametrize("vocab", [5001, 40000])
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
def test_scores_of_peaks_anywhere(vocab, kind):
    """Smooth peaks: the best logits lie side by side, many equal after rounding, at and around the ends of chunks and of a
    row's parts; each is found once."""
    step = torch.arange(vocab, dtype=torch.float32)
    at = list(range(0, vocab, 977)) + [2559, 2560, 4095, 4096, 5119, vocab - 1]
    x = torch.stack([-(step - p).abs() / 50 for p in at if p < vocab]).to(kind).to(DEV)
    target = torch.zeros(len(x), dtype=torch.int32, device=DEV)
    check_scores(x, target, vocab, 32)
    check_scores(x[:3], target[:3], vocab, 32)


@pytest.mark.parametrize("vocab", [257, 9001])
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
def test_scores_of_masked_rows(vocab, kind):
    """Forbidden tokens (-inf): most, all but one, all; the lowest finite value as a mask; huge logits."""
    gen = torch.Generator().manual_seed(vocab)
    x = torch.randn(6, vocab, generator=gen)
    x[0, torch.rand(vocab, generator=gen) < 0.97] = -float("inf")
    x[1] = -float("inf")
    x[1, 100] = 2.0
    x[2] = -float("inf")
    x[3, torch.rand(vocab, generator=gen) < 0.5] = torch.finfo(kind).min / 2
    x[4] = x[4] * 1e30
    x = x.to(kind).to(DEV)
    target = torch.tensor([0, 100, 3, 4, 5, -1], dtype=torch.int32, device=DEV)
    check_scores(x, target, vocab, 8)


def test_scores_of_nan_rows():
    """A NaN makes the row's statistics NaN, ranks last and leaves the other rows alone."""
    for vocab in (257, 20000):
        x, target = logits(4, vocab, vocab, torch.float32, 5)
        x[1, vocab // 2] = float("nan")
        x[2, 7] = float("inf")
        got = run_scores(x, target, vocab, 5)
        want = oracle.scores(x[[0, 3]].double().cpu().numpy(), target[[0, 3]].cpu().numpy(), 5)
        assert np.isnan([got[1][1], got[2][1], *got[4][1]]).all()
        assert vocab // 2 not in got[3][1]
        assert got[3][2][0] == 7 and np.isnan(got[2][2])
        np.testing.assert_array_equal(got[3][[0, 3]], want[3])
        assert np.isfinite(got[4][[0, 3]]).all()


def test_scores_of_unaligned_rows_and_no_statistics():
    base = torch.randn(40 * 1003 + 3, device=DEV)
    x = base[3:].view(40, 1003)[:, :1000]  # rows at odd 4-byte offsets
    target = torch.randint(0, 1000, (40,), dtype=torch.int32, device=DEV)
    check_scores(x, target, 1000, 20)
    only = run_scores(x, target, 1000, 3, optional=False)
    assert (only[0] == 9.0).all()
    np.testing.assert_array_equal(only[3], oracle.scores(x.double().cpu().numpy(), target.cpu().numpy(), 3)[3])


@pytest.mark.parametrize("bad", [-2, 100])
def test_scores_report_a_target_out_of_range(bad):
    x, _ = logits(3, 100, 100, torch.float32, 1)
    target = torch.tensor([1, bad, 2], dtype=torch.int32, device=DEV)
    got = run_scores(x, target, 100, 1)
    assert device_error() == 110
    assert got[0][1] == 0.0 and np.isfinite(got[1]).all()
    g = run_gradient(x, target, 100, 100, torch.ones(3, device=DEV), None)
    assert device_error() == 110
    assert (g[1] == 0).all() and (g[0] != 0).any()


# ---------------------------------------------------------------- gradient
def statistics(x, vocab):
    lse, entropy, _ = oracle.statistics(x[:, :vocab].double().cpu().numpy())
    return (torch.as_tensor(a, dtype=torch.float32).to(DEV) for a in (lse, entropy))


def run_gradient(x, target, vocab, ldd, d_logp, d_entropy, in_place=False):
    from sejong_b200 import _lib
    rows = x.shape[0]
    lse, entropy = statistics(x, vocab)
    d = x.clone() if in_place else torch.full((rows, ldd), 9.0, dtype=x.dtype, device=DEV)
    src = d if in_place else x
    _lib.call("sj_token_scores_bwd", ptr(src), F32 if x.dtype == torch.float32 else BF16, src.stride(0), ptr(target), rows,
              vocab, ptr(lse), ptr(entropy) if d_entropy is not None else 0, ptr(d_logp), ptr(d_entropy), ptr(d), ldd, stream())
    return d


def check_gradient(x, target, vocab, ldd, d_logp, d_entropy, in_place=False):
    got = run_gradient(x, target, vocab, ldd, d_logp, d_entropy, in_place).double().cpu().numpy()
    rows = x.shape[0]
    host = [np.zeros(rows) if t is None else t.double().cpu().numpy() for t in (d_logp, d_entropy)]
    exact, tgt = x[:, :vocab].double().cpu().numpy(), target.cpu().numpy()
    want = oracle.gradient(exact, tgt, *host)
    assert (got[:, vocab:] == 0).all()
    lse, entropy, logp = oracle.statistics(exact)
    lp = np.where(np.isneginf(logp), 0.0, logp)
    p = np.where(np.isneginf(logp), 0.0, np.exp(logp))
    a = np.abs(host[0])[:, None]
    size = p * (a + np.abs(host[1])[:, None] * (np.abs(lp) + entropy[:, None] + 1))
    # the kept lse and entropy are rounded to f32, too: 2^-24 of their size
    bound = size * (2.0 ** -20 + 2.0 ** -23 * (np.abs(lp) + np.abs(lse)[:, None])) + 1e-37
    hit = np.arange(vocab)[None, :] == tgt[:, None]
    bound = bound + np.where(hit, 2.0 ** -23 * a, 0.0)
    if x.dtype == torch.bfloat16:
        bound = bound + 2.0 ** -8 * np.abs(want)
    assert (np.abs(got[:, :vocab] - want) <= bound).all()


@pytest.mark.parametrize("rows,vocab,ld,ldd", [(1, 1, 1, 1), (5, 2, 3, 2), (64, 257, 264, 264), (1000, 257, 257, 264),
                                               (33, 1000, 1001, 1007), (9, 5003, 5008, 5008), (3, 50001, 50008, 50008),
                                               (2, 131075, 131075, 131080)])
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
def test_gradient_matches_the_restatement(rows, vocab, ld, ldd, kind):
    x, target = logits(rows, vocab, ld, kind, rows + vocab)
    gen = torch.Generator().manual_seed(rows)
    a, b = (torch.randn(rows, generator=gen).to(DEV) for _ in range(2))
    check_gradient(x, target, vocab, ldd, a, b)
    check_gradient(x, target, vocab, ldd, a, None)
    check_gradient(x, target, vocab, ldd, None, b)
    if ld == ldd:
        check_gradient(x, target, vocab, ldd, a, b, in_place=True)


@pytest.mark.parametrize("vocab,ld", [(1, 8), (3, 8), (3, 800), (257, 320), (259, 4096), (100, 8200), (2049, 9000)])
@pytest.mark.parametrize("rows", [1, 3, 6, 9])
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
def test_gradient_of_rows_with_padding(vocab, ld, rows, kind):
    """Columns after the last whole 16 bytes: fewer and many more than a warp's lanes, in rows of one to nine."""
    x, target = logits(rows, vocab, ld, kind, rows + ld)
    target[-1] = vocab - 1
    gen = torch.Generator().manual_seed(ld)
    a, b = (torch.randn(rows, generator=gen).to(DEV) for _ in range(2))
    check_gradient(x, target, vocab, ld, a, b)
    check_gradient(x, target, vocab, ld, a, b, in_place=True)


@pytest.mark.parametrize("kind,vocab", [(torch.float32, 8193), (torch.float32, 12291), (torch.bfloat16, 16385),
                                        (torch.float32, 4097), (torch.bfloat16, 8195)])
def test_gradient_in_place_where_a_part_ends_with_the_whole_pieces(kind, vocab):
    """The columns after the last whole 16 bytes are read and written by one CTA alone."""
    ld = -(-vocab // 8) * 8 + 8
    x, target = logits(40, vocab, ld, kind, vocab)
    target[:20] = vocab - 1
    gen = torch.Generator().manual_seed(vocab)
    a, b = (torch.randn(40, generator=gen).to(DEV) for _ in range(2))
    for _ in range(5):
        check_gradient(x, target, vocab, ld, a, b, in_place=True)


@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
def test_gradient_of_masked_rows(kind):
    gen = torch.Generator().manual_seed(2)
    x = torch.randn(4, 300, generator=gen)
    x[0, torch.rand(300, generator=gen) < 0.9] = -float("inf")
    x[0, 7] = 0.5
    x[1] = -float("inf")
    x[1, 9] = 1.0
    x[3, ::2] = torch.finfo(kind).min / 2
    x = x.to(kind).to(DEV)
    target = torch.tensor([7, 9, 3, 4], dtype=torch.int32, device=DEV)
    check_gradient(x, target, 300, 300, torch.ones(4, device=DEV), torch.ones(4, device=DEV))
    x[2] = -float("inf")  # nothing allowed: no gradient
    g = run_gradient(x, target, 300, 300, torch.ones(4, device=DEV), torch.ones(4, device=DEV))
    assert (g[2] == 0).all()


def test_gradient_against_differences_of_the_forward_kernel():
    """Central differences of the forward kernel's own outputs; step 2^-6, so the difference quotient is
    off by h^2 / 6 times a third derivative (below 2) and by 2^-18 / h from the rounding of the values."""
    vocab, rows, h = 257, 6, 2.0 ** -6
    x, target = logits(rows, vocab, vocab, torch.float32, 3, scale=1.0)
    target = target.clamp(min=0)
    gen = torch.Generator().manual_seed(7)
    a, b = (torch.randn(rows, generator=gen).to(DEV) for _ in range(2))
    g = run_gradient(x, target, vocab, vocab, a, b).cpu().numpy()
    for j in (0, 5, 100, 256, *target[:3].tolist()):
        up, down = x.clone(), x.clone()
        up[:, j] += h
        down[:, j] -= h
        f = [run_scores(y, target, vocab, 0) for y in (up, down)]
        step = (up[:, j] - down[:, j]).double().cpu().numpy()
        value = [a.cpu().numpy().astype(np.float64) * y[0] + b.cpu().numpy().astype(np.float64) * y[1] for y in f]
        quotient = (value[0] - value[1]) / step
        size = 1 + np.abs(a.cpu().numpy()) + np.abs(b.cpu().numpy())
        assert (np.abs(quotient - g[:, j]) <= size * (h * h / 3 + 2.0 ** -17 / h)).all()


# ---------------------------------------------------------------- workspaces and parts of rows
def test_one_workspace_serves_any_sizes_in_turn():
    """Zeroed once: what a call leaves in it is no count of a later call with more or fewer rows, columns or
    alternatives.  Each call equals one with a workspace of its own."""
    from sejong_b200 import _lib
    sizes = [(8, 50001, 20), (128, 50001, 20), (8, 50001, 20), (1, 9001, 3), (400, 9001, 32), (64, 131072, 0), (413, 5001, 7),
             (2, 50001, 1)]
    size = max(_lib.load().sj_token_scores_workspace(*s) for s in sizes)
    work = torch.zeros(size, dtype=torch.uint8, device=DEV)
    for i, (rows, vocab, top) in enumerate(sizes):
        x, target = logits(rows, vocab, vocab, torch.float32, 100 + i)
        stats = [torch.full((rows,), 9.0, device=DEV) for _ in range(3)]
        ids, best = torch.full((rows, top), -9, dtype=torch.int32, device=DEV), torch.full((rows, top), 9.0, device=DEV)
        _lib.call("sj_token_scores", ptr(x), F32, vocab, ptr(target), rows, vocab, top, *[ptr(t) for t in stats], ptr(ids),
                  ptr(best), ptr(work), size, stream())
        for got, own in zip((*stats, ids, best), run_scores(x, target, vocab, top)):
            np.testing.assert_array_equal(got.cpu().numpy(), own, err_msg=str((rows, vocab, top)))


@pytest.mark.parametrize("rows,vocab", [(64, 5000), (32, 50001), (3, 8193), (100, 16400)])
@pytest.mark.parametrize("top", [0, 20])
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
def test_no_part_of_a_row_is_empty(rows, vocab, top, kind):
    """The part that is done last writes the row with the target's logit that it has read; one of no columns would have
    read none.  It would also leave its maximum, -inf, in the workspace."""
    from sejong_b200 import _lib
    x, target = logits(rows, vocab, vocab, kind, rows)
    target = target.clamp(min=0)
    check_scores(x, target, vocab, top)
    out = [torch.empty(rows, device=DEV) for _ in range(3)]
    ids, best = torch.empty(rows, top, dtype=torch.int32, device=DEV), torch.empty(rows, top, device=DEV)
    size = _lib.load().sj_token_scores_workspace(rows, vocab, top)
    work = torch.zeros(size, dtype=torch.uint8, device=DEV)
    _lib.call("sj_token_scores", ptr(x), F32 if kind == torch.float32 else BF16, vocab, ptr(target), rows, vocab, top,
              *[ptr(t) for t in out], ptr(ids), ptr(best), ptr(work), size, stream())
    assert not torch.isneginf(work.view(torch.float32)).any()
