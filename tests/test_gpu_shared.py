"""Several continuations of one prompt on a paged cache, against the 64-bit restatements (oracle/beams.py,
oracle/paged.py): the books of forked, copied and compacted pages (exact), a beam search's selection (indices exact), and
the attention of rows that share keys.

Bounds, from the arithmetic.  Selection: a sum of f32 exponentials of 2 ulp each (2^-22 of a term, and as much for the
rounding of its exponent, at most 2^6) is off by less than 2^-16 of itself in the worst case, its logarithm by 2^-16, and
the total is rounded once (2^-24 of it).  Attention: as in test_gpu_paged.py.
"""
import ctypes

import numpy as np
import pytest
import torch

from oracle import beams as oracle
from oracle import paged as opaged

pytestmark = pytest.mark.gpu

DEV = "cuda"
BAD_INDEX = 110


@pytest.fixture(scope="module", autouse=True)
def lib():
    from sejong_b200 import _lib
    lib = _lib.load()
    _lib.call("sj_device_init", 0)
    return lib


@pytest.fixture(autouse=True)
def share_always(monkeypatch):
    """Small cases go the way of large ones."""
    monkeypatch.setenv("SJ_ATTN_SHARE", "always")


@pytest.fixture(autouse=True)
def no_device_error(lib):
    yield
    assert device_error() == 0


def device_error():
    from sejong_b200._lib import call
    code = ctypes.c_int(0)
    call("sj_device_error", ctypes.byref(code), 1, stream())
    return code.value


def call(name, *args):
    from sejong_b200 import _lib
    return _lib.call(name, *args)


def ptr(t):
    return 0 if t is None else t.data_ptr()


def stream():
    return torch.cuda.current_stream().cuda_stream


def ints(a):
    return torch.as_tensor(np.ascontiguousarray(a), dtype=torch.int32, device=DEV)


# ---------------------------------------------------------------- selection
def select(x, score, keep, dtype=torch.float32, pad=0, workspace=None):
    from sejong_b200 import _lib
    requests, beams, vocab = x.shape
    wide = torch.full((requests * beams, vocab + pad), 1e30, dtype=dtype)  # what lies past the row is not looked at
    wide[:, :vocab] = x.reshape(-1, vocab).to(dtype)
    logits = wide.to(DEV)
    out = [torch.full((requests, keep), 9, dtype=d, device=DEV) for d in (torch.int32, torch.int32, torch.float32)]
    size = _lib.load().sj_beam_select_workspace(requests, beams, vocab, keep)
    work = torch.zeros(max(size, 1), dtype=torch.uint8, device=DEV) if workspace is None else workspace
    s = score.float().to(DEV).contiguous()
    code = {torch.float32: 0, torch.bfloat16: 4}[dtype]
    for _ in range(2):  # the workspace is ready for the next call
        call("sj_beam_select", ptr(logits), code, vocab + pad, ptr(s), requests, beams, vocab, keep, *(ptr(t) for t in out),
             ptr(work), work.numel(), stream())
        got = [t.cpu().numpy() for t in out]
    return wide[:, :vocab].double().view(requests, beams, vocab).numpy(), score.float().double().numpy(), got


def check_select(x, score, keep, dtype=torch.float32, pad=0):
    exact, s, (parent, token, total) = select(x, score, keep, dtype, pad)
    with np.errstate(invalid="ignore", divide="ignore"):
        want = oracle.select(exact, s, keep)
    assert np.array_equal(parent, want[0]) and np.array_equal(token, want[1])
    there = want[2] > -np.inf
    assert np.array_equal(np.isneginf(total), ~there)
    total, exact = total[there].astype(np.float64), want[2][there]
    assert (np.abs(total - exact) <= 2.0 ** -16 + 2.0 ** -23 * np.abs(exact)).all()


def logits(requests, beams, vocab, seed, spread=3.0):
    gen = torch.Generator().manual_seed(seed)
    score = -torch.rand(requests, beams, generator=gen) * 6 - 20
    return torch.randn(requests, beams, vocab, generator=gen) * spread, score


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("requests,beams,vocab,keep,pad", [
    (1, 1, 1, 1, 0), (1, 1, 2, 2, 5), (3, 4, 257, 8, 7), (2, 1, 257, 40, 0), (1, 32, 257, 64, 3), (2, 40, 100, 64, 0),
    (2, 3, 1024, 33, 0), (5, 2, 1025, 4, 0), (2, 8, 5000, 16, 3), (1, 5, 50001, 10, 6), (1, 1, 131075, 64, 1),
    (40, 8, 2049, 1, 0), (3, 64, 1500, 64, 1), (10, 20, 5000, 40, 0), (2, 64, 9000, 64, 2), (30, 25, 257, 50, 0), (3, 12, 700, 24, 1),
    (2, 2, 1100, 64, 0)])
def test_selection(dtype, requests, beams, vocab, keep, pad):
    check_select(*logits(requests, beams, vocab, requests * beams + vocab), keep, dtype, pad)


@pytest.mark.parametrize("vocab", [257, 4097])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_selection_of_ties(vocab, dtype):
    """Equal logits, equal beams: the lowest index first, more of them than any list holds."""
    x = torch.zeros(2, 3, vocab)
    x[1, :, 7::5] = 1.0
    check_select(x, torch.tensor([[-1.0, -1.0, -1.0], [-3.0, -2.0, -2.0]]), 20, dtype)
    check_select(torch.full((1, 64, vocab), 2.5), torch.zeros(1, 64), 64, dtype)
    x, _ = logits(1, 1, vocab, 6)  # beams that are alike, in rows that begin anywhere
    for pad in (0, 1, 2, 5):
        check_select(x.expand(1, 7, vocab).contiguous(), torch.full((1, 7), -2.0), 25, dtype, pad)
    x = torch.arange(vocab).flip(0).float().expand(1, 2, vocab) / 64  # falling along the row
    check_select(x, torch.tensor([[-1.0, -1.5]]), 30)
    check_select(x.flip(2), torch.tensor([[-1.0, -1.5]]), 30)


@pytest.mark.parametrize("keep", [1, 8, 9, 16, 17])
@pytest.mark.parametrize("vocab", [257, 1000, 3000])
def test_selection_of_few_among_ties(vocab, keep):
    x = torch.zeros(2, 3, vocab)
    x[1, :, 7::5] = 1.0
    check_select(x, torch.tensor([[-1.0, -1.0, -1.0], [-3.0, -2.0, -2.0]]), keep)
    x, _ = logits(1, 1, vocab, 6)
    check_select(x.expand(1, 9, vocab).contiguous(), torch.full((1, 9), -2.0), keep)


@pytest.mark.parametrize("beams,keep", [(1, 16), (15, 16), (16, 16), (17, 16), (1, 17), (8, 24), (8, 32), (32, 8), (33, 8), (1, 64)])
@pytest.mark.parametrize("vocab", [100, 257, 1000])
def test_selection_about_the_ways_to_a_bar(vocab, beams, keep):
    """Both sides of the rule by which a small vocabulary's bar is found."""
    check_select(*logits(3, beams, vocab, beams * vocab + keep), keep)
    check_select(*logits(3, beams, vocab, beams * vocab + keep, spread=0.1), keep, torch.bfloat16)


@pytest.mark.parametrize("vocab", [257, 4097, 40000])
def test_selection_of_forbidden_tokens_and_empty_beams(vocab):
    inf = float("inf")
    x, score = logits(4, 3, vocab, 1)
    x[0, :, 5:] = -inf                       # five tokens of each beam
    x[1] = -inf                              # none
    x[2, :2] = -inf                          # of one beam
    x[2, 2, ::3] = -inf
    score[3, 1:] = -inf                      # a first step
    check_select(x, score, 20)
    x, score = logits(5, 2, vocab, 2)
    x[0, 0, 3] = float("nan")                # such rows have no candidates
    x[1, 1, vocab - 1] = inf
    x[2, 0] = float("nan")
    score[3, 0] = float("nan")
    lowest = torch.finfo(torch.float32).min
    x[4, 0] = lowest                         # a mask that leaves nothing, by the lowest value instead
    x[4, 1, 10:] = lowest
    check_select(x, score, 12)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("at", [1234, 21000, 37999])
def test_selection_keeps_the_nan_of_a_part_without_other_values(dtype, at):
    """A row of 20 parts, of which one has a NaN and forbidden tokens only, and the next one nothing but those."""
    x, _ = logits(1, 2, 40000, 4)
    score = torch.tensor([[-1.0, -9.0]])  # the row with the NaN would bring the best
    first = at // 2000 * 2000
    x[0, 0, first:first + 4000] = -float("inf")
    x[0, 0, at] = float("nan")
    check_select(x, score, 8, dtype)


@pytest.mark.parametrize("vocab", [257, 5000])
def test_selection_without_scores_that_are_no_numbers(vocab):
    """A score of +inf would make every total of its beam equal, and which tokens are kept would not follow from them."""
    x, score = logits(3, 3, vocab, 5)
    score[0, 1] = float("inf")
    score[1, 0] = float("nan")
    score[2] = float("inf")
    check_select(x, score, 12)


def test_selection_of_extreme_logits():
    x, score = logits(2, 2, 3000, 3)
    x[0] *= 1e30
    x[1] = x[1] * 1e-30 - 1e4
    x[1, 0, :5] = 0.0
    x[1, 0, 5:9] = -0.0
    check_select(x, score, 16)


def test_selection_of_the_most_requests():
    check_select(*logits(4096, 2, 1030, 1), 3)
    check_select(*logits(4096, 3, 40, 2), 5, torch.bfloat16)


def test_selection_offsets_past_32_bits():
    """Three rows of more than 2^30 columns, which begin past 2^31 and 2^32 bytes and elements."""
    free, _ = torch.cuda.mem_get_info()
    if free < 16 << 30:
        pytest.skip("needs 16 GB of device memory")
    from sejong_b200 import _lib
    vocab, keep = (1 << 31) - (1 << 17) - 3, 4
    x = torch.full((3, vocab + 3), -200.0, dtype=torch.bfloat16, device=DEV)  # nothing beside the rest: e^-200 is 0 in f32
    want = []
    for r, places in enumerate(((5, vocab - 1, 1 << 30, 77), (vocab - 1, vocab - 2, 0, 1), (1 << 30, vocab // 2, 9, vocab - 9))):
        for i, at in enumerate(places):
            x[r, at] = 4.0 - i
        want.append(list(places))
    score = torch.tensor([-1.0, -2.0, -3.0], device=DEV)
    out = [torch.empty(3, keep, dtype=d, device=DEV) for d in (torch.int32, torch.int32, torch.float32)]
    size = _lib.load().sj_beam_select_workspace(3, 1, vocab, keep)
    work = torch.zeros(size, dtype=torch.uint8, device=DEV)
    call("sj_beam_select", ptr(x), 4, vocab + 3, ptr(score), 3, 1, vocab, keep, *(ptr(t) for t in out), ptr(work), size, stream())
    assert out[1].tolist() == want and (out[0] == 0).all()
    top = torch.arange(4, 0, -1).double()
    exact = score.cpu().double()[:, None] + torch.log_softmax(top, 0)
    assert ((out[2].cpu().double() - exact).abs() <= 2.0 ** -16 + 2.0 ** -23 * exact.abs()).all()


def test_selection_shares_a_workspace_between_sizes():
    from sejong_b200 import _lib
    sizes = [(1, 2, 9000), (60, 4, 1100), (2, 1, 70000), (3, 5, 300)]
    work = torch.zeros(max(_lib.load().sj_beam_select_workspace(*s, 8) for s in sizes), dtype=torch.uint8, device=DEV)
    for requests, beams, vocab in sizes + sizes:
        x, score = logits(requests, beams, vocab, vocab)
        exact, s, got = select(x, score, 8, workspace=work)
        want = oracle.select(exact, s, 8)
        assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


def test_selection_captured_and_on_another_stream():
    from sejong_b200 import _lib
    x, score = logits(3, 4, 6000, 8)
    logit, s = x.reshape(12, -1).to(DEV), score.to(DEV)
    out = [torch.empty(3, 8, dtype=d, device=DEV) for d in (torch.int32, torch.int32, torch.float32)]
    work = torch.zeros(_lib.load().sj_beam_select_workspace(3, 4, 6000, 8), dtype=torch.uint8, device=DEV)

    def run():
        call("sj_beam_select", ptr(logit), 0, 6000, ptr(s), 3, 4, 6000, 8, *(ptr(t) for t in out), ptr(work), work.numel(),
             stream())

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for k in range(3):
        logit.copy_(torch.roll(x, k, 0).reshape(12, -1))
        s.copy_(torch.roll(score, k, 0))
        graph.replay()
        want = oracle.select(torch.roll(x, k, 0).double().numpy(), torch.roll(score, k, 0).double().numpy(), 8)
        assert np.array_equal(out[0].cpu().numpy(), want[0]) and np.array_equal(out[1].cpu().numpy(), want[1])


# ---------------------------------------------------------------- forks
class Books:
    """A paged cache's books on the GPU in two sets, and the same in Python."""

    def __init__(self, cached, table, shares, free, page):
        self.page, self.batch, self.pages = page, len(cached), len(shares)
        self.cached, self.table, self.shares, self.free = list(cached), np.array(table), list(shares), list(free)
        stack = self.free + [-1] * (self.pages - len(self.free))
        self.now = [ints(self.cached), ints(self.table), ints(self.shares), ints(stack), ints([len(self.free)])]
        self.copies, self.summary = ints(np.full((self.batch, 3), 9)), ints([9] * 4)

    def fork(self, parent):
        new = [torch.full_like(t, -1) for t in self.now]
        par = ints(parent)
        for _ in range(2):  # the state is only read
            call("sj_paged_fork", ptr(par), self.batch, self.page, ptr(self.now[0]), ptr(self.now[1]),
                 self.now[1].shape[1], ptr(self.now[2]), ptr(self.now[3]), ptr(self.now[4]), self.pages, *(ptr(t) for t in new),
                 ptr(self.copies), ptr(self.summary), stream())
        return new

    def expect(self, new, want):
        lengths, table, shares, free, copies, back, status = want
        assert new[0].tolist() == list(lengths)
        assert np.array_equal(new[1].cpu().numpy(), table)
        assert new[2].tolist() == list(shares)
        assert new[4].tolist() == [len(free)] and new[3].tolist()[:len(free)] == list(free)
        assert self.summary.tolist() == [len(copies), back, status, len(free)]
        rows = self.copies.tolist()
        assert [tuple(r) for r in rows[:len(copies)]] == [tuple(int(v) for v in c) for c in copies]
        assert all(r == [-1, -1, 0] for r in rows[len(copies):])


def start(lengths, page, spare, width_pad=1, seed=0):
    """Requests that hold pages of their own."""
    rng = np.random.default_rng(seed)
    held = [opaged.ceil_div(n, page) for n in lengths]
    pages = sum(held) + spare
    ids = rng.permutation(pages)
    table = np.full((len(lengths), max(max(held) + width_pad, 1)), -1)
    at = 0
    for b, n in enumerate(held):
        table[b, :n] = ids[at:at + n]
        at += n
    return Books(lengths, table, [0] * pages, [int(i) for i in ids[at:]], page)


@pytest.mark.parametrize("lengths,page,seed", [
    ([0], 16, 0), ([1], 1, 1), ([5, 0, 16], 16, 2), ([40, 33, 64, 1, 0, 17, 100, 3], 16, 3), ([1000, 37], 3, 4),
    (list(range(0, 700, 7)), 8, 5), ([9000] * 3, 4, 6)])
def test_forks_one_after_the_other(lengths, page, seed):
    rng = np.random.default_rng(seed)
    books = start(lengths, page, 6 * len(lengths) + 3, seed=seed)
    batch = len(lengths)
    for step in range(6):
        parent = rng.integers(-1 if step % 2 else 0, batch, batch)
        if step == 3:
            parent = np.full(batch, parent[0])
        want = oracle.fork([int(p) for p in parent], page, books.cached, books.table, books.shares, books.free)
        new = books.fork(parent)
        books.expect(new, want)
        if want[-1]:
            break
        table = np.where(np.arange(want[1].shape[1])[None, :] < opaged.ceil_div(np.array(want[0]), page)[:, None], want[1], -1)
        books = Books([int(n) for n in want[0]], table, [int(s) for s in want[2]], [int(p) for p in want[3]], page)


def test_fork_of_the_largest_batch():
    """4096 requests, 512 of which are taken over eight times; every page is counted."""
    books = start([21 + b % 40 for b in range(4096)], 16, 5000)
    parent = (np.arange(4096) // 8) * 8 % 4096
    books.expect(books.fork(parent), oracle.fork(parent.tolist(), 16, books.cached, books.table, books.shares, books.free))


def test_fork_of_the_largest_cache():
    pages = 1 << 18
    table = np.full((2, 70001), -1)
    ids = np.random.default_rng(0).permutation(pages)
    table[0, :70000], table[1, :50000] = ids[:70000], ids[70000:120000]
    books = Books([70000 * 2 - 1, 50000 * 2], table, [0] * pages, ids[120000:].tolist(), 2)
    new = books.fork([1, 1])
    assert books.summary.tolist() == [0, 70000, 0, pages - 50000]
    assert new[3][:pages - 50000].tolist() == ids[120000:].tolist() + sorted(ids[:70000].tolist())
    new = books.fork([0, 0])
    assert books.summary.tolist() == [1, 50000, 0, pages - 70001]
    assert new[2].sum().item() == 69999


def test_fork_and_compaction_of_the_largest_batch_and_cache():
    """4096 requests on 2^18 pages: the most shared memory that either takes."""
    pages, rng = 1 << 18, np.random.default_rng(1)
    lengths = [16 * (1 + b % 60) - 5 * (b % 3) for b in range(4096)]
    ids = rng.permutation(pages)
    table = np.full((4096, 62), -1)
    at = 0
    for b, n in enumerate(lengths):
        held = opaged.ceil_div(n, 16)
        table[b, :held] = ids[at:at + held]
        at += held
    books = Books(lengths, table, [0] * pages, ids[at:].tolist(), 16)
    parent = rng.integers(-1, 4096, 4096)
    want = oracle.fork(parent.tolist(), 16, books.cached, books.table, books.shares, books.free)
    assert want[-1] == 0 and len(want[4]) > 100
    books.expect(books.fork(parent), want)
    table, shares, free, moves = oracle.compact(16, books.cached, books.table, books.shares, books.free, pages)
    new, got = compact(books, len(moves))
    assert [tuple(m) for m in got] == [(a, b, 16) for a, b in moves]
    assert np.array_equal(new[0].cpu().numpy(), table) and new[2].tolist()[:len(free)] == free
    assert books.summary.tolist() == [len(moves), at, 0, len(free)]


@pytest.mark.parametrize("parent,cached,status", [
    ([0, 0, 0], [10, 3, 0], 2), ([3, 0, 1], [10, 3, 0], 4), ([-2, 0, 1], [10, 3, 0], 4), ([0, 1, 2], [10, -1, 0], 4),
    ([0, 1, 2], [10, 300, 0], 3), ([0, 1, 2], [10, 2 ** 31 - 4, 0], 4)])
def test_fork_refuses_as_a_whole(parent, cached, status):
    books = start([10, 3, 0], 4, 1)
    books.now[0].copy_(ints(cached))
    new = books.fork(parent)
    assert books.summary.tolist() == [0, 0, status, 1]
    assert new[0].tolist() == cached and new[2].tolist() == books.shares and new[4].tolist() == [1]
    assert new[3].tolist()[:1] == books.free and new[1][0, :3].tolist() == books.table[0, :3].tolist()
    assert (books.copies == ints([-1, -1, 0])).all()


def test_fork_refuses_a_stack_out_of_bounds():
    books = start([10, 3], 4, 2)
    for count in (-1, books.pages + 1):
        books.now[4].fill_(count)
        books.fork([0, 1])
        assert books.summary.tolist() == [0, 0, 4, count]


@pytest.mark.parametrize("bad", [-1, -7, 10 ** 6])
def test_fork_reports_pages_out_of_range(bad):
    books = start([16, 16], 4, 3)
    books.now[1][0, 1] = bad
    new = books.fork([1, 1])  # request 0's pages come back, but for the one that is none
    assert device_error() == BAD_INDEX
    assert books.summary.tolist() == [0, 3, 0, 6]
    assert new[2].sum().item() == 4


@pytest.mark.parametrize("parent", [[0, 1], [1, 0], [1, 1], [0, 0], [-1, -1]])
@pytest.mark.parametrize("bad", [-1, -7, 10 ** 6, -2 ** 31])
def test_fork_reports_pages_out_of_range_whoever_goes_on(parent, bad):
    """Of requests with one child, with several, and with none."""
    books = start([14, 16], 4, 3)
    books.now[1][0, 1] = bad
    new = books.fork(parent)
    assert device_error() == BAD_INDEX and books.summary[2].item() == 0
    assert all(new[1][b, 1].item() == bad for b, p in enumerate(parent) if p == 0)
    start([14, 16], 4, 3).fork(parent)
    assert device_error() == 0


def test_fork_reports_pages_given_back_too_often():
    books = start([8, 8], 4, 3)
    books.now[1][1, 0] = books.now[1][0, 0].item()  # in two tables, but counted once
    books.fork([-1, -1])
    assert device_error() == BAD_INDEX


# ---------------------------------------------------------------- copies
def caches(layers, pages, hk, page, dim, layout, seed=0):
    gen = torch.Generator().manual_seed(seed)
    shape = (hk, page, dim) if layout == "head" else (page, hk, dim)
    pair = [torch.randn(layers, pages, *shape, generator=gen).bfloat16() for _ in range(2)]
    pair = [t.to(DEV) for t in pair]
    return pair if layout == "head" else [t.transpose(2, 3) for t in pair]


@pytest.mark.parametrize("layout", ["head", "token"])
@pytest.mark.parametrize("layers,hk,page,dim,copies", [(1, 1, 1, 64, [(0, 1, 1)]), (3, 2, 16, 64, [(4, 2, 5), (4, 3, 16)]),
                                                       (1, 8, 64, 128, [(0, 9, 63), (5, 1, 0), (3, 2, 1)]),
                                                       (2, 3, 24, 128, [(9, 0, 24)]), (1, 4, 200, 64, [(1, 0, 199)])])
def test_copies(layout, layers, hk, page, dim, copies):
    k, v = caches(layers, 10, hk, page, dim, layout)
    want = [t.clone() for t in (k, v)]
    for src, dst, rows in copies:
        for t in want:
            t[:, dst, :, :rows] = t[:, src, :, :rows]
    todo = ints(copies + [(-1, -1, 0)] * 3)
    call("sj_paged_copy", ptr(todo), len(copies) + 3, ptr(k), ptr(v), layers, k.stride(0), 10, page, k.stride(1), k.stride(2),
         k.stride(3), hk, dim, stream())
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])


@pytest.mark.parametrize("entry", [(10, 1, 4), (0, 10, 4), (0, -1, 4), (-2, 1, 4), (0, 1, 17), (0, 1, -1)])
def test_copy_reports_what_is_out_of_range(entry):
    k, v = caches(1, 10, 2, 16, 64, "head")
    want = k.clone(), v.clone()
    call("sj_paged_copy", ptr(ints([entry])), 1, ptr(k), ptr(v), 1, k.stride(0), 10, 16, *k.stride()[1:4], 2, 64, stream())
    assert device_error() == BAD_INDEX
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])


# ---------------------------------------------------------------- compaction
def compact(books, most):
    new = [torch.full_like(t, -1) for t in books.now[1:4]]
    moves = ints(np.full((max(most, 1), 3), 9))
    call("sj_paged_compact", ptr(books.now[0]), books.batch, books.page, ptr(books.now[1]), books.now[1].shape[1],
         ptr(books.now[2]), ptr(books.now[3]), ptr(books.now[4]), books.pages, *(ptr(t) for t in new), ptr(moves), most,
         ptr(books.summary), stream())
    return new, moves.tolist()[:most]


@pytest.mark.parametrize("lengths,page,spare", [([0], 16, 1), ([5], 16, 0), ([33, 0, 64, 1, 17], 16, 40),
                                                (list(range(0, 900, 13)), 8, 500), ([20000, 3], 1, 4000), ([7, 9], 4, 200)])
def test_compaction(lengths, page, spare):
    books = start(lengths, page, spare, seed=spare)
    table, shares, free, moves = oracle.compact(page, books.cached, books.table, books.shares, books.free, books.pages)
    most = len(moves) + 5
    new, got = compact(books, most)
    assert [tuple(m) for m in got] == [(a, b, page) for a, b in moves] + [(-1, -1, 0)] * 5
    assert np.array_equal(new[0].cpu().numpy(), table) and new[1].tolist() == list(shares)
    assert new[2].tolist()[:len(free)] == free
    assert books.summary.tolist() == [len(moves), books.pages - len(free), 0, len(free)]


def test_compaction_refuses_as_a_whole():
    books = start([30, 40, 50], 4, 60, seed=3)
    moves = oracle.compact(4, books.cached, books.table, books.shares, books.free, books.pages)[3]
    assert len(moves) > 2
    used = books.pages - len(books.free)
    new, got = compact(books, len(moves) - 1)
    assert books.summary.tolist() == [0, used, 1, len(books.free)] and all(m == [-1, -1, 0] for m in got)
    inside = books.table >= 0
    assert np.array_equal(new[0].cpu().numpy()[inside], books.table[inside]) and new[1].tolist() == books.shares
    assert new[2].tolist()[:len(books.free)] == books.free
    for bad in (books.free[1], -1, books.pages):  # twice, or out of range
        books.now[3][0] = bad
        compact(books, 100)
        assert books.summary[2].item() == 4


def test_compaction_reports_free_and_absent_pages():
    books = start([8, 8], 4, 3)
    books.now[1][0, 0] = books.free[0]
    books.now[1][0, 1] = -3
    new, _ = compact(books, 10)
    assert device_error() == BAD_INDEX
    assert new[0][0, :2].tolist() == [books.free[0], -3]


# ---------------------------------------------------------------- attention
def shared_case(groups, hq, hk, dim, page, window=0, layout="head", loose=0, seed=0, scale=1.0, pad=0, poison=True):
    """groups: (tokens in common, [tokens of each row, from 0, or None for a row without a request]).  `loose` rows before the
    first group have requests of their own.  Compares with the restatement, and with rows that do not share."""
    from sejong_b200 import _lib
    gen, rng = torch.Generator().manual_seed(seed), np.random.default_rng(seed)
    request, length, group, table, content = [], [], [], [], []
    for i in range(loose):
        n = 1 + 37 * i
        request.append(len(table))
        length.append(n)
        table.append(["own"] * opaged.ceil_div(n, page))
        content.append(n)
    for common, rows in groups:
        group.append((len(request), len(table), common))
        base = len(table)
        whole = common // page  # pages in common
        table.append(["own"] * opaged.ceil_div(max(common, 1), page))
        content.append(common)
        for n in rows:
            length.append(n or 0)
            if n is None:
                request.append(-1)
                continue
            request.append(len(table))
            table.append([(base, j) if j < whole else "own" for j in range(opaged.ceil_div(n, page))])
            content.append(n)
    ids = iter(rng.permutation(sum(row.count("own") for row in table) + 2))
    pages = sum(row.count("own") for row in table) + 2
    width = max(len(row) for row in table) + 1
    tables = np.full((len(table), width), -1, dtype=np.int64)
    shape = (pages, hk, page, dim) if layout == "head" else (pages, page, hk, dim)
    exact = [torch.full(shape, float("nan") if poison else 0.0) for _ in range(2)]
    exact = [t if layout == "head" else t.transpose(1, 2) for t in exact]
    for b, (row, n) in enumerate(zip(table, content)):
        for j, what in enumerate(row):
            if what == "own":
                tables[b, j] = next(ids)
                rows_here = min(page, max(n - j * page, 0))
                for t in exact:
                    t[tables[b, j], :, :rows_here] = torch.randn(hk, rows_here, dim, generator=gen)
            else:
                tables[b, j] = tables[what[0], what[1]]
    # a group's tokens past its whole pages are the rows' own copies of the same values
    for (first, base, common), (_, rows) in zip(group, groups):
        tail = common % page
        if tail:
            for r in range(first, first + len(rows)):
                b = request[r]
                if b >= 0 and len(table[b]) > common // page:
                    n = min(tail, length[r] - common // page * page)
                    for t in exact:
                        t[tables[b, common // page], :, :n] = t[tables[base, common // page], :, :n]
    exact = [t.bfloat16() for t in exact]
    k, v = (t.to(DEV) for t in exact)
    if layout == "token":
        k, v = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v))
    rows = len(request)
    q = (torch.randn(rows, hq * dim + pad, generator=gen) * scale).bfloat16()
    qd, tab, req, pos, grp = q.to(DEV), ints(tables), ints(request), ints(np.array(length) - 1), ints(group or [(0, 0, 0)])
    o = torch.full((rows, hq * dim + pad), 5.0, dtype=torch.bfloat16, device=DEV)
    lse = torch.full((rows, hq), 7.0, device=DEV)
    size = _lib.load().sj_attn_paged_shared_workspace(rows, len(group), hq, hk, dim)
    work = torch.zeros(size, dtype=torch.uint8, device=DEV)
    results = []
    for _ in range(2):
        call("sj_attn_paged_shared", ptr(qd), qd.shape[1], ptr(k), ptr(v), pages, page, *k.stride()[:3], ptr(tab), width,
             len(table), ptr(req), ptr(pos), rows, ptr(grp), len(group), hq, hk, dim, window, ptr(o), o.shape[1], ptr(lse),
             ptr(work), size, stream())
        assert device_error() == 0
        results.append((o.clone(), lse.clone()))
    assert torch.equal(results[0][0], results[1][0]) and torch.equal(results[0][1], results[1][1])
    assert (o[:, hq * dim:] == 5.0).all()
    kd, vd = (torch.nan_to_num(t.double(), nan=0.0) for t in exact)
    want, want_lse, mean, reach = opaged.attention(q[:, :hq * dim].double().view(rows, hq, dim), kd, vd,
                                                   torch.as_tensor(tables), request, np.array(length) - 1, page, window)
    got = o.cpu()[:, :hq * dim].double().view(rows, hq, dim)
    off = (got - want).abs() - (2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -9) * mean)
    assert (off <= 0).all(), float(off.max())
    got_lse = lse.cpu().double()
    empty = torch.isneginf(want_lse)
    assert torch.equal(torch.isneginf(got_lse), empty)
    bound = (dim + 8) * 2.0 ** -24 * reach + 2.0 ** -20
    assert ((got_lse - want_lse).abs()[~empty] <= bound[~empty]).all()
    assert (got[empty] == 0).all()


@pytest.mark.parametrize("hq,hk", [(4, 4), (4, 2), (12, 4), (9, 1), (16, 1), (40, 2), (100, 1), (130, 1)])
@pytest.mark.parametrize("dim", [64, 128])
def test_shared_head_layouts(hq, hk, dim):
    shared_case([(160, [161, 200, 160, 170]), (300, [301] * 3)], hq, hk, dim, 16, seed=hq + dim)


@pytest.mark.parametrize("layout", ["head", "token"])
@pytest.mark.parametrize("page", [1, 3, 16, 24, 128, 200])
def test_shared_pages_and_orders(page, layout):
    shared_case([(130, [140, 131, 150]), (257, [258, 300]), (0, [5, 9])], 4, 2, 64, page, layout=layout, seed=page)


@pytest.mark.parametrize("dim", [64, 128])
def test_shared_lengths(dim):
    """From nothing in common, or one token, over whole tiles and one more, to rows with no token of their own."""
    for n in (0, 1, 63, 64, 65, 127, 128, 129, 255, 256, 257, 384, 385, 640, 1500):
        shared_case([(n, [n + 1, n + 40, max(n, 1)])], 4, 2, dim, 16, seed=n)


@pytest.mark.parametrize("dim", [64, 128])
def test_shared_rows_that_see_less(dim):
    """Rows that end inside what is shared, rows without a request, rows of length zero."""
    shared_case([(400, [401, None, 390, 0, 450]), (300, [None, None]), (200, [0]), (333, [5, 340, 334])], 4, 2, dim, 16, seed=1)


@pytest.mark.parametrize("window", [1, 5, 64, 200, 380, 5000])
def test_shared_windows(window):
    shared_case([(400, [401, 420, 500, 410]), (100, [120, 101])], 4, 2, 64, 16, window=window, loose=2, seed=window)


def test_shared_large_groups():
    """More rows than a tile of queries, than two; groups of one row; rows of no group."""
    shared_case([(520, [521 + i % 7 for i in range(90)])], 4, 1, 64, 16, seed=2)
    shared_case([(700, [701 + i % 30 for i in range(140)]), (64, [80])], 6, 2, 128, 64, loose=3, seed=3)
    shared_case([(300 + i, [301 + i]) for i in range(40)], 2, 1, 64, 16, seed=4)


@pytest.mark.parametrize("rows", [1030, 2048, 2100])
def test_shared_many_rows(rows):
    shared_case([(64, [65 + i % 3 for i in range(rows - 30)]), (32, [40] * 30)], 2, 1, 64, 16, seed=rows)


def test_shared_sharp_scores():
    shared_case([(500, [520, 501, 530])], 4, 2, 64, 16, scale=30.0, seed=5)
    shared_case([(3000, [3001] * 40)], 4, 2, 128, 16, scale=30.0, seed=6)


def test_shared_long():
    shared_case([(40000, [40001, 40100])], 2, 1, 64, 64, seed=7)
    shared_case([(9000, [9001 + 50 * i for i in range(20)]), (20000, [20010] * 3)], 8, 2, 128, 32, seed=8, pad=8)


def test_shared_without_groups():
    shared_case([], 4, 2, 64, 16, loose=4)


@pytest.mark.parametrize("dim", [64, 128])
def test_shared_where_it_does_not_pay(monkeypatch, dim):
    """The same by the rule: too little to share for the host to see, and for the GPU (wide block tables)."""
    monkeypatch.delenv("SJ_ATTN_SHARE")
    shared_case([(160, [161, 200, 0, 170]), (300, [301, None])], 4, 2, dim, 16, loose=1, seed=dim)
    shared_case([(160, [161, 200, 0, 170] * 20), (300, [300, None]), (200, [30000])], 8, 8, dim, 128, loose=1, seed=dim)


def test_shared_where_it_pays(monkeypatch):
    monkeypatch.delenv("SJ_ATTN_SHARE")
    shared_case([(2500, [2501 + i % 40 for i in range(80)])], 8, 4, 128, 64, seed=9)


@pytest.mark.parametrize("group", [[(0, 9, 32)], [(0, -1, 32)], [(-1, 0, 32)], [(5, 0, 32)], [(0, 0, -3)], [(0, 0, 1000)],
                                   [(2, 0, 32), (1, 0, 32)], [(1, 0, 32), (1, 0, 32)]])
def test_shared_reports_groups_out_of_range(group):
    """Such a group has nothing in common: its rows read their own tables."""
    from sejong_b200 import _lib
    gen = torch.Generator().manual_seed(1)
    k, v = (torch.randn(8, 2, 16, 64, generator=gen).bfloat16().to(DEV) for _ in range(2))
    q = torch.randn(4, 256, generator=gen).bfloat16().to(DEV)
    table = ints([[0, 1, 2], [0, 1, 3], [0, 1, 4], [0, 1, 5]])
    pos, grp = ints([40, 39, 41, 33]), ints(group)
    out = []
    for name, extra, size in (("sj_attn_paged", [], _lib.load().sj_attn_paged_workspace(4, 4, 2, 64)),
                              ("sj_attn_paged_shared", [ptr(grp), len(group)],
                               _lib.load().sj_attn_paged_shared_workspace(4, len(group), 4, 2, 64))):
        o, lse = torch.empty_like(q), torch.empty(4, 4, device=DEV)
        work = torch.zeros(size, dtype=torch.uint8, device=DEV)
        call(name, ptr(q), 256, ptr(k), ptr(v), 8, 16, *k.stride()[:3], ptr(table), 3, 4, 0, ptr(pos), 4, *extra, 4, 2, 64, 0,
             ptr(o), 256, ptr(lse), ptr(work), size, stream())
        out.append((o, lse))
    assert device_error() == BAD_INDEX
    assert (out[0][0].float() - out[1][0].float()).abs().max() < 0.02
    assert (out[0][1] - out[1][1]).abs().max() < 1e-4


@pytest.mark.parametrize("group", [[(0, 0, 32), (4, 0, 0), (2, 0, 32)], [(0, 0, 32), (4, 0, 0), (2, 0, 32), (4, 0, 0)],
                                   [(4, 0, 0), (0, 0, 32)]])
def test_shared_reports_groups_after_the_end(group):
    test_shared_reports_groups_out_of_range(group)


BAD_GROUPS = [[(0, 9, 32)], [(0, -1, 32)], [(-1, 0, 32)], [(5, 0, 32)], [(0, 0, -3)], [(0, 0, 1000)], [(2, 0, 32), (1, 0, 32)],
              [(1, 0, 32), (1, 0, 32)], [(0, 0, 32), (4, 0, 0), (2, 0, 32)]]


@pytest.mark.parametrize("group", BAD_GROUPS)
def test_shared_reports_groups_where_rows_are_left_apart(monkeypatch, group):
    """The same where the rule sees too little to share."""
    monkeypatch.delenv("SJ_ATTN_SHARE")
    test_shared_reports_groups_out_of_range(group)
    gen = torch.Generator().manual_seed(1)  # and nothing to report of groups that are in order
    k, v = (torch.randn(8, 2, 16, 64, generator=gen).bfloat16().to(DEV) for _ in range(2))
    q = torch.randn(4, 256, generator=gen).bfloat16().to(DEV)
    shared_call(q, k, v, ints([[0, 1, 2]] * 4), ints([0, 1, 2, 3]), ints([40, 39, 41, 33]), ints([(0, 1, 32), (2, 3, 48), (4, 0, 0)]),
                4, 2, 64)
    assert device_error() == 0


@pytest.mark.parametrize("rows,hq", [(1030, 2), (4, 130)])
def test_shared_reports_groups_of_shapes_that_never_share(rows, hq):
    """More than 1024 groups, or more than 128 query heads a KV head."""
    gen = torch.Generator().manual_seed(2)
    k, v = (torch.randn(8, 1, 16, 64, generator=gen).bfloat16().to(DEV) for _ in range(2))
    q = torch.randn(rows, hq * 64, generator=gen).bfloat16().to(DEV)
    table, req, pos = ints([[0, 1, 2]] * rows), ints(np.arange(rows)), ints([40] * rows)
    group = np.array([(r, r, 32) for r in range(rows)])
    want = shared_call(q, k, v, table, req, pos, ints(group), hq, 1, 64)
    assert device_error() == 0
    group[rows - 2, 2] = 49
    got = shared_call(q, k, v, table, req, pos, ints(group), hq, 1, 64)
    assert device_error() == BAD_INDEX
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def shared_call(q, k, v, table, request, position, group, hq, hk, dim, window=0, work=None, out=None):
    from sejong_b200 import _lib
    rows, groups = q.shape[0], group.shape[0]
    o, lse = out or (torch.empty_like(q), torch.empty(rows, hq, device=DEV))
    size = _lib.load().sj_attn_paged_shared_workspace(rows, groups, hq, hk, dim)
    work = torch.zeros(size, dtype=torch.uint8, device=DEV) if work is None else work
    call("sj_attn_paged_shared", ptr(q), q.shape[1], ptr(k), ptr(v), k.shape[0], k.shape[2], *k.stride()[:3], ptr(table),
         table.shape[1], table.shape[0], ptr(request), ptr(position), rows, ptr(group), groups, hq, hk, dim, window, ptr(o),
         o.shape[1], ptr(lse), ptr(work), work.numel(), stream())
    return o, lse


def test_shared_passes_nan_and_infinity_to_rows_that_see_them():
    """In common: to every row.  Before a window, past a row's end, in the tile's rest: to no row that does not see it."""
    gen = torch.Generator().manual_seed(3)
    for where, seen in ((5, [True, True, True]), (130, [True, False, True]), (199, [True, False, False]), (203, [False] * 3)):
        k, v = (torch.randn(20, 1, 16, 64, generator=gen).bfloat16().to(DEV) for _ in range(2))
        table = ints(np.arange(20)[None].repeat(3, 0))
        q = torch.randn(3, 128, generator=gen).bfloat16().to(DEV)
        v[where // 16, 0, where % 16, 7] = float("nan")
        k[where // 16, 0, where % 16] = float("inf")
        o, lse = shared_call(q, k, v, table, ints([0, 1, 2]), ints([201, 100, 180]), ints([(0, 0, 200)]), 2, 1, 64)
        assert torch.isfinite(lse).all(1).tolist() == [not s for s in seen]
        assert torch.isfinite(o.float()).all(1).tolist() == [not s for s in seen]
    k, v = (torch.randn(20, 1, 16, 64, generator=gen).bfloat16().to(DEV) for _ in range(2))
    v[2, 0, 3] = float("nan")  # token 35
    o, _ = shared_call(q, k, v, table, ints([0, 1, 2]), ints([201, 150, 134]), ints([(0, 0, 120)]), 2, 1, 64, window=100)
    assert torch.isfinite(o.float()).all(1).tolist() == [True, True, False]


def test_shared_on_another_stream_and_captured():
    """The same call on a side stream, and replayed from a CUDA graph over other lengths and groups."""
    from sejong_b200 import _lib
    gen = torch.Generator().manual_seed(8)
    k, v = (torch.randn(300, 2, 16, 64, generator=gen).bfloat16().to(DEV) for _ in range(2))
    q = torch.randn(6, 4 * 64, generator=gen).bfloat16().to(DEV)
    ids = np.random.default_rng(0).permutation(300)
    table = np.concatenate((np.tile(ids[:50], (6, 1)), ids[50:290].reshape(6, 40)), axis=1)
    table, req = ints(table), ints(np.arange(6))
    pos, group = ints([900, 850, 801, 1000, 830, 1400]), ints([(0, 0, 800), (4, 4, 790), (6, 0, 0)])
    work = torch.zeros(_lib.load().sj_attn_paged_shared_workspace(6, 3, 4, 2, 64), dtype=torch.uint8, device=DEV)
    out = torch.empty_like(q), torch.empty(6, 4, device=DEV)

    def run():
        return shared_call(q, k, v, table, req, pos, group, 4, 2, 64, work=work, out=out)

    first = [t.clone() for t in run()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = [t.clone() for t in run()]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for new, groups in (([900, 850, 801, 1000, 830, 1400], [(0, 0, 800), (4, 4, 790), (6, 0, 0)]),
                        ([700, -1, 10, 799, 800, 801], [(0, 0, 640), (3, 3, 700), (6, 0, 0)]),
                        ([-1] * 6, [(0, 0, 0), (6, 0, 0), (6, 0, 0)]),
                        ([1439] * 6, [(0, 5, 800), (6, 0, 0), (6, 0, 0)])):
        pos.copy_(ints(new))
        group.copy_(ints(groups))
        graph.replay()
        got = [t.clone() for t in out]
        want = [t.clone() for t in run()]
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        plain = shared_call(q, k, v, table, req, pos, ints([(0, 0, 0)]), 4, 2, 64)
        assert (got[0].float() - plain[0].float()).abs().max() < 0.02


def random_shared(seed, rows, keys, hq, hk, dim):
    """Rows that share all but their last page, and the call's arguments."""
    gen, page = torch.Generator().manual_seed(seed), 16
    common = keys // page
    k, v = (torch.randn(common + rows, hk, page, dim, generator=gen).bfloat16().to(DEV) for _ in range(2))
    table = np.concatenate((np.tile(np.arange(common), (rows, 1)), common + np.arange(rows)[:, None]), axis=1)
    q = torch.randn(rows, hq * dim, generator=gen).bfloat16().to(DEV)
    return q, k, v, ints(table), ints(np.arange(rows)), ints([common * page + i % page for i in range(rows)]), \
        ints([(0, 0, common * page)]), hq, hk, dim


def test_shared_calls_at_once_and_graphs_that_share_a_workspace():
    """Two streams with workspaces of their own; then two captured calls of different sizes on one workspace, in turn."""
    from sejong_b200 import _lib
    calls = [random_shared(1, 40, 4000, 12, 4, 64), random_shared(2, 150, 2500, 8, 2, 128)]
    want = [[t.clone() for t in shared_call(*c)] for c in calls]
    size = [_lib.load().sj_attn_paged_shared_workspace(c[0].shape[0], 1, c[7], c[8], c[9]) for c in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    works = [torch.zeros(n, dtype=torch.uint8, device=DEV) for n in size]
    outs = [[(torch.empty_like(c[0]), torch.empty(c[0].shape[0], c[7], device=DEV)) for _ in range(8)] for c in calls]
    torch.cuda.synchronize()
    for i in range(8):
        for c, s, w, out in zip(calls, streams, works, outs):
            with torch.cuda.stream(s):
                shared_call(*c, work=w, out=out[i])
    torch.cuda.synchronize()
    for out, w in zip(outs, want):
        assert all(torch.equal(a, b) for pair in out for a, b in zip(pair, w))
    work = torch.zeros(max(size), dtype=torch.uint8, device=DEV)
    graphs = []
    for c, out in zip(calls, outs):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            shared_call(*c, work=work, out=out[0])
    for i in (0, 1, 1, 0, 1, 0, 0):
        for t in outs[i][0]:
            t.fill_(3.0)
        graphs[i].replay()
        assert all(torch.equal(a, b) for a, b in zip(outs[i][0], want[i]))


def test_selections_at_once_and_graphs_that_share_a_workspace():
    from sejong_b200 import _lib
    sizes = [(3, 4, 9000, 8), (1, 2, 70000, 20)]
    inputs, want, outs, need = [], [], [], []
    for requests, beams, vocab, keep in sizes:
        x, score = logits(requests, beams, vocab, vocab)
        inputs.append((x.reshape(-1, vocab).to(DEV), score.to(DEV)))
        want.append(oracle.select(x.double().numpy(), score.double().numpy(), keep))
        outs.append([[torch.full((requests, keep), 9, dtype=d, device=DEV) for d in (torch.int32, torch.int32, torch.float32)]
                     for _ in range(8)])
        need.append(_lib.load().sj_beam_select_workspace(requests, beams, vocab, keep))

    def run(i, out, work):
        requests, beams, vocab, keep = sizes[i]
        call("sj_beam_select", ptr(inputs[i][0]), 0, vocab, ptr(inputs[i][1]), requests, beams, vocab, keep, *(ptr(t) for t in out),
             ptr(work), work.numel(), stream())

    def right(i, out):
        return np.array_equal(out[0].cpu().numpy(), want[i][0]) and np.array_equal(out[1].cpu().numpy(), want[i][1])

    streams, works = [torch.cuda.Stream() for _ in sizes], [torch.zeros(n, dtype=torch.uint8, device=DEV) for n in need]
    torch.cuda.synchronize()
    for k in range(8):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                run(i, outs[i][k], works[i])
    torch.cuda.synchronize()
    assert all(right(i, out) for i in (0, 1) for out in outs[i])
    work = torch.zeros(max(need), dtype=torch.uint8, device=DEV)
    graphs = []
    for i in (0, 1):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            run(i, outs[i][0], work)
    for i in (0, 1, 1, 0, 1, 0, 0):
        for t in outs[i][0]:
            t.fill_(7)
        graphs[i].replay()
        assert right(i, outs[i][0])


def test_shared_and_copied_offsets_past_32_bits():
    """Cache buffers of more than 2^32 elements: the last pages are read, by boxes and by pieces, and copied."""
    free, _ = torch.cuda.mem_get_info()
    if free < 24 << 30:
        pytest.skip("needs 24 GB of device memory")
    gen = torch.Generator().manual_seed(12)
    page, hk, dim = 64, 8, 128
    pages = (1 << 32) // (page * hk * dim) + 6
    k = torch.empty(pages, hk, page, dim, dtype=torch.bfloat16, device=DEV)
    v = torch.empty_like(k)
    small = [torch.randn(4, hk, page, dim, generator=gen).bfloat16() for _ in range(2)]
    for cache, x in ((k, small[0]), (v, small[1])):
        cache[-4:] = x.to(DEV)
    q = torch.randn(2, hk * dim, generator=gen).bfloat16()
    table = ints([[pages - 4, pages - 3, pages - 2, pages - 1]] * 2)
    o, lse = shared_call(q.to(DEV), k, v, table, ints([0, 1]), ints([210, 215]), ints([(0, 0, 200)]), hk, hk, dim)
    want, _, mean, _ = opaged.attention(q.double().view(2, hk, dim), small[0].double(), small[1].double(),
                                        torch.tensor([[0, 1, 2, 3]] * 2), [0, 1], [210, 215], page)
    assert ((o.cpu().double().view(2, hk, dim) - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -9) * mean).all()
    call("sj_paged_copy", ptr(ints([(pages - 4, pages - 5, 64)])), 1, ptr(k), ptr(v), 1, 0, pages, page, *k.stride()[:3], hk,
         dim, stream())
    assert torch.equal(k[-5], k[-4]) and torch.equal(v[-5], v[-4])


# ---------------------------------------------------------------- together
def test_a_beam_search_on_the_books():
    """Steps of plan, commit, select, fork and copy, as a server runs them, against sequences kept in Python: after every step
    each request's pages hold exactly its own tokens."""
    page, beams, requests, vocab, pages, width = 4, 3, 2, 50, 80, 12
    batch = beams * requests
    rng = np.random.default_rng(0)
    state = [torch.zeros(batch, dtype=torch.int32, device=DEV), ints(np.full((batch, width), -1)),
             torch.zeros(pages, dtype=torch.int32, device=DEV), ints(np.arange(pages)), ints([pages])]
    spare = [t.clone() for t in state]
    k, v = (torch.zeros(1, pages, 1, page, 64, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    lengths, summary = ints([0] * batch), ints([0] * 4)
    copies, info = ints(np.zeros((batch, 3))), ints([0] * 4)
    texts = [[int(t) for t in rng.integers(0, vocab, 5 + b // beams)] for b in range(batch)]
    written = [0] * batch
    for step in range(9):
        cached, table, shares, free, count = state
        added = [len(t) - n for t, n in zip(texts, written)]
        if step == 0:
            added = [n if b % beams == 0 else 0 for b, n in enumerate(added)]
        rows = sum(added)
        request, position, slot = (ints([-1] * rows) for _ in range(3))
        call("sj_paged_plan", ptr(cached), ptr(ints(added)), batch, page, ptr(free), ptr(count), ptr(table), width, ptr(lengths),
             ptr(request), ptr(position), ptr(slot), rows, ptr(summary), stream())
        assert summary[2].item() == 0
        for r, p, s in zip(request.tolist(), position.tolist(), slot.tolist()):
            for cache in (k, v):
                cache[0, s // page, 0, s % page] = float(texts[r][p])
        call("sj_paged_commit", ptr(cached), ptr(lengths), 0, batch, page, ptr(table), width, ptr(free), ptr(count), pages,
             ptr(summary), stream())
        written = [w + a for w, a in zip(written, added)]
        x = torch.from_numpy(rng.standard_normal((requests, beams, vocab))) * 2
        score = torch.full((requests, beams), -1.0)
        if step == 0:
            score[:, 1:] = float("-inf")
        parent, token, _ = select(x, score, beams)[2]
        parent = (parent + np.arange(requests)[:, None] * beams).reshape(-1)
        texts = [texts[p] + [int(t)] for p, t in zip(parent, token.reshape(-1))]
        written = [written[p] for p in parent]
        par = ints(parent)
        call("sj_paged_fork", ptr(par), batch, page, ptr(cached), ptr(table), width, ptr(shares), ptr(free), ptr(count), pages,
             *(ptr(t) for t in spare), ptr(copies), ptr(info), stream())
        assert info[2].item() == 0
        call("sj_paged_copy", ptr(copies), batch, ptr(k), ptr(v), 1, k.stride(0), pages, page, *k.stride()[1:4], 1, 64, stream())
        state, spare = spare, state
        held = state[1].tolist()
        assert state[0].tolist() == written
        for b in range(batch):
            for p in range(written[b]):
                assert k[0, held[b][p // page], 0, p % page, 0].item() == texts[b][p]
        used = {i for b in range(batch) for i in held[b][:opaged.ceil_div(written[b], page)]}
        assert state[4].item() == pages - len(used) and not used & set(state[3].tolist()[:state[4].item()])
