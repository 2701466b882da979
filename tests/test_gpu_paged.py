"""Batched decoding on a paged cache against the 64-bit restatement (oracle/paged.py): the step's maps
(exact), scaled rotary tables, the rotary append and the attention over pages.

Bounds, from the arithmetic.  A bf16 has 8 significant bits, so a rounding to it is at most 2^-8 of the
value.  Append: two f32 products, a sum and one bf16 rounding.  Attention: products of bf16 are exact in f32
and a score sums `dim` of them, so it is off by at most (dim + 8) 2^-24 sum |q_i k_i| / sqrt(dim) (the eight covers the scaling and the shift by
the maximum); the probabilities are rounded to bf16 for the product with V (2^-8 of each weight, and
another 2^-9 for the f32 exponentials, sums and the scores' error at the sizes here) and the result
once more.
"""
import ctypes

import numpy as np
import pytest
import torch

from oracle import paged as oracle

pytestmark = pytest.mark.gpu

DEV = "cuda"


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


def call(name, *args):
    from sejong_b200 import _lib
    return _lib.call(name, *args)


def ptr(t):
    return 0 if t is None else t.data_ptr()


def stream():
    return torch.cuda.current_stream().cuda_stream


def ints(a):
    return torch.as_tensor(np.ascontiguousarray(a), dtype=torch.int32, device=DEV)


# ---------------------------------------------------------------- plan and commit
class Planner:
    def __init__(self, cached, added, page, pages, width, rows, seed=0):
        rng = np.random.default_rng(seed)
        self.page, self.rows, self.batch, self.pages = page, rows, len(cached), pages
        held = [max(0, oracle.ceil_div(int(c), page)) for c in cached]
        ids = rng.permutation(pages)
        self.table0 = np.full((self.batch, width), -1, dtype=np.int64)
        at = 0
        for b, n in enumerate(held):
            self.table0[b, :min(n, width)] = ids[at:at + n][:width]
            at += n
        self.free0 = ids[at:]
        self.cached0, self.added0 = np.asarray(cached), np.asarray(added)
        self.cached, self.added, self.table = ints(cached), ints(added), ints(self.table0)
        stack = np.full(pages, -7)
        stack[:len(self.free0)] = self.free0
        self.free, self.count = ints(stack), ints([len(self.free0)])
        self.lengths, self.summary = ints(np.zeros(self.batch)), ints(np.zeros(4))
        self.maps = [ints(np.full(max(rows, 1), 77)) for _ in range(3)]

    def plan(self):
        call("sj_paged_plan", ptr(self.cached), ptr(self.added), self.batch, self.page, ptr(self.free), ptr(self.count),
             ptr(self.table), self.table.shape[1], ptr(self.lengths), *[ptr(m) for m in self.maps], self.rows,
             ptr(self.summary), stream())

    def commit(self, release=None):
        call("sj_paged_commit", ptr(self.cached), ptr(self.lengths), ptr(release), self.batch, self.page,
             ptr(self.table), self.table.shape[1], ptr(self.free), ptr(self.count), self.pages, ptr(self.summary),
             stream())

    def check(self):
        want = oracle.plan(self.cached0, self.added0, self.page, self.free0, self.table0, self.rows)
        got = [self.table, self.lengths, *[m[:self.rows] for m in self.maps], self.summary]
        for name, g, w in zip(("table", "lengths", "request", "position", "slot", "summary"), got, want):
            np.testing.assert_array_equal(g.cpu().numpy(), w, err_msg=name)
        return want


@pytest.mark.parametrize("batch,page,high,rows", [(1, 16, 40, 1), (3, 1, 9, 8), (65, 7, 300, 200), (256, 16, 900, 777),
                                                  (1024, 64, 500, 4000), (1025, 16, 200, 1500), (4096, 32, 100, 9000)])
def test_plan_matches_the_restatement_and_repeats(batch, page, high, rows):
    rng = np.random.default_rng(batch + page)
    cached = rng.integers(0, high, batch)
    added = rng.integers(0, 3, batch)
    if rows > batch:
        added[rng.integers(0, batch)] += min(high, (rows - int(added.sum())) // 2) if rows > added.sum() else 0
    while added.sum() > rows:
        added[np.argmax(added)] -= 1
    need = sum(oracle.ceil_div(int(c + n), page) for c, n in zip(cached, added))
    p = Planner(cached, added, page, need + 5, oracle.ceil_div(2 * high, page) + 1, rows, seed=batch)
    p.plan()
    p.check()
    p.plan()  # nothing of the first call is counted twice
    p.check()


def test_plan_adds_nothing_for_a_batch_at_rest():
    p = Planner([5, 0, 16], [0, 0, 0], 8, 10, 4, 4)
    p.plan()
    want = p.check()
    assert list(want[5][:3]) == [0, 0, 0]


@pytest.mark.parametrize("cached,added,rows,width,spare,status", [
    ([5, 5], [3, 4], 6, 4, 9, 1),            # more rows than the maps hold
    ([16, 16], [1, 1], 4, 9, 1, 2),          # one free page for two requests
    ([16, 3], [17, 1], 30, 2, 9, 3),         # a table of two pages of 16
    ([16, -1], [1, 1], 4, 9, 9, 4),          # a negative length
    ([16, 1], [1, -2], 4, 9, 9, 4),          # a negative count
    ([16, 2 ** 31 - 2], [1, 5], 9, 9, 9, 4)  # a length past 32 bits
])
def test_plan_refuses_as_a_whole(cached, added, rows, width, spare, status):
    held = sum(oracle.ceil_div(max(c, 0), 16) for c in cached if c < 10 ** 6)
    small = [c if c < 10 ** 6 else 0 for c in cached]
    p = Planner(small, added, 16, held + spare, width, rows)
    p.cached = ints(np.array(cached))
    p.plan()
    np.testing.assert_array_equal(p.table.cpu().numpy(), p.table0)
    np.testing.assert_array_equal(p.lengths.cpu().numpy(), cached)
    for m in p.maps:
        assert (m[:rows].cpu().numpy() == -1).all()
    assert p.summary.tolist() == [0, 0, status, len(p.free0)]


def test_plan_of_the_largest_counts():
    """4096 requests that each ask for as many rows as a plan can have: refused, although the sum fills 31 bits."""
    most = (1 << 19) - 1
    p = Planner(np.zeros(4096), np.full(4096, most), 1, 4, 2, most)
    p.plan()
    assert p.summary.tolist() == [0, 0, 1, 4]
    assert (p.maps[0] == -1).all() and (p.lengths == 0).all()


def test_commit_takes_and_returns_pages():
    """Steps with growing and finishing requests: no page is ever held twice or lost."""
    rng = np.random.default_rng(4)
    page, pages, batch = 4, 60, 6
    p = Planner(np.zeros(batch), np.zeros(batch), page, pages, 20, 64)
    lengths = np.zeros(batch, dtype=int)
    for step in range(30):
        added = rng.integers(0, 6, batch)
        gone = rng.random(batch) < 0.25
        p.added = ints(added)
        p.plan()
        assert p.summary[2].item() == 0
        lengths = lengths + added
        np.testing.assert_array_equal(p.lengths.cpu().numpy(), lengths)
        p.commit(ints(gone) if step % 3 else None)
        if step % 3:
            lengths = np.where(gone, 0, lengths)
        p.commit(ints(np.zeros(batch)))  # a second commit changes nothing
        np.testing.assert_array_equal(p.cached.cpu().numpy(), lengths)
        table = p.table.cpu().numpy()
        held = [i for b in range(batch) for i in table[b, :oracle.ceil_div(int(lengths[b]), page)]]
        free = p.free.cpu().numpy()[:p.count.item()]
        assert sorted(list(held) + list(free)) == list(range(pages))


# ---------------------------------------------------------------- rotary tables
@pytest.mark.parametrize("rope_dim,offset", [(64, 0), (2, 3), (48, 100000)])
@pytest.mark.parametrize("kind,code,factor", [("plain", 0, 1.0), ("linear", 1, 4.0), ("base", 2, 8.0),
                                              ("ramp", 3, 16.0)])
def test_scaled_rotary_table(rope_dim, offset, kind, code, factor):
    t = 513
    table = torch.empty(t, rope_dim // 2, 2, device=DEV)
    call("sj_rope_table_scaled", ptr(table), t, rope_dim, offset, 10000.0, code, factor, 2048, 32.0, 1.0, stream())
    want = oracle.rope_table(t, rope_dim, 10000.0, offset=offset, scaling=kind, factor=factor, original=2048)
    # f64 angles up to 1e5 (relative 1e-15) and one rounding to f32 of values up to the amplitude (< 1.4)
    np.testing.assert_allclose(table.cpu().numpy(), want, rtol=0, atol=2 ** -23)


# ---------------------------------------------------------------- append
def pages_of(pages, hk, page, dim, layout, gen, fill=None):
    """K and V [pages, hk, page, dim] views of one of three storages."""
    shape = {"head": (pages, hk, page, dim), "token": (pages, page, hk, dim), "both": (pages, 2, page, hk, dim)}[layout]
    make = (lambda: torch.full(shape, fill, dtype=torch.bfloat16)) if fill is not None else \
        (lambda: torch.randn(shape, generator=gen).bfloat16())
    if layout == "both":  # K and V of a page side by side in one buffer
        kv = make().to(DEV)
        return kv[:, 0].transpose(1, 2), kv[:, 1].transpose(1, 2)
    k, v = make().to(DEV), make().to(DEV)
    return (k, v) if layout == "head" else (k.transpose(1, 2), v.transpose(1, 2))


def strides(k):
    return k.stride(0), k.stride(1), k.stride(2)


@pytest.mark.parametrize("rows,hq,hk,dim,rot,half,page,layout,pad", [
    (1, 4, 2, 64, 64, 0, 16, "head", 0), (37, 12, 4, 64, 64, 1, 7, "token", 8), (130, 3, 1, 128, 48, 1, 16, "both", 16),
    (65, 5, 5, 128, 16, 0, 3, "head", 0), (9, 0, 2, 64, 32, 0, 1, "token", 0), (33, 8, 2, 64, 0, 1, 32, "head", 24),
    (3000, 16, 4, 64, 64, 0, 64, "head", 0)])
def test_append_matches_the_restatement(rows, hq, hk, dim, rot, half, page, layout, pad):
    gen = torch.Generator().manual_seed(rows + dim + rot)
    rng = np.random.default_rng(rows)
    pages, context = oracle.ceil_div(rows, page) + 2, 1000
    slot = rng.permutation(pages * page)[:rows]
    slot[rng.random(rows) < 0.2] = -1
    position = np.where(slot >= 0, rng.integers(0, context, rows), -1)
    qkv = torch.randn(rows, (hq + 2 * hk) * dim + pad, generator=gen).bfloat16().to(DEV)
    table = torch.as_tensor(oracle.rope_table(context, max(rot, 2), 10000.0)).float().to(DEV)
    k, v = pages_of(pages, hk, page, dim, layout, gen)
    k0, v0 = k.cpu().clone(), v.cpu().clone()
    q = torch.full((rows, hq * dim + pad), 3.0, dtype=torch.bfloat16, device=DEV)
    slots, positions = ints(slot), ints(position)
    call("sj_paged_append", ptr(qkv), qkv.shape[1], ptr(positions), ptr(slots), rows, hq, hk, dim, ptr(table), context,
         rot, half, ptr(q), q.shape[1], ptr(k), ptr(v), pages, page, *strides(k), stream())
    x = qkv.cpu()[:, :(hq + 2 * hk) * dim].double().view(rows, hq + 2 * hk, dim)
    y = x.clone()
    if rot:
        y[:, :hq + hk] = oracle.rotate(x[:, :hq + hk], table.cpu().double(), torch.as_tensor(np.maximum(position, 0)), rot,
                                       bool(half))
    live = torch.as_tensor(slot >= 0)
    want_k, want_v = k0.double(), v0.double()
    at = torch.as_tensor(slot)[live]
    want_k[at // page, :, at % page] = y[live][:, hq:hq + hk]
    want_v[at // page, :, at % page] = x[live][:, hq + hk:]
    # two products and a sum of values below 8, in f32, then one bf16 rounding
    close = lambda got, want: (got.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -20  # noqa: E731
    if hq:
        want_q = torch.where(live[:, None, None], y[:, :hq], 0.0).reshape(rows, hq * dim)
        assert close(q.cpu()[:, :hq * dim], want_q).all()
    assert (q[:, hq * dim:] == 3.0).all()
    assert close(k.cpu(), want_k).all()
    assert torch.equal(v.cpu().double(), want_v)  # values are copied; slots of no row keep their contents


def test_append_rotates_queries_in_place():
    gen = torch.Generator().manual_seed(1)
    rows, hq, hk, dim = 50, 4, 2, 64
    qkv = torch.randn(rows, (hq + 2 * hk) * dim, generator=gen).bfloat16().to(DEV)
    table = torch.as_tensor(oracle.rope_table(64, 64, 10000.0)).float().to(DEV)
    k, v = pages_of(8, hk, 16, dim, "head", gen)
    slot, position = ints(np.arange(rows)), ints(np.arange(rows))
    q = torch.empty(rows, hq * dim, dtype=torch.bfloat16, device=DEV)
    again = qkv.clone()
    for src, dst in ((qkv, q), (again, again)):
        call("sj_paged_append", ptr(src), src.shape[1], ptr(position), ptr(slot), rows, hq, hk, dim, ptr(table), 64, 64, 0,
             ptr(dst), dst.shape[1], ptr(k), ptr(v), 8, 16, *strides(k), stream())
    assert torch.equal(again[:, :hq * dim], q)
    assert torch.equal(again[:, hq * dim:], qkv[:, hq * dim:])


@pytest.mark.parametrize("slot,position", [(128, 3), (5, 64), (5, -1)])
def test_append_skips_and_reports_what_is_out_of_range(slot, position):
    gen = torch.Generator().manual_seed(2)
    qkv = torch.randn(2, 6 * 64, generator=gen).bfloat16().to(DEV)
    table = torch.zeros(64, 32, 2, device=DEV)
    k, v = pages_of(8, 1, 16, 64, "head", gen)
    k0, v0 = k.clone(), v.clone()
    q = torch.ones(2, 4 * 64, dtype=torch.bfloat16, device=DEV)
    s, p = ints([slot, -1]), ints([position, -1])
    call("sj_paged_append", ptr(qkv), 6 * 64, ptr(p), ptr(s), 2, 4, 1, 64, ptr(table), 64, 64, 0, ptr(q), 256, ptr(k),
         ptr(v), 8, 16, *strides(k), stream())
    assert device_error() == 110
    assert (q == 0).all() and torch.equal(k, k0) and torch.equal(v, v0)


# ---------------------------------------------------------------- attention
def attention_case(lengths, hq, hk, dim, page, window, layout="head", request=None, seed=0, ldq_pad=0, scale=1.0,
                   requests=None, poison=True):
    """Runs sj_attn_paged and compares.  Slots that no length covers hold NaN."""
    from sejong_b200 import _lib
    gen = torch.Generator().manual_seed(seed)
    rng = np.random.default_rng(seed)
    rows = len(lengths)
    request = np.arange(rows) if request is None else np.asarray(request)
    requests = requests or max(int(request.max()) + 1, 1)
    whole = np.zeros(requests, dtype=int)  # the longest view of each request
    for b, n in zip(request, lengths):
        if b >= 0:
            whole[b] = max(whole[b], n)
    held = [oracle.ceil_div(int(n), page) for n in whole]
    pages, width = sum(held) + 2, max(max(held), 1) + 1
    ids = rng.permutation(pages)
    table = np.full((requests, width), -1, dtype=np.int64)
    k, v = pages_of(pages, hk, page, dim, layout, gen, fill=float("nan") if poison else 0.0)
    kd, vd = torch.zeros(pages, hk, page, dim, dtype=torch.float64), torch.zeros(pages, hk, page, dim, dtype=torch.float64)
    at = 0
    for b in range(requests):
        n = int(whole[b])
        table[b, :held[b]] = ids[at:at + held[b]]
        at += held[b]
        j = torch.arange(n)
        own = torch.as_tensor(table[b])[j // page]
        for cache, exact in ((k, kd), (v, vd)):
            x = torch.randn(n, hk, dim, generator=gen).bfloat16()
            exact[own, :, j % page] = x.double()
            cache[own.to(DEV), :, (j % page).to(DEV)] = x.to(DEV)
    q = (torch.randn(rows, hq * dim + ldq_pad, generator=gen) * scale).bfloat16()
    qd = q.to(DEV)
    o = torch.full((rows, hq * dim + ldq_pad), 5.0, dtype=torch.bfloat16, device=DEV)
    lse = torch.full((rows, hq), 7.0, device=DEV)
    size = _lib.load().sj_attn_paged_workspace(rows, hq, hk, dim)
    work = torch.zeros(size, dtype=torch.uint8, device=DEV)
    tables, req = ints(table), ints(request)
    position = ints(np.asarray(lengths) - 1)
    results = []
    for _ in range(2):  # the workspace is ready for the next call
        call("sj_attn_paged", ptr(qd), qd.shape[1], ptr(k), ptr(v), pages, page, *strides(k), ptr(tables), width, requests,
             ptr(req), ptr(position), rows, hq, hk, dim, window, ptr(o), o.shape[1], ptr(lse), ptr(work), size, stream())
        results.append((o.clone(), lse.clone()))
    assert torch.equal(results[0][0], results[1][0]) and torch.equal(results[0][1], results[1][1])
    assert (o[:, hq * dim:] == 5.0).all()
    exact_q = q[:, :hq * dim].double().view(rows, hq, dim)
    want, want_lse, mean, reach = oracle.attention(exact_q, kd, vd, torch.as_tensor(table), request,
                                                   np.asarray(lengths) - 1, page, window)
    got = o.cpu()[:, :hq * dim].double().view(rows, hq, dim)
    off = (got - want).abs() - (2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -9) * mean)
    assert (off <= 0).all(), float(off.max())
    got_lse = lse.cpu().double()
    empty = torch.isneginf(want_lse)
    assert torch.equal(torch.isneginf(got_lse), empty)
    bound = (dim + 8) * 2.0 ** -24 * reach + 2.0 ** -20
    assert ((got_lse - want_lse).abs()[~empty] <= bound[~empty]).all()
    assert (got[empty] == 0).all()


@pytest.mark.parametrize("hq,hk", [(4, 4), (4, 2), (12, 4), (8, 1), (9, 1), (16, 1), (20, 1), (40, 2)])
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_head_layouts(hq, hk, dim):
    attention_case([1, 2, 31, 32, 33, 0, 200], hq, hk, dim, 16, 0, seed=hq + dim)


@pytest.mark.parametrize("page", [1, 3, 8, 16, 24, 64, 128])
@pytest.mark.parametrize("layout", ["head", "token", "both"])
def test_attention_pages_and_orders(page, layout):
    attention_case([130, 1, 257, 64, 500], 6, 2, 64, page, 0, layout=layout, seed=page, ldq_pad=8)


@pytest.mark.parametrize("window", [1, 2, 17, 128, 1000])
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_windows(window, dim):
    attention_case([1, 16, 129, 700, 0, 128, 127], 4, 2, dim, 16, window, seed=window)


@pytest.mark.parametrize("lengths", [[1], [5000], [0], [20011, 3], [4096] * 9, [1] * 300, [63, 64, 65] * 50])
def test_attention_lengths_and_batches(lengths):
    attention_case(lengths, 6, 2, 64, 16, 0, seed=len(lengths))


def test_attention_one_long_row_of_wide_heads():
    attention_case([30000], 4, 1, 128, 64, 0, seed=5)


def test_attention_rows_of_shared_and_absent_requests():
    """Several rows of one request see their own prefixes; padded rows see nothing."""
    attention_case([10, 11, 12, 0, 700, 40, 0], 4, 2, 64, 16, 0, request=[2, 2, 2, -1, 0, 1, 3], requests=5, seed=9)


def test_attention_sharp_scores():
    """Scores of some hundreds: the running maximum moves far, and weights underflow."""
    attention_case([900, 33, 4000], 4, 2, 64, 16, 0, scale=60.0, seed=11)


def test_attention_shares_pages_between_requests():
    """Two requests with the same first pages (a common prompt) give what copies would."""
    from sejong_b200 import _lib
    gen = torch.Generator().manual_seed(3)
    k, v = pages_of(6, 2, 16, 64, "head", gen)
    q = torch.randn(1, 4 * 64, generator=gen).bfloat16().repeat(2, 1).to(DEV)
    table, position = ints([[0, 1, 2], [0, 1, 3]]), ints([31, 31])
    o, lse = torch.empty_like(q), torch.empty(2, 4, device=DEV)
    size = _lib.load().sj_attn_paged_workspace(2, 4, 2, 64)
    work = torch.zeros(size, dtype=torch.uint8, device=DEV)
    call("sj_attn_paged", ptr(q), 256, ptr(k), ptr(v), 6, 16, *strides(k), ptr(table), 3, 2, 0, ptr(position), 2, 4, 2, 64,
         0, ptr(o), 256, ptr(lse), ptr(work), size, stream())
    assert torch.equal(o[0], o[1]) and torch.equal(lse[0], lse[1])


@pytest.mark.parametrize("request_id,position,page_id", [(3, 4, 0), (-2, 4, 0), (0, 32, 0), (0, -2, 0), (0, 2 ** 31 - 1, 0),
                                                         (0, 4, 6), (0, 4, -1)])
def test_attention_reports_what_is_out_of_range(request_id, position, page_id):
    from sejong_b200 import _lib
    gen = torch.Generator().manual_seed(4)
    k, v = pages_of(6, 2, 16, 64, "head", gen)
    q = torch.randn(2, 4 * 64, generator=gen).bfloat16().to(DEV)
    table, req, pos = ints([[page_id, 5], [1, 2], [3, 4]]), ints([request_id, 1]), ints([position, 20])
    o, lse = torch.ones_like(q), torch.zeros(2, 4, device=DEV)
    size = _lib.load().sj_attn_paged_workspace(2, 4, 2, 64)
    work = torch.zeros(size, dtype=torch.uint8, device=DEV)
    call("sj_attn_paged", ptr(q), 256, ptr(k), ptr(v), 6, 16, *strides(k), ptr(table), 2, 3, ptr(req), ptr(pos), 2, 4, 2,
         64, 0, ptr(o), 256, ptr(lse), ptr(work), size, stream())
    assert device_error() == 110
    assert (o[0] == 0).all() and torch.isneginf(lse[0]).all()
    assert torch.isfinite(lse[1]).all() and (o[1] != 0).any()


def test_attention_passes_nan_and_infinity_of_seen_keys():
    """A NaN in a seen key or value reaches the rows and heads that see it and no others."""
    from sejong_b200 import _lib
    gen = torch.Generator().manual_seed(6)
    k, v = pages_of(4, 2, 16, 64, "head", gen)
    k[0, 0, 3, 5] = float("nan")
    v[1, 1, 2, 7] = float("nan")
    q = torch.randn(2, 4 * 64, generator=gen).bfloat16().to(DEV)
    table, pos = ints([[0], [1]]), ints([10, 10])
    o, lse = torch.empty_like(q), torch.empty(2, 4, device=DEV)
    size = _lib.load().sj_attn_paged_workspace(2, 4, 2, 64)
    work = torch.zeros(size, dtype=torch.uint8, device=DEV)
    call("sj_attn_paged", ptr(q), 256, ptr(k), ptr(v), 4, 16, *strides(k), ptr(table), 1, 2, 0, ptr(pos), 2, 4, 2, 64, 0,
         ptr(o), 256, ptr(lse), ptr(work), size, stream())
    bad = torch.isnan(o.view(2, 4, 64))
    assert bad[0, :2].all() and not bad[0, 2:].any()
    assert not bad[1, :2].any() and bad[1, 2:, 7].all() and bad[1].sum() == 2
    assert torch.isnan(lse[0, :2]).all() and torch.isfinite(lse[0, 2:]).all() and torch.isfinite(lse[1]).all()


def test_attention_on_another_stream_and_captured():
    """The same call on a side stream, and replayed from a CUDA graph over changing lengths."""
    from sejong_b200 import _lib
    gen = torch.Generator().manual_seed(8)
    k, v = pages_of(300, 2, 16, 64, "head", gen)
    q = torch.randn(3, 4 * 64, generator=gen).bfloat16().to(DEV)
    table = ints(np.random.default_rng(0).permutation(300).reshape(3, 100))
    pos = ints([1500, 3, 200])
    o, lse = torch.empty_like(q), torch.empty(3, 4, device=DEV)
    size = _lib.load().sj_attn_paged_workspace(3, 4, 2, 64)
    work = torch.zeros(size, dtype=torch.uint8, device=DEV)

    def attend():
        call("sj_attn_paged", ptr(q), 256, ptr(k), ptr(v), 300, 16, *strides(k), ptr(table), 100, 3, 0, ptr(pos), 3, 4, 2, 64,
             0, ptr(o), 256, ptr(lse), ptr(work), size, stream())
        return o.clone(), lse.clone()

    first = attend()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = attend()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first[0], second[0]) and torch.equal(first[1], second[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call("sj_attn_paged", ptr(q), 256, ptr(k), ptr(v), 300, 16, *strides(k), ptr(table), 100, 3, 0, ptr(pos), 3, 4, 2, 64,
             0, ptr(o), 256, ptr(lse), ptr(work), size, stream())
    for new in ([1500, 3, 200], [0, 1599, 17], [-1, -1, 900]):
        pos.copy_(ints(new))
        graph.replay()
        got = o.clone(), lse.clone()
        want = attend()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_attention_offsets_past_32_bits():
    """A cache buffer of more than 2^32 bytes (and 2^31 elements): the last pages are read."""
    free, _ = torch.cuda.mem_get_info()
    if free < 24 << 30:
        pytest.skip("needs 24 GB of device memory")
    from sejong_b200 import _lib
    gen = torch.Generator().manual_seed(12)
    page, hk, dim = 64, 8, 128
    pages = (1 << 32) // (page * hk * dim) + 3  # 2^32 elements: 8.6 GB each
    k = torch.empty(pages, hk, page, dim, dtype=torch.bfloat16, device=DEV)
    v = torch.empty_like(k)
    small = [torch.randn(2, hk, page, dim, generator=gen).bfloat16() for _ in range(2)]
    for cache, x in ((k, small[0]), (v, small[1])):
        cache[-2:] = x.to(DEV)
    q = torch.randn(1, hk * dim, generator=gen).bfloat16()
    qd, table, pos = q.to(DEV), ints([[pages - 2, pages - 1]]), ints([99])
    o, lse = torch.empty_like(qd), torch.empty(1, hk, device=DEV)
    size = _lib.load().sj_attn_paged_workspace(1, hk, hk, dim)
    work = torch.zeros(size, dtype=torch.uint8, device=DEV)
    call("sj_attn_paged", ptr(qd), hk * dim, ptr(k), ptr(v), pages, page, *strides(k), ptr(table), 2, 1, 0, ptr(pos), 1, hk,
         hk, dim, 0, ptr(o), hk * dim, ptr(lse), ptr(work), size, stream())
    want, want_lse, mean, reach = oracle.attention(q.double().view(1, hk, dim), small[0].double(), small[1].double(),
                                                   torch.tensor([[0, 1]]), [0], [99], page)
    assert ((o.cpu().double().view(1, hk, dim) - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -9) * mean).all()
    # the append reaches them too
    qkv = torch.randn(1, 3 * hk * dim, generator=gen).bfloat16().to(DEV)
    rope = torch.zeros(128, dim // 2, 2, device=DEV)
    rope[..., 0] = 1.0
    slot = ints([(pages - 1) * page + 36])
    call("sj_paged_append", ptr(qkv), 3 * hk * dim, ptr(ints([100])), ptr(slot), 1, hk, hk, dim, ptr(rope), 128, dim, 0,
         ptr(o), hk * dim, ptr(k), ptr(v), pages, page, *strides(k), stream())
    assert torch.equal(k[-1, :, 36].reshape(-1), qkv[0, hk * dim:2 * hk * dim])
    assert torch.equal(v[-1, :, 36].reshape(-1), qkv[0, 2 * hk * dim:])


@pytest.mark.parametrize("bad", [-1, -7, 60, 1 << 30])
def test_commit_refuses_as_a_whole_what_a_page_id_out_of_range_would_return(bad):
    p = Planner([5, 9, 0], [1, 4, 2], 4, 60, 6, 16)
    p.plan()
    p.check()
    state = (p.cached, p.lengths, p.free, p.count, p.table, p.summary)
    good = p.table[1, 2].item()
    p.table[1, 2] = bad
    before = [t.clone() for t in state]
    gone = ints([1, 1, 0])
    p.commit(gone)
    assert device_error() == 110
    assert all(torch.equal(a, b) for a, b in zip(state, before))
    p.table[1, 2] = good
    p.commit(gone)
    assert p.cached.tolist() == p.lengths.tolist() == [0, 0, 2]
    held = [p.table[2, 0].item()]
    assert sorted(held + p.free[:p.count.item()].tolist()) == list(range(60))


@pytest.mark.parametrize("count,pages", [(None, 50), (2, 60)])
def test_commit_refuses_as_a_whole_a_stack_out_of_bounds(count, pages):
    """More pages than the stack has room for, or fewer on it than the step took."""
    p = Planner([5, 9, 0], [1, 4, 2], 4, 60, 6, 16)
    p.plan()
    if count is not None:
        p.count.fill_(count)
        p.summary[1] = count + 1
    p.pages = pages
    state = (p.cached, p.lengths, p.free, p.count, p.table, p.summary)
    before = [t.clone() for t in state]
    p.commit(ints([1, 1, 0]))
    assert device_error() == 110
    assert all(torch.equal(a, b) for a, b in zip(state, before))


@pytest.mark.parametrize("bad", [-1, -9, 134217727, 1 << 28, 1 << 30, 2 ** 31 - 1])
@pytest.mark.parametrize("where", ["table", "stack"])
def test_plan_reports_page_ids_without_slots(bad, where):
    """Ids below 0, and those whose slots would not fit 31 bits (id * 16 would wrap to another request's slot)."""
    p = Planner([5, 16], [2, 2], 16, 40, 4, 6)
    if where == "table":
        p.table[0, 0] = bad  # the page that request 0's new tokens go on with
    else:
        p.free[p.count.item() - 1] = bad  # the page that request 1 gets
    p.plan()
    assert device_error() == 110
    own = [p.table0[0, 0] * 16 + 5, p.table0[0, 0] * 16 + 6, p.free0[-1] * 16, p.free0[-1] * 16 + 1, -1, -1]
    own = [-1, -1] + own[2:] if where == "table" else own[:2] + [-1] * 4
    assert p.maps[2].tolist() == own
    assert p.summary.tolist() == [4, 1, 0, len(p.free0) - 1]


def test_plan_of_the_largest_page_id():
    p = Planner([5], [2], 16, 40, 4, 2)
    p.table[0, 0] = 134217726
    p.plan()
    assert p.maps[2].tolist() == [134217726 * 16 + 5, 134217726 * 16 + 6]


@pytest.mark.parametrize("slot", [-2, -128, -2 ** 31])
def test_append_reports_slots_below_minus_one(slot):
    test_append_skips_and_reports_what_is_out_of_range(slot, 3)
