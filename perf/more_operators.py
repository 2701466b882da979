"""Cases that measure the operators of several continuations of one prompt on a paged key-value cache:

  select   sj_beam_select        the best continuations of each request over its beams and the vocabulary
  fork     sj_paged_fork         requests take over one another's pages, which they share and count; pages come back
  copy     sj_paged_copy         rows of pages copied to other pages, keys and values of every layer
  compact  sj_paged_compact      the pages in use moved to the front of the cache
  share    sj_attn_paged_shared  attention of rows that share their first pages, whose keys are read once for all

`run` makes either the library's calls (`own`) or the same computation in elementary torch operations.
"""
import math

import numpy as np
import torch

own = False

NO_PAGE = -1


# ---------------------------------------------------------------- cases
def listed():
    return [
        # a step of the byte model's beam search: a small vocabulary, latency counts
        {"name": "select bytes", "op": "select", "requests": 16, "beams": 4, "vocab": 257, "ld": 264, "keep": 8,
         "f32": True, "masked": False, "first": False},
        # a full server with a word vocabulary and 16-bit logits
        {"name": "select words", "op": "select", "requests": 128, "beams": 8, "vocab": 50001, "ld": 50008, "keep": 16,
         "f32": False, "masked": False, "first": False},
        # the reordering after one step of a few short beams
        {"name": "fork beams", "op": "fork", "requests": 8, "beams": 4, "page": 16, "low": 20, "high": 2000,
         "ended": 1},
        # the same on a large server with long texts, where many pages are counted and come back
        {"name": "fork server", "op": "fork", "requests": 128, "beams": 8, "page": 64, "low": 500, "high": 32768,
         "ended": 9},
        # the half-filled last pages of those few beams, every layer of the byte model's global stage
        {"name": "copy beams", "op": "copy", "copies": 13, "padded": 32, "pages": 300, "page": 16, "full": False,
         "hk": 4, "dim": 64, "layers": 6, "layout": "head"},
        # pages moved before a cache is made smaller
        {"name": "copy moves", "op": "copy", "copies": 2003, "padded": 2100, "pages": 5000, "page": 64, "full": True,
         "hk": 8, "dim": 128, "layers": 1, "layout": "token"},
        # a small cache, a third of it in use
        {"name": "compact beams", "op": "compact", "requests": 8, "beams": 4, "page": 16, "low": 20, "high": 2000,
         "spare": 2.0},
        # a large one
        {"name": "compact server", "op": "compact", "requests": 128, "beams": 8, "page": 16, "low": 500,
         "high": 16384, "spare": 1.0},
        # the least a server meets: four beams of one short text
        {"name": "share beams", "op": "share", "kind": "requests", "groups": 1, "per_low": 4, "per_high": 4,
         "low": 240, "high": 240, "own_low": 9, "own_high": 9, "hq": 4, "hk": 2, "dim": 64, "page": 16, "window": 0,
         "layout": "head"},
        # 16 samples of each of 16 prompts on the byte model's global heads
        {"name": "share samples", "op": "share", "kind": "requests", "groups": 16, "per_low": 16, "per_high": 16,
         "low": 2048, "high": 16384, "own_low": 1, "own_high": 500, "hq": 12, "hk": 4, "dim": 64, "page": 16,
         "window": 0, "layout": "head"},
        # a full server whose requests all begin with one long text
        {"name": "share prompt", "op": "share", "kind": "requests", "groups": 1, "per_low": 509, "per_high": 509,
         "low": 32768, "high": 32768, "own_low": 1, "own_high": 400, "hq": 16, "hk": 4, "dim": 128, "page": 64,
         "window": 0, "layout": "head"},
        # a piece of a long prompt: rows of one request, which share all that came before
        {"name": "share piece", "op": "share", "kind": "piece", "groups": 2, "per_low": 250, "per_high": 333,
         "low": 20001, "high": 60003, "own_low": 0, "own_high": 0, "hq": 16, "hk": 2, "dim": 128, "page": 64,
         "window": 0, "layout": "token"},
    ]


def _log(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def _heads(rng):
    while True:
        dim, hk, group = rng.choice((64, 64, 128)), rng.choice((1, 2, 4, 8)), rng.choice((1, 2, 3, 4, 5, 8, 12, 16))
        if hk * group <= 64:
            return dim, hk, hk * group


def draw(rng):
    op = rng.choice(("select", "select", "fork", "copy", "compact", "share", "share", "share"))
    page = rng.choice((8, 16, 16, 24, 32, 64, 128))
    if op == "select":
        vocab = rng.choice((257, _log(rng, 2, 130000)))
        beams = _log(rng, 1, 32)
        requests = _log(rng, 1, max(2, min(256, int(5e7 / vocab / beams))))
        return {"op": op, "requests": requests, "beams": beams, "vocab": vocab,
                "ld": vocab + rng.choice((0, 7, -vocab % 8)), "keep": min(beams * vocab, rng.choice((beams, 2 * beams))),
                "f32": rng.random() < 0.5, "masked": rng.random() < 0.3, "first": rng.random() < 0.15}
    if op in ("fork", "compact"):
        beams = _log(rng, 1, 32)
        requests = _log(rng, 1, 1024 // beams)
        most = min(32768, int(5e5 * page / requests / beams))  # at most half a million entries of block tables
        high = _log(rng, 16, max(17, most))
        case = {"op": op, "requests": requests, "beams": beams, "page": page, "low": _log(rng, 1, high), "high": high}
        if op == "fork":
            case["ended"] = rng.choice((0, rng.randint(0, requests)))
        else:
            case["spare"] = rng.choice((0.02, 0.3, 1.0, 2.0))
        return case
    if op == "copy":
        dim, hk, _ = _heads(rng)
        layers = rng.choice((1, 2, 5, 12))
        full = rng.random() < 0.5
        copies = _log(rng, 1, max(2, min(3000, int(1.2e8 / (page * hk * dim * layers)))))
        return {"op": op, "copies": copies, "padded": copies + rng.choice((0, rng.randint(0, 50))),
                "pages": 2 * copies + rng.randint(1, 100), "page": page, "full": full, "hk": hk, "dim": dim,
                "layers": layers, "layout": rng.choice(("head", "token"))}
    dim, hk, hq = _heads(rng)
    kind = rng.choice(("requests", "requests", "requests", "piece"))
    window = rng.choice((0, 0, 0, 0, _log(rng, 1, 4096)))
    groups = _log(rng, 1, 40)
    per = _log(rng, 1, max(2, 512 // groups))
    rows = groups * per
    high = _log(rng, 16, max(17, min(60000, int(1e11 / (rows * hq * dim)), int(1e9 / (groups * hk * dim * 4)))))
    own = 0 if kind == "piece" else _log(rng, 1, max(2, min(500, int(2e8 / (rows * hk * dim * 4)))))
    return {"op": op, "kind": kind, "groups": groups, "per_low": _log(rng, 1, per), "per_high": per,
            "low": _log(rng, 1, high), "high": high, "own_low": min(1, own), "own_high": own, "hq": hq, "hk": hk,
            "dim": dim, "page": page, "window": window, "layout": rng.choice(("head", "token"))}


def _spread(count, low, high):
    """`count` whole numbers between low and high, even over their logarithm."""
    at = (np.arange(count) + 0.5) / count
    return np.rint(low * (max(high, 1) / max(low, 1)) ** at).astype(np.int64).clip(low, high)


def _ceil(a, b):
    return -(-a // b)


# ---------------------------------------------------------------- inputs
def prepare(case, seed):
    host = np.random.default_rng(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = {"case": case}
    {"select": _prepare_select, "fork": _prepare_fork, "copy": _prepare_copy, "compact": _prepare_compact,
     "share": _prepare_share}[case["op"]](case, state, host, gen)
    return state


def _int(a):
    return torch.as_tensor(np.ascontiguousarray(a), dtype=torch.int32, device="cuda")


def _filled(*shape):
    return torch.full(shape, NO_PAGE, dtype=torch.int32, device="cuda")


def _prepare_select(case, state, host, gen):
    requests, beams, vocab, ld, keep = (case[n] for n in ("requests", "beams", "vocab", "ld", "keep"))
    rows = requests * beams
    x = torch.randn(rows, ld, device="cuda", generator=gen) * 3.0
    if case["masked"]:  # about a third of the tokens are forbidden
        x.masked_fill_(torch.rand(rows, ld, device="cuda", generator=gen) < 0.33, -math.inf)
    score = -torch.rand(requests, beams, device="cuda", generator=gen) * 6.0 - 20.0
    score = score.sort(dim=1, descending=True).values
    if case["first"]:  # a request's first step: its other beams hold nothing yet
        score[:, 1:] = -math.inf
    state.update(logits=x if case["f32"] else x.to(torch.bfloat16), score=score.contiguous(),
                 parent=_filled(requests, keep), token=_filled(requests, keep),
                 best=torch.empty(requests, keep, dtype=torch.float32, device="cuda"))


def _beams(case, host, spare):
    """Block tables of requests of several beams each, as steps of a beam search leave them: a request's first pages are
    shared by all of its beams, the next ones by pairs, the last are a beam's own.  Lengths, tables, further owners of
    each page, and the free pages."""
    requests, beams, page = case["requests"], case["beams"], case["page"]
    length = _spread(requests, case["low"], case["high"])[host.permutation(requests)]
    held, width = _ceil(length, page), int(_ceil(length, page).max()) + 2
    cached = np.repeat(length, beams)
    table = np.full((requests * beams, width), NO_PAGE, dtype=np.int64)
    taken = 0
    for i in range(requests):
        n = int(held[i])
        common, pairs = int(n * 0.7), int(n * 0.85)
        pairs = min(pairs, int(length[i]) // page)
        common = min(common, pairs)
        at = slice(i * beams, (i + 1) * beams)
        table[at, :common] = taken + np.arange(common)
        taken += common
        pair = np.arange(beams) // 2
        table[at, common:pairs] = taken + pair[:, None] * (pairs - common) + np.arange(pairs - common)
        taken += (int(pair[-1]) + 1) * (pairs - common)
        table[at, pairs:n] = taken + np.arange(beams)[:, None] * (n - pairs) + np.arange(n - pairs)
        taken += beams * (n - pairs)
    pages = taken + max(int(taken * spare), requests * beams + 5)
    ids = host.permutation(pages)
    owners = np.zeros(pages, dtype=np.int64)
    np.add.at(owners, ids[table[table >= 0]], 1)
    table = np.where(table >= 0, ids[table], NO_PAGE)
    return cached, table, np.maximum(owners - 1, 0), ids[taken:]


def _paged(state, cached, table, shares, free):
    pages = shares.size
    stack = np.full(pages, NO_PAGE, dtype=np.int64)
    stack[:free.size] = free
    state.update(cached=_int(cached), table=_int(table), shares=_int(shares), free=_int(stack),
                 free_count=_int([free.size]), pages=pages, table_out=_filled(*table.shape), shares_out=_filled(pages),
                 free_out=_filled(pages), summary=_filled(4))


def _prepare_fork(case, state, host, gen):
    requests, beams = case["requests"], case["beams"]
    parent = host.integers(0, beams, (requests, beams)) + np.arange(requests)[:, None] * beams
    parent[host.permutation(requests)[:case["ended"]]] = -1
    _paged(state, *_beams(case, host, 0.1))
    state.update(parent=_int(parent.reshape(-1)), cached_out=_filled(requests * beams), count_out=_filled(1),
                 copies=_filled(requests * beams, 3))


def _prepare_compact(case, state, host, gen):
    _paged(state, *_beams(case, host, case["spare"]))
    state.update(moves=_filled(state["pages"] // 2, 3))


def _cache(case, gen, *lead):
    """K and V pages as [..., page, head, token, dim] views of either storage order; every slot holds something."""
    shape = ((case["hk"], case["page"], case["dim"]) if case["layout"] == "head"
             else (case["page"], case["hk"], case["dim"]))
    k, v = (torch.randn(*lead, *shape, dtype=torch.bfloat16, device="cuda", generator=gen) for _ in range(2))
    return (k, v) if case["layout"] == "head" else (k.transpose(-3, -2), v.transpose(-3, -2))


def _prepare_copy(case, state, host, gen):
    copies, pages, page = case["copies"], case["pages"], case["page"]
    ids = host.permutation(pages)[:2 * copies]
    rows = np.full(copies, page) if case["full"] else host.integers(1, page, copies) if page > 1 else np.ones(copies)
    todo = np.full((case["padded"], 3), NO_PAGE, dtype=np.int64)
    todo[:, 2] = 0
    todo[:copies] = np.stack((ids[:copies], ids[copies:], rows), axis=1)
    k, v = _cache(case, gen, case["layers"], pages)
    state.update(copies=_int(todo), k=k, v=v)


def _prepare_share(case, state, host, gen):
    groups, page, dim, hq = (case[n] for n in ("groups", "page", "dim", "hq"))
    per = _spread(groups, case["per_low"], case["per_high"])[host.permutation(groups)]
    shared = _spread(groups, case["low"], case["high"])[host.permutation(groups)]
    rows = int(per.sum())
    first = np.concatenate(([0], per.cumsum()))
    if case["kind"] == "piece":  # rows at consecutive positions of one request
        source = np.arange(groups)
        request = np.repeat(source, per)
        position = np.repeat(shared, per) + np.arange(rows) - np.repeat(first[:-1], per)
        held = _ceil(shared + per, page)
        width, pages = int(held.max()) + 2, int(held.sum()) + 3
        table = np.full((groups, width), NO_PAGE, dtype=np.int64)
        table[np.arange(width)[None, :] < held[:, None]] = host.permutation(pages)[:int(held.sum())]
    else:  # requests that forked: whole pages in common, then pages of their own
        shared = np.maximum(shared // page, 1) * page
        source, request = first[:-1], np.arange(rows)
        tail = _spread(rows, case["own_low"], case["own_high"])[host.permutation(rows)]
        length = np.repeat(shared, per) + tail
        position = length - 1
        held, common = _ceil(length, page), np.repeat(shared // page, per)
        width, total = int(held.max()) + 2, int((shared // page).sum() + (held - common).sum())
        pages = total + 3
        ids = host.permutation(pages)
        table = np.full((rows, width), NO_PAGE, dtype=np.int64)
        at = np.arange(width)[None, :]
        begin = np.concatenate(([0], (shared // page).cumsum()))
        np.copyto(table, np.repeat(begin[:-1], per)[:, None] + at, where=at < common[:, None])
        mine = (at >= common[:, None]) & (at < held[:, None])
        table[mine] = begin[-1] + np.arange(int(mine.sum()))
        table = np.where(table >= 0, ids[table], NO_PAGE)
    k, v = _cache(case, gen, pages)
    q = torch.randn(rows, hq * dim, dtype=torch.bfloat16, device="cuda", generator=gen)
    state.update(q=q, k=k, v=v, table=_int(table), request=_int(request), position=_int(position),
                 group=_int(np.stack((first[:-1], source, shared), axis=1)), rows=rows,
                 o=torch.empty(rows, hq * dim, dtype=torch.bfloat16, device="cuda"),
                 lse=torch.empty(rows, hq, dtype=torch.float32, device="cuda"),
                 # what the caller knows on the host, for the plain form
                 per=per.tolist(), shared=shared.tolist(), source=source.tolist(),
                 tail=int((position + 1 - np.repeat(shared, per)).max()))


# ---------------------------------------------------------------- one pass
def run(state):
    op = state["case"]["op"]
    if own:
        return {"select": _own_select, "fork": _own_fork, "copy": _own_copy, "compact": _own_compact,
                "share": _own_share}[op](state, state["case"])
    return {"select": _plain_select, "fork": _plain_fork, "copy": _plain_copy, "compact": _plain_compact,
            "share": _plain_share}[op](state, state["case"])


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _own_select(s, c):
    from sejong_b200._lib import SJ_BF16, SJ_F32, call, load
    if "workspace" not in s:  # kept by the program, zero before its first use
        size = load().sj_beam_select_workspace(c["requests"], c["beams"], c["vocab"], c["keep"])
        s["workspace"] = torch.zeros(max(size, 1), dtype=torch.uint8, device="cuda")
    call("sj_beam_select", s["logits"].data_ptr(), SJ_F32 if c["f32"] else SJ_BF16, c["ld"], s["score"].data_ptr(),
         c["requests"], c["beams"], c["vocab"], c["keep"], s["parent"].data_ptr(), s["token"].data_ptr(),
         s["best"].data_ptr(), s["workspace"].data_ptr(), s["workspace"].numel(), _stream())
    return [s["parent"], s["token"], s["best"]]


def _plain_select(s, c):
    requests, beams, vocab, keep = (c[n] for n in ("requests", "beams", "vocab", "keep"))
    x = s["logits"][:, :vocab]
    e = x.double()  # totals of different beams lie next to one another
    m = e.amax(1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    lse = m + (e - m).exp_().sum(1, keepdim=True).log()
    ranked, order = x.float().sort(dim=1, descending=True, stable=True)
    short = min(keep, vocab)
    ranked, order = ranked[:, :short], order[:, :short]
    total = s["score"].double().view(-1, 1) + (ranked.double() - lse)
    total = torch.where(total > -math.inf, total, -math.inf)  # a row of forbidden tokens has none
    total, order = total.view(requests, beams * short), order.reshape(requests, beams * short)
    best, at = total.sort(dim=1, descending=True, stable=True)
    best, at = best[:, :keep], at[:, :keep]
    there = best > -math.inf
    parent = torch.where(there, at // short, -1).int()
    token = torch.where(there, order.gather(1, at), -1).int()
    return [parent, token, torch.where(there, best, -math.inf).float()]


def _own_fork(s, c):
    from sejong_b200._lib import call
    call("sj_paged_fork", s["parent"].data_ptr(), c["requests"] * c["beams"], c["page"], s["cached"].data_ptr(),
         s["table"].data_ptr(), s["table"].shape[1], s["shares"].data_ptr(), s["free"].data_ptr(),
         s["free_count"].data_ptr(), s["pages"], s["cached_out"].data_ptr(), s["table_out"].data_ptr(),
         s["shares_out"].data_ptr(), s["free_out"].data_ptr(), s["count_out"].data_ptr(), s["copies"].data_ptr(),
         s["summary"].data_ptr(), _stream())
    return [s["cached_out"], s["table_out"], s["shares_out"], s["free_out"], s["count_out"], s["copies"], s["summary"]]


def _plain_fork(s, c):
    batch, page, pages = c["requests"] * c["beams"], c["page"], s["pages"]
    parent, cached, table = s["parent"].long(), s["cached"].long(), s["table"].long()
    count = s["free_count"].long()
    index = torch.arange(batch, device="cuda")
    live = parent >= 0
    source = torch.where(live, parent, 0)
    children = torch.zeros(batch + 1, dtype=torch.long, device="cuda")
    children = children.scatter_add(0, torch.where(live, parent, batch), torch.ones_like(parent))[:batch]
    lowest = torch.full((batch + 1,), batch, dtype=torch.long, device="cuda")
    lowest = lowest.scatter_reduce(0, torch.where(live, parent, batch), index, "amin")
    full, part = cached // page, cached % page
    copied = live & (part[source] > 0) & (lowest[source] != index)
    rank = copied.long().cumsum(0) - 1
    taken = copied.long().sum()
    stack = s["free"].long()
    fresh = stack[(count - 1 - rank).clamp(0, pages - 1)]
    # tables
    at = torch.arange(table.shape[1], device="cuda")[None, :]
    held = (cached + page - 1) // page
    moved = torch.where(copied[:, None] & (at == full[source][:, None]), fresh[:, None], table[source])
    inside = live[:, None] & (at < held[source][:, None])
    table_out = torch.where(inside, moved, s["table_out"].long())
    # owners
    change = torch.where(at < full[:, None], (children - 1)[:, None], -(children == 0).long()[:, None])
    change = torch.where(at < held[:, None], change, 0)
    left = torch.zeros(pages, dtype=torch.long, device="cuda")
    left = left.scatter_add(0, table.clamp(min=0).view(-1), change.view(-1)) + s["shares"]
    gone = left < 0
    # the stack: what is left of it, then the pages that come back, the lowest first
    back = gone.long().cumsum(0)
    depth = count - taken
    free_out = torch.where(torch.arange(pages, device="cuda") < depth, stack, s["free_out"].long())
    free_out = torch.cat((free_out, free_out[:1]))
    place = torch.where(gone, depth + back - 1, pages)
    free_out = free_out.scatter(0, place, torch.arange(pages, device="cuda"))[:pages]
    copies = torch.full((batch + 1, 3), -1, dtype=torch.long, device="cuda")
    copies[:, 2] = 0
    place = torch.where(copied, rank, batch)[:, None].expand(-1, 3)
    last = table.gather(1, full.clamp(max=table.shape[1] - 1)[:, None])[:, 0][source]
    copies = copies.scatter(0, place, torch.stack((last, fresh, part[source]), dim=1))[:batch]
    summary = torch.stack((taken, back[-1], torch.zeros_like(taken), (depth + back[-1])[0]))
    return [x.int() for x in (torch.where(live, cached[source], 0), table_out, torch.where(gone, 0, left), free_out,
                              depth + back[-1], copies, summary)]


def _own_copy(s, c):
    from sejong_b200._lib import call
    k, v = s["k"], s["v"]
    call("sj_paged_copy", s["copies"].data_ptr(), c["padded"], k.data_ptr(), v.data_ptr(), c["layers"], k.stride(0),
         c["pages"], c["page"], k.stride(1), k.stride(2), k.stride(3), c["hk"], c["dim"], _stream())
    return [k, v]


def _plain_copy(s, c):
    todo = s["copies"].long()
    # rows that are not copied are written with what they hold; entries without a page write what one that has writes
    todo = torch.where(todo[:, :1] >= 0, todo, todo[:1])
    row = (torch.arange(c["page"], device="cuda")[None, :] < todo[:, 2:])[None, :, None, :, None]
    for x in (s["k"], s["v"]):
        x[:, todo[:, 1]] = torch.where(row, x[:, todo[:, 0]], x[:, todo[:, 1]])
    return [s["k"], s["v"]]


def _own_compact(s, c):
    from sejong_b200._lib import call
    call("sj_paged_compact", s["cached"].data_ptr(), c["requests"] * c["beams"], c["page"], s["table"].data_ptr(),
         s["table"].shape[1], s["shares"].data_ptr(), s["free"].data_ptr(), s["free_count"].data_ptr(), s["pages"],
         s["table_out"].data_ptr(), s["shares_out"].data_ptr(), s["free_out"].data_ptr(), s["moves"].data_ptr(),
         s["moves"].shape[0], s["summary"].data_ptr(), _stream())
    return [s["table_out"], s["shares_out"], s["free_out"], s["moves"], s["summary"]]


def _plain_compact(s, c):
    page, pages, most = c["page"], s["pages"], s["moves"].shape[0]
    index = torch.arange(pages, device="cuda")
    count = s["free_count"].long()
    used = pages - count
    free = torch.zeros(pages + 1, dtype=torch.bool, device="cuda")
    free[torch.where(index < count, s["free"].long(), pages)] = True
    free = free[:pages]
    moves, hole = ~free & (index >= used), free & (index < used)
    i, j = moves.long().cumsum(0) - 1, hole.long().cumsum(0) - 1
    spare = torch.full((pages + 1,), -1, dtype=torch.long, device="cuda")
    holes = spare.scatter(0, torch.where(hole, j, pages), index)
    to = torch.where(moves, holes[i.clamp(min=0)], index)
    table, held = s["table"].long(), (s["cached"].long() + page - 1) // page
    inside = torch.arange(table.shape[1], device="cuda")[None, :] < held[:, None]
    table_out = torch.where(inside, to[table.clamp(min=0)], s["table_out"].long())
    shares = torch.zeros(pages + 1, dtype=torch.long, device="cuda")
    shares = shares.scatter(0, torch.where(free, pages, to), s["shares"].long())[:pages]
    free_out = torch.where(index < count, pages - 1 - index, s["free_out"].long())
    todo = torch.full((max(most, pages) + 1, 3), -1, dtype=torch.long, device="cuda")
    todo[:, 2] = 0
    place = torch.where(moves, i, max(most, pages))[:, None].expand(-1, 3)
    todo = todo.scatter(0, place, torch.stack((index, to, torch.full_like(index, page)), dim=1))[:most]
    summary = torch.stack((moves.long().sum(), used[0], torch.zeros_like(used[0]), count[0]))
    return [x.int() for x in (table_out, shares, free_out, todo, summary)]


def _own_share(s, c):
    from sejong_b200._lib import call, load
    k, v = s["k"], s["v"]
    if "workspace" not in s:
        size = load().sj_attn_paged_shared_workspace(s["rows"], c["groups"], c["hq"], c["hk"], c["dim"])
        s["workspace"] = torch.zeros(size, dtype=torch.uint8, device="cuda")
    call("sj_attn_paged_shared", s["q"].data_ptr(), s["q"].shape[1], k.data_ptr(), v.data_ptr(), k.shape[0], c["page"],
         k.stride(0), k.stride(1), k.stride(2), s["table"].data_ptr(), s["table"].shape[1], s["table"].shape[0],
         s["request"].data_ptr(), s["position"].data_ptr(), s["rows"], s["group"].data_ptr(), c["groups"], c["hq"],
         c["hk"], c["dim"], c["window"], s["o"].data_ptr(), s["o"].shape[1], s["lse"].data_ptr(),
         s["workspace"].data_ptr(), s["workspace"].numel(), _stream())
    return [s["o"], s["lse"]]


def _part(score, seen):
    """The maximum, the sum and the weights of scores under a mask; nothing seen: -inf, 0 and zeros."""
    score = torch.where(seen, score, -math.inf)
    m = score.amax(-1, keepdim=True)
    p = (score - torch.where(m == -math.inf, 0.0, m)).exp()
    return m, p.sum(-1, keepdim=True), p


def _plain_share(s, c):
    hq, hk, dim, page, window, rows = *(c[n] for n in ("hq", "hk", "dim", "page", "window")), s["rows"]
    fan, scale = hq // hk, 1.0 / math.sqrt(dim)
    q = s["q"].float().view(rows, hk, fan, dim)
    count = s["position"].long() + 1
    least = (count - window).clamp(min=0) if window else torch.zeros_like(count)
    m = torch.empty(rows, hk, fan, 1, device="cuda")
    total, o = torch.empty_like(m), torch.empty(rows, hk, fan, dim, device="cuda")
    first, border = 0, []
    for per, shared, source in zip(s["per"], s["shared"], s["source"]):  # the keys in common, for all rows of a group
        part = slice(first, first + per)
        ids = s["table"][source, :_ceil(shared, page)].long()
        k, v = (x[ids].transpose(0, 1).reshape(hk, -1, dim)[:, :shared].float() for x in (s["k"], s["v"]))
        x = q[part].permute(1, 0, 2, 3).reshape(hk, per * fan, dim)
        key = torch.arange(shared, device="cuda")[None, :]
        seen = (key >= least[part, None]) & (key < count[part, None])
        a, b, p = _part((x @ k.transpose(1, 2) * scale).view(hk, per, fan, shared), seen[None, :, None, :])
        back = lambda y: y.view(hk, per, fan, -1).permute(1, 0, 2, 3)  # noqa: E731
        m[part], total[part], o[part] = back(a), back(b), back(p.view(hk, per * fan, shared) @ v)
        border += [torch.full((per,), shared, device="cuda")]
        first += per
    if s["tail"] > 0:  # each row's own
        border = torch.cat(border)
        step = max(1, int(4e8 / (s["tail"] * hk * dim * 4)))
        for at in range(0, rows, step):
            part = slice(at, min(at + step, rows))
            key = border[part, None] + torch.arange(s["tail"], device="cuda")[None, :]
            seen = (key < count[part, None]) & (key >= least[part, None])
            ids = s["table"][s["request"][part].long()].gather(1, (key // page).clamp(max=s["table"].shape[1] - 1))
            ids = ids.clamp(min=0).long()
            k, v = (torch.where(seen[:, :, None, None], x[ids, :, key % page], 0.0).float().transpose(1, 2)
                    for x in (s["k"], s["v"]))
            a, b, p = _part(q[part] @ k.transpose(2, 3) * scale, seen[:, None, None, :])
            top = torch.maximum(m[part], a)
            base = torch.where(top == -math.inf, 0.0, top)
            f, g = (m[part] - base).exp(), (a - base).exp()
            m[part], total[part], o[part] = top, f * total[part] + g * b, f * o[part] + g * (p @ v)
    lse = (m + total.log()).view(rows, hq)
    o = torch.where(total > 0, o / total, 0.0).reshape(rows, hq * dim)
    return [o.to(s["o"].dtype), lse]


# ---------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    return {"select": _exact_select, "fork": _exact_none, "copy": _exact_copy, "compact": _exact_none,
            "share": _exact_share}[case["op"]](state, case)


def _exact_none(s, c):
    return None  # whole numbers only


def _exact_copy(s, c):
    k, v = s["k"].double(), s["v"].double()
    for source, to, rows in s["copies"].tolist():
        if source >= 0:
            k[:, to, :, :rows], v[:, to, :, :rows] = k[:, source, :, :rows], v[:, source, :, :rows]
    return [k, v]


def _exact_select(s, c):
    requests, beams, vocab, keep = (c[n] for n in ("requests", "beams", "vocab", "keep"))
    best = torch.full((requests, keep), -math.inf, dtype=torch.float64, device="cuda")
    x = s["logits"][:, :vocab].view(requests, beams, vocab)
    for r in range(requests):
        logp = torch.log_softmax(x[r].double(), dim=-1)
        total = (logp + s["score"][r].double()[:, None]).reshape(-1)
        best[r] = total.nan_to_num(nan=-math.inf, neginf=-math.inf).topk(keep).values
    return [None, None, best]


def _exact_share(s, c):
    hq, hk, dim, page = c["hq"], c["hk"], c["dim"], c["page"]
    rows = s["rows"]
    if rows * hq * max(s["shared"]) * dim > 6e11:
        return None
    o = torch.zeros(rows, hq, dim, dtype=torch.float64, device="cuda")
    lse = torch.full((rows, hq), -math.inf, dtype=torch.float64, device="cuda")
    for r, (count, b) in enumerate(zip((s["position"].long() + 1).tolist(), s["request"].tolist())):
        low = max(0, count - c["window"]) if c["window"] else 0
        ids = s["table"][b, low // page:_ceil(count, page)].long()
        skip = low - low // page * page
        k, v = (t[ids].permute(1, 0, 2, 3).reshape(hk, -1, dim)[:, skip:skip + count - low].double()
                for t in (s["k"], s["v"]))
        score = s["q"][r].double().view(hk, hq // hk, dim) @ k.transpose(1, 2) / math.sqrt(dim)
        lse[r] = torch.logsumexp(score, -1).reshape(hq)
        o[r] = (torch.softmax(score, -1) @ v).reshape(hq, dim)
    return [o.reshape(rows, hq * dim), lse]


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    op = case["op"]
    if op == "select":
        requests, beams, vocab = case["requests"], case["beams"], case["vocab"]
        size = 4 if case["f32"] else 2
        live = requests * (1 if case["first"] else beams)
        return {"bytes": live * vocab * size + 4 * requests * beams + 12 * requests * case["keep"],
                "flops": 4 * live * vocab}
    if op in ("fork", "compact"):
        requests, beams, page = case["requests"], case["beams"], case["page"]
        held = _ceil(_spread(requests, case["low"], case["high"]), page)
        entries = int(held.sum()) * beams
        pages = int((held * 0.7).sum() + (held * 0.15).sum() * (beams + 1) // 2 + (held * 0.15).sum() * beams)
        if op == "fork":  # tables, lengths and parents, owners, the stack; in and out
            pages = int(pages * 1.1)
            return {"bytes": 8 * entries + 24 * requests * beams + 8 * pages + 8 * int(pages * 0.1), "flops": 0}
        free = int(pages * case["spare"])
        moved = min(pages, free)
        return {"bytes": 8 * entries + 8 * (pages + free) + 8 * free + 12 * moved, "flops": 0}
    if op == "copy":
        rows = case["copies"] * (case["page"] if case["full"] else (case["page"] + 1) // 2)
        return {"bytes": 8 * rows * case["hk"] * case["dim"] * case["layers"] + 12 * case["padded"], "flops": 0}
    groups, hq, hk, dim, page, window = (case[n] for n in ("groups", "hq", "hk", "dim", "page", "window"))
    per, shared = (_spread(groups, case[n + "low"], case[n + "high"]) for n in ("per_", ""))
    rows = int(per.sum())
    if case["kind"] == "piece":
        tail = (per + 1) / 2  # of a row, on average
        kept = int((shared + per).sum())
    else:
        tail = np.full(groups, _spread(rows, case["own_low"], case["own_high"]).mean())
        kept = int(shared.sum() + rows * tail[0])
    seen = shared + tail
    if window:
        seen = np.minimum(seen, window)
        kept = min(kept, rows * window)
    return {"bytes": int(4 * kept * hk * dim + 4 * rows * hq * dim + 4 * rows * hq + 4 * kept // page + 8 * rows),
            "flops": int(4 * float((per * seen).sum()) * hq * dim)}
