"""Cases that measure the operators of batched serving on a paged key-value cache, and of scoring tokens:

  plan        sj_paged_plan        block tables, positions and cache slots of a step's rows, from the requests' lengths
  append      sj_paged_append      rotary positions of the step's queries and keys; keys and values into their cache slots
  attend      sj_attn_paged        attention of each row over its request's pages
  score       sj_token_scores      log probability of given tokens, entropy and the best alternatives of each row of logits
  score_bwd   sj_token_scores_bwd  the logits' gradient from those of the log probabilities and entropies

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
        # one decoding step of a middling batch: a new token each, some requests start a page with it
        {"name": "plan decode", "op": "plan", "batch": 64, "page": 16, "low": 1, "high": 8192, "chunks": 0, "chunk": 1,
         "rows": 64},
        # a step of a large server: most requests decode, 32 bring a piece of their prompt; rows padded for a graph
        {"name": "plan mixed", "op": "plan", "batch": 1021, "page": 64, "low": 1, "high": 32768, "chunks": 32,
         "chunk": 1500, "rows": 50000},
        # the decode step of the byte model's global heads (12 query, 4 key heads), padded to the graph's 64 rows
        {"name": "append decode", "op": "append", "rows": 64, "live": 50, "hq": 12, "hk": 4, "dim": 64, "rot": 64,
         "half": False, "page": 16, "context": 8192, "layout": "head"},
        # a prompt batch with wide heads of which a part is rotated, in halves
        {"name": "append prompt", "op": "append", "rows": 32003, "live": 32003, "hq": 16, "hk": 2, "dim": 128,
         "rot": 64, "half": True, "page": 64, "context": 131072, "layout": "head"},
        # the least a server meets: a few short requests of the small dense model; latency counts
        {"name": "attend short", "op": "attend", "rows": 3, "low": 7, "high": 250, "hq": 4, "hk": 2, "dim": 64,
         "page": 16, "window": 0, "layout": "head"},
        # the byte model's local stages: every head its own keys, 128 keys in sight
        {"name": "attend window", "op": "attend", "rows": 192, "low": 1, "high": 8192, "hq": 4, "hk": 4, "dim": 64,
         "page": 16, "window": 128, "layout": "token"},
        # few requests with a long context: the length has to be split over the GPU
        {"name": "attend long", "op": "attend", "rows": 2, "low": 150001, "high": 200003, "hq": 16, "hk": 4, "dim": 64,
         "page": 64, "window": 0, "layout": "head"},
        # a full server with ragged lengths
        {"name": "attend ragged", "op": "attend", "rows": 256, "low": 512, "high": 16384, "hq": 12, "hk": 4, "dim": 64,
         "page": 16, "window": 0, "layout": "head"},
        # alternatives beside the sampled byte of a decode step; bytes outside a grammar masked
        {"name": "score decode", "op": "score", "rows": 64, "vocab": 257, "ld": 264, "top": 5, "f32": True,
         "masked": True},
        # scores of a scored or sampled batch with a word vocabulary
        {"name": "score words", "op": "score", "rows": 2048, "vocab": 50001, "ld": 50008, "top": 20, "f32": False,
         "masked": False},
        # a policy or distillation step of the byte model: batch 32 x 1024
        {"name": "gradient bytes", "op": "score_bwd", "rows": 32768, "vocab": 257, "ld": 264, "f32": True,
         "masked": False},
        # the same with a word vocabulary, 16-bit logits
        {"name": "gradient words", "op": "score_bwd", "rows": 2048, "vocab": 65537, "ld": 65544, "f32": False,
         "masked": False},
    ]


def _log(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def _heads(rng):
    while True:
        dim, hk, group = rng.choice((64, 64, 128)), rng.choice((1, 2, 4, 8)), rng.choice((1, 2, 3, 4, 5, 8, 12, 16))
        widths = (hk * dim, hk * group * dim, (hk * group + 2 * hk) * dim)
        if hk * group <= 64 and 3072 not in widths:
            return dim, hk, hk * group


def draw(rng):
    op = rng.choice(("plan", "append", "attend", "attend", "score", "score_bwd"))
    page = rng.choice((8, 16, 16, 24, 32, 64, 128))
    if op == "plan":
        batch = _log(rng, 1, 1500)
        chunks = rng.choice((0, 0, rng.randint(0, min(batch, 40))))
        chunk = _log(rng, 2, 1500)
        rows = batch - chunks + chunks * chunk
        return {"op": op, "batch": batch, "page": page, "low": 1, "high": _log(rng, 64, 32768), "chunks": chunks,
                "chunk": chunk, "rows": rows + rng.choice((0, rng.randint(0, 500)))}
    if op == "append":
        dim, hk, hq = _heads(rng)
        live = _log(rng, 1, 20000)
        return {"op": op, "rows": live + rng.choice((0, rng.randint(0, 40))), "live": live, "hq": hq, "hk": hk,
                "dim": dim, "rot": rng.choice((dim, dim, dim // 2, 16, 48)), "half": rng.random() < 0.5, "page": page,
                "context": _log(rng, 1000, 131072), "layout": rng.choice(("head", "token"))}
    if op == "attend":
        dim, hk, hq = _heads(rng)
        window = rng.choice((0, 0, 0, _log(rng, 1, 4096)))
        rows = _log(rng, 1, 300)
        most = int(8e8 / (rows * hk * dim * 4))  # tokens of the longest request: a cache of at most 0.8 GB
        high = _log(rng, 16, max(17, min(200000, most)))
        return {"op": op, "rows": rows, "low": _log(rng, 1, high), "high": high, "hq": hq, "hk": hk, "dim": dim,
                "page": page, "window": window, "layout": rng.choice(("head", "token"))}
    vocab = rng.choice((257, _log(rng, 2, 130000)))
    rows = _log(rng, 1, max(2, min(32768, int(6e7 / vocab))))
    case = {"op": op, "rows": rows, "vocab": vocab, "ld": vocab + rng.choice((0, 7, -vocab % 8)),
            "f32": rng.random() < 0.5, "masked": rng.random() < 0.3}
    if op == "score":
        case["top"] = min(vocab, rng.choice((0, 1, 5, 20, 32)))
    return case


def _lengths(count, low, high):
    """`count` lengths between low and high, even over their logarithm."""
    at = (np.arange(count) + 0.5) / count
    return np.maximum(1, np.rint(low * (high / low) ** at)).astype(np.int64)


def _ceil(a, b):
    return -(-a // b)


# ---------------------------------------------------------------- inputs
def prepare(case, seed):
    host = np.random.default_rng(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = {"case": case}
    {"plan": _prepare_plan, "append": _prepare_append, "attend": _prepare_attend, "score": _prepare_score,
     "score_bwd": _prepare_score}[case["op"]](case, state, host, gen)
    return state


def _int(a):
    return torch.as_tensor(np.ascontiguousarray(a), dtype=torch.int32, device="cuda")


def _empty(*shape, dtype=torch.int32):
    return torch.empty(*shape, dtype=dtype, device="cuda")


def _added(case):
    added = np.ones(case["batch"], dtype=np.int64)
    added[:case["chunks"]] = case["chunk"]
    return added


def _prepare_plan(case, state, host, gen):
    batch, page = case["batch"], case["page"]
    order = host.permutation(batch)
    cached = _lengths(batch, case["low"], case["high"])[order]
    added = _added(case)[host.permutation(batch)]
    held, need = _ceil(cached, page), _ceil(cached + added, page)
    width = int(need.max()) + 3
    pages = int(need.sum()) + 100
    ids = host.permutation(pages)
    table = np.full((batch, width), NO_PAGE, dtype=np.int64)
    inside = np.arange(width)[None, :] < held[:, None]
    table[inside] = ids[:int(held.sum())]
    free = ids[int(held.sum()):]
    rows = case["rows"]
    state.update(cached=_int(cached), added=_int(added), table=_int(table), free=_int(free),
                 free_count=_int([free.size]), lengths=_empty(batch), request=_empty(rows), position=_empty(rows),
                 slot=_empty(rows), summary=_empty(4))


def _cache(case, pages, gen):
    """K and V pages as [page, head, token, dim] views of either storage order; every slot holds something."""
    shape = ((pages, case["hk"], case["page"], case["dim"]) if case["layout"] == "head"
             else (pages, case["page"], case["hk"], case["dim"]))
    k, v = (torch.randn(shape, dtype=torch.bfloat16, device="cuda", generator=gen) for _ in range(2))
    return (k, v) if case["layout"] == "head" else (k.transpose(1, 2), v.transpose(1, 2))


def _rope_table(context, rot):
    """(cos, sin) of each position's rot / 2 angles, base 10000."""
    at = torch.arange(context, dtype=torch.float64, device="cuda")
    freq = 10000.0 ** (torch.arange(rot // 2, dtype=torch.float64, device="cuda") * (-2.0 / rot))
    angle = at[:, None] * freq
    return torch.stack((angle.cos(), angle.sin()), dim=-1).float().contiguous()


def _prepare_append(case, state, host, gen):
    rows, live, page, dim, hq, hk = (case[n] for n in ("rows", "live", "page", "dim", "hq", "hk"))
    pages = _ceil(live, page) + 8
    slots = np.full(rows, -1, dtype=np.int64)
    slots[:live] = host.permutation((pages - 1) * page)[:live]  # none in the last page
    position = np.where(slots >= 0, host.integers(0, case["context"], rows), -1)
    k, v = _cache(case, pages, gen)
    qkv = torch.randn(rows, (hq + 2 * hk) * dim, dtype=torch.bfloat16, device="cuda", generator=gen)
    state.update(qkv=qkv, position=_int(position), slot=_int(slots), k=k, v=v,
                 rope=_rope_table(case["context"], case["rot"]), q=_empty(rows, hq * dim, dtype=torch.bfloat16))


def _prepare_attend(case, state, host, gen):
    rows, page, dim, hq = (case[n] for n in ("rows", "page", "dim", "hq"))
    length = _lengths(rows, case["low"], case["high"])[host.permutation(rows)]
    held = _ceil(length, page)
    pages, width = int(held.sum()) + 3, int(held.max()) + 2
    table = np.full((rows, width), NO_PAGE, dtype=np.int64)
    table[np.arange(width)[None, :] < held[:, None]] = host.permutation(pages)[:int(held.sum())]
    k, v = _cache(case, pages, gen)
    q = torch.randn(rows, hq * dim, dtype=torch.bfloat16, device="cuda", generator=gen)
    state.update(q=q, k=k, v=v, table=_int(table), position=_int(length - 1), longest=int(length.max()),
                 o=_empty(rows, hq * dim, dtype=torch.bfloat16), lse=_empty(rows, hq, dtype=torch.float32))


def _prepare_score(case, state, host, gen):
    rows, vocab, ld = case["rows"], case["vocab"], case["ld"]
    kind = torch.float32 if case["f32"] else torch.bfloat16
    x = torch.randn(rows, ld, device="cuda", generator=gen) * 3.0
    target = _int(host.integers(0, vocab, rows))
    if case["masked"]:  # about a third of the entries are forbidden, never the target
        out = torch.rand(rows, ld, device="cuda", generator=gen) < 0.33
        out.scatter_(1, target.long()[:, None], False)
        x.masked_fill_(out, -math.inf)
    x = x.to(kind)
    state.update(logits=x, target=target)
    if case["op"] == "score":
        top = case["top"]
        state.update(logp=_empty(rows, dtype=torch.float32), entropy=_empty(rows, dtype=torch.float32),
                     lse=_empty(rows, dtype=torch.float32), top_id=_empty(rows, top),
                     top_logp=_empty(rows, top, dtype=torch.float32))
        return
    # what the forward pass kept, and the gradients that came back for it
    step = max(1, (1 << 25) // vocab)
    lse, entropy = [], []
    for at in range(0, rows, step):
        a, b, _ = _statistics(x[at:at + step, :vocab].double())
        lse.append(a)
        entropy.append(b)
    state.update(lse=torch.cat(lse).float(), entropy=torch.cat(entropy).float(),
                 d_logp=torch.randn(rows, device="cuda", generator=gen),
                 d_entropy=torch.randn(rows, device="cuda", generator=gen) * 0.1, d_logits=_empty(rows, ld, dtype=kind))


def _statistics(x):
    """lse, entropy and the log probabilities of each row, in the type of x."""
    m = x.amax(1, keepdim=True)
    shifted = x - m
    e = shifted.exp()
    s = e.sum(1, keepdim=True)
    logp = shifted - s.log()
    entropy = -(torch.where(e > 0, logp, 0.0) * e).sum(1) / s[:, 0]
    return (m + s.log())[:, 0], entropy, logp


# ---------------------------------------------------------------- one pass
def run(state):
    op = state["case"]["op"]
    if own:
        return {"plan": _own_plan, "append": _own_append, "attend": _own_attend, "score": _own_score,
                "score_bwd": _own_score_bwd}[op](state, state["case"])
    return {"plan": _plain_plan, "append": _plain_append, "attend": _plain_attend, "score": _plain_score,
            "score_bwd": _plain_score_bwd}[op](state, state["case"])


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _own_plan(s, c):
    from sejong_b200._lib import call
    call("sj_paged_plan", s["cached"].data_ptr(), s["added"].data_ptr(), c["batch"], c["page"], s["free"].data_ptr(),
         s["free_count"].data_ptr(), s["table"].data_ptr(), s["table"].shape[1], s["lengths"].data_ptr(),
         s["request"].data_ptr(), s["position"].data_ptr(), s["slot"].data_ptr(), c["rows"], s["summary"].data_ptr(),
         _stream())
    return [s["table"], s["lengths"], s["request"], s["position"], s["slot"], s["summary"]]


def _plain_plan(s, c):
    page, rows, table = c["page"], c["rows"], s["table"]
    cached, added = s["cached"].long(), s["added"].long()
    lengths = cached + added
    held, need = (cached + page - 1) // page, (lengths + page - 1) // page
    taken = (need - held).cumsum(0)
    at = torch.arange(table.shape[1], device="cuda")[None, :]
    order = (taken - (need - held))[:, None] + at - held[:, None]
    new = (at >= held[:, None]) & (at < need[:, None])
    pick = s["free"][(s["free_count"].long() - 1 - order).clamp(0, s["free"].shape[0] - 1)]
    table = torch.where(new, pick, table)
    ends = added.cumsum(0)
    r = torch.arange(rows, device="cuda")
    live = r < ends[-1]
    request = torch.searchsorted(ends, r, right=True).clamp(max=c["batch"] - 1)
    position = cached[request] + r - (ends - added)[request]
    slot = table[request, (position // page).clamp(max=table.shape[1] - 1)].long() * page + position % page
    summary = torch.stack((ends[-1], taken[-1], torch.zeros_like(ends[-1]), s["free_count"][0] - taken[-1]))
    return [table, lengths.int(), torch.where(live, request, -1).int(), torch.where(live, position, -1).int(),
            torch.where(live, slot, -1).int(), summary.int()]


def _own_append(s, c):
    from sejong_b200._lib import call
    k, v = s["k"], s["v"]
    call("sj_paged_append", s["qkv"].data_ptr(), s["qkv"].shape[1], s["position"].data_ptr(), s["slot"].data_ptr(),
         c["rows"], c["hq"], c["hk"], c["dim"], s["rope"].data_ptr(), c["context"], c["rot"], int(c["half"]),
         s["q"].data_ptr(), s["q"].shape[1], k.data_ptr(), v.data_ptr(), k.shape[0], c["page"], k.stride(0),
         k.stride(1), k.stride(2), _stream())
    return [s["q"], k, v]


def _rotate(x, table, position, rot, half):
    """x [rows, heads, dim]: the first `rot` of each head turned by its row's angles."""
    at = table[position.clamp(min=0).long()]
    cos, sin = at[:, None, :, 0], at[:, None, :, 1]
    turned, rest = x[..., :rot], x[..., rot:]
    if half:
        a, b = turned[..., :rot // 2], turned[..., rot // 2:]
        return torch.cat((a * cos - b * sin, a * sin + b * cos, rest), dim=-1)
    a, b = turned[..., 0::2], turned[..., 1::2]
    return torch.cat((torch.stack((a * cos - b * sin, a * sin + b * cos), dim=-1).flatten(-2), rest), dim=-1)


def _append(s, c, kind):
    """Queries, keys and values of each row in `kind`, where the keys and values go, and which rows there are."""
    rows, hq, hk, dim, page = c["rows"], c["hq"], c["hk"], c["dim"], c["page"]
    x = s["qkv"].to(kind).view(rows, hq + 2 * hk, dim)
    live = (s["slot"] >= 0)[:, None, None]
    last = s["k"].shape[0] * page - 1  # a slot that no row of the batch owns
    slot = torch.where(s["slot"] >= 0, s["slot"], last).long()
    turned = _rotate(x[:, :hq + hk], s["rope"].to(kind), s["position"], c["rot"], c["half"])
    q = torch.where(live, turned[:, :hq], 0.0).reshape(rows, hq * dim)
    return q, turned[:, hq:], x[:, hq + hk:], slot // page, slot % page, live


def _plain_append(s, c):
    q, k, v, at, off, live = _append(s, c, torch.float32)
    for cache, new in ((s["k"], k), (s["v"], v)):
        cache[at, :, off] = torch.where(live, new.to(cache.dtype), cache[at, :, off])
    return [q.to(s["q"].dtype), s["k"], s["v"]]


def _own_attend(s, c):
    from sejong_b200._lib import call, load
    k, v = s["k"], s["v"]
    if "workspace" not in s:  # kept by the program, zero before its first use
        size = load().sj_attn_paged_workspace(c["rows"], c["hq"], c["hk"], c["dim"])
        s["workspace"] = torch.zeros(size, dtype=torch.uint8, device="cuda")
    call("sj_attn_paged", s["q"].data_ptr(), s["q"].shape[1], k.data_ptr(), v.data_ptr(), k.shape[0], c["page"],
         k.stride(0), k.stride(1), k.stride(2), s["table"].data_ptr(), s["table"].shape[1], c["rows"], 0,
         s["position"].data_ptr(), c["rows"], c["hq"], c["hk"], c["dim"], c["window"], s["o"].data_ptr(),
         s["o"].shape[1], s["lse"].data_ptr(), s["workspace"].data_ptr(), s["workspace"].numel(), _stream())
    return [s["o"], s["lse"]]


def _plain_attend(s, c):
    rows, hq, hk, dim, page = c["rows"], c["hq"], c["hk"], c["dim"], c["page"]
    span = min(s["longest"], c["window"]) if c["window"] else s["longest"]
    count = s["position"].long() + 1
    first = (count - span).clamp(min=0) if c["window"] else torch.zeros_like(count)
    key = first[:, None] + torch.arange(span, device="cuda")[None, :]
    seen = (key < count[:, None])[:, None, :, None]
    at = s["table"].gather(1, (key // page).clamp(max=s["table"].shape[1] - 1)).clamp(min=0).long()
    k = torch.where(seen, s["k"][at, :, key % page].transpose(1, 2), 0.0).float()  # [rows, hk, span, dim]
    q = s["q"].float().view(rows, hk, hq // hk, dim)
    score = torch.where(seen.transpose(2, 3), q @ k.transpose(2, 3) / math.sqrt(dim), -math.inf)
    del k
    m = score.amax(-1, keepdim=True)
    p = (score - m).exp()
    total = p.sum(-1, keepdim=True)
    v = torch.where(seen, s["v"][at, :, key % page].transpose(1, 2), 0.0).float()
    o = (p @ v / total).reshape(rows, hq * dim)
    return [o.to(s["o"].dtype), (m + total.log()).reshape(rows, hq)]


def _own_score(s, c):
    from sejong_b200._lib import SJ_BF16, SJ_F32, call, load
    if "workspace" not in s:
        size = load().sj_token_scores_workspace(c["rows"], c["vocab"], c["top"])
        s["workspace"] = torch.zeros(max(size, 1), dtype=torch.uint8, device="cuda")
    call("sj_token_scores", s["logits"].data_ptr(), SJ_F32 if c["f32"] else SJ_BF16, c["ld"], s["target"].data_ptr(),
         c["rows"], c["vocab"], c["top"], s["logp"].data_ptr(), s["entropy"].data_ptr(), s["lse"].data_ptr(),
         s["top_id"].data_ptr(), s["top_logp"].data_ptr(), s["workspace"].data_ptr(), s["workspace"].numel(),
         _stream())
    return [s["logp"], s["entropy"], s["lse"], s["top_logp"], s["top_id"]]


def _plain_score(s, c):
    x = s["logits"][:, :c["vocab"]].float()
    lse, entropy, logp = _statistics(x)
    ranked, order = x.sort(dim=1, descending=True, stable=True)
    top = c["top"]
    best = logp.gather(1, order[:, :top])
    return [logp.gather(1, s["target"].long()[:, None])[:, 0], entropy, lse, best, order[:, :top].int()]


def _own_score_bwd(s, c):
    from sejong_b200._lib import SJ_BF16, SJ_F32, call
    call("sj_token_scores_bwd", s["logits"].data_ptr(), SJ_F32 if c["f32"] else SJ_BF16, c["ld"],
         s["target"].data_ptr(), c["rows"], c["vocab"], s["lse"].data_ptr(), s["entropy"].data_ptr(),
         s["d_logp"].data_ptr(), s["d_entropy"].data_ptr(), s["d_logits"].data_ptr(), c["ld"], _stream())
    return [s["d_logits"]]


def _gradient(s, c, rows, kind):
    """d logits [rows, ld] of a slice of rows: d_logp (1[target] - p) - d_entropy p (log p + entropy)."""
    vocab = c["vocab"]
    logp = s["logits"][rows, :vocab].to(kind) - s["lse"][rows, None].to(kind)
    p = logp.exp()
    a, b, h = (s[n][rows, None].to(kind) for n in ("d_logp", "d_entropy", "entropy"))
    g = -p * (a + b * (torch.where(p > 0, logp, 0.0) + h))
    hit = torch.arange(vocab, device="cuda")[None, :] == s["target"][rows, None]
    out = torch.zeros(g.shape[0], c["ld"], dtype=kind, device="cuda")
    out[:, :vocab] = torch.where(hit, g + a, g)
    return out


def _plain_score_bwd(s, c):
    return [_gradient(s, c, slice(None), torch.float32).to(s["d_logits"].dtype)]


# ---------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    return {"plan": _exact_plan, "append": _exact_append, "attend": _exact_attend, "score": _exact_score,
            "score_bwd": _exact_score_bwd}[case["op"]](state, case)


def _exact_plan(s, c):
    return None  # whole numbers only


def _exact_append(s, c):
    rows, hq, hk, dim, page, rot = (c[n] for n in ("rows", "hq", "hk", "dim", "page", "rot"))
    x = s["qkv"].double().view(rows, hq + 2 * hk, dim)
    slot, position = s["slot"].long(), s["position"].long()
    live = slot >= 0
    angle = torch.view_as_complex(s["rope"].double().contiguous())[position.clamp(min=0)][:, None, :]
    y = x[:, :hq + hk].clone()
    index = torch.arange(rot, device="cuda")
    first, second = (index[:rot // 2], index[rot // 2:]) if c["half"] else (index[0::2], index[1::2])
    z = torch.complex(x[:, :hq + hk, first], x[:, :hq + hk, second]) * angle
    y[:, :, first], y[:, :, second] = z.real, z.imag
    q = (y[:, :hq] * live[:, None, None]).reshape(rows, hq * dim)
    k, v = s["k"].double(), s["v"].double()
    k[slot[live] // page, :, slot[live] % page] = y[live, hq:]
    v[slot[live] // page, :, slot[live] % page] = x[live, hq + hk:]
    return [q, k, v]


def _exact_attend(s, c):
    rows, hq, hk, dim, page = (c[n] for n in ("rows", "hq", "hk", "dim", "page"))
    counts = (s["position"].long() + 1).tolist()
    o = torch.zeros(rows, hq, dim, dtype=torch.float64, device="cuda")
    lse = torch.full((rows, hq), -math.inf, dtype=torch.float64, device="cuda")
    for r, count in enumerate(counts):
        low = max(0, count - c["window"]) if c["window"] else 0
        ids = s["table"][r, low // page:_ceil(count, page)].long()
        skip = low - low // page * page
        k, v = (t[ids].permute(1, 0, 2, 3).reshape(hk, -1, dim)[:, skip:skip + count - low].double()
                for t in (s["k"], s["v"]))
        score = s["q"][r].double().view(hk, hq // hk, dim) @ k.transpose(1, 2) / math.sqrt(dim)
        lse[r] = torch.logsumexp(score, -1).reshape(hq)
        o[r] = (torch.softmax(score, -1) @ v).reshape(hq, dim)
    return [o.reshape(rows, hq * dim), lse]


def _exact_score(s, c):
    rows, vocab, top = c["rows"], c["vocab"], c["top"]
    out = [[], [], [], []]
    step = max(1, (1 << 25) // vocab)
    for at in range(0, rows, step):
        logp = torch.log_softmax(s["logits"][at:at + step, :vocab].double(), 1)
        target = s["target"][at:at + step].long()[:, None]
        out[0].append(logp.gather(1, target)[:, 0])
        out[1].append(torch.special.entr(logp.exp()).sum(1))
        out[2].append(torch.logsumexp(s["logits"][at:at + step, :vocab].double(), 1))
        out[3].append(logp.topk(top, dim=1).values)
    return [torch.cat(x) for x in out] + [None]


def _exact_score_bwd(s, c):
    rows, vocab = c["rows"], c["vocab"]
    step = max(1, (1 << 25) // vocab)
    out = torch.zeros(rows, c["ld"], dtype=torch.float64, device="cuda")
    for at in range(0, rows, step):
        part = slice(at, at + step)
        x = s["logits"][part, :vocab].double()
        p = (x - s["lse"][part, None].double()).exp()
        a, b, h = (s[n][part, None].double() for n in ("d_logp", "d_entropy", "entropy"))
        g = -a * p + b * (torch.special.entr(p) - h * p)
        out[part, :vocab] = g.scatter_add(1, s["target"][part].long()[:, None], a)
    return [out]


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    op = case["op"]
    if op == "plan":
        batch, page = case["batch"], case["page"]
        # lengths in and out, the new rows' three maps and the summary; the new pages read and entered
        new = int(_added(case).sum()) // page
        return {"bytes": 4 * (4 * batch + 3 * case["rows"] + 2 * new + 4), "flops": 0}
    if op == "append":
        rows, live, dim, hq, hk = (case[n] for n in ("rows", "live", "dim", "hq", "hk"))
        moved = 2 * 2 * live * (hq + 2 * hk) * dim + 2 * (rows - live) * hq * dim
        table = min(live, case["context"]) * case["rot"] * 4
        return {"bytes": moved + table + 8 * rows, "flops": 3 * live * (hq + hk) * case["rot"]}
    if op == "attend":
        rows, dim, hq, hk = (case[n] for n in ("rows", "dim", "hq", "hk"))
        length = _lengths(rows, case["low"], case["high"])
        pages = int(_ceil(length, case["page"]).sum())
        keys = int((np.minimum(length, case["window"]) if case["window"] else length).sum())
        if case["window"]:
            pages = min(pages, keys // case["page"] + rows)
        return {"bytes": 2 * 2 * keys * hk * dim + 2 * 2 * rows * hq * dim + 4 * rows * hq + 4 * pages + 4 * rows,
                "flops": 4 * keys * hq * dim}
    rows, vocab, size = case["rows"], case["vocab"], 4 if case["f32"] else 2
    if op == "score":
        return {"bytes": rows * (vocab * size + 4 + 12 + 8 * case["top"]), "flops": 5 * rows * vocab}
    return {"bytes": rows * ((vocab + case["ld"]) * size + 20), "flops": 7 * rows * vocab}
