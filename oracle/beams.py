"""FP64 / integer restatement of several continuations of one prompt: a beam search's selection, and the books of a
paged cache whose pages are shared (numpy, one request or page at a time)."""
import numpy as np

from .paged import ceil_div


def select(logits, score, keep):
    """(parent, token, total) [requests, keep] of logits f64 [requests, beams, vocab] and scores f64 [requests, beams];
    -1 and -inf past the last candidate."""
    requests, beams, vocab = logits.shape
    parent, token = (np.full((requests, keep), -1, dtype=np.int64) for _ in range(2))
    best = np.full((requests, keep), -np.inf)
    for r in range(requests):
        total = np.full((beams, vocab), -np.inf)
        for b in range(beams):
            x, m = logits[r, b], np.max(logits[r, b])
            if not (np.isfinite(m) and np.isfinite(score[r, b])):  # NaN, +inf, or nothing allowed
                continue
            total[b] = score[r, b] + ((x - m) - np.log(np.sum(np.exp(x - m))))
        order = np.argsort(-total.reshape(-1), kind="stable")[:keep]
        there = total.reshape(-1)[order] > -np.inf
        order = order[there]
        n = len(order)
        parent[r, :n], token[r, :n], best[r, :n] = order // vocab, order % vocab, total.reshape(-1)[order]
    return parent, token, best


def fork(parent, page, cached, table, shares, free):
    """(cached, table, shares, free, copies, back, status) after the requests took over one another's pages.  `free` is
    the stack, its top last; table rows are as long as given, entries that hold no page are -1."""
    batch, width = len(cached), len(table[0])
    old = [np.array(cached), np.array(table), np.array(shares), list(free), [], 0]
    if any(not -1 <= p < batch for p in parent) or any(c < 0 for c in cached):
        return (*old, 4)
    if any(ceil_div(c, page) > width for c in cached):
        return (*old, 3)
    stack = list(free)
    owners = {p: 0 for p in range(len(shares))}
    for b in range(batch):
        for j in range(ceil_div(cached[b], page)):
            owners[table[b][j]] += 1
    for p in owners:  # owners that the tables do not show (none in a whole state)
        owners[p] += (shares[p] + 1 - owners[p]) if owners[p] else 0
    held_before = {p for p in owners if owners[p] > 0}
    out, lengths, copies, seen = np.full((batch, width), -1), [], [], set()
    for b in range(batch):
        for j in range(ceil_div(cached[b], page)):
            owners[table[b][j]] -= 1
    for b, p in enumerate(parent):
        lengths.append(0 if p < 0 else cached[p])
        if p < 0:
            continue
        for j in range(ceil_div(cached[p], page)):
            partly = j == cached[p] // page
            if partly and p in seen:
                if not stack:
                    return (*old, 2)
                fresh = stack.pop()
                copies.append((table[p][j], fresh, cached[p] % page))
                out[b][j] = fresh
                owners[fresh] += 1
            else:
                out[b][j] = table[p][j]
                owners[table[p][j]] += 1
        seen.add(p)
    back = sorted(p for p in held_before if owners[p] == 0)
    return np.array(lengths), out, np.array([max(owners[p] - 1, 0) for p in range(len(shares))]), stack + back, copies, \
        len(back), 0


def compact(page, cached, table, shares, free, pages):
    """(table, shares, free, moves) with the pages in use at the lowest ids."""
    gone = set(free)
    used = pages - len(gone)
    front = [p for p in range(used) if p in gone]
    moves = list(zip([p for p in range(used, pages) if p not in gone], front))
    to = {p: p for p in range(pages)}
    to.update(dict(moves))
    out = np.full_like(np.array(table), -1)
    for b, c in enumerate(cached):
        for j in range(ceil_div(c, page)):
            out[b, j] = to[table[b][j]]
    more = np.zeros(pages, dtype=np.int64)
    for p in range(pages):
        if p not in gone:
            more[to[p]] = shares[p]
    return out, more, list(range(pages - 1, used - 1, -1)), moves
