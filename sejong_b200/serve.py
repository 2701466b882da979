"""Batched generation and scoring for the dense byte model on a paged key-value cache.

The reference generates for one prompt at a time (crates/sejong-runtime/src/lib.rs:84-126) on one contiguous
cache (crates/sejong-model/src/architecture.rs:395-533); `Generator` restates that.  `BatchGenerator` keeps up
to `batch` requests in one cache of `pages` pages a layer and steps them together:

  * a step is a sj_paged_commit of the one before (which returns the pages of finished requests) and a
    sj_paged_plan of the new tokens: block tables, positions and slots, all on the GPU;
  * a prompt runs through the training kernels (GEMMs with the rotary epilogue, tcgen05 attention), and
    sj_paged_append files its keys and values;
  * a decode step is one CUDA graph for `batch` rows, whatever number of them is live: the QKV GEMM, the rotary
    append at each row's own position, sj_attn_paged, the rest of the block, the head;
  * prompts are run one at a time, between decode steps;
  * bytes are sampled on the host as `Generator` does, each request with its own Sampling and Rng, and
    sj_token_scores gives the sampled bytes' log probabilities, the entropies and the best alternatives;
  * requests wait until the pages that they may come to need are free, so a step never runs out of them; a full
    context restarts from its last `context` tokens, as the reference does;
  * a call that raises leaves an empty cache.

`generate` with `samples`, and `beam_search`, keep several continuations of each prompt.  The prompt runs once, and its
requests share its pages: a step begins with a sj_paged_fork of the requests (which counts the owners of pages, and takes
back those that nobody holds), a sj_paged_copy of half-filled pages, and its attention is sj_attn_paged_shared;
sj_beam_select finds the best continuations of a request's beams.

`score` gives the same figures for the bytes of a given text of at most `context` bytes.  `rope_scaling` stretches the
rotary positions beyond the trained context (sj_rope_table_scaled).
"""
import ctypes
from collections import deque
from dataclasses import dataclass, field
from typing import Optional

import numpy as np
import torch

from . import _lib
from ._lib import (EPI_RESIDUAL, EPI_ROPE, EPI_STORE, EPI_SWIGLU, ROPE_BASE, ROPE_LINEAR, ROPE_RAMP, SJ_BF16, SJ_F32,
                   call)
from .generate import Sampling, _ptr, check_sampling, sample
from .model import EOS, HEAD_DIM, VOCAB, VOCAB_PAD, FlatLayout, global_stage, initialize


SHARED_PAGES = 1 << 18  # that sj_paged_fork takes


@dataclass
class RopeScaling:
    """Rotary positions for contexts longer than the trained one: "linear" (positions divided by the factor),
    "base" (a larger base) or "ramp" (each frequency by its turns over `original` positions)."""
    kind: str
    factor: float
    original: int = 0
    fast: float = 32.0
    slow: float = 1.0

    def code(self):
        kinds = {"linear": ROPE_LINEAR, "base": ROPE_BASE, "ramp": ROPE_RAMP}
        if self.kind not in kinds:
            raise ValueError(f"rope scaling {self.kind!r}: linear, base or ramp")
        return kinds[self.kind]


@dataclass
class Scores:
    """Of each byte: its log probability, the entropy of the distribution it was drawn from, and the best
    alternatives as (token, log probability)."""
    logp: list = field(default_factory=list)
    entropy: list = field(default_factory=list)
    alternatives: list = field(default_factory=list)


@dataclass
class Completion:
    text: bytes
    ended: bool                       # EOS was drawn
    scores: Optional[Scores] = None   # with one more entry than `text` when it ended: the EOS


@dataclass
class Hypothesis:
    """A beam search's result: `score` is the sum of the bytes' log probabilities, `ranked` what they are ordered by."""
    text: bytes
    ended: bool
    score: float
    ranked: float


@dataclass
class _Beams:
    index: int
    tokens: list
    reserved: int
    live: list = field(default_factory=list)     # (drawn bytes, score) of each beam
    ended: list = field(default_factory=list)    # hypotheses


@dataclass
class _Request:
    index: int
    tokens: list
    options: Sampling
    state: ctypes.c_uint64
    reserved: int
    length: int = 0
    out: list = field(default_factory=list)
    scores: Optional[Scores] = None


class BatchGenerator:
    def __init__(self, config, params=None, device=None, context=None, batch=32, page=16, pages=None,
                 rope_scaling=None):
        if config.hierarchy is not None or config.experts is not None:
            raise ValueError("batched generation covers the dense byte model without experts")
        if batch < 1 or batch > 4096 or page < 1:
            raise ValueError("batch must be 1 to 4096 and page at least 1")
        self.c = c = config
        self.dev = torch.device("cuda", torch.cuda.current_device() if device is None else device)
        torch.cuda.set_device(self.dev)
        self.lib = _lib.load()
        call("sj_device_init", self.dev.index)
        self.context, self.batch, self.page = L, B, P = int(context or c.context), int(batch), int(page)
        if not 0 < L < 1 << 19:
            raise ValueError("the context must be 1 to 524287")
        self.width = -(-L // P)
        self.pages = int(pages or self.default_pages())
        if self.pages < 1:
            raise ValueError("the cache needs at least one page")
        self.layout = FlatLayout(c)
        params = initialize(c, self.lib) if params is None else params
        self.w = torch.from_numpy(self.layout.pack(params)).to(self.dev)
        self.wb = torch.empty(self.layout.total, dtype=torch.bfloat16, device=self.dev)
        call("sj_cast", _ptr(self.w), SJ_F32, _ptr(self.wb), SJ_BF16, self.layout.total, self._stream())
        self.s = s = global_stage(c)
        d, f, cq, rows = s.width, s.ffn, s.qkv_width, max(L, B)
        f32 = torch.float32
        e = lambda *shape, dt=torch.bfloat16: torch.empty(*shape, dtype=dt, device=self.dev)  # noqa: E731
        z = lambda *shape, dt=torch.int32: torch.zeros(*shape, dtype=dt, device=self.dev)  # noqa: E731
        # caches: heads outermost inside a page, so a page of a head is one run of memory
        self.k, self.v = (e(s.layers, self.pages, s.kv_heads, P, HEAD_DIM) for _ in range(2))
        self.strides = self.k.stride()[1:4]
        self.rope = e(L * HEAD_DIM, dt=f32)
        if rope_scaling is None:
            call("sj_rope_table", _ptr(self.rope), L, HEAD_DIM, 0, float(c.rope_theta), self._stream())
        else:
            call("sj_rope_table_scaled", _ptr(self.rope), L, HEAD_DIM, 0, float(c.rope_theta), rope_scaling.code(),
                 float(rope_scaling.factor), int(rope_scaling.original), float(rope_scaling.fast),
                 float(rope_scaling.slow), self._stream())
        self.x, self.x1 = e(rows, d, dt=f32), e(rows, d, dt=f32)
        self.z, self.qkv, self.o = e(rows, d), e(rows, cq), e(rows, d)
        self.gu, self.h = e(rows, 2 * f), e(rows, f)
        self.inv, self.lse = e(rows, dt=f32), e(rows * s.heads, dt=f32)
        self.logits = e(B, VOCAB_PAD, dt=f32)
        # what the host writes for a step: tokens added, requests to release, token ids
        self.host = torch.zeros(2 * B + rows, dtype=torch.int32, pin_memory=True)
        self.input = z(2 * B + rows)
        self.added, self.release, self.ids = self.input[:B], self.input[B:2 * B], self.input[2 * B:]
        self.lengths, self.summary = z(B), z(4)
        self.planned = torch.zeros(4, dtype=torch.int32, pin_memory=True)  # the host's copy of the summary
        # the cache's books in one buffer, so that they are replaced as a whole
        self.state = z(B + B * self.width + 2 * self.pages + 1)
        self.cached, self.table, self.shares, self.free, self.free_count = self._books(self.state)
        self.table.fill_(-1)
        torch.arange(self.pages, out=self.free)
        self.free_count.fill_(self.pages)
        self.spare = None  # what sharing needs, made when it is first used
        self.shared_graph = None
        self.request, self.position, self.slot = z(rows), z(rows), z(rows)
        self.work = z(self.lib.sj_attn_paged_workspace(B, s.heads, s.kv_heads, HEAD_DIM), dt=torch.uint8)
        self.score_work = z(self.lib.sj_token_scores_workspace(rows, VOCAB, 32), dt=torch.uint8)
        self.graph = None
        self.slots = [None] * B
        self.finished = set()
        self.reserved = 0
        torch.cuda.current_stream(self.dev).synchronize()  # calls run on whichever stream is current then

    def default_pages(self):
        """As many as a whole batch of full contexts holds, and as a fork of it takes before it returns others."""
        return self.batch * self.width + self.batch - 1

    def _books(self, state):
        B, W, N = self.batch, self.width, self.pages
        parts = torch.split(state, [B, B * W, N, N, 1])
        return parts[0], parts[1].view(B, W), *parts[2:]

    # ---------------------------------------------------------------- kernels
    def _stream(self):
        return torch.cuda.current_stream(self.dev).cuda_stream

    def _wb(self, name):
        return _ptr(self.wb, self.layout[name].offset)

    def _gemm(self, a, lda, b, ldb, c, ldc, c_dtype, m, n, k, epi=EPI_STORE, aux=0, ld_aux=0, rope_cols=0, rope_t=0):
        call("sj_gemm", a, lda, 0, b, ldb, 0, c, ldc, c_dtype, m, n, k, epi, 1.0, aux, ld_aux, rope_cols, rope_t,
             float(self.c.rope_theta) if epi == EPI_ROPE else 0.0, 0, self._stream())

    def _norm(self, x, name, rows):
        call("sj_rmsnorm_fwd", _ptr(x), SJ_F32, _ptr(self.w, self.layout[name].offset), _ptr(self.z), _ptr(self.inv),
             rows, self.s.width, float(self.c.norm_epsilon), self._stream())

    def _commit_and_plan(self, rows):
        call("sj_paged_commit", _ptr(self.cached), _ptr(self.lengths), _ptr(self.release), self.batch, self.page,
             _ptr(self.table), self.width, _ptr(self.free), _ptr(self.free_count), self.pages, _ptr(self.summary),
             self._stream())
        call("sj_paged_plan", _ptr(self.cached), _ptr(self.added), self.batch, self.page, _ptr(self.free),
             _ptr(self.free_count), _ptr(self.table), self.width, _ptr(self.lengths), _ptr(self.request),
             _ptr(self.position), _ptr(self.slot), rows, _ptr(self.summary), self._stream())

    def _append(self, layer, qkv, rows, hq, rope_dim, q):
        s = self.s
        call("sj_paged_append", qkv, s.qkv_width, _ptr(self.position), _ptr(self.slot), rows, hq, s.kv_heads, HEAD_DIM,
             _ptr(self.rope), self.context, rope_dim, 0, q, s.qkv_width, _ptr(self.k[layer]), _ptr(self.v[layer]),
             self.pages, self.page, *self.strides, self._stream())

    def _blocks(self, rows, attend):
        """The blocks on x [rows, width]; attend(layer) goes from the normalised rows in z to o."""
        s = self.s
        d, f = s.width, s.ffn
        for i in range(s.layers):
            p = f"{s.prefix}.{i}"
            self._norm(self.x, f"{p}.attention_norm", rows)
            attend(i, p)
            self._gemm(_ptr(self.o), d, self._wb(f"{p}.attention_output"), d, _ptr(self.x1), d, SJ_F32, rows, d, d,
                       EPI_RESIDUAL, aux=_ptr(self.x), ld_aux=d)
            self._norm(self.x1, f"{p}.ffn_norm", rows)
            self._gemm(_ptr(self.z), d, self._wb(f"{p}.gate_up"), 2 * f, _ptr(self.gu), 2 * f, SJ_BF16, rows, 2 * f, d,
                       EPI_SWIGLU, aux=_ptr(self.h), ld_aux=f)
            self._gemm(_ptr(self.h), f, self._wb(f"{p}.down"), d, _ptr(self.x), d, SJ_F32, rows, d, f, EPI_RESIDUAL,
                       aux=_ptr(self.x1), ld_aux=d)
        self._norm(self.x, "final_norm", rows)

    def _embed(self, rows):
        call("sj_embedding_fwd", self._wb("embedding"), _ptr(self.ids), _ptr(self.x), SJ_F32, rows, self.s.width, VOCAB,
             self._stream())

    def _head(self, first, rows, out):
        d = self.s.width
        self._gemm(_ptr(self.z, first * d), d, self._wb("output"), VOCAB_PAD, _ptr(out), VOCAB_PAD, SJ_F32, rows, VOCAB,
                   d)

    def _prompt(self, n, file):
        """Rows 0 .. n - 1 at positions 0 .. n - 1 through the blocks; their keys and values filed when `file`."""
        s = self.s
        d, cq, kq, vq = s.width, s.qkv_width, s.heads * HEAD_DIM, (s.heads + s.kv_heads) * HEAD_DIM

        def attend(i, p):
            self._gemm(_ptr(self.z), d, self._wb(f"{p}.qkv"), cq, _ptr(self.qkv), cq, SJ_BF16, n, cq, d, EPI_ROPE,
                       aux=_ptr(self.rope), rope_cols=vq, rope_t=self.context)
            if file:  # rotated by the epilogue: keys and values only
                self._append(i, _ptr(self.qkv, kq), n, 0, 0, 0)
            call("sj_attn_gqa_fwd", _ptr(self.qkv), cq, _ptr(self.qkv, kq), cq, _ptr(self.qkv, vq), cq, _ptr(self.o), d,
                 _ptr(self.lse), 1, n, s.heads, s.kv_heads, HEAD_DIM, s.window, self._stream())

        self._embed(n)
        self._blocks(n, attend)

    def _decode(self):
        """One step of every live request: `batch` rows, those past the live ones empty."""
        s, B = self.s, self.batch
        d, cq = s.width, s.qkv_width

        def attend(i, p):
            self._gemm(_ptr(self.z), d, self._wb(f"{p}.qkv"), cq, _ptr(self.qkv), cq, SJ_BF16, B, cq, d)
            self._append(i, _ptr(self.qkv), B, s.heads, HEAD_DIM, _ptr(self.qkv))
            call("sj_attn_paged", _ptr(self.qkv), cq, _ptr(self.k[i]), _ptr(self.v[i]), self.pages, self.page,
                 *self.strides, _ptr(self.table), self.width, B, _ptr(self.request), _ptr(self.position), B, s.heads,
                 s.kv_heads, HEAD_DIM, s.window, _ptr(self.o), d, 0, _ptr(self.work), self.work.numel(), self._stream())

        self._commit_and_plan(B)
        self._embed(B)
        self._blocks(B, attend)
        self._head(0, B, self.logits)

    # ---------------------------------------------------------------- steps
    def _clear(self):
        """An empty cache without requests, whatever a call that was broken off has left."""
        self.slots = [None] * self.batch
        self.finished.clear()
        self.reserved = 0
        for t in (self.cached, self.lengths, self.summary, self.shares):
            t.zero_()
        self.table.fill_(-1)
        torch.arange(self.pages, out=self.free)
        self.free_count.fill_(self.pages)
        self._device_error()

    def _device_error(self):
        """The device error word, which is cleared."""
        code = ctypes.c_int(0)
        call("sj_device_error", ctypes.byref(code), 1, self._stream())
        return code.value

    def _write(self, added, ids):
        """The host's part of a step: tokens added by slot, pages to return, token ids of the rows."""
        B = self.batch
        torch.cuda.current_stream(self.dev).synchronize()  # the last step's copy has been read
        host = self.host.numpy()
        host[:2 * B + self.batch] = 0
        for b, n in added.items():
            host[b] = n
        for b in self.finished:
            host[B + b] = 1
        self.finished.clear()
        host[2 * B:2 * B + len(ids)] = ids
        used = 2 * B + max(len(ids), B)
        self.input[:used].copy_(self.host[:used], non_blocking=True)

    def _start(self, slot, tokens):
        """A prompt (or the tail of a full context) into an empty slot; its last row's logits are row 0."""
        self._write({slot: len(tokens)}, tokens)
        self._commit_and_plan(len(tokens))
        self._prompt(len(tokens), True)
        self._head(len(tokens) - 1, 1, self.logits)
        self.slots[slot].length = len(tokens)

    def _step(self, live):
        self._write({b: 1 for b in live}, [self.slots[b].tokens[-1] for b in live])
        if self.graph is None:
            self._decode()  # what a first call sets up is not captured; the captured step runs from the next one on
            torch.cuda.current_stream(self.dev).synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                self._decode()
            self.graph = graph
        else:
            self.graph.replay()
        for b in live:
            self.slots[b].length += 1

    def _scores(self, logits, targets, top):
        """Scores of the targets under rows of logits (device), as lists on the host."""
        n = len(targets)
        target = torch.tensor(targets, dtype=torch.int32).to(self.dev)
        stats = torch.empty(2, n, dtype=torch.float32, device=self.dev)
        ids = torch.empty(n, top, dtype=torch.int32, device=self.dev)
        best = torch.empty(n, top, dtype=torch.float32, device=self.dev)
        call("sj_token_scores", _ptr(logits), SJ_F32, VOCAB_PAD, _ptr(target), n, VOCAB, top, _ptr(stats[0]),
             _ptr(stats[1]), 0, _ptr(ids), _ptr(best), _ptr(self.score_work), self.score_work.numel(), self._stream())
        logp, entropy = stats.cpu().numpy()
        ids, best = ids.cpu().numpy(), best.cpu().numpy()
        pairs = [[(int(t), float(p)) for t, p in zip(a, b)] for a, b in zip(ids, best)]
        return Scores([float(v) for v in logp], [float(v) for v in entropy], pairs)

    def _draw(self, slots, top):
        """A byte for each of the slots from its row of logits; finished requests leave.  Returns what finished."""
        self.planned.copy_(self.summary, non_blocking=True)  # here when the logits are
        logits = self.logits[:len(slots), :VOCAB].cpu().numpy()
        status = int(self.planned[2])
        if status:
            raise RuntimeError(f"a step could not be planned: status {status}")
        tokens = [sample(logits[r], self.slots[b].options, self.slots[b].state) for r, b in enumerate(slots)]
        scores = None if top is None else self._scores(self.logits, tokens, top)
        done = []
        for r, b in enumerate(slots):
            q = self.slots[b]
            if scores is not None:
                q.scores.logp.append(scores.logp[r])
                q.scores.entropy.append(scores.entropy[r])
                q.scores.alternatives.append(scores.alternatives[r])
            ended = tokens[r] == EOS
            if not ended:
                q.out.append(tokens[r])
                q.tokens.append(tokens[r])
            if ended or len(q.out) >= q.options.max_bytes:
                done.append((q.index, Completion(bytes(q.out), ended, q.scores)))
                self.slots[b] = None
                self.finished.add(b)
                self.reserved -= q.reserved
        return done

    # ---------------------------------------------------------------- requests that share pages
    def _share(self):
        """Buffers of steps whose requests share pages."""
        if self.spare is not None:
            return
        B, s = self.batch, self.s
        z = lambda *shape, dt=torch.int32: torch.zeros(*shape, dtype=dt, device=self.dev)  # noqa: E731
        spare = torch.full_like(self.state, -1)
        self.spare_books = self._books(spare)
        # what the host writes for a step: tokens added, token ids, parents, groups (first row, request, tokens)
        self.shared_host = torch.zeros(6 * B, dtype=torch.int32, pin_memory=True)
        self.shared_input = z(6 * B)
        self.shared_added, self.shared_ids, self.parent, self.group = torch.split(self.shared_input, [B, B, B, 3 * B])
        self.copies, self.forked = z(B, 3), z(4)
        self.shared_planned = torch.zeros(8, dtype=torch.int32, pin_memory=True)
        self.shared_work = z(self.lib.sj_attn_paged_shared_workspace(B, B, s.heads, s.kv_heads, HEAD_DIM), dt=torch.uint8)
        self.spare = spare

    def _fork_and_plan(self, rows):
        B, P, W = self.batch, self.page, self.width
        call("sj_paged_commit", _ptr(self.cached), _ptr(self.lengths), 0, B, P, _ptr(self.table), W, _ptr(self.free),
             _ptr(self.free_count), self.pages, _ptr(self.summary), self._stream())
        cached, table, shares, free, count = self.spare_books
        call("sj_paged_fork", _ptr(self.parent), B, P, _ptr(self.cached), _ptr(self.table), W, _ptr(self.shares),
             _ptr(self.free), _ptr(self.free_count), self.pages, _ptr(cached), _ptr(table), _ptr(shares), _ptr(free),
             _ptr(count), _ptr(self.copies), _ptr(self.forked), self._stream())
        self.state.copy_(self.spare)
        call("sj_paged_copy", _ptr(self.copies), B, _ptr(self.k), _ptr(self.v), self.s.layers, self.k.stride(0), self.pages,
             P, *self.strides, self.s.kv_heads, HEAD_DIM, self._stream())
        call("sj_paged_plan", _ptr(self.cached), _ptr(self.shared_added), B, P, _ptr(self.free), _ptr(self.free_count),
             _ptr(self.table), W, _ptr(self.lengths), _ptr(self.request), _ptr(self.position), _ptr(self.slot), rows,
             _ptr(self.summary), self._stream())

    def _decode_shared(self):
        """As _decode, after a fork of the requests, for rows that share keys."""
        s, B = self.s, self.batch
        d, cq = s.width, s.qkv_width

        def attend(i, p):
            self._gemm(_ptr(self.z), d, self._wb(f"{p}.qkv"), cq, _ptr(self.qkv), cq, SJ_BF16, B, cq, d)
            self._append(i, _ptr(self.qkv), B, s.heads, HEAD_DIM, _ptr(self.qkv))
            call("sj_attn_paged_shared", _ptr(self.qkv), cq, _ptr(self.k[i]), _ptr(self.v[i]), self.pages, self.page,
                 *self.strides, _ptr(self.table), self.width, B, _ptr(self.request), _ptr(self.position), B,
                 _ptr(self.group), B, s.heads, s.kv_heads, HEAD_DIM, s.window, _ptr(self.o), d, 0, _ptr(self.shared_work),
                 self.shared_work.numel(), self._stream())

        self._fork_and_plan(B)
        call("sj_embedding_fwd", self._wb("embedding"), _ptr(self.shared_ids), _ptr(self.x), SJ_F32, B, s.width, VOCAB,
             self._stream())
        self._blocks(B, attend)
        self._head(0, B, self.logits)

    def _write_shared(self, parents, added, ids=(), groups=()):
        """The host's part of a step.  `added`: tokens by slot; `groups`: (first row, slot, tokens in common)."""
        B = self.batch
        torch.cuda.current_stream(self.dev).synchronize()  # the last step's copy has been read
        host = self.shared_host.numpy()
        host[:2 * B] = 0
        for b, n in added.items():
            host[b] = n
        host[B:B + len(ids)] = ids
        host[2 * B:3 * B] = parents
        rows = host[3 * B:].reshape(B, 3)
        rows[:] = (B, 0, 0)  # an empty group
        rows[:len(groups)] = np.asarray(groups, dtype=np.int32).reshape(-1, 3)
        self.shared_input.copy_(self.shared_host, non_blocking=True)

    def _start_shared(self, slot, tokens, pending):
        """A prompt into a slot that is empty or has finished; its last row's logits are row 0.  `pending`: the next step's
        parents, whose pages stay until then."""
        gone = self.finished - {p for b, p in enumerate(pending) if p != b}
        self.finished -= gone
        self._write_shared([-1 if b in gone else b for b in range(self.batch)], {slot: len(tokens)})
        self.ids[:len(tokens)].copy_(torch.tensor(tokens, dtype=torch.int32))
        self._fork_and_plan(len(tokens))
        self._prompt(len(tokens), True)
        self._head(len(tokens) - 1, 1, self.logits)

    def _step_shared(self, parents, live, ids, common):
        """One step of the live slots, slot b going on from what parents[b] holds; common[b]: (block, tokens) that its
        neighbours of the same block share."""
        groups, last = [], None
        for r, b in enumerate(live):
            if common[b] is None or common[b] != last:
                groups.append((r, b, 0 if common[b] is None else common[b][1]))
            last = common[b]
        for b in self.finished:
            parents[b] = -1
        self.finished.clear()
        self._write_shared(parents, {b: 1 for b in live}, ids, groups)
        if self.shared_graph is None:
            self._decode_shared()  # what a first call sets up is not captured
            torch.cuda.current_stream(self.dev).synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                self._decode_shared()
            self.shared_graph = graph
        else:
            self.shared_graph.replay()

    def _check_shared(self):
        """After the step's results have been waited for."""
        self.shared_planned[:4].copy_(self.summary)
        self.shared_planned[4:].copy_(self.forked)
        status, forked = int(self.shared_planned[2]), int(self.shared_planned[6])
        if status or forked:
            raise RuntimeError(f"a step could not be planned: status {status}, of the fork {forked}")

    def _check_sharing(self):
        """Before a call stages anything: a cache whose pages can be shared."""
        if self.pages > SHARED_PAGES:
            raise ValueError(f"several continuations of a prompt take a cache of at most {SHARED_PAGES} pages, not {self.pages}")

    def _reserve(self, tokens, most_bytes, count, forks):
        """Pages that `count` continuations of a prompt may come to need: its full pages once, the rest for each; all of them
        for each where a full context may start again.  `forks`: those of a beam search, whose forks copy half-filled pages
        for all but one before they return others; the copies of samples, made once, are pages that they go on to fill."""
        most = -(-min(self.context, len(tokens) + most_bytes) // self.page)
        shared = len(tokens) // self.page if len(tokens) + most_bytes <= self.context else 0
        pages = shared + count * (most - shared) + (count - 1 if forks else 0)
        if pages > self.pages:
            raise ValueError(f"{count} continuations of a prompt may need {pages} pages of a cache of {self.pages}")
        return pages

    def _run_samples(self, waiting, count, top):
        """`count` continuations of each prompt: (tokens, options, reserved) in, lists of completions out."""
        results = [[None] * count for _ in waiting]
        blocks = [None] * (self.batch // count)  # slots b * count .. of a prompt
        todo = deque(enumerate(waiting))
        parents, ids, common = list(range(self.batch)), {}, [None] * self.batch
        left = {}  # pages and continuations of a block

        def draw(slots, rows):
            """A byte for each slot from a row of logits; finished ones leave."""
            logits = self.logits[:max(rows) + 1, :VOCAB].cpu().numpy()
            self._check_shared()
            tokens = [sample(logits[r], self.slots[b].options, self.slots[b].state) for b, r in zip(slots, rows)]
            scores = None
            if top is not None:
                scores = self._scores(self.logits[torch.tensor(rows, device=self.dev)], tokens, top)
            for i, (b, token) in enumerate(zip(slots, tokens)):
                q = self.slots[b]
                if scores is not None:
                    q.scores.logp.append(scores.logp[i])
                    q.scores.entropy.append(scores.entropy[i])
                    q.scores.alternatives.append(scores.alternatives[i])
                if token != EOS:
                    q.out.append(token)
                    q.tokens.append(token)
                if token == EOS or len(q.out) >= q.options.max_bytes:
                    results[q.index][b % count] = Completion(bytes(q.out), token == EOS, q.scores)
                    self.slots[b], parents[b] = None, b
                    self.finished.add(b)
                    left[b // count][1] -= 1
                    if left[b // count][1] == 0:
                        self.reserved -= left.pop(b // count)[0]
                        blocks[b // count] = None
                else:
                    ids[b] = token

        while todo or left:
            for n, block in enumerate(blocks):
                if block is None and todo and self.reserved + todo[0][1][2] <= self.pages:
                    index, (tokens, options, reserved) = todo.popleft()
                    blocks[n], left[n] = index, [reserved, count]
                    self.reserved += reserved
                    first = n * count
                    self._start_shared(first, tokens, parents)
                    for b in range(first, first + count):
                        state = ctypes.c_uint64((int(options.seed) + b - first) & (2**64 - 1))
                        self.slots[b] = _Request(index, list(tokens), options, state, 0, len(tokens),
                                                 scores=None if top is None else Scores())
                        parents[b], common[b] = first, (n, len(tokens))
                    draw(list(range(first, first + count)), [0] * count)
            for b, q in enumerate(self.slots):
                if q is not None and q.length == self.context:  # a full context starts again from its tail, by itself
                    self.finished.add(b)
                    tail = q.tokens[-self.context:]
                    self._start_shared(b, tail, parents)
                    q.length, common[b] = len(tail), None
                    draw([b], [0])
            live = [b for b, q in enumerate(self.slots) if q is not None and q.length < self.context]
            if live:
                self._step_shared(parents, live, [ids[b] for b in live], common)
                parents[:] = range(self.batch)
                for b in live:
                    self.slots[b].length += 1
                draw(live, list(range(len(live))))
        return results

    def _select(self, rows, scores, beams, keep):
        """(parent, token, score) [requests, keep] of the first rows of logits and the beams' scores."""
        requests = rows // beams
        score = torch.tensor(scores, dtype=torch.float32).to(self.dev)
        ids = torch.empty(2, requests, keep, dtype=torch.int32, device=self.dev)
        best = torch.empty(requests, keep, dtype=torch.float32, device=self.dev)
        size = self.lib.sj_beam_select_workspace(requests, beams, VOCAB, keep)
        work = torch.zeros(max(size, 1), dtype=torch.uint8, device=self.dev)
        call("sj_beam_select", _ptr(self.logits), SJ_F32, VOCAB_PAD, _ptr(score), requests, beams, VOCAB, keep, _ptr(ids[0]),
             _ptr(ids[1]), _ptr(best), _ptr(work), work.numel(), self._stream())
        parent, token = ids.cpu().tolist()
        self._check_shared()
        return parent, token, best.cpu().tolist()

    def _run_beams(self, waiting, beams, most_bytes, penalty):
        results = [None] * len(waiting)
        blocks = [None] * (self.batch // beams)
        todo = deque(waiting)
        parents, ids = list(range(self.batch)), {}

        def rank(score, length):
            return score / max(length, 1) ** penalty

        def advance(n, parent, token, score):
            """The best continuations of a block's beams: those that end are kept aside, the others go on."""
            q, first, live = blocks[n], n * beams, []
            for at, (p, t, total) in enumerate(zip(parent, token, score)):
                if p < 0 or len(live) == beams:
                    break
                drawn = q.live[p][0]
                if t == EOS:
                    if at < beams:
                        q.ended.append(Hypothesis(bytes(drawn), True, total, rank(total, len(drawn) + 1)))
                    continue
                parents[first + len(live)], ids[first + len(live)] = first + p, t
                live.append((drawn + [t], total))
            q.ended.sort(key=lambda h: -h.ranked)
            del q.ended[beams:]
            q.live = live
            length = len(live[0][0]) if live else 0
            # what goes on can come to be worth no more than its score at the length that is best for it: the largest, or
            # where a greater length makes less of it, the next one, by an end
            hope = max((max(rank(s, length + 1), rank(s, most_bytes)) for _, s in live), default=-float("inf"))
            done = not live or length >= most_bytes or (len(q.ended) == beams and q.ended[-1].ranked >= hope)
            if done:
                whole = length >= most_bytes
                rest = [Hypothesis(bytes(d), False, s, rank(s, len(d))) for d, s in live if whole]
                results[q.index] = sorted(q.ended + rest, key=lambda h: -h.ranked)[:beams]
                blocks[n] = None
                self.reserved -= q.reserved
                parents[first:first + beams] = range(first, first + beams)
                self.finished.update(range(first, first + beams))
            else:
                for b in range(first + len(live), first + beams):  # fewer tokens are allowed than there are beams
                    parents[b], ids[b] = first, live[0][0][-1]
                q.live += [(live[0][0], -float("inf"))] * (beams - len(live))

        while todo or any(q is not None for q in blocks):
            for n in range(len(blocks)):
                if blocks[n] is None and todo and self.reserved + todo[0].reserved <= self.pages:
                    blocks[n] = q = todo.popleft()
                    self.reserved += q.reserved
                    self._start_shared(n * beams, q.tokens, parents)
                    q.live = [([], 0.0)]
                    found = self._select(1, [0.0], 1, min(2 * beams, VOCAB))
                    advance(n, *(f[0] for f in found))
            running = [n for n, q in enumerate(blocks) if q is not None]
            if not running:
                continue
            live = [n * beams + i for n in running for i in range(beams)]
            common = [None] * self.batch
            for b in live:
                common[b] = (b // beams, len(blocks[b // beams].tokens))
            self._step_shared(parents, live, [ids[b] for b in live], common)
            parents[:] = range(self.batch)
            scores = [s for n in running for _, s in blocks[n].live]
            found = self._select(len(live), scores, beams, 2 * beams)
            for i, n in enumerate(running):
                advance(n, *(f[i] for f in found))
        return results

    def _guard(self, run, *args):
        """run(*args), which leaves no requests behind, whether it ends or raises."""
        try:
            self._share()
            results = run(*args)
            code = self._device_error()
            if code:
                raise RuntimeError(f"device error {code} during generation")
        except BaseException:
            self._clear()
            raise
        self._clear()  # pages that were shared are counted anew
        return results

    def beam_search(self, prompts, beams=4, max_bytes=64, length_penalty=1.0):
        """For each prompt the `beams` best continuations found (Hypothesis, the best first): those that end, or have
        `max_bytes` bytes, ordered by their log probability over length ** length_penalty (an end counts as a byte).  The
        search stops early only where no beam can come to be worth more."""
        if not 1 <= beams <= min(self.batch, 32):
            raise ValueError("beams must be 1 to 32, and at most the batch")
        if max_bytes < 1:
            raise ValueError("max_bytes must be positive")
        if not abs(float(length_penalty)) <= 50:  # nor NaN; a length to a much larger power leaves f64
            raise ValueError("the length penalty must be -50 to 50")
        self._check_sharing()
        waiting = []
        for i, prompt in enumerate(prompts):
            tokens = [EOS] + list(bytes(prompt))
            if len(tokens) + max_bytes > self.context:
                raise ValueError("a prompt and its continuations have to fit the context")
            waiting.append(_Beams(i, tokens, self._reserve(tokens, max_bytes, beams, True)))
        return self._guard(self._run_beams, waiting, beams, max_bytes, float(length_penalty))

    def _admit(self, index, prompt, options, top):
        tokens = ([EOS] + list(bytes(prompt)))[-self.context:]
        most = min(self.context, len(tokens) + options.max_bytes)
        return _Request(index, tokens, options, ctypes.c_uint64(int(options.seed) & (2**64 - 1)), -(-most // self.page),
                        scores=None if top is None else Scores())

    def generate(self, prompts, options=None, top=None, samples=1):
        """Completions of the prompts (bytes), in their order.  `options`: one Sampling for all, or one each.
        `top`: None for no scores, else how many alternatives (0 to 32) beside each drawn token's.  `samples` > 1: a
        list of that many completions for each prompt, drawn with its seed, its seed + 1, ...; they share its pages."""
        if options is None or isinstance(options, Sampling):
            options = [options or Sampling()] * len(prompts)
        if len(options) != len(prompts):
            raise ValueError("one Sampling for all prompts, or one for each")
        if top is not None and not 0 <= top <= 32:
            raise ValueError("top must be 0 to 32")
        if not 1 <= samples <= self.batch:
            raise ValueError("samples must be 1 to the batch")
        if samples > 1:
            self._check_sharing()
            shared = []
            for prompt, o in zip(prompts, options):
                if o.max_bytes < 1:
                    raise ValueError("max_bytes must be positive")
                check_sampling(o)
                tokens = ([EOS] + list(bytes(prompt)))[-self.context:]
                if len(tokens) == self.context:
                    raise ValueError("a prompt that fills the context cannot be shared")
                shared.append((tokens, o, self._reserve(tokens, o.max_bytes, samples, False)))
            return self._guard(self._run_samples, shared, samples, top)
        waiting = deque(self._admit(i, p, o, top) for i, (p, o) in enumerate(zip(prompts, options)))
        for q in waiting:
            if q.reserved > self.pages:
                raise ValueError(f"a request may need {q.reserved} pages of a cache of {self.pages}")
            if q.options.max_bytes < 1:
                raise ValueError("max_bytes must be positive")
            check_sampling(q.options)
        try:
            return self._run(waiting, top)
        except BaseException:
            self._clear()
            raise

    def _run(self, waiting, top):
        """The completions of the waiting requests, in the order of their indices."""
        results = [None] * len(waiting)

        def take(done):
            for i, completion in done:
                results[i] = completion

        while waiting or any(q is not None for q in self.slots):
            for b in range(self.batch):
                if self.slots[b] is None and waiting and self.reserved + waiting[0].reserved <= self.pages:
                    self.slots[b] = q = waiting.popleft()
                    self.reserved += q.reserved
                    self._start(b, q.tokens)
                    take(self._draw([b], top))
            for b, q in enumerate(self.slots):
                if q is not None and q.length == self.context:  # a full context starts again from its tail
                    self.finished.add(b)
                    self._start(b, q.tokens[-self.context:])
                    take(self._draw([b], top))
            live = [b for b, q in enumerate(self.slots) if q is not None and q.length < self.context]
            if live:
                self._step(live)
                take(self._draw(live, top))
        code = self._device_error()
        if code:
            raise RuntimeError(f"device error {code} during generation")
        return results

    def score(self, text, top=0):
        """Scores of each byte of `text` after EOS and the bytes before it."""
        tokens = [EOS] + list(bytes(text))
        if len(tokens) > self.context + 1:
            raise ValueError("the text is longer than the context")
        if not 0 <= top <= 32:
            raise ValueError("top must be 0 to 32")
        n = len(tokens) - 1
        if n == 0:
            return Scores()
        torch.cuda.current_stream(self.dev).synchronize()
        self.ids[:n].copy_(torch.tensor(tokens[:n], dtype=torch.int32))
        self._prompt(n, False)
        logits = torch.empty(n, VOCAB_PAD, dtype=torch.float32, device=self.dev)
        self._head(0, n, logits)
        return self._scores(logits, tokens[1:], top)
