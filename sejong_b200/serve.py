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
        self.pages = int(pages or B * self.width)
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
        self.k = [e(self.pages, s.kv_heads, P, HEAD_DIM) for _ in range(s.layers)]
        self.v = [e(self.pages, s.kv_heads, P, HEAD_DIM) for _ in range(s.layers)]
        self.strides = self.k[0].stride()[:3]
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
        self.cached, self.lengths, self.summary = z(B), z(B), z(4)
        self.planned = torch.zeros(4, dtype=torch.int32, pin_memory=True)  # the host's copy of the summary
        self.table = torch.full((B, self.width), -1, dtype=torch.int32, device=self.dev)
        self.free = torch.arange(self.pages, dtype=torch.int32, device=self.dev)
        self.free_count = torch.full((1,), self.pages, dtype=torch.int32, device=self.dev)
        self.request, self.position, self.slot = z(rows), z(rows), z(rows)
        self.work = z(self.lib.sj_attn_paged_workspace(B, s.heads, s.kv_heads, HEAD_DIM), dt=torch.uint8)
        self.score_work = z(self.lib.sj_token_scores_workspace(rows, VOCAB, 32), dt=torch.uint8)
        self.graph = None
        self.slots = [None] * B
        self.finished = set()
        self.reserved = 0
        torch.cuda.current_stream(self.dev).synchronize()  # calls run on whichever stream is current then

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
        for t in (self.cached, self.lengths, self.summary):
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

    def _admit(self, index, prompt, options, top):
        tokens = ([EOS] + list(bytes(prompt)))[-self.context:]
        most = min(self.context, len(tokens) + options.max_bytes)
        return _Request(index, tokens, options, ctypes.c_uint64(int(options.seed) & (2**64 - 1)), -(-most // self.page),
                        scores=None if top is None else Scores())

    def generate(self, prompts, options=None, top=None):
        """Completions of the prompts (bytes), in their order.  `options`: one Sampling for all, or one each.
        `top`: None for no scores, else how many alternatives (0 to 32) beside each drawn token's."""
        if options is None or isinstance(options, Sampling):
            options = [options or Sampling()] * len(prompts)
        if len(options) != len(prompts):
            raise ValueError("one Sampling for all prompts, or one for each")
        if top is not None and not 0 <= top <= 32:
            raise ValueError("top must be 0 to 32")
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
