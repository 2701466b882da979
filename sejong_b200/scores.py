"""Differentiable token scores for training on log probabilities and entropies (policy gradients, distillation):
`token_scores` on torch tensors, through sj_token_scores and sj_token_scores_bwd."""
from typing import NamedTuple

import torch

from . import _lib
from ._lib import SJ_BF16, SJ_F32, call

_DTYPES = {torch.float32: SJ_F32, torch.bfloat16: SJ_BF16}


class TokenScores(NamedTuple):
    logp: torch.Tensor      # f32 [rows], differentiable
    entropy: torch.Tensor   # f32 [rows], differentiable
    top_id: torch.Tensor    # int32 [rows, top]
    top_logp: torch.Tensor  # f32 [rows, top], not differentiated


def _row_stride(logits):
    """Of rows that token_scores has seen to; one row has any."""
    return logits.stride(0) if logits.shape[0] > 1 else logits.shape[1]


def _stream(t):
    return torch.cuda.current_stream(t.device).cuda_stream


class _Undifferentiable(torch.autograd.Function):
    """The gradient as it is, a function of `inputs` whose own derivative is an error.  (A backward that is marked as
    once differentiable leaves out in silence what it depends on through the saved logits.)"""
    @staticmethod
    def forward(ctx, gradient, *inputs):
        return gradient.view_as(gradient)

    @staticmethod
    def backward(ctx, _):
        raise RuntimeError("the gradient of token_scores has no derivative")


class _Scores(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, top):
        rows, vocab = logits.shape
        dev = logits.device
        logp, entropy, lse = (torch.empty(rows, dtype=torch.float32, device=dev) for _ in range(3))
        ids = torch.empty(rows, top, dtype=torch.int32, device=dev)
        best = torch.empty(rows, top, dtype=torch.float32, device=dev)
        with torch.cuda.device(dev):  # the library works on the current one
            size = max(_lib.load().sj_token_scores_workspace(rows, vocab, top), 1)
            work = torch.zeros(size, dtype=torch.uint8, device=dev)
            call("sj_token_scores", logits.data_ptr(), _DTYPES[logits.dtype], _row_stride(logits), targets.data_ptr(),
                 rows, vocab, top, logp.data_ptr(), entropy.data_ptr(), lse.data_ptr(), ids.data_ptr(),
                 best.data_ptr(), work.data_ptr(), size, _stream(logits))
        ctx.save_for_backward(logits, targets, lse, entropy)
        ctx.mark_non_differentiable(ids, best)
        return logp, entropy, ids, best

    @staticmethod
    def backward(ctx, d_logp, d_entropy, _ids, _best):
        logits, targets, lse, entropy = ctx.saved_tensors
        rows, vocab = logits.shape
        d_logp, d_entropy = d_logp.float().contiguous(), d_entropy.float().contiguous()
        out = torch.empty(rows, vocab, dtype=logits.dtype, device=logits.device)
        with torch.cuda.device(logits.device):
            call("sj_token_scores_bwd", logits.data_ptr(), _DTYPES[logits.dtype], _row_stride(logits),
                 targets.data_ptr(), rows, vocab, lse.data_ptr(), entropy.data_ptr(), d_logp.data_ptr(),
                 d_entropy.data_ptr(), out.data_ptr(), vocab, _stream(logits))
        if torch.is_grad_enabled():  # a graph of the gradient is asked for
            out = _Undifferentiable.apply(out, logits, d_logp, d_entropy)
        return out, None, None


def token_scores(logits, targets, top=0):
    """Log probability of targets[r] (int32; -1: none) and entropy under each row of logits (f32 or bf16 [rows, vocab]
    on the GPU, any row stride), and the `top` best alternatives (0 to 32).  First derivatives only."""
    if logits.dim() != 2 or targets.shape != logits.shape[:1]:
        raise ValueError("logits [rows, vocab] and targets [rows]")
    if logits.dtype not in _DTYPES:
        raise ValueError(f"logits of {logits.dtype}: float32 or bfloat16")
    if not logits.is_cuda or targets.device != logits.device:
        raise ValueError("logits and targets on the same GPU")
    if logits.stride(1) != 1 or (logits.shape[0] > 1 and not logits.shape[1] <= logits.stride(0) < 1 << 31):
        logits = logits.contiguous()
    return TokenScores(*_Scores.apply(logits, targets.to(torch.int32).contiguous(), top))
