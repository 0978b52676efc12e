"""The operators at the two ends of a model over a vocabulary table.

  token_embedding          rows of the table by token, scaled; differentiable
  token_embedding_grad     the table's gradient, summed by token, the same bits every time
  token_logprobs           log probabilities of given tokens, entropy, top alternatives; differentiable
  token_logprobs_grad      the gradient of the logits from gradients of the first two
  topk_distillation_loss   loss of a student's logits against a teacher's top logits; differentiable
  topk_distillation_step   that loss with the gradient of the logits, in one call

HIP tensors only; calls are asynchronous on the current stream.  float32, float16 and
bfloat16; sums and softmax statistics are in 32 bits.  A token outside the table or the
vocabulary contributes nothing.  Differentiable ones have a backward pass of first order; forward
mode raises.  The same kernels are registered as torch.ops.tbe.*, for HIP tensors alone: those
are not differentiable (their results do not require a gradient) and have no fake kernel for
tracing.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _ext

_NO_PADDING = -1


def _tracks(x: torch.Tensor) -> bool:
    """Whether the call goes through autograd, which refuses a tangent: there is no forward-mode rule."""
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(x).tangent is not None:
        return True
    return x.requires_grad and torch.is_grad_enabled()


# ---------------------------------------------------------------- the table

class _TokenEmbeddingFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weight, token_ids, scale, padding_idx, out_dtype):
        ctx.save_for_backward(token_ids)
        ctx.rest = (weight.shape[0], scale, padding_idx, weight.dtype)
        return _ext.token_embedding(weight, token_ids, scale, out_dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        (token_ids,) = ctx.saved_tensors
        num_rows, scale, padding_idx, dtype = ctx.rest
        return _ext.token_embedding_grad(grad, token_ids, num_rows, scale, padding_idx, dtype), None, None, None, None


def token_embedding(weight: torch.Tensor, token_ids: torch.Tensor, scale: float = 1.0,
                    padding_idx: Optional[int] = None, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """scale * weight[token_ids], in out_dtype (default: the weight's).

    token_ids: int32 or int64, any shape; a token outside the table gives a row of zeros.
    padding_idx: a token whose row gets no gradient (it is looked up like any other).  None or
    a number below 0 is no token: it does not count from the table's end."""
    pad = _NO_PADDING if padding_idx is None else padding_idx
    if _tracks(weight):
        return _TokenEmbeddingFn.apply(weight, token_ids, scale, pad, out_dtype)
    return _ext.token_embedding(weight, token_ids, scale, out_dtype)


def token_embedding_grad(grad_output: torch.Tensor, token_ids: torch.Tensor, num_rows: int, scale: float = 1.0,
                         padding_idx: Optional[int] = None,
                         grad_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """The gradient [num_rows, width] of the table, from that of token_embedding's result
    (padding_idx as there)."""
    return _ext.token_embedding_grad(grad_output, token_ids, num_rows, scale,
                                     _NO_PADDING if padding_idx is None else padding_idx, grad_dtype)


def token_embedding_grad_add_(grad_weight: torch.Tensor, grad_output: torch.Tensor, token_ids: torch.Tensor,
                              scale: float = 1.0, padding_idx: Optional[int] = None) -> torch.Tensor:
    """Adds that gradient to grad_weight: only the rows that a token names are read and
    written (a table tied to the output layer, several batches to one step)."""
    return _ext.token_embedding_grad_add_(grad_weight, grad_output, token_ids, scale,
                                          _NO_PADDING if padding_idx is None else padding_idx)


class TokenEmbedding(torch.nn.Module):
    """A trainable table of token rows: token_embedding with its own weight."""

    def __init__(self, num_rows: int, width: int, scale: float = 1.0, padding_idx: Optional[int] = None,
                 device="cuda", dtype: torch.dtype = torch.float32, out_dtype: Optional[torch.dtype] = None):
        super().__init__()
        self.scale, self.padding_idx, self.out_dtype = float(scale), padding_idx, out_dtype
        self.weight = torch.nn.Parameter(torch.empty(num_rows, width, device=device, dtype=dtype))
        torch.nn.init.normal_(self.weight, std=width ** -0.5)

    def forward(self, token_ids: torch.Tensor) -> torch.Tensor:
        return token_embedding(self.weight, token_ids, self.scale, self.padding_idx, self.out_dtype)


# ---------------------------------------------------------------- log probabilities

class TokenLogprobs(NamedTuple):
    """logprobs has the shape of the given tokens, entropy that of the rows, the top lists
    [..., top_k]; stats is what token_logprobs_grad needs.  top_logprobs carry no gradient."""
    logprobs: torch.Tensor
    entropy: torch.Tensor
    top_logprobs: torch.Tensor
    top_tokens: torch.Tensor
    stats: torch.Tensor


class _TokenLogprobsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, temperature, top_k):
        out = _ext.token_logprobs(logits, tokens, temperature, top_k)
        ctx.save_for_backward(logits, tokens, out[4], out[1])
        ctx.temperature = temperature
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(out[2], out[3], out[4])
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_logprobs, grad_entropy, *_):
        logits, tokens, stats, entropy = ctx.saved_tensors
        return _ext.token_logprobs_grad(logits, tokens, stats, entropy, grad_logprobs, grad_entropy,
                                        ctx.temperature), None, None, None


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, temperature: float = 1.0,
                   top_k: int = 0) -> TokenLogprobs:
    """Log probabilities of `tokens` under softmax(logits / temperature), the entropy of every
    row and its top_k (at most 64) most probable tokens, in one pass over the logits.

    logits: [..., vocabulary], rows at any stride; tokens: [...] or [..., n], n at most 256.
    Equal logits are listed lowest token first.  A row whose logits are all -inf has log
    probabilities -inf, entropy 0 and gradient 0; a given token outside the vocabulary has
    log probability 0 and no gradient."""
    if _tracks(logits):
        return TokenLogprobs(*_TokenLogprobsFn.apply(logits, tokens, temperature, top_k))
    return TokenLogprobs(*_ext.token_logprobs(logits, tokens, temperature, top_k))


def token_logprobs_grad(logits: torch.Tensor, tokens: torch.Tensor, scores: TokenLogprobs,
                        grad_logprobs: Optional[torch.Tensor] = None, grad_entropy: Optional[torch.Tensor] = None,
                        temperature: float = 1.0) -> torch.Tensor:
    """The gradient of the logits from those (float32) of scores.logprobs and scores.entropy,
    where scores = token_logprobs(logits, tokens, temperature)."""
    return _ext.token_logprobs_grad(logits, tokens, scores.stats, scores.entropy, grad_logprobs, grad_entropy,
                                    temperature)


# ---------------------------------------------------------------- distillation

class _TopkDistillFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, teacher_tokens, teacher_values, row_weights, temperature, renormalize):
        loss, stats = _ext.topk_distill_loss(logits, teacher_tokens, teacher_values, row_weights, temperature,
                                             renormalize)
        ctx.save_for_backward(logits, teacher_tokens, teacher_values, row_weights, stats)
        ctx.how = (temperature, renormalize)
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        logits, tokens, values, weights, stats = ctx.saved_tensors
        grad = grad if weights is None else grad * weights
        return _ext.topk_distill_grad(logits, tokens, values, stats, grad, *ctx.how), None, None, None, None, None


def topk_distillation_loss(logits: torch.Tensor, teacher_tokens: torch.Tensor, teacher_values: torch.Tensor,
                           row_weights: Optional[torch.Tensor] = None, temperature: float = 1.0,
                           renormalize: bool = True) -> torch.Tensor:
    """Per row, w T^2 KL(q || softmax(logits / T)) over a teacher's top tokens.

    logits: [..., vocabulary]; teacher_tokens, teacher_values: [..., k], k at most 256, as
    token_logprobs(teacher_logits, ...).top_tokens / .top_logprobs give them; a shorter list
    is filled up with -1.  renormalize: q = softmax(teacher_values / T) over the list;
    otherwise q = exp(teacher_values), the teacher's probabilities as they are.
    row_weights: float32 [...]; a row of weight 0 (padding) is not read.  The teacher and the
    weights are constants: only the logits get a gradient."""
    if _tracks(logits):
        return _TopkDistillFn.apply(logits, teacher_tokens, teacher_values, row_weights, temperature, renormalize)
    return _ext.topk_distill_loss(logits, teacher_tokens, teacher_values, row_weights, temperature, renormalize)[0]


def topk_distillation_step(logits: torch.Tensor, teacher_tokens: torch.Tensor, teacher_values: torch.Tensor,
                           row_weights: Optional[torch.Tensor] = None, temperature: float = 1.0,
                           renormalize: bool = True) -> Tuple[torch.Tensor, torch.Tensor]:
    """topk_distillation_loss and the gradient of its sum with respect to the logits.

    For a training step that knows its row weights beforehand: the logits are read once for
    both where a row fits a work-group's registers."""
    return _ext.topk_distill_step(logits, teacher_tokens, teacher_values, row_weights, temperature, renormalize)


class TopKDistillationLoss(torch.nn.Module):
    """topk_distillation_loss summed over the rows and divided by their weights' sum (or number);
    0 where every row has weight 0."""

    def __init__(self, temperature: float = 1.0, renormalize: bool = True):
        super().__init__()
        self.temperature, self.renormalize = float(temperature), bool(renormalize)

    def forward(self, logits: torch.Tensor, teacher_tokens: torch.Tensor, teacher_values: torch.Tensor,
                row_weights: Optional[torch.Tensor] = None) -> torch.Tensor:
        rows = topk_distillation_loss(logits, teacher_tokens, teacher_values, row_weights, self.temperature,
                                      self.renormalize)
        if row_weights is None:
            return rows.mean()
        total = row_weights.sum()
        return rows.sum() / torch.where(total == 0, 1.0, total)
