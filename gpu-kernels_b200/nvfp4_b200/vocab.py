"""The two ends of a model that share its vocabulary: rows of an embedding table by token id,
and log probabilities of tokens from rows of logits, with their gradients.  torch tensors in,
kernels of libnvfp4_b200.so underneath; asynchronous on torch's current stream of the tensors'
device.  ValueError for arguments of the wrong shape, type or device, NVFP4Error for a bad
status.

    x = embedding(tokens, table, scale=K ** 0.5)
    logits = linear(h, table)                                  # a tied output projection
    r = token_logprobs(logits, targets, top_k=5, entropy=True)
    dlogits = token_logprobs_backward(dlogprobs, logits, targets, r, dentropy=dentropy)

These functions record no autograd graph; the operators of the same names in
torch.ops.nvfp4_b200 do.
"""
from typing import NamedTuple, Optional

import torch

from ._bind import native


def embedding(tokens: torch.Tensor, table: torch.Tensor, scale: float = 1.0) -> torch.Tensor:
    """scale * table[tokens], rounded once (scale 1 copies the bits).

    tokens int32 or int64 of any shape, contiguous; table [V, K] bf16 or fp16 (rows may be a slice of wider
    ones, 16-byte aligned; K a multiple of 8); the result is tokens.shape + [K].  A token
    outside [0, V), such as the -1 of padding, gives zeros."""
    return native.embedding(tokens, table, scale)


def embedding_backward(dy: torch.Tensor, tokens: torch.Tensor, rows: int, scale: float = 1.0) -> torch.Tensor:
    """Gradient [rows, K] of the table: scale * the sum of dy over equal tokens, in fp32 and in
    an order that the tokens and the sizes decide, rounded once; zero for rows that no token names."""
    return native.embedding_backward(dy, tokens, rows, scale)


class TokenLogprobs(NamedTuple):
    """What token_logprobs returns, fp32 [T] unless stated."""
    logprobs: torch.Tensor                # log p of the targets, 0 for an ignored one
    entropy: Optional[torch.Tensor]       # of each row's distribution
    top_logprobs: Optional[torch.Tensor]  # [T, top_k], highest first
    top_tokens: Optional[torch.Tensor]    # int32 [T, top_k], -1 where fewer tokens are left
    lse: torch.Tensor                     # log sum exp(logits / temperature), for the gradient


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor, vocab: Optional[int] = None, top_k: int = 0,
                   temperature: float = 1.0, entropy: bool = False) -> TokenLogprobs:
    """Log probabilities of targets [T] (int32 or int64) under softmax(logits / temperature),
    in one pass over logits [T, W] (bf16, fp16 or fp32; rows may be a slice of wider ones).

    vocab: the first so many columns are tokens, the others padding.  top_k <= 32: also the
    most probable tokens, the lowest first among equals.  entropy: also each row's entropy.
    A target outside [0, vocab) is ignored: log probability 0.  A logit of -inf or NaN masks
    its token (probability 0, no alternative), finite ones of any size are ordinary; a row with nothing left has log probability
    -inf and entropy 0; a logit of +inf makes its row's results NaN."""
    return TokenLogprobs._make(native.token_logprobs(logits, targets, vocab, top_k, temperature, entropy))


def token_logprobs_backward(dlogprobs: torch.Tensor, logits: torch.Tensor, targets: torch.Tensor,
                            result: TokenLogprobs, dentropy: Optional[torch.Tensor] = None,
                            vocab: Optional[int] = None, temperature: float = 1.0,
                            out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Gradient of the logits [T, W] from those of the log probabilities (fp32 [T]; no effect
    where the target is ignored) and, with dentropy, of the entropies: result is
    token_logprobs(..., the same vocab and temperature), with entropy=True for dentropy.
    Masked tokens and padding columns get zero; the alternatives carry no gradient.  Rows whose
    log sum exp is past 256 in size (64 for fp32 logits) are summed again, for which lse alone
    says too little.
    out: where it goes; it may be the logits themselves."""
    return native.token_logprobs_backward(dlogprobs, dentropy, logits, targets, result[4], result[1], vocab,
                                          temperature, out)
