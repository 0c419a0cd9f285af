"""Token embedding: the first layer of the reference's prediction network (``nn.Embedding`` at
src/decoder/decoder.py:9) with a scale, and its gradient by sorted tokens.

``rnnt_token_embedding_forward`` / ``_backward`` (include/rnnt_mi355.h) through the compiled binding.  The gradient
sums each token's rows in position order in fp32 and rounds once: two runs give the same bits, and frequent tokens
(the padding of a ragged batch, a vocabulary's common words) cost no more per position than rare ones.
"""
from __future__ import annotations

import math
from typing import Optional

import torch
import torch.nn as nn

from . import _torch_binding


def token_embedding(tokens: torch.Tensor, weight: torch.Tensor, scale: float = 1.0,
                    padding_idx: Optional[int] = None) -> torch.Tensor:
    """``scale * weight[tokens]``, ``[*tokens.shape, dim]`` in ``weight``'s type; differentiable in ``weight`` (once, and not in
    forward mode).

    Args:
        tokens: int32 or int64, any shape.  A token outside ``[0, vocab)`` gives a row of NaN and no gradient.
        weight: ``[vocab, dim]`` fp32, bf16 or fp16.
        scale: factor applied in fp32 before the one rounding.
        padding_idx: a row that receives no gradient, as in ``nn.Embedding`` (its values are still looked up).
    """
    if padding_idx is not None and not 0 <= int(padding_idx) < weight.shape[0]:
        raise ValueError("padding_idx must be None or a row of weight")
    return _torch_binding.load().token_embedding(tokens, weight, float(scale), -1 if padding_idx is None else int(padding_idx))


class TokenEmbedding(nn.Module):
    """``nn.Embedding`` as the reference uses it (src/decoder/decoder.py:9: ``padding_idx=0``), same parameter name, over
    :func:`token_embedding`.  ``scale="sqrt"``: the square root of the width."""

    def __init__(self, vocab_size: int, dim: int, padding_idx: Optional[int] = None, scale=1.0):
        super().__init__()
        self.padding_idx = padding_idx
        self.scale = math.sqrt(dim) if scale == "sqrt" else float(scale)
        self.weight = nn.Parameter(torch.empty(vocab_size, dim))
        nn.init.normal_(self.weight)
        if padding_idx is not None:
            with torch.no_grad():
                self.weight[padding_idx].zero_()

    def forward(self, tokens: torch.Tensor) -> torch.Tensor:
        return token_embedding(tokens, self.weight, self.scale, self.padding_idx)

    def extra_repr(self) -> str:
        return f"{self.weight.shape[0]}, {self.weight.shape[1]}, padding_idx={self.padding_idx}, scale={self.scale}"
