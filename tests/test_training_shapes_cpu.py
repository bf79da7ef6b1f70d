"""What the scoring's and the embedding's nodes say to rows of no element: a ``ValueError`` by name, of any leading
shape. No kernel runs here."""

from __future__ import annotations

import pytest
import torch

from hsn_amd import embedding, scoring


@pytest.mark.parametrize("shape", [(), (0,), (3,), (2, 3), (2, 0)])
def test_scoring_of_no_vocabulary(shape):
    with pytest.raises(ValueError, match="logits are on cpu"):
        scoring.token_logprobs(torch.zeros(*shape, 0), torch.zeros(shape, dtype=torch.int64))


@pytest.mark.parametrize("shape", [(0,), (3,), (2, 3), (2, 3, 4), (2, 0, 4)])
def test_the_embedding_of_no_width(shape):
    tokens = torch.zeros(shape, dtype=torch.int64)
    with pytest.raises(ValueError, match="d_out is on cpu"):
        embedding.backward(tokens, torch.zeros(*shape, 0), 5)
    with pytest.raises(ValueError, match="table is on cpu"):
        embedding.forward(tokens, torch.zeros(5, 0))
