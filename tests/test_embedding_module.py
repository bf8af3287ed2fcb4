"""The Embedding module's constructors (no GPU: nothing is looked up)."""

from __future__ import annotations

import pytest
import torch

from opaque_amd.vocabulary import Embedding


@pytest.mark.parametrize("freeze", [True, False])
def test_from_pretrained_shares_the_table(freeze):
    table = torch.randn(7, 5)
    m = Embedding.from_pretrained(table, freeze, -2, scale=3.0)
    assert m.weight.data_ptr() == table.data_ptr() and m.weight.requires_grad is not freeze
    assert (m.num_embeddings, m.embedding_dim, m.padding_idx, m.scale) == (7, 5, 5, 3.0)
    assert torch.equal(m.weight.detach(), table) and set(m.state_dict()) == {"weight"}
    assert Embedding.from_pretrained(table).scale == 1.0


def test_from_pretrained_refuses_what_the_module_does_not_do():
    with pytest.raises(ValueError):
        Embedding.from_pretrained(torch.randn(7))
    with pytest.raises(TypeError):
        Embedding.from_pretrained(torch.randn(7, 5), max_norm=1.0)
