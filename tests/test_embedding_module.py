"""The embedding module's construction: what ``nn.Embedding`` has beside its forward."""
import pytest
import torch
import torch.nn as nn

from gmdn_amd.embedding import Embedding


def test_from_pretrained():
    table = torch.randn(7, 4)
    e = Embedding.from_pretrained(table, scale=3.0, padding_idx=2)
    assert type(e) is Embedding and e.scale == 3.0 and e.padding_idx == 2 and not e.weight.requires_grad
    assert e.weight.data_ptr() == table.data_ptr()
    assert Embedding.from_pretrained(table, freeze=False).weight.requires_grad and Embedding.from_pretrained(table).scale == 1.0


def test_device_and_type():
    e = Embedding(7, 4, device="meta", dtype=torch.bfloat16)
    assert e.weight.is_meta and e.weight.dtype == torch.bfloat16
    assert (Embedding(7, 4, 1, 2.0).weight[1] == 0).all() and "scale=2.0" in repr(Embedding(7, 4, 1, 2.0))
    assert isinstance(e, nn.Embedding)


@pytest.mark.parametrize("option", [dict(max_norm=1.0), dict(scale_grad_by_freq=True), dict(sparse=True)])
def test_options_that_it_does_not_have(option):
    with pytest.raises(ValueError, match="not supported"):
        Embedding(7, 4, **option)
    with pytest.raises(ValueError, match="not supported"):
        Embedding.from_pretrained(torch.randn(7, 4), **option)
