"""Prompts of equal lengths make the rotary angles' table once where a kernel reads it, and not at all where none does."""
import pytest
import torch

from test_gpu_serving_model import make, texts

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens,incoherent,tables", [(3, True, 0), (12, True, 1), (12, False, 0)])
def test_tables_of_a_prompt(monkeypatch, tokens, incoherent, tables):
    from rptc_b200 import ops
    model = make(rows=2, incoherent=incoherent)
    made, table = [], ops.rope_angles
    monkeypatch.setattr(ops, "rope_angles", lambda *a: made.append(a) or table(*a))
    model.prefill(torch.stack(texts([tokens, tokens])))
    assert len(made) == tables and model.pos.tolist() == [tokens, tokens]
