"""The logits that texts are scored by: products in 32 bits, not rounded to the model's 16."""
import pytest
import torch

from test_gpu_serving_model import make, texts

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lengths", [[30, 1, 9], [2100, 40]])
def test_scores_are_made_from_products_in_32_bits(monkeypatch, lengths):
    """A sum of n products in 32 bits, in any order, is off by 2 n 2^-24 sum |x w| at most; rounded to fp16 it would be off by 2^-11 of itself."""
    from rptc_b200 import ops
    model = make(rows=2, max_pos=2200)
    seen, normed = [], []
    logprobs, rmsnorm = ops.token_logprobs, ops.rmsnorm

    def scored(logits, targets, top):
        seen.append((logits.clone(), normed[-1].clone()))
        return logprobs(logits, targets, top)

    def norm(h, w, out, eps):
        normed.append(out)
        return rmsnorm(h, w, out, eps)
    monkeypatch.setattr(ops, "token_logprobs", scored)
    monkeypatch.setattr(ops, "rmsnorm", norm)
    found = model.score(texts(lengths), top=2)
    assert [len(f[0]) for f in found] == [n - 1 for n in lengths]
    row, last = 0, None
    for logits, xn in seen:
        row = row if last is not None and torch.equal(xn, last) else 0
        last, x, w = xn, xn[row:row + len(logits)].double(), model.head.double()
        row += len(logits)
        assert logits.dtype == torch.float32
        assert ((logits.double() - x @ w.t()).abs() <= 2 * model.cfg.hidden * 2.0**-24 * (x.abs() @ w.abs().t()) + 2.0**-149).all()
