"""Attention between ragged sets: what its rows may hold (no number, infinities, weights and gradients of very different size), and what
it refuses.  Formulas and the derivation of the bounds are those of test_cross_attention_gpu."""
import pytest
import torch

from test_cross_attention_gpu import assert_near, inputs, reference, splits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [72, 100, 128])
@pytest.mark.parametrize("dtype", ["float"])
def test_queries_that_see_no_key_hold_anything(cuda, dtype, dim):
    """Events without keys, with masked keys alone, and rows behind the last event: zeros, whatever their queries are, in heads whose rows
    are copied one step at a time as in narrower ones."""
    from hgcalml_b200.cross_attention_op import CrossAttention
    nq, nk = [130, 70, 5, 64], [0, 90, 200, 0]
    q, k, v, grad = inputs(nq, nk, 4, 2, dim, dtype, cuda, seed=71, extra=(40, 3))
    mask = torch.ones(len(k), dtype=torch.bool, device=cuda)
    mask[90:290] = False
    blind = torch.ones(len(q), dtype=torch.bool, device=cuda)
    blind[130:200] = False
    q[blind] = torch.tensor([float("nan"), float("inf"), -float("inf")], device=cuda).to(q.dtype)[torch.arange(int(blind.sum()), device=cuda) % 3, None, None]
    want, _ = reference(torch.where(blind[:, None, None], torch.zeros_like(q), q), k, v, nq, nk, dim ** -0.5, mask, grad)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    rs = splits(nq, cuda), splits(nk, cuda)
    for _ in range(20):
        out, lse = CrossAttention(*leaves, *rs, key_mask=mask, with_lse=True)
        assert (out[blind] == 0).all() and (lse[blind] == -float("inf")).all()
        assert_near(out.detach(), want["out"], "out")
    assert (torch.autograd.grad(out, leaves, grad)[0][blind] == 0).all()
