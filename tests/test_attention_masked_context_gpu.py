"""The attention layer on a context of which some rows hold anything and are masked."""
import pytest
import torch

from test_attention_layer_gpu import _rows, _splits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("prepared", [False, True])
@pytest.mark.parametrize("kind", [torch.bool, torch.uint8])
def test_what_masked_rows_hold_does_not_matter(cuda, dtype, prepared, kind):
    """Result and all gradients as with zeros there, bit by bit; the masked rows of the context get zeros."""
    from hgcalml_b200.AttentionLayersRagged import RaggedCrossAttention
    torch.manual_seed(7)
    nq, nk = [50, 0, 170, 1], [400, 7, 33, 0]
    layer = RaggedCrossAttention(4, 32, 24, n_in=20, n_context=28, n_key_heads=2).to(cuda).to(dtype)
    x, clean = _rows(sum(nq), 20, cuda, 1, dtype).requires_grad_(True), _rows(sum(nk), 28, cuda, 2, dtype)
    pq, clean_p = 5. * _rows(sum(nq), 4, cuda, 3, torch.float32), 5. * _rows(sum(nk), 4, cuda, 4, torch.float32)
    mask = torch.ones(sum(nk), dtype=kind, device=cuda)
    mask[::5] = 0
    mask[400:407] = 0
    hidden = mask == 0
    rs, grad = (_splits(nq, cuda), _splits(nk, cuda)), _rows(sum(nq), 24, cuda, 5, dtype)

    def run(fill):
        context, pk = clean.clone(), clean_p.clone()
        context[hidden], pk[hidden] = fill, fill
        context.requires_grad_(True)
        if prepared:
            y = layer([x, layer.prepare(context, pk, mask), *rs], pq, key_mask=mask)
        else:
            y = layer([x, context, *rs], pq, pk, key_mask=mask)
        return [y] + list(torch.autograd.grad(y, [x, context] + list(layer.parameters()), grad))

    want = run(0.)
    for fill in (float("nan"), float("inf"), 1e4):
        got = run(fill)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert (want[2][hidden] == 0).all() and all(t.isfinite().all() for t in want)
    with torch.no_grad():
        context = clean.clone()
        context[hidden] = float("nan")
        assert torch.equal(layer([x, context, *rs], pq, clean_p, key_mask=mask), want[0])


def test_masks_and_positions_that_do_not_fit_are_refused(cuda):
    from hgcalml_b200 import _capi as C
    from hgcalml_b200.AttentionLayersRagged import RaggedCrossAttention
    layer = RaggedCrossAttention(2, 8, 4, n_in=5, n_context=6).to(cuda)
    x, context, rs = _rows(3, 5, cuda, 1, torch.float32), _rows(7, 6, cuda, 2, torch.float32), (_splits([3], cuda), _splits([7], cuda))
    mask = torch.ones(7, dtype=torch.bool, device=cuda)
    for bad in (*(torch.ones(n, dtype=torch.bool, device=cuda) for n in (1, 6, 8)), mask.cpu(), mask.float()):
        with pytest.raises(C.HgcError, match="key_mask"):
            layer([x, context, *rs], key_mask=bad)
    for bad in (torch.zeros(6, device=cuda), torch.zeros(7, 2, 1, device=cuda), torch.zeros(7), torch.zeros(7, device=cuda, requires_grad=True)):
        with pytest.raises(C.HgcError, match="positions|CUDA"):
            layer([x, context, *rs], None, bad, key_mask=mask)
