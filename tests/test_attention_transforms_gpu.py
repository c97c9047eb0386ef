"""Attention between ragged sets, and norm and rotation, under torch's transforms: followed, or refused rather than passed over."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _calls(dev):
    from hgcalml_b200.cross_attention_op import CrossAttention
    from hgcalml_b200.norm_rotate_op import NormRotate
    rs_q, rs_k = (torch.tensor(r, dtype=torch.int32, device=dev) for r in ([0, 4, 9], [0, 6, 7]))
    q, k, v = (torch.randn((n, 2, 16), generator=torch.Generator(device=dev).manual_seed(i), device=dev) for i, n in enumerate((9, 7, 7)))
    w, p = torch.ones(16, device=dev), torch.arange(9., device=dev)
    return [(lambda *t: CrossAttention(*t, rs_q, rs_k), (q, k, v)), (lambda x, y, s: NormRotate(x, y, s, None, p)[0], (q, k, w)),
            (lambda x, t: NormRotate(x, None, None, None, t)[0], (q, p))]


@pytest.mark.parametrize("which", [0, 1, 2])
def test_tangents_are_refused(cuda, which):
    from hgcalml_b200 import _capi as C
    call, args = _calls(cuda)[which]
    want = call(*args)
    for i in range(len(args)):
        with torch.autograd.forward_ad.dual_level():
            duals = [torch.autograd.forward_ad.make_dual(t, torch.ones_like(t)) if j == i else t for j, t in enumerate(args)]
            with pytest.raises(C.HgcError, match="forward-mode"):
                call(*duals)
            with torch.no_grad(), pytest.raises(C.HgcError, match="forward-mode"):
                call(*duals)
            assert torch.equal(call(*args), want)  # no tangent among these
        with pytest.raises(RuntimeError):
            torch.func.jvp(lambda t: call(*args[:i], t, *args[i + 1:]), (args[i],), (torch.ones_like(args[i]),))
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda t: call(t, *args[1:]))(torch.stack([args[0]] * 3))
    assert torch.equal(call(*args), want)


@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning", "ignore::DeprecationWarning")
def test_a_trace_does_not_keep_a_result_as_a_constant(cuda, which, grad):
    call, args = _calls(cuda)[which]
    leaves = [args[0].clone().requires_grad_(grad), *args[1:]]
    traced = torch.jit.trace(call, tuple(leaves), check_trace=False)
    other = [2. * args[0].roll(1, 0) + 1., *args[1:]]
    assert torch.equal(traced(*other), call(*other)) and not torch.equal(call(*other), call(*args))


def test_gradients_of_given_tensors_refuse_tangents(cuda):
    from hgcalml_b200 import _capi as C
    from hgcalml_b200.cross_attention_op import CrossAttention, CrossAttentionGrad
    rs = torch.tensor([0, 5], dtype=torch.int32, device=cuda)
    x = torch.randn((5, 2, 16), device=cuda)
    out, lse = CrossAttention(x, x, x, rs, rs, with_lse=True)
    with torch.autograd.forward_ad.dual_level(), pytest.raises(C.HgcError, match="forward-mode"):
        CrossAttentionGrad(torch.autograd.forward_ad.make_dual(x, x), x, x, x, out, lse, rs, rs)
