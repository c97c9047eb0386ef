"""Attention between ragged sets: gradients of sharp weights, of few keys, of batches of very different events, and of many ragged ones.
Formulas and bounds are those of test_cross_attention_gpu."""
import random

import pytest
import torch

from test_cross_attention_gpu import E, assert_near, check, inputs, reference, splits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["half", "bfloat"])
@pytest.mark.parametrize("dim,heads,kv_heads", [(64, 2, 1), (128, 2, 2), (22, 2, 1), (16, 2, 2)])
def test_gradients_at_large_scores(cuda, dtype, dim, heads, kv_heads):
    nq, nk = [40, 100, 300], [130, 70, 900]
    q, k, v, grad = inputs(nq, nk, heads, kv_heads, dim, dtype, cuda, seed=110, size=6.)
    check(q, k, v, grad, nq, nk, what="large")


@pytest.mark.parametrize("dtype", ["half", "bfloat"])
@pytest.mark.parametrize("dim", [22, 64, 128])
def test_what_rounding_left_of_the_result_makes_up_for_it(cuda, dtype, dim):
    """Events of a few keys: products in float32, and the sum of out and grad from the unrounded result, so that the bound has the rounding of the
    gradient alone: o is off by u^2 |o| and what sums and scores are.  Without the rest the gradient of queries is further off."""
    from hgcalml_b200.cross_attention_op import CrossAttention, CrossAttentionGrad
    nq, nk, heads = [200] * 6, [8, 3, 2, 12, 5, 9], 2
    q, k, v, grad = inputs(nq, nk, heads, heads, dim, dtype, cuda, seed=111, size=2.)
    u, scale = torch.finfo(q.dtype).eps / 2, dim ** -0.5
    tiny = torch.finfo(q.dtype).smallest_normal * torch.finfo(q.dtype).eps
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    rs = splits(nq, cuda), splits(nk, cuda)
    dq, dk, _ = torch.autograd.grad(CrossAttention(*leaves, *rs), leaves, grad)
    out, lse = CrossAttention(q, k, v, *rs, with_lse=True)
    without, _, _ = CrossAttentionGrad(grad, q, k, v, out, lse, *rs, out_rest=torch.zeros_like(out))
    assert torch.equal(CrossAttentionGrad(grad, q, k, v, out, lse, *rs)[0], without)
    a = b = 0
    off = [0., 0.]  # squares, with the rest and without
    for n, m in zip(nq, nk):
        rows, keys = slice(a, a + n), slice(b, b + m)
        a, b = a + n, b + m
        for h in range(heads):
            qh, kh, vh, gh = (t.double() for t in (q[rows, h], k[keys, h], v[keys, h], grad[rows, h]))
            s = scale * qh @ kh.T
            p = torch.softmax(s, 1)
            x = scale * (3 * dim + 22) * E * (qh.abs() @ kh.abs().T).amax(1) + 4 * E * torch.logsumexp(s, 1).abs()
            rel = (2 * x + 2. ** -21)[:, None]
            o = p @ vh
            err_o = u * u * o.abs() + (rel + (m + 100) * E) * (p @ vh.abs())
            ds = p * (gh @ vh.T - (gh * o).sum(1, keepdim=True))
            err_ds = rel * ds.abs() + p * (2 * (3 * dim + 22) * E * (gh.abs() @ vh.abs().T) + (gh.abs() * err_o).sum(1, keepdim=True)
                                           + (dim + 8) * E * (gh.abs() * o.abs()).sum(1, keepdim=True))
            want = scale * ds @ kh
            bound = u * want.abs() + tiny + scale * ((err_ds + (m + 100) * E * ds.abs()) @ kh.abs())
            assert_near(dq[rows, h], (want, bound), "dq")
            off = [e + float((g[rows, h].double() - want).square().sum()) for e, g in zip(off, (dq, without))]
            want = scale * ds.T @ qh
            bound = u * want.abs() + tiny + scale * ((err_ds + (n + 100) * E * ds.abs()).T @ qh.abs())
            assert_near(dk[keys, h], (want, bound), "dk")
    assert off[1] > off[0]


@pytest.mark.parametrize("dtype", ["float", "half", "bfloat"])
@pytest.mark.parametrize("dim", [16, 64, 128])
def test_events_of_very_different_size(cuda, dtype, dim):
    """Events of a few keys and of one beside one of thousands, and few queries beside many: the kernels are chosen for the mean event, every
    result is within the bounds of its own.  In 16 bits a quarter of a sum may come from the polynomial: its logarithm is off by 2^-13."""
    from hgcalml_b200.cross_attention_op import CrossAttention
    for nq, nk in (([300, 40, 500, 1], [8, 1, 10000, 2]), ([5000, 1, 3], [4, 6000, 0]), ([1, 1, 900], [20, 5000, 3])):
        q, k, v, grad = inputs(nq, nk, 2, 1, dim, dtype, cuda, seed=112)
        want, lse = reference(q, k, v, nq, nk, dim ** -0.5, None, grad)
        leaves = [t.requires_grad_(True) for t in (q, k, v)]
        out, got = CrossAttention(*leaves, splits(nq, cuda), splits(nk, cuda), with_lse=True)
        assert_near(out.detach(), want["out"], f"{nq} on {nk}: out")
        for name, g in zip(("dq", "dk", "dv"), torch.autograd.grad(out, leaves, grad)):
            assert_near(g, want[name], f"{nq} on {nk}: {name}")
        seen = ~lse.isinf()
        assert torch.equal(~got.isinf(), seen)
        assert ((got.double() - lse).abs()[seen] <= (0. if dtype == "float" else 2. ** -13) + 1e-5 * (1 + lse.abs()[seen])).all()


@pytest.mark.parametrize("dtype,dim,group", [("float", 24, 1), ("float", 96, 3), ("half", 64, 1), ("bfloat", 64, 3), ("bfloat", 128, 2), ("bfloat", 10, 5)])
def test_many_ragged_events(cuda, dtype, dim, group):
    """Every row of every event in one tile: random lengths with empty events, ones around those of tiles and steps, and rows behind the last."""
    rng = random.Random(dim + group)
    for most in (3, 70, 300):
        n = rng.randint(30, 70)
        length = lambda: rng.choice([0, 0, 1, rng.randint(0, most), most, 63, 64, 65, 127, 128, 129][:5 if most < 60 else None])  # noqa: E731
        nq, nk = [length() for _ in range(n)], [length() for _ in range(n)]
        q, k, v, grad = inputs(nq, nk, group, 1, dim, dtype, cuda, seed=113, extra=(rng.randint(0, 200), rng.randint(0, 200)))
        out = check(q, k, v, grad, nq, nk, what=f"lengths up to {most}")
        assert (out[sum(nq):] == 0).all()
