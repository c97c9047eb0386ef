"""Attention between ragged sets: what its rows may hold (no number, infinities, weights and gradients of very different size), and what
it refuses.  Formulas and the derivation of the bounds are those of test_cross_attention_gpu."""
import pytest
import torch

from test_cross_attention_gpu import assert_near, inputs, reference, splits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [72, 100, 128])
@pytest.mark.parametrize("dtype", ["float", "half", "bfloat"])
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


# one query, a few, as many as fill half a tile with keys for both halves, several tiles; widths without whole vectors; short calls
CALLS = [([1, 1], [700, 900], 4, 2, 64), ([1, 1], [700, 900], 2, 2, 128), ([3, 2], [9000, 400], 4, 2, 64), ([100, 90], [6000, 500], 2, 2, 64),
         ([100, 90], [6000, 500], 4, 1, 128), ([700, 300], [900, 400], 2, 1, 64), ([700, 300], [900, 400], 2, 1, 96), ([200, 90], [300, 400], 2, 1, 22),
         ([20, 30], [30, 40], 2, 1, 32), ([1, 1], [300, 20], 2, 1, 7)]


@pytest.mark.parametrize("call", range(len(CALLS)))
@pytest.mark.parametrize("dtype", ["float", "half", "bfloat"])
@pytest.mark.parametrize("where", ["query", "keys", "value"])
def test_what_is_no_number_stays_none(cuda, call, dtype, where):
    """A NaN in a query, in all keys of a part, or in a value that is seen gives NaN in every result that it is a term of, and changes
    no other."""
    from hgcalml_b200.cross_attention_op import CrossAttention
    nq, nk, heads, kv_heads, dim = CALLS[call]
    q, k, v, _ = inputs(nq, nk, heads, kv_heads, dim, dtype, cuda, seed=81 + call)
    rs = splits(nq, cuda), splits(nk, cuda)
    clean, clean_lse = CrossAttention(q, k, v, *rs, with_lse=True)
    group, nan = heads // kv_heads, float("nan")
    gone = torch.zeros(clean.shape, dtype=torch.bool, device=cuda)
    if where == "query":
        q[nq[0] - 1, heads - 1, dim // 2] = nan
        gone[nq[0] - 1, heads - 1] = True
    elif where == "value":
        v[nk[0] // 2, 0, dim - 1] = nan
        gone[:nq[0], :group, dim - 1] = True
    else:
        k[nk[0] // 2:nk[0], 0, 0] = nan
        gone[:nq[0], :group] = True
    out, lse = CrossAttention(q, k, v, *rs, with_lse=True)
    assert torch.equal(out.isnan(), gone) and torch.equal(out[~gone], clean[~gone])
    rows = gone.all(-1)
    assert torch.equal(lse.isnan(), rows) and torch.equal(lse[~rows], clean_lse[~rows])


@pytest.mark.parametrize("dtype", ["half", "bfloat"])
@pytest.mark.parametrize("call", [2, 3, 4, 5, 6])
def test_a_key_that_is_no_number_is_one_in_every_column(cuda, dtype, call):
    """Some of the weights' powers of two are worked out on the multipliers: NaN in any of eight neighbouring keys gives NaN."""
    from hgcalml_b200.cross_attention_op import CrossAttention
    nq, nk, heads, kv_heads, dim = CALLS[call]
    q, k, v, _ = inputs(nq, nk, heads, kv_heads, dim, dtype, cuda, seed=95)
    rs = splits(nq, cuda), splits(nk, cuda)
    clean = CrossAttention(q, k, v, *rs)
    for at in range(nk[0] // 2, nk[0] // 2 + 8):
        bad = k.clone()
        bad[at, 0, 0] = float("nan")
        out, lse = CrossAttention(q, bad, v, *rs, with_lse=True)
        group = heads // kv_heads
        assert out[:nq[0], :group].isnan().all() and lse[:nq[0], :group].isnan().all()
        assert torch.equal(out[nq[0]:], clean[nq[0]:]) and torch.equal(out[:, group:], clean[:, group:])


@pytest.mark.parametrize("dtype", ["half", "bfloat", "float"])
@pytest.mark.parametrize("call", range(len(CALLS)))
def test_a_row_does_not_depend_on_its_neighbours(cuda, dtype, call):
    """Other queries of the event, some with much larger scores, change no bit of a query's result."""
    from hgcalml_b200.cross_attention_op import CrossAttention
    nq, nk, heads, kv_heads, dim = CALLS[call]
    q, k, v, _ = inputs(nq, nk, heads, kv_heads, dim, dtype, cuda, seed=97)
    rs = splits(nq, cuda), splits(nk, cuda)
    clean = CrossAttention(q, k, v, *rs)
    stay = torch.arange(len(q), device=cuda) % 3 != 1
    for size in (0.01, 1., 30.):
        other = torch.where(stay[:, None, None], q, size * q.flip(0, 1))
        assert torch.equal(CrossAttention(other, k, v, *rs)[stay], clean[stay])
