"""Attention between ragged sets: what its rows may hold (no number, infinities, weights and gradients of very different size), and what
it refuses.  Formulas and the derivation of the bounds are those of test_cross_attention_gpu."""
import math

import pytest
import torch

from test_cross_attention_gpu import E, TYPES, assert_near, inputs, reference, splits

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


@pytest.mark.parametrize("dtype", ["half", "bfloat"])
@pytest.mark.parametrize("n_q,heads", [(100, 2), (300, 1), (1, 2), (4, 4)])
@pytest.mark.parametrize("n_k", [200_000, 400_000])
def test_one_key_far_above_all_others(cuda, dtype, n_q, heads, n_k):
    """One key dominates, and hundreds of thousands have a share together, wherever the one is.  Values are one but for its zero, so a
    result is the others' share.  With u the rounding of the type it is off by 2 u + 2^-12 (its own, the weights' and their powers of two),
    by 2 x for the scores (see test_cross_attention_gpu), by 2^-23 for each of n / 16 sums that are cut off, and in half
    precision by n 2^-37 for weights below its normal numbers."""
    from hgcalml_b200.cross_attention_op import CrossAttention
    dim, one = 64, 1 if n_q == 4 else heads
    q = torch.zeros((n_q, heads, dim), dtype=TYPES[dtype], device=cuda)
    q[..., 0] = 8.  # the score is the key's first column
    v = torch.ones((n_k, one, dim), dtype=q.dtype, device=cuda)
    rs = splits([n_q], cuda), splits([n_k], cuda)
    for gap in (10., 14., 16., 17., 17.5, 18., 20.):
        for at in (0, 5, n_k // 2, n_k - 1):
            k = torch.zeros_like(v)
            k[at, :, 0], v[at] = gap, 0.
            out, lse = CrossAttention(q, k, v, *rs, with_lse=True)
            v[at] = 1.
            others = (n_k - 1) * math.exp(-gap)
            share = others / (1. + others)
            u = torch.finfo(q.dtype).eps / 2
            bound = share * (2 * u + 2. ** -12 + 2 * (3 * dim + 22) * E * gap + n_k / 16 * 2. ** -23)
            if dtype == "half":
                bound += n_k * 2. ** -37 + 2. ** -25
            assert float((out.double() - share).abs().max()) <= bound, (gap, at, share, float(out.min()), float(out.max()))
            assert float((lse.double() - gap - math.log1p(others)).abs().max()) <= 1e-5 * (1 + gap)


@pytest.mark.parametrize("dtype,dim", [("float", 64), ("float", 128), ("half", 64), ("bfloat", 64), ("bfloat", 128), ("bfloat", 22)])
def test_gradients_of_hidden_keys_are_zero_whatever_the_queries_are(cuda, dtype, dim):
    """Masked keys of events whose queries, or their gradients, hold NaN and infinities: exactly zero; other events as without."""
    from hgcalml_b200.cross_attention_op import CrossAttention
    nq, nk = [140, 70, 300], [200, 90, 400]
    q, k, v, grad = inputs(nq, nk, 4, 2, dim, dtype, cuda, seed=91)
    mask = torch.rand(len(k), generator=torch.Generator(device=cuda).manual_seed(1), device=cuda) < 0.7
    mask[200:290] = False
    rs = splits(nq, cuda), splits(nk, cuda)

    def run():
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        return torch.autograd.grad(CrossAttention(*leaves, *rs, key_mask=mask), leaves, grad)

    clean = run()
    q[7], q[150], grad[9], grad[160] = float("nan"), float("inf"), float("inf"), float("nan")
    dq, dk, dv = run()
    for got, before in ((dk, clean[1]), (dv, clean[2])):
        assert (got[~mask] == 0).all() and torch.equal(got[290:], before[290:])
    assert (dq[140:210] == 0).all() and torch.equal(dq[210:], clean[0][210:])


@pytest.mark.parametrize("dim,heads,kv_heads", [(64, 2, 2), (128, 2, 1), (40, 3, 1)])
def test_gradients_in_half_do_not_depend_on_other_events(cuda, dim, heads, kv_heads):
    """Rows of another event that are 2^20 times as large, or infinite, change no bit."""
    from hgcalml_b200.cross_attention_op import CrossAttention
    nq, nk = [150, 7, 300, 0, 90], [2000, 300, 700, 50, 4000]
    q, k, v, grad = inputs(nq, nk, heads, kv_heads, dim, "half", cuda, seed=101)
    rs = splits(nq, cuda), splits(nk, cuda)
    mask = torch.ones(len(k), dtype=torch.bool, device=cuda)
    mask[2001] = mask[5] = False
    grad *= 2. ** -10

    def run():
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        return torch.autograd.grad(CrossAttention(*leaves, *rs, key_mask=mask), leaves, grad)

    clean = run()
    want, _ = reference(q, k, v, nq, nk, dim ** -0.5, mask, grad)
    for got, name in zip(clean, ("dq", "dk", "dv")):
        assert_near(got, want[name], name)
    for large in (1024., 60000., float("inf")):
        grad[151:153], grad[200:210], v[2001:2010], v[2400:2410], v[5] = large, -large, large, large, large  # of events 1 and 2, and a masked key
        for got, before, gone in zip(run(), clean, (slice(150, 457), slice(2000, 3000), slice(2000, 3000))):
            keep = torch.ones(len(got), dtype=torch.bool, device=cuda)
            keep[gone] = False
            assert torch.equal(got[keep], before[keep])


@pytest.mark.parametrize("dim,heads,kv_heads", [(64, 2, 1), (128, 1, 1)])
def test_gradients_of_very_different_size_in_half(cuda, dim, heads, kv_heads):
    """Rows of the gradient 2^20 apart in an event, on so many keys that a weight is 2^-15.  A slope of half precision is off by 2^-25 where it is below
    the normal numbers, in units of 2^14 times a power of two of at least 1 / (2 |do| max|v|), with do the row's gradient for dq and
    the event's largest for dk: by 2^-38 |do| max|v|; a weight by 2^-39."""
    from hgcalml_b200.cross_attention_op import CrossAttention
    nq, nk = [300, 40], [40000, 3000]
    q, k, v, grad = inputs(nq, nk, heads, kv_heads, dim, "half", cuda, seed=102)
    grad[::7] *= 2. ** 10
    grad[1::7] *= 2. ** -10
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    got = torch.autograd.grad(CrossAttention(*leaves, splits(nq, cuda), splits(nk, cuda)), leaves, grad)
    want, _ = reference(q.detach(), k.detach(), v.detach(), nq, nk, dim ** -0.5, None, grad)
    with torch.no_grad():
        a = b = 0
        for n, m in zip(nq, nk):
            rows, keys = slice(a, a + n), slice(b, b + m)
            a, b = a + n, b + m
            do, vs = grad[rows].double().norm(dim=-1), v[keys].double().norm(dim=-1).max()
            for h in range(heads):
                kv = h * kv_heads // heads
                want["dq"][1][rows, h] += dim ** -0.5 * 2. ** -38 * do[:, h, None] * vs * k[keys, kv].double().abs().sum(0)
                want["dk"][1][keys, kv] += dim ** -0.5 * 2. ** -38 * do.max() * vs * q[rows, h].double().abs().sum(0)
                want["dv"][1][keys, kv] += 2. ** -39 * grad[rows, h].double().abs().sum(0)
        for g, name in zip(got, ("dq", "dk", "dv")):
            assert_near(g, want[name], name)
    # the gradient of a query depends on its own row alone
    small = torch.arange(len(q), device=cuda) % 7 == 1
    grad[~small] *= 2. ** -10
    again, = torch.autograd.grad(CrossAttention(*leaves, splits(nq, cuda), splits(nk, cuda)), leaves[:1], grad)
    assert torch.equal(again[small], got[0][small])


@pytest.mark.parametrize("dtype", ["float", "bfloat"])
def test_what_the_device_finds_wrong_is_raised_on_demand(cuda, dtype, monkeypatch):
    from hgcalml_b200 import _capi as C
    from hgcalml_b200.cross_attention_op import CrossAttention, CrossAttentionGrad
    q, k, v, grad = inputs([100], [200], 2, 2, 64, dtype, cuda)
    good = splits([40, 60], cuda), splits([50, 100], cuda)
    bad = splits([40, 60], cuda), torch.tensor([0, 150, 100], dtype=torch.int32, device=cuda)
    want, lse = CrossAttention(q, k, v, *good, with_lse=True)
    CrossAttention(q, k, v, *bad)  # unspecified, and nothing waits
    monkeypatch.setattr(C, "CHECK_STATUS", True)
    assert torch.equal(CrossAttention(q, k, v, *good), want)
    CrossAttentionGrad(grad, q, k, v, want, lse, *good)
    assert CrossAttention(q[:0], k, v, *[torch.zeros_like(good[0])] * 2).shape == (0, 2, 64)
    with pytest.raises(C.HgcError, match="row splits"):
        CrossAttention(q, k, v, *bad)
    with pytest.raises(C.HgcError, match="row splits"):
        CrossAttentionGrad(grad, q, k, v, want, lse, *bad)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):  # a capture cannot wait
        held = CrossAttention(q, k, v, *good)
    graph.replay()
    assert torch.equal(held, want)


@pytest.mark.parametrize("dtype", ["float", "half", "bfloat"])
@pytest.mark.parametrize("call", range(len(CALLS)))
def test_gradients_of_what_is_no_number_are_none(cuda, dtype, call):
    """A NaN in a query: its gradient, and those of all keys and values that it sees, and no others."""
    from hgcalml_b200.cross_attention_op import CrossAttention
    nq, nk, heads, kv_heads, dim = CALLS[call]
    q, k, v, grad = inputs(nq, nk, heads, kv_heads, dim, dtype, cuda, seed=98)
    mask = torch.rand(len(k), generator=torch.Generator(device=cuda).manual_seed(3), device=cuda) < 0.8
    rs = splits(nq, cuda), splits(nk, cuda)

    def run():
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        return torch.autograd.grad(CrossAttention(*leaves, *rs, key_mask=mask), leaves, grad)

    clean = run()
    q[0, 0, 0] = float("nan")
    got = run()
    seen = mask.clone()
    seen[nk[0]:] = False
    for g, before, rows in zip(got, clean, (torch.arange(len(q), device=cuda) == 0, seen, seen)):
        gone = torch.zeros(g.shape, dtype=torch.bool, device=cuda)
        gone[rows, 0] = True
        assert torch.equal(g.isnan(), gone) and torch.equal(g[~gone], before[~gone])


@pytest.mark.parametrize("dtype", ["float", "half", "bfloat"])
@pytest.mark.parametrize("call", range(len(CALLS)))
def test_keys_that_are_masked_first_or_last(cuda, dtype, call):
    """Whole steps and parts without a key that is seen, before the first one and behind the last, hold anything and change nothing."""
    from hgcalml_b200.cross_attention_op import CrossAttention
    nq, nk, heads, kv_heads, dim = CALLS[call]
    q, k, v, grad = inputs(nq, nk, heads, kv_heads, dim, dtype, cuda, seed=99)
    for event in (slice(0, nk[0]), slice(nk[0], nk[0] + nk[1])):
        for hide in (slice(event.start, event.stop - 2), slice(event.start + 2, event.stop), slice(event.start, (event.start + event.stop) // 2)):
            mask = torch.ones(len(k), dtype=torch.bool, device=cuda)
            mask[hide] = False
            want, _ = reference(q, k, v, nq, nk, dim ** -0.5, mask, grad)
            bad = [t.masked_fill(~mask[:, None, None], float("nan")).requires_grad_(True) for t in (k, v)]
            leaves = [q.detach().requires_grad_(True), *bad]
            out = CrossAttention(*leaves, splits(nq, cuda), splits(nk, cuda), key_mask=mask)
            assert_near(out.detach(), want["out"], "out")
            for name, g in zip(("dq", "dk", "dv"), torch.autograd.grad(out, leaves, grad)):
                assert_near(g, want[name], name)
