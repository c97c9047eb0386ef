"""Attention between ragged sets against its formulas in 64 bits, at the sizes, layouts and masks where it can go wrong.

Tolerances are bounds, not fits.  With u the largest relative error of a rounding to the tensors' type (eps / 2), e = 2^-24
that of float32 and w what weights are off by before they meet the values (0 in float32; in 16 bits their rounding u and, in the
weight and in the sum that it is divided by, the polynomial for their power of two, 1.0e-4 < 2^-13: u + 2^-12):
  a product on the tensor cores in float32 parts by 20 e: with x = big + small of 11 bits each, |x - big| <= 2^-11 |x|, of which small
  loses less than 2^-10, so 2 x 2^-21 for two operands, and small small, 2^-22, is left out; an addition of 8 products and what was
  there cuts off up to 2 e of each of the 9, 18 e for 8 products, less than 3 e for each one;
  a score is off by at most x = scale (3 D + 22) e sum|q_d k_d| + 4 e |lse|, so a weight by the share 2 x + 2^-21 (two scores; exp);
  o_d by u |o_d| + (w + 2 x + 2^-21 + (n + 100) e) sum_j p_j |v_jd| for n summed keys, 32 of them in one sum (72 e, and 20 e);
  ds_j = p_j (dp_j - delta) by (w + 2 x + 2^-21) |ds_j| + p_j (2 (3 D + 22) e sum|do_d v_jd| + sum_d |do_d| err(o_d));
the gradients by their sums over these, their own rounding and that of the sum."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

E = 2. ** -24
TYPES = {"float": torch.float32, "half": torch.float16, "bfloat": torch.bfloat16}


def splits(sizes, dev):
    return torch.tensor(np.concatenate([[0], np.cumsum(sizes)]), dtype=torch.int32, device=dev)


def reference(q, k, v, nq, nk, scale, mask=None, grad=None):
    """{name: (value, bound of the error)} in 64 bits; rows behind the last event are zero."""
    heads, kv_heads, dim = q.shape[1], k.shape[1], q.shape[2]
    group = heads // kv_heads
    u = torch.finfo(q.dtype).eps / 2
    w = 0. if q.dtype == torch.float32 else u + 2. ** -12
    f = lambda t: t.double()  # noqa: E731
    zero = lambda t: torch.zeros(t.shape, dtype=torch.float64, device=t.device)  # noqa: E731
    res = {n: [zero(t), zero(t)] for n, t in (("out", q), ("dq", q), ("dk", k), ("dv", k))}
    lse = torch.full(q.shape[:2], -float("inf"), dtype=torch.float64, device=q.device)
    a = b = 0
    for n, m in zip(nq, nk):
        keys = torch.arange(b, b + m, device=q.device)
        if mask is not None:
            keys = keys[mask[b:b + m] != 0]
        rows = slice(a, a + n)
        a, b = a + n, b + m
        if n == 0 or len(keys) == 0:
            continue
        for h in range(heads):
            kv = h // group
            qh, kh, vh = f(q[rows, h]), f(k[keys, kv]), f(v[keys, kv])
            s = scale * qh @ kh.T
            lh = torch.logsumexp(s, 1)
            lse[rows, h] = lh
            p = torch.exp(s - lh[:, None])
            x = scale * (3 * dim + 22) * E * (qh.abs() @ kh.abs().T).amax(1) + 4 * E * lh.abs()
            rel = (w + 2 * x + 2. ** -21)[:, None]
            o = p @ vh
            tol_o = u * o.abs() + (rel + (len(keys) + 100) * E) * (p @ vh.abs())
            res["out"][0][rows, h], res["out"][1][rows, h] = o, tol_o
            if grad is None:
                continue
            gh = f(grad[rows, h])
            # the sum of out and grad is taken from the rounded result
            ds = p * (gh @ vh.T - (gh * o).sum(1, keepdim=True))
            tol_ds = rel * ds.abs() + p * (2 * (3 * dim + 22) * E * (gh.abs() @ vh.abs().T) + ((gh.abs() * tol_o).sum(1, keepdim=True)))
            if len(keys) == 1:
                ds, tol_ds = zero(ds), zero(ds)
            dq = scale * ds @ kh
            res["dq"][0][rows, h] = dq
            res["dq"][1][rows, h] = u * dq.abs() + scale * ((tol_ds + (len(keys) + 100) * E * ds.abs()) @ kh.abs())
            res["dk"][0][keys, kv] += scale * ds.T @ qh
            res["dk"][1][keys, kv] += scale * ((tol_ds + (n * group + 100) * E * ds.abs()).T @ qh.abs())
            res["dv"][0][keys, kv] += p.T @ gh
            res["dv"][1][keys, kv] += ((rel + (n * group + 100) * E) * p).T @ gh.abs()
    for name in ("dk", "dv"):
        res[name][1] += u * res[name][0].abs()
    # half precision: what lies below its normal numbers is rounded in steps of its smallest one
    tiny = torch.finfo(q.dtype).smallest_normal * torch.finfo(q.dtype).eps
    return {name: (value, bound + tiny) for name, (value, bound) in res.items()}, lse


def assert_near(got, want, what):
    value, bound = want
    assert got.shape == value.shape
    bad = ~((got.double() - value).abs() <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} values are off, by up to " \
                          f"{float(((got.double() - value).abs() / bound)[bad].nan_to_num(float('inf')).max()):.3g} times the bound"


def inputs(nq, nk, heads, kv_heads, dim, dtype, dev, seed=1, extra=(0, 0), size=1.):
    g = torch.Generator(device=dev).manual_seed(seed)
    make = lambda *s: (size * torch.randn(s, generator=g, device=dev)).to(TYPES[dtype])  # noqa: E731
    q, k, v = make(sum(nq) + extra[0], heads, dim), make(sum(nk) + extra[1], kv_heads, dim), make(sum(nk) + extra[1], kv_heads, dim)
    return q, k, v, make(sum(nq) + extra[0], heads, dim)


def check(q, k, v, grad, nq, nk, mask=None, scale=None, both=True, what=""):
    """Forward, and backward through autograd, against the reference."""
    from hgcalml_b200.cross_attention_op import CrossAttention
    dev = q.device
    want, lse = reference(q, k, v, nq, nk, q.shape[2] ** -0.5 if scale is None else scale, mask, grad)
    rs_q, rs_k = splits(nq, dev), splits(nk, dev)
    out, got_lse = CrossAttention(q, k, v, rs_q, rs_k, scale=scale, key_mask=mask, with_lse=True)
    assert out.dtype == q.dtype and out.is_contiguous()
    assert_near(out, want["out"], what + " out")
    assert torch.equal(got_lse.isinf(), lse.isinf())
    assert ((got_lse.double() - lse).abs()[~lse.isinf()] <= 1e-5 * (1 + lse.abs()[~lse.isinf()])).all()
    if both:
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        again = CrossAttention(*leaves, rs_q, rs_k, scale=scale, key_mask=mask)
        assert torch.equal(again, out)
        for name, g in zip(("dq", "dk", "dv"), torch.autograd.grad(again, leaves, grad)):
            assert g.dtype == q.dtype
            assert_near(g, want[name], f"{what} {name}")
    return out


SHAPES = [  # events' queries, events' keys, heads, key heads
    ([1], [1], 1, 1), ([1], [700], 8, 8), ([5, 0, 1, 130], [3, 4, 0, 257], 4, 2), ([64, 128], [64, 128], 2, 2),
    ([127, 129, 1], [63, 65, 300], 3, 1), ([0, 0, 7], [9, 0, 1], 6, 2), ([33] * 40, [1 + 5 * i for i in range(40)], 2, 1),
    ([300], [1500], 5, 5), ([2, 3], [2000, 900], 7, 1),
]


@pytest.mark.parametrize("dtype", ["float", "half", "bfloat"])
@pytest.mark.parametrize("dim", [1, 8, 22, 32, 40, 64, 96, 127, 128])
def test_shapes(cuda, dtype, dim):
    for i, (nq, nk, heads, kv_heads) in enumerate(SHAPES):
        q, k, v, grad = inputs(nq, nk, heads, kv_heads, dim, dtype, cuda, seed=100 + i)
        check(q, k, v, grad, nq, nk, what=f"shape {i}")


@pytest.mark.parametrize("dtype,dim", [("float", 32), ("half", 64), ("bfloat", 64), ("bfloat", 128), ("bfloat", 22)])
def test_masked_keys_hold_anything(cuda, dtype, dim):
    """Infinities, NaN and the type's lowest value in masked keys, an event without a visible key, one with a single one, and
    rows behind the last event that hold NaN."""
    nq, nk = [70, 200, 3, 9], [90, 300, 40, 20]
    for seed in (1, 2):
        q, k, v, grad = inputs(nq, nk, 4, 2, dim, dtype, cuda, seed=seed, extra=(3, 5))
        g = torch.Generator(device=cuda).manual_seed(seed)
        mask = torch.rand((len(k),), generator=g, device=cuda) < 0.7
        mask[390:430] = False
        mask[430:450] = False
        mask[437] = True
        fill = torch.tensor([float("inf"), float("nan"), -float("inf"), torch.finfo(k.dtype).min], device=cuda).to(k.dtype)
        hidden = ~mask
        hidden[-5:] = True
        for t in (k, v):
            t[hidden] = fill[torch.randint(0, 4, (int(hidden.sum()), 1, 1), generator=g, device=cuda)].expand(-1, *t.shape[1:])
        kk, vv = (torch.where(hidden[:, None, None], torch.zeros_like(t), t) for t in (k, v))
        qq, gg = q.clone(), grad.clone()
        q[-3:], grad[-3:] = float("nan"), float("inf")
        qq[-3:], gg[-3:] = 0, 0
        want, _ = reference(qq, kk, vv, nq, nk, dim ** -0.5, mask, gg)
        from hgcalml_b200.cross_attention_op import CrossAttention
        leaves = [t.requires_grad_(True) for t in (q, k, v)]
        out = CrossAttention(*leaves, splits(nq, cuda), splits(nk, cuda), key_mask=mask)
        assert_near(out.detach(), want["out"], "out")
        for name, got in zip(("dq", "dk", "dv"), torch.autograd.grad(out, leaves, grad)):
            assert_near(got, want[name], name)
            # a key that is not seen, an event with one key, a row behind the last event: exactly zero
            rows = {"dq": slice(sum(nq), None), "dk": slice(430, 450), "dv": slice(390, 430)}[name]
            assert (got[rows] == 0).all()
            if name != "dq":
                assert (got[hidden] == 0).all()


@pytest.mark.parametrize("dtype", ["float", "bfloat"])
def test_a_neighbouring_event_does_not_leak(cuda, dtype):
    """The last tile of an event ends in rows of the next one, which may be infinite."""
    nq, nk = [10, 90, 30], [70, 20, 200]
    q, k, v, grad = inputs(nq, nk, 2, 2, 64, dtype, cuda, seed=3)
    whole = check(q, k, v, grad, nq, nk)
    from hgcalml_b200.cross_attention_op import CrossAttention
    k[70:90], v[70:90], q[10:100], grad[10:100] = float("nan"), float("inf"), float("nan"), float("inf")
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    out = CrossAttention(*leaves, splits(nq, cuda), splits(nk, cuda))
    assert torch.equal(out[:10], whole[:10]) and torch.equal(out[100:], whole[100:])
    for g, gone in zip(torch.autograd.grad(out, leaves, grad), (slice(10, 100), slice(70, 90), slice(70, 90))):
        keep = torch.ones(len(g), dtype=torch.bool, device=cuda)
        keep[gone] = False
        assert g[keep].isfinite().all()


@pytest.mark.parametrize("dtype,dim", [("float", 24), ("bfloat", 64), ("half", 128), ("bfloat", 20)])
def test_layouts(cuda, dtype, dim):
    """Views of joint projections, heads before rows, odd distances, unaligned starts and a row for all."""
    from hgcalml_b200.cross_attention_op import CrossAttention
    nq, nk, heads, kv_heads = [150, 20], [100, 333], 4, 2
    q, k, v, grad = inputs(nq, nk, heads, kv_heads, dim, dtype, cuda, seed=7)
    rs = splits(nq, cuda), splits(nk, cuda)
    want = CrossAttention(q, k, v, *rs)
    joint = torch.cat([q.flatten(1), q.flatten(1)], 1)[:, :heads * dim].unflatten(1, (heads, dim))
    packed = torch.stack([k, v], 1)
    by_head = q.transpose(0, 1).contiguous().transpose(0, 1)
    odd = torch.zeros((len(k), kv_heads, dim + 3), dtype=k.dtype, device=cuda)
    odd[:, :, 1:dim + 1] = k
    spread = torch.zeros((len(v), kv_heads, dim, 2), dtype=v.dtype, device=cuda)
    spread[..., 0] = v
    for args in ((joint, packed[:, 0], packed[:, 1]), (by_head, k, v), (q, odd[:, :, 1:dim + 1], v), (q, k, spread[..., 0])):
        out = CrossAttention(*args, *rs)
        # other kernels may take other layouts: equal up to the rounding of both
        assert (out.double() - want.double()).abs().max() <= 4 * torch.finfo(q.dtype).eps * v.abs().max()
        leaves = [t.detach().requires_grad_(True) for t in args]
        ref, _ = reference(q, k, v, nq, nk, dim ** -0.5, None, grad)
        for name, g in zip(("dq", "dk", "dv"), torch.autograd.grad(CrossAttention(*leaves, *rs), leaves, grad)):
            assert_near(g, ref[name], name)
    one = k[:1].expand(len(k), -1, -1)
    ref, _ = reference(q, one, v, nq, nk, dim ** -0.5)
    assert_near(CrossAttention(q, one, v, *rs), ref["out"], "one key for all")


@pytest.mark.parametrize("dtype", ["float", "half", "bfloat"])
def test_scales_and_large_scores(cuda, dtype):
    nq, nk = [40, 100], [130, 70]
    q, k, v, grad = inputs(nq, nk, 2, 1, 64, dtype, cuda, seed=9)
    for scale in (1e-3, 1.):
        check(q, k, v, grad, nq, nk, scale=scale, what=f"scale {scale}")
    q, k, v, grad = inputs(nq, nk, 2, 1, 64, dtype, cuda, seed=10, size=6.)
    out = check(q, k, v, grad, nq, nk, both=dtype == "float", what="large")
    assert out.isfinite().all()


@pytest.mark.parametrize("dtype,dim,heads,kv_heads", [("bfloat", 64, 8, 2), ("half", 128, 4, 4), ("float", 32, 4, 1), ("bfloat", 22, 2, 2),
                                                      ("bfloat", 32, 32, 1), ("half", 64, 40, 1)])
def test_single_queries_over_long_keys(cuda, dtype, dim, heads, kv_heads):
    """A query per event, and a few, over thousands of keys: the keys are split, and joined in a fixed order."""
    for nq, nk in (([1], [5000]), ([1, 1, 1], [7000, 0, 1234]), ([3], [9001])):
        q, k, v, grad = inputs(nq, nk, heads, kv_heads, dim, dtype, cuda, seed=21)
        out = check(q, k, v, grad, nq, nk)
        from hgcalml_b200.cross_attention_op import CrossAttention
        for _ in range(3):
            assert torch.equal(CrossAttention(q, k, v, splits(nq, cuda), splits(nk, cuda)), out)


@pytest.mark.parametrize("dtype", ["float", "half", "bfloat"])
@pytest.mark.parametrize("dim", [8, 24, 64, 120, 128])
@pytest.mark.parametrize("group", [1, 2, 3, 5, 8])
def test_a_few_queries_of_every_event(cuda, dtype, dim, group):
    """Single tokens with one to eight heads to a key head: masks that leave events some keys, one and none, what masked and foreign
    rows hold, events without queries or keys, lengths around those of a step, and rows behind the last event."""
    nq, nk = [1, 0, 1, 1, 1, 0, 1, 1], [1, 40, 0, 129, 700, 31, 1500, 64]
    q, k, v, grad = inputs(nq, nk, 2 * group, 2, dim, dtype, cuda, seed=23, extra=(1, 9))
    mask = torch.rand(k.shape[0], generator=torch.Generator(device=cuda).manual_seed(1), device=cuda) < 0.6
    mask[41:170] = False
    mask[100] = True  # one key of the event of 129
    mask[-73 - 9:] = False  # and none of the last one
    k[~mask], v[~mask] = float("nan"), float("inf")
    k[-9:], v[-9:] = float("nan"), float("nan")
    out = check(q, k, v, grad, nq, nk, mask=mask)
    assert (out[-2:] == 0).all()
    mask[:] = True
    k, v = k.nan_to_num(1.), v.nan_to_num(1., 1., 1.)
    k[-9:], v[-9:] = float("nan"), float("nan")
    check(q, k, v, grad, nq, nk, both=False)


@pytest.mark.parametrize("dtype,dim", [("bfloat", 64), ("float", 32)])
def test_many_queries_over_few_keys(cuda, dtype, dim):
    """The other long axis: gradients of a few keys are split over the queries."""
    nq, nk = [6000, 2500], [30, 3]
    q, k, v, grad = inputs(nq, nk, 4, 2, dim, dtype, cuda, seed=22)
    check(q, k, v, grad, nq, nk)


@pytest.mark.parametrize("dim,masked", [(32, True), (64, False), (128, True), (128, False)])
def test_tiles_with_and_without_a_second_half(cuda, dim, masked):
    """Events of 12 to 236 queries, three heads to a key head, on 195 to 3714 keys: tiles whose second half has rows follow ones whose has
    none, with any number of steps between; and a few queries on keys of one step and of many.  The same results every time."""
    from hgcalml_b200.cross_attention_op import CrossAttention
    for sizes in (lambda i: (12 + i * 97 % 225, 195 + i * 1013 % 3520), lambda i: (i % 4, [40, 1, 6000, 300, 0, 129, 9000, 64][i % 8])):
        nq, nk = zip(*[sizes(i) for i in range(44)])
        q, k, v, grad = inputs(nq, nk, 6, 2, dim, "bfloat", cuda, seed=24)
        mask = torch.rand(k.shape[0], generator=torch.Generator(device=cuda).manual_seed(2), device=cuda) < 0.7 if masked else None
        out = check(q, k, v, grad, nq, nk, mask=mask, both=False)
        for _ in range(20):
            assert torch.equal(CrossAttention(q, k, v, splits(nq, cuda), splits(nk, cuda), key_mask=mask), out)


def test_gradients_are_those_of_differences(cuda):
    """Central differences of a scalar of the result, in float32."""
    from hgcalml_b200.cross_attention_op import CrossAttention
    nq, nk = [6, 3], [11, 5]
    q, k, v, grad = inputs(nq, nk, 2, 1, 12, "float", cuda, seed=31)
    rs = splits(nq, cuda), splits(nk, cuda)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    grads = torch.autograd.grad(CrossAttention(*leaves, *rs), leaves, grad)
    gen = torch.Generator(device=cuda).manual_seed(5)
    for i in range(3):
        step = torch.randn(leaves[i].shape, generator=gen, device=cuda)
        h = 2. ** -6
        moved = [[t.detach() + (sign * h * step if j == i else 0.) for j, t in enumerate(leaves)] for sign in (1., -1.)]
        diff = sum(s * (CrossAttention(*m, *rs).double() * grad.double()).sum() for s, m in zip((1., -1.), moved)) / (2 * h)
        exact = (grads[i].double() * step.double()).sum()
        # third order: h^2 / 6 of a third derivative of order |step|^3 |grad|, and rounding of about 1e-6 / h
        assert abs(float(diff - exact)) <= 2e-2 * (1 + float((grads[i].double() * step.double()).abs().sum()))


def test_what_is_not_needed_is_not_computed(cuda):
    from hgcalml_b200.cross_attention_op import CrossAttention, CrossAttentionGrad
    nq, nk = [50, 10], [20, 300]
    q, k, v, grad = inputs(nq, nk, 2, 2, 64, "bfloat", cuda, seed=41)
    rs = splits(nq, cuda), splits(nk, cuda)
    out, lse = CrossAttention(q, k, v, *rs, with_lse=True)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    dq, dk, dv = torch.autograd.grad(CrossAttention(*leaves, *rs), leaves, grad)
    assert torch.equal(CrossAttentionGrad(grad, q, k, v, out, lse, *rs)[2], dv)
    assert CrossAttentionGrad(grad, q, k, v, out, lse, *rs, need_keys=False)[1:] == (None, None)
    ql = q.clone().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(CrossAttention(ql, k, v, *rs), ql, grad)[0], dq)
    vl = v.clone().requires_grad_(True)
    o, l2 = CrossAttention(q, k, vl, *rs, with_lse=True)
    assert not l2.requires_grad
    assert torch.equal(torch.autograd.grad(o, vl, grad)[0], dv)
    # the gradient of a sum comes as one value for all rows
    kl = k.clone().requires_grad_(True)
    g1, = torch.autograd.grad(CrossAttention(q, kl, v, *rs).sum(), kl)
    assert torch.equal(g1, torch.autograd.grad(CrossAttention(*leaves, *rs), leaves, torch.ones_like(out))[1])
    with pytest.raises(RuntimeError):  # once differentiable
        g, = torch.autograd.grad(CrossAttention(q, kl, v, *rs).float().square().sum(), kl, create_graph=True)
        g.sum().backward()


def test_parts_of_the_keys_join(cuda):
    """The logarithms of the sums put results over two halves of the keys together."""
    from hgcalml_b200.cross_attention_op import CrossAttention
    q, k, v, _ = inputs([77], [500], 2, 2, 32, "float", cuda, seed=51)
    rs = splits([77], cuda)
    whole = CrossAttention(q, k, v, rs, splits([500], cuda))
    (a, la), (b, lb) = (CrossAttention(q, k[s], v[s], rs, splits([n], cuda), with_lse=True) for s, n in ((slice(0, 200), 200), (slice(200, 500), 300)))
    w = torch.sigmoid(la - lb)[..., None]
    assert (a * w + b * (1 - w) - whole).abs().max() < 1e-5


def test_empty_batches(cuda):
    from hgcalml_b200.cross_attention_op import CrossAttention
    for nq, nk in (([0], [0]), ([0, 0], [5, 0]), ([4, 2], [0, 0]), ([], [])):
        for dtype in ("float", "bfloat"):
            q, k, v, grad = inputs(nq, nk, 2, 1, 64, dtype, cuda)
            leaves = [t.requires_grad_(True) for t in (q, k, v)]
            out = CrossAttention(*leaves, splits(nq, cuda), splits(nk, cuda))
            assert (out == 0).all() and out.shape == q.shape
            for g, t in zip(torch.autograd.grad(out, leaves, grad), leaves):
                assert g.shape == t.shape and (g == 0).all()
    q, k, v, _ = inputs([4], [6], 2, 1, 64, "bfloat", cuda)
    none = torch.zeros((1,), dtype=torch.int32, device=cuda)
    assert (CrossAttention(q, k, v, none, none) == 0).all()


@pytest.mark.parametrize("dtype", ["float", "bfloat"])
def test_streams_graphs_and_calls_at_once(cuda, dtype):
    from hgcalml_b200.cross_attention_op import CrossAttention, CrossAttentionGrad
    nq, nk = [200, 30], [1500, 800]
    q, k, v, grad = inputs(nq, nk, 4, 2, 64, dtype, cuda, seed=61)
    rs = splits(nq, cuda), splits(nk, cuda)
    want, lse = CrossAttention(q, k, v, *rs, with_lse=True)
    grads = CrossAttentionGrad(grad, q, k, v, want, lse, *rs)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    results = []
    for s in streams:
        with torch.cuda.stream(s):
            results.append(CrossAttentionGrad(grad, q, k, v, CrossAttention(q, k, v, *rs), lse, *rs))
    torch.cuda.synchronize()
    for r in results:
        assert all(torch.equal(a, b) for a, b in zip(r, grads))
    # two graphs in one pool, replayed in turn, with other splits and inputs in the same memory
    static = [t.clone() for t in (q, k, v, grad)]
    s_rs = [t.clone() for t in rs]
    graphs, outs = [], []
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        CrossAttention(*static[:3], *s_rs)
    torch.cuda.synchronize()
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=graphs[0].pool() if graphs else None):
            o, l2 = CrossAttention(*static[:3], *s_rs, with_lse=True)
            outs.append((o, *CrossAttentionGrad(static[3], *static[:3], o, l2, *s_rs)))
        graphs.append(g)
    for g, r in zip(graphs, outs):
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(r[0], want) and all(torch.equal(a, b) for a, b in zip(r[1:], grads))
    other_q, other_k = [100, 40], [2000, 77]  # fewer queries than the tensors have rows
    s_rs[0].copy_(splits(other_q, cuda))
    s_rs[1].copy_(splits(other_k, cuda))
    for g, r in zip(graphs, outs):
        g.replay()
        torch.cuda.synchronize()
        ref, _ = reference(q, k, v, other_q, other_k, 64 ** -0.5, None, grad)
        for got, name in zip(r, ("out", "dq", "dk", "dv")):
            assert_near(got, ref[name], name)


def test_splits_that_make_no_sense_are_reported(cuda):
    """Results are unspecified then, but nothing is read or written outside the tensors."""
    import ctypes
    from hgcalml_b200 import _capi as C
    q, k, v, grad = inputs([100], [200], 2, 2, 64, "bfloat", cuda)
    for rs_q, rs_k, bad in (([0, 40, 100], [0, 50, 200], 0), ([0, 40, 90], [0, 50, 150], 0), ([0, 60, 40], [0, 50, 200], 16),
                            ([0, 40, 101], [0, 50, 200], 16), ([5, 40, 100], [0, 50, 200], 16), ([0, 40, 100], [0, -5, 200], 16),
                            ([0, 2 ** 31 - 1, 100], [0, -2 ** 31, 2 ** 31 - 1], 16)):
        t = [torch.tensor(r, dtype=torch.int32, device=cuda) for r in (rs_q, rs_k)]
        out, lse = torch.zeros_like(q), torch.zeros((100, 2), device=cuda)
        d = [torch.zeros_like(x) for x in (q, k, v)]
        ws = C.workspace(C.lib.hgc_cross_attention_workspace_bytes(100, 200, 3, 2, 2, 64, 2), cuda)
        tail = (100, 200, 3, 2, 2, 64, None, ctypes.c_float(0.125), 2)
        rc = C.lib.hgc_cross_attention(C.ptr(q), C.ptr(k), C.ptr(v), C.ptr(t[0]), C.ptr(t[1]), None, C.ptr(out), None, C.ptr(lse), *tail,
                                       C.ptr(ws), ws.numel(), C.stream_of(q))
        assert rc == 0 and C.read_status(ws, raise_on_flag=False) == bad
        ws = C.workspace(C.lib.hgc_cross_attention_grad_workspace_bytes(100, 200, 3, 2, 2, 64, 2), cuda)
        rc = C.lib.hgc_cross_attention_grad(C.ptr(grad), C.ptr(q), C.ptr(k), C.ptr(v), C.ptr(out), None, C.ptr(lse), C.ptr(t[0]), C.ptr(t[1]),
                                            None, *[C.ptr(x) for x in d], *tail, C.ptr(ws), ws.numel(), C.stream_of(q))
        assert rc == 0 and C.read_status(ws, raise_on_flag=False) == bad


def test_offsets_beyond_32_bits(cuda):
    """Keys whose elements lie more than 2^31 elements, and queries more than 2^31 bytes, into their tensors."""
    from hgcalml_b200.cross_attention_op import CrossAttention
    n, heads, dim = 4_400_000, 4, 128
    k = torch.zeros((n, heads, dim), dtype=torch.bfloat16, device=cuda)  # 2.25e9 elements
    far = 700
    g = torch.Generator(device=cuda).manual_seed(3)
    k[-far:] = torch.randn((far, heads, dim), generator=g, device=cuda).to(k.dtype)
    q = torch.randn((3, heads, dim), generator=g, device=cuda).to(k.dtype)
    rs_q = torch.tensor([0, 0, 3], dtype=torch.int32, device=cuda)
    rs_k = torch.tensor([0, n - far, n], dtype=torch.int32, device=cuda)
    ref, _ = reference(q, k[-far:], k[-far:], [3], [far], dim ** -0.5)
    assert_near(CrossAttention(q, k, k, rs_q, rs_k), ref["out"], "out")
    del ref
    kq = k[-far:].clone()
    rs_k2 = torch.tensor([0, 0, far], dtype=torch.int32, device=cuda)
    out = CrossAttention(k, kq, kq, rs_k, rs_k2)
    ref, _ = reference(kq, kq, kq, [far], [far], dim ** -0.5)
    assert_near(out[-far:], ref["out"], "far queries")
    assert (out[:1000] == 0).all()
