"""Norm and rotation of heads against the formulas in 64 bits.

Tolerances are bounds: with u = eps / 2 of the tensors' type and e = 2^-24, the norm's factor is off by (D + 6) e at most, an angle's
sine and cosine by 4 e, a turned value is a sum of two products: u |y| + (D + 16) e (|n_a| + |n_b|).  In the gradient the mean adds
a sum over the columns, the weights' sums one over all rows."""
import pytest
import torch

pytestmark = pytest.mark.gpu

E = 2. ** -24
TYPES = {"float": torch.float32, "half": torch.float16, "bfloat": torch.bfloat16}


def reference(x, w, pos, rotary, interleaved, base, eps, grad=None):
    """((y, bound), (dx, bound), (dw, bound))"""
    n, heads, dim = x.shape
    u = torch.finfo(x.dtype).eps / 2
    tiny = torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps
    x64 = x.double()
    w64 = torch.ones(dim, dtype=torch.float64, device=x.device) if w is None else w.double()
    r = 1 / torch.sqrt(x64.square().mean(-1, keepdim=True) + eps)
    m = x64 * r * w64
    # column d turns with its partner: y_d = cos n_d + sin n_partner, where sin has the sign of the side of the pair
    partner = torch.arange(dim, device=x.device)
    cos, sin = torch.ones((n, dim), dtype=torch.float64, device=x.device), torch.zeros((n, dim), dtype=torch.float64, device=x.device)
    if pos is not None and rotary:
        p = pos.double() if pos.dim() == 2 else pos.double()[:, None]
        axes = p.shape[1]
        pairs = rotary // (2 * axes)
        i = torch.arange(pairs, device=x.device)
        for a in range(axes):
            t = p[:, a, None] * base ** (-i.double() / pairs)
            one = a * 2 * pairs + (2 * i if interleaved else i)
            two = one + (1 if interleaved else pairs)
            partner[one], partner[two] = two, one
            cos[:, one], cos[:, two], sin[:, one], sin[:, two] = torch.cos(t), torch.cos(t), -torch.sin(t), torch.sin(t)
    cos, sin = cos[:, None], sin[:, None]
    y = cos * m + sin * m[..., partner]
    size = m.abs() + (sin != 0) * m[..., partner].abs()
    res = [(y, u * y.abs() + (dim + 16) * E * size + tiny)]
    if grad is not None:
        g = cos * grad.double() - sin * grad.double()[..., partner]
        gs = grad.double().abs() + (sin != 0) * grad.double()[..., partner].abs()
        gw, gws = g * w64, gs * w64.abs()
        mean = (gw * x64).mean(-1, keepdim=True)
        dx = r * (gw - x64 * r * r * mean)
        bound = (dim + 16) * E * r * (gws + 3 * x64.abs() * r * r * (gws * x64.abs()).mean(-1, keepdim=True))
        res.append((dx, u * dx.abs() + bound + tiny))
        dw = (g * x64 * r).sum((0, 1))
        uw = 0. if w is None else torch.finfo(w.dtype).eps / 2
        res.append((dw, uw * dw.abs() + (dim + 16 + n * heads / 64 + 64) * E * (gs * x64.abs() * r).sum((0, 1)) + tiny))
    return res


def assert_near(got, want, what):
    value, bound = want
    bad = ~((got.double() - value).abs() <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} values are off, by up to " \
                          f"{float(((got.double() - value).abs() / bound)[bad].nan_to_num(float('inf')).max()):.3g} times the bound"


def inputs(n, heads, dim, dtype, axes, kind, dev, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    x = (3. * torch.randn((n, heads, dim), generator=g, device=dev)).to(TYPES[dtype])
    w = 1. + 0.2 * torch.randn((dim,), generator=g, device=dev)
    grad = torch.randn((n, heads, dim), generator=g, device=dev).to(TYPES[dtype])
    shape = (n, axes) if axes else (n,)
    if kind == torch.float32:
        pos = 150. * torch.randn(shape, generator=g, device=dev)
    else:
        pos = torch.randint(-2_000_000, 2_000_000, shape, generator=g, device=dev).to(kind)
    return x, w, pos, grad


@pytest.mark.parametrize("dtype", ["float", "half", "bfloat"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rotary,axes", [(64, 64, 0), (32, 32, 4), (22, 12, 3), (128, 128, 1), (128, 64, 2), (8, 8, 1), (2, 2, 0), (96, 32, 2),
                                             (72, 64, 0), (1, 0, 0), (127, 126, 3), (40, 24, 1), (16, 16, 1)] + [
                             # axes of few columns, which end inside a 16-byte vector
                             (16, 4, 1), (32, 12, 3), (8, 6, 3), (64, 20, 5), (24, 8, 4), (16, 6, 1), (128, 8, 1),
                             # two columns at a time
                             (124, 100, 1), (50, 46, 0), (46, 40, 2), (60, 12, 6), (64, 60, 3), (66, 66, 0), (33, 32, 2), (61, 60, 5)])
def test_forward_and_backward(cuda, dtype, interleaved, dim, rotary, axes):
    from hgcalml_b200.norm_rotate_op import NormRotate
    kinds = [torch.float32, torch.int32, torch.int64]
    for i, (n, heads, m, kv_heads) in enumerate([(1, 1, 0, 1), (33, 8, 50, 2), (130, 3, 7, 1), (1000, 5, 1, 40)]):
        q, wq, pq, gq = inputs(n, heads, dim, dtype, axes, kinds[i % 3], cuda, 10 + i)
        k, wk, pk, gk = inputs(m, kv_heads, dim, dtype, axes, kinds[i % 3], cuda, 20 + i)
        if i % 2:
            wq, wk = wq.to(q.dtype), wk.to(q.dtype)
        how = dict(rotary_dim=rotary, interleaved=interleaved, eps=1e-5, base=500.)
        y, z = NormRotate(q, k, wq, wk, pq, pk, **how)
        want_q = reference(q, wq, pq, rotary, interleaved, 500., 1e-5, gq)
        want_k = reference(k, wk, pk, rotary, interleaved, 500., 1e-5, gk)
        assert_near(y, want_q[0], "queries")
        assert_near(z, want_k[0], "keys")
        leaves = [t.detach().requires_grad_(True) for t in (q, k, wq, wk)]
        out = NormRotate(*leaves, pq, pk, **how)
        assert torch.equal(out[0], y) and torch.equal(out[1], z)
        dq, dk, dwq, dwk = torch.autograd.grad(out, leaves, (gq, gk))
        assert dwq.dtype == wq.dtype and dq.dtype == q.dtype
        for got, want, name in ((dq, want_q[1], "dq"), (dk, want_k[1], "dk"), (dwq, want_q[2], "dwq"), (dwk, want_k[2], "dwk")):
            assert_near(got, want, name)


@pytest.mark.parametrize("dtype,dim", [("bfloat", 64), ("float", 20)])
def test_parts_that_are_left_out(cuda, dtype, dim):
    from hgcalml_b200.norm_rotate_op import NormRotate
    q, wq, pq, gq = inputs(50, 4, dim, dtype, 0, torch.int32, cuda, 1)
    k, wk, pk, gk = inputs(70, 2, dim, dtype, 0, torch.int32, cuda, 2)
    y, z = NormRotate(q, k, wq, wk, pq, pk)
    alone, none = NormRotate(q, None, wq, None, pq)
    assert none is None and torch.equal(alone, y)
    assert_near(NormRotate(q)[0], reference(q, None, None, 0, False, 2., 1e-6)[0], "no weight")
    still = NormRotate(q, k, wq, wk, pq, None)
    assert torch.equal(still[0], y)
    assert_near(still[1], reference(k, wk, None, 0, False, 2., 1e-6)[0], "no positions")
    # gradients of one set, of rows alone, of weights alone; a result that is not used
    full = torch.autograd.grad(NormRotate(*[t.requires_grad_(True) for t in (q, k, wq, wk)], pq, pk), (q, k, wq, wk), (gq, gk))
    a, b = NormRotate(q, k, wq, wk, pq, pk)
    dk, dwk = torch.autograd.grad(b, (k, wk), gk)
    assert torch.equal(dk, full[1]) and torch.equal(dwk, full[3])
    for pick in ((0,), (2,), (1,), (3,), (0, 3)):
        t = [x.detach().requires_grad_(i in pick) for i, x in enumerate((q, k, wq, wk))]
        out = NormRotate(*t, pq, pk)
        got = torch.autograd.grad([o for o in out], [t[i] for i in pick], (gq, gk), allow_unused=True)
        for g, i in zip(got, pick):
            assert torch.equal(g, full[i])
    with pytest.raises(RuntimeError):
        g, = torch.autograd.grad(NormRotate(q, None, wq, None, pq)[0].float().square().sum(), q, create_graph=True)
        g.sum().backward()


@pytest.mark.parametrize("dtype,dim", [("bfloat", 64), ("half", 32), ("float", 22)])
def test_layouts(cuda, dtype, dim):
    from hgcalml_b200.norm_rotate_op import NormRotate
    q, w, pos, grad = inputs(90, 4, dim, dtype, 1, torch.float32, cuda, 3)
    want, _ = NormRotate(q, None, w, None, pos)
    joint = torch.cat([q, q, q], 1)
    odd = torch.zeros((90, 4, dim + 3), dtype=q.dtype, device=cuda)
    odd[..., 1:dim + 1] = q
    flipped = q.permute(2, 0, 1).contiguous().permute(1, 2, 0)
    by_head = q.transpose(0, 1).contiguous().transpose(0, 1)
    for x in (joint[:, 4:8], odd[..., 1:dim + 1], flipped, by_head):
        x = x.detach().requires_grad_(True)
        y, _ = NormRotate(x, None, w, None, pos)
        ref = reference(q, w, pos, dim // 2 * 2, False, 10000., 1e-6, grad)
        assert y.is_contiguous()
        assert_near(y, ref[0], "y")
        assert_near(torch.autograd.grad(y, x, grad)[0], ref[1], "dx")
    one = q[:1].expand(90, -1, -1)
    assert_near(NormRotate(one, None, w, None, pos)[0], reference(one, w, pos, dim // 2 * 2, False, 10000., 1e-6)[0], "one row for all")
    two = torch.stack([pos, pos], 2)[..., 0]
    assert torch.equal(NormRotate(q, None, w, None, two)[0], want)


def test_far_positions_and_odd_values(cuda):
    from hgcalml_b200.norm_rotate_op import NormRotate
    x, w, _, _ = inputs(6, 2, 64, "float", 0, torch.int64, cuda, 4)
    pos = torch.tensor([2 ** 40 + 1, -2 ** 40, 2 ** 31 - 1, -2 ** 31, 0, 123456789], device=cuda)
    # an angle of 2^40 is known to 2^-13 in double; that of the reference as well
    got, want = NormRotate(x, None, w, None, pos)[0], reference(x, w, pos, 64, False, 10000., 1e-6)[0]
    assert ((got.double() - want[0]).abs() <= want[1] + 2. ** -11 * want[0].abs().max()).all()
    assert_near(got[2:], (want[0][2:], want[1][2:] + 2. ** -20 * want[0].abs().max()), "31 bits")
    zero, _ = NormRotate(torch.zeros_like(x), None, w, None, pos)
    assert (zero == 0).all()
    bad = x.clone()
    bad[1, 0, 3] = float("nan")
    bad[2, 1, 60] = float("inf")
    y, _ = NormRotate(bad, None, w, None, pos)
    assert y[1, 0].isnan().all() and torch.equal(y[1, 1], got[1, 1]) and torch.equal(y[0], got[0]) and torch.equal(y[2, 0], got[2, 0])
    small = NormRotate((x * 1e-22), None, None, None, None)[0]
    assert small.isfinite().all()


def test_repeated_captured_and_concurrent_calls(cuda):
    from hgcalml_b200.norm_rotate_op import NormRotate
    q, wq, pq, gq = inputs(3000, 8, 64, "bfloat", 3, torch.float32, cuda, 5)
    k, wk, pk, gk = inputs(5000, 2, 64, "bfloat", 3, torch.float32, cuda, 6)

    def step():
        leaves = [t.detach().requires_grad_(True) for t in (q, k, wq, wk)]
        out = NormRotate(*leaves, pq, pk, rotary_dim=48)
        return [o.detach() for o in out] + list(torch.autograd.grad(out, leaves, (gq, gk)))

    want = step()
    torch.cuda.synchronize()
    streams, results = [torch.cuda.Stream() for _ in range(3)], []
    for s in streams:
        with torch.cuda.stream(s):
            results.append(step())
    torch.cuda.synchronize()
    for r in results + [step()]:
        assert all(torch.equal(a, b) for a, b in zip(r, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, z = NormRotate(q, k, wq, wk, pq, pk, rotary_dim=48)
    y.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want[0]) and torch.equal(z, want[1])


def test_gradients_are_those_of_differences(cuda):
    from hgcalml_b200.norm_rotate_op import NormRotate
    x, w, pos, grad = inputs(5, 2, 12, "float", 2, torch.float32, cuda, 7)
    x, w = x.requires_grad_(True), w.requires_grad_(True)
    dx, dw = torch.autograd.grad(NormRotate(x, None, w, None, pos)[0], (x, w), grad)
    g = torch.Generator(device=cuda).manual_seed(1)
    for t, d in ((x, dx), (w, dw)):
        step, h = torch.randn(t.shape, generator=g, device=cuda), 2. ** -6
        value = [(NormRotate(*[(u + s * h * step if u is t else u).detach() for u in (x,)], None, (w + s * h * step if t is w else w).detach(), None,
                             pos)[0].double() * grad.double()).sum() for s in (1., -1.)]
        exact = (d.double() * step.double()).sum()
        assert abs(float((value[0] - value[1]) / (2 * h) - exact)) <= 1e-2 * (1 + float((d.double() * step.double()).abs().sum()))


def test_offsets_beyond_32_bits(cuda):
    from hgcalml_b200.norm_rotate_op import NormRotate
    n = 4_300_000
    x = torch.ones((n, 4, 128), dtype=torch.bfloat16, device=cuda)  # 2.2e9 elements
    g = torch.Generator(device=cuda).manual_seed(3)
    x[-9:] = torch.randn((9, 4, 128), generator=g, device=cuda).to(x.dtype)
    pos = torch.arange(n, device=cuda)
    y, _ = NormRotate(x, None, None, None, pos)
    for rows in (slice(0, 9), slice(n - 9, n)):
        assert_near(y[rows], reference(x[rows], None, pos[rows], 128, False, 10000., 1e-6)[0], "far rows")


@pytest.mark.parametrize("dtype", ["float", "bfloat"])
def test_more_rows_than_the_chip_holds(cuda, dtype):
    from hgcalml_b200.norm_rotate_op import NormRotate
    q, wq, pq, gq = inputs(90001, 8, 32, dtype, 4, torch.float32, cuda, 8)
    k, wk, pk, gk = inputs(30011, 1, 32, dtype, 4, torch.float32, cuda, 9)
    leaves = [t.requires_grad_(True) for t in (q, k, wq, wk)]
    out = NormRotate(*leaves, pq, pk)
    got = out + torch.autograd.grad(out, leaves, (gq, gk))
    want_q, want_k = (reference(x.detach(), w.detach(), p, 32, False, 10000., 1e-6, g) for x, w, p, g in ((q, wq, pq, gq), (k, wk, pk, gk)))
    for i, name in enumerate(("y", "dx", "dw")):
        assert_near(got[2 * i].detach(), want_q[i], "queries " + name)
        assert_near(got[2 * i + 1].detach(), want_k[i], "keys " + name)


def test_without_an_eps(cuda):
    """Nothing but the rows' own squares under the root; groups of lanes that have no row divide by zero, which is no one's concern."""
    from hgcalml_b200.norm_rotate_op import NormRotate
    x, w, pos, grad = inputs(7, 3, 64, "bfloat", 1, torch.float32, cuda, 11)
    leaves = [t.requires_grad_(True) for t in (x, w)]
    y, _ = NormRotate(leaves[0], None, leaves[1], None, pos, eps=0.)
    dx, dw = torch.autograd.grad(y, leaves, grad)
    want = reference(x.detach(), w.detach(), pos, 64, False, 10000., 0., grad)
    for got, ref, name in zip((y.detach(), dx, dw), want, ("y", "dx", "dw")):
        assert_near(got, ref, name)
