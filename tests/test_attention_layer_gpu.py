"""Projection, norm and rotation, attention and output transform together, as the layer calls them."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def _rows(n, width, dev, seed, dtype):
    return torch.randn((n, width), generator=torch.Generator(device=dev).manual_seed(seed), device=dev).to(dtype)


def _splits(sizes, dev):
    return torch.tensor(np.concatenate([[0], np.cumsum(sizes)]), dtype=torch.int32, device=dev)


def _plain(layer, x, context, nq, nk, pq, pk, mask):
    """The layer from elementary operations in 64 bits, differentiable."""
    f = lambda t: t.double()  # noqa: E731
    dim, heads, kv = layer.n_head_features, layer.n_heads, layer.n_key_heads

    def norm(t, w):
        return t / torch.sqrt(t.square().mean(-1, keepdim=True) + 1e-6) * f(w)

    def turn(t, pos):
        axes = pos.shape[1]
        pairs = dim // (2 * axes)
        theta = f(pos)[:, :, None] * layer.how["base"] ** (-torch.arange(pairs, device=t.device).double() / pairs)
        t = t[..., :2 * axes * pairs].unflatten(-1, (axes, 2, pairs))
        c, s = torch.cos(theta)[:, None], torch.sin(theta)[:, None]
        return torch.stack([t[..., 0, :] * c - t[..., 1, :] * s, t[..., 1, :] * c + t[..., 0, :] * s], -2).flatten(-3)

    q = (f(x) @ f(layer.query_transform.kernel) + f(layer.query_transform.bias)).unflatten(-1, (heads, dim))
    both = (f(context) @ f(layer.context_transform.kernel) + f(layer.context_transform.bias)).unflatten(-1, (2, kv, dim))
    q, k, v = turn(norm(q, layer.query_scale), pq), turn(norm(both[:, 0], layer.key_scale), pk), both[:, 1]
    k, v = (t.repeat_interleave(heads // kv, 1) for t in (k, v))
    out, a, b = [], 0, 0
    for n, m in zip(nq, nk):
        s = torch.einsum("nhd,mhd->hnm", q[a:a + n], k[b:b + m]) * dim ** -0.5
        s = s.masked_fill(~mask[b:b + m], -float("inf"))
        p = torch.softmax(s, -1) if m and mask[b:b + m].any() else torch.zeros_like(s)
        out.append(torch.einsum("hnm,mhd->nhd", p, v[b:b + m]))
        a, b = a + n, b + m
    return torch.cat(out).flatten(1) @ f(layer.output_transform.kernel) + f(layer.output_transform.bias)


# The layer rounds its intermediate results (projections, turned rows, attention, output) to its type: five roundings of up to u
# on the way to the result and as many on the way back, each of a quantity whose size is that of the result, here allowed twice.
@pytest.mark.parametrize("dtype,tol", [(torch.float32, 2e-5), (torch.bfloat16, 20 * 2. ** -8), (torch.float16, 20 * 2. ** -11)])
@pytest.mark.parametrize("kv", [4, 2])
def test_layer_and_its_gradients(cuda, dtype, tol, kv):
    from hgcalml_b200.AttentionLayersRagged import RaggedCrossAttention
    torch.manual_seed(3)
    nq, nk = [50, 0, 170, 1], [400, 7, 33, 0]
    layer = RaggedCrossAttention(4, 32, 24, n_in=20, n_context=28, n_key_heads=kv).to(cuda).to(dtype)
    x, context = _rows(sum(nq), 20, cuda, 1, dtype).requires_grad_(True), _rows(sum(nk), 28, cuda, 2, dtype).requires_grad_(True)
    pq, pk = 5. * _rows(sum(nq), 4, cuda, 3, torch.float32), 5. * _rows(sum(nk), 4, cuda, 4, torch.float32)
    mask = torch.ones(sum(nk), dtype=torch.bool, device=cuda)
    mask[::7] = False
    rs = _splits(nq, cuda), _splits(nk, cuda)
    y = layer([x, context, *rs], pq, pk, key_mask=mask)
    grad = _rows(*y.shape, cuda, 5, dtype)
    inputs = [x, context] + list(layer.parameters())
    got = torch.autograd.grad(y, inputs, grad)
    want = _plain(layer, x, context, nq, nk, pq, pk, mask)
    ref = torch.autograd.grad(want, inputs, grad.double())
    assert y.dtype == dtype and (y.double() - want).norm() <= tol * want.norm()
    for g, r, t in zip(got, ref, inputs):
        assert g.shape == t.shape and (g.double() - r.double()).norm() <= tol * r.double().norm() + 1e-30
    # a context that was prepared ahead of time
    with torch.no_grad():
        ahead = layer([x, layer.prepare(context, pk), *rs], pq, key_mask=mask)
        assert torch.equal(ahead, layer([x, context, *rs], pq, pk, key_mask=mask))
    with pytest.raises(RuntimeError):
        layer([x, layer.prepare(context, pk), *rs], pq, pk)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_captured_step(cuda, dtype):
    """Forward and gradients in one graph, replayed on other inputs, with other lengths, and beside an eager step on another stream."""
    from hgcalml_b200.AttentionLayersRagged import RaggedCrossAttention
    torch.manual_seed(5)
    layer = RaggedCrossAttention(4, 32, 24, n_in=20, n_context=28, n_key_heads=2).to(cuda).to(dtype)

    def inputs(seed, nq, nk):
        return [_rows(300, 20, cuda, seed, dtype), _rows(900, 28, cuda, seed + 1, dtype), _splits(nq, cuda), _splits(nk, cuda),
                5. * _rows(300, 4, cuda, seed + 2, torch.float32), 5. * _rows(900, 4, cuda, seed + 3, torch.float32), _rows(300, 24, cuda, seed + 4, dtype)]

    def step(x, context, rs_q, rs_k, pq, pk, grad):
        x, context = x.detach().requires_grad_(True), context.detach().requires_grad_(True)
        y = layer([x, context, rs_q, rs_k], pq, pk)
        return [y.detach()] + list(torch.autograd.grad(y, [x, context] + list(layer.parameters()), grad))

    first, second = inputs(11, [100, 0, 200], [500, 300, 100]), inputs(21, [1, 150, 40], [30, 0, 800])
    static = [t.clone() for t in first]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(*static)
    for given in (first, second, first):
        want = step(*given)
        for s, g in zip(static, given):
            s.copy_(g)
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            beside = step(*given)
        torch.cuda.synchronize()
        # our kernels give the same every time; products of the dense layers may be taken another way under capture
        for a, b, c in zip(held, want, beside):
            tol = 20 * torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 2e-5
            assert (a.double() - b.double()).norm() <= tol * b.double().norm() and (c.double() - b.double()).norm() <= tol * b.double().norm()


def test_one_new_query_after_the_other(cuda):
    """As a service asks them: the context is prepared once, and queries come one per event."""
    from hgcalml_b200.AttentionLayersRagged import RaggedCrossAttention
    torch.manual_seed(4)
    nk = [700, 3000, 5]
    layer = RaggedCrossAttention(8, 64, 16, n_in=32, n_context=32, n_key_heads=2).to(cuda).to(torch.bfloat16)
    context, rs_k = _rows(sum(nk), 32, cuda, 1, torch.bfloat16), _splits(nk, cuda)
    x = _rows(12, 32, cuda, 2, torch.bfloat16)
    with torch.no_grad():
        ready = layer.prepare(context, torch.arange(sum(nk), device=cuda))
        steps = [layer([x[3 * i:3 * i + 3].contiguous(), ready, _splits([1, 1, 1], cuda), rs_k], torch.full((3,), 1000 + i, device=cuda)) for i in range(4)]
        order = torch.arange(12, device=cuda).reshape(4, 3).T.reshape(-1)
        together = layer([x[order], ready, _splits([4, 4, 4], cuda), rs_k], 1000 + torch.arange(12, device=cuda) % 4)
    got = torch.stack(steps).transpose(0, 1).reshape(12, 16)
    # other numbers of rows may take other kernels: the roundings of weights, attention and output
    assert (got.double() - together.double()).norm() <= 3 * 2. ** -8 * together.double().norm()
