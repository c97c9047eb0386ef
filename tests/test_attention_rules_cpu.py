"""What the attention between ragged sets, and norm and rotation, refuse: on the host, before anything runs on a device."""
import ctypes
import random

import pytest
import torch

NUL = ctypes.c_void_p(None)
F = ctypes.c_float


def _attend(L, n_q=4, n_k=6, n_rs=2, heads=2, kv=1, dim=8, strides=None, scale=1., dtype=0):
    return L.hgc_cross_attention(*[NUL] * 9, n_q, n_k, n_rs, heads, kv, dim, strides, F(scale), dtype, NUL, 0, NUL)


def _attend_grad(L, n_q=4, n_k=6, n_rs=2, heads=2, kv=1, dim=8, strides=None, scale=1., dtype=0):
    return L.hgc_cross_attention_grad(*[NUL] * 13, n_q, n_k, n_rs, heads, kv, dim, strides, F(scale), dtype, NUL, 0, NUL)


@pytest.mark.parametrize("call", [_attend, _attend_grad])
def test_attention_entries_check_their_arguments(call):
    from hgcalml_b200 import _capi
    L = _capi.lib
    inf, nan = float("inf"), float("nan")
    for bad in (dict(n_q=-1), dict(n_k=-1), dict(n_rs=0), dict(heads=0), dict(kv=0), dict(heads=3, kv=2), dict(dim=0), dict(dtype=3), dict(dtype=-1),
                dict(scale=0.), dict(scale=-1.), dict(scale=inf), dict(scale=nan), dict(strides=(ctypes.c_longlong * 6)(-1, 0, 0, 0, 0, 0))):
        assert call(L, **bad) == -1, bad
    for much in (dict(dim=129), dict(heads=65536, kv=65536), dict(n_q=2 ** 31 - 1), dict(n_k=2 ** 31 - 8192), dict(n_rs=2 ** 31 - 1)):
        assert call(L, **much) == -3, much
    assert call(L) == -1  # null tensors
    assert call(L, n_q=0, n_k=0) == 0  # nothing to do
    assert _attend(L, n_q=0) == 0


def test_attention_workspaces():
    from hgcalml_b200 import _capi
    L = _capi.lib
    for query in (L.hgc_cross_attention_workspace_bytes, L.hgc_cross_attention_grad_workspace_bytes):
        assert query(1, 1, 2, 1, 1, 129, 0) == 0 and query(-1, 1, 2, 1, 1, 8, 0) == 0 and query(1, 1, 2, 3, 2, 8, 0) == 0
        rng = random.Random(1)
        for _ in range(2000):  # any sizes, and no more than sixteen parts a multiprocessor of a block's results
            kv = rng.choice([1, 2, 3, 8])
            heads, dim = kv * rng.choice([1, 2, 5, 32, 40]), rng.randint(1, 128)
            n_q, n_k, n_rs = (int(10 ** rng.uniform(0, 7)) - 1 for _ in range(3))
            size = query(n_q, n_k, n_rs % 5000 + 1, heads, kv, dim, rng.randint(0, 2))
            assert 256 <= size <= 2 ** 40
    assert L.hgc_cross_attention_grad_workspace_bytes(10 ** 6, 10, 2, 8, 8, 64, 0) >= 8 * 8 * 10 ** 6


def _set(C, **kw):
    class Rows(ctypes.Structure):
        _fields_ = [("x", ctypes.c_void_p), ("w", ctypes.c_void_p), ("p", ctypes.c_void_p), ("y", ctypes.c_void_p), ("gy", ctypes.c_void_p),
                    ("gx", ctypes.c_void_p), ("gw", ctypes.c_void_p), ("row", ctypes.c_longlong), ("head", ctypes.c_longlong), ("n", ctypes.c_int),
                    ("heads", ctypes.c_int), ("wt", ctypes.c_int)]
    r = Rows()
    r.n, r.heads, r.row, r.head = 0, 1, 8, 8
    for k, v in kw.items():
        setattr(r, k, v)
    return ctypes.byref(r)


def test_norm_rotate_entries_check_their_arguments():
    from hgcalml_b200 import _capi
    L = _capi.lib

    def call(r=None, sets=1, dim=8, rotary=8, axes=1, kind=0, base=1e4, eps=1e-6, dtype=0):
        r = r or _set(_capi)
        d = ctypes.c_double(base)
        return (L.hgc_norm_rotate(r, sets, dim, rotary, axes, kind, 0, d, F(eps), dtype, NUL),
                L.hgc_norm_rotate_grad(r, sets, dim, rotary, axes, kind, 0, d, F(eps), dtype, NUL, 0, NUL))

    assert call()[0] == 0  # no rows
    for bad in (dict(sets=0), dict(sets=3), dict(dim=0), dict(rotary=-2), dict(rotary=10), dict(rotary=7), dict(axes=0), dict(axes=3), dict(kind=3),
                dict(base=1.), dict(base=float("nan")), dict(eps=-1.), dict(eps=float("nan")), dict(dtype=3), dict(r=_set(_capi, n=-1)),
                dict(r=_set(_capi, heads=0)), dict(r=_set(_capi, row=-1)), dict(r=_set(_capi, n=3)), dict(r=_set(_capi, w=1, wt=2))):
        assert call(**bad) == (-1, -1), bad
    assert call(dim=129, rotary=8) == call(r=_set(_capi, n=2 ** 31 - 1)) == call(r=_set(_capi, heads=65536)) == (-3, -3)
    assert L.hgc_norm_rotate(None, 1, 8, 8, 1, 0, 0, ctypes.c_double(1e4), F(0.), 0, NUL) == -1
    assert L.hgc_norm_rotate_grad_workspace_bytes(_set(_capi, n=1000, heads=3), 1, 64) > 256


def test_python_layer_takes_cuda_tensors_only():
    from hgcalml_b200 import _capi as C
    from hgcalml_b200.AttentionLayersRagged import RaggedCrossAttention
    from hgcalml_b200.cross_attention_op import CrossAttention
    from hgcalml_b200.norm_rotate_op import NormRotate
    q, rs = torch.zeros(4, 2, 8), torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(C.HgcError):
        CrossAttention(q, q, q, rs, rs)
    with pytest.raises(C.HgcError):
        NormRotate(q)
    layer = RaggedCrossAttention(4, 8, 12, n_in=5, n_context=6, n_key_heads=2)
    assert layer.context_transform.kernel.shape == (6, 32) and layer.output_transform.kernel.shape == (32, 12)
    with pytest.raises(ValueError):
        RaggedCrossAttention(4, 8, 12, n_in=5, n_context=6, n_key_heads=3)


def test_tiles_of_ragged_batches():
    """The arithmetic by which blocks find their rows, as the kernels do it: every row of every event in one tile, none in two, and
    every access inside the tensor whatever the splits hold."""
    def find(rs, n, rows, tile):
        events = len(rs) - 1
        at = lambda i: min(max(rs[i], 0), n)  # noqa: E731
        lo, hi = 0, events + 1
        while hi - lo > 1:
            step = (hi - lo + 31) // 32
            votes = [lo + l * step < hi and at(lo + l * step) // rows + lo + l * step <= tile for l in range(32)]
            ahead = max(votes.index(False) if False in votes else 32, 1)
            lo += (ahead - 1) * step
            hi = min(lo + step, hi)
        first, last = at(lo), at(lo + 1) if lo < events else n
        begin = first + (tile - first // rows - lo) * rows
        begin = last if begin < 0 or begin > last else begin
        return lo, begin, min(last, begin + rows)

    rng = random.Random(2)
    for _ in range(300):
        sizes = [rng.choice([0, 1, rng.randint(0, 40), rng.randint(0, 400)]) for _ in range(rng.choice([0, 1, 3, 40, 100]))]
        rs = [0]
        for s in sizes:
            rs.append(rs[-1] + s)
        n, rows = rs[-1] + rng.choice([0, 0, 5, 300]), rng.choice([1, 4, 21, 64, 128])
        owner = [None] * n
        for tile in range(n // rows + len(sizes) + 1):
            e, begin, end = find(rs, n, rows, tile)
            for r in range(begin, end):
                assert owner[r] is None and (rs[e] <= r < rs[e + 1] if e < len(sizes) else r >= rs[-1])
                owner[r] = e
        assert None not in owner
        bad = [rng.choice([-5, 0, n, n + 7, 2 ** 31 - 1, -2 ** 31, rng.randint(0, n + 1)]) for _ in rs]
        for tile in range(n // rows + len(sizes) + 1):
            e, begin, end = find(bad, n, rows, tile)
            assert 0 <= e <= len(sizes) and 0 <= begin <= n and end <= n
