"""Workspaces of the attention between ragged sets: what the sizes need, and not many times that."""
import random

SMS = 148  # of a B200; what the library takes where there is no device


def test_workspaces_are_no_larger_than_their_parts():
    """Forward: float32 parts of rows, dim + 1 values each.  A split gives a multiprocessor at most 8 blocks of 64 rows, 6 of 256 (twice as many
    parts of 128) or 20 of 8; two parts of every row where events fit half a tile.  Backward: of each row 8 bytes and in half precision 4 more, of each event 12, and parts of dq and of dk
    and dv: 20 blocks of 64 rows, or 4 of 128.  Sixteen tensors' alignment on top."""
    from hgcalml_b200 import _capi
    L = _capi.lib
    rng = random.Random(3)
    for _ in range(3000):
        kv = rng.choice([1, 2, 3, 8])
        heads, dim, dtype = kv * rng.choice([1, 2, 5, 32, 40]), rng.randint(1, 128), rng.randint(0, 2)
        n_q, n_k = (int(10 ** rng.uniform(0, 7)) - 1 for _ in range(2))
        n_rs = int(10 ** rng.uniform(0, 4))
        size = n_q, n_k, n_rs, heads, kv, dim, dtype
        rows = n_q * heads
        parts = max(SMS * max(8 * 64, 2 * 6 * 256, 20 * 8), 2 * rows)
        assert 512 <= L.hgc_cross_attention_workspace_bytes(*size) <= 16 * 256 + 4 * (dim + 1) * parts
        parts = SMS * max(20 * 64, 4 * 128)
        most = 16 * 256 + 8 * rows + (4 * rows if dtype == 1 else 0) + 12 * n_rs + 3 * 4 * dim * parts
        least = 8 * rows + (4 * rows if dtype == 1 else 0) + 12 * (n_rs - 1)
        assert least <= L.hgc_cross_attention_grad_workspace_bytes(*size) <= most, size
