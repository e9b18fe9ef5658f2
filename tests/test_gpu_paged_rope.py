"""RoPE settings of the paged cache at the edges of what the contiguous one takes, on the GPU."""
import numpy as np
import pytest

import jxai_b200 as jx
from tests.paged_model import Model
from tests.test_gpu_paged import cuda

pytestmark = pytest.mark.gpu


def keys_after(rope_dim, base, neox, hd=64, n=20, factors=None):
    """Keys that a prompt of n tokens leaves in a paged cache, and the call's k."""
    import torch
    cache = jx.PagedKVCache(1, 1, 64, 1, hd, dtype="int8")
    rng = np.random.default_rng(rope_dim)
    q, k, v = (rng.standard_normal((n, 1, hd)).astype(np.float32) for _ in range(3))
    out = torch.zeros(n, 1, hd, device="cuda")
    jx.attn_prefill(cache, [jx.Layer(hd, rope_dim, base, 0, rope_freqs=factors)], *(cuda(x) for x in (q, k, v)),
                    out, range(n), 1, 1, neox=neox)
    assert np.isfinite(out.cpu().numpy()).all()
    return cache.read([0], [0], n, dtype=torch.float32)[0, 0, 0].cpu().numpy(), k


@pytest.mark.parametrize("neox", [False, True])
@pytest.mark.parametrize("rope_dim", [3, 33, 63, 64, 65])
def test_odd_numbers_of_rotated_dims(rope_dim, neox):
    """Frequencies are powers of -2 j / rope_dim, an odd one too, over rope_dim // 2 pairs."""
    got, k = keys_after(rope_dim, 1e4, neox)
    rd = min(64, rope_dim)
    j = np.arange(rd // 2)
    a = np.arange(20)[:, None] * 1e4 ** (-2.0 * j / rd)
    c, s = np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)
    u, w = (j, j + rd // 2) if neox else (2 * j, 2 * j + 1)
    x = k[:, 0].copy()
    x[:, u], x[:, w] = k[:, 0][:, u] * c - k[:, 0][:, w] * s, k[:, 0][:, u] * s + k[:, 0][:, w] * c
    m = Model(1, 1, 64, 1, 64, "int8")
    m.write(0, 0, 0, 0, x[:, None])
    assert np.array_equal(got.astype(np.float64), m.values(0, 0, 0, 0, 20))


@pytest.mark.parametrize("rope_dim", [0, 1])
@pytest.mark.parametrize("base", [0.0, -1.0, float("nan")])
def test_a_layer_without_rotation_needs_no_base(rope_dim, base):
    got, k = keys_after(rope_dim, base, True)
    m = Model(1, 1, 64, 1, 64, "int8")
    m.write(0, 0, 0, 0, k)
    assert np.array_equal(got.astype(np.float64), m.values(0, 0, 0, 0, 20))
