"""What the Python calls take for positions and sequences."""
import numpy as np
import pytest

import jxai_b200 as jx
from jxai_b200.attention import _call_ints


@pytest.mark.filterwarnings("ignore::DeprecationWarning")
def test_positions_of_any_kind_that_int_takes():
    for x in ([3, 1], (3, 1), np.array([3, 1]), np.array([3.0, 1.0]), np.array([3, 1], np.uint8),
              np.array([[3], [1]]), [3.0, np.float32(1)], np.array([3.0, 1.0], np.float16)):
        assert list(_call_ints(x)) == [3, 1]
    assert list(_call_ints(np.array([True, False]))) == [1, 0]
    assert list(_call_ints(np.zeros(3))) == [0, 0, 0]
    assert list(_call_ints(range(100))) == list(range(100))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_contiguous_cache_takes_them(dtype):
    """Positions and sequences as arrays of floats, and sequences that are listed for the first rows
    alone (the others are rows of sequence 0): the same outputs as with lists of integers."""
    import torch
    H, HK, HD, n = 4, 2, 64, 9
    g = torch.Generator(device="cuda").manual_seed(0)
    q, k, v = (torch.randn(n, 1, h * HD, generator=g, device="cuda") for h in (H, HK, HK))
    layers = [jx.Layer(HD, HD, 1e4, 0)]

    def run(call, rows, pos, **kw):
        cache = jx.KVCache(3, 1, 32, HK * HD, dtype=dtype)
        out = torch.zeros_like(q[:rows])
        call(cache, layers, q[:rows], k[:rows], v[:rows], out, pos, H, HK, **kw)
        torch.cuda.synchronize()
        return out
    want = run(jx.attn_prefill, n, list(range(n)), seq_ids=[0] * n)
    assert torch.equal(want, run(jx.attn_prefill, n, np.arange(n, dtype=np.float64), seq_ids=[0]))
    assert torch.equal(want, run(jx.attn_prefill, n, np.arange(n), seq_ids=np.zeros(n)))
    want = run(jx.attn_step, 2, [0, 0], seq_ids=[2, 0])
    assert torch.equal(want, run(jx.attn_step, 2, np.zeros(2), seq_ids=[2]))
    assert torch.equal(want, run(jx.attn_step, 2, np.zeros(2, bool), seq_ids=np.array([2.0, 0.0])))
