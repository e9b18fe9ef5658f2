"""Values at the edges of what the paged cache's attention takes, on the GPU, compared with the
plain 64-bit model or with what the values say by themselves."""
import numpy as np
import pytest

import jxai_b200 as jx
from tests.test_gpu_paged import Pair, cuda

pytestmark = pytest.mark.gpu


def attend(p, s, pos0, q, k, v, prompt, scale=None):
    """Outputs [n, layers, H, HD] of tokens pos0 .. of sequence s; `out` starts as NaN."""
    import torch
    n = len(q)
    wide = [cuda(x) for x in (q, k, v)]
    out = torch.full_like(wide[0], float("nan"))
    (jx.attn_prefill if prompt else jx.attn_step)(
        p.cache, p.layers, *wide, out, list(range(pos0, pos0 + n)), p.H, p.HK,
        scale=p.scale if scale is None else scale, softcap=p.softcap, sliding_window=p.window,
        neox=p.kw["neox"], seq_ids=[s] * n)
    torch.cuda.synchronize()
    assert p.cache.check_device_error() == 0
    return out.cpu().numpy().reshape(n, p.L, p.H, p.HD)


def expect(p, s, l, pos0, q, k, v):
    """The model's outputs and bounds [n, H, HD] for layer l."""
    n = len(q)
    with np.errstate(all="ignore"):
        ref, tol = p.model.step(s, l, pos0, q[:, l], k[:, l], v[:, l], p.H, p.scale, p.softcap,
                                p.window if p.swa[l] else 0, **p.kw)
    return ref.reshape(n, p.H, p.HD), tol.reshape(n, p.H, p.HD)


SHAPES = [(4, 1, 64), (2, 2, 64), (7, 1, 64), (4, 2, 128), (8, 1, 128), (4, 1, 256), (3, 1, 32)]


@pytest.mark.parametrize("tc", [0, 1])
@pytest.mark.parametrize("size", [np.inf, -np.inf, 2.0 ** 30, -2.0 ** 44])
@pytest.mark.parametrize("H,HK,HD", SHAPES)
def test_a_query_does_not_reach_other_heads_and_tokens(H, HK, HD, size, tc):
    """One token's query of one head is infinite or far larger than the rest: every other head and
    token keeps the model's value, within the model's bound (which is the head's own)."""
    p = Pair(H, HK, HD, "int8", cap=64, seed=H + HD, tc=tc)
    q, k, v = p.inputs(30)
    h, at = H - 1, 21
    qh = q.reshape(30, 1, H, HD)
    if np.isinf(size):
        qh[at, 0, h, 3] = size
    else:
        qh[at, 0, h] *= np.float32(size)
    got = attend(p, 0, 0, q, k, v, True)
    ref, tol = expect(p, 0, 0, 0, q, k, v)
    ok = np.ones((30, H), bool)
    ok[at, h] = False
    assert (np.abs(got[:, 0] - ref) <= tol)[ok].all()
    q, k, v = p.inputs(1)
    q.reshape(1, 1, H, HD)[0, 0, h, :2] = size
    got = attend(p, 0, 30, q, k, v, False)
    ref, tol = expect(p, 0, 0, 30, q, k, v)
    assert (np.abs(got[:, 0] - ref) <= tol)[0, :h].all()


@pytest.mark.parametrize("tc", [0, 1])
def test_small_queries_beside_large_ones_keep_their_bits(tc):
    """Queries of the heads of a group 2^24 apart."""
    p = Pair(4, 1, 64, "int8", cap=128, seed=2, tc=tc)
    q, k, v = p.inputs(100)
    # a head whose scores are ordinary, beside one whose scores are 2^24 times as large
    q.reshape(100, 1, 4, 64)[:, :, 1::2] *= np.float32(2.0 ** 24)
    got = attend(p, 0, 0, q, k, v, True)
    ref, tol = expect(p, 0, 0, 0, q, k, v)
    assert (np.abs(got[:, 0] - ref) <= tol)[:, ::2].all()
