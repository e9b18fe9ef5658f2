"""Values at the edges of what the paged cache's attention takes, on the GPU, compared with the
plain 64-bit model or with what the values say by themselves."""
import numpy as np
import pytest

import jxai_b200 as jx
from tests.paged_model import Model, rotate
from tests.test_gpu_paged import Pair, cuda, load_prompt

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


def far_case(rng, n, HD, H, HK, spread):
    """Keys that are one direction times 1, 0.5 or -1 (each block of 16 holds a 1), and values whose
    blocks are 2^-spread .. 2^spread large.  No rotation."""
    f = rng.choice([1.0, 0.5, -1.0], n)
    f[::16] = 1.0
    u = rng.standard_normal((HK, HD)).astype(np.float32)
    k = (f[:, None, None] * u).reshape(n, 1, HK * HD)
    v = rng.standard_normal((n, 1, HK * HD))
    v *= np.exp2(rng.integers(-spread, spread + 1, n // 16 + 1))[np.arange(n) // 16][:, None, None]
    q = rng.standard_normal((n, 1, H * HD))
    return f, u, [x.astype(np.float32) for x in (q, k, v)]


@pytest.mark.parametrize("tc", [0, 1])
@pytest.mark.parametrize("size", [1e4, 1e6, 2.0 ** 26, 1e12, 1e18, 1e24, 1e33])
@pytest.mark.parametrize("H,HK,HD,dtype", [(2, 1, 64, "int8"), (4, 2, 128, "e4m3"), (4, 1, 256, "int8"),
                                           (8, 4, 32, "e4m3"), (7, 1, 64, "e4m3")])
def test_scores_of_any_size(H, HK, HD, dtype, size, tc):
    """Scores so far apart that the largest wins alone, and several equal largest: the output is the
    mean of their values, whatever the scales of the blocks that these lie in."""
    rng = np.random.default_rng(int(np.log2(size)) + HD)
    n = 150
    f, u, (q, k, v) = far_case(rng, n, HD, H, HK, 10)
    G = H // HK
    # every query at an angle to the keys that keeps |q.u| near its largest
    q = np.sign(rng.standard_normal((n, 1, HK, G, 1))) * (u[:, None] + 0.1 * q.reshape(n, 1, HK, G, HD))
    q = (q * np.float32(size)).astype(np.float32).reshape(n, 1, H * HD)
    p = Pair(H, HK, HD, dtype, cap=256, seed=1, tc=tc, rope_dim=0)

    def check(got, at, q):
        V = p.model.values(0, 0, 1, 0, at + len(got))
        for i in range(len(got)):
            for h in range(H):
                g = h // G
                s = np.sign(q[i].reshape(H, HD)[h].astype(np.float64) @ u[g])
                x = s * f[:at + i + 1]
                w = x == x.max()
                want = V[:at + i + 1, g][w].mean(0)
                # Weights of equal scores: 2^-22 from exp2 and 2^-22 as two fp16 parts; what the
                # second part loses below the largest weight, 2^-25 each; the sums over rows, one
                # rounding (2^-23) per 16 rows and a few more.
                tol = np.abs(V[:at + i + 1, g][w]).max() * (2.0 ** -21 + (at + i + 1) * 2.0 ** -25
                                                           + ((at + i + 1) / 16 + 4) * 2.0 ** -23)
                assert (np.abs(got[i, 0, h] - want) <= tol).all(), (i, h)
    got = attend(p, 0, 0, q, k, v, True)
    p.model.write(0, 0, 0, 0, k.reshape(n, HK, HD))
    p.model.write(0, 0, 1, 0, v.reshape(n, HK, HD))
    check(got, 0, q)
    f = np.append(f, 1.0)
    one = [q[:1], u.reshape(1, 1, HK * HD), v[-1:]]
    got = attend(p, 0, n, *one, False)
    p.model.write(0, 0, 0, n, u.reshape(1, HK, HD))
    p.model.write(0, 0, 1, n, v[-1:].reshape(1, HK, HD))
    check(got, n, one[0])


@pytest.mark.parametrize("dtype", ["int8", "e4m3"])
def test_far_scores_over_a_split_segment(dtype):
    """A long row whose parts are joined over CTAs: equal far scores count alike, and a part without
    any of the largest counts for nothing."""
    rng = np.random.default_rng(5)
    n, HD = 6000, 64
    f, u, (_, k, v) = far_case(rng, n, HD, 1, 1, 8)
    f[:2000] = np.where(f[:2000] == 1.0, 0.5, f[:2000])  # the first third holds none of the largest
    f[:2000:16] = -1.0
    k = (f[:, None, None] * u).reshape(n, 1, HD).astype(np.float32)
    p = Pair(1, 1, HD, dtype, cap=6016, seed=1, rope_dim=0)
    load_prompt(p, 0, (None, k, v))
    V = p.model.values(0, 0, 1, 0, n)[:, 0]
    w = f == 1.0
    for size in (1.0, 2.0 ** 20, 2.0 ** 27, 2.0 ** 60):
        q = (u * np.float32(size * 30)).reshape(1, 1, HD)
        # a new key that scores least, dropped again
        got = attend(p, 0, n, q, -u.reshape(1, 1, HD), v[:1], False)[0, 0, 0]
        p.cache.rollback(0, n)
        # the largest score is at least 30 |u|^2 / 8 / 2 above the next: e^-100 and less of the rest
        tol = np.abs(V[w]).max() * (2.0 ** -21 + n * 2.0 ** -25 + (n / 16 + 4) * 2.0 ** -23)
        assert (np.abs(got - V[w].mean(0)) <= tol).all(), size


@pytest.mark.parametrize("tc", [0, 1])
@pytest.mark.parametrize("window", [1, 40, 3000, 0])
@pytest.mark.parametrize("size", [30.0, 2.0 ** 24, 2.0 ** 50])
def test_far_scores_of_blocks_with_windows(size, window, tc):
    """Tokens whose windows begin and end inside pages, behind rows that several CTAs read: pages and
    parts without rows for some of the tokens, scores near zero and far from it."""
    rng = np.random.default_rng(window)
    n, more, HD, H = 3000, 21, 64, 2
    f, u, (_, k, v) = far_case(rng, n + more, HD, H, 1, 6)
    p = Pair(H, 1, HD, "int8", cap=3040, seed=1, tc=tc, rope_dim=0, swa=[window > 0], window=window)
    load_prompt(p, 0, (None, k[:n], v[:n]))
    at = n - n % 16
    f[at:] = np.where(np.arange(at, n + more) % 16 == 0, 1.0, f[at:])
    k[at:] = (f[at:, None, None] * u).reshape(-1, 1, HD)
    p.cache.rollback(0, at)
    q = (np.array([1.0, -1.0])[None, None, :, None] * u[:, None] * size).astype(np.float32)
    q = np.ascontiguousarray(np.broadcast_to(q, (n + more - at, 1, H, HD))).reshape(-1, 1, H * HD)
    got = attend(p, 0, at, q, k[at:], v[at:], True)[:, 0]
    p.model.write(0, 0, 0, at, k[at:].reshape(-1, 1, HD))
    p.model.write(0, 0, 1, at, v[at:].reshape(-1, 1, HD))
    V = p.model.values(0, 0, 1, 0, n + more)[:, 0]
    for i, pos in enumerate(range(at, n + more)):
        lo = max(0, pos - window + 1) if window else 0
        for h in range(H):
            x = (1.0, -1.0)[h] * f[lo:pos + 1]
            won = V[lo:pos + 1][x == x.max()]
            # the next score is 30 |u|^2 / 16 = 100 or more below: e^-100 of the rest
            m = pos + 1 - lo
            tol = np.abs(won).max() * (2.0 ** -21 + m * 2.0 ** -25 + (m / 16 + 4) * 2.0 ** -23)
            assert (np.abs(got[i, h] - won.mean(0)) <= tol).all(), (pos, h)


@pytest.mark.parametrize("flip", [False, True])
@pytest.mark.parametrize("at,up,down", [(0, 6, -6), (2 ** 21, 6, -6), (2 ** 22, 6, -6), (2 ** 22, 3, -12),
                                        (2 ** 22, 13, 2), (-2 ** 22, 2, -9)])
def test_parts_on_both_sides_of_far_scores(at, up, down, flip):
    """Scores of -at + up and -at + down (in powers of two) in the two halves of a long row, the
    lower ones with larger values: parts whose sums are taken against references near zero and far
    from it count alike."""
    n, HD = 6000, 64
    j = np.where((np.arange(n) < n // 2) ^ flip, float(up), float(down))
    k, v = np.zeros((n, 1, HD), np.float32), np.random.default_rng(abs(at)).standard_normal((n, 1, HD))
    k[:, 0, 0], k[:, 0, 1] = 64.0, j
    v = (v * np.where(j == up, 2.0 ** 13, 2.0 ** 25)[:, None, None]).astype(np.float32)
    p = Pair(1, 1, HD, "int8", cap=6016, seed=1, rope_dim=0)
    load_prompt(p, 0, (None, k, v))
    K, V = (p.model.values(0, 0, w, 0, n)[:, 0] for w in range(2))
    assert np.array_equal(K[:, :2], k[:, 0, :2])
    q, new = np.zeros((1, 1, HD), np.float32), np.zeros((1, 1, HD), np.float32)
    q[0, 0, :3] = -at / 64, 1.0, -1.0
    new[0, 0, :3] = 64.0, 0.0, 100.0  # the new row's score: -at - 100
    # times log2(e) in fp32, the scale is 1: every score a whole number
    scale = np.float32(np.log(2))
    assert np.float32(scale * np.float32(1.4426950408889634)) == 1.0
    got = attend(p, 0, n, q, new, v[:1], False, scale=float(scale))[0, 0, 0]
    w = np.exp2(j - up)
    want = (w @ V) / w.sum()
    # a weight, in the sum of values and in that of weights: 2^-22 from exp2, 2^-22 as two parts;
    # each sum over rows: one rounding (2^-23) per 16 rows and a few more
    tol = (w @ np.abs(V)) / w.sum() * 2 * (2.0 ** -21 + (n / 16 + 8) * 2.0 ** -23)
    assert (np.abs(got - want) <= tol).all(), np.abs(got / want - 1).max()


class Clipped(Model):
    """The model with values cut at `top`, as prompts on the tensor cores take them."""
    top = np.inf

    def values(self, *a):
        return np.clip(super().values(*a), -self.top, self.top)


@pytest.mark.parametrize("tc", [0, 1])
@pytest.mark.parametrize("dtype", ["int8", "e4m3"])
def test_rows_with_infinities_count_as_they_are_held(dtype, tc):
    """NaN, infinities, huge and tiny values and blocks of zeros in K and V: every output is the
    model's, over the rows as they are held."""
    p = Pair(2, 1, 64, dtype, cap=128, seed=3, tc=tc)
    p.model = Clipped(1, 1, 128, 1, 64, dtype)
    if tc:
        # fp16 ends at 65504; the unit of a head's rows is at most 2^8 (int8) or 2^9
        p.model.top = 65504.0 * 2.0 ** (8 if dtype == "int8" else 9)
    q, k, v = p.inputs(60)
    k[0, 0, :8] = [np.nan, np.inf, -np.inf, 0, 1e30, -1e-40, 1e-30, 3e38]
    v[1, 0, :8] = [np.nan, np.inf, -np.inf, 0, 1e30, -1e-40, 1e-30, 3e38]
    k[16:32] = 0.0
    v[16:32] = 0.0
    q[0:16] = 0.0
    got = attend(p, 0, 0, q, k, v, True)[:, 0]
    ref, _ = expect(p, 0, 0, 0, q, k, v)
    V = np.abs(p.model.values(0, 0, 1, 0, 60)[:, 0])
    K = p.model.values(0, 0, 0, 0, 60)[:, 0]
    qr = rotate(q.reshape(60, 2, 64), np.arange(60), **p.kw).astype(np.float64)
    checked = 0
    for i in range(60):
        for h in range(2):
            e = K[:i + 1] @ qr[i, h] * p.scale
            if abs(e[0]) < 1e4 and abs(e[0]) > 1e-9:
                continue  # (the infinite row's score is not far from the others')
            # Scores but the first row's are ordinary: 64 products of 2^-21 and less.  Values
            # that lie more than 2^22 below the head's largest are rounded when an e4m3 row is
            # widened: by 2^-25 of the unit 2^9.
            wide = 2.0 ** -16 if tc and dtype == "e4m3" else 0.0
            ds = np.abs(qr[i, h]).sum() * p.scale * (wide + np.abs(K[1:i + 1]).max(initial=0.0) * 2.0 ** -20)
            tol = V[:i + 1].max(0) * (4 * ds + 2.0 ** -18) + wide
            assert (np.abs(got[i, h] - ref[i, h]) <= tol).all(), (i, h)
            checked += 1
    assert checked > 100


@pytest.mark.parametrize("tc", [0, 1])
@pytest.mark.parametrize("dtype,spread", [("int8", 30), ("e4m3", 20), ("e4m3", 30)])
def test_values_far_below_those_of_later_rows(dtype, spread, tc):
    """Tokens that attend small values alone, 2^spread below those of later rows: right to the last
    bit of their own size, as far as one fp16 unit per head holds both."""
    p = Pair(4, 1, 64, dtype, cap=256, seed=spread, tc=tc)
    q, k, v = p.inputs(200)
    v[:128] *= np.float32(2.0 ** -spread)
    got = attend(p, 0, 0, q, k, v, True)[:, 0]
    ref, tol = expect(p, 0, 0, 0, q, k, v)
    # e4m3 beyond 2^22: off by at most 2^-32 of the largest scale
    wide = 2.0 ** (p.model.k[0, 0, 1, :12].max() - 32) if tc and dtype == "e4m3" and spread > 22 else 0.0
    assert (np.abs(got - ref) <= tol + wide).all()


def test_a_scale_that_almost_vanishes():
    """Scores that underflow are zeros, not NaN where a later row is masked."""
    for tc in (0, 1):
        p = Pair(2, 1, 64, "int8", cap=256, seed=6, tc=tc)
        q, k, v = p.inputs(200)
        for scale in (1e-30, 1e-38, 1e-45):
            p.cache.clear(0)
            got = attend(p, 0, 0, q, k, v, True, scale=scale)[:, 0]
            p.model.write(0, 0, 1, 0, v.reshape(200, 1, 64))
            V = p.model.values(0, 0, 1, 0, 200)[:, 0]
            mean = np.cumsum(V, 0) / np.arange(1, 201)[:, None]
            tol = np.abs(V).max() * (2.0 ** -21 + 200 * 2.0 ** -25 + (200 / 16 + 4) * 2.0 ** -23)
            assert (np.abs(got - mean[:, None]) <= tol).all()


@pytest.mark.parametrize("dtype", ["int8", "e4m3"])
@pytest.mark.parametrize("H,HK,HD,rows", [(4, 1, 64, 1100), (8, 1, 64, 700), (2, 1, 128, 1700), (8, 1, 128, 2300)])
def test_prompts_behind_many_rows(H, HK, HD, rows, dtype):
    """Several partial sums of the tensor-core kernel are added up (every 4 or 6 tiles of 128 rows),
    the reference moving between them: keys that grow along the rows."""
    p = Pair(H, HK, HD, dtype, cap=rows + 100, seed=rows, tc=1)
    q, k, v = p.inputs(rows)
    k *= (0.05 + 6.0 * (np.arange(rows) / rows) ** 2).astype(np.float32)[:, None, None]
    load_prompt(p, 0, (q, k, v))
    p.run([(0, rows, 5)], True, spread=8.0)
    p.run([(0, rows + 5, 70)], True, spread=0.5)


@pytest.mark.parametrize("H", [8, 16])
def test_prompts_of_many_layers_behind_many_rows(H):
    """More fp16 rows than stay in L2 (items ordered by stream), more layers than one group takes,
    several items per CTA."""
    rows, L = 1150, 70
    p = Pair(H, 8, 64, "int8", L=L, cap=1184, seed=H, tc=1)
    x = p.inputs(rows)
    load_prompt(p, 0, x)
    p.run([(0, rows, 9)], True)
