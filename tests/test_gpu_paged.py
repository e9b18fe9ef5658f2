"""The paged 8-bit cache on the GPU against a plain 64-bit model: what it holds is
compared exactly, attention within a bound derived from 32-bit arithmetic."""
import math

import numpy as np
import pytest

import jxai_b200 as jx
from jxai_b200 import _lib
from tests.paged_model import Model

pytestmark = pytest.mark.gpu


def cuda(x):
    import torch
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


class Pair:
    """A cache and its model, driven together."""

    def __init__(self, H, HK, HD, dtype, n_seqs=1, L=1, cap=256, n_pages=None, seed=0, **kw):
        self.H, self.HK, self.HD, self.L = H, HK, HD, L
        self.cache = jx.PagedKVCache(n_seqs, L, cap, HK, HD, n_pages=n_pages, dtype=dtype)
        self.cache.set_option("prefill_tc", kw.get("tc", 1))
        self.model = Model(n_seqs, L, cap, HK, HD, dtype)
        self.rng = np.random.default_rng(seed)
        self.kw = dict(rope_dim=kw.get("rope_dim", HD), base=kw.get("base", 1e4), neox=kw.get("neox", True))
        self.kw_layer = {}  # layer -> RoPE settings of its own
        self.swa = kw.get("swa", [False] * L)
        self.window, self.softcap = kw.get("window", 0), kw.get("softcap", 0.0)
        self.shares = kw.get("shares", {})  # layer -> layer whose rows it reads
        self.layers = [jx.Layer(HD, self.kw["rope_dim"], self.kw["base"], self.shares.get(l, l),
                                is_swa=self.swa[l], shares_kv=l in self.shares) for l in range(L)]
        self.scale = 1.0 / math.sqrt(HD)

    def inputs(self, n, spread=1.0):
        r = self.rng
        q = r.standard_normal((n, self.L, self.H * self.HD))
        k, v = (r.standard_normal((n, self.L, self.HK * self.HD)) * spread for _ in range(2))
        return [x.astype(np.float32) for x in (q, k, v)]

    def run(self, jobs, prompt, spread=1.0, inputs=None, stream=None, pad=0):
        """jobs: (sequence, first position, tokens).  Runs both, checks outputs and rows."""
        import torch
        n = sum(j[2] for j in jobs)
        q, k, v = inputs or self.inputs(n, spread)
        seqs = [s for s, p, m in jobs for _ in range(m)]
        pos = [p + i for s, p, m in jobs for i in range(m)]
        wide = [cuda(np.pad(x, ((0, 0), (0, 0), (0, pad)))) for x in (q, k, v)]
        out = torch.full_like(wide[0], 7.5)
        call = jx.attn_prefill if prompt else jx.attn_step
        call(self.cache, self.layers, *wide, out, pos, self.H, self.HK, scale=self.scale,
             softcap=self.softcap, sliding_window=self.window, neox=self.kw["neox"], seq_ids=seqs,
             stream=stream)
        torch.cuda.synchronize()
        assert self.cache.check_device_error() == 0
        got = out.cpu().numpy()
        if pad:
            assert (got[..., -pad:] == 7.5).all()
            got = got[..., :-pad]
        at, worst = 0, 0.0
        for s, p, m in jobs:
            order = sorted(range(self.L), key=lambda l: l in self.shares)
            for l in order:
                ref, tol = self.model.step(
                    s, l, p, q[at:at + m, l], k[at:at + m, l], v[at:at + m, l], self.H, self.scale,
                    self.softcap, self.window if self.swa[l] else 0, append=l not in self.shares,
                    src=self.shares.get(l, l), **self.kw_layer.get(l, self.kw))
                err = np.abs(got[at:at + m, l] - ref)
                assert np.isfinite(got[at:at + m, l]).all()
                assert (err <= tol).all(), (s, l, float((err / tol).max()), float(err.max()))
                worst = max(worst, float((err / tol).max()))
            self.model.rows[s] = p + m
            at += m
            self.check_rows(s)
        return worst

    def check_rows(self, s):
        n = self.model.rows[s]
        assert self.cache.seq_pos(s) == n
        assert self.cache.held_pages(s) == -(-n // 32)
        if n == 0:
            return
        import torch
        got = self.cache.read([s], [0], n, dtype=torch.float32)[0].cpu().numpy()
        for l in range(self.L):
            if l in self.shares:
                continue
            for w in range(2):
                want = self.model.values(s, l, w, 0, n)
                assert np.array_equal(got[l, w].astype(np.float64), want), (s, l, w)


SHAPES = [(4, 1, 64), (14, 2, 64), (8, 8, 64), (8, 1, 128), (6, 2, 128), (4, 2, 128), (4, 1, 256),
          (8, 1, 256), (8, 4, 32), (5, 1, 32)]


@pytest.mark.parametrize("tc", [0, 1])
@pytest.mark.parametrize("dtype", ["int8", "e4m3"])
@pytest.mark.parametrize("H,HK,HD", SHAPES)
def test_steps_after_a_prompt(H, HK, HD, dtype, tc):
    p = Pair(H, HK, HD, dtype, n_seqs=2, cap=160, seed=H * HD, tc=tc)
    p.run([(1, 0, 37)], True)
    p.run([(0, 0, 1), (1, 37, 1)], False)
    p.run([(1, 38, 1), (0, 1, 1)], False, spread=3.0)
    p.run([(1, 39, 70), (0, 2, 14)], True)
    p.run([(0, 16, 1), (1, 109, 1)], False)


@pytest.mark.parametrize("tc", [0, 1])
@pytest.mark.parametrize("dtype", ["int8", "e4m3"])
@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200])
def test_prompt_lengths(n, dtype, tc):
    p = Pair(4, 1, 64, dtype, cap=256, seed=n, tc=tc)
    p.run([(0, 0, n)], True)
    p.run([(0, n, 1)], False)


@pytest.mark.parametrize("dtype", ["int8", "e4m3"])
@pytest.mark.parametrize("T", [1, 16, 31, 32, 33, 500, 2048, 3001])
def test_step_lengths(T, dtype):
    p = Pair(4, 2, 64, dtype, n_seqs=3, L=2, cap=3040, seed=T)
    if T > 1:
        x = p.inputs(T - 1)
        for s in (0, 2):
            load_prompt(p, s, x)
    else:
        x = None
    p.run([(2, T - 1, 1), (1, 0, 1)], False)


def load_prompt(p, s, x):
    """Rows without their attention (a long prompt is slow in the model): written by the model and
    loaded into the cache."""
    import torch
    from tests.paged_model import rotate
    q, k, v = x
    n = len(k)
    for l in range(p.L):
        p.model.write(s, l, 0, 0, rotate(k[:, l].reshape(n, p.HK, p.HD), np.arange(n), **p.kw))
        p.model.write(s, l, 1, 0, v[:, l].reshape(n, p.HK, p.HD))
    p.model.rows[s] = n
    args = []
    nb = -(-n // 16)
    for w in range(2):
        c = torch.from_numpy(p.model.code[s, :, w, :n].astype(np.float32)).cuda()
        args.append(c.to(torch.int8 if p.model.dtype == "int8" else torch.float8_e4m3fn))
        args.append(cuda(np.exp2(p.model.k[s, :, w, :nb]).astype(np.float32)))
    p.cache.load(s, 0, *args)
    p.check_rows(s)


@pytest.mark.parametrize("tc", [0, 1])
@pytest.mark.parametrize("dtype", ["int8", "e4m3"])
@pytest.mark.parametrize("HD,G", [(64, 4), (128, 2), (256, 4), (32, 3)])
def test_window_softcap_and_shared_layers(HD, G, dtype, tc):
    p = Pair(G * 2, 2, HD, dtype, L=4, cap=300, swa=[True, False, True, False], window=40,
             softcap=20.0, shares={2: 0, 3: 1}, neox=False, rope_dim=HD // 2, seed=HD, tc=tc)
    p.run([(0, 0, 150)], True)
    p.run([(0, 150, 1)], False)
    p.run([(0, 151, 20)], True)
    p.window = 1  # only the row itself
    p.run([(0, 171, 1)], False)
    p.run([(0, 172, 3)], True)


@pytest.mark.parametrize("dtype", ["int8", "e4m3"])
def test_padded_strides(dtype):
    p = Pair(4, 2, 64, dtype, L=2, cap=100, seed=5)
    p.run([(0, 0, 40)], True, pad=3)
    p.run([(0, 40, 1)], False, pad=3)


@pytest.mark.parametrize("dtype", ["int8", "e4m3"])
def test_long_prompts_after_rows(dtype):
    """Prompts on the tensor cores: every group, both head widths, windows, soft caps, two RoPE
    settings, rows cached before, several sequences of unlike lengths in one call."""
    for H, HK, HD in [(2, 2, 64), (4, 2, 128), (4, 1, 64), (8, 1, 128), (8, 2, 128)]:
        p = Pair(H, HK, HD, dtype, n_seqs=3, L=3, cap=420, swa=[False, True, True], window=70,
                 softcap=15.0 if HD == 64 else 0.0, neox=HD == 64, rope_dim=HD // 2 if H == 4 else HD,
                 seed=H + HD)
        p.layers[2].rope_base = 1e6
        x = p.inputs(130)
        p.kw_layer = {2: dict(p.kw, base=1e6)}
        p.run([(1, 0, 130)], True, inputs=x)
        p.run([(0, 0, 49), (1, 130, 150), (2, 0, 131)], True, spread=2.0)
        p.run([(1, 280, 1), (0, 49, 1)], False)


@pytest.mark.parametrize("dtype", ["int8", "e4m3"])
def test_scales_far_apart(dtype):
    """Blocks whose scales differ by powers of two up to 2^24, and one head far larger than the
    other: what each row is worth stays what it is."""
    p = Pair(4, 2, 64, dtype, cap=300, seed=31)
    q, k, v = p.inputs(200)
    f = 2.0 ** (-8 * (np.arange(200) // 50))
    k, v = k * f[:, None, None], v * f[:, None, None]
    k[..., 64:] *= 1e-3
    v[..., 64:] *= 1e3
    p.run([(0, 0, 200)], True, inputs=[q, k.astype(np.float32), v.astype(np.float32)])
    p.run([(0, 200, 1)], False)


@pytest.mark.parametrize("dtype", ["int8", "e4m3"])
def test_scales_grow_row_by_row(dtype):
    """Magnitudes that rise and fall by powers of ten, appended one by one and then in pieces:
    every re-rounding of a block is the model's."""
    p = Pair(2, 1, 64, dtype, cap=128, seed=9)
    for t in range(36):
        p.run([(0, t, 1)], False, spread=10.0 ** ((t * 7) % 5 - 2))
    at = 36
    for n in (1, 3, 20, 2, 30):
        p.run([(0, at, n)], True, spread=10.0 ** (n % 4 - 1))
        at += n


@pytest.mark.parametrize("tc", [0, 1])
@pytest.mark.parametrize("dtype", ["int8", "e4m3"])
def test_extreme_values(dtype, tc):
    """NaN counts as 0, infinities and magnitudes over 2^62 as 2^62, tiny values and zeros stay in
    the format; what attends them is finite."""
    import torch
    from tests.paged_model import rotate
    p = Pair(2, 1, 64, dtype, cap=128, seed=3, tc=tc)
    q, k, v = p.inputs(40)
    k[0, 0, :8] = [np.nan, np.inf, -np.inf, 0, 1e30, -1e-40, 1e-30, 3e38]
    v[1, 0, :8] = [np.nan, np.inf, -np.inf, 0, 1e30, -1e-40, 1e-30, 3e38]
    k[16:32] = 0.0
    v[16:32] = 0.0
    q[0:16] = 0.0
    wide = [cuda(x) for x in (q, k, v)]
    out = torch.zeros_like(wide[0])
    jx.attn_prefill(p.cache, p.layers, *wide, out, list(range(40)), 2, 1, neox=True)
    p.model.write(0, 0, 0, 0, rotate(k[:, 0].reshape(40, 1, 64), np.arange(40), **p.kw))
    p.model.write(0, 0, 1, 0, v[:, 0].reshape(40, 1, 64))
    p.model.rows[0] = 40
    p.check_rows(0)
    assert np.isfinite(out.cpu().numpy()).all()


@pytest.mark.parametrize("tc", [0, 1])
@pytest.mark.parametrize("size", [1e3, 1e6, 1e12])
def test_scores_far_from_zero(size, tc):
    """Scores of any size: the softmax becomes a choice of the largest, and stays a softmax where
    two are equal."""
    p = Pair(2, 1, 64, "int8", cap=300, seed=8, tc=tc)
    q, k, v = p.inputs(200)
    k[:] = k[:1] * 0.25                # equal keys but for the position's rotation
    p.layers[0].rope_dim = 0           # none: all scores of a query are equal
    p.kw = dict(p.kw, rope_dim=0)
    q = (q * size).astype(np.float32)
    p.run([(0, 0, 200)], True, inputs=[q, k, v])
    p.run([(0, 200, 1)], False, inputs=[q[:1], k[:1], v[:1]])


@pytest.mark.parametrize("tc", [0, 1])
def test_later_rows_do_not_reach_earlier_ones(tc):
    """A token whose key and value are infinite or NaN: the tokens before it are right."""
    import torch
    for dtype in ("int8", "e4m3"):
        p, ok = (Pair(4, 1, 64, dtype, cap=256, seed=14, tc=tc) for _ in range(2))
        q, k, v = p.inputs(200)
        ok.run([(0, 0, 200)], True, inputs=(q, k, v))
        bad_k, bad_v = k.copy(), v.copy()
        bad_k[150], bad_v[150] = np.inf, -np.inf
        bad_k[170], bad_v[171] = np.nan, np.nan
        outs = []
        for pair, kv in ((p, (bad_k, bad_v)), (ok, (k, v))):
            pair.cache.clear(0)
            wide = [cuda(x) for x in (q, *kv)]
            out = torch.empty_like(wide[0])
            jx.attn_prefill(pair.cache, pair.layers, *wide, out, list(range(200)), 4, 1, neox=True)
            outs.append(out.cpu().numpy())
        # rows before the block that holds the token: the same, but for the exponent the
        # sums are taken against
        assert np.abs(outs[0][:144] - outs[1][:144]).max() <= 2.0 ** -18 * np.abs(v).max()
        assert np.isfinite(outs[0]).all()


@pytest.mark.parametrize("tc", [0, 1])
def test_rows_behind_a_window_do_not_reach_it(tc):
    """Rows with infinities and NaN in front of a sliding window leave its output alone."""
    p = Pair(4, 1, 64, "e4m3", cap=128, swa=[True], window=16, seed=4, tc=tc)
    x = p.inputs(64)
    x[1][:48], x[2][:48] = np.inf, np.nan
    load_prompt(p, 0, x)
    p.run([(0, 64, 1)], False)
    p.run([(0, 65, 5)], True)


def test_rope_settings():
    """Frequency factors, a YaRN scale, a far position, and a second setting in one call."""
    import torch
    fac = np.linspace(1, 4, 32).astype(np.float32)
    cache = jx.PagedKVCache(1, 2, 100000, 1, 64, n_pages=3200, dtype="int8")
    layers = [jx.Layer(64, 64, 5e5, 0, rope_freqs=fac), jx.Layer(64, 32, 1e4, 1)]
    m = Model(1, 2, 99872, 1, 64, "int8")
    # a far position: the rows before it are zeros
    n = 99840
    zero = torch.zeros(2, n, 1, 64, dtype=torch.int8, device="cuda")
    one = torch.ones(2, n // 16, 1, device="cuda")
    cache.load(0, 0, zero, one, zero, one)
    rng = np.random.default_rng(0)
    q, k, v = (rng.standard_normal((1, 2, 64)).astype(np.float32) for _ in range(3))
    out = torch.zeros(1, 2, 64, device="cuda")
    jx.attn_step(cache, layers, *(cuda(x) for x in (q, k, v)), out, [n], 1, 1, yarn_scale=1.5, neox=True)
    from tests.paged_model import rotate
    for l, (f, rd, b) in enumerate([(fac, 64, 5e5), (None, 32, 1e4)]):
        m.write(0, l, 0, n, rotate(k[:, l].reshape(1, 1, 64), [n], rd, b, True, f, 1.5))
        m.write(0, l, 1, n, v[:, l].reshape(1, 1, 64))
        got = cache.read([0], [n], 1, dtype=torch.float32)[0, l].cpu().numpy()
        assert np.array_equal(got[0], m.values(0, l, 0, n, n + 1))
        assert np.array_equal(got[1], m.values(0, l, 1, n, n + 1))


@pytest.mark.parametrize("dtype", ["int8", "e4m3"])
def test_fork_writes_do_not_meet(dtype):
    p = Pair(4, 2, 64, dtype, n_seqs=3, L=2, cap=128, seed=11)
    p.run([(0, 0, 50)], True)
    free = p.cache.free_pages
    p.cache.fork(0, 1)
    p.model.fork(0, 1)
    p.cache.fork(0, 2, 33)
    p.model.fork(0, 2, 33)
    assert p.cache.free_pages == free
    p.run([(1, 50, 1)], False)          # its own copy of the shared tail page
    assert p.cache.free_pages == free - 1
    p.check_rows(0)
    p.run([(2, 33, 40)], True, spread=4.0)
    p.run([(0, 50, 1), (1, 51, 1), (2, 73, 1)], False)
    for s in range(3):
        p.check_rows(s)
    p.cache.clear(0)
    p.model.rows[0] = 0
    for s in range(3):
        p.check_rows(s)
    p.cache.clear(1)
    p.cache.clear(2)
    assert p.cache.free_pages == p.cache.n_pages


def test_a_page_shared_by_all_writers_of_a_call():
    """The last holder of a shared page keeps it: two writers need one free page."""
    p = Pair(2, 1, 32, "int8", n_seqs=2, cap=64, n_pages=2)
    p.run([(0, 0, 20)], True)
    p.cache.fork(0, 1)
    p.model.fork(0, 1)
    p.run([(0, 20, 1), (1, 20, 1)], False)
    assert p.cache.free_pages == 0
    p.check_rows(0)


def test_streams_and_tensors():
    import torch
    cache = jx.PagedKVCache(1, 1, 64, 1, 32, dtype="int8")
    st = torch.cuda.Stream()
    codes = torch.randint(-127, 128, (1, 2 * 40, 1, 32), dtype=torch.int8, device="cuda")
    scales = torch.ones(1, 3, 1, device="cuda")
    refuses(_lib.JX_ERR_INVALID, cache.load, 0, 0, codes[:, ::2], scales, codes[:, 1::2], scales, stream=st)
    cache.load(0, 0, codes[:, ::2], scales, codes[:, 1::2], scales)
    refuses(_lib.JX_ERR_INVALID, cache.read, [0], [0], 40, stream=st)
    out = torch.empty(1, 1, 2, 40, 1, 32, device="cuda")
    torch.cuda.synchronize()
    cache.read([0], [0], 40, out=out, stream=st)
    st.synchronize()
    assert torch.equal(out[0, 0, 0], codes[0, ::2].float()) and torch.equal(out[0, 0, 1], codes[0, 1::2].float())


def test_a_fork_onto_its_own_fork():
    p = Pair(2, 1, 32, "int8", n_seqs=2, cap=96, n_pages=4)
    p.run([(0, 0, 70)], True)
    for n in (70, 40, 70):
        p.cache.fork(0, 1, n)
        p.model.fork(0, 1, n)
        p.check_rows(1)
    p.cache.clear(0)
    p.check_rows(1)
    p.cache.clear(1)
    assert p.cache.free_pages == 4


def test_copy():
    p = Pair(4, 2, 128, "e4m3", n_seqs=2, L=3, cap=128, seed=2)
    p.run([(0, 0, 77)], True)
    p.run([(1, 0, 100)], True)
    p.cache.copy(0, 1)
    p.model.fork(0, 1)
    p.check_rows(1)
    p.run([(0, 77, 1)], False)
    p.check_rows(1)
    assert p.cache.free_pages == p.cache.n_pages - 6


KEPT = [[0], [5], list(range(40)), list(range(32)) + [40, 50, 99], list(range(0, 100, 3)),
        list(range(4)) + list(range(60, 100)), list(range(1, 100)), list(range(99, 100)), []]


@pytest.mark.parametrize("dtype", ["int8", "e4m3"])
@pytest.mark.parametrize("case", range(len(KEPT)))
@pytest.mark.parametrize("full", [False, True])
def test_keep(case, dtype, full):
    rows = KEPT[case]
    p = Pair(4, 2, 64, dtype, L=2, cap=128, n_pages=4 if full else 8, seed=case)
    p.run([(0, 0, 60)], True)
    p.run([(0, 60, 40)], True, spread=20.0)
    p.cache.keep(0, rows)
    p.model.keep(0, rows)
    p.check_rows(0)
    assert p.cache.free_pages == p.cache.n_pages - -(-len(rows) // 32)
    p.run([(0, len(rows), 1)], False)


def test_keep_of_a_fork_leaves_the_other():
    p = Pair(4, 2, 128, "int8", n_seqs=2, L=2, cap=128, seed=8)
    p.run([(0, 0, 100)], True)
    p.cache.fork(0, 1)
    p.model.fork(0, 1)
    rows = list(range(32)) + list(range(33, 100, 2))
    p.cache.keep(1, np.array(rows))
    p.model.keep(1, rows)
    p.check_rows(0)
    p.check_rows(1)
    # the page that stayed in place is still shared
    assert p.cache.free_pages == 8 - 4 - 2


def test_compact_and_slots():
    p = Pair(4, 2, 64, "int8", n_seqs=2, cap=128, seed=6)
    slot = jx.KVCacheSlot(p.cache, 0)
    p.run([(0, 0, 100)], True)
    assert slot.seq_pos == 100
    slot.compact(20)
    p.model.keep(0, list(range(4)) + list(range(80, 100)))
    assert slot.seq_pos == 24 and slot.compactions == 1
    p.check_rows(0)
    slot.compact(20)
    assert slot.seq_pos == 24
    slot.rollback(10)
    p.model.rows[0] = 10
    p.check_rows(0)
    p.run([(0, 10, 1)], False)
    slot.clear()
    assert p.cache.free_pages == p.cache.n_pages


def test_rollback_then_write_again():
    p = Pair(4, 2, 64, "e4m3", cap=128, seed=13)
    p.run([(0, 0, 90)], True, spread=9.0)
    p.cache.rollback(0, 41)
    p.model.rows[0] = 41
    p.check_rows(0)
    p.run([(0, 41, 30)], True, spread=0.1)
    p.run([(0, 64, 1)], False)           # writes inside the sequence: it ends there
    assert p.cache.seq_pos(0) == 65
    p.cache.set_seq_pos(0, 65)
    p.run([(0, 65, 1)], False)


def test_load_takes_any_codes_and_scales():
    import torch
    for dtype in ("int8", "e4m3"):
        cache = jx.PagedKVCache(1, 1, 64, 1, 32, dtype=dtype)
        codes = (torch.arange(32 * 32, device="cuda") % 256).to(torch.uint8).view(1, 32, 1, 32)
        scales = torch.tensor([3.0, float("nan")], device="cuda").view(1, 2, 1)
        cache.load(0, 0, codes, scales, codes, torch.tensor([0.0, 1e30], device="cuda").view(1, 2, 1))
        got = cache.read([0], [0], 32, dtype=torch.float32)[0, 0, :, :, 0]
        c = codes[0, :, 0].view(torch.int8 if dtype == "int8" else torch.float8_e4m3fn).float()
        c = c.clamp(min=-127) if dtype == "int8" else c.nan_to_num(nan=0.0)
        assert torch.equal(got[0, :16], c[:16] * 2.0)
        assert torch.equal(got[0, 16:], c[16:] * 2.0 ** 56)
        assert torch.equal(got[1, :16], c[:16] * 2.0 ** -40)
        assert torch.equal(got[1, 16:], c[16:] * 2.0 ** 56)
        assert torch.equal(cache.read([0], [3], 20)[0, 0, :, :, 0].float(), got[:, 3:23])


def test_a_serving_run():
    """Prompts, steps, a fork, an eviction, a compaction and more steps on one cache, on a stream of
    their own."""
    import torch
    p = Pair(8, 2, 64, "int8", n_seqs=3, L=3, cap=256, n_pages=20, swa=[True, False, True],
             window=48, seed=21, tc=-1)
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        p.run([(0, 0, 61), (2, 0, 90)], True)
        for i in range(5):
            p.run([(2, 90 + i, 1), (0, 61 + i, 1)], False)
        p.cache.fork(2, 1)
        p.model.fork(2, 1)
        p.run([(1, 95, 20)], True, spread=2.0)
        rows = [0, 1, 2, 3] + list(range(20, 115, 5))
        p.cache.keep(1, rows)
        p.model.keep(1, rows)
        p.cache.compact(2, 40)
        p.model.keep(2, [0, 1, 2, 3] + list(range(55, 95)))
        for i in range(3):
            p.run([(0, 66 + i, 1), (1, 23 + i, 1), (2, 44 + i, 1)], False)
        p.run([(0, 69, 64)], True)
        for s in range(3):
            p.check_rows(s)


@pytest.mark.parametrize("dtype", ["int8", "e4m3"])
def test_layer_by_layer(dtype):
    """One call per layer at the same positions, as an engine runs a token."""
    import torch
    H, HK, HD, L = 4, 2, 64, 3
    p = Pair(H, HK, HD, dtype, n_seqs=2, L=L, cap=128, seed=77)
    for jobs, prompt in [([(1, 0, 60)], True), ([(1, 60, 1), (0, 0, 1)], False), ([(0, 1, 5)], True),
                         ([(0, 6, 1), (1, 61, 1)], False)]:
        n = sum(j[2] for j in jobs)
        q, k, v = p.inputs(n)
        seqs = [s for s, a, m in jobs for _ in range(m)]
        pos = [a + i for s, a, m in jobs for i in range(m)]
        for l in range(L):
            wide = [cuda(x[:, l:l + 1]) for x in (q, k, v)]
            out = torch.empty_like(wide[0])
            (jx.attn_prefill if prompt else jx.attn_step)(
                p.cache, [p.layers[l]], *wide, out, pos, H, HK, neox=True, seq_ids=seqs)
            got, at = out.cpu().numpy()[:, 0], 0
            for s, a, m in jobs:
                ref, tol = p.model.step(s, l, a, q[at:at + m, l], k[at:at + m, l], v[at:at + m, l], H,
                                        p.scale, **p.kw)
                assert (np.abs(got[at:at + m] - ref) <= tol).all()
                at += m
        for s, a, m in jobs:
            p.model.rows[s] = a + m
            p.check_rows(s)


@pytest.mark.parametrize("tokens,tc", [(3, 0), (3, 1), (50, 1)])
def test_more_sequences_than_a_launch_takes(tokens, tc):
    """Prompts and steps of 131 sequences of unlike lengths, with a window."""
    p = Pair(2, 1, 64, "int8", n_seqs=131, L=2, cap=64, swa=[False, True], window=20, seed=5, tc=tc)
    jobs = [(s, 0, tokens + s % 4) for s in range(131)]
    p.run(jobs, True)
    p.run([(s, n, 1) for s, _, n in reversed(jobs)], False)


@pytest.mark.parametrize("dtype", ["int8", "e4m3"])
def test_padded_rows_on_the_tensor_cores(dtype):
    p = Pair(8, 2, 128, dtype, cap=200, seed=15)
    p.run([(0, 0, 150)], True, pad=4)


@pytest.mark.parametrize("HD", [64, 128])
def test_a_wait_that_runs_out_is_reported(HD):
    """A CTA whose wait runs out sets the error word; the kernel ends, and the next step is right."""
    import torch
    p = Pair(4, 2, HD, "int8", cap=2000, seed=3)
    load_prompt(p, 0, p.inputs(1500))
    q, k, v = p.inputs(1)
    wide = [cuda(x) for x in (q, k, v)]
    out = torch.empty_like(wide[0])
    p.cache.set_option("wait_limit_ms", 20)
    p.cache.set_option("test_wait_cta", 1)
    jx.attn_step(p.cache, p.layers, *wide, out, [1500], 4, 2, neox=True)
    torch.cuda.synchronize()
    assert p.cache.check_device_error() == 1
    assert p.cache.check_device_error() == 0
    p.cache.set_option("test_wait_cta", 0)
    p.cache.set_option("wait_limit_ms", 0)
    p.cache.rollback(0, 1488)  # drops the block that step may have written
    p.model.rows[0] = 1488
    p.run([(0, 1488, 1)], False)
    p.run([(0, 1489, 1)], False)


def test_calls_in_a_row_share_their_buffers():
    """Prompts of several sizes, keeps and steps queued without a wait between them: lists, widened
    rows and totals are used in turn."""
    import torch
    H, HK, HD = 8, 2, 64
    caches = [jx.PagedKVCache(2, 2, 600, HK, HD, dtype="int8") for _ in range(2)]
    for c in caches:
        c.set_option("prefill_tc", 1)
    layers = [jx.Layer(HD, HD, 1e4, l) for l in range(2)]
    g = torch.Generator(device="cuda").manual_seed(0)
    sizes = [300, 64, 500, 65, 600, 130]
    data = [[torch.randn(n, 2, w, generator=g, device="cuda") for w in (H * HD, HK * HD, HK * HD)] for n in sizes]
    torch.cuda.synchronize()

    def go(cache, wait):
        outs = []
        for i, (n, (q, k, v)) in enumerate(zip(sizes, data)):
            out = torch.empty_like(q)
            jx.attn_prefill(cache, layers, q, k, v, out, np.arange(n), H, HK, seq_ids=np.zeros(n, int))
            cache.fork(0, 1)
            cache.keep(1, np.arange(i, n, 2))
            m = cache.seq_pos(1)
            one = torch.empty_like(q[:1])
            jx.attn_step(cache, layers, q[:1], k[:1], v[:1], one, [m], H, HK, seq_ids=[1])
            outs += [out, one, cache.read([1], [0], m + 1)]
            if wait:
                torch.cuda.synchronize()
        torch.cuda.synchronize()
        return outs
    for a, b in zip(go(caches[0], False), go(caches[1], True)):
        assert torch.equal(a, b)


def refuses(code, fn, *args, **kw):
    with pytest.raises(jx.JxError) as e:
        fn(*args, **kw)
    assert e.value.code == code, str(e.value)


def test_refusals():
    import torch
    p = Pair(4, 2, 64, "int8", n_seqs=2, L=2, cap=64, n_pages=3, seed=1)
    p.run([(0, 0, 40)], True)
    z = lambda n=1, w=256: torch.zeros(n, 2, w, device="cuda")  # noqa: E731

    def step(pos, layers=None, q=None, k=None, seqs=None, H=4, HK=2, call=jx.attn_step, **kw):
        n = len(pos)
        call(p.cache, layers or p.layers, z(n) if q is None else q, z(n, 128) if k is None else k,
             z(n, 128), z(n), pos, H, HK, seq_ids=seqs, **kw)

    refuses(_lib.JX_ERR_RANGE, step, [41])                     # leaves a gap
    refuses(_lib.JX_ERR_RANGE, step, [64])                     # beyond the capacity
    refuses(_lib.JX_ERR_INVALID, step, [-1])
    refuses(_lib.JX_ERR_INVALID, step, [40], seqs=[2])
    refuses(_lib.JX_ERR_INVALID, step, [40, 40], seqs=[0, 0])
    refuses(_lib.JX_ERR_INVALID, step, [40, 42], seqs=[0, 0], call=jx.attn_prefill)
    refuses(_lib.JX_ERR_INVALID, step, [40, 0, 41], seqs=[0, 1, 0], call=jx.attn_prefill)
    refuses(_lib.JX_ERR_INVALID, step, [40], H=2, HK=1)
    refuses(_lib.JX_ERR_INVALID, step, [40], yarn_scale=float("nan"))
    refuses(_lib.JX_ERR_UNSUPPORTED, step, [40], layers=[jx.Layer(32, 32, 1e4, l) for l in range(2)])
    refuses(_lib.JX_ERR_INVALID, step, [40], layers=[jx.Layer(64, 64, 1e4, 0) for l in range(2)])
    refuses(_lib.JX_ERR_INVALID, step, [40], layers=[jx.Layer(64, 64, 1e4, l + 1) for l in range(2)])
    refuses(_lib.JX_ERR_INVALID, step, [40], layers=[jx.Layer(64, 64, 0.0, l) for l in range(2)])
    refuses(_lib.JX_ERR_INVALID, step, [40], q=z().cpu().pin_memory())
    # a layer that only reads cannot run ahead of what is held
    refuses(_lib.JX_ERR_RANGE, step, [40], layers=[jx.Layer(64, 64, 1e4, l, shares_kv=True) for l in range(2)])
    # too few pages: nothing changes
    refuses(_lib.JX_ERR_NOMEM, step, list(range(40)), seqs=[1] * 40, call=jx.attn_prefill)
    assert p.cache.seq_pos(1) == 0 and p.cache.free_pages == 1
    refuses(_lib.JX_ERR_RANGE, p.cache.set_seq_pos, 0, 41)
    refuses(_lib.JX_ERR_INVALID, p.cache.set_option, "prefill_tc", 2)
    refuses(_lib.JX_ERR_INVALID, p.cache.set_option, "wait_limit_ms", -1)
    refuses(_lib.JX_ERR_INVALID, p.cache.set_option, "no_such_option", 1)
    refuses(_lib.JX_ERR_INVALID, p.cache.fork, 0, 0)
    refuses(_lib.JX_ERR_RANGE, p.cache.fork, 0, 1, 41)
    refuses(_lib.JX_ERR_NOMEM, p.cache.copy, 0, 1)
    refuses(_lib.JX_ERR_INVALID, p.cache.keep, 0, [3, 3])
    refuses(_lib.JX_ERR_INVALID, p.cache.keep, 0, [3, 40])
    refuses(_lib.JX_ERR_RANGE, p.cache.read, [0], [39], 2)
    refuses(_lib.JX_ERR_UNSUPPORTED, jx.attn_step_partial, p.cache, p.layers, z(), z(1, 128), z(1, 128),
            torch.zeros(2 * 4 * 66, device="cuda"), [40], 4, 2)
    p.cache.fork(0, 1)
    refuses(_lib.JX_ERR_NOMEM, p.cache.keep, 1, list(range(1, 40)))  # shared, and no pages
    p.cache.clear(1)
    p.check_rows(0)
    # capture
    g = torch.cuda.CUDAGraph()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    args = (z(), z(1, 128), z(1, 128), z())
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=st):
        args[3].zero_()
        refuses(_lib.JX_ERR_UNSUPPORTED, jx.attn_step, p.cache, p.layers, *args, [40], 4, 2)
        refuses(_lib.JX_ERR_UNSUPPORTED, p.cache.keep, 0, [1])
        refuses(_lib.JX_ERR_UNSUPPORTED, p.cache.fork, 0, 1)
    p.run([(0, 40, 1)], False)


def test_many_sequences_and_layers():
    """More sequences and more layers than one launch's plan holds."""
    p = Pair(2, 1, 32, "e4m3", n_seqs=150, L=70, cap=32, seed=17)
    jobs = [(s, 0, 1) for s in range(150)]
    x = p.inputs(150)
    import torch
    wide = [cuda(a) for a in x]
    out = torch.zeros_like(wide[0])
    jx.attn_step(p.cache, p.layers, *wide, out, [0] * 150, 2, 1, seq_ids=list(range(150)))
    # one row: attention returns the row's values
    got = p.cache.read(range(150), [0] * 150, 1, dtype=torch.float32)[:, :, 1, 0]
    want = got.repeat_interleave(2, dim=2).view(150, 70, 64)
    assert torch.allclose(out, want, rtol=2.0 ** -20, atol=0)
    del jobs
