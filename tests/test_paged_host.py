"""The paged cache's host side where no GPU is needed."""
import ctypes as C
import os
import random
import subprocess
import tempfile

import numpy as np
import pytest

import jxai_b200 as jx
from jxai_b200 import _lib
from jxai_b200.attention import _i32_array

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_desc_layout_matches_header():
    src = ('#include <stdio.h>\n#include <stddef.h>\n#include "jx_attn.h"\nint main(void) {'
           'printf("%zu %zu %zu %d %d", sizeof(jx_pkv_desc), offsetof(jx_pkv_desc, n_pages),'
           'offsetof(jx_pkv_desc, device), JX_I8, JX_E4M3); return 0; }')
    with tempfile.TemporaryDirectory() as d:
        with open(os.path.join(d, "t.c"), "w") as fh:
            fh.write(src)
        exe = os.path.join(d, "t")
        subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), os.path.join(d, "t.c"), "-o", exe],
                       check=True)
        got = [int(x) for x in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [C.sizeof(_lib.PkvDesc), _lib.PkvDesc.n_pages.offset, _lib.PkvDesc.device.offset,
                   jx.JX_I8, jx.JX_E4M3]


def create(**kw):
    d = dict(n_seqs=1, n_layers=1, capacity=64, n_kv_heads=1, head_dim=64, n_pages=2, dtype=jx.JX_I8, device=0)
    d.update(kw)
    h = C.c_void_p()
    return jx.load_library().jx_pkv_create(C.byref(_lib.PkvDesc(*d.values())), C.byref(h))


@pytest.mark.parametrize("bad,code", [
    (dict(n_seqs=0), _lib.JX_ERR_INVALID), (dict(n_pages=0), _lib.JX_ERR_INVALID),
    (dict(capacity=0), _lib.JX_ERR_INVALID), (dict(dtype=jx.JX_F32), _lib.JX_ERR_INVALID),
    (dict(dtype=5), _lib.JX_ERR_INVALID), (dict(head_dim=96), _lib.JX_ERR_UNSUPPORTED),
    (dict(capacity=1 << 31), _lib.JX_ERR_INVALID), (dict(n_kv_heads=600), _lib.JX_ERR_UNSUPPORTED),
    (dict(n_layers=9000, n_kv_heads=8), _lib.JX_ERR_UNSUPPORTED),
    (dict(n_seqs=1 << 20, capacity=1 << 20), _lib.JX_ERR_INVALID)])
def test_descriptions_refused(bad, code):
    assert create(**bad) == code


def test_null_arguments_refused():
    lib = jx.load_library()
    bad = _lib.JX_ERR_INVALID
    assert lib.jx_pkv_create(None, None) == bad
    assert lib.jx_pkv_destroy(None) == _lib.JX_OK
    assert lib.jx_pkv_attn_step(None, None, 0, None, None) == bad
    assert lib.jx_pkv_attn_prefill(None, None, 0, None, None) == bad
    for call, args in [("get_desc", (None,)), ("get_seq_pos", (0, None)), ("set_seq_pos", (0, 0)),
                       ("free_pages", (None,)), ("held_pages", (0, None)), ("clear", (0,)),
                       ("rollback", (0, 0)), ("fork", (0, 1, 0, None)), ("copy", (0, 1, None)),
                       ("keep", (0, None, 0, None)), ("compact", (0, 4, None)),
                       ("load_rows", (0, 0, 1, None, None, None, None, None)),
                       ("read_rows", (None, None, 1, 1, 0, None, None)),
                       ("check_device_error", (None, None)), ("set_option", (None, 0)),
                       ("last_launch_count", (None,))]:
        assert getattr(lib, "jx_pkv_" + call)(None, *args) == bad, call
        assert lib.jx_last_error_string()


def test_python_refusals():
    with pytest.raises(jx.JxError):
        jx.PagedKVCache(1, 1, 64, 1, 64, dtype="bf16")
    try:
        import torch
        if torch.cuda.is_available():
            pytest.skip("a GPU is present")
    except ImportError:
        pass
    with pytest.raises(jx.JxError) as e:
        jx.PagedKVCache(1, 1, 64, 1, 64)
    assert e.value.code == _lib.JX_ERR_CUDA


def test_integer_lists():
    assert list(_i32_array([1, 2])) == [1, 2]
    assert list(_i32_array(range(3, 9, 2))) == [3, 5, 7]
    assert list(_i32_array(np.arange(4)[::-1])) == [3, 2, 1, 0]
    assert list(_i32_array(np.array([], dtype=np.int64))) == []
    for bad in (np.zeros(2), np.zeros((2, 2), int), np.array([1 << 31])):
        with pytest.raises(jx.JxError):
            _i32_array(bad)


class Bar:
    """An mbarrier: `count` arrivals complete a phase; a wait names a phase by its parity."""

    def __init__(self):
        self.phase = 0

    def arrive(self):
        self.phase += 1

    def passes(self, parity):
        return (self.phase & 1) != parity


def prompt_barriers(items, stages, rng):
    """The waits and arrivals of jx_paged_prompt.cu's roles for items of (tiles of query tile 0,
    of tile 1), taken in a random order.  Every wait has to end, and on the phase it means."""
    full, empty = [[Bar() for _ in range(stages)] for _ in range(2)]
    q, s, p, pv, o = [[Bar(), Bar()] for _ in range(5)]
    pipe, copies = [], []  # MMA commits and TMA copies, in order

    def producer():
        n = 0
        for c in items:
            for _ in range(2 * max(c)):
                if n >= stages:
                    yield empty[n % stages], ((n // stages) & 1) ^ 1, n // stages
                copies.append(n % stages)
                n += 1

    def issuer():
        n0, done = 0, [0, 0]

        def tile(n):
            return full[n % stages], (n // stages) & 1, n // stages + 1
        for i, c in enumerate(items):
            for x in range(2):
                yield q[x], i & 1, i + 1
                if c[x]:
                    if done[x]:
                        yield pv[x], (done[x] - 1) & 1, done[x]
                    yield tile(n0)
                pipe.append(s[x])
            if max(c):
                pipe.append(empty[n0 % stages])
            for t in range(max(c)):
                for x in range(2):
                    if t >= c[x]:
                        continue
                    yield p[x], done[x] & 1, done[x] + 1
                    if t == 0 and i:
                        yield o[x], (i - 1) & 1, i
                    yield tile(n0 + 2 * t + 1)
                    pipe.append(pv[x])
                    if t + 1 < c[x]:
                        yield pv[x], done[x] & 1, done[x] + 1
                        yield tile(n0 + 2 * t + 2)
                        pipe.append(s[x])
                    done[x] += 1
                for k in (1, 2) if t + 1 < max(c) else (1,):
                    pipe.append(empty[(n0 + 2 * t + k) % stages])
            n0 += 2 * max(c)

    def softmax(x):
        g = n = 0
        q[x].arrive()
        for i, c in enumerate(items):
            for t in range(c[x]):
                if t and t % 4 == 0:
                    yield pv[x], (n - 1) & 1, n
                yield s[x], g & 1, g + 1
                p[x].arrive()
                g, n = g + 1, n + 1
            if not c[x]:
                yield s[x], g & 1, g + 1
                g += 1
            if i + 1 < len(items):
                q[x].arrive()
            if c[x]:
                yield pv[x], (n - 1) & 1, n
            o[x].arrive()

    roles = [producer(), issuer(), softmax(0), softmax(1)]
    waits = {i: next(r, None) for i, r in enumerate(roles)}
    while any(waits.values()):
        ready = [i for i, w in waits.items() if w and w[0].passes(w[1])]
        acts = ready + ["pipe"] * bool(pipe) + ["copy"] * bool(copies)
        assert acts, "a wait never ends"
        act = rng.choice(acts)
        if act == "pipe":
            pipe.pop(0).arrive()
        elif act == "copy":
            full[copies.pop(0)].arrive()
        else:
            assert waits[act][0].phase == waits[act][2], "a wait ends on another phase"
            waits[act] = next(roles[act], None)


def test_prompt_kernel_barriers():
    rng = random.Random(0)
    for _ in range(1500):
        items = []
        for _ in range(rng.randint(1, 6)):
            a = rng.randint(1, 9)
            items.append((a, rng.choice([0, a, a + 1, max(1, a - 1)])))
        prompt_barriers(items, rng.choice([3, 8]), rng)
