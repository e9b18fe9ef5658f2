"""The paged cache's host side where no GPU is needed."""
import ctypes as C
import os
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
