"""Calls on the paged cache that find too little memory, or memory that they cannot use, on the GPU:
they say so and change nothing."""
import numpy as np
import pytest

import jxai_b200 as jx
from jxai_b200 import _lib
from tests.test_gpu_paged import Pair, refuses

pytestmark = pytest.mark.gpu


def state(p):
    c = p.cache
    return [(c.seq_pos(s), c.held_pages(s)) for s in range(c.n_seqs)] + [c.free_pages]


def test_a_prompt_without_its_workspaces_changes_nothing():
    """The fp16 rows, totals and lists of a tensor-core prompt cannot be allocated: the sequence is as
    long as it was, with the rows it held, and the same call succeeds afterwards."""
    import torch
    p = Pair(4, 2, 64, "int8", n_seqs=2, cap=400, seed=1, tc=0)
    p.run([(0, 0, 50), (1, 0, 70)], True)
    p.cache.fork(0, 1, 45)  # a page that the prompt would have to copy
    p.model.fork(0, 1, 45)
    p.cache.set_option("prefill_tc", 1)
    p.cache.set_option("test_fail", 1)
    before = state(p)
    q, k, v = (torch.from_numpy(x).cuda() for x in p.inputs(200))
    out = torch.full_like(q, 3.0)
    call = lambda pos: jx.attn_prefill(p.cache, p.layers, q, k, v, out, pos, 4, 2, seq_ids=[1] * 200)  # noqa: E731
    for first in (45, 20):  # behind its rows, and over the last of them
        refuses(_lib.JX_ERR_NOMEM, call, range(first, first + 200))
        torch.cuda.synchronize()
        assert state(p) == before and (out == 3.0).all()
        p.check_rows(0)
        p.check_rows(1)
    p.cache.set_option("test_fail", 0)
    p.run([(1, 45, 200)], True)
    p.run([(1, 245, 10)], True)
    p.cache.set_option("test_fail", 1)  # what calls have allocated stays
    p.run([(1, 255, 20)], True)
    p.check_rows(0)


def test_too_few_pages_after_the_workspaces_change_nothing():
    p = Pair(4, 2, 64, "int8", n_seqs=2, cap=400, n_pages=6, seed=1, tc=1)
    p.run([(0, 0, 100)], True)
    before = state(p)
    q, k, v = p.inputs(70)
    refuses(_lib.JX_ERR_NOMEM, p.run, [(1, 0, 70)], True, inputs=(q, k, v))
    assert state(p) == before
    p.check_rows(0)
    p.run([(1, 0, 60)], True)


def test_a_keep_without_its_list_changes_nothing():
    p = Pair(4, 2, 64, "int8", cap=128, seed=4)
    p.cache.set_option("prefill_tc", 0)
    p.run([(0, 0, 100)], True)
    p.cache.set_option("test_fail", 1)
    before = state(p)
    rows = list(range(0, 100, 3))
    refuses(_lib.JX_ERR_NOMEM, p.cache.keep, 0, rows)
    refuses(_lib.JX_ERR_NOMEM, p.cache.compact, 0, 20)
    assert state(p) == before
    p.check_rows(0)
    p.cache.set_option("test_fail", 0)
    p.cache.keep(0, np.array(rows))
    p.model.keep(0, rows)
    p.check_rows(0)


@pytest.mark.parametrize("pages", [4, 8])
def test_a_keep_that_fails_late_loses_no_page(pages):
    """After the pages for the result were taken (or, in a full pool, in place)."""
    p = Pair(4, 2, 64, "int8", cap=128, n_pages=pages, seed=4)
    p.run([(0, 0, 100)], True)
    before = state(p)
    rows = list(range(0, 100, 2))
    p.cache.set_option("test_fail", 2)
    for _ in range(3):
        refuses(_lib.JX_ERR_CUDA, p.cache.keep, 0, rows)
        assert state(p) == before
    p.check_rows(0)
    p.cache.set_option("test_fail", 0)
    p.cache.keep(0, rows)
    p.model.keep(0, rows)
    p.check_rows(0)
    p.run([(0, 50, 1)], False)


@pytest.mark.parametrize("prompt", [False, True])
@pytest.mark.parametrize("which", ["q", "k", "v", "out"])
def test_misaligned_rows_are_refused(which, prompt):
    """Addresses that no float has are refused on the host; those that only lack the alignment of
    wide loads are taken."""
    import torch
    p = Pair(2, 1, 64, "int8", cap=64, seed=4)
    p.run([(0, 0, 40)], True)
    before = state(p)
    z = [torch.zeros(2, 1, w * 64, device="cuda") for w in (2, 1, 1, 2)]
    plan = jx.StepPlan(p.cache, p.layers, *z, [40], 2, 1, seq_ids=[0], prefill=prompt)
    at = getattr(plan.args, which)
    for offset in (1, 2, 3):
        setattr(plan.args, which, at + offset)
        refuses(_lib.JX_ERR_INVALID, plan.run)
        assert state(p) == before
    setattr(plan.args, which, at + 4)
    plan.run()
    torch.cuda.synchronize()
    assert p.cache.check_device_error() == 0 and p.cache.seq_pos(0) == 41
