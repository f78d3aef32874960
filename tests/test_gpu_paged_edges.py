"""Attention over a paged cache at the edges of what its arrays and scores may hold.  Oracle and tolerances as in
test_gpu_paged.py."""

import numpy as np
import pytest
import torch

from helpers import assert_attn_close, randn_bf16, t2bits, t2f32
from oracle import attention_paged_ref
from test_gpu_paged import Step, check_attention, cke, pages_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("HD", [64, 128])
@pytest.mark.parametrize("rows,sequences,max_new", [(880, 48, 0), (880, 48, 880), (880, 150, 0), (2, 48, 2), (2, 150, 1), (7, 9000, 1)])
def test_offsets_that_decrease_give_zeros(gpu, rows, sequences, max_new, HD):
    """Sequences that overlap have more blocks than the launch has workgroups (of 880 rows and 48 sequences the pieces of 61 blocks
    would belong to none), and weights beyond 64 bits: no row is anyone's then.  The next step is served as ever."""
    QH, KVH, page, width = 4, 1, 1024, 128
    offsets = torch.tensor([0, rows] * (sequences // 2 + 1), dtype=torch.int32)[:sequences + 1]
    lens = torch.full((sequences,), 5616, dtype=torch.int32)
    lens[0] = 11120
    table = (torch.arange(sequences * width, dtype=torch.int32) % 12).view(sequences, width)
    q = randn_bf16((rows, QH, HD), 21).to(gpu)
    k, v = (randn_bf16((12, page, KVH, HD), s).to(gpu) for s in (22, 23))
    args = (table.to(gpu), offsets.to(gpu), lens.to(gpu))
    for at in (None, sequences // 2):      # decreasing throughout; and by one row in one place
        if at is not None:
            some = torch.arange(sequences + 1, dtype=torch.int32).clamp_(max=rows)
            some[at + 1:] = some[at] - 1 if some[at] > 0 else 0
            args[1].copy_(some)
        print(f"decreasing offsets: {rows} rows, {sequences} sequences, max_new {max_new}, HD {HD}, from {at}", flush=True)
        torch.full((rows, QH, HD), float("nan"), dtype=torch.bfloat16, device=gpu)      # (what the output's memory held before)
        out = cke().flash_attention_paged(q, k, v, *args, max_new)
        torch.cuda.synchronize()
        assert not t2bits(out).any()
    check_attention(gpu, Step(gpu, [(min(rows, 300), 5616), (1, 40)], 16), 4, 1, HD, what="the next step")


@pytest.mark.parametrize("HD", [64, 128])
@pytest.mark.parametrize("lengths", [[(300, 6000), (150, 700), (2, 40)], [(5, 9000), (3, 700), (2, 40)], [(1, 9000), (1, 700), (1, 40)]])
def test_scores_of_minus_infinity(gpu, lengths, HD):
    """All scores of a row minus infinity: the softmax is undefined, NaN as the formula has it, in blocks that are cut as in those
    that are not.  Some of them: those tokens have no part."""
    QH, KVH = 8, 2
    step = Step(gpu, lengths, 16)
    q = randn_bf16((step.rows, QH, HD), 41).abs()
    k, v = pages_of(step, KVH, HD, 42)
    tokens = k.view(-1, KVH, HD)
    tokens[torch.from_numpy(step.slots(0, 0, step.kv[0]))] = -float("inf")
    tokens[torch.from_numpy(step.slots(1, 0, 650)), 1] = -float("inf")
    tokens[torch.from_numpy(step.slots(2, 0, 40)), 0] = -float("inf")
    seen = [step.offsets[1] + i for i in range(step.new[1]) if step.kv[1] - step.new[1] + i >= 650]
    finite = np.zeros((step.rows, KVH), dtype=bool)
    finite[step.offsets[1]:step.offsets[2], 0] = True
    finite[seen, 1] = True
    finite[step.offsets[2]:, 1] = True
    finite = np.repeat(finite, QH // KVH, axis=1)
    with np.errstate(invalid="ignore"):
        ref = attention_paged_ref(t2f32(q), t2f32(k), t2f32(v), step.table, step.offsets, step.kv)
    assert np.isnan(ref[~finite]).all() and np.isfinite(ref[finite]).all()
    for most in (0, max(step.new)):
        print(f"scores of minus infinity: {lengths} HD={HD} max_new={most}", flush=True)
        out = cke().flash_attention_paged(q.to(gpu), k.to(gpu), v.to(gpu), *step.args, most)
        torch.cuda.synchronize()
        got = t2f32(out)
        assert np.isnan(got[~finite]).all()
        assert_attn_close(torch.from_numpy(got[finite]), ref[finite], what=f"beside scores of minus infinity, {lengths}")
