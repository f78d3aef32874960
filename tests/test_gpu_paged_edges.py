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
