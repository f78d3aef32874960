"""Refusals of the paged entry points through the C ABI: every check runs before the first HIP call, so no GPU is needed."""

import ctypes

import pytest

from custom_kernels import _l3lib
from custom_kernels._l3lib import PagedStep

FAKE = 1 << 20   # an aligned address that is never read

NULL, HEAD_SIZE, HEAD_RATIO, SHAPE, STRIDE, ALIGNMENT, WORKSPACE, SCALE = -1, -2, -3, -4, -5, -6, -7, -12


def step(**changes):
    fields = dict(q_offsets=FAKE, kv_lens=FAKE, page_table=FAKE, table_stride=8, rows=5, sequences=3, max_pages=8, pages=20, page_size=16,
                  max_new=0)
    return PagedStep(**{**fields, **changes})


def i64(*values):
    return (ctypes.c_int64 * len(values))(*values)


STEPS = [(dict(q_offsets=None), NULL), (dict(kv_lens=None), NULL), (dict(page_table=None), NULL), (dict(rows=0), SHAPE),
         (dict(sequences=0), SHAPE), (dict(sequences=65537), SHAPE), (dict(max_pages=0), SHAPE), (dict(pages=0), SHAPE),
         (dict(page_size=4), SHAPE), (dict(page_size=24), SHAPE), (dict(page_size=0), SHAPE), (dict(page_size=-16), SHAPE),
         (dict(max_pages=2 ** 27), SHAPE), (dict(max_new=-1), SHAPE), (dict(table_stride=-8), STRIDE), (dict(kv_lens=FAKE + 2), ALIGNMENT)]


def attend(s=None, q=FAKE, k=FAKE, v=FAKE, out=FAKE, ws=None, nbytes=0, heads=(8, 2, 64), qs=(512, 64), ks=(2048, 128, 64),
           vs=(2048, 128, 64), os=(512, 64), scale=0.125):
    return _l3lib.load().l3_attn_paged(q, k, v, out, ws, nbytes, s if s is not None else step(), *heads, i64(*qs), i64(*ks), i64(*vs),
                                       i64(*os), scale, None)


def append(s=None, x=FAKE, f=FAKE, qw=None, kw=None, q=FAKE, k=FAKE, v=FAKE, heads=(8, 2, 64), rows=32, xs=768, ks=(2048, 128, 64),
           vs=(2048, 128, 64)):
    return _l3lib.load().l3_rot_embed_append_paged(x, f, qw, kw, 1e-5, q, k, v, s if s is not None else step(), *heads, rows, xs, i64(*ks),
                                                   i64(*vs), None)


def norm(q=FAKE, k=FAKE, qw=FAKE, kw=FAKE, f=FAKE, qo=FAKE, ko=FAKE, dims=(2, 3, 8, 2, 64), qs=(2304, 768, 64), ks=(2304, 768, 64)):
    return _l3lib.load().l3_norm_rot_embed(q, k, qw, kw, 1e-5, f, qo, ko, *dims, i64(*qs), i64(*ks), None)


@pytest.mark.parametrize("changes,code", STEPS)
def test_a_step_is_checked(changes, code):
    assert attend(step(**changes)) == code
    assert append(step(**changes)) == code
    assert _l3lib.load().l3_attn_paged_workspace_bytes(step(**changes), 8, 2, 64) == 0


@pytest.mark.parametrize("changes,code", [
    (dict(q=None), NULL), (dict(k=None), NULL), (dict(v=None), NULL), (dict(out=None), NULL), (dict(heads=(8, 2, 96)), HEAD_SIZE),
    (dict(heads=(8, 3, 64)), SHAPE), (dict(heads=(0, 2, 64)), SHAPE), (dict(heads=(34, 2, 64)), HEAD_RATIO), (dict(scale=0.0), SCALE),
    (dict(scale=float("nan")), SCALE), (dict(scale=float("inf")), SCALE), (dict(qs=(508, 64)), STRIDE), (dict(qs=(-512, 64)), STRIDE),
    (dict(os=(512, 0)), STRIDE), (dict(ks=(2048, 132, 64)), STRIDE), (dict(vs=(2048, 128, 4)), STRIDE), (dict(ks=(2048, 2 ** 24, 64)), STRIDE),
    (dict(q=FAKE + 8), ALIGNMENT), (dict(out=FAKE + 2), ALIGNMENT), (dict(v=FAKE + 4), ALIGNMENT), (dict(ws=FAKE + 16, nbytes=1 << 40), ALIGNMENT)])
def test_attention_arguments(changes, code):
    assert attend(**changes) == code


def test_a_workspace_that_is_too_small():
    needed = _l3lib.load().l3_attn_paged_workspace_bytes(step(), 8, 2, 64)
    if needed:
        assert attend(ws=FAKE, nbytes=needed - 1) == WORKSPACE


@pytest.mark.parametrize("changes,code", [
    (dict(x=None), NULL), (dict(f=None), NULL), (dict(q=None), NULL), (dict(k=None), NULL), (dict(heads=(8, 2, 32)), HEAD_SIZE),
    (dict(heads=(8, 0, 64)), SHAPE), (dict(rows=0), SHAPE), (dict(xs=764), STRIDE), (dict(ks=(0, 128, 64)), STRIDE),
    (dict(vs=(2048, 128, 0)), STRIDE), (dict(qw=FAKE + 2), ALIGNMENT), (dict(kw=FAKE + 8), ALIGNMENT), (dict(x=FAKE + 8), ALIGNMENT)])
def test_append_arguments(changes, code):
    assert append(**changes) == code


@pytest.mark.parametrize("changes,code", [
    (dict(qw=None), NULL), (dict(kw=None), NULL), (dict(ko=None), NULL), (dict(dims=(2, 3, 8, 2, 80)), HEAD_SIZE), (dict(dims=(0, 3, 8, 2, 64)), SHAPE),
    (dict(dims=(2, 3, 8, 70000, 64)), SHAPE), (dict(qs=(2300, 768, 64)), STRIDE), (dict(ks=(2304, 768, -64)), STRIDE), (dict(f=FAKE + 4), ALIGNMENT),
    (dict(q=FAKE + 8), ALIGNMENT)])
def test_norm_rot_embed_arguments(changes, code):
    assert norm(**changes) == code


def test_more_rows_than_a_launch_holds():
    rows = 2 ** 23
    assert attend(step(rows=rows + 1)) == SHAPE and append(step(rows=rows + 1)) == SHAPE
    assert norm(dims=(2, rows + 1, 8, 2, 64)) == SHAPE
    heads = 512
    assert attend(step(rows=rows, sequences=60000), heads=(heads, heads, 64), qs=(heads * 64, 64), os=(heads * 64, 64),
                  ks=(16 * heads * 64, heads * 64, 64), vs=(16 * heads * 64, heads * 64, 64)) == SHAPE


@pytest.mark.parametrize("rows,max_pages,max_new", [(5, 64, 1), (5, 64, 0), (300, 256, 0), (300, 256, 300)])
def test_a_workspace_of_a_step_that_may_be_cut_is_checked(rows, max_pages, max_new):
    """Page tables wide enough for both forms to cut blocks."""
    s = step(rows=rows, max_pages=max_pages, table_stride=max_pages, max_new=max_new)
    needed = _l3lib.load().l3_attn_paged_workspace_bytes(s, 8, 2, 64)
    assert needed > 0
    for nbytes in (0, 1, needed - 1):
        assert attend(s, ws=FAKE, nbytes=nbytes) == WORKSPACE
    assert attend(s, ws=FAKE + 128, nbytes=needed) == ALIGNMENT
