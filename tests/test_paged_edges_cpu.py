"""CPU tests of the paged cache's boundary: calls that are almost empty, workspaces (the host decides
both before anything is enqueued)."""
import ctypes as C
import re

import pytest

import cactus_amd.hip as H
from tests.test_paged_cpu import append, attend, cache, ragged, read, refused


@pytest.mark.parametrize("call", [append, attend])
@pytest.mark.parametrize("batch,tokens", [(0, 3), (3, 0)])
def test_without_offsets_rows_and_sequences_are_the_same_number_also_when_one_is_none(call, batch, tokens):
    assert refused(call(batch=batch, tokens=tokens), "one row per sequence")
    assert call(batch=batch, tokens=tokens, cu=1 << 20) == 0


def test_calls_without_sequences_or_rows_do_nothing():
    assert append(batch=0, tokens=0) == 0 and attend(batch=0, tokens=0) == 0
    assert read(batch=0) == 0 and read(rows=0) == 0 and ragged(batch=0) == 0 and ragged(tokens=0) == 0


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("context", [0, 500, 1 << 20])
def test_chunks_of_more_than_1024_sequences_need_no_workspace(dim, context):
    """Their row tiles fill the chip without splitting keys (64 rows each: all of them the tile kernel's)."""
    c = cache(head_dim=dim, kv_heads=1)
    need = lambda batch: H.lib.cactus_hip_attention_paged_workspace_bytes(C.byref(c), batch, 64 * batch, context, 1, 0, 0, 0)  # noqa: E731
    assert need(1025) == 0 and need(1 << 16) == 0
    # three sequences: two splits of the least number of keys, 256 at head_dim 64 and 128 above
    assert (need(3) > 0) == (context >= 2 * (256 if dim == 64 else 128))


def test_two_groups_of_waves_are_for_fp16_prompts_only():
    """max_context 0 is a legal bound over pages, and no sign of FP16 prompts: no kernel over pages has two groups."""
    names = set(re.findall(rb"attention_tile_kernelILi(\d+)ELb([01])ELi([12])E", open(H.SO_PATH, "rb").read()))
    assert names == {(d, p, g) for d in (b"64", b"128", b"256") for p in (b"0", b"1") for g in (b"1", b"2")
                     if g == b"1" or (p == b"0" and d != b"256")}


@pytest.mark.parametrize("call", [attend, ragged])
@pytest.mark.parametrize("scale", [1e16, -1e16, 1e30, 3e38])
def test_refuses_a_scale_whose_scores_leave_the_running_maximum_s_range(call, scale):
    assert refused(call(scale=scale), "scale")
