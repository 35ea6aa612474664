"""Numbers that the paged operators' C interface cannot hold are refused with the framework's error, whichever way they come."""
import ctypes
import types

import pytest
import torch

from test_paged_refusals import cache

FAR = [2 ** 31, 2 ** 32 + 3, 2 ** 64, -1, -2 ** 40]


@pytest.fixture
def some(pkg):
    args = cache(pkg)
    return types.SimpleNamespace(args=args, _ref=ctypes.byref(args), dim=64)


@pytest.mark.parametrize("far", FAR)
def test_scratch_memory(pkg, some, far):
    for at in ((far, 3, 4), (5, far, 4), (5, 3, far)):
        with pytest.raises(pkg.W4A32Error):
            pkg.op_paged_attention_scratch(some, *at)
        with pytest.raises(pkg.W4A32Error):
            pkg.op_verify_drafts_scratch(*at)
    for at in ((far, 0), (5, far)):
        with pytest.raises(pkg.W4A32Error):
            pkg.op_paged_attention_scratch(some, 5, 3, 4, False, *at)
    with pytest.raises(pkg.W4A32Error):
        pkg.op_paged_evict_scratch(some, far)


@pytest.mark.gpu
def test_calls(pkg):
    k, v = (torch.randn(4, 2, 16, 64, device="cuda") for _ in range(2))
    table, length = torch.arange(4, dtype=torch.int32, device="cuda")[None], torch.zeros(1, dtype=torch.int32, device="cuda")
    c = pkg.PagedCache(k, v, table, length)
    q, starts = torch.randn(2, 256, device="cuda"), torch.tensor([0, 2], dtype=torch.int32, device="cuda")
    kv, scratch = torch.randn(2, 128, device="cuda"), pkg.op_paged_attention_scratch(c, 2, 2, 4)
    logits, tokens = torch.randn(2, 50, device="cuda"), torch.zeros(2, dtype=torch.int64, device="cuda")
    u, choice = torch.rand(2, device="cuda"), torch.rand(1, device="cuda")
    room = pkg.op_verify_drafts_scratch(2, 50, 1)
    for far in FAR:
        with pytest.raises(pkg.W4A32Error):
            pkg.op_paged_append(c, q, kv, kv, starts, max_rows=far)
        for mine in (scratch, None):
            with pytest.raises(pkg.W4A32Error):
                pkg.op_paged_attention(c, q, starts, far, 4, 0.1, scratch=mine)
        with pytest.raises(pkg.W4A32Error):
            pkg.op_verify_drafts(logits, starts, far, tokens, u, choice, 1.0, scratch=room)
    for temperature in (1e39, -1e300, float("inf"), float("nan")):
        with pytest.raises(pkg.W4A32Error):
            pkg.op_verify_drafts(logits, starts, 2, tokens, u, choice, temperature, scratch=room)


@pytest.mark.gpu
def test_rows_farther_apart_than_an_int(pkg):
    """A stride of 2^32 + 128 elements is not one of 128"""
    k, v = (torch.zeros(2, 1, 16, 64, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    c = pkg.PagedCache(k, v, torch.arange(2, dtype=torch.int32, device="cuda")[None], torch.zeros(1, dtype=torch.int32, device="cuda"))
    wide = torch.empty(2 ** 32 + 256, dtype=torch.bfloat16, device="cuda").as_strided((2, 64), (2 ** 32 + 128, 1))
    near, starts = torch.ones(2, 64, dtype=torch.bfloat16, device="cuda"), torch.tensor([0, 2], dtype=torch.int32, device="cuda")
    for rows in ((wide, near, near), (near, wide, near), (near, near, wide)):
        with pytest.raises(pkg.W4A32Error):
            pkg.op_paged_append(c, *rows, starts)
    assert not bool(c.k.any()) and not bool(c.v.any())
