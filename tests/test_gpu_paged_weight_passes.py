"""Added-up weights of steps whose scores are too many to lie in scratch memory at once."""
import numpy as np
import pytest
import torch

import paged_model as pm
from test_gpu_paged import TYPES, dev, fill_new, on_gpu, run_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act,kind", TYPES)
@pytest.mark.parametrize("window,first", [(0, 0), (70, 5)])
@pytest.mark.parametrize("heads,kv,dim,lens,rows,ld", [
    (24, 2, 64, [90, 300, 0, 40], [200, 3, 0, 150], 6000),    # passes of 128 or 192 rows end within a sequence and between two
    (24, 2, 128, [700, 0], [300, 29], 12000),
])
def test_passes(pkg, act, kind, window, first, heads, kv, dim, lens, rows, ld):
    B = pm.Batch(48, lens, rows, kv, dim, 16, table_ld=ld, weights=True)
    fill_new(B)
    run_attention(pkg, B, act, kind, heads, window, first, accumulate=True, pad_rows=5, stride=8)


def test_passes_follow_the_scratch_memory(pkg):
    """Less of it, more passes, down to 128 rows; then the call is refused. What a row gets does not depend on them, and what a token
    gets by the order of sums alone: 600 weights below 1."""
    heads, kv, dim, rows = 12, 2, 64, 600
    B = pm.Batch(49, [50], [rows], kv, dim, 16, table_ld=100, weights=True)
    fill_new(B)
    cache, _, _ = on_gpu(pkg, B, "bf16")
    old = cache.weight.clone()
    q = torch.randn(rows, heads * dim, device="cuda")
    full = pkg.op_paged_attention_scratch(cache, rows, rows, heads, True)
    least = pkg.op_paged_attention_scratch(cache, 128, 128, heads, True).numel()
    assert least < full.numel()
    got = []
    for size in (full.numel(), full.numel() - 1, 2 * least, least):
        cache.weight.copy_(old)
        out = pkg.op_paged_attention(cache, q, dev(B.row_start), rows, heads, 0.125, accumulate=True, scratch=full[:size])
        got.append((out, cache.weight.clone()))
    with pytest.raises(pkg.W4A32Error):
        pkg.op_paged_attention(cache, q, dev(B.row_start), rows, heads, 0.125, accumulate=True, scratch=full[:least - 1])
    there = ~torch.isnan(old)
    for out, weight in got[1:]:
        assert bool(((out - got[0][0]).abs() <= 1e-5).all())
        assert bool(((weight - got[0][1]).abs()[there] <= 2.0 ** -24 * 2 * (rows * heads // kv) ** 0.5 * (1 + weight[there])).all())


def test_a_window_and_its_own_scratch_memory(pkg):
    """512 rows on a table for 131072 tokens"""
    B = pm.Batch(50, [2000], [512], 2, 64, 64, table_ld=2048, weights=True)
    fill_new(B)
    cache, _, _ = on_gpu(pkg, B, "bf16")
    own = pkg.op_paged_attention_scratch(cache, 512, 512, 12, True, 1024, 4)
    every = pkg.op_paged_attention_scratch(cache, 512, 512, 12, True)
    assert own.numel() < every.numel() // 4
    run_attention(pkg, B, "f32", "bf16", 12, 1024, 4, accumulate=True, scratch=own)
    run_attention(pkg, B, "f32", "bf16", 12, 1024, 4, accumulate=True, scratch=every)
    run_attention(pkg, B, "f32", "bf16", 12, 1024, 4, accumulate=True)


def test_a_captured_step_of_passes(pkg):
    heads, kv, dim, rows = 12, 2, 64, 500
    B = pm.Batch(51, [50, 9], [300, 200], kv, dim, 16, table_ld=100, weights=True)
    fill_new(B)
    cache, _, _ = on_gpu(pkg, B, "f16")
    old = torch.nan_to_num(cache.weight, nan=0.25)
    q, out, starts = torch.randn(rows, heads * dim, device="cuda"), torch.empty(rows, heads * dim, device="cuda"), dev(B.row_start)
    scratch = pkg.op_paged_attention_scratch(cache, 128, 128, heads, True)
    scratch = torch.empty(2 * scratch.numel(), dtype=scratch.dtype, device="cuda")

    def step():
        cache.weight.copy_(old)
        pkg.op_paged_attention(cache, q, starts, 300, heads, 0.125, accumulate=True, scratch=scratch, out=out)

    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
    for split in ([0, 300, 500], [0, 1, 129], [0, 0, 190], [0, 300, 500]):
        starts.copy_(torch.tensor(split, dtype=torch.int32))
        out.fill_(3.0)
        step()
        want = out.clone(), cache.weight.clone()
        out.fill_(3.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[0]) and torch.equal(cache.weight, want[1])
        assert bool((out[split[-1]:] == 3.0).all())
