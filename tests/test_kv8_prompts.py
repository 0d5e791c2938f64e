"""Prompt attention over the 8-bit cache: what the calls of the other tests leave out."""
import math

import pytest
import torch

from test_kv8 import DT, attend, batch, check

gpu = pytest.mark.gpu


def leave_nan_behind(mb=512):
    """Free memory that holds no numbers in any type, for the allocator to hand out again."""
    torch.cuda.empty_cache()
    held = [torch.full((n,), 255, dtype=torch.uint8, device="cuda") for n in (mb << 20, *[64 << 20] * 4, *[4 << 20] * 8, *[1 << 19] * 16, *[512] * 64)]
    torch.cuda.synchronize()
    del held


@gpu
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("new", [40, 300])
@pytest.mark.parametrize("window,lengths", [(100, (800, 5000)), (1, (641, 940)), (700, (5000, 700)), (0, (5000, 900))])
def test_requests_longer_than_their_block_table(D, new, window, lengths):
    """Keys without an entry in the table are not there: rows that see nothing else give zeros, whatever memory held before the call."""
    b = batch([new, new], [640 - new, 640 - new], 4, 2, D, 64, torch.bfloat16, "cuda", table_pad=0)
    b["lens"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    b["max_len"] = max(lengths)
    for _ in range(3):
        leave_nan_behind()
        check(attend(b, window), b, window)


@gpu
@pytest.mark.parametrize("D", [64, 128, 256, 96])
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("new,lengths,window", [(2, (1, 90), 0), (40, (12, 90), 0), (300, (12, 400), 0), (300, (12, 400), 5)])
def test_queries_that_are_not_numbers_and_see_nothing(D, dt, new, lengths, window):
    """A row in front of its request's first key gives zeros whatever its query holds."""
    b = batch([new, new], [0, 64], 4, 2, D, 64, DT[dt], "cuda", seed=new)
    b["lens"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")         # more queries than keys in the first request
    b["max_len"] = max(lengths)
    q = b["q"].clone()
    blind = new - lengths[0]
    q[0, 1, 3], q[blind - 1, 3, D - 1] = math.nan, math.inf
    q[blind, 0, 0] = -math.inf
    got = attend({**b, "q": q}, window).cpu()
    assert (got[:blind] == 0).all()
    assert got[blind, 1:].isfinite().all()
    got[blind, 0] = attend(b, window).cpu()[blind, 0]
    check(got, b, window)


@gpu
@pytest.mark.parametrize("D", [64, 128, 256, 96])
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("new,context,window", [(2, 0, 0), (40, 0, 0), (300, 0, 0), (300, 0, 1), (60, 5000, 1), (60, 5000, 0)])
def test_infinite_queries(D, dt, new, context, window):
    """A query with an infinity gives NaN, the one whose scores are all minus infinity (a single visible key, one sign) like the others."""
    b = batch([new], [context], 4, 2, D, 64, DT[dt], "cuda", seed=new + context)
    q = b["q"].clone()
    for h in range(4):
        q[h % 2, h, 0] = math.inf if h & 2 else -math.inf
    got = attend({**b, "q": q}, window).cpu()
    for h in range(4):
        assert got[h % 2, h].isnan().all()
        got[h % 2, h] = attend(b, window).cpu()[h % 2, h]
    check(got, b, window)


def scratch_of(f):
    """What ``f`` gives, and the bytes that it holds at most on top of that."""
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    out = f()
    torch.cuda.synchronize()
    return out, torch.cuda.max_memory_allocated() - before - out.numel() * out.element_size()


@gpu
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("new,window", [(300, 128), (300, 1000), (1, 128), (500, 1)])
def test_windows_behind_long_contexts(D, new, window):
    """Only what the window leaves is widened, at any place; the keys in front of it do not matter."""
    group = 8 if new > 1 else 32                   # one token of 32 heads a group is a prompt
    b = batch([new, new, new], [2000, 2100, 2303], 2 * group, 2, D, 64, torch.bfloat16, "cuda", seed=new)
    want = attend(b, window)
    check(want, b, window)
    front = 200_064 // 64                          # even: bits are the same only where tiles of 128 keys start at the same keys
    table = torch.zeros(3, front + b["table"].shape[1], dtype=torch.int32, device="cuda")
    for r, shift in enumerate((front, front - 2, front // 2 * 2 - 100)):           # whole tiles of 128 keys in front
        table[r, shift:shift + b["table"].shape[1]] = b["table"][r]
        b["lens"][r] += 64 * shift
    b["table"], b["max_len"] = table, int(b["lens"].max())
    got, scratch = scratch_of(lambda: attend(b, window))
    assert torch.equal(got, want)
    assert scratch < 3 * 2 * D * 4 * (window + new + 256) + 3 * new * 2 * group * (D + 1) * 4 * 32 + (1 << 20)


def limits(b, heads, window, D):
    """Bounds of the scratch that make one, two or more heads of a request fit, and one and two requests; a head's bytes."""
    new = b["max_q"]
    rows = -(-b["max_len"] // 128) * 128
    if window:
        rows = min(rows, -(-(window + new + 127) // 128) * 128)
    head = rows * D * 4
    return (1, 2 * head, 4 * head, heads * head, (heads + 1) * head, 2 * heads * head), head


@gpu
@pytest.mark.parametrize("D,heads", [(64, 6), (128, 6), (256, 5)])
@pytest.mark.parametrize("new,context,window", [([300, 257, 1], [40, 0, 900], 0), ([280], [3000], 0), ([300, 260], [900, 77], 150)])
def test_groups_of_requests_and_heads(monkeypatch, D, heads, new, context, window):
    from vllm_kunlun_b200.ops import kv8_cuda
    b = batch(new, context, 2 * heads, heads, D, 64, torch.bfloat16, "cuda", seed=D)
    check(attend(b, window, b["sinks"]), b, window, b["sinks"])
    for limit in limits(b, heads, window, D)[0]:
        monkeypatch.setattr(kv8_cuda, "SCRATCH", limit)
        check(attend(b, window, b["sinks"]), b, window, b["sinks"])


@gpu
@pytest.mark.parametrize("D,heads", [(64, 6), (128, 6), (256, 5)])
@pytest.mark.parametrize("window", [0, 2000])
def test_scratch_is_bounded(monkeypatch, D, heads, window):
    """Never more than the bound, or one head's rows: prompts that fill the GPU with one head, so that no row is split."""
    from vllm_kunlun_b200.ops import kv8_cuda
    b = batch([9700, 5000], [0, 1200], 2 * heads, heads, D, 64, torch.bfloat16, "cuda", seed=D)
    want = attend(b, window)
    bounds, head = limits(b, heads, window, D)
    for limit in bounds:
        monkeypatch.setattr(kv8_cuda, "SCRATCH", limit)
        got, scratch = scratch_of(lambda: attend(b, window))
        assert torch.equal(got, want)
        # the allocator counts whole blocks and splits none for a remainder of up to 1 MiB: three of them, with the result
        assert scratch <= max(limit, head) + (3 << 20), (limit, scratch)


def test_blocks_are_planned_beside_the_scratch(monkeypatch):
    """What prompts widen is not given to the pool."""
    from types import SimpleNamespace as NS

    from vllm_kunlun_b200.engine.runner import ModelRunner
    from vllm_kunlun_b200.ops import kv8_cuda
    monkeypatch.setattr(torch.cuda, "mem_get_info", lambda device=None: (40 << 30, 100 << 30))
    planned = {}
    for kind, per in (("auto", 4096), ("fp8_e4m3", 4096)):
        fake = NS(cfg=NS(cache=NS(num_blocks=None, gpu_memory_utilization=0.9, cache_dtype=kind), model=NS(hidden_size=4096)),
                  is_cuda=True, device="cuda", max_tokens=8192, max_bs=1 << 20, max_blocks_per_seq=1 << 20, _bytes_per_block=lambda: per)
        planned[kind] = ModelRunner._plan_num_blocks(fake)
    assert planned["auto"] - planned["fp8_e4m3"] == kv8_cuda.SCRATCH // 4096
