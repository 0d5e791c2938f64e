"""Prompt attention over the 8-bit cache: what the calls of the other tests leave out."""
import math

import pytest
import torch

from test_kv8 import DT, attend, batch, check

pytestmark = pytest.mark.gpu


def leave_nan_behind(mb=512):
    """Free memory that holds no numbers in any type, for the allocator to hand out again."""
    torch.cuda.empty_cache()
    held = [torch.full((n,), 255, dtype=torch.uint8, device="cuda") for n in (mb << 20, *[64 << 20] * 4, *[4 << 20] * 8, *[1 << 19] * 16, *[512] * 64)]
    torch.cuda.synchronize()
    del held


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
