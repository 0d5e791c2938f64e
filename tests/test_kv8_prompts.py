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
