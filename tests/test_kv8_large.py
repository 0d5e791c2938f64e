"""The 8-bit cache where offsets pass 32 bits: writes, reads and every attention kernel on blocks beyond 4 GiB."""
import pytest
import torch

from test_kv8 import DT, attend, batch, check, new_cache
from vllm_kunlun_b200 import ops
from vllm_kunlun_b200.ops.reference import attention as ra

pytestmark = pytest.mark.gpu


def far(b, D, block):
    """The batch's blocks as the last ones of a pool of 5 GiB whose other blocks hold no numbers."""
    small = b["cache"]
    page = small[0].numel()
    blocks = (5 << 30) // page + small.shape[0]
    first = blocks - small.shape[0]
    cache = torch.full((blocks, *small.shape[1:]), 255, dtype=torch.uint8, device="cuda")
    cache[first:] = small
    assert first * page > 1 << 32
    return {**b, "cache": cache, "table": torch.where(b["table"] >= 0, b["table"] + first, b["table"])}


@pytest.mark.parametrize("D,block", [(128, 64), (64, 16), (256, 64), (80, 16)])
def test_blocks_beyond_four_gigabytes(D, block):
    for new, context in (([1, 2], [700, 40]), ([30, 5], [100, 0]), ([300], [77])):
        b = batch(new, context, 4, 2, D, block, torch.bfloat16, "cuda", seed=D)
        want = attend(b)
        check(want, b)
        assert torch.equal(attend(far(b, D, block)), want)


@pytest.mark.parametrize("D,fused", [(128, True), (64, True), (128, False), (256, False)])
def test_writes_and_reads_beyond_four_gigabytes(D, fused):
    block, Hkv, T = 64, 2, 40
    blocks = (5 << 30) // (2 * Hkv * block * (D + 4))
    cache = new_cache(blocks, Hkv, block, D, "cuda", 0x11)
    g = torch.Generator(device="cuda").manual_seed(D)
    slots = blocks * block - 1 - torch.randperm(3 * block, generator=g, device="cuda")[:T]
    near = new_cache(4, Hkv, block, D, "cuda", 0x11)
    shift = (blocks - 4) * block
    x = torch.randn(T, (4 + 2 * Hkv) * D, generator=g, device="cuda").to(DT["bf16"])
    for c, s in ((cache, slots), (near, slots - shift)):
        if fused:
            cs = torch.cat([torch.ones(T, D // 2), torch.zeros(T, D // 2)], 1).cuda()
            ops.qkv_split_norm_rope_cache(x, torch.arange(T, device="cuda"), cs, None, None, 1e-6, 4, Hkv, D, True, c, s)
        else:
            k, v = x.view(T, -1, D)[:, 4:4 + Hkv], x.view(T, -1, D)[:, 4 + Hkv:]
            ops.reshape_and_cache(k, v, c, s)
    assert torch.equal(cache[-4:], near)
    assert int((cache[:-4] != 0x11).sum()) == 0
    for a, b in zip(ops.gather_kv_cache(cache, slots), ra.gather_kv_cache(near, slots - shift, torch.bfloat16)):
        assert torch.equal(a, b)
