"""Decode attention over the 8-bit cache where weights and values of a row lie far apart, against 64-bit results.

Limits.  With p the softmax weights, s a value row's scale and c its codes, an output may be off by

* the score's error (fp32 sums of D products; queries in pieces whose last step leaves 2^-24 of the row's largest element at most), which
  multiplies weights by at most ``1 + 2 * off``,
* the rounding of a weight: 2^-8 of it for bf16 queries (three e5m2 pieces take 2^-9, the fp16 number in front of them 2^-11), 2^-11 + 2^-12
  of it for fp16 (an fp16 number and three e4m3 pieces),
* for weights that are tiny beside the row's largest, half a step of the last piece: no more than ``FLOOR`` times the largest ``p * s`` that
  the row sees per key, times that key's codes,
* and one rounding at the end, half a unit of the type.
"""
import math

import pytest
import torch

from vllm_kunlun_b200 import ops
from vllm_kunlun_b200.ops.reference import attention as ra

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16}
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
ROUND = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11 + 2.0 ** -12}
FLOOR = 2.0 ** -25
BLOCK = 64


def pool(k, v):
    """An 8-bit cache of whole blocks holding ``k, v [n, heads, D]`` in the order of ``table``, and that table."""
    n, H, D = k.shape
    blocks = -(-n // BLOCK)
    table = torch.randperm(blocks, generator=torch.Generator().manual_seed(n)).cuda()
    cache = torch.zeros(blocks, 2, H, BLOCK, D + 4, dtype=torch.uint8, device="cuda")
    codes, scales = ra.kv8_views(cache)
    c, s = ra.kv8_rows(k, v)
    pad = blocks * BLOCK - n
    c = torch.nn.functional.pad(c.view(torch.uint8), (0, 0, 0, 0, 0, 0, 0, pad)).view(blocks, BLOCK, 2, H, D).permute(0, 2, 3, 1, 4)
    s = torch.nn.functional.pad(s, (0, 0, 0, 0, 0, pad)).view(blocks, BLOCK, 2, H).permute(0, 2, 3, 1)
    codes.view(torch.uint8)[table] = c
    scales[table] = s
    return cache, table.int()[None]


def stored(k, v):
    """Codes and scales as the cache holds them, in 64 bits: ``(ck, sk, cv, sv)``, ``[n, heads, D]`` and ``[n, heads, 1]``."""
    c, s = ra.kv8_rows(k, v)
    return c[:, 0].double(), s[:, 0, :, None].double(), c[:, 1].double(), s[:, 1, :, None].double()


def results(q, k, v, window=0):
    """What the last ``len(q)`` tokens' queries give, the weights, and how far a result may be off; ``[new, H, D]``, ``[H, new, n]``."""
    ck, sk, cv, sv = stored(k, v)
    g, n, D = q.shape[1] // k.shape[1], len(k), q.shape[2]
    kk, vv, cc, ss = (x.repeat_interleave(g, 1) for x in (ck * sk, cv * sv, cv, sv))
    x, scale = q.double(), D ** -0.5
    pos = torch.arange(n - len(q), n, device="cuda")[:, None]
    j = torch.arange(n, device="cuda")
    seen = j <= pos
    if window:
        seen &= j > pos - window
    s = (torch.einsum("ihd,jhd->hij", x, kk) * scale).masked_fill(~seen, -math.inf)
    mag = torch.einsum("ihd,jhd->hij", x.abs(), kk.abs()) * scale
    off = (D + 8) * 2.0 ** -24 * mag + 2.0 ** -24 * x.abs().amax(-1).T[:, :, None] * kk.abs().sum(-1).T[:, None] * scale
    off = torch.where(seen, off, 0.0).amax(2).T[..., None]
    p = torch.softmax(s, 2)
    out = torch.einsum("hij,jhd->ihd", p, vv)
    lim = torch.einsum("hij,jhd->ihd", p, vv.abs()) * (ROUND[q.dtype] + 2 * off + 2.0 ** -17)
    top = (p * ss[:, :, 0].T[:, None]).amax(2)
    lim += FLOOR * top.T[..., None] * torch.einsum("ij,jhd->ihd", seen.double(), cc.abs())
    return out, p, lim


def attend(q, k, v, window=0, requests=1):
    """``[requests, new, H, D]``: so many requests of the same tokens, over the same blocks."""
    cache, table = pool(k, v)
    n, new = len(k), len(q)
    lens = torch.full((requests,), n, dtype=torch.int32, device="cuda")
    qsl = torch.arange(requests + 1, device="cuda").int() * new
    out = ops.paged_attention(q.repeat(requests, 1, 1), cache, table.repeat(requests, 1), lens, qsl, q.shape[2] ** -0.5, new, n,
                              window or None)
    return out.double().unflatten(0, (requests, new))


def compare(got, want, lim, dt, whole=True):
    """Element by element, and every row as a whole to 2^-7: two roundings to bf16."""
    d = (got - want).abs()
    over = (d - lim - UNIT[dt] * want.abs() * 1.001 - (2.0 ** -25 if dt == torch.float16 else 0)).amax()
    rows = d.norm(dim=-1) / want.norm(dim=-1)
    assert not whole or float(rows.max()) <= 2.0 ** -7, f"a row is off by {float(rows.max()):.2%}"
    assert float(over) <= 0, f"{float(over)} over"


def rows_of(n, new, H, Hkv, D, dt, seed):
    """Queries, keys and values with components in common, so that sums over many keys do not cancel."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.randn(new, H, D, generator=g, device="cuda")
    k = torch.randn(n, Hkv, D, generator=g, device="cuda")
    v = 1 + 0.5 * torch.randn(n, Hkv, D, generator=g, device="cuda")
    return q.to(dt), k, v


@pytest.mark.parametrize("n,share", [(4096, 0.95), (8192, 0.8), (8192, 0.95), (8192, 0.99), (16384, 0.9), (32768, 0.8), (32768, 0.9),
                                     (32768, 0.97)])
@pytest.mark.parametrize("D,group", [(64, 4), (64, 16), (128, 4), (128, 8), (128, 16), (256, 4), (256, 8)])
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("size", [0.05, 1.0])
def test_a_key_that_holds_most_of_a_row(n, share, D, group, dt, size):
    """The first key has ``share`` of every row's weight and a value of ``size``: the others, each tiny beside it, keep their part, in a
    row that is cut into many pieces (one request) and in rows that are not (many)."""
    q, k, v = rows_of(n, 1, group, 1, D, DT[dt], n + group)
    k[:, :, 0] = 0
    k[0] = 0
    k[0, 0, 0] = 16.0                        # a power of two: its code is exact
    v[0] *= size
    ck, sk, _, _ = stored(k, v)
    s = torch.einsum("hd,jd->hj", q[0].double(), (ck * sk)[1:, 0]) * D ** -0.5
    # the first element of a query meets the first key alone
    q[0, :, 0] = ((torch.logsumexp(s, 1) + math.log(share / (1 - share))) / (16.0 * D ** -0.5)).to(q.dtype)
    want, p, lim = results(q, k, v)
    assert (p[:, 0, 0] - share).abs().max() < 0.03
    for requests in (1, 300):
        compare(attend(q, k, v, requests=requests), want, lim, q.dtype)


@pytest.mark.parametrize("size,others", [(2.0 ** 10, 1.0), (2.0 ** 13, 1.0), (6e4, 1.0), (6e4, 2.0 ** -8)])
@pytest.mark.parametrize("D,group", [(64, 2), (64, 8), (128, 4), (128, 8), (256, 2), (256, 8)])
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("where", ["in front of the window", "a later token", "hardly any weight", "a small scale of its own"])
def test_a_value_far_larger_than_the_others(where, dt, D, group, size, others):
    """A row that does not see the large value, or gives it next to no weight, has its result from the others."""
    n, new, window = 3000, 2, 0
    q, k, v = rows_of(n, new, group, 1, D, DT[dt], D + group)
    v *= others                                        # 2^-8: the smallest scale of the format, beside its largest
    big = torch.ones(D, device="cuda") * size
    check = slice(None)
    if where == "in front of the window":
        window = 700                                   # the first row's window starts at 2299; tiles start at multiples of 128 or 256
        v[2290:2299, 0] = big
    elif where == "a later token":
        v[n - 1, 0] = big
        check = slice(0, 1)                            # the second row sees it
    elif where == "hardly any weight":
        k[:, :, 0] = 0
        k[100, 0] = 0
        k[100, 0, 0] = -256.0
        q[..., 0] = 60.0 * D ** 0.5 / 256              # its score is -60, the others' are around 0
        v[100, 0] = big
    else:
        v[5:900] *= 2.0 ** -20                         # small, large and ordinary ones in one tile, the large one with no weight
        k[:, :, 0] = 0
        k[100, 0] = 0
        k[100, 0, 0] = -256.0
        q[..., 0] = 60.0 * D ** 0.5 / 256
        v[100, 0] = big
    want, p, lim = results(q, k, v, window)
    for requests in (1, 300):
        compare(attend(q, k, v, window, requests)[:, check], want[check], lim[check], q.dtype)


@pytest.mark.parametrize("ratio", [2.0 ** 7, 2.0 ** 11, 2.0 ** 13, 2.0 ** 15])
@pytest.mark.parametrize("D,group", [(64, 2), (64, 16), (128, 4), (128, 16), (256, 4)])
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("new", [1, 20, 300])
def test_a_query_element_far_larger_than_the_others(new, dt, D, group, ratio):
    """One element of every query is ``ratio`` times the others and meets keys of zero there: the others' digits make the scores."""
    n = new + 4                                        # few keys: errors of single scores show
    q, k, v = rows_of(n, new, group, 1, D, DT[dt], D + group)
    k *= 2
    v[::2] *= -1
    k[:, :, 5] = 0
    q[..., 5] = ratio
    want, p, lim = results(q, k, v)
    compare(attend(q, k, v), want, lim, q.dtype, whole=ratio < 2.0 ** 15)


@pytest.mark.parametrize("D", [128])
def test_a_kernel_in_front_that_takes_its_time(D):
    """A decode call that starts while the kernel in front of it runs on: its bounded waits do not count that kernel's time (three
    seconds of attention over 2^27 keys of one block)."""
    from vllm_kunlun_b200.ops import gemm_cuda
    q, k, v = rows_of(500, 1, 4, 2, D, torch.bfloat16, D)
    cache, table = pool(k, v)
    lens, qsl = torch.tensor([500], dtype=torch.int32, device="cuda"), torch.tensor([0, 1], dtype=torch.int32, device="cuda")

    def step():
        return ops.paged_attention(q, cache, table, lens, qsl, D ** -0.5, 1, 500, stable_metadata=True)

    want = step()
    block, n = 1 << 16, 1 << 27
    slow = torch.zeros(1, 2, 1, block, 20, dtype=torch.uint8, device="cuda")
    blocks = torch.zeros(1, n // block, dtype=torch.int32, device="cuda")
    long_lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    one = torch.zeros(1, 1, 16, device="cuda")
    ops.paged_attention(one, slow, blocks, lens, qsl, 1.0, 1, 500)                # loads the kernel
    torch.cuda.synchronize()
    start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    start.record()
    ops.paged_attention(one, slow, blocks, long_lens, qsl, 1.0, 1, n)
    got = step()
    end.record()
    torch.cuda.synchronize()
    gemm_cuda.check_status()
    assert torch.equal(got, want)
    assert start.elapsed_time(end) > 100, "the kernel in front was over too soon to show anything"
