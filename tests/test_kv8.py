"""The 8-bit key / value cache: writes, reads and attention against 64-bit oracles.

Tolerances.  A rounding to a type with unit u (``torch.finfo(t).eps / 2``) is off by at most u of the value: bf16 2^-8, fp16 2^-11,
e4m3 2^-4 (2^-10 of a scale below its smallest normal number).  fp32 sums of n products are off by at most about n 2^-24 of the
sum of magnitudes.
"""
import math

import pytest
import torch

from vllm_kunlun_b200 import ops
from vllm_kunlun_b200.ops.reference import attention as ra

gpu = pytest.mark.gpu
DEVICES = ["cpu", pytest.param("cuda", marks=gpu)]
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def new_cache(blocks, heads, block, dim, device, fill=0):
    return torch.full((blocks, 2, heads, block, dim + 4), fill, dtype=torch.uint8, device=device)


def special_rows(T, H, D, dt, seed=0):
    """Rows of very different sizes; NaN, infinities, zeros, exact powers, the ends of the range."""
    g = torch.Generator().manual_seed(seed)
    k, v = (torch.randn(T, H, D, generator=g) * torch.exp2(torch.randint(-30, 18, (T, H, 1), generator=g).float()) for _ in range(2))
    big = 60000.0
    for i, x in enumerate((0.0, 448.0, 449.0, 448.0 * 128, big, 2.0 ** -24, 1.75, 1.0)):
        k[i % T, i % H] = 0
        k[i % T, i % H, i % D] = -x
    v[1 % T, 0, 3 % D] = math.inf
    k[2 % T, H - 1, 5 % D] = -math.inf
    if T > 4:
        v[3, 0, 1] = math.nan
        k[4, H - 1, 0] = math.nan
    return k.to(dt), v.to(dt)


# ----------------------------------------------------------------------------- writing and reading back

def test_rows_against_the_definition():
    """The oracle's codes and scales from the definition, one value at a time."""
    k, v = special_rows(9, 2, 16, torch.float32)
    codes, scales = ra.kv8_rows(k, v)
    grid = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    grid = grid[grid.isfinite()]
    for t in range(9):
        for h in range(2):
            rows = torch.stack([k[t, h], v[t, h]]).double()
            if rows.isnan().any():
                assert scales[t, :, h].isnan().all() and (codes[t, :, h].view(torch.uint8) == 0).all()
                continue
            for w in range(2):
                amax = float(rows[w].abs().max())
                e = next((e for e in range(-15, 8) if amax <= 448 * 2.0 ** e), 7)
                assert float(scales[t, w, h]) == 2.0 ** e
                x = (rows[w] / 2.0 ** e).clamp(-448, 448)
                c = codes[t, w, h].double()
                assert ((c - x).abs() <= (grid[None] - x[:, None]).abs().amin(1)).all()    # nothing of the grid is nearer


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("H,D,block", [(1, 16, 4), (2, 64, 16), (8, 128, 64), (3, 80, 12), (2, 256, 32), (1, 512, 64)])
def test_put_and_read_back(device, dt, H, D, block):
    T, blocks = 21, 9
    k, v = special_rows(T, H, D, DT[dt], seed=D)
    g = torch.Generator().manual_seed(1)
    slots = torch.randperm(blocks * block, generator=g)[:T]
    slots[5], slots[6] = -1, blocks * block            # padding, and a slot behind the pool
    want = new_cache(blocks, H, block, D, "cpu", 0x5a)
    ra.reshape_and_cache_kv8(k, v, want, slots)
    got = new_cache(blocks, H, block, D, device, 0x5a)
    # values as a slice of a wider projection row, as a split leaves them
    wide = torch.cat([torch.zeros_like(v[:, :1]), v], 1).to(device)[:, 1:]
    ops.reshape_and_cache(k.to(device), wide, got, slots.to(device))
    (wc, ws), (gc, gs) = ra.kv8_views(want), ra.kv8_views(got.cpu())
    assert torch.equal(wc.view(torch.uint8), gc.view(torch.uint8))
    assert torch.equal(ws.isnan(), gs.isnan()) and torch.equal(ws.nan_to_num(), gs.nan_to_num())
    pick = torch.cat([slots, torch.tensor([-7, blocks * block + 3, int(slots[0])])])
    for out in (torch.float32, torch.bfloat16, torch.float16):
        wk, wv = ra.gather_kv_cache(want, pick, torch.float32)
        gk, gv = ops.gather_kv_cache(got, pick.to(device), out)
        for a, b in ((wk, gk), (wv, gv)):
            assert torch.equal(a.nan_to_num(7e4), b.cpu().float().nan_to_num(7e4))     # every value is exact in each type
            assert (b[-3:-1] == 0).all()


@pytest.mark.parametrize("device", DEVICES)
def test_read_back_of_a_16_bit_cache(device):
    cache = torch.randn(5, 2, 3, 16, 64, dtype=torch.bfloat16, device=device)
    slots = torch.tensor([79, 0, -1, 33, 80, 33], device=device)
    k, v = ops.gather_kv_cache(cache, slots)
    for i, s in enumerate(slots.tolist()):
        for w, x in enumerate((k, v)):
            assert torch.equal(x[i], cache[s // 16, w, :, s % 16] if 0 <= s < 80 else torch.zeros_like(x[i]))
    with pytest.raises(ValueError):
        ops.gather_kv_cache(cache, slots, torch.float16)


def rotated64(x, cs, neox):
    hr = cs.shape[-1] // 2
    c, s = cs[:, None, :hr], cs[:, None, hr:]
    out = x.clone()
    a, b = (x[..., :hr], x[..., hr:2 * hr]) if neox else (x[..., 0:2 * hr:2], x[..., 1:2 * hr:2])
    ra_, rb_ = a * c - b * s, b * c + a * s
    if neox:
        out[..., :hr], out[..., hr:2 * hr] = ra_, rb_
    else:
        out[..., 0:2 * hr:2], out[..., 1:2 * hr:2] = ra_, rb_
    return out


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dt,H,Hkv,D,rot,neox,norm,gemma,block,T", [
    ("bf16", 32, 8, 128, 128, True, False, False, 64, 5),
    ("bf16", 5, 1, 128, 128, True, True, False, 16, 33),
    ("fp16", 4, 2, 128, 128, True, True, True, 64, 401),
    ("bf16", 3, 3, 128, 128, False, True, False, 64, 7),
    ("bf16", 8, 2, 256, 64, True, True, True, 32, 9),
    ("fp16", 14, 2, 64, 64, True, False, False, 16, 3),
    ("fp32", 2, 1, 80, 32, True, True, False, 12, 6),
    ("bf16", 2, 1, 512, 512, True, False, False, 64, 2)])
def test_fused_write(device, dt, H, Hkv, D, rot, neox, norm, gemma, block, T):
    g = torch.Generator().manual_seed(D + T)
    t = DT[dt]
    wide = (torch.randn(T, (H + 2 * Hkv) * D + 8, generator=g) * 2).to(t).to(device)
    qkv = wide[:, 8:]                                            # strided rows
    pos = torch.randint(0, 50, (T,), generator=g)
    angle = torch.arange(50).double()[:, None] * 10000.0 ** (-torch.arange(0, rot, 2).double() / rot)
    cos_sin = torch.cat([angle.cos(), angle.sin()], -1).float()
    qw, kw = ((1.0 - gemma + 0.2 * torch.randn(D, generator=g)).to(t) if norm else None for _ in range(2))
    blocks = T // block + 2
    slots = torch.randperm(blocks * block, generator=g)[:T]
    if T > 2:
        slots[1] = -1
    cache = new_cache(blocks, Hkv, block, D, device, 0x33)
    dev = [x if x is None else x.to(device) for x in (pos, cos_sin, qw, kw)]
    q = ops.qkv_split_norm_rope_cache(qkv, *dev, 1e-6, H, Hkv, D, neox, cache, slots.to(device), gemma).cpu()
    x = qkv.cpu().double().view(T, H + 2 * Hkv, D)
    rows = [x[:, :H], x[:, H:H + Hkv]]
    if norm:
        rows = [y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6) * (w.double() + gemma) for y, w in zip(rows, (qw, kw))]
    cs = cos_sin.double()[pos]
    # fp32 between load and rounding: a dozen roundings of sums up to the pair's magnitudes
    near = [16 * 2.0 ** -24 * y.abs().amax(-1, keepdim=True) * 2 for y in rows]
    wq, wk = (rotated64(y, cs, neox) for y in rows)
    assert ((q.view(T, H, D).double() - wq).abs() <= UNIT[t] * wq.abs() * 1.001 + near[0] + (2.0 ** -25 if t == torch.float16 else 0)).all()
    codes, scales = ra.kv8_views(cache.cpu())
    for which, (want, slack) in enumerate(((wk, near[1]), (x[:, H + Hkv:], torch.zeros(())))):
        for i in range(T):
            s = int(slots[i])
            if s < 0:
                continue
            sc = scales[s // block, which, :, s % block].double()[:, None]
            y = want[i]
            lim = slack[i] if slack.dim() else slack
            amax = y.abs().amax(-1, keepdim=True)
            assert (amax <= 448 * sc + lim).all() and ((amax > 224 * sc - lim) | (sc == 2.0 ** -15)).all()
            got = codes[s // block, which, :, s % block].double() * sc
            assert ((got - y).abs() <= torch.maximum(2.0 ** -4 * y.abs(), sc * 2.0 ** -10) + lim * 1.1).all()
    untouched = torch.ones(blocks * block, dtype=torch.bool)
    untouched[slots[slots >= 0]] = False
    raw = codes.view(torch.uint8).permute(0, 3, 1, 2, 4).reshape(blocks * block, -1)[untouched]
    assert (raw == 0x33).all()


@gpu
@pytest.mark.parametrize("H,Hkv,norm", [(32, 4, True), (7, 3, False), (1, 1, True)])
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
def test_fused_write_of_many_tokens(dt, H, Hkv, norm):
    """The same bits as in small calls; a NaN or an infinity in a key or value marks its token and head alone."""
    T, D, block = 3700, 128, 16
    g = torch.Generator().manual_seed(H)
    qkv = torch.randn(T, (H + 2 * Hkv) * D, generator=g).to(DT[dt])
    x = qkv.view(T, H + 2 * Hkv, D)
    x[10, H, 5] = math.nan                       # key
    x[11, H + 2 * Hkv - 1, 127] = math.nan       # value
    x[12, H + Hkv, 64] = math.inf                # value: saturates
    qkv = qkv.cuda()
    w = [(1 + 0.1 * torch.randn(D, generator=g)).to(DT[dt]).cuda() if norm else None for _ in range(2)]
    angle = torch.rand(T, 64, generator=g) * 6.3
    cs = torch.cat([angle.cos(), angle.sin()], -1).cuda()
    pos = torch.arange(T).cuda()
    slots = torch.randperm(T + 60, generator=g)[:T].cuda()
    caches = [new_cache((T + 60 + block) // block, Hkv, block, D, "cuda", 0x11) for _ in range(2)]
    q = ops.qkv_split_norm_rope_cache(qkv, pos, cs, *w, 1e-6, H, Hkv, D, True, caches[0], slots)
    parts = [ops.qkv_split_norm_rope_cache(qkv[i:i + 370], pos[i:i + 370], cs, *w, 1e-6, H, Hkv, D, True, caches[1], slots[i:i + 370])
             for i in range(0, T, 370)]
    assert torch.equal(q, torch.cat(parts)) and torch.equal(*caches)
    k, v = ops.gather_kv_cache(caches[0], slots)
    nan = (k.isnan() | v.isnan()).any(-1).cpu()
    want = torch.zeros(T, Hkv, dtype=torch.bool)
    want[10, 0] = want[11, Hkv - 1] = True
    assert torch.equal(nan, want)
    assert float(v[12, 0, 64]) == 448 * 128


@pytest.mark.parametrize("device", DEVICES)
def test_blocks_move_whole(device):
    k, v = special_rows(32, 2, 64, torch.bfloat16)
    cache = new_cache(4, 2, 16, 64, device)
    ops.reshape_and_cache(k.to(device), v.to(device), cache, torch.arange(32, device=device))
    ops.copy_blocks([cache], [(0, 2), (1, 3)])
    at = torch.arange(32, device=device)
    for a, b in zip(ops.gather_kv_cache(cache, at), ops.gather_kv_cache(cache, at + 32)):
        assert torch.equal(a.nan_to_num(), b.nan_to_num())


# ----------------------------------------------------------------------------- attention

def batch(new, context, H, Hkv, D, block, dt, device, seed=0, spare=2, table_pad=1):
    """A pool of cached rows, block tables in any order, queries."""
    g = torch.Generator().manual_seed(seed)
    lens = [n + c for n, c in zip(new, context)]
    per = [-(-n // block) for n in lens]
    blocks = sum(per) + spare
    cache = new_cache(blocks, Hkv, block, D, "cpu")
    n = blocks * block
    size = torch.exp(0.5 * torch.randn(n, Hkv, 1, generator=g))
    k, v = torch.randn(n, Hkv, D, generator=g) * size, torch.randn(n, Hkv, D, generator=g) * size.flip(0)
    codes, scales = ra.kv8_views(cache)
    c, s = ra.kv8_rows(k, v)
    codes.view(torch.uint8).copy_(c.view(torch.uint8).view(blocks, block, 2, Hkv, D).permute(0, 2, 3, 1, 4))
    scales.copy_(s.view(blocks, block, 2, Hkv).permute(0, 2, 3, 1))
    order = torch.randperm(blocks, generator=g).int()
    table = torch.full((len(new), max(per + [0]) + table_pad), -1, dtype=torch.int32)
    at = 0
    for r, m in enumerate(per):
        table[r, :m] = order[at:at + m]
        at += m
    qsl = torch.tensor([0] + new).cumsum(0).int()
    q = (torch.randn(int(qsl[-1]), H, D, generator=g) * 1.5).to(dt)
    sinks = torch.randn(H, generator=g)
    move = lambda *x: [y.to(device) for y in x]  # noqa: E731
    return dict(zip(("q", "cache", "table", "lens", "qsl", "sinks"), move(q, cache, table, torch.tensor(lens, dtype=torch.int32), qsl, sinks)),
                new=new, context=context, scale=D ** -0.5, max_q=max(new), max_len=max(lens))


def oracle(b, window=0, sinks=None):
    """64-bit result ``[T, H, D]`` and how far a result may be off before its last rounding, from the cache as it is."""
    cache, q = b["cache"].cpu(), b["q"].cpu().double()
    nb, block, Hkv = cache.shape[0], cache.shape[3], cache.shape[2]
    codes, scales = ra.kv8_views(cache)
    T, H, D = q.shape
    out, lim = torch.zeros(T, H, D, dtype=torch.float64), torch.zeros(T, H, D, dtype=torch.float64)
    # weights: two e4m3 pieces (2^-8) for bf16, three or fp16 (2^-11) for fp16, fp32 otherwise
    eps_p = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -22}[b["q"].dtype]
    table, at = b["table"].cpu().long(), 0
    for r, (n, c) in enumerate(zip(b["new"], b["context"])):
        L = int(b["lens"][r])
        j = torch.arange(max(0, min(L, table.shape[1] * block)))
        blk = table[r, j // block]
        j, blk = j[(blk >= 0) & (blk < nb)], blk[(blk >= 0) & (blk < nb)]
        k, v = (codes[blk, w, :, j % block].double() * scales[blk, w, :, j % block].double()[..., None] for w in (0, 1))
        k, v = (x.repeat_interleave(H // Hkv, 1) for x in (k, v))
        qq = q[at:at + n]
        pos = torch.arange(L - n, L)[:, None]
        seen = j <= pos
        if window:
            seen &= j > pos - window
        s = torch.einsum("ihd,jhd->hij", qq, k) * b["scale"]
        mag = torch.einsum("ihd,jhd->hij", qq.abs(), k.abs()) * b["scale"]
        amax_q, sum_k = qq.abs().amax(-1).T[:, :, None], k.abs().sum(-1).T[:, None]
        # scores: fp32 sums of D products, and queries in e4m3 pieces whose last step is 2^-18 of the row's largest element
        off = (D + 8) * 2.0 ** -24 * mag + 2.0 ** -18 * amax_q * sum_k * b["scale"]
        s = torch.where(seen, s, -math.inf)
        if sinks is not None:
            s = torch.cat([s, sinks.cpu().double()[:, None, None].expand(-1, n, 1)], 2)
        p = torch.softmax(s, 2).nan_to_num() if not s.isnan().any() else torch.softmax(s, 2)
        p = torch.where(s.isneginf().all(2, keepdim=True), 0.0, p)[..., :len(j)]
        keep = seen.any(1)
        worst = torch.where(seen, off, 0.0).amax(2) if len(j) else torch.zeros(H, n, dtype=torch.float64)
        pv = torch.where(seen, p, 0.0)
        nan_rows = torch.einsum("hij,jhd->ihd", seen.double().expand_as(p), v.isnan().double()) > 0
        out[at:at + n] = torch.einsum("hij,jhd->ihd", pv.nan_to_num(), v.nan_to_num()).masked_fill(nan_rows, math.nan)
        mag_o = torch.einsum("hij,jhd->ihd", pv.nan_to_num(), v.nan_to_num().abs())
        lim[at:at + n] = mag_o * (eps_p + 2 * worst.T[..., None].nan_to_num() + 2.0 ** -17)
        # Weights far below a row's largest lose digits absolutely, too: exp(s - m) <= 1 for the largest is held in fp16, whose smallest step
        # is 2^-24 (off by 2^-25), or, times 2^3 and v's scale over the largest one, as e4m3 pieces of which the last of two counts 2^-5:
        # steps of 2^-9 / 2^5 / 2^3 = 2^-17 (off by 2^-18; three: 2^-23).  The sum of weights is 1 at least, so a result is off by no more
        # than that times the sum of what the weights multiply, codes times the largest scale.
        if b["q"].dtype != torch.float32 and len(j):
            unit = 2.0 ** (-18 if b["q"].dtype == torch.bfloat16 else -23)
            sc = scales[blk, 1, :, j % block].double().nan_to_num().amax(0).repeat_interleave(H // Hkv)
            cd = codes[blk, 1, :, j % block].double().nan_to_num().abs().repeat_interleave(H // Hkv, 1)
            lim[at:at + n] += unit * torch.einsum("ij,jhd->ihd", seen.double(), cd) * sc[:, None]
        out[at:at + n][~keep] = 0
        at += n
    return out, lim


def check(got, b, window=0, sinks=None):
    want, lim = oracle(b, window, sinks)
    got = got.cpu().double()
    assert torch.equal(got.isnan(), want.isnan())
    u = UNIT[b["q"].dtype]
    d = (got - want).nan_to_num().abs()
    worst = (d - lim - u * want.nan_to_num().abs() * 1.001 - (2.0 ** -25 if u == 2.0 ** -11 else 0)).max() if d.numel() else torch.tensor(0.0)
    assert worst <= 0, f"{float(worst)} over; largest difference {float(d.max())}"


def attend(b, window=0, sinks=None, **kw):
    return ops.paged_attention(b["q"], b["cache"], b["table"], b["lens"], b["qsl"], b["scale"], b["max_q"], b["max_len"],
                               window or None, sinks, **kw)


SHAPES = [(4, 1, 128, 64), (8, 2, 128, 16), (16, 1, 128, 32), (2, 2, 128, 128), (6, 2, 128, 48), (14, 2, 64, 16), (16, 2, 256, 64),
          (3, 1, 80, 12), (2, 1, 512, 64), (8, 8, 64, 64), (20, 1, 128, 64)]
LENGTHS = [([1], [0]), ([1, 1, 1], [0, 126, 127]), ([1, 1], [128, 700]), ([2, 1, 2], [5, 255, 1030]), ([1] * 9, [17 * i for i in range(9)]),
           ([7], [0]), ([130, 1, 64], [3, 40, 257]), ([300], [0]), ([129, 257], [1000, 64])]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("at", range(len(LENGTHS)))
def test_attention(device, dt, shape, at):
    if device == "cpu" and (dt != "bf16" or at % 3 or shape[2] > 256):
        pytest.skip("the oracle walks rows one at a time")
    H, Hkv, D, block = shape
    b = batch(*LENGTHS[at], H, Hkv, D, block, DT[dt], device, seed=at)
    window, sinks = ((0, 100)[at % 2], b["sinks"] if at % 3 == 1 else None)
    check(attend(b, window, sinks), b, window, sinks)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("D,block", [(128, 64), (128, 16), (64, 16), (256, 64), (96, 8)])
@pytest.mark.parametrize("new,context", [([1, 1, 2], [70, 130, 199]), ([40, 150], [30, 0])])
def test_what_a_row_does_not_see_does_not_reach_it(device, D, block, new, context):
    """NaN in later tokens, in rows behind a request's end and in blocks of nobody; a NaN that is seen gives NaN."""
    b = batch(new, context, 4, 2, D, block, torch.bfloat16, "cpu", seed=3)
    codes, scales = ra.kv8_views(b["cache"])
    used = torch.zeros(b["cache"].shape[0] * block, dtype=torch.bool)
    for r, n in enumerate(b["lens"].tolist()):
        j = torch.arange(n)
        used[b["table"][r].long()[j // block] * block + j % block] = True
    free = (~used).view(-1, block)
    blk, off = free.nonzero(as_tuple=True)
    codes.view(torch.uint8)[blk, :, :, off] = 0x7f                 # e4m3 NaN, as an unwritten pool may hold
    scales[blk, :, :, off] = math.nan
    clean = {**b, "cache": b["cache"].clone()}
    # the last token of the last request: seen by its own row only
    last = int(b["lens"][-1]) - 1
    s = int(b["table"][-1, last // block]) * block + last % block
    k = torch.randn(1, 2, D)
    v = torch.randn(1, 2, D)
    v[0, 1, D - 1] = math.nan
    ops.reshape_and_cache(k, v, b["cache"], torch.tensor([s]))
    for x in (clean, b):
        for name in ("q", "cache", "table", "lens", "qsl"):
            x[name] = x[name].to(device)
        check(attend(x), x)
    got = attend(b)
    assert got[-1, 2:].isnan().all() and got[:-1].isfinite().all() and got[-1, :2].isfinite().all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("D", [128, 64, 256])
def test_rows_that_see_nothing(device, D):
    """More queries than tokens, no tokens at all, blocks outside the pool, a table that is too short; a request without queries."""
    b = batch([3, 2, 1, 0, 20, 1], [4, 3, 90, 50, 80, 700], 4, 2, D, 64, torch.bfloat16, device, table_pad=0)
    b["lens"][0], b["lens"][1] = 1, 0              # queries at positions -2, -1, 0 and at -2, -1
    b["table"][2, 0] = b["cache"].shape[0]         # keys 0 .. 63 of the third request are not there
    b["table"][4, 1] = -5
    b["lens"][5] += 64                              # ... and its last block has no entry
    b["table"] = b["table"][:, :11].contiguous()
    out = torch.full_like(b["q"], 7.0)
    for sinks in (None, b["sinks"]):
        got = attend(b, 0, sinks, out=out if device == "cuda" else None)
        check(got, b, 0, sinks)
        assert (got[:2] == 0).all() and (got[3:5] == 0).all()


@gpu
@pytest.mark.parametrize("D,dt", [(128, "bf16"), (64, "fp16"), (256, "bf16"), (96, "bf16")])
def test_rows_of_no_request_stay(D, dt):
    """A padded batch: rows behind the last request, and in front of the first of a part of a batch."""
    for new in ([1, 2], [40, 3]):
        b = batch(new, [50, 3], 4, 2, D, 64, DT[dt], "cuda")
        T = b["q"].shape[0]
        q = torch.full((T + 9, 4, D), math.nan, dtype=DT[dt], device="cuda")
        q[4:4 + T] = b["q"]
        out = torch.full_like(q, 5.0)
        ops.paged_attention(q, b["cache"], b["table"], b["lens"], b["qsl"] + 4, b["scale"], b["max_q"], b["max_len"], out=out)
        check(out[4:4 + T], b)
        assert (out[:4] == 5).all() and (out[4 + T:] == 5).all()


@gpu
@pytest.mark.parametrize("D,new", [(128, 40), (128, 200), (64, 70), (64, 300), (256, 30)])
@pytest.mark.parametrize("window", [1, 5, 130, 700])
def test_windows_of_prompts(D, new, window):
    """Windows inside a tile, over several and beyond the start, with a context; both prompt kernels."""
    b = batch([new, 17, new + 1], [0, 600, 333], 4, 2, D, 32, torch.bfloat16, "cuda", seed=new)
    check(attend(b, window), b, window)


@gpu
@pytest.mark.parametrize("new", [1, 30, 300])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 + 5, 2 ** 40])
def test_windows_wider_than_any_length(new, window):
    b = batch([new, 2], [300, 7], 4, 2, 128, 64, torch.bfloat16, "cuda")
    assert torch.equal(attend(b, window), attend(b))


@gpu
@pytest.mark.parametrize("new", [1, 9])
def test_more_requests_than_a_launch_takes(new):
    """4100 requests are three launches of 2048 at most, each with items that are cut."""
    n = [new if i % 5 else 0 for i in range(4100)]
    n[2047] = n[2048] = new
    b = batch(n, [(17 * i) % 50 if i % 1000 else 900 for i in range(4100)], 2, 1, 64, 16, torch.bfloat16, "cuda")
    check(attend(b), b)


@gpu
def test_long_bounds_and_wide_tables():
    """Lengths far below what the call allows for: the scratch of a prompt is that of a few requests at a time."""
    b = batch([70, 1, 300, 90, 5], [600, 20, 0, 130, 64], 8, 4, 128, 64, torch.bfloat16, "cuda")
    want = attend(b)
    check(want, b)
    table = torch.full((5, 4000), -1, dtype=torch.int32, device="cuda")
    table[:, :b["table"].shape[1]] = b["table"]
    got = ops.paged_attention(b["q"], b["cache"], table, b["lens"], b["qsl"], b["scale"], b["max_q"], 250000)
    check(got, b)
    # the decode kernel cuts its line of tiles by the lengths, not by their bound
    b = batch([1, 1, 2], [600, 20, 4000], 4, 2, 128, 64, torch.bfloat16, "cuda")
    got = ops.paged_attention(b["q"], b["cache"], b["table"], b["lens"], b["qsl"], b["scale"], b["max_q"], 250000)
    check(got, b)


@gpu
@pytest.mark.parametrize("D", [64, 128, 256, 96])
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("new,context", [([1, 2, 1], [400, 37, 3]), ([50, 3], [30, 0]), ([300, 20], [100, 4])])
def test_queries_that_are_not_numbers(D, dt, new, context):
    """A NaN or an infinity in a query is its row's alone."""
    b = batch(new, context, 4, 2, D, 64, DT[dt], "cuda", seed=5)
    bad = torch.zeros(b["q"].shape[:2], dtype=torch.bool)
    bad[0, 1] = bad[2, 3] = bad[-1, 0] = True
    q = b["q"].clone()
    q[0, 1, 3], q[2, 3, D - 1], q[-1, 0, 0] = math.nan, math.inf, -math.inf
    got = attend({**b, "q": q}).cpu()
    assert got[bad].isnan().all()
    got[bad] = attend(b).cpu()[bad]
    check(got, b)


@gpu
@pytest.mark.parametrize("D,group", [(64, 2), (64, 5), (64, 8), (64, 16), (128, 4), (128, 8), (128, 13), (256, 3), (256, 8), (256, 16)])
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
def test_maxima_that_keep_moving(D, group, dt):
    """Keys that grow tile by tile: every tile rescales what the ones in front of it left, for all rows of a head at once."""
    lens = [900 + 61 * i for i in range(24)]
    b = batch([1] * 24, [n - 1 for n in lens], 2 * group, 2, D, 64, DT[dt], "cpu", seed=group)
    scales = ra.kv8_views(b["cache"])[1]
    for r, n in enumerate(lens):
        j = torch.arange(n)
        scales[b["table"][r].long()[j // 64], 0, :, j % 64] *= torch.exp2((j // 256).float())[:, None]
    for name in ("q", "cache", "table", "lens", "qsl"):
        b[name] = b[name].cuda()
    first = attend(b)
    check(first, b)
    for _ in range(20):
        assert torch.equal(attend(b), first)


@gpu
def test_items_around_the_cuts():
    """One to many tiles a request and every number of requests up to 40: cuts on, next to and far from the ends of items."""
    for n in (1, 2, 3, 7, 19, 40):
        b = batch([1 + (i % 2) for i in range(n)], [(389 * i) % 1900 for i in range(n)], 8, 2, 128, 64, torch.bfloat16, "cuda", seed=n)
        check(attend(b), b)
        assert torch.equal(attend(b), attend(b))


def test_refusals():
    b = batch([1, 1], [5, 9], 4, 2, 64, 16, torch.bfloat16, "cpu")
    for kw in (dict(bias=torch.zeros(4, 1)), dict(gate=torch.zeros(2, 4, dtype=torch.bfloat16)), dict(keep_first=4), dict(sigmoid=True)):
        with pytest.raises(ValueError):
            attend(b, **kw)
    with pytest.raises(ValueError):
        attend(b, -1)


@gpu
def test_refusals_on_the_gpu():
    b = batch([1, 1], [5, 9], 4, 2, 128, 64, torch.bfloat16, "cuda")
    k = torch.zeros(3, 2, 128, dtype=torch.bfloat16, device="cuda")
    slots = torch.arange(3, device="cuda")
    bad = [
        lambda: ops.reshape_and_cache(k, k[:2], b["cache"], slots),
        lambda: ops.reshape_and_cache(k, k, b["cache"], slots[:2]),
        lambda: ops.reshape_and_cache(k, k, b["cache"], slots.int()),
        lambda: ops.reshape_and_cache(k[:, :1], k[:, :1], b["cache"], slots),
        lambda: ops.reshape_and_cache(k, k, b["cache"].cpu(), slots),
        lambda: ops.reshape_and_cache(k.transpose(1, 2), k.transpose(1, 2), b["cache"], slots),
        lambda: ops.reshape_and_cache(k[..., :40], k[..., :40], new_cache(2, 2, 16, 40, "cuda"), slots),
        lambda: ops.gather_kv_cache(b["cache"], slots.cpu()),
        lambda: attend({**b, "q": b["q"][..., :64]}),
        lambda: attend({**b, "q": b["q"].transpose(1, 2)}),
        lambda: attend({**b, "lens": b["lens"].long()}),
        lambda: attend({**b, "qsl": b["qsl"][:2]}),
        lambda: attend({**b, "table": b["table"][:1]}),
        lambda: attend({**b, "q": b["q"].cpu()}),
        lambda: attend({**b, "cache": b["cache"][:, :, :1]}),
        lambda: attend(b, 0, torch.zeros(3, device="cuda")),
        lambda: attend(b, out=torch.empty_like(b["q"]).float()),
    ]
    for i, f in enumerate(bad):
        with pytest.raises((RuntimeError, ValueError)):
            f()
            pytest.fail(f"call {i} was taken")
    torch.cuda.synchronize()


@gpu
@pytest.mark.parametrize("D", [128, 256])
def test_streams_graphs_and_two_calls_at_once(D):
    """The same bits from another stream, from a captured and replayed call with other contents, and from two calls that overlap."""
    b1 = batch([1, 2, 1], [4000, 9, 700], 8, 2, D, 64, torch.bfloat16, "cuda", seed=1)
    b2 = batch([200, 31], [300, 1], 8, 2, D, 64, torch.bfloat16, "cuda", seed=2)
    want = [attend(b) for b in (b1, b2)]
    check(want[0], b1)
    check(want[1], b2)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for s in (s1, s2):
        s.wait_stream(torch.cuda.current_stream())
    got = {}
    for i in range(20):
        for s in (s1, s2):
            with torch.cuda.stream(s):
                got[s, i] = [attend(b) for b in (b1, b2)]
    torch.cuda.synchronize()
    for pair in got.values():
        assert all(torch.equal(a, w) for a, w in zip(pair, want))
    for b, w in zip((b1, b2), want):
        q = torch.zeros_like(b["q"])
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = attend({**b, "q": q})
        q.copy_(b["q"])
        for _ in range(3):
            out.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, w)


@gpu
def test_write_then_attend_in_one_go():
    """Prompt, then decode steps: the fused write feeds the attention that reads it, in a mixed batch as the engine issues it."""
    H, Hkv, D, block, dt = 8, 2, 128, 64, torch.bfloat16
    g = torch.Generator().manual_seed(0)
    n0, steps, blocks = 150, 4, 8
    cos_sin = torch.cat([torch.ones(400, 64), torch.zeros(400, 64)], -1).cuda()
    rows = (torch.randn(2 * (n0 + steps), (H + 2 * Hkv) * D, generator=g)).to(dt).cuda()
    cache = new_cache(blocks, Hkv, block, D, "cuda")
    table = torch.tensor([[5, 2, 7], [0, 3, 1]], dtype=torch.int32, device="cuda")
    ref = []
    for r in range(2):
        x = rows[r * (n0 + steps):(r + 1) * (n0 + steps)].view(-1, H + 2 * Hkv, D).float().cpu()
        c, s = ra.kv8_rows(x[:, H:H + Hkv], x[:, H + Hkv:])
        kv = c.double() * s.double()[..., None]
        k, v = (kv[:, w].repeat_interleave(H // Hkv, 1) for w in (0, 1))
        sc = torch.einsum("ihd,jhd->hij", x[:, :H].double(), k) * D ** -0.5
        sc = sc.masked_fill(torch.ones(sc.shape[1:]).triu(1).bool(), -math.inf)
        ref.append(torch.einsum("hij,jhd->ihd", torch.softmax(sc, 2), v))
    done = [0, 0]

    def step(counts, decodes):
        pos = torch.cat([torch.arange(d, d + n) for d, n in zip(done, counts)]).cuda()
        x = torch.cat([rows[r * (n0 + steps) + done[r]:r * (n0 + steps) + done[r] + n] for r, n in enumerate(counts)])
        req = torch.cat([torch.full((n,), r) for r, n in enumerate(counts)]).cuda()
        slots = table[req, pos // block].long() * block + pos % block
        q = ops.qkv_split_norm_rope_cache(x, pos, cos_sin, None, None, 1e-6, H, Hkv, D, True, cache, slots)
        lens = torch.tensor([d + n for d, n in zip(done, counts)], dtype=torch.int32, device="cuda")
        qsl = torch.tensor([0, counts[0], sum(counts)], dtype=torch.int32, device="cuda")
        o = ops.paged_attention(q.view(-1, H, D), cache, table, lens, qsl, D ** -0.5, max(counts), int(lens.max()),
                                num_decodes=decodes, decode_query_len=1, num_decode_tokens=decodes, stable_metadata=True)
        want = torch.cat([ref[r][done[r]:done[r] + n] for r, n in enumerate(counts)])
        off = (o.cpu().double() - want).abs()
        assert (off <= 2.0 ** -8 * want.abs() + 2.0 ** -7 * want.abs().mean() + 2.0 ** -8).all(), float(off.max())
        for r, n in enumerate(counts):
            done[r] += n
    step([1, n0], 1)          # one token of the first request beside the second one's prompt
    step([n0 - 1, 2], 0)
    for _ in range(2):
        step([1, 1], 2)


# ----------------------------------------------------------------------------- the engine

@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("head_dim,heads", [(128, 4), (64, 4), (32, 4)])
def test_engine_generates_from_an_8_bit_cache(device, head_dim, heads):
    """``kv_cache_dtype="fp8_e4m3"``: pages are uint8; chunks, decode steps and prefix reuse run."""
    from vllm_kunlun_b200 import LLM, SamplingParams
    from vllm_kunlun_b200.config import ModelConfig
    cfg = dict(architecture="Qwen3ForCausalLM", name="tiny", vocab_size=512, hidden_size=256, num_layers=2, num_heads=heads,
               num_kv_heads=2, head_dim=head_dim, intermediate_size=256, rms_norm_eps=1e-6, rope_theta=1e6, qk_norm=True, max_position=512)
    prompts = [[(7 * i + j) % 500 for i in range(n)] for j, n in enumerate((70, 3, 33))]
    outs = {}
    for kvd in ("auto", "fp8_e4m3"):
        llm = LLM(ModelConfig(**cfg), device=device, block_size=16, max_model_len=256, max_num_seqs=4, max_num_batched_tokens=64,
                  num_gpu_blocks=64, seed=3, kv_cache_dtype=kvd, enable_prefix_caching=True)
        cache = llm.engine.runner.kv_caches[0]
        assert (cache.dtype == torch.uint8 and cache.shape[-1] == head_dim + 4) == (kvd != "auto")
        sp = SamplingParams(max_tokens=6, temperature=0.0, ignore_eos=True)
        outs[kvd] = [list(o.token_ids) for o in llm.generate(prompts, sp)]
        assert all(len(o.token_ids) == 6 for o in llm.generate(prompts, sp))      # again, from reused prefixes
    assert all(len(x) == 6 for x in outs["fp8_e4m3"])


def test_models_that_keep_other_caches_refuse():
    from vllm_kunlun_b200 import LLM
    from vllm_kunlun_b200.config import PRESETS
    import dataclasses
    mla = next(p() for n, p in PRESETS.items() if p().use_mla)
    small = dataclasses.replace(mla, num_layers=1, vocab_size=64, hidden_size=64, intermediate_size=64, num_experts=2,
                                num_experts_per_tok=1, moe_intermediate_size=64, quantization=None, num_heads=2, num_kv_heads=2,
                                q_lora_rank=64, max_position=64, n_group=1, topk_group=1, first_dense_layers=1)
    with pytest.raises(ValueError):
        LLM(small, device="cpu", kv_cache_dtype="fp8_e4m3", num_gpu_blocks=4, max_model_len=32)
