"""Keys and values kept in 8 bits: writing them into the paged cache, reading them back, and the attention that reads them in place.

The cache is ``uint8 [blocks, 2, kv_heads, block_size, D + 4]``: of every block, K or V and head first ``block_size`` rows of D e4m3
codes, then ``block_size`` fp32 scales.  A row x (one token's key or value of one head) is held as

    scale = 2^e,  e the smallest of -15 .. 7 with max |x| <= 448 * 2^e  (7 if there is none),    code = e4m3(x / scale), saturating

so that what a row stands for, code * scale, is an exact number in fp16 and in bf16.  Attention of the query at position p of a
request over its keys j with p - window < j <= p:

    s_j = scale * q . k_j,    out = sum_j exp(s_j) v_j / (exp(sink) + sum_j exp(s_j))        (no window: all j <= p; no sink: no such term)

``listed()``: the fixed cases; ``draw(rng)``: one more of the same ranges; ``prepare(case, seed)``: what a serving process has in hand
before the call; ``run(state)``: one pass, in plain torch operations or, with ``own``, through the framework's op layer;
``work(case)``: the bytes and operations that a pass cannot do without; ``exact(case, seed)``: the same in 64 bits.
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-6
ROPE_THETA = 1e6

# heads, key / value heads, head size: Llama-3.1-8B and Qwen3-8B, Qwen3-30B-A3B, the "small" layer-benchmark size, a 64-wide head
# layout with sinks and a window, the full-attention layers of Qwen3-Next
HEADS = [(32, 8, 128), (32, 4, 128), (16, 4, 128), (64, 8, 64), (16, 2, 256)]


# ----------------------------------------------------------------------------- the cases

def listed():
    return [
        # Projections of 16 decoding requests (one token each): rotation, and keys and values into the cache.
        dict(name="write_decode_16", kind="write", heads=32, kv_heads=8, dim=128, tokens=16, norm=False, block=64, dtype="bf16"),
        # The same of a prompt step at the batch limit of the scheduler, with normed queries and keys.
        dict(name="write_prompt_8192", kind="write", heads=32, kv_heads=4, dim=128, tokens=8192, norm=True, block=64, dtype="bf16"),
        # Keys and values that were rotated elsewhere (positions with several axes), in fp16, an odd number of tokens.
        dict(name="put_2179", kind="put", heads=32, kv_heads=8, dim=128, tokens=2179, block=16, dtype="fp16"),
        # Reading a cached prefix back: a short one, where latency counts, and a long one.
        dict(name="read_back_131", kind="read", heads=16, kv_heads=4, dim=128, tokens=131, block=16, dtype="fp16"),
        dict(name="read_back_16384", kind="read", heads=32, kv_heads=8, dim=128, tokens=16384, block=64, dtype="bf16"),
        # One interactive request with a short history: the smallest attention call.
        dict(name="decode_1x900", kind="attn", heads=32, kv_heads=8, dim=128, requests=1, new=1, context=899, ragged=False,
             window=0, sinks=False, block=16, dtype="bf16"),
        # A decode step of the serving benchmark's batch, 4096 tokens each.
        dict(name="decode_16x4096", kind="attn", heads=32, kv_heads=8, dim=128, requests=16, new=1, context=4095, ragged=False,
             window=0, sinks=False, block=64, dtype="bf16"),
        # Many requests of uneven lengths, as a running server has them.
        dict(name="decode_ragged_48", kind="attn", heads=32, kv_heads=4, dim=128, requests=48, new=1, context=8191, ragged=True,
             window=0, sinks=False, block=64, dtype="bf16"),
        # Verification of one drafted token per request, heads of 64 with sinks, fp16.
        dict(name="verify_12x2", kind="attn", heads=64, kv_heads=8, dim=64, requests=12, new=2, context=2500, ragged=True,
             window=0, sinks=True, block=16, dtype="fp16"),
        # Prompts of the headline benchmark: four of 2048 tokens in one step.
        dict(name="prompt_4x2048", kind="attn", heads=32, kv_heads=8, dim=128, requests=4, new=2048, context=0, ragged=False,
             window=0, sinks=False, block=64, dtype="bf16"),
        # Short prompts of uneven lengths behind a cached prefix.
        dict(name="prompt_ragged_11", kind="attn", heads=32, kv_heads=8, dim=128, requests=11, new=371, context=200, ragged=True,
             window=0, sinks=False, block=16, dtype="bf16"),
        # A chunk of a long prompt: 4096 new tokens behind 28672.
        dict(name="chunk_4096_of_32768", kind="attn", heads=32, kv_heads=4, dim=128, requests=1, new=4096, context=28672,
             ragged=False, window=0, sinks=False, block=64, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["write", "put", "read", "decode", "decode", "verify", "prompt", "chunk"])
    heads, kv, dim = rng.choice(HEADS[:3] + HEADS)
    c = dict(kind="attn", heads=heads, kv_heads=kv, dim=dim, block=rng.choice([16, 32, 64, 64]), dtype=rng.choice(["bf16", "bf16", "fp16"]))
    if kind in ("write", "put", "read"):
        c.update(kind=kind, tokens=_log(rng, 1, 8192 if kind == "write" else 16384))
        return dict(c, norm=rng.random() < 0.5) if kind == "write" else c
    c.update(ragged=rng.random() < 0.6, window=rng.choice([0, 0, 0, 128, 1024]), sinks=rng.random() < 0.3)
    if kind == "decode":
        requests = _log(rng, 1, 64)
        return dict(c, requests=requests, new=1, context=_log(rng, 1, min(32767, 262144 // requests)))
    if kind == "verify":
        requests = _log(rng, 1, 32)
        return dict(c, requests=requests, new=2, context=_log(rng, 1, 131072 // requests))
    if kind == "prompt":
        requests = _log(rng, 1, 12)
        return dict(c, requests=requests, new=_log(rng, 17, 4096 // requests), context=0)
    requests = _log(rng, 1, 4)
    return dict(c, requests=requests, new=_log(rng, 17, 2048 // requests), context=_log(rng, 16, 24576 // requests))


# ----------------------------------------------------------------------------- inputs

def _lengths(case):
    """New tokens and earlier tokens of every request; ragged: between a third of the given size and all of it."""
    n, c, R = case["new"], case["context"], case["requests"]
    if not case["ragged"]:
        return [n] * R, [c] * R
    share = [(1 + (5 * i + 3) % 7 / 3) / 3 for i in range(R)]
    return [max(1, round(n * s)) if n > 2 else n for s in share], [round(c * s) for s in share]


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _cache(g, blocks, kv_heads, block, dim):
    """A pool that earlier tokens have filled: keys with a few strong channels, tokens of differing size."""
    x = _randn(g, blocks, 2, kv_heads, block, dim)
    x[:, 0] *= torch.exp(0.6 * _randn(g, kv_heads, 1, dim))
    x *= torch.exp(0.4 * _randn(g, blocks, 2, kv_heads, block, 1))
    scale = _scale(x)
    cache = torch.empty(blocks, 2, kv_heads, block * (dim + 4), dtype=torch.uint8, device=DEV)
    cache[..., :block * dim] = _codes(x, scale).view(torch.uint8).flatten(-2)
    cache[..., block * dim:] = scale.view(torch.uint8).flatten(-2)
    return cache.view(blocks, 2, kv_heads, block, dim + 4)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    kind, H, Hkv, D, block, dt = case["kind"], case["heads"], case["kv_heads"], case["dim"], case["block"], DTYPES[case["dtype"]]
    s = dict(case=case)
    if kind != "attn":
        # requests write wherever the block table has put them: whole blocks in any order
        T = case["tokens"]
        blocks = -(-T // block) + 3
        s["cache"] = _cache(g, blocks, Hkv, block, D)
        start = seed % block
        at = torch.arange(start, start + T, device=DEV)
        s["slots"] = torch.randperm(blocks, generator=g, device=DEV)[at // block] * block + at % block
        if kind == "put":
            s["k"], s["v"] = ((_randn(g, T, Hkv, D) * torch.exp(0.5 * _randn(g, T, Hkv, 1))).to(dt) for _ in range(2))
        if kind == "write":
            rot = 64 if D == 256 else D
            s["qkv"] = (_randn(g, T, (H + 2 * Hkv) * D) * 1.5).to(dt)
            s["positions"] = torch.randint(0, 8192, (T,), generator=g, device=DEV)
            inv = ROPE_THETA ** (-torch.arange(0, rot, 2, device=DEV, dtype=torch.float64) / rot)
            angle = torch.arange(8192, device=DEV, dtype=torch.float64)[:, None] * inv
            s["cos_sin"] = torch.cat([angle.cos(), angle.sin()], -1).float().contiguous()
            s["gemma"] = D == 256
            w = 0.0 if s["gemma"] else 1.0
            s["q_w"], s["k_w"] = ((w + 0.1 * _randn(g, D)).to(dt) if case["norm"] else None for _ in range(2))
        return s
    new, context = _lengths(case)
    lens = [n + c for n, c in zip(new, context)]
    per = [-(-n // block) for n in lens]
    blocks = sum(per) + 2
    s["cache"] = _cache(g, blocks, Hkv, block, D)
    order = torch.randperm(blocks, generator=g, device=DEV).int()
    table = torch.zeros(len(lens), max(per), dtype=torch.int32)
    starts = [0]
    for n in per:
        starts.append(starts[-1] + n)
    order = order.cpu()
    for r, n in enumerate(per):
        table[r, :n] = order[starts[r]:starts[r] + n]
    s["table"] = table.to(DEV)
    s["seq_lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
    qsl = [0]
    for n in new:
        qsl.append(qsl[-1] + n)
    s["qsl"] = torch.tensor(qsl, dtype=torch.int32, device=DEV)
    s["q"] = (_randn(g, qsl[-1], H, D) * 1.5).to(dt)
    s["sinks"] = _randn(g, H) if case["sinks"] else None
    s.update(max_new=max(new), max_len=max(lens), scale=D ** -0.5)
    return s


# ----------------------------------------------------------------------------- plain form

def _scale(x):
    """Power of two per row ``[..., 1]``, fp32."""
    m, e = torch.frexp(x.abs().amax(-1, keepdim=True).clamp(2.0 ** -24, 448.0 * 128) / 448.0)
    return torch.ldexp(torch.ones_like(m), (e - (m == 0.5).int()).clamp(-15, 7))


def _codes(x, scale):
    return (x / scale).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)


def _parts(cache, D):
    """Codes ``[blocks, 2, heads, block * D]`` in e4m3 and scales ``[blocks, 2, heads, block]`` as views; a power of two in fp32 is
    the bf16 number in its upper half."""
    pages = cache.flatten(-2)
    n = cache.shape[3] * D
    return pages[..., :n].view(torch.float8_e4m3fn), pages[..., n:].view(torch.bfloat16)[..., 1::2]


def _put(cache, k, v, slots):
    """Plain write of fp32 rows ``[T, heads, D]``."""
    D, block = k.shape[-1], cache.shape[3]
    pages = cache.flatten(-2)
    codes = pages[..., :block * D].unflatten(-1, (block, D))
    scales = pages[..., block * D:].unflatten(-1, (block, 4))
    x = torch.stack([k, v], 1)
    s = _scale(x)
    b, o = slots // block, slots % block
    codes[b, :, :, o] = _codes(x, s).view(torch.uint8)
    scales[b, :, :, o] = s.view(torch.uint8)


def _values(cache, D, b, o, dtype=torch.float32):
    """Rows at blocks ``b`` and offsets ``o``: ``[..., 2, heads, D]``."""
    block = cache.shape[3]
    pages = cache.flatten(-2)
    codes = pages[..., :block * D].unflatten(-1, (block, D))[b, :, :, o]
    scales = pages[..., block * D:].unflatten(-1, (block, 4))[b, :, :, o].contiguous()
    return codes.view(torch.float8_e4m3fn).to(dtype) * scales.view(torch.float32).to(dtype)


def _rotated(x, cs, rot):
    c, sn = cs[:, None, :rot // 2], cs[:, None, rot // 2:]
    a, b = x[..., :rot // 2], x[..., rot // 2:rot]
    return torch.cat([a * c - b * sn, b * c + a * sn, x[..., rot:]], -1)


def _split_rotated(s, dtype):
    """Rotated queries and keys and the values of a fused projection row, in ``dtype``."""
    case = s["case"]
    H, Hkv, D = case["heads"], case["kv_heads"], case["dim"]
    q, k, v = s["qkv"].to(dtype).unflatten(-1, (H + 2 * Hkv, D)).split([H, Hkv, Hkv], 1)
    if s["q_w"] is not None:
        one = 1.0 if s["gemma"] else 0.0
        q, k = (x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * (w.to(dtype) + one) for x, w in ((q, s["q_w"]), (k, s["k_w"])))
    cs = s["cos_sin"].to(dtype)[s["positions"]]
    return _rotated(q, cs, cs.shape[-1]), _rotated(k, cs, cs.shape[-1]), v


@torch.inference_mode()
def run(s):
    case = s["case"]
    kind, H, Hkv, D, dt = case["kind"], case["heads"], case["kv_heads"], case["dim"], DTYPES[case["dtype"]]
    if own:
        from vllm_kunlun_b200 import ops
        if kind == "write":
            q = ops.qkv_split_norm_rope_cache(s["qkv"], s["positions"], s["cos_sin"], s["q_w"], s["k_w"], EPS, H, Hkv, D, True,
                                              s["cache"], s["slots"], s["gemma"])
            return q, *_parts(s["cache"], D)
        if kind == "put":
            ops.reshape_and_cache(s["k"], s["v"], s["cache"], s["slots"])
            return _parts(s["cache"], D)
        if kind == "read":
            return ops.gather_kv_cache(s["cache"], s["slots"], dt)
        return ops.paged_attention(s["q"], s["cache"], s["table"], s["seq_lens"], s["qsl"], s["scale"], s["max_new"],
                                   s["max_len"], case["window"] or None, s["sinks"])
    if kind == "write":
        q, k, v = _split_rotated(s, torch.float32)
        _put(s["cache"], k, v, s["slots"])
        return q.flatten(1).to(dt), *_parts(s["cache"], D)
    if kind == "put":
        _put(s["cache"], s["k"].float(), s["v"].float(), s["slots"])
        return _parts(s["cache"], D)
    block = case["block"]
    if kind == "read":
        kv = _values(s["cache"], D, s["slots"] // block, s["slots"] % block).to(dt)
        return kv[:, 0].contiguous(), kv[:, 1].contiguous()
    # attention: requests padded to the longest, everything in one batch of products
    lens, qsl = s["seq_lens"].long(), s["qsl"].long()
    B, Q, L = len(lens), s["max_new"], s["max_len"]
    j = torch.arange(L, device=DEV)
    kv = _values(s["cache"], D, s["table"].long()[:, j // block], (j % block).expand(B, L))      # [B, L, 2, Hkv, D]
    k, v = kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2)                                # [B, Hkv, L, D]
    n = qsl[1:] - qsl[:-1]
    i = torch.arange(Q, device=DEV)
    there = i < n[:, None]
    rows = torch.where(there, qsl[:-1, None] + i, 0)
    q = s["q"].float()[rows].transpose(1, 2).unflatten(1, (Hkv, H // Hkv)).flatten(2, 3)           # [B, Hkv, g * Q, D]
    p = (q * s["scale"]) @ k.transpose(-1, -2)
    pos = (lens - n)[:, None] + i                                                                  # [B, Q]
    hidden = j > pos[..., None]
    if case["window"]:
        hidden |= j <= pos[..., None] - case["window"]
    p = p.unflatten(2, (H // Hkv, Q)).masked_fill_(hidden[:, None, None], -math.inf)              # [B, Hkv, g, Q, L]
    top = p.amax(-1, keepdim=True)
    if s["sinks"] is not None:
        sink = s["sinks"].view(Hkv, H // Hkv, 1, 1)
        top = torch.maximum(top, sink)
    p = p.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    if s["sinks"] is not None:
        total = total + torch.exp(sink - top)
    o = (p.flatten(2, 3) @ v).unflatten(2, (H // Hkv, Q)) / total
    return o.flatten(1, 2).transpose(1, 2)[there].to(dt)


# ----------------------------------------------------------------------------- what a pass cannot do without

def work(case):
    kind, H, Hkv, D = case["kind"], case["heads"], case["kv_heads"], case["dim"]
    row = 2 * Hkv * (D + 4)                   # one token's keys and values in the cache
    if kind == "write":
        T = case["tokens"]
        rot = 64 if D == 256 else D
        return dict(bytes=T * (2 * (H + 2 * Hkv) * D + 2 * H * D + row + 16) + min(T, 8192) * 4 * rot,
                    flops=T * (H + Hkv) * (3 * rot + 4 * D * case["norm"]) + 4 * T * Hkv * D)
    if kind in ("put", "read"):
        return dict(bytes=case["tokens"] * (row + 4 * Hkv * D + 8), flops=case["tokens"] * 4 * Hkv * D)
    w = case["window"]
    pairs = keys = 0
    for n, c in zip(*_lengths(case)):
        if w:
            full = max(0, min(n, w - c))       # rows that see everything in front of them
            pairs += full * c + full * (full + 1) // 2 + (n - full) * w
            keys += min(c + n, w + n - 1)
        else:
            pairs += n * c + n * (n + 1) // 2
            keys += c + n
    return dict(bytes=4 * sum(_lengths(case)[0]) * H * D + keys * row, flops=4 * H * D * pairs)


# ----------------------------------------------------------------------------- 64 bits

@torch.inference_mode()
def exact(case, seed):
    """A cache's codes are compared with what they stand for before rounding; its scales are powers of two, which have no such value."""
    s = prepare(case, seed)
    kind, H, Hkv, D, block = case["kind"], case["heads"], case["kv_heads"], case["dim"], case["block"]
    f64 = torch.float64
    raw = s["cache"].reshape(-1, block * (D + 4))                        # a page of one head a row
    codes = raw[:, :block * D].contiguous().view(torch.float8_e4m3fn).to(f64).view(-1, block, D)
    scales = raw[:, block * D:].contiguous().view(torch.float32).to(f64).view(-1, block, 1)

    def rows(slots, which):
        """Page and row of every (slot, head)."""
        page = ((slots // block)[:, None] * 2 + which) * Hkv + torch.arange(Hkv, device=DEV)
        return page, (slots % block)[:, None].expand_as(page)

    if kind in ("write", "put"):
        if kind == "put":
            k, v, q = s["k"].to(f64), s["v"].to(f64), None
        else:
            x = s["qkv"].to(f64).view(-1, H + 2 * Hkv, D)
            q, k, v = x[:, :H], x[:, H:H + Hkv], x[:, H + Hkv:]
            if case["norm"]:
                def normed(y, w):
                    return y / (y.pow(2).sum(-1, keepdim=True) / D + EPS).sqrt() * (w.to(f64) + (1.0 if s["gemma"] else 0.0))
                q, k = normed(q, s["q_w"]), normed(k, s["k_w"])
            table = s["cos_sin"].to(f64)[s["positions"]]
            half = table.shape[1] // 2
            z = torch.complex(table[:, :half], table[:, half:])[:, None]

            def turned(y):
                t = torch.complex(y[..., :half], y[..., half:2 * half]) * z
                return torch.cat([t.real, t.imag, y[..., 2 * half:]], -1)
            q, k = turned(q), turned(k)
            q = q.reshape(-1, H * D)
        for which, y in ((0, k), (1, v)):
            e = torch.ceil(torch.log2(y.abs().amax(-1, keepdim=True) / 448)).clamp(-15, 7)
            codes[rows(s["slots"], which)] = (y / torch.exp2(e)).clamp(-448, 448)
        out = codes.view(-1, 2, Hkv, block * D)
        return [out, None] if kind == "put" else [q, out, None]
    if kind == "read":
        return [codes[rows(s["slots"], w)] * scales[rows(s["slots"], w)] for w in (0, 1)]
    g, outs, at = H // Hkv, [], 0
    for r, (n, c) in enumerate(zip(*_lengths(case))):
        keys = torch.arange(c + n, device=DEV)
        slots = s["table"][r].long()[keys // block] * block + keys % block
        k, v = (codes[rows(slots, w)] * scales[rows(slots, w)] for w in (0, 1))         # [L, Hkv, D]
        out = torch.empty(n, H, D, dtype=f64, device=DEV)
        step = max(1, 2 ** 28 // (c + n))
        for h in range(H):
            for a in range(0, n, step):
                b = min(n, a + step)
                w = torch.softmax(torch.cat([
                    (s["q"][at + a:at + b, h].to(f64) @ k[:, h // g].T * s["scale"]).masked_fill(
                        _unseen(c + a, b - a, keys, case["window"]), -math.inf),
                    (torch.full((b - a, 1), -math.inf, dtype=f64, device=DEV) if s["sinks"] is None
                     else s["sinks"][h].to(f64).expand(b - a, 1))], 1), 1)
                out[a:b, h] = w[:, :-1] @ v[:, h // g]
        outs.append(out)
        at += n
    return torch.cat(outs)


def _unseen(first, n, keys, window):
    pos = torch.arange(first, first + n, device=DEV)[:, None]
    return (keys > pos) | (keys <= pos - window) if window else keys > pos
