"""CUDA attention over the 8-bit paged cache (``csrc/attention/kv8_*.cu``).

A batch is decode-first, as in :func:`ops.paged_attention`: requests with few query rows per key / value head go to the decode
kernel, the others to the prompt kernels; what neither takes (fp32 models, other head or block sizes) to the generic one.
"""
from __future__ import annotations

import os

import torch

from . import _ext

# B200_KV8_UMMA=0 keeps every call on the generic kernel
TENSOR_CORES = [os.environ.get("B200_KV8_UMMA", "1") != "0"]
DECODE_ROWS = 16                # query rows (heads of a group x query tokens) that the decode kernel takes
# Bytes of keys and values that a prompt call widens at a time: all requests, some of them, or some heads of one (one head at least)
SCRATCH = 1 << 30


def paged_attention_kv8(out, q, kv_cache, block_tables, seq_lens, query_start_loc, scale: float, max_query_len: int,
                        max_seq_len: int, window: int, sinks, workspace, num_decodes: int, decode_query_len: int,
                        num_decode_tokens: int, stable_metadata: bool):
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    n = num_decodes
    if 0 < n < seq_lens.shape[0]:       # start offsets are absolute: both parts work on the whole q and out
        _attend(out, q, kv_cache, block_tables[:n], seq_lens[:n], query_start_loc[:n + 1], scale, decode_query_len, max_seq_len,
                window, sinks, workspace, stable_metadata)
        _attend(out, q, kv_cache, block_tables[n:], seq_lens[n:], query_start_loc[n:], scale, max_query_len, max_seq_len, window,
                sinks, workspace, False)
    else:
        _attend(out, q, kv_cache, block_tables, seq_lens, query_start_loc, scale, max_query_len, max_seq_len, window, sinks,
                workspace, stable_metadata)
    return out


def _attend(out, q, kv_cache, block_tables, seq_lens, query_start_loc, scale, max_query_len, max_seq_len, window, sinks, workspace,
            stable_metadata):
    D, group = q.shape[2], q.shape[1] // kv_cache.shape[2]
    if TENSOR_CORES[0] and kv_cache.shape[3] % 16 == 0 and q.dtype != torch.float32 and q.stride(0) % 8 == 0 and q.data_ptr() % 16 == 0:
        if max_query_len * group <= DECODE_ROWS and D in (64, 128, 256):
            ws = (workspace.o, workspace.lse, workspace.tickets) if workspace is not None else (None, None, None)
            _ext.C().kv8_decode(out, q, kv_cache, block_tables, seq_lens, query_start_loc, sinks, *ws, max_query_len, max_seq_len,
                                window, scale, stable_metadata)
            return
        if D in (64, 128, 256) and group <= 128 and scale > 0:
            # widened once for all query tiles where more than one pair of them (128 // group tokens each) reads the same keys.
            # us widened inside and first, one request behind 16000 tokens, by tiles: 32 / 8 heads of 128: one 44 / 58, two 57 / 65, three
            # 74 / 76, four 100 / 92, six 127 / 110, ten 328 / 235; 64 / 8 heads of 64: 36 / 41, 48 / 44, 61 / 53, 80 / 66, 102 / 79, 269 / 188.
            # 40 requests behind 1000: 96 / 120, 117 / 138, 176 / 176, 188 / 188, 270 / 245, 451 / 382; heads of 64: 67 / 68, 95 / 90,
            # 143 / 119, 160 / 129, 227 / 169, 364 / 258.  Heads of 256 have no kernel that widens inside.
            wide = D == 256 or max_query_len > 2 * (128 // group)
            _ext.C().kv8_prompt(out, q, kv_cache, block_tables, seq_lens, query_start_loc, sinks, max_query_len, max_seq_len, window,
                                scale, wide, SCRATCH)
            return
    _ext.C().kv8_attention_generic(out, q, kv_cache, block_tables, seq_lens, query_start_loc, sinks, window, scale)
