"""CUDA attention over the 8-bit paged cache (``csrc/attention/kv8_*.cu``).

A batch is decode-first, as in :func:`ops.paged_attention`: requests with few query rows per key / value head go to the decode
kernel, the others to the prompt kernel; what neither takes (fp32 models, other head or block sizes) to the generic one.
"""
from __future__ import annotations

import torch

from . import _ext


def paged_attention_kv8(out, q, kv_cache, block_tables, seq_lens, query_start_loc, scale: float, max_query_len: int,
                        max_seq_len: int, window: int, sinks, workspace, num_decodes: int, decode_query_len: int,
                        num_decode_tokens: int, stable_metadata: bool):
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    _ext.C().kv8_attention_generic(out, q, kv_cache, block_tables, seq_lens, query_start_loc, sinks, window, scale)
    return out
