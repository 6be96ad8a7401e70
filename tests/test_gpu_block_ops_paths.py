"""GPU numerics of the encoder-block operators on paths that sizes select: both kernels of masked
attention, their splits and lookups of documents, and rows that a CTA of the norm walks over.

Each attention test checks which kernel its sizes take and how many splits, so that it keeps
testing what it was written for.  References and bounds: those of ``test_gpu_block_ops``.
"""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

from test_gpu_block_ops import _assert_close, _i32, _of_heads, _random_qkv, _reference, _starts

pytestmark = pytest.mark.gpu

TILES, ROWS = 1, 0


def _plan(q_rows, kv_rows, documents, heads, kv_heads, d, causal=False, batch=None):
    """(kernel, splits) of a call; ``batch``: (rows, keys) of each item."""
    from musc_b200 import _lib
    at = 1 << 20  # looked at for being null only
    q_len, kv_len = batch or (0, 0)
    args = _lib.MaskedAttentionArgs(dtype=_lib.F16, heads=heads, kv_heads=kv_heads, head_dim=d, q_rows=q_rows, kv_rows=kv_rows,
                                    documents=documents, causal=causal, q_offsets=None if batch else at,
                                    kv_offsets=None if batch else at, q_len=q_len, kv_len=kv_len, kv_pitch=kv_len, scale=1.0)
    kernel, splits = ctypes.c_int(), ctypes.c_int()
    _lib.check(_lib.lib().musc_b200_masked_attention_plan(ctypes.byref(args), ctypes.byref(kernel), ctypes.byref(splits)),
               'musc_b200_masked_attention_plan')
    return kernel.value, splits.value


def _assert_heads(got, q, k, v, heads, kv_heads, q_off, k_off, rows=None, slopes=None, **options):
    """The query heads of the first and of the last key head against the formula (``rows``: of these rows)."""
    d, group = q.shape[1] // heads, heads // kv_heads
    for h in sorted({0, kv_heads - 1}):
        part = None if slopes is None else slopes[h * group:(h + 1) * group]
        want, tol = _reference(_of_heads(q, d, h * group, group), _of_heads(k, d, h, 1), _of_heads(v, d, h, 1), group, 1,
                               q_off, k_off, slopes=part, **options)
        out = _of_heads(got, d, h * group, group)
        rows = ~want.isnan().all(1) if rows is None else rows
        _assert_close(out[rows], want[rows], tol[rows])


# ----------------------------------------------------------------------------- offsets
@pytest.mark.parametrize('kernel,n,heads', [(ROWS, 20, 2), (ROWS, 21, 16), (TILES, 900, 64)])
def test_query_offsets_past_the_tensor(cuda_device, kernel, n, heads):
    """Documents that begin before the first row or end behind the last one are cut to the rows there are,
    positions too; documents that lie outside have none."""
    from musc_b200 import ops
    d, kv_heads = 64, heads // 2
    lens = [40, 600, 33, n + 200, 7]
    k_off = _starts(lens)
    q, k, v = _random_qkv(cuda_device, n, k_off[-1], heads, kv_heads, d, torch.float16, 60, False)
    slopes = 2.0 ** (-(torch.arange(heads, device=cuda_device) % 5).float())
    assert _plan(n, k_off[-1], 5, heads, kv_heads, d, True)[0] == kernel
    for q_off in ([-30, -9, n // 3, n // 3, n + 50, n + 60], [-3, 1, 2, 9, 1 << 30, 1 << 30]):
        got = ops.attention_masked(q, k, v, heads, kv_heads, offsets=_i32(q_off, cuda_device), kv_offsets=_i32(k_off, cuda_device),
                                   causal=True, slopes=slopes)
        cut = [min(max(o, 0), n) for o in q_off]
        _assert_heads(got, q, k, v, heads, kv_heads, cut, k_off, causal=True, slopes=slopes)
