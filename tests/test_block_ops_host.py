"""Encoder-block operators (masked attention, rotary positions, RMS norm): contracts that the
library and the wrappers check before any device work."""
from __future__ import annotations

import ctypes

import pytest
import torch

from musc_b200 import _lib, ops

vp = ctypes.c_void_p


def _attention_args(**changes):
    at = 1 << 20
    kwargs = dict(q=at, k=2 * at, v=3 * at, out=4 * at, dtype=_lib.F16, heads=4, kv_heads=2, head_dim=64, q_rows=10,
                  kv_rows=20, q_stride=256, k_stride=128, v_stride=128, out_stride=256, documents=2, causal=1,
                  q_offsets=5 * at, kv_offsets=6 * at, scale=0.125, softcap=0.0)
    kwargs.update(changes)
    return _lib.MaskedAttentionArgs(**kwargs)


@pytest.mark.parametrize('changes,message', [
    (dict(dtype=_lib.F32), 'dtype'), (dict(head_dim=80), 'head_dim'), (dict(heads=3), 'multiple of kv_heads'),
    (dict(kv_heads=0), 'multiple of kv_heads'), (dict(q_rows=-1), 'q_rows'), (dict(kv_rows=1 << 31), 'q_rows'),
    (dict(documents=-1), 'documents'), (dict(scale=0.0), 'scale'), (dict(scale=float('nan')), 'scale'),
    (dict(scale=float('inf')), 'scale'), (dict(softcap=-1.0), 'softcap'), (dict(softcap=float('nan')), 'softcap'),
    (dict(softcap=1e-20), 'softcap'), (dict(softcap=1e20), 'softcap'), (dict(scale=-1.0), 'scale'),
    (dict(causal=0, prefix=1 << 20), 'prefix'), (dict(kv_offsets=None), 'go together'),
    (dict(q_offsets=None), 'go together'),
    (dict(q_offsets=None, kv_offsets=None, q_len=4, kv_len=10, kv_pitch=10), 'make q_rows'),
    (dict(q_offsets=None, kv_offsets=None, q_len=5, kv_len=10, kv_pitch=9), 'kv_pitch'),
    (dict(q_offsets=None, kv_offsets=None, q_len=5, kv_len=10, kv_pitch=11), 'within kv_rows'),
    (dict(q_offsets=None, kv_offsets=None, q_len=1 << 62, kv_len=10, kv_pitch=10, documents=8), 'q_len'),
    (dict(q=None), 'null'), (dict(k=None), 'null'), (dict(out=None), 'null'),
    (dict(q_stride=255), 'strides'), (dict(q_stride=260), 'multiples of 8'), (dict(v_stride=120), 'strides'),
    (dict(q=(1 << 20) + 8), '16-byte'), (dict(slopes=(1 << 20) + 2), '4-byte'),
    (dict(out=(1 << 20) + 256), 'overlap'), (dict(out=(2 << 20) + 16), 'overlap'), (dict(out=(3 << 20) - 2048), 'overlap'),
])
def test_attention_contract(changes, message):
    st = _lib.lib().musc_b200_masked_attention(ctypes.byref(_attention_args(**changes)), None)
    assert st == _lib.ERR_INVALID and message in _lib.last_error()


def test_attention_without_rows_or_arguments():
    lib = _lib.lib()
    assert lib.musc_b200_masked_attention(None, None) == _lib.ERR_INVALID
    assert lib.musc_b200_masked_attention_bytes(None) == 0
    assert lib.musc_b200_masked_attention(ctypes.byref(_attention_args(q_rows=0, q=None, out=None)), None) == _lib.OK
    assert lib.musc_b200_masked_attention(ctypes.byref(_attention_args(documents=0)), None) == _lib.OK


def test_attention_workspace():
    """Few rows against many keys split the keys: the call asks for its workspace and checks it."""
    lib = _lib.lib()
    args = _attention_args(kv_rows=100_000, v=64 << 20, out=128 << 20)
    need = lib.musc_b200_masked_attention_bytes(ctypes.byref(args))
    assert need > 0
    assert lib.musc_b200_masked_attention(ctypes.byref(args), None) == _lib.ERR_WORKSPACE
    args.workspace, args.workspace_bytes = 1 << 30, need - 1
    assert lib.musc_b200_masked_attention(ctypes.byref(args), None) == _lib.ERR_WORKSPACE
    args.workspace, args.workspace_bytes = (1 << 30) + 16, need
    assert lib.musc_b200_masked_attention(ctypes.byref(args), None) == _lib.ERR_INVALID
    assert lib.musc_b200_masked_attention_bytes(ctypes.byref(_attention_args(head_dim=80))) == 0


def _rotary(**changes):
    at = 1 << 20
    a = dict(q=at, k=2 * at, q_out=3 * at, k_out=4 * at, dtype=_lib.F16, tokens=10, heads=4, kv_heads=2, head_dim=64,
             q_stride=256, k_stride=128, q_out_stride=256, k_out_stride=128, positions=5 * at, float_positions=0, axes=2,
             frequencies=6 * at, axis=7 * at, pairs=32, adjacent=0)
    a.update(changes)
    return _lib.lib().musc_b200_rotary(*a.values(), None)


@pytest.mark.parametrize('changes,message', [
    (dict(dtype=_lib.E4M3), 'dtype'), (dict(tokens=-1), 'tokens'), (dict(heads=0), 'heads'), (dict(axes=0), 'axes'),
    (dict(pairs=33), 'pairs'), (dict(pairs=0), 'pairs'), (dict(head_dim=514), 'head_dim'), (dict(q=None), 'null'),
    (dict(k_out=None), 'null'), (dict(positions=None), 'null'), (dict(q_stride=255), 'strides'),
    (dict(q=(1 << 20) + 1), 'aligned'), (dict(positions=(5 << 20) + 2), 'aligned'), (dict(axis=(7 << 20) + 1), 'aligned'),
    (dict(q_out=(1 << 20) + 16), 'overlap'),                       # shifted by half a row
    (dict(q_out=2 << 20), 'overlap'),                              # onto the other input
    (dict(k_out=3 << 20), 'overlap'),                              # two outputs in one place
    (dict(q_out=1 << 20, q_out_stride=512), 'overlap'),            # its own input at another stride
])
def test_rotary_contract(changes, message):
    assert _rotary(**changes) == _lib.ERR_INVALID and message in _lib.last_error()


def test_rotary_accepts_columns_of_one_buffer_and_no_tokens():
    assert _rotary(tokens=0, q=None) == _lib.OK
    at = 1 << 20
    # q and k as columns of one projection, turned in place: past the checks (what is missing here is the device)
    inplace = dict(q=at, q_out=at, k=at + 512, k_out=at + 512, q_stride=384, q_out_stride=384, k_stride=384, k_out_stride=384)
    assert _rotary(**inplace) != _lib.ERR_INVALID
    assert _rotary(**dict(inplace, k=at + 510, k_out=at + 510)) == _lib.ERR_INVALID


def _norm(**changes):
    at = 1 << 20
    a = dict(x=at, x_dtype=_lib.F32, delta=2 * at, delta_dtype=_lib.F16, weight=3 * at, eps=1e-6, out=4 * at,
             out_dtype=_lib.E4M3, scales=5 * at, group=128, rows=4, channels=1000, x_stride=1000, delta_stride=1000,
             out_stride=1000)
    a.update(changes)
    return _lib.lib().musc_b200_add_rmsnorm(*a.values(), None)


@pytest.mark.parametrize('changes,message', [
    (dict(x_dtype=_lib.E4M3), 'x and delta'), (dict(delta_dtype=7), 'x and delta'), (dict(out_dtype=9), 'out dtype'),
    (dict(rows=-1), 'rows'), (dict(channels=0), 'channels'), (dict(channels=32769), 'channels'), (dict(eps=-1.0), 'eps'),
    (dict(eps=float('nan')), 'eps'), (dict(group=100), 'group'), (dict(group=128, out_dtype=_lib.F16), 'group'),
    (dict(x=None), 'null'), (dict(scales=None), 'null'), (dict(weight=None), 'null'), (dict(x_stride=999), 'strides'),
    (dict(delta_stride=5), 'strides'), (dict(x=(1 << 20) + 2), 'aligned'), (dict(out=(1 << 20) + 16), 'overlap'),
    (dict(out=(2 << 20) + 16), 'overlap'), (dict(delta=(1 << 20) + 4000), 'overlap'),
    (dict(out=(3 << 20) + 16), 'overlap'), (dict(weight=(1 << 20) + 16), 'overlap'),
    (dict(scales=(1 << 20) + 8), 'overlap'), (dict(scales=(4 << 20) + 8), 'overlap'),
])
def test_norm_contract(changes, message):
    assert _norm(**changes) == _lib.ERR_INVALID and message in _lib.last_error()


@pytest.mark.parametrize('changes,message', [(dict(scales=(5 << 20) + 2), 'scales must be aligned'),
                                             (dict(scales=(3 << 20) + 8), 'overlap')])
def test_norm_scales_contract(changes, message):
    assert _norm(**changes) == _lib.ERR_INVALID and message in _lib.last_error()


def test_norm_without_rows():
    assert _norm(rows=0, x=None) == _lib.OK


def test_wrappers_refuse_cpu_tensors():
    q = torch.zeros(4, 128, dtype=torch.float16)
    off = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(ValueError, match='CUDA'):
        ops.attention_masked(q, q, q, 2, offsets=off)
    with pytest.raises(ValueError, match='CUDA'):
        ops.rotary(q, q, torch.zeros(4, 1, dtype=torch.int32), torch.ones(4), torch.zeros(4, dtype=torch.int32), 2)
    with pytest.raises(ValueError, match='CUDA'):
        ops.add_rmsnorm(q, None, torch.ones(128))


def test_rotary_frequencies():
    f, a = ops.rotary_frequencies([2, 3], base=100.0, device='cpu')
    assert a.tolist() == [0, 0, 1, 1, 1] and a.dtype == torch.int32 and f.dtype == torch.float32
    torch.testing.assert_close(f, torch.tensor([1.0, 0.1, 1.0, 100.0 ** (-1 / 3), 100.0 ** (-2 / 3)]))
    f, a = ops.rotary_frequencies([1, 0, 3], base=16.0, shared=True, device='cpu')
    assert a.tolist() == [0, 2, 2, 2]
    torch.testing.assert_close(f, torch.tensor([1.0, 0.5, 0.25, 0.125]))
    for bad in ([], [0, 0], [-1, 3]):
        with pytest.raises(ValueError):
            ops.rotary_frequencies(bad, device='cpu')


@pytest.mark.parametrize('q_len,kv_len', [(70, 70), (1, 8192), (0, 0), (1 << 40, 5)])
def test_attention_of_an_empty_batch(q_len, kv_len):
    """A batch of no items has no rows, whatever the items' length."""
    args = _attention_args(q=None, k=None, v=None, out=None, q_offsets=None, kv_offsets=None, documents=0, q_rows=0, kv_rows=0,
                           q_len=q_len, kv_len=kv_len, kv_pitch=kv_len)
    assert _lib.lib().musc_b200_masked_attention(ctypes.byref(args), None) == _lib.OK
    assert _lib.lib().musc_b200_masked_attention_bytes(ctypes.byref(args)) == 0
    args.documents = 1  # an item without its rows
    if q_len:
        assert _lib.lib().musc_b200_masked_attention(ctypes.byref(args), None) == _lib.ERR_INVALID


def _plan(**changes):
    """(tile kernel, splits) of a call."""
    tiles, splits = ctypes.c_int(-1), ctypes.c_int(-1)
    st = _lib.lib().musc_b200_masked_attention_plan(ctypes.byref(_attention_args(**changes)), ctypes.byref(tiles),
                                                    ctypes.byref(splits))
    assert st == _lib.OK, _lib.last_error()
    return tiles.value, splits.value


def test_attention_plan():
    lib, one = _lib.lib(), ctypes.c_int(7)
    assert lib.musc_b200_masked_attention_plan(None, ctypes.byref(one), ctypes.byref(one)) == _lib.ERR_INVALID
    assert lib.musc_b200_masked_attention_plan(ctypes.byref(_attention_args()), None, ctypes.byref(one)) == _lib.ERR_INVALID
    bad = _attention_args(head_dim=80)
    assert lib.musc_b200_masked_attention_plan(ctypes.byref(bad), ctypes.byref(one), ctypes.byref(one)) == _lib.ERR_INVALID
    assert _plan(q_rows=0) == (0, 0) and _plan(documents=0) == (0, 0)
    assert _plan(kv_rows=0) == (0, 1)                                        # no keys: nothing to split
    assert _plan(q_rows=8192, kv_rows=8192, heads=16, kv_heads=16, documents=1, causal=0) == (1, 1)
    assert _plan(q_rows=32, kv_rows=32 * 8192, heads=32, kv_heads=8, documents=32)[0] == 0
    # above eight splits the row kernel's sums go through the workspace, as the tile kernel's do above one
    for sizes in (dict(q_rows=8, kv_rows=40_000, heads=8, kv_heads=1, head_dim=128, documents=2),
                  dict(q_rows=512, kv_rows=8192, documents=1, causal=0)):
        args = _attention_args(**sizes)
        tiles, splits = _plan(**sizes)
        assert splits > (1 if tiles else 8)
        rows = sizes['q_rows'] * args.heads * splits
        assert lib.musc_b200_masked_attention_bytes(ctypes.byref(args)) >= rows * (args.head_dim * 4 + 8)


@pytest.mark.parametrize('head_dim', [64, 128])
def test_attention_plan_of_long_contexts(head_dim):
    """Few heads over very long keys: the tile kernel divides a row tile's keys into 32 at most, the row kernel into
    64, so one row goes to the row kernel and 256 rows to the tile kernel, however long the keys."""
    for keys in (300_000, 1_000_000):
        for heads in (1, 2):
            sizes = dict(kv_rows=keys, heads=heads, kv_heads=heads, head_dim=head_dim, documents=1)
            tiles, splits = _plan(q_rows=1, **sizes)
            assert tiles == 0 and splits > 32
            assert _plan(q_rows=256, **dict(sizes, heads=2, kv_heads=1)) == (1, 32)


def test_forward_only_refuses_gradients_and_tangents():
    from torch.autograd import forward_ad
    x, asks = torch.ones(3), torch.ones(3, requires_grad=True)
    ops._forward_only('op', x, None)
    with pytest.raises(ValueError, match='gradient'):
        ops._forward_only('op', x, None, asks)
    with torch.no_grad():
        ops._forward_only('op', asks)
    with forward_ad.dual_level():
        ops._forward_only('op', x, None)
        for enabled in (True, False):
            with torch.set_grad_enabled(enabled), pytest.raises(ValueError, match='tangent'):
                ops._forward_only('op', None, forward_ad.make_dual(x, x))
