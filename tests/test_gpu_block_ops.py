"""GPU numerics of the encoder-block operators: masked attention, rotary positions over several
axes, residual add + RMS norm.

Every operator is compared with its formula evaluated in float64 on the same inputs.  With
u = finfo(type).eps / 2 (the error of one rounding to the type):

* attention: the probabilities are rounded once (u of each) and the output once, so
  |error| <= u (A + |out|) + 2 e A, where A is the same average of |v| and e bounds the relative error
  of a probability from its 32-bit score: a dot product of D terms is off by at most
  (D + 8) 2^-24 of the sum of its terms' magnitudes, the cap by 2^-20 of cap + 1, the bias by 2^-22 of
  its value, exponential and sums by 2^-18.
* rotary: cosine and sine are off by less than 2^-21 (angle of 64 bits rounded to a 32-bit fraction of
  a turn, 2 ulp of the function, two products), the result is rounded once.
* norm: a sum of n squares in runs of 32 and a tree of 10 levels is off by 42 2^-24, its root by half,
  the products by 4 2^-24: 2^-18 in all, and one rounding; e4m3 rounds by 2^-4 of the value or half
  its smallest step, 2^-10.
"""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _unit(dtype):
    return torch.finfo(dtype).eps / 2


# ----------------------------------------------------------------------------- attention
def _intervals(q_off, k_off, k_len, causal, prefix):
    """Per row (document, first key, end of the visible keys, key position); rows of no document: None."""
    rows = {}
    for d in range(len(q_off) - 1):
        nq, k0 = q_off[d + 1] - q_off[d], k_off[d]
        nk = k_off[d + 1] - k0 if k_len is None else k_len[d]
        for i in range(nq):
            seen = nk
            if causal:
                seen = min(max(i + nk - nq + 1, prefix[d] if prefix is not None else 0, 0), nk)
            rows[q_off[d] + i] = (k0, k0 + seen, k0 + i + nk - nq)
    return rows


def _reference(q, k, v, heads, kv_heads, q_off, k_off, k_len=None, causal=False, prefix=None, softcap=0.0, slopes=None,
               scale=None):
    """(out, tolerance) in float64; rows of no document stay NaN."""
    d = q.shape[1] // heads
    scale = d ** -0.5 if scale is None else scale
    u = _unit(q.dtype)
    rows = _intervals(q_off, k_off, k_len, causal, prefix)
    want = torch.full(q.shape, math.nan, dtype=torch.float64, device=q.device)
    tol = torch.full_like(want, math.nan)
    if not rows:
        return want, tol
    index = torch.tensor(sorted(rows), device=q.device)
    lo, hi, pos = (torch.tensor([rows[int(r)][c] for r in index], device=q.device)[:, None] for c in range(3))
    key = torch.arange(k.shape[0], device=q.device)[None]
    visible = (key >= lo) & (key < hi)
    for h in range(heads):
        at = h // (heads // kv_heads) * d
        qh = q[index, h * d:(h + 1) * d].double()
        kh, vh = (torch.where(visible.any(0)[:, None], t[:, at:at + d].double(), 0.0) for t in (k, v))
        z = qh @ kh.T * scale
        size = qh.abs() @ kh.abs().T * scale
        e = torch.where(visible, size, 0.0).amax(1, keepdim=True) * (d + 8) * 2.0 ** -24 + 2.0 ** -18
        if softcap:
            z = softcap * torch.tanh(z / softcap)
            e = e + (softcap + 1) * 2.0 ** -20
        if slopes is not None:
            bias = float(slopes[h]) * (key - pos).abs()
            z = z - bias
            e = e + torch.where(visible, bias, 0.0).amax(1, keepdim=True) * 2.0 ** -22
        z = torch.where(visible, z, -math.inf)
        top = z.amax(1, keepdim=True)
        p = torch.exp(z - torch.where(torch.isfinite(top), top, 0.0))
        p = torch.where(visible, p / p.sum(1, keepdim=True), 0.0)
        out, mean = p @ vh, p @ vh.abs()
        want[index, h * d:(h + 1) * d] = out
        tol[index, h * d:(h + 1) * d] = u * (mean + out.abs()) * (1 + 2.0 ** -6) + 2 * e * mean + 2.0 ** -24
    return want, tol


def _assert_close(got, want, tol):
    bad = ~((got.double() - want).abs() <= tol)
    assert not bool(bad.any()), (int(bad.sum()), got[bad][:4], want[bad][:4], tol[bad][:4])


def _random_qkv(dev, tq, tk, heads, kv_heads, d, dtype, seed, self_attention):
    g = torch.Generator(device=dev).manual_seed(seed)
    rand = lambda *shape: torch.randn(*shape, generator=g, device=dev).to(dtype)
    if self_attention:  # columns of one projection
        qkv = rand(tq, (heads + 2 * kv_heads) * d)
        return qkv[:, :heads * d], qkv[:, heads * d:(heads + kv_heads) * d], qkv[:, (heads + kv_heads) * d:]
    return rand(tq, heads * d), rand(tk, kv_heads * d), rand(tk, kv_heads * d)


def _starts(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return out


def _i32(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


# documents (queries, keys), heads, kv_heads, head_dim, options
CASES = [
    ([(1, 1)], 1, 1, 64, {}),
    ([(1, 17)], 3, 3, 128, {}),
    ([(1, 1370)] * 3, 4, 4, 64, {}),
    ([(1, 700), (1, 1), (1, 0), (1, 129)], 8, 2, 128, dict(softcap=30.0)),
    ([(3, 65), (5, 5), (1, 300), (0, 9), (2, 1)], 6, 2, 64, dict(causal=True, bias=True)),
    ([(7, 2)], 2, 1, 64, dict(causal=True)),                                  # the first five rows see no key
    ([(1, 513)], 40, 1, 64, dict(bias=True, softcap=20.0)),                    # a group of 40 heads
    ([(200, 200)], 2, 2, 64, {}),
    ([(256, 256), (129, 129)], 2, 1, 128, dict(causal=True)),
    ([(300, 300), (1, 1), (0, 0), (77, 77), (128, 128), (1, 1)], 4, 2, 64, dict(causal=True, prefix=[100, 1, 0, 90, 0, 1])),
    ([(37, 37)] * 20, 3, 3, 64, {}),                                           # several documents in a tile
    ([(5, 5)] * 70 + [(600, 600)] + [(1, 1)] * 40, 2, 2, 128, dict(causal=True, softcap=50.0, bias=True)),
    ([(130, 700), (260, 300)], 4, 1, 128, dict(causal=True, prefix=[650, 0], bias=True)),
    ([(900, 40)], 2, 2, 64, dict(causal=True)),                                # most rows see no key
    ([(1370, 1370), (1025, 1025)], 2, 2, 64, {}),
    ([(257, 1111)], 3, 1, 128, dict(softcap=5.0)),
    ([(640, 640)], 2, 2, 64, dict(bias=True)),                                 # the bias on both sides
]


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16])
@pytest.mark.parametrize('case', range(len(CASES)))
def test_attention_matches_formula(cuda_device, case, dtype):
    from musc_b200 import ops
    docs, heads, kv_heads, d, options = CASES[case]
    options = dict(options)
    q_off, k_off = _starts([n for n, _ in docs]), _starts([m for _, m in docs])
    same = all(n == m for n, m in docs)
    q, k, v = _random_qkv(cuda_device, q_off[-1], k_off[-1], heads, kv_heads, d, dtype, 100 + case, same)
    slopes = 2.0 ** (-torch.arange(1, heads + 1, device=cuda_device).float()) if options.pop('bias', False) else None
    prefix = options.pop('prefix', None)
    got = ops.attention_masked(q, k, v, heads, kv_heads, offsets=_i32(q_off, cuda_device),
                               kv_offsets=None if same else _i32(k_off, cuda_device),
                               prefix=None if prefix is None else _i32(prefix, cuda_device), slopes=slopes, **options)
    _assert_close(got, *_reference(q, k, v, heads, kv_heads, q_off, k_off, prefix=prefix, slopes=slopes, **options))


@pytest.mark.parametrize('d', [64, 128])
@pytest.mark.parametrize('n_q', [1, 3, 40, 300])
@pytest.mark.parametrize('causal', [False, True])
def test_attention_cache_slots_ignore_what_lies_behind(cuda_device, n_q, causal, d):
    """Key slots used to differing lengths: what lies behind a slot's keys (NaN, infinities) and in rows
    that no document owns changes nothing, bit for bit."""
    from musc_b200 import ops
    heads, kv_heads, slot, lengths = 4, 2, 333, [333, 301, 0, 128, 300]
    docs = len(lengths)
    q, k, v = _random_qkv(cuda_device, docs * n_q, docs * slot, heads, kv_heads, d, torch.bfloat16, 5 + n_q, False)
    for fill in (0.0, math.nan, math.inf):
        for i, n in enumerate(lengths):
            k[i * slot + n:(i + 1) * slot] = fill
            v[i * slot + n:(i + 1) * slot] = -fill
        got = ops.attention_masked(q, k, v, heads, kv_heads, offsets=_i32(_starts([n_q] * docs), cuda_device),
                                   kv_offsets=_i32(_starts([slot] * docs), cuda_device),
                                   kv_lengths=_i32(lengths, cuda_device), causal=causal)
        if fill == 0.0:
            clean = got
            _assert_close(got, *_reference(q, k, v, heads, kv_heads, _starts([n_q] * docs), _starts([slot] * docs),
                                           lengths, causal))
        else:
            assert torch.equal(got, clean)
    # the same as a batch: the host knows a document's keys there, so the sums may be split in another order
    batched = ops.attention_masked(q.view(docs, n_q, -1), k.view(docs, slot, -1), v.view(docs, slot, -1), heads, kv_heads,
                                   kv_lengths=_i32(lengths, cuda_device), causal=causal)
    for i, n in enumerate(lengths):
        k[i * slot + n:(i + 1) * slot] = v[i * slot + n:(i + 1) * slot] = 0.0
    _assert_close(batched.view_as(clean), *_reference(q, k, v, heads, kv_heads, _starts([n_q] * docs),
                                                      _starts([slot] * docs), lengths, causal))


@pytest.mark.parametrize('d,dtype', [(64, torch.float16), (128, torch.bfloat16)])
@pytest.mark.parametrize('poison', [math.nan, math.inf, -math.inf])
def test_attention_masked_values_do_not_leak(cuda_device, poison, d, dtype):
    """Keys and values that a row does not see may hold anything: later tokens of its own document, other
    documents in the same tile, the type's lowest value in scores."""
    from musc_b200 import ops
    heads, lens = 2, [150, 30, 200, 9]
    off = _starts(lens)
    q, k, v = _random_qkv(cuda_device, off[-1], off[-1], heads, heads, d, dtype, 77, False)
    late = [off[1] - 1, off[3] - 2]            # the last key of one document, the last but one of another
    k[late] = torch.finfo(dtype).min
    v[late] = poison
    want, tol = _reference(q, torch.where(k < -1e4, 0.0, k), torch.where(torch.isfinite(v), v, 0.0), heads, heads, off, off,
                           causal=True)
    got = ops.attention_masked(q, k, v, heads, offsets=_i32(off, cuda_device), causal=True)
    clean = [r for r in range(off[-1]) if not (off[1] - 1 <= r < off[1] or off[3] - 2 <= r < off[3])]
    _assert_close(got[clean], want[clean], tol[clean])
    # documents of their own: only the poisoned ones are touched
    got = ops.attention_masked(q, k, v, heads, offsets=_i32(off, cuda_device))
    want, tol = _reference(q, torch.where(k < -1e4, 0.0, k), torch.where(torch.isfinite(v), v, 0.0), heads, heads, off, off)
    for first, end in ((off[1], off[2]), (off[3], off[4])):
        _assert_close(got[first:end], want[first:end], tol[first:end])


def test_attention_visible_nan_and_infinity(cuda_device):
    """A value that a row does see reaches it."""
    from musc_b200 import ops
    q, k, v = _random_qkv(cuda_device, 300, 300, 1, 1, 64, torch.float16, 8, False)
    k = k * 0.1
    v[280, 3], v[40, 5] = math.nan, math.inf
    got = ops.attention_masked(q, k, v, 1, offsets=_i32([0, 300], cuda_device), causal=True)
    assert torch.isnan(got[280:, 3]).all() and torch.isfinite(got[:280, 3]).all()
    assert torch.isinf(got[40:, 5]).all() and torch.isfinite(got[:40, 5]).all()
    q[7] = math.nan
    got = ops.attention_masked(q, k, v, 1, offsets=_i32([0, 300], cuda_device), causal=True)
    assert torch.isnan(got[7]).all() and torch.isfinite(got[:7]).all() and torch.isfinite(got[8:40]).all()


@pytest.mark.parametrize('d,n', [(64, 5), (128, 400)])
def test_attention_leaves_rows_outside_documents(cuda_device, d, n):
    from musc_b200 import ops
    q, k, v = _random_qkv(cuda_device, n + 20, n + 20, 2, 2, d, torch.float16, 9, True)
    out = torch.full((n + 20, 2 * d), 7.0, dtype=torch.float16, device=cuda_device)
    off = _i32([10, 10 + n], cuda_device)
    ops.attention_masked(q, k, v, 2, offsets=off, out=out)
    assert bool((out[:10] == 7).all()) and bool((out[10 + n:] == 7).all())
    want, tol = _reference(q, k, v, 2, 2, [10, 10 + n], [10, 10 + n])
    _assert_close(out[10:10 + n], want[10:10 + n], tol[10:10 + n])
    # no documents, no queries, no keys
    ops.attention_masked(q, k, v, 2, offsets=_i32([0], cuda_device), out=out)
    assert bool((out[:10] == 7).all())
    assert ops.attention_masked(q[:0], k, v, 2, offsets=_i32([0, 0], cuda_device), kv_offsets=off).shape == (0, 2 * d)
    none = ops.attention_masked(q, k[:0], v[:0], 2, offsets=_i32([0, n + 20], cuda_device), kv_offsets=_i32([0, 0], cuda_device))
    assert bool((none == 0).all())


@pytest.mark.parametrize('n', [3, 500])
def test_attention_offsets_out_of_range_stay_inside(cuda_device, n):
    """Offsets and lengths past the tensors are clamped to them."""
    from musc_b200 import ops
    q, k, v = _random_qkv(cuda_device, n, 600, 2, 1, 64, torch.float16, 10, False)
    got = ops.attention_masked(q, k, v, 2, 1, offsets=_i32([0, n], cuda_device), kv_offsets=_i32([-50, 100_000], cuda_device),
                               kv_lengths=_i32([1 << 30], cuda_device))
    _assert_close(got, *_reference(q, k, v, 2, 1, [0, n], [0, 600]))


def test_attention_batch_forms_and_strides(cuda_device):
    """(B, L, W) views: items a cache slot apart, a slice of longer items, one token of each."""
    from musc_b200 import ops
    g = torch.Generator(device=cuda_device).manual_seed(11)
    b, length, slot, heads, d = 3, 70, 100, 2, 64
    cache = torch.randn(b, slot, 4 * d + 8, generator=g, device=cuda_device).to(torch.bfloat16)
    x = torch.randn(b, length, heads * d, generator=g, device=cuda_device).to(torch.bfloat16)
    k, v = cache[:, :length, :d], cache[:, :length, d:2 * d]
    flat = lambda t: t.reshape(b * length, -1)
    off = _starts([length] * b)
    _assert_close(flat(ops.attention_masked(x, k, v, heads, 1, causal=True)),
                  *_reference(flat(x), flat(k), flat(v), heads, 1, off, off, causal=True))
    last = x[:, -1:]   # one token of each item: its rows lie a whole item apart
    got = ops.attention_masked(last, k, v, heads, 1, causal=True)
    _assert_close(got.reshape(b, -1), *_reference(last.reshape(b, -1), flat(k), flat(v), heads, 1, _starts([1] * b), off))
    one = ops.attention_masked(x[:1], k[:1], v[:1], heads, 1)
    _assert_close(one[0], *_reference(x[0], k[0], v[0], heads, 1, [0, length], [0, length]))


@pytest.mark.parametrize('n_q', [1, 130])
def test_attention_far_rows(cuda_device, n_q):
    """Keys whose element offsets pass 32 bits."""
    from musc_b200 import ops
    rows, d, width = 1_060_000, 64, 2048
    cache = torch.zeros(rows, width, dtype=torch.bfloat16, device=cuda_device)
    g = torch.Generator(device=cuda_device).manual_seed(12)
    tail = torch.randn(700, width, generator=g, device=cuda_device).to(torch.bfloat16)
    cache[rows - 700:] = tail
    q = torch.randn(n_q, d, generator=g, device=cuda_device).to(torch.bfloat16)
    got = ops.attention_masked(q, cache[:, width - d:], cache[:, :d], 1, offsets=_i32([0, n_q], cuda_device),
                               kv_offsets=_i32([rows - 700, rows], cuda_device))
    _assert_close(got, *_reference(q, tail[:, width - d:], tail[:, :d], 1, 1, [0, n_q], [0, 700]))


@pytest.mark.parametrize('n_q,n_k', [(1, 40_000), (200, 30_000)])
@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16])
def test_attention_long_axis(cuda_device, n_q, n_k, dtype):
    """Few rows against many keys: the keys are split and joined.  Scores grow along the keys, so that
    running maxima rise from split to split; fp16 probabilities of a flat tail are not lost."""
    from musc_b200 import ops
    q, k, v = _random_qkv(cuda_device, n_q, n_k, 2, 1, 64, dtype, 13, False)
    k = (k.float() * torch.linspace(0.1, 4.0, n_k, device=cuda_device)[:, None]).to(dtype)
    got = ops.attention_masked(q, k, v, 2, 1, offsets=_i32([0, n_q], cuda_device), kv_offsets=_i32([0, n_k], cuda_device))
    _assert_close(got, *_reference(q, k, v, 2, 1, [0, n_q], [0, n_k]))
    # one key at score 16, the others at 0: weights of e^-16 that add up to half a percent
    q, k = torch.zeros_like(q), torch.zeros_like(k)
    q[:, 0::64], k[0, 0] = 11.3125, 11.3125
    got = ops.attention_masked(q, k, v, 2, 1, offsets=_i32([0, n_q], cuda_device), kv_offsets=_i32([0, n_k], cuda_device))
    _assert_close(got, *_reference(q, k, v, 2, 1, [0, n_q], [0, n_k]))


def _lengths(kind, seed):
    g = torch.Generator().manual_seed(seed)
    if kind == 'middling':      # 60 documents, some longer than a row tile, some empty
        n = torch.randint(0, 160, (60,), generator=g)
        n[::9] += 300
        n[5] = n[6] = 0
    elif kind == 'tiny':        # more documents than are looked up in shared memory
        n = torch.randint(8, 28, (1100,), generator=g)
    elif kind == 'one_of_many': # one long document among short ones
        n = torch.randint(1, 90, (33,), generator=g)
        n[20] = 1500
    else:                       # long ones, ending at and beside tile borders
        n = torch.tensor([256, 255, 257, 512, 1, 64, 65, 700])
    return n.tolist()


@pytest.mark.parametrize('causal', [False, True])
@pytest.mark.parametrize('kind,d', [('middling', 64), ('tiny', 64), ('one_of_many', 128), ('long', 128)])
def test_attention_many_documents(cuda_device, kind, d, causal):
    """Row tiles of many documents, packed rows before the first and behind the last one left alone."""
    from musc_b200 import ops
    lens = _lengths(kind, 40)
    off = [13 + o for o in _starts(lens)]
    q, k, v = _random_qkv(cuda_device, off[-1] + 30, off[-1] + 30, 2, 1, d, torch.bfloat16, 41, True)
    out = torch.full_like(q, 3.0)
    ops.attention_masked(q, k, v, 2, 1, offsets=_i32(off, cuda_device), causal=causal, out=out)
    assert bool((out[:13] == 3).all()) and bool((out[off[-1]:] == 3).all())
    want, tol = _reference(q, k, v, 2, 1, off, off, causal=causal)
    _assert_close(out[13:off[-1]], want[13:off[-1]], tol[13:off[-1]])


@pytest.mark.parametrize('length', [17, 100, 256, 300, 515])
def test_attention_batches_of_one_length(cuda_device, length):
    from musc_b200 import ops
    q, k, v = _random_qkv(cuda_device, 5 * length, 5 * length, 4, 2, 64, torch.float16, 42, True)
    view = lambda t: t.unflatten(0, (5, length))
    got = ops.attention_masked(view(q), view(k), view(v), 4, 2, causal=True, softcap=20.0)
    off = _starts([length] * 5)
    _assert_close(got.flatten(0, 1), *_reference(q, k, v, 4, 2, off, off, causal=True, softcap=20.0))


@pytest.mark.parametrize('d', [64, 128])
@pytest.mark.parametrize('n_q', [4, 150])
@pytest.mark.parametrize('poison', [0.0, math.nan])
def test_attention_split_documents(cuda_device, n_q, poison, d):
    """Several documents of few rows over long keys: both kernels split the keys; a NaN in a value that only the
    last rows see stays with them."""
    from musc_b200 import ops
    docs, keys = 2, [9001, 5003]
    q, k, v = _random_qkv(cuda_device, docs * n_q, sum(keys), 2, 1, d, torch.float16, 43, False)
    q_off, k_off = _starts([n_q] * docs), _starts(keys)
    prefix = [4000, 5003]
    clean = v.clone()
    v[k_off[1] - 2, 5] = poison                    # the last but one key of the first document
    got = ops.attention_masked(q, k, v, 2, 1, offsets=_i32(q_off, cuda_device), kv_offsets=_i32(k_off, cuda_device),
                               causal=True, prefix=_i32(prefix, cuda_device))
    want, tol = _reference(q, k, clean if math.isnan(poison) else v, 2, 1, q_off, k_off, causal=True, prefix=prefix)
    rows = [r for r in range(docs * n_q) if not (math.isnan(poison) and n_q - 2 <= r < n_q)]
    _assert_close(got[rows], want[rows], tol[rows])
    if math.isnan(poison):
        assert torch.isnan(got[n_q - 2:n_q, [5, 5 + d]]).all()
        others = [c for c in range(2 * d) if c % d != 5]
        _assert_close(got[n_q - 2:n_q][:, others], want[n_q - 2:n_q][:, others], tol[n_q - 2:n_q][:, others])


@pytest.mark.parametrize('heads,kv_heads,d', [(1, 1, 64), (6, 2, 128), (5, 1, 64), (9, 1, 64), (16, 1, 128), (17, 1, 64)])
@pytest.mark.parametrize('keys', [3, 700, 9000])
@pytest.mark.parametrize('options', [{}, dict(causal=True), dict(causal=True, bias=True, softcap=8.0, prefix=True)])
def test_attention_few_rows_of_each_document(cuda_device, heads, kv_heads, d, keys, options):
    from musc_b200 import ops
    docs = [(n, keys + n % 5) for n in (2, 1, 15, 0, 3, 16, 7, 4, 9, 31, 5)]
    options, dtype = dict(options), torch.bfloat16 if heads % 2 else torch.float16
    q_off, k_off = _starts([n for n, _ in docs]), _starts([m for _, m in docs])
    q, k, v = _random_qkv(cuda_device, q_off[-1], k_off[-1], heads, kv_heads, d, dtype, 7 * keys + heads, False)
    prefix = [m - n // 2 for n, m in docs] if options.pop('prefix', False) else None
    slopes = 2.0 ** (-torch.arange(1, heads + 1, device=cuda_device).float()) if options.pop('bias', False) else None
    got = ops.attention_masked(q, k, v, heads, kv_heads, offsets=_i32(q_off, cuda_device), kv_offsets=_i32(k_off, cuda_device),
                               prefix=None if prefix is None else _i32(prefix, cuda_device), slopes=slopes, **options)
    _assert_close(got, *_reference(q, k, v, heads, kv_heads, q_off, k_off, prefix=prefix, slopes=slopes, **options))


@pytest.mark.parametrize('poison', [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize('keys', [40, 5000])
@pytest.mark.parametrize('bias', [False, True])
def test_attention_last_keys_reach_only_the_rows_behind_them(cuda_device, keys, poison, bias):
    """Rows of one document that share a product: values that are not finite at the last keys stay with the
    rows that see them."""
    from musc_b200 import ops
    n, heads, d = 6, 4, 128
    q, k, v = _random_qkv(cuda_device, n, keys, heads, 2, d, torch.float16, keys, False)
    v = v.clone()
    v[keys - 2, ::3] = poison  # seen by the last two rows
    slopes = torch.tensor([0.5, 0.25, 0.0, 1.0], device=cuda_device) if bias else None
    got = ops.attention_masked(q, k, v, heads, 2, offsets=_i32([0, n], cuda_device), kv_offsets=_i32([0, keys], cuda_device),
                               causal=True, slopes=slopes)
    clean = v.clone()
    clean[keys - 2] = 0
    want, tol = _reference(q, k, clean, heads, 2, [0, n], [0, keys], causal=True, slopes=slopes)
    _assert_close(got[:n - 2], want[:n - 2], tol[:n - 2])
    hit = torch.arange(d * 2, device=cuda_device) % 3 == 0
    hit = torch.cat([hit[:d], hit[:d], hit[d:], hit[d:]])  # two heads for each key head
    assert not bool(got[n - 2:, hit].isfinite().any())
    assert bool(got[n - 2:, ~hit].isfinite().all())
    k = k.clone()
    k[keys - 1] = poison  # its scores reach the last row alone
    got = ops.attention_masked(q, k, clean, heads, 2, offsets=_i32([0, n], cuda_device), kv_offsets=_i32([0, keys], cuda_device),
                               causal=True, slopes=slopes)
    _assert_close(got[:n - 1], want[:n - 1], tol[:n - 1])


def _of_heads(t, d, first, count):
    return t[:, first * d:(first + count) * d]


@pytest.mark.parametrize('case', [i for i, c in enumerate(CASES) if sum(n for n, _ in c[0]) >= 16])
def test_attention_of_many_heads(cuda_device, case):
    """The same documents with 128 and more key heads, of which the first and the last are compared."""
    from musc_b200 import ops
    docs, heads, kv_heads, d, options = CASES[case]
    options, dtype, group = dict(options), torch.bfloat16 if case % 2 else torch.float16, heads // kv_heads
    kv_heads, heads = 128, 128 * group
    q_off, k_off = _starts([n for n, _ in docs]), _starts([m for _, m in docs])
    q, k, v = _random_qkv(cuda_device, q_off[-1], k_off[-1], heads, kv_heads, d, dtype, 900 + case, False)
    slopes = 2.0 ** (-(torch.arange(heads, device=cuda_device) % 9).float()) if options.pop('bias', False) else None
    prefix = options.pop('prefix', None)
    got = ops.attention_masked(q, k, v, heads, kv_heads, offsets=_i32(q_off, cuda_device), kv_offsets=_i32(k_off, cuda_device),
                               prefix=None if prefix is None else _i32(prefix, cuda_device), slopes=slopes, **options)
    for h in (0, kv_heads - 1):
        part = None if slopes is None else slopes[h * group:(h + 1) * group]
        want, tol = _reference(_of_heads(q, d, h * group, group), _of_heads(k, d, h, 1), _of_heads(v, d, h, 1), group, 1,
                               q_off, k_off, prefix=prefix, slopes=part, **options)
        _assert_close(_of_heads(got, d, h * group, group), want, tol)


@pytest.mark.parametrize('d', [64, 128])
@pytest.mark.parametrize('poison', [math.nan, math.inf, -math.inf])
def test_attention_of_many_heads_masked_values_do_not_leak(cuda_device, poison, d):
    """Documents of 300, 40 and 170 rows; the second one's last key and what lies behind the third's are not finite."""
    from musc_b200 import ops
    heads, lengths = 160, [300, 40, 170]
    off = _starts(lengths)
    q, k, v = _random_qkv(cuda_device, off[-1] + 30, off[-1] + 30, heads, heads, d, torch.float16, d, False)
    k, v = k.clone(), v.clone()
    k[off[2] - 1], v[off[2] - 1], k[off[3]:], v[off[3]:] = poison, poison, poison, poison
    got = ops.attention_masked(q, k, v, heads, heads, offsets=_i32(off, cuda_device), causal=True)
    clean_k, clean_v = k.clone(), v.clone()
    clean_k[off[2] - 1], clean_v[off[2] - 1] = 0, 0
    rows = torch.arange(off[-1], device=cuda_device) != off[2] - 1
    for h in (0, heads // 2, heads - 1):
        want, tol = _reference(*(_of_heads(t, d, h, 1) for t in (q, clean_k, clean_v)), 1, 1, off, off, causal=True)
        _assert_close(_of_heads(got, d, h, 1)[:off[-1]][rows], want[:off[-1]][rows], tol[:off[-1]][rows])
    assert not bool(got[off[2] - 1].isfinite().any())


@pytest.mark.parametrize('n,rows,heads,kv_heads,d', [(400, 12, 16, 16, 128), (290, 8, 16, 16, 64), (330, 3, 32, 16, 128),
                                                     (1500, 5, 12, 4, 64)])
def test_attention_many_short_documents_of_many_heads(cuda_device, n, rows, heads, kv_heads, d):
    from musc_b200 import ops
    lengths = [rows + (i % 3) - 1 for i in range(n)]
    off = _starts(lengths)
    q, k, v = _random_qkv(cuda_device, off[-1], off[-1], heads, kv_heads, d, torch.bfloat16, n, True)
    got = ops.attention_masked(q, k, v, heads, kv_heads, offsets=_i32(off, cuda_device), causal=True)
    group, last = heads // kv_heads, kv_heads - 1
    want, tol = _reference(_of_heads(q, d, last * group, group), _of_heads(k, d, last, 1), _of_heads(v, d, last, 1), group, 1,
                           off, off, causal=True)
    _assert_close(_of_heads(got, d, last * group, group), want, tol)


@pytest.mark.parametrize('n_q,n_k', [(40, 3000), (300, 700)])
@pytest.mark.parametrize('causal', [False, True])
def test_attention_cache_slots_of_many_heads(cuda_device, n_q, n_k, causal):
    """Slots in use to differing lengths; NaN behind them."""
    from musc_b200 import ops
    b, heads, kv_heads, d = 3, 192, 96, 64
    g = torch.Generator(device=cuda_device).manual_seed(n_q)
    q = torch.randn(b, n_q, heads * d, generator=g, device=cuda_device).half()
    k, v = (torch.randn(b, n_k, kv_heads * d, generator=g, device=cuda_device).half() for _ in range(2))
    used = [n_k, n_k // 2 + 1, n_q - 7]
    for i, n in enumerate(used):
        k[i, n:], v[i, n:] = math.nan, math.nan
    got = ops.attention_masked(q, k, v, heads, kv_heads, kv_lengths=_i32(used, cuda_device), causal=causal)
    for i, n in enumerate(used):
        h = kv_heads - 1
        want, tol = _reference(q[i, :, h * 2 * d:], k[i, :n, h * d:], v[i, :n, h * d:], 2, 1, [0, n_q], [0, n], causal=causal)
        _assert_close(got[i, :, h * 2 * d:], want, tol)


@pytest.mark.parametrize('n', [20, 900])
def test_attention_disordered_offsets_stay_inside(cuda_device, n):
    """Offsets that fall, repeat or leave the tensors: results are undefined, accesses are not."""
    from musc_b200 import ops
    q, k, v = _random_qkv(cuda_device, n, n, 2, 1, 64, torch.float16, 44, True)
    top = (1 << 31) - 1
    for q_off, k_off in (([0, n, 5, n], [0, 3, 2, n]), ([-7, 3, n // 2, top], [top, 0, -top, 9]), ([0, top, 0, n], [5, 5, 5, 5]),
                         ([n, n - 1, 2, 0], [0, n, 0, n]), ([-top - 1, top, -5, top], [-1, -1, top, top])):
        for causal in (False, True):
            ops.attention_masked(q, k, v, 2, 1, offsets=_i32(q_off, cuda_device), kv_offsets=_i32(k_off, cuda_device),
                                 kv_lengths=_i32([top, -3, 4], cuda_device), causal=causal)
    torch.cuda.synchronize()
    ops.check_device_error(cuda_device)
    got = ops.attention_masked(q, k, v, 2, 1, offsets=_i32([0, n], cuda_device))
    _assert_close(got, *_reference(q, k, v, 2, 1, [0, n], [0, n]))


@pytest.mark.parametrize('n_q', [2, 200])
@pytest.mark.parametrize('softcap', [0.01, 3.0, 1e4, 1e7])
def test_attention_cap_far_from_the_scores(cuda_device, n_q, softcap):
    """Caps far below the scores (all of them at the cap) and far above: tanh(z / cap) * cap keeps the relative
    accuracy of 32 bits for small z / cap too, so the bound is the uncapped one's and 2^-20 of min(|z|, cap)."""
    from musc_b200 import ops
    q, k, v = _random_qkv(cuda_device, n_q, 700, 2, 1, 64, torch.float16, 31, False)
    q = q * 3
    offsets = dict(offsets=_i32([0, n_q], cuda_device), kv_offsets=_i32([0, 700], cuda_device))
    got = ops.attention_masked(q, k, v, 2, 1, softcap=softcap, **offsets)
    want, _ = _reference(q, k, v, 2, 1, [0, n_q], [0, 700], softcap=softcap)
    _, tol = _reference(q, k, v, 2, 1, [0, n_q], [0, 700])
    mean = torch.cat([_reference(q[:, h * 64:(h + 1) * 64], k, v.abs(), 1, 1, [0, n_q], [0, 700], softcap=softcap)[0]
                      for h in range(2)], 1)
    size = float((q.double().view(-1, 64) @ k.double().T / 8).abs().max())
    # the rounding of P and of the result, on the capped scores' own average
    tol = torch.maximum(tol, 2.0 ** -11 * (mean + want.abs()) * (1 + 2.0 ** -6) + 2.0 ** -24)
    tol = tol + 2 * mean * ((64 + 8) * 2.0 ** -24 * 8 * size + 2.0 ** -18 + min(size, softcap) * 2.0 ** -20)
    _assert_close(got, want, tol)


def test_attention_captured_and_on_other_streams(cuda_device):
    """Replays of two graphs and eager calls on two streams give the eager result bit for bit."""
    from musc_b200 import ops
    calls = []
    for n, heads in ((1, 2), (300, 2)):
        q, k, v = _random_qkv(cuda_device, n, 900, heads, 1, 64, torch.float16, 14 + n, False)
        kwargs = dict(offsets=_i32([0, n], cuda_device), kv_offsets=_i32([0, 900], cuda_device), causal=True)
        calls.append(lambda q=q, k=k, v=v, heads=heads, kwargs=kwargs: ops.attention_masked(q, k, v, heads, 1, **kwargs))
    want = [c() for c in calls]
    graphs = []
    for c in calls:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = c()
        graphs.append((g, out))
    streams = [torch.cuda.Stream(cuda_device) for _ in calls]
    torch.cuda.synchronize()
    eager = []
    for _ in range(5):
        for (g, _), s, c in zip(graphs, streams, calls):
            with torch.cuda.stream(s):
                g.replay()
                eager.append(c())
    torch.cuda.synchronize()
    for (_, out), w in zip(graphs, want):
        assert torch.equal(out, w)
    for i, e in enumerate(eager):
        assert torch.equal(e, want[i % 2])


def test_attention_refusals(cuda_device):
    from musc_b200 import ops
    q = torch.zeros(8, 128, dtype=torch.float16, device=cuda_device)
    off = _i32([0, 8], cuda_device)
    for bad, message in ((dict(offsets=off.long()), 'offsets'), (dict(offsets=off.cpu()), 'offsets'),
                         (dict(offsets=off, prefix=off), 'prefix'), (dict(offsets=off, prefix=off[:1]), 'causal'),
                         (dict(offsets=off, softcap=-1.0), 'softcap'), (dict(offsets=off, scale=0.0), 'scale'),
                         (dict(offsets=off, slopes=torch.ones(3, device=cuda_device)), 'slopes'),
                         (dict(), 'expected'), (dict(offsets=off, out=q), 'overlap'),
                         (dict(offsets=off, out=q.float()), 'out'), (dict(offsets=off[:0]), 'offsets')):
        with pytest.raises(ValueError, match=message):
            ops.attention_masked(q, q, q, 2, **bad)
    with pytest.raises(ValueError, match='float16'):
        ops.attention_masked(q, q.float(), q, 2, offsets=off)
    with pytest.raises(ValueError, match='head_dim'):
        ops.attention_masked(q, q, q, 4, offsets=off)
    with pytest.raises(ValueError, match='multiple'):
        ops.attention_masked(q, q, q, 2, 3, offsets=off)
    with pytest.raises(ValueError, match='gradient'):
        ops.attention_masked(q.requires_grad_(), q, q, 2, offsets=off)
    with torch.no_grad():
        ops.attention_masked(q, q, q, 2, offsets=off)
    with pytest.raises(ValueError, match='16-byte|multiples'):
        odd = torch.zeros(8 * 129, dtype=torch.float16, device=cuda_device)
        ops.attention_masked(odd[1:1 + 8 * 128].view(8, 128), q.detach(), q.detach(), 2, offsets=off)


# ----------------------------------------------------------------------------- rotary
def _turned(x, heads, positions, frequencies, axis, adjacent):
    n = frequencies.numel()
    x = x.double().reshape(*x.shape[:-1], heads, -1)
    angle = positions.double()[..., axis.long()] * frequencies.double()
    c, s = torch.cos(angle)[..., None, :], torch.sin(angle)[..., None, :]
    i0 = torch.arange(n, device=x.device) * (2 if adjacent else 1)
    i1 = i0 + (1 if adjacent else n)
    y, size = x.clone(), torch.zeros_like(x)
    y[..., i0] = x[..., i0] * c - x[..., i1] * s
    y[..., i1] = x[..., i1] * c + x[..., i0] * s
    size[..., i0] = size[..., i1] = x[..., i0].abs() + x[..., i1].abs()
    return y.flatten(-2), size.flatten(-2)


@pytest.mark.parametrize('dtype', [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize('tokens,heads,kv_heads,d,sections,adjacent', [
    (1, 1, 1, 64, [32], False), (5, 3, 1, 64, [16, 16], True), (1000, 4, 2, 128, [16, 24, 24], False),
    (33, 2, 2, 80, [20, 20], False), (7, 2, 1, 80, [13, 11], True), (9, 1, 1, 2, [1], False), (4, 2, 2, 6, [1, 1], True),
    (300, 5, 5, 96, [8, 8, 8], False), (20, 2, 1, 512, [256], True), (3000, 16, 16, 64, [16, 16], False)])
def test_rotary_matches_formula(cuda_device, tokens, heads, kv_heads, d, sections, adjacent, dtype):
    from musc_b200 import ops
    g = torch.Generator(device=cuda_device).manual_seed(tokens + d)
    qk = torch.randn(tokens, (heads + kv_heads) * d, generator=g, device=cuda_device).to(dtype)
    q, k = qk[:, :heads * d], qk[:, heads * d:]
    f, a = ops.rotary_frequencies(sections, device=cuda_device)
    positions = torch.randint(-5, 300_000, (tokens, len(sections)), generator=g, device=cuda_device).to(torch.int32)
    u = _unit(dtype)
    for pos in (positions, positions.float() / 7):
        got = ops.rotary(q, k, pos, f, a, heads, kv_heads, adjacent)
        for out, x, h in zip(got, (q, k), (heads, kv_heads)):
            want, size = _turned(x, h, pos, f, a, adjacent)
            _assert_close(out, want, size * 2.0 ** -21 + want.abs() * u * (size > 0) + 2.0 ** -25)
    want = ops.rotary(q, k, positions, f, a, heads, kv_heads, adjacent)
    ops.rotary(q, k, positions, f, a, heads, kv_heads, adjacent, out=(q, k))          # in place
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])


def test_rotary_forms(cuda_device):
    from musc_b200 import ops
    g = torch.Generator(device=cuda_device).manual_seed(2)
    f, a = ops.rotary_frequencies([16, 16], device=cuda_device)
    x = torch.randn(3, 50, 128, generator=g, device=cuda_device)
    pos = torch.randint(0, 40, (3, 50, 2), generator=g, device=cuda_device).to(torch.int32)
    q, k = ops.rotary(x, None, pos, f, a, 2)
    assert k is None and torch.equal(q.view(150, 128), ops.rotary(x.view(150, 128), None, pos.view(150, 2), f, a, 2)[0])
    # rows that start off a 16-byte boundary take the narrow path, to the same values
    buf = torch.empty(150 * 131 + 1, device=cuda_device)
    odd = buf[1:].as_strided((150, 128), (131, 1))
    odd.copy_(x.view(150, 128))
    assert torch.equal(ops.rotary(odd, None, pos.view(150, 2), f, a, 2)[0], q.view(150, 128))
    # an axis that does not exist is taken as the nearest, positions of zero turn nothing
    far = ops.rotary(x, None, pos, f, torch.full_like(a, 9), 2)[0]
    assert torch.equal(far, ops.rotary(x, None, pos, f, torch.ones_like(a), 2)[0])
    assert torch.equal(ops.rotary(x, None, torch.zeros_like(pos), f, a, 2)[0], x)
    assert ops.rotary(x[:0], None, pos[:0], f, a, 2)[0].shape == (0, 50, 128)
    for bad, message in ((dict(positions=pos.long()), 'positions'), (dict(positions=pos[:2]), 'positions'),
                         (dict(axis=a.long()), 'axis'), (dict(frequencies=f.double()), 'frequencies'),
                         (dict(heads=3), 'heads'), (dict(heads=8), 'pairs'), (dict(out=(x[:, :1], None)), 'out'),
                         (dict(k=x[..., :64]), 'expected')):
        args = dict(q=x, k=None, positions=pos, frequencies=f, axis=a, heads=2)
        args.update(bad)
        with pytest.raises(ValueError, match=message):
            ops.rotary(**args)
    with pytest.raises(ValueError, match='gradient'):
        ops.rotary(x.clone().requires_grad_(), None, pos, f, a, 2)


# ----------------------------------------------------------------------------- norm
def _normed(x, delta, w, eps):
    h = x.double() if delta is None else (x.float() + delta.float()).double()
    return h * torch.rsqrt(h.square().mean(-1, keepdim=True) + eps) * w.double()


@pytest.mark.parametrize('x_dtype', [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize('delta_dtype', [torch.float32, torch.float16, torch.bfloat16, None])
@pytest.mark.parametrize('out_dtype', [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize('rows,c', [(1, 1), (3, 7), (5, 1024), (4, 1025), (2, 1480), (3, 4096), (1, 32768), (2, 20001)])
def test_norm_matches_formula(cuda_device, rows, c, x_dtype, delta_dtype, out_dtype):
    from musc_b200 import ops
    g = torch.Generator(device=cuda_device).manual_seed(rows + c)
    x = (3 * torch.randn(rows, c, generator=g, device=cuda_device)).to(x_dtype)
    delta = torch.randn(rows, c, generator=g, device=cuda_device).to(delta_dtype) if delta_dtype else None
    w = 1 + 0.2 * torch.randn(c, generator=g, device=cuda_device)
    want_x = x if delta is None else (x.float() + delta.float()).to(x_dtype)
    want = _normed(x, delta, w, 1e-5)
    x = x.clone()
    got = ops.add_rmsnorm(x, delta, w, 1e-5, out_dtype)
    assert torch.equal(x, want_x)
    _assert_close(got, want, want.abs() * (2.0 ** -18 + _unit(out_dtype)) + 2.0 ** -25)


@pytest.mark.parametrize('group', [0, 32, 64, 128, 256])
@pytest.mark.parametrize('rows,c', [(1, 1), (3, 100), (6, 1024), (5, 1480), (2, 4096), (3, 5003), (1, 32768)])
def test_norm_eight_bits(cuda_device, rows, c, group):
    from musc_b200 import ops
    g = torch.Generator(device=cuda_device).manual_seed(rows + c + group)
    x = torch.randn(rows, c, generator=g, device=cuda_device) * torch.exp(torch.randn(rows, c, generator=g, device=cuda_device))
    x[-1, : c // 2] = 0
    delta = torch.zeros(rows, c, dtype=torch.bfloat16, device=cuda_device)
    w = 1 + 0.2 * torch.randn(c, generator=g, device=cuda_device)
    want = _normed(x, None, w, 1e-6)
    values, scales = ops.add_rmsnorm(x, delta, w, 1e-6, torch.float8_e4m3fn, group=group)
    size = group or c
    n = -(-c // size)
    assert values.shape == (rows, c) and scales.shape == (rows, n)
    padded = torch.zeros(rows, n * size, dtype=torch.float64, device=cuda_device)
    padded[:, :c] = want
    top = padded.view(rows, n, size).abs().amax(-1) / 448
    _assert_close(scales, top, top * 2.0 ** -17 + 2.0 ** -125)
    want = want / scales.double().repeat_interleave(size, 1)[:, :c]
    _assert_close(values.float(), want, want.abs() * (2.0 ** -4 + 2.0 ** -16) + 2.0 ** -10)


def test_norm_edges(cuda_device):
    from musc_b200 import ops
    w = torch.ones(256, device=cuda_device)
    x = torch.zeros(4, 256, device=cuda_device)
    x[1, 7], x[2, 9], x[3] = math.nan, math.inf, 1e-20
    values, scales = ops.add_rmsnorm(x.clone(), None, w, 1e-6, torch.float8_e4m3fn)
    assert bool((values[0].float() == 0).all()) and float(scales[0]) == 2.0 ** -126       # a row of zeros
    assert torch.isnan(values[1].float()).all()                                            # NaN spreads over its row only
    assert torch.isnan(values[2].float()[9]) and bool((values[2].float()[:9] == 0).all())
    torch.testing.assert_close(values[3].float() * scales[3], torch.full((256,), 1e-17, device=cuda_device), rtol=0.07, atol=0)
    # rows a stride apart, off 16-byte boundaries; rows of nothing
    buf = torch.randn(10, 301, device=cuda_device)
    view = buf[:, 1:257]
    want = _normed(view, None, w, 1e-6)
    keep = buf.clone()
    out = torch.empty(10, 300, dtype=torch.float16, device=cuda_device)[:, 3:259]
    ops.add_rmsnorm(view, torch.ones(10, 256, dtype=torch.float16, device=cuda_device), w, out=out)
    assert torch.equal(buf[:, :1], keep[:, :1]) and torch.equal(buf[:, 257:], keep[:, 257:])
    want = _normed(keep[:, 1:257], torch.ones(10, 256, device=cuda_device), w, 1e-6)
    _assert_close(out, want, want.abs() * (2.0 ** -18 + 2.0 ** -11) + 2.0 ** -25)
    assert ops.add_rmsnorm(x[:0], None, w).shape == (0, 256)
    three = torch.randn(2, 3, 256, device=cuda_device)
    v, s = ops.add_rmsnorm(three, None, w, out_dtype=torch.float8_e4m3fn, group=64)
    assert v.shape == (2, 3, 256) and s.shape == (2, 3, 4)
    for bad, message in ((dict(weight=w.half()), 'weight'), (dict(delta=x[:2]), 'delta'), (dict(out_dtype=torch.int8), 'out_dtype'),
                         (dict(group=64), 'group'), (dict(out_dtype=torch.float8_e4m3fn, group=100), 'group'),
                         (dict(out=x), 'out'), (dict(scales=w), 'scales'), (dict(eps=-1.0), 'eps'),
                         (dict(x=three[:, :2]), 'contiguous')):
        args = dict(x=x, delta=None, weight=w)
        args.update(bad)
        with pytest.raises(ValueError, match=message):
            ops.add_rmsnorm(**args)
    with pytest.raises(ValueError, match='gradient'):
        ops.add_rmsnorm(x, None, w.clone().requires_grad_())


# ----------------------------------------------------------------------------- together
def test_block_of_packed_images(cuda_device):
    """One block over three images of differing grids packed into one sequence: norm, projection, two-axis
    rotary, attention within each image, projection, norm in 8 bits -- each step against its formula on
    its own inputs, then the whole block replayed from a graph, bit for bit."""
    from musc_b200 import ops
    grids, heads, kv_heads, d, c = [(9, 14), (1, 1), (20, 11)], 4, 2, 64, 256
    g = torch.Generator(device=cuda_device).manual_seed(21)
    off = _starts([h * w for h, w in grids])
    t = off[-1]
    positions = torch.tensor([[i // w, i % w] for h, w in grids for i in range(h * w)], dtype=torch.int32, device=cuda_device)
    offsets = _i32(off, cuda_device)
    f, a = ops.rotary_frequencies([16, 16], device=cuda_device)
    x0 = torch.randn(t, c, generator=g, device=cuda_device)
    branch = (0.3 * torch.randn(t, c, generator=g, device=cuda_device)).half()
    w1, w2 = (1 + 0.1 * torch.randn(c, generator=g, device=cuda_device) for _ in range(2))
    w_qkv = (torch.randn((heads + 2 * kv_heads) * d, c, generator=g, device=cuda_device) * c ** -0.5).half()
    w_out = (torch.randn(c, heads * d, generator=g, device=cuda_device) * c ** -0.5).half()

    def block(x):
        steps = dict(x_in=x.clone(), h=ops.add_rmsnorm(x, branch, w1))
        steps['qkv'] = torch.nn.functional.linear(steps['h'], w_qkv)
        q, k, v = steps['qkv'].split([heads * d, kv_heads * d, kv_heads * d], 1)
        steps['q'], steps['k'] = ops.rotary(q, k, positions, f, a, heads, kv_heads)
        steps['a'] = ops.attention_masked(steps['q'], steps['k'], v, heads, kv_heads, offsets=offsets)
        steps['o'] = torch.nn.functional.linear(steps['a'], w_out)
        steps['x_mid'] = x.clone()
        steps['y'], steps['s'] = ops.add_rmsnorm(x, steps['o'], w2, out_dtype=torch.float8_e4m3fn, group=128)
        return steps

    s = block(x0.clone())
    want = _normed(s['x_in'], branch, w1, 1e-6)
    _assert_close(s['h'], want, want.abs() * (2.0 ** -18 + 2.0 ** -11) + 2.0 ** -25)
    q, k, v = s['qkv'].split([heads * d, kv_heads * d, kv_heads * d], 1)
    for out, x, n in ((s['q'], q, heads), (s['k'], k, kv_heads)):
        want, size = _turned(x, n, positions, f, a, False)
        _assert_close(out, want, size * 2.0 ** -21 + want.abs() * 2.0 ** -11 + 2.0 ** -25)
    _assert_close(s['a'], *_reference(s['q'], s['k'], v, heads, kv_heads, off, off))
    want = _normed(s['x_mid'], s['o'], w2, 1e-6) / s['s'].double().repeat_interleave(128, 1)
    _assert_close(s['y'].float(), want, want.abs() * (2.0 ** -4 + 2.0 ** -16) + 2.0 ** -10)

    x = x0.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = block(x)
    x.copy_(x0)
    graph.replay()
    torch.cuda.synchronize()
    for name in s:
        assert torch.equal(out[name].float(), s[name].float()), name
    ops.check_device_error(cuda_device)
