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

from test_gpu_block_ops import _assert_close, _i32, _normed, _of_heads, _random_qkv, _reference, _starts

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


def test_empty_batches(cuda_device):
    from musc_b200 import ops
    x = torch.zeros(3, 70, 128, dtype=torch.float16, device=cuda_device)
    assert ops.attention_masked(x[:0], x[:0], x[:0], 2, causal=True).shape == (0, 70, 128)
    assert ops.attention_masked(x[:, :0], x, x, 2).shape == (3, 0, 128)
    x[:] = 1
    assert bool((ops.attention_masked(x, x[:, :0], x[:, :0], 2) == 0).all())


# ----------------------------------------------------------------------------- the row kernel's sums in a workspace
# rows and keys of the documents, heads, kv_heads, head_dim, splits (above, up to)
LONG = [
    ([(4, 30_000), (4, 30_000)], 8, 1, 128, (8, 32)),
    ([(3, 20_011), (0, 5), (6, 40_000)], 2, 1, 64, (8, 32)),
    ([(10, 100_000)], 4, 2, 64, (32, 64)),
    ([(1, 100_000)], 1, 1, 64, (32, 64)),
    ([(9, 200_003), (7, 197_001)], 6, 2, 128, (32, 64)),
]


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16])
@pytest.mark.parametrize('options', [{}, dict(causal=True, softcap=9.0, bias=True), dict(causal=True, prefix=True)])
@pytest.mark.parametrize('case', range(len(LONG)))
def test_rows_over_long_keys_in_many_splits(cuda_device, case, options, dtype):
    """More splits than a cluster joins: unnormalised sums through the workspace.  Scores grow along the keys, so that
    the splits' maxima differ; a document without keys gives zeros."""
    from musc_b200 import ops
    docs, heads, kv_heads, d, (above, most) = LONG[case]
    options, empty = dict(options), (3, 0)
    docs = docs + [empty]
    q_off, k_off = _starts([n for n, _ in docs]), _starts([m for _, m in docs])
    q, k, v = _random_qkv(cuda_device, q_off[-1], k_off[-1], heads, kv_heads, d, dtype, 200 + case, False)
    k = (k.float() * torch.linspace(0.2, 2.0, k_off[-1], device=cuda_device)[:, None]).to(dtype)
    slopes = 2.0 ** (-6 - torch.arange(heads, device=cuda_device).float()) if options.pop('bias', False) else None
    prefix = [m - n // 2 for n, m in docs] if options.pop('prefix', False) else None
    kernel, splits = _plan(q_off[-1], k_off[-1], len(docs), heads, kv_heads, d)
    assert kernel == ROWS and above < splits <= most
    got = ops.attention_masked(q, k, v, heads, kv_heads, offsets=_i32(q_off, cuda_device), kv_offsets=_i32(k_off, cuda_device),
                               prefix=None if prefix is None else _i32(prefix, cuda_device), slopes=slopes, **options)
    _assert_close(got, *_reference(q, k, v, heads, kv_heads, q_off, k_off, prefix=prefix, slopes=slopes, **options))
    assert bool((got[q_off[-2]:] == 0).all())


@pytest.mark.parametrize('poison', [math.nan, math.inf])
@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16])
@pytest.mark.parametrize('case', [0, 2])
def test_rows_over_long_keys_last_values_not_finite(cuda_device, case, dtype, poison):
    """A value at the last key that is not finite reaches the rows that see it: their split is taken again key by key
    and joined with the other splits' sums."""
    from musc_b200 import ops
    docs, heads, kv_heads, d, (above, most) = LONG[case]
    q_off, k_off = _starts([n for n, _ in docs]), _starts([m for _, m in docs])
    kernel, splits = _plan(q_off[-1], k_off[-1], len(docs), heads, kv_heads, d)
    assert kernel == ROWS and above < splits <= most
    q, k, v = _random_qkv(cuda_device, q_off[-1], k_off[-1], heads, kv_heads, d, dtype, 220 + case, False)
    clean = v.clone()
    v[k_off[1] - 2, 5] = poison                               # seen by the last two rows of the first document
    got = ops.attention_masked(q, k, v, heads, kv_heads, offsets=_i32(q_off, cuda_device), kv_offsets=_i32(k_off, cuda_device),
                               causal=True)
    want, tol = _reference(q, k, clean, heads, kv_heads, q_off, k_off, causal=True)
    hit = torch.zeros(got.shape, dtype=torch.bool, device=cuda_device)
    hit[q_off[1] - 2:q_off[1], [h * d + 5 for h in range(heads // kv_heads)]] = True
    assert not bool(got[hit].isfinite().any())
    others = ~hit
    others[q_off[1] - 2:q_off[1]] = False                     # (their bound would need the poisoned row's other values)
    _assert_close(got[others], want[others], tol[others])
    assert bool(got[~hit].isfinite().all())


@pytest.mark.parametrize('kernel,n_q,n_k,heads,d', [(ROWS, 1, 100_000, 2, 64), (ROWS, 2, 60_000, 8, 128), (ROWS, 2, 3000, 4, 64),
                                                    (TILES, 300, 9000, 4, 64), (TILES, 300, 500, 96, 128)])
def test_keys_of_minus_infinity(cuda_device, kernel, n_q, n_k, heads, d):
    """Visible scores of -infinity weigh nothing, in the middle of a split or in all of one; a row that has no other
    score is 0 / 0."""
    from musc_b200 import ops
    q, k, v = _random_qkv(cuda_device, n_q, n_k, heads, 1, d, torch.bfloat16, 61, False)
    q[:, ::d] = 1.0
    first = n_k * 3 // 5
    k[:first, 0] = -math.inf
    assert _plan(n_q, n_k, 1, heads, 1, d)[0] == kernel
    offsets = dict(offsets=_i32([0, n_q], cuda_device), kv_offsets=_i32([0, n_k], cuda_device))
    got = ops.attention_masked(q, k, v, heads, 1, **offsets)
    _assert_close(got, *_reference(q, k[first:], v[first:], heads, 1, [0, n_q], [0, n_k - first]))
    k[:, 0] = -math.inf
    assert bool(ops.attention_masked(q, k, v, heads, 1, **offsets).isnan().all())


def test_splits_captured_and_on_other_streams(cuda_device):
    """Calls that need a workspace, of both kernels: replays of their graphs and eager calls on two streams at once
    give the eager result bit for bit."""
    from musc_b200 import ops
    calls = []
    for kernel, above, n, keys, docs, heads, kv_heads, d in ((ROWS, 8, 8, 40_000, 2, 8, 1, 128), (TILES, 1, 300, 9000, 1, 4, 2, 64)):
        got, splits = _plan(n, keys, docs, heads, kv_heads, d, True)
        assert got == kernel and splits > above
        q, k, v = _random_qkv(cuda_device, n, keys, heads, kv_heads, d, torch.float16, 62 + n, False)
        kwargs = dict(offsets=_i32([n * i // docs for i in range(docs + 1)], cuda_device),
                      kv_offsets=_i32([keys * i // docs for i in range(docs + 1)], cuda_device), causal=True)
        calls.append(lambda q=q, k=k, v=v, h=heads, hk=kv_heads, kwargs=kwargs: ops.attention_masked(q, k, v, h, hk, **kwargs))
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
    for i in range(6):
        for j, (s, c) in enumerate(zip(streams, calls)):
            with torch.cuda.stream(s):
                graphs[(i + j) % 2][0].replay()   # each graph on both streams in turn, never on both at once
                eager.append((j, c()))
        torch.cuda.synchronize()
    for (_, out), w in zip(graphs, want):
        assert torch.equal(out, w)
    for j, e in eager:
        assert torch.equal(e, want[j])


# ----------------------------------------------------------------------------- the tile kernel's lookup of documents
def _lengths(kind):
    g = torch.Generator().manual_seed(63)
    if kind == '8 long':              # ending at and beside tile borders
        return [256, 255, 257, 512, 1, 64, 65, 700]
    if kind == '32':                  # the most documents that one warp looks up
        return [70 + 5 * (i % 3) for i in range(30)] + [900, 0]
    if kind == '33':
        n = torch.randint(1, 90, (33,), generator=g)
        n[20] = 1500
    elif kind == '60':
        n = torch.randint(0, 160, (60,), generator=g)
        n[::9] += 300
        n[5] = n[6] = 0
    elif kind == '1024':              # the most that are looked up in shared memory: long, short and empty ones
        n = torch.randint(0, 41, (1024,), generator=g)
        n[torch.rand(1024, generator=g) < 0.15] += 420
        n[torch.rand(1024, generator=g) < 0.1] = 0
    elif kind == '1100':
        n = torch.randint(8, 28, (1100,), generator=g)
    else:                             # '40 short': tiles cut from the packed rows
        n = torch.randint(0, 30, (40,), generator=g)
    return n.tolist()


@pytest.mark.parametrize('causal', [False, True])
@pytest.mark.parametrize('kind,heads,d', [('8 long', 16, 64), ('8 long', 8, 128), ('32', 16, 64), ('33', 16, 64), ('33', 8, 128),
                                          ('60', 8, 64), ('1024', 2, 64), ('1100', 8, 64), ('40 short', 160, 64)])
def test_tiles_of_many_documents(cuda_device, kind, heads, d, causal):
    """Row tiles of many documents, packed rows before the first and behind the last one left alone."""
    from musc_b200 import ops
    lens = _lengths(kind)
    off = [13 + o for o in _starts(lens)]
    rows, kv_heads = off[-1] + 30, heads // 2
    assert _plan(rows, rows, len(lens), heads, kv_heads, d, causal)[0] == TILES
    q, k, v = _random_qkv(cuda_device, rows, rows, heads, kv_heads, d, torch.bfloat16, 64, True)
    out = torch.full_like(q, 3.0)
    ops.attention_masked(q, k, v, heads, kv_heads, offsets=_i32(off, cuda_device), causal=causal, out=out)
    assert bool((out[:13] == 3).all()) and bool((out[off[-1]:] == 3).all())
    first = 0
    while first < len(lens):              # documents together that have up to 4000 rows
        last = first + 1
        while last < len(lens) and off[last + 1] - off[first] <= 4000:
            last += 1
        a, b = off[first], off[last]
        part = [o - a for o in off[first:last + 1]]
        _assert_heads(out[a:b], q[a:b], k[a:b], v[a:b], heads, kv_heads, part, part, causal=causal,
                      rows=torch.ones(b - a, dtype=torch.bool, device=cuda_device))
        first = last


@pytest.mark.parametrize('length,heads', [(17, 512), (100, 64), (256, 16), (300, 16), (515, 16)])
def test_tiles_of_batches_of_one_length(cuda_device, length, heads):
    from musc_b200 import ops
    kv_heads = heads // 2
    assert _plan(5 * length, 5 * length, 5, heads, kv_heads, 64, True, (length, length))[0] == TILES
    q, k, v = _random_qkv(cuda_device, 5 * length, 5 * length, heads, kv_heads, 64, torch.float16, 65, True)
    view = lambda t: t.unflatten(0, (5, length))
    got = ops.attention_masked(view(q), view(k), view(v), heads, kv_heads, causal=True, softcap=20.0)
    off = _starts([length] * 5)
    _assert_heads(got.flatten(0, 1), q, k, v, heads, kv_heads, off, off, causal=True, softcap=20.0)


@pytest.mark.parametrize('documents', [3, 40])
def test_tiles_disordered_offsets_stay_inside(cuda_device, documents):
    """Offsets that fall, repeat or leave the tensors: results are undefined, accesses are not."""
    from musc_b200 import ops
    n, heads, kv_heads = 3000, 32, 16
    assert _plan(n, n, documents, heads, kv_heads, 64, True)[0] == TILES
    q, k, v = _random_qkv(cuda_device, n, n, heads, kv_heads, 64, torch.float16, 66, True)
    top = (1 << 31) - 1
    g = torch.Generator().manual_seed(67)
    anywhere = lambda lo, hi: torch.randint(lo, hi, (documents + 1,), generator=g).tolist()
    sets = [(anywhere(0, n + 1), anywhere(0, n + 1)), (anywhere(-top, top), anywhere(-top, top)),
            (sorted(anywhere(0, n), reverse=True), sorted(anywhere(0, n))), ([n] * (documents + 1), [0] * (documents + 1)),
            ([-top - 1, top] * ((documents + 1) // 2) + [-5] * ((documents + 1) % 2), anywhere(0, n))]
    for q_off, k_off in sets:
        for causal in (False, True):
            ops.attention_masked(q, k, v, heads, kv_heads, offsets=_i32(q_off, cuda_device), kv_offsets=_i32(k_off, cuda_device),
                                 kv_lengths=_i32(anywhere(-9, n)[1:], cuda_device), causal=causal)
    torch.cuda.synchronize()
    ops.check_device_error(cuda_device)
    got = ops.attention_masked(q, k, v, heads, kv_heads, offsets=_i32([0, n], cuda_device))
    _assert_heads(got, q, k, v, heads, kv_heads, [0, n], [0, n])


@pytest.mark.parametrize('heads,d', [(64, 64), (16, 128)])
def test_tiles_key_offsets_past_the_tensor(cuda_device, heads, d):
    from musc_b200 import ops
    n, kv_heads = 500, heads // 2
    assert _plan(n, 600, 1, heads, kv_heads, d)[0] == TILES
    q, k, v = _random_qkv(cuda_device, n, 600, heads, kv_heads, d, torch.float16, 68, False)
    got = ops.attention_masked(q, k, v, heads, kv_heads, offsets=_i32([0, n], cuda_device),
                               kv_offsets=_i32([-50, 100_000], cuda_device), kv_lengths=_i32([1 << 30], cuda_device))
    _assert_heads(got, q, k, v, heads, kv_heads, [0, n], [0, 600])


# ----------------------------------------------------------------------------- the tile kernel's masks and scores
@pytest.mark.parametrize('d,dtype', [(64, torch.float16), (128, torch.bfloat16)])
@pytest.mark.parametrize('poison', [math.nan, math.inf, -math.inf])
def test_tiles_masked_values_do_not_leak(cuda_device, poison, d, dtype):
    """Keys and values that a row does not see may hold anything: later tokens of its own document, other
    documents in the same tile, the type's lowest value in scores."""
    from musc_b200 import ops
    heads, lens = 160, [150, 30, 200, 9]
    off = _starts(lens)
    assert _plan(off[-1], off[-1], 4, heads, heads, d, True)[0] == TILES
    q, k, v = _random_qkv(cuda_device, off[-1], off[-1], heads, heads, d, dtype, 69, False)
    late = [off[1] - 1, off[3] - 2]            # the last key of one document, the last but one of another
    k[late] = torch.finfo(dtype).min
    v[late] = poison
    clean_k, clean_v = k.clone(), v.clone()
    clean_k[late], clean_v[late] = 0, 0
    got = ops.attention_masked(q, k, v, heads, offsets=_i32(off, cuda_device), causal=True)
    clean = torch.ones(off[-1], dtype=torch.bool, device=cuda_device)
    clean[off[1] - 1], clean[off[3] - 2:off[3]] = False, False
    _assert_heads(got, q, clean_k, clean_v, heads, heads, off, off, causal=True, rows=clean)
    # whole documents: only the poisoned ones are touched
    got = ops.attention_masked(q, k, v, heads, offsets=_i32(off, cuda_device))
    clean[:off[1]], clean[off[2]:off[3]] = False, False
    _assert_heads(got, q, clean_k, clean_v, heads, heads, off, off, rows=clean)


def test_tiles_visible_nan_and_infinity(cuda_device):
    """A value that a row does see reaches it."""
    from musc_b200 import ops
    heads = 128
    assert _plan(300, 300, 1, heads, heads, 64, True)[0] == TILES
    q, k, v = _random_qkv(cuda_device, 300, 300, heads, heads, 64, torch.float16, 70, False)
    k = k * 0.1
    v[280, 3::64], v[40, 5::64] = math.nan, math.inf
    got = ops.attention_masked(q, k, v, heads, offsets=_i32([0, 300], cuda_device), causal=True)
    assert torch.isnan(got[280:, 3::64]).all() and torch.isfinite(got[:280, 3::64]).all()
    assert torch.isinf(got[40:, 5::64]).all() and torch.isfinite(got[:40, 5::64]).all()
    q[7] = math.nan
    got = ops.attention_masked(q, k, v, heads, offsets=_i32([0, 300], cuda_device), causal=True)
    assert torch.isnan(got[7]).all() and torch.isfinite(got[:7]).all() and torch.isfinite(got[8:40]).all()


@pytest.mark.parametrize('d', [64, 128])
def test_tiles_leave_rows_outside_documents(cuda_device, d):
    """Rows outside every document are not written: one document, and tiles that documents begin themselves."""
    from musc_b200 import ops
    heads = 64
    for lens in ([400], [300, 0, 290], [33] * 12):
        off = [10 + o for o in _starts(lens)]
        rows = off[-1] + 10
        assert _plan(rows, rows, len(lens), heads, heads, d)[0] == TILES
        q, k, v = _random_qkv(cuda_device, rows, rows, heads, heads, d, torch.float16, 71, True)
        out = torch.full((rows, heads * d), 7.0, dtype=torch.float16, device=cuda_device)
        ops.attention_masked(q, k, v, heads, offsets=_i32(off, cuda_device), out=out)
        assert bool((out[:10] == 7).all()) and bool((out[off[-1]:] == 7).all())
        _assert_heads(out, q, k, v, heads, heads, off, off)


@pytest.mark.parametrize('d', [64, 128])
@pytest.mark.parametrize('causal', [False, True])
def test_tiles_cache_slots_ignore_what_lies_behind(cuda_device, causal, d):
    """Key slots used to differing lengths: what lies behind a slot's keys changes nothing, bit for bit."""
    from musc_b200 import ops
    n_q, heads, kv_heads, slot, lengths = 300, 32, 16, 333, [333, 301, 0, 128, 300]
    docs = len(lengths)
    assert _plan(docs * n_q, docs * slot, docs, heads, kv_heads, d, causal)[0] == TILES
    q, k, v = _random_qkv(cuda_device, docs * n_q, docs * slot, heads, kv_heads, d, torch.bfloat16, 72, False)
    q_off, k_off = _starts([n_q] * docs), _starts([slot] * docs)
    results = []
    for fill in (0.0, math.nan, math.inf):
        for i, n in enumerate(lengths):
            k[i * slot + n:(i + 1) * slot] = fill
            v[i * slot + n:(i + 1) * slot] = -fill
        results.append(ops.attention_masked(q, k, v, heads, kv_heads, offsets=_i32(q_off, cuda_device),
                                            kv_offsets=_i32(k_off, cuda_device), kv_lengths=_i32(lengths, cuda_device),
                                            causal=causal))
        if fill == 0.0:
            _assert_heads(results[0], q, k, v, heads, kv_heads, q_off, k_off, k_len=lengths, causal=causal)
    assert torch.equal(results[0], results[1]) and torch.equal(results[0], results[2])


@pytest.mark.parametrize('d', [64, 128])
@pytest.mark.parametrize('softcap', [0.01, 3.0, 1e4, 1e7])
def test_tiles_cap_far_from_the_scores(cuda_device, softcap, d):
    """As the test of few heads: the rounding of P and of the result on the capped scores' own average, a dot product off
    by (d + 8) 2^-24 of its terms' magnitudes, and 2^-20 of min(|z|, cap)."""
    from musc_b200 import ops
    n_q, n_k, heads = 200, 700, 64
    assert _plan(n_q, n_k, 1, heads, heads, d)[0] == TILES
    q, k, v = _random_qkv(cuda_device, n_q, n_k, heads, heads, d, torch.float16, 73, False)
    q = q * 3
    got = ops.attention_masked(q, k, v, heads, softcap=softcap, offsets=_i32([0, n_q], cuda_device),
                               kv_offsets=_i32([0, n_k], cuda_device))
    for h in (0, heads - 1):
        qh, kh, vh = (_of_heads(t, d, h, 1) for t in (q, k, v))
        want, _ = _reference(qh, kh, vh, 1, 1, [0, n_q], [0, n_k], softcap=softcap)
        mean, _ = _reference(qh, kh, vh.abs(), 1, 1, [0, n_q], [0, n_k], softcap=softcap)
        size = float((qh.double().abs() @ kh.double().abs().T).max()) * d ** -0.5
        top = float((qh.double() @ kh.double().T).abs().max()) * d ** -0.5
        tol = 2.0 ** -11 * (mean + want.abs()) * (1 + 2.0 ** -6) + 2.0 ** -24
        tol = tol + 2 * mean * ((d + 8) * 2.0 ** -24 * size + 2.0 ** -18 + min(top, softcap) * 2.0 ** -20)
        _assert_close(_of_heads(got, d, h, 1), want, tol)


# ----------------------------------------------------------------------------- writes that autograd has to know of
def _block_writes(dev):
    """(name, call, tensor that it writes): every block operator that writes a tensor of the caller's."""
    from musc_b200 import ops
    half = lambda *shape: torch.randn(*shape, device=dev).half()
    qkv = [half(2, 40, 128) for _ in range(3)]
    rows = [half(40, 128) for _ in range(3)]
    off = _i32([0, 40], dev)
    f, a = ops.rotary_frequencies([32], device=dev)
    pos = torch.arange(40, dtype=torch.int32, device=dev)[:, None]
    x, h, delta, w = torch.randn(40, 128, device=dev), half(40, 128), half(40, 128), torch.ones(128, device=dev)
    scales, eight = torch.zeros(40, 1, device=dev), torch.zeros(40, 128, device=dev).to(torch.float8_e4m3fn)
    o3, o2 = half(2, 40, 128), half(40, 128)
    return [
        ('attention out', lambda: ops.attention(*qkv, 2, out=o3), o3),
        ('attention_masked out', lambda: ops.attention_masked(*rows, 2, offsets=off, out=o2), o2),
        ('rotary q', lambda: ops.rotary(rows[0], rows[1], pos, f, a, 2, out=(rows[0], rows[1])), rows[0]),
        ('rotary k', lambda: ops.rotary(rows[0], rows[1], pos, f, a, 2, out=(rows[0], rows[1])), rows[1]),
        ('add_layernorm x', lambda: ops.add_layernorm(x, delta, w, w), x),
        ('add_layernorm out', lambda: ops.add_layernorm(x, None, w, w, out=o2), o2),
        ('add_rmsnorm x', lambda: ops.add_rmsnorm(x, delta, w), x),
        ('add_rmsnorm 16-bit x', lambda: ops.add_rmsnorm(h, delta, w), h),
        ('add_rmsnorm out', lambda: ops.add_rmsnorm(x, None, w, out=o2), o2),
        ('add_rmsnorm scales', lambda: ops.add_rmsnorm(x, None, w, out_dtype=torch.float8_e4m3fn, out=eight, scales=scales), scales),
    ]


@pytest.mark.parametrize('which', range(10))
def test_writes_reach_autograd(cuda_device, which):
    """A tensor that a backward pass still needs and a block operator then overwrites is noticed by it, also where
    the operator was given a view."""
    name, call, written = _block_writes(cuda_device)[which]
    factor = torch.ones_like(written).requires_grad_()
    y = (factor * written).sum()                              # keeps `written` for the gradient of `factor`
    with torch.no_grad():
        call()
    with pytest.raises(RuntimeError, match='inplace'):
        y.backward()
    with torch.inference_mode():
        _block_writes(cuda_device)[which][1]()                # tensors without a version


def test_reads_leave_versions_alone(cuda_device):
    from musc_b200 import ops
    x, w = torch.randn(40, 128, device=cuda_device), torch.ones(128, device=cuda_device)
    q = torch.randn(40, 128, device=cuda_device).half()
    versions = x._version, q._version
    ops.add_rmsnorm(x, None, w)
    ops.add_layernorm(x, None, w, w)
    ops.attention_masked(q, q, q, 2, offsets=_i32([0, 40], cuda_device))
    f, a = ops.rotary_frequencies([32], device=cuda_device)
    ops.rotary(q, q, torch.zeros(40, 1, dtype=torch.int32, device=cuda_device), f, a, 2)
    assert (x._version, q._version) == versions


def test_gradients_and_tangents_are_refused(cuda_device):
    """Inputs and given outputs that ask for a gradient, and inputs with a tangent of forward mode."""
    from torch.autograd import forward_ad

    from musc_b200 import ops
    q = torch.randn(40, 128, device=cuda_device).half()
    x, w = torch.randn(40, 128, device=cuda_device), torch.ones(128, device=cuda_device)
    off, pos = _i32([0, 40], cuda_device), torch.zeros(40, 1, dtype=torch.int32, device=cuda_device)
    f, a = ops.rotary_frequencies([32], device=cuda_device)
    asks = lambda t: t.clone().requires_grad_()
    scales = torch.zeros(40, 1, device=cuda_device)
    for call in (lambda t: ops.attention_masked(q, q, q, 2, offsets=off, out=t(q)),
                 lambda t: ops.attention_masked(q, t(q), q, 2, offsets=off),
                 lambda t: ops.rotary(q, q, pos, f, a, 2, out=(t(q), q.clone())),
                 lambda t: ops.rotary(q, None, pos.float(), t(f), a, 2),
                 lambda t: ops.add_rmsnorm(t(x), None, w), lambda t: ops.add_rmsnorm(x, t(q), w),
                 lambda t: ops.add_rmsnorm(x, None, w, out=t(q)),
                 lambda t: ops.add_rmsnorm(x, None, w, out_dtype=torch.float8_e4m3fn, scales=t(scales))):
        with pytest.raises(ValueError, match='gradient'):
            call(asks)
        with torch.no_grad():
            call(asks)
        with forward_ad.dual_level(), pytest.raises(ValueError, match='tangent'):
            call(lambda t: forward_ad.make_dual(t.clone(), torch.ones_like(t)))


# ----------------------------------------------------------------------------- the norm's walk over rows
# Rows enough that every CTA takes at least three (a warp's or its own) on 148 SMs with a last step that some leave out.
WALKS = [(60_001, 64), (60_001, 100), (20_003, 1480), (9001, 1481), (5003, 5000), (5003, 5003), (2501, 12_296), (2000, 20_001),
         (2003, 16_384), (1999, 32_768), (60_001, 1024)]


def _walk_inputs(rows, c, dev, x_dtype=torch.float32):
    g = torch.Generator(device=dev).manual_seed(rows + c)
    x = torch.randn(rows, c, generator=g, device=dev) * torch.exp(2 * torch.randn(rows, 1, generator=g, device=dev))
    delta = (0.5 * torch.randn(rows, c, generator=g, device=dev)).to(torch.bfloat16)
    w = 1 + 0.2 * torch.randn(c, generator=g, device=dev)
    return x.to(x_dtype), delta, w


@pytest.mark.parametrize('x_dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('rows,c', WALKS)
def test_norm_walk_over_rows(cuda_device, rows, c, x_dtype):
    from musc_b200 import ops
    x, delta, w = _walk_inputs(rows, c, cuda_device, x_dtype)
    want_x = (x.float() + delta.float()).to(x_dtype)
    want = _normed(x, delta, w, 1e-6)
    got = ops.add_rmsnorm(x, delta, w, 1e-6, torch.float16)
    assert torch.equal(x, want_x)
    _assert_close(got, want, want.abs() * (2.0 ** -18 + 2.0 ** -11) + 2.0 ** -25)


@pytest.mark.parametrize('group', [0, 32, 128, 256])
@pytest.mark.parametrize('rows,c', WALKS)
def test_norm_walk_over_rows_eight_bits(cuda_device, rows, c, group):
    from musc_b200 import ops
    x, delta, w = _walk_inputs(rows, c, cuda_device)
    want = _normed(x, delta, w, 1e-6)
    values, scales = ops.add_rmsnorm(x, delta, w, 1e-6, torch.float8_e4m3fn, group=group)
    size = group or c
    n = -(-c // size)
    top = torch.nn.functional.pad(want, (0, n * size - c)).view(rows, n, size).abs().amax(-1) / 448
    _assert_close(scales, top, top * 2.0 ** -17 + 2.0 ** -125)
    want /= scales.double().repeat_interleave(size, 1)[:, :c]
    _assert_close(values.float(), want, want.abs() * (2.0 ** -4 + 2.0 ** -16) + 2.0 ** -10)


# ----------------------------------------------------------------------------- given outputs with rows a stride apart
@pytest.mark.parametrize('kernel,above,n_q,n_k,docs,heads,kv_heads,d', [
    (ROWS, 0, 9, 700, 1, 8, 8, 64), (ROWS, 1, 4, 3000, 1, 4, 2, 64), (ROWS, 8, 8, 40_000, 2, 8, 1, 128),
    (TILES, 0, 500, 500, 1, 64, 64, 64), (TILES, 1, 300, 9000, 1, 4, 2, 64)])
def test_attention_into_columns(cuda_device, kernel, above, n_q, n_k, docs, heads, kv_heads, d):
    """q, k, v and out as columns of wider buffers, each with its own row stride; the columns beside out stay."""
    from musc_b200 import ops
    got, splits = _plan(n_q, n_k, docs, heads, kv_heads, d, True)
    assert got == kernel and splits > above
    g = torch.Generator(device=cuda_device).manual_seed(74)
    rand = lambda rows, width, extra: torch.randn(rows, width + extra, generator=g, device=cuda_device).half()
    q, k, v = rand(n_q, heads * d, 24)[:, 16:-8], rand(n_k, kv_heads * d, 8)[:, 8:], rand(n_k, kv_heads * d, 72)[:, :-72]
    buf = torch.full((n_q, heads * d + 40), 5.0, dtype=torch.float16, device=cuda_device)
    q_off, k_off = [n_q * i // docs for i in range(docs + 1)], [n_k * i // docs for i in range(docs + 1)]
    out = buf[:, 8:-32]
    assert ops.attention_masked(q, k, v, heads, kv_heads, offsets=_i32(q_off, cuda_device), kv_offsets=_i32(k_off, cuda_device),
                                causal=True, out=out) is out
    assert bool((buf[:, :8] == 5).all()) and bool((buf[:, -32:] == 5).all())
    _assert_heads(out, q, k, v, heads, kv_heads, q_off, k_off, causal=True)


@pytest.mark.parametrize('kernel,n_q,n_k,docs,heads,kv_heads,d', [
    (ROWS, 4, 5480, 4, 16, 16, 64), (ROWS, 8, 40_000, 2, 8, 1, 128), (ROWS, 9, 900, 3, 8, 2, 128), (TILES, 900, 900, 3, 64, 64, 64),
    (TILES, 300, 9000, 1, 4, 2, 64)])
def test_attention_repeats_itself(cuda_device, kernel, n_q, n_k, docs, heads, kv_heads, d):
    """The same call gives the same bits: no sum depends on the order in which CTAs run."""
    from musc_b200 import ops
    assert _plan(n_q, n_k, docs, heads, kv_heads, d, True)[0] == kernel
    q, k, v = _random_qkv(cuda_device, n_q, n_k, heads, kv_heads, d, torch.bfloat16, 75, False)
    offsets = dict(offsets=_i32([n_q * i // docs for i in range(docs + 1)], cuda_device),
                   kv_offsets=_i32([n_k * i // docs for i in range(docs + 1)], cuda_device))
    first = ops.attention_masked(q, k, v, heads, kv_heads, causal=True, softcap=30.0, **offsets)
    for _ in range(20):
        assert torch.equal(ops.attention_masked(q, k, v, heads, kv_heads, causal=True, softcap=30.0, **offsets), first)


# ----------------------------------------------------------------------------- far rows, many documents, many splits
@pytest.mark.parametrize('kernel,n_q,n_k,heads,d', [(ROWS, 6, 40, 2, 64), (TILES, 300, 290, 160, 64)])
def test_rows_whose_offsets_pass_32_bits(cuda_device, kernel, n_q, n_k, heads, d):
    """Queries, keys, values and outputs 2^31 elements and more from their first row."""
    from musc_b200 import ops
    assert _plan(n_q, n_k, 1, heads, heads, d, True)[0] == kernel
    size, width = (1 << 31) + (1 << 30), heads * d
    buf, into = (torch.empty(size, dtype=torch.bfloat16, device=cuda_device) for _ in range(2))
    far = lambda t, of: of.as_strided(t.shape, ((size - width) // t.shape[0] // 8 * 8, 1))
    q, k, v = _random_qkv(cuda_device, n_q, n_k, heads, heads, d, torch.bfloat16, 76, False)
    offsets = dict(offsets=_i32([0, n_q], cuda_device), kv_offsets=_i32([0, n_k], cuda_device), causal=True)
    for which in range(3):
        given = [q, k, v]
        given[which] = far(given[which], buf).copy_(given[which])
        out = ops.attention_masked(*given, heads, out=far(q, into), **offsets)
        _assert_heads(out.clone(), q, k, v, heads, heads, [0, n_q], [0, n_k], causal=True)


@pytest.mark.parametrize('most', [1, 6])
def test_rows_of_more_documents_than_a_warp_counts(cuda_device, most):
    """Above 1024 documents their rows are searched for; documents of no rows and of no keys among them."""
    from musc_b200 import ops
    docs, heads, d = 2000, 4, 128
    g = torch.Generator().manual_seed(77 + most)
    q_lens, k_lens = (torch.randint(0, n + 1, (docs,), generator=g).tolist() for n in (most, 60))
    q_off, k_off = [3 + o for o in _starts(q_lens)], _starts(k_lens)
    rows = q_off[-1] + 3
    assert _plan(rows, k_off[-1], docs, heads, 1, d, True)[0] == ROWS and (rows > docs) == (most > 1)
    q, k, v = _random_qkv(cuda_device, rows, k_off[-1], heads, 1, d, torch.float16, 78, False)
    out = torch.full_like(q, 4.0)
    ops.attention_masked(q, k, v, heads, 1, offsets=_i32(q_off, cuda_device), kv_offsets=_i32(k_off, cuda_device), causal=True, out=out)
    assert bool((out[:3] == 4).all()) and bool((out[-3:] == 4).all())
    for first in range(0, docs, 250):
        a, b, ka, kb = q_off[first], q_off[first + 250], k_off[first], k_off[first + 250]
        want, tol = _reference(q[a:b], k[ka:kb], v[ka:kb], heads, 1, [o - a for o in q_off[first:first + 251]],
                               [o - ka for o in k_off[first:first + 251]], causal=True)
        _assert_close(out[a:b], want, tol)


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16])
@pytest.mark.parametrize('poison', [0.0, math.nan])
@pytest.mark.parametrize('n_q,n_k,docs,kv_heads,d', [(300, 60_000, 1, 1, 64), (500, 90_000, 2, 2, 128)])
def test_tiles_over_long_keys_in_many_splits(cuda_device, n_q, n_k, docs, kv_heads, d, poison, dtype):
    """The tile kernel's most splits, with maxima that differ from split to split; a NaN in a value that only the last
    rows see stays with them."""
    from musc_b200 import ops
    heads = 2
    assert _plan(n_q, n_k, docs, heads, kv_heads, d, True) == (TILES, 32)
    q, k, v = _random_qkv(cuda_device, n_q, n_k, heads, kv_heads, d, dtype, 79, False)
    k = (k.float() * torch.linspace(0.2, 2.0, n_k, device=cuda_device)[:, None]).to(dtype)
    q_off, k_off = [n_q * i // docs for i in range(docs + 1)], [n_k * i // docs for i in range(docs + 1)]
    clean = v.clone()
    v[k_off[1] - 2, 5] += poison
    got = ops.attention_masked(q, k, v, heads, kv_heads, offsets=_i32(q_off, cuda_device), kv_offsets=_i32(k_off, cuda_device),
                               causal=True, softcap=20.0)
    want, tol = _reference(q, k, clean, heads, kv_heads, q_off, k_off, causal=True, softcap=20.0)
    hit = torch.zeros(got.shape, dtype=torch.bool, device=cuda_device)
    if poison:
        hit[q_off[1] - 2:q_off[1], [h * d + 5 for h in range(heads // kv_heads)]] = True
        assert bool(got[hit].isnan().all())
    _assert_close(got[~hit], want[~hit], tol[~hit])


@pytest.mark.parametrize('c', [1024, 1001, 8192])
def test_norm_and_rotary_of_far_rows(cuda_device, c):
    """Rows 2^31 elements and more from the first one give what they give near by, in place too."""
    from musc_b200 import ops
    n, size = 6, (1 << 31) + (1 << 30)
    bufs = [torch.empty(size, dtype=torch.bfloat16, device=cuda_device) for _ in range(2)]
    stride = (size - c) // n // 8 * 8
    far = lambda t, i: bufs[i].as_strided(t.shape, (stride, 1)).copy_(t)
    g = torch.Generator(device=cuda_device).manual_seed(80)
    x, delta = (torch.randn(n, c, generator=g, device=cuda_device).bfloat16() for _ in range(2))
    w = 1 + 0.2 * torch.randn(c, generator=g, device=cuda_device)
    near_x = x.clone()
    want = ops.add_rmsnorm(near_x, delta, w, out_dtype=torch.bfloat16)
    far_x = far(x, 0)
    assert torch.equal(ops.add_rmsnorm(far_x, far(delta, 1), w, out_dtype=torch.bfloat16), want) and torch.equal(far_x, near_x)
    out = far(torch.zeros_like(x), 1)
    ops.add_rmsnorm(near_x, None, w, out_dtype=torch.bfloat16, out=out)
    assert torch.equal(out, ops.add_rmsnorm(near_x, None, w, out_dtype=torch.bfloat16))
    if c % 64 == 0:
        f, a = ops.rotary_frequencies([16, 16], device=cuda_device)
        pos = torch.randint(0, 1000, (n, 2), generator=g, device=cuda_device).to(torch.int32)
        want, _ = ops.rotary(x, None, pos, f, a, c // 64)
        far_x = far(x, 0)
        ops.rotary(far_x, None, pos, f, a, c // 64, out=(far_x, None))
        assert torch.equal(far_x, want)
