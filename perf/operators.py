"""Measured cases of the encoder-block operators: masked attention, rotary positions over several
axes, and the residual add + root-mean-square norm.

``run`` computes an operator in its plain form (elementary torch operations in 32 bits) or, where the
module's ``own`` is true, through ``musc_b200.ops``.  ``exact`` evaluates the definition in 64 bits.
"""
import functools
import math
import os
import random
import sys

import torch

own = False

_TYPES = {'f32': torch.float32, 'f16': torch.float16, 'bf16': torch.bfloat16, 'e4m3': torch.float8_e4m3fn}
_SIZE = {'f32': 4, 'f16': 2, 'bf16': 2, 'e4m3': 1}
_E4M3_MAX = 448.0


@functools.cache
def _ops():
    path = os.path.join(os.getcwd(), 'musc-gpu_b200')
    if path not in sys.path:
        sys.path.insert(0, path)
    from musc_b200 import ops
    return ops


# ----------------------------------------------------------------------------- cases
def listed():
    return [
        # Attention pooling: one probe query per image over the tokens of a ViT-L/14 at 518 pixels,
        # for a batch of four images.  The smallest call: latency counts.
        _attention('probe', docs=4, q_len=1, k_len=1370, heads=16, kv_heads=16, head_dim=64, dtype='f16'),
        # One token of each of 32 requests over caches of up to 8192 tokens, used to differing lengths.
        _attention('token_cache', docs=32, q_len=1, k_len=8192, heads=32, kv_heads=8, head_dim=128, dtype='bf16',
                   slots=True, causal=True, softcap=30.0),
        # Images of differing sizes packed into one sequence: each attends to its own patches only.
        _attention('packed_images', docs=9, q_len=1370, k_len=0, heads=16, kv_heads=16, head_dim=64, dtype='f16',
                   ragged=True),
        # Image tokens as a prefix that all tokens see, text after it; scores capped.
        _attention('prefix_text', docs=4, q_len=2003, k_len=0, heads=16, kv_heads=4, head_dim=128, dtype='bf16',
                   ragged=True, causal=True, prefix=True, softcap=50.0),
        # One long document, causal, with a bias that falls with the distance: the largest.
        _attention('long_distance', docs=1, q_len=16384, k_len=0, heads=8, kv_heads=2, head_dim=128, dtype='bf16',
                   causal=True, bias=True),
        # Rotary positions of one new token in each of 32 requests.
        _rotary('rotary_token', tokens=32, heads=32, kv_heads=8, head_dim=128, axes=1, dtype='bf16'),
        # Rows and columns of a batch of eight 37 x 37 patch grids with class tokens.
        _rotary('rotary_image', tokens=10960, heads=16, kv_heads=16, head_dim=64, axes=2, dtype='f16', adjacent=True),
        # Time, height and width of a long video.
        _rotary('rotary_video', tokens=65001, heads=16, kv_heads=4, head_dim=128, axes=3, dtype='bf16'),
        # The norm before one token's projections.
        _norm('norm_token', rows=4, channels=1024, residual='bf16', delta='bf16', out='bf16'),
        # A block of the encoder: batch of four images, fp32 residual stream, 16-bit branch and output.
        _norm('norm_image', rows=5480, channels=1024, residual='f32', delta='f16', out='f16'),
        # 8-bit input of the next product, one scale for each row.
        _norm('norm_rows_8bit', rows=16389, channels=4096, residual='bf16', delta='bf16', out='e4m3'),
        # 8-bit with a scale for each group of 128 columns, a width that is no multiple of the group.
        _norm('norm_groups_8bit', rows=8191, channels=1480, residual='f32', delta='bf16', out='e4m3', group=128),
    ]


def _attention(name, *, docs, q_len, k_len, heads, kv_heads, head_dim, dtype, ragged=False, slots=False, causal=False,
               prefix=False, softcap=0.0, bias=False):
    """``k_len`` 0: self-attention.  ``ragged``: document lengths from a fifth of ``q_len`` up.
    ``slots``: each document's keys lie in a slot of ``k_len`` rows, used from a quarter up."""
    return {'name': name, 'op': 'attention', 'docs': docs, 'q_len': q_len, 'k_len': k_len, 'heads': heads,
            'kv_heads': kv_heads, 'head_dim': head_dim, 'dtype': dtype, 'ragged': ragged, 'slots': slots,
            'causal': causal, 'prefix': prefix, 'softcap': softcap, 'bias': bias}


def _rotary(name, *, tokens, heads, kv_heads, head_dim, axes, dtype, adjacent=False):
    return {'name': name, 'op': 'rotary', 'tokens': tokens, 'heads': heads, 'kv_heads': kv_heads,
            'head_dim': head_dim, 'axes': axes, 'dtype': dtype, 'adjacent': adjacent}


def _norm(name, *, rows, channels, residual, delta, out, group=0):
    return {'name': name, 'op': 'norm', 'rows': rows, 'channels': channels, 'residual': residual, 'delta': delta,
            'out': out, 'group': group}


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(('token', 'packed', 'causal', 'rotary', 'norm'))
    dtype = rng.choice(('f16', 'bf16'))
    if op in ('token', 'packed', 'causal'):
        head_dim = rng.choice((64, 128))
        kv_heads = rng.choice((1, 2, 4, 8))
        group = rng.choice((1, 2, 3, 4, 8))
        heads = kv_heads * group
        common = dict(heads=heads, kv_heads=kv_heads, head_dim=head_dim, dtype=dtype,
                      softcap=rng.choice((0.0, 30.0, 50.0)), bias=rng.random() < 0.4)
        if op == 'token':  # one or a few new tokens over caches: the keys fill 400 MB at most
            q_len = rng.choice((1, 1, 2, 5))
            rows = 400_000_000 // (kv_heads * head_dim * 4)
            docs = _log_int(rng, 1, 64)
            k_len = _log_int(rng, 8, min(32768, rows // docs, 400_000_000 // (heads * docs * docs * q_len)))
            case = _attention('', docs=docs, q_len=q_len, k_len=k_len, slots=True, causal=rng.random() < 0.5, **common)
        else:  # whole prompts and images: the scores of the plain form fill 4 GB at most
            total = _log_int(rng, 60, int(math.sqrt(1e9 / heads)))
            docs = _log_int(rng, 1, 24) if op == 'packed' else rng.choice((1, 1, 2))
            case = _attention('', docs=docs, q_len=max(5, total // docs), k_len=0, ragged=docs > 1,
                              causal=op == 'causal', prefix=op == 'causal' and rng.random() < 0.5, **common)
    elif op == 'rotary':
        kv_heads = rng.choice((1, 2, 4, 8, 16))
        head_dim = rng.choice((64, 80, 128))
        heads = kv_heads * rng.choice((1, 2, 4))
        case = _rotary('', tokens=_log_int(rng, 1, min(65000, 160_000_000 // (head_dim * (heads + kv_heads)))),
                       heads=heads, kv_heads=kv_heads, head_dim=head_dim, axes=rng.choice((1, 2, 3)), dtype=dtype,
                       adjacent=rng.random() < 0.5)
    else:
        channels = rng.choice((rng.randrange(16, 500) * 16, rng.randrange(200, 8000), 1024, 4096))
        out = rng.choice(('f16', 'bf16', 'e4m3', 'e4m3'))
        case = _norm('', rows=_log_int(rng, 1, 60_000_000 // channels), channels=channels,
                     residual=rng.choice(('f32', 'bf16')), delta=rng.choice(('f16', 'bf16')), out=out,
                     group=rng.choice((0, 128)) if out == 'e4m3' else 0)
    del case['name']
    return case


# ----------------------------------------------------------------------------- inputs
def _lengths(case):
    """Host lengths of a case's documents: queries, keys, prefixes and key slots.  They are the case's own,
    so that its work is known without its inputs."""
    rng = random.Random(case['docs'] * 1009 + case['q_len'] * 31 + case['k_len'])
    docs, q_len, k_len = case['docs'], case['q_len'], case['k_len']
    q = [rng.randint(max(1, q_len // 5), q_len) if case['ragged'] else q_len for _ in range(docs)]
    if k_len == 0:
        k, slot = list(q), list(q)
    elif case['slots']:
        k = [rng.randint(min(k_len, max(q_len, k_len // 4)), k_len) for _ in range(docs)]
        slot = [k_len] * docs
    else:
        k, slot = [k_len] * docs, [k_len] * docs
    prefix = [rng.randint(0, n) for n in k]
    return q, k, slot, prefix


def _starts(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return out


def prepare(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    return {'attention': _prepare_attention, 'rotary': _prepare_rotary, 'norm': _prepare_norm}[case['op']](case, gen)


def _prepare_attention(case, gen):
    dtype = _TYPES[case['dtype']]
    h, hk, d = case['heads'], case['kv_heads'], case['head_dim']
    q_lens, k_lens, slots, prefix = _lengths(case)
    tq, tk = sum(q_lens), sum(slots)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device='cuda')
    state = dict(case, q_offsets=ints(_starts(q_lens)), k_offsets=ints(_starts(slots)), k_lengths=ints(k_lens),
                 prefix_lengths=ints(prefix) if case['prefix'] else None,
                 slopes=2.0 ** (-8.0 * torch.arange(1, h + 1, device='cuda') / h) if case['bias'] else None)
    rand = lambda *shape: torch.randn(*shape, generator=gen, device='cuda').to(dtype)
    if case['k_len'] == 0:  # queries, keys and values are columns of one projection
        qkv = rand(tq, (h + 2 * hk) * d)
        qkv[:, :h * d] *= 1.5
        state.update(q=qkv[:, :h * d], k=qkv[:, h * d:(h + hk) * d], v=qkv[:, (h + hk) * d:])
    else:
        state.update(q=rand(tq, h * d) * 1.5, k=rand(tk, hk * d), v=rand(tk, hk * d))
    return state


def _prepare_rotary(case, gen):
    dtype = _TYPES[case['dtype']]
    t, h, hk, d, axes = (case[n] for n in ('tokens', 'heads', 'kv_heads', 'head_dim', 'axes'))
    qk = torch.randn(t, (h + hk) * d, generator=gen, device='cuda').to(dtype)
    index = torch.arange(t, device='cuda')
    first = int(torch.randint(0, 30000, (1,), generator=gen, device='cuda'))
    if axes == 1:    # each token somewhere in its own request
        positions = torch.randint(0, 131072, (t, 1), generator=gen, device='cuda')
    elif axes == 2:  # a class token at (0, 0), then rows and columns of 37 x 37 patches, image after image
        patch = index % 1370 - 1
        positions = torch.stack([patch.clamp_min(0) // 37, patch.clamp_min(0) % 37], 1)
    else:            # frames of 24 x 30 patches, from some time on
        positions = torch.stack([first + index // 720, index // 30 % 24, index % 30], 1)
    pairs = d // 2
    per_axis = [pairs // axes + (a < pairs % axes) for a in range(axes)]
    frequencies = torch.cat([10000.0 ** (-torch.arange(n, dtype=torch.float64, device='cuda') / n) for n in per_axis])
    axis = torch.cat([torch.full((n,), a, device='cuda') for a, n in enumerate(per_axis)])
    return dict(case, q=qk[:, :h * d], k=qk[:, h * d:], positions=positions.to(torch.int32),
                frequencies=frequencies.float(), axis=axis.to(torch.int32))


def _prepare_norm(case, gen):
    rows, c = case['rows'], case['channels']
    x = torch.randn(rows, c, generator=gen, device='cuda')
    x *= torch.exp(0.5 * torch.randn(rows, 1, generator=gen, device='cuda'))  # the residual stream's rows differ in size
    x[:, torch.randint(0, c, (3,), generator=gen, device='cuda')] *= 20.0     # and a few channels stand out
    delta = 0.5 * torch.randn(rows, c, generator=gen, device='cuda')
    weight = 1.0 + 0.1 * torch.randn(c, generator=gen, device='cuda')
    return dict(case, x=x.to(_TYPES[case['residual']]), d=delta.to(_TYPES[case['delta']]), weight=weight, eps=1e-6)


# ----------------------------------------------------------------------------- one pass
def run(state):
    if state['op'] == 'attention':
        return _own_attention(state) if own else _plain_attention(state)
    if state['op'] == 'rotary':
        return _own_rotary(state) if own else _plain_rotary(state)
    return _own_norm(state) if own else _plain_norm(state)


def _own_attention(s):
    kwargs = dict(kv_heads=s['kv_heads'], offsets=s['q_offsets'], causal=s['causal'], prefix=s['prefix_lengths'],
                  softcap=s['softcap'], slopes=s['slopes'])
    if s['k_len']:
        kwargs['kv_offsets'] = s['k_offsets']
    if s['slots']:
        kwargs['kv_lengths'] = s['k_lengths']
    return _ops().attention_masked(s['q'], s['k'], s['v'], s['heads'], **kwargs)


def _plain_attention(s):
    h, hk, d = s['heads'], s['kv_heads'], s['head_dim']
    q, k, v = (s[n].float() for n in 'qkv')
    tq, tk = q.shape[0], k.shape[0]
    q = q.view(tq, hk, h // hk, d).permute(1, 2, 0, 3).reshape(hk, -1, d)
    k, v = (t.view(tk, hk, d).transpose(0, 1) for t in (k, v))
    scores = ((q @ k.transpose(1, 2)) * d ** -0.5).view(h, tq, tk)
    if s['softcap']:
        scores = s['softcap'] * torch.tanh(scores / s['softcap'])
    # the keys that a row sees, as one interval of the packed keys
    row = torch.arange(tq, device=q.device)
    doc = torch.searchsorted(s['q_offsets'], row, right=True) - 1
    begin, count = s['k_offsets'][doc].long(), s['k_lengths'][doc].long()
    q_begin, q_count = s['q_offsets'][doc].long(), (s['q_offsets'][1:] - s['q_offsets'][:-1])[doc].long()
    position = row - q_begin + count - q_count
    end = begin + count
    if s['causal']:
        seen = position + 1
        if s['prefix_lengths'] is not None:
            seen = torch.maximum(seen, s['prefix_lengths'][doc].long())
        end = begin + torch.minimum(seen.clamp_min(0), count)
    key = torch.arange(tk, device=q.device)
    if s['slopes'] is not None:
        distance = (key - (begin + position)[:, None]).abs().float()
        scores = scores - s['slopes'][:, None, None] * distance
    hidden = (key < begin[:, None]) | (key >= end[:, None])
    scores.masked_fill_(hidden, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(torch.isfinite(top), top, 0.0))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, 1.0)
    out = p.view(hk, -1, tk) @ v
    return out.view(h, tq, d).transpose(0, 1).reshape(tq, h * d).to(s['q'].dtype)


def _own_rotary(s):
    return _ops().rotary(s['q'], s['k'], s['positions'], s['frequencies'], s['axis'], s['heads'],
                         kv_heads=s['kv_heads'], adjacent=s['adjacent'])


def _plain_rotary(s):
    # the angle of a far position needs more than 32 bits
    angle = s['positions'].double()[:, s['axis'].long()] * s['frequencies'].double()
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]

    def turn(x, heads):
        x32 = x.float().view(x.shape[0], heads, -1)
        if s['adjacent']:
            a, b = x32[..., 0::2], x32[..., 1::2]
            y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1)
        else:
            a, b = x32.chunk(2, -1)
            y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        return y.reshape(x.shape).to(x.dtype)

    return turn(s['q'], s['heads']), turn(s['k'], s['kv_heads'])


def _own_norm(s):
    out = _ops().add_rmsnorm(s['x'], s['d'], s['weight'], s['eps'], _TYPES[s['out']], group=s['group'])
    return (s['x'], *out) if s['out'] == 'e4m3' else (s['x'], out)


def _plain_norm(s):
    h = s['x'].float() + s['d'].float()
    s['x'].copy_(h)
    y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + s['eps']) * s['weight']
    if s['out'] != 'e4m3':
        return s['x'], y.to(_TYPES[s['out']])
    rows, c = y.shape
    group = s['group'] or c
    groups = -(-c // group)
    padded = torch.zeros(rows, groups * group, device=y.device)
    padded[:, :c] = y
    scale = padded.view(rows, groups, group).abs().amax(-1) / _E4M3_MAX
    values = y / scale.repeat_interleave(group, 1)[:, :c]
    return s['x'], values.clamp(-_E4M3_MAX, _E4M3_MAX).to(torch.float8_e4m3fn), scale


# ----------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    """The definitions, document by document and head by head, in float64 and unrounded."""
    state = prepare(case, seed)
    if case['op'] == 'attention':
        return _exact_attention(state)
    if case['op'] == 'rotary':
        return tuple(_exact_turn(state, state[n], heads) for n, heads in (('q', case['heads']), ('k', case['kv_heads'])))
    h = state['x'].double() + state['d'].double()
    y = h / torch.sqrt((h * h).sum(1, keepdim=True) / h.shape[1] + state['eps']) * state['weight'].double()
    if case['out'] != 'e4m3':
        return h, y
    group = case['group'] or case['channels']
    scales, values = [], []
    for part in y.split(group, 1):
        scales.append(part.abs().max(1, keepdim=True).values / _E4M3_MAX)
        values.append(part / scales[-1])
    return h, torch.cat(values, 1), torch.cat(scales, 1)


def _exact_attention(s):
    q_lens, k_lens, slots, prefix = _lengths(s)
    h, hk, d = s['heads'], s['kv_heads'], s['head_dim']
    out = torch.zeros(sum(q_lens), h * d, dtype=torch.float64, device='cuda')
    q0 = k0 = 0
    for nq, nk, slot, pre in zip(q_lens, k_lens, slots, prefix):
        i = torch.arange(nq, device='cuda')[:, None] + (nk - nq)
        j = torch.arange(nk, device='cuda')[None]
        visible = torch.ones(nq, nk, dtype=torch.bool, device='cuda')
        if s['causal']:
            visible = j <= i
            if s['prefix']:
                visible |= j < pre
        for head in range(h):
            at = head // (h // hk) * d
            z = s['q'][q0:q0 + nq, head * d:(head + 1) * d].double() @ s['k'][k0:k0 + nk, at:at + d].double().T
            z /= math.sqrt(d)
            if s['softcap']:
                z = torch.tanh(z / s['softcap']) * s['softcap']
            if s['bias']:
                z -= s['slopes'][head].double() * (i - j).abs()
            z[~visible] = -math.inf
            p = torch.softmax(z, -1).nan_to_num(0.0)
            out[q0:q0 + nq, head * d:(head + 1) * d] = p @ s['v'][k0:k0 + nk, at:at + d].double()
            del z, p
        q0, k0 = q0 + nq, k0 + slot
    return out


def _exact_turn(s, x, heads):
    angle = s['positions'].double()[:, s['axis'].long()] * s['frequencies'].double()
    factor = torch.polar(torch.ones_like(angle), angle)[:, None]
    x = x.double().reshape(x.shape[0], heads, -1)
    n = angle.shape[1]
    if s['adjacent']:
        y = torch.view_as_real(torch.view_as_complex(x.reshape(x.shape[0], heads, n, 2).contiguous()) * factor).flatten(2)
    else:
        z = torch.complex(x[..., :n].contiguous(), x[..., n:].contiguous()) * factor
        y = torch.cat([z.real, z.imag], -1)
    return y.reshape(x.shape[0], -1)


# ----------------------------------------------------------------------------- work
def work(case):
    if case['op'] == 'attention':
        q_lens, k_lens, _, prefix = _lengths(case)
        h, hk, d, size = case['heads'], case['kv_heads'], case['head_dim'], _SIZE[case['dtype']]
        pairs = 0
        for nq, nk, pre in zip(q_lens, k_lens, prefix):
            if not case['causal']:
                pairs += nq * nk
                continue
            first = nk - nq + 1  # keys that the first query sees; one more for each after it
            least = min(pre, nk) if case['prefix'] else 0
            lifted = min(nq, max(0, least - first + 1))  # queries whose prefix reaches further
            pairs += lifted * least + (nq - lifted) * (first + lifted + nk) // 2
        return {'bytes': size * d * (2 * h * sum(q_lens) + 2 * hk * sum(k_lens)), 'flops': 4 * d * h * pairs}
    if case['op'] == 'rotary':
        values = case['tokens'] * (case['heads'] + case['kv_heads']) * case['head_dim']
        return {'bytes': 2 * values * _SIZE[case['dtype']] + 4 * case['tokens'] * case['axes'], 'flops': 3 * values}
    values = case['rows'] * case['channels']
    size = 2 * _SIZE[case['residual']] + _SIZE[case['delta']] + _SIZE[case['out']]
    scales = case['rows'] * -(-case['channels'] // (case['group'] or case['channels'])) * 4 if case['out'] == 'e4m3' else 0
    return {'bytes': values * size + scales + 4 * case['channels'], 'flops': 5 * values}
