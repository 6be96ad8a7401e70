"""The encoder with two-axis rotary positions, over batches and over packed images of differing sizes.

Reference: the tower's formula in float64, image by image.  Bounds: those of the 24-block tower's
test (tokens within 5e-3 RMS and 5e-2 maximum of the layer's RMS), here for two blocks.
"""
from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F


def _tower(device, **kwargs):
    from musc_b200.encoder import VisionEncoder, random_vit_state
    state = random_vit_state(5, image_size=56, patch_size=14, width=128, layers=2, heads=2, output_dim=64)
    del state['positional_embedding']
    return state, VisionEncoder(state, image_size=56, patch_size=14, width=128, layers=2, heads=2, device=device,
                                rotary=100.0, **kwargs)


def _reference(state, image):
    st = {k: v.double() for k, v in state.items()}
    gh, gw = image.shape[1] // 14, image.shape[2] // 14
    x = F.conv2d(image.double()[None], st['conv1.weight'], stride=14)[0].flatten(1).T
    x = torch.cat([st['class_embedding'][None], x])
    ln = lambda t, name: F.layer_norm(t, (128,), st[name + '.weight'], st[name + '.bias'])
    x = ln(x, 'ln_pre')
    rows = torch.cat([torch.zeros(1), torch.arange(gh).repeat_interleave(gw)]).double()
    cols = torch.cat([torch.zeros(1), torch.arange(gw).repeat(gh)]).double()
    f = 100.0 ** (-torch.arange(16).double() / 16)
    angle = torch.cat([rows[:, None] * f, cols[:, None] * f], 1)[:, None]            # (L, 1, 32)

    def turn(t):
        a, b = t.view(-1, 2, 64).chunk(2, -1)
        return torch.cat([a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()], -1)

    tokens = []
    for i in range(2):
        pre = f'transformer.resblocks.{i}.'
        qkv = ln(x, pre + 'ln_1') @ st[pre + 'attn.in_proj_weight'].T + st[pre + 'attn.in_proj_bias']
        q, k, v = qkv.chunk(3, -1)
        p = torch.softmax(torch.einsum('lhd,mhd->hlm', turn(q), turn(k)) / 8, -1)
        a = torch.einsum('hlm,mhd->lhd', p, v.view(-1, 2, 64)).reshape(-1, 128)
        x = x + a @ st[pre + 'attn.out_proj.weight'].T + st[pre + 'attn.out_proj.bias']
        h = F.gelu(ln(x, pre + 'ln_2') @ st[pre + 'mlp.c_fc.weight'].T + st[pre + 'mlp.c_fc.bias'])
        x = x + h @ st[pre + 'mlp.c_proj.weight'].T + st[pre + 'mlp.c_proj.bias']
        tokens.append(x)
    return ln(x[:1], 'ln_post')[0] @ st['proj'], tokens


def _near(got, want):
    want = want.to(got.device)
    rms = want.square().mean().sqrt()
    err = (got.double() - want).abs()
    assert float(err.square().mean().sqrt() / rms) < 5e-3 and float(err.max() / rms) < 5e-2


@pytest.mark.gpu
def test_packed_images_match_formula(cuda_device):
    state, enc = _tower(cuda_device)
    g = torch.Generator().manual_seed(6)
    images = [torch.rand(3, 14 * h, 14 * w, generator=g) for h, w in ((4, 4), (1, 1), (20, 23), (9, 3), (4, 4))]
    pooled, tokens = enc.forward_packed([im.to(cuda_device) for im in images], [1, 2])
    assert pooled.shape == (5, 64) and [len(t) for t in tokens] == [5, 5]
    for i, im in enumerate(images):
        want_pooled, want = _reference(state, im)
        _near(pooled[i], want_pooled)
        for layer in range(2):
            assert tokens[layer][i].shape == want[layer].shape
            _near(tokens[layer][i], want[layer])


@pytest.mark.gpu
@pytest.mark.parametrize('graph', [False, True])
def test_batch_with_rotary_matches_formula(cuda_device, graph):
    state, enc = _tower(cuda_device)
    g = torch.Generator().manual_seed(7)
    images = torch.rand(3, 3, 56, 56, generator=g)
    for _ in range(3):  # the graph's capture, then replays
        pooled, tokens = enc.forward(images.to(cuda_device), [2], graph=graph)
        for i in range(3):
            want_pooled, want = _reference(state, images[i])
            _near(pooled[i], want_pooled)
            _near(tokens[0][i], want[1])


def test_packed_refusals():
    from musc_b200.encoder import VisionEncoder, random_vit_state
    _, enc = _tower('cpu')
    with pytest.raises(ValueError, match='no images'):
        enc.forward_packed([], [1])
    for bad in ((3, 15, 14), (1, 14, 14), (3, 0, 14)):
        with pytest.raises(ValueError, match='multiples of 14'):
            enc.forward_packed([torch.zeros(3, 14, 14), torch.zeros(*bad)], [1])
    state = random_vit_state(5, image_size=56, patch_size=14, width=128, layers=1, heads=2, output_dim=64)
    learned = VisionEncoder(state, image_size=56, patch_size=14, width=128, layers=1, heads=2, device='cpu')
    with pytest.raises(ValueError, match='rotary'):
        learned.forward_packed([torch.zeros(3, 14, 14)], [1])
    del state['positional_embedding']
    with pytest.raises(KeyError):
        VisionEncoder(state, image_size=56, patch_size=14, width=128, layers=1, heads=2, device='cpu')
