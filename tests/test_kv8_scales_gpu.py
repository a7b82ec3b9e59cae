"""Attention over cached pages whose V scales are 0, subnormal or far apart, against 64 bits.

Bounds.  Logits, weights and their 16-bit form are off as ``test_kv8_gpu.py`` says: with
``d = 12 2^-22 S + 2^-20 max|logit|``, S the largest ``sum |q| |k| scale``, and 2^-18 for the exponents (numbers
of up to 2^8, each rounded to 24 bits), a weight is within ``2 (d + 2^-18)`` of itself and within 2^-11 more in 16
bits.  Weights are kept relative to a reference that goes by the largest V scale of the keys a warp has seen, so the
smallest are off by 2^-35 of it, and pages 2^-60 below it count as 0: 2^-34 N max|v| covers both.  The output is
rounded to bf16: 2^-8 of itself, and 2^-133 where it is subnormal.
"""
import numpy as np
import pytest
import torch

from mes_b200 import _C
from test_kv8_gpu import D, DEV, KINDS, Cache, _cu

pytestmark = pytest.mark.gpu


def _expect(cache, q, news, heads, scale):
    """64-bit outputs, their bounds, and for each sequence the summed weights and their relative bound."""
    T, hkv = q.shape[0], cache.hkv
    G = heads // hkv
    qd = q.double().cpu().numpy().reshape(T, heads, D)
    want, tol = np.zeros((T, heads, D)), np.zeros((T, heads, D))
    add, r0 = [], 0
    for b, (c, m) in enumerate(zip(cache.ctx, news)):
        kv = cache.values(b)
        add.append([])
        for h in range(hkv):
            at = np.s_[r0:r0 + m, h * G:(h + 1) * G]
            x = np.einsum("igd,td->igt", qd[at], kv[0, h]) * scale
            size = (np.einsum("igd,td->igt", np.abs(qd[at]), np.abs(kv[0, h])) * scale).max()
            d = 12 * 2.0 ** -22 * size + 2.0 ** -20 * np.abs(x).max() + 2.0 ** -18
            x = np.where(np.arange(c)[None, None] > (c - m + np.arange(m))[:, None, None], -np.inf, x)
            w = np.exp(x - x.max(-1, keepdims=True))
            w = w / w.sum(-1, keepdims=True)
            want[at] = np.einsum("igt,td->igd", w, kv[1, h])
            tol[at] = ((2 * d + 2.0 ** -11) * np.einsum("igt,td->igd", w, np.abs(kv[1, h])) +
                       2.0 ** -34 * c * np.abs(kv[1, h]).max() + 2.0 ** -8 * np.abs(want[at]) + 2.0 ** -133)
            add[b].append((w.sum((0, 1)), 2 * d + 2.0 ** -20 * m * G))
        r0 += m
    return want, tol, add


def _attend_and_check(cache, news, heads, sums, seed=2):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(sum(news), heads * D, generator=g).to(torch.bfloat16).to(DEV)
    want, tol, add = _expect(cache, q, news, heads, D ** -0.5)
    before = cache.sums.double().cpu().numpy()
    got = _C.kv8_attention(q, cache.codes, cache.scales, cache.table, _cu(news), cache.lens, heads, D ** -0.5, max(news),
                           sums=cache.sums if sums else None)
    assert _C.take_device_error() == 0
    off = np.abs(got.double().cpu().numpy().reshape(want.shape) - want)
    assert (off <= tol).all(), (np.argwhere(~(off <= tol))[0], np.nanmax(off / tol))
    if not sums:
        return
    after = cache.sums.double().cpu().numpy()
    for b, c in enumerate(cache.ctx):
        t = np.arange(c)
        p = cache.table[b].cpu().numpy()[t // cache.page]
        for h in range(cache.hkv):
            w, rel = add[b][h]
            old = before[p, h, t % cache.page]
            assert (np.abs(after[p, h, t % cache.page] - (old + w)) <= rel * w + 2.0 ** -22 * (old + w) + 1e-30).all(), (b, h)


# V scales of a sequence's pages, in turn.
ZEROS = [[1e-12, 0.0], [0.0, 1e-12], [0.0, 1e-6, 0.0], [0.0] * 9 + [1e-9], [1e-9] + [0.0] * 9, [0.0]]
SMALL = [[1e-37], [1e-38], [1e-40], [1e-38, 0.0], [0.0, 1e-38]]
APART = [[1.0, 1e-38], [1e-38, 1.0], [1.0, 1e-38, 0.0], [1e-20, 1e20], [1e20, 0.0, 1e-20], [1e30, 1.0, 1e-30], [1e-30] * 4 + [1e30]]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("heads", [2, 12])
@pytest.mark.parametrize("sums", [False, True])
@pytest.mark.parametrize("amp", ZEROS + SMALL + APART, ids=str)
def test_v_scales(kind, page, heads, sums, amp):
    """Short texts (dealt whole), longer ones and one cut among blocks; K scales are ordinary."""
    for ctx, news in (([100, 40, 500, 1, 33], [1, 2, 1, 1, 2]), ([700, 40, 9000, 1], [1, 2, 1, 1])):
        cache = Cache(kind, page, 1, ctx).fill(amp=amp)
        cache.scales[:, 0] = cache.scales[:, 0].clamp(max=0.1, min=1e-3)
        _attend_and_check(cache, news, heads, sums)


@pytest.mark.parametrize("kind", KINDS)
def test_tiny_values_as_they_are_written(kind):
    """Pages of tiny and of zero values beside ordinary ones, stored by the cache write."""
    page, hkv, n = 16, 2, 150
    g = torch.Generator().manual_seed(9)
    for tiny in (1e-37, 3e-38, 1e-39, 0.0):
        for ordinary in (1.0, 1e-9, tiny):
            cache = Cache(kind, page, hkv, [n])
            v = torch.randn(n, hkv * D, generator=g)
            v *= torch.tensor([tiny, ordinary]).repeat_interleave(2 * page).repeat(3)[:n].view(-1, 1)
            k = torch.randn(n, hkv * D, generator=g)
            k, v = k.to(torch.bfloat16).to(DEV), v.to(torch.bfloat16).to(DEV)
            _C.kv8_append(k, v, cache.codes, cache.scales, cache.table, _cu([n]), cache.lens, n, sums=cache.sums)
            _attend_and_check(cache, [3], 6, True)
