"""The 4-bit matrix-vector products (``mes_awq_gemv``) against 64-bit arithmetic.

Bounds.  The kernel's weights are exact, so what differs from 64 bits is its fp32 summation, at
most (K / 16 + K / group + 40) adds and multiplies in a row, each off by at most 2^-22 of the sum
of magnitudes ``mag = sum |x| |w|`` (a tensor-core add may truncate), and the rounding of the
result.  With ``e = (K / 16 + K / group + 40) 2^-22 mag``: fp32 sums are within ``e`` + 2^-23 of
the result, bf16 results within ``e`` + 2^-8 of theirs, and silu(g) u, |silu'| < 1.1, within
``1.1 e_g |u| + |silu(g)| e_u + 1.1 e_g e_u`` + 2^-8 of its own.
"""
import numpy as np
import pytest
import torch

from mes_b200 import _C
from oracle import awq as oawq

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _weights(K, N, group, seed):
    """(kernel-layout tensors on the GPU, exact fp64 weights [K, N])."""
    rng = np.random.default_rng(seed)
    q = rng.integers(0, 16, (K, N), dtype=np.uint8)
    z = rng.integers(0, 16, (K // group, N), dtype=np.uint8)
    s = rng.uniform(0.002, 0.02, (K // group, N)).astype(np.float16)
    s[0, :3] = (6e-8, 1.0, 0.0)                     # the least subnormal, one, and a dead feature
    w = (q.astype(np.float64) - np.repeat(z, group, 0)) * np.repeat(s.astype(np.float64), group, 0)
    qw = _C.awq_repack(torch.from_numpy(oawq.awq_pack(q)).to(DEV))
    return (qw, torch.from_numpy(oawq.awq_pack(z)).to(DEV), torch.from_numpy(s).to(DEV)), w


def _x(M, K, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(M, K, generator=g).to(torch.bfloat16)


def _expect(x, w, group):
    xd = x.double().numpy()
    mag = np.abs(xd) @ np.abs(w)
    K = w.shape[0]
    return xd @ w, (K / 16 + K / group + 40) * 2.0 ** -22 * mag


def _near(got, want, tol):
    got = got.double().cpu().numpy()
    assert got.shape == want.shape
    off = np.abs(got - want) - tol
    assert not (off > 0).any(), f"{off.max():.3g} past the bound at {np.unravel_index(off.argmax(), off.shape)}"


SHAPES = [(128, 8, 128), (128, 40, 32), (256, 32, 64), (384, 1000, 128), (1536, 2048, 128), (1024, 1024, 64),
          (2048, 72, 32), (9728, 256, 128), (512, 20000, 128)]


@pytest.mark.parametrize("K,N,group", SHAPES)
@pytest.mark.parametrize("M", [1, 3, 8, 9, 16])
@pytest.mark.parametrize("bias", [False, True])
def test_bf16(K, N, group, M, bias):
    wt, w = _weights(K, N, group, K + N)
    x = _x(M, K, M)
    b = torch.randn(N, generator=torch.Generator().manual_seed(5)).to(torch.bfloat16) if bias else None
    y, e = _expect(x, w, group)
    if bias:
        y = y + b.double().numpy()
    got = _C.awq_gemv(x.to(DEV), *wt, None if b is None else b.to(DEV), group_size=group)
    assert got.dtype == torch.bfloat16
    _near(got, y, e + 2.0 ** -8 * np.abs(y))
    assert _C.take_device_error() == 0


@pytest.mark.parametrize("K,N,group", SHAPES)
@pytest.mark.parametrize("M", [1, 7, 16])
def test_residual(K, N, group, M):
    wt, w = _weights(K, N, group, 3)
    x = _x(M, K, M)
    r = torch.randn(M, N, generator=torch.Generator().manual_seed(6))
    y, e = _expect(x, w, group)
    want = y + r.double().numpy()
    res = r.to(DEV)
    out = _C.awq_gemv_residual(x.to(DEV), *wt, res, group_size=group)
    assert out is res
    _near(res, want, e + 2.0 ** -22 * (np.abs(y) + np.abs(want)))


@pytest.mark.parametrize("K,N,group", [(128, 32, 128), (1024, 6144, 128), (256, 96, 32), (512, 2080, 64)])
@pytest.mark.parametrize("M", [1, 8, 13])
def test_silu(K, N, group, M):
    wt, w = _weights(K, N, group, 4)
    x = (_x(M, K, M).float() * 0.2).to(torch.bfloat16)
    y, e = _expect(x, w, group)
    f = np.arange(N // 2)
    gi, ui = f // 16 * 32 + f % 16, f // 16 * 32 + 16 + f % 16
    silu = y[:, gi] / (1 + np.exp(-y[:, gi]))
    want = silu * y[:, ui]
    eg, eu = e[:, gi], e[:, ui]
    tol = 1.1 * eg * np.abs(y[:, ui]) + np.abs(silu) * eu + 1.1 * eg * eu + (2.0 ** -8 + 1e-6) * np.abs(want)
    _near(_C.awq_gemv_silu(x.to(DEV), *wt, group_size=group), want, tol)


def test_silu_matches_the_models_interleaving():
    """Gate and up projections put together by ``interleave_gate_up`` as the model's layer does."""
    K, I, M = 256, 64, 3
    rng = np.random.default_rng(8)
    q = rng.integers(0, 16, (K, 2 * I), dtype=np.uint8)
    z = rng.integers(0, 16, (K // 128, 2 * I), dtype=np.uint8)
    s = rng.uniform(0.002, 0.02, (K // 128, 2 * I)).astype(np.float16)
    w = (q.astype(np.float64) - np.repeat(z, 128, 0)) * np.repeat(s.astype(np.float64), 128, 0)
    qw, qz, sc = _C.interleave_gate_up(*(torch.from_numpy(a).to(DEV) for a in
                                         (oawq.awq_pack(q), oawq.awq_pack(z), s)))
    x = (_x(M, K, 1).float() * 0.2).to(torch.bfloat16)
    y, e = _expect(x, w, 128)
    gate, up = y[:, :I], y[:, I:]
    silu = gate / (1 + np.exp(-gate))
    tol = (1.1 * e[:, :I] * np.abs(up) + np.abs(silu) * e[:, I:] + 1.1 * e[:, :I] * e[:, I:] +
           (2.0 ** -8 + 1e-6) * np.abs(silu * up))
    _near(_C.awq_gemv_silu(x.to(DEV), _C.awq_repack(qw), qz, sc), silu * up, tol)


def test_strided_rows_and_outputs():
    K, N, M = 256, 104, 5
    wt, w = _weights(K, N, 128, 9)
    x = _x(M, K + 24, 2)
    xs = x.to(DEV)[:, 8:8 + K]                     # rows of pitch K + 24, 16-byte aligned
    y, e = _expect(x[:, 8:8 + K], w, 128)
    buf = torch.full((M, N + 7), float("nan"), dtype=torch.bfloat16, device=DEV)
    out = _C.awq_gemv(xs, *wt, out=buf[:, 3:3 + N])
    _near(out, y, e + 2.0 ** -8 * np.abs(y))
    assert buf[:, :3].isnan().all() and buf[:, 3 + N:].isnan().all()
    res = torch.zeros(M, N + 5, device=DEV)
    _C.awq_gemv_residual(xs, *wt, res[:, 1:1 + N])
    _near(res[:, 1:1 + N], y, e + 2.0 ** -22 * np.abs(y))
    assert (res[:, 0] == 0).all() and (res[:, 1 + N:] == 0).all()


def test_a_row_does_not_see_the_others():
    """Rows with infinities and NaN leave the other rows' bits alone, and a call repeats."""
    K, N = 1024, 264
    wt, _ = _weights(K, N, 128, 10)
    x = _x(8, K, 3).to(DEV)
    base = _C.awq_gemv(x, *wt)
    assert torch.equal(base, _C.awq_gemv(x, *wt))
    bad = x.clone()
    bad[2, 5] = float("nan")
    bad[6, 700] = float("inf")
    got = _C.awq_gemv(bad, *wt)
    ok = [0, 1, 3, 4, 5, 7]
    assert torch.equal(got[ok], base[ok])
    assert got[2].isnan().all() and not got[6].isfinite().all()
    for m in range(8):
        assert torch.equal(_C.awq_gemv(x[m:m + 1], *wt)[0], base[m])


def test_no_rows_and_side_stream():
    wt, w = _weights(128, 64, 128, 11)
    assert _C.awq_gemv(torch.empty(0, 128, dtype=torch.bfloat16, device=DEV), *wt).shape == (0, 64)
    x = _x(2, 128, 4)
    y, e = _expect(x, w, 128)
    side = torch.cuda.Stream()
    xd = x.to(DEV)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _C.awq_gemv(xd, *wt)
    side.synchronize()
    _near(got, y, e + 2.0 ** -8 * np.abs(y))


def test_refusals():
    wt, _ = _weights(256, 64, 128, 12)
    x = torch.zeros(17, 256, dtype=torch.bfloat16, device=DEV)
    for bad in (lambda: _C.awq_gemv(x, *wt), lambda: _C.awq_gemv(x[:2, :128], *wt),
                lambda: _C.awq_gemv(x[:2], *wt, group_size=64), lambda: _C.awq_gemv(x[:2, ::2], *wt),
                lambda: _C.awq_gemv(x[:2].float(), *wt), lambda: _C.awq_gemv(x[:2].cpu(), *wt),
                lambda: _C.awq_gemv_residual(x[:2], *wt, torch.zeros(2, 63, device=DEV)),
                lambda: _C.awq_gemv(torch.zeros(2, 260, dtype=torch.bfloat16, device=DEV)[:, 4:], *wt)):
        with pytest.raises(_C.MesError):
            bad()


def test_rows_of_any_size():
    """A power of two on x is one on the result, bit for bit, where nothing leaves fp32's range.  Small sums are kept to
    2^-76: K / 16 + 2 K / group roundings for each scale, one for each group and row of sums."""
    K, N, M, group = 512, 72, 3, 128
    wt, w = _weights(K, N, group, 13)
    x = _x(M, K, 5)
    x[x.abs() < 2.0 ** -8] = 1.0
    base = _C.awq_gemv_residual(x.to(DEV), *wt, torch.zeros(M, N, device=DEV))
    for e in (-28, -20, 40, 64):
        got = _C.awq_gemv_residual((x * 2.0 ** e).to(DEV), *wt, torch.zeros(M, N, device=DEV))
        # Sums of q x are multiples of 2^(e - 15 - 73), their products with a scale (11 bits from 2^-9 on, or the least,
        # 2^-24) of 2^(e - 107) and 2^(e - 112): for e = -28 and -20 no bit is below 2^-149.
        if e < -20:
            assert torch.equal(got[:, 3:], base[:, 3:] * 2.0 ** e)
        else:
            assert torch.equal(got, base * 2.0 ** e)
    for e in (-60, -70, -90):
        small = x * 2.0 ** e
        got = _C.awq_gemv_residual(small.to(DEV), *wt, torch.zeros(M, N, device=DEV)).double().cpu().numpy()
        y, rel = _expect(small, w, group)
        most = 1.0 * (K / 16 + 2 * K / group) + K / group + 16          # the largest scale is 1
        assert (np.abs(got - y) <= rel + most * 2.0 ** -76).all(), e
