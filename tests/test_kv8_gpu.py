"""The 8-bit paged KV cache (``mes_kv8_*``) against plain implementations.

Codes and scales are compared bit for bit with the same fp32 arithmetic in numpy (one division
or product and one rounding a value) and, in 64 bits, with half a step of the type around the
value.  Attention is compared with 64-bit attention over the stored values.

Attention bounds.  Products are exact and summed in fp32, so a logit is off by at most
``d = 12 2^-22 S`` with S the largest ``sum |q| |k| scale`` (8 tensor-core steps that may truncate,
three scalings), plus 2^-20 of its own size for the scalings.  A weight is then off by ``2 d'``,
``d' = d + 2^-20 max|logit| + 2^-20`` (the exponentials), relative, and by 2^-11 where it enters the
product with V in 16 bits; the smallest weights are off by 2^-35 of the largest.  So the output is
within ``(2 d' + 2^-11 + 2^-18) sum_t w_t |v_t|`` + 2^-35 N max|v|, and 2^-8 of itself for bf16.
A sum of weights is within ``2 d' + 2^-20`` of itself for each addition of up to rows * G weights,
plus 2^-22 of the sum it is added to.
"""
import numpy as np
import pytest
import torch

from mes_b200 import _C

pytestmark = pytest.mark.gpu
DEV = "cuda"
D = 128
QMAX = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
KINDS = [torch.int8, torch.float8_e4m3fn]
PAGES = [16, 32, 64, 128]


class Cache:
    """A cache on the GPU with a shuffled page pool; unused pages and slots hold the worst."""

    def __init__(self, kind, page, hkv, ctx, extra=2, seed=0):
        self.kind, self.page, self.hkv, self.ctx = kind, page, hkv, list(ctx)
        g = torch.Generator().manual_seed(seed)
        need = [-(-c // page) for c in ctx]
        self.num_pages = sum(need) + extra
        order = torch.randperm(self.num_pages, generator=g).tolist()
        width = max(max(need, default=1), 1)
        table = torch.full((len(ctx), width), -7, dtype=torch.int32)     # unused entries: nonsense
        for b, n in enumerate(need):
            for j in range(n):
                table[b, j] = order.pop()
        self.table = table.to(DEV)
        # NaN codes of e4m3 (0x7f); for int8 the one code that is never written.
        poison = 0x7F if kind == torch.float8_e4m3fn else -128
        self.codes = torch.full((self.num_pages, 2, hkv, page, D), poison, dtype=torch.int8, device=DEV).view(kind)
        self.scales = torch.full((self.num_pages, 2, hkv), float("nan"), device=DEV)
        self.sums = torch.full((self.num_pages, hkv, page), float("nan"), device=DEV)
        self.lens = torch.tensor(self.ctx, dtype=torch.int32, device=DEV)

    def fill(self, seed=1, amp=None):
        """Codes and scales of the first ``ctx`` tokens of every sequence at random."""
        g = torch.Generator().manual_seed(seed)
        for b, c in enumerate(self.ctx):
            for j in range(-(-c // self.page)):
                p, n = int(self.table[b, j]), min(self.page, c - j * self.page)
                v = (torch.randn(2, self.hkv, n, D, generator=g) * QMAX[self.kind] / 3.5).clamp(-QMAX[self.kind], QMAX[self.kind])
                v = (v.round() if self.kind == torch.int8 else v).to(self.kind)
                self.codes.view(torch.int8)[p, :, :, :n] = v.view(torch.int8).to(DEV)
                s = (torch.rand(2, self.hkv, generator=g) + 0.5) * 3.5 / QMAX[self.kind]
                self.scales[p] = (s if amp is None else s * amp[j % len(amp)]).to(DEV)
                self.sums[p, :, :n] = torch.rand(self.hkv, n, generator=g).to(DEV)
        return self

    def values(self, b, count=None, dtype=np.float64):
        """[2, Hkv, count, D] stored values of sequence b."""
        count = self.ctx[b] if count is None else count
        pages = self.table[b, :-(-count // self.page)].long()
        v = self.codes.view(torch.int8)[pages].view(self.kind).float().cpu().numpy().astype(dtype)
        s = self.scales[pages].cpu().numpy().astype(dtype)
        return (v * s[..., None, None]).transpose(1, 2, 0, 3, 4).reshape(2, self.hkv, -1, D)[:, :, :count]

    def raw(self, b, count):
        pages = self.table[b, :-(-count // self.page)].long()
        v = self.codes.view(torch.int8)[pages].cpu().numpy()
        return v.transpose(1, 2, 0, 3, 4).reshape(2, self.hkv, -1, D)[:, :, :count]


def _cu(news):
    return torch.tensor([0, *np.cumsum(news)], dtype=torch.int32, device=DEV)


def _encode(x, kind):
    """fp32 values over their scale -> code bytes."""
    q = np.float32(QMAX[kind])
    x = np.clip(x, -q, q)
    if kind == torch.int8:
        return np.rint(x).astype(np.int8)
    return torch.from_numpy(np.ascontiguousarray(x)).to(torch.float8_e4m3fn).view(torch.int8).numpy()


def _decode(codes, kind):
    return torch.from_numpy(np.ascontiguousarray(codes)).view(kind).float().numpy()


# ------------------------------------------------------------------------------ append
def _plain_append(old_codes, old_scale, old_n, new, kind):
    """One run: codes int8 [old_n, D], scale, new fp32 [n, D] -> (codes [old_n + n, D], scale)."""
    f = np.float32
    finite = np.where(np.isfinite(new), np.abs(new), 0).max(initial=0).astype(f)
    was = f(old_scale) if old_n else f(0)
    now = max(was, f(finite / f(QMAX[kind])))
    safe = now if now > 0 else f(1)
    with np.errstate(invalid="ignore", over="ignore"):
        new_codes = _encode(np.where(np.isnan(new), f(0), new / safe).astype(f), kind)
    if now > was and old_n:
        old_codes = _encode((_decode(old_codes, kind) * was / safe).astype(f), kind)
    return np.concatenate([old_codes, new_codes]), now


def _append_and_check(cache, news, seed=3, amp=1.0, edit=None, sums=True):
    g = torch.Generator().manual_seed(seed)
    T, hkv = sum(news), cache.hkv
    qkv = (torch.randn(T, (3 + 2 * hkv) * D, generator=g) * amp).to(torch.bfloat16)
    if edit is not None:
        edit(qkv)
    dev = qkv.to(DEV)
    k, v = dev[:, 3 * D:(3 + hkv) * D], dev[:, (3 + hkv) * D:]
    before = [cache.raw(b, c - m) for b, (c, m) in enumerate(zip(cache.ctx, news))]
    scales0 = cache.scales.cpu().numpy().copy()
    untouched = cache.codes.view(torch.int8).cpu().clone()
    sums0 = cache.sums.cpu().clone()
    _C.kv8_append(k, v, cache.codes, cache.scales, cache.table, _cu(news), cache.lens, max_new=max(news),
                  sums=cache.sums if sums else None)
    assert _C.take_device_error() == 0
    codes, scales = cache.codes.view(torch.int8).cpu(), cache.scales.cpu().numpy()
    sums1 = cache.sums.cpu()
    x = torch.stack([k, v]).float().cpu().numpy().reshape(2, T, hkv, D)
    seen = torch.zeros(untouched.shape[:4], dtype=torch.bool)
    r0, P = 0, cache.page
    for b, (c, m) in enumerate(zip(cache.ctx, news)):
        for j in range((c - m) // P, -(-c // P) if m else 0):
            p = int(cache.table[b, j])
            lo, hi = max(j * P, c - m), min((j + 1) * P, c)
            old_n = lo - j * P
            for side in range(2):
                for h in range(hkv):
                    new = x[side, r0 + lo - (c - m):r0 + hi - (c - m), h]
                    want, now = _plain_append(before[b][side, h, j * P:lo], scales0[p, side, h], old_n, new, cache.kind)
                    assert scales[p, side, h] == now, (b, j, side, h)
                    assert np.array_equal(codes[p, side, h, :hi - j * P].numpy(), want), (b, j, side, h)
                    # in 64 bits: within half a step of the type (plus the rounding of the scale)
                    fin = np.isfinite(new)
                    val = _decode(want[old_n:], cache.kind).astype(np.float64) * np.float64(now)
                    step = 0.5 * now if cache.kind == torch.int8 else np.maximum(np.abs(new) / 16, now * 2.0 ** -10)
                    assert (np.abs(val - new) <= step * (1 + 1e-5) + 1e-37)[fin].all()
            seen[p, :, :, :hi - j * P] = True
            if sums:
                assert (sums1[p, :, lo - j * P:hi - j * P] == 0).all()
                sums0[p, :, lo - j * P:hi - j * P] = 0
        r0 += m
    keep = ~seen.unsqueeze(-1).expand_as(codes)
    assert torch.equal(codes[keep], untouched[keep])            # nothing else was written
    assert torch.equal(sums1.nan_to_num(nan=-1.0), sums0.nan_to_num(nan=-1.0))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page", PAGES)
@pytest.mark.parametrize("hkv", [1, 2, 5])
def test_append_first_pass(kind, page, hkv):
    ctx = [1, page - 1, page, page + 1, 3 * page + 5, 200]
    _append_and_check(Cache(kind, page, hkv, ctx), ctx)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page", PAGES)
@pytest.mark.parametrize("amp", [0.01, 1.0, 50.0])     # scales that stay, may grow, and grow
def test_append_to_filled_pages(kind, page, amp):
    ctx, news = [3, page + 1, 2 * page, 2 * page + 7, 150, 260], [1, 1, 3, 0, page + 9, 2]
    _append_and_check(Cache(kind, page, 3, ctx).fill(), news, amp=amp)


@pytest.mark.parametrize("kind", KINDS)
def test_append_token_by_token(kind):
    """Every token is within the steps it was rounded with: at most half a step of the final scale
    for each time that the scale grew (int8), and its own."""
    hkv, n = 2, 70
    cache = Cache(kind, 32, hkv, [n])
    g = torch.Generator().manual_seed(5)
    x = (torch.randn(2, n, hkv * D, generator=g) * torch.linspace(0.2, 3.0, n).view(1, -1, 1)).to(torch.bfloat16).to(DEV)
    grew = torch.zeros(3, 2, hkv)
    for t in range(n):
        was = cache.scales[cache.table[0].long()].cpu()
        _C.kv8_append(x[0, t:t + 1], x[1, t:t + 1], cache.codes, cache.scales, cache.table, _cu([1]),
                      torch.tensor([t + 1], dtype=torch.int32, device=DEV), max_new=1)
        grew += (cache.scales[cache.table[0].long()].cpu() != was).float()
    got = cache.values(0)
    want = x.view(2, n, hkv, D).double().cpu().numpy().transpose(0, 2, 1, 3)
    s = cache.scales[cache.table[0].long()].cpu().numpy().transpose(1, 2, 0).repeat(32, 2)[:, :, :n, None]
    times = grew.numpy().transpose(1, 2, 0).repeat(32, 2)[:, :, :n, None]
    step = 0.5 * s if kind == torch.int8 else np.maximum(np.abs(want) / 16 * 1.2, s * 2.0 ** -10)
    assert (np.abs(got - want) <= step * times * (1 + 1e-4)).all()


@pytest.mark.parametrize("kind", KINDS)
def test_append_special_values(kind):
    def edit(qkv):
        qkv[0, 3 * D:] = 0                                   # a token of zeros
        qkv[2, 3 * D + 5] = float("inf")
        qkv[2, 3 * D + 6] = float("-inf")
        qkv[3, 3 * D + 7] = float("nan")
        qkv[4, 4 * D:5 * D] = 1e-38                           # near the least normal number
        qkv[5, 4 * D + 1] = 3e38
    _append_and_check(Cache(kind, 16, 2, [1, 3, 2]), [1, 3, 2], edit=edit)
    zero = Cache(kind, 16, 2, [20])
    _append_and_check(zero, [20], edit=lambda q: q.zero_())
    assert (zero.scales[zero.table[0].long()] == 0).all()


def test_append_reports_bad_pages_and_lengths():
    cache = Cache(torch.int8, 16, 2, [20, 20])
    k = torch.randn(4, 2 * D, device=DEV).to(torch.bfloat16)
    before = cache.codes.clone()
    for table, cu, lens in (
            (torch.full_like(cache.table, cache.num_pages), _cu([2, 2]), cache.lens),
            (torch.full_like(cache.table, -1), _cu([2, 2]), cache.lens),
            (cache.table, _cu([2, 7]), cache.lens),                       # more rows than there are
            (cache.table, _cu([2, 2]), cache.lens + 100),                 # past the table
            (cache.table, _cu([2, 2]), torch.zeros_like(cache.lens))):    # fewer tokens than new ones
        _C.kv8_append(k, k, cache.codes, cache.scales, table, cu, lens, max_new=2)
        assert _C.take_device_error() == 1
    # (sequence 0 of the third call is in order and was written)
    diff = (cache.codes != before).nonzero()[:, 0].unique().tolist()
    assert set(diff) <= set(cache.table[0].tolist())


# ------------------------------------------------------------------------------ read
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page", PAGES)
def test_read(kind, page):
    cache = Cache(kind, page, 3, [2 * page, page]).fill()
    pages = cache.table[0, :2].repeat(2)
    got = _C.kv8_read(cache.codes, cache.scales, pages)
    want = cache.codes.view(torch.int8)[pages.long()].view(kind).float() * cache.scales[pages.long()][..., None, None]
    assert torch.equal(got, want.to(torch.bfloat16))
    got = _C.kv8_read(cache.codes, cache.scales, torch.tensor([-1, cache.num_pages], dtype=torch.int32, device=DEV))
    assert (got == 0).all() and _C.take_device_error() == 1
    assert _C.kv8_read(cache.codes, cache.scales, pages[:0]).shape == (0, 2, 3, page, D)


# ------------------------------------------------------------------------------ attention
def _attend_and_check(cache, news, heads, seed=7, sums=False, amp=1.0, max_new=None, special=None, ctx=None):
    ctx = cache.ctx if ctx is None else ctx
    g = torch.Generator().manual_seed(seed)
    T, hkv = sum(news), cache.hkv
    G = heads // hkv
    q = (torch.randn(T, (heads + 2 * hkv) * D, generator=g) * amp).to(torch.bfloat16).to(DEV)[:, :heads * D]
    if special is not None:
        special(q)
    scale = D ** -0.5
    out = torch.full((T, heads * D), float("nan"), dtype=torch.bfloat16, device=DEV)
    sums0 = cache.sums.double().cpu().numpy()
    got = _C.kv8_attention(q, cache.codes, cache.scales, cache.table, _cu(news), cache.lens, heads, scale,
                           max_new=max(max(news), 1) if max_new is None else max_new, out=out,
                           sums=cache.sums if sums else None)
    assert got is out and _C.take_device_error() == 0
    got = got.double().cpu().numpy().reshape(T, heads, D)
    sums1 = cache.sums.double().cpu().numpy()
    qd = q.double().cpu().numpy().reshape(T, heads, D)
    r0 = 0
    for b, (c, m) in enumerate(zip(ctx, news)):
        if m == 0:
            continue
        kv = cache.values(b, c) if c else np.zeros((2, hkv, 0, D))
        for h in range(hkv):
            rows = qd[r0:r0 + m, h * G:(h + 1) * G]                      # [m, G, D]
            x = np.einsum("igd,td->igt", rows, kv[0, h]) * scale
            size = (np.einsum("igd,td->igt", np.abs(rows), np.abs(kv[0, h])) * scale).max(initial=0)
            d = 12 * 2.0 ** -22 * size + 2.0 ** -20 * np.abs(x).max(initial=0) + 2.0 ** -20
            x = np.where(np.arange(c)[None, None] > (c - m + np.arange(m))[:, None, None], -np.inf, x)
            top = x.max(-1, keepdims=True, initial=-np.inf)
            w = np.exp(x - np.where(np.isfinite(top), top, 0))
            w = w / np.maximum(w.sum(-1, keepdims=True), 1e-300)
            want = np.einsum("igt,td->igd", w, kv[1, h])
            mag = np.einsum("igt,td->igd", w, np.abs(kv[1, h]))
            tol = (2 * d + 2.0 ** -11 + 2.0 ** -18) * mag + 2.0 ** -35 * c * np.abs(kv[1, h]).max(initial=0) + 2.0 ** -8 * np.abs(want)
            off = np.abs(got[r0:r0 + m, h * G:(h + 1) * G] - want)
            assert (off <= tol).all(), (b, h, (off - tol).max(), np.argwhere(~(off <= tol))[0])
            if sums:
                t = np.arange(c)
                p = cache.table[b].cpu().numpy()[t // cache.page] if c else t
                have = sums1[p, h, t % cache.page]
                old = sums0[p, h, t % cache.page]
                add = w.sum((0, 1))
                assert (np.abs(have - (old + add)) <= (2 * d + 2.0 ** -20 * m * G) * add + 2.0 ** -22 * (old + add) + 1e-30).all(), (b, h)
        r0 += m
    if not sums:
        assert np.array_equal(np.nan_to_num(sums1, nan=-1), np.nan_to_num(sums0, nan=-1))
    return got


EDGE_CTX = [1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 500, 1000]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page", PAGES)
@pytest.mark.parametrize("heads,hkv", [(2, 2), (4, 2), (3, 1), (8, 1), (10, 2), (16, 1), (20, 1)])
@pytest.mark.parametrize("sums", [False, True])
def test_attention_single_tokens(kind, page, heads, hkv, sums):
    _attend_and_check(Cache(kind, page, hkv, EDGE_CTX).fill(), [1] * len(EDGE_CTX), heads, sums=sums)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("heads,hkv", [(2, 2), (6, 1), (8, 2)])
@pytest.mark.parametrize("sums", [False, True])
def test_attention_several_tokens(kind, page, heads, hkv, sums):
    ctx, news = [1, 5, 33, 64, 130, 300, 700], [1, 5, 2, 0, 17, 40, 3]
    _attend_and_check(Cache(kind, page, hkv, ctx).fill(), news, heads, sums=sums)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("batch", [1, 3, 40, 700])
def test_attention_work_split(kind, batch):
    """One long sequence cut among many blocks; many short ones sharing them; both at once."""
    rng = np.random.default_rng(batch)
    ctx = [6000] + [int(n) for n in np.exp(rng.uniform(0, np.log(400), batch - 1))]
    _attend_and_check(Cache(kind, 32, 2, ctx).fill(), [1] * batch, 4)


@pytest.mark.parametrize("new", [1, 5, 17])
@pytest.mark.parametrize("sums", [False, True])
def test_attention_many_items(new, sums):
    """More units than blocks, so that shares count the items' beginnings; sequences without new tokens
    among them, tiles of 8, 16 and 32 rows, the last of an item not full."""
    rng = np.random.default_rng(new)
    ctx = [1, 4000] + [int(n) for n in np.exp(rng.uniform(np.log(20), np.log(2500), 68))]
    news = [min(c, int(n)) for c, n in zip(ctx, rng.integers(0, new + 1, 70))]
    news[5] = new
    _attend_and_check(Cache(torch.int8, 16, 3, ctx).fill(), news, 6, sums=sums, max_new=new)


def test_one_row_may_have_any_stride():
    cache = Cache(torch.int8, 16, 2, [40]).fill()
    other = Cache(torch.int8, 16, 2, [40]).fill()
    rows = torch.randn(3, 4 * D, device=DEV).to(torch.bfloat16)
    got = []
    for c, (q, k, v) in ((cache, [r[None] for r in rows]), (other, [r[:, None].t() for r in rows])):
        k, v = k[:, :2 * D], v[:, :2 * D]
        _C.kv8_append(k, v, c.codes, c.scales, c.table, _cu([1]), c.lens, max_new=1)
        got.append((_C.kv8_attention(q, c.codes, c.scales, c.table, _cu([1]), c.lens, 4, 0.1, max_new=1), c.codes))
    assert got[1][0].isfinite().all() and all(torch.equal(a, b) for a, b in zip(*got))


@pytest.mark.parametrize("sums", [False, True])
def test_attention_of_a_long_text_by_itself(sums):
    """Every token of a text in one call: the first sees itself only."""
    _attend_and_check(Cache(torch.int8, 64, 2, [300, 1]).fill(), [300, 1], 4, sums=sums)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads", [2, 24])
def test_attention_rows_that_see_nothing(kind, heads):
    """More query rows than cached tokens: the first rows see nothing and are zeros."""
    cache = Cache(kind, 16, 2, [0, 2, 40]).fill()
    got = _attend_and_check(cache, [2, 5, 1], heads, sums=True)
    assert (got[:2] == 0).all() and (got[2:5] == 0).all() and not (got[5:] == 0).all()


@pytest.mark.parametrize("kind", KINDS)
def test_attention_scales_of_any_size(kind):
    """V scales far apart, far from 1, and pages of zeros: weights stay what they are."""
    for amp in ([1e-12, 1.0, 1e-3], [1e10, 1.0], [1.0, 0.0]):
        cache = Cache(kind, 16, 1, [100, 40]).fill(amp=amp)
        cache.scales[:, 0] = cache.scales[:, 0].clamp(max=0.1, min=1e-3).nan_to_num(nan=float("nan"))
        _attend_and_check(cache, [1, 2], 2, sums=True)


def test_attention_large_logits():
    """Logits of hundreds, one key taking all the weight."""
    _attend_and_check(Cache(torch.int8, 32, 2, [400, 33]).fill(), [1, 1], 4, amp=60.0)


def test_attention_tiny_and_nonfinite_queries():
    cache = Cache(torch.int8, 32, 1, [50, 50, 50]).fill()
    _attend_and_check(cache, [1, 1, 1], 2, amp=1e-30)
    q = torch.randn(3, 2 * D, device=DEV).to(torch.bfloat16)
    base = _C.kv8_attention(q, cache.codes, cache.scales, cache.table, _cu([1, 1, 1]), cache.lens, 2, 0.1, max_new=1)
    q[1, 3] = float("nan")
    got = _C.kv8_attention(q, cache.codes, cache.scales, cache.table, _cu([1, 1, 1]), cache.lens, 2, 0.1, max_new=1)
    assert got[1, :D].isnan().all()
    assert torch.equal(got[1, D:], base[1, D:]) and torch.equal(got[[0, 2]], base[[0, 2]])


def test_attention_bounds_may_be_loose():
    """max_new above the real one picks the larger row tiles; the result stays right."""
    cache = Cache(torch.float8_e4m3fn, 32, 2, [90, 300]).fill()
    _attend_and_check(cache, [4, 4], 4, max_new=8)
    _attend_and_check(cache, [1, 7], 4, max_new=8)


def test_attention_repeats_bit_for_bit_and_on_another_stream():
    cache = Cache(torch.int8, 64, 2, [3000, 70, 1]).fill()
    q = torch.randn(3, 8 * D, device=DEV).to(torch.bfloat16)

    def call():
        return _C.kv8_attention(q, cache.codes, cache.scales, cache.table, _cu([1, 1, 1]), cache.lens, 8, 0.1, max_new=1)
    a = call()
    assert torch.equal(a, call())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = call()
    side.synchronize()
    assert torch.equal(a, b)


def test_attention_leaves_sms_to_others():
    """With SMs reserved for other kernels the shares change, the result does not."""
    cache = Cache(torch.int8, 64, 2, [5000, 70]).fill()
    _C.set_sm_reserve(32)
    try:
        _attend_and_check(cache, [1, 1], 4)
    finally:
        _C.set_sm_reserve(0)


def test_cache_of_more_than_32_bits():
    """Pages whose bytes lie past 2^32: written, read and attended to."""
    page, hkv = 128, 8
    num = 2 ** 32 // (2 * hkv * page * D) + 40
    codes = torch.empty(num, 2, hkv, page, D, dtype=torch.int8, device=DEV)
    scales = torch.empty(num, 2, hkv, device=DEV)
    sums = torch.zeros(num, hkv, page, device=DEV)
    small = Cache(torch.int8, page, hkv, [300])
    table = torch.tensor([[num - 1, 3, num - 20]], dtype=torch.int32, device=DEV)
    k, v = (torch.randn(300, hkv * D, device=DEV).to(torch.bfloat16) for _ in range(2))
    q = torch.randn(1, 16 * D, device=DEV).to(torch.bfloat16)
    got, lens = [], small.lens
    for c, s, t in ((codes, scales, table), (small.codes, small.scales, small.table)):
        w = sums if c is codes else small.sums
        _C.kv8_append(k, v, c, s, t, _cu([300]), lens, max_new=300, sums=w)
        o = _C.kv8_attention(q, c, s, t, _cu([1]), lens, 16, 0.09, max_new=1, sums=w)
        got.append((o, _C.kv8_read(c, s, t.reshape(-1))[:2], w[t.reshape(-1).long()][:2]))
    assert _C.take_device_error() == 0
    for a, b in zip(*got):
        assert torch.equal(a, b)
    # and moved: the other end of the pool keeps the last 200 of them
    kept, new = _C.kv8_evict(codes, scales, sums, table, lens, torch.tensor([[num - 2, num - 30]], dtype=torch.int32, device=DEV), 200, 200)
    assert torch.equal(kept, torch.arange(100, 300, dtype=torch.int32, device=DEV).expand(1, hkv, 200))
    last = _C.kv8_read(codes, scales, torch.tensor([num - 30], dtype=torch.int32, device=DEV))
    kv = torch.stack([k, v]).view(2, 300, hkv, D)[:, 228:].transpose(1, 2).float()
    assert ((last[0, :, :, :72].float() - kv).abs() < 0.05).all()


def test_attention_reports_bad_pages_and_lengths():
    cache = Cache(torch.int8, 16, 2, [20, 20]).fill()
    q = torch.randn(2, 4 * D, device=DEV).to(torch.bfloat16)

    def call(table, cu, lens):
        return _C.kv8_attention(q, cache.codes, cache.scales, table, cu, lens, 4, 0.1, max_new=1)
    good = call(cache.table, _cu([1, 1]), cache.lens)
    assert _C.take_device_error() == 0
    bad = cache.table.clone()
    bad[1] = cache.num_pages + 5
    got = call(bad, _cu([1, 1]), cache.lens)
    assert _C.take_device_error() == 1
    assert torch.allclose(got[0].float(), good[0].float(), rtol=0.02, atol=1e-3)
    call(cache.table, _cu([1, 1]), cache.lens + 1000)
    assert _C.take_device_error() == 1
    call(cache.table, _cu([1, 5]), cache.lens)
    assert _C.take_device_error() == 1
    call(cache.table, _cu([2, 0]), cache.lens)               # more new tokens than max_new
    assert _C.take_device_error() == 1


# ------------------------------------------------------------------------------ evict
def _evict_and_check(kind, page, hkv, ctx, keep, recent, sums=None, seed=11, amp=None):
    per = -(-keep // page)
    cache = Cache(kind, page, hkv, ctx, extra=2 + len(ctx) * per).fill(amp=amp)
    if sums is not None:
        sums(cache)
    used = set(cache.table[cache.table >= 0].tolist())
    free = [p for p in range(cache.num_pages) if p not in used][:len(ctx) * per]
    new_table = torch.tensor(free, dtype=torch.int32, device=DEV).view(len(ctx), per)
    before, scales0, sums0 = cache.codes.view(torch.int8).cpu().numpy().copy(), cache.scales.cpu().numpy().copy(), cache.sums.cpu().numpy().copy()
    kept, lens = _C.kv8_evict(cache.codes, cache.scales, cache.sums, cache.table, cache.lens, new_table, keep, recent)
    assert _C.take_device_error() == 0
    codes, scales, sums1 = cache.codes.view(torch.int8).cpu().numpy(), cache.scales.cpu().numpy(), cache.sums.cpu().numpy()
    kept, f = kept.cpu().numpy(), np.float32
    assert lens.tolist() == [min(c, keep) for c in ctx]
    table, nt = cache.table.cpu().numpy(), new_table.cpu().numpy()
    for b, c in enumerate(ctx):
        t = np.arange(c)
        for h in range(hkv):
            mine = sums0[table[b, t // page], h, t % page].astype(np.float64)
            if c <= keep:
                want = t
            else:
                old = c - recent
                rank = np.where(np.isnan(mine[:old]), -np.inf, mine[:old])
                best = np.lexsort((np.arange(old), np.isnan(mine[:old]), -rank))[:keep - recent]
                want = np.concatenate([np.sort(best), t[old:]])
            assert np.array_equal(kept[b, h, :len(want)], want), (b, h)
            assert (kept[b, h, len(want):] == -1).all()
            for j in range(per):
                src = want[j * page:(j + 1) * page]
                p, n = nt[b, j], len(want[j * page:(j + 1) * page])
                assert np.array_equal(sums1[p, h, :n], sums0[table[b, src // page], h, src % page], equal_nan=True)
                assert (sums1[p, h, n:] == 0).all()
                for side in range(2):
                    was = scales0[table[b, src // page], side, h]
                    now = was.max(initial=0).astype(f)
                    assert scales[p, side, h] == now
                    got = codes[p, side, h]
                    assert (got[n:] == 0).all()
                    raw = before[table[b, src // page], side, h, src % page]
                    safe = now if now > 0 else f(1)
                    again = _encode((_decode(raw, kind) * was[:, None] / safe).astype(f), kind) if n else raw
                    expect = np.where((was == now)[:, None], raw, again)
                    assert np.array_equal(got[:n], expect), (b, h, j, side)
    old_pages = sorted(used)
    assert np.array_equal(codes[old_pages], before[old_pages])            # the sources are left alone
    assert np.array_equal(scales[old_pages], scales0[old_pages])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page", PAGES)
@pytest.mark.parametrize("keep,recent", [(1, 0), (1, 1), (50, 0), (50, 13), (50, 50), (257, 100)])
def test_evict(kind, page, keep, recent):
    _evict_and_check(kind, page, 2, [1, 49, 50, 51, 300, 700], keep, recent)


@pytest.mark.parametrize("ctx,keep,recent", [([5000, 4097, 20], 1000, 77), ([40000], 12345, 1), ([9000, 33], 8999, 4000)])
def test_evict_long(ctx, keep, recent):
    """Selections spread over several blocks."""
    _evict_and_check(torch.int8, 64, 3, ctx, keep, recent)


def test_evict_ties_and_special_sums():
    def equal(cache):
        cache.sums.fill_(0.25)

    def few(cache):
        cache.sums.copy_((cache.sums * 3).nan_to_num().floor())

    def special(cache):
        flat = cache.sums.view(-1)
        flat[::3] = 0.0
        flat[1::7] = -0.0
        flat[2::11] = float("inf")
        flat[3::13] = float("nan")
        flat[4::17] = 1e-40
        flat[5::19] = -2.0
    for sums in (equal, few, special):
        _evict_and_check(torch.int8, 16, 2, [100, 333, 6000], 90, 10, sums)


@pytest.mark.parametrize("kind", KINDS)
def test_evict_scales_far_apart(kind):
    _evict_and_check(kind, 16, 2, [200, 90], 64, 20, amp=[1.0, 1e-4, 300.0, 0.0])


# ------------------------------------------------------------------------------ refusals
def test_short_tables_need_no_workspace():
    """Up to 512 tokens of table one kernel and no workspace; past it, and with sums, both are needed."""
    lib, stream = _C.lib(), torch.cuda.current_stream().cuda_stream
    for page, width, sums, want in ((16, 32, False, 0), (16, 33, False, 2), (128, 4, False, 0), (128, 5, False, 2), (16, 32, True, 2)):
        cache = Cache(torch.int8, page, 2, [page * width]).fill()
        q, out = torch.randn(1, 4 * D, device=DEV).to(torch.bfloat16), torch.zeros(1, 4 * D, dtype=torch.bfloat16, device=DEV)
        cu = _cu([1])
        st = lib.mes_kv8_attention(0, q.data_ptr(), 4 * D, cache.codes.data_ptr(), cache.scales.data_ptr(),
                                   cache.sums.data_ptr() if sums else None, cache.table.data_ptr(), width, cu.data_ptr(),
                                   cache.lens.data_ptr(), 1, 1, 1, 4, 2, D, page, cache.num_pages, 0.1, out.data_ptr(), None,
                                   0, stream)
        assert (st != 0) == (want != 0), (page, width, sums, st)
        before = _C.launch_count
        got = _C.kv8_attention(q, cache.codes, cache.scales, cache.table, cu, cache.lens, 4, 0.1, max_new=1,
                               sums=cache.sums if sums else None)
        assert _C.launch_count - before == (1 if page * width <= 512 else 2) + sums
        assert st != 0 or torch.equal(got, out)


def test_refusals():
    cache = Cache(torch.int8, 32, 2, [40]).fill()
    k = torch.zeros(1, 2 * D, dtype=torch.bfloat16, device=DEV)
    q = torch.zeros(1, 4 * D, dtype=torch.bfloat16, device=DEV)
    c, s, w, t, l, cu = cache.codes, cache.scales, cache.sums, cache.table, cache.lens, _cu([1])
    nt = torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    for bad in (
            lambda: _C.kv8_append(k, k, c.view(torch.uint8), s, t, cu, l, 1),
            lambda: _C.kv8_append(k.float(), k, c, s, t, cu, l, 1),
            lambda: _C.kv8_append(k, k[:, :D], c, s, t, cu, l, 1),
            lambda: _C.kv8_append(k, k, c, s.double(), t, cu, l, 1),
            lambda: _C.kv8_append(k, k, c, s, t.long(), cu, l, 1),
            lambda: _C.kv8_append(k, k, c, s, t, cu[:1], l, 1),
            lambda: _C.kv8_append(k, k, c, s, t, cu, l, 2),                    # max_new above T
            lambda: _C.kv8_append(k.cpu(), k, c, s, t, cu, l, 1),
            lambda: _C.kv8_append(k, k, c[:, :, :, :8], s, t, cu, l, 1),      # no page of 8
            lambda: _C.kv8_append(torch.zeros(1, 2 * D + 4, dtype=torch.bfloat16, device=DEV)[:, 4:], k, c, s, t, cu, l, 1),
            lambda: _C.kv8_read(c, s, t),
            lambda: _C.kv8_attention(q, c, s, t, cu, l, 3, 0.1, 1),
            lambda: _C.kv8_attention(q[:, :3 * D], c, s, t, cu, l, 3, 0.1, 1),   # 3 heads over 2
            lambda: _C.kv8_attention(q, c, s, t, cu, l, 4, 0.1, 1, sums=w[:1]),
            lambda: _C.kv8_attention(q, c, s, t, cu, l, 4, 0.1, 1, out=torch.empty(1, 4 * D, device=DEV)),
            lambda: _C.kv8_attention(q, c, s, t.expand(1025, -1).contiguous(), _cu([1] + [0] * 1024),
                                     l.expand(1025).contiguous(), 4, 0.1, 1),
            lambda: _C.kv8_evict(c, s, None, t, l, nt, 20, 5),
            lambda: _C.kv8_evict(c, s, w, t, l, nt, 20, 21),
            lambda: _C.kv8_evict(c, s, w, t, l, nt, 0, 0),
            lambda: _C.kv8_evict(c, s, w, t, l, nt, 33, 5)):                   # needs two new pages
        with pytest.raises(_C.MesError):
            bad()
    assert _C.take_device_error() == 0


def test_empty_batches():
    cache = Cache(torch.int8, 32, 2, [40]).fill()
    none = torch.zeros(0, 4 * D, dtype=torch.bfloat16, device=DEV)
    assert _C.kv8_attention(none, cache.codes, cache.scales, cache.table, _cu([0]), cache.lens, 4, 0.1, max_new=0).shape == (0, 4 * D)
    before = cache.codes.clone()
    _C.kv8_append(none[:, :2 * D], none[:, :2 * D], cache.codes, cache.scales, cache.table, _cu([0]), cache.lens, max_new=0)
    assert torch.equal(cache.codes.view(torch.int8), before.view(torch.int8))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("news,max_new", [([5, 1, 2], 2), ([1, 100, 2], 2), ([70, 70, 3], 69), ([2, 2, 2], 1)])
def test_append_skips_more_new_tokens_than_max_new(kind, page, news, max_new):
    """Whether they would fit the pages that the call reckons with or not: the sequence's pages stay as they are, the
    others are written, and the call is recorded."""
    ctx, hkv = [8 + news[0], 150, 40], 2
    made = [Cache(kind, page, hkv, ctx).fill() for _ in range(2)]
    g = torch.Generator().manual_seed(4)
    k, v = ((torch.randn(sum(news), hkv * D, generator=g) * 3).to(torch.bfloat16).to(DEV) for _ in range(2))
    got, want = made
    _C.kv8_append(k, v, got.codes, got.scales, got.table, _cu(news), got.lens, max_new=max_new, sums=got.sums)
    assert _C.take_device_error() == 1
    r0 = 0
    for b, n in enumerate(news):
        if n <= max_new:
            _C.kv8_append(k[r0:r0 + n], v[r0:r0 + n], want.codes, want.scales, want.table[b:b + 1], _cu([n]),
                          want.lens[b:b + 1], max_new=n, sums=want.sums)
        r0 += n
    assert _C.take_device_error() == 0
    for a, b in ((got.codes.view(torch.int8), want.codes.view(torch.int8)), (got.scales, want.scales), (got.sums, want.sums)):
        assert torch.equal(a.nan_to_num(nan=-1) if a.is_floating_point() else a, b.nan_to_num(nan=-1) if b.is_floating_point() else b)


def test_evict_counts_a_length_outside_the_table_as_nothing():
    """It is recorded, keeps no token and has empty new pages; the other sequences are not affected."""
    ctx, keep, page = [100, 90, 80], 40, 16
    for bad in (-1, 7 * page + 1, 2 ** 31 - 1):
        cache = Cache(torch.int8, page, 2, ctx, extra=9).fill()
        used = set(cache.table[cache.table >= 0].tolist())
        new_table = torch.tensor([p for p in range(cache.num_pages) if p not in used], dtype=torch.int32, device=DEV).view(3, 3)
        lens = cache.lens.clone()
        want, want_lens = _C.kv8_evict(cache.codes, cache.scales, cache.sums, cache.table, lens, new_table, keep, 8)
        pages = [t.clone() for t in (cache.codes, cache.scales, cache.sums)]
        assert _C.take_device_error() == 0
        lens[1] = bad
        got, got_lens = _C.kv8_evict(cache.codes, cache.scales, cache.sums, cache.table, lens, new_table, keep, 8)
        assert _C.take_device_error() == 1
        assert got_lens.tolist() == [40, 0, 40] and want_lens.tolist() == [40, 40, 40]
        assert (got[1] == -1).all() and torch.equal(got[[0, 2]], want[[0, 2]])
        empty = new_table[1].long()
        for a, b in zip((cache.codes, cache.scales, cache.sums), pages):
            assert (a[empty] == 0).all()
            b[empty] = 0
            assert torch.equal(a.nan_to_num(nan=-1) if a.is_floating_point() else a, b.nan_to_num(nan=-1) if b.is_floating_point() else b)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page", [16, 32])
def test_values_through_many_evictions(kind, page):
    """A window that slides over a stream.  A value is rounded when it is written, each time its page's scale
    grows and each time a compaction changes its scale, and scales never shrink on the way, so int8 values are
    within half a step of the present scale for each of those.  An e4m3 rounding is within 2^-4 of the present value
    or 2^-10 of the scale, and the value itself drifts by no more than those."""
    hkv, keep, rounds = 2, 48, 40
    per = -(-keep // page)
    pool = list(range(2 * per + 6))
    cache = Cache(kind, page, hkv, [1], extra=len(pool))
    g = torch.Generator().manual_seed(21)
    true, times, scale = (np.zeros((2, hkv, 0, D)), np.zeros((2, hkv, 0)), np.zeros((2, hkv, 0)))
    pages, most, rounded = [], 0, 0

    def present(pages, n):
        s = cache.scales[torch.tensor(pages, device=DEV)].double().cpu().numpy()      # [pages, 2, hkv]
        return np.repeat(s.transpose(1, 2, 0), page, 2)[:, :, :n]
    cache.sums.zero_()
    for r in range(rounds):
        m = int(torch.randint(1, 20, (1,), generator=g))
        new = torch.randn(2, m, hkv * D, generator=g) * torch.exp(torch.randn(1, m, 1, generator=g))
        new = new.to(torch.bfloat16)
        n = true.shape[2] + m
        while len(pages) * page < n:
            pages.append(pool.pop())
        table = torch.tensor([pages], dtype=torch.int32, device=DEV)
        lens = torch.tensor([n], dtype=torch.int32, device=DEV)
        _C.kv8_append(new[0].to(DEV), new[1].to(DEV), cache.codes, cache.scales, table, _cu([m]), lens, max_new=m, sums=cache.sums)
        now = present(pages, n)
        assert (now[:, :, :n - m] >= scale).all()
        times = np.concatenate([times + (now[:, :, :n - m] != scale), np.ones((2, hkv, m))], 2)
        true = np.concatenate([true, new.double().numpy().reshape(2, m, hkv, D).transpose(0, 2, 1, 3)], 2)
        scale = now
        if n > keep:
            to = [pool.pop() for _ in range(per)]
            kept, _ = _C.kv8_evict(cache.codes, cache.scales, cache.sums, table, lens,
                                   torch.tensor([to], dtype=torch.int32, device=DEV), keep, keep)
            assert torch.equal(kept[0, 0], torch.arange(n - keep, n, dtype=torch.int32, device=DEV))
            pool += pages
            pages, n = to, keep
            true, times, scale = true[:, :, -keep:], times[:, :, -keep:], scale[:, :, -keep:]
            now = present(pages, n)
            assert (now >= scale).all()
            times, scale = times + (now != scale), now
            rounded += 1
        p = torch.tensor(pages, device=DEV)
        codes = cache.codes.view(torch.int8)[p].view(kind).float().double().cpu().numpy()
        got = (codes * cache.scales[p].double().cpu().numpy()[..., None, None]).transpose(1, 2, 0, 3, 4).reshape(2, hkv, -1, D)[:, :, :n]
        t, s = times[..., None], scale[..., None]
        if kind == torch.int8:
            bound = 0.5 * s * t
        else:
            bound = t * ((1 + 2.0 ** -4) ** t * np.abs(true) / 16 + s * 2.0 ** -10 * (1 + 2.0 ** -4) ** t)
        assert (np.abs(got - true) <= bound * (1 + 1e-4)).all(), r
        most = max(most, int(times.max()))
    # it reaches what it is about: many compactions, values rounded more than twice again
    assert rounded > 20 and most > 3 and _C.take_device_error() == 0
