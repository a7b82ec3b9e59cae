"""The token-step operators' host side, on CPU: what the C entry points and the wrappers refuse before
anything is launched, and the page accounting of ``IncrementalEmbedder`` against a recording
stand-in for the library's launchers."""
import numpy as np
import pytest
import torch

from mes_b200 import _C, synthetic
from mes_b200.core.incremental import IncrementalEmbedder
from mes_b200.layers.kv_cache import CacheStep, KV8Cache
from mes_b200.models import Qwen3ForCausalLM
from mes_b200.schemas.config import MESConfig

A, ODD2, ODD4, ODD8 = 0x10000, 0x10002, 0x10004, 0x10008     # never dereferenced


def test_gemv_entry_point_refuses():
    f = _C.lib().mes_awq_gemv

    def call(epi=0, x=A, ldx=256, qw=A, qz=A, sc=A, bias=None, y=A, ldy=64, M=1, N=64, K=256, group=128):
        return f(epi, x, ldx, qw, qz, sc, bias, y, ldy, M, N, K, group, None)
    for kw in (dict(epi=3), dict(epi=-1), dict(M=17), dict(M=-1), dict(N=0), dict(N=60), dict(K=192), dict(K=0),
               dict(group=16), dict(group=256), dict(ldx=248), dict(ldx=260), dict(ldy=56), dict(epi=2, N=40, ldy=64),
               dict(epi=2, bias=A), dict(x=None), dict(qw=None), dict(qz=None), dict(sc=None), dict(y=None)):
        assert call(**kw) == 1, kw
    for kw in (dict(x=ODD8), dict(qw=ODD8), dict(sc=ODD4), dict(qz=ODD2), dict(bias=A + 1), dict(y=A + 1),
               dict(epi=1, y=ODD2)):
        assert call(**kw) == 2, kw
    assert call(M=0, x=None) == 0                               # no rows: nothing to do


def _append(dtype=0, k=A, ldk=256, v=A, ldv=256, codes=A, scales=A, sums=None, table=A, width=4, cu=A, lens=A, B=2,
            T=8, max_new=4, hkv=2, D=128, page=32, pages=100):
    return _C.lib().mes_kv8_append(dtype, k, ldk, v, ldv, codes, scales, sums, table, width, cu, lens, B, T, max_new, hkv,
                                   D, page, pages, None)


def _attention(dtype=0, q=A, ldq=512, codes=A, scales=A, sums=None, table=A, width=4, cu=A, lens=A, B=2, T=8, max_new=4,
               hq=4, hkv=2, D=128, page=32, pages=100, out=A, ws=A, size=1 << 40):
    return _C.lib().mes_kv8_attention(dtype, q, ldq, codes, scales, sums, table, width, cu, lens, B, T, max_new, hq, hkv, D,
                                      page, pages, 0.1, out, ws, size, None)


def _evict(dtype=0, codes=A, scales=A, sums=A, table=A, width=4, lens=A, B=2, new=A, new_width=2, keep=40, recent=10,
           hkv=2, D=128, page=32, pages=100, kept=A, new_lens=A):
    return _C.lib().mes_kv8_evict(dtype, codes, scales, sums, table, width, lens, B, new, new_width, keep, recent, hkv, D,
                                  page, pages, kept, new_lens, None)


def _read(dtype=0, codes=A, scales=A, pages=A, n=3, hkv=2, D=128, page=32, num=100, out=A):
    return _C.lib().mes_kv8_read(dtype, codes, scales, pages, n, hkv, D, page, num, out, None)


CACHE = [dict(dtype=2), dict(dtype=-1), dict(hkv=0), dict(D=64), dict(page=24), dict(page=256)]


def test_cache_entry_points_refuse():
    for f in (_append, _attention, _evict, _read):
        for kw in CACHE:
            assert f(**kw) == 1, (f.__name__, kw)
    too_many = 2 ** 31 // (2 * 2 * 32)                           # rows are counted in 32 bits
    for f in (_append, _attention, _evict):
        for kw in (dict(pages=0), dict(pages=too_many), dict(B=-1), dict(width=0), dict(codes=None), dict(scales=None),
                   dict(table=None), dict(lens=None)):
            assert f(**kw) == 1, (f.__name__, kw)
        for kw in (dict(codes=ODD8), dict(scales=ODD2), dict(sums=ODD2), dict(table=ODD2), dict(lens=ODD2)):
            assert f(**kw) == 2, (f.__name__, kw)
        assert f(B=0) == 0
    for kw in (dict(T=-1), dict(max_new=9), dict(max_new=-1), dict(ldk=248), dict(ldv=260), dict(k=None), dict(v=None),
               dict(cu=None)):
        assert _append(**kw) == 1, kw
    for kw in (dict(k=ODD8), dict(v=ODD8), dict(cu=ODD2)):
        assert _append(**kw) == 2, kw
    assert _append(T=0, max_new=0) == 0 and _append(max_new=0) == 0
    for kw in (dict(T=-1), dict(max_new=9), dict(hq=3), dict(hq=0), dict(ldq=504), dict(ldq=516), dict(B=1025), dict(q=None),
               dict(cu=None), dict(out=None), dict(ws=None, width=17), dict(size=0, width=17), dict(ws=None, sums=A),
               dict(size=0, sums=A)):       # a short table without sums needs no workspace
        assert _attention(**kw) == 1, kw
    for kw in (dict(q=ODD8), dict(out=ODD8), dict(ws=A + 128), dict(cu=ODD2)):
        assert _attention(**kw) == 2, kw
    assert _attention(T=0, max_new=0) == 0
    for kw in (dict(keep=0, new_width=0), dict(recent=41), dict(recent=-1), dict(new_width=1), dict(new_width=3), dict(sums=None),
               dict(new=None), dict(kept=None), dict(new_lens=None)):
        assert _evict(**kw) == 1, kw
    for kw in (dict(new=ODD2), dict(kept=ODD2), dict(new_lens=ODD2)):
        assert _evict(**kw) == 2, kw
    for kw in (dict(n=-1), dict(num=0), dict(codes=None), dict(scales=None), dict(pages=None), dict(out=None)):
        assert _read(**kw) == 1, kw
    for kw in (dict(codes=ODD8), dict(out=ODD8), dict(scales=ODD2), dict(pages=ODD2)):
        assert _read(**kw) == 2, kw
    assert _read(n=0) == 0


def test_attention_workspace_size():
    size = _C.lib().mes_kv8_attention_workspace_size
    base = size(4, 4, 8, 2, 1, 0)
    assert base > 0 and size(64, 64, 8, 2, 1, 0) == base         # lengths and sequences add nothing
    assert size(4, 4, 16, 2, 1, 0) == base and size(4, 4, 32, 2, 1, 0) > base        # 8 rows a kv head, then 16
    assert size(4, 4, 8, 2, 1, 1000) >= base + 4 * 4 * 8 * 1000                      # logits for the sums
    for bad in ((-1, 4, 8, 2, 1, 0), (4, 1025, 8, 2, 1, 0), (4, 4, 7, 2, 1, 0), (4, 4, 8, 0, 1, 0), (4, 4, 8, 2, 5, 0),
                (4, 4, 8, 2, 1, -1)):
        assert size(*bad) == -1, bad


class _RecordingLib:
    def __init__(self, real):
        self.real, self.calls = real, []

    def __getattr__(self, name):
        if name.endswith("_size") or name == "mes_status_string":
            return getattr(self.real, name)

        def launch(*args):
            self.calls.append(name)
            return 0
        return launch


@pytest.fixture
def rec(monkeypatch):
    fake = _RecordingLib(_C.lib())
    monkeypatch.setattr(_C, "lib", lambda: fake)
    monkeypatch.setattr(_C, "_stream", lambda t: 0)
    return fake


def test_wrappers_refuse_before_the_library(rec):
    bf, i32 = torch.bfloat16, torch.int32
    qw, qz, sc = (torch.zeros(32, 64, dtype=i32), torch.zeros(2, 8, dtype=i32), torch.zeros(2, 64, dtype=torch.float16))
    x = torch.zeros(3, 256, dtype=bf)
    codes, scales, sums = torch.zeros(9, 2, 2, 32, 128, dtype=torch.int8), torch.zeros(9, 2, 2), torch.zeros(9, 2, 32)
    table, lens, cu = torch.zeros(2, 3, dtype=i32), torch.zeros(2, dtype=i32), torch.zeros(3, dtype=i32)
    k, q, new = torch.zeros(4, 256, dtype=bf), torch.zeros(4, 512, dtype=bf), torch.zeros(2, 2, dtype=i32)
    c = (codes, scales, table, cu, lens)
    bad = [
        lambda: _C.awq_gemv(x.float(), qw, qz, sc), lambda: _C.awq_gemv(x[:, :128], qw, qz, sc),
        lambda: _C.awq_gemv(x[0], qw, qz, sc), lambda: _C.awq_gemv(x.expand(17, 3, 256)[:, 0], qw, qz, sc),
        lambda: _C.awq_gemv(x, qw, qz[:1], sc), lambda: _C.awq_gemv(x, qw, qz, sc[:, :32]),
        lambda: _C.awq_gemv(x, qw.to(torch.int64), qz, sc), lambda: _C.awq_gemv(x, qw.to("meta"), qz, sc),
        lambda: _C.awq_gemv(x, qw, qz, sc, group_size=0), lambda: _C.awq_gemv(x, qw, qz, sc, torch.zeros(63, dtype=bf)),
        lambda: _C.awq_gemv(x, qw, qz, sc, out=torch.zeros(3, 64)),
        lambda: _C.awq_gemv_residual(x, qw, qz, sc, torch.zeros(3, 64, dtype=bf)),
        lambda: _C.awq_gemv_silu(x, qw, qz, sc, out=torch.zeros(3, 64, dtype=bf)),
        lambda: _C.kv8_append(k, k, codes.to(torch.int16), *c[1:], 4), lambda: _C.kv8_append(k, k, codes[:, :1], *c[1:], 4),
        lambda: _C.kv8_append(k, k, codes, scales[:8], *c[2:], 4), lambda: _C.kv8_append(k, k[:3], *c, 4),
        lambda: _C.kv8_append(k, k, *c, 4, sums[:, :1]), lambda: _C.kv8_append(k, k, codes, scales, table, cu[:2], lens, 4),
        lambda: _C.kv8_append(k, k, codes, scales, table[0], cu, lens, 4), lambda: _C.kv8_append(k.to("meta"), k, *c, 4),
        lambda: _C.kv8_read(codes, scales, lens.long()), lambda: _C.kv8_read(codes, scales, lens, torch.zeros(2, 2, 2, 32, 128)),
        lambda: _C.kv8_attention(q, *c, 3, 0.1, 4), lambda: _C.kv8_attention(q[:, :384], *c, 3, 0.1, 4),
        lambda: _C.kv8_attention(q, *c, 4, 0.1, 5), lambda: _C.kv8_attention(q, *c, 4, 0.1, 4, out=torch.zeros(4, 512)),
        lambda: _C.kv8_attention(q, codes, scales, table, cu, lens[:1], 4, 0.1, 4),
        lambda: _C.kv8_evict(codes, scales, None, table, lens, new, 40, 10), lambda: _C.kv8_evict(codes, scales, sums, table, lens, new, 40, 41),
        lambda: _C.kv8_evict(codes, scales, sums, table, lens, new, 70, 1), lambda: _C.kv8_evict(codes, scales, sums, table, lens, new.long(), 40, 1),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(_C.MesError):
            call()
        assert rec.calls == [], (i, rec.calls)
    _C.awq_gemv(x, qw, qz, sc, torch.zeros(64, dtype=bf))
    _C.kv8_append(k, k, *c, 4, sums)
    _C.kv8_attention(q, *c, 4, 0.1, 4, sums=sums)
    _C.kv8_evict(codes, scales, sums, table, lens, new, 40, 10)
    _C.kv8_read(codes.view(torch.float8_e4m3fn), scales, lens)
    assert rec.calls == ["mes_awq_gemv", "mes_kv8_append", "mes_kv8_attention", "mes_kv8_evict", "mes_kv8_read"]


def test_cache_object_checks(rec):
    with pytest.raises(ValueError):
        KV8Cache(4, 32, 2, torch.float16, "cpu")
    with pytest.raises(ValueError):
        KV8Cache(4, 20, 2, torch.int8, "cpu")
    cache = KV8Cache(4, 32, 2, torch.float8_e4m3fn, "cpu")
    assert cache.page_size == 32 and cache.codes.dtype == torch.float8_e4m3fn and cache.sums is None
    i32 = torch.int32
    step = CacheStep(torch.zeros(1, 1, dtype=i32), torch.zeros(2, dtype=i32), torch.zeros(1, dtype=i32), 1)
    with pytest.raises(ValueError):
        cache.evict(step, torch.zeros(1, 1, dtype=i32), 10, 5)


def test_incremental_pages_and_launches(rec):
    cfg = synthetic.qwen3_0_6b(num_hidden_layers=2, vocab_size=500)
    model = Qwen3ForCausalLM(MESConfig(model_config=cfg))
    emb = IncrementalEmbedder(model, num_pages=12, page_size=16, budget=32, recent=8, observe=4)
    handles, out = emb.add([np.arange(40), np.arange(3)])            # 3 pages and 1; 40 <= 32 + 8 stays
    assert out.shape == (2, cfg.hidden_size) and len(emb._free) == 8
    # the new text's rows are many: GEMMs and the 16-bit attention, then its last tokens' weights
    assert {"mes_awq_gemm_ws", "mes_varlen_attention", "mes_kv8_append", "mes_kv8_attention", "mes_last_token_l2"} <= set(rec.calls)
    assert "mes_kv8_evict" not in rec.calls and "mes_awq_gemv" not in rec.calls
    rec.calls.clear()
    emb.extend(handles, [[1], [2, 3]])                               # 41 tokens: cut to 32, two pages
    assert [emb.cached_tokens(h) for h in handles] == [32, 5]
    assert [emb._texts[h].position for h in handles] == [41, 5]
    assert rec.calls.count("mes_kv8_evict") == 2 and len(emb._free) == 9
    assert rec.calls.count("mes_awq_gemv") == 8 and rec.calls.count("mes_kv8_attention") == 2     # 4 projections a layer
    assert not {"mes_awq_gemm_ws", "mes_varlen_attention"} & set(rec.calls)
    forks = emb.fork(handles[1], 2)
    assert len(emb._free) == 7 and all(emb.cached_tokens(f) == 5 for f in forks)
    with pytest.raises(_C.MesError):
        emb.add([np.arange(16 * 8)])                                 # eight pages are not free
    assert len(emb._free) == 7 and len(emb._texts) == 4
    emb.drop(handles + forks)
    assert sorted(emb._free) == list(range(12)) and not emb._texts


def test_texts_end_with_the_rotary_table(rec):
    """Positions go on counting under a budget; past the table there is no rotation to give."""
    cfg = synthetic.qwen3_0_6b(num_hidden_layers=1, vocab_size=500, max_position_embeddings=64)
    emb = IncrementalEmbedder(Qwen3ForCausalLM(MESConfig(model_config=cfg)), num_pages=40, page_size=16, budget=32)
    (h,), _ = emb.add([np.arange(30)])
    for _ in range(34):
        emb.extend([h], [[1]])
    assert emb._texts[h].position == 64
    (other,) = emb.fork(h, 1)
    rec.calls.clear()
    state = (list(emb._free), list(emb._texts[h].pages), emb.cached_tokens(h))
    for call in (lambda: emb.extend([h], [[1]]), lambda: emb.extend([other], [[1, 2]]), lambda: emb.add([np.arange(65)]),
                 lambda: emb.add([[1], np.arange(70)])):
        with pytest.raises(_C.MesError, match="64 positions"):
            call()
        assert rec.calls == []
    assert (emb._free, emb._texts[h].pages, emb.cached_tokens(h)) == state and set(emb._texts) == {h, other}
    emb.add([np.arange(64)])


def _cached_texts(model, count, tokens=1, **kw):
    """``count`` texts whose one page is taken, as if ``add`` had run."""
    emb = IncrementalEmbedder(model, num_pages=4 * count, page_size=16, **kw)
    handles, _ = emb.add([np.arange(tokens)] * count)
    return emb, handles


@pytest.mark.parametrize("budget", [None, 8])
def test_more_texts_than_one_attention_call_takes(rec, budget):
    """1024 sequences are what ``mes_kv8_attention`` takes: longer lists run in parts, in order."""
    cfg = synthetic.qwen3_0_6b(num_hidden_layers=2, vocab_size=500)
    model = Qwen3ForCausalLM(MESConfig(model_config=cfg))
    emb, handles = _cached_texts(model, 1500, tokens=9, budget=budget, observe=2)
    rec.calls.clear()
    assert emb.extend(handles, [[1]] * 1500).shape == (1500, cfg.hidden_size)
    # two parts of two layers, one write and one attention each
    assert rec.calls.count("mes_kv8_append") == rec.calls.count("mes_kv8_attention") == 4
    assert all(emb._texts[h].position == 10 for h in handles)
    emb.drop(handles)
    assert sorted(emb._free) == list(range(6000))


def test_a_step_past_what_the_attention_counts(rec):
    """The attention counts its units in 32 bits: a call past that is split, a single text past it refused,
    and the refusal changes nothing."""
    assert _C.kv8_attention_fits(1024, 1, 16, 8, 4096) and not _C.kv8_attention_fits(1025, 1, 16, 8, 4096)
    assert _C.kv8_attention_fits(4, 60000, 16, 8, 65536) and not _C.kv8_attention_fits(64, 60000, 16, 8, 65536)
    cfg = synthetic.qwen3_0_6b(num_hidden_layers=1, vocab_size=500)
    emb, handles = _cached_texts(Qwen3ForCausalLM(MESConfig(model_config=cfg)), 3)
    rec.calls.clear()
    fits = []
    real = _C.kv8_attention_fits

    def tight(B, max_new, heads, kv_heads, tokens):
        fits.append((B, max_new, heads, kv_heads, tokens))
        return real(B, max_new, heads, kv_heads, tokens) and B * max_new <= 6
    _C.kv8_attention_fits = tight
    try:
        emb.extend(handles, [[1] * 4, [2] * 3, [3]])           # 4 | 3, 1 (two texts of at most 3)
        assert rec.calls.count("mes_kv8_append") == 2
        rec.calls.clear()
        state = list(emb._free), [(list(emb._texts[h].pages), emb.cached_tokens(h)) for h in handles]
        with pytest.raises(_C.MesError, match="one call"):
            emb.extend(handles, [[1], [2], [3] * 7])
        assert rec.calls == [] and state == (list(emb._free), [(list(emb._texts[h].pages), emb.cached_tokens(h)) for h in handles])
    finally:
        _C.kv8_attention_fits = real


def test_fork_into_no_texts(rec):
    cfg = synthetic.qwen3_0_6b(num_hidden_layers=1, vocab_size=500)
    emb = IncrementalEmbedder(Qwen3ForCausalLM(MESConfig(model_config=cfg)), num_pages=4, page_size=16)
    (h,), _ = emb.add([np.arange(20)])
    assert emb.fork(h, 0) == [] and len(emb._free) == 2 and set(emb._texts) == {h}
    with pytest.raises(_C.MesError):
        emb.fork(h, -1)
    with pytest.raises(_C.MesError):
        emb.fork(h, 2)
    assert len(emb._free) == 2 and set(emb._texts) == {h}
