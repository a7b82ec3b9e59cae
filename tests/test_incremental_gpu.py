"""Texts that grow: ``IncrementalEmbedder`` against the worker's forward over the whole text.

What differs is the 8-bit cache (and, for few new tokens, weights that are not rounded to bf16).
A cached value is off by at most half a step of its page's scale: relative to a head's typical value,
whose largest of a page is some four times it, about 1% for int8 (4 / 127 / sqrt(12)) and 2.6% for
e4m3 (2^-4 / sqrt(12) and its rounding to fewer steps).  Attention averages keys' and values' errors, and
each layer adds them to a residual stream that they reach after a projection, so the angle between
embeddings is a few times that at most: 0.03 to 0.05 for int8, 0.1 for e4m3, cosines of 0.998 and
0.99.
"""
import numpy as np
import pytest
import torch

from mes_b200 import _C, synthetic
from mes_b200.core.gpu_worker import GPUWorker
from mes_b200.core.incremental import IncrementalEmbedder
from mes_b200.schemas.config import MESConfig
from mes_b200.ultils.loader import load_weights

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
COS = {torch.int8: 0.998, torch.float8_e4m3fn: 0.99}


def _worker(make, seed=0, **kw):
    cfg = make(num_hidden_layers=3, vocab_size=3000, max_position_embeddings=4096, **kw)
    worker = GPUWorker(MESConfig(model_config=cfg), device=DEV)
    load_weights(worker.model, synthetic.quantize_dense_checkpoint(synthetic.dense_weights(cfg, seed=seed)))
    worker.use_cuda_graphs = False
    return worker, cfg


@pytest.fixture(scope="module")
def qwen3():
    return _worker(synthetic.qwen3_0_6b)


@pytest.fixture(scope="module")
def qwen2():
    return _worker(synthetic.qwen2_1_5b)


def _whole(worker, texts):
    pos = np.concatenate([np.arange(len(t)) for t in texts])
    return worker.embed(np.concatenate(texts), pos, np.cumsum([len(t) for t in texts]) - 1).numpy()


def _cos(a, b):
    return (a * b).sum(1) / np.linalg.norm(a, axis=1) / np.linalg.norm(b, axis=1)


def _ids(rng, n, vocab=3000):
    return rng.integers(0, vocab, n)


@pytest.mark.parametrize("name", ["qwen3", "qwen2"])
@pytest.mark.parametrize("dtype", list(COS))
@pytest.mark.parametrize("page", [16, 64])
def test_growing_texts_match_the_whole(request, name, dtype, page):
    worker, _ = request.getfixturevalue(name)
    rng = np.random.default_rng(page)
    emb = IncrementalEmbedder(worker.model, num_pages=200, page_size=page, dtype=dtype)
    texts = [_ids(rng, n) for n in (37, 1, 300, 64)]
    handles, got = emb.add(texts)
    assert got.shape == (4, worker.mes_config.model_config.hidden_size) and got.dtype == torch.float32
    # nothing cached is used yet: only the row counts of the GEMMs differ
    assert (_cos(got.cpu().numpy(), _whole(worker, texts)) > 0.9995).all()
    for more in ([1, 1, 1, 1], [2, 5, 1, 3], [40, 1, 7, 130], [1, 1, 1, 1]):
        new = [_ids(rng, n) for n in more]
        texts = [np.concatenate(p) for p in zip(texts, new)]
        got = emb.extend(handles, new)
        cos = _cos(got.cpu().numpy(), _whole(worker, texts))
        assert (cos > COS[dtype]).all(), cos
    assert _C.take_device_error() == 0
    assert [emb.cached_tokens(h) for h in handles] == [len(t) for t in texts]
    free = len(emb._free)
    emb.drop(handles[1:3])
    assert len(emb._free) == free + sum(-(-len(t) // page) for t in texts[1:3])
    # the others go on
    new = [_ids(rng, 1), _ids(rng, 4)]
    got = emb.extend([handles[3], handles[0]], new)
    cos = _cos(got.cpu().numpy(), _whole(worker, [np.concatenate([texts[3], new[0]]), np.concatenate([texts[0], new[1]])]))
    assert (cos > COS[dtype]).all(), cos


def test_queries_after_one_instruction(qwen3):
    worker, _ = qwen3
    rng = np.random.default_rng(3)
    emb = IncrementalEmbedder(worker.model, num_pages=100, page_size=32)
    instruction = _ids(rng, 70)
    (h,), _ = emb.add([instruction])
    queries = [_ids(rng, n) for n in (5, 1, 19, 9)]
    got = emb.extend(emb.fork(h, 4), queries).cpu().numpy()
    cos = _cos(got, _whole(worker, [np.concatenate([instruction, q]) for q in queries]))
    assert (cos > COS[torch.int8]).all(), cos
    assert emb.cached_tokens(h) == 70


def test_a_budget_keeps_the_cache_small(qwen3):
    worker, _ = qwen3
    rng = np.random.default_rng(4)
    budget, page = 64, 16
    emb = IncrementalEmbedder(worker.model, num_pages=60, page_size=page, budget=budget)
    handles, _ = emb.add([_ids(rng, 50), _ids(rng, 200)])
    assert [emb.cached_tokens(h) for h in handles] == [50, 64]
    for _ in range(40):
        got = emb.extend(handles, [_ids(rng, 1), _ids(rng, 2)])
        assert got.isfinite().all()
        assert all(emb.cached_tokens(h) <= budget + budget // 4 for h in handles)
    assert _C.take_device_error() == 0
    emb.drop(handles)
    assert sorted(emb._free) == list(range(60))


def test_the_last_tokens_of_a_run_give_the_weights(qwen3):
    """Every observed query adds weights of sum 1 for each of its heads: after a text, a long and a short
    addition the sums of a kv head tell how many queries were observed."""
    worker, cfg = qwen3
    rng = np.random.default_rng(12)
    G = cfg.num_attention_heads // cfg.num_key_value_heads
    emb = IncrementalEmbedder(worker.model, num_pages=20, page_size=16, budget=256, observe=4)
    (h,), _ = emb.add([_ids(rng, 50)])
    for more, seen in ((0, 4), (40, 8), (3, 11), (1, 12)):
        if more:
            emb.extend([h], [_ids(rng, more)])
        n, pages = emb.cached_tokens(h), torch.tensor(emb._texts[h].pages, device=DEV)
        for cache in emb.caches:
            total = cache.sums[pages].transpose(0, 1).reshape(cache.sums.shape[1], -1)[:, :n].double().sum(1)
            assert ((total - seen * G).abs() < 1e-3 * seen * G).all(), (more, total)


@pytest.mark.parametrize("budget", [None, 40])
def test_captured_steps_match_eager_ones(qwen3, budget):
    """Steps whose sizes come back run as graphs, with the lengths and pages of each call, across page
    and eviction boundaries; what differs is how the attention is cut (fp32 rounding)."""
    worker, cfg = qwen3
    G = cfg.num_attention_heads // cfg.num_key_value_heads
    embs, got = [], []
    for graphs in (True, False):
        rng = np.random.default_rng(13)
        emb = IncrementalEmbedder(worker.model, num_pages=60, page_size=16, budget=budget, observe=2)
        emb.use_cuda_graphs = graphs
        handles, _ = emb.add([_ids(rng, 20), _ids(rng, 33), _ids(rng, 1)])
        out = []
        for i in range(14):
            some = handles[:2] if i % 3 == 2 else handles
            out.append(emb.extend(some, [_ids(rng, 1 + (i + j) % 2) for j in range(len(some))]))
        embs.append(emb)
        got.append([o.cpu().numpy() for o in out])
    captured = [g for g in embs[0]._graphs.values() if g is not None]
    assert len(captured) >= 3 and not embs[1]._graphs
    for a, b in zip(*got):
        assert (_cos(a, b) > 0.9999).all(), _cos(a, b)
    if budget is None:
        return
    for a, b in zip(embs[0].caches, embs[1].caches):     # every step's weights are counted once
        ta, tb = ([c.sums[torch.tensor(e._texts[0].pages, device=DEV)].transpose(0, 1).reshape(c.sums.shape[1], -1)
                   [:, :e.cached_tokens(0)].double().sum(1) for e, c in zip(embs, (a, b))])
        assert ((ta - tb).abs() < 0.02 * tb).all()
    embs[0].release_graphs()
    assert not embs[0]._graphs


def test_no_room_for_an_eviction_changes_nothing(qwen3):
    worker, _ = qwen3
    rng = np.random.default_rng(11)
    emb = IncrementalEmbedder(worker.model, num_pages=8, page_size=16, budget=64)
    (h,), _ = emb.add([_ids(rng, 80)])            # 5 pages, and no eviction yet
    with pytest.raises(_C.MesError, match="free pages"):
        emb.extend([h], [_ids(rng, 1)])           # 1 more, and 4 to copy to
    assert emb.cached_tokens(h) == 80 and len(emb._free) == 3
    with pytest.raises(_C.MesError, match="free pages"):
        emb.add([_ids(rng, 81)])
    assert len(emb._free) == 3
    emb.drop([h])
    assert sorted(emb._free) == list(range(8))


def test_a_window_keeps_the_last_tokens(qwen3):
    """With as many recent tokens as the budget, what is kept is the end of the unlimited cache,
    re-rounded at most once a page."""
    worker, _ = qwen3
    rng = np.random.default_rng(5)
    text = _ids(rng, 150)
    caches = []
    for kw in (dict(), dict(budget=100, recent=100)):
        emb = IncrementalEmbedder(worker.model, num_pages=40, page_size=16, **kw)
        (h,), _ = emb.add([text])
        pages = torch.tensor(emb._texts[h].pages, dtype=torch.int32, device=DEV)
        n = emb.cached_tokens(h)
        caches.append([(c.read(pages).transpose(1, 3).reshape(-1, c.codes.shape[2], 2, 128)[:n].float(),
                        c.scales[pages.long()].amax()) for c in emb.caches])
    for (whole, scale), (kept, _) in zip(*caches):
        assert kept.shape[0] == 100
        # half a step of the largest scale, and two roundings to bf16
        assert ((kept - whole[50:]).abs() <= 0.5 * scale + 2.0 ** -7 * whole[50:].abs()).all()


def test_sixteen_rows_and_more_agree(qwen3):
    """The same new tokens through the matrix-vector kernels and through the GEMMs."""
    worker, _ = qwen3
    rng = np.random.default_rng(6)
    text, new = _ids(rng, 40), [_ids(rng, 1) for _ in range(20)]
    emb = IncrementalEmbedder(worker.model, num_pages=200, page_size=16)
    (h,), _ = emb.add([text])
    together = emb.extend(emb.fork(h, 20), new)
    apart = torch.cat([emb.extend(emb.fork(h, 10), new[:10]), emb.extend(emb.fork(h, 10), new[10:])])
    assert (_cos(together.cpu().numpy(), apart.cpu().numpy()) > 0.9995).all()


def test_refusals(qwen3):
    worker, _ = qwen3
    emb = IncrementalEmbedder(worker.model, num_pages=4, page_size=16)
    for bad in (lambda: emb.add([[]]), lambda: emb.add([np.zeros(100, dtype=np.int64)]), lambda: emb.extend([0], [[1], [2]])):
        with pytest.raises(_C.MesError):
            bad()
    assert len(emb._free) == 4 and not emb._texts
    (h,), _ = emb.add([[1, 2, 3]])
    with pytest.raises(_C.MesError):
        emb.extend([h], [[]])
    assert emb.add([])[0] == []
    with pytest.raises(ValueError):
        IncrementalEmbedder(worker.model, 4, 24)
    with pytest.raises(ValueError):
        IncrementalEmbedder(worker.model, 4, dtype=torch.float16)
    with pytest.raises(ValueError):
        IncrementalEmbedder(worker.model, 4, budget=10, recent=11)


def test_more_texts_than_one_attention_call(qwen3):
    """1100 forks of a text, some with two tokens more and some with one, against the same extensions in a short list."""
    worker, _ = qwen3
    rng = np.random.default_rng(14)
    emb = IncrementalEmbedder(worker.model, num_pages=2400, page_size=16)
    (h,), _ = emb.add([_ids(rng, 20)])
    new = [[7], [5, 9]]
    want = torch.stack([emb.extend(emb.fork(h, 1), [t])[0] for t in new])
    got = emb.extend(emb.fork(h, 1100), [new[i % 3 == 0] for i in range(1100)])
    assert got.shape == (1100, want.shape[1])
    # the long list takes the GEMMs, the short ones the matrix-vector products
    pick = torch.tensor([int(i % 3 == 0) for i in range(1100)], device=DEV)
    assert (_cos(got.cpu().numpy(), want[pick].cpu().numpy()) > 0.9995).all()
    assert _C.take_device_error() == 0
