"""Cases for the token-step operators: what a decoder runs when it extends sequences that it has
already seen, instead of running them again from their first token.

* ``gemv``: a 4-bit (AWQ) projection of a few rows, in its three forms: to bf16 with an
  optional bias, added to the fp32 residual stream, and gate/up with SiLU-and-mul.
* ``append``: new keys and values written to a paged cache held in 8 bits (int8 or e4m3) with one
  fp32 scale for each page of tokens, kv head and side (K or V).
* ``attend``: causal grouped-query attention of the new tokens over that cache, optionally
  adding every cached token's attention weight to a running sum per kv head.
* ``evict``: a cache cut down to the tokens with the largest sums and the most recent ones.

Cache layout: ``codes [pages, 2, Hkv, P, 128]`` (K, then V), ``scales [pages, 2, Hkv]``,
``sums [pages, Hkv, P]``; a sequence's token t is in slot ``t % P`` of page
``block_table[b, t // P]``.  New tokens are packed rows, ``cu`` their offsets per sequence, and
``ctx`` counts each sequence's cached tokens, the new ones among them.

``own`` selects what ``run`` calls: the plain torch forms below, or the package's operators.
"""
import math

import numpy as np
import torch

own = False

D = 128                       # head size of every supported model
QMAX = {"int8": 127.0, "e4m3": 448.0}
DTYPE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
_lib = []


def _ops():
    if not _lib:
        import __graft_entry__
        _lib.append(__graft_entry__.load_package()._C)
    return _lib[0]


# ------------------------------------------------------------------------------------- cases
def listed():
    return [
        # One token through a small projection (the 0.6B model's o_proj): launch latency.
        dict(name="gemv o 1 row", op="gemv", rows=1, k=2048, n=1024, group=128, form="residual"),
        # One token through the Qwen2-1.5B QKV projection, which has a bias.
        dict(name="gemv qkv 3 rows bias", op="gemv", rows=3, k=1536, n=2048, group=128, form="bias"),
        # A group of concurrent streams through the largest gate/up projection (8B).
        dict(name="gemv gate_up 8 rows", op="gemv", rows=8, k=4096, n=24576, group=128, form="silu"),
        # One new token in each of 32 streams, some of them at a page's first slot.
        dict(name="append 1 token x 32", op="append", kind="int8", seqs=32, lo=5, hi=3000, new=1, page=32,
             kv_heads=8),
        # The benchmark batch, 20 prompts of 1000 tokens, stored after its first pass.
        dict(name="append 20 x 1000", op="append", kind="e4m3", seqs=20, lo=1000, hi=1000, new=1000, page=64,
             kv_heads=8),
        # One short stream: latency.
        dict(name="attend 1 x 500", op="attend", kind="int8", seqs=1, lo=500, hi=500, new=1, page=16, heads=16,
             kv_heads=8, sums=False),
        # Many streams of very different lengths, one new token each (8B heads).
        dict(name="attend 64 ragged", op="attend", kind="e4m3", seqs=64, lo=100, hi=8192, new=1, page=64, heads=32,
             kv_heads=8, sums=False),
        # Two long documents, one new token each: the cache is all the traffic.
        dict(name="attend 2 x 131072", op="attend", kind="int8", seqs=2, lo=131072, hi=131072, new=1, page=128,
             heads=16, kv_heads=8, sums=False),
        # A short text after a cached prefix: several query tokens for each kv head.
        dict(name="attend suffix 8 x 23", op="attend", kind="e4m3", seqs=8, lo=1500, hi=4000, new=23, page=32,
             heads=12, kv_heads=2, sums=False),
        # A step that also tracks the weights that eviction goes by.
        dict(name="attend sums 16", op="attend", kind="int8", seqs=16, lo=2000, hi=6000, new=1, page=32, heads=32,
             kv_heads=8, sums=True),
        # A batch of streams cut down to half of their budget.
        dict(name="evict 8 x 4096", op="evict", kind="int8", seqs=8, lo=3000, hi=4096, page=32, kv_heads=8, keep=2048,
             recent=256),
        # One long document cut to a sixth.
        dict(name="evict 1 x 100003", op="evict", kind="e4m3", seqs=1, lo=100003, hi=100003, page=64, kv_heads=8,
             keep=16384, recent=1000),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["gemv", "gemv", "append", "attend", "attend", "attend", "evict"])
    if op == "gemv":
        form = rng.choice(["plain", "bias", "residual", "silu"])
        unit = 128 if form == "silu" else 8
        return dict(op=op, rows=rng.choice([1, 1, 2, 3, 5, 8, 11, 16]), k=128 * _log_int(rng, 4, 96),
                    n=unit * _log_int(rng, 512 // unit, 24576 // unit), group=rng.choice([32, 64, 128, 128]), form=form)
    kind, page, kv_heads = rng.choice(["int8", "e4m3"]), rng.choice([16, 32, 64, 128]), rng.choice([1, 2, 4, 8])
    if op == "append":
        seqs = _log_int(rng, 1, 64)
        new = _log_int(rng, 1, 20000 // seqs)
        hi = new + rng.choice([0, 7, 1000])
        return dict(op=op, kind=kind, seqs=seqs, lo=max(1, min(new, hi // 3)), hi=hi, new=new, page=page,
                    kv_heads=kv_heads)
    seqs = _log_int(rng, 1, 64)
    if op == "evict":
        hi = _log_int(rng, 40, 160000 // seqs)
        keep = max(2, int(hi * rng.uniform(0.15, 0.9)))
        return dict(op=op, kind=kind, seqs=seqs, lo=max(1, hi // rng.choice([1, 4])), hi=hi, page=page,
                    kv_heads=kv_heads, keep=keep, recent=int(keep * rng.uniform(0.0, 0.5)))
    hi = _log_int(rng, 1, 262144 // seqs)
    heads = kv_heads * rng.choice([1, 2, 4, 5, 6, 8])
    # Several new tokens as far as that costs no more than the longest listed cache.
    new = rng.choice([1, 1, 1, max(1, min(hi, _log_int(rng, 2, 32), 40_000_000 // (hi * seqs * heads)))])
    return dict(op=op, kind=kind, seqs=seqs, lo=max(1, hi // rng.choice([1, 3, 20])), hi=hi, new=new, page=page,
                heads=heads, kv_heads=kv_heads, sums=hi * seqs <= 65536 and rng.random() < 0.3)


def _lengths(case):
    """Cached tokens and new tokens of each sequence: spread over [lo, hi] by the golden ratio."""
    lo, hi = case["lo"], case["hi"]
    ctx = [hi if i == 0 else lo + int((hi - lo) * ((i * 0.6180339887) % 1.0)) for i in range(case["seqs"])]
    return ctx, [min(case.get("new", 1), c) for c in ctx]


# ------------------------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def prepare(case, seed):
    g = _gen(seed)
    if case["op"] == "gemv":
        rows, k, n, group = case["rows"], case["k"], case["n"], case["group"]

        def words(*shape):
            return torch.randint(-2 ** 31, 2 ** 31, shape, generator=g, device="cuda", dtype=torch.int64).to(torch.int32)

        s = dict(case)
        s["x"] = torch.randn(rows, k, generator=g, device="cuda").to(torch.bfloat16)
        # The weights as the package keeps them after loading: eight k of one feature in a word.
        s["qweight"], s["qzeros"] = words(k // 8, n), words(k // group, n // 8)
        s["scales"] = (torch.rand(k // group, n, generator=g, device="cuda") * 0.018 + 0.002).to(torch.float16)
        if case["form"] == "silu":   # gates of a few units, where silu is neither 0 nor linear
            s["scales"] = (s["scales"].float() * (8.0 / math.sqrt(k))).to(torch.float16)
        s["bias"] = torch.randn(n, generator=g, device="cuda").to(torch.bfloat16) if case["form"] == "bias" else None
        s["residual"] = torch.randn(rows, n, generator=g, device="cuda") if case["form"] == "residual" else None
        return s

    ctx, new = _lengths(case)
    page, hkv, kind = case["page"], case["kv_heads"], case["kind"]
    npages = [-(-c // page) for c in ctx]
    total, width = sum(npages) + 3, max(npages)
    s = dict(case, ctx_host=ctx, new_host=new)
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(case["seqs"], width, dtype=torch.int32, device="cuda")
    first = 0
    for b, p in enumerate(npages):
        table[b, :p] = order[first:first + p]
        first += p
    s["table"] = table
    s["ctx"] = torch.tensor(ctx, dtype=torch.int32, device="cuda")
    s["cu"] = torch.tensor([0, *np.cumsum(new)], dtype=torch.int32, device="cuda")
    # A cache that earlier calls filled: codes spread as quantised normal values are, one scale
    # for each page, side and head.
    codes = torch.empty(total, 2, hkv, page, D, dtype=DTYPE[kind], device="cuda")
    step = max(1, 2 ** 25 // (2 * hkv * page * D))
    for p in range(0, total, step):
        v = torch.randn(codes[p:p + step].shape, generator=g, device="cuda") * (QMAX[kind] / 3.5)
        v = v.clamp(-QMAX[kind], QMAX[kind])
        codes[p:p + step] = (v.round() if kind == "int8" else v).to(DTYPE[kind])
    s["codes"] = codes
    s["scales"] = (torch.rand(total, 2, hkv, generator=g, device="cuda") + 0.5) * (3.5 / QMAX[kind])
    s["sums"] = None
    if case["op"] == "evict" or case.get("sums"):
        # Sums of attention weights: a few large ones, many small ones.
        s["sums"] = torch.rand(total, hkv, page, generator=g, device="cuda").pow(6.0) * 4.0
    if case["op"] == "append":
        rows = sum(new)
        # The packed QKV projection's k and v columns, channels of different sizes.
        qkv = torch.randn(rows, (2 * hkv + 2 * hkv) * D, generator=g, device="cuda")
        qkv *= torch.rand(qkv.shape[1], generator=g, device="cuda") * 2 + 0.1
        qkv = qkv.to(torch.bfloat16)
        s["k"], s["v"] = qkv[:, 2 * hkv * D:3 * hkv * D], qkv[:, 3 * hkv * D:]
        touched = [table[b, (c - m) // page:(c - 1) // page + 1] for b, (c, m) in enumerate(zip(ctx, new))]
        s["touched"] = torch.cat(touched)
        # A page that holds no tokens yet has no scale yet; stale slots hold zeros.
        start = torch.tensor([c - m for c, m in zip(ctx, new)], device="cuda")
        slot = torch.arange(width * page, device="cuda").view(1, width, page)
        stale = (slot >= start.view(-1, 1, 1)) & (torch.arange(width, device="cuda").view(1, -1, 1) <
                                                  torch.tensor(npages, device="cuda").view(-1, 1, 1))
        b, p, t = stale.nonzero(as_tuple=True)
        codes.view(torch.int8)[table[b, p].long(), :, :, t] = 0
    elif case["op"] == "attend":
        s["scale"] = D ** -0.5
        s["q"] = torch.randn(sum(new), (case["heads"] + 2 * hkv) * D, generator=g, device="cuda").to(torch.bfloat16)
        s["q"] = s["q"][:, :case["heads"] * D]     # the q columns of the packed projection
    else:
        keep_pages = -(-case["keep"] // page)
        s["codes"] = torch.cat([codes.view(torch.int8), torch.zeros(
            case["seqs"] * keep_pages, *codes.shape[1:], dtype=torch.int8, device="cuda")]).view(DTYPE[kind])
        s["scales"] = torch.cat([s["scales"], torch.zeros(case["seqs"] * keep_pages, 2, hkv, device="cuda")])
        s["sums"] = torch.cat([s["sums"], torch.zeros(case["seqs"] * keep_pages, hkv, page, device="cuda")])
        s["new_table"] = torch.arange(total, total + case["seqs"] * keep_pages, dtype=torch.int32,
                                      device="cuda").view(case["seqs"], keep_pages)
        s["new_pages"] = s["new_table"].reshape(-1)
    return s


# --------------------------------------------------------------------------------- plain forms
def _nibbles(words):
    """int32 ``[R, C]`` -> the eight codes of each word in order, int32 ``[R, 8, C]``: code i of a
    word is its nibble (0, 4, 1, 5, 2, 6, 3, 7)[i]."""
    shift = torch.tensor([0, 16, 4, 20, 8, 24, 12, 28], dtype=torch.int32, device=words.device)
    return (words.unsqueeze(1) >> shift.view(1, 8, 1)) & 15


def _plain_gemv(s):
    k, n, group = s["k"], s["n"], s["group"]
    q = _nibbles(s["qweight"]).reshape(k // group, group, n)
    z = _nibbles(s["qzeros"]).transpose(1, 2).reshape(k // group, 1, n)
    w = ((q - z).float() * s["scales"].float().unsqueeze(1)).view(k, n)
    y = s["x"].float() @ w
    if s["form"] == "bias":
        y = y + s["bias"].float()
    if s["form"] == "residual":
        s["residual"] += y
        return s["residual"]
    if s["form"] == "silu":   # blocks of 16 gate features and 16 up features alternate
        y = y.view(-1, n // 32, 2, 16)
        y = (y[:, :, 0] / (1.0 + torch.exp(-y[:, :, 0])) * y[:, :, 1]).reshape(-1, n // 2)
    return y.to(torch.bfloat16)


def _encode(v, kind):
    """Values over their scale -> codes, ties to even, held within the type's finite range."""
    v = v.clamp(-QMAX[kind], QMAX[kind])
    return (v.round() if kind == "int8" else v).to(DTYPE[kind])


def _pages(s, pages):
    """The codes of pages ``[n, 2, Hkv, P, D]`` (indexed as bytes)."""
    return s["codes"].view(torch.int8)[pages.long()].view(s["codes"].dtype)


def _read(s, pages):
    """The values that pages stand for, bf16 ``[n, 2, Hkv, P, D]``."""
    return (_pages(s, pages).float() * s["scales"][pages.long()][..., None, None]).to(torch.bfloat16)


def _plain_append(s):
    page, hkv, kind = s["page"], s["kv_heads"], s["kind"]
    cu, ctx, table, touched = s["cu"].long(), s["ctx"].long(), s["table"].long(), s["touched"].long()
    row = torch.arange(s["k"].shape[0], device="cuda")
    b = torch.searchsorted(cu[1:], row, right=True)
    pos = ctx[b] - (cu[b + 1] - row)                       # where each new token goes
    at, slot = table[b, pos // page], pos % page
    kv = torch.stack([s["k"].reshape(-1, hkv, D), s["v"].reshape(-1, hkv, D)], 1).float()   # [T, 2, Hkv, D]
    new_max = torch.zeros_like(s["scales"]).index_reduce_(0, at, kv.abs().amax(-1), "amax")[touched]
    # A page's old tokens are the slots before the first new one.
    old = torch.full((s["scales"].shape[0],), page, device="cuda").index_reduce_(0, at, slot, "amin")[touched]
    had = old.view(-1, 1, 1) > 0
    was = torch.where(had, s["scales"][touched], torch.zeros_like(new_max))
    now = torch.maximum(was, new_max / QMAX[kind])
    safe = torch.where(now > 0, now, torch.ones_like(now))
    grown = (torch.arange(page, device="cuda").view(1, 1, 1, page) < old.view(-1, 1, 1, 1)) & (now > was)[..., None]
    was_codes = _pages(s, touched)
    again = _encode(was_codes.float() * was[..., None, None] / safe[..., None, None], kind)
    codes = s["codes"].view(torch.int8)
    codes[touched] = torch.where(grown[..., None], again.view(torch.int8), was_codes.view(torch.int8))
    s["scales"][touched] = now
    full = torch.ones_like(s["scales"])
    full[touched] = safe
    codes[at, :, :, slot] = _encode(kv / full[at][..., None], kind).view(torch.int8)
    return [_read(s, s["touched"]), s["scales"][touched]]


def _by_sequence(s, width):
    """(K, V) of every sequence, fp32 ``[B, Hkv, width * P, D]``."""
    t = s["table"][:, :width].long()
    v = _pages(s, t).float() * s["scales"][t][..., None, None]       # [B, width, 2, Hkv, P, D]
    v = v.permute(2, 0, 3, 1, 4, 5)
    return v.reshape(2, v.shape[1], v.shape[2], -1, D)


def _plain_attend(s):
    heads, hkv, page = s["heads"], s["kv_heads"], s["page"]
    B, n = s["seqs"], max(s["new_host"])
    cu, ctx = s["cu"].long(), s["ctx"].long()
    row = torch.arange(s["q"].shape[0], device="cuda")
    b = torch.searchsorted(cu[1:], row, right=True)
    i = row - cu[b]
    q = torch.zeros(B, n, heads, D, device="cuda")
    q[b, i] = s["q"].reshape(-1, heads, D).float()
    q = q.view(B, n, hkv, heads // hkv, D).permute(0, 2, 3, 1, 4).reshape(B, hkv, -1, D)   # rows (head, token)
    kv = _by_sequence(s, s["table"].shape[1])
    logits = (q @ kv[0].transpose(-1, -2)) * s["scale"]
    key = torch.arange(kv.shape[3], device="cuda")
    last = (ctx - (cu[1:] - cu[:-1])).view(-1, 1) + torch.arange(n, device="cuda")         # [B, n]
    seen = (key.view(1, 1, -1) <= last.unsqueeze(-1)) & (key.view(1, 1, -1) < ctx.view(-1, 1, 1))
    seen = seen.view(B, 1, 1, n, -1)
    logits = logits.view(B, hkv, -1, n, key.shape[0]).masked_fill_(~seen, float("-inf"))
    w = torch.exp(logits - logits.amax(-1, keepdim=True))
    w = w / w.sum(-1, keepdim=True)
    o = w.view(B, hkv, -1, key.shape[0]) @ kv[1]
    o = o.view(B, hkv, -1, n, D).permute(0, 3, 1, 2, 4).reshape(B, n, heads * D)
    out = o[b, i].to(torch.bfloat16)
    if s["sums"] is None:
        return out
    real = (torch.arange(n, device="cuda") < (cu[1:] - cu[:-1]).view(-1, 1)).view(B, 1, 1, n, 1)
    add = torch.where(real, w, torch.zeros_like(w)).sum((2, 3))                            # [B, Hkv, keys]
    at = s["table"].long()[:, key // page]              # [B, keys]; past the end the weight is 0
    s["sums"].index_put_((at.unsqueeze(1), torch.arange(hkv, device="cuda").view(1, -1, 1), (key % page).view(1, 1, -1)),
                         add, accumulate=True)
    return [out, s["sums"]]


def _plain_evict(s):
    page, hkv, kind, keep = s["page"], s["kv_heads"], s["kind"], s["keep"]
    B, width = s["seqs"], s["table"].shape[1]
    ctx, t = s["ctx"].long(), s["table"].long()
    sums = s["sums"][t].permute(0, 2, 1, 3).reshape(B, hkv, width * page)
    key = torch.arange(width * page, device="cuda")
    # The most recent tokens come first, tokens past the end last, ties by the lower index.
    recent = key >= (ctx - s["recent"]).view(-1, 1, 1)
    sums = torch.where(recent, float("inf"), sums)
    sums = torch.where(key < ctx.view(-1, 1, 1), sums, float("-inf"))
    order = torch.sort(sums, dim=-1, descending=True, stable=True).indices[..., :keep]
    if order.shape[-1] < keep:
        order = torch.nn.functional.pad(order, (0, keep - order.shape[-1]), value=width * page)
    lens = torch.minimum(ctx, torch.full_like(ctx, keep))
    order = torch.where(torch.arange(keep, device="cuda") < lens.view(-1, 1, 1), order, width * page)
    kept = torch.sort(order, dim=-1).values
    live = kept < width * page
    src = torch.where(live, kept, torch.zeros_like(kept))
    b = torch.arange(B, device="cuda").view(-1, 1, 1).expand_as(src)
    h = torch.arange(hkv, device="cuda").view(1, -1, 1).expand_as(src)
    at = t[b, src // page]
    pages = s["new_table"].shape[1]
    pad = (0, pages * page - keep)
    was = torch.where(live[..., None], s["scales"][at, :, h], 0.0)                         # [B, Hkv, keep, 2]
    was = torch.nn.functional.pad(was, (0, 0, *pad)).view(B, hkv, pages, page, 2)
    now = was.amax(3)                                                                      # [B, Hkv, pages, 2]
    safe = torch.where(now > 0, now, torch.ones_like(now)).unsqueeze(3)
    v = s["codes"].view(torch.int8)[at, :, h, src % page]                                  # [B, Hkv, keep, 2, D]
    v = torch.where(live[..., None, None], v, torch.zeros_like(v))
    v = torch.nn.functional.pad(v, (0, 0, 0, 0, *pad)).view(DTYPE[kind]).view(B, hkv, pages, page, 2, D)
    v = _encode(v.float() * was[..., None] / safe[..., None], kind)
    to = s["new_table"].long()
    s["codes"].view(torch.int8)[to] = v.view(torch.int8).permute(0, 2, 4, 1, 3, 5)
    s["scales"][to] = now.permute(0, 2, 3, 1)
    kept_sums = torch.where(live, s["sums"][at, h, src % page], 0.0)
    s["sums"][to] = torch.nn.functional.pad(kept_sums, pad).view(B, hkv, pages, page).transpose(1, 2)
    kept = torch.where(live, kept, torch.full_like(kept, -1)).to(torch.int32)
    return [kept, lens.to(torch.int32), _read(s, s["new_pages"]), s["sums"][to]]


# ----------------------------------------------------------------------------------------- run
def run(state):
    s = state
    if not own:
        return {"gemv": _plain_gemv, "append": _plain_append, "attend": _plain_attend, "evict": _plain_evict}[s["op"]](s)
    C = _ops()
    if s["op"] == "gemv":
        if s["form"] == "silu":
            return C.awq_gemv_silu(s["x"], s["qweight"], s["qzeros"], s["scales"], group_size=s["group"])
        if s["form"] == "residual":
            return C.awq_gemv_residual(s["x"], s["qweight"], s["qzeros"], s["scales"], s["residual"],
                                       group_size=s["group"])
        return C.awq_gemv(s["x"], s["qweight"], s["qzeros"], s["scales"], s["bias"], group_size=s["group"])
    if s["op"] == "append":
        C.kv8_append(s["k"], s["v"], s["codes"], s["scales"], s["table"], s["cu"], s["ctx"], max_new=s["new"])
        return [C.kv8_read(s["codes"], s["scales"], s["touched"]), s["scales"][s["touched"].long()]]
    if s["op"] == "attend":
        out = C.kv8_attention(s["q"], s["codes"], s["scales"], s["table"], s["cu"], s["ctx"], s["heads"], s["scale"],
                              max_new=s["new"], sums=s["sums"])
        return out if s["sums"] is None else [out, s["sums"]]
    kept, lens = C.kv8_evict(s["codes"], s["scales"], s["sums"], s["table"], s["ctx"], s["new_table"], s["keep"],
                             s["recent"])
    return [kept, lens, C.kv8_read(s["codes"], s["scales"], s["new_pages"]), s["sums"][s["new_table"].long()]]


# --------------------------------------------------------------------------------------- exact
def _exact_gemv(s):
    k, n, group = s["k"], s["n"], s["group"]
    qw = s["qweight"].cpu().numpy().view(np.uint32)
    qz = s["qzeros"].cpu().numpy().view(np.uint32)
    place = {0: 0, 2: 1, 4: 2, 6: 3, 1: 4, 3: 5, 5: 6, 7: 7}          # code -> nibble of its word
    x = s["x"].double().cpu().numpy()
    scales = s["scales"].double().cpu().numpy()
    zeros = np.empty((k // group, n))
    for c in range(8):
        zeros[:, c::8] = (qz >> np.uint32(4 * place[c])) & np.uint32(15)
    y = np.zeros((s["rows"], n))
    part = np.zeros((k // group, s["rows"], n))
    for c in range(8):
        q = ((qw >> np.uint32(4 * place[c])) & np.uint32(15)).astype(np.float64)
        for g in range(k // group):
            rows = slice(g * group // 8, (g + 1) * group // 8)
            part[g] += x[:, g * group + c:(g + 1) * group:8] @ q[rows]
    for g in range(k // group):
        y += (part[g] - x[:, g * group:(g + 1) * group].sum(1, keepdims=True) * zeros[g]) * scales[g]
    if s["form"] == "bias":
        y += s["bias"].double().cpu().numpy()
    if s["form"] == "residual":
        y += s["residual"].double().cpu().numpy()
    if s["form"] == "silu":
        f = np.arange(n // 2)
        gate = y[:, f // 16 * 32 + f % 16]
        y = gate / (1.0 + np.exp(-gate)) * y[:, f // 16 * 32 + 16 + f % 16]
    return y


def _tokens(s, b, side, h, count):
    """The first ``count`` cached K or V rows of one sequence and head, in 64 bits."""
    pages = s["table"][b, :-(-count // s["page"])].long()
    v = s["codes"].view(torch.int8)[pages, side, h].view(s["codes"].dtype).double() * s["scales"][pages, side, h].double().view(-1, 1, 1)
    return v.reshape(-1, D)[:count]


def _exact_attend(s):
    heads, hkv, page = s["heads"], s["kv_heads"], s["page"]
    out = torch.zeros(sum(s["new_host"]), heads, D, dtype=torch.float64, device="cuda")
    sums = None if s["sums"] is None else s["sums"].double()
    r0 = 0
    for b, (c, m) in enumerate(zip(s["ctx_host"], s["new_host"])):
        for h in range(hkv):
            k, v = _tokens(s, b, 0, h, c), _tokens(s, b, 1, h, c)
            mine = slice(h * heads // hkv, (h + 1) * heads // hkv)
            q = s["q"][r0:r0 + m].reshape(m, heads, D)[:, mine].double()
            x = torch.einsum("igd,td->igt", q, k) * s["scale"]
            hidden = torch.arange(c, device="cuda").view(1, 1, -1) > torch.arange(c - m, c, device="cuda").view(-1, 1, 1)
            w = torch.softmax(x.masked_fill(hidden, float("-inf")), -1)
            out[r0:r0 + m, mine] = torch.einsum("igt,td->igd", w, v)
            if sums is not None:
                t = torch.arange(c, device="cuda")
                sums[s["table"][b].long()[t // page], h, t % page] += w.sum((0, 1))
        r0 += m
    out = out.reshape(-1, heads * D)
    return out if sums is None else [out, sums]


def _round_codes(x, kind):
    if kind == "int8":
        return np.clip(np.rint(x), -127, 127)
    a = np.minimum(np.abs(x), 448.0)     # e4m3: 3 bits after the leading one, subnormals below 2^-6
    step = np.exp2(np.floor(np.log2(np.maximum(a, 2.0 ** -6))) - 3)
    return np.sign(x) * np.minimum(np.rint(a / step) * step, 448.0)


def _exact_append(s):
    page, kind, hkv = s["page"], s["kind"], s["kv_heads"]
    table = s["table"].cpu().numpy()
    kv = np.stack([s[x].double().cpu().numpy().reshape(-1, hkv, D) for x in ("k", "v")], 1)
    touched = s["touched"].long()
    codes, scales = _pages(s, touched).double().cpu().numpy(), s["scales"][touched].double().cpu().numpy()
    values = codes * scales[..., None, None]
    place = {int(p): i for i, p in enumerate(s["touched"].tolist())}
    r0 = 0
    for b, (c, m) in enumerate(zip(s["ctx_host"], s["new_host"])):
        for p in range((c - m) // page, (c - 1) // page + 1):
            lo, hi = max(p * page, c - m), min((p + 1) * page, c)
            i, old = place[int(table[b, p])], max(0, (c - m) - p * page)
            x = kv[r0 + lo - (c - m):r0 + hi - (c - m)].transpose(1, 2, 0, 3)          # [2, Hkv, new, D]
            was = scales[i] if old else np.zeros_like(scales[i])
            now = np.maximum(was, np.abs(x).max((2, 3)) / QMAX[kind])
            safe = np.where(now > 0, now, 1.0)[..., None, None]
            again = _round_codes(values[i, :, :, :old] / safe, kind) * safe
            values[i, :, :, :old] = np.where((now > was)[..., None, None], again, values[i, :, :, :old])
            values[i, :, :, lo - p * page:hi - p * page] = _round_codes(x / safe, kind) * safe
            values[i, :, :, hi - p * page:] = codes[i, :, :, hi - p * page:] * now[..., None, None]
            scales[i] = now
        r0 += m
    return [values, scales]


def _exact_evict(s):
    page, kind, hkv, keep = s["page"], s["kind"], s["kv_heads"], s["keep"]
    if sum(s["ctx_host"]) * hkv > 1_000_000:
        return None
    table = s["table"].cpu().numpy()
    codes, scales = s["codes"].float().cpu().numpy(), s["scales"].double().cpu().numpy()
    sums = s["sums"].double().cpu().numpy()
    pages = s["new_table"].shape[1]
    out = np.zeros((s["seqs"], pages, 2, hkv, page, D))
    moved = np.zeros((s["seqs"], pages, hkv, page))
    for b, c in enumerate(s["ctx_host"]):
        t = np.arange(c)
        for h in range(hkv):
            mine = sums[table[b, t // page], h, t % page]
            old = max(0, c - s["recent"])
            best = np.argsort(-mine[:old], kind="stable")[:max(0, min(c, keep) - (c - old))]
            kept = np.concatenate([np.sort(best), t[old:]])[-keep:]
            for p in range(-(-len(kept) // page)):
                src = kept[p * page:(p + 1) * page]
                at = table[b, src // page]
                was = scales[at, :, h]                                               # [n, 2]
                now = was.max(0)
                v = codes[at, :, h, src % page] * (was / np.where(now > 0, now, 1.0))[..., None]
                out[b, p, :, h, :len(src)] = (_round_codes(v, kind) * now[:, None]).transpose(1, 0, 2)
                moved[b, p, h, :len(src)] = sums[at, h, src % page]
    return [None, None, out.reshape(-1, 2, hkv, page, D), moved]


def exact(case, seed):
    s = prepare(case, seed)
    return {"gemv": _exact_gemv, "append": _exact_append, "attend": _exact_attend, "evict": _exact_evict}[case["op"]](s)


# ---------------------------------------------------------------------------------------- work
def work(case):
    if case["op"] == "gemv":
        m, k, n, group, form = case["rows"], case["k"], case["n"], case["group"], case["form"]
        weights = k * n / 2 + k / group * n * 2.5
        io = 2 * m * k + {"plain": 2 * m * n, "bias": 2 * m * n + 2 * n, "residual": 8 * m * n, "silu": m * n}[form]
        return {"bytes": weights + io, "flops": 2.0 * m * k * n}
    ctx, new = _lengths(case)
    page, hkv = case["page"], case["kv_heads"]
    if case["op"] == "append":
        touched = sum((c - 1) // page - (c - m) // page + 1 for c, m in zip(ctx, new))
        # each new value read in 16 bits and written in 8; the touched pages read back to bf16
        return {"bytes": sum(new) * hkv * 2 * D * 3 + touched * hkv * 2 * page * D * 3, "flops": sum(new) * hkv * 2 * D * 3}
    if case["op"] == "attend":
        heads = case["heads"]
        pairs = sum(m * c - m * (m - 1) // 2 for c, m in zip(ctx, new))
        extra = 8 * sum(ctx) * hkv if case["sums"] else 0
        return {"bytes": sum(ctx) * hkv * 2 * D + sum(new) * heads * D * 4 + extra, "flops": 4.0 * pairs * heads * D}
    left = [min(c, case["keep"]) for c in ctx]
    stored = case["seqs"] * -(-case["keep"] // page) * page
    # sums read; kept rows read and written (with sums and indices); the new pages read back to bf16
    return {"bytes": 4 * sum(ctx) * hkv + sum(left) * hkv * (4 * D + 12) + stored * hkv * 2 * D * 3,
            "flops": sum(ctx) * hkv + sum(left) * hkv * 2 * D * 2}
