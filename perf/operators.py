"""Measured cases of the attention operators: attention over the 8-bit paged cache, sliding-window attention over
ragged 16-bit inputs, quantising appends, and the cache's page operations.

`run` has two forms of every operator: where `own` is false, elementary torch operations in 32 bits on the same tensors;
where it is true, the calls of the package. `exact` states the results in 64 bits.

Cache layout (page = 64 tokens): codes int8 [layers, pages, 2 (K, V), kv heads, 64 * D], a head's K block as
[D/64][64 tokens][64 dims] and its V block as [D][64 tokens]; scales f32 [layers, pages, 2, kv heads]; tables int32
[sequences, pages per sequence] (-1: no page); lens int32 [sequences]; refs int32 [pages].
"""
import math
import os
import random
import sys

import torch

own = False

PAGE = 64
INV127 = 1.0 / 127.0  # a page's scale is its largest magnitude times this, in 32 bits
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _package():
    path = os.path.join(ROOT, "mrl-index-rust-vector_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import mrl_b200

    return mrl_b200


# ---- cases ------------------------------------------------------------------------------------------------------------


def listed():
    return [
        # one user, a short prompt, one kv head of 256 dims: the smallest call, all latency
        dict(name="decode_one_short", op="attend", n=1, len_lo=37, len_hi=37, q_lo=1, q_hi=1, hq=3, hkv=1, d=256, window=0,
             sinks=0, dtype="bf16", ragged=1),
        # a serving batch in mid-flight: sequences of very different lengths, four query heads per kv head
        dict(name="decode_batch_ragged", op="attend", n=48, len_lo=100, len_hi=8000, q_lo=1, q_hi=1, hq=32, hkv=8, d=128,
             window=0, sinks=0, dtype="bf16", ragged=2),
        # few readers of very long contexts: the work is one stream over the cache
        dict(name="decode_long", op="attend", n=4, len_lo=120001, len_hi=131071, q_lo=1, q_hi=1, hq=32, hkv=8, d=128,
             window=0, sinks=0, dtype="bf16", ragged=3),
        # a windowed layer of a big batch: old pages are gone, the first tokens stay
        dict(name="decode_window_sinks", op="attend", n=128, len_lo=500, len_hi=20000, q_lo=1, q_hi=1, hq=16, hkv=8, d=64,
             window=1024, sinks=4, dtype="f16", ragged=4),
        # queries' own tokens on top of a cached prefix of retrieved passages
        dict(name="chunk_on_prefix", op="attend", n=4, len_lo=3000, len_hi=6000, q_lo=257, q_hi=700, hq=32, hkv=8, d=128,
             window=0, sinks=0, dtype="bf16", ragged=5),
        # every sequence of a batch gains the token it just answered
        dict(name="append_token", op="append", n=256, len_lo=1, len_hi=700, q_lo=1, q_hi=1, hkv=8, d=128, dtype="bf16",
             ragged=6),
        # passages enter the cache, some behind an older partial page
        dict(name="append_passages", op="append", n=9, len_lo=700, len_hi=4200, q_lo=600, q_hi=4000, hkv=8, d=128,
             dtype="bf16", ragged=7),
        # a batch of search queries through an encoder layer: short, ragged, both directions visible
        dict(name="window_queries", op="window", n=64, len_lo=5, len_hi=60, hq=3, hkv=1, d=256, window=512, sinks=0,
             causal=False, dtype="bf16", ragged=8),
        # documents through a full layer of a small encoder, one kv head per query head
        dict(name="window_documents", op="window", n=6, len_lo=500, len_hi=3001, hq=12, hkv=12, d=64, window=0, sinks=0,
             causal=False, dtype="f16", ragged=9),
        # a long prompt through a windowed causal layer with sinks
        dict(name="window_long_causal", op="window", n=2, len_lo=7001, len_hi=8192, hq=16, hkv=4, d=128, window=1024, sinks=4,
             causal=True, dtype="bf16", ragged=10),
        # beams: every step the children are dropped and forked again from their parents
        dict(name="pages_fork", op="fork", n=8, children=6, len_lo=700, len_hi=3000, layers=8, hkv=8, d=128, ragged=11),
        # requests retire, the cache closes the holes, others are admitted
        dict(name="pages_compact", op="compact", n=48, len_lo=100, len_hi=2000, layers=4, hkv=8, d=128, ragged=12),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["decode", "decode", "chunk", "append", "window", "window", "fork", "compact"])
    ragged = rng.randrange(1 << 30)
    d = rng.choice([64, 128, 256])
    hkv = rng.choice([1, 2, 3, 4, 8])
    g = rng.choice([1, 2, 3, 4, 6, 8])
    dtype = rng.choice(["bf16", "f16"])
    windowed = rng.random() < 0.4
    window, sinks = (_log(rng, 16, 4096), rng.choice([0, 1, 4, 70])) if windowed else (0, 0)
    if op == "decode":
        n = _log(rng, 1, 128)
        top = int(min(131071, 9.0e8 / (n * hkv * 2 * d)))
        hi = _log(rng, 1, max(2, top))
        return dict(op="attend", n=n, len_lo=max(1, hi // rng.choice([1, 2, 20])), len_hi=hi, q_lo=1, q_hi=1, hq=hkv * g, hkv=hkv, d=d,
                    window=window, sinks=sinks, dtype=dtype, ragged=ragged)
    if op == "chunk":
        n = _log(rng, 1, 16)
        q_hi = _log(rng, 2, 800)
        top = int(min(32768, 1.2e9 / (n * hkv * g * q_hi), 4.0e8 / (n * hkv * 2 * d)))
        hi = max(q_hi, _log(rng, 16, max(17, top)))
        return dict(op="attend", n=n, len_lo=max(1, q_hi, hi // 2), len_hi=hi, q_lo=max(1, q_hi // 3), q_hi=q_hi, hq=hkv * g, hkv=hkv,
                    d=d, window=window, sinks=sinks, dtype=dtype, ragged=ragged)
    if op == "append":
        n = _log(rng, 1, 256)
        q_hi = _log(rng, 1, max(2, min(4000, 20000 // n)))
        return dict(op="append", n=n, len_lo=q_hi, len_hi=q_hi + _log(rng, 1, 700), q_lo=max(1, q_hi // 4), q_hi=q_hi, hkv=hkv, d=d,
                    dtype=dtype, ragged=ragged)
    if op == "window":
        n = _log(rng, 1, 64)
        hi = _log(rng, 1, int(min(8192, math.sqrt(1.5e9 / (n * hkv * g)))))
        return dict(op="window", n=n, len_lo=max(1, hi // rng.choice([1, 3, 10])), len_hi=hi, hq=hkv * g, hkv=hkv, d=d, window=window,
                    sinks=sinks, causal=rng.random() < 0.5, dtype=dtype, ragged=ragged)
    if op == "fork":
        n, children = _log(rng, 1, 16), _log(rng, 1, 8)
        return dict(op="fork", n=n, children=children, len_lo=1, len_hi=_log(rng, 65, 3000), layers=rng.choice([1, 2, 4, 8]), hkv=hkv,
                    d=d, ragged=ragged)
    n = _log(rng, 2, 48)
    return dict(op="compact", n=n, len_lo=1, len_hi=_log(rng, 65, 2000), layers=rng.choice([1, 2, 4]), hkv=hkv, d=d, ragged=ragged)


def _lens(case):
    """The case's sequence lengths and tokens per sequence: part of the case, the same for every seed."""
    rng = random.Random(case["ragged"])
    lens = [_log(rng, case["len_lo"], case["len_hi"]) for _ in range(case["n"])]
    if "q_lo" not in case:
        return lens, lens
    toks = [min(n, _log(rng, case["q_lo"], case["q_hi"])) for n in lens]
    return lens, toks


def _cu(toks):
    cu = [0]
    for t in toks:
        cu.append(cu[-1] + t)
    return cu


def _pages(tokens):
    return (tokens + PAGE - 1) // PAGE


# ---- inputs -----------------------------------------------------------------------------------------------------------


def _pool(case, gen, layers, pages):
    """A pool as appends leave it: codes that fill their range, scales that differ from page to page."""
    h, d = case["hkv"], case["d"]
    codes = torch.empty(layers, pages, 2, h, PAGE * d, dtype=torch.int8, device="cuda")
    for la in range(layers):
        step = max(1, (1 << 28) // (2 * h * PAGE * d))
        for at in range(0, pages, step):
            part = codes[la, at:at + step]
            x = torch.empty(part.shape, dtype=torch.float16, device="cuda").normal_(0.0, 35.0, generator=gen)
            part.copy_(x.clamp_(-127, 127).round_())
    scales = torch.exp(torch.randn(layers, pages, 2, h, generator=gen, device="cuda") * 0.3) / 35.0
    return codes, scales


def _tables(lens, spare, gen, first_seen=None):
    """Sequence i's pages at random places of the pool; pages below first_seen(i) that no query sees any more are gone."""
    need = [_pages(n) for n in lens]
    width = max(need) + 2
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32).cpu()
    tables = torch.full((len(lens), width), -1, dtype=torch.int32)
    at = 0
    for i, m in enumerate(need):
        tables[i, :m] = order[at:at + m]
        at += m
        if first_seen is not None:
            lo, keep = first_seen[i]
            tables[i, keep:max(keep, lo)] = -1
    refs = torch.zeros(pages, dtype=torch.int32)
    live = tables[tables >= 0].long()
    refs[live] = 1
    return tables, refs, pages


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed * 1000003 + 17)
    op = case["op"]
    lens, toks = _lens(case)
    st = {"case": dict(case), "seqs": torch.arange(len(lens), dtype=torch.int32, device="cuda")}
    if op == "window":
        return _prepare_window(case, gen, st, lens)
    layers = case.get("layers", 1)
    if op == "fork":
        return _prepare_fork(case, gen, st, lens, layers)
    if op == "compact":
        return _prepare_compact(case, gen, st, lens, layers)
    seen = None
    if case.get("window"):
        keep = _pages(case["sinks"])
        seen = [(max(0, n - t - case["window"] + 1) // PAGE, keep) for n, t in zip(lens, toks)]
        need = [min(_pages(n), keep) + max(0, _pages(n) - max(lo, keep)) for n, (lo, _) in zip(lens, seen)]
        tables, _, _ = _tables(lens, 0, gen, seen)
        pages = sum(need) + 3
        order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32).cpu()
        live = tables >= 0
        tables[live] = order[:int(live.sum())]
        refs = torch.zeros(pages, dtype=torch.int32)
        refs[tables[live].long()] = 1
    else:
        tables, refs, pages = _tables(lens, 3, gen)
    st["codes"], st["scales"] = _pool(case, gen, layers, pages)
    st["tables"], st["refs"] = tables.cuda(), refs.cuda()
    st["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    cu = _cu(toks)
    st["cu"] = torch.tensor(cu, dtype=torch.int32, device="cuda")
    st["max_q"] = max(toks)
    dt = DTYPES[case["dtype"]]
    total = cu[-1]
    if op == "attend":
        # queries of a trained layer: logits with a spread of a few units
        q = torch.randn(total, case["hq"], case["d"], generator=gen, device="cuda") * 1.5
        st["q"] = q.to(dt)
    else:
        # keys have a few large channels, values do not
        chan = torch.exp(torch.randn(case["hkv"], case["d"], generator=gen, device="cuda") * 0.7)
        kv = torch.empty(total, 2, case["hkv"], case["d"], dtype=dt, device="cuda")
        kv[:, 0] = (torch.randn(total, case["hkv"], case["d"], generator=gen, device="cuda") * chan).to(dt)
        kv[:, 1] = torch.randn(total, case["hkv"], case["d"], generator=gen, device="cuda").to(dt)
        st["k"], st["v"] = kv[:, 0], kv[:, 1]  # halves of one projection's output
    _handle(st)
    return st


def _handle(st):
    if own:
        M = _package()
        dev = M.default_device()
        dev.use_torch_stream()
        st["cache"] = M.KvCache(st["codes"], st["scales"], st["tables"], st["lens"], st["refs"], dev=dev)


def _prepare_window(case, gen, st, lens):
    cu = _cu(lens)
    dt = DTYPES[case["dtype"]]
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    # one projection's output holds q, k and v side by side
    qkv = torch.empty(cu[-1], hq + 2 * hkv, d, dtype=dt, device="cuda")
    qkv[:, :hq] = (torch.randn(cu[-1], hq, d, generator=gen, device="cuda") * 1.5).to(dt)
    qkv[:, hq:] = torch.randn(cu[-1], 2 * hkv, d, generator=gen, device="cuda").to(dt)
    st["q"], st["k"], st["v"] = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    st["cu"] = torch.tensor(cu, dtype=torch.int32, device="cuda")
    st["max_len"] = max(lens)
    if own:
        M = _package()
        st["dev"] = M.default_device()
        st["dev"].use_torch_stream()
    return st


def _prepare_fork(case, gen, st, lens, layers):
    """n parents, `children` forks of each; a pass drops the children and forks them again, from other parents' order."""
    n, c = case["n"], case["children"]
    tables, refs, pages = _tables(lens, n * c + 5, gen)
    kids = n * c
    full = torch.full((n + kids, tables.shape[1]), -1, dtype=torch.int32)
    full[:n] = tables
    st["codes"], st["scales"] = _pool(case, gen, layers, pages)
    st["tables"], st["refs"] = full.cuda(), refs.cuda()
    st["lens"] = torch.tensor(lens + [0] * kids, dtype=torch.int32, device="cuda")
    st["children"] = torch.arange(n, n + kids, dtype=torch.int32, device="cuda")
    st["parents"] = torch.randint(0, n, (kids,), generator=gen, device="cuda").to(torch.int32)
    _handle(st)
    return st


def _prepare_compact(case, gen, st, lens, layers):
    """Two halves of the sequences retire in turn; a pass releases one, compacts, and admits as many tokens again."""
    tables, refs, pages = _tables(lens, 7, gen)
    st["codes"], st["scales"] = _pool(case, gen, layers, pages)
    st["tables"], st["refs"] = tables.cuda(), refs.cuda()
    st["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    st["halves"] = [st["seqs"][0::2].contiguous(), st["seqs"][1::2].contiguous()]
    st["admit"] = [st["lens"][0::2].clone(), st["lens"][1::2].clone()]
    st["turn"] = 0
    _handle(st)
    return st


# ---- one pass ---------------------------------------------------------------------------------------------------------


def run(state):
    case = state["case"]
    return {"attend": _run_attend, "append": _run_append, "window": _run_window, "fork": _run_fork,
            "compact": _run_compact}[case["op"]](state, case)


def _run_attend(st, case):
    if own:
        if st["max_q"] == 1:
            return {"out": st["cache"].attend(0, st["q"], st["seqs"], window=case["window"], sinks=case["sinks"])}
        out, lse = st["cache"].attend(0, st["q"], st["seqs"], st["cu"], max_q=st["max_q"], window=case["window"],
                                      sinks=case["sinks"], return_lse=True)
        return {"out": out, "lse": lse}
    h, d, hq = case["hkv"], case["d"], case["hq"]
    n, g, mq = case["n"], hq // h, st["max_q"]
    rows = st["tables"][st["seqs"].long()]
    width = rows.shape[1]
    pick = rows.clamp(min=0).long()
    page = st["codes"][0][pick]  # [n, width, 2, h, 64 * d]
    sc = st["scales"][0][pick]   # [n, width, 2, h]
    k = page[:, :, 0].view(n, width, h, d // 64, PAGE, 64).permute(0, 2, 1, 4, 3, 5).float()
    k = (k * sc[:, :, 0].permute(0, 2, 1)[..., None, None, None]).reshape(n, h, width * PAGE, d)
    v = page[:, :, 1].view(n, width, h, d, PAGE).permute(0, 2, 1, 4, 3).float()
    v = (v * sc[:, :, 1].permute(0, 2, 1)[..., None, None]).reshape(n, h, width * PAGE, d)
    tok = torch.arange(st["q"].shape[0], device="cuda")
    of = torch.searchsorted(st["cu"][1:].long(), tok, right=True)
    at = tok - st["cu"].long()[of]
    q = torch.zeros(n, mq, hq, d, device="cuda")
    q[of, at] = st["q"].float()
    lens = st["lens"][st["seqs"].long()].long()
    count = (st["cu"][1:] - st["cu"][:-1]).long()
    pos = (lens - count)[:, None] + torch.arange(mq, device="cuda")[None]
    key = torch.arange(width * PAGE, device="cuda")
    gone = (rows < 0).repeat_interleave(PAGE, 1)
    see = _visible(pos, key, case["window"], case["sinks"], True) & (key < lens[:, None])[:, None] & ~gone[:, None]
    out, lse = _plain(q, k, v, see, g)
    if mq == 1:
        return {"out": out[of, at].to(st["q"].dtype)}
    return {"out": out[of, at].to(st["q"].dtype), "lse": lse[of, at]}


def _visible(pos, key, window, sinks, causal):
    """[n, queries, keys]: which keys each query sees."""
    off = pos[:, :, None] - key
    see = off >= 0 if causal else torch.ones_like(off, dtype=torch.bool)
    if window:
        see = see & ((off.abs() < window) | (key < sinks))
    return see


def _plain(q, k, v, see, g):
    """Softmax attention in 32 bits: q [n, mq, hq, d], k and v [n, h, keys, d], see [n, mq, keys]."""
    n, mq, hq, d = q.shape
    h = k.shape[1]
    qh = q.view(n, mq, h, g, d).permute(0, 2, 1, 3, 4).reshape(n, h, mq * g, d)
    s = torch.matmul(qh, k.transpose(2, 3)).view(n, h, mq, g, -1) / math.sqrt(d)
    s = s.masked_fill_(~see[:, None, :, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    p = s.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(n, h, mq * g, -1), v).view(n, h, mq, g, d) / torch.where(total > 0, total, torch.ones_like(total))
    lse = (m + total.log())[..., 0]
    return o.permute(0, 2, 1, 3, 4).reshape(n, mq, hq, d), lse.permute(0, 2, 1, 3).reshape(n, mq, hq)


def _run_append(st, case):
    if own:
        c = st["cache"]
        c.append(0, st["k"], st["v"], st["seqs"], st["cu"])
        k, v = c.read(0, st["seqs"], st["cu"], tokens=st["k"].shape[0])
        return {"k": k, "v": v, "codes": st["codes"], "scales": st["scales"]}
    h, d = case["hkv"], case["d"]
    cu = st["cu"].long()
    tok = torch.arange(st["k"].shape[0], device="cuda")
    of = torch.searchsorted(cu[1:], tok, right=True)
    seq = st["seqs"].long()[of]
    start = st["lens"].long()[seq] - (cu[of + 1] - cu[of])
    pos = start + tok - cu[of]
    page = st["tables"][seq, pos // PAGE].long()
    slot = pos % PAGE
    x = torch.stack([st["k"], st["v"]], 1).float()  # [t, 2, h, d]
    pages = st["refs"].shape[0]
    fine = torch.where(torch.isfinite(x), x, torch.zeros_like(x))
    top = torch.zeros(pages, 2, h, device="cuda").index_reduce_(0, page, fine.abs().amax(-1), "amax")
    older = torch.zeros(pages, dtype=torch.long, device="cuda")
    older[page] = (start - (pos - slot)).clamp(min=0)  # tokens that the page held before: the same for each of its new tokens
    was = st["scales"][0]
    touched = torch.zeros(pages, dtype=torch.bool, device="cuda")
    touched[page] = True
    had = (older > 0)[:, None, None]
    grown = torch.maximum(top * INV127, 2.0 * was)
    now = torch.where(had, torch.where(top <= 127.0 * was, was, grown), top * INV127)
    now = torch.where(touched[:, None, None], now, was)
    redo = (had & (now > was))
    which = redo.any(-1).any(-1).nonzero()[:, 0]
    ratio = torch.where(redo, was / now, torch.ones_like(now))[which]
    old = st["codes"][0][which].float()
    st["codes"][0][which] = (old * ratio[..., None]).round().to(torch.int8)
    st["scales"][0].copy_(now)
    s = now[page][..., None]
    code = torch.where(s > 0, x / s, torch.zeros_like(x))
    code = torch.where(torch.isnan(code), torch.zeros_like(code), code).round().clamp(-127, 127).to(torch.int8)
    k_view = st["codes"][0].view(pages, 2, h, d // 64, PAGE, 64)
    v_view = st["codes"][0].view(pages, 2, h, d, PAGE)
    k_view[page, 0, :, :, slot] = code[:, 0].view(-1, h, d // 64, 64)
    v_view[page, 1, :, :, slot] = code[:, 1]
    sk, sv = now[page, 0][..., None], now[page, 1][..., None]
    return {"k": code[:, 0].float() * sk, "v": code[:, 1].float() * sv, "codes": st["codes"], "scales": st["scales"]}


def _run_window(st, case):
    if own:
        out, lse = _package().window_attention(st["q"], st["k"], st["v"], st["cu"], max_len=st["max_len"], causal=case["causal"],
                                               window=case["window"], sinks=case["sinks"], return_lse=True, dev=st["dev"])
        return {"out": out, "lse": lse}
    n, mq = case["n"], st["max_len"]
    hq, h, d = case["hq"], case["hkv"], case["d"]
    cu = st["cu"].long()
    tok = torch.arange(st["q"].shape[0], device="cuda")
    of = torch.searchsorted(cu[1:], tok, right=True)
    at = tok - cu[of]
    q = torch.zeros(n, mq, hq, d, device="cuda")
    k = torch.zeros(n, mq, h, d, device="cuda")
    v = torch.zeros(n, mq, h, d, device="cuda")
    q[of, at], k[of, at], v[of, at] = st["q"].float(), st["k"].float(), st["v"].float()
    lens = cu[1:] - cu[:-1]
    pos = torch.arange(mq, device="cuda")
    see = _visible(pos[None].expand(n, -1), pos, case["window"], case["sinks"], case["causal"]) & (pos < lens[:, None])[:, None]
    out, lse = _plain(q, k.transpose(1, 2), v.transpose(1, 2), see, hq // h)
    return {"out": out[of, at].to(st["q"].dtype), "lse": lse[of, at]}


def _whole(st):
    return {"tables": st["tables"], "lens": st["lens"], "refs": st["refs"], "codes": st["codes"], "scales": st["scales"]}


def _release(st, seqs):
    s = seqs.long()
    rows = st["tables"][s]
    held = rows[rows >= 0].long()
    st["refs"].index_add_(0, held, torch.full_like(held, -1, dtype=torch.int32))
    st["tables"][s] = -1
    st["lens"][s] = 0


def _run_fork(st, case):
    if own:
        c = st["cache"]
        c.release(st["children"])
        c.fork(st["parents"], st["children"])
        return _whole(st)
    _release(st, st["children"])
    par, kid = st["parents"].long(), st["children"].long()
    rows = st["tables"][par]
    lens = st["lens"][par].long()
    full, part = lens // PAGE, lens % PAGE > 0
    col = torch.arange(rows.shape[1], device="cuda")
    share = rows[(col < full[:, None]) & (rows >= 0)].long()
    st["refs"].index_add_(0, share, torch.ones_like(share, dtype=torch.int32))
    with_tail = part.nonzero()[:, 0]
    fresh = (st["refs"] == 0).nonzero()[:, 0][:with_tail.shape[0]]
    src = rows[with_tail, full[with_tail]].long()
    st["codes"][:, fresh] = st["codes"][:, src]
    st["scales"][:, fresh] = st["scales"][:, src]
    st["refs"][fresh] = 1
    rows[with_tail, full[with_tail]] = fresh.to(torch.int32)
    st["tables"][kid] = rows
    st["lens"][kid] = lens.to(torch.int32)
    return _whole(st)


def _run_compact(st, case):
    turn = st["turn"]
    st["turn"] = 1 - turn
    gone, admit = st["halves"][turn], st["admit"][turn]
    if own:
        c = st["cache"]
        c.release(gone)
        c.compact()
        c.reserve(gone, admit)
        return _whole(st)
    _release(st, gone)
    refs = st["refs"]
    live = (refs > 0).sum()
    ids = torch.arange(refs.shape[0], device="cuda")
    holes = ((refs == 0) & (ids < live)).nonzero()[:, 0]
    high = ((refs > 0) & (ids >= live)).nonzero()[:, 0]
    st["codes"][:, holes] = st["codes"][:, high]
    st["scales"][:, holes] = st["scales"][:, high]
    to = ids.to(torch.int32)
    to[high] = holes.to(torch.int32)
    refs[holes] = refs[high]
    refs[high] = 0
    t = st["tables"]
    t.copy_(torch.where(t >= 0, to[t.clamp(min=0).long()], t))
    s = gone.long()
    was = st["lens"][s].long()
    need = (was + admit + PAGE - 1) // PAGE - (was + PAGE - 1) // PAGE
    fresh = (refs == 0).nonzero()[:, 0][:int(need.sum())]
    refs[fresh] = 1
    col = torch.arange(t.shape[1], device="cuda")
    first = (was + PAGE - 1) // PAGE
    new = (col >= first[:, None]) & (col < (first + need)[:, None])
    rows = t[s]
    rows[new] = fresh.to(torch.int32)
    t[s] = rows
    st["lens"][s] = (was + admit).to(torch.int32)
    return _whole(st)


# ---- what a pass cannot do without ------------------------------------------------------------------------------------


def _pairs(n_keys, first, count, window, sinks, causal):
    """(visible pairs, keys that any query sees) of queries at positions first .. first + count - 1."""
    pairs, lo_seen = 0, n_keys
    for p in range(first, first + count):
        hi = min(n_keys, p + 1) if causal else n_keys
        lo = 0
        if window:
            lo = max(0, p - window + 1)
            hi = min(hi, p + window)
        pairs += max(0, hi - lo) + (min(lo, sinks) if window else 0)
        lo_seen = min(lo_seen, lo)
    top = n_keys if not causal else min(n_keys, first + count)
    return pairs, max(0, top - lo_seen) + (min(lo_seen, sinks) if window else 0)


def work(case):
    lens, toks = _lens(case)
    h, d = case["hkv"], case["d"]
    op = case["op"]
    if op in ("attend", "window"):
        pairs = keys = 0
        for n, t in zip(lens, toks):
            a, b = _pairs(n, n - t, t, case["window"], case["sinks"], case.get("causal", True))
            pairs, keys = pairs + a, keys + b
        rows = sum(toks) * case["hq"]
        io = rows * d * 2 * 2 + (rows * 4 if op == "window" or max(toks) > 1 else 0)
        per_key = 2 * h * d * (1 if op == "attend" else 2) + (2 * h * 4 / PAGE if op == "attend" else 0)
        return {"bytes": io + keys * per_key, "flops": 4.0 * d * case["hq"] * pairs}
    if op == "append":
        t = sum(toks)
        return {"bytes": t * 2 * h * d * (2 + 1 + 4), "flops": 4.0 * t * 2 * h * d}
    page = case["layers"] * 2 * h * (PAGE * d + 4)
    if op == "fork":
        # of the parents that the seed picks, the share with a partial last page
        part = sum(1 for n in lens if n % PAGE) / len(lens) * case["n"] * case["children"]
        return {"bytes": part * page * 2 + case["n"] * case["children"] * (2 * _pages(sum(lens) // len(lens)) * 4), "flops": 0.0}
    a, b = lens[0::2], lens[1::2]
    left = sum(_pages(n) for n in b)
    total = left + sum(_pages(n) for n in a)
    moved = left * (1 - left / total)  # of pages at random places, those above the live count
    return {"bytes": moved * page * 2 + total * 8, "flops": 0.0}


# ---- in 64 bits -------------------------------------------------------------------------------------------------------


def _exact_rows(q, k, v, pos, window, sinks, causal):
    """One sequence: q [t, hq, d], k and v [keys, h, d], all float64; out [t, hq, d], lse [t, hq]."""
    g = q.shape[1] // k.shape[1]
    j = torch.arange(k.shape[0], device=q.device)
    out, lse = torch.empty_like(q), torch.empty(q.shape[:2], dtype=torch.float64, device=q.device)
    for at in range(0, q.shape[0], 512):
        p = pos[at:at + 512, None]
        ok = torch.ones(p.shape[0], j.shape[0], dtype=torch.bool, device=q.device)
        if causal:
            ok &= j <= p
        if window:
            ok &= ((p - j < window) & (j - p < window)) | (j < sinks)
        for head in range(q.shape[1]):
            s = (q[at:at + 512, head] @ k[:, head // g].T) * q.shape[2] ** -0.5
            s[~ok] = -math.inf
            z = torch.logsumexp(s, 1)
            w = torch.where(ok, torch.exp(s - torch.where(torch.isfinite(z), z, 0.0)[:, None]), 0.0)
            lse[at:at + 512, head] = z
            out[at:at + 512, head] = w @ v[:, head // g]
    return out, lse


def _exact_page(codes, scales, which, d):
    """K or V rows [64, h, d] of one page in float64."""
    c = codes[which].double()
    h = c.shape[0]
    rows = c.view(h, d // 64, PAGE, 64).permute(2, 0, 1, 3).reshape(PAGE, h, d) if which == 0 else c.view(h, d, PAGE).permute(2, 0, 1)
    return rows * scales[which].double()[:, None]


def exact(case, seed):
    lens, toks = _lens(case)
    global own
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    op = case["op"]
    if op == "window":
        outs = []
        cu = _cu(lens)
        for a, b in zip(cu, cu[1:]):
            q, k, v = (st[x][a:b].double() for x in ("q", "k", "v"))
            outs.append(_exact_rows(q, k, v, torch.arange(b - a, device="cuda"), case["window"], case["sinks"], case["causal"]))
        return {"out": torch.cat([o for o, _ in outs]), "lse": torch.cat([e for _, e in outs])}
    if op == "attend":
        outs = []
        cu = _cu(toks)
        d = case["d"]
        tables = st["tables"].cpu().tolist()
        for i, n in enumerate(lens):
            ids = tables[i][:_pages(n)]
            k, v = (torch.stack([_exact_page(st["codes"][0, max(p, 0)], st["scales"][0, max(p, 0)], w, d) for p in ids])
                    .reshape(-1, case["hkv"], d)[:n] for w in (0, 1))
            q = st["q"][cu[i]:cu[i + 1]].double()
            outs.append(_exact_rows(q, k, v, torch.arange(n - toks[i], n, device="cuda"), case["window"], case["sinks"], True))
        out = {"out": torch.cat([o for o, _ in outs])}
        if max(toks) > 1:
            out["lse"] = torch.cat([e for _, e in outs])
        return out
    if op == "append":
        return _exact_append(case, st, lens, toks)
    return _exact_pages(case, st, lens)


def _exact_append(case, st, lens, toks):
    """Page by page, in 64 bits: the scales and the values that the cache holds for the new tokens."""
    cu = _cu(toks)
    tables = st["tables"].cpu().tolist()
    scales = st["scales"].double().cpu()
    held = [torch.zeros(cu[-1], case["hkv"], case["d"], dtype=torch.float64) for _ in (0, 1)]
    new = [st[x].double().cpu() for x in ("k", "v")]
    for i, n in enumerate(lens):
        pos = n - toks[i]
        while pos < n:
            end = min(n, (pos // PAGE + 1) * PAGE)
            rows = slice(cu[i] + pos - (n - toks[i]), cu[i] + end - (n - toks[i]))
            page = tables[i][pos // PAGE]
            for w in (0, 1):
                x = new[w][rows]
                top = x.abs().amax(dim=(0, 2))
                s = top / 127
                if pos % PAGE:
                    old = scales[0, page, w]
                    s = torch.where(top <= 127 * old, old, torch.maximum(s, 2 * old))
                scales[0, page, w] = s
                held[w][rows] = torch.round(x / s[:, None]).clamp(-127, 127) * s[:, None]
            pos = end
    return {"k": held[0], "v": held[1], "codes": None, "scales": scales}


def _exact_pages(case, st, lens):
    """The page bookkeeping step by step on the host."""
    t = st["tables"].cpu().numpy().copy()
    lens = st["lens"].cpu().numpy().copy()
    refs = st["refs"].cpu().numpy().copy()
    scales = st["scales"].double().cpu()
    src = list(range(len(refs)))  # whose contents each page holds

    def release(s):
        for p in t[s]:
            if p >= 0:
                refs[p] -= 1
        t[s] = -1
        lens[s] = 0

    def take():
        p = int((refs == 0).argmax())
        refs[p] = 1
        return p

    if case["op"] == "fork":
        par, kid = st["parents"].cpu().tolist(), st["children"].cpu().tolist()
        for c in kid:
            release(c)
        for p in par:
            for x in t[p][:lens[p] // PAGE]:
                refs[x] += 1
        for p, c in zip(par, kid):
            t[c], lens[c] = t[p], lens[p]
            if lens[p] % PAGE:
                new = take()
                src[new] = src[t[p][lens[p] // PAGE]]
                t[c][lens[p] // PAGE] = new
    else:
        gone, admit = st["halves"][0].cpu().tolist(), st["admit"][0].cpu().tolist()
        for s in gone:
            release(s)
        live = int((refs > 0).sum())
        low = [p for p in range(live) if refs[p] == 0]
        high = [p for p in range(live, len(refs)) if refs[p] > 0]
        for a, b in zip(low, high):
            src[a], refs[a], refs[b] = src[b], refs[b], 0
            t[t == b] = a
        for s, n in zip(gone, admit):
            for i in range(_pages(int(n))):
                t[s][i] = take()
            lens[s] = n
    return {"tables": torch.from_numpy(t), "lens": torch.from_numpy(lens), "refs": torch.from_numpy(refs), "codes": None,
            "scales": scales[:, src]}
