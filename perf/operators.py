"""The serving operators around a windowed paged cache, as measured workloads.

Five operators over the paged K/V cache ``[num_blocks, block_size, Hkv, D]``:

* ``decode``: attention of one new token per sequence under a sliding window
  with a few first tokens (sinks) that stay visible,
* ``prompt``: the same attention for chunks of new tokens (causal),
* ``resize``: page accounting of a step: pages that left the window or a
  shortened sequence are freed, new ones are taken, shared tails are copied,
* ``fork``: a sequence continued several times: full pages shared, the partly
  filled last page copied in every layer,
* ``compact``: live pages moved to the front of the pool in every layer.

``run`` computes them in plain torch (``own`` false) or through the package.
Query position p sees token t when t <= p and (t < sinks or t > p - window).
"""
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
SENTINEL = -1e30


def _package():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                        "paged-attention-triton_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import paged_attention
    return paged_attention


# ---------------------------------------------------------------- cases
def listed():
    return [
        # a single chat stream far beyond its window: one token's latency
        dict(name="decode_b1_s32768_w1024", op="decode", dtype="bf16", b=1, hq=32, hkv=8, d=128,
             bs=16, smin=32768, smax=32768, window=1024, sinks=4, lens=1),
        # a serving batch of mixed lengths, full heads, pages of 32 tokens
        dict(name="decode_b48_mha_f16_w511", op="decode", dtype="f16", b=48, hq=16, hkv=16, d=64,
             bs=32, smin=1, smax=4096, window=511, sinks=5, lens=2),
        # a large batch of long streams with grouped heads
        dict(name="decode_b128_gqa8_w4096", op="decode", dtype="bf16", b=128, hq=64, hkv=8, d=128,
             bs=16, smin=512, smax=32768, window=4096, sinks=16, lens=3),
        # a few draft tokens verified on long streams: short chunks
        dict(name="prompt_b4_q7_s8192_w1024", op="prompt", dtype="bf16", b=4, hq=32, hkv=8, d=128,
             bs=16, qmin=5, qmax=7, smin=4096, smax=8192, window=1024, sinks=4, lens=4),
        # a mixed batch of prompt chunks, ragged in both lengths
        dict(name="prompt_b8_ragged_f16_d64", op="prompt", dtype="f16", b=8, hq=16, hkv=4, d=64,
             bs=32, qmin=33, qmax=1000, smin=1000, smax=4096, window=777, sinks=3, lens=5),
        # one long prompt in one pass
        dict(name="prompt_b1_q8192_w4096", op="prompt", dtype="bf16", b=1, hq=32, hkv=8, d=128,
             bs=16, qmin=8192, qmax=8192, smin=8192, smax=8192, window=4096, sinks=4, lens=6),
        # one decode step of a large batch: a page every few rows, old pages freed
        dict(name="resize_step_b256_w4096", op="resize", mode="step", dtype="bf16", b=256, hkv=8,
             d=128, bs=16, layers=1, smin=512, smax=32768, window=4096, sinks=4, share=0, lens=7),
        # a scheduler's turn: some rows end, some begin, some go on from shared tails
        dict(name="resize_turn_b64_shared", op="resize", mode="turn", dtype="f16", b=64, hkv=4,
             d=64, bs=32, layers=16, smin=1, smax=4096, window=0, sinks=0, share=1, lens=8),
        # parallel sampling of one short prompt
        dict(name="fork_1to4_s700", op="fork", dtype="bf16", b=1, ways=4, hkv=8, d=128, bs=16,
             layers=8, smin=700, smax=700, lens=9),
        # beam search over a batch: every row continued three more times
        dict(name="fork_32x3_l16_bs64", op="fork", dtype="f16", b=32, ways=3, hkv=8, d=128, bs=64,
             layers=16, smin=17, smax=1024, lens=10),
        # a small pool after half of its rows ended
        dict(name="compact_512_pages_l4", op="compact", dtype="f16", b=24, hkv=8, d=64, bs=16,
             layers=4, pool=512, fill=0.45, lens=11),
        # a whole model's pool, thinned out
        dict(name="compact_4096_pages_l16", op="compact", dtype="bf16", b=96, hkv=8, d=128, bs=16,
             layers=16, pool=4096, fill=0.6, lens=12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["decode", "decode", "prompt", "prompt", "resize", "fork", "compact"])
    c = dict(op=op, dtype=rng.choice(["f16", "bf16"]), lens=rng.randrange(1 << 20))
    d = rng.choice([64, 128])
    bs = rng.choice([8, 16, 32, 64, 128])
    hkv = rng.choice([1, 2, 4, 8])
    if op == "decode":
        g = rng.choice([1, 2, 3, 4, 8])
        window, smax = _log(rng, 16, 4096), _log(rng, 64, 32768)
        c.update(b=_log(rng, 1, 128), hq=hkv * g, hkv=hkv, d=d, bs=bs,
                 smin=rng.choice([1, max(1, smax // 2), smax]), smax=smax, window=window,
                 sinks=rng.choice([0, 1, 4, 5, 16, 33]))
    elif op == "prompt":
        g = rng.choice([1, 2, 4, 5, 8])
        b = _log(rng, 1, 12)
        qmax = _log(rng, 1, 4096 // b)
        smax = qmax + _log(rng, 1, 4096)
        c.update(b=b, hq=hkv * g, hkv=hkv, d=d, bs=bs, qmin=rng.choice([1, (qmax + 1) // 2, qmax]),
                 qmax=qmax, smin=(qmax + smax) // 2, smax=smax, window=_log(rng, 16, 4096),
                 sinks=rng.choice([0, 1, 4, 17]))
    elif op == "resize":
        smax = _log(rng, 64, 16384)
        c.update(mode=rng.choice(["step", "turn"]), b=_log(rng, 1, 200), hkv=hkv, d=64, bs=bs,
                 layers=rng.randint(1, 4), smin=1, smax=smax,
                 window=rng.choice([0, _log(rng, 16, 4096)]), sinks=rng.choice([0, 4, 33]),
                 share=rng.choice([0, 1]))
        if c["share"] or c["mode"] == "turn":
            c["smax"] = min(smax, 2048)
            c["b"] = min(c["b"], 48)
    elif op == "fork":
        c.update(b=_log(rng, 1, 24), ways=rng.randint(1, 4), hkv=hkv, d=d, bs=bs,
                 layers=rng.randint(1, 16), smin=1, smax=_log(rng, 16, 2048))
    else:
        c.update(b=_log(rng, 1, 96), hkv=hkv, d=d, bs=min(bs, 32), layers=rng.randint(1, 12),
                 pool=_log(rng, 128, 2048), fill=round(rng.uniform(0.1, 0.95), 3))
    return c


def _lengths(c):
    """Sequence lengths of a case (log-uniform), the same for every seed."""
    r = random.Random(c["lens"])
    lo, hi = c["smin"], c["smax"]
    return [min(hi, max(lo, _log(r, lo, hi))) for _ in range(c["b"])]


def _chunks(c):
    """(new tokens, whole length) of each sequence of a prompt case."""
    r = random.Random(c["lens"])
    out = []
    for _ in range(c["b"]):
        q = r.randint(c["qmin"], c["qmax"])
        out.append((q, max(q, r.randint(c["smin"], c["smax"]))))
    return out


def _first(pos, c):
    """First token inside the window of position `pos`."""
    return max(0, pos - c["window"] + 1)


def _pages_needed(first, length, c):
    """Pages of a stream whose tokens in [sinks, first) have been given up."""
    bs = c["bs"]
    return [j for j in range(-(-length // bs))
            if j * bs < c["sinks"] or (j + 1) * bs > first]


# ---------------------------------------------------------------- inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(shape, g, dtype):
    return torch.randn(shape, generator=g, device="cuda", dtype=dtype)


def _table(rows, width, perm):
    """Block table whose row r has the next shuffled pages at the logical pages rows[r], -1 elsewhere."""
    flat = [(r, j) for r, js in enumerate(rows) for j in js]
    t = torch.full((len(rows), width), -1, dtype=torch.int32)
    if flat:
        at = torch.tensor(flat)
        t[at[:, 0], at[:, 1]] = perm[: len(flat)]
    return t


def _attention_state(c, seed, qlens, slens, firsts):
    g = _gen(seed)
    dt = DTYPES[c["dtype"]]
    rows = [_pages_needed(f, s, c) for f, s in zip(firsts, slens)]
    pool = sum(map(len, rows)) + 7
    perm = torch.randperm(pool, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    width = max(-(-s // c["bs"]) for s in slens)
    shape = (pool, c["bs"], c["hkv"], c["d"])
    st = dict(c=c, q=_normal((sum(qlens), c["hq"], c["d"]), g, dt), k=_normal(shape, g, dt),
              v=_normal(shape, g, dt), table=_table(rows, width, perm).cuda(),
              lens=torch.tensor(slens, dtype=torch.int32).cuda())
    if c["sinks"]:
        # the first tokens draw attention: their keys are longer than the others'
        st["k"][st["table"][:, 0].long(), : min(c["sinks"], c["bs"])] *= 1.5
    return st


def _pool_state(c, seed, slens, new_rows=0):
    """A pool of `layers` layers' caches, tables and lengths of the rows, counts of each page's users."""
    g = _gen(seed)
    bs, b = c["bs"], len(slens)
    window = c.get("window", 0)
    sub = dict(c, sinks=c.get("sinks", 0))
    rows = [_pages_needed(max(0, s - 1 - window + 1) if window else 0, s, sub) for s in slens]
    grown = [s + 1 for s in slens] if c.get("mode") == "step" else slens
    width = max(1, max(-(-s // bs) for s in grown + [c.get("smax", 1)])) + 1
    need = sum(map(len, rows))
    pool = c.get("pool", need + need // 4 + 4 * b + 2 * new_rows + 8)
    perm = torch.randperm(pool, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    table = _table(rows + [[]] * new_rows, width, perm)
    lens = torch.tensor(list(slens) + [0] * new_rows, dtype=torch.int32)
    if c.get("share"):
        # every fourth row goes on from the pages of the row before it, the partly filled one among them
        for r in range(1, b, 4):
            table[r] = table[r - 1]
            lens[r] = lens[r - 1]
    used = table[table >= 0].long()
    refs = torch.zeros(pool, dtype=torch.int32).index_add_(0, used, torch.ones(len(used), dtype=torch.int32))
    kv = _normal((c["layers"], 2, pool, bs, c["hkv"], c["d"]), g, DTYPES[c["dtype"]])
    # table, lengths and counts as one buffer each for the start and the working copy, so that a
    # pass begins from the same accounting
    start = torch.cat([table.reshape(-1), lens]).cuda()
    st = dict(c=c, kv=kv, start=start, work=start.clone(), refs0=refs.cuda(), shape=tuple(table.shape))
    n = table.numel()
    st["table"], st["lens"] = st["work"][:n].view(table.shape), st["work"][n:]
    if own:
        pa = _package()
        st["pool"] = pa.PagePool([kv[l, 0] for l in range(c["layers"])], [kv[l, 1] for l in range(c["layers"])])
        st["pool"].adopt(st["table"], st["lens"])
        st["pool0"] = st["pool"].state.clone()
    else:
        st["refs"] = st["refs0"].clone()
    return st


def prepare(case, seed):
    c = dict(case)
    op = c["op"]
    if op == "decode":
        slens = _lengths(c)
        return _attention_state(c, seed, [1] * c["b"], slens, [_first(s - 1, c) for s in slens])
    if op == "prompt":
        ch = _chunks(c)
        st = _attention_state(c, seed, [q for q, _ in ch], [s for _, s in ch],
                              [_first(s - q, c) for q, s in ch])
        starts = [0]
        for q, _ in ch:
            starts.append(starts[-1] + q)
        st["starts"] = torch.tensor(starts, dtype=torch.int32).cuda()
        return st
    if op == "compact":
        st = _pool_state(c, seed, _compact_lengths(c))
        return st
    slens = _lengths(c)
    if op == "fork":
        n = c["b"] * c["ways"]
        st = _pool_state(c, seed, slens, new_rows=n)
        st["parents"] = torch.tensor([i % c["b"] for i in range(n)], dtype=torch.int32).cuda()
        st["children"] = torch.arange(c["b"], c["b"] + n, dtype=torch.int32).cuda()
        return st
    st = _pool_state(c, seed, slens)
    st["new"] = torch.tensor(_new_lengths(c, st["lens"].tolist()), dtype=torch.int32).cuda()
    return st


def _compact_lengths(c):
    """Rows that fill the wanted share of the pool's pages."""
    want = int(c["fill"] * c["pool"])
    base = [want // c["b"] + (i < want % c["b"]) for i in range(c["b"])]
    r = random.Random(c["lens"])
    return [max(0, n * c["bs"] - r.randint(0, c["bs"] - 1)) if n else 0 for n in base]


def _new_lengths(c, lens):
    if c["mode"] == "step":
        return [s + 1 for s in lens]
    r = random.Random(c["lens"] + 1)
    out = []
    for i, s in enumerate(lens):
        kind = r.randrange(4) if not (c["share"] and i % 4 < 2) else 3
        out.append([0, max(0, s - 5), -1, min(c["smax"], s + 1 + r.randrange(9))][kind])
    return out


# ---------------------------------------------------------------- the operators
def run(state):
    c = state["c"]
    op = c["op"]
    if op in ("decode", "prompt"):
        if own:
            return _attention_own(state)
        return _decode_plain(state) if op == "decode" else _prompt_plain(state)
    state["work"].copy_(state["start"])
    if own:
        state["pool"].state.copy_(state["pool0"])
        return _pages_own(state)
    state["refs"].copy_(state["refs0"])
    return {"resize": _resize_plain, "fork": _fork_plain, "compact": _compact_plain}[op](state)


def _attention_own(st):
    pa, c = _package(), st["c"]
    if c["op"] == "decode":
        o, lse = pa.paged_attention(st["q"], st["k"], st["v"], st["table"], st["lens"], c["bs"],
                                    window=c["window"], num_sinks=c["sinks"], return_lse=True)
    else:
        o, lse = pa.paged_prompt_attention(st["q"], st["k"], st["v"], st["table"], st["starts"],
                                           st["lens"], c["bs"], window=c["window"],
                                           num_sinks=c["sinks"], return_lse=True)
    return {"o": o, "lse": lse}


def _pages_own(st):
    c, pool = st["c"], st["pool"]
    out = {"table": st["table"], "refs": pool.refs}
    if c["op"] == "compact":
        out["live"] = pool.compact(st["table"])
    elif c["op"] == "fork":
        pool.fork(st["table"], st["lens"], st["parents"], st["children"])
        out["lens"] = st["lens"]
    else:
        pool.resize(st["table"], st["lens"], st["new"], window=c["window"] or None,
                    num_sinks=c["sinks"] if c["window"] else 0)
        out["lens"] = st["lens"]
    if c["op"] != "resize" or c["share"]:
        out["kv"] = st["kv"]
    return out


def _softmax_v(s, seen, v):
    """softmax(s) v over the last axis of s where `seen`; (output, log of the sum of exp)."""
    s = torch.where(seen, s, torch.full_like(s, -math.inf))
    top = s.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    p = torch.exp(s - top)
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v) / total.clamp_min(1e-30)
    lse = torch.where(total > 0, top + torch.log(total), torch.full_like(total, SENTINEL))
    return o, lse[..., 0]


def _decode_plain(st):
    c = st["c"]
    bs, hkv, d, g = c["bs"], c["hkv"], c["d"], c["hq"] // c["hkv"]
    s = st["lens"].long()
    most = min(c["smax"], c["window"] + c["sinks"])
    first = (s - c["window"]).clamp_min(0)
    heads = first.clamp_max(c["sinks"])
    i = torch.arange(most, device="cuda")
    tok = torch.where(i < heads[:, None], i, first[:, None] + i - heads[:, None])
    seen = tok < s[:, None]
    tok = torch.where(seen, tok, s[:, None] - 1)
    at = st["table"].long().gather(1, tok // bs) * bs + tok % bs
    k = st["k"].view(-1, hkv, d)[at].float().permute(0, 2, 3, 1)       # [B, Hkv, D, V]
    v = st["v"].view(-1, hkv, d)[at].float().permute(0, 2, 1, 3)       # [B, Hkv, V, D]
    q = st["q"].float().view(-1, hkv, g, d)
    o, lse = _softmax_v(torch.matmul(q, k) / math.sqrt(d), seen[:, None, None], v)
    return {"o": o.reshape(-1, c["hq"], d).to(st["q"].dtype), "lse": lse.reshape(-1, c["hq"])}


def _prompt_plain(st):
    c = st["c"]
    bs, hkv, d, g, b = c["bs"], c["hkv"], c["d"], c["hq"] // c["hkv"], c["b"]
    starts, s = st["starts"].long(), st["lens"].long()
    n = starts[1:] - starts[:-1]
    wide = c["qmax"]
    i = torch.arange(wide, device="cuda")
    valid = i < n[:, None]                                             # [B, Q]
    row = torch.where(valid, starts[:-1, None] + i, torch.zeros_like(i))
    pos = s[:, None] - n[:, None] + i
    t = torch.arange(st["table"].shape[1] * bs, device="cuda")
    page = st["table"].long().clamp_min(0).repeat_interleave(bs, 1)
    at = page * bs + t % bs                                            # [B, S]
    k = st["k"].view(-1, hkv, d)[at].float().permute(0, 2, 3, 1)
    v = st["v"].view(-1, hkv, d)[at].float().permute(0, 2, 1, 3)
    q = st["q"][row].float().view(b, wide, hkv, g, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, g * wide, d)
    seen = (t <= pos[..., None]) & ((t < c["sinks"]) | (t > pos[..., None] - c["window"]))
    seen = seen[:, None, None].expand(b, 1, g, wide, t.numel()).reshape(b, 1, g * wide, t.numel())
    o, lse = _softmax_v(torch.matmul(q, k) / math.sqrt(d), seen, v)
    o = o.view(b, hkv, g, wide, d).permute(0, 3, 1, 2, 4).reshape(b, wide, c["hq"], d)
    lse = lse.view(b, hkv, g, wide).permute(0, 3, 1, 2).reshape(b, wide, c["hq"])
    # rows in order of the packed queries
    total = st["q"].shape[0]
    r = torch.arange(total, device="cuda")
    seq = (r[:, None] >= starts[None, 1:]).sum(1)
    off = r - starts[seq]
    return {"o": o[seq, off].to(st["q"].dtype), "lse": lse[seq, off]}


def _free_list(refs):
    """Indices of the free pages in ascending order, then the others."""
    return torch.sort((refs > 0).to(torch.int32), stable=True).indices


def _copy_slots(kv, src, dst, used, do):
    """Pages src -> dst (their first `used` slots) in every layer where `do`; elsewhere a page onto itself."""
    slot = torch.arange(kv.shape[3], device="cuda")
    src = torch.where(do, src, dst)
    keep = (slot < used[:, None])[None, None, :, :, None, None]
    kv[:, :, dst] = torch.where(keep, kv[:, :, src], kv[:, :, dst])


def _resize_plain(st):
    c = st["c"]
    bs, table, lens, refs = c["bs"], st["table"], st["lens"], st["refs"]
    pool = refs.numel()
    j = torch.arange(table.shape[1], device="cuda")
    s = lens.long()
    n = torch.where(st["new"] >= 0, st["new"].long(), s)
    used, want, q0 = (s + bs - 1) // bs, (n + bs - 1) // bs, torch.minimum(s, n)
    drop = j >= want[:, None]
    if c["window"]:
        drop = drop | ((j >= -(-c["sinks"] // bs)) & ((j + 1) * bs <= (q0 - c["window"] + 1)[:, None]))
    drop = drop & (j < used[:, None]) & (st["new"] >= 0)[:, None] & (table >= 0)
    refs.index_add_(0, table.clamp_min(0).reshape(-1).long(), -drop.reshape(-1).to(torch.int32))
    table.masked_fill_(drop, -1)
    last = (s // bs).clamp_max(table.shape[1] - 1)
    tail = table.gather(1, last[:, None])[:, 0].long()
    cow = (n > s) & (s % bs != 0) & (tail >= 0) & (refs[tail.clamp_min(0)] > 1)
    need = (want - used).clamp_min(0) + cow
    end = need.cumsum(0)
    ok = end <= (refs == 0).sum()
    begin = end - need
    free = _free_list(refs)
    grow = ok[:, None] & (j >= used[:, None]) & (j < want[:, None])
    page = free[((begin + cow)[:, None] + j - used[:, None]).clamp(0, pool - 1)]
    table.copy_(torch.where(grow, page.to(torch.int32), table))
    cow = cow & ok
    fresh = free[begin.clamp_max(pool - 1)]
    here = table.gather(1, last[:, None])[:, 0]
    table.scatter_(1, last[:, None], torch.where(cow, fresh.to(torch.int32), here)[:, None])
    refs.index_add_(0, page.reshape(-1), grow.reshape(-1).to(torch.int32))
    refs.index_add_(0, fresh, cow.to(torch.int32))
    refs.index_add_(0, tail.clamp_min(0), -cow.to(torch.int32))
    lens.copy_(torch.where(ok | (n < s), n, s))
    out = {"table": table, "refs": refs, "lens": lens}
    if c["share"]:
        at = cow.nonzero()[:, 0]
        _copy_slots(st["kv"], tail[at], fresh[at], (s % bs)[at], cow[at])
        out["kv"] = st["kv"]
    return out


def _fork_plain(st):
    c = st["c"]
    bs, table, lens, refs = c["bs"], st["table"], st["lens"], st["refs"]
    pool = refs.numel()
    p, ch = st["parents"].long(), st["children"].long()
    j = torch.arange(table.shape[1], device="cuda")
    s = lens[p].long()
    full, rest = s // bs, s % bs
    need = (rest > 0).long()
    end = need.cumsum(0)
    ok = end <= (refs == 0).sum()
    fresh = _free_list(refs)[(end - need).clamp_max(pool - 1)]
    rows = table[p]
    tail = rows.gather(1, full[:, None])[:, 0].long()
    share = ok[:, None] & (j < full[:, None])
    mine = torch.where(share, rows, torch.full_like(rows, -1))
    copied = ok & (rest > 0)
    mine.scatter_(1, full[:, None], torch.where(copied, fresh, torch.full_like(fresh, -1)).to(torch.int32)[:, None])
    table[ch] = mine
    lens[ch] = torch.where(ok, s, torch.zeros_like(s)).to(torch.int32)
    refs.index_add_(0, rows.clamp_min(0).reshape(-1).long(), (share & (rows >= 0)).reshape(-1).to(torch.int32))
    refs.index_add_(0, fresh, copied.to(torch.int32))
    at = copied.nonzero()[:, 0]
    _copy_slots(st["kv"], tail[at], fresh[at], rest[at], copied[at])
    return {"table": table, "refs": refs, "lens": lens, "kv": st["kv"]}


def _compact_plain(st):
    table, refs, kv = st["table"], st["refs"], st["kv"]
    i = torch.arange(refs.numel(), device="cuda")
    live = refs > 0
    n = live.sum()
    holes, movers = (~live & (i < n)).nonzero()[:, 0], (live & (i >= n)).nonzero()[:, 0]
    kv[:, :, holes] = kv[:, :, movers]
    to = i.to(torch.int32)
    to[movers] = holes.to(torch.int32)
    table.copy_(torch.where(table >= 0, to[table.clamp_min(0).long()], table))
    refs[holes] = refs[movers]
    refs[movers] = 0
    return {"table": table, "refs": refs, "live": n.to(torch.int32).reshape(1), "kv": kv}


# ---------------------------------------------------------------- cost and definition
def work(case):
    c = case
    op = c["op"]
    e = 2
    if op in ("decode", "prompt"):
        chunks = [(1, s) for s in _lengths(c)] if op == "decode" else _chunks(c)
        pairs = tokens = rows = 0
        for q, s in chunks:
            for pos in range(s - q, s):
                f = _first(pos, c)
                pairs += pos + 1 - f + min(c["sinks"], f)
            f = _first(s - q, c)
            tokens += s - f + min(c["sinks"], f)
            rows += q
        kv = 2 * tokens * c["hkv"] * c["d"] * e
        return {"bytes": kv + rows * c["hq"] * (2 * c["d"] * e + 4), "flops": 4 * pairs * c["hq"] * c["d"]}
    slot = c["hkv"] * c["d"] * e * 2 * c["layers"]
    if op == "compact":
        # on average a share (1 - fill) of the live pages lies behind the live count
        live = sum(-(-s // c["bs"]) for s in _compact_lengths(c))
        moved = live * (c["pool"] - live) // c["pool"]
        return {"bytes": 2 * moved * c["bs"] * slot + 8 * live + 8 * c["pool"], "flops": 0}
    lens = _lengths(c)
    pages = sum(-(-s // c["bs"]) for s in lens)
    if op == "fork":
        copied = c["ways"] * sum(s % c["bs"] for s in lens)
        return {"bytes": 2 * copied * slot + 16 * c["ways"] * pages, "flops": 0}
    new, copied = _new_lengths(c, _shared(c, lens)), 0
    if c["share"]:
        lens = _shared(c, lens)
        for r in range(1, c["b"], 4):
            copied += sum(lens[x] % c["bs"] for x in (r - 1, r) if new[x] > lens[x])
    touched = sum(abs(-(-max(n, 0) // c["bs"]) - -(-s // c["bs"])) for n, s in zip(new, lens) if n >= 0)
    return {"bytes": 2 * copied * slot + 12 * touched + 12 * c["b"] + 4 * pages, "flops": 0}


def _shared(c, lens):
    lens = list(lens)
    if c.get("share"):
        for r in range(1, len(lens), 4):
            lens[r] = lens[r - 1]
    return lens


def exact(case, seed):
    """Attention by its definition in 64 bits, sequence by sequence; page operators only move and count."""
    if case["op"] not in ("decode", "prompt"):
        return None
    st = prepare(case, seed)
    c, q = st["c"], st["q"].double()
    g = c["hq"] // c["hkv"]
    starts = list(range(c["b"] + 1)) if c["op"] == "decode" else st["starts"].tolist()
    o, lse = torch.empty_like(q), torch.empty(q.shape[:2], dtype=torch.float64, device="cuda")
    for b, length in enumerate(st["lens"].tolist()):
        n = starts[b + 1] - starts[b]
        low = max(0, length - n - c["window"] + 1)
        tokens = torch.cat([torch.arange(min(c["sinks"], low)), torch.arange(low, length)]).cuda()
        pages = st["table"][b][tokens // c["bs"]].long()
        keys, values = (st[x][pages, tokens % c["bs"]].double() for x in ("k", "v"))
        at = torch.arange(length - n, length, device="cuda")[:, None]
        hidden = (tokens > at) | ((tokens >= c["sinks"]) & (tokens <= at - c["window"]))
        for h in range(c["hq"]):
            rows = slice(starts[b], starts[b + 1])
            score = q[rows, h] @ keys[:, h // g].T * c["d"] ** -0.5
            score.masked_fill_(hidden, -math.inf)
            norm = torch.logsumexp(score, 1, keepdim=True)
            o[rows, h] = (score - norm).exp_() @ values[:, h // g]
            lse[rows, h] = norm[:, 0]
    return {"o": o, "lse": lse}
