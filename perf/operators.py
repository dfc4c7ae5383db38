"""Cases of the bounded-memory cache operators: paged decode attention, quantize-append into pages (and the read-back),
sliding-window decode attention with sinks, decode attention that accumulates attention weights, and eviction by them.

`run` computes a case in plain torch operations (`own = False`) or through the package's entry points (`own = True`);
`exact` computes it from the definition in 64 bits.

Sizes: the head counts are those of the package's benchmark configurations (12 / 2, 28 / 4, 40 / 8 heads of 128
channels) plus 64-channel heads; groups of 32 and 128 channels per scale.
"""
import math

import torch

own = False
DEV = "cuda"
HEADS = ((12, 2, 128), (28, 4, 128), (40, 8, 128), (14, 2, 64))
FORMATS = ("fp16", "int8", "int4", "int4z")


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # one user, a short chat: pages of 16 tokens, the launch latency is what counts
        dict(name="paged_int8_single", op="paged", fmt="int8", B=1, Hq=12, Hkv=2, D=128, gs=32, page=16, lo=300, hi=300,
             window=0, sinks=0),
        # a serving batch with contexts of every age between one token and 16 K
        dict(name="paged_int8_ragged", op="paged", fmt="int8", B=32, Hq=28, Hkv=4, D=128, gs=128, page=64, lo=1, hi=16384,
             window=0, sinks=0),
        # four long documents in 4 bits with zero-points, odd lengths
        dict(name="paged_int4z_long", op="paged", fmt="int4z", B=4, Hq=40, Hkv=8, D=128, gs=32, page=32, lo=20001, hi=49999,
             window=0, sinks=0),
        # unquantized pages under a window with sinks
        dict(name="paged_fp16_window", op="paged", fmt="fp16", B=16, Hq=28, Hkv=4, D=128, gs=128, page=16, lo=2000, hi=12000,
             window=4096, sinks=4),
        # one decode step of a batch writes one token per sequence
        dict(name="append_int8_step", op="append", fmt="int8", B=64, Hkv=4, D=128, gs=128, page=64, T=1, lo=5, hi=4000,
             ragged=False),
        # a chunk of prompts of different lengths, padded to the longest
        dict(name="append_int4_prompts", op="append", fmt="int4", B=8, Hkv=8, D=128, gs=32, page=32, T=2048, lo=0, hi=3000,
             ragged=True),
        # contiguous cache, long contexts, the last 4 K tokens and 4 sinks
        dict(name="window_int8_batch", op="window", fmt="int8", B=8, Hq=28, Hkv=4, D=128, gs=32, S=32768, lo=9000, hi=32768,
             window=4096, sinks=4),
        # one very long sequence, a wide window
        dict(name="window_int4_single", op="window", fmt="int4", B=1, Hq=40, Hkv=8, D=128, gs=32, S=131072, lo=131001,
             hi=131001, window=16384, sinks=64),
        # attention that also keeps the sums the eviction ranks by
        dict(name="weights_int8_batch", op="weights", fmt="int8", B=16, Hq=28, Hkv=4, D=128, gs=128, S=8192, lo=4097, hi=8192),
        # the same right after a prompt of one user
        dict(name="weights_int4z_single", op="weights", fmt="int4z", B=1, Hq=12, Hkv=2, D=128, gs=32, S=4096, lo=4001,
             hi=4001),
        # steady state of a bounded cache: one token came in, one has to go
        dict(name="evict_one", op="evict", B=16, Hkv=4, D=128, cap=2304, lo=2049, hi=2049, budget=2048, sinks=4, recent=256,
             fresh=False),
        # after the prompt: the cache shrinks to its budget
        dict(name="evict_prompt", op="evict", B=4, Hkv=8, D=128, cap=32768, lo=32001, hi=32001, budget=4096, sinks=4,
             recent=512, fresh=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_BIGGEST = 2.7e8        # bytes: the largest listed case moves as many


def draw(rng):
    while True:
        op = rng.choice(("paged", "paged", "append", "window", "weights", "evict"))
        Hq, Hkv, D = rng.choice(HEADS)
        fmt = rng.choice(FORMATS)
        gs = rng.choice((32, 64, 128))
        gs = D if fmt == "fp16" else min(gs, D)
        B = _log(rng, 1, 64)
        hi = _log(rng, 1, 50000)
        lo = rng.choice((hi, _log(rng, 1, hi)))
        window = rng.choice((0, _log(rng, 1, 16384)))
        sinks = rng.choice((0, 4, rng.randint(1, 200)))
        page = rng.choice((16, 32, 48, 64, 128))
        if op == "paged":
            c = dict(op=op, fmt=fmt, B=B, Hq=Hq, Hkv=Hkv, D=D, gs=gs, page=page, lo=lo, hi=hi, window=window,
                     sinks=sinks if window else 0)
        elif op == "append":
            c = dict(op=op, fmt=fmt, B=B, Hkv=Hkv, D=D, gs=gs, page=page, T=rng.choice((1, 1, _log(rng, 2, 2048))),
                     lo=min(lo, 4000) - 1, hi=min(hi, 4000) - 1, ragged=rng.random() < 0.5)
        elif op == "window":
            c = dict(op=op, fmt=fmt, B=B, Hq=Hq, Hkv=Hkv, D=D, gs=gs, S=hi + rng.randint(0, 300), lo=lo, hi=hi,
                     window=window or 512, sinks=sinks)
        elif op == "weights":
            hi, lo = min(hi, 16384), min(lo, 16384)
            c = dict(op=op, fmt=fmt, B=B, Hq=Hq, Hkv=Hkv, D=D, gs=gs, S=hi + rng.randint(0, 300), lo=lo, hi=hi)
        else:
            hi = max(hi, 600)
            budget = _log(rng, 300, 8192)
            s, r = rng.choice((0, 4, 32)), _log(rng, 1, 250)
            fresh = rng.random() < 0.5
            n = hi if fresh else budget + rng.randint(1, 8)
            c = dict(op=op, B=min(B, 16), Hkv=Hkv, D=D, cap=max(n, budget) + rng.randint(0, 100), lo=n, hi=n, budget=budget,
                     sinks=s, recent=r, fresh=fresh)
        full = dict(c, window=0) if "window" in c else c        # what has to be made and held
        if work(full)["bytes"] <= _BIGGEST and _held(c) <= 1.0e9:
            return c


def _lens(case):
    """Row lengths, evenly spread over [lo, hi]; the seed only decides which row has which."""
    B, lo, hi = case["B"], case["lo"], case["hi"]
    return [lo + (hi - lo) * i // max(B - 1, 1) for i in range(B)] if B > 1 else [hi]


def _new_lens(case):
    B, T = case["B"], case["T"]
    return [T - (T * i) // (2 * B) for i in range(B)] if case["ragged"] else [T] * B


def _side_bytes(case):
    """Bytes of one cached token of one head, K and V."""
    D, gs, fmt = case["D"], case["gs"], case["fmt"]
    if fmt == "fp16":
        return 4 * D
    G = D // gs
    return 2 * (D if fmt == "int8" else D // 2) + 4 * G * (2 if fmt == "int4z" else 1)


def _visible(n, window, sinks):
    return n if window == 0 else min(n, window + min(sinks, max(n - window, 0)))


def _held(case):
    if case["op"] == "evict":
        return case["B"] * case["Hkv"] * case["cap"] * (4 * case["D"] + 8)
    if case["op"] == "append":
        return 3 * case["B"] * case["Hkv"] * (case["hi"] + case["T"]) * 4 * case["D"]
    S = case.get("S", case["hi"])
    return case["B"] * case["Hkv"] * S * 4 * case["D"]


def work(case):
    """Bytes and operations of one pass: every input read once, every output written once."""
    B, Hkv, D, op = case["B"], case["Hkv"], case["D"], case["op"]
    if op in ("paged", "window", "weights"):
        Hq = case["Hq"]
        vis = sum(_visible(n, case.get("window", 0), case.get("sinks", 0)) for n in _lens(case))
        b = vis * Hkv * _side_bytes(case) + 4 * B * Hq * D + 4 * B
        if op == "paged":
            b += 4 * sum(-(-n // case["page"]) for n in _lens(case))
        if op == "weights":
            b += vis * Hkv * 8
        return {"bytes": b, "flops": 4 * D * Hq * vis}
    if op == "append":
        tok = sum(_new_lens(case)) * Hkv
        # read the tokens, write them to the pages; read the pages, write the values (zeros for the padding)
        b = tok * (4 * D + 2 * _side_bytes(case)) + B * case["T"] * Hkv * 4 * D
        return {"bytes": b, "flops": 8 * tok * D}
    n, m = case["hi"], min(case["hi"], case["budget"])
    # the sums and positions, and the rows that have to move: at least those of the protected tail of the context
    moved = min(max(n - m, 0), case["recent"])
    rows = B * Hkv
    return {"bytes": rows * (n * 8 + moved * 2 * (4 * D + 8)), "flops": rows * n * 4}


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(1 + seed * 7919)


def _values(shape, gen):
    """fp16 keys or values: normal, with a spread of the channels' sizes between 0.3 and 3."""
    std = torch.exp(torch.empty(shape[-1], device=DEV).uniform_(math.log(0.3), math.log(3.0), generator=gen))
    x = torch.randn(shape, generator=gen, device=DEV, dtype=torch.float16)
    return x.mul_(std.to(torch.float16))


def _encode(x, fmt, gs):
    """(payload, scale, zero-point) of fp16 values [..., D]: absmax groups, or min / max groups with a zero-point.
    Divisors are tensors: torch turns a division by a Python number into a product with its reciprocal."""
    if fmt == "fp16":
        return x.clone(), None, None
    D = x.shape[-1]
    g = x.float().unflatten(-1, (D // gs, gs))

    def over(a, d):
        return a / torch.full_like(a, d)

    zp = None
    if fmt == "int4z":
        lo, hi = g.amin(-1), g.amax(-1)
        s = over((hi - lo).clamp_min(15.0 * 2.0 ** -14), 15.0)
        zp = lo + 8.0 * s
        c = torch.round((g - zp.unsqueeze(-1)) / s.unsqueeze(-1)).clamp_(-8, 7)
    else:
        amax = g.abs().amax(-1).clamp_min(1e-5).half().float()      # the clamp is one of fp16 values
        if fmt == "int8":
            s = over(amax, 127.0).half().float()
            # the quotient is rounded to the values' type before it becomes an integer
            c = torch.round((g / s.unsqueeze(-1)).half().float()).clamp_(-127, 127)
        else:
            s = over(amax.clamp_min(1e-5), 7.0)
            c = torch.round(g / s.unsqueeze(-1)).clamp_(-7, 7)
    c = c.flatten(-2).to(torch.int8)
    if fmt != "int8":
        u = (c + 8).to(torch.uint8)
        c = ((u[..., 0::2] << 4) | u[..., 1::2]).view(torch.int8)
    return c, s.half(), (None if zp is None else zp.half())


def _encode_rows(x, fmt, gs):
    """_encode, a slice of the first dimension at a time."""
    step = max(1, (1 << 26) // max(1, x[0].numel()))
    parts = [_encode(x[i:i + step], fmt, gs) for i in range(0, x.shape[0], step)]
    return tuple(None if parts[0][j] is None else torch.cat([p[j] for p in parts]) for j in range(3))


def _decode32(payload, scale, zp, fmt):
    """Cached values in 32 bits (the product of a code and an fp16 scale is exact there)."""
    if fmt == "fp16":
        return payload.float()
    if fmt != "int8":
        u = payload.view(torch.uint8)
        payload = torch.stack(((u >> 4).to(torch.int8) - 8, (u & 15).to(torch.int8) - 8), -1).flatten(-2)
    G = scale.shape[-1]
    x = payload.float().unflatten(-1, (G, payload.shape[-1] // G)) * scale.float().unsqueeze(-1)
    if zp is not None:
        x = x + zp.float().unsqueeze(-1)
    return x.flatten(-2)


def _row_lens(case, gen):
    lens = torch.tensor(_lens(case), device=DEV, dtype=torch.int32)
    return lens[torch.randperm(case["B"], generator=gen, device=DEV)]


def _pages(case, lens_max, gen):
    """A pool with spare pages in random order and the table of every row; entries past a row's pages are -1."""
    B, page = case["B"], case["page"]
    per = [-(-n // page) for n in lens_max.tolist()]
    width = max(max(per), 1)
    total = sum(per)
    pool = total + max(1, total // 16)
    order = torch.randperm(pool, generator=gen, device=DEV).to(torch.int32)
    table = torch.full((B, width), -1, device=DEV, dtype=torch.int32)
    at = 0
    for b, p in enumerate(per):
        table[b, :p] = order[at:at + p]
        at += p
    return pool, table


def prepare(case, seed):
    gen = _gen(seed)
    op, B, Hkv, D = case["op"], case["B"], case["Hkv"], case["D"]
    st = {"case": case}
    if op == "evict":
        cap, n, budget, sinks, recent = case["cap"], case["hi"], case["budget"], case["sinks"], case["recent"]
        st["lengths"] = torch.full((B,), n, device=DEV, dtype=torch.int32)
        w = torch.exp(2.0 * torch.randn(B, Hkv, cap, generator=gen, device=DEV))
        # tokens nobody looked at: their sums are equal
        st["weights"] = torch.where(torch.rand(B, Hkv, cap, generator=gen, device=DEV) < 0.05, 0.0, w)
        st["weights"][:, :, n:] = 0
        st["positions"] = torch.full((B, Hkv, cap), -1, device=DEV, dtype=torch.int32)
        if case["fresh"]:
            st["seen"] = torch.full((B,), n, device=DEV, dtype=torch.int32)
        else:
            # `budget` slots hold what earlier rounds kept: sinks first, then older tokens in no order, the recent ones
            # spread over the freed slots; the newest n - budget tokens were appended since
            seen = 4 * budget
            st["seen"] = torch.full((B,), seen, device=DEV, dtype=torch.int32)
            old = seen - (n - budget)
            late = max(0, min(recent, budget - sinks))
            mid = budget - sinks - late
            pos = torch.empty(B * Hkv, budget, device=DEV, dtype=torch.int32)
            for r in range(B * Hkv):
                pick = sinks + torch.randperm(old - late - sinks, generator=gen, device=DEV)[:mid]
                rest = torch.cat((pick, torch.arange(old - late, old, device=DEV)))
                pos[r, :sinks] = torch.arange(sinks, device=DEV)
                pos[r, sinks:] = rest[torch.randperm(rest.numel(), generator=gen, device=DEV)]
            st["positions"][:, :, :budget] = pos.view(B, Hkv, budget)
        st["k"] = torch.randn(B, Hkv, cap, D, generator=gen, device=DEV, dtype=torch.float16)
        st["v"] = torch.randn(B, Hkv, cap, D, generator=gen, device=DEV, dtype=torch.float16)
        return st
    fmt, gs = case["fmt"], case["gs"]
    if op == "append":
        start = _row_lens(case, gen)
        st["start"] = start
        st["new_lens"] = torch.tensor(_new_lens(case), device=DEV, dtype=torch.int32) if case["ragged"] else None
        pool, st["table"] = _pages(case, start + case["T"], gen)
        G = D // gs
        width = {"fp16": D, "int8": D}.get(fmt, D // 2)
        for s in ("k", "v"):
            st[s] = torch.zeros(pool, Hkv, case["page"], width, device=DEV, dtype=torch.float16 if fmt == "fp16" else torch.int8)
            st[s + "s"] = None if fmt == "fp16" else torch.zeros(pool, Hkv, case["page"], G, device=DEV, dtype=torch.float16)
            st[s + "z"] = torch.zeros_like(st[s + "s"]) if fmt == "int4z" else None
            st[s + "_new"] = _values((B, Hkv, case["T"], D), gen)
        return st
    st["q"] = torch.randn(B, case["Hq"], D, generator=gen, device=DEV, dtype=torch.float16)
    lens = _row_lens(case, gen)
    st["lens"] = lens
    if op == "paged":
        pool, st["table"] = _pages(case, lens, gen)
        shape = (pool, Hkv, case["page"], D)
    else:
        shape = (B, Hkv, case["S"], D)
    for s in ("k", "v"):
        st[s], st[s + "s"], st[s + "z"] = _encode_rows(_values(shape, gen), fmt, gs)
    if op == "weights":
        w = torch.exp(torch.randn(B, Hkv, case["S"], generator=gen, device=DEV)) * 0.01
        # the newest token has no sum yet
        slot = torch.arange(case["S"], device=DEV)
        st["weights"] = torch.where(slot < (lens - 1).clamp_min(0)[:, None, None], w, torch.zeros_like(w))
    return st


# ------------------------------------------------------------------------------------------------ plain forms
def _plain_row(q, k, v, n, window, sinks, Hkv):
    """One row: q [Hq, D], k / v fp32 [Hkv, S, D] -> (out fp32 [Hq, D], probabilities [Hkv, rep, S])."""
    Hq, D = q.shape
    S = k.shape[1]
    slot = torch.arange(S, device=q.device)
    seen = slot < n
    if window:
        seen = seen & ((slot < sinks) | (slot >= n - window))
    x = torch.matmul(q.float().view(Hkv, Hq // Hkv, D), k.transpose(1, 2)) * (1.0 / math.sqrt(D))
    x = x.masked_fill(~seen, float("-inf"))
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(m == float("-inf"), torch.zeros_like(m), m))
    total = e.sum(-1, keepdim=True)
    p = torch.where(total > 0, e / total, torch.zeros_like(e))
    v = torch.where(seen[:, None], v, torch.zeros_like(v))
    return torch.matmul(p, v).reshape(Hq, D), p


def _plain_attention(st):
    case = st["case"]
    fmt, Hkv, page = case["fmt"], case["Hkv"], case.get("page")
    window, sinks = case.get("window", 0), case.get("sinks", 0)
    outs = []
    for b in range(case["B"]):
        n = st["lens"][b]
        side = []
        for s in ("k", "v"):
            parts = (st[s], st[s + "s"], st[s + "z"])
            if case["op"] == "paged":
                idx = st["table"][b].clamp_min(0).long()
                parts = tuple(None if t is None else t[idx].transpose(0, 1).flatten(1, 2) for t in parts)
            else:
                parts = tuple(None if t is None else t[b] for t in parts)
            side.append(_decode32(*parts, fmt))
        out, p = _plain_row(st["q"][b], side[0], side[1], n, window, sinks, Hkv)
        outs.append(out)
        if case["op"] == "weights":
            st["weights"][b] += p.sum(1)
    return torch.stack(outs).half()


def _plain_append(st):
    case = st["case"]
    B, T, page = case["B"], case["T"], case["page"]
    t = torch.arange(T, device=DEV)
    pos = st["start"][:, None].long() + t
    new = st["new_lens"] if st["new_lens"] is not None else torch.full((B,), T, device=DEV, dtype=torch.int32)
    live = t < new[:, None]
    pid = st["table"].long().gather(1, pos // page).clamp_min(0)
    row = pos % page
    bb, tt = live.nonzero(as_tuple=True)
    pg, rw = pid[bb, tt], row[bb, tt]
    outs = {}
    for s in ("k", "v"):
        enc = _encode(st[s + "_new"].transpose(1, 2)[bb, tt], case["fmt"], case["gs"])        # [N, Hkv, .]
        for name, x in zip((s, s + "s", s + "z"), enc):
            if x is not None:
                st[name][pg, :, rw] = x
        got = _decode32(*(None if st[n] is None else st[n][pg, :, rw] for n in (s, s + "s", s + "z")), case["fmt"]).half()
        back = torch.zeros_like(st[s + "_new"])
        back.transpose(1, 2)[bb, tt] = got
        outs[s] = back
    return outs


def _plain_evict(st):
    case = st["case"]
    budget, sinks, recent = case["budget"], case["sinks"], case["recent"]
    w, pos = st["weights"], st["positions"]
    cap = w.shape[-1]
    slot = torch.arange(cap, device=DEV)
    n, seen = st["lengths"][:, None, None], st["seen"][:, None, None]
    m = n.clamp_max(budget)
    where = torch.where(pos >= 0, pos, seen - n + slot)
    live = (slot < n).expand_as(w)
    kept = live & ((where < sinks) | (where >= seen - recent))
    rank = torch.where(w != w, torch.full_like(w, float("-inf")), w)
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices
    cls = torch.where(kept, 0, torch.where(live, 1, 2)).gather(-1, order)
    order = order.gather(-1, torch.sort(cls, dim=-1, stable=True).indices)
    keep = torch.zeros_like(live).scatter_(-1, order, slot.expand_as(order) < m)
    # the i-th kept token behind the budget goes to the i-th freed slot before it, row by row
    src = (keep & (slot >= m)).nonzero(as_tuple=True)
    dst = (~keep & (slot < m)).nonzero(as_tuple=True)
    for t in (st["k"], st["v"], w):
        t[dst] = t[src]
    shrink = (n > budget) & live
    new_pos = where.to(torch.int32).clone()
    new_pos[dst] = new_pos[src]
    pos.copy_(torch.where(shrink, torch.where(slot < m, new_pos, -1), pos))
    w.masked_fill_(shrink & (slot >= m), 0.0)
    return st["lengths"].clamp_max(budget)


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    st, case = state, state["case"]
    op = case["op"]
    if own:
        import llm_kvcache_quantization_b200 as kvq
    if op == "paged":
        if not own:
            return _plain_attention(st)
        return kvq.decode_attn_paged(st["q"], st["k"], st["v"], st["ks"], st["vs"], st["table"], st["lens"],
                                     window=case["window"] or None, sinks=case["sinks"], k_zp=st["kz"], v_zp=st["vz"])
    if op == "window":
        if not own:
            return _plain_attention(st)
        return kvq.decode_attn_window(st["q"], st["k"], st["v"], st["ks"], st["vs"], st["lens"], case["window"],
                                      case["sinks"], k_zp=st["kz"], v_zp=st["vz"])
    if op == "weights":
        if own:
            out = kvq.decode_attn_weights(st["q"], st["k"], st["v"], st["ks"], st["vs"], st["lens"], st["weights"],
                                          k_zp=st["kz"], v_zp=st["vz"])
        else:
            out = _plain_attention(st)
        return {"out": out, "weights": st["weights"]}
    if op == "append":
        if own:
            kvq.paged_append(st["k_new"], st["v_new"], st["k"], st["v"], st["ks"], st["vs"], st["table"], st["start"],
                             st["new_lens"], k_zp=st["kz"], v_zp=st["vz"])
            k, v = kvq.paged_read(st["k"], st["v"], st["ks"], st["vs"], st["table"], st["start"], case["T"], st["new_lens"],
                                  head_dim=case["D"], k_zp=st["kz"], v_zp=st["vz"])
            outs = {"k": k, "v": v}
        else:
            outs = _plain_append(st)
        for name in ("ks", "vs", "kz", "vz"):
            if st[name] is not None:
                outs[name] = st[name]
        return outs
    if own:
        lengths = kvq.evict_tokens(st["weights"], st["positions"], st["lengths"], st["seen"], case["budget"],
                                   (st["k"], st["v"]), sinks=case["sinks"], recent=case["recent"])
    else:
        lengths = _plain_evict(st)
    return {"lengths": lengths, "weights": st["weights"], "positions": st["positions"], "k": st["k"], "v": st["v"]}


# ------------------------------------------------------------------------------------------------ 64 bits
def _exact_tokens(st, s, index, fmt):
    """float64 values [len, Hkv, D] of the cached tokens that `index` selects (a tuple into the leading dimensions, the
    head dimension a slice)."""
    x = st[s][index]
    if fmt == "fp16":
        return x.double()
    if fmt in ("int4", "int4z"):
        byte = x.long() & 255
        x = torch.empty(*byte.shape[:-1], byte.shape[-1] * 2, device=byte.device, dtype=torch.long)
        x[..., 0::2] = torch.div(byte, 16, rounding_mode="floor") - 8
        x[..., 1::2] = byte % 16 - 8
    sc = st[s + "s"][index].double()
    rep = x.shape[-1] // sc.shape[-1]
    y = x.double() * sc.repeat_interleave(rep, dim=-1)
    return y + st[s + "z"][index].double().repeat_interleave(rep, dim=-1) if fmt == "int4z" else y


def exact(case, seed):
    st = prepare(case, seed)
    op, B, Hkv, D = case["op"], case["B"], case["Hkv"], case["D"]
    every = slice(None)
    if op in ("paged", "window", "weights"):
        rep = case["Hq"] // Hkv
        out = torch.zeros(B, case["Hq"], D, device=DEV, dtype=torch.float64)
        sums = st["weights"].double() if op == "weights" else None
        for b, n in enumerate(st["lens"].tolist()):
            if n == 0:
                continue
            first = 0 if not case.get("window") else max(0, n - case["window"])
            tok = torch.cat((torch.arange(min(case.get("sinks", 0), first), device=DEV), torch.arange(first, n, device=DEV)))
            for part in range(Hkv):
                one = slice(part, part + 1)
                if op == "paged":
                    index = (st["table"][b].long()[tok // case["page"]], one, tok % case["page"])
                else:
                    index = (b, one, tok)
                k, v = (_exact_tokens(st, s, index, case["fmt"]).reshape(tok.numel(), D) for s in ("k", "v"))
                z = st["q"][b, part * rep:(part + 1) * rep].double() @ k.t() / math.sqrt(D)
                p = torch.exp(z - torch.logsumexp(z, -1, keepdim=True))
                out[b, part * rep:(part + 1) * rep] = p @ v
                if sums is not None:
                    sums[b, part, :n] += p.sum(0)
        return out if sums is None else {"out": out, "weights": sums}
    if op == "append":
        fmt, gs, page = case["fmt"], case["gs"], case["page"]
        res = {}
        new = st["new_lens"].tolist() if st["new_lens"] is not None else [case["T"]] * B

        def r32(a):
            return a.float().double()

        for s in ("k", "v"):
            val = torch.zeros(B, Hkv, case["T"], D, device=DEV, dtype=torch.float64)
            for b, count in enumerate(new):
                if count == 0:
                    continue
                x = st[s + "_new"][b, :, :count].double()
                if fmt == "fp16":
                    val[b, :, :count] = x
                    continue
                g = x.reshape(Hkv, count, D // gs, gs)
                if fmt == "int4z":
                    top, low = g.max(-1).values, g.min(-1).values
                    # a cached code is defined by 32-bit steps: scale, zero-point, difference and quotient are rounded
                    step = r32(torch.clamp(r32(top - low), min=15 / 2 ** 14) / 15)
                    zero = r32(low + 8 * step)
                    code = torch.clamp(torch.round(r32(r32(g - zero[..., None]) / step[..., None])), -8, 7)
                else:
                    top = torch.clamp(g.abs().max(-1).values, min=1e-5).to(torch.float16).double()
                    if fmt == "int8":
                        step = r32(top / 127).to(torch.float16).double()
                        code = torch.clamp(torch.round(r32(g / step[..., None]).to(torch.float16).double()), -127, 127)
                    else:
                        step = r32(top / 7)
                        code = torch.clamp(torch.round(r32(g / step[..., None])), -7, 7)
                kept = step.to(torch.float16).double()
                y = code * kept[..., None]
                place = torch.arange(count, device=DEV) + st["start"][b]
                pg, rw = st["table"][b].long()[place // page], (place % page).long()
                st[s + "s"][pg, :, rw] = step.to(torch.float16).transpose(0, 1)
                if fmt == "int4z":
                    y = y + zero.to(torch.float16).double()[..., None]
                    st[s + "z"][pg, :, rw] = zero.to(torch.float16).transpose(0, 1)
                val[b, :, :count] = y.reshape(Hkv, count, D)
            res[s] = val
        for name in ("ks", "vs", "kz", "vz"):
            if st[name] is not None:
                res[name] = st[name].double()
        return res
    import numpy as np
    w, pos = st["weights"].cpu().numpy(), st["positions"].cpu().numpy()
    left = []
    for b in range(B):
        n, seen = int(st["lengths"][b]), int(st["seen"][b])
        left.append(min(n, case["budget"]))
        if n <= case["budget"]:
            continue
        m = case["budget"]
        for h in range(Hkv):
            at = np.where(pos[b, h, :n] < 0, seen - n + np.arange(n), pos[b, h, :n])
            safe = (at < case["sinks"]) | (at >= seen - case["recent"])
            score = np.where(np.isnan(w[b, h, :n]), -np.inf, w[b, h, :n].astype(np.float64))
            best = np.lexsort((np.arange(n), -score, ~safe))[:m]
            chosen = np.zeros(n, dtype=bool)
            chosen[best] = True
            home = np.flatnonzero(~chosen[:m])
            away = m + np.flatnonzero(chosen[m:])
            at[home] = at[away]
            w[b, h, home] = w[b, h, away]
            w[b, h, m:n] = 0
            pos[b, h, :m] = at[:m]
            pos[b, h, m:n] = -1
            i, j = torch.from_numpy(home).to(DEV), torch.from_numpy(away).to(DEV)
            for s in ("k", "v"):
                st[s][b, h, i] = st[s][b, h, j]
    return {"lengths": torch.tensor(left, device=DEV, dtype=torch.int32), "weights": torch.from_numpy(w).to(DEV).double(),
            "positions": torch.from_numpy(pos).to(DEV), "k": st["k"].double(), "v": st["v"].double()}
