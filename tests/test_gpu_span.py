"""GPU tests of the bounded and paged cache operators against plain 64-bit implementations (span_reference.py)."""
import ctypes as C
import math

import pytest
import torch

import llm_kvcache_quantization_b200 as kvq
from llm_kvcache_quantization_b200 import _lib, ops
from span_reference import attention, check, evict, make_cache, make_table, paginate, values, visible

pytestmark = pytest.mark.gpu
DEV = "cuda"
FORMATS = ("fp16", "int8", "int8z", "int4", "int4z")


def _d(*ts):
    return tuple(None if t is None else t.to(DEV) for t in ts)


def _flag():
    return _lib.load().kvq_debug_error_flag(1)


def _case(B, Hq, Hkv, D, S, fmt, gs, seed):
    gen = torch.Generator().manual_seed(seed)
    q = torch.randn(B, Hq, D, generator=gen).half()
    k, ks, kz = make_cache((B, Hkv, S), D, fmt, gs, gen)
    v, vs, vz = make_cache((B, Hkv, S), D, fmt, gs, gen)
    return gen, q, k, v, ks, vs, kz, vz


def _poison(t, lens, window=0, sinks=0):
    """NaN / extreme codes in every slot outside the visible span."""
    if t is None:
        return None
    t = t.clone()
    for b, n in enumerate(lens):
        t[b, :, ~visible(n, t.shape[2], window, sinks)] = float("nan") if t.dtype.is_floating_point else 127
    return t


# ------------------------------------------------------------------------------------------------ paged attention
PAGED = [
    # B, Hq, Hkv, D, lens, page, gs, window, sinks
    (1, 12, 2, 128, [1], 16, 32, 0, 0),
    (3, 12, 2, 128, [300, 0, 17], 16, 32, 0, 0),
    (4, 28, 4, 128, [1, 64, 65, 2049], 64, 128, 0, 0),
    (2, 40, 8, 128, [1025, 4097], 32, 64, 0, 0),
    (2, 14, 2, 64, [700, 31], 48, 64, 0, 0),
    (2, 4, 4, 256, [513, 90], 32, 128, 0, 0),
    (2, 20, 1, 128, [777, 1300], 128, 128, 0, 0),          # 20 heads per kv head: three chunks of 8
    (3, 28, 4, 128, [2000, 5, 900], 16, 128, 100, 4),
    (2, 12, 2, 128, [1500, 64], 32, 32, 1, 0),
    (2, 14, 2, 64, [1500, 333], 16, 32, 257, 33),
    (130, 2, 1, 128, [(37 * i) % 300 for i in range(130)], 16, 128, 0, 0),
    (1, 8, 2, 128, [200], 7, 32, 0, 0),                     # a page size only the generic kernel takes
]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("case", range(len(PAGED)))
def test_paged_attention(case, fmt):
    B, Hq, Hkv, D, lens, page, gs, window, sinks = PAGED[case]
    S = max(lens)
    gen, q, k, v, ks, vs, kz, vz = _case(B, Hq, Hkv, D, S, fmt, gs, 100 + case)
    out, tol, _, _ = attention(q, k, v, ks, vs, kz, vz, lens, window, sinks)
    pool, table = make_table(lens, page, gen)
    pages = [paginate(_poison(t, lens, window, sinks), lens, page, pool, table) for t in (k, v, ks, vs, kz, vz)]
    for b, n in enumerate(lens):                            # pages that the window has left may be gone
        for j in range(-(-n // page)):
            if not visible(n, table.shape[1] * page, window, sinks)[j * page:(j + 1) * page].any():
                table[b, j] = -1
    qd, kd, vd, ksd, vsd, kzd, vzd, td = _d(q, *pages, table)
    lend = torch.tensor(lens, dtype=torch.int32, device=DEV)
    got = kvq.decode_attn_paged(qd, kd, vd, ksd, vsd, td, lend, window=window or None, sinks=sinks, k_zp=kzd, v_zp=vzd)
    check(got, out, tol, f"{PAGED[case]} {fmt}")
    again = kvq.decode_attn_paged(qd, kd, vd, ksd, vsd, td, lend, window=window or None, sinks=sinks, k_zp=kzd, v_zp=vzd)
    assert torch.equal(got, again)
    assert _flag() == 0


def test_paged_attention_max_ctx_strided_query_out_and_dtype():
    B, Hq, Hkv, D, page = 2, 12, 2, 128, 32
    lens = [500, 170]
    gen, q, k, v, ks, vs, kz, vz = _case(B, Hq, Hkv, D, 512, "int8", 32, 7)
    pool, table = make_table(lens, page, gen)
    pages = _d(*[paginate(t, lens, page, pool, table) for t in (k, v, ks, vs)])
    tau = torch.empty(Hq).uniform_(0.8, 1.2, generator=gen)
    lend = torch.tensor(lens, device=DEV)                   # int64: cast
    td = table.to(DEV)
    out, tol, _, _ = attention(q, k, v, ks, vs, None, None, [300, 170], inv_tau=tau, sm=0.07)
    qd = torch.empty(B, D, Hq, dtype=torch.float16, device=DEV).transpose(1, 2)
    qd.copy_(q)
    dst = torch.full((B, Hq + 1, D + 8), 7.0, dtype=torch.float16, device=DEV)
    got = kvq.decode_attn_paged(qd, *pages, td, lend, 0.07, max_ctx=300, inv_tau=tau.to(DEV), out=dst[:, 1:, :D])
    check(got, out, tol)
    assert got.data_ptr() == dst[:, 1:, :D].data_ptr()
    assert (dst[:, 0] == 7).all() and (dst[:, :, D:] == 7).all()
    bf = kvq.decode_attn_paged(q.to(DEV).float(), *pages, td, lend, 0.07, max_ctx=300, inv_tau=tau.to(DEV))
    assert bf.dtype == torch.float32 and torch.equal(bf, got.float())


def test_page_outside_the_pool_is_refused_by_the_kernel():
    gen, q, k, v, ks, vs, kz, vz = _case(2, 12, 2, 128, 200, "int8", 32, 8)
    lens = [200, 100]
    pool, table = make_table(lens, 32, gen)
    pages = _d(*[paginate(t, lens, 32, pool, table) for t in (k, v, ks, vs)])
    lend = torch.tensor(lens, dtype=torch.int32, device=DEV)
    good = kvq.decode_attn_paged(q.to(DEV), *pages, table.to(DEV), lend)
    assert _flag() == 0
    for bad in (pool, -1, 2 ** 31 - 1):
        t = table.clone()
        t[0, 3] = bad
        got = kvq.decode_attn_paged(q.to(DEV), *pages, t.to(DEV), lend)
        assert _flag() == 8
        assert torch.equal(got[1], good[1])                 # the other row is untouched
        kvq.paged_read(*pages, t.to(DEV), None, 200, lend, head_dim=128)
        assert _flag() == 8


def test_zero_rows_zero_context_and_empty_batch():
    q = torch.randn(2, 4, 128, device=DEV).half()
    pool = torch.zeros(3, 2, 16, 128, dtype=torch.float16, device=DEV)
    table = torch.full((2, 2), -1, dtype=torch.int32, device=DEV)
    lens = torch.zeros(2, dtype=torch.int32, device=DEV)
    assert (kvq.decode_attn_paged(q, pool, pool, None, None, table, lens) == 0).all()
    neg = torch.full((2,), -5, dtype=torch.int32, device=DEV)
    assert (kvq.decode_attn_paged(q, pool, pool, None, None, table, neg) == 0).all()
    assert kvq.decode_attn_paged(q[:0], pool, pool, None, None, table[:0], lens[:0]).shape == (0, 4, 128)
    empty = torch.zeros(2, 2, 0, 128, dtype=torch.float16, device=DEV)
    assert (kvq.decode_attn_window(q, empty, empty, None, None, None, 8) == 0).all()
    assert _flag() == 0


def test_which_kernel_serves_which_layout():
    def kind(fmt, D, gs, page, zp=False):
        gen = torch.Generator().manual_seed(0)
        k, ks, kz = _d(*make_cache((4, 2, page or 96), D, fmt, gs, gen))
        s = _lib.KvqSpanAttnArgs()
        a = s.attn
        a.format, a.B, a.Hq, a.Hkv, a.D, a.group_size = ops.cache_format(k, D), 4, 8, 2, D, gs
        a.sm_scale, a.max_ctx = 0.1, k.shape[2]
        a.k = a.v = ops._cache_side(k, ks, kz, None)
        if page:
            s.pages = _lib.KvqPageTable(k.data_ptr(), 1, 1, page, 4)
        return _lib.load().kvq_span_attn_kernel_kind(C.byref(s))
    for fmt in FORMATS:
        for D in (64, 128):
            for gs in ((D,) if fmt == "fp16" else (32, D)):
                for page in (0, 32, 64, 128):
                    assert kind(fmt, D, gs, page) == 1, (fmt, D, gs, page)
                assert kind(fmt, D, gs, 16) == (0 if fmt.startswith("int4") and D == 64 else 1)
                assert kind(fmt, D, gs, 8) == 0
        assert kind(fmt, 256, 128, 32) == 0
    assert kind("int8", 128, 16, 32) == 0


# ------------------------------------------------------------------------------------------------ window
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("window,sinks", ((1, 0), (1, 5), (31, 33), (64, 4), (640, 100), (5000, 7)))
@pytest.mark.parametrize("D,gs", ((128, 32), (128, 128), (64, 32)))
def test_window_attention(window, sinks, fmt, D, gs):
    lens = [1, 0, 33, 1024, 1025, 1500]
    S = 1503
    gen, q, k, v, ks, vs, kz, vz = _case(6, 12, 2, D, S, fmt, gs, window * 7 + sinks)
    out, tol, _, _ = attention(q, k, v, ks, vs, kz, vz, lens, window, sinks)
    parts = _d(*[_poison(t, lens, window, sinks) for t in (k, v, ks, vs)])
    kzd, vzd = _d(_poison(kz, lens, window, sinks), _poison(vz, lens, window, sinks))
    lend = torch.tensor(lens, dtype=torch.int32, device=DEV)
    got = kvq.decode_attn_window(q.to(DEV), *parts, lend, window, sinks, k_zp=kzd, v_zp=vzd)
    check(got, out, tol, f"{fmt} window {window} sinks {sinks}")
    assert _flag() == 0


@pytest.mark.parametrize("fmt", ("fp16", "int8", "int4"))
@pytest.mark.parametrize("S", (1, 2, 3, 5, 31, 513))
def test_window_on_tight_odd_caches_reads_nothing_behind_them(fmt, S):
    """The cache tensors end with their last token, in an allocation whose next bytes are NaN / 0x7f."""
    gen, q, k, v, ks, vs, kz, vz = _case(1, 4, 1, 128, S, fmt, 32, S)
    parts = []
    for t in (k, v, ks, vs):
        if t is None:
            parts.append(None)
            continue
        big = torch.full((t.numel() + 4096,), float("nan") if t.dtype.is_floating_point else 127, dtype=t.dtype, device=DEV)
        big[:t.numel()] = t.flatten().to(DEV)
        parts.append(big[:t.numel()].view(t.shape))
    out, tol, _, _ = attention(q, k, v, ks, vs, None, None, [S], 3, 1)
    check(kvq.decode_attn_window(q.to(DEV), *parts, None, 3, 1), out, tol)
    out, tol, _, _ = attention(q, k, v, ks, vs, None, None, [S])
    check(kvq.decode_attn_window(q.to(DEV), *parts, None, 10 ** 6), out, tol)


@pytest.mark.parametrize("fmt", ("int8", "int4", "fp16"))
def test_window_as_long_as_the_context_is_full_attention(fmt):
    lens = [700, 350]
    gen, q, k, v, ks, vs, kz, vz = _case(2, 28, 4, 128, 704, fmt, 64, 11)
    parts = _d(k, v, ks, vs)
    lend = torch.tensor(lens, dtype=torch.int32, device=DEV)
    a = kvq.decode_attn_window(q.to(DEV), *parts, lend, 704, 9)
    full = {"int8": kvq.decode_attn_int8, "int4": kvq.decode_attn_int4}.get(fmt)
    b = kvq.decode_attn_fp16(q.to(DEV), parts[0], parts[1], lend) if full is None else full(q.to(DEV), *parts, lend)
    # the package's other kernels promise 2e-3 + 1e-2 |x|
    assert ((a - b).abs() <= 2e-3 + 1e-2 * b.abs()).all()


@pytest.mark.parametrize("fmt", ("fp16", "int8", "int4z"))
def test_extreme_values(fmt):
    """Logits far apart, the largest and smallest scales: the joined runs must neither overflow nor lose the small ones."""
    B, Hq, Hkv, D, S = 2, 8, 1, 128, 2100
    gen, q, k, v, ks, vs, kz, vz = _case(B, Hq, Hkv, D, S, fmt, 128 if fmt == "int8" else 32, 5)
    q = (q * 8).half()
    if fmt == "fp16":
        v[:, :, ::2] *= 2000
        v[:, :, 1::2] *= 2.0 ** -12
    else:
        vs[:, :, 0:700] *= 2000
        vs[:, :, 700:1400] *= 2.0 ** -9
        ks[:, :, 5] *= 40
    out, tol, _, _ = attention(q, k, v, ks, vs, kz, vz, [S, 1401])
    parts = _d(k, v, ks, vs)
    kzd, vzd = _d(kz, vz)
    got = kvq.decode_attn_window(q.to(DEV), *parts, torch.tensor([S, 1401], dtype=torch.int32, device=DEV), S, k_zp=kzd, v_zp=vzd)
    check(got, out, tol, fmt)


def test_minus_infinity_keys_and_nan():
    """A visible key of -inf has weight zero; rows with nothing else give zeros; NaN in a visible key stays visible."""
    q = torch.ones(3, 2, 128).half()
    k = torch.zeros(3, 1, 40, 128).half()
    v = torch.randn(3, 1, 40, 128, generator=torch.Generator().manual_seed(0)).half()
    k[0, 0, 0:33] = float("-inf")
    k[1] = float("-inf")
    k[2, 0, 7] = float("nan")
    got = kvq.decode_attn_window(*_d(q, k, v), None, None, None, 40).cpu()
    want = v[0, 0, 33:].double().mean(0)
    assert ((got[0].double() - want).abs() <= 2.0 ** -10).all()
    assert (got[1] == 0).all()
    assert torch.isnan(got[2]).all()


# ------------------------------------------------------------------------------------------------ weights
WEIGHTS = [(1, 12, 2, 128, 1, [1], 32), (2, 28, 4, 128, 300, [300, 77], 128), (3, 14, 2, 64, 1030, [1029, 0, 64], 32),
           (2, 20, 1, 128, 2050, [2050, 1111], 128), (1, 40, 8, 128, 5000, [4999], 64), (2, 4, 4, 256, 600, [600, 599], 256)]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("case", range(len(WEIGHTS)))
def test_weights(case, fmt):
    B, Hq, Hkv, D, S, lens, gs = WEIGHTS[case]
    gen, q, k, v, ks, vs, kz, vz = _case(B, Hq, Hkv, D, S, fmt, gs, 40 + case)
    out, tol, w, wtol = attention(q, k, v, ks, vs, kz, vz, lens)
    parts = _d(*[_poison(t, lens) for t in (k, v, ks, vs)])
    kzd, vzd = _d(_poison(kz, lens), _poison(vz, lens))
    lend = torch.tensor(lens, dtype=torch.int32, device=DEV)
    start = torch.rand(B, Hkv, S + 5, generator=gen)
    buf = start.to(DEV)
    got = kvq.decode_attn_weights(q.to(DEV), *parts, lend, buf, k_zp=kzd, v_zp=vzd)
    check(got, out, tol, fmt)
    first = buf.clone()
    ref = start.double()
    ref[:, :, :S] += w
    check(buf[:, :, :S], ref[:, :, :S], wtol + ref[:, :, :S].abs() * 2.0 ** -24, fmt)
    for b, n in enumerate(lens):
        assert torch.equal(buf[b, :, n:].cpu(), start[b, :, n:]), "a sum behind the context was touched"
    kvq.decode_attn_weights(q.to(DEV), *parts, lend, buf, k_zp=kzd, v_zp=vzd)
    ref[:, :, :S] += w
    check(buf[:, :, :S], ref[:, :, :S], 2 * wtol + ref[:, :, :S].abs() * 2.0 ** -23, fmt)
    buf2 = start.to(DEV)
    kvq.decode_attn_weights(q.to(DEV), *parts, lend, buf2, k_zp=kzd, v_zp=vzd)
    assert torch.equal(buf2, first), "results change from call to call"


# ------------------------------------------------------------------------------------------------ append and read
def _contiguous_append(fmt, k, v, gs, pct):
    """The contiguous caches' codes of the same tokens: what the pages must hold, bit for bit."""
    cls = {"fp16": lambda: kvq.FP16KVCache(1, device=DEV),
           "int8": lambda: kvq.INT8KVCache(1, device=DEV, group_size=gs, clip_percentile=pct),
           "int4": lambda: kvq.INT4KVCache(1, device=DEV, group_size=gs, clip_percentile=pct),
           "int4z": lambda: kvq.INT4KVCache(1, device=DEV, group_size=gs, asymmetric=True)}[fmt]
    c = cls()
    c.append(0, k, v)
    return {n: t[:, :, :k.shape[2]] for n, t in c._bufs[0].items()}


@pytest.mark.parametrize("fmt", ("fp16", "int8", "int4", "int4z"))
@pytest.mark.parametrize("B,H,T,D,gs,page,pct", ((3, 2, 1, 128, 32, 16, 100.0), (5, 4, 37, 128, 128, 32, 99.9),
                                                (2, 2, 2500, 128, 32, 64, 100.0), (4, 3, 1100, 64, 64, 48, 99.9),
                                                (2, 2, 40, 128, 16, 16, 90.0), (1, 1, 9, 256, 64, 7, 100.0)))
def test_paged_append_and_read(fmt, B, H, T, D, gs, page, pct):
    gen = torch.Generator().manual_seed(B * 1000 + T)
    k, v = (torch.randn(B, H, T, D, generator=gen).half() for _ in range(2))
    start = torch.tensor([(11 * b) % 50 for b in range(B)], dtype=torch.int32)
    new = torch.tensor([T if b % 3 == 0 else max(0, T - 1 - 5 * b) for b in range(B)], dtype=torch.int32)
    pool, table = make_table((start + new).tolist(), page, gen)
    want = _contiguous_append(fmt, k.to(DEV), v.to(DEV), gs, pct)
    pools = {n: torch.full((pool, H, page, t.shape[3]), 3, dtype=t.dtype, device=DEV) for n, t in want.items()}
    before = {n: t.clone() for n, t in pools.items()}
    td, sd, nd = _d(table, start, new)
    kvq.paged_append(k.to(DEV), v.to(DEV), pools["k"], pools["v"], pools.get("ks"), pools.get("vs"), td, sd, nd,
                     k_zp=pools.get("kz"), v_zp=pools.get("vz"), clip_percentile=pct)
    touched = torch.zeros(pool, page, dtype=torch.bool)
    for b in range(B):
        for t in range(int(new[b])):
            pos = int(start[b]) + t
            touched[int(table[b, pos // page]), pos % page] = True
    for b in range(B):
        pos = torch.arange(int(new[b])) + int(start[b])
        pg, rw = table[b].long()[pos // page].to(DEV), (pos % page).to(DEV)
        for n, t in pools.items():
            assert torch.equal(t[pg, :, rw].transpose(0, 1), want[n][b, :, :int(new[b])]), (n, b)
    for n, t in pools.items():
        keep = (~touched).to(DEV)
        assert torch.equal(t.transpose(1, 2)[keep], before[n].transpose(1, 2)[keep]), f"{n}: rows of other tokens changed"
    kr, vr = kvq.paged_read(pools["k"], pools["v"], pools.get("ks"), pools.get("vs"), td, sd, T + 2, nd, head_dim=D,
                            k_zp=pools.get("kz"), v_zp=pools.get("vz"))
    for got, s in ((kr, "k"), (vr, "v")):
        for b in range(B):
            n = int(new[b])
            if n:
                x, _, _ = values(want[s][b, :, :n].cpu(), want[s + "s"][b, :, :n].cpu() if fmt != "fp16" else None,
                                 want[s + "z"][b, :, :n].cpu() if fmt == "int4z" else None, D)
                # code * scale is exact and code * scale + zp one fp32 rounding (2^-24) before the rounding to fp16
                exact = x.half() if fmt != "int4z" else None
                if exact is not None:
                    assert torch.equal(got[b, :, :n].cpu(), exact)
                else:
                    err = (got[b, :, :n].cpu().double() - x).abs()
                    assert (err <= x.abs() * (2.0 ** -11 + 2.0 ** -23) + 2.0 ** -25).all()
            assert (got[b, :, n:] == 0).all()
    assert _flag() == 0


@pytest.mark.parametrize("T", (1, 600))
def test_paged_append_static_scales_strided_sources_and_bad_pages(T):
    B, H, D, page = 8, 2, 128, 32
    gen = torch.Generator().manual_seed(3)
    src = torch.randn(B, T, H, 2, D, generator=gen).half().to(DEV)
    k, v = src[:, :, :, 0].transpose(1, 2), src[:, :, :, 1].transpose(1, 2)     # views of a fused projection's output
    tab = torch.rand(H, 4, generator=gen).mul(0.02).add(0.01).half().to(DEV)
    c = kvq.INT8KVCache(1, device=DEV, group_size=32, static_k_scale=tab[None], static_v_scale=tab[None])
    c.append(0, k, v)
    lens = [T] * B
    pool, table = make_table(lens, page, gen)
    pk, pv = (torch.zeros(pool, H, page, D, dtype=torch.int8, device=DEV) for _ in range(2))
    sk, sv = (torch.zeros(pool, H, page, 4, dtype=torch.float16, device=DEV) for _ in range(2))
    zero = torch.zeros(B, dtype=torch.int32, device=DEV)
    kvq.paged_append(k, v, pk, pv, sk, sv, table.to(DEV), zero, k_static=tab, v_static=tab)
    want_k, want_v = c.get_kv(0)
    got_k, got_v = kvq.paged_read(pk, pv, sk, sv, table.to(DEV), None, T, head_dim=D)
    assert torch.equal(got_k, want_k) and torch.equal(got_v, want_v)
    assert _flag() == 0
    # a bad page, a position behind the table, a negative position: nothing is stored, the flag says so
    for what in ("page", "behind", "negative"):
        t2, s2 = table.clone(), torch.zeros(B, dtype=torch.int32)
        if what == "page":
            t2[0, 0] = pool
        else:
            s2[0] = t2.shape[1] * page if what == "behind" else -T
        a, b_ = pk.clone(), sk.clone()
        a.zero_(), b_.zero_()
        kvq.paged_append(k, v, a, pv.clone(), b_, sv.clone(), t2.to(DEV), s2.to(DEV), k_static=tab, v_static=tab)
        assert _flag() == 8
        own = t2[0][(t2[0] >= 0) & (t2[0] < pool)].long()
        if T == 1 or what != "page":
            assert (a[own.to(DEV)] == 0).all()
        rest = table[1][table[1] >= 0].long().to(DEV)
        assert torch.equal(a[rest], pk[rest]) and torch.equal(b_[rest], sk[rest])


@pytest.mark.parametrize("fmt", FORMATS[1:])
@pytest.mark.parametrize("D,gs", ((128, 128), (128, 64), (128, 32), (64, 64), (64, 32)))
@pytest.mark.parametrize("S,off", ((1301, 0), (1302, 0), (1304, 0), (1300, 1), (1296, 2), (333, 4)))
def test_scale_rows_of_every_alignment(S, off, D, gs, fmt):
    """Contiguous caches whose scale rows start on 2 to 16 bytes, by the number of slots or as views that skip some: the
    same kernel as for aligned ones, bit for bit (the products and their order do not depend on how scales arrive)."""
    gen, q, k, v, ks, vs, kz, vz = _case(2, 12, 2, D, S, fmt, gs, S + off)
    lens = [S - off, 40]

    def run(pad):
        def scales(t):
            if t is None:
                return None
            wide = torch.full((2, 2, S + pad, t.shape[3]), float("nan")).half().to(DEV)
            wide[:, :, :S] = t.to(DEV)
            return wide[:, :, off:S]
        kk, vv = k[:, :, off:].contiguous().to(DEV), v[:, :, off:].contiguous().to(DEV)
        return kvq.decode_attn_window(q.to(DEV), kk, vv, scales(ks), scales(vs), torch.tensor(lens, device=DEV, dtype=torch.int32),
                                      S, k_zp=scales(kz), v_zp=scales(vz))
    got = run(0)
    cut = [None if t is None else t[:, :, off:] for t in (k, v, ks, vs, kz, vz)]
    ref, tol, _, _ = attention(q, *cut, lens, S, 0)
    check(got, ref, tol, f"{fmt} S={S} off={off}")
    assert torch.equal(run(0), got)
    if off == 0:
        assert torch.equal(run(-S % 8), got)                # rows on 16 bytes


# ------------------------------------------------------------------------------------------------ eviction
EVICT = [
    # B, H, cap, lengths, budget, sinks, recent, seen offset
    (1, 1, 2, [2], 1, 0, 0, 0),
    (2, 2, 40, [33, 40], 32, 4, 8, 0),
    (3, 2, 700, [700, 5, 650], 640, 0, 0, 100),
    (2, 3, 2300, [2049, 2048], 2048, 4, 256, 5000),
    (1, 2, 9000, [8999], 1024, 4, 1020, 0),
    (2, 1, 5000, [5000, 4097], 100, 100, 0, 0),
    (1, 2, 40000, [40000], 39990, 4, 32, 7),
    (1, 1, 100, [-3], 50, 0, 0, 0),
    (2, 2, 64, [64, 64], 64, 4, 4, 0),
]


def _evict_inputs(case, kind, gen):
    B, H, cap, lengths, budget, sinks, recent, off = EVICT[case]
    if kind == "random":
        w = torch.exp(2 * torch.randn(B, H, cap, generator=gen))
    elif kind == "ties":
        w = torch.randint(0, 3, (B, H, cap), generator=gen).float()
    elif kind == "equal":
        w = torch.zeros(B, H, cap)
        w[:, :, ::2] = -0.0
    else:
        w = torch.randn(B, H, cap, generator=gen)
        pick = torch.rand(B, H, cap, generator=gen)
        w[pick < 0.1] = float("nan")
        w[(pick > 0.1) & (pick < 0.2)] = float("inf")
        w[(pick > 0.2) & (pick < 0.3)] = float("-inf")
        w[(pick > 0.3) & (pick < 0.4)] = 1e-42
    lens = torch.tensor(lengths, dtype=torch.int32)
    seen = lens.clamp(0, cap) + off
    pos = torch.full((B, H, cap), -1, dtype=torch.int32)
    if off:                                                # the first slots hold survivors of earlier evictions
        for b in range(B):
            n = int(lens[b])
            old = max(n - 3, 0)
            for h in range(H):
                pos[b, h, :old] = torch.randperm(int(seen[b]) - (n - old), generator=gen)[:old].to(torch.int32)
    return w, pos, lens, seen


@pytest.mark.parametrize("kind", ("random", "ties", "equal", "special"))
@pytest.mark.parametrize("case", range(len(EVICT)))
def test_evict(case, kind):
    B, H, cap, lengths, budget, sinks, recent, off = EVICT[case]
    gen = torch.Generator().manual_seed(case)
    w, pos, lens, seen = _evict_inputs(case, kind, gen)
    bufs = [torch.randint(-128, 128, (B, H, cap, 64), generator=gen, dtype=torch.int16).to(torch.int8),
            torch.randn(B, H, cap + 3, 128, generator=gen).half(), torch.randn(B, H, cap, 3, generator=gen).half(),
            torch.randint(0, 2 ** 31, (B, H, cap), generator=gen), torch.randint(0, 100, (B, H, cap, 5), generator=gen).to(torch.int8)]
    rw, rp, rn, moves = evict(w, pos, lens, seen, budget, sinks, recent)
    want = [t.clone() for t in bufs]
    for (b, h), (dst, src) in moves.items():
        for t, u in zip(want, bufs):
            t[b, h, dst] = u[b, h, src]
    wd, pd, ld, sd = _d(w, pos, lens, seen)
    bd = _d(*bufs)
    got = kvq.evict_tokens(wd, pd, ld, sd, budget, bd, sinks=sinks, recent=recent)
    assert torch.equal(got.cpu(), rn)
    assert torch.equal(pd.cpu(), rp)
    assert torch.equal(wd.cpu().view(torch.int32), rw.view(torch.int32))        # moved bit for bit (NaN, -0)
    for i, (t, u) in enumerate(zip(bd, want)):
        assert torch.equal(t.cpu(), u), i
    assert torch.equal(ld.cpu(), lens) and torch.equal(sd.cpu(), seen)


@pytest.mark.parametrize("kind", ("random", "ties", "equal", "special"))
@pytest.mark.parametrize("cap,n,budget", ((4096, 4096, 2000), (4097, 4097, 4000), (32768, 32768, 300), (32769, 32769, 30000),
                                          (70000, 69999, 20000)))
def test_evict_long_rows(cap, n, budget, kind):
    """Runs of one slot more or less than a CTA's, runs that are read again by every pass, large and small shares."""
    gen = torch.Generator().manual_seed(cap)
    EVICT.append((1, 1, cap, [n], budget, 4, 64, 0))
    try:
        w, pos, lens, seen = _evict_inputs(len(EVICT) - 1, kind, gen)
    finally:
        EVICT.pop()
    k = torch.arange(cap, dtype=torch.int32).view(1, 1, cap, 1)
    rw, rp, rn, moves = evict(w, pos, lens, seen, budget, 4, 64)
    wd, pd, ld, sd, kd = _d(w, pos, lens, seen, k)
    got = kvq.evict_tokens(wd, pd, ld, sd, budget, [kd], sinks=4, recent=64)
    dst, src = moves[0, 0]
    k[0, 0, dst, 0] = torch.tensor(src, dtype=torch.int32)
    assert torch.equal(got.cpu(), rn) and torch.equal(pd.cpu(), rp) and torch.equal(kd.cpu(), k)
    assert torch.equal(wd.cpu().view(torch.int32), rw.view(torch.int32))


@pytest.mark.parametrize("cap", (300, 20000, 40000))
def test_evict_more_protected_tokens_than_the_budget(cap):
    """Positions that do not differ: more protected tokens than fit; the lowest slots among them are kept."""
    gen = torch.Generator().manual_seed(2)
    w = torch.rand(1, 1, cap, generator=gen)
    pos = torch.randint(0, 8, (1, 1, cap), generator=gen, dtype=torch.int32)
    lens = torch.tensor([cap], dtype=torch.int32)
    rw, rp, rn, moves = evict(w, pos, lens, lens, 100, 4, 0)
    wd, pd, ld = _d(w, pos, lens)
    got = kvq.evict_tokens(wd, pd, ld, ld.clone(), 100, [], sinks=4)
    assert torch.equal(got.cpu(), rn) and torch.equal(pd.cpu(), rp) and torch.equal(wd.cpu(), rw)


def test_evict_strided_rows_and_views():
    """Weights, positions and buffers as views of larger tensors; slots and heads outside the views keep their bytes."""
    gen = torch.Generator().manual_seed(9)
    B, H, cap, n, budget = 2, 3, 300, 290, 100
    w = torch.rand(B, H + 2, cap + 16, generator=gen)
    p = torch.full((B, H + 2, cap + 16), -1, dtype=torch.int32)
    k = torch.randn(cap + 20, H + 2, B, 32, generator=gen).half()               # slots outermost
    wd, pd, kd = _d(w, p, k)
    lens = torch.full((B,), n, dtype=torch.int32)
    rw, rp, rn, moves = evict(w[:, 1:1 + H, :n], p[:, 1:1 + H, :n], lens, lens, budget, 2, 10)
    kv = kd.permute(2, 1, 0, 3)[:, 1:1 + H, :n]
    kvq.evict_tokens(wd[:, 1:1 + H, :n], pd[:, 1:1 + H, :n], lens.to(DEV), lens.to(DEV), budget, [kv], sinks=2, recent=10)
    want_w, want_k = w.clone(), k.clone()
    want_w[:, 1:1 + H, :n] = rw
    view = want_k.permute(2, 1, 0, 3)[:, 1:1 + H]
    old = k.permute(2, 1, 0, 3)[:, 1:1 + H].clone()
    for (b, h), (dst, src) in moves.items():
        view[b, h, dst] = old[b, h, src]
    assert torch.equal(wd.cpu(), want_w) and torch.equal(kd.cpu(), want_k)


# ------------------------------------------------------------------------------------------------ streams, graphs, devices
def test_other_stream_and_captured_graphs_do_not_share_scratch():
    lens = [1500, 900]
    gen, q, k, v, ks, vs, kz, vz = _case(2, 28, 4, 128, 1500, "int8", 128, 21)
    parts = _d(k, v, ks, vs)
    lend = torch.tensor(lens, dtype=torch.int32, device=DEV)
    qs = [torch.randn(2, 28, 128, generator=gen).half().to(DEV) for _ in range(2)]
    ws = [torch.zeros(2, 4, 1500, device=DEV) for _ in range(2)]
    want = [kvq.decode_attn_weights(x, *parts, lend, torch.zeros(2, 4, 1500, device=DEV)) for x in qs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(kvq.decode_attn_weights(qs[0], *parts, lend, torch.zeros(2, 4, 1500, device=DEV)), want[0])
    torch.cuda.synchronize()
    graphs, outs = [], [torch.empty(2, 28, 128, dtype=torch.float16, device=DEV) for _ in range(2)]
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            kvq.decode_attn_weights(qs[i], *parts, lend, ws[i], out=outs[i])
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for i in range(2):
        assert torch.equal(outs[i], want[i])
        assert abs(float(ws[i].double().sum()) / (20 * 2 * 28) - 1) < 1e-4       # every head's weights sum to 1


def test_evict_and_append_in_a_graph():
    gen = torch.Generator().manual_seed(2)
    B, H, cap, budget = 2, 2, 600, 512
    w0 = torch.rand(B, H, cap, generator=gen).to(DEV)
    k0 = torch.randn(B, H, cap, 128, generator=gen).half().to(DEV)
    lens = torch.tensor([600, 513], dtype=torch.int32, device=DEV)
    w, p, k = w0.clone(), torch.full((B, H, cap), -1, dtype=torch.int32, device=DEV), k0.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        new = kvq.evict_tokens(w, p, lens, lens, budget, [k], sinks=4, recent=16)
    for _ in range(2):
        w.copy_(w0), k.copy_(k0), p.fill_(-1)
        g.replay()
        rw, rp, rn, _ = evict(w0.cpu(), torch.full((B, H, cap), -1, dtype=torch.int32), lens.cpu(), lens.cpu(), budget, 4, 16)
        assert torch.equal(w.cpu(), rw) and torch.equal(p.cpu(), rp) and torch.equal(new.cpu(), rn)


# ------------------------------------------------------------------------------------------------ the caches
@pytest.mark.parametrize("fmt", ("fp16", "int8", "int4", "int4_asym"))
@pytest.mark.parametrize("window", (None, 50))
def test_paged_cache_serves_sequences_that_come_and_go(fmt, window):
    """Prompts of different lengths, joint decode steps, one sequence leaves, another takes its pages: every step's attention
    against a 64-bit reference over the tokens of each sequence as the contiguous cache would hold them."""
    L, H, Hq, D, page, gs = 2, 2, 12, 128, 16, 32
    gen = torch.Generator().manual_seed(31)
    c = kvq.PagedKVCache(L, 16, H, D, page_size=page, kv_format=fmt, group_size=gs, clip_percentile=100.0, window=window,
                         sinks=3 if window else 0, device=DEV)
    hist = {}                                              # (seq, layer) -> [k, v]

    def step(T, counts):
        rows = c.sequences
        for l in range(L):
            k, v = (torch.randn(len(rows), H, T, D, generator=gen).half() for _ in range(2))
            c.append(l, k.to(DEV), v.to(DEV), new_lens=None if all(x == T for x in counts) else counts)
            for i, s in enumerate(rows):
                for j, x in enumerate((k, v)):
                    hist.setdefault((s, l), [[], []])[j].append(x[i, :, :counts[i]])
            q = torch.randn(len(rows), Hq, D, generator=gen).half()
            got = c.fused_decode(l, q.to(DEV), 1 / math.sqrt(D))
            kr, vr = c.get_kv(l)
            for i, s in enumerate(rows):
                kk, vv = (torch.cat(x, 1)[None] for x in hist[s, l])
                n = kk.shape[2]
                assert c.get_seq_lens()[i] == n
                if n == 0:
                    assert (got[i] == 0).all()
                    continue
                enc = _contiguous_append(fmt.replace("_asym", "z"), kk.to(DEV), vv.to(DEV), gs, 100.0)
                enc = {m: t.cpu() for m, t in enc.items()}
                ref, tol, _, _ = attention(q[i:i + 1], enc["k"], enc["v"], enc.get("ks"), enc.get("vs"), enc.get("kz"),
                                           enc.get("vz"), [n], window or 0, 3 if window else 0)
                check(got[i:i + 1], ref, tol, f"{fmt} seq {s} layer {l}")
                x, _, _ = values(enc["k"], enc.get("ks"), enc.get("kz"), D)
                err = (kr[i:i + 1, :, :n].cpu().double() - x).abs()
                assert (err <= x.abs() * (2.0 ** -11 + 2.0 ** -23) + 2.0 ** -25).all() and (kr[i, :, n:] == 0).all()

    a, b = c.add_sequence(), c.add_sequence()
    step(70, [70, 33])
    for _ in range(3):
        step(1, [1, 1])
    c.free_sequence(a)
    d = c.add_sequence()
    assert c.sequences == (b, d)
    step(40, [0, 40])                                      # the old row sits out while the new one is filled
    step(1, [1, 1])
    assert c.num_free_pages == 16 - sum(-(-n // page) for n in c.get_seq_lens())
    for tokens, match in ((300, "max_pages_per_seq"), (120, "exhausted")):
        with pytest.raises(ValueError, match=match):
            c.append(0, *(torch.zeros(2, H, tokens, D).half().to(DEV) for _ in range(2)))
    step(1, [1, 1])                                        # the refused step changed nothing
    c.clear()
    assert c.num_free_pages == 16 and c.get_seq_len() == 0
    assert _flag() == 0


@pytest.mark.parametrize("kind", ("fp16", "int8", "int4", "int4z"))
def test_contiguous_cache_with_a_window(kind):
    gen = torch.Generator().manual_seed(5)
    B, H, Hq, D, T = 2, 2, 12, 128, 150
    make = {"fp16": lambda: kvq.FP16KVCache(1, device=DEV), "int8": lambda: kvq.INT8KVCache(1, device=DEV, group_size=32),
            "int4": lambda: kvq.INT4KVCache(1, device=DEV), "int4z": lambda: kvq.INT4KVCache(1, device=DEV, asymmetric=True)}
    c = make[kind]()
    c.set_attention_window(20, 2)
    k, v = (torch.randn(B, H, T, D, generator=gen).half().to(DEV) for _ in range(2))
    c.append(0, k, v)
    q = torch.randn(B, Hq, D, generator=gen).half()
    n = {name: t[:, :, :T].cpu() for name, t in c._bufs[0].items()}
    for args in ((20, 2), (7, 0), None):
        c.set_attention_window(*(args or (None,)))
        got = c.fused_decode(0, q.to(DEV), 1 / math.sqrt(D))
        out, tol, _, _ = attention(q, n["k"], n["v"], n.get("ks"), n.get("vs"), n.get("kz"), n.get("vz"), [T] * B,
                                   *(args or (0, 0)))
        if args:
            check(got, out, tol)
        else:
            assert ((got.cpu().double() - out).abs() <= 2e-3 + 1e-2 * out.abs()).all()
    # a graph with device-side lengths sees the window as well
    c.set_attention_window(20, 2)
    ctx = torch.tensor([100, 100], dtype=torch.int32, device=DEV)
    c.use_device_positions(torch.tensor([99], dtype=torch.int32, device=DEV), ctx, T)
    got = c.fused_decode(0, q.to(DEV), 1 / math.sqrt(D))
    c.use_host_positions()
    out, tol, _, _ = attention(q, n["k"], n["v"], n.get("ks"), n.get("vs"), n.get("kz"), n.get("vz"), [100] * B, 20, 2)
    check(got, out, tol)


@pytest.mark.parametrize("kind", ("fp16", "int8", "int4z"))
def test_contiguous_cache_with_eviction(kind):
    """Prompt, then decode steps under a budget: the whole run against a plain replay (64-bit attention over the slots, the
    plain eviction on the kernel's own sums) and the invariants of a bounded cache."""
    gen = torch.Generator().manual_seed(6)
    B, H, Hq, D, T, budget, sinks, recent = 2, 2, 12, 128, 100, 40, 4, 8
    make = {"fp16": lambda: kvq.FP16KVCache(1, device=DEV), "int8": lambda: kvq.INT8KVCache(1, device=DEV, group_size=128),
            "int4z": lambda: kvq.INT4KVCache(1, device=DEV, asymmetric=True)}
    c = make[kind]()
    c.append(0, *(torch.randn(B, H, T, D, generator=gen).half().to(DEV) for _ in range(2)))
    c.enable_eviction(budget, sinks, recent)
    w = torch.zeros(B, H, 0)
    pos = torch.zeros(B, H, 0, dtype=torch.int32)
    seen = T
    for step in range(30):
        new = 3 if step == 11 else 1                       # a chunk of several tokens in between
        c.append(0, *(torch.randn(B, H, new, D, generator=gen).half().to(DEV) for _ in range(2)))
        seen += new
        n = c.get_seq_len()
        snap = {m: t.clone()[:, :, :n] for m, t in c._bufs[0].items()}         # same strides: the same kernel serves them
        bufs = {m: t.cpu() for m, t in snap.items()}
        q = torch.randn(B, Hq, D, generator=gen).half()
        before = torch.zeros(B, H, n, dtype=torch.float64)
        before[:, :, :w.shape[2]] = w.double()
        pos = torch.cat((pos, torch.full((B, H, n - pos.shape[2]), -1, dtype=torch.int32)), 2)
        got = c.fused_decode(0, q.to(DEV), 1 / math.sqrt(D))
        out, tol, dw, dwtol = attention(q, bufs["k"], bufs["v"], bufs.get("ks"), bufs.get("vs"), bufs.get("kz"),
                                        bufs.get("vz"), [n] * B)
        check(got, out, tol, f"step {step}")
        # the sums that the eviction saw differ from the 64-bit ones by rounding: rank by a second, identical pass
        again = before.float().to(DEV)
        ops.span_attn(q.to(DEV), snap["k"], snap["v"], snap.get("ks"), snap.get("vs"), None, 1 / math.sqrt(D),
                      weights=again, k_zp=snap.get("kz"), v_zp=snap.get("vz"))
        check(again, before + dw, dwtol + (before + dw) * 2.0 ** -23)
        i32 = torch.full((B,), n, dtype=torch.int32)
        w, pos, lens, moves = evict(again.cpu(), pos, i32, torch.full((B,), seen, dtype=torch.int32), budget, sinks, recent)
        w, pos = w[:, :, :budget], pos[:, :, :budget]
        assert c.get_seq_len() == budget == int(lens[0]) and c.get_tokens_seen() == seen
        assert torch.equal(c._evict_state[0]["w"][:, :, :budget].cpu(), w)
        assert torch.equal(c._evict_state[0]["p"][:, :, :budget].cpu(), pos)
        assert (c._evict_state[0]["w"][:, :, budget:] == 0).all()
        for m, t in c._bufs[0].items():
            x = bufs[m].clone()
            for (b, h), (dst, src) in moves.items():
                x[b, h, dst] = bufs[m][b, h, src]
            assert torch.equal(t[:, :, :budget].cpu(), x[:, :, :budget]), m
        for b in range(B):
            for h in range(H):
                have = set(pos[b, h].tolist())
                assert set(range(sinks)) <= have and set(range(seen - recent, seen)) <= have and len(have) == budget
    c.clear()
    assert c.get_tokens_seen() == 0


@pytest.mark.parametrize("fmt", ("fp16", "int8", "int4z"))
@pytest.mark.parametrize("S", (256, 257, 1024, 1025, 2048, 2049))
def test_many_rows_around_the_lengths_that_are_cut(S, fmt):
    """1024 rows (more than the chip takes at once) and 256 of them; ragged, with empty ones; with weights too."""
    B, Hq, Hkv, D = 128, 16, 8, 64
    gen, q, k, v, ks, vs, kz, vz = _case(2, Hq, Hkv, D, S, fmt, 64, S)
    lens = [S if b % 5 == 0 else (b * 97) % S for b in range(B)]
    rep = [None if t is None else t.to(DEV).repeat_interleave(B // 2, 0) for t in (q, k, v, ks, vs, kz, vz)]
    lend = torch.tensor(lens, dtype=torch.int32, device=DEV)
    got = kvq.decode_attn_window(rep[0], *rep[1:5], lend, S, k_zp=rep[5], v_zp=rep[6])
    few = kvq.decode_attn_window(rep[0][:32].contiguous(), *[None if t is None else t[:32].contiguous() for t in rep[1:5]],
                                 lend[:32].contiguous(), S, k_zp=None if kz is None else rep[5][:32].contiguous(),
                                 v_zp=None if vz is None else rep[6][:32].contiguous())
    w = torch.zeros(B, Hkv, S, device=DEV)
    kvq.decode_attn_weights(rep[0], *rep[1:5], lend, w, k_zp=rep[5], v_zp=rep[6])
    for b in (0, 1, 2, 5, 31, 64, 100, 127):
        i = b // (B // 2)
        one = [None if t is None else t[i:i + 1] for t in (q, k, v, ks, vs, kz, vz)]
        ref, tol, rw, wtol = attention(*one, [lens[b]])
        check(got[b:b + 1], ref, tol, f"{fmt} row {b}")
        if b < 32:
            check(few[b:b + 1], ref, tol, f"{fmt} row {b} of few")
        assert ((w[b:b + 1].double().cpu() - rw).abs() <= wtol + 2.0 ** -22).all()


def test_a_step_with_eviction_is_not_captured():
    """Its lengths are the host's; the call is refused before anything is launched or kept, and works afterwards."""
    c = kvq.INT8KVCache(1, device=DEV, group_size=32)
    c.enable_eviction(40, 2, 8)
    gen = torch.Generator().manual_seed(4)
    k = torch.randn(1, 2, 50, 128, generator=gen).half().to(DEV)
    q = torch.randn(1, 4, 128, generator=gen).half().to(DEV)
    c.append(0, k, k)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = q + 1                                          # a graph that is not empty
        with pytest.raises(ValueError, match="captured"):
            c.fused_decode(0, q, 0.09)
    assert c.get_seq_len() == 50
    g.replay()
    out = c.fused_decode(0, q, 0.09)
    assert c.get_seq_len() == 40 and torch.isfinite(out).all() and torch.equal(y, q + 1)


def test_a_step_of_a_paged_cache_is_not_captured():
    c = kvq.PagedKVCache(1, 8, 2, 128, page_size=16, device=DEV, group_size=32)
    c.add_sequence()
    k = torch.randn(1, 2, 20, 128, device=DEV).half()
    q = torch.randn(1, 4, 128, device=DEV).half()
    c.append(0, k, k)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = q + 1
        for call in (lambda: c.append(0, k, k), lambda: c.fused_decode(0, q), lambda: c.get_kv(0)):
            with pytest.raises(ValueError, match="captured"):
                call()
    assert c.get_seq_lens() == (20,) and c.num_free_pages == 6
    assert torch.isfinite(c.fused_decode(0, q)).all()
