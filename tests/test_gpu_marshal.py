"""The two host forms of a bounded- or paged-cache call - _marshal.so and the Python one - give the same bits, and what the
Python form refuses or converts is not taken by the other."""
import pytest
import torch

from llm_kvcache_quantization_b200 import ops
from span_reference import make_cache, make_table, paginate
import test_span_cpu

pytestmark = pytest.mark.gpu
DEV = "cuda"


class _None:
    """A marshalling module that takes no call."""
    def __getattr__(self, name):
        return lambda *a: None


class _Seen:
    """The real one, noting which calls it took."""
    def __init__(self):
        self.real, self.took = ops._lib.marshal(), []

    def __getattr__(self, name):
        def call(*a):
            r = getattr(self.real, name)(*a)
            self.took.append(r is not None)
            return r
        return call


def _both(monkeypatch, call):
    """Results of the two forms; the first must have been taken by _marshal.so."""
    seen = _Seen()
    monkeypatch.setattr(ops, "_MARSHAL", seen)
    a = call()
    assert seen.took == [True]
    monkeypatch.setattr(ops, "_MARSHAL", _None())
    b = call()
    for x, y in zip(a, b):
        assert torch.equal(x, y) and x.stride() == y.stride() and x.dtype == y.dtype
    return a


def _paged(fmt, seed=3):
    gen = torch.Generator().manual_seed(seed)
    lens, page, D = [70, 0, 33], 16, 128
    k, ks, kz = make_cache((3, 2, 70), D, fmt, 32, gen)
    v, vs, vz = make_cache((3, 2, 70), D, fmt, 32, gen)
    pool, table = make_table(lens, page, gen)
    t = [None if x is None else paginate(x, lens, page, pool, table).to(DEV) for x in (k, v, ks, vs, kz, vz)]
    q = torch.randn(3, 12, D, generator=gen).half().to(DEV)
    return q, t, table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV), gen


@pytest.mark.parametrize("fmt", ("fp16", "int8", "int8z", "int4", "int4z"))
def test_both_forms_agree(monkeypatch, fmt):
    q, (k, v, ks, vs, kz, vz), table, lens, gen = _paged(fmt)
    tau = torch.full((12,), 0.9, device=DEV)
    for kw in (dict(), dict(window=20, sinks=3), dict(max_ctx=50), dict(inv_tau=tau, sm_scale=0.11)):
        _both(monkeypatch, lambda: (ops.span_attn(q, k, v, ks, vs, lens, block_table=table, k_zp=kz, v_zp=vz, **{
            "sm_scale": None, **kw}),))
    _both(monkeypatch, lambda: ops.paged_read(k, v, ks, vs, table, None, 40, lens, head_dim=128, k_zp=kz, v_zp=vz))
    new = [torch.randn(3, 2, 5, 128, generator=gen).half().to(DEV) for _ in range(2)]
    n = torch.tensor([5, 0, 2], dtype=torch.int32, device=DEV)
    start = torch.tensor([60, 0, 33], dtype=torch.int32, device=DEV)

    def append(**kw):
        pools = [None if t is None else t.clone() for t in (k, v, ks, vs, kz, vz)]
        ops.paged_append(*new, *pools[:4], table, start, n, k_zp=pools[4], v_zp=pools[5], **kw)
        return [t.view(torch.int16) if t.dtype == torch.float16 else t for t in pools if t is not None]
    _both(monkeypatch, append)
    if fmt in ("int8", "int4"):
        tab = torch.full((2, 4), 0.02, device=DEV)
        _both(monkeypatch, lambda: append(k_static=tab, v_static=tab.half()))
        _both(monkeypatch, lambda: append(clip_percentile=99.0))


def test_both_forms_agree_on_weights_and_eviction(monkeypatch):
    gen = torch.Generator().manual_seed(8)
    k, ks, _ = make_cache((2, 2, 300), 128, "int8", 32, gen)
    k, ks = k.to(DEV), ks.to(DEV)
    q = torch.randn(2, 12, 128, generator=gen).half().to(DEV)
    lens = torch.tensor([300, 41], dtype=torch.int32, device=DEV)
    out = torch.empty_like(q)

    def weights():
        w = torch.ones(2, 2, 310, device=DEV)
        r = ops.span_attn(q, k, k, ks, ks, lens, weights=w[:, :, :300], out=out)
        assert r is out
        return r.clone(), w
    w = _both(monkeypatch, weights)[1][:, :, :300].contiguous()

    def evict():
        ww, p, kk, ss = w.clone(), torch.full((2, 2, 300), -1, dtype=torch.int32, device=DEV), k.clone(), ks.clone()
        n = ops.evict(ww, p, lens, lens, 200, [kk, ss], sinks=4, recent=8)
        return n, ww, p, kk, ss
    _both(monkeypatch, evict)


@pytest.mark.parametrize("case", range(len(test_span_cpu.test_paged_attention_argument_checks.pytestmark[0].args[1])))
def test_what_is_refused_in_python_is_refused(case):
    edit, match = test_span_cpu.test_paged_attention_argument_checks.pytestmark[0].args[1][case]
    k, ks = test_span_cpu._pool()
    a = dict(q=torch.zeros(1, 4, 128).half(), k=k, v=k.clone(), ks=ks, vs=ks.clone(), table=torch.zeros(1, 2, dtype=torch.int32),
             lens=torch.zeros(1, dtype=torch.int32))
    edit(a)
    a = {n: t.to(DEV) if torch.is_tensor(t) else t for n, t in a.items()}
    args = [a.pop(n) for n in ("q", "k", "v", "ks", "vs", "lens")]
    with pytest.raises(ValueError, match=match):
        ops.span_attn(*args, block_table=a.pop("table"), **a)


def test_what_needs_a_conversion_is_converted():
    q, (k, v, ks, vs, _, _), table, lens, _ = _paged("int8")
    ref = ops.span_attn(q, k, v, ks, vs, lens, block_table=table)
    wide = torch.zeros(3, 12, 129, dtype=torch.float16, device=DEV)[..., 1:]
    wide.copy_(q)                                          # rows that do not start on 4 bytes
    for qq, nn in ((q, lens.long()), (wide, lens), (q, torch.stack((lens, lens), 1)[:, 0])):
        assert torch.equal(ops.span_attn(qq, k, v, ks, vs, nn, block_table=table), ref)
    with pytest.raises(ValueError, match="CUDA"):
        ops.span_attn(q, k, v, ks, vs, lens.cpu(), block_table=table)

