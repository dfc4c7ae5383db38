"""CPU-side checks of the bounded and paged cache operators: refusals before any launch, and the page bookkeeping."""
import contextlib
import ctypes as C

import pytest
import torch

import llm_kvcache_quantization_b200 as kvq
from llm_kvcache_quantization_b200 import _lib, build, ops
from span_reference import evict


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


def _span_args():
    s = _lib.KvqSpanAttnArgs()
    a = s.attn
    a.format, a.B, a.Hq, a.Hkv, a.D, a.group_size, a.max_ctx = _lib.FMT_INT8, 2, 12, 2, 128, 32, 100
    a.q = a.out = a.workspace = 4096
    a.workspace_bytes = 1 << 40
    for side in (a.k, a.v):
        side.payload, side.pay_stride_b, side.pay_stride_h, side.pay_stride_s = 4096, 25600, 12800, 128
        side.scale, side.sc_stride_b, side.sc_stride_h, side.sc_stride_s = 4096, 800, 400, 4
    return s


def test_struct_sizes():
    assert C.sizeof(_lib.KvqPageTable) == 2 * 8 + 3 * 4 + 4
    assert C.sizeof(_lib.KvqSpanAttnArgs) == C.sizeof(_lib.KvqAttnArgs) + 32 + 8 + 24
    assert C.sizeof(_lib.KvqPagedAppendArgs) == C.sizeof(_lib.KvqAppendArgs) + 32 + 16
    assert C.sizeof(_lib.KvqEvictArgs) == 6 * 4 + 3 * 8 + 6 * 8 + 8 + 10 * 40 + 16


def test_null_arguments(lib):
    for name in ("kvq_span_attn", "kvq_paged_append", "kvq_paged_read", "kvq_evict"):
        assert getattr(lib, name)(None, None) == _lib.KVQ_EINVAL
    assert lib.kvq_span_attn_workspace_bytes(None) == 0
    assert lib.kvq_span_attn_kernel_kind(None) == _lib.KVQ_EINVAL


@pytest.mark.parametrize("change,code", (
    (dict(Hq=5), _lib.KVQ_EINVAL), (dict(D=96), _lib.KVQ_EUNSUPPORTED), (dict(group_size=48), _lib.KVQ_EINVAL),
    (dict(format=7), _lib.KVQ_EINVAL), (dict(splits=2), _lib.KVQ_EINVAL), (dict(tail_tokens=1), _lib.KVQ_EINVAL),
    (dict(stages=1), _lib.KVQ_EINVAL), (dict(n_out=1), _lib.KVQ_EUNSUPPORTED), (dict(q=None), _lib.KVQ_EINVAL),
    (dict(out=None), _lib.KVQ_EINVAL), (dict(max_ctx=-1), _lib.KVQ_EINVAL), (dict(B=-1), _lib.KVQ_EINVAL),
    (dict(max_ctx=2000, workspace_bytes=1024), _lib.KVQ_EWORKSPACE), (dict(max_ctx=2000, workspace=None), _lib.KVQ_EWORKSPACE),
    (dict(q=4097), _lib.KVQ_EINVAL), (dict(B=70000), _lib.KVQ_ELIMIT), (dict(max_ctx=2 ** 31 - 1, B=64), _lib.KVQ_ELIMIT)))
def test_span_attn_refusals(lib, change, code):
    s = _span_args()
    for k, x in change.items():
        setattr(s.attn, k, x)
    assert lib.kvq_span_attn(C.byref(s), None) == code


def test_span_attn_refusals_of_the_span_fields(lib):
    def call(**kw):
        s = _span_args()
        for k, x in kw.items():
            setattr(s, k, x)
        return lib.kvq_span_attn(C.byref(s), None)
    table = _lib.KvqPageTable(4096, 4, 4, 32, 9)
    assert call(window=-1) == _lib.KVQ_EINVAL
    assert call(sinks=4) == _lib.KVQ_EINVAL                 # sinks without a window
    assert call(window=4, sinks=-1) == _lib.KVQ_EINVAL
    assert call(window=4, weights=4096) == _lib.KVQ_EUNSUPPORTED
    assert call(pages=table, weights=4096) == _lib.KVQ_EUNSUPPORTED
    for bad in ((4096, 4, 4, 0, 9), (4096, 4, 0, 32, 9), (4096, 4, 4, 32, 0), (4096, 4, 3, 32, 9)):
        assert call(pages=_lib.KvqPageTable(*bad)) == _lib.KVQ_EINVAL          # the last: 96 < max_ctx tokens
    s = _span_args()
    s.attn.k.pay_stride_s = 120
    assert lib.kvq_span_attn(C.byref(s), None) == _lib.KVQ_EINVAL
    s = _span_args()
    s.attn.v.scale = None
    assert lib.kvq_span_attn(C.byref(s), None) == _lib.KVQ_EINVAL
    s = _span_args()
    s.attn.k.zp = 4096                                      # zero-points on one side only
    assert lib.kvq_span_attn(C.byref(s), None) == _lib.KVQ_EINVAL


def test_paged_append_and_read_refusals(lib):
    def args():
        p = _lib.KvqPagedAppendArgs()
        a = p.append
        a.format, a.policy, a.B, a.Hkv, a.T, a.D, a.group_size = _lib.FMT_INT8, _lib.SCALE_DYNAMIC_PCT, 2, 2, 3, 128, 32
        a.quantile = 1.0
        for side in (a.k, a.v):
            side.src = side.payload = side.scale = 4096
            side.pay_stride_b, side.pay_stride_h, side.pay_stride_s = 8192, 4096, 128
        p.pages = _lib.KvqPageTable(4096, 4, 4, 32, 9)
        p.start_pos = 4096
        return p
    for path, x, code in (("write_pos", 1, _lib.KVQ_EINVAL), ("max_slots", 5, _lib.KVQ_EINVAL), ("n_out", 1, _lib.KVQ_EUNSUPPORTED),
                          ("rope_cos", 4096, _lib.KVQ_EUNSUPPORTED), ("policy", 3, _lib.KVQ_EINVAL), ("format", 9, _lib.KVQ_EINVAL),
                          ("group_size", 24, _lib.KVQ_EINVAL), ("T", -1, _lib.KVQ_EINVAL)):
        p = args()
        setattr(p.append, path, x)
        assert lib.kvq_paged_append(C.byref(p), None) == code, path
    p = args()
    p.start_pos = None
    assert lib.kvq_paged_append(C.byref(p), None) == _lib.KVQ_EINVAL
    p = args()
    p.pages.table = None
    assert lib.kvq_paged_append(C.byref(p), None) == _lib.KVQ_EINVAL
    p = args()
    p.append.k.pay_stride_s = 136
    assert lib.kvq_paged_append(C.byref(p), None) == _lib.KVQ_EINVAL
    r = _lib.KvqPagedReadArgs()
    r.format, r.B, r.Hkv, r.T, r.D, r.group_size = _lib.FMT_INT8, 2, 2, 3, 96, 32
    assert lib.kvq_paged_read(C.byref(r), None) == _lib.KVQ_EUNSUPPORTED
    r.D = 128
    assert lib.kvq_paged_read(C.byref(r), None) == _lib.KVQ_EINVAL             # no table


def test_evict_refusals(lib):
    def args():
        e = _lib.KvqEvictArgs()
        e.B, e.Hkv, e.cap, e.budget, e.sinks, e.recent = 2, 2, 100, 50, 4, 8
        e.lengths = e.seen = e.new_lengths = e.weights = e.positions = e.workspace = 4096
        e.workspace_bytes = 1 << 30
        e.n_bufs = 1
        e.bufs[0] = _lib.KvqEvictBuf(4096, 25600, 12800, 128, 128)
        return e
    for path, x, code in (("budget", 0, -1), ("sinks", 43, -1), ("recent", -1, -1), ("n_bufs", 11, -1), ("lengths", None, -1),
                          ("workspace", None, _lib.KVQ_EWORKSPACE), ("workspace_bytes", 10, _lib.KVQ_EWORKSPACE),
                          ("B", 70000, _lib.KVQ_ELIMIT), ("cap", -1, -1)):
        e = args()
        setattr(e, path, x)
        assert lib.kvq_evict(C.byref(e), None) == code, path
    e = args()
    e.bufs[0].row_bytes = 0
    assert lib.kvq_evict(C.byref(e), None) == _lib.KVQ_EINVAL
    e = args()
    e.bufs[0].row_bytes = (1 << 30) + 1
    assert lib.kvq_evict(C.byref(e), None) == _lib.KVQ_ELIMIT
    for new in (4096, 4100, 4092):                                              # overlaps the lengths that every head reads
        e = args()
        e.new_lengths = new
        assert lib.kvq_evict(C.byref(e), None) == _lib.KVQ_EINVAL


def test_wrappers_refuse_cpu_tensors():
    q = torch.zeros(1, 4, 128, dtype=torch.float16)
    k = torch.zeros(1, 2, 8, 128, dtype=torch.float16)
    ctx = torch.tensor([8], dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        kvq.decode_attn_window(q, k, k, None, None, ctx, 4)
    with pytest.raises(ValueError, match="CUDA"):
        kvq.decode_attn_paged(q, k, k, None, None, ctx[None], ctx)
    with pytest.raises(ValueError, match="CUDA"):
        kvq.decode_attn_weights(q, k, k, None, None, ctx, torch.zeros(1, 2, 8))
    with pytest.raises(ValueError, match="CUDA"):
        kvq.evict_tokens(torch.zeros(1, 2, 8), torch.zeros(1, 2, 8, dtype=torch.int32), ctx, ctx, 4, [k])
    with pytest.raises(ValueError, match="needs a window"):
        kvq.decode_attn_window(q, k, k, None, None, ctx, None)
    with pytest.raises(ValueError, match="weights tensor"):
        kvq.decode_attn_weights(q, k, k, None, None, ctx, None)


@pytest.fixture
def no_device_check(monkeypatch):
    """The wrappers' own argument checks, without a device: everything before the first library call."""
    monkeypatch.setattr(ops, "_require_cuda", lambda *t: torch.device("cpu"))


def _pool(fmt="int8", pages=4, heads=2, page=16, D=128, G=4):
    w = {"fp16": D, "int8": D, "int4": D // 2}[fmt]
    k = torch.zeros(pages, heads, page, w, dtype=torch.float16 if fmt == "fp16" else torch.int8)
    return k, (None if fmt == "fp16" else torch.zeros(pages, heads, page, G, dtype=torch.float16))


@pytest.mark.parametrize("edit,match", (
    (lambda a: a.update(q=a["q"][0]), "q must have shape"),
    (lambda a: a.update(q=a["q"].double()), "fp16 query"),
    (lambda a: a.update(q=torch.zeros(1, 4, 96).half()), "head_dim must be"),
    (lambda a: a.update(k=a["k"].float()), "payload must be"),
    (lambda a: a.update(k=a["k"][..., :100]), "width"),
    (lambda a: a.update(v=a["v"][:, :, :8]), "k/v cache mismatch"),
    (lambda a: a.update(ks=None), "needs k_scale"),
    (lambda a: a.update(ks=a["ks"].float()), "k_scale must be fp16"),
    (lambda a: a.update(ks=a["ks"][..., :3], vs=a["vs"][..., :3]), "num_groups 3"),
    (lambda a: a.update(vs=a["vs"][..., :2]), "num_groups mismatch"),
    (lambda a: a.update(k_zp=a["ks"]), "go together"),
    (lambda a: a.update(k_zp=a["ks"][..., :2], v_zp=a["vs"][..., :2]), "shape and strides"),
    (lambda a: a.update(q=torch.zeros(1, 3, 128).half()), "GQA head mismatch"),
    (lambda a: a.update(table=a["table"].long()), "block_table must be int32"),
    (lambda a: a.update(table=torch.zeros(2, 2, dtype=torch.int32)), "block_table must be int32"),
    (lambda a: a.update(lens=torch.zeros(2, dtype=torch.int32)), "context_lens must be 1D"),
    (lambda a: a.update(lens=None), "needs context_lens"),
    (lambda a: a.update(window=0), "window must be >= 1"),
    (lambda a: a.update(sinks=3), "sinks go with a window"),
    (lambda a: a.update(window=3, sinks=-1), "sinks >= 0"),
    (lambda a: a.update(max_ctx=-1), "max_ctx"),
    (lambda a: a.update(inv_tau=torch.ones(3)), "inv_tau"),
    (lambda a: a.update(out=torch.zeros(1, 4, 128)), "out must be"),
))
def test_paged_attention_argument_checks(no_device_check, edit, match):
    k, ks = _pool()
    a = dict(q=torch.zeros(1, 4, 128).half(), k=k, v=k.clone(), ks=ks, vs=ks.clone(), table=torch.zeros(1, 2, dtype=torch.int32),
             lens=torch.zeros(1, dtype=torch.int32))
    edit(a)
    args = [a.pop(n) for n in ("q", "k", "v", "ks", "vs", "lens")]
    with pytest.raises(ValueError, match=match):
        ops.span_attn(*args, block_table=a.pop("table"), **a)


def test_misaligned_caches_and_weights_are_refused(no_device_check):
    q = torch.zeros(1, 4, 128).half()
    base = torch.zeros(1, 2, 8, 130, dtype=torch.float16)
    with pytest.raises(ValueError, match="16-byte"):
        ops.span_attn(q, base[..., :128], base[..., :128], None, None, None, window=4)
    k = torch.zeros(1, 2, 8, 128, dtype=torch.float16)
    for w in (torch.zeros(1, 2, 7), torch.zeros(1, 2, 8).double(), torch.zeros(1, 1, 8), torch.zeros(1, 2, 16)[:, :, ::2],
              torch.zeros(1, 1, 8).expand(1, 2, 8)):
        with pytest.raises(ValueError, match="weights must be"):
            ops.span_attn(q, k, k, None, None, None, weights=w)
    with pytest.raises(ValueError, match="no scales"):
        ops.span_attn(q, k, k, k[..., :1], None, None)


def test_append_and_read_argument_checks(no_device_check):
    k, ks = _pool()
    new = torch.zeros(1, 2, 3, 128).half()
    table, one = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)

    def app(k_new=new, v_new=new, kp=k, sc=ks, t=table, start=one, n=None, **kw):
        ops.paged_append(k_new, v_new, kp, kp, sc, sc, t, start, n, **kw)
    for kw, match in ((dict(v_new=new[:, :, :2]), "shape mismatch"), (dict(k_new=new[:, :1], v_new=new[:, :1]), "heads mismatch"),
                      (dict(k_static=torch.ones(2, 4)), "go together"), (dict(clip_percentile=0.0), "clip_percentile"),
                      (dict(k_static=torch.ones(2, 3), v_static=torch.ones(2, 3)), "k_static must be"),
                      (dict(k_static=torch.ones(2, 4), v_static=torch.ones(2, 4), k_zp=ks, v_zp=ks), "static scales"),
                      (dict(start=torch.zeros(2, dtype=torch.int32)), "start_pos must be"),
                      (dict(n=torch.zeros(2, dtype=torch.int32)), "new_lens must be"), (dict(t=table.long()), "block_table")):
        with pytest.raises(ValueError, match=match):
            app(**kw)
    for kw, match in ((dict(head_dim=96), "head_dim must be"), (dict(head_dim=256), "num_groups|width|multiple"), (dict(tokens=-1), "tokens")):
        args = dict(tokens=3, head_dim=128)
        args.update(kw)
        with pytest.raises(ValueError, match=match):
            t = args.pop("tokens")
            ops.paged_read(k, k, ks if args["head_dim"] != 256 else ks[..., :3], ks if args["head_dim"] != 256 else ks[..., :3],
                           table, one, t, **args)


def test_evict_argument_checks(no_device_check):
    w, p = torch.zeros(2, 2, 8), torch.full((2, 2, 8), -1, dtype=torch.int32)
    lens = torch.zeros(2, dtype=torch.int32)
    k = torch.zeros(2, 2, 8, 4)

    def ev(w=w, p=p, lens=lens, budget=4, bufs=(k,), **kw):
        ops.evict(w, p, lens, lens, budget, bufs, **kw)
    for kw, match in ((dict(w=w.double()), "weights must be"), (dict(p=p.long()), "positions must be"),
                      (dict(budget=0), "budget"), (dict(sinks=3, recent=2), "budget"), (dict(bufs=(k,) * 11), "at most 10"),
                      (dict(bufs=(k[:1],)), "buffer 0"), (dict(bufs=(k, k[:, :, :7])), "buffer 1"),
                      (dict(bufs=(k.transpose(2, 3).contiguous().transpose(2, 3),)), "contiguous"),
                      (dict(bufs=(k[..., :0],)), "empty rows"), (dict(bufs=(k[:, :1].expand(2, 2, 8, 4),)), "overlap"),
                      (dict(lens=torch.zeros(3, dtype=torch.int32)), "lengths"),
                      (dict(w=w[:, :1].expand(2, 2, 8)), "rows that do not overlap")):
        with pytest.raises(ValueError, match=match):
            ev(**kw)


def test_numbers_beyond_32_bits(no_device_check, monkeypatch):
    """A window that 32 bits do not hold is the whole row, not what is left of the number; such a budget is refused."""
    k, ks = _pool()
    seen = []

    class Fake:
        def kvq_span_attn_workspace_bytes(self, s):
            return 256

        def kvq_span_attn(self, s, stream):
            seen.append((s._obj.window, s._obj.sinks))
            return 0
    monkeypatch.setattr(_lib, "load", lambda: Fake())
    monkeypatch.setattr(ops, "_stream_ptr", lambda d: 0)
    monkeypatch.setattr(ops, "_MARSHAL", type("N", (), {"span_attn": lambda *a: None})())
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    for window, sinks in ((2 ** 32 + 5, 4), (7, 2 ** 33 + 1)):
        ops.span_attn(torch.zeros(4, 4, 128).half(), k, k, ks, ks, None, window=window, sinks=sinks)
    assert seen == [(2 ** 31 - 1, 4), (7, 2 ** 31 - 1)]
    w, p = torch.zeros(1, 1, 8), torch.full((1, 1, 8), -1, dtype=torch.int32)
    n = torch.full((1,), 8, dtype=torch.int32)
    monkeypatch.undo()
    monkeypatch.setattr(ops, "_require_cuda", lambda *t: torch.device("cpu"))
    with pytest.raises(ValueError, match="2.31"):
        ops.evict(w, p, n, n, 2 ** 32 + 1, ())


def test_plain_eviction_by_hand():
    """The reference itself: budget 3 of 5 tokens, one sink, one recent; slot 1 beats 2 and 3 only by its sum."""
    w = torch.tensor([[[0.0, 5.0, 1.0, 2.0, 0.0]]])
    p = torch.full((1, 1, 5), -1, dtype=torch.int32)
    n = torch.tensor([5], dtype=torch.int32)
    rw, rp, rn, moves = evict(w, p, n, n, 3, 1, 1)
    assert moves[0, 0] == ([2], [4]) and rp.tolist() == [[[0, 1, 4, -1, -1]]] and rn.tolist() == [3]
    assert rw.tolist() == [[[0.0, 5.0, 0.0, 0.0, 0.0]]]
    # ties: the lowest slots stay
    rw, rp, _, moves = evict(torch.ones(1, 1, 5), p, n, n, 3, 0, 0)
    assert moves[0, 0] == ([], []) and rp.tolist() == [[[0, 1, 2, -1, -1]]]


# ------------------------------------------------------------------------------------------------ host bookkeeping
def _cache(**kw):
    args = dict(page_size=16, kv_format="int8", group_size=32, device="cpu")
    args.update(kw)
    return kvq.PagedKVCache(2, 6, 2, 128, **args)


@pytest.mark.parametrize("kw", (dict(page_size=20), dict(page_size=0), dict(kv_format="int2"), dict(group_size=48),
                                dict(window=0), dict(sinks=4), dict(clip_percentile=0.0),
                                dict(static_k_scale=torch.ones(2, 2, 4)),
                                dict(static_k_scale=torch.ones(2, 2, 3), static_v_scale=torch.ones(2, 2, 3)),
                                dict(kv_format="int4_asym", static_k_scale=torch.ones(2, 2, 4), static_v_scale=torch.ones(2, 2, 4))))
def test_paged_cache_constructor_checks(kw):
    with pytest.raises(ValueError):
        _cache(**kw)


def test_paged_cache_pages_are_reserved_shared_and_returned():
    c = _cache()
    with pytest.raises(ValueError, match="0 sequences"):
        c._begin(1, 1, None)
    a, b = c.add_sequence(), c.add_sequence()
    assert c.sequences == (a, b) and c.num_free_pages == 6
    c._begin(2, 20, [20, 16])
    c._step_layer = 2
    table, start, lens, longest, counts = c._step
    assert start.tolist() == [0, 0] and lens.tolist() == [20, 16] and longest == 20 and counts.tolist() == [20, 16]
    assert table.tolist() == [[0, 1], [2, -1]] and c.num_free_pages == 3
    c._begin(2, 1, None)
    table, start, lens, longest, counts = c._step
    assert start.tolist() == [20, 16] and lens.tolist() == [21, 17] and counts is None
    assert table.tolist() == [[0, 1], [2, 3]]
    c._step_layer = 2
    with pytest.raises(ValueError, match="exhausted"):
        c._begin(2, 30, None)                               # 2 more pages each, 2 free
    assert c.get_seq_lens() == (21, 17) and c.num_free_pages == 2
    c.free_sequence(a)
    assert c.sequences == (b,) and c.num_free_pages == 4
    with pytest.raises(ValueError, match="unknown"):
        c.free_sequence(a)
    with pytest.raises(ValueError, match="counts"):
        c._begin(1, 4, [5])
    with pytest.raises(ValueError, match="nothing was appended"):
        c.fused_decode(0, torch.zeros(1, 2, 128).half())
    with pytest.raises(ValueError, match="CPU tensors"):
        c.append(0, torch.zeros(1, 2, 1, 128).half(), torch.zeros(1, 2, 1, 128).half())
    c._begin(1, 1, None)
    c._step_layer = 1
    with pytest.raises(ValueError, match="middle of a step"):
        c.add_sequence()
    with pytest.raises(ValueError, match="middle of a step"):
        c._begin(1, 1, None)
    c.clear()
    assert c.num_free_pages == 6 and c.sequences == () and c.get_seq_len() == 0


def test_max_pages_per_sequence():
    c = _cache(max_pages_per_seq=2)
    c.add_sequence()
    c._begin(1, 32, None)
    c._step_layer = 2
    with pytest.raises(ValueError, match="max_pages_per_seq"):
        c._begin(1, 1, None)


def test_bounded_cache_settings():
    c = kvq.INT8KVCache(2, device="cpu")
    for bad in ((0, 0), (5, -1)):
        with pytest.raises(ValueError, match="window"):
            c.set_attention_window(*bad)
    with pytest.raises(ValueError, match="sinks go with"):
        c.set_attention_window(None, 3)
    c.set_attention_window(10, 2)
    with pytest.raises(ValueError, match="attention window takes no eviction"):
        c.enable_eviction(100)
    c.set_attention_window(None)
    with pytest.raises(ValueError, match="budget"):
        c.enable_eviction(30, sinks=4, recent=32)
    c.enable_eviction(100)
    with pytest.raises(ValueError, match="already"):
        c.enable_eviction(100)
    with pytest.raises(ValueError, match="no attention window"):
        c.set_attention_window(10)
    with pytest.raises(ValueError, match="device-side positions"):
        c.use_device_positions(torch.zeros(1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), 1)
    o = kvq.INT4KVCache(1, device="cpu", outlier_idx=torch.zeros(1, 2, 1, dtype=torch.int16))
    for call in (lambda: o.set_attention_window(4), lambda: o.enable_eviction(100)):
        with pytest.raises(ValueError, match="outlier"):
            call()
    t = kvq.INT8KVCache(1, device="cpu", decode_attn_impl="torch_ref")
    with pytest.raises(ValueError, match="torch_ref"):
        t.set_attention_window(4)
    from llm_kvcache_quantization_b200.runtime import GraphedKVStackStep
    with pytest.raises(ValueError, match="no attention window and no eviction"):
        GraphedKVStackStep(c, 4, 1.0)
