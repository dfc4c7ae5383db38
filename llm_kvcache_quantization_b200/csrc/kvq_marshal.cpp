// Python module _marshal: fills the argument structs of the bounded- and paged-cache entry points from torch tensors and
// calls libkvq.  ops.py offers the same operations in Python with every check spelled out; there a call of some 60 field
// assignments and 40 tensor attributes costs the host 30 to 42 us, more than the kernels of a short decode step take.  Here
// the ordinary call - tensors of the documented types and layouts, on one CUDA device, nothing to convert - takes the
// marshalling out of the interpreter: paged attention 40 -> 9 us a call, with weights 42 -> 11, append 30 -> 3, read-back
// 30 -> 5, eviction 30 -> 7 (launches included).
// A function returns None, with nothing done, for whatever is not that ordinary call; the caller then takes the Python
// form, which converts, or says what is wrong.  So every condition here is at least as strict as its check there.
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <climits>
#include <cmath>
#include <exception>

#include "kvq.h"

namespace {

struct Lib {
    int (*span_attn)(const KvqSpanAttnArgs*, kvq_stream_t);
    size_t (*span_attn_ws)(const KvqSpanAttnArgs*);
    int (*paged_append)(const KvqPagedAppendArgs*, kvq_stream_t);
    int (*paged_read)(const KvqPagedReadArgs*, kvq_stream_t);
    int (*evict)(const KvqEvictArgs*, kvq_stream_t);
    size_t (*evict_ws)(int32_t, int32_t, int32_t, int32_t);
};
Lib lib{};
PyObject* check_fn = nullptr;      // check(name, status): raises for a status that is not 0

// An optional tensor argument: a plain strided CUDA tensor on the device of the call, or None.
struct Arg {
    const at::Tensor* t = nullptr;
    explicit operator bool() const { return t != nullptr; }
    const at::Tensor* operator->() const { return t; }
    void* ptr() const { return t ? t->data_ptr() : nullptr; }
    bool is(at::ScalarType s) const { return t->scalar_type() == s; }
};

struct Call {
    c10::Device dev{c10::kCPU};
    bool ok = true;
    Arg opt(PyObject* o) {
        Arg a;
        if (o == Py_None) return a;
        if (!THPVariable_CheckExact(o)) { ok = false; return a; }
        const at::Tensor& t = THPVariable_Unpack(o);
        if (!t.is_cuda() || t.layout() != at::kStrided) { ok = false; return a; }
        if (dev.is_cpu()) dev = t.device();
        if (t.device() != dev) { ok = false; return a; }
        a.t = &t;
        return a;
    }
    Arg need(PyObject* o) {
        Arg a = opt(o);
        if (!a) ok = false;
        return a;
    }
    // A Python int in [lo, hi]; `none` for None.
    long long integer(PyObject* o, long long lo, long long hi, long long none) {
        if (o == Py_None) return none;
        if (!PyLong_CheckExact(o)) { ok = false; return 0; }
        int over = 0;
        const long long v = PyLong_AsLongLongAndOverflow(o, &over);
        if (over || v < lo || v > hi) { ok = false; return 0; }
        return v;
    }
};

struct Cache {
    int format = 0, group = 0;
    int64_t major = 0, heads = 0, slots = 0;
};

// One side (K or V) of a cache: alignment, scales, zero-points.
bool side(KvqCacheSide& s, const Arg& p, const Arg& sc, const Arg& zp) {
    const int64_t es = p->element_size();
    if (p->stride(3) != 1 || ((uintptr_t)p.ptr() & 15)) return false;
    for (int d = 0; d < 3; ++d)
        if (p->size(d) > 1 && p->stride(d) * es % 16) return false;
    s = KvqCacheSide{};
    s.payload = p.ptr();
    s.pay_stride_b = p->stride(0) * es, s.pay_stride_h = p->stride(1) * es, s.pay_stride_s = p->stride(2) * es;
    if (!sc) return !zp;
    if (!sc.is(at::kHalf) || sc->dim() != 4 || sc->sizes().slice(0, 3) != p->sizes().slice(0, 3)) return false;
    if (sc->size(3) > 1 && sc->stride(3) != 1) return false;
    s.scale = sc.ptr();
    s.sc_stride_b = sc->stride(0), s.sc_stride_h = sc->stride(1), s.sc_stride_s = sc->stride(2);
    if (zp) {
        if (!zp.is(at::kHalf) || zp->sizes() != sc->sizes() || zp->strides() != sc->strides()) return false;
        s.zp = zp.ptr();
    }
    return true;
}

bool cache(Cache& c, KvqCacheSide& ks, KvqCacheSide& vs, int64_t D, const Arg& k, const Arg& v, const Arg& k_scale,
           const Arg& v_scale, const Arg& k_zp, const Arg& v_zp) {
    if (k->dim() != 4 || k->sizes() != v->sizes() || k->scalar_type() != v->scalar_type() || k->numel() == 0) return false;
    c.major = k->size(0), c.heads = k->size(1), c.slots = k->size(2);
    if (c.major > INT_MAX || c.heads > INT_MAX || c.slots > INT_MAX) return false;
    const int64_t w = k->size(3);
    if (k.is(at::kHalf)) {
        if (w != D || k_scale || v_scale || k_zp || v_zp) return false;
        c.format = KVQ_FMT_FP16, c.group = (int)D;
    } else {
        if (!k.is(at::kChar) || (w != D && 2 * w != D)) return false;
        if (!k_scale || !v_scale || (bool)k_zp != (bool)v_zp || k_scale->dim() != 4) return false;
        const int64_t groups = k_scale->size(3);
        if (groups < 1 || D % groups || D / groups % 8 || v_scale->dim() != 4 || v_scale->size(3) != groups) return false;
        c.format = w == D ? KVQ_FMT_INT8 : KVQ_FMT_INT4, c.group = (int)(D / groups);
    }
    return side(ks, k, k_scale, k_zp) && side(vs, v, v_scale, v_zp);
}

bool lengths(const Arg& t, int64_t B) { return t.is(at::kInt) && t->dim() == 1 && t->size(0) == B && t->is_contiguous(); }

bool table(KvqPageTable& p, const Arg& t, int64_t B, const Cache& c) {
    if (!t.is(at::kInt) || t->dim() != 2 || t->size(0) != B || t->size(1) < 1 || t->size(1) > INT_MAX) return false;
    if (t->size(1) > 1 && t->stride(1) != 1) return false;
    p.table = (const int32_t*)t.ptr();
    p.stride_b = t->stride(0), p.cols = (int32_t)t->size(1), p.page_size = (int32_t)c.slots, p.num_pages = (int32_t)c.major;
    return true;
}

// fp32 [B, Hkv, slots] / int32 alike, contiguous in its slots, rows apart
bool slot_rows(const Arg& t) {
    const int64_t n = t->size(2);
    if (n > 1 && t->stride(2) != 1) return false;
    return !(t->size(0) > 1 && t->stride(0) < n) && !(t->size(1) > 1 && t->stride(1) < n);
}

at::Tensor empty(at::IntArrayRef size, at::ScalarType type, c10::Device dev) {
    return at::empty(size, at::TensorOptions().dtype(type).device(dev));
}

template <class F>
bool launch(const char* name, F f) {
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = f();
    Py_END_ALLOW_THREADS
    if (rc == KVQ_OK) return true;
    PyObject* r = PyObject_CallFunction(check_fn, "si", name, rc);
    Py_XDECREF(r);
    if (!PyErr_Occurred()) PyErr_Format(PyExc_RuntimeError, "%s failed (code %d)", name, rc);
    return false;
}

kvq_stream_t stream_of(c10::Device dev) { return (kvq_stream_t)c10::cuda::getCurrentCUDAStream(dev.index()).stream(); }

// ------------------------------------------------------------------------------------------------------------------
// span_attn(q, k, v, k_scale, v_scale, context_lens, sm_scale, k_zp, v_zp, block_table, window, sinks, weights, max_ctx,
//           inv_tau, out)
PyObject* span_attn(PyObject* const* o, Py_ssize_t n) {
    if (n != 16) Py_RETURN_NONE;
    Call c;
    const Arg q = c.need(o[0]), k = c.need(o[1]), v = c.need(o[2]), ks = c.opt(o[3]), vs = c.opt(o[4]), lens = c.opt(o[5]),
              kz = c.opt(o[7]), vz = c.opt(o[8]), tab = c.opt(o[9]), w = c.opt(o[12]), tau = c.opt(o[14]), out = c.opt(o[15]);
    const long long window = c.integer(o[10], 1, INT_MAX, 0), sinks = c.integer(o[11], 0, INT_MAX, 0),
                    bound = c.integer(o[13], 0, LLONG_MAX, LLONG_MAX);
    if (!c.ok || (o[6] != Py_None && !PyFloat_CheckExact(o[6])) || (window == 0 && sinks)) Py_RETURN_NONE;
    if (q->dim() != 3 || !q.is(at::kHalf) || q->numel() == 0) Py_RETURN_NONE;
    const int64_t B = q->size(0), Hq = q->size(1), D = q->size(2);
    if ((D != 64 && D != 128 && D != 256) || B > INT_MAX || Hq > INT_MAX) Py_RETURN_NONE;
    if (q->stride(2) != 1 || q->stride(0) % 2 || q->stride(1) % 2 || ((uintptr_t)q.ptr() & 3)) Py_RETURN_NONE;
    KvqSpanAttnArgs s{};
    KvqAttnArgs& a = s.attn;
    Cache ch;
    if (!cache(ch, a.k, a.v, D, k, v, ks, vs, kz, vz) || Hq % ch.heads) Py_RETURN_NONE;
    long long span;
    if (tab) {
        if (!lens || !table(s.pages, tab, B, ch)) Py_RETURN_NONE;
        span = std::min<long long>((long long)s.pages.cols * s.pages.page_size, INT_MAX);
    } else {
        if (ch.major != B) Py_RETURN_NONE;
        span = ch.slots;
    }
    span = std::min(span, bound);
    if (lens && !lengths(lens, B)) Py_RETURN_NONE;
    if (tau && (!tau.is(at::kFloat) || !tau->is_contiguous() || tau->numel() != Hq)) Py_RETURN_NONE;
    if (w) {
        if (!w.is(at::kFloat) || w->dim() != 3 || w->size(0) != B || w->size(1) != ch.heads || w->size(2) < span) Py_RETURN_NONE;
        if (!slot_rows(w)) Py_RETURN_NONE;
        s.weights = (float*)w.ptr(), s.w_stride_b = w->stride(0), s.w_stride_h = w->stride(1);
    }
    if (out && (!out.is(at::kHalf) || out->sizes() != q->sizes() || out->stride(2) != 1)) Py_RETURN_NONE;
    c10::cuda::CUDAGuard guard(c.dev);
    at::Tensor made;
    if (!out) made = empty({B, Hq, D}, at::kHalf, c.dev);
    const at::Tensor& dst = out ? *out.t : made;
    a.format = ch.format, a.B = (int32_t)B, a.Hq = (int32_t)Hq, a.Hkv = (int32_t)ch.heads, a.D = (int32_t)D;
    a.group_size = ch.group, a.max_ctx = (int32_t)span;
    a.q = q.ptr(), a.q_stride_b = q->stride(0), a.q_stride_h = q->stride(1);
    a.out = dst.data_ptr(), a.out_stride_b = dst.stride(0), a.out_stride_h = dst.stride(1);
    a.sm_scale = (float)(o[6] == Py_None ? 1.0 / std::sqrt((double)D) : PyFloat_AS_DOUBLE(o[6]));
    a.inv_tau = (const float*)tau.ptr();
    a.context_lens = (const int32_t*)lens.ptr();
    s.window = (int32_t)window, s.sinks = (int32_t)sinks;
    // scratch of this call only: inside a graph capture it comes from that graph's pool
    const size_t bytes = std::max<size_t>(lib.span_attn_ws(&s), 256);
    const at::Tensor ws = empty({(int64_t)bytes}, at::kByte, c.dev);
    a.workspace = ws.data_ptr(), a.workspace_bytes = bytes;
    if (!launch("kvq_span_attn", [&] { return lib.span_attn(&s, stream_of(c.dev)); })) return nullptr;
    if (out) return Py_NewRef(o[15]);
    return THPVariable_Wrap(std::move(made));
}

// paged_append(k_new, v_new, k_pages, v_pages, k_scale, v_scale, block_table, start_pos, new_lens, k_zp, v_zp, k_static,
//              v_static, clip_percentile) -> True
bool append_side(KvqAppendSide& d, const KvqCacheSide& p, const Arg& src, const Arg& fixed, int64_t H, int64_t groups) {
    if (src->stride(3) != 1) return false;
    d.src = src.ptr(), d.src_stride_b = src->stride(0), d.src_stride_h = src->stride(1), d.src_stride_t = src->stride(2);
    d.payload = (void*)p.payload, d.pay_stride_b = p.pay_stride_b, d.pay_stride_h = p.pay_stride_h, d.pay_stride_s = p.pay_stride_s;
    d.scale = (void*)p.scale, d.zp = (void*)p.zp;
    d.sc_stride_b = p.sc_stride_b, d.sc_stride_h = p.sc_stride_h, d.sc_stride_s = p.sc_stride_s;
    if (fixed) {
        if (!(fixed.is(at::kHalf) || fixed.is(at::kFloat)) || fixed->dim() != 2 || fixed->size(0) != H ||
            fixed->size(1) != groups || !fixed->is_contiguous()) return false;
        d.static_scale = fixed.ptr(), d.static_scale_is_f32 = fixed.is(at::kFloat);
    }
    return true;
}

PyObject* paged_append(PyObject* const* o, Py_ssize_t n) {
    if (n != 14) Py_RETURN_NONE;
    Call c;
    const Arg kn = c.need(o[0]), vn = c.need(o[1]), k = c.need(o[2]), v = c.need(o[3]), ks = c.opt(o[4]), vs = c.opt(o[5]),
              tab = c.need(o[6]), start = c.need(o[7]), lens = c.opt(o[8]), kz = c.opt(o[9]), vz = c.opt(o[10]),
              kf = c.opt(o[11]), vf = c.opt(o[12]);
    if (!c.ok || !PyFloat_CheckExact(o[13])) Py_RETURN_NONE;
    const double clip = PyFloat_AS_DOUBLE(o[13]);
    if (!(clip > 0.0 && clip <= 100.0)) Py_RETURN_NONE;
    if (kn->dim() != 4 || kn->sizes() != vn->sizes() || !kn.is(at::kHalf) || !vn.is(at::kHalf) || kn->numel() == 0) Py_RETURN_NONE;
    const int64_t B = kn->size(0), H = kn->size(1), T = kn->size(2), D = kn->size(3);
    if (B > INT_MAX || T > INT_MAX || D > INT_MAX) Py_RETURN_NONE;
    Cache ch;
    KvqCacheSide kc, vc;
    if (!cache(ch, kc, vc, D, k, v, ks, vs, kz, vz) || ch.heads != H) Py_RETURN_NONE;
    if ((bool)kf != (bool)vf || (kf && (kz || ch.format == KVQ_FMT_FP16))) Py_RETURN_NONE;
    KvqPagedAppendArgs p{};
    KvqAppendArgs& a = p.append;
    if (!append_side(a.k, kc, kn, kf, H, D / ch.group) || !append_side(a.v, vc, vn, vf, H, D / ch.group)) Py_RETURN_NONE;
    if (!table(p.pages, tab, B, ch) || !lengths(start, B) || (lens && !lengths(lens, B))) Py_RETURN_NONE;
    p.start_pos = (const int32_t*)start.ptr(), p.new_lens = (const int32_t*)lens.ptr();
    a.format = ch.format, a.B = (int32_t)B, a.Hkv = (int32_t)H, a.T = (int32_t)T, a.D = (int32_t)D, a.group_size = ch.group;
    a.adaptive_margin = 1.f;
    a.quantile = clip < 100.0 ? (float)(clip / 100.0) : 1.f;
    a.policy = ch.format == KVQ_FMT_FP16 || kf ? KVQ_SCALE_STATIC : kz ? KVQ_SCALE_ASYM_MINMAX : KVQ_SCALE_DYNAMIC_PCT;
    c10::cuda::CUDAGuard guard(c.dev);
    if (!launch("kvq_paged_append", [&] { return lib.paged_append(&p, stream_of(c.dev)); })) return nullptr;
    Py_RETURN_TRUE;
}

// paged_read(k_pages, v_pages, k_scale, v_scale, block_table, start_pos, tokens, lens, head_dim, k_zp, v_zp) -> (k, v)
PyObject* paged_read(PyObject* const* o, Py_ssize_t n) {
    if (n != 11) Py_RETURN_NONE;
    Call c;
    const Arg k = c.need(o[0]), v = c.need(o[1]), ks = c.opt(o[2]), vs = c.opt(o[3]), tab = c.need(o[4]), start = c.opt(o[5]),
              lens = c.opt(o[7]), kz = c.opt(o[9]), vz = c.opt(o[10]);
    const long long T = c.integer(o[6], 1, INT_MAX, 0), D = c.integer(o[8], 64, 256, 0);
    if (!c.ok || T == 0 || (D != 64 && D != 128 && D != 256) || tab->dim() != 2 || tab->numel() == 0) Py_RETURN_NONE;
    KvqPagedReadArgs p{};
    Cache ch;
    if (!cache(ch, p.k, p.v, D, k, v, ks, vs, kz, vz)) Py_RETURN_NONE;
    const int64_t B = tab->size(0);
    if (B > INT_MAX || !table(p.pages, tab, B, ch)) Py_RETURN_NONE;
    if ((start && !lengths(start, B)) || (lens && !lengths(lens, B))) Py_RETURN_NONE;
    p.start_pos = (const int32_t*)start.ptr(), p.lens = (const int32_t*)lens.ptr();
    p.format = ch.format, p.B = (int32_t)B, p.Hkv = (int32_t)ch.heads, p.T = (int32_t)T, p.D = (int32_t)D, p.group_size = ch.group;
    c10::cuda::CUDAGuard guard(c.dev);
    at::Tensor kout = empty({B, ch.heads, T, D}, at::kHalf, c.dev), vout = empty({B, ch.heads, T, D}, at::kHalf, c.dev);
    p.k_out = kout.data_ptr(), p.v_out = vout.data_ptr();
    p.out_stride_t = D, p.out_stride_h = T * D, p.out_stride_b = ch.heads * T * D;
    if (!launch("kvq_paged_read", [&] { return lib.paged_read(&p, stream_of(c.dev)); })) return nullptr;
    PyObject* r = PyTuple_New(2);
    if (!r) return nullptr;
    PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(std::move(kout)));
    PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(std::move(vout)));
    return r;
}

// evict(weights, positions, lengths, seen, budget, buffers (a tuple), sinks, recent) -> new lengths
PyObject* evict(PyObject* const* o, Py_ssize_t n) {
    if (n != 8 || !PyTuple_CheckExact(o[5])) Py_RETURN_NONE;
    Call c;
    const Arg w = c.need(o[0]), pos = c.need(o[1]), len = c.need(o[2]), seen = c.need(o[3]);
    const long long budget = c.integer(o[4], 1, INT_MAX, 0), sinks = c.integer(o[6], 0, INT_MAX, -1),
                    recent = c.integer(o[7], 0, INT_MAX, -1);
    const Py_ssize_t nb = PyTuple_GET_SIZE(o[5]);
    if (!c.ok || budget < 1 || sinks < 0 || recent < 0 || sinks + recent > budget || nb > KVQ_EVICT_MAX_BUFS) Py_RETURN_NONE;
    if (!w.is(at::kFloat) || w->dim() != 3 || w->numel() == 0 || !pos.is(at::kInt) || pos->sizes() != w->sizes()) Py_RETURN_NONE;
    if (!slot_rows(w) || !slot_rows(pos)) Py_RETURN_NONE;
    const int64_t B = w->size(0), H = w->size(1), cap = w->size(2);
    if (B > INT_MAX || H > INT_MAX || cap > INT_MAX || !lengths(len, B) || !lengths(seen, B)) Py_RETURN_NONE;
    KvqEvictArgs e{};
    for (Py_ssize_t i = 0; i < nb; ++i) {
        const Arg t = c.need(PyTuple_GET_ITEM(o[5], i));
        if (!c.ok || t->dim() < 3 || t->size(0) != B || t->size(1) != H || t->size(2) < cap) Py_RETURN_NONE;
        int64_t row = 1;
        for (int64_t d = t->dim() - 1; d > 2; --d) {
            if (t->size(d) > 1 && t->stride(d) != row) Py_RETURN_NONE;
            row *= t->size(d);
        }
        if (row == 0) Py_RETURN_NONE;
        for (int d = 0; d < 3; ++d)
            if (t->size(d) > 1 && t->stride(d) < row) Py_RETURN_NONE;
        const int64_t es = t->element_size();
        e.bufs[i] = KvqEvictBuf{t.ptr(), t->stride(0) * es, t->stride(1) * es, t->stride(2) * es, row * es};
    }
    c10::cuda::CUDAGuard guard(c.dev);
    at::Tensor made = empty({B}, at::kInt, c.dev);
    e.B = (int32_t)B, e.Hkv = (int32_t)H, e.cap = (int32_t)cap, e.n_bufs = (int32_t)nb;
    e.budget = (int32_t)budget, e.sinks = (int32_t)sinks, e.recent = (int32_t)recent;
    e.lengths = (const int32_t*)len.ptr(), e.seen = (const int32_t*)seen.ptr(), e.new_lengths = (int32_t*)made.data_ptr();
    e.weights = (float*)w.ptr(), e.w_stride_b = w->stride(0), e.w_stride_h = w->stride(1);
    e.positions = (int32_t*)pos.ptr(), e.p_stride_b = pos->stride(0), e.p_stride_h = pos->stride(1);
    const size_t bytes = lib.evict_ws(e.B, e.Hkv, e.cap, e.budget);
    at::Tensor ws = empty({(int64_t)bytes}, at::kByte, c.dev);
    e.workspace = ws.data_ptr(), e.workspace_bytes = bytes;
    if (!launch("kvq_evict", [&] { return lib.evict(&e, stream_of(c.dev)); })) return nullptr;
    return THPVariable_Wrap(std::move(made));
}

// bind(check, address, ...): the entry points of the library that the package has loaded, in the order of Lib
PyObject* bind(PyObject* const* o, Py_ssize_t n) {
    void* f[6];
    if (n != 7) { PyErr_SetString(PyExc_TypeError, "bind takes check and 6 addresses"); return nullptr; }
    for (int i = 0; i < 6; ++i) {
        f[i] = PyLong_AsVoidPtr(o[i + 1]);
        if (PyErr_Occurred()) return nullptr;
    }
    lib = Lib{(decltype(Lib::span_attn))f[0], (decltype(Lib::span_attn_ws))f[1], (decltype(Lib::paged_append))f[2],
              (decltype(Lib::paged_read))f[3], (decltype(Lib::evict))f[4], (decltype(Lib::evict_ws))f[5]};
    Py_XSETREF(check_fn, Py_NewRef(o[0]));
    Py_RETURN_NONE;
}

// No C++ exception (torch's allocator raises them) leaves through the interpreter.
template <PyObject* (*F)(PyObject* const*, Py_ssize_t)>
PyObject* guarded(PyObject*, PyObject* const* o, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    return F(o, n);
    END_HANDLE_TH_ERRORS
}

#define KVQ_METHOD(f) {#f, (PyCFunction)(void (*)(void))guarded<f>, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {KVQ_METHOD(span_attn), KVQ_METHOD(paged_append), KVQ_METHOD(paged_read), KVQ_METHOD(evict),
                         KVQ_METHOD(bind), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_marshal", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__marshal() {
    PyObject* m = PyModule_Create(&module);
    if (!m) return nullptr;
    PyModule_AddIntConstant(m, "SPAN_ATTN", sizeof(KvqSpanAttnArgs));
    PyModule_AddIntConstant(m, "PAGED_APPEND", sizeof(KvqPagedAppendArgs));
    PyModule_AddIntConstant(m, "PAGED_READ", sizeof(KvqPagedReadArgs));
    PyModule_AddIntConstant(m, "EVICT", sizeof(KvqEvictArgs));
    return m;
}
