"""64-bit reference of attention over the visible span of a cache, and the error a kernel may make.

Bounds (u = 2^-24, half a step of fp32; h = 2^-11, half a step of fp16):
 * a logit is an fp32 sum of D products (and, for quantized keys, of one product per group) whose codes carry an offset of
   8 or 128 that is subtracted again; summed in any order, with accumulation that may truncate (a whole step, 2u, per
   addition), it is off by at most 2 (D + 8) u X, X = sm_scale sum_d |q_d| ((|code| + offset) scale + |zp|);
 * e^x turns that into a relative error of a probability; numerator and denominator both carry it, and the exponentials
   and the fp32 sums over tokens add less than 2^-19: eps_p = 4 (D + 8) u X + 2^-19;
 * P and P * scale_v are each rounded to fp16 before the product with V, 2 h relative to A = sum_s p_s (|c s| + |z|)
   (a factor 1 + 2^-4 covers the product of the errors);
 * the output is rounded to fp16: h |out|, or 2^-25 below the normal range.
"""
import math

import torch

U, H = 2.0 ** -24, 2.0 ** -11


def unpack(payload, D):
    """int8 codes of an int8 [.., D] or nibble-packed [.., D/2] payload."""
    if payload.shape[-1] == D:
        return payload.double()
    b = payload.to(torch.int16) & 255
    return torch.stack(((b >> 4) - 8, (b & 15) - 8), -1).flatten(-2).double()


def values(payload, scale, zp, D):
    """(value, |c s| + |z|, (|c| + offset) s + |z|) in 64 bits."""
    if payload.dtype == torch.float16:
        x = payload.double()
        return x, x.abs(), x.abs()
    off = 128.0 if payload.shape[-1] == D else 8.0
    c = unpack(payload, D)
    rep = D // scale.shape[-1]
    s = scale.double().repeat_interleave(rep, -1)
    z = torch.zeros_like(s) if zp is None else zp.double().repeat_interleave(rep, -1)
    return c * s + z, (c * s).abs() + z.abs(), (c.abs() + off) * s.abs() + z.abs()


def visible(n, S, window, sinks):
    t = torch.arange(S)
    ok = t < n
    if window:
        ok &= (t < sinks) | (t >= n - window)
    return ok


def attention(q, k, v, ks, vs, kz, vz, lens, window=0, sinks=0, sm=None, inv_tau=None):
    """Contiguous cache tensors on the CPU -> (out, tolerance, weight sums, their tolerance)."""
    B, Hq, D = q.shape
    Hkv, S = k.shape[1], k.shape[2]
    rep = Hq // Hkv
    sm = 1.0 / math.sqrt(D) if sm is None else sm
    out = torch.zeros(B, Hq, D, dtype=torch.float64)
    tol = torch.full((B, Hq, D), 2.0 ** -25, dtype=torch.float64)
    w = torch.zeros(B, Hkv, S, dtype=torch.float64)
    wtol = torch.zeros(B, Hkv, S, dtype=torch.float64)
    if inv_tau is not None:
        q = q * inv_tau.half().view(1, -1, 1)              # rounded to fp16, as the kernels do
    for b in range(B):
        ok = visible(int(lens[b]), S, window, sinks)
        if not ok.any():
            continue
        for h in range(Hq):
            g = h // rep

            def side(x, sc, z):
                return values(x[b, g][ok], None if sc is None else sc[b, g][ok], None if z is None else z[b, g][ok], D)
            kv, _, kx = side(k, ks, kz)
            vv, va, _ = side(v, vs, vz)
            x = (kv @ q[b, h].double()) * sm
            X = float((kx @ q[b, h].double().abs()).max()) * abs(sm)
            eps = 4 * (D + 8) * U * X + 2.0 ** -19
            p = torch.softmax(x, 0)
            out[b, h] = p @ vv
            A = p @ va
            tol[b, h] += H * out[b, h].abs() + A * (2 * H * (1 + 2.0 ** -4) + eps)
            w[b, g, ok] += p
            wtol[b, g, ok] += p * (eps + (rep + 2) * 2 * U)
    return out, tol, w, wtol


def check(got, ref, tol, what=""):
    got = got.double().cpu()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    over = (got - ref).abs() - tol
    assert (over <= 0).all(), f"{what}: {int((over > 0).sum())} values off by up to {float((got - ref).abs().max()):.3e} " \
                              f"(bound there {float(tol.flatten()[over.argmax()]):.3e})"


def make_cache(shape, D, fmt, gs, gen):
    """Random cache tensors [*, *, *, .] of a format: (payload, scale, zp); scales of the size that N(0, 1) data has."""
    if fmt == "fp16":
        return torch.randn(*shape, D, generator=gen).half(), None, None
    lo, hi, unit = (-127, 128, 3.0 / 127) if fmt.startswith("int8") else (-8, 8, 3.0 / 7)
    c = torch.randint(lo, hi, (*shape, D), generator=gen, dtype=torch.int16)
    s = (torch.rand(*shape, D // gs, generator=gen) + 0.5).mul(unit).half()
    z = torch.randn(*shape, D // gs, generator=gen).mul(0.5).half() if fmt.endswith("z") else None
    if fmt.startswith("int4"):
        u = (c + 8)
        c = ((u[..., 0::2] << 4) | u[..., 1::2])
        c = torch.where(c > 127, c - 256, c)
    return c.to(torch.int8), s, z


def paginate(x, lens, page, pool_pages, table):
    """Scatter contiguous [B, H, S, .] into a pool of NaN- or 0x7f-filled pages along `table`."""
    if x is None:
        return None
    B, Hh, S = x.shape[:3]
    pool = torch.full((pool_pages, Hh, page, x.shape[3]), float("nan") if x.dtype.is_floating_point else 127, dtype=x.dtype)
    for b in range(B):
        for j in range(-(-int(lens[b]) // page)):
            t = x[b, :, j * page:(j + 1) * page]
            pool[int(table[b, j]), :, :t.shape[1]] = t
    return pool


def make_table(lens, page, gen, spare=3, extra_cols=1):
    per = [-(-int(n) // page) for n in lens]
    pool = sum(per) + spare
    order = torch.randperm(pool, generator=gen).to(torch.int32)
    table = torch.full((len(per), max(per + [1]) + extra_cols), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(per):
        table[b, :n] = order[at:at + n]
        at += n
    return pool, table


def evict(weights, positions, lengths, seen, budget, sinks, recent):
    """Plain eviction of one cache: per (b, h) the list (dst, src) of moves, and the new weights / positions / lengths."""
    w, p = weights.clone(), positions.clone()
    moves = {}
    new = lengths.clone()
    for b in range(w.shape[0]):
        n = max(0, min(int(lengths[b]), w.shape[2]))
        new[b] = min(n, budget)
        if n <= budget:
            continue
        for h in range(w.shape[1]):
            where = [int(x) if x >= 0 else int(seen[b]) - n + s for s, x in enumerate(p[b, h, :n].tolist())]

            def key(s):
                x = float(w[b, h, s])
                safe = where[s] < sinks or where[s] >= int(seen[b]) - recent
                return (not safe, -(float("-inf") if x != x else x) if not safe else 0.0, s)
            keep = set(sorted(range(n), key=key)[:budget])
            dst = [s for s in range(budget) if s not in keep]
            src = [s for s in range(budget, n) if s in keep]
            moves[b, h] = (dst, src)
            kept_w = w[b, h].clone()
            for d, s in zip(dst, src):
                kept_w[d] = w[b, h, s]
                where[d] = where[s]
            w[b, h] = kept_w
            w[b, h, budget:n] = 0
            p[b, h, :budget] = torch.tensor(where[:budget], dtype=torch.int32)
            p[b, h, budget:n] = -1
    return w, p, new, moves
