"""Bodies of the decoder-operator tests (tests/test_decoder_ops_emu_cpu.py on the host emulator of the kernels,
tests/test_decoder_ops_gpu.py on the device): every case against a plain implementation in 64 bits.

Tolerances are bounds by arithmetic, per output element.  With e(t) = finfo(t).eps / 2 the largest relative error of one
rounding to t:
  score s = scale q.k in fp32, D products and sums:      |ds| <= (D + 4) e(f32) scale sum_d |q_d k_d|
  probability p = exp(s - max) / sum, n terms:           |dp| / p <= 2 max|ds| + (n + 16) e(f32)
  bf16 probabilities enter products as high + low parts (decode) -> e(bf16)^2, or as one bf16 (training) -> e(bf16)
  the result is rounded to the output type once:         e(t) |result|
and an error of the terms of sum_j p_j v_j is at most that relative error times sum_j p_j |v_j|."""
import math

import pytest
import torch

E32 = torch.finfo(torch.float32).eps / 2
E16 = torch.finfo(torch.bfloat16).eps / 2


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def attention_ref(q, k, v, n, scale=None):
    """q [R,D], k / v [T,D] of one head in their own types, the first n keys visible -> (out [R,D], |dp|/p bound [R,1],
    sum_j p_j |v_j| [R,D]) in 64 bits; n <= 0: all keys alike; no key: zeros"""
    q, k, v = q.double(), k.double(), v.double()
    D = q.shape[1]
    scale = D ** -0.5 if scale is None else scale
    if k.shape[0] == 0:
        return torch.zeros_like(q), torch.zeros(q.shape[0], 1, dtype=torch.float64), torch.zeros_like(q)
    if n <= 0:
        P = torch.full((q.shape[0], k.shape[0]), 1.0 / k.shape[0], dtype=torch.float64)
        ds = torch.zeros(q.shape[0], 1, dtype=torch.float64)
    else:
        k, v = k[:n], v[:n]
        P = torch.softmax(q @ k.t() * scale, dim=1)
        ds = (D + 4) * E32 * abs(scale) * (q.abs() @ k.abs().t()).max(dim=1, keepdim=True).values
    return P @ v, 2 * ds + (k.shape[0] + 16) * E32, P @ v.abs()


def check_close(got, ref, tol, what):
    got = got.detach().double().cpu()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    assert torch.isfinite(got).all(), what
    bad = (got - ref).abs() > tol
    assert not bad.any(), '%s: %d of %d outside, worst %.3g of its tolerance' % (
        what, int(bad.sum()), bad.numel(), float(((got - ref).abs() / tol.clamp(min=1e-300)).max()))


def make_pages(B, need, page, Hkv, D, dtype, dev, gen, layout='heads_first', extra=2):
    """a cache whose unused slots hold NaN, and the pages of the sequences in a random order; table entries behind a
    sequence's pages are -1"""
    total = sum(need) + extra
    order = torch.randperm(total, generator=gen)
    width = max(1, max(need))
    table = torch.full((B, width), -1, dtype=torch.int32)
    at = 0
    for b in range(B):
        table[b, :need[b]] = order[at:at + need[b]].to(torch.int32)
        at += need[b]
    shape = (total, Hkv, page, D) if layout == 'heads_first' else (total, page, Hkv, D)
    pages = []
    for _ in range(2):
        x = torch.full(shape, float('nan'), dtype=dtype)
        pages.append(x if layout == 'heads_first' else x.transpose(1, 2))
    return pages[0], pages[1], table


def put(pages, table, b, j, page, x):
    pages[int(table[b, j // page]), :, j % page] = x


def paged_case(ops, dev, dtype, B, H, Hkv, D, page, lens, append, layout='heads_first', seed=0, q_std=2.0, scale=None):
    gen = torch.Generator().manual_seed(seed)
    need = [(max(n, 0) + (1 if append and n >= 0 else 0) + page - 1) // page for n in lens]
    kp, vp, table = make_pages(B, need, page, Hkv, D, dtype, dev, gen, layout)
    keys = [torch.randn(max(n, 0), Hkv, D, generator=gen).to(dtype) for n in lens]
    vals = [torch.randn(max(n, 0), Hkv, D, generator=gen).to(dtype) for n in lens]
    for b in range(B):
        for j in range(max(lens[b], 0)):
            put(kp, table, b, j, page, keys[b][j])
            put(vp, table, b, j, page, vals[b][j])
    q = (torch.randn(B, H, D, generator=gen) * q_std).to(dtype)
    kn, vn = torch.randn(B, Hkv, D, generator=gen).to(dtype), torch.randn(B, Hkv, D, generator=gen).to(dtype)
    want_k, want_v = kp.clone(), vp.clone()
    kpd, vpd = kp.to(dev), vp.to(dev)
    if layout != 'heads_first':       # (the transposed storage must survive the move)
        kpd, vpd = kp.transpose(1, 2).contiguous().to(dev).transpose(1, 2), vp.transpose(1, 2).contiguous().to(dev).transpose(1, 2)
    out = ops.paged_attention(q.to(dev), kpd, vpd, table.to(dev), torch.tensor(lens, dtype=torch.int32).to(dev),
                              k_new=kn.to(dev) if append else None, v_new=vn.to(dev) if append else None, scale=scale)
    assert out.dtype == dtype
    G = H // Hkv
    for b in range(B):
        K, V = keys[b], vals[b]
        if append and lens[b] >= 0:
            K, V = torch.cat([K, kn[b:b + 1]]), torch.cat([V, vn[b:b + 1]])
            put(want_k, table, b, lens[b], page, kn[b])
            put(want_v, table, b, lens[b], page, vn[b])
        for h in range(Hkv):
            ref, dp, av = attention_ref(q[b, h * G:(h + 1) * G], K[:, h], V[:, h], K.shape[0], scale)
            split = E16 * E16 if dtype == torch.bfloat16 else 0.0
            check_close(out[b, h * G:(h + 1) * G], ref, half_step(dtype) * ref.abs() + (dp + split) * av * (1 + half_step(dtype)),
                        'b=%d head group %d' % (b, h))
    # the cache: the new tokens and nothing else (NaN slots stay NaN)
    for got, want in ((kpd, want_k), (vpd, want_v)):
        assert torch.equal(torch.nan_to_num(got.cpu().float(), nan=-77.0), torch.nan_to_num(want.float(), nan=-77.0))
    return out


def append_case(ops, dev, src, dtype, B, n, Hkv, D, page, starts, counts, layout='heads_first', seed=0, strided=True):
    gen = torch.Generator().manual_seed(seed)
    need = [(max(s, 0) + c + page - 1) // page if s >= 0 else 0 for s, c in zip(starts, counts)]
    kp, vp, table = make_pages(B, need, page, Hkv, D, dtype, dev, gen, layout)
    kv = torch.randn(B, n, 2, Hkv, D, generator=gen).to(src)
    k, v = kv[:, :, 0], kv[:, :, 1]
    if not strided:
        k, v = k.contiguous(), v.contiguous()
    want_k, want_v = kp.clone(), vp.clone()
    for b in range(B):
        if starts[b] >= 0:
            for t in range(min(n, counts[b])):
                put(want_k, table, b, starts[b] + t, page, k[b, t].to(dtype))
                put(want_v, table, b, starts[b] + t, page, v[b, t].to(dtype))
    if layout == 'heads_first':
        kpd, vpd = kp.to(dev), vp.to(dev)
    else:
        kpd, vpd = (x.transpose(1, 2).contiguous().to(dev).transpose(1, 2) for x in (kp, vp))
    kvd = kv.to(dev)
    kd, vd = (kvd[:, :, 0], kvd[:, :, 1]) if strided else (k.to(dev), v.to(dev))
    ops.paged_append(kd, vd, kpd, vpd, table.to(dev), torch.tensor(starts, dtype=torch.int32).to(dev),
                     torch.tensor(counts, dtype=torch.int32).to(dev))
    for got, want in ((kpd, want_k), (vpd, want_v)):
        assert torch.equal(torch.nan_to_num(got.cpu().float(), nan=-77.0), torch.nan_to_num(want.float(), nan=-77.0))


def sample_ref(x, u, t, k, tp, mp):
    """one row, in Python floats (64 bits), straight from the definition"""
    x = [(-math.inf if math.isnan(v) else v) for v in x.double().tolist()]
    V = len(x)
    order = sorted(range(V), key=lambda i: (-x[i], i))
    top = x[order[0]]
    if not t > 0 or top == -math.inf:
        return order[0]
    k = V if k <= 0 or k > V else k
    w = [1.0 if v == top else (math.exp((v - top) / t) if top != math.inf else 0.0) for v in x]
    kept = order[:k]
    if tp < 1:
        whole, before, n = math.fsum(w[i] for i in kept), [], 0
        acc = 0.0
        for i in kept:
            if n > 0 and not acc < tp * whole:
                break
            acc += w[i]
            n += 1
        kept = kept[:max(n, 1)]
    kept = [kept[0]] + [i for i in kept[1:] if w[i] >= mp]
    kept.sort()
    whole, acc = math.fsum(w[i] for i in kept), 0.0
    for i in kept:
        acc += w[i]
        if acc > u * whole:
            return i
    return max(i for i in kept if w[i] > 0)


def f32(x):
    return torch.tensor(x, dtype=torch.float32).double().item()


def sample_case(ops, dev, x, u, t=1.0, k=0, tp=1.0, mp=0.0):
    """settings: numbers or per-row lists"""
    rows = x.shape[0]

    def per_row(s, as_int=False):
        return [int(v) if as_int else f32(v) for v in (s if isinstance(s, (list, tuple)) else [s] * rows)]

    def arg(s, dt):
        return torch.tensor(s, dtype=dt).to(dev) if isinstance(s, (list, tuple)) else s
    got = ops.sample_rows(x.to(dev), torch.tensor(u, dtype=torch.float32).to(dev), arg(t, torch.float32), arg(k, torch.int32),
                          arg(tp, torch.float32), arg(mp, torch.float32))
    assert got.dtype == torch.int32 and tuple(got.shape) == (rows,)
    T, K, TP, MP, U = per_row(t), per_row(k, True), per_row(tp), per_row(mp), per_row(u)
    want = [sample_ref(x[b], U[b], T[b], K[b], TP[b], MP[b]) for b in range(rows)]
    assert got.cpu().tolist() == want, (got.cpu().tolist(), want)


# what can stay, gathered: (V, settings) where equal logits, the list's size (two entries per thread: 512 up to 1024 logits, 1024
# above) or its bins of several indices are met
SAMPLE_GATHERED = [
    (1000, dict(k=511)), (1000, dict(k=512, tp=.9)), (1000, dict(k=513, tp=.9)), (1000, dict(k=999, tp=.99)),
    (1025, dict(k=1024, tp=.97)), (3000, dict(k=1023, tp=.8)), (3000, dict(k=1024, mp=.02)), (3000, dict(k=1025, tp=.8)),
    (3000, dict(tp=.5)), (3000, dict(tp=.98, t=1.5)), (12000, dict(k=300, tp=.9)), (12000, dict(tp=.6)),
    (40000, dict(k=900, tp=.95, t=2.)), (40000, dict(tp=.3)),
]


def gathered_case(ops, dev, V, kw):
    """normal logits; 400 equal ones within the list before the border's bin (top_p ends among them); one outlier so low
    that all others share a bin"""
    g = torch.Generator().manual_seed(V)
    x = torch.randn(3, V, generator=g) * 2
    at = torch.randperm(V, generator=g)[:400]
    x[1, at] = 7.5
    x[1, at[:3]] = 12.0
    x[2, V // 2] = -1e30
    sample_case(ops, dev, x, [0.03, 0.5, 0.98], **kw)


def cross_ref(q, k, v, dout, klens, dtype, scale=None, keep=None):
    """forward and formula gradients in 64 bits, with a bound for every element.  keep [B,H,Tq,Tk]: dropout factors (0 or
    1 / (1 - p)).  -> {'out': (ref, tol), 'dq': ..., 'dk': ..., 'dv': ...}"""
    q, k, v = q.double(), k.double(), v.double()
    dout = dout.double() if dout is not None else None
    B, Tq, H, D = q.shape
    Tk, Hkv = k.shape[1], k.shape[2]
    G = H // Hkv
    scale = D ** -0.5 if scale is None else scale
    eo = half_step(dtype)
    ep = E16 if dtype == torch.bfloat16 else 0.0          # P, dS as operands of the second products
    z = torch.zeros_like
    out, t_out = z(q), z(q)
    dq, t_dq, dk, t_dk, dv, t_dv = z(q), z(q), z(k), z(k), z(v), z(v)
    for b in range(B):
        n = Tk if klens is None else min(int(klens[b]), Tk)
        uniform = n <= 0
        n = Tk if uniform else n
        for h in range(H):
            g = h // G
            qh, kh, vh = q[b, :, h], k[b, :n, g], v[b, :n, g]
            S = z(qh @ kh.t()) if uniform else qh @ kh.t() * scale
            P = torch.softmax(S, dim=1)
            ds = z(S[:, :1]) if uniform else (D + 4) * E32 * scale * (qh.abs() @ kh.abs().t()).max(1, keepdim=True).values
            dp = 2 * ds + (n + 16) * E32
            kp = keep[b, h, :, :n].double() if keep is not None else torch.ones_like(P)
            Pd = P * kp
            O, aO = Pd @ vh, Pd @ vh.abs()
            out[b, :, h] = O
            t_out[b, :, h] = eo * O.abs() + (dp + ep + 2 * E32) * aO * (1 + eo)
            if dout is None:
                continue
            dO = dout[b, :, h]
            dv[b, :n, g] += Pd.t() @ dO
            t_dv[b, :n, g] += (Pd * (dp + ep + (Tq * G + 16) * E32)).t() @ dO.abs()
            if uniform:
                continue
            dP = (dO @ vh.t()) * kp
            Dv = (P * dP).sum(1, keepdim=True)
            dS = P * (dP - Dv)
            e_dP = (D + 4) * E32 * (dO.abs() @ vh.abs().t()) * kp
            e_D = (dO.abs() * ((dp + ep) * aO + (eo * eo + (D + 4) * E32) * O.abs())).sum(1, keepdim=True)
            e_dS = P * (dp * (dP - Dv).abs() + e_dP + e_D) + (ep + 2 * E32) * dS.abs()
            dq[b, :, h] = scale * (dS @ kh)
            t_dq[b, :, h] = scale * ((e_dS + (n + 16) * E32 * dS.abs()) @ kh.abs())
            dk[b, :n, g] += scale * (dS.t() @ qh)
            t_dk[b, :n, g] += scale * ((e_dS + (Tq * G + 16) * E32 * dS.abs()).t() @ qh.abs())
    r = {'out': (out, t_out)}
    if dout is not None:
        for name, x, t in (('dq', dq, t_dq), ('dk', dk, t_dk), ('dv', dv, t_dv)):
            r[name] = (x, t * (1 + eo) + eo * x.abs())
    return r


def cross_case(ops, dev, dtype, B, H, Hkv, D, Tq, Tk, klens, grad=True, layout='packed', seed=0, scale=None, q_std=2.0,
               poison=True):
    """layout: 'packed' = k and v views of one stacked projection, 'heads' = [B,H,T,d] storage, 'dense'"""
    gen = torch.Generator().manual_seed(seed)
    q = (torch.randn(B, Tq, H, D, generator=gen) * q_std).to(dtype)
    kv = torch.randn(B, Tk, 2, Hkv, D, generator=gen).to(dtype)
    dout = torch.randn(B, Tq, H, D, generator=gen).to(dtype) if grad else None
    ref = cross_ref(q, kv[:, :, 0], kv[:, :, 1], dout, klens, dtype, scale)
    if poison and klens is not None:          # what lies behind an utterance's end: NaN and infinities
        for b in range(B):
            if 0 < klens[b] < Tk:
                kv[b, klens[b]:, 0] = float('nan')
                kv[b, klens[b]:, 1] = float('inf')
    if layout == 'packed':
        kvd, qd = kv.to(dev), q.to(dev)
        kd, vd = kvd[:, :, 0], kvd[:, :, 1]
    elif layout == 'heads':
        qd = q.transpose(1, 2).contiguous().to(dev).transpose(1, 2)
        kd, vd = (kv[:, :, i].transpose(1, 2).contiguous().to(dev).transpose(1, 2) for i in (0, 1))
    else:
        qd, kd, vd = q.to(dev), kv[:, :, 0].contiguous().to(dev), kv[:, :, 1].contiguous().to(dev)
    lens = torch.tensor(klens, dtype=torch.int32).to(dev) if klens is not None else None
    if grad:
        qd, kd, vd = (x.detach().requires_grad_(True) for x in (qd, kd, vd))
    out = ops.cross_attention(qd, kd, vd, lens, scale=scale)
    assert out.dtype == dtype and out.shape == q.shape
    check_close(out, *ref['out'], 'out')
    if grad:
        for name, x in zip(('dq', 'dk', 'dv'), torch.autograd.grad(out, (qd, kd, vd), dout.to(dev))):
            assert x.dtype == dtype
            check_close(x, *ref[name], name)
    return out


def absent_pages_case(ops, dev, dtype, page):
    """entries outside [0, n_pages) inside a sequence: their keys do not count; a new token on such a page or behind the table
    is neither stored nor attended to; a length behind the table counts as the table"""
    gen = torch.Generator().manual_seed(3)
    B, Hkv, D, width = 4, 2, 32, 4
    kp = torch.randn(9, Hkv, page, D, generator=gen).to(dtype)
    vp = torch.randn(9, Hkv, page, D, generator=gen).to(dtype)
    kp[0] = vp[0] = float('nan')                     # what a clamped entry would read
    table = torch.tensor([[3, -1, 4, 5], [99, 2, -7, 6], [-1, -1, -1, -1], [1, 7, 8, 9]], dtype=torch.int32)
    lens = [3 * page - 1, 2 * page, page, 40 * page]
    q = torch.randn(B, Hkv, D, generator=gen).to(dtype)
    kn, vn = torch.randn(B, Hkv, D, generator=gen).to(dtype), torch.randn(B, Hkv, D, generator=gen).to(dtype)
    kd, vd = kp.to(dev), vp.to(dev)
    out = ops.paged_attention(q.to(dev), kd, vd, table.to(dev), torch.tensor(lens, dtype=torch.int32).to(dev), kn.to(dev), vn.to(dev))
    for b in range(B):
        n = min(lens[b], width * page)
        seen = [j for j in range(n) if 0 <= int(table[b, j // page]) < 9]
        new = lens[b] < width * page and 0 <= int(table[b, lens[b] // page]) < 9
        for h in range(Hkv):
            K = [kp[int(table[b, j // page]), h, j % page] for j in seen] + ([kn[b, h]] if new else [])
            V = [vp[int(table[b, j // page]), h, j % page] for j in seen] + ([vn[b, h]] if new else [])
            K = torch.stack(K) if K else torch.zeros(0, D)
            V = torch.stack(V) if V else torch.zeros(0, D)
            ref, dp, av = attention_ref(q[b, h:h + 1], K, V, K.shape[0])
            check_close(out[b, h:h + 1], ref, half_step(dtype) * ref.abs() + (dp + E16 * E16) * av * (1 + half_step(dtype)), 'b=%d' % b)
        if new:
            put(kp, table, b, lens[b], page, kn[b])
            put(vp, table, b, lens[b], page, vn[b])
    for got, want in ((kd, kp), (vd, vp)):
        assert torch.equal(torch.nan_to_num(got.cpu().float(), nan=-77.0), torch.nan_to_num(want.float(), nan=-77.0))


def dropout_case(ops, dev, dtype, B=2, H=2, Tq=7, Tk=70, D=32, p=0.3):
    """the factors are read off with values that are rows of the identity; then out and gradients against 64 bits with them,
    and against the mask AttentionFn draws from the same site"""
    gen = torch.Generator().manual_seed(11)
    klens = [Tk, Tk - 13]
    q, k = torch.randn(B, Tq, H, D, generator=gen), torch.randn(B, Tk, H, D, generator=gen)
    v, dout = torch.randn(B, Tk, H, D, generator=gen), torch.randn(B, Tq, H, D, generator=gen)
    lens = torch.tensor(klens, dtype=torch.int32).to(dev)
    # the mask of this site, from the materialised softmax: q = 0 makes every visible probability 1 / klen
    mode = ops.get_compute_mode()
    ops.set_compute_mode('f32')
    ops.manual_dropout_seed(5)
    keep = torch.zeros(B, H, Tq, Tk)
    for j0 in range(0, Tk, D):
        eye = torch.zeros(B, Tk, H, D)
        for j in range(j0, min(j0 + D, Tk)):
            eye[:, j, :, j - j0] = 1.0
        ops.manual_dropout_seed(5)
        cv, _ = ops.AttentionFn.apply(torch.zeros(B, Tq, H, D).to(dev), None, k.to(dev), eye.to(dev), None, lens,
                                      {'dropout': p, 'training': True})
        cv = cv.detach().cpu().view(B, Tq, H, D)
        for b in range(B):
            keep[b, :, :, j0:j0 + D] = (cv[b] * klens[b]).permute(1, 0, 2)[:, :, :min(D, Tk - j0)]
    ops.set_compute_mode(mode)
    kept = keep > 0.5
    share = float(kept[0].float().mean())
    assert abs(share - (1 - p)) < 0.1, share
    keep = kept.double() / (1 - p)
    q, k, v, dout = (x.to(dtype) for x in (q, k, v, dout))
    ref = cross_ref(q, k, v, dout, klens, dtype, keep=keep)
    qd, kd, vd = (x.to(dev).requires_grad_(True) for x in (q, k, v))
    ops.manual_dropout_seed(5)
    out = ops.cross_attention(qd, kd, vd, lens, dropout_p=p)
    check_close(out, *ref['out'], 'out')
    for name, x in zip(('dq', 'dk', 'dv'), torch.autograd.grad(out, (qd, kd, vd), dout.to(dev))):
        check_close(x, *ref[name], name)


def difference_case(ops, dev):
    """directional derivatives: the kernel's difference quotient against its gradient.  The quotient's own truncation is taken
    from the same quotient in 64 bits; its rounding is at most the outputs' tolerance over the step."""
    gen = torch.Generator().manual_seed(7)
    B, Tq, Tk, H, Hkv, D, h = 2, 6, 37, 4, 2, 16, 2.0 ** -5
    klens = [37, 20]
    lens = torch.tensor(klens, dtype=torch.int32).to(dev)
    x = [torch.randn(B, Tq, H, D, generator=gen), torch.randn(B, Tk, Hkv, D, generator=gen), torch.randn(B, Tk, Hkv, D, generator=gen)]
    d = [torch.randn(t.shape, generator=gen).mul_(64).round_().div_(64) for t in x]
    x = [t.mul_(256).round_().div_(256) for t in x]                 # x +- h d without a rounding
    w = torch.randn(B, Tq, H, D, generator=gen)
    dev_x = [t.clone().to(dev).requires_grad_(True) for t in x]
    grads = torch.autograd.grad(ops.cross_attention(*dev_x, lens), dev_x, w.to(dev))
    g64 = cross_ref(*x, w, klens, torch.float32)
    for i in range(3):
        lo, hi = list(x), list(x)
        lo[i], hi[i] = x[i] - h * d[i], x[i] + h * d[i]
        with torch.enable_grad():
            got = [ops.cross_attention(*[t.clone().to(dev).requires_grad_(True) for t in y], lens).detach().double().cpu() for y in (lo, hi)]
        ref = [cross_ref(*y, None, klens, torch.float32)['out'] for y in (lo, hi)]
        quot = float(((got[1] - got[0]) * w).sum() / (2 * h))
        quot64 = float(((ref[1][0] - ref[0][0]) * w).sum() / (2 * h))
        slope, (r, t) = float((grads[i].double().cpu() * d[i]).sum()), g64[('dq', 'dk', 'dv')[i]]
        slope64 = float((r * d[i]).sum())
        tol = abs(quot64 - slope64) + float(((ref[0][1] + ref[1][1]) * w.abs()).sum()) / (2 * h) + float((t * d[i].abs()).sum())
        assert abs(quot - slope) <= tol, (i, quot, slope, tol)
        assert tol < 0.2 * abs(slope64), (i, tol, slope64)


def backward_case(ops, dev):
    """a second backward pass finds everything as the first one left it, also on saved tensors that hooks laid out anew"""
    g = torch.Generator().manual_seed(3)
    def leaf(B, h, t):      # (a view of [B,h,t,d]: strides that a copy does not keep)
        return torch.randn(B, h, t, 32, generator=g).to(dev).transpose(1, 2).detach().requires_grad_()
    q, k, v = leaf(2, 4, 5), leaf(2, 2, 70), leaf(2, 2, 70)
    klens = torch.tensor([70, 33], dtype=torch.int32).to(dev)
    d1, d2 = (torch.randn(2, 5, 4, 32, generator=g).to(dev) for _ in range(2))
    kept = []

    def pack(t):
        kept.append((t, t.detach().clone()))
        return t
    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
        out = ops.cross_attention(q, k, v, klens, scale=0.25)
    first = torch.autograd.grad(out, (q, k, v), d1, retain_graph=True)
    other = torch.autograd.grad(out, (q, k, v), d2, retain_graph=True)
    again = torch.autograd.grad(out, (q, k, v), d1, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    assert not any(torch.equal(a, b) for a, b in zip(first, other))
    assert kept and all(torch.equal(t, was) for t, was in kept)      # nothing saved is written to
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.contiguous().clone(), lambda t: t):
        out = ops.cross_attention(q, k, v, klens, scale=0.25)
    laid_out = torch.autograd.grad(out, (q, k, v), d1)
    assert all(torch.equal(a, b) for a, b in zip(first, laid_out))
    out = ops.cross_attention(q, k, v, klens)
    with pytest.raises(RuntimeError):
        gq = torch.autograd.grad(out.square().sum(), q, create_graph=True)[0]
        torch.autograd.grad(gq.sum(), k)


def infinite_scores_case(ops, dev, dtype):
    """keys with a score of -inf have no probability, also where they fill the first tiles"""
    g = torch.Generator().manual_seed(8)
    q, k, v = torch.randn(1, 9, 2, 64, generator=g), torch.randn(1, 150, 2, 64, generator=g), torch.randn(1, 150, 2, 64, generator=g)
    q, k, v = (x.to(dtype) for x in (q, k, v))
    q[..., 0] = 1.0
    k[:, :130, :, 0] = float('-inf')
    want = cross_ref(q[:, :, :, :], k[:, 130:], v[:, 130:], None, None, dtype)['out']
    for grad in (True, False):
        check_close(ops.cross_attention(q.to(dev).requires_grad_(grad), k.to(dev), v.to(dev)).detach(), want[0], want[1], 'out')


def infinite_scores_in_the_last_dimension_case(ops, dev, dtype, D):
    """the same for head sizes between the kernels' widths, where the last dimension's chunk borders on what is not there"""
    g = torch.Generator().manual_seed(D)
    q, k, v = torch.randn(1, 70, 2, D, generator=g), torch.randn(1, 150, 1, D, generator=g), torch.randn(1, 150, 1, D, generator=g)
    q, k, v = (x.to(dtype) for x in (q, k, v))
    q[..., -1] = 1.0
    k[:, :130, :, -1] = float('-inf')
    want = cross_ref(q, k[:, 130:], v[:, 130:], None, None, dtype)['out']
    for rows in (70, 3):
        for grad in (True, False):
            out = ops.cross_attention(q[:, :rows].to(dev).requires_grad_(grad), k.to(dev), v.to(dev)).detach()
            check_close(out, want[0][:, :rows], want[1][:, :rows], 'out')


def check_close_but_for_infinities(got, ref, tol, what):
    """infinities where the reference has them, and only there"""
    got, far = got.detach().double().cpu(), torch.isinf(ref)
    assert far.any() and torch.equal(got[far], ref[far]), what
    check_close(got[~far], ref[~far], tol[~far], what)


def infinite_last_row_case(ops, dev, dtype, D, Tq, Tk, klens, train=True):
    """an infinite value in the last visible row of v, and an infinite gradient of the last query: the sums they enter are
    infinite, by the definition"""
    g = torch.Generator().manual_seed(Tk)
    B = len(klens)
    q, k, v, dout = (torch.randn(B, t, 2, D, generator=g).to(dtype) for t in (Tq, Tk, Tk, Tq))
    inf_v, inf_d = v.clone(), dout.clone()
    for b, n in enumerate(klens):
        inf_v[b, n - 1, :, 5] = float('inf')
        inf_d[b, Tq - 1, :, D - 1] = float('-inf')
    lens = torch.tensor(klens, dtype=torch.int32).to(dev)
    ref = cross_ref(q, k, inf_v, None, klens, dtype)['out']
    check_close_but_for_infinities(ops.cross_attention(q.to(dev).requires_grad_(train), k.to(dev), inf_v.to(dev), lens), *ref, 'out')
    if train:
        ref, vd = cross_ref(q, k, v, inf_d, klens, dtype)['dv'], v.to(dev).requires_grad_()
        got = torch.autograd.grad(ops.cross_attention(q.to(dev), k.to(dev), vd, lens), vd, inf_d.to(dev))[0]
        check_close_but_for_infinities(got, *ref, 'dv')


INFINITE_LAST_ROW = [dict(D=64, Tq=70, Tk=150, klens=[150, 33]), dict(D=72, Tq=37, Tk=50, klens=[50]),
                     dict(D=32, Tq=5, Tk=33, klens=[1, 33, 32])]


def infinite_values_paged_case(ops, dev, dtype, D, page, n):
    """infinite values of an inner key and of the last one (behind which a tile is partly empty): the sums they enter are
    infinite, whatever the parts a probability is split into"""
    g = torch.Generator().manual_seed(n)
    width = (n + page - 1) // page
    k, v = (torch.randn(n, 2, D, generator=g).to(dtype) for _ in range(2))
    v[n // 3, :, 1] = float('inf')
    v[n - 1, :, D - 2] = float('-inf')
    kp, vp = (torch.full((width, 2, page, D), float('nan'), dtype=dtype) for _ in range(2))
    table = torch.randperm(width, generator=g).to(torch.int32).view(1, width)
    for j in range(n):
        put(kp, table, 0, j, page, k[j])
        put(vp, table, 0, j, page, v[j])
    q = torch.randn(1, 4, D, generator=g).to(dtype)
    lens = torch.tensor([n], dtype=torch.int32).to(dev)
    paged = ops.paged_attention(q.to(dev), kp.to(dev), vp.to(dev), table.to(dev), lens)[0]
    plain = ops.cross_attention(q.to(dev).unsqueeze(1), k.to(dev).unsqueeze(0), v.to(dev).unsqueeze(0))[0, 0]
    split = E16 * E16 if dtype == torch.bfloat16 else 0.0
    for out in (paged, plain):
        for h in range(2):
            ref, dp, av = attention_ref(q[0, 2 * h:2 * h + 2], k[:, h], v[:, h], n)
            check_close_but_for_infinities(out[2 * h:2 * h + 2], ref, half_step(dtype) * ref.abs() + (dp + split) * av * (1 + half_step(dtype)), h)


INFINITE_VALUES = [dict(D=64, page=16, n=37), dict(D=128, page=64, n=700), dict(D=40, page=7, n=50), dict(D=32, page=16, n=2)]


def no_softmax_case(ops, dev, dtype, Tk):
    """every score of a row -inf: NaN in both forms, and only there"""
    g = torch.Generator().manual_seed(Tk)
    q, k, v = (torch.randn(2, t, 2, 32, generator=g).to(dtype) for t in (3, Tk, Tk))
    q[:, :, :, 0] = 1.0
    k[1, :, 1, 0] = float('-inf')
    for grad in (True, False):
        out = ops.cross_attention(q.to(dev).requires_grad_(grad), k.to(dev), v.to(dev)).detach().cpu()
        assert out[1, :, 1].isnan().all()
        assert torch.isfinite(out[0]).all() and torch.isfinite(out[1, :, 0]).all()


def nan_among_minus_infinities_case(ops, dev, V):
    """a NaN counts as -inf, also against -inf: rows without a larger logit give their first entry, others are not disturbed"""
    inf, nan = float('inf'), float('nan')
    x = torch.full((5, V), -inf)
    x[0, 0] = nan
    x[1, 1:] = nan
    x[2, ::2] = nan
    x[3, V - 1] = nan
    x[4, ::2] = nan
    x[4, V - 2:] = 1.0
    for kw in (dict(), dict(t=0.0), dict(k=2), dict(tp=0.9), dict(k=V - 1, tp=0.5)):
        sample_case(ops, dev, x, [0.0, 0.3, 0.5, 0.7, 0.9], **kw)


def forward_mode_case(ops, dev, tokens, dropout_p=0.0):
    """dual tensors are refused, whichever kernel would take the call; duals of another level's end and plain tensors are not"""
    import torch.autograd.forward_ad as fw
    x = [torch.ones(1, t, 2, 16).to(dev) for t in (tokens, 9, 9)]
    with fw.dual_level():
        for i in range(3):
            y = list(x)
            y[i] = fw.make_dual(y[i], torch.ones_like(y[i]))
            with pytest.raises(NotImplementedError):
                ops.cross_attention(*y, dropout_p=dropout_p)
        assert ops.cross_attention(*x, dropout_p=dropout_p).shape == x[0].shape
    assert ops.cross_attention(*y, dropout_p=dropout_p).shape == x[0].shape


def no_backward_case(ops, dev):
    """paged_attention under autograd: the same values, and an error where a gradient would get lost"""
    import torch.autograd.forward_ad as fw
    g = torch.Generator().manual_seed(2)
    q, kn, vn = (torch.randn(2, 2, 16, generator=g).to(dev) for _ in range(3))
    kp, vp = (torch.randn(3, 2, 4, 16, generator=g).to(dev) for _ in range(2))
    table, lens = torch.tensor([[0], [2]], dtype=torch.int32).to(dev), torch.tensor([3, 0], dtype=torch.int32).to(dev)
    want = ops.paged_attention(q, kp, vp, table, lens, kn, vn)
    assert not want.requires_grad
    w = torch.ones(16, 16, device=dev, requires_grad=True)
    for i in range(3):
        y = [q, kn, vn]
        y[i] = y[i].clone().requires_grad_()
        out = ops.paged_attention(y[0], kp, vp, table, lens, y[1], y[2])
        assert torch.equal(out, want)
        assert torch.autograd.grad((out.detach() @ w).sum(), w)[0].shape == w.shape
        with pytest.raises(NotImplementedError, match='paged_attention'):
            out.sum().backward()
        with torch.no_grad():
            assert not ops.paged_attention(y[0], kp, vp, table, lens, y[1], y[2]).requires_grad
    out = ops.paged_attention(q.clone().requires_grad_(), kp, vp, table[:, :0], lens)      # no key: zeros
    with pytest.raises(NotImplementedError, match='paged_attention'):
        out.sum().backward()
    with fw.dual_level(), pytest.raises(NotImplementedError):
        ops.paged_attention(fw.make_dual(q, q), kp, vp, table, lens)


def overwritten_pages_case(ops, dev):
    """autograd notices that pages changed behind its back; pages of its own are not written to"""
    q = torch.ones(1, 1, 8).to(dev)
    table, lens = torch.zeros(1, 1, dtype=torch.int32).to(dev), torch.zeros(1, dtype=torch.int32).to(dev)

    def attend(kp, vp):
        ops.paged_attention(q, kp, vp, table, lens, q, q)

    def append(kp, vp):
        ops.paged_append(q.unsqueeze(1), q.unsqueeze(1), kp, vp, table, lens)
    for write in (attend, append):
        both = torch.zeros(2, 1, 1, 4, 8).to(dev)
        for i in range(2):
            w = torch.ones(8, device=dev, requires_grad=True)
            loss = (both[i] * w).sum()                    # saves the pages
            write(both[0], both[1])
            with pytest.raises(RuntimeError, match='modified by an inplace operation'):
                loss.backward()
        own = both[0].clone().requires_grad_()
        with pytest.raises(ValueError):
            write(own, both[1])
        with torch.no_grad():
            write(own, both[1])
        with torch.inference_mode():                      # (tensors without a version)
            write(torch.zeros(1, 1, 4, 8).to(dev), torch.zeros(1, 1, 4, 8).to(dev))
    kp = torch.zeros(1, 1, 4, 8).to(dev)
    ops.paged_attention(q, kp, kp, table, lens)
    assert kp._version == 0                               # reading is no change


def far_tokens_case(ops, dev):
    """tokens 2^24 elements and more apart, and a single token whose stride means nothing: the results of dense tensors"""
    g = torch.Generator().manual_seed(4)
    far = 1 << 24

    def apart(x, step):
        n = (x.shape[1] - 1) * step + x.shape[2] * x.shape[3]
        return torch.zeros(n, dtype=x.dtype, device=dev).as_strided(x.shape, (8, step, x.shape[3], 1)).copy_(x)

    def run(q, k, v, dout):
        q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
        out = ops.cross_attention(q, k, v)
        return [out.detach()] + list(torch.autograd.grad(out, (q, k, v), dout))
    for Tq, steps in ((2, (far, 64, 64, 64)), (2, (64, far + 8, far, 64)), (2, (64, 64, 64, far)), (1, (3 * far, 64, 64, 3 * far))):
        x = [torch.randn(1, t, 4, 16, generator=g).to(torch.bfloat16) for t in (Tq, 2, 2, Tq)]
        want = run(*(t.to(dev) for t in x))
        assert all(torch.equal(a, b) for a, b in zip(run(*(apart(t, s) for t, s in zip(x, steps))), want))
        # (the single-token form reads them as they are)
        assert torch.equal(ops.cross_attention(x[0].to(dev), apart(x[1], far), apart(x[2], far)),
                           ops.cross_attention(*(t.to(dev) for t in x[:3])))


def many_pages_case(ops, dev, page):
    """a cache of more pages than 31 or 32 bits count (one page, expanded): its pages are there, negative entries are not"""
    g = torch.Generator().manual_seed(5)
    k, v = (torch.randn(1, 1, page, 32, generator=g).to(dev) for _ in range(2))
    q = torch.randn(3, 1, 32, generator=g)
    table = torch.tensor([[7, 2 ** 31 - 1], [-1, -2 ** 31], [0, -5]], dtype=torch.int32)
    lens = [2 * page, 2 * page, 2 * page - 1]
    for n_pages in (2 ** 31, 2 ** 31 + 5, 2 ** 32 + 1):
        out = ops.paged_attention(q.to(dev), k.expand(n_pages, 1, page, 32), v.expand(n_pages, 1, page, 32), table.to(dev),
                                  torch.tensor(lens, dtype=torch.int32).to(dev))
        ref, dp, av = attention_ref(torch.cat([q[0], q[2]]), k[0, 0].cpu(), v[0, 0].cpu(), page)      # (a key twice: the same softmax)
        dp = dp + page * E32
        check_close(torch.stack([out[0, 0], out[2, 0]]), ref, E32 * ref.abs() + dp * av * (1 + E32), n_pages)
        assert not out[1].any()


def dropout_widths_case(ops, dev, dtype, B, H, Hkv, Tq, Tk, D, klens, p=0.25, seed=6):
    """dropout at every width of the kernels, odd lengths over several tiles of either side, shared heads: the factors are those
    that the training softmax draws from the same site (q = 0: every visible probability is 1 / klen), read off with values that
    are rows of the identity"""
    gen = torch.Generator().manual_seed(D)
    lens = torch.tensor(klens, dtype=torch.int32).to(dev)
    mode, W = ops.get_compute_mode(), 64
    ops.set_compute_mode('f32')
    keep = torch.zeros(B, H, Tq, Tk)
    for j0 in range(0, Tk, W):
        n = min(W, Tk - j0)
        eye = torch.zeros(B, Tk, H, W)
        eye[:, range(j0, j0 + n), :, range(n)] = 1.0
        ops.manual_dropout_seed(seed)
        cv, _ = ops.AttentionFn.apply(torch.zeros(B, Tq, H, W).to(dev), None, torch.zeros(B, Tk, H, W).to(dev), eye.to(dev), None, lens,
                                      {'dropout': p, 'training': True})
        cv = cv.detach().cpu().view(B, Tq, H, W)
        for b in range(B):
            keep[b, :, :, j0:j0 + n] = (cv[b] * klens[b]).permute(1, 0, 2)[:, :, :n]
    ops.set_compute_mode(mode)
    keep = (keep > 0.5).double() / (1 - p)
    q, k, v, dout = (torch.randn(B, t, h, D, generator=gen).to(dtype) for t, h in ((Tq, H), (Tk, Hkv), (Tk, Hkv), (Tq, H)))
    ref = cross_ref(q, k, v, dout, klens, dtype, keep=keep)
    qd, kd, vd = (x.to(dev).requires_grad_(True) for x in (q, k, v))
    ops.manual_dropout_seed(seed)
    out = ops.cross_attention(qd, kd, vd, lens, dropout_p=p)
    check_close(out, *ref['out'], 'out')
    for name, x in zip(('dq', 'dk', 'dv'), torch.autograd.grad(out, (qd, kd, vd), dout.to(dev))):
        check_close(x, *ref[name], name)


DROPOUT_WIDTHS = [dict(B=2, H=2, Hkv=2, Tq=67, Tk=201, D=64, klens=[201, 139]), dict(B=1, H=4, Hkv=2, Tq=131, Tk=67, D=32, klens=[66]),
                  dict(B=1, H=2, Hkv=1, Tq=67, Tk=203, D=128, klens=[203]), dict(B=1, H=2, Hkv=2, Tq=5, Tk=71, D=72, klens=[70]),
                  dict(B=2, H=3, Hkv=1, Tq=70, Tk=69, D=64, klens=[1, 69])]


# the kernels for rows that LDS holds with their masses, without them, and not at all, with and without settings
SAMPLE_WIDE = [(V, kw) for V in (9000, 12000, 31000) for kw in (dict(), dict(tp=.9), dict(k=40, t=.7), dict(mp=.05))]


def wide_case(ops, dev, dtype, V, kw):
    x = torch.randn(2, V + 1, generator=torch.Generator().manual_seed(V)).mul_(3).to(dtype)[:, 1:]
    sample_case(ops, dev, x, [0.25, 0.75], **kw)
