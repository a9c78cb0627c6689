"""Cases that measure the decoder operators of neural_sp_amd.ops: attention of target tokens over encoder states of
another length (forward and backward, and one token at a time), attention of one new token over a paged key / value cache
with and without the append, the append of a whole prompt, and sampling from given random numbers.

`run` computes an operator in its plain form (elementary torch operations, 32 bits, 64 where a border is compared) unless
the module's `own` is true: then it makes the calls a user of the package makes.
"""
import math

import torch

own = False

DTYPE = {'bf16': torch.bfloat16, 'f32': torch.float32}
BYTES = {'bf16': 2, 'f32': 4}
FLT_MAX = torch.finfo(torch.float32).max


# ------------------------------------------------------------------------------------------------ cases
def _cross(name, dtype, B, H, Hkv, D, Tq, Tk, kmin, grad):
    return dict(name=name, op='cross', dtype=dtype, B=B, H=H, Hkv=Hkv, D=D, Tq=Tq, Tk=Tk, kmin=kmin, grad=grad)


def _paged(name, dtype, B, H, Hkv, D, page, lmin, lmax, append):
    return dict(name=name, op='paged', dtype=dtype, B=B, H=H, Hkv=Hkv, D=D, page=page, lmin=lmin, lmax=lmax,
                append=append)


def _append(name, src, dtype, B, Hkv, D, page, n, nmin, start):
    return dict(name=name, op='append', src=src, dtype=dtype, B=B, Hkv=Hkv, D=D, page=page, n=n, nmin=nmin, start=start)


def _sample(name, dtype, B, V, temperature, top_k, top_p, min_p, per_row):
    return dict(name=name, op='sample', dtype=dtype, B=B, V=V, temperature=temperature, top_k=top_k, top_p=top_p,
                min_p=min_p, per_row=per_row)


def listed():
    return [
        # a training step's source attention: 32 utterances of a Transformer decoder with d_model 512, word pieces against
        # encoder frames after 8-fold subsampling
        _cross('cross train', 'bf16', 32, 8, 8, 64, 61, 187, 90, True),
        # the same in the fp32 parity mode, the 256-wide decoder, odd lengths, one utterance without a valid frame
        _cross('cross train fp32', 'f32', 8, 4, 4, 64, 45, 301, 0, True),
        # long utterances and character targets at 128 utterances per GPU: the largest training call
        _cross('cross train large', 'bf16', 128, 8, 8, 64, 256, 800, 600, True),
        # wide shared heads (four query heads on each key head) over long states
        _cross('cross train shared', 'bf16', 4, 16, 4, 128, 500, 2048, 1111, True),
        # one step of decoding a single utterance: latency
        _cross('cross token', 'bf16', 1, 4, 4, 64, 1, 200, 200, False),
        # one step of decoding a batch of long utterances
        _cross('cross token batch', 'bf16', 64, 8, 8, 64, 1, 1500, 700, False),
        # one step of decoding a single utterance over its own prefix: append and attend, latency
        _paged('paged token', 'bf16', 1, 4, 4, 64, 16, 37, 37, True),
        # fp32 parity mode, ragged prefixes, one of them empty before the append
        _paged('paged token fp32', 'f32', 16, 4, 4, 64, 16, 0, 333, True),
        # many long prefixes with shared heads: the largest serving call
        _paged('paged long shared', 'bf16', 16, 32, 8, 128, 64, 9000, 32000, True),
        # a batch's prompts into the cache: fp32 projections rounded to the cache's bf16
        _append('append prompts', 'f32', 'bf16', 32, 8, 64, 16, 300, 40, 0),
        # sampling one utterance's next word piece, latency
        _sample('sample one', 'f32', 1, 1000, 0.8, 20, 0.95, 0.0, False),
        # sampling for a whole batch over a large vocabulary, every row with its own settings
        _sample('sample batch', 'f32', 256, 10000, 1.0, 500, 0.9, 0.01, True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))


def draw(rng):
    op = rng.choice(['cross', 'cross', 'token', 'paged', 'paged', 'append', 'sample', 'sample'])
    dtype = rng.choice(['bf16', 'bf16', 'f32'])
    if op in ('cross', 'token'):
        D = rng.choice([32, 64, 64, 72, 128])
        Hkv = rng.choice([1, 2, 4, 8])
        H = Hkv * rng.choice([1, 1, 1, 2, 4])
        if op == 'token':
            c = _cross('', dtype, _log(rng, 1, 128), H, Hkv, D, rng.choice([1, 1, 1, 2, 5]), _log(rng, 1, 4000), 0, False)
        else:
            c = _cross('', dtype, _log(rng, 1, 64), H, Hkv, D, _log(rng, 2, 700), _log(rng, 1, 2500), 0, True)
        c['kmin'] = rng.choice([0, c['Tk'] // 2, c['Tk']])
        most = 3e9 if dtype == 'bf16' else 5e8          # score elements x head size: stay below the largest listed call
        while c['B'] > 1 and c['B'] * c['H'] * c['Tq'] * c['Tk'] * c['D'] > most:
            c['B'] = (c['B'] + 1) // 2
        while c['Tq'] > 2 and c['B'] * c['H'] * c['Tq'] * c['Tk'] * c['D'] > most:
            c['Tq'] = (c['Tq'] + 1) // 2
    elif op == 'paged':
        Hkv = rng.choice([1, 2, 4, 8])
        c = _paged('', dtype, _log(rng, 1, 128), Hkv * rng.choice([1, 1, 2, 4, 7]), Hkv, rng.choice([32, 64, 64, 72, 128]),
                   rng.choice([8, 16, 16, 32, 64, 100]), 0, _log(rng, 1, 20000), rng.choice([True, False]))
        while c['B'] > 1 and c['B'] * c['Hkv'] * c['lmax'] * c['D'] > 2e8:
            c['B'] = (c['B'] + 1) // 2
        c['lmin'] = rng.choice([0, c['lmax'] // 3, c['lmax']])
    elif op == 'append':
        n = _log(rng, 1, 2000)
        c = _append('', rng.choice(['f32', dtype]), dtype, _log(rng, 1, 64), rng.choice([1, 2, 4, 8]),
                    rng.choice([32, 64, 64, 72, 128]), rng.choice([8, 16, 16, 32, 64, 100]), n,
                    rng.choice([0, n // 2, n]), rng.choice([0, 0, _log(rng, 1, 500)]))
    else:
        V = _log(rng, 20, 50000)
        c = _sample('', dtype, _log(rng, 1, 256), V, rng.choice([0.0, 0.5, 0.7, 1.0, 1.3]),
                    rng.choice([0, 1, 10, 50, V // 3, V]), rng.choice([1.0, 0.95, 0.9, 0.5]),
                    rng.choice([0.0, 0.0, 0.02, 0.1]), rng.choice([True, False]))
    del c['name']
    return c


# ------------------------------------------------------------------------------------------------ inputs
def _spread(lo, hi, n, gen):
    """n whole numbers spread evenly over lo..hi (their sum does not depend on the seed), in an order of the seed's."""
    x = torch.tensor([lo + (hi - lo) * i // max(1, n - 1) for i in range(n)] if n > 1 else [hi], dtype=torch.int32)
    return x[torch.randperm(n, generator=gen)]


def _sum_spread(lo, hi, n):
    return sum(lo + (hi - lo) * i // max(1, n - 1) for i in range(n)) if n > 1 else hi


def _pages(c, lens, gen, dev):
    """A cache of one layer that has served other sequences before: the pages of a sequence lie anywhere, entries behind a
    sequence's last page are -1."""
    B, page = c['B'], c['page']
    need = [(int(n) + page - 1) // page for n in lens]
    width = max(1, max(need))
    n_pages = sum(need) + 3
    order = torch.randperm(n_pages, generator=gen).to(torch.int32)
    table = torch.full((B, width), -1, dtype=torch.int32)
    at = 0
    for b in range(B):
        table[b, :need[b]] = order[at:at + need[b]]
        at += need[b]
    return n_pages, table.to(dev)


def prepare(case, seed):
    c = case
    dev = torch.device('cuda')
    gen = torch.Generator().manual_seed(int(seed))
    dgen = torch.Generator(device=dev).manual_seed(int(seed))
    dt = DTYPE[c['dtype']]

    def randn(*shape, std=1.0, dtype=dt):
        return (torch.randn(shape, device=dev, dtype=torch.float32, generator=dgen) * std).to(dtype)

    if c['op'] == 'cross':
        s = dict(case=c, q=randn(c['B'], c['Tq'], c['H'], c['D'], std=2.0))
        # keys and values leave one stacked projection side by side, as a decoder layer makes them
        kv = randn(c['B'], c['Tk'], 2, c['Hkv'], c['D'])
        s['k'], s['v'] = kv[:, :, 0], kv[:, :, 1]
        s['klens'] = _spread(c['kmin'], c['Tk'], c['B'], gen).to(dev)
        if c['grad']:
            s['dout'] = randn(c['B'], c['Tq'], c['H'], c['D'])
        return s
    if c['op'] == 'paged':
        # lengths before the append; with it every sequence has one key more
        lens = _spread(c['lmin'], c['lmax'], c['B'], gen)
        n_pages, table = _pages(c, lens + 1, gen, dev)
        shape = (n_pages, c['Hkv'], c['page'], c['D'])
        s = dict(case=c, table=table, lens=lens.to(dev), q=randn(c['B'], c['H'], c['D'], std=2.0))
        s['k_pages'] = torch.randn(shape, device=dev, dtype=dt, generator=dgen)
        s['v_pages'] = torch.randn(shape, device=dev, dtype=dt, generator=dgen)
        s['k_new'], s['v_new'] = randn(c['B'], c['Hkv'], c['D']), randn(c['B'], c['Hkv'], c['D'])
        return s
    if c['op'] == 'append':
        counts = _spread(c['nmin'], c['n'], c['B'], gen)
        n_pages, table = _pages(c, counts + c['start'], gen, dev)
        shape = (n_pages, c['Hkv'], c['page'], c['D'])
        kv = randn(c['B'], c['n'], 2, c['Hkv'], c['D'], dtype=DTYPE[c['src']])
        return dict(case=c, table=table, counts=counts.to(dev), k=kv[:, :, 0], v=kv[:, :, 1],
                    starts=torch.full((c['B'],), c['start'], dtype=torch.int32, device=dev),
                    k_pages=torch.zeros(shape, device=dev, dtype=dt), v_pages=torch.zeros(shape, device=dev, dtype=dt))
    s = dict(case=c, logits=randn(c['B'], c['V'], std=3.0),
             u=torch.rand((c['B'],), device=dev, dtype=torch.float32, generator=dgen))
    s['temperature'], s['top_k'], s['top_p'], s['min_p'] = c['temperature'], c['top_k'], c['top_p'], c['min_p']
    if c['per_row']:
        # requests of one batch with settings of their own, around the case's
        f = torch.linspace(0.5, 1.0, c['B'], device=dev)
        s['temperature'] = c['temperature'] * (0.5 + f)
        s['top_k'] = (c['top_k'] * f).to(torch.int32)
        s['top_p'] = 1.0 - (1.0 - c['top_p']) * f
        s['min_p'] = c['min_p'] * f
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _cross_plain(q, k, v, klens):
    B, Tq, H, D = q.shape
    Tk, Hkv = k.shape[1], k.shape[2]
    qf = q.float().view(B, Tq, Hkv, H // Hkv, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, (H // Hkv) * Tq, D)
    kf, vf = k.float().permute(0, 2, 3, 1), v.float().permute(0, 2, 1, 3)
    s = torch.matmul(qf, kf.contiguous()) * (1.0 / math.sqrt(D))
    hidden = torch.arange(Tk, device=q.device).view(1, 1, 1, Tk) >= klens.view(B, 1, 1, 1)
    s = s.masked_fill(hidden, -FLT_MAX)                       # a row without a visible key: all keys alike
    e = torch.exp(s - s.max(dim=-1, keepdim=True).values)
    p = e / e.sum(dim=-1, keepdim=True)
    o = torch.matmul(p, vf.contiguous()).view(B, Hkv, H // Hkv, Tq, D).permute(0, 3, 1, 2, 4).reshape(B, Tq, H, D)
    return o.to(q.dtype)


def _write_plain(pages, table, pos, row, x):
    """pages[table[row, pos // page], :, pos % page] = x, token by token"""
    page = pages.shape[2]
    pages[table[row, pos // page].long(), :, (pos % page).long()] = x.to(pages.dtype)


def _paged_plain(q, k_pages, v_pages, table, lens, k_new=None, v_new=None):
    B, H, D = q.shape
    Hkv, page = k_pages.shape[1], k_pages.shape[2]
    if k_new is not None:
        row = torch.arange(B, device=q.device)
        _write_plain(k_pages, table, lens, row, k_new)
        _write_plain(v_pages, table, lens, row, v_new)
        lens = lens + 1
    idx = table.clamp(min=0).long()
    L = table.shape[1] * page
    kf = k_pages[idx].float().permute(0, 2, 1, 3, 4).reshape(B, Hkv, L, D)
    vf = v_pages[idx].float().permute(0, 2, 1, 3, 4).reshape(B, Hkv, L, D)
    s = torch.matmul(q.float().view(B, Hkv, H // Hkv, D), kf.transpose(2, 3)) * (1.0 / math.sqrt(D))
    seen = torch.arange(L, device=q.device).view(1, 1, 1, L) < lens.view(B, 1, 1, 1)
    s = s.masked_fill(~seen, -FLT_MAX)
    e = torch.exp(s - s.max(dim=-1, keepdim=True).values) * seen
    o = torch.matmul(e, vf.masked_fill(~seen.view(B, 1, L, 1), 0.0)) / e.sum(dim=-1, keepdim=True).clamp(min=1e-30)
    return o.view(B, H, D).to(q.dtype)                        # no key at all: zeros


def _append_plain(k, v, k_pages, v_pages, table, starts, counts):
    n = k.shape[1]
    row, t = torch.nonzero(torch.arange(n, device=k.device).view(1, n) < counts.view(-1, 1), as_tuple=True)
    pos = starts[row] + t
    _write_plain(k_pages, table, pos, row, k[row, t])
    _write_plain(v_pages, table, pos, row, v[row, t])


def _setting(x, like):
    return torch.as_tensor(x, device=like.device).to(torch.float32).double().expand(like.shape[0]).unsqueeze(1)


def _sample_plain(logits, u, temperature, top_k, top_p, min_p):
    """the order is by falling logit, the lower index first among equals; what is kept is its first entries: at most top_k, up
    to the one whose mass completes top_p of theirs, none below min_p of the largest.  The token is the first kept index
    whose mass with all kept indices before it exceeds u of the whole."""
    B, V = logits.shape
    t, tp, mp = _setting(temperature, u), _setting(top_p, u), _setting(min_p, u)
    k = torch.as_tensor(top_k, device=u.device).to(torch.int64).expand(B).unsqueeze(1)
    k = torch.where((k <= 0) | (k > V), torch.full_like(k, V), k)
    k = torch.where(t <= 0, torch.ones_like(k), k)            # temperature 0: the largest logit
    z, order = torch.sort(logits.double(), dim=1, descending=True, stable=True)
    w = torch.exp((z - z[:, :1]) / torch.where(t <= 0, torch.ones_like(t), t))
    first = torch.arange(V, device=u.device).unsqueeze(0) < k
    w = w * first
    before = torch.cumsum(w, dim=1) - w
    keep = first & ((before < tp * w.sum(dim=1, keepdim=True)) | (tp >= 1)) & (w >= mp)
    keep[:, 0] = True
    mass = torch.zeros_like(w).scatter_(1, order, w * keep)   # by index again
    cum = torch.cumsum(mass, dim=1)
    hit = (cum > u.double().unsqueeze(1) * cum[:, -1:]) & (mass > 0)
    return torch.argmax(hit.to(torch.int8), dim=1).to(torch.int32)


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    s = state
    c = s['case']
    if own:
        from neural_sp_amd import ops
    if c['op'] == 'cross':
        q, k, v = s['q'], s['k'], s['v']
        if not c['grad']:
            if own:
                return ops.cross_attention(q, k, v, s['klens'])
            return _cross_plain(q, k, v, s['klens'])
        q, k, v = (x.detach().requires_grad_(True) for x in (q, k, v))
        if own:
            out = ops.cross_attention(q, k, v, s['klens'])
        else:
            out = _cross_plain(q, k, v, s['klens'])
        return (out.detach(),) + torch.autograd.grad(out, (q, k, v), s['dout'])
    if c['op'] == 'paged':
        new = (s['k_new'], s['v_new']) if c['append'] else (None, None)
        if own:
            out = ops.paged_attention(s['q'], s['k_pages'], s['v_pages'], s['table'], s['lens'], k_new=new[0],
                                      v_new=new[1])
        else:
            out = _paged_plain(s['q'], s['k_pages'], s['v_pages'], s['table'], s['lens'], *new)
        return (out, s['k_pages'], s['v_pages']) if c['append'] else out
    if c['op'] == 'append':
        if own:
            ops.paged_append(s['k'], s['v'], s['k_pages'], s['v_pages'], s['table'], s['starts'], s['counts'])
        else:
            _append_plain(s['k'], s['v'], s['k_pages'], s['v_pages'], s['table'], s['starts'], s['counts'])
        return s['k_pages'], s['v_pages']
    if own:
        return ops.sample_rows(s['logits'], s['u'], s['temperature'], s['top_k'], s['top_p'], s['min_p'])
    return _sample_plain(s['logits'], s['u'], s['temperature'], s['top_k'], s['top_p'], s['min_p'])


# ------------------------------------------------------------------------------------------------ the least there is to do
def work(case):
    c = case
    if c['op'] == 'cross':
        e = BYTES[c['dtype']]
        keys = _sum_spread(c['kmin'], c['Tk'], c['B'])
        rows = c['B'] * c['Tq'] * c['H'] * c['D']
        bytes_ = e * (2 * rows + 2 * keys * c['Hkv'] * c['D'])
        flops = 4.0 * keys * c['Tq'] * c['H'] * c['D']
        if c['grad']:
            bytes_ += e * (2 * rows + 2 * c['B'] * c['Tk'] * c['Hkv'] * c['D'])      # the output's gradient, dq; dk, dv
            flops *= 3.5
        return {'bytes': bytes_, 'flops': flops}
    if c['op'] == 'paged':
        e = BYTES[c['dtype']]
        keys = _sum_spread(c['lmin'], c['lmax'], c['B'])
        row = c['Hkv'] * c['D']
        bytes_ = e * (2 * keys * row + 2 * c['B'] * c['H'] * c['D'] + (4 * c['B'] * row if c['append'] else 0))
        bytes_ += 4 * (keys // c['page'] + c['B'])
        return {'bytes': bytes_, 'flops': 4.0 * (keys + (c['B'] if c['append'] else 0)) * c['H'] * c['D']}
    if c['op'] == 'append':
        n = _sum_spread(c['nmin'], c['n'], c['B']) * c['Hkv'] * c['D']
        return {'bytes': 2.0 * n * (BYTES[c['src']] + BYTES[c['dtype']]) + 8 * c['B'], 'flops': 0.0}
    return {'bytes': BYTES[c['dtype']] * c['B'] * c['V'] + 8 * c['B'], 'flops': 2.0 * c['B'] * c['V']}


# ------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    """from the definitions, sequence by sequence (and head by head where that is much), in 64 bits; caches are written, not
    computed, and tokens are whole numbers: no value for either"""
    c = case
    if c['op'] in ('append', 'sample'):
        return None
    s = prepare(case, seed)
    if c['op'] == 'cross':
        q, k, v = s['q'].double(), s['k'].double(), s['v'].double()
        G, scale = c['H'] // c['Hkv'], c['D'] ** -0.5
        out = torch.empty_like(q)
        dq, dk, dv = torch.zeros_like(q), torch.zeros(k.shape, device=k.device, dtype=k.dtype), None
        dv = torch.zeros_like(dk)
        lens = s['klens'].tolist()
        for b in range(c['B']):
            n = lens[b] if lens[b] > 0 else c['Tk']           # none visible: the mean of all values
            for h in range(c['H']):
                g = h // G
                S = (q[b, :, h] @ k[b, :n, g].t()) * scale
                P = torch.softmax(S if lens[b] > 0 else torch.zeros_like(S), dim=1)
                out[b, :, h] = P @ v[b, :n, g]
                if c['grad']:
                    dO = s['dout'][b, :, h].double()
                    dv[b, :n, g] += P.t() @ dO
                    if lens[b] > 0:
                        dP = dO @ v[b, :n, g].t()
                        dS = P * (dP - (dP * P).sum(1, keepdim=True)) * scale
                        dq[b, :, h] = dS @ k[b, :n, g]
                        dk[b, :n, g] += dS.t() @ q[b, :, h]
        return (out, dq, dk, dv) if c['grad'] else out
    lens, table, page = s['lens'].tolist(), s['table'].cpu(), c['page']
    out = torch.zeros(s['q'].shape, device=s['q'].device, dtype=torch.float64)
    for b in range(c['B']):
        ids = table[b, :(lens[b] + page - 1) // page].long().to(out.device)
        K = s['k_pages'][ids].double().transpose(0, 1).reshape(c['Hkv'], -1, c['D'])[:, :lens[b]]
        V = s['v_pages'][ids].double().transpose(0, 1).reshape(c['Hkv'], -1, c['D'])[:, :lens[b]]
        if c['append']:
            K = torch.cat([K, s['k_new'][b].double().unsqueeze(1)], dim=1)
            V = torch.cat([V, s['v_new'][b].double().unsqueeze(1)], dim=1)
        if K.shape[1]:
            S = torch.matmul(s['q'][b].double().view(c['Hkv'], -1, c['D']), K.transpose(1, 2)) * c['D'] ** -0.5
            out[b] = torch.matmul(torch.softmax(S, dim=2), V).reshape(c['H'], c['D'])
    return (out, None, None) if c['append'] else out
