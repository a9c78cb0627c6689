"""Bodies of the tests of cached decoding (TransformerDecoder.sample, PagedKVCache, the fused source attention of a training
step), run on the host emulator and on the device."""
import numpy as np
import torch

from tests.decoder_ops_common import f32, sample_ref


def tiny_model(dev, n_layers=2, vocab=37, seed=0, **kw):
    from neural_sp_amd.configs import conformer_ctc_att_args
    from neural_sp_amd.speech2text import Speech2Text
    torch.manual_seed(seed)
    args = conformer_ctc_att_args('XS', n_layers=2, vocab=vocab, dec_n_layers=n_layers, transformer_enc_n_heads=4,
                                  transformer_dec_n_heads=4, **kw)
    model = Speech2Text(args).to(dev)
    with torch.no_grad():           # an untrained decoder hardly looks at anything: let it
        for layer in model.dec_fwd.layers:
            for att in (layer.self_attn, layer.src_attn):
                for w in (att.w_query, att.w_key, att.w_value):
                    w.weight.mul_(3.0)
        model.dec_fwd.output.weight.mul_(2.0)
    return model


def states(dev, B=3, T=21, d=64, seed=1):
    g = torch.Generator().manual_seed(seed)
    eouts = torch.randn(B, T, d, generator=g)
    return eouts.to(dev), torch.tensor([T, T - 8, 3][:B], dtype=torch.int32)


def uncached_logits(dec, eouts, elens, prefix):
    """logits of the token behind every prefix of the given tokens, by the training path (whole prefix, causal mask)"""
    from neural_sp_amd import ops
    from neural_sp_amd.modules import AttnMask
    dev = eouts.device
    B, L = prefix.shape
    with torch.no_grad():
        yy = AttnMask(torch.full((B,), L, dtype=torch.int32).to(dev), causal=True, lookahead=0)
        xy = AttnMask(elens.to(dev))
        out = dec.pos_enc(dec.embed(prefix.to(dev)), scale=True)
        for layer in dec.layers:
            out = layer(out, yy, eouts, xy)
        out = ops.layer_norm(out, dec.norm_out.weight, dec.norm_out.bias, dec.norm_out.eps)
        return ops.linear(out, dec.output.weight, dec.output.bias).view(B, L, -1).float().cpu()


def sample_case(dev, settings, seed=5, ratio=1.0, page_size=4, check_every=3):
    """fp32 mode: every token of TransformerDecoder.sample is the one the definition of sample_rows takes from the logits of the
    training path on the same prefix, with the same random numbers"""
    model = tiny_model(dev)
    model.eval()
    dec = model.dec_fwd
    eouts, elens = states(dev)
    hyps, aws = dec.sample(eouts, elens, ratio, seed=seed, page_size=page_size, check_every=check_every, **settings)
    assert aws is None and len(hyps) == 3
    ymax = int(np.ceil(eouts.shape[1] * ratio))
    u = torch.rand((ymax, 3), generator=torch.Generator().manual_seed(seed))
    L = max(len(h) for h in hyps)
    ys = torch.full((3, L), dec.eos, dtype=torch.int64)
    for b, h in enumerate(hyps):
        ys[b, 1:len(h)] = torch.from_numpy(np.ascontiguousarray(h[:L - 1 if len(h) == L else len(h)])[:max(0, len(h) - 1)].astype(np.int64))
    logits = uncached_logits(dec, eouts, elens, ys)
    s = dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0)
    s.update(settings)
    for b, h in enumerate(hyps):
        assert len(h) == ymax or h[-1] == dec.eos
        assert dec.eos not in h[:-1].tolist()
        for n, tok in enumerate(h.tolist()):
            want = sample_ref(logits[b, n], u[n, b].double().item(), f32(s['temperature']), s['top_k'], f32(s['top_p']), f32(s['min_p']))
            assert tok == want, (b, n, tok, want)
    again, _ = dec.sample(eouts, elens, ratio, seed=seed, page_size=16, check_every=1, **settings)
    assert all(np.array_equal(x, y) for x, y in zip(hyps, again))
    short, _ = dec.sample(eouts, elens, ratio, seed=seed, exclude_eos=True, **settings)
    for h, x in zip(hyps, short):
        assert np.array_equal(x, h[:-1] if h[-1] == dec.eos else h)
    return hyps


def position_table_case(dev):
    """no more tokens than there are positions"""
    model = tiny_model(dev)
    model.eval()
    dec = model.dec_fwd
    assert dec.pe_type == 'add'
    eouts, elens = states(dev)
    with torch.no_grad():
        dec.output.bias[dec.eos] = -1e4           # never ends by itself
    long, _ = dec.sample(eouts, elens, seed=2)
    dec.pos_enc.pe = dec.pos_enc.pe[:, :6].contiguous()
    hyps, _ = dec.sample(eouts, elens, 3.0, seed=2)
    assert [len(h) for h in long] == [21] * 3 and [h.tolist() for h in hyps] == [h[:6].tolist() for h in long]


def decode_case(dev):
    """Speech2Text.decode routes recog_sampling there, and nowhere else without it"""
    from neural_sp_amd.configs import synthetic_batch
    import pytest
    model = tiny_model(dev)
    batch = synthetic_batch(B=2, t_range=(40, 52), u_range=(2, 5), vocab=37, seed=0)
    p = dict(recog_sampling=True, recog_temperature=0.9, recog_top_k=10, recog_seed=3, recog_max_len_ratio=0.5)
    a, _ = model.decode(batch['xs'], p, None)
    b, _ = model.decode(batch['xs'], p, None)
    c, _ = model.decode(batch['xs'], dict(p, recog_seed=4), None)
    assert [x[0].tolist() for x in a] == [x[0].tolist() for x in b] != [x[0].tolist() for x in c]
    assert all(len(x) == 1 and 1 <= len(x[0]) for x in a)
    model.dec_fwd.attn_type = 'mocha'
    with pytest.raises(NotImplementedError):
        model.dec_fwd.sample(*states(dev))
    model.dec_fwd.attn_type = 'scaled_dot'
    model.dec_fwd.pos_enc.pe_type = model.dec_fwd.pe_type = '1dconv3L'
    with pytest.raises(NotImplementedError):
        model.dec_fwd.sample(*states(dev))


def training_step(dev, monkeypatch, mode, fused):
    from neural_sp_amd import ops
    from neural_sp_amd.configs import synthetic_batch
    batch = synthetic_batch(B=3, t_range=(40, 64), u_range=(2, 6), vocab=37, seed=0)
    monkeypatch.setenv('NSP_CROSS_ATTN', '1' if fused else '0')
    model = tiny_model(dev)
    with ops.compute_mode(mode):
        loss, _ = model(batch, task='all')
        loss.backward()
    return float(loss.detach()), {n: p.grad.detach().double().cpu() for n, p in model.named_parameters() if p.grad is not None}


def fused_bf16_case(dev, monkeypatch):
    """bf16 mode: both paths round (scores and probabilities here, the context there), and behind a ReLU a rounding can change an
    element of a gradient by its whole value, so single elements say nothing.  Each gradient as a whole: the fused path is as
    near to the fp32 mode's as the other is -- twice that distance, and one bf16 rounding for gradients that it does not touch."""
    l32, g32 = training_step(dev, monkeypatch, 'f32', False)
    l0, g0 = training_step(dev, monkeypatch, 'bf16', False)
    l1, g1 = training_step(dev, monkeypatch, 'bf16', True)
    assert abs(l1 - l32) <= 1e-3 * abs(l32), (l32, l0, l1)
    for n in g32:
        if n.endswith('_attn.w_key.bias'):
            continue                    # 0 but for roundings, see fused_training_case
        norm = float(g32[n].norm())
        d0, d1 = float((g0[n] - g32[n]).norm()), float((g1[n] - g32[n]).norm())
        assert d1 <= 2 * d0 + 2.0 ** -8 * norm, (n, d0 / norm, d1 / norm)


def fused_training_case(dev, monkeypatch, mode, tol_loss, tol_grad):
    """the same training step with and without the fused source attention: loss and every gradient, at the repository's own
    parity gates (largest difference over largest value of each gradient)"""
    from neural_sp_amd import ops
    from neural_sp_amd.configs import synthetic_batch
    batch = synthetic_batch(B=3, t_range=(40, 64), u_range=(2, 6), vocab=37, seed=0)
    got = []
    for on in ('0', '1'):
        monkeypatch.setenv('NSP_CROSS_ATTN', on)
        model = tiny_model(dev)
        calls = []
        real = ops.cross_attention
        monkeypatch.setattr(ops, 'cross_attention', lambda *a, **k: (calls.append(1), real(*a, **k))[1])
        with ops.compute_mode(mode):
            loss, _ = model(batch, task='all')
            loss.backward()
        monkeypatch.setattr(ops, 'cross_attention', real)
        assert len(calls) == (2 if on == '1' else 0)
        got.append((float(loss.detach()), {n: p.grad.detach().float().cpu() for n, p in model.named_parameters() if p.grad is not None}))
    (l0, g0), (l1, g1) = got
    assert abs(l1 - l0) <= tol_loss * abs(l0), (l0, l1)
    assert g0.keys() == g1.keys()
    floor = 1e-5 * sorted(float(g.abs().max()) for g in g0.values())[int(0.9 * (len(g0) - 1))]
    for n in g0:
        if n.endswith('_attn.w_key.bias'):
            # a key bias adds q_i . b to every score of row i, which the softmax does not see: its gradient sum_i q_i sum_j dS_ij is
            # 0 because every sum_j dS_ij is, and what either path gives is rounding.  Measured against the query bias's, a sum of
            # the same dS with keys in the queries' place.
            like = float(g0[n.replace('w_key', 'w_query')].abs().max())
            assert max(float(g0[n].abs().max()), float(g1[n].abs().max())) <= tol_grad * like, n
            continue
        d = float((g1[n] - g0[n]).abs().max()) / max(float(g0[n].abs().max()), floor)
        assert d <= tol_grad, (n, d)


def cache_case(dev):
    import pytest
    from neural_sp_amd.kv_cache import PagedKVCache
    c = PagedKVCache(2, 3, 20, 2, 16, torch.float32, dev, page_size=8, n_pages=5)
    assert c.k(0).shape == (5, 2, 8, 16) and c.block_table.shape == (3, 3) and c.lens.tolist() == [-1, -1, -1]
    c.reserve([0, 2, 0], 9)
    t = c.block_table.cpu()
    used = t[t >= 0].tolist()
    assert (t >= 0).sum(1).tolist() == [2, 0, 2] and len(set(used)) == 4 and c.free_pages == 1
    with pytest.raises(RuntimeError):
        c.reserve([0, 2], 20)                       # all or none
    assert torch.equal(c.block_table.cpu(), t) and c.free_pages == 1
    with pytest.raises(ValueError):
        c.reserve([1], 25)
    c.reserve([0], 5)                               # never fewer
    old = c.block_table
    c.release([0, 0])
    assert c.free_pages == 3 and c.block_table[0].tolist() == [-1, -1, -1] and old[0].tolist() == t[0].tolist()
    c.reserve([1], 20)
    t = c.block_table.cpu()
    assert c.free_pages == 0 and len(set(t[t >= 0].tolist())) == 5
    with pytest.raises(ValueError):
        PagedKVCache(1, 1, 0, 1, 8, torch.float32, dev)


def cache_rows_case(dev):
    """a row named twice, once from the end, is one row; a wrong row changes nothing"""
    import pytest
    from neural_sp_amd.kv_cache import PagedKVCache
    c = PagedKVCache(1, 3, 16, 1, 8, torch.float32, dev, page_size=8, n_pages=3)
    c.reserve([2, -1], 16)
    c.reserve([0], 8)
    t = c.block_table.cpu()
    assert (t >= 0).sum(1).tolist() == [1, 0, 2] and c.free_pages == 0
    for wrong in (3, -4):
        with pytest.raises(IndexError):
            c.reserve([0, wrong], 16)
        with pytest.raises(IndexError):
            c.release([0, wrong])
        assert torch.equal(c.block_table.cpu(), t) and c.free_pages == 0
        c.reserve([0], 8)                               # still its own page
        assert torch.equal(c.block_table.cpu(), t)
    c.release([-1, 2])
    assert c.free_pages == 2 and c.block_table.cpu()[2].tolist() == [-1, -1]
    c.reserve([1], 16)
    t = c.block_table.cpu()
    used = t[t >= 0].tolist()
    assert len(used) == len(set(used)) == 3


def bf16_logits_case(dev, monkeypatch, steps=12):
    """bf16 mode: the logits that the cached steps hand to the sampler, against the training path's on the same prefixes.  Both
    round, in different places, so each step's logits as a whole: as near to the fp32 mode's as the training path's are -- twice
    that distance, and one bf16 rounding (of the norm)."""
    from neural_sp_amd import ops
    model = tiny_model(dev)
    model.eval()
    dec = model.dec_fwd
    eouts, elens = states(dev)
    with torch.no_grad():
        dec.output.bias[dec.eos] = -1e4               # all utterances take every step
    got, real = [], ops.sample_rows
    monkeypatch.setattr(ops, 'sample_rows', lambda x, *a: (got.append(x.detach().float().cpu()), real(x, *a))[1])
    with ops.compute_mode('bf16'):
        hyps, _ = dec.sample(eouts, elens, steps / eouts.shape[1], seed=3, page_size=4)
    monkeypatch.setattr(ops, 'sample_rows', real)
    assert len(got) == steps and [len(h) for h in hyps] == [steps] * 3
    ys = torch.full((3, steps), dec.eos, dtype=torch.int64)
    for b, h in enumerate(hyps):
        ys[b, 1:] = torch.from_numpy(np.ascontiguousarray(h[:-1]).astype(np.int64))
    with ops.compute_mode('f32'):
        want = uncached_logits(dec, eouts, elens, ys).double()
    with ops.compute_mode('bf16'):
        other = uncached_logits(dec, eouts, elens, ys).double()
    seen = [i for i in range(want.shape[2]) if i != dec.eos]
    for n in range(steps):
        w, o, x = want[:, n, seen], other[:, n, seen], got[n].double()[:, seen]
        assert float((x - w).norm()) <= 2 * float((o - w).norm()) + 2.0 ** -8 * float(w.norm()), n
