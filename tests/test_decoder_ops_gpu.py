"""The decoder operators on the device: sizes, masks, layouts and the ways a program uses them (streams, captured graphs,
repeated calls), every value against 64 bits (tests/decoder_ops_common.py)."""
import pytest
import torch

from tests import decoder_ops_common as C

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
DEV = 'cuda'


@pytest.fixture(autouse=True)
def random_state_of_the_process():
    """the tests behind these draw the numbers and the dropout masks that they draw without them"""
    from neural_sp_amd import ops
    was = dict(ops._DROPOUT_STATE)
    with torch.random.fork_rng():
        yield
    ops._DROPOUT_STATE.update(was)


@pytest.fixture
def ops():
    from neural_sp_amd import ops
    return ops


CROSS = [
    dict(B=2, H=2, Hkv=2, D=64, Tq=5, Tk=70, klens=[70, 33]),
    dict(B=3, H=4, Hkv=2, D=32, Tq=70, Tk=20, klens=[0, 1, -3], layout='heads'),
    dict(B=1, H=3, Hkv=1, D=72, Tq=66, Tk=130, klens=None, layout='dense'),
    dict(B=2, H=1, Hkv=1, D=8, Tq=1, Tk=1, klens=[1, 9]),
    dict(B=9, H=8, Hkv=8, D=64, Tq=131, Tk=257, klens=[257, 256, 255, 193, 192, 129, 65, 64, 63]),
    dict(B=2, H=16, Hkv=4, D=128, Tq=129, Tk=515, klens=[515, 100]),
    dict(B=1, H=6, Hkv=1, D=40, Tq=1, Tk=3001, klens=[3000]),
    dict(B=1, H=2, Hkv=2, D=64, Tq=700, Tk=64, klens=[64], scale=0.5),
    dict(B=64, H=8, Hkv=8, D=64, Tq=70, Tk=131, klens=[131 - 2 * i for i in range(64)]),      # two owned fragments per wave
    dict(B=32, H=16, Hkv=16, D=128, Tq=130, Tk=66, klens=[66 - i for i in range(32)]),
    dict(B=520, H=2, Hkv=1, D=24, Tq=129, Tk=129, klens=[(i * 5) % 131 for i in range(520)]),
    dict(B=17, H=2, Hkv=1, D=96, Tq=16, Tk=100, klens=[100 - 5 * i for i in range(17)], layout='heads'),
]


@pytest.mark.parametrize('dtype', [BF, F32])
@pytest.mark.parametrize('a', CROSS, ids=str)
@pytest.mark.parametrize('grad', [True, False])
def test_cross_attention(ops, dtype, a, grad):
    C.cross_case(ops, DEV, dtype, grad=grad, **a)


@pytest.mark.parametrize('dtype', [BF, F32])
@pytest.mark.parametrize('a', [
    dict(B=2, H=4, Hkv=4, D=64, page=16, lens=[0, 37], append=True),
    dict(B=3, H=8, Hkv=2, D=128, page=32, lens=[0, 5, 300], append=False),
    dict(B=3, H=6, Hkv=2, D=40, page=7, lens=[-1, 50, 0], append=True),
    dict(B=1, H=2, Hkv=1, D=32, page=100, lens=[1100], append=True, layout='slots_first'),
    dict(B=1, H=20, Hkv=1, D=72, page=1, lens=[70], append=True),
    dict(B=2, H=8, Hkv=8, D=64, page=16, lens=[15, 16], append=True, layout='slots_first'),
    dict(B=2, H=7, Hkv=1, D=128, page=64, lens=[5000, 2], append=True),
    dict(B=1, H=1, Hkv=1, D=64, page=256, lens=[4096], append=False),
], ids=str)
def test_paged_attention(ops, dtype, a):
    C.paged_case(ops, DEV, dtype, **a)


def test_paged_attention_absent_pages_and_full_tables(ops):
    for dtype in (BF, F32):
        for page in (16, 5):
            C.absent_pages_case(ops, DEV, dtype, page)


@pytest.mark.parametrize('src,dtype', [(F32, BF), (F32, F32), (BF, BF)])
@pytest.mark.parametrize('a', [
    dict(B=3, n=9, Hkv=2, D=40, page=4, starts=[0, -1, 3], counts=[9, 4, 0]),
    dict(B=3, n=90, Hkv=2, D=32, page=16, starts=[0, 20, 3], counts=[90, 4, 70], layout='slots_first', strided=False),
    dict(B=1, n=1, Hkv=1, D=128, page=1, starts=[5], counts=[1]),
    dict(B=5, n=200, Hkv=8, D=64, page=16, starts=[0, 1, 15, 16, 17], counts=[200, 199, 17, 1, 0]),
], ids=str)
def test_paged_append(ops, src, dtype, a):
    C.append_case(ops, DEV, src, dtype, **a)


SAMPLE = [dict(), dict(k=5), dict(tp=.9), dict(mp=.05), dict(k=40, tp=.7, mp=.01, t=.7), dict(t=0.0), dict(k=1), dict(t=1e-4),
          dict(t=1e4), dict(tp=0.0), dict(mp=2.0)]


@pytest.mark.parametrize('dtype', [BF, F32])
@pytest.mark.parametrize('kw', SAMPLE, ids=str)
@pytest.mark.parametrize('V', [1, 40, 1000, 4097])
def test_sample_rows(ops, dtype, kw, V):
    g = torch.Generator().manual_seed(V)
    x = torch.randn(6, V, generator=g) * 3
    C.sample_case(ops, DEV, x.to(dtype), [0.0, 0.3, 0.5, 0.7, 0.9, 0.99999], **kw)


def test_sample_rows_long_rows_and_ties(ops):
    g = torch.Generator().manual_seed(2)
    for V in (32768, 32769, 50001):
        x = torch.randn(3, V + 1, generator=g)[:, :V] * 2
        C.sample_case(ops, DEV, x, [0.1, 0.5, 0.9], k=[50, 0, V // 2], tp=[0.9, 0.8, 1.0], t=[1.0, 0.5, 2.0])
    for kw in (dict(), dict(k=1650), dict(tp=.9), dict(k=600, tp=.7)):
        C.sample_case(ops, DEV, torch.zeros(2, 3001), [0.2, 0.9], **kw)
        x = torch.where(torch.arange(3001) % 3 == 0, 1.0, -0.0).repeat(2, 1)
        C.sample_case(ops, DEV, x, [0.2, 0.9], **kw)


@pytest.mark.parametrize('V,kw', C.SAMPLE_GATHERED, ids=str)
def test_sample_rows_gathered(ops, V, kw):
    C.gathered_case(ops, DEV, V, kw)


def test_sample_rows_temperature_zero_is_argmax_rows(ops):
    x = torch.randn(33, 777, generator=torch.Generator().manual_seed(4)).to(DEV).round()
    assert torch.equal(ops.sample_rows(x, torch.zeros(33, device=DEV), temperature=0.0), ops.argmax_rows(x))


def test_cross_attention_dropout_is_the_training_softmax_mask(ops):
    for dtype in (F32, BF):
        C.dropout_case(ops, DEV, dtype, B=2, H=3, Tq=37, Tk=150, D=32)


def test_cross_attention_against_differences(ops):
    C.difference_case(ops, DEV)


def test_single_token_form_agrees_with_the_training_form(ops):
    """the two kernels behind cross_attention, on the same call: within both their bounds of each other"""
    g = torch.Generator().manual_seed(9)
    for dtype in (BF, F32):
        q, k, v = (torch.randn(4, t, 4, 64, generator=g).to(dtype) for t in (2, 400, 400))
        klens = [400, 0, 17, 257]
        _, tol = C.cross_ref(q, k, v, None, klens, dtype)['out']
        lens = torch.tensor(klens, dtype=torch.int32).to(DEV)
        a = ops.cross_attention(q.to(DEV), k.to(DEV), v.to(DEV), lens)
        b = ops.cross_attention(q.to(DEV).requires_grad_(True), k.to(DEV), v.to(DEV), lens)
        assert ((a.double() - b.detach().double()).abs().cpu() <= 2 * tol).all()


def test_same_bits_every_time_and_on_another_stream(ops):
    g = torch.Generator().manual_seed(6)
    q, k, v = (torch.randn(3, t, 8, 64, generator=g).to(BF).to(DEV).requires_grad_(True) for t in (100, 333, 333))
    dout = torch.randn(3, 100, 8, 64, generator=g).to(BF).to(DEV)
    lens = torch.tensor([333, 200, 64], dtype=torch.int32, device=DEV)
    kp, vp = torch.randn(90, 8, 16, 64, device=DEV).to(BF), torch.randn(90, 8, 16, 64, device=DEV).to(BF)
    table = torch.randperm(90, generator=g)[:84].to(torch.int32).view(3, 28).to(DEV)
    plens = torch.tensor([440, 100, 0], dtype=torch.int32, device=DEV)
    logits, u = torch.randn(40, 5000, device=DEV) * 2, torch.rand(40, device=DEV)

    def all_of_them():
        out = ops.cross_attention(q, k, v, lens)
        r = [out.detach()] + list(torch.autograd.grad(out, (q, k, v), dout))
        with torch.no_grad():
            r.append(ops.cross_attention(q[:, :1], k, v, lens))
        r.append(ops.paged_attention(q.detach()[:, 0], kp, vp, table, plens))
        r.append(ops.sample_rows(logits, u, 0.9, 100, 0.9, 0.01))
        return r
    first = all_of_them()
    side = torch.cuda.Stream()
    for _ in range(3):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            again = all_of_them()
        torch.cuda.current_stream().wait_stream(side)
        here = all_of_them()
        for a, b, c in zip(first, again, here):
            assert torch.equal(a, b) and torch.equal(a, c)


def test_two_captured_graphs_with_eager_work_between(ops):
    """a decoding step captured twice at different sizes (each graph with its own workspace) and a training pass, replayed
    several times with new inputs and with eager calls of the same sizes in between"""
    g = torch.Generator().manual_seed(8)

    def step(B, pages):
        s = dict(q=torch.randn(B, 4, 64, generator=g).to(DEV), kn=torch.randn(B, 4, 64, generator=g).to(DEV),
                 vn=torch.randn(B, 4, 64, generator=g).to(DEV), kp=torch.randn(B * pages, 4, 16, 64, generator=g).to(DEV),
                 vp=torch.randn(B * pages, 4, 16, 64, generator=g).to(DEV), lens=torch.zeros(B, dtype=torch.int32, device=DEV),
                 table=torch.randperm(B * pages, generator=g).to(torch.int32).view(B, pages).to(DEV),
                 enc=torch.randn(B, 900, 2, 4, 64, generator=g).to(DEV), u=torch.rand(B, generator=g).to(DEV),
                 w=torch.randn(256, 500, generator=g).to(DEV))

        def run():
            o = ops.paged_attention(s['q'], s['kp'], s['vp'], s['table'], s['lens'], s['kn'], s['vn'])
            o = ops.cross_attention(o.unsqueeze(1), s['enc'][:, :, 0], s['enc'][:, :, 1])
            return o, ops.sample_rows(o.reshape(o.shape[0], -1) @ s['w'], s['u'], 1.0, 20, 0.9)
        return s, run
    made = []
    for B, pages in ((1, 40), (3, 90)):
        s, run = step(B, pages)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run()
        made.append((s, run, graph, out))
    for n in (0, 5, 16, 300, 639, 1):
        for s, run, graph, out in made:
            s['lens'].fill_(n)
            s['q'].copy_(torch.randn(s['q'].shape, generator=g))
        for s, run, graph, out in made:      # both in flight before anything is compared
            graph.replay()
        for s, run, graph, out in made:
            want = run()
            torch.cuda.synchronize()
            assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1]), n


def test_captured_training_pass(ops):
    g = torch.Generator().manual_seed(10)
    q, k, v = (torch.randn(2, t, 4, 64, generator=g).to(BF).to(DEV) for t in (40, 200, 200))
    dout = torch.randn(2, 40, 4, 64, generator=g).to(BF).to(DEV)
    lens = torch.tensor([200, 77], dtype=torch.int32, device=DEV)

    def run():
        x = [t.detach().requires_grad_(True) for t in (q, k, v)]
        out = ops.cross_attention(*x, lens)
        return [out.detach()] + list(torch.autograd.grad(out, x, dout))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for i in range(4):
        q.copy_(torch.randn(q.shape, generator=g))
        lens.copy_(torch.tensor([200 - 30 * i, 77 * (i % 2)], dtype=torch.int32))
        graph.replay()
        want = run()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_cache_offsets_behind_32_bits(ops):
    """a cache of more than 2^32 bytes: pages at its far end"""
    n_pages, page, Hkv, D = 33000, 64, 8, 128                    # 4.3 GB per tensor
    kp = torch.zeros(n_pages, Hkv, page, D, device=DEV, dtype=BF)
    vp = torch.zeros(n_pages, Hkv, page, D, device=DEV, dtype=BF)
    g = torch.Generator().manual_seed(12)
    table = torch.tensor([[n_pages - 1, 5, n_pages - 2]], dtype=torch.int32, device=DEV)
    k, v = (torch.randn(1, 150, Hkv, D, generator=g).to(BF) for _ in range(2))
    ops.paged_append(k.to(DEV), v.to(DEV), kp, vp, table, torch.zeros(1, dtype=torch.int32, device=DEV))
    assert torch.equal(kp[n_pages - 2, :, :22].cpu(), k[0, 128:].transpose(0, 1))
    q = torch.randn(1, 16, D, generator=g).to(BF)
    out = ops.paged_attention(q.to(DEV), kp, vp, table, torch.tensor([150], dtype=torch.int32, device=DEV))
    for h in range(Hkv):
        ref, dp, av = C.attention_ref(q[0, 2 * h:2 * h + 2], k[0, :, h], v[0, :, h], 150)
        C.check_close(out[0, 2 * h:2 * h + 2], ref, C.half_step(BF) * ref.abs() + (dp + C.E16 ** 2) * av * (1 + C.half_step(BF)), h)


def test_cross_attention_backward_passes_do_not_meet(ops):
    C.backward_case(ops, DEV)


@pytest.mark.parametrize('dtype', [BF, F32])
def test_cross_attention_scores_of_minus_infinity(ops, dtype):
    C.infinite_scores_case(ops, DEV, dtype)


def test_cross_attention_of_more_sequences_than_a_grid_has_rows(ops):
    """(the single-token kernel has a sequence per grid row, 65535 at most; the other one takes over)"""
    g = torch.Generator().manual_seed(1)
    B = 65540
    q, k, v = (torch.randn(2, t, 1, 8, generator=g).repeat(B // 2, 1, 1, 1) for t in (1, 2, 2))
    out = ops.cross_attention(q.to(DEV), k.to(DEV), v.to(DEV)).cpu()
    want = C.cross_ref(q[:2], k[:2], v[:2], None, None, F32)['out']
    C.check_close(out[:2], want[0], want[1], 'out')
    assert torch.equal(out, out[:2].repeat(B // 2, 1, 1, 1))


@pytest.mark.parametrize('D', [8, 40, 72, 96])
@pytest.mark.parametrize('dtype', [BF, F32])
def test_cross_attention_scores_of_minus_infinity_by_the_last_dimension(ops, dtype, D):
    C.infinite_scores_in_the_last_dimension_case(ops, DEV, dtype, D)


@pytest.mark.parametrize('dtype', [BF, F32])
@pytest.mark.parametrize('a', C.INFINITE_LAST_ROW, ids=str)
def test_cross_attention_of_an_infinite_last_row(ops, dtype, a):
    C.infinite_last_row_case(ops, DEV, dtype, **a)


@pytest.mark.parametrize('dtype', [BF, F32])
@pytest.mark.parametrize('a', C.INFINITE_VALUES, ids=str)
def test_decoding_with_infinite_values(ops, dtype, a):
    C.infinite_values_paged_case(ops, DEV, dtype, **a)


@pytest.mark.parametrize('dtype', [BF, F32])
@pytest.mark.parametrize('Tk', [40, 1300])
def test_cross_attention_of_a_row_without_a_softmax(ops, dtype, Tk):
    C.no_softmax_case(ops, DEV, dtype, Tk)


@pytest.mark.parametrize('V', [3, 700, 12000, 33000])
def test_sample_rows_of_nan_among_minus_infinities(ops, V):
    C.nan_among_minus_infinities_case(ops, DEV, V)


@pytest.mark.parametrize('tokens', [1, 40])
def test_cross_attention_of_dual_tensors(ops, tokens):
    C.forward_mode_case(ops, DEV, tokens)
    C.forward_mode_case(ops, DEV, tokens, 0.1)


def test_paged_attention_has_no_backward_pass(ops):
    C.no_backward_case(ops, DEV)


def test_pages_that_autograd_has_saved(ops):
    C.overwritten_pages_case(ops, DEV)


def test_cross_attention_of_tokens_far_apart(ops):
    C.far_tokens_case(ops, DEV)


@pytest.mark.parametrize('page', [16, 5])
def test_paged_attention_of_more_pages_than_an_int_counts(ops, page):
    C.many_pages_case(ops, DEV, page)


@pytest.mark.parametrize('dtype', [BF, F32])
@pytest.mark.parametrize('a', C.DROPOUT_WIDTHS, ids=str)
def test_cross_attention_dropout_widths(ops, dtype, a):
    C.dropout_widths_case(ops, DEV, dtype, **a)


@pytest.mark.parametrize('dtype', [BF, F32])
@pytest.mark.parametrize('V,kw', C.SAMPLE_WIDE, ids=str)
def test_sample_rows_wide(ops, dtype, V, kw):
    C.wide_case(ops, DEV, dtype, V, kw)


def test_captured_calls_of_large_shared_memory_and_split_keys(ops):
    """sampling from long rows (more LDS than a launch has without asking), decoding over split keys: captured before their first
    eager call of these sizes, replayed with new inputs"""
    g = torch.Generator().manual_seed(11)
    x = [torch.randn(5, V, generator=g).to(DEV) for V in (10007, 29000, 33001)]
    u = torch.rand(5, generator=g).to(DEV)
    q, k, v = (torch.randn(2, t, 4, 72, generator=g).to(BF).to(DEV) for t in (1, 1777, 1777))
    lens = torch.tensor([1777, 901], dtype=torch.int32, device=DEV)

    def run():
        return [ops.sample_rows(y, u, 0.8, 300, 0.9) for y in x] + [ops.sample_rows(x[0], u), ops.cross_attention(q, k, v, lens)]
    ops.sample_rows(x[0][:, :10], u)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for i in range(4):
        for t in x + [u, q]:
            t.copy_(torch.rand(t.shape, generator=g))
        lens.copy_(torch.tensor([1777 - 400 * i, 5 * i], dtype=torch.int32))
        graph.replay()
        want = run()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i
