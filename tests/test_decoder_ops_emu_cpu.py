"""The decoder operators (ops.cross_attention, paged_attention, paged_append, sample_rows) on the host emulator of their
kernels, through the real ctypes glue: every case against 64 bits (tests/decoder_ops_common.py), and what they refuse."""
import pytest
import torch

from tests import decoder_ops_common as C
from tests.hipemu import build_emu

pytestmark = pytest.mark.skipif(not build_emu.available(), reason='no host clang++ for the HIP emulator')
BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def random_state_of_the_process():
    """the tests behind these draw the numbers and the dropout masks that they draw without them"""
    from neural_sp_amd import ops
    was = dict(ops._DROPOUT_STATE)
    with torch.random.fork_rng():
        yield
    ops._DROPOUT_STATE.update(was)


@pytest.fixture
def emu():
    from neural_sp_amd import ops
    from tests.hipemu.shim import emulated_kernels
    with emulated_kernels():
        yield ops


@pytest.mark.parametrize('dtype', [BF, F32])
@pytest.mark.parametrize('a', [
    dict(B=2, H=2, Hkv=2, D=64, Tq=5, Tk=70, klens=[70, 33]),
    dict(B=3, H=4, Hkv=2, D=32, Tq=70, Tk=20, klens=[0, 1, -3], layout='heads'),     # rows without a visible key
    dict(B=1, H=3, Hkv=1, D=72, Tq=66, Tk=130, klens=None, layout='dense'),           # head size between the kernels' sizes
    dict(B=1, H=2, Hkv=1, D=128, Tq=3, Tk=65, klens=[64]),
    dict(B=2, H=1, Hkv=1, D=8, Tq=1, Tk=1, klens=[1, 9]),                             # length behind the tensor's end
    dict(B=1, H=1, Hkv=1, D=40, Tq=17, Tk=129, klens=[128], scale=0.9),
], ids=str)
@pytest.mark.parametrize('grad', [True, False])
def test_cross_attention(emu, dtype, a, grad):
    C.cross_case(emu, 'cpu', dtype, grad=grad, **a)


@pytest.mark.parametrize('dtype', [BF, F32])
@pytest.mark.parametrize('a', [
    dict(B=2, H=4, Hkv=4, D=64, page=16, lens=[0, 37], append=True),
    dict(B=3, H=8, Hkv=2, D=128, page=32, lens=[0, 5, 300], append=False),
    dict(B=3, H=6, Hkv=2, D=40, page=7, lens=[-1, 50, 0], append=True),               # an unused row; pages of odd size
    dict(B=1, H=2, Hkv=1, D=32, page=100, lens=[1100], append=True, layout='slots_first'),
    dict(B=1, H=20, Hkv=1, D=72, page=1, lens=[70], append=True),                     # more than 16 rows on one key head
    dict(B=2, H=2, Hkv=1, D=64, page=16, lens=[15, 16], append=True),                 # the new token fills / opens a page
], ids=str)
def test_paged_attention(emu, dtype, a):
    C.paged_case(emu, 'cpu', dtype, **a)


def test_paged_attention_absent_pages_and_full_tables(emu):
    C.absent_pages_case(emu, 'cpu', BF, 16)
    C.absent_pages_case(emu, 'cpu', F32, 5)


@pytest.mark.parametrize('src,dtype', [(F32, BF), (F32, F32), (BF, BF)])
@pytest.mark.parametrize('a', [
    dict(B=3, n=9, Hkv=2, D=40, page=4, starts=[0, -1, 3], counts=[9, 4, 0]),
    dict(B=3, n=9, Hkv=2, D=32, page=16, starts=[0, 20, 3], counts=[9, 4, 7], layout='slots_first', strided=False),
    dict(B=1, n=1, Hkv=1, D=128, page=1, starts=[5], counts=[1]),
], ids=str)
def test_paged_append(emu, src, dtype, a):
    C.append_case(emu, 'cpu', src, dtype, **a)


def test_paged_append_drops_what_has_no_place(emu):
    k = torch.ones(2, 4, 1, 8)
    pages = torch.zeros(3, 1, 2, 8)
    vp = torch.zeros(3, 1, 2, 8)
    table = torch.tensor([[0, 7], [-1, 2]], dtype=torch.int32)       # page 7 does not exist, page -1 neither
    emu.paged_append(k, 2 * k, pages, vp, table, torch.tensor([1, 0], dtype=torch.int32))
    want = torch.zeros(3, 1, 2, 8)
    want[0, 0, 1] = 1.0            # row 0: position 1 only (2, 3 on page 7, 4 behind the table)
    want[2, 0, :] = 1.0            # row 1: positions 2 and 3
    assert torch.equal(pages, want) and torch.equal(vp, 2 * want)


SAMPLE = [dict(), dict(k=5), dict(tp=.9), dict(mp=.05), dict(k=40, tp=.7, mp=.01, t=.7), dict(t=0.0), dict(tp=0.0), dict(mp=1.0),
          dict(mp=2.0), dict(k=1), dict(k=10 ** 9), dict(k=-4), dict(t=1e-4), dict(t=1e4),
          dict(k=[0, 1, 300, 299], tp=[1.0, .5, .2, .99], t=[1., 2., .5, 1.], mp=[0., .1, 0., .3])]


@pytest.mark.parametrize('dtype', [BF, F32])
@pytest.mark.parametrize('kw', SAMPLE, ids=str)
def test_sample_rows(emu, dtype, kw):
    x = torch.randn(4, 300, generator=torch.Generator().manual_seed(1)) * 3
    C.sample_case(emu, 'cpu', x.to(dtype), [0.0, 0.3, 0.7, 0.99999], **kw)


@pytest.mark.parametrize('kw', [dict(), dict(k=650), dict(tp=.9), dict(k=600, tp=.7), dict(k=3)], ids=str)
def test_sample_rows_of_equal_logits(emu, kw):
    """one value everywhere, and two values: the border falls inside a class of equal logits larger than what is ranked
    entry by entry"""
    u = [0.0, 0.3, 0.7, 0.99999]
    C.sample_case(emu, 'cpu', torch.zeros(4, 700), u, **kw)
    x = torch.where(torch.arange(1500) % 3 == 0, 1.0, -0.0).repeat(4, 1)
    x[:, 6] = 0.0
    C.sample_case(emu, 'cpu', x, u, **kw)


@pytest.mark.parametrize('V,kw', C.SAMPLE_GATHERED, ids=str)
def test_sample_rows_gathered(emu, V, kw):
    C.gathered_case(emu, 'cpu', V, kw)


def test_sample_rows_infinities_and_nan(emu):
    inf, nan = float('inf'), float('nan')
    x = torch.tensor([[nan, 1.0, nan, 2.0], [-inf, -inf, -inf, -inf], [0.0, inf, 1.0, inf], [nan, nan, nan, nan],
                      [-inf, 0.5, -inf, 0.5]])
    for u, want in ((0.0, [1, 0, 1, 0, 1]), (0.6, [3, 0, 3, 0, 3])):
        got = emu.sample_rows(x, torch.full((5,), u))
        assert got.tolist() == want
    # random numbers outside [0, 1) stay inside the kept entries
    for u, want in ((-1.0, [1, 0, 1, 0, 1]), (1.0, [3, 0, 3, 0, 3]), (nan, [3, 0, 3, 0, 3])):
        assert emu.sample_rows(x, torch.full((5,), u)).tolist() == want


def test_sample_rows_sizes_and_strides(emu):
    g = torch.Generator().manual_seed(5)
    for V in (1, 2, 63, 4096, 4097, 33000):          # 33000: more than the LDS holds
        x = torch.randn(2, V + 3, generator=g)[:, :V]
        C.sample_case(emu, 'cpu', x, [0.2, 0.8], k=[7, 0], tp=[1.0, 0.6])
    assert emu.sample_rows(torch.zeros(0, 5), torch.zeros(0)).shape == (0,)
    one = torch.randn(1, 50, generator=g).expand(3, 50)
    assert len(set(emu.sample_rows(one, torch.full((3,), 0.4)).tolist())) == 1


def test_empty_calls(emu):
    """no sequence, no query, no key"""
    i32 = torch.int32
    for B, Tq, Tk in ((0, 3, 4), (2, 0, 4), (2, 3, 0)):
        q, k, v = (torch.randn(B, t, 2, 16, requires_grad=True) for t in (Tq, Tk, Tk))
        out = emu.cross_attention(q, k, v, torch.zeros(B, dtype=i32))
        assert out.shape == q.shape and not out.any()
        for x, g in zip((q, k, v), torch.autograd.grad(out.sum(), (q, k, v))):
            assert g.shape == x.shape and not g.any()
        with torch.no_grad():
            assert not emu.cross_attention(q, k, v).any()
    pages = torch.zeros(1, 2, 4, 16)
    assert emu.paged_attention(torch.zeros(0, 2, 16), pages, pages, torch.zeros(0, 1, dtype=i32), torch.zeros(0, dtype=i32)).shape == (0, 2, 16)
    out = emu.paged_attention(torch.ones(2, 2, 16), pages, pages, torch.zeros(2, 0, dtype=i32), torch.tensor([3, 0], dtype=i32),
                              torch.ones(2, 2, 16), torch.ones(2, 2, 16))
    assert not out.any()          # a table without columns: no key, no room
    emu.paged_append(torch.zeros(2, 0, 2, 16), torch.zeros(2, 0, 2, 16), pages, pages, torch.zeros(2, 1, dtype=i32), torch.zeros(2, dtype=i32))


def test_refusals(emu):
    i32 = torch.int32
    q, k = torch.zeros(2, 3, 4, 16), torch.zeros(2, 5, 2, 16)
    lens = torch.zeros(2, dtype=i32)
    for bad in (lambda: emu.cross_attention(q, k, k.bfloat16()), lambda: emu.cross_attention(q.half(), k.half(), k.half()),
                lambda: emu.cross_attention(q, k[:1], k[:1]), lambda: emu.cross_attention(q[:, :, :3], k, k),
                lambda: emu.cross_attention(q[..., :12], k[..., :12], k[..., :12]),
                lambda: emu.cross_attention(torch.zeros(1, 1, 1, 136), torch.zeros(1, 1, 1, 136), torch.zeros(1, 1, 1, 136)),
                lambda: emu.cross_attention(q, k, k, lens.long()), lambda: emu.cross_attention(q, k, k, lens[:1]),
                lambda: emu.cross_attention(q, k, k, scale=0.0), lambda: emu.cross_attention(q, k, k, dropout_p=1.0),
                lambda: emu.cross_attention(q, k, k[:, :4]), lambda: emu.cross_attention(q[0], k, k)):
        with pytest.raises(ValueError):
            bad()
    q, kp, t = torch.zeros(2, 4, 16), torch.zeros(3, 2, 4, 16), torch.zeros(2, 2, dtype=i32)
    n = torch.zeros(2, 2, 16)
    for bad in (lambda: emu.paged_attention(q.bfloat16(), kp, kp, t, lens), lambda: emu.paged_attention(q, kp, kp[:2], t, lens),
                lambda: emu.paged_attention(q, kp, kp, t.long(), lens), lambda: emu.paged_attention(q, kp, kp, t[:1], lens),
                lambda: emu.paged_attention(q, kp, kp, t, lens[:1]), lambda: emu.paged_attention(q, kp, kp, t, lens, n),
                lambda: emu.paged_attention(q, kp, kp, t, lens, n[:1], n[:1]), lambda: emu.paged_attention(q[:, :3], kp, kp, t, lens),
                lambda: emu.paged_attention(q, kp, kp, t, lens, n.bfloat16(), n.bfloat16()),
                lambda: emu.paged_attention(q, kp.transpose(2, 3), kp.transpose(2, 3), t, lens),
                lambda: emu.paged_append(n.unsqueeze(1), n.unsqueeze(1), torch.zeros(3, 2, 4, 18)[..., 1:17], kp, t, lens),
                lambda: emu.paged_append(n.unsqueeze(1).bfloat16(), n.unsqueeze(1).bfloat16(), kp, kp, t, lens),
                lambda: emu.paged_append(n, n, kp, kp, t, lens),
                lambda: emu.paged_append(n.unsqueeze(1), n.unsqueeze(1), kp, kp, t, lens, lens[:1])):
        with pytest.raises(ValueError):
            bad()
    x, u = torch.zeros(2, 9), torch.zeros(2)
    for bad in (lambda: emu.sample_rows(x.half(), u), lambda: emu.sample_rows(x, u[:1]), lambda: emu.sample_rows(x, u.double()),
                lambda: emu.sample_rows(x, u, top_k=torch.zeros(2)), lambda: emu.sample_rows(x, u, temperature=torch.zeros(1)),
                lambda: emu.sample_rows(torch.zeros(1, (1 << 18) + 1), u[:1]), lambda: emu.sample_rows(x[:, :0], u)):
        with pytest.raises(ValueError):
            bad()


def test_host_tensors_are_rejected_loudly():
    """without the emulator: no CPU fallback"""
    from neural_sp_amd import ops
    x = torch.zeros(1, 1, 1, 8)
    i = torch.zeros(1, dtype=torch.int32)
    for call in (lambda: ops.cross_attention(x, x, x), lambda: ops.paged_attention(x[0], x, x, i.view(1, 1), i),
                 lambda: ops.paged_append(x, x, x, x, i.view(1, 1), i), lambda: ops.sample_rows(x[0, 0], x[0, 0, 0, :1])):
        with pytest.raises((AssertionError, RuntimeError)):
            call()


def test_cross_attention_dropout_is_the_training_softmax_mask(emu):
    """same site, same mask as AttentionFn (attn_softmax_fwd), forward and backward"""
    C.dropout_case(emu, 'cpu', F32)
    C.dropout_case(emu, 'cpu', BF)


def test_cross_attention_against_differences(emu):
    C.difference_case(emu, 'cpu')


def test_cross_attention_backward_passes_do_not_meet(emu):
    C.backward_case(emu, 'cpu')


@pytest.mark.parametrize('dtype', [BF, F32])
def test_cross_attention_scores_of_minus_infinity(emu, dtype):
    C.infinite_scores_case(emu, 'cpu', dtype)


def test_refusals_of_memory_and_settings(emu):
    """pages that one write would change in several places, and settings that are tensors"""
    i32 = torch.int32
    q, t, lens, n = torch.zeros(2, 4, 16), torch.zeros(2, 2, dtype=i32), torch.zeros(2, dtype=i32), torch.zeros(2, 2, 16)
    kp, vp = torch.zeros(3, 2, 4, 16), torch.zeros(3, 2, 4, 16)
    wide = torch.zeros(1, 2, 4, 16).expand(3, 2, 4, 16)
    x = torch.zeros(2, 1, 2, 16)
    emu.paged_attention(q, kp, kp, t, lens)             # one tensor for both, and an expanded one, may be read
    emu.paged_attention(q, wide, wide, t, lens)
    c = torch.zeros(2, 3, 4, 16)
    for bad in (lambda: emu.paged_attention(q, kp, kp, t, lens, n, n), lambda: emu.paged_attention(q, wide, vp, t, lens, n, n),
                lambda: emu.paged_append(x, x, kp, kp, t, lens), lambda: emu.paged_append(x, x, kp, wide, t, lens),
                lambda: emu.paged_attention(q, kp, vp, t, lens, scale=torch.tensor(0.5)),
                lambda: emu.cross_attention(c, c, c, scale=torch.tensor(0.5)),
                lambda: emu.cross_attention(c, c, c, dropout_p=torch.tensor(0.5))):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize('D', [8, 40, 72, 96])
@pytest.mark.parametrize('dtype', [BF, F32])
def test_cross_attention_scores_of_minus_infinity_by_the_last_dimension(emu, dtype, D):
    C.infinite_scores_in_the_last_dimension_case(emu, 'cpu', dtype, D)


@pytest.mark.parametrize('dtype', [BF, F32])
@pytest.mark.parametrize('a', C.INFINITE_LAST_ROW, ids=str)
def test_cross_attention_of_an_infinite_last_row(emu, dtype, a):
    C.infinite_last_row_case(emu, 'cpu', dtype, **a)


@pytest.mark.parametrize('dtype', [BF, F32])
@pytest.mark.parametrize('a', C.INFINITE_VALUES, ids=str)
def test_decoding_with_infinite_values(emu, dtype, a):
    C.infinite_values_paged_case(emu, 'cpu', dtype, **a)


@pytest.mark.parametrize('dtype', [BF, F32])
@pytest.mark.parametrize('Tk', [40, 1300])
def test_cross_attention_of_a_row_without_a_softmax(emu, dtype, Tk):
    C.no_softmax_case(emu, 'cpu', dtype, Tk)


@pytest.mark.parametrize('V', [3, 700, 12000, 33000])
def test_sample_rows_of_nan_among_minus_infinities(emu, V):
    C.nan_among_minus_infinities_case(emu, 'cpu', V)


@pytest.mark.parametrize('tokens', [1, 40])
def test_cross_attention_of_dual_tensors(emu, tokens):
    C.forward_mode_case(emu, 'cpu', tokens)
    C.forward_mode_case(emu, 'cpu', tokens, 0.1)


def test_paged_attention_has_no_backward_pass(emu):
    C.no_backward_case(emu, 'cpu')


def test_pages_that_autograd_has_saved(emu):
    C.overwritten_pages_case(emu, 'cpu')


def test_c_entries_of_cross_attention_without_queries_or_keys(emu):
    """nothing is read or written, in both directions"""
    from neural_sp_amd import _lib
    for B, Tq, Tk in ((0, 3, 4), (2, 0, 4), (2, 3, 0)):
        sizes = emu._CROSS_TAIL(B, 2, 2, 16, Tq, Tk, 0, *(512, 32, 16) * 3, 0.25, 0.0)
        for name in ('nsp_cross_attn_fwd', 'nsp_cross_attn_bwd'):
            assert getattr(_lib.lib(), name)(emu._CROSS_PTRS(*[0] * 11, 512, 32, 16, 0, 0) + sizes, 0) == 0


def test_cross_attention_of_tokens_far_apart(emu):
    C.far_tokens_case(emu, 'cpu')


@pytest.mark.parametrize('page', [16, 5])
def test_paged_attention_of_more_pages_than_an_int_counts(emu, page):
    C.many_pages_case(emu, 'cpu', page)


@pytest.mark.parametrize('dtype', [BF, F32])
@pytest.mark.parametrize('a', C.DROPOUT_WIDTHS, ids=str)
def test_cross_attention_dropout_widths(emu, dtype, a):
    C.dropout_widths_case(emu, 'cpu', dtype, **a)


@pytest.mark.parametrize('dtype', [BF, F32])
@pytest.mark.parametrize('V,kw', C.SAMPLE_WIDE, ids=str)
def test_sample_rows_wide(emu, dtype, V, kw):
    C.wide_case(emu, 'cpu', dtype, V, kw)


def test_c_entry_of_decode_attention_over_no_state(emu):
    """table == NULL, width 0: there is no key, so zeros"""
    from neural_sp_amd import _lib
    q, out = torch.ones(2, 1, 2, 16), torch.full((2, 1, 2, 16), 7.0)
    tail, floats = emu._decode_tail(2, 2, 2, 16, 1, 1, 0, 0, F32, (32, 32, 16), (0, 32, 16), (0, 32, 16), (0, 0, 0, 0), 0.25)
    assert floats == 0
    assert _lib.lib().nsp_decode_attn(emu._DECODE_PTRS(q.data_ptr(), out.data_ptr(), 0, 0, 0, 0, 0, 0, 0) + tail, 0) == 0
    assert not out.any()
