"""Cached decoding and the fused source attention through the model, on the device."""
import pytest
import torch

from tests import decoder_serving_common as S

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def random_state_of_the_process():
    """the tests behind these draw the numbers and the dropout masks that they draw without them"""
    from neural_sp_amd import ops
    was = dict(ops._DROPOUT_STATE)
    with torch.random.fork_rng():
        yield
    ops._DROPOUT_STATE.update(was)


@pytest.mark.parametrize('settings', [dict(temperature=0.0), dict(), dict(temperature=0.8, top_k=7, top_p=0.9, min_p=0.01)], ids=str)
def test_sample_is_what_the_training_path_gives_token_by_token(settings):
    from neural_sp_amd import ops
    with ops.compute_mode('f32'):
        S.sample_case('cuda', settings)


def test_sample_in_bf16_mode():
    """the throughput mode draws from nearly the same distribution: logits of the cached path on a fixed prefix against the
    uncached ones would need the same roundings; here it has to run, to end and to repeat"""
    from neural_sp_amd import ops
    with ops.compute_mode('bf16'):
        model = S.tiny_model('cuda')
        model.eval()
        eouts, elens = S.states('cuda')
        a, _ = model.dec_fwd.sample(eouts, elens, seed=1)
        b, _ = model.dec_fwd.sample(eouts, elens, seed=1)
        assert [x.tolist() for x in a] == [x.tolist() for x in b]
        assert all(0 <= int(t) < 37 for x in a for t in x)


def test_sample_ends_with_the_position_table():
    S.position_table_case('cuda')


def test_decode_samples_when_asked():
    S.decode_case('cuda')


def test_fused_source_attention_in_a_training_step(monkeypatch):
    S.fused_training_case('cuda', monkeypatch, 'f32', 1e-4, 2e-3)


def test_fused_source_attention_in_a_bf16_training_step(monkeypatch):
    S.fused_bf16_case('cuda', monkeypatch)


def test_paged_cache_hands_out_pages():
    S.cache_case('cuda')
    torch.cuda.synchronize()


def test_paged_cache_rows_from_the_end_and_wrong_ones():
    S.cache_rows_case('cuda')


def test_logits_of_cached_steps_in_bf16_mode(monkeypatch):
    S.bf16_logits_case('cuda', monkeypatch)
