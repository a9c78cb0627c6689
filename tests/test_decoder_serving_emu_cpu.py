"""Cached decoding and the fused source attention through the model, on the host emulator of the kernels."""
import pytest
import torch

from tests import decoder_serving_common as S
from tests.hipemu import build_emu

pytestmark = pytest.mark.skipif(not build_emu.available(), reason='no host clang++ for the HIP emulator')


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
    from tests.cpu_ops_shim import host_logic_on_cpu
    with host_logic_on_cpu(real_kernels=True, real_conv=False):
        yield


@pytest.mark.parametrize('settings', [dict(temperature=0.0), dict(), dict(temperature=0.8, top_k=7, top_p=0.9, min_p=0.01)], ids=str)
def test_sample_is_what_the_training_path_gives_token_by_token(emu, settings):
    S.sample_case('cpu', settings)


def test_sample_ends_with_the_position_table(emu):
    S.position_table_case('cpu')


def test_decode_samples_when_asked(emu):
    S.decode_case('cpu')


def test_fused_source_attention_in_a_training_step(emu, monkeypatch):
    S.fused_training_case('cpu', monkeypatch, 'f32', 1e-4, 2e-3)


def test_paged_cache_hands_out_pages():
    S.cache_case('cpu')


def test_paged_cache_rows_from_the_end_and_wrong_ones():
    S.cache_rows_case('cpu')


def test_logits_of_cached_steps_in_bf16_mode(emu, monkeypatch):
    S.bf16_logits_case('cpu', monkeypatch)
