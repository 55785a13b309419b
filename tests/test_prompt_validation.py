"""Operators around a prompt: calls that are refused, before anything is launched, and the frequencies."""
import math

import pytest
import torch

import pypto_b200 as pto
from pypto_b200 import _lib

BF = torch.bfloat16


def heads(**over):
    t, hq, hk, d = 5, 4, 2, 64
    a = dict(query=torch.zeros(t, hq, d, dtype=BF), key=torch.zeros(t, hk, d, dtype=BF), positions=torch.arange(t),
             rotary=pto.RotaryFrequencies(32, device="cpu"), query_out=torch.zeros(t, hq, d, dtype=BF),
             key_out=torch.zeros(t, hk, d, dtype=BF))
    a.update(over)
    return a


@pytest.mark.parametrize("over,exc", [
    ({}, RuntimeError),  # no CPU path
    (dict(query=torch.zeros(5, 4, 64)), ValueError),
    (dict(query=torch.zeros(5, 4 * 64, dtype=BF)), ValueError),
    (dict(query=torch.zeros(5, 64, 4, dtype=BF).transpose(1, 2)), ValueError),
    (dict(query=torch.zeros(5, 4, 68, dtype=BF)[..., :64]), ValueError),  # rows off 16-byte boundaries
    (dict(query_out=torch.zeros(5, 4, 64, dtype=torch.float16)), ValueError),
    (dict(key_out=None), ValueError),
    (dict(key=torch.zeros(6, 2, 64, dtype=BF), key_out=torch.zeros(6, 2, 64, dtype=BF)), ValueError),
    (dict(positions=torch.arange(4)), ValueError),
    (dict(positions=torch.arange(5).float()), ValueError),
    (dict(query_weight=torch.ones(64)), ValueError),
    (dict(key_weight=torch.ones(32, dtype=BF)), ValueError),
    (dict(layout="sideways"), ValueError),
    (dict(rotary=10000.0), ValueError),
    (dict(eps=-1.0), ValueError),
    (dict(eps=math.nan), ValueError),
    (dict(query=[1, 2]), TypeError),
])
def test_norm_rope_refuses(over, exc):
    with pytest.raises(exc):
        pto.qk_norm_rope(**heads(**over))


def cache(**over):
    a = dict(key_nope=torch.zeros(3, 512, dtype=BF), key_rope=torch.zeros(3, 64, dtype=BF), cache_index=torch.arange(3),
             key_nope_2d=torch.zeros(128, 512, dtype=torch.int8), key_rope_2d=torch.zeros(128, 64, dtype=BF),
             k_nope_scales=torch.zeros(128, 4))
    a.update(over)
    return a


@pytest.mark.parametrize("over,exc", [
    ({}, RuntimeError),
    (dict(key_nope=torch.zeros(3, 500, dtype=BF)), ValueError),
    (dict(key_nope=torch.zeros(3, 512)), ValueError),
    (dict(cache_index=torch.arange(3).int()), ValueError),
    (dict(cache_index=torch.arange(4)), ValueError),
    (dict(key_rope=None), ValueError),
    (dict(key_rope_2d=None), ValueError),
    (dict(k_nope_scales=torch.zeros(128, 3)), ValueError),
    (dict(k_nope_scales=torch.zeros(128, 4, dtype=BF)), ValueError),
    (dict(key_nope_2d=None), ValueError),
    (dict(key_nope_2d=None, key_rope_2d=None, k_nope_scales=None), ValueError),
    (dict(packed_kv_cache=torch.zeros(127, 656, dtype=torch.int8)), ValueError),
    (dict(key_nope_2d=torch.zeros(512, 128, dtype=torch.int8).t()), RuntimeError),
])
def test_cache_write_refuses(over, exc):
    with pytest.raises(exc):
        pto.kv_cache_write(**cache(**over))


def read(**over):
    a = dict(key_nope_2d=torch.zeros(128, 512, dtype=torch.int8), key_rope_2d=torch.zeros(128, 64, dtype=BF),
             k_nope_scales=torch.zeros(128, 4), block_table=torch.zeros(2, 1, dtype=torch.int32),
             cu_seqlens=torch.tensor([0, 3, 5], dtype=torch.int32), key_nope_out=torch.zeros(5, 512, dtype=BF),
             key_rope_out=torch.zeros(5, 64, dtype=BF))
    a.update(over)
    return a


@pytest.mark.parametrize("over,exc", [
    ({}, RuntimeError),
    (dict(packed_kv_cache=torch.zeros(128, 656, dtype=torch.int8)), ValueError),
    (dict(key_nope_2d=None), ValueError),
    (dict(key_rope_2d=None), ValueError),
    (dict(cu_seqlens=torch.tensor([0, 3, 5])), ValueError),
    (dict(block_table=torch.zeros(3, 1, dtype=torch.int32)), ValueError),
    (dict(key_rope_out=torch.zeros(4, 64, dtype=BF)), ValueError),
    (dict(key_nope_out=torch.zeros(5, 512, dtype=torch.float16)), ValueError),
    (dict(block_size=0), ValueError),
    (dict(block_size=(1 << 32) + 1), ValueError),
    (dict(first=torch.zeros(3, dtype=torch.int32)), ValueError),
])
def test_cache_read_refuses(over, exc):
    with pytest.raises(exc):
        pto.kv_cache_read(**read(**over))


def prompt(**over):
    a = dict(query=torch.zeros(5, 4, 128, dtype=BF), key=torch.zeros(9, 2, 128, dtype=BF), value=torch.zeros(9, 2, 128, dtype=BF),
             cu_seqlens_q=torch.tensor([0, 2, 5], dtype=torch.int32), cu_seqlens_k=torch.tensor([0, 4, 9], dtype=torch.int32),
             attention_out=torch.zeros(5, 4, 128, dtype=BF))
    a.update(over)
    return a


@pytest.mark.parametrize("over,exc", [
    ({}, RuntimeError),
    (dict(query=torch.zeros(5, 3, 128, dtype=BF), attention_out=torch.zeros(5, 3, 128, dtype=BF)), ValueError),  # heads
    (dict(query=torch.zeros(5, 4, 96, dtype=BF)), ValueError),
    (dict(key=torch.zeros(9, 2, 64, dtype=BF)), ValueError),
    (dict(value=torch.zeros(8, 2, 128, dtype=BF)), ValueError),
    (dict(value=torch.zeros(9, 2, 64, dtype=BF), attention_out=torch.zeros(5, 4, 64, dtype=BF)), ValueError),
    (dict(key=torch.zeros(9, 2, 128, dtype=torch.float16)), ValueError),
    (dict(query=torch.zeros(5, 4, 128)), ValueError),
    (dict(attention_out=torch.zeros(5, 4, 64, dtype=BF)), ValueError),
    (dict(cu_seqlens_q=torch.tensor([0, 2, 5])), ValueError),
    (dict(cu_seqlens_k=torch.tensor([0, 9], dtype=torch.int32)), ValueError),
    (dict(softmax_scale=0.0), ValueError),
    (dict(softmax_scale=-1.0), ValueError),
    (dict(softmax_scale=math.nan), ValueError),
    (dict(lse_out=torch.zeros(5, 4)), ValueError),
    (dict(lse_out=torch.zeros(4, 5, dtype=BF)), ValueError),
    (dict(query=torch.zeros(4, 5, 136, dtype=BF).transpose(0, 1)[..., 4:132]), ValueError),  # off 16-byte boundaries
    (dict(key=None), TypeError),
])
def test_prompt_attention_refuses(over, exc):
    with pytest.raises(exc):
        pto.prompt_attention(**prompt(**over))


def test_prompt_attention_workspace():
    lib = _lib.load()
    # short contexts are never cut into pieces: status words and tables only
    assert lib.pto_prompt_attention_workspace_bytes(17, 17, 1, 8, 2, 64) < 1 << 20
    # the pieces of one token's context: at most 8 x 148 of the group's rows
    one = lib.pto_prompt_attention_workspace_bytes(1, 1 << 20, 1, 8, 1, 128)
    assert 0 < one < (1 << 20) + 8 * 148 * 8 * 130 * 4
    assert lib.pto_prompt_attention_workspace_bytes(1 << 17, 1 << 17, 4, 128, 8, 128) < 200 << 20
    assert lib.pto_prompt_attention_workspace_bytes(1, 1, 0, 1, 1, 64) == 0
    assert lib.pto_prompt_attention_workspace_bytes(1 << 30, 1, (1 << 31) - 1, 1, 1, 64) == 0  # more sequences than tiles are counted for


def test_c_entries_refuse_before_any_cuda_call():
    lib = _lib.load()
    assert lib.pto_prompt_attention(None, None, None, None, None, None, None, 2, 1, 1, 1, 1, 1, 64, 64, None, 1.0, 1, None, 0,
                                    None) == -1
    assert lib.pto_qk_norm_rope(None, None, None, 0, None, None, None, None, None, 2, 1, 1, 64, 0, 64, None, 0, 0, 0, 1.0, 1e-6,
                                None) == -1
    assert lib.pto_kv_cache_write(None, 512, None, 0, None, 2, 1, 512, None, None, None, 1, None, 128, None, 0, None) == -1
    assert lib.pto_kv_cache_read(None, None, None, 1, None, 128, None, None, None, 1, 1, 128, 1, 512, None, 512, None, 0, 2, None, 0,
                                 None) == -1


def test_frequencies():
    plain = pto.RotaryFrequencies(64, device="cpu")
    assert plain.amplitude == 1.0 and plain.inv_freq[0] == 1.0 and plain.inv_freq[31] == pytest.approx(10000 ** (-62 / 64))
    turns = [t % (1 << 64) for t in plain.turns.tolist()]
    # a frequency is held to half a step of 2^-64 turns (2^-64 pi), and a few 64-bit operations
    for f, t in zip(plain.inv_freq, turns):
        assert abs(t / 2.0 ** 64 * 2 * math.pi - f) <= 2.0 ** -64 * math.pi + 2.0 ** -50 * f
    assert pto.RotaryFrequencies(64, scaling=dict(type="linear", factor=4), device="cpu").inv_freq[5] == plain.inv_freq[5] / 4
    ntk = pto.RotaryFrequencies(64, scaling=dict(type="ntk", factor=8), device="cpu")
    assert ntk.inv_freq[0] == 1.0 and ntk.inv_freq[31] == pytest.approx(plain.inv_freq[31] / 8)
    yarn = pto.RotaryFrequencies(64, scaling=dict(type="yarn", factor=40, original_max_position=4096), device="cpu")
    assert yarn.inv_freq[0] == 1.0 and yarn.inv_freq[31] == pytest.approx(plain.inv_freq[31] / 40)
    assert yarn.amplitude == pytest.approx(0.1 * math.log(40) + 1)
    wave = pto.RotaryFrequencies(64, scaling=dict(type="by_wavelength", factor=8, low_freq_factor=1, high_freq_factor=4,
                                                  original_max_position=8192), device="cpu")
    assert wave.inv_freq[0] == 1.0 and wave.inv_freq[31] == pytest.approx(plain.inv_freq[31] / 8)
    for bad in (dict(type="linear", factor=0.5), dict(type="yarn", factor=2), dict(type="spiral", factor=2),
                dict(type="linear", factor=2, offset=1)):
        with pytest.raises(ValueError):
            pto.RotaryFrequencies(64, scaling=bad, device="cpu")
    with pytest.raises(ValueError):
        pto.RotaryFrequencies(24, device="cpu")
