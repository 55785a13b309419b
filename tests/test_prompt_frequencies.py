"""Scaled rotary frequencies against what their kinds mean, counted out pair by pair in numpy (64 bits)."""
import math

import numpy as np
import pytest

import pypto_b200 as pto


def plain(r, base):
    return np.exp(-np.arange(r // 2) * (2.0 / r) * np.log(base))


def close(rotary, want):
    # powers, logarithms and a blend in 64 bits: a few steps of 2^-53, more where the base's power multiplies them by log(base)
    np.testing.assert_allclose(rotary.inv_freq, want, rtol=2.0 ** -44)
    turns = np.array([t % (1 << 64) for t in rotary.turns.tolist()], dtype=object)
    for f, t in zip(want, turns):  # what the kernel reads: half a step of 2^-64 turns, and the above
        assert abs(float(t) / 2.0 ** 64 * 2 * math.pi - f) <= 2.0 ** -64 * math.pi + 2.0 ** -44 * f


@pytest.mark.parametrize("r,base,trained,factor,betas,attention", [
    (64, 10000.0, 4096, 40.0, {}, None),
    (128, 10000.0, 32768, 4.0, {}, None),
    (128, 500000.0, 8192, 16.0, dict(beta_fast=16.0, beta_slow=2.0), None),
    (32, 150000.0, 4096, 2.5, dict(beta_fast=48.0), 1.0),
    (64, 10000.0, 2048, 8.0, dict(beta_slow=0.5), 0.75),
])
def test_yarn_slows_the_pairs_that_turn_seldom(r, base, trained, factor, betas, attention):
    s = dict(type="yarn", factor=factor, original_max_position=trained, **betas)
    if attention is not None:
        s["attention_factor"] = attention
    rotary = pto.RotaryFrequencies(r, base, scaling=s, device="cpu")
    f = plain(r, base)
    turns = trained * f / (2 * math.pi)  # of a pair over the trained length; fewer from pair to pair
    kept = np.flatnonzero(turns >= betas.get("beta_fast", 32.0))
    slowed = np.flatnonzero(turns <= betas.get("beta_slow", 1.0))
    assert len(kept) and len(slowed) and slowed[0] - kept[-1] > 2  # (there is a ramp to look at)
    keep = np.ones(r // 2)
    for i in range(r // 2):  # a line over the pairs from the last one that is kept to the first one that is slowed
        if i >= slowed[0]:
            keep[i] = 0.0
        elif i > kept[-1]:
            keep[i] = (slowed[0] - i) / (slowed[0] - kept[-1])
    close(rotary, f * keep + f / factor * (1 - keep))
    assert rotary.amplitude == pytest.approx(1 + math.log(factor) / 10 if attention is None else attention, rel=1e-14)


@pytest.mark.parametrize("r,base,trained,factor,lo,hi", [
    (128, 500000.0, 8192, 8.0, 1.0, 4.0), (64, 500000.0, 8192, 32.0, 1.0, 4.0), (64, 10000.0, 2048, 3.0, 0.5, 16.0)])
def test_by_wavelength_blends_between_two_wavelengths(r, base, trained, factor, lo, hi):
    rotary = pto.RotaryFrequencies(r, base, scaling=dict(type="by_wavelength", factor=factor, low_freq_factor=lo, high_freq_factor=hi,
                                                         original_max_position=trained), device="cpu")
    want, between = [], 0
    for f in plain(r, base):
        wave = 2 * math.pi / f
        if wave < trained / hi:
            want.append(f)
        elif wave > trained / lo:
            want.append(f / factor)
        else:
            smooth = (trained / wave - lo) / (hi - lo)
            want.append((1 - smooth) * f / factor + smooth * f)
            between += 1
    assert between > 1
    close(rotary, np.array(want))
    assert rotary.amplitude == 1.0


@pytest.mark.parametrize("r,base", [(16, 10000.0), (128, 1e6), (256, 1.5)])
def test_plain_linear_and_ntk(r, base):
    f = plain(r, base)
    close(pto.RotaryFrequencies(r, base, device="cpu"), f)
    close(pto.RotaryFrequencies(r, base, scaling=dict(type="linear", factor=3.0), device="cpu"), f / 3)
    # the slowest pair factor times slower, the others by the same power of their place
    place = np.arange(r // 2) / (r // 2 - 1)
    close(pto.RotaryFrequencies(r, base, scaling=dict(type="ntk", factor=6.0), device="cpu"), f * 6.0 ** -place)
