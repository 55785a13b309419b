"""Norm and rotation of heads, quantised rows into the paged caches and back, on the GPU against their formulas in 64 bits (the
quantisation, whose whole numbers have one right value, against its fp32 operations one by one)."""
import math

import numpy as np
import pytest
import torch

import pypto_b200 as pto
from pypto_b200 import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F16 = torch.bfloat16, torch.float16


def rand(*shape, dtype=BF, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


# ---- norm and rotation ----------------------------------------------------------------------------------------------
def want_heads(x, w, positions, rotary, layout, last, eps):
    """The definition in 64 bits, and the magnitude that fp32 errors scale with."""
    y = x.double()
    if w is not None:
        y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    size = y.abs()
    if rotary is not None:
        r = rotary.rotary_dim
        at = y.shape[-1] - r if last else 0
        angle = positions.double()[:, None, None] * torch.tensor(rotary.inv_freq, dtype=torch.float64)
        cos, sin = angle.cos() * rotary.amplitude, angle.sin() * rotary.amplitude
        z = y[..., at:at + r].clone()
        a, b = (z[..., :r // 2], z[..., r // 2:]) if layout == "half" else (z[..., 0::2], z[..., 1::2])
        p, q, s = a * cos - b * sin, a * sin + b * cos, (a.abs() + b.abs()) * abs(rotary.amplitude)
        y, size = y.clone(), size.clone()
        if layout == "interleaved":
            y[..., at:at + r], size[..., at:at + r] = torch.stack([p, q], -1).flatten(-2), torch.stack([s, s], -1).flatten(-2)
        else:
            y[..., at:at + r], size[..., at:at + r] = torch.cat([p, q], -1), torch.cat([s, s], -1)
    return y, size


def close_heads(got, x, w, positions, rotary, layout, last, eps=1e-6):
    """One rounding (half a step of the type), and fp32: sum of up to 256 squares, reciprocal root, angle (2^-25 of half a turn), cosine,
    two products: below 24 steps of 2^-23 of the pair's magnitude. f16 below its normal range has an absolute half step."""
    want, size = want_heads(x.cpu(), w.cpu() if w is not None else None, positions.cpu() if positions is not None else None, rotary,
                            layout, last, eps)
    half = torch.finfo(got.dtype).eps / 2
    bound = half * want.abs() + 24 * 2.0 ** -23 * size * (1 + half) + (2.0 ** -25 if got.dtype == F16 else 0)
    err = (got.cpu().double() - want).abs()
    assert bool((err <= bound).all()), (err - bound).max()


@pytest.mark.parametrize("t,hq,hk,dq,dk,r,layout,last,norm,dtype", [
    (1, 1, 1, 16, 16, 16, "half", False, True, BF),
    (64, 32, 8, 128, 128, 128, "half", False, True, BF),
    (65, 32, 8, 128, 128, 64, "interleaved", True, True, F16),
    (33, 128, 1, 192, 64, 64, "deinterleave", True, False, BF),
    (7, 5, 3, 96, 96, 32, "half", True, True, F16),
    (3, 3, 2, 256, 256, 128, "deinterleave", False, True, BF),
    (5, 7, 1, 24, 40, 16, "interleaved", False, False, BF),
    (6000, 9, 2, 64, 64, 64, "half", False, False, F16),
    (5001, 4, 1, 128, 128, 48, "half", True, True, BF),
])
def test_heads_follow_the_definition(t, hq, hk, dq, dk, r, layout, last, norm, dtype):
    q, k = rand(t, hq, dq, dtype=dtype, seed=1, scale=1.7).to(DEV), rand(t, hk, dk, dtype=dtype, seed=2, scale=0.5).to(DEV)
    wq, wk = (rand(dq, dtype=dtype, seed=3).to(DEV), rand(dk, dtype=dtype, seed=4).to(DEV)) if norm else (None, None)
    pos = (torch.arange(t) * 37 % 5000).to(DEV)
    rot = pto.RotaryFrequencies(r)
    qo, ko = torch.full_like(q, 7), torch.full_like(k, 7)
    pto.qk_norm_rope(q, k, pos, rot, qo, ko, query_weight=wq, key_weight=wk, layout=layout, rope_last=last)
    close_heads(qo, q, wq, pos, rot, layout, last)
    close_heads(ko, k, wk, pos, rot, layout, last)
    # in place, and with 32-bit positions: the same bits
    pto.qk_norm_rope(q, k, pos.int(), rot, q, k, query_weight=wq, key_weight=wk, layout=layout, rope_last=last)
    assert torch.equal(q, qo) and torch.equal(k, ko)


@pytest.mark.parametrize("scaling", [None, dict(type="linear", factor=4), dict(type="ntk", factor=8.0),
                                     dict(type="yarn", factor=40, original_max_position=4096),
                                     dict(type="by_wavelength", factor=8, low_freq_factor=1, high_freq_factor=4,
                                          original_max_position=8192)], ids=lambda s: s["type"] if s else "none")
def test_far_positions_keep_their_angles(scaling):
    pos = torch.tensor([0, 1, 131071, 1 << 20, (1 << 31) - 1, -5, 999_999_937])
    rot = pto.RotaryFrequencies(64, 10000.0, scaling=scaling)
    x = rand(len(pos), 2, 64, dtype=F16, seed=5).to(DEV)
    out = torch.empty_like(x)
    pto.qk_norm_rope(x, None, pos.to(DEV), rot, out, None)
    # (64-bit angles of positions up to 2^31 are themselves within 2^31 * 2^-53 * 2 of the exact ones: 5e-7)
    want, size = want_heads(x.cpu(), None, pos, rot, "half", False, 0)
    err = (out.cpu().double() - want).abs()
    assert bool((err <= 2.0 ** -11 * want.abs() + 5e-6 * size + 2.0 ** -25).all()), err.max()


def test_views_of_a_fused_projection_in_place():
    t, hq, hk, d = 70, 8, 2, 128
    buf = rand(t, (hq + 2 * hk) * d, seed=6).to(DEV)
    before = buf.clone()
    q, k = buf[:, :hq * d].view(t, hq, d), buf[:, hq * d:(hq + hk) * d].view(t, hk, d)
    wq, wk = rand(d, seed=7).to(DEV), rand(d, seed=8).to(DEV)
    pos, rot = torch.arange(t, device=DEV), pto.RotaryFrequencies(128)
    pto.qk_norm_rope(q, k, pos, rot, q, k, query_weight=wq, key_weight=wk)
    close_heads(q, before[:, :hq * d].view(t, hq, d), wq, pos, rot, "half", False)
    close_heads(k, before[:, hq * d:(hq + hk) * d].view(t, hk, d), wk, pos, rot, "half", False)
    assert torch.equal(buf[:, (hq + hk) * d:], before[:, (hq + hk) * d:])


def test_heads_first_storage_and_a_head_that_all_tokens_share():
    t, h, d = 19, 6, 64
    q = rand(h, t, d, seed=9).to(DEV).transpose(0, 1)
    k = rand(1, 1, d, seed=10).to(DEV).expand(t, 3, d)
    ko = torch.empty(t, 3, d, dtype=BF, device=DEV)
    qo = torch.empty(h, t, d, dtype=BF, device=DEV).transpose(0, 1)
    pos, rot = torch.arange(t, device=DEV) + 100, pto.RotaryFrequencies(32)
    pto.qk_norm_rope(q, k, pos, rot, qo, ko, layout="interleaved", rope_last=True)
    close_heads(qo, q, None, pos, rot, "interleaved", True)
    close_heads(ko, k, None, pos, rot, "interleaved", True)


def test_pairs_taken_apart_in_place():
    """Every lane writes dims that two others have read."""
    pos, rot = torch.arange(333, device=DEV), pto.RotaryFrequencies(192)
    x = rand(333, 9, 256, seed=31).to(DEV)
    y = x.clone()
    pto.qk_norm_rope(y, None, pos, rot, y, None, layout="deinterleave", rope_last=True)
    close_heads(y, x, None, pos, rot, "deinterleave", True)


def test_dims_that_are_not_rotated_are_copied_whatever_they_are():
    for layout, last in (("half", False), ("interleaved", True), ("deinterleave", True)):
        x = rand(9, 2, 96, seed=30).to(DEV)
        at = 5 if last else 90
        x[4, 1, at], x[5, 0, at], x[6, 0, at + 1] = math.inf, -math.inf, math.nan
        out = torch.empty_like(x)
        pto.qk_norm_rope(x, None, torch.arange(9, device=DEV), pto.RotaryFrequencies(64), out, None, layout=layout, rope_last=last)
        kept = slice(0, 32) if last else slice(64, 96)
        assert torch.equal(out[..., kept].isnan(), x[..., kept].isnan())
        assert torch.equal(out[..., kept].nan_to_num(3), x[..., kept].nan_to_num(3))
        assert bool(out[..., 32:].isfinite().all() if last else out[..., :64].isfinite().all())


def test_one_side_with_a_norm():
    q, k = rand(50, 4, 128, seed=31).to(DEV), rand(50, 2, 128, seed=32).to(DEV)
    w, pos, rot = rand(128, seed=33).to(DEV), torch.arange(50, device=DEV), pto.RotaryFrequencies(64)
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    pto.qk_norm_rope(q, k, pos, rot, qo, ko, key_weight=w)
    close_heads(qo, q, None, pos, rot, "half", False)
    close_heads(ko, k, w, pos, rot, "half", False)


def test_norm_alone_and_rows_of_zeros():
    x = rand(40, 4, 128, seed=11).to(DEV)
    x[3] = 0
    w = rand(128, seed=12).to(DEV)
    out = torch.empty_like(x)
    pto.qk_norm_rope(x, None, None, None, out, None, query_weight=w, eps=1e-5)
    close_heads(out, x, w, None, None, "half", False, 1e-5)
    assert bool((out[3] == 0).all())
    pto.qk_norm_rope(x[:0], None, None, None, out[:0], None, query_weight=w)


# ---- quantised rows ---------------------------------------------------------------------------------------------
def quantised(x, f16_scales=False):
    """q = rint(x * (127 / max)), scale = 1 / (127 / max) per 128 dims, every operation rounded to fp32."""
    y = x.float().numpy().reshape(x.shape[0], -1, 128)
    top = np.abs(y).max(-1, keepdims=True)
    with np.errstate(all="ignore"):
        up = np.where(top < 2.0 ** -120, np.float32(0), np.float32(127) / top).astype(np.float32)
        q = np.rint(y * up).astype(np.int8)
        scale = np.where(up == 0, np.float32(0), np.float32(1) / up).astype(np.float32)[..., 0]
    return torch.from_numpy(q.reshape(x.shape[0], -1)), torch.from_numpy(scale.astype(np.float16 if f16_scales else np.float32))


def rows_of(t, width, dtype, seed):
    x = rand(t, width, dtype=dtype, seed=seed)
    x[:, ::97] *= 8
    if t > 2:
        x[1, :128] = 0
        x[2, -128:] = x[2, -128:] * 1e-4
    return x


@pytest.mark.parametrize("t,width,dtype,rope,f16_scales", [
    (1, 128, BF, False, True), (65, 512, BF, True, False), (3, 384, F16, False, False), (130, 1152, BF, False, False),
    (4099, 512, BF, True, False), (17, 512, F16, False, True)])
def test_written_rows_are_the_quantised_ones(t, width, dtype, rope, f16_scales):
    rows = 40 * 128
    x = rows_of(t, width, dtype, 13)
    xr = rand(t, 64, seed=14) if rope else None
    idx = torch.randperm(rows, generator=torch.Generator().manual_seed(15))[:t]
    kn = torch.full((rows, width), 5, dtype=torch.int8, device=DEV)
    sc = torch.full((rows, width // 128), 3.0, dtype=F16 if f16_scales else torch.float32, device=DEV)
    kr = torch.full((rows, 64), 2.0, dtype=BF, device=DEV) if rope else None
    packed = torch.full((rows, 656), 9, dtype=torch.int8, device=DEV) if rope else None
    pto.kv_cache_write(x.to(DEV), xr.to(DEV) if rope else None, idx.to(DEV), kn, kr, sc, packed_kv_cache=packed)
    assert pto.workspace_status()[0] == 0
    q, s = quantised(x, f16_scales)
    want, want_s = torch.full((rows, width), 5, dtype=torch.int8), torch.full(sc.shape, 3.0, dtype=sc.dtype)
    want[idx], want_s[idx] = q, s
    assert torch.equal(kn.cpu(), want) and torch.equal(sc.cpu(), want_s)
    if rope:
        want_r = torch.full((rows, 64), 2.0, dtype=BF)
        want_r[idx] = xr
        assert torch.equal(kr.cpu(), want_r)
        again = torch.full((rows, 656), 9, dtype=torch.int8, device=DEV)
        pto.pack_kv_cache(kn, kr, sc, again)
        assert torch.equal(packed.cpu()[idx], again.cpu()[idx])
        rest = torch.ones(rows, dtype=torch.bool)
        rest[idx] = False
        assert bool((packed.cpu()[rest] == 9).all())
        alone = torch.full((rows, 656), 9, dtype=torch.int8, device=DEV)
        pto.kv_cache_write(x.to(DEV), xr.to(DEV), idx.to(DEV), None, None, None, packed_kv_cache=alone)
        assert torch.equal(alone, packed)


def test_rows_of_a_wider_projection_padding_and_indices_outside():
    t, rows = 9, 256
    kv = rand(t, 576, seed=16).to(DEV)
    idx = torch.tensor([4, -1, 255, rows, 7, -1, -2, 0, 1 << 40], device=DEV)
    kn, kr = torch.zeros(rows, 512, dtype=torch.int8, device=DEV), torch.zeros(rows, 64, dtype=BF, device=DEV)
    sc = torch.zeros(rows, 4, device=DEV)
    pto.reset_workspace_status()
    pto.kv_cache_write(kv[:, :512], kv[:, 512:], idx, kn, kr, sc)
    assert pto.workspace_status()[0] == _lib.PTO_ST_BAD_PAGE
    pto.reset_workspace_status()
    q, s = quantised(kv[:, :512].cpu())
    want, want_r = torch.zeros(rows, 512, dtype=torch.int8), torch.zeros(rows, 64, dtype=BF)
    for i, at in enumerate(idx.tolist()):
        if 0 <= at < rows:
            want[at], want_r[at] = q[i], kv[i, 512:].cpu()
    assert torch.equal(kn.cpu(), want) and torch.equal(kr.cpu(), want_r)
    # padding alone is no error
    pto.kv_cache_write(kv[:2, :512], kv[:2, 512:], torch.full((2,), -1, device=DEV), kn, kr, sc)
    assert pto.workspace_status()[0] == 0 and torch.equal(kn.cpu(), want)
    pto.kv_cache_write(kv[:0, :512], kv[:0, 512:], idx[:0], kn, kr, sc)


def test_groups_that_are_not_numbers_and_tiny_ones():
    x = rand(4, 512, seed=17)
    x[0, 5], x[1, 200], x[2, 300] = math.nan, math.inf, -math.inf
    x[3, :128] = 2.0 ** -126
    kn, sc = torch.zeros(128, 512, dtype=torch.int8, device=DEV), torch.zeros(128, 4, device=DEV)
    pto.kv_cache_write(x.to(DEV), None, torch.arange(4, device=DEV), kn, None, sc)
    s = sc.cpu()
    assert math.isnan(s[0, 0]) and not math.isfinite(s[1, 1]) and not math.isfinite(s[2, 2])
    assert s[3, 0] == 0 and bool((kn[3, :128] == 0).all())
    cu, table = torch.tensor([0, 4], dtype=torch.int32, device=DEV), torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    out = torch.empty(4, 512, dtype=BF, device=DEV)
    pto.kv_cache_read(kn, None, sc, table, cu, out, None)
    back = out.cpu().float()
    assert not bool(back[0, :128].isfinite().any()) and not bool(back[1, 128:256].isfinite().any())
    assert bool(back[0, 128:].isfinite().all()) and bool(back[1, :128].isfinite().all()) and bool((back[3, :128] == 0).all())


@pytest.mark.parametrize("lens,width,dtype,form,block,with_first", [
    ([129], 512, BF, "packed", 128, False), ([1, 0, 300, 17, 0], 512, BF, "split", 128, True), ([5, 64], 128, F16, "split", 1, False),
    ([1000, 3, 77] * 12, 512, BF, "split", 16, True), ([250], 1152, BF, "split", 128, False),
    ([9000, 11000, 1, 30000], 512, BF, "packed", 128, True)])
def test_rows_read_back(lens, width, dtype, form, block, with_first):
    g = torch.Generator().manual_seed(18)
    b, groups = len(lens), width // 128
    first = [7 * i % 50 if with_first else 0 for i in range(b)]
    need = [-(-(f + n) // block) for f, n in zip(first, lens)]
    pages = sum(need) + 3
    rows = pages * block
    kn = torch.randint(-128, 128, (rows, width), generator=g, dtype=torch.int8)
    kr, sc = torch.randn(rows, 64, generator=g).to(BF), torch.rand(rows, groups, generator=g) * 0.05
    order = torch.randperm(pages, generator=g)
    table = torch.full((b, max(need) + 1), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    cu = torch.tensor([0] + lens).cumsum(0).int()
    total, extra = int(cu[-1]), 5
    rope = dtype == BF and width == 512
    out = torch.full((total + extra, width + 64), 7.0, dtype=dtype, device=DEV)
    ro = torch.full((total + extra, 64), 7.0, dtype=BF, device=DEV) if rope else None
    args = (kn.to(DEV), kr.to(DEV) if rope else None, sc.to(DEV))
    packed = None
    if form == "packed":
        packed = torch.cat([kn, kr.view(torch.int8), sc.view(torch.int8)], 1).to(DEV)
        args = (None, None, None)
    pto.kv_cache_read(*args, table.to(DEV), cu.to(DEV), out[:, :width], ro, block,
                      first=torch.tensor(first, dtype=torch.int32, device=DEV) if with_first else None, packed_kv_cache=packed)
    assert pto.workspace_status()[0] == 0
    src = torch.cat([table[i, (f + torch.arange(n)) // block].long() * block + (f + torch.arange(n)) % block
                     for i, (f, n) in enumerate(zip(first, lens))])
    want = (kn[src].float().view(total, groups, 128) * sc[src][..., None]).view(total, width).to(dtype)
    assert torch.equal(out[:total, :width].cpu(), want)
    assert bool((out[total:] == 7).all()) and bool((out[:, width:] == 7).all())
    if rope:
        assert torch.equal(ro[:total].cpu(), kr[src]) and bool((ro[total:] == 7).all())


def test_positions_without_a_page_read_as_zeros():
    kn, sc = torch.ones(256, 128, dtype=torch.int8, device=DEV), torch.ones(256, 1, device=DEV)
    table = torch.tensor([[1, -1, 0], [0, 2, 1]], dtype=torch.int32, device=DEV)  # page 2 is outside
    cu = torch.tensor([0, 300, 700], dtype=torch.int32, device=DEV)  # 400 positions of 384 in the table
    out = torch.full((700, 128), 7.0, dtype=BF, device=DEV)
    pto.reset_workspace_status()
    pto.kv_cache_read(kn, None, sc, table, cu, out, None)
    assert pto.workspace_status()[0] == _lib.PTO_ST_BAD_PAGE
    pto.reset_workspace_status()
    want = torch.ones(700, 128)
    want[128:256] = 0
    want[300 + 128:300 + 256] = 0
    want[300 + 384:] = 0
    assert torch.equal(out.cpu().float(), want)


def test_offsets_beyond_32_bits():
    rows = (1 << 31) // 512 + 4096  # an int8 cache of 2.1 GB
    kn, sc = torch.zeros(rows, 512, dtype=torch.int8, device=DEV), torch.zeros(rows, 4, device=DEV)
    x = rand(300, 512, seed=19).to(DEV)
    idx = torch.arange(rows - 300, rows, device=DEV)
    pto.kv_cache_write(x, None, idx, kn, None, sc)
    table = torch.arange((rows - 384) // 128, rows // 128, dtype=torch.int32, device=DEV)[None]
    cu = torch.tensor([0, 300], dtype=torch.int32, device=DEV)
    out = torch.empty(300, 512, dtype=BF, device=DEV)
    pto.kv_cache_read(kn, None, sc, table, cu, out, None, first=torch.tensor([84], dtype=torch.int32, device=DEV))
    q, s = quantised(x.cpu())
    assert torch.equal(out.cpu(), (q.float().view(300, 4, 128) * s[..., None]).view(300, 512).to(BF))
    assert pto.workspace_status()[0] == 0


def test_recorded_calls_see_new_rows():
    kn, sc = torch.zeros(512, 512, dtype=torch.int8, device=DEV), torch.zeros(512, 4, device=DEV)
    kr = torch.zeros(512, 64, dtype=BF, device=DEV)
    x, xr = rand(33, 512, seed=20).to(DEV), rand(33, 64, seed=21).to(DEV)
    idx = torch.arange(100, 133, device=DEV)
    step = pto.CapturedCall(pto.kv_cache_write, x, xr, idx, kn, kr, sc)
    x.copy_(rand(33, 512, seed=22))
    idx.add_(200)
    step.replay()
    q, s = quantised(x.cpu())
    assert torch.equal(kn[300:333].cpu(), q) and torch.equal(sc[300:333].cpu(), s) and torch.equal(kr[300:333], xr)
