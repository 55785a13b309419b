"""Attention over packed prompts on the GPU against its definition in 64 bits.

Tolerance, per value, with h half a step of the rows' type and A = sum_j p_j |v_j| / sum_j p_j: the rounding of the output h |o|, of
every probability h A, and fp32: scores (12 accumulations of a value below 16, each 2^-22 of it at most: 5e-5 of a probability), value
products (a step of 16 keys each 2^-23 of the running sum: 2^-23 n / 16 A)."""
import math

import pytest
import torch

import pypto_b200 as pto
from pypto_b200 import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F16 = torch.bfloat16, torch.float16


def cu(lens):
    return torch.tensor([0] + list(lens)).cumsum(0).int().to(DEV)


def make(ql, kl, hq, hkv, dqk, dv, dtype, seed=0, extra=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    q = torch.randn(sum(ql) + extra, hq, dqk, generator=g, device=DEV).to(dtype)
    k = torch.randn(sum(kl) + extra, hkv, dqk, generator=g, device=DEV).to(dtype)
    v = torch.randn(sum(kl) + extra, hkv, dv, generator=g, device=DEV).to(dtype)
    return q, k, v


def definition(q, k, v, ql, kl, scale, causal):
    """Outputs, sum p|v| / sum p and log sum exp in 64 bits; a hidden key takes no part, whatever it holds."""
    tq, hq, _ = q.shape
    g = hq // k.shape[1]
    out = torch.zeros(tq, hq, v.shape[2], dtype=torch.float64, device=DEV)
    size, lse = torch.zeros_like(out), torch.full((hq, tq), -math.inf, dtype=torch.float64, device=DEV)
    q0 = k0 = 0
    for nq, nk in zip(ql, kl):
        seen = torch.ones(nq, nk, dtype=torch.bool, device=DEV)
        if causal:
            seen = seen.tril(nk - nq)
        some = seen.any(1)
        if nq and nk:
            for h in range(hq):
                x = (q[q0:q0 + nq, h].double() @ k[k0:k0 + nk, h // g].double().T * scale).masked_fill(~seen, -math.inf)
                lse[h, q0:q0 + nq] = torch.where(some, torch.logsumexp(x, 1), -math.inf)
                p = torch.softmax(x, 1).masked_fill(~seen, 0.0)
                vh = v[k0:k0 + nk, h // g].double()
                bad = ~vh.isfinite()
                o = p @ vh.masked_fill(bad, 0)
                if bad.any():  # a value that is not finite reaches the rows that see it
                    for j, c in bad.nonzero().tolist():
                        o[:, c] += torch.where(seen[:, j], vh[j, c], 0.0)
                out[q0:q0 + nq, h] = torch.where(some[:, None], o, 0.0)
                size[q0:q0 + nq, h] = torch.where(some[:, None], p @ vh.masked_fill(bad, 0).abs(), 0.0)
        q0, k0 = q0 + nq, k0 + nk
    return out, size, lse


def check(out, lse, q, k, v, ql, kl, scale, causal):
    n = sum(ql)
    want, size, want_lse = definition(q, k, v, ql, kl, scale, causal)
    h = torch.finfo(out.dtype).eps / 2
    bound = h * want.abs() + (h + 1e-4 + 2.0 ** -23 * max(list(kl) + [1]) / 16) * size + 1e-7
    got = out[:n].double()
    finite = want[:n].isfinite()
    assert torch.equal(got.isfinite(), finite) and torch.equal(got.isnan(), want[:n].isnan())
    assert torch.equal(got[~finite].nan_to_num(7, 8, 9), want[:n][~finite].nan_to_num(7, 8, 9))
    err = torch.where(finite, (got - want[:n]).abs() - bound[:n], -1.0)
    assert bool((err <= 0).all()), (float(err.max()), (err > 0).nonzero()[:4].tolist(), int((err > 0).sum()))
    if lse is not None:
        a, b = lse[:, :n].double(), want_lse[:, :n]
        assert torch.equal(a == -math.inf, b == -math.inf)
        d = torch.where(b == -math.inf, 0.0, (a - b).abs())
        assert bool((d <= 1e-4 + 2.0 ** -22 * b.abs().nan_to_num(0, 0, 0)).all()), float(d.max())


def run(ql, kl, hq, hkv, dqk, dv, dtype, causal=True, seed=0, scale=None, edit=None):
    q, k, v = make(ql, kl, hq, hkv, dqk, dv, dtype, seed)
    if edit is not None:
        edit(q, k, v)
    out = torch.full((sum(ql), hq, dv), 7.0, dtype=dtype, device=DEV)
    lse = torch.full((hq, sum(ql)), 7.0, device=DEV)
    pto.prompt_attention(q, k, v, cu(ql), cu(kl), out, scale, causal=causal, lse_out=lse)
    assert pto.workspace_status()[0] == 0
    check(out, lse, q, k, v, ql, kl, dqk ** -0.5 if scale is None else scale, causal)
    again = torch.empty_like(out)
    pto.prompt_attention(q, k, v, cu(ql), cu(kl), again, scale, causal=causal)
    bits = torch.int16
    assert torch.equal(again.view(bits), out.view(bits))
    return out


@pytest.mark.parametrize("dqk,dv", [(64, 64), (128, 128), (192, 128)])
@pytest.mark.parametrize("dtype", [BF, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("ql,kl,hq,hkv", [
    ([1], [1], 1, 1),
    ([17], [17], 8, 2),
    ([128], [128], 1, 1),
    ([129], [129], 2, 1),
    ([300], [300], 4, 4),
    ([700], [700], 2, 2),
    ([5, 130, 1, 64, 257], [5, 130, 1, 64, 257], 4, 2),
], ids=lambda x: str(x))
def test_prompts(ql, kl, hq, hkv, dqk, dv, dtype):
    run(ql, kl, hq, hkv, dqk, dv, dtype)


@pytest.mark.parametrize("ql,kl,hq,hkv,dqk,dv,dtype,causal", [
    ([1], [5000], 8, 1, 128, 128, BF, True),  # one token, in pieces
    ([1] * 5, [4096, 1, 129, 777, 2048], 16, 2, 128, 128, F16, True),
    ([3, 1, 2], [999, 600, 2], 12, 4, 64, 64, BF, True),
    ([200, 77], [3333, 500], 8, 2, 128, 128, BF, True),  # chunks behind earlier keys
    ([60], [9000], 5, 1, 192, 128, BF, True),
    ([40, 30], [10, 0], 4, 2, 128, 128, BF, True),  # tokens without a key
    ([0, 9, 0, 300, 0], [4, 9, 0, 100, 7], 6, 2, 64, 64, F16, True),
    ([3, 200], [0, 0], 2, 1, 128, 128, BF, True),  # no keys at all
    ([5, 0], [700, 900], 2, 2, 192, 128, F16, False),
    ([255, 1, 513], [4000, 4000, 4000], 16, 1, 64, 64, BF, True),
    ([1] * 40, [2500] * 40, 32, 8, 128, 128, BF, True),  # more items than one round
    ([50, 20], [300, 64], 4, 4, 128, 128, BF, False),
    ([600], [600], 7, 1, 128, 128, F16, True),  # groups that are no power of two
    ([33], [1000], 128, 1, 64, 64, BF, True),  # one key head for all
    ([300], [300], 200, 1, 64, 64, BF, True),
    ([8300], [8300], 8, 1, 128, 128, BF, True),  # a table of more than 256 row tiles
    ([1] * 300, list(range(1, 301)), 4, 1, 128, 128, BF, True),
    ([1000, 3000, 2000] * 2, [1000, 3000, 2000] * 2, 16, 8, 64, 64, F16, True),
    ([1], [40000], 1, 1, 192, 128, F16, False),
    ([0, 3, 0, 0, 1, 9, 2, 0] * 3 + [4] * 7, [0, 9, 5, 0, 1, 2, 16, 0] * 3 + [5, 4, 0, 8, 30, 4, 7], 2, 1, 64, 64, BF, True),  # 31 short ones
    ([0, 0, 1200, 0, 700, 0], [3, 0, 400, 0, 90, 0], 4, 1, 128, 128, F16, False),  # row tiles of two sequences between empty ones
], ids=lambda x: str(x)[:24])
def test_shapes(ql, kl, hq, hkv, dqk, dv, dtype, causal):
    run(ql, kl, hq, hkv, dqk, dv, dtype, causal)


@pytest.mark.parametrize("scale", [1e-3, 0.5, 3.0])
def test_scores_of_any_spread(scale):
    """Probabilities from nearly equal to one key's alone; a running maximum that rises late."""
    def rising(q, k, v):
        k.mul_(torch.linspace(0.05, 1.0, k.shape[0], device=DEV)[:, None, None])
    # (scores up to 3 * 128: their fp32 error, 12 * 2^-22 of 400, is 1e-3 of a probability, within the bf16 half step of 4e-3 that the
    # bound holds twice and a half of which typical roundings use)
    run([513], [513], 4, 2, 128, 128, BF, seed=3, scale=scale, edit=rising)


@pytest.mark.parametrize("dtype", [BF, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_what_a_token_does_not_see_does_not_reach_it(bad, dtype):
    ql, kl = [100, 140, 1], [100, 300, 50]

    def edit(q, k, v):
        v[60, 0, 3], v[60, 1, 100] = bad, bad  # tokens from 60 on see it
        v[100 + 299, 0, 7] = bad               # the last key of a sequence: its last token sees it
        v[100 + 10, 1, 9] = bad                # a key that all tokens of a sequence see
        v[99, 1, 0] = bad
    out = run(ql, kl, 8, 2, 128, 128, dtype, edit=edit)
    assert bool(out[:60].isfinite().all()) and bool(out[100:239, :4].isfinite().all()) and bool(out[240].isfinite().all())
    assert not bool(out[60:100, :4, 3].isfinite().any())


def test_values_that_are_not_finite_in_items_of_many_tiles():
    def edit(q, k, v):
        v[1300, 0, 5] = math.inf
        v[1999, 0, 6] = math.nan
    run([700], [2000], 2, 1, 64, 64, BF, edit=edit)
    run([1], [2000], 2, 1, 64, 64, BF, edit=lambda q, k, v: v[1999].fill_(math.nan))


def test_keys_that_are_not_numbers_stay_with_who_sees_them():
    ql = kl = [200, 90]
    q, k, v = make(ql, kl, 2, 1, 128, 128, BF, seed=5)
    k[150], k[200 + 89, 0, 5] = math.nan, math.inf
    out = torch.empty(290, 2, 128, dtype=BF, device=DEV)
    pto.prompt_attention(q, k, v, cu(ql), cu(kl), out)
    assert bool(out[:150].isfinite().all()) and bool(out[150:200].isnan().all()) and bool(out[200:289].isfinite().all())
    check(out[:150], None, q[:150], k[:150], v[:150], [150], [150], 128 ** -0.5, True)


def test_rows_behind_the_last_sequence_and_what_lies_there():
    ql, kl = [70, 20], [70, 200]
    q, k, v = make(ql, kl, 4, 2, 128, 128, BF, seed=6, extra=150)
    k[270:], v[270:], q[90:] = math.nan, math.nan, math.nan
    out = torch.full((240, 4, 128), 7.0, dtype=BF, device=DEV)
    lse = torch.full((4, 240), 7.0, device=DEV)
    pto.prompt_attention(q, k, v, cu(ql), cu(kl), out, lse_out=lse)
    assert bool((out[90:] == 7).all()) and bool((lse[:, 90:] == 7).all())
    check(out[:90], lse[:, :90].contiguous(), q[:90], k[:270], v[:270], ql, kl, 128 ** -0.5, True)


def test_views():
    """Keys and values of one up-projection, heads before tokens, an output inside a wider one."""
    ql, kl, h = [33, 150], [33, 260], 6
    g = torch.Generator(device=DEV).manual_seed(7)
    up = torch.randn(293, h, 256, generator=g, device=DEV).to(BF)
    k, v = up[..., :128], up[..., 128:]
    q = torch.randn(h, 183, 128, generator=g, device=DEV).to(BF).transpose(0, 1)
    wide = torch.full((183, h, 192), 7.0, dtype=BF, device=DEV)
    pto.prompt_attention(q, k, v, cu(ql), cu(kl), wide[..., 64:])
    assert bool((wide[..., :64] == 7).all())
    check(wide[..., 64:], None, q, k, v, ql, kl, 128 ** -0.5, True)
    shared = q[:, :1].expand(183, h, 128)  # the same query row for all heads
    pto.prompt_attention(shared, k, v, cu(ql), cu(kl), wide[..., 64:])
    check(wide[..., 64:], None, shared, k, v, ql, kl, 128 ** -0.5, True)


def test_offsets_beyond_32_bits():
    tk = (1 << 31) // (8 * 128) + 3000  # keys of 4.3 GB
    k = torch.zeros(tk, 8, 128, dtype=BF, device=DEV)
    v = torch.zeros(tk, 8, 128, dtype=BF, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(8)
    k[-700:], v[-700:] = torch.randn(700, 8, 128, generator=g, device=DEV).to(BF), torch.randn(700, 8, 128, generator=g, device=DEV).to(BF)
    q = torch.randn(20, 8, 128, generator=g, device=DEV).to(BF)
    out = torch.empty(20, 8, 128, dtype=BF, device=DEV)
    ck = torch.tensor([0, tk - 700, tk], dtype=torch.int32, device=DEV)
    pto.prompt_attention(q, k, v, torch.tensor([0, 0, 20], dtype=torch.int32, device=DEV), ck, out)
    check(out, None, q, k[-700:].contiguous(), v[-700:].contiguous(), [20], [700], 128 ** -0.5, True)


def test_offsets_out_of_order_reach_nothing_outside():
    q, k, v = make([64], [64], 2, 1, 64, 64, BF)
    out = torch.full((64, 2, 64), 7.0, dtype=BF, device=DEV)
    pto.reset_workspace_status()
    bad = torch.tensor([0, 50, 10, 900], dtype=torch.int32, device=DEV)
    pto.prompt_attention(q, k, v, bad, bad, out)
    assert pto.workspace_status()[0] == _lib.PTO_ST_BAD_PAGE
    pto.reset_workspace_status()
    check(out[:10], None, q[:10], k[:10], v[:10], [10], [10], 64 ** -0.5, True)


def test_a_recorded_call_sees_new_lengths():
    q, k, v = make([300], [3000], 4, 2, 128, 128, BF, seed=9)
    out = torch.zeros(300, 4, 128, dtype=BF, device=DEV)
    cq, ck = cu([300, 0, 0]), cu([3000, 0, 0])
    step = pto.CapturedCall(pto.prompt_attention, q, k, v, cq, ck, out)
    for ql, kl in (([100, 1, 150], [100, 2000, 600]), ([1, 1, 1], [3000 - 2, 1, 1]), ([0, 0, 300], [0, 0, 3000])):
        cq.copy_(cu(ql)), ck.copy_(cu(kl))
        step.replay()
        check(out, None, q[:sum(ql)], k, v, ql, kl, 128 ** -0.5, True)
    assert step.workspace_status()[0] == 0


def test_two_streams_at_once():
    cases = [make([500, 3], [500, 9000], 8, 2, 128, 128, BF, seed=10), make([250], [6000], 4, 4, 128, 128, BF, seed=11)]
    lens = [([500, 3], [500, 9000]), ([250], [6000])]
    outs = [torch.empty(c[0].shape[0], c[0].shape[1], 128, dtype=BF, device=DEV) for c in cases]
    offs = [(cu(a), cu(b)) for a, b in lens]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(5):
        for c, o, (cq, ck), st in zip(cases, outs, offs, streams):
            with torch.cuda.stream(st):
                pto.prompt_attention(*c, cq, ck, o)
    torch.cuda.synchronize()
    for c, o, (ql, kl) in zip(cases, outs, lens):
        check(o, None, *c, ql, kl, 128 ** -0.5, True)


def test_results_over_different_keys_join():
    """An earlier context without a mask and the chunk itself, joined by their lse, are the whole."""
    n, past = 90, 1100
    q, k, v = make([n], [past + n], 8, 2, 128, 128, BF, seed=12)
    part = [torch.empty(n, 8, 128, dtype=BF, device=DEV) for _ in range(2)]
    lse = [torch.empty(8, n, device=DEV) for _ in range(2)]
    pto.prompt_attention(q, k[:past], v[:past], cu([n]), cu([past]), part[0], causal=False, lse_out=lse[0])
    pto.prompt_attention(q, k[past:], v[past:], cu([n]), cu([n]), part[1], lse_out=lse[1])
    w = torch.softmax(torch.stack(lse).double(), 0).permute(0, 2, 1)[..., None]
    both = (w * torch.stack(part).double()).sum(0)
    want, size, _ = definition(q, k, v, [n], [past + n], 128 ** -0.5, True)
    assert bool(((both - want).abs() <= 2 ** -8 * (w * torch.stack(part).double().abs()).sum(0) + (2 ** -8 + 3e-4) * size).all())
