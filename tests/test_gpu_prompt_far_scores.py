"""Prompt attention with scores so far from zero that fp32 does not hold their product with log2(e) to a fraction of one, on the GPU
against the definition in 64 bits."""
import pytest
import torch

import pypto_b200 as pto
from test_gpu_prompt_attention import check, cu

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F16 = torch.bfloat16, torch.float16


@pytest.mark.parametrize("ql,kl,hq,hkv,dqk,dv,dtype,power,scale,sign", [
    ([513], [513], 4, 2, 128, 128, BF, 0, 2.0 ** 40, 0),       # a scale that leaves the largest score alone
    ([300, 1, 70], [300, 40, 70], 4, 2, 64, 64, F16, 0, 2.0 ** 30, 0),
    ([300], [700], 2, 2, 192, 128, F16, 13, 2.0 ** -3, 0),     # rows of large values under an ordinary scale
    ([300], [300], 2, 1, 128, 128, BF, 40, 2.0 ** -3, 0),
    ([1], [5000], 8, 1, 128, 128, BF, 0, 2.0 ** 40, 0),        # pieces of an item, and both streams of one
    ([60, 1], [9000, 200], 5, 1, 64, 64, F16, 12, 2.0 ** -3, 0),
    ([200], [3333], 8, 2, 128, 128, BF, 0, 2.0 ** 40, -1),     # scores below zero only
    ([1, 5], [4000, 90], 4, 1, 128, 128, BF, 0, 2.0 ** 99, 1),
    ([130], [1500], 2, 1, 128, 128, BF, 20, 2.0 ** 99, 0),     # the exponents leave fp32, the scores do not
], ids=lambda x: str(x)[:16])
def test_scores_far_from_zero(ql, kl, hq, hkv, dqk, dv, dtype, power, scale, sign):
    """Rows of small whole numbers times a power of two: scores are exact, and those below a row's largest are so far below that they
    take no part. Equal largest ones share."""
    g = torch.Generator(device=DEV).manual_seed(45)
    ints = lambda n, h, d: torch.randint(-2, 3, (n, h, d), generator=g, device=DEV).double()  # noqa: E731
    q, k = ints(sum(ql), hq, dqk), ints(sum(kl), hkv, dqk)
    if sign:
        q, k = q.abs(), k.abs() * sign
    q, k = (q * 2.0 ** power).to(dtype), (k * 2.0 ** power).to(dtype)
    v = torch.randn(sum(kl), hkv, dv, generator=g, device=DEV).to(dtype)
    out = torch.full((sum(ql), hq, dv), 7.0, dtype=dtype, device=DEV)
    lse = torch.full((hq, sum(ql)), 7.0, device=DEV)
    pto.prompt_attention(q, k, v, cu(ql), cu(kl), out, scale, lse_out=lse)
    assert pto.workspace_status()[0] == 0
    fits = dqk * 4.0 ** (power + 1) * scale < 2.0 ** 126  # (otherwise the log of the sum has no fp32 value)
    check(out, lse if fits else None, q, k, v, ql, kl, scale, True)


@pytest.mark.parametrize("ql,kl,hq,hkv,dqk,dv,dtype,late", [
    ([300], [700], 4, 2, 128, 128, BF, False),
    ([513], [513], 2, 1, 64, 64, F16, True),
    ([1], [5000], 8, 1, 128, 128, BF, False),
    ([60, 7], [3000, 200], 5, 1, 192, 128, F16, True),
], ids=lambda x: str(x)[:16])
def test_far_scores_that_differ_little(ql, kl, hq, hkv, dqk, dv, dtype, late):
    """Scores of 2^23 and a few, whole numbers that fp32 holds; under a scale of 2 their exponents are steps of 2 apart, their differences
    are exact. Every other query head has ordinary scores in the same warp; with `late`, keys have the large part from the middle on."""
    g = torch.Generator(device=DEV).manual_seed(46)
    q, k = torch.zeros(sum(ql), hq, dqk, device=DEV), torch.zeros(sum(kl), hkv, dqk, device=DEV)
    q[..., 8:16] = torch.randint(-1, 2, (sum(ql), hq, 8), generator=g, device=DEV).float()
    k[..., 8:16] = torch.randint(-1, 2, (sum(kl), hkv, 8), generator=g, device=DEV).float()
    q[:, ::2, 0], k[..., 0] = 2.0 ** 11, 2.0 ** 12
    if late:
        k[:kl[0] // 2, :, 0] = 0
    q, k = q.to(dtype), k.to(dtype)
    v = torch.randn(sum(kl), hkv, dv, generator=g, device=DEV).to(dtype)
    out = torch.full((sum(ql), hq, dv), 7.0, dtype=dtype, device=DEV)
    lse = torch.full((hq, sum(ql)), 7.0, device=DEV)
    pto.prompt_attention(q, k, v, cu(ql), cu(kl), out, 2.0, lse_out=lse)
    assert pto.workspace_status()[0] == 0
    check(out, lse, q, k, v, ql, kl, 2.0, True)
