"""Norm and rotation of rows and weights that are not finite, on the GPU against the definition in 64 bits."""
import math

import pytest
import torch

import pypto_b200 as pto
from test_gpu_prompt_rows import rand, want_heads

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F16 = torch.bfloat16, torch.float16


@pytest.mark.parametrize("layout,last", [("half", False), ("half", True), ("interleaved", False), ("interleaved", True),
                                         ("deinterleave", False), ("deinterleave", True)])
@pytest.mark.parametrize("dtype", [BF, F16], ids=["bf16", "f16"])
def test_norm_keeps_what_is_not_finite_to_its_dim(layout, last, dtype):
    """A row with an infinity has an infinite norm: zeros everywhere but in that dim (and its pair, where it is rotated). Six steps of a
    warp, whole rows of ordinary values between them."""
    t, h, d, r = 9, 24, 96, 64
    x = rand(t, h, d, dtype=dtype, seed=40)
    kept, turned = (5, 32 + 11) if last else (90, 11)
    x[1, 0, kept], x[2, 23, kept], x[3, 7, kept + 1], x[4, 20, turned] = math.inf, -math.inf, math.nan, math.inf
    x[5, 3, kept], x[5, 3, kept + 1] = math.inf, -math.inf
    w = rand(d, dtype=dtype, seed=41)
    pos, rot = torch.arange(t) * 100, pto.RotaryFrequencies(r)
    for norm in (w, w.clone()):
        if norm is not w:  # a weight that is not finite reaches its own dim
            norm[kept + 2], norm[kept - 1] = math.inf, math.nan
        want, size = want_heads(x, norm, pos, rot, layout, last, 1e-6)
        out = torch.full_like(x, 7, device=DEV)
        pto.qk_norm_rope(x.to(DEV), None, pos.to(DEV), rot, out, None, query_weight=norm.to(DEV), layout=layout, rope_last=last)
        got = out.cpu().double()
        finite = want.isfinite()
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got[~finite].nan_to_num(7, 8, 9), want[~finite].nan_to_num(7, 8, 9))
        half = torch.finfo(dtype).eps / 2  # (the bound of finite values is that of ordinary rows)
        bound = half * want.abs() + 24 * 2.0 ** -23 * size * (1 + half) + (2.0 ** -25 if dtype == F16 else 0)
        assert bool(((got - want).abs()[finite] <= bound[finite]).all())
