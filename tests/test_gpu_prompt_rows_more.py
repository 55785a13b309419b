"""Rows around a prompt: float16 scales on the way back, and recorded calls that work in place."""
import pytest
import torch

import pypto_b200 as pto
from test_gpu_prompt_rows import quantised, rand

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F16 = torch.bfloat16, torch.float16


@pytest.mark.parametrize("width,dtype", [(128, BF), (640, F16), (512, BF)])
def test_rows_with_float16_scales_come_back(width, dtype):
    """Exactly the stored scale times the stored whole number, rounded once."""
    t, rows = 77, 256
    x = rand(t, width, dtype=dtype, seed=60)
    at = torch.randperm(128, generator=torch.Generator().manual_seed(61))[:t].sort().values
    kn = torch.zeros(rows, width, dtype=torch.int8, device=DEV)
    sc = torch.zeros(rows, width // 128, dtype=F16, device=DEV)
    pto.kv_cache_write(x.to(DEV), None, (at + 128).to(DEV), kn, None, sc)
    out = torch.full((128, width), 7.0, dtype=dtype, device=DEV)
    table, cu = torch.tensor([[1]], dtype=torch.int32, device=DEV), torch.tensor([0, 128], dtype=torch.int32, device=DEV)
    pto.kv_cache_read(kn, None, sc, table, cu, out, None)
    q, s = quantised(x, f16_scales=True)
    want = torch.zeros(128, width, dtype=dtype)
    want[at] = (q.float().view(t, -1, 128) * s.float()[..., None]).view(t, width).to(dtype)
    assert torch.equal(out.cpu(), want) and pto.workspace_status()[0] == 0


@pytest.mark.parametrize("norm", [False, True])
def test_a_recorded_call_in_place_takes_the_rows_of_its_replay(norm):
    x, k = torch.zeros(40, 8, 128, dtype=BF, device=DEV), torch.zeros(40, 2, 128, dtype=BF, device=DEV)
    w = rand(128, seed=62).to(DEV) if norm else None
    pos, rot = torch.arange(40, device=DEV), pto.RotaryFrequencies(64)
    step = pto.CapturedCall(pto.qk_norm_rope, x, k, pos, rot, x, k, query_weight=w, key_weight=w, layout="deinterleave")
    for seed in (63, 64):
        new, new_k = rand(40, 8, 128, seed=seed).to(DEV), rand(40, 2, 128, seed=seed + 10).to(DEV)
        x.copy_(new), k.copy_(new_k), pos.add_(1000)
        step.replay()
        want, want_k = torch.empty_like(new), torch.empty_like(new_k)
        pto.qk_norm_rope(new, new_k, pos, rot, want, want_k, query_weight=w, key_weight=w, layout="deinterleave")
        assert torch.equal(x, want) and torch.equal(k, want_k)
