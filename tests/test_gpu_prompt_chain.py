"""The operators around a prompt as a layer runs them, one after the other, and through every host path."""
import math

import pytest
import torch

import oracle
import pypto_b200 as pto
import pypto_b200.torch_ops  # noqa: F401  (registers the operators)
from pypto_b200 import prompt
from test_gpu_prompt_attention import check, cu

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, I8 = torch.bfloat16, torch.int8


def randn(*shape, seed, dtype=BF, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)


def pages(lens, seed, spare=3):
    """A block table of permuted pages and the cache row of every position of every sequence."""
    need = [-(-n // 128) for n in lens]
    order = torch.randperm(sum(need) + spare, generator=torch.Generator().manual_seed(seed))
    table = torch.full((len(lens), max(need) + 1), -1, dtype=torch.int32)
    at, rows = 0, []
    for i, (n, k) in enumerate(zip(lens, need)):
        table[i, :k] = order[at:at + k]
        at += k
        pos = torch.arange(n)
        rows.append(table[i, pos // 128].long() * 128 + pos % 128)
    return table.to(DEV), [r.to(DEV) for r in rows], (sum(need) + spare) * 128


class GroupedLayer:
    """A chunk of new tokens of sequences that have `past` earlier ones, 8 query heads on 2 key heads: norm and rotation in the fused
    projection, keys and values quantised into paged caches, everything read back, attention."""

    def __init__(self, past, new, seed=0):
        self.past, self.new, self.hq, self.hk, self.d = past, new, 8, 2, 128
        t, total = sum(new), [p + n for p, n in zip(past, new)]
        self.table, rows, n_rows = pages(total, seed)
        self.rotary = pto.RotaryFrequencies(128, 10000.0, scaling=dict(type="yarn", factor=8, original_max_position=512))
        self.wq, self.wk = randn(128, seed=seed + 1), randn(128, seed=seed + 2)
        w = self.hk * self.d
        self.k_cache, self.v_cache = (torch.zeros(n_rows, w, dtype=I8, device=DEV) for _ in range(2))
        self.k_scale, self.v_scale = (torch.zeros(n_rows, self.hk, device=DEV) for _ in range(2))
        for cache, scale, s in ((self.k_cache, self.k_scale, 3), (self.v_cache, self.v_scale, 4)):
            for i, p in enumerate(past):
                if p:
                    pto.kv_cache_write(randn(p, w, seed=seed + 10 * i + s), None, rows[i][:p], cache, None, scale)
        self.slots = torch.cat([r[p:] for r, p in zip(rows, past)])
        self.positions = torch.cat([torch.arange(p, p + n) for p, n in zip(past, new)]).to(DEV)
        self.qkv = torch.zeros(t, (self.hq + 2 * self.hk) * self.d, dtype=BF, device=DEV)
        self.cq, self.ck = cu(new), cu(total)
        self.total = total
        self.k_all, self.v_all = (torch.zeros(sum(total), w, dtype=BF, device=DEV) for _ in range(2))
        self.out = torch.zeros(t, self.hq, self.d, dtype=BF, device=DEV)

    def parts(self):
        t, a, b = self.qkv.shape[0], self.hq * self.d, (self.hq + self.hk) * self.d
        return self.qkv[:, :a].view(t, self.hq, self.d), self.qkv[:, a:b].view(t, self.hk, self.d), self.qkv[:, b:]

    def step(self):
        q, k, v = self.parts()
        pto.qk_norm_rope(q, k, self.positions, self.rotary, q, k, query_weight=self.wq, key_weight=self.wk)
        pto.kv_cache_write(self.qkv[:, self.hq * self.d:(self.hq + self.hk) * self.d], None, self.slots, self.k_cache, None, self.k_scale)
        pto.kv_cache_write(v, None, self.slots, self.v_cache, None, self.v_scale)
        pto.kv_cache_read(self.k_cache, None, self.k_scale, self.table, self.ck, self.k_all, None)
        pto.kv_cache_read(self.v_cache, None, self.v_scale, self.table, self.ck, self.v_all, None)
        n = self.k_all.shape[0]
        pto.prompt_attention(q, self.k_all.view(n, self.hk, self.d), self.v_all.view(n, self.hk, self.d), self.cq, self.ck, self.out)

    def verify(self):
        q, k, v = self.parts()
        n = self.k_all.shape[0]
        # a value reads back within half a step of its group (max / 127), and its bf16 rounding
        at = torch.cat([torch.arange(c - m, c) for c, m in zip(torch.tensor(self.total).cumsum(0).tolist(), self.new)]).to(DEV)
        for rows, back in ((k.reshape(k.shape[0], -1), self.k_all), (v, self.v_all)):
            x = rows.float().view(rows.shape[0], -1, 128)
            top = x.abs().amax(-1, keepdim=True)
            err = (back[at].float().view_as(x) - x).abs()
            assert bool((err <= top * (0.5 / 127 + 2.0 ** -8 + 1e-6)).all())
        check(self.out, None, q, self.k_all.view(n, self.hk, self.d), self.v_all.view(n, self.hk, self.d), self.new, self.total,
              self.d ** -0.5, True)
        assert pto.workspace_status()[0] == 0


@pytest.mark.parametrize("past,new", [([0], [70]), ([300, 0, 129], [60, 33, 1]), ([1500, 40, 128], [1, 1, 1])])
def test_a_chunk_of_a_layer_with_grouped_heads(past, new):
    layer = GroupedLayer(past, new)
    layer.qkv.copy_(randn(*layer.qkv.shape, seed=50))
    layer.step()
    layer.verify()


def test_the_chunk_recorded_and_replayed():
    layer = GroupedLayer([200, 0], [40, 24], seed=7)
    layer.qkv.copy_(randn(*layer.qkv.shape, seed=60))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer.step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        layer.step()
    for seed in (61, 62):
        layer.qkv.copy_(randn(*layer.qkv.shape, seed=seed))
        layer.out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        layer.verify()


def test_latent_rows_written_here_are_what_the_sparse_attention_reads():
    """Prompt rows quantised by `kv_cache_write` into split and packed caches; the sparse attention over them, all positions selected,
    against the oracle over the same caches; and the same rows expanded to heads for the dense attention."""
    lens = [300, 129]
    table, rows, n_rows = pages(lens, 11)
    slots, t = torch.cat(rows), sum(lens)
    kv = randn(t, 576, seed=70)
    rope = torch.empty(t, 1, 64, dtype=BF, device=DEV)
    rotary = pto.RotaryFrequencies(64)
    positions = torch.cat([torch.arange(n) for n in lens]).to(DEV)
    pto.qk_norm_rope(kv[:, 512:].view(t, 1, 64), None, positions, rotary, rope, None, layout="deinterleave")
    kn, kr = torch.zeros(n_rows, 512, dtype=I8, device=DEV), torch.zeros(n_rows, 64, dtype=BF, device=DEV)
    sc, packed = torch.zeros(n_rows, 4, device=DEV), torch.zeros(n_rows, 656, dtype=I8, device=DEV)
    pto.kv_cache_write(kv[:, :512], rope.view(t, 64), slots, kn, kr, sc, packed_kv_cache=packed)

    b, nq = len(lens), 128
    qn, qr = randn(b * nq, 512, seed=71, scale=0.5), randn(b * nq, 64, seed=72)
    idx = torch.full((b, 2048), -1, dtype=torch.int32, device=DEV)
    for i, n in enumerate(lens):
        idx[i, :n] = torch.arange(n, dtype=torch.int32)
    act = torch.tensor(lens, dtype=torch.int32, device=DEV)
    outs = [torch.empty(b, 1, nq, 512, dtype=BF, device=DEV) for _ in range(2)]
    pto.sparse_flash_attention_quant_d(qn, qr, kn, kr, sc, idx, table, act, outs[0], nq, 1, 576 ** -0.5, 2048, 128, table.shape[1])
    pto.sparse_attention_antiquant_d(qn, qr, packed, idx, table, act, outs[1], nq, 1, 576 ** -0.5, 2048, 128, table.shape[1])
    assert torch.equal(*outs)
    want = oracle.sparse_attention(qn.cpu(), qr.cpu(), kn.cpu(), kr.cpu(), sc.cpu(), idx.cpu(), table.cpu(), lens, 1)
    e = oracle.attention_errors(outs[0].cpu(), want)
    assert e["max_abs"] <= 2e-2 and e["rel_l2"] <= 5e-3, e

    # the dense side: the prompt's own rows back, expanded to 16 heads of 192 | 128
    h = 16
    back, back_r = torch.empty(t, 512, dtype=BF, device=DEV), torch.empty(t, 64, dtype=BF, device=DEV)
    pto.kv_cache_read(None, None, None, table, cu(lens), back, back_r, packed_kv_cache=packed)
    assert torch.equal(back_r, rope.view(t, 64))
    up = (back @ randn(512, h * 256, seed=73, scale=512 ** -0.5)).view(t, h, 256)
    k = torch.cat([up[..., :128], back_r[:, None].expand(-1, h, -1)], -1)
    q = randn(t, h, 192, seed=74)
    pto.qk_norm_rope(q, None, positions, rotary, q, None, layout="deinterleave", rope_last=True)
    out = torch.empty(t, h, 128, dtype=BF, device=DEV)
    pto.prompt_attention(q, k, up[..., 128:], cu(lens), cu(lens), out)
    check(out, None, q, k, up[..., 128:], lens, lens, 192 ** -0.5, True)


def _calls():
    """One call of each operator, with its outputs made anew."""
    t, lens = 37, [37, 300]
    table, rows, n_rows = pages(lens, 21)
    rotary = pto.RotaryFrequencies(64, scaling=dict(type="linear", factor=2))
    x, xr = randn(337, 512, seed=80), randn(337, 64, seed=81)
    caches = (torch.zeros(n_rows, 512, dtype=I8, device=DEV), torch.zeros(n_rows, 64, dtype=BF, device=DEV),
              torch.zeros(n_rows, 4, device=DEV))
    pto.kv_cache_write(x, xr, torch.cat(rows), *caches)
    q, k, pos = randn(t, 6, 128, seed=82), randn(t, 2, 128, seed=83), torch.arange(t, device=DEV)
    wq, wk = randn(128, seed=84), randn(128, seed=85)
    kk, vv = randn(337, 2, 128, seed=86), randn(337, 2, 128, seed=87)
    cq, ck = cu([30, 7]), cu(lens)

    def rope(op):
        o = torch.empty_like(q), torch.empty_like(k)
        op(q, k, pos, rotary, *o, wq, wk)
        return o

    def write(op):
        o = tuple(torch.zeros_like(c) for c in caches) + (torch.zeros(n_rows, 656, dtype=I8, device=DEV),)
        op(x, xr, torch.cat(rows), *o)
        return o

    def read(op):
        o = torch.zeros(337, 512, dtype=BF, device=DEV), torch.zeros(337, 64, dtype=BF, device=DEV)
        op(*caches, table, ck, *o)
        return o

    def attend(op):
        o = torch.zeros(t, 6, 128, dtype=BF, device=DEV), torch.zeros(6, t, device=DEV)
        op(q, kk, vv, cq, ck, *o)
        return o

    eager = {"qk_norm_rope": lambda q, k, p, r, qo, ko, a, b: pto.qk_norm_rope(q, k, p, r, qo, ko, query_weight=a, key_weight=b),
             "kv_cache_write": lambda x, r, i, a, b, c, d: pto.kv_cache_write(x, r, i, a, b, c, packed_kv_cache=d),
             "kv_cache_read": lambda a, b, c, t, u, o, r: pto.kv_cache_read(a, b, c, t, u, o, r),
             "prompt_attention": lambda q, k, v, a, b, o, l: pto.prompt_attention(q, k, v, a, b, o, 128 ** -0.5, lse_out=l)}
    ns = torch.ops.pypto_b200
    registered = {"qk_norm_rope": lambda q, k, p, r, qo, ko, a, b: ns.qk_norm_rope(q, k, p, r.turns, qo, ko, a, b, r.amplitude),
                  "kv_cache_write": lambda x, r, i, a, b, c, d: ns.kv_cache_write(x, r, i, a, b, c, d),
                  "kv_cache_read": lambda a, b, c, t, u, o, r: ns.kv_cache_read(a, b, c, t, u, o, r),
                  "prompt_attention": lambda q, k, v, a, b, o, l: ns.prompt_attention(q, k, v, a, b, o, 128 ** -0.5, True, l)}
    return dict(qk_norm_rope=rope, kv_cache_write=write, kv_cache_read=read, prompt_attention=attend), eager, registered


@pytest.mark.parametrize("op", ["qk_norm_rope", "kv_cache_write", "kv_cache_read", "prompt_attention"])
def test_every_host_path_makes_the_same_call(op, monkeypatch):
    calls, eager, registered = _calls()
    call = calls[op]
    want = call(eager[op])  # (the workspace exists from here on)
    compiled = call(torch.compile(registered[op], backend="eager", fullgraph=True))

    class Watched:
        def __init__(self, native):
            self.native, self.taken = native, []

        def __getattr__(self, name):
            return lambda *args: self.taken.append(getattr(self.native, name)(*args)) or self.taken[-1]

    native = Watched(prompt._native)
    monkeypatch.setattr(prompt, "_native", native)
    taken = call(eager[op])
    monkeypatch.setattr(prompt, "_native", None)
    checked = call(eager[op])
    torch.cuda.synchronize()
    assert native.taken == [True]
    for other in (compiled, taken, checked):
        for a, b in zip(want, other):
            assert torch.equal(a, b)


def test_c_entries_refuse_what_python_does_not_see():
    """Arguments that pass the Python checks and the C entry turns down, with a message and without a launch."""
    q = torch.zeros(4, 1, 264, dtype=BF, device=DEV)  # a head of more than 256 dims
    before = pto.launch_count()
    with pytest.raises(pto._lib.PtoError, match="dims"):
        pto.qk_norm_rope(q, None, None, None, q.clone(), None, query_weight=torch.ones(264, dtype=BF, device=DEV))
    x = torch.zeros(4, 2, 64, dtype=BF, device=DEV)
    with pytest.raises(pto._lib.PtoError, match="overlap"):  # every head written to the same place
        pto.qk_norm_rope(x, None, None, None, torch.zeros(4, 1, 64, dtype=BF, device=DEV).expand(4, 2, 64), None)
    k = torch.zeros(9, 1, 64, dtype=BF, device=DEV)
    with pytest.raises(pto._lib.PtoError, match="overlap"):
        pto.prompt_attention(x, k.expand(9, 2, 64), k.expand(9, 2, 64), cu([4]), cu([9]), torch.empty_like(x))
    with pytest.raises(ValueError):
        pto.prompt_attention(x, k, k, cu([4]), cu([9]), torch.empty_like(x), math.inf)
    with pytest.raises(ValueError):
        pto.qk_norm_rope(x, None, torch.arange(4, device=DEV), pto.RotaryFrequencies(64), torch.empty_like(x), None, eps=math.nan)
    assert pto.launch_count() == before
