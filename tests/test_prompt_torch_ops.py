"""Calls of the operators around a prompt that leave out what is optional, through their `torch.library` registration."""
import pytest
import torch

import pypto_b200 as pto
import pypto_b200.torch_ops  # noqa: F401  (registers the operators)

BF, I8 = torch.bfloat16, torch.int8


def _ns():
    return torch.ops.pypto_b200


def _attention(x, cu, out, lse=None):
    if lse is None:
        _ns().prompt_attention(x, x, x, cu, cu, out, 0.125)
        _ns().prompt_attention(x, x, x, cu, cu, out, 0.125, True, None)
    else:
        _ns().prompt_attention(x, x, x, cu, cu, out, 0.125, lse_out=lse)
    return out + 1


def _write(x, rope, index, caches, packed=None):
    if packed is None:
        _ns().kv_cache_write(x, rope, index, *caches)
    else:
        _ns().kv_cache_write(x, rope, index, None, None, None, packed)


def _inputs(dev):
    g = torch.Generator(device=dev).manual_seed(50)
    x = torch.randn(70, 4, 128, generator=g, device=dev).to(BF)
    return x, torch.tensor([0, 50, 70], dtype=torch.int32, device=dev)


def _rows(dev):
    g = torch.Generator(device=dev).manual_seed(51)
    caches = (torch.zeros(128, 512, dtype=I8, device=dev), torch.zeros(128, 64, dtype=BF, device=dev), torch.zeros(128, 4, device=dev))
    return (torch.randn(30, 512, generator=g, device=dev).to(BF), torch.randn(30, 64, generator=g, device=dev).to(BF),
            torch.arange(30, device=dev) + 17, caches)


def test_schemas_name_the_buffers_that_are_written():
    for name, written in (("qk_norm_rope", {"query_out", "key_out"}), ("kv_cache_read", {"key_nope_out", "key_rope_out"}),
                          ("kv_cache_write", {"key_nope_2d", "key_rope_2d", "k_nope_scales", "packed_kv_cache"}),
                          ("prompt_attention", {"attention_out", "lse_out"})):
        schema = getattr(_ns(), name).default._schema
        assert {a.name for a in schema.arguments if a.alias_info is not None and a.alias_info.is_write} == written
        assert len(schema.returns) == 0


def test_calls_without_optional_buffers_trace_without_a_device():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        x, cu = torch.empty(70, 4, 128, dtype=BF), torch.empty(3, dtype=torch.int32)
        _attention(x, cu, torch.empty_like(x))
        _attention(x, cu, torch.empty_like(x), torch.empty(4, 70))
        rows = torch.empty(30, 512, dtype=BF), torch.empty(30, 64, dtype=BF), torch.empty(30, dtype=torch.int64)
        _write(*rows, (torch.empty(128, 512, dtype=I8), torch.empty(128, 64, dtype=BF), torch.empty(128, 4)))
        _write(*rows, None, torch.empty(128, 656, dtype=I8))


def test_host_tensors_are_refused():
    x, cu = _inputs("cpu")
    with pytest.raises(RuntimeError, match="device"):
        _attention(x, cu, torch.empty_like(x))
    with pytest.raises(RuntimeError, match="device"):
        _write(*_rows("cpu"))


@pytest.mark.gpu
@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_compiled_calls_without_optional_buffers(backend):
    x, cu = _inputs("cuda")
    want, want_lse, out, lse = torch.zeros_like(x), torch.zeros(4, 70, device="cuda"), torch.zeros_like(x), torch.zeros(4, 70, device="cuda")
    pto.prompt_attention(x, x, x, cu, cu, want, 0.125, lse_out=want_lse)
    attention = torch.compile(_attention, backend=backend, fullgraph=True)
    version = out._version
    assert torch.equal(attention(x, cu, out), want + 1) and torch.equal(out, want) and out._version > version
    assert torch.equal(attention(x, cu, out.zero_(), lse), want + 1) and torch.equal(out, want) and torch.equal(lse, want_lse)

    rows = _rows("cuda")
    again = tuple(torch.zeros_like(c) for c in rows[3])
    packed, want_packed = (torch.zeros(128, 656, dtype=I8, device="cuda") for _ in range(2))
    pto.kv_cache_write(*rows[:3], *rows[3], packed_kv_cache=want_packed)
    write = torch.compile(_write, backend=backend, fullgraph=True)
    write(*rows[:3], again)
    write(*rows[:3], None, packed)
    for a, b in zip((*rows[3], want_packed), (*again, packed)):
        assert torch.equal(a, b) and bool(a.any())


def _norm_alone(x, w, out):
    _ns().qk_norm_rope(x, None, None, None, out, None, w, None)


def _default_scale(x, cu, out):
    _ns().prompt_attention(x, x, x, cu, cu, out)


def test_norm_alone_and_the_default_scale_trace_without_a_device():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        x = torch.empty(5, 4, 128, dtype=BF)
        _norm_alone(x, torch.empty(128, dtype=BF), torch.empty_like(x))
        _default_scale(x, torch.empty(2, dtype=torch.int32), torch.empty_like(x))


def test_norm_alone_and_the_default_scale_reach_the_operators_checks():
    x, cu = _inputs("cpu")
    with pytest.raises(RuntimeError, match="device"):
        _norm_alone(x, torch.ones(128, dtype=BF), torch.empty_like(x))
    with pytest.raises(RuntimeError, match="device"):
        _default_scale(x, cu, torch.empty_like(x))
    turns = pto.RotaryFrequencies(64, device="cpu").turns
    with pytest.raises(TypeError, match="positions"):  # a rotation without positions
        _ns().qk_norm_rope(x, None, None, turns, torch.empty_like(x), None, None, None)


@pytest.mark.gpu
@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_compiled_norm_alone_and_default_scale(backend):
    x, cu = _inputs("cuda")
    w, want, got = x[0, 0].clone(), torch.zeros_like(x), torch.zeros_like(x)
    pto.qk_norm_rope(x, None, None, None, want, None, query_weight=w)
    torch.compile(_norm_alone, backend=backend, fullgraph=True)(x, w, got)
    assert torch.equal(want, got) and bool(got.any())
    pto.prompt_attention(x, x, x, cu, cu, want)
    torch.compile(_default_scale, backend=backend, fullgraph=True)(x, cu, got)
    assert torch.equal(want, got)
