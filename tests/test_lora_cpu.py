"""The LoRA registry of unquantised linears (runtime/lora.py:206-226 contract), on CPU.

Registry contents, the ``adapters`` lists and the one-time wrapping follow
the reference; a layer without adapters runs its own forward and inputs the
fused GEMM cannot take (here: CPU tensors) get the reference's two-step
``out + sum scale (x A^T) B^T``.
"""
import contextlib

import torch
import torch.nn as nn

from minimaxh3_b200.kernels.lora import attach_lora_registry, fused_supported


class _Block(nn.Module):
    def __init__(self):
        super().__init__()
        self.proj = nn.Linear(16, 24)
        self.out = nn.Linear(24, 16, bias=False)
        self.norm = nn.LayerNorm(16)


def test_registry_wraps_linears_once():
    m = nn.Sequential(_Block(), _Block())
    reg = attach_lora_registry(m)
    assert sorted(reg) == ["0.out", "0.proj", "1.out", "1.proj"]
    for mod in reg.values():
        assert mod.adapters == [] and mod._lora_wrapped
    fwd = m[0].proj.forward
    attach_lora_registry(m)
    assert m[0].proj.forward is fwd                      # not wrapped twice


def test_no_adapters_is_the_plain_forward_and_cpu_gets_two_step_lora():
    torch.manual_seed(0)
    lin = nn.Linear(16, 24)
    attach_lora_registry(nn.Sequential(lin))
    x = torch.randn(5, 16)
    assert torch.equal(lin(x), x @ lin.weight.t() + lin.bias)
    A, B = torch.randn(4, 16), torch.randn(24, 4)
    lin.adapters = [(A, B, 0.5)]
    assert not fused_supported(lin, x)
    ref = x @ lin.weight.t() + lin.bias + 0.5 * ((x @ A.t()) @ B.t())
    assert torch.allclose(lin(x), ref, atol=1e-5)


def test_folded_lora_operands_are_cached_until_an_input_changes():
    """ops._lora_operands reuses the folded (A_cat, B_cat) of a layer until an adapter tensor,
    its scale or the weight scale changes (an in-place edit bumps a tensor's version)."""
    from minimaxh3_b200 import ops

    g = torch.Generator().manual_seed(3)
    A = torch.randn(8, 64, generator=g).to(torch.bfloat16)
    Bm = torch.randn(32, 8, generator=g).to(torch.bfloat16)
    ws = torch.rand(1, 32, generator=g) + 0.5
    first = ops._lora_operands([(A, Bm, 1.0)], 32, 64, "cpu", col_scale=ws.reshape(-1), scale_src=ws)
    again = ops._lora_operands([(A, Bm, 1.0)], 32, 64, "cpu", col_scale=ws.reshape(-1), scale_src=ws)
    assert again[0] is first[0] and again[1] is first[1]
    fresh = ops._fold_lora([(A, Bm, 1.0)], 32, 64, "cpu", col_scale=ws.reshape(-1))
    assert torch.equal(fresh[0], first[0]) and torch.equal(fresh[1], first[1])
    Bm.mul_(2.0)
    edited = ops._lora_operands([(A, Bm, 1.0)], 32, 64, "cpu", col_scale=ws.reshape(-1), scale_src=ws)
    assert edited[1] is not first[1] and not torch.equal(edited[1], first[1])
    rescaled = ops._lora_operands([(A, Bm, 0.5)], 32, 64, "cpu", col_scale=ws.reshape(-1), scale_src=ws)
    assert torch.equal(rescaled[1].float(), (edited[1].float() * 0.5).to(torch.bfloat16).float())
    ws.mul_(2.0)
    new_scale = ops._lora_operands([(A, Bm, 0.5)], 32, 64, "cpu", col_scale=ws.reshape(-1), scale_src=ws)
    assert new_scale[1] is not rescaled[1]


class _Stream:
    """What ops._lora_operands asks of a CUDA stream, without a device."""

    def __init__(self):
        self.waited = []

    def record_event(self):
        return ("after the fold on", self)

    def wait_event(self, event):
        self.waited.append(event)


class _Folded:
    def __init__(self):
        self.used_on = []

    def record_stream(self, stream):
        self.used_on.append(stream)


def _fake_device(monkeypatch):
    """Streams, capture and the fold as fakes: (state with the current stream, adapters to fold)."""
    from types import SimpleNamespace

    from minimaxh3_b200 import ops

    state = SimpleNamespace(stream=_Stream(), capturing=False)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: state.stream)
    monkeypatch.setattr(torch.cuda, "device", contextlib.nullcontext)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: state.capturing)
    monkeypatch.setattr(ops, "_fold_lora", lambda *a: (_Folded(), _Folded()))
    monkeypatch.setattr(ops, "_LORA_CACHE", type(ops._LORA_CACHE)())
    return state, [(torch.zeros(16, 32), torch.zeros(8, 16), 1.0)]


def test_folded_lora_operands_on_another_stream_wait_for_the_fold(monkeypatch):
    from minimaxh3_b200 import ops

    state, adapters = _fake_device(monkeypatch)
    first, filled = state.stream, ops._lora_operands(adapters, 8, 32, "cuda:0")
    assert ops._lora_operands(adapters, 8, 32, "cuda:0") == filled and first.waited == []
    state.stream = other = _Stream()
    again = ops._lora_operands(adapters, 8, 32, "cuda:0")
    assert again[0] is filled[0] and again[1] is filled[1]
    assert other.waited == [("after the fold on", first)]
    assert all(t.used_on == [other] for t in filled)  # their memory outlives the reads there


def test_captured_lora_operands_are_neither_kept_nor_taken(monkeypatch):
    """A capture only records its fold, and a graph must not read memory that the cache may drop."""
    from minimaxh3_b200 import ops

    state, adapters = _fake_device(monkeypatch)
    state.capturing = True
    captured = ops._lora_operands(adapters, 8, 32, "cuda:0")
    state.capturing = False
    eager = ops._lora_operands(adapters, 8, 32, "cuda:0")
    assert eager[0] is not captured[0]
    state.capturing = True
    assert ops._lora_operands(adapters, 8, 32, "cuda:0")[0] is not eager[0]
