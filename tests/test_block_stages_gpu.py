"""A block's operators in their chain, each against its 64-bit formula on what the stage before it gave on the GPU.

So only one operator's rounding lies between a result and its reference, and a bound is tight enough to tell
an operator that is left out, or works on the wrong rows, from one that is there.  With |.| the norm of a whole
tensor, h = 2^-8 half a step of bf16 and activations rounded by the definition (its bytes are tested elsewhere):
  norms, gated residual   h |ref|: one rounding of the result (f32 before it: 2^-14)
  4-bit linear            h |ref|, and with an adapter h | |x A^T| |B|^T |: the low-rank operand in bf16
  8-bit linear            h |ref|
  attention               cosine 0.9995 and 2e-2 of the largest value, the package's contract on its operands
A tenth is added for what f32 sums leave.  Every mistake below, planted in the reference, is at least twice the
bound away (attention's: outside its contract).
"""
import math

import pytest
import torch

import test_block_chain_gpu as chain
from oracle import fp8_attention_ref as OA
from oracle import fp8_linear_ref as OL
from test_fp4_gpu import _ref as fp4_ref
from test_fp4_gpu import _values as fp4_values

DEV, LENS, H, D, C, AXES = "cuda", chain.LENS, chain.H, chain.D, chain.C, chain.AXES
T = sum(LENS)
REP = torch.repeat_interleave(torch.arange(len(LENS)), torch.tensor(LENS))
h = 1.1 * 2.0 ** -8


def _ln(t):
    t = t - t.mean(-1, keepdim=True)
    return t / (t.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt()


def _rms(t):
    return t / (t.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt()


def ref_norm(x, sc, sh, rep=REP):
    return _ln(x.double()) * (1 + sc.double()[rep]) + sh.double()[rep]


def ref_linear4(x, w, bias, lora=None):
    y = fp4_values(*fp4_ref(x)) @ w.t() + bias
    return y if lora is None else y + (x.double() @ lora[0].t()) @ lora[1].t()


def bound_linear4(x, ref, lora):
    low = 0.0 if lora is None else float(((x.double() @ lora[0].t()).abs() @ lora[1].abs().t()).norm())
    return h * (float(ref.norm()) + low)


def ref_linear8(x, w, bias):
    x8, s = OL.quantize_rows(x)
    return (x8.double() * s.double().view(-1, 1)) @ w.t() + bias


def ref_turn(t, pos, sign=1.0):
    ang = torch.cat([pos[:, i, None].double() * 10000.0 ** (-2 * torch.arange(d // 2, dtype=torch.float64) / d) for i, d in enumerate(AXES)], -1)[:, None] * sign
    a, b = t.double()[..., 0::2], t.double()[..., 1::2]
    return torch.stack([a * ang.cos() - b * ang.sin(), a * ang.sin() + b * ang.cos()], -1).flatten(-2).to(torch.bfloat16)


def ref_attention(q, k, v, lens):
    def operand(x, dt):
        s = (torch.clamp(x.float().abs().amax(dim=(0, 2)), min=1e-12).double() / 448.0).float()
        y = x.float() / s[None, :, None]
        y = (torch.clamp(y, -448, 448) if dt == torch.float8_e4m3fn else y).to(dt)
        return (y.double() * s.double()[None, :, None]).permute(1, 0, 2)[None]

    out, at = [], 0
    for n in lens:
        s = slice(at, at + n)
        out.append(OA.sdpa_dequant_oracle(operand(q[s], torch.float8_e4m3fn), operand(k[s], torch.float8_e4m3fn), operand(v[s], torch.float16),
                                          OA.LOG2E / math.sqrt(D), base2=True)[0].permute(1, 0, 2))
        at += n
    return torch.cat(out)


def ref_gated(x, y, g, sc=None, sh=None, y_norm=None, norm=_ln, rep=REP):
    y = y.double() if y_norm is None else y_norm(y.double())
    r = x.double() + g.double()[rep] * y
    n = norm(r)
    return r, n if sc is None else n * (1 + sc.double()[rep]) + sh.double()[rep]


def _stages():
    """Every stage's input and output on the device, on the CPU."""
    from minimaxh3_b200.kernels.block_norm import gated_residual_norm, norm_modulate
    from minimaxh3_b200.kernels.fp8_attention import fp8_attention_varlen
    from minimaxh3_b200.kernels.rotary import Rotary

    cu = torch.tensor([0, LENS[0], T], dtype=torch.int32, device=DEV)
    pos = torch.randint(0, 60, (T, 3), generator=torch.Generator().manual_seed(5), dtype=torch.int32).to(DEV)
    layers, val = chain._layers()
    x, mod = chain._rand(1, T, C), chain._mods(40)
    with torch.no_grad():
        h1 = norm_modulate(x, mod["sc1"], mod["sh1"], cu_seqlens=cu)
        qkv = layers["qkv"](h1).view(-1, 3, H, D)
        a = fp8_attention_varlen(*qkv.unbind(1), cu, cu, max(LENS), rotary=Rotary(pos, AXES))
        o = layers["out"](a.reshape(-1, C))
        r, h2 = gated_residual_norm(x, o, mod["g1"], mod["sc2"], mod["sh2"], cu_seqlens=cu)
        u = layers["up"](h2)
        act = torch.nn.functional.gelu(u)
        y = layers["down"](act)
        last = gated_residual_norm(r, y, mod["g2"], y_norm="rms", norm="rms", cu_seqlens=cu)
        whole = chain._block(x, layers, mod, cu, pos)
    assert all(torch.equal(s, w) for s, w in zip(last, whole))  # these are the chain's stages
    cpu = lambda t: tuple(v.cpu() for v in t) if isinstance(t, tuple) else t.cpu()  # noqa: E731
    out = dict(x=x, h1=h1, qkv=qkv, a=a, o=o, r=r, h2=h2, u=u, act=act, y=y, last=last, pos=pos)
    return {n: cpu(t) for n, t in out.items()}, {n: cpu(t) for n, t in val.items()}, {n: cpu(t) for n, t in mod.items()}


@pytest.mark.gpu
def test_each_stage_of_a_block():
    s, val, mod = _stages()
    swapped = REP.flip(0)  # the rows of the other sequence

    def check(name, got, ref, bound, **wrong):
        err = float((got.double() - ref).norm())
        assert err <= bound, (name, err, bound)
        for what, bad in wrong.items():
            assert float((bad - ref).norm()) > 2 * bound, (name, what)

    m = mod
    ref = ref_norm(s["x"], m["sc1"], m["sh1"])
    check("norm", s["h1"], ref, h * float(ref.norm()), other_sequences=ref_norm(s["x"], m["sc1"], m["sh1"], swapped),
          no_shift=ref_norm(s["x"], m["sc1"], 0 * m["sh1"]), no_scale=ref_norm(s["x"], 0 * m["sc1"], m["sh1"]))

    qkv, lora = s["qkv"].reshape(T, 3 * C), val["lora"]
    ref = ref_linear4(s["h1"], *val["qkv"], lora)
    check("qkv", qkv, ref, bound_linear4(s["h1"], ref, lora), no_adapter=ref_linear4(s["h1"], *val["qkv"]),
          no_bias=ref_linear4(s["h1"], val["qkv"][0], 0, lora))

    q, k, v = s["qkv"].unbind(1)
    tq, tk = ref_turn(q, s["pos"]), ref_turn(k, s["pos"])
    ref, got = ref_attention(tq, tk, v, LENS), s["a"].float()
    for i in range(len(LENS)):
        assert OA.within_tolerance(OA.compare(got[REP == i], ref[REP == i]))
    for what, bad in dict(not_turned=ref_attention(q, k, v, LENS), turned_back=ref_attention(ref_turn(q, s["pos"], -1), tk, v, LENS),
                          one_sequence=ref_attention(tq, tk, v, [T]), zero=0 * ref + 1e-9).items():
        assert not OA.within_tolerance(OA.compare(bad, ref)), what

    for name, into, out in (("out", s["a"].reshape(T, C), s["o"]), ("down", s["act"], s["y"])):
        ref = ref_linear4(into, *val[name])
        check(name, out, ref, bound_linear4(into, ref, None), no_bias=ref_linear4(into, val[name][0], 0), zero=0 * ref)

    ref = ref_linear8(s["h2"], *val["up"])
    check("up", s["u"], ref, h * float(ref.norm()), no_bias=ref_linear8(s["h2"], val["up"][0], 0))

    both = lambda *a, **kw: torch.stack(ref_gated(*a, **kw))  # noqa: E731
    args = (s["x"], s["o"], m["g1"], m["sc2"], m["sh2"])
    ref = both(*args)
    for i, name in enumerate(("r", "h2")):
        check(name, s[name], ref[i], h * float(ref[i].norm()), no_block=both(s["x"], 0 * s["o"], *args[2:])[i], no_gate=both(*args[:2], 1 + 0 * m["g1"], *args[3:])[i])
    check("h2", s["h2"], ref[1], h * float(ref[1].norm()), other_sequences=both(*args, rep=swapped)[1], rms=both(*args, norm=_rms)[1])
    ref = both(s["r"], s["y"], m["g2"], y_norm=_rms, norm=_rms)
    for i in range(2):
        check("last", s["last"][i], ref[i], h * float(ref[i].norm()), no_y_norm=both(s["r"], s["y"], m["g2"], norm=_rms)[i])
