"""The measured cases of the block operators: rotary positions with several axes, the norms
before and after a block with their modulation, gate and residual, and the 4-bit linear.

``run`` computes a case either in its plain form (elementary torch operations in
32 bits, 64 where a value next to a rounding border or a far position's angle
needs them) or, with ``own`` true, through the package's public functions.
"""
import math

import torch

own = False

DEV = "cuda" if torch.cuda.is_available() else "cpu"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------


def _rotary(batch, heads, kv_heads, grid, dim, axes, dtype, interleaved=True, heads_first=False, grad=False):
    return dict(op="rotary", batch=batch, heads=heads, kv_heads=kv_heads, grid=grid, dim=dim, axes=axes, dtype=dtype,
                interleaved=interleaved, heads_first=heads_first, grad=grad)


def _norm(batch, tokens, channels, norm, dtype, mod, affine=False, per_token=False, grad=False):
    return dict(op="norm_modulate", batch=batch, tokens=tokens, channels=channels, norm=norm, dtype=dtype, mod=mod,
                affine=affine, per_token=per_token, grad=grad)


def _gated(lengths, channels, y_norm, norm, dtype, mod, alpha=1.0, grad=False):
    return dict(op="gated_residual_norm", lengths=lengths, channels=channels, y_norm=y_norm, norm=norm, dtype=dtype,
                mod=mod, alpha=alpha, grad=grad)


def listed():
    cases = [
        # one denoising step's self-attention: Q and K of 21 latent frames x 30 x 52 patches, as views of the fused projection
        dict(_rotary(1, 40, 40, "21x30x52", 128, "44,42,42", "bf16"), name="rotary video bf16"),
        # one token of two streams with shared key heads: the smallest call
        dict(_rotary(2, 8, 2, "1x1x1", 64, "16,24,24", "f16", interleaved=False, heads_first=True), name="rotary one token f16"),
        # fine-tuning on an image of odd size: forward and the gradients of q and k
        dict(_rotary(2, 24, 24, "1x45x77", 128, "32,48,48", "bf16", interleaved=False, grad=True), name="rotary image grad"),
        # the norm before self-attention of the same step, its modulation kept in 32 bits
        dict(_norm(1, 32760, 5120, "layer", "bf16", "f32"), name="norm video bf16"),
        # a training step's norm on a ragged batch: forward and every gradient
        dict(_norm(2, 4097, 1536, "layer", "bf16", "f32", affine=True, grad=True), name="norm grad"),
        # packed video and audio sequences: gate, residual and the next norm in one pass
        dict(_gated("33784,16892", 5120, "none", "layer", "bf16", "f32"), name="gated packed bf16"),
        # the same with a norm on the block's output, trained in 32 bits
        dict(_gated("1000,37,0,2053", 1544, "rms", "rms", "f32", "f32", alpha=0.5, grad=True), name="gated grad f32"),
        # rounding the MLP's activations to 4 bits, as a check of which layers may be converted does
        dict(op="fp4_round_trip", rows=32760, k=13824, dtype="bf16", name="fp4 round trip mlp"),
        # the same of a text stream
        dict(op="fp4_round_trip", rows=512, k=5120, dtype="f16", name="fp4 round trip text"),
        # the linear of a text stream
        dict(op="fp4_linear", rows=509, k=5120, n=5120, bias=True, dtype="bf16", name="fp4 linear text"),
        # the modulation's linear: one row, where reading the weight is the work
        dict(op="fp4_linear", rows=1, k=5120, n=5120, bias=True, dtype="bf16", name="fp4 linear one row"),
        # the MLP's first linear over a whole video
        dict(op="fp4_linear", rows=32760, k=5120, n=13824, bias=True, dtype="bf16", name="fp4 linear video"),
    ]
    return cases


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "norm_modulate", "gated_residual_norm", "fp4_round_trip", "fp4_linear"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    grad = rng.random() < 0.4
    if op == "rotary":
        dim, axes = rng.choice([(64, "16,24,24"), (64, "32,32"), (128, "44,42,42"), (128, "32,48,48"), (128, "16,56,56"),
                                (128, "128"), (80, "20,30,30"), (96, "32,32"), (72, "24,24,24")])
        kv = rng.choice([1, 2, 4, 8, 12])
        heads = kv * rng.choice([1, 1, 1, 3])
        grid = "%dx%dx%d" % (_log(rng, 1, 24), _log(rng, 1, 48), _log(rng, 1, 64))
        return _rotary(rng.choice([1, 1, 2, 3]), heads, kv, grid, dim, axes, dtype, rng.random() < 0.5, rng.random() < 0.3, grad)
    if op == "norm_modulate":
        tokens, channels = _log(rng, 1, 20000), _log(rng, 48, 6000)
        if rng.random() < 0.7:
            channels = max(64, channels // 64 * 64)
        return _norm(rng.choice([1, 1, 2, 3]), tokens, channels, rng.choice(["layer", "rms"]), dtype, rng.choice([dtype, "f32"]),
                     rng.random() < 0.5, rng.random() < 0.3, grad)
    if op == "gated_residual_norm":
        channels = _log(rng, 48, 5200)
        if rng.random() < 0.7:
            channels = max(64, channels // 64 * 64)
        lengths = ",".join(str(_log(rng, 1, 12000)) for _ in range(rng.choice([1, 2, 3, 5])))
        return _gated(lengths, channels, rng.choice(["none", "rms", "layer"]), rng.choice(["layer", "rms"]), dtype,
                      rng.choice([dtype, "f32"]), rng.choice([1.0, 0.5]), grad)
    rows = _log(rng, 1, 16000)
    if op == "fp4_round_trip":
        return dict(op=op, rows=rows, k=32 * _log(rng, 1, 400), dtype=dtype)
    return dict(op=op, rows=rows, k=32 * _log(rng, 1, 200), n=8 * _log(rng, 1, 1000), bias=rng.random() < 0.5, dtype=dtype)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _hidden(g, *shape, dtype):
    """N(0, 1) with one channel in a hundred eight times as large, as the outlier channels of a transformer's stream."""
    x = torch.randn(*shape, generator=g, device=DEV)
    x.mul_(torch.where(torch.rand(shape[-1], generator=g, device=DEV) < 0.01, 8.0, 1.0))
    return x.to(dtype)


def _randn(g, *shape, scale=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)


def _ints(text, sep=","):
    return [int(v) for v in text.split(sep)]


def prepare(case, seed):
    g, dt = _gen(seed), TYPES[case["dtype"]]
    s = dict(case=case)
    op = case["op"]
    if op == "rotary":
        f, h, w = _ints(case["grid"], "x")
        B, S, D, H, Hk = case["batch"], f * h * w, case["dim"], case["heads"], case["kv_heads"]
        axes = _ints(case["axes"])
        t, i, j = torch.meshgrid(torch.arange(f), torch.arange(h), torch.arange(w), indexing="ij")
        pos = torch.stack([t, i, j], -1).reshape(S, 3)[:, 3 - len(axes):] + int(torch.randint(0, 1000, (1,), generator=g, device=DEV))
        s["positions"] = pos.to(torch.int32).to(DEV)
        if case["heads_first"]:
            s["q"], s["k"] = _randn(g, B, H, S, D, dtype=dt), _randn(g, B, Hk, S, D, dtype=dt)
        else:  # views of one projection's output
            qkv = _randn(g, B, S, H + 2 * Hk, D, dtype=dt)
            s["q"], s["k"] = qkv[:, :, :H].transpose(1, 2), qkv[:, :, H:H + Hk].transpose(1, 2)
        if case["grad"]:
            s["dq"], s["dk"] = _randn(g, B, H, S, D, dtype=dt), _randn(g, B, Hk, S, D, dtype=dt)
            s["q"], s["k"] = s["q"].contiguous().requires_grad_(True), s["k"].contiguous().requires_grad_(True)
    elif op == "norm_modulate":
        B, S, C, md = case["batch"], case["tokens"], case["channels"], TYPES[case["mod"]]
        lead = (B, S) if case["per_token"] else (B,)
        s["x"] = _hidden(g, B, S, C, dtype=dt)
        s["scale"], s["shift"] = _randn(g, *lead, C, scale=0.3, dtype=md), _randn(g, *lead, C, scale=0.3, dtype=md)
        s["weight"] = (1 + _randn(g, C, scale=0.2)).to(md) if case["affine"] else None
        s["bias"] = _randn(g, C, scale=0.2, dtype=md) if case["affine"] and case["norm"] == "layer" else None
        if case["grad"]:
            s["dh"] = _randn(g, B, S, C, dtype=dt)
            s["leaves"] = [s[n].requires_grad_(True) for n in ("x", "scale", "shift", "weight", "bias") if s[n] is not None]
    elif op == "gated_residual_norm":
        lens, C, md = _ints(case["lengths"]), case["channels"], TYPES[case["mod"]]
        T, n = sum(lens), len(lens)
        s["cu"] = torch.tensor([sum(lens[:i]) for i in range(n + 1)], dtype=torch.int32, device=DEV)
        s["x"], s["y"] = _hidden(g, T, C, dtype=dt), _hidden(g, T, C, dtype=dt)
        s["gate"] = _randn(g, n, C, scale=0.5, dtype=md)
        s["scale"], s["shift"] = _randn(g, n, C, scale=0.3, dtype=md), _randn(g, n, C, scale=0.3, dtype=md)
        s["y_weight"] = (1 + _randn(g, C, scale=0.2)).to(md) if case["y_norm"] != "none" else None
        if case["grad"]:
            s["dr"], s["dh"] = _randn(g, T, C, dtype=dt), _randn(g, T, C, dtype=dt)
            s["leaves"] = [s[m].requires_grad_(True) for m in ("x", "y", "gate", "scale", "shift", "y_weight") if s[m] is not None]
    else:
        s["x"] = _hidden(g, case["rows"], case["k"], dtype=dt)
        if op == "fp4_linear":  # the weight as a converted layer keeps it
            w = _randn(g, case["n"], case["k"], scale=0.02, dtype=torch.bfloat16)
            codes, block, row = _round_fp4(w)
            s["w4"], s["w_block"], s["w_scale"] = _pack(codes), _tile(block), row
            s["bias"] = _randn(g, case["n"], scale=0.01, dtype=torch.bfloat16) if case["bias"] else None
    return s


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------

E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)


def _round_fp4(x):
    """4-bit codes [M, K] (bit 3 the sign), e4m3 scales [M, K/16] and power-of-two row scales [M, 1]."""
    M, K = x.shape
    v = x.double().reshape(M, K // 16, 16)
    top = v.abs().amax(dim=2)
    m, e = torch.frexp(top.amax(dim=1, keepdim=True) / 2688.0)
    e = torch.where(m > 0, torch.where(m > 0.5, e, e - 1), torch.full_like(e, -100)).clamp(min=-100)
    row = ((e + 127) << 23).to(torch.int32).view(torch.float32).double()  # 2^e from its bits: a rounded power would move ties
    block = (top / (6.0 * row)).float().to(torch.float8_e4m3fn)
    q = v / (block.double() * row).unsqueeze(2)
    a = torch.where(block.float().unsqueeze(2) > 0, q.abs(), torch.zeros_like(q))
    code = sum(c.to(torch.uint8) for c in (a > 0.25, a >= 0.75, a > 1.25, a >= 1.75, a > 2.5, a >= 3.5, a > 5.0))  # ties to the even code
    code = code + 8 * (v < 0).to(torch.uint8)
    return code.reshape(M, K), block, row.float()


def _pack(code):
    return (code[:, 0::2] + 16 * code[:, 1::2]).contiguous()


def _unpack(packed):
    return torch.stack([packed & 15, packed >> 4], dim=2).reshape(packed.shape[0], -1)


def _tile(block):
    """Scales [M, K/16] as blocks of 128 rows x 4: [ceil(M/128), ceil(K/64), 32, 4, 4], row 32 i + j at [j, i]."""
    M, n = block.shape
    pad = torch.zeros((-(-M // 128) * 128, -(-n // 4) * 4), dtype=torch.uint8, device=block.device)
    pad[:M, :n] = block.view(torch.uint8)
    return pad.view(pad.shape[0] // 128, 4, 32, pad.shape[1] // 4, 4).permute(0, 3, 2, 1, 4).contiguous().view(torch.float8_e4m3fn)


def _untile(tiled, M, n):
    t = tiled.view(torch.uint8).permute(0, 3, 2, 1, 4)
    return t.reshape(t.shape[0] * 128, -1)[:M, :n].contiguous().view(torch.float8_e4m3fn)


def _values(code, block, row):
    """The numbers that codes and scales stand for, in 32 bits (exact: at most 6 significant bits)."""
    v = torch.tensor(E2M1, device=code.device)[code.int()]
    return (v.reshape(*block.shape, 16) * block.float().unsqueeze(2)).reshape(code.shape) * row


def _plain_rotate(x, cos, sin, interleaved):
    R = 2 * cos.shape[-1]
    v = x.float()
    a, b = (v[..., 0:R:2], v[..., 1:R:2]) if interleaved else (v[..., :R // 2], v[..., R // 2:R])
    u, w = a * cos - b * sin, a * sin + b * cos
    rot = torch.stack([u, w], -1).flatten(-2) if interleaved else torch.cat([u, w], -1)
    return torch.cat([rot, v[..., R:]], -1).to(x.dtype)


def _plain_norm(v, norm, eps=1e-6):
    if norm == "layer":
        v = v - v.mean(-1, keepdim=True)
    return v * torch.rsqrt((v * v).mean(-1, keepdim=True) + eps)


def _rows_of(m, cu, T):
    """A per-sequence tensor [n, C] as one row for each token."""
    at = torch.arange(T, device=m.device)[:, None]
    return ((at >= cu[None, :-1]) & (at < cu[None, 1:])).float() @ m.float()


def _grads(outs, leaves, douts):
    return list(torch.autograd.grad(outs, leaves, douts))


def run(s):
    c = s["case"]
    op = c["op"]
    if op == "rotary":
        axes = _ints(c["axes"])
        if own:
            from minimaxh3_b200.kernels.rotary import rotary_axes

            q, k = rotary_axes(s["q"], s["k"], s["positions"], axes, theta=10000.0, interleaved=c["interleaved"])
        else:
            turn = [s["positions"][:, a, None].double() * 10000.0 ** (-2.0 * torch.arange(d // 2, device=DEV, dtype=torch.float64) / d)
                    for a, d in enumerate(axes)]
            angle = torch.cat(turn, -1)
            cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
            q, k = _plain_rotate(s["q"], cos, sin, c["interleaved"]), _plain_rotate(s["k"], cos, sin, c["interleaved"])
        return [q, k] + (_grads([q, k], [s["q"], s["k"]], [s["dq"], s["dk"]]) if c["grad"] else [])
    if op == "norm_modulate":
        if own:
            from minimaxh3_b200.kernels.block_norm import norm_modulate

            h = norm_modulate(s["x"], s["scale"], s["shift"], weight=s["weight"], bias=s["bias"], norm=c["norm"], eps=1e-6)
        else:
            n = _plain_norm(s["x"].float(), c["norm"])
            n = n * s["weight"].float() if s["weight"] is not None else n
            n = n + s["bias"].float() if s["bias"] is not None else n
            scale, shift = ((m if c["per_token"] else m.unsqueeze(1)).float() for m in (s["scale"], s["shift"]))
            h = (n * (1 + scale) + shift).to(s["x"].dtype)
        return [h] + (_grads([h], s["leaves"], [s["dh"]]) if c["grad"] else [])
    if op == "gated_residual_norm":
        if own:
            from minimaxh3_b200.kernels.block_norm import gated_residual_norm

            r, h = gated_residual_norm(s["x"], s["y"], s["gate"], s["scale"], s["shift"], y_norm=c["y_norm"],
                                       y_weight=s["y_weight"], residual_scale=c["alpha"], norm=c["norm"], eps=1e-6, cu_seqlens=s["cu"])
        else:
            T = s["x"].shape[0]
            z = s["y"].float() if c["y_norm"] == "none" else _plain_norm(s["y"].float(), c["y_norm"]) * s["y_weight"].float()
            r = c["alpha"] * s["x"].float() + _rows_of(s["gate"], s["cu"], T) * z
            h = _plain_norm(r, c["norm"]) * (1 + _rows_of(s["scale"], s["cu"], T)) + _rows_of(s["shift"], s["cu"], T)
            r, h = r.to(s["x"].dtype), h.to(s["x"].dtype)
        return [r, h] + (_grads([r, h], s["leaves"], [s["dr"], s["dh"]]) if c["grad"] else [])
    if op == "fp4_round_trip":
        if own:
            from minimaxh3_b200.kernels.fp4_linear import dequantize_fp4, quantize_fp4

            return dequantize_fp4(*quantize_fp4(s["x"]))
        return _values(*_round_fp4(s["x"])).to(torch.bfloat16)
    if own:
        from minimaxh3_b200.kernels.fp4_linear import fp4_linear

        return fp4_linear(s["x"], s["w4"], s["w_block"], s["w_scale"], bias=s["bias"])
    w = _values(_unpack(s["w4"]), _untile(s["w_block"], c["n"], c["k"] // 16), s["w_scale"])
    out = _values(*_round_fp4(s["x"])) @ w.t()
    return (out + s["bias"].float() if s["bias"] is not None else out).to(torch.bfloat16)


# ---------------------------------------------------------------------------
# what a case cannot do without
# ---------------------------------------------------------------------------


def work(case):
    op, e = case["op"], TYPES[case["dtype"]].itemsize
    if op == "rotary":
        f, h, w = _ints(case["grid"], "x")
        n = case["batch"] * f * h * w * (case["heads"] + case["kv_heads"]) * case["dim"]
        passes = 2 if case["grad"] else 1
        return {"bytes": passes * (2 * n * e + 12 * f * h * w), "flops": passes * 3 * n}
    if op in ("norm_modulate", "gated_residual_norm"):
        md = TYPES[case["mod"]].itemsize
        C = case["channels"]
        if op == "norm_modulate":
            rows, groups, mods, streams, back = case["batch"] * case["tokens"], case["batch"], 2, 2, 3
            groups = rows if case["per_token"] else groups
        else:
            lens = _ints(case["lengths"])
            rows, groups, mods, streams, back = sum(lens), len(lens), 3, 4, 6
        n = rows * C
        b = streams * n * e + mods * groups * C * md
        if case["grad"]:
            b += back * n * e + 2 * mods * groups * C * md
        return {"bytes": b, "flops": (10 if op == "norm_modulate" else 16) * n * (3 if case["grad"] else 1)}
    M, K = case["rows"], case["k"]
    if op == "fp4_round_trip":
        return {"bytes": M * K * (e + 2 + 2 * 0.5625), "flops": 6 * M * K}
    N = case["n"]
    return {"bytes": M * K * e + N * K * 0.5625 + 2 * M * N + 4 * N, "flops": 2 * M * N * K}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------


def _exact_norm(v, kind, eps=1e-6):
    """(xhat, rstd) of each row."""
    if kind == "none":
        return v, None
    mu = v.sum(-1, keepdim=True) / v.shape[-1] if kind == "layer" else torch.zeros_like(v[..., :1])
    rstd = 1.0 / torch.sqrt(((v - mu) ** 2).sum(-1, keepdim=True) / v.shape[-1] + eps)
    return (v - mu) * rstd, rstd


def _exact_norm_grad(dn, n, rstd, kind):
    """The gradient of the input of a norm from that of its result: (dn - mean(dn) - n mean(n dn)) rstd."""
    if kind == "none":
        return dn
    d = dn - n * (dn * n).mean(-1, keepdim=True)
    return rstd * (d - dn.mean(-1, keepdim=True) if kind == "layer" else d)


def _floor_log2(v):
    return (v.view(torch.int64) >> 52) - 1023


def _pow2(e):
    return ((e + 1023) << 52).view(torch.float64)


def _exact_fp4(x):
    """The values that rounding to 4 bits leaves: steps of 1/2 below 2, 1 below 4 and 2 above, ties to even."""
    M, K = x.shape
    v = x.to(torch.float64).view(M, -1, 16)
    amax = v.abs().amax((1, 2)).clamp(min=1e-300)
    up = _floor_log2(amax / 1344)  # 2^up <= amax / 1344, so 2^up >= amax / 2688 unless amax / 1344 is a power of two itself
    up = torch.where(_pow2(up) * 1344 == amax, up - 1, up)
    row = _pow2(up.clamp(min=-100)).view(M, 1, 1)
    t = v.abs().amax(2, keepdim=True) / (6 * row)
    step = _pow2(_floor_log2(t.clamp(min=2.0 ** -6)) - 3)
    s = torch.minimum(torch.round(t / step) * step, torch.full_like(t, 448.0))
    q = torch.where(s > 0, v / (s * row).clamp(min=1e-300), torch.zeros_like(v))
    step = torch.where(q.abs() < 2, 0.5, torch.where(q.abs() < 4, 1.0, 2.0))
    return (torch.round(q / step) * step).clamp(-6, 6).mul(s * row).view(M, K)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    with torch.no_grad():
        if op == "rotary":
            f, h, w = _ints(case["grid"], "x")
            axes = _ints(case["axes"])
            which = torch.tensor([a for a, d in enumerate(axes) for _ in range(d // 2)], device=DEV)
            rate = torch.tensor([math.pow(10000.0, -2.0 * j / d) for d in axes for j in range(d // 2)], dtype=torch.float64, device=DEV)
            z = torch.polar(torch.ones((), dtype=torch.float64, device=DEV), s["positions"].double()[:, which] * rate)
            R = sum(axes)

            def turn(x, z):
                v = x.double()
                p = v[..., :R].unflatten(-1, (R // 2, 2)) if case["interleaved"] else v[..., :R].unflatten(-1, (2, R // 2)).transpose(-1, -2)
                p = torch.view_as_real(torch.view_as_complex(p.contiguous()) * z)
                p = p if case["interleaved"] else p.transpose(-1, -2)
                return torch.cat([p.flatten(-2), v[..., R:]], -1)

            out = [turn(s["q"], z), turn(s["k"], z)]
            return out + ([turn(s["dq"], z.conj()), turn(s["dk"], z.conj())] if case["grad"] else [])
        if op == "norm_modulate":
            n, rstd = _exact_norm(s["x"].double(), case["norm"])
            sc, sh = ((m if case["per_token"] else m[:, None]).double() for m in (s["scale"], s["shift"]))
            w = s["weight"].double() if s["weight"] is not None else torch.ones(case["channels"], dtype=torch.float64, device=DEV)
            b = s["bias"].double() if s["bias"] is not None else torch.zeros_like(w)
            out = [(n * w + b) * (1 + sc) + sh]
            if case["grad"]:
                dh = s["dh"].double()
                tok = (lambda t: t) if case["per_token"] else (lambda t: t.sum(1))
                dw = [(dh * (1 + sc) * n).sum((0, 1))] if s["weight"] is not None else []
                db = [(dh * (1 + sc)).sum((0, 1))] if s["bias"] is not None else []
                out += [_exact_norm_grad(dh * (1 + sc) * w, n, rstd, case["norm"]), tok(dh * (n * w + b)), tok(dh)] + dw + db
            return out
        if op == "gated_residual_norm":
            lens = _ints(case["lengths"])
            rep = torch.repeat_interleave(torch.arange(len(lens), device=DEV), torch.tensor(lens, device=DEV))
            x, gate, sc, sh = s["x"].double(), s["gate"].double()[rep], s["scale"].double()[rep], s["shift"].double()[rep]
            ny, ry = _exact_norm(s["y"].double(), case["y_norm"])
            wy = s["y_weight"].double() if s["y_weight"] is not None else 1.0
            r = case["alpha"] * x + gate * (ny * wy)
            n, rstd = _exact_norm(r, case["norm"])
            out = [r, n * (1 + sc) + sh]
            if case["grad"]:
                dh = s["dh"].double()
                d = s["dr"].double() + _exact_norm_grad(dh * (1 + sc), n, rstd, case["norm"])

                def per(t):
                    return torch.zeros(len(lens), t.shape[1], dtype=torch.float64, device=DEV).index_add_(0, rep, t)

                out += [case["alpha"] * d, _exact_norm_grad(d * gate * wy, ny, ry, case["y_norm"]), per(d * ny * wy), per(dh * n), per(dh)]
                if s["y_weight"] is not None:
                    out.append((d * gate * ny).sum(0))
            return out
        if op == "fp4_round_trip":
            return _exact_fp4(s["x"])
        N, K = case["n"], case["k"]
        v = torch.tensor([0, 1, 2, 3, 4, 6, 8, 12], dtype=torch.float64, device=DEV) / 2
        byte = s["w4"].long()
        w = torch.empty(N, K, dtype=torch.float64, device=DEV)
        for half, code in ((0, byte % 16), (1, byte // 16)):
            w[:, half::2] = v[code % 8] * (1 - 2 * (code // 8)).double()
        rows, col = torch.arange(N, device=DEV)[:, None], torch.arange(K // 16, device=DEV)[None]
        w = w.view(N, -1, 16) * s["w_block"].float()[rows // 128, col // 4, rows % 32, rows % 128 // 32, col % 4].double()[..., None]
        out = _exact_fp4(s["x"]) @ (w.view(N, K) * s["w_scale"].double()).t()
        return out + s["bias"].double() if s["bias"] is not None else out
