"""The norms before and after a block against their definition in 64 bits, forward and backward.

Tolerances, with u = 2^-24: a row's sums go through at most 8 + 5 + 5 additions, so
its mean is off by 20 u max|v| and its deviation sigma by a relative 24 u (1 + 2
max|v| / sigma); the reciprocal root adds 2 u.  xhat is then off by at most
F = 64 u (1 + max|v| / sigma) times (1 + |xhat|).  Products with the modulation
add a few u each (within F), and the result is rounded once: half a step of its
type.  A column sum of n terms is off by at most n u times the sum of their
magnitudes, in any order, beside the terms' own F.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24


def _rand(seed, *shape, dtype=torch.bfloat16, scale=1.0, shift=0.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=DEV) * scale + shift).to(dtype)


def _norm(v, kind, eps):
    """(xhat, rstd, F)."""
    if kind == "none":
        return v, torch.ones_like(v[..., :1]), torch.zeros_like(v[..., :1])
    mu = v.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(v[..., :1])
    rstd = ((v - mu) ** 2).mean(-1, keepdim=True).add(eps).rsqrt()
    return (v - mu) * rstd, rstd, 64 * U * (1 + v.abs().amax(-1, keepdim=True) * rstd)


def _back(dn, n, rstd, kind):
    """(gradient, sum of the magnitudes it is made of)."""
    if kind == "none":
        return dn, dn.abs()
    m1 = (dn * n).mean(-1, keepdim=True)
    m0 = dn.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(m1)
    mag = dn.abs() + dn.abs().mean(-1, keepdim=True) + n.abs() * (dn * n).abs().mean(-1, keepdim=True)
    return rstd * (dn - m0 - n * m1), rstd * mag


def _half(t, v):
    f = torch.finfo(t.dtype)
    return f.eps / 2 * v.abs() + f.smallest_normal * f.eps


def _close(got, ref, err, what=""):
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    d = (got.double() - ref).abs()
    tol = _half(got, ref.abs() + err) + err
    assert bool((d <= tol).all()), (what, float((d - tol).max()))


class Case:
    """One call with its 64-bit values; modulation tensors are given per row (``rows_of`` expands them)."""

    def __init__(self, x, y=None, gate=None, scale=None, shift=None, weight=None, bias=None, y_weight=None, norm="layer", y_norm="none",
                 alpha=1.0, eps=1e-6, rows_of=lambda t: t):
        d = lambda t, dflt: dflt if t is None else rows_of(t.detach()).double()
        c = lambda t, dflt: dflt if t is None else t.detach().double()
        self.x, self.norm, self.y_norm, self.alpha = x, norm, y_norm, alpha
        x64 = x.detach().double()
        self.g, self.sc, self.sh = d(gate, 1.0), d(scale, 0.0), d(shift, 0.0)
        self.w, self.b, self.wy = c(weight, 1.0), c(bias, 0.0), c(y_weight, 1.0)
        if y is None:
            self.r, self.er, self.yh = x64, torch.zeros_like(x64), None
        else:
            self.yh, self.ry, self.Fy = _norm(y.detach().double(), y_norm, eps)
            gz = self.g * self.wy
            self.gz = gz
            self.r = alpha * x64 + gz * self.yh
            self.er = abs(gz) * self.Fy * (1 + self.yh.abs()) + 4 * U * (abs(alpha) * x64.abs() + abs(gz * self.yh))
        if norm != "none":
            self.xh, self.rstd, self.F = _norm(self.r, norm, eps)
            # an error of r moves xhat by itself over sigma, and sigma by at most the largest of the row's
            self.F = self.F + 3 * self.er.amax(-1, keepdim=True) * self.rstd
            A = self.w * (1 + self.sc)
            self.A = A
            self.h = (self.xh * self.w + self.b) * (1 + self.sc) + self.sh
            self.eh = abs(A) * self.F * (1 + self.xh.abs()) + 8 * U * (abs(A * self.xh) + abs(self.b * (1 + self.sc)) + abs(self.sh))

    def grads(self, dr, dh, group_sum):
        """{name: (gradient, error)}; ``group_sum`` adds rows as the modulation belongs to them."""
        z = torch.zeros_like(self.r)
        dr, dh = z if dr is None else dr.double(), z if dh is None else dh.double()
        out, n = {}, self.x[..., 0].numel()
        d, mag, F = dr, dr.abs() * 4 * U, torch.zeros_like(z[..., :1])
        if self.norm != "none":
            F = self.F
            dn = dh * self.A
            g, m = _back(dn, self.xh, self.rstd, self.norm)
            d, mag = dr + g, mag + m * F * 4 * (1 + self.xh.abs())

            def col(name, terms, err):
                out[name] = (group_sum(terms), group_sum(terms.abs() * (n + 64) * U + err))

            xw = self.xh * self.w + self.b
            col("scale", dh * xw, dh.abs() * abs(self.w) * F * (1 + self.xh.abs()) + 8 * U * abs(dh * xw))
            col("shift", dh, z)
            t = dh * (1 + self.sc)
            S = lambda v: v.reshape(-1, v.shape[-1]).sum(0)
            out["weight"] = (S(t * self.xh), S((t * self.xh).abs() * (n + 64) * U + t.abs() * F * (1 + self.xh.abs())))
            out["bias"] = (S(t), S(t.abs() * (n + 64) * U))
        k = self.alpha if self.yh is not None else 1.0
        out["x"] = (k * d, abs(k) * mag + 2 * U * abs(k * d))
        if self.yh is not None:
            ey = self.Fy * (1 + self.yh.abs())
            t = d * self.yh * self.wy
            out["gate"] = (group_sum(t), group_sum(t.abs() * (n + 64) * U + abs(self.wy) * (mag * self.yh.abs() + d.abs() * ey)))
            dz = d * self.gz
            g, m = _back(dz, self.yh, self.ry, self.y_norm)
            em, _ = _back(z, self.yh, self.ry, self.y_norm)
            _, spread = _back(mag * abs(self.gz), self.yh, self.ry, self.y_norm)
            out["y"] = (g, m * (4 * self.Fy * (1 + self.yh.abs()) + 8 * U) + spread)
            t = d * self.g * self.yh
            S = lambda v: v.reshape(-1, v.shape[-1]).sum(0)
            out["y_weight"] = (S(t), S(t.abs() * (n + 64) * U + abs(self.g) * (mag * self.yh.abs() + d.abs() * ey)))
        return out


SIZES = [(1, 1, 8), (2, 3, 64), (3, 37, 104), (1, 5, 1), (2, 9, 7), (1, 70, 1544), (2, 300, 128), (1, 3, 8192), (2, 11, 5120)]


@pytest.mark.parametrize("B,S,C", SIZES)
@pytest.mark.parametrize("dtype,mod", [(torch.bfloat16, torch.float32), (torch.float16, torch.float16), (torch.float32, torch.float32)])
@pytest.mark.parametrize("norm", ["layer", "rms"])
def test_norm_modulate_forward(B, S, C, dtype, mod, norm):
    from minimaxh3_b200.kernels.block_norm import norm_modulate

    x = _rand(1, B, S, C, dtype=dtype, scale=2.0, shift=1.5)
    sc, sh = _rand(2, B, C, dtype=mod, scale=0.3), _rand(3, B, C, dtype=mod, scale=0.3)
    w, b = _rand(4, C, dtype=mod, shift=1.0), _rand(5, C, dtype=mod)
    per = lambda t: t[:, None].expand(B, S, C)
    for kw in (dict(scale=sc, shift=sh, weight=w, bias=b), dict(scale=sc), dict(shift=sh, weight=w), dict(bias=b), dict()):
        c = Case(x, norm=norm, rows_of=per, **kw)
        _close(norm_modulate(x, norm=norm, **kw), c.h, c.eh)
    # the same modulation as [B, 1, C] and as a row for each token
    full = norm_modulate(x, sc, sh, norm=norm)
    assert torch.equal(norm_modulate(x, sc[:, None], sh[:, None], norm=norm), full)
    c = Case(x, scale=sc, shift=sh, norm=norm, rows_of=per)  # another kernel, another order of the sums: the same bound
    tok = norm_modulate(x, per(sc).contiguous(), per(sh).contiguous(), norm=norm)
    _close(tok, c.h, c.eh)
    assert torch.equal(norm_modulate(x, per(sc).contiguous(), sh, norm=norm), tok)


@pytest.mark.parametrize("B,S,C", [(1, 1, 8), (3, 37, 104), (2, 9, 7), (1, 70, 1544), (2, 11, 5120)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("y_norm,norm", [("none", "layer"), ("rms", "rms"), ("layer", "layer"), ("rms", "none")])
def test_gated_residual_forward(B, S, C, dtype, y_norm, norm):
    from minimaxh3_b200.kernels.block_norm import gated_residual_norm

    x, y = _rand(6, B, S, C, dtype=dtype, shift=0.5), _rand(7, B, S, C, dtype=dtype, scale=3.0, shift=-1.0)
    f = torch.float32
    kw = dict(gate=_rand(8, B, C, dtype=f))
    if y_norm != "none":
        kw["y_weight"] = _rand(9, C, dtype=f, shift=1.0)
    if norm != "none":
        kw |= dict(scale=_rand(10, B, C, dtype=f, scale=0.3), shift=_rand(11, B, C, dtype=f), weight=_rand(12, C, dtype=dtype, shift=1.0))
    for alpha in (1.0, -0.75):
        c = Case(x, y, norm=norm, y_norm=y_norm, alpha=alpha, rows_of=lambda t: t[:, None].expand(B, S, C), **kw)
        r, h = gated_residual_norm(x, y, norm=norm, y_norm=y_norm, residual_scale=alpha, **kw)
        _close(r, c.r, c.er, "r")
        assert (h is None) == (norm == "none")
        if h is not None:
            _close(h, c.h, c.eh, "h")


@pytest.mark.parametrize("lens,before,after", [([5, 0, 33, 1], 0, 0), ([100], 3, 4), ([1] * 40, 0, 1), ([0, 0], 2, 2), ([700, 2, 650], 0, 9)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_packed_sequences(lens, before, after, dtype):
    """Modulation by sequence; rows outside every sequence give zeros, and zero gradients."""
    from minimaxh3_b200.kernels.block_norm import gated_residual_norm

    C, n = 136, len(lens)
    cu = torch.tensor([before + sum(lens[:i]) for i in range(n + 1)], dtype=torch.int32, device=DEV)
    T = before + sum(lens) + after
    rep = torch.repeat_interleave(torch.arange(n), torch.tensor(lens)).to(DEV)
    inside = slice(before, before + sum(lens))
    f = torch.float32
    leaf = lambda t: t.requires_grad_(True)
    x, y = leaf(_rand(13, T, C, dtype=dtype)), leaf(_rand(14, T, C, dtype=dtype))
    kw = dict(gate=leaf(_rand(15, n, C, dtype=f)), scale=leaf(_rand(16, n, C, dtype=f, scale=0.3)), shift=leaf(_rand(17, n, C, dtype=f)),
              y_weight=leaf(_rand(18, C, dtype=f, shift=1.0)))
    r, h = gated_residual_norm(x, y, y_norm="rms", norm="layer", residual_scale=0.5, cu_seqlens=cu, **kw)
    dr, dh = _rand(19, T, C, dtype=dtype), _rand(20, T, C, dtype=dtype)
    grads = torch.autograd.grad((r, h), (x, y, *kw.values()), (dr, dh))
    c = Case(x[inside], y[inside], norm="layer", y_norm="rms", alpha=0.5, rows_of=lambda t: t[rep], **kw)
    _close(r[inside], c.r, c.er, "r")
    _close(h[inside], c.h, c.eh, "h")
    want = c.grads(dr[inside], dh[inside], lambda t: torch.zeros(n, C, dtype=t.dtype, device=DEV).index_add_(0, rep, t))
    for name, g in zip(("x", "y", *kw), grads):
        if name in ("x", "y"):
            _close(g[inside], *want[name], name)
        else:
            _close(g, *want[name], name)
    for t in (r, h, grads[0], grads[1]):
        assert bool((t[:before] == 0).all()) and bool((t[before + sum(lens):] == 0).all())


@pytest.mark.parametrize("B,S,C", [(1, 1, 8), (2, 45, 104), (2, 9, 7), (1, 700, 1544), (3, 11, 5120), (1, 2, 8192), (5, 400, 64)])
@pytest.mark.parametrize("dtype,mod", [(torch.bfloat16, torch.float32), (torch.float16, torch.float16), (torch.float32, torch.float32)])
@pytest.mark.parametrize("norm,y_norm,per_token", [("layer", None, False), ("rms", None, True), ("layer", "none", False), ("rms", "layer", False),
                                                   ("layer", "rms", True), ("none", "rms", False)])
def test_gradients(B, S, C, dtype, mod, norm, y_norm, per_token):
    from minimaxh3_b200.kernels.block_norm import gated_residual_norm, norm_modulate

    leaf = lambda t: t.requires_grad_(True)
    shape = (B, S, C) if per_token else (B, C)
    x, kw = leaf(_rand(21, B, S, C, dtype=dtype, shift=0.5)), {}
    if norm != "none":
        kw |= dict(scale=leaf(_rand(22, *shape, dtype=mod, scale=0.3)), shift=leaf(_rand(23, *shape, dtype=mod)),
                   weight=leaf(_rand(24, C, dtype=mod, shift=1.0)), bias=leaf(_rand(25, C, dtype=mod)))
    if y_norm is not None:
        kw["gate"] = leaf(_rand(26, *shape, dtype=mod))
        if y_norm != "none":
            kw["y_weight"] = leaf(_rand(27, C, dtype=mod, shift=1.0))
    per = (lambda t: t) if per_token else (lambda t: t[:, None].expand(B, S, C))
    total = (lambda t: t) if per_token else (lambda t: t.sum(1))
    dr, dh = _rand(28, B, S, C, dtype=dtype), _rand(29, B, S, C, dtype=dtype)
    if y_norm is None:
        c = Case(x, norm=norm, rows_of=per, **kw)
        grads = torch.autograd.grad(norm_modulate(x, norm=norm, **kw), (x, *kw.values()), dh)
        want, names = c.grads(None, dh, total), ("x", *kw)
    else:
        y = leaf(_rand(30, B, S, C, dtype=dtype, scale=2.0, shift=-0.5))
        c = Case(x, y, norm=norm, y_norm=y_norm, alpha=0.5, rows_of=per, **kw)
        r, h = gated_residual_norm(x, y, norm=norm, y_norm=y_norm, residual_scale=0.5, **kw)
        outs, douts = ((r,), (dr,)) if h is None else ((r, h), (dr, dh))
        grads = torch.autograd.grad(outs, (x, y, *kw.values()), douts)
        want, names = c.grads(dr, None if h is None else dh, total), ("x", "y", *kw)
    for name, g in zip(names, grads):
        assert g.dtype == dict(x=x, y=x, **kw)[name].dtype
        _close(g, *want[name], name)


@pytest.mark.parametrize("C", [64, 1928, 5120])
@pytest.mark.parametrize("dtype,mods", [(torch.bfloat16, (torch.float32,) * 3), (torch.bfloat16, (torch.bfloat16,) * 3),
                                        (torch.float32, (torch.float32, torch.bfloat16, torch.float32))])
def test_modulation_by_token_of_several_groups(C, dtype, mods):
    """Rows of one modulation beside groups of another, views of a wider tensor, and more rows than one block's."""
    from minimaxh3_b200.kernels.block_norm import gated_residual_norm, norm_modulate

    B, S = 3, 331
    leaf = lambda t: t.requires_grad_(True)
    x, y = leaf(_rand(110, B, S, C, dtype=dtype)), leaf(_rand(111, B, S, C, dtype=dtype, shift=0.3))
    wide = _rand(112, B, S, 2 * C, dtype=mods[0], scale=0.3)
    gate, scale, shift = leaf(wide[..., C:]), leaf(_rand(113, B, C, dtype=mods[1], scale=0.3)), leaf(_rand(114, B, S, C, dtype=mods[2]))
    per = lambda t: t if t.dim() == 3 else t[:, None].expand(B, S, C)
    c = Case(x, y, gate=per(gate), scale=per(scale), shift=shift, norm="layer", y_norm="none")
    r, h = gated_residual_norm(x, y, gate, scale, shift)
    _close(r, c.r, c.er)
    _close(h, c.h, c.eh)
    dr, dh = _rand(115, B, S, C, dtype=dtype), _rand(116, B, S, C, dtype=dtype)
    names = ("x", "y", "gate", "scale", "shift")
    want = c.grads(dr, dh, lambda t: t)
    got = dict(zip(names, torch.autograd.grad((r, h), (x, y, gate, scale, shift), (dr, dh), retain_graph=True)))
    for name in ("x", "y", "gate", "shift"):
        _close(got[name], *want[name], name)
    # the rows' gradients of scale are rounded to its type one by one, and their sum once more
    terms, err = want["scale"]
    u = torch.finfo(mods[1]).eps / 2
    tol = (err + u * (terms.abs() + err)).sum(1) * (1 + u) + u * terms.sum(1).abs() + S * U * terms.abs().sum(1)
    assert bool(((got["scale"].double() - terms.sum(1)).abs() <= tol).all())
    # h unused, r unused
    want = c.grads(dr, None, lambda t: t)
    for name, g in zip(names, torch.autograd.grad(r, (x, y, gate, scale, shift), dr, retain_graph=True)):
        if name in ("scale", "shift"):
            assert bool((g == 0).all())
        else:
            _close(g, *want[name], name)
    want = c.grads(None, dh, lambda t: t)
    for name, g in zip(("x", "y", "gate", "shift"), torch.autograd.grad(h, (x, y, gate, shift), dh)):
        _close(g, *want[name], name)
    # the same rows packed, with rows outside every sequence
    flat = lambda t: t.detach().reshape(B * S, C)
    cu = torch.tensor([7, 7, 500, B * S - 20], dtype=torch.int32, device=DEV)
    sc, sh = leaf(flat(per(scale)).to(mods[0]).clone()), leaf(flat(shift).to(mods[0]).clone())
    xs = leaf(flat(x).clone())
    c = Case(xs, scale=sc, shift=sh, norm="rms")
    h = norm_modulate(xs, sc, sh, norm="rms", cu_seqlens=cu)
    inside = slice(7, B * S - 20)
    _close(h[inside], c.h[inside], c.eh[inside])
    dh = flat(dh)
    want = c.grads(None, dh, lambda t: t)
    for name, g in zip(("x", "scale", "shift"), torch.autograd.grad(h, (xs, sc, sh), dh)):
        _close(g[inside], want[name][0][inside], want[name][1][inside], name)
        assert bool((g[:7] == 0).all()) and bool((g[B * S - 20:] == 0).all())
    assert bool((h[:7] == 0).all()) and bool((h[B * S - 20:] == 0).all())


def test_gradients_against_differences():
    """The kernel's gradients along random directions, against central differences of the 64-bit forward (step 1e-5:
    the truncation is of order 1e-10, far below f32's 1e-6 of the slope)."""
    from minimaxh3_b200.kernels.block_norm import gated_residual_norm

    B, S, C, f = 2, 13, 72, torch.float32
    shapes = dict(x=(B, S, C), y=(B, S, C), gate=(B, C), scale=(B, C), shift=(B, C), weight=(C,), bias=(C,), y_weight=(C,))
    t = {n: _rand(40 + i, *s, dtype=f, scale=0.7, shift=0.2).requires_grad_(True) for i, (n, s) in enumerate(shapes.items())}
    dr, dh = _rand(50, B, S, C, dtype=f), _rand(51, B, S, C, dtype=f)
    conf = dict(norm="layer", y_norm="rms")
    grads = dict(zip(t, torch.autograd.grad(gated_residual_norm(residual_scale=0.5, **conf, **t), tuple(t.values()), (dr, dh))))

    def value(moved):
        c = Case(alpha=0.5, rows_of=lambda m: m[:, None].expand(B, S, C), **conf, **moved)
        return float((c.r * dr.double()).sum() + (c.h * dh.double()).sum())

    base = {n: v.detach().double() for n, v in t.items()}
    for i, n in enumerate(t):
        v = _rand(60 + i, *shapes[n], dtype=torch.float64)
        step = 1e-5
        slope = (value(base | {n: base[n] + step * v}) - value(base | {n: base[n] - step * v})) / (2 * step)
        got = float((grads[n].double() * v).sum())
        size = float((grads[n].double() * v).abs().sum())
        assert abs(got - slope) <= 1e-5 * size + 1e-6, (n, got, slope)


def test_broadcast_inputs_and_partial_gradients():
    from minimaxh3_b200.kernels.block_norm import gated_residual_norm, norm_modulate

    B, S, C, f = 3, 20, 64, torch.float32
    x = _rand(70, B, S, C, dtype=f)
    sc = _rand(71, C, dtype=f).requires_grad_(True)      # one row for every batch item
    sh = _rand(72, 1, 1, C, dtype=f).requires_grad_(True)
    dh = _rand(73, B, S, C, dtype=f)
    gs, gh = torch.autograd.grad(norm_modulate(x, sc, sh), (sc, sh), dh)
    c = Case(x, scale=sc.detach().expand(B, S, C), shift=sh.detach().expand(B, S, C))
    want = c.grads(None, dh, lambda t: t.sum((0, 1)))
    _close(gs, *want["scale"])
    _close(gh, want["shift"][0].view(1, 1, C), want["shift"][1].view(1, 1, C))
    # only r is used: h's gradient is absent
    y, g = _rand(74, B, S, C, dtype=f).requires_grad_(True), _rand(75, B, C, dtype=f).requires_grad_(True)
    r, h = gated_residual_norm(x, y, g)
    dy, dg = torch.autograd.grad(r, (y, g), dh)
    c = Case(x, y, gate=g, rows_of=lambda t: t[:, None].expand(B, S, C))
    want = c.grads(dh, None, lambda t: t.sum(1))
    _close(dy, *want["y"])
    _close(dg, *want["gate"])
    # only h is used
    r, h = gated_residual_norm(x, y, g)
    (dy,) = torch.autograd.grad(h, y, dh)
    _close(dy, *c.grads(None, dh, lambda t: t.sum(1))["y"])
    # what only h depends on has the gradient 0 when h is not used, by group and by token
    for lead in ((B,), (B, S)):
        sc = _rand(77, *lead, C, dtype=f).requires_grad_(True)
        w = _rand(78, C, dtype=f).requires_grad_(True)
        r, _ = gated_residual_norm(x, y, g, sc, sc, weight=w)
        ds, dw, dy2 = torch.autograd.grad(r, (sc, w, y), dh)
        assert bool((ds == 0).all()) and bool((dw == 0).all())
        want = Case(x, y, gate=g, rows_of=lambda t: t[:, None].expand(B, S, C)).grads(dh, None, lambda t: t.sum(1))
        _close(dy2, *want["y"])
    # x and y are the same tensor, and an input is shared by two calls
    xs = _rand(76, B, S, C, dtype=f).requires_grad_(True)
    r, h = gated_residual_norm(xs, xs, g.detach())
    (dx,) = torch.autograd.grad(r, xs, dh)
    torch.testing.assert_close(dx, dh + dh * g.detach()[:, None], rtol=2.0 ** -21, atol=2.0 ** -21)


def test_strides_streams_graphs_and_repeatability():
    from minimaxh3_b200.kernels.block_norm import gated_residual_norm, norm_modulate

    B, S, C = 2, 50, 128
    wide = _rand(80, B, S, 3 * C + 8)
    x, y = wide[..., :C], wide[..., C:2 * C]
    odd = wide[..., 2 * C + 1:3 * C + 1]  # one element off a vector
    sc, g = _rand(81, B, 2 * C, dtype=torch.float32), _rand(82, B, C, dtype=torch.float32)
    ref = gated_residual_norm(x.contiguous(), y.contiguous(), g, sc[:, C:].contiguous())
    got = gated_residual_norm(x, y, g, sc[:, C:])
    assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
    assert torch.equal(norm_modulate(odd), norm_modulate(odd.contiguous()))
    assert torch.equal(norm_modulate(_rand(83, C, B, S).permute(1, 2, 0)), norm_modulate(_rand(83, C, B, S).permute(1, 2, 0).contiguous()))
    leaves = [t.detach().clone().requires_grad_(True) for t in (x, y, g, sc[:, C:])]
    dh = _rand(84, B, S, C)
    step = lambda: torch.autograd.grad(gated_residual_norm(*leaves)[1], leaves, dh)
    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, again))  # column sums have one order
    graphs, caps = [], []
    for _ in range(2):  # two captured steps, each with its own workspace
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            caps.append(step())
        graphs.append(graph)
    for graph in graphs:
        graph.replay()
    torch.cuda.synchronize()
    for cap in caps:
        assert all(torch.equal(a, b) for a, b in zip(first, cap))


def test_empty_inputs_and_large_offsets():
    from minimaxh3_b200.kernels.block_norm import norm_modulate

    for shape in ((0, 4, 64), (2, 0, 64)):
        x = _rand(85, *shape, dtype=torch.float32).requires_grad_(True)
        sc = _rand(86, shape[0], 64, dtype=torch.float32).requires_grad_(True)
        h = norm_modulate(x, sc)
        assert h.shape == x.shape
        dx, ds = torch.autograd.grad(h, (x, sc), torch.zeros_like(h))
        assert dx.shape == x.shape and ds.shape == sc.shape and bool((ds == 0).all())
    far = 2 ** 30 + 64  # elements between rows: the third starts past 2^31
    buf = torch.zeros(2 * far + 256, dtype=torch.bfloat16, device=DEV)
    x = buf.as_strided((3, 256), (far, 1))
    x.copy_(_rand(87, 3, 256))
    assert torch.equal(norm_modulate(x), norm_modulate(x.contiguous()))


def test_bad_offsets_stay_inside():
    """Offsets are data: entries outside [0, T] are clamped, and rows that no sequence holds give zeros."""
    from minimaxh3_b200.kernels.block_norm import norm_modulate

    x = _rand(88, 40, 64)
    sc = _rand(89, 2, 64)
    got = norm_modulate(x, sc, cu_seqlens=torch.tensor([-7, 10, 99], dtype=torch.int32, device=DEV))
    assert torch.equal(got, norm_modulate(x, sc, cu_seqlens=torch.tensor([0, 10, 40], dtype=torch.int32, device=DEV)))


def test_infinite_rows_keep_to_themselves():
    from minimaxh3_b200.kernels.block_norm import norm_modulate

    x = _rand(90, 9, 128)
    clean = norm_modulate(x)
    bad = x.clone()
    bad[3, 5], bad[6, 7] = float("inf"), float("nan")
    got = norm_modulate(bad)
    keep = [0, 1, 2, 4, 5, 7, 8]
    assert torch.equal(got[keep], clean[keep]) and bool(got[3].isnan().all()) and bool(got[6].isnan().all())
    assert bool((norm_modulate(torch.full((2, 64), 3.0, device=DEV)) == 0).all())  # a constant row: its variance is 0


@pytest.mark.parametrize("shift", [0.0, 2.8, 2.9, 40.0, -3000.0])
@pytest.mark.parametrize("C", [64, 1000, 5120])
def test_streams_far_from_zero(shift, C):
    """Means on both sides of the border where the variance is summed again (8 times it), and far past it."""
    from minimaxh3_b200.kernels.block_norm import gated_residual_norm, norm_modulate

    f = torch.float32
    x = _rand(95, 1, 41, C, dtype=f, shift=shift)
    x[:, ::5] -= shift  # rows of both kinds side by side
    c = Case(x)
    _close(norm_modulate(x), c.h, c.eh)
    y, g = _rand(96, 1, 41, C, dtype=f, shift=-shift), _rand(97, C, dtype=f)
    c = Case(x, y, gate=g, y_norm="layer")
    r, h = gated_residual_norm(x, y, g, y_norm="layer")
    _close(r, c.r, c.er)
    _close(h, c.h, c.eh)


@pytest.mark.parametrize("C", [256, 251])
def test_squares_past_the_largest_float(C):
    """Rows near 10^20 whose squares overflow while those around their mean do not."""
    from minimaxh3_b200.kernels.block_norm import norm_modulate

    x = 1e20 * (1 + 1e-3 * _rand(101, 1, 9, C, dtype=torch.float32))
    x[:, ::3] = _rand(102, 1, 3, C, dtype=torch.float32)
    c = Case(x)
    _close(norm_modulate(x), c.h, c.eh)


def test_compiled():
    from minimaxh3_b200.kernels.block_norm import gated_residual_norm

    x, y, g = (_rand(91 + i, 2, 30, 64, dtype=torch.float32).requires_grad_(True) for i in range(3))
    g = _rand(94, 2, 64, dtype=torch.float32).requires_grad_(True)
    f = torch.compile(lambda a, b, c: gated_residual_norm(a, b, c), fullgraph=True, backend="aot_eager")
    r, h = f(x, y, g)
    er, eh = gated_residual_norm(x, y, g)
    assert torch.equal(r, er) and torch.equal(h, eh)
    d = torch.ones_like(h)
    for a, b in zip(torch.autograd.grad((r, h), (x, y, g), (d, d)), torch.autograd.grad((er, eh), (x, y, g), (d, d))):
        assert torch.equal(a, b)


def test_modulation_forms_of_packed_rows():
    """x [T, C]: one row for all, a row for each token, and both at once; other float types beside x."""
    from minimaxh3_b200.kernels.block_norm import gated_residual_norm, norm_modulate

    T, C, f = 33, 136, torch.float32
    x, y = _rand(100, T, C), _rand(101, T, C)
    one, tok, g = _rand(102, C, dtype=f, scale=0.3), _rand(103, T, C, scale=0.3), _rand(104, 1, C, dtype=torch.float16)
    per = lambda t: t.expand(T, C)
    for sc, sh in ((one, one), (one[None], tok), (tok, one), (tok, tok)):
        c = Case(x, scale=per(sc), shift=per(sh))
        _close(norm_modulate(x, sc, sh), c.h, c.eh)
        c = Case(x, y, gate=per(g), scale=per(sc), shift=per(sh), y_norm="layer")
        r, h = gated_residual_norm(x, y, g, sc, sh, y_norm="layer")
        _close(r, c.r, c.er, "r")
        _close(h, c.h, c.eh, "h")
    # gradients of a token's modulation beside one that all tokens share
    leaf = lambda t: t.detach().clone().requires_grad_(True)
    lo, lt, lg = leaf(one), leaf(tok), leaf(g)
    dr, dh = _rand(105, T, C), _rand(106, T, C)
    r, h = gated_residual_norm(x, y, lg, lo, lt)
    go, gt, gg = torch.autograd.grad((r, h), (lo, lt, lg), (dr, dh))
    c = Case(x, y, gate=per(g), scale=per(one), shift=per(tok))
    want = c.grads(dr, dh, lambda t: t)
    _close(gt, *want["shift"])
    # those of the shared rows are rounded per token to their type before they are added: one half step of it each
    for got, name in ((go, "scale"), (gg, "gate")):
        ref, err = want[name]
        err = (err + torch.finfo(got.dtype).eps / 2 * ref.abs()).sum(0) + T * torch.finfo(got.dtype).eps / 2 * ref.abs().sum(0)
        _close(got.view(-1), ref.sum(0), err, name)
    # an 8-wide row that no vector fits, and strides of the modulation
    wide = _rand(107, 2, 3, 4 * 24 + 1, dtype=f)
    c = Case(x.view(1, T, C)[:, :3, :24].expand(2, 3, 24), scale=wide[..., 1:25], shift=wide[..., 25:49])
    _close(norm_modulate(x.view(1, T, C)[:, :3, :24].expand(2, 3, 24), wide[..., 1:25], wide[..., 25:49]), c.h, c.eh)


def test_long_and_short_sequences_share_a_stage():
    """Sequences that end inside the rows a CTA takes at once, and many empty ones."""
    from minimaxh3_b200.kernels.block_norm import norm_modulate

    lens = [1, 0, 0, 2, 1, 3, 700, 1, 1, 0, 5000, 2, 1]
    n, T, C, f = len(lens), sum(lens), 64, torch.float32
    cu = torch.tensor([sum(lens[:i]) for i in range(n + 1)], dtype=torch.int32, device=DEV)
    rep = torch.repeat_interleave(torch.arange(n), torch.tensor(lens)).to(DEV)
    x, sc = _rand(110, T, C).requires_grad_(True), _rand(111, n, C, dtype=f).requires_grad_(True)
    h = norm_modulate(x, sc, cu_seqlens=cu)
    c = Case(x, scale=sc, rows_of=lambda t: t[rep])
    _close(h, c.h, c.eh)
    dh = _rand(112, T, C)
    dx, ds = torch.autograd.grad(h, (x, sc), dh)
    want = c.grads(None, dh, lambda t: torch.zeros(n, C, dtype=t.dtype, device=DEV).index_add_(0, rep, t))
    _close(dx, *want["x"], "x")
    _close(ds, *want["scale"], "scale")


@pytest.mark.parametrize("C", [104, 1928, 2051])
@pytest.mark.parametrize("dtype,by_token", [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float16, torch.float16),
                                            (torch.float32, torch.float32), (torch.float32, torch.bfloat16)])
@pytest.mark.parametrize("shared", ["token", "group", "packed"])
def test_gradients_of_shared_modulations_are_rounded_once(C, dtype, by_token, shared):
    """16-bit modulations that tokens or batch items share: the sum over them is in f32 (a term is off by its own F
    and the sum by n u of their magnitudes) and rounded once - where terms cancel, rounding each would show."""
    from minimaxh3_b200.kernels.block_norm import gated_residual_norm

    B, S, low = 3, 150, torch.float16 if dtype == torch.float16 else torch.bfloat16
    leaf = lambda t: t.requires_grad_(True)  # noqa: E731
    lead = (B, S) if shared != "packed" else (B * S,)
    x, y = leaf(_rand(210, *lead, C, dtype=dtype)), leaf(_rand(211, *lead, C, dtype=dtype, shift=0.3))
    dr, dh = _rand(212, *lead, C, dtype=dtype), _rand(213, *lead, C, dtype=dtype)
    cu = torch.tensor([0, 70, 70 + S, B * S], dtype=torch.int32, device=DEV) if shared == "packed" else None
    gate = leaf(_rand(214, C, dtype=low))
    scale = leaf(_rand(215, *((1, S, C) if shared == "token" else (1, C) if shared == "packed" else (C,)), dtype=low, scale=0.3))
    shift = leaf(_rand(216, *((B, S, C) if shared == "token" else (B, C)), dtype=by_token if shared == "token" else low))
    if shared == "token":
        rows = lambda t: t.expand(B, S, C)  # noqa: E731
    elif shared == "group":
        rows = lambda t: (t if t.dim() == 1 else t[:, None]).expand(B, S, C)  # noqa: E731
    else:
        rep = torch.repeat_interleave(torch.arange(3, device=DEV), torch.tensor([70, S, B * S - 70 - S], device=DEV))
        rows = lambda t: t[rep] if t.shape[:-1] == (3,) else t.expand(B * S, C)  # noqa: E731
    c = Case(x, y, gate=gate, scale=scale, shift=shift, rows_of=rows)
    r, h = gated_residual_norm(x, y, gate, scale, shift, cu_seqlens=cu)
    got = torch.autograd.grad((r, h), (x, y, gate, scale, shift), (dr, dh))
    want = c.grads(dr, dh, lambda t: t)
    _close(got[0], *want["x"], "x")
    _close(got[1], *want["y"], "y")
    for name, m, g in zip(("gate", "scale", "shift"), (gate, scale, shift), got[2:]):
        assert g.dtype == m.dtype and g.shape == m.shape
        terms, err = want[name]
        if shared == "packed" and m.shape[0] == 3:
            total = lambda t: torch.zeros(3, C, dtype=t.dtype, device=DEV).index_add_(0, rep, t)  # noqa: E731
        elif shared == "group" and m.shape[:-1] == (B,):
            total = lambda t: t.sum(1)  # noqa: E731
        else:
            total = lambda t: t.sum_to_size(m.shape)  # noqa: E731
        _close(g, total(terms), total(err + terms.abs() * B * S * U), name)


@pytest.mark.parametrize("C", [64, 1928, 2051])
@pytest.mark.parametrize("dtype,mods", [(torch.bfloat16, (torch.float32,) * 3), (torch.float32, (torch.bfloat16, torch.float32, torch.float16))])
def test_many_batch_items_of_one_row(C, dtype, mods):
    """[B, 1, C] with modulation [B, C]: each row has its own, and the call's memory does not grow by f32 rows for each."""
    from minimaxh3_b200.kernels.block_norm import gated_residual_norm

    B = 3001
    leaf = lambda t: t.requires_grad_(True)  # noqa: E731
    x, y = leaf(_rand(220, B, 1, C, dtype=dtype)), leaf(_rand(221, B, 1, C, dtype=dtype, shift=0.3))
    kw = dict(gate=leaf(_rand(222, B, C, dtype=mods[0])), scale=leaf(_rand(223, B, C, dtype=mods[1], scale=0.3)),
              shift=leaf(_rand(224, B, C, dtype=mods[2])), weight=leaf(_rand(225, C, dtype=torch.float32, shift=1.0)),
              bias=leaf(_rand(226, C, dtype=torch.float32)), y_weight=leaf(_rand(227, C, dtype=dtype, shift=1.0)))
    dr, dh = _rand(228, B, 1, C, dtype=dtype), _rand(229, B, 1, C, dtype=dtype)
    c = Case(x, y, norm="layer", y_norm="rms", rows_of=lambda t: t[:, None], **kw)
    r, h = gated_residual_norm(x, y, norm="layer", y_norm="rms", **kw)
    _close(r, c.r, c.er, "r")
    _close(h, c.h, c.eh, "h")
    want = c.grads(dr, dh, lambda t: t.sum(1))
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    grads = torch.autograd.grad((r, h), (x, y, *kw.values()), (dr, dh))
    made = sum(g.numel() * g.element_size() for g in grads)
    # the gradients, and partial sums of at most 16 CTAs an SM
    assert torch.cuda.max_memory_allocated() - before <= made + (16 * 148 + 2) * 3 * C * 4 + (1 << 20)
    for name, g in zip(("x", "y", *kw), grads):
        _close(g, *want[name], name)
