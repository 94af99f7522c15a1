"""Transformer-block operators (GPU): layer norm, rotary positions and the gated feed-forward block against their formulas in
64 bits on the CPU, at the sizes, strides and types where they can go wrong; gradients also against differences; the block as
it is used, around dm_attention."""
import math

import pytest
import torch

import diffusion_model_amd as d
from diffusion_model_amd import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
# half a step of each type, relative to the value
HALF = {t: torch.finfo(t).eps / 2 for t in DTYPES.values()}


def rand(g, *shape, dtype=torch.float32, scale=1.0, shift=0.0):
    return (torch.randn(*shape, generator=g) * scale + shift).to(dtype)


def close(got, want, tol, what):
    """|got - want| <= tol elementwise; `want` and `tol` in 64 bits on the CPU."""
    got = got.detach().cpu().double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {((got - want).abs() - tol).max().item():.3e} above the bound"


# ------------------------------------------------------------------ layer norm

def norm_oracle(x, w, b, eps, dy=None):
    x = x.double()
    mu = x.mean(-1, keepdim=True)
    rstd = ((x - mu) ** 2).mean(-1, keepdim=True).add(eps).rsqrt()
    z = (x - mu) * rstd
    y = z * (1 if w is None else w.double()) + (0 if b is None else b.double())
    if dy is None:
        return y, z, mu[..., 0], rstd[..., 0]
    gz = dy.double() * (1 if w is None else w.double())
    dx = rstd * (gz - gz.mean(-1, keepdim=True) - z * (gz * z).mean(-1, keepdim=True))
    flat = lambda t: t.reshape(-1, t.shape[-1])  # noqa: E731
    return y, z, mu[..., 0], rstd[..., 0], gz, dx, flat(dy.double() * z).sum(0), flat(dy.double()).sum(0)


# widths: one element, odd, below and above a wave's vectors, a block's, 1024 threads', and beyond registers
NORM_WIDTHS = [1, 2, 7, 8, 64, 100, 129, 256, 1000, 2049, 4096, 5001, 8200, 20000, 40000]


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("width", NORM_WIDTHS)
def test_layer_norm_forward_and_backward(width, dtype):
    dt = DTYPES[dtype]
    g = torch.Generator().manual_seed(width)
    for rows, params in ((1, "same"), (37 if width <= 8200 else 3, "fp32"), (5, "none")):
        x = rand(g, rows, width, dtype=dt, scale=1.5, shift=0.5)
        dy = rand(g, rows, width, dtype=dt)
        pt = torch.float32 if params == "fp32" else dt
        w, b = (None, None) if params == "none" else (rand(g, width, dtype=pt, scale=0.2, shift=1.0), rand(g, width, dtype=pt))
        y, z, mu, rstd, gz, dx, dw, db = norm_oracle(x, w, b, 1e-5, dy)
        dev = lambda t: None if t is None else t.to(DEV)  # noqa: E731
        gy, gmu, grs = d.layer_norm(dev(x), dev(w), dev(b), return_stats=True)
        # fp32 sums of n terms in a tree of at most 32 + 10 sequential additions, then a handful of operations: 64 half steps of what is added up.
        # rstd amplifies the error of the centred values: (|x| + |mu|) rstd half steps of z's operands.
        e = 64 * 2.0 ** -24
        ez = e * (((x.double().abs() + x.double().abs().mean(-1, keepdim=True)) * rstd[:, None]) + 1 + z.abs())
        wa = torch.ones(width, dtype=torch.float64) if w is None else w.double().abs()
        ba = torch.zeros(width, dtype=torch.float64) if b is None else b.double().abs()
        close(gmu, mu, e * x.double().abs().mean(-1), f"mean {rows}x{width}")
        # the variance's error relative to var + eps: that of the squares, and the mean's error against the deviation
        em = e * x.double().abs().mean(-1) * rstd
        close(grs, rstd, rstd * (e + em + em * em), f"rstd {rows}x{width}")
        close(gy, y, HALF[dt] * y.abs() + ez * wa + e * ba + 1e-7 * (dt == torch.float16), f"y {rows}x{width}")
        gdx, gdw, gdb = d.layer_norm_backward(dev(dy), dev(x), dev(w), gmu, grs)
        span = rstd[:, None] * (gz.abs() + gz.abs().mean(-1, keepdim=True) + z.abs() * (gz * z).abs().mean(-1, keepdim=True))
        drift = rstd[:, None] * ((ez * (gz * z).abs().mean(-1, keepdim=True)) + z.abs() * (gz.abs() * ez).mean(-1, keepdim=True))
        close(gdx, dx, HALF[dt] * dx.abs() + 2 * e * span + 2 * drift + 1e-7 * (dt == torch.float16), f"dx {rows}x{width}")
        if w is None:
            assert gdw is None and gdb is None
            continue
        assert gdw.dtype == pt
        close(gdw, dw, HALF[pt] * dw.abs() + (dy.double().abs() * (ez + e * z.abs())).sum(0) + 1e-7 * (pt == torch.float16), f"dw {rows}x{width}")
        close(gdb, db, HALF[pt] * db.abs() + e * dy.double().abs().sum(0) + 1e-7 * (pt == torch.float16), f"db {rows}x{width}")


@pytest.mark.parametrize("rows,width", [(3000, 64), (5000, 257), (2050, 1024), (70000, 8)])
def test_layer_norm_backward_sums_over_many_rows(rows, width):
    """More rows than one pass of the blocks takes: the parameters' sums, and the same bits in a second call."""
    g = torch.Generator().manual_seed(rows)
    x, dy, w = rand(g, rows, width), rand(g, rows, width), rand(g, width, shift=1.0)
    _, z, _, _, _, dx, dw, db = norm_oracle(x, w, None, 1e-5, dy)
    xd, dyd, wd = x.to(DEV), dy.to(DEV), w.to(DEV)
    _, mu, rs = d.layer_norm(xd, wd, return_stats=True)
    a = d.layer_norm_backward(dyd, xd, wd, mu, rs)
    e = 200 * 2.0 ** -24  # up to rows/1024 + 64 + 16 sequential additions
    close(a[1], dw, e * (dy.double().abs() * (z.abs() + 4)).sum(0), "dw")
    close(a[2], db, e * dy.double().abs().sum(0), "db")
    for p, q in zip(a, d.layer_norm_backward(dyd, xd, wd, mu, rs)):
        assert torch.equal(p, q)


def test_layer_norm_views_strides_and_edges():
    g = torch.Generator().manual_seed(1)
    base = rand(g, 6, 5, 48, dtype=torch.bfloat16).to(DEV)
    w = rand(g, 16, dtype=torch.bfloat16).to(DEV)
    for x in (base[..., 3:19], base[..., ::3], base.transpose(0, 1)[..., :16], base[:1, :1, :16].expand(4, 3, 16), base[0, 0, 5:21]):
        want = norm_oracle(x.cpu(), w.cpu(), None, 1e-5)[0]
        close(d.layer_norm(x, w), want, HALF[torch.bfloat16] * want.abs() + 1e-4, str(x.stride()))
        dy = torch.randn(x.shape, device=DEV).to(torch.bfloat16)
        _, mu, rs = d.layer_norm(x, w, return_stats=True)
        o = norm_oracle(x.cpu(), w.cpu(), None, 1e-5, dy.cpu())
        for got, ref in zip(d.layer_norm_backward(dy, x, w, mu, rs), o[5:]):
            close(got, ref, 2 * HALF[torch.bfloat16] * ref.abs() + 1e-3, "view gradient")
    # constant rows have no deviation: y = bias, rstd = 1/sqrt(eps)
    x = torch.full((3, 40), 7.0, device=DEV)
    y, mu, rs = d.layer_norm(x, None, torch.full((40,), 0.25, device=DEV), return_stats=True)
    assert torch.equal(y, torch.full_like(y, 0.25)) and torch.equal(mu, torch.full_like(mu, 7.0))
    close(rs, torch.full((3,), 1e5 ** 0.5, dtype=torch.float64), 1e-3, "rstd of a constant row")
    # infinities and NaN stay in their rows
    x = torch.randn(4, 100, device=DEV)
    ref = d.layer_norm(x)
    x[1, 3], x[2, 7] = float("inf"), float("nan")
    y = d.layer_norm(x)
    assert y[1:3].isnan().all() and torch.equal(y[0], ref[0]) and torch.equal(y[3], ref[3])
    # no rows
    e = torch.empty(0, 40, device=DEV)
    y, mu, rs = d.layer_norm(e, torch.ones(40, device=DEV), return_stats=True)
    dx, dw, db = d.layer_norm_backward(e, e, torch.ones(40, device=DEV), mu, rs)
    assert y.shape == (0, 40) and dx.shape == (0, 40) and not dw.any() and not db.any() and dw.shape == (40,)


# ------------------------------------------------------------------ rotary positions

def rotary_oracle(x, inv, pos, layout, scale, inverse):
    """x [B,T,H,D]; pos [axes,B,T]."""
    x = x.double()
    pairs = inv.numel()
    axis = torch.arange(pairs) // max(1, pairs // pos.shape[0])
    phi = pos.double()[axis].movedim(0, -1) * inv if pairs else pos.double()[0][..., None][..., :0]
    if inverse:
        phi = -phi
    c, s = scale * phi.cos()[:, :, None], scale * phi.sin()[:, :, None]
    out = x.clone()
    i = torch.arange(pairs)
    ia, ib = (i, i + pairs) if layout == "half" else (2 * i, 2 * i + 1)
    a, b = x[..., ia], x[..., ib]
    out[..., ia], out[..., ib] = a * c - b * s, a * s + b * c
    mag = torch.zeros_like(x)
    mag[..., ia] = mag[..., ib] = a.abs() + b.abs()
    return out, mag * scale


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("head_dim,rotary_dim", [(128, 128), (64, 48), (80, 40), (2, 2), (7, 6), (100, 34), (32, 0), (256, 64)])
def test_rotary(head_dim, rotary_dim, layout, dtype):
    dt = DTYPES[dtype]
    g = torch.Generator().manual_seed(head_dim + rotary_dim)
    for b, t, hq, hk, far, inverse, scale in ((2, 5, 3, 1, 0, False, 1.0), (1, 1, 9, 2, 10 ** 6, True, 1.3), (3, 33, 4, 4, 2 ** 40, False, 1.0)):
        q, k = rand(g, b, t, hq, head_dim, dtype=dt), rand(g, b, t, hk, head_dim, dtype=dt)
        inv, _ = d.rotary_frequencies(rotary_dim)
        pos = torch.randint(-far, far + 1, (b, t), generator=g) + torch.arange(t)
        got = d.apply_rotary(q.to(DEV), k.to(DEV), inv.to(DEV), pos.to(DEV), layout=layout, scale=scale, inverse=inverse)
        # the angle's error: position * frequency in 64 bits on both sides, then 32-bit sine and cosine (4 half steps)
        e = 6 * 2.0 ** -24 + 4 * (far + t) * 2.0 ** -52
        for x, y in zip((q, k), got):
            want, mag = rotary_oracle(x, inv, pos[None], layout, scale, inverse)
            close(y, want, HALF[dt] * want.abs() + e * mag + 1e-7 * (dt == torch.float16), f"{layout} {head_dim}/{rotary_dim} at {far}")
            assert torch.equal(y[..., rotary_dim:].cpu(), x[..., rotary_dim:])


def test_rotary_views_axes_in_place_and_gradient():
    g = torch.Generator().manual_seed(3)
    b, t, h, hk, dd = 2, 12, 4, 2, 32
    for dt in (torch.float32, torch.bfloat16):
        qkv = rand(g, b, t, (h + 2 * hk) * dd, dtype=dt).to(DEV)
        before = qkv.clone()
        q, k = qkv[..., :h * dd].unflatten(-1, (h, dd)), qkv[..., h * dd:(h + hk) * dd].unflatten(-1, (hk, dd))
        inv, _ = d.rotary_frequencies(24, axes=3)
        inv = inv.to(DEV)
        pos = torch.stack([torch.arange(t) // 4, torch.arange(t) % 4, torch.full((t,), 7)])[:, None]  # [3, 1, T]: shared by the images
        new = d.apply_rotary(q, k, inv, pos.to(DEV), layout="interleaved")
        for x, y in zip((q, k), new):
            want, mag = rotary_oracle(x.cpu(), inv.cpu(), pos.expand(3, b, t), "interleaved", 1.0, False)
            close(y, want, HALF[dt] * want.abs() + 6 * 2.0 ** -24 * mag, "three axes")
        assert torch.equal(qkv, before)
        d.apply_rotary(q, k, inv, pos.to(DEV), layout="interleaved", inplace=True)
        assert torch.equal(q, new[0]) and torch.equal(k, new[1]) and torch.equal(qkv[..., (h + hk) * dd:], before[..., (h + hk) * dd:])
        # heads-first storage, a position for every token from the default
        x = rand(g, b, h, t, dd, dtype=dt).to(DEV).transpose(1, 2)
        want, mag = rotary_oracle(x.cpu(), inv.cpu(), torch.arange(t).expand(1, b, t), "half", 1.0, False)
        close(d.apply_rotary(x, None, inv)[0], want, HALF[dt] * want.abs() + 6 * 2.0 ** -24 * mag, "heads first")
    # the gradient of sum(dy * rotary(x)) is the inverse turn of dy: against central differences of the oracle
    x, dy = rand(g, 1, 3, 2, 6), rand(g, 1, 3, 2, 6)
    inv, pos = d.rotary_frequencies(4)[0], torch.tensor([[5, 0, 9]])
    got = d.apply_rotary(dy.to(DEV), None, inv.to(DEV), pos.to(DEV), inverse=True, scale=1.2)[0].cpu().double()
    num = torch.zeros_like(got)
    for i in range(x.numel()):
        for sgn in (1, -1):
            v = x.double().clone()
            v.view(-1)[i] += sgn * 0.5
            num.view(-1)[i] += sgn * (rotary_oracle(v, inv, pos[None], "half", 1.2, False)[0] * dy.double()).sum()
    close(got, num, 1e-6, "rotary gradient")  # linear: the difference is exact to 64 bits; 32-bit results of order 1
    # nothing to do
    e = torch.empty(0, 4, 2, 8, device=DEV)
    assert d.apply_rotary(e, None, d.rotary_frequencies(8)[0].to(DEV))[0].shape == (0, 4, 2, 8)
    # one image's tokens do not see another's positions: a batch equals its images
    q = rand(g, 3, 40, 4, 64, dtype=torch.bfloat16).to(DEV)
    pos = torch.randint(0, 10 ** 5, (3, 40), generator=g).to(DEV)
    inv = d.rotary_frequencies(64)[0].to(DEV)
    whole = d.apply_rotary(q, None, inv, pos)[0]
    for i in range(3):
        assert torch.equal(whole[i:i + 1], d.apply_rotary(q[i:i + 1], None, inv, pos[i:i + 1])[0])


# ------------------------------------------------------------------ gated feed-forward block

def act_oracle(name, v):
    if name == "relu":
        return v.clamp_min(0), (v > 0).double()
    if name == "gelu":
        cdf = 0.5 * torch.erfc(-v / math.sqrt(2))
        return v * cdf, cdf + v * torch.exp(-v * v / 2) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        k = math.sqrt(2 / math.pi)
        t = torch.tanh(k * (v + 0.044715 * v ** 3))
        return 0.5 * v * (1 + t), 0.5 * (1 + t) + 0.5 * v * (1 - t * t) * k * (1 + 3 * 0.044715 * v * v)
    s = torch.sigmoid(v)
    return (s, s * (1 - s)) if name == "sigmoid" else (v * s, s * (1 + v * (1 - s)))


def ffn_case(g, m, dd, f, n, dt, bias):
    x, dy = rand(g, m, dd, dtype=dt), rand(g, m, n, dtype=dt)
    w = [rand(g, f, dd, dtype=dt, scale=dd ** -0.5), rand(g, f, dd, dtype=dt, scale=dd ** -0.5), rand(g, n, f, dtype=dt, scale=f ** -0.5)]
    b = [rand(g, f, dtype=dt, scale=0.3), rand(g, f, dtype=dt, scale=0.3), rand(g, n, dtype=dt, scale=0.3)] if bias else [None] * 3
    return x, dy, w, b


def ffn_oracle(x, dy, w, b, act):
    """Results in 64 bits, and for each the sum of the absolute values of what is added up (a bound on what rounding can do)."""
    x, dy, (wg, wu, wd) = x.double(), dy.double(), [t.double() for t in w]
    bg, bu, bd = [0.0 if t is None else t.double() for t in b]
    g, u = x @ wg.T + bg, x @ wu.T + bu
    ga, ua = x.abs() @ wg.abs().T + abs(bg), x.abs() @ wu.abs().T + abs(bu)
    a, da = act_oracle(act, g)
    h = a * u
    dh = dy @ wd
    dha = dy.abs() @ wd.abs()
    dg, du = dh * u * da, dh * a
    # what an error of one unit relative to ga, ua does to h, dg, du (|act'|, |act''| <= 1.3 for all five activations)
    ha = 1.3 * ga * u.abs() + a.abs() * ua
    dga = dha * u.abs() * da.abs() + dh.abs() * ua * da.abs() + 1.3 * dh.abs() * u.abs() * ga
    dua = dha * a.abs() + 1.3 * dh.abs() * ga
    res = {"y": h @ wd.T + bd, "dx": dg @ wg + du @ wu, "dw_gate": dg.T @ x, "dw_up": du.T @ x, "dw_down": dy.T @ h,
           "db_gate": dg.sum(0), "db_up": du.sum(0), "db_down": dy.sum(0)}
    exact = {"y": ha @ wd.abs().T + (h.abs() @ wd.abs().T) + abs(bd), "dx": (dga + dg.abs()) @ wg.abs() + (dua + du.abs()) @ wu.abs(),
             "dw_gate": (dga + dg.abs()).T @ x.abs(), "dw_up": (dua + du.abs()).T @ x.abs(), "dw_down": dy.abs().T @ (ha + h.abs()),
             "db_gate": (dga + dg.abs()).sum(0), "db_up": (dua + du.abs()).sum(0), "db_down": dy.abs().sum(0)}
    # what rounding g, u, and then h, dg, du to the type does: half steps of the values themselves
    hr = 1.3 * g.abs() * u.abs() + a.abs() * u.abs() + h.abs()
    dgr = 3 * dg.abs() + 1.3 * (dh * u * g).abs()
    dur = 2 * du.abs() + 1.3 * (dh * g).abs()
    rounded = {"y": h.abs() @ wd.abs().T, "dx": dgr @ wg.abs() + dur @ wu.abs(), "dw_gate": dgr.T @ x.abs(), "dw_up": dur.T @ x.abs(),
               "dw_down": dy.abs().T @ hr, "db_gate": dgr.sum(0), "db_up": dur.sum(0), "db_down": torch.zeros(dy.shape[1], dtype=torch.float64)}
    return res, exact, rounded


FFN_SIZES = [  # rows, width, hidden, out: one row, both sides of the change of path, widths of no whole vector, tiles' edges, long k
    (1, 64, 256, 64), (1, 7, 9, 3), (3, 40, 24, 56), (17, 100, 130, 100), (33, 64, 72, 33), (64, 128, 256, 128), (65, 128, 256, 128),
    (65, 1, 1, 1), (100, 33, 65, 17), (129, 72, 136, 264), (257, 256, 520, 256), (130, 1000, 200, 130), (1500, 64, 96, 64), (700, 520, 1032, 136)]


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("size", FFN_SIZES, ids=lambda s: "x".join(map(str, s)))
def test_gated_ffn_forward_and_backward(size, dtype):
    m, dd, f, n = size
    dt = DTYPES[dtype]
    act = ["silu", "gelu", "gelu_tanh", "relu", "sigmoid"][(m + dd) % 5]
    if act == "relu" and dt != torch.float32:
        act = "silu"  # (a rounded g may fall on the other side of the kink: its slope has no bound in the rounding)
    g = torch.Generator().manual_seed(m * 31 + f)
    x, dy, w, b = ffn_case(g, m, dd, f, n, dt, bias=(m + f) % 2 == 0)
    res, exact, rounded = ffn_oracle(x, dy, w, b, act)
    dev = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    xd, dyd, wd, bd = dev(x), dev(dy), [dev(t) for t in w], [dev(t) for t in b]
    y, saved = d.gated_ffn(xd, *wd, *bd, activation=act, save=True)
    assert torch.equal(y, d.gated_ffn(xd, *wd, *bd, activation=act))
    grads = d.gated_ffn_backward(dyd, xd, *wd, saved, activation=act, bias=True)
    # fp32 sums of K terms: at most K half steps, in practice chains of K/16 instructions; 16 per operand split and activation on top
    e = 2.0 ** -24 * (32 + max(dd, f, n, m) / 8)
    half = HALF[dt] if dt != torch.float32 else 0.0
    for name, got in zip(("y", "dx", "dw_gate", "dw_up", "dw_down", "db_gate", "db_up", "db_down"), (y, *grads)):
        tol = HALF[dt] * res[name].abs() + e * exact[name] + half * 1.01 * rounded[name] + (1e-6 if dt == torch.float16 else 0)
        close(got, res[name], tol, f"{name} {size} {dtype} {act}")
    for p, q in zip(grads, d.gated_ffn_backward(dyd, xd, *wd, saved, activation=act, bias=True)):
        assert torch.equal(p, q)
    nobias = d.gated_ffn_backward(dyd, xd, *wd, saved, activation=act)
    assert nobias[4:] == (None, None, None) and all(torch.equal(p, q) for p, q in zip(nobias[:4], grads[:4]))


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh", "relu", "sigmoid"])
def test_gated_ffn_gradients_against_differences(act):
    """Central differences of the 64-bit forward formula along random directions, every input in turn."""
    g = torch.Generator().manual_seed(11)
    x, dy, w, b = ffn_case(g, 70, 24, 40, 16, torch.float32, True)
    dev = lambda t: t.to(DEV)  # noqa: E731
    _, saved = d.gated_ffn(dev(x), *map(dev, w), *map(dev, b), activation=act, save=True)
    grads = [t.cpu().double() for t in d.gated_ffn_backward(dev(dy), dev(x), *map(dev, w), saved, activation=act, bias=True)]
    params = [t.double() for t in (x, *w, *b)]
    loss = lambda p: (ffn_oracle(p[0], dy, p[1:4], p[4:], act)[0]["y"] * dy.double()).sum()  # noqa: E731
    for i, grad in enumerate(grads):
        v = torch.randn(params[i].shape, generator=g, dtype=torch.float64)
        step = 1e-5 if act != "relu" else 1e-7
        num = (loss([p + step * v * (j == i) if j == i else p for j, p in enumerate(params)]) -
               loss([p - step * v if j == i else p for j, p in enumerate(params)])) / (2 * step)
        got = (grad * v).sum()
        scale = (grad * v).abs().sum()
        assert abs(got - num) <= 1e-5 * scale, (act, i, got.item(), num.item())


def test_gated_ffn_strides_edges_and_neighbours():
    g = torch.Generator().manual_seed(5)
    dt = torch.bfloat16
    x, dy, w, b = ffn_case(g, 96, 48, 72, 40, dt, True)
    wd, bd = [t.to(DEV) for t in w], [t.to(DEV) for t in b]
    wide = torch.full((96, 104), float("nan"), dtype=dt, device=DEV)
    for off in (0, 8, 3):  # rows inside a wider array, on and off 16-byte boundaries; what lies beside them is not read into results
        wide[:, off:off + 48] = x.to(DEV)
        view = wide[:, off:off + 48]
        y, saved = d.gated_ffn(view, *wd, *bd, save=True)
        ref, rsaved = d.gated_ffn(x.to(DEV), *wd, *bd, save=True)
        assert torch.equal(y, ref)
        pad = torch.full((96, 88), float("nan"), dtype=dt, device=DEV)
        pad[:, off:off + 40] = dy.to(DEV)
        for p, q in zip(d.gated_ffn_backward(pad[:, off:off + 40], view, *wd, saved, bias=True),
                        d.gated_ffn_backward(dy.to(DEV), x.to(DEV), *wd, rsaved, bias=True)):
            assert torch.equal(p, q)
        wide.fill_(float("nan"))
    # leading dimensions, transposed weights, the rows of a batch independent of each other where the path is the same
    y3 = d.gated_ffn(x.to(DEV).view(2, 3, 16, 48), *wd, *bd)
    assert y3.shape == (2, 3, 16, 40) and torch.equal(y3.view(96, 40), ref)
    wt = wd[2].t().contiguous().t()
    assert torch.equal(d.gated_ffn(x.to(DEV), wd[0], wd[1], wt, *bd), ref)
    # a row of NaN or infinity spoils its own row only
    for bad in (float("nan"), float("inf")):
        for rows in (5, 96):
            xb = x[:rows].to(DEV).clone()
            good = d.gated_ffn(xb, *wd, *bd)
            xb[2, 5] = bad
            y = d.gated_ffn(xb, *wd, *bd)
            keep = torch.arange(rows, device=DEV) != 2
            assert torch.equal(y[keep], good[keep]) and not y[2].isfinite().any()
    # no rows
    e = torch.empty(0, 48, dtype=dt, device=DEV)
    y, saved = d.gated_ffn(e, *wd, *bd, save=True)
    out = d.gated_ffn_backward(torch.empty(0, 40, dtype=dt, device=DEV), e, *wd, saved, bias=True)
    assert y.shape == (0, 40) and out[0].shape == (0, 48) and not any(t.any() for t in out[1:])


def test_fp32_products_keep_fp32_range():
    """Values near the ends of the fp32 range survive the split into three terms: no overflow of a leading term, no loss of small ones."""
    m, dd = 70, 16
    x = torch.zeros(m, dd)
    x[:, 0], x[:, 1] = 3.4e38, 1.5e-30
    wg, wu = torch.zeros(8, dd), torch.zeros(8, dd)
    wg[0, 0] = 1.0              # g = 3.4e38
    wu[0, 1] = 1.0              # u = 1.5e-30
    wd = torch.zeros(4, 8)
    wd[1, 0] = 1.0
    y = d.gated_ffn(x.to(DEV), wg.to(DEV), wu.to(DEV), wd.to(DEV), activation="relu").cpu().double()
    want = x[0, 0].double() * x[0, 1].double()
    assert abs(y[:, 1] - want).max() <= 4 * 2.0 ** -24 * want and not y[:, [0, 2, 3]].any()


# ------------------------------------------------------------------ together, streams, graphs

def block_params(g, c, hidden):
    p = {"n1": rand(g, c, shift=1.0, scale=0.1), "n1b": rand(g, c, scale=0.1), "qkv": rand(g, 3 * c, c, scale=c ** -0.5),
         "proj": rand(g, c, c, scale=c ** -0.5), "n2": rand(g, c, shift=1.0, scale=0.1), "n2b": rand(g, c, scale=0.1),
         "wg": rand(g, hidden, c, scale=c ** -0.5), "wu": rand(g, hidden, c, scale=c ** -0.5), "wd": rand(g, c, hidden, scale=hidden ** -0.5)}
    return p


def attention(qkv, b, t, c):
    o = torch.empty(b, t, c, device=DEV)
    _lib.check(_lib.lib().dm_attention(_lib.ptr(qkv), _lib.ptr(o), b, t, c, torch.cuda.current_stream().cuda_stream))
    return o


def test_transformer_block_over_image_tokens():
    """norm -> projections -> rotary over rows and columns (in place, in the packed qkv) -> dm_attention -> norm -> gated block, as a user
    strings them together, against the block in 64 bits."""
    b, side, c, hidden = 3, 8, 64, 160
    t = side * side
    g = torch.Generator().manual_seed(21)
    x, p = rand(g, b, t, c), block_params(g, c, hidden)
    inv, _ = d.rotary_frequencies(c, axes=2)
    pos = torch.stack([torch.arange(t) // side, torch.arange(t) % side])[:, None]

    def dev(name):
        return p[name].to(DEV)
    xd = x.to(DEV)
    qkv = (d.layer_norm(xd, dev("n1"), dev("n1b")) @ dev("qkv").T).contiguous()
    d.apply_rotary(qkv[..., :c].unflatten(-1, (1, c)), qkv[..., c:2 * c].unflatten(-1, (1, c)), inv.to(DEV), pos.to(DEV), inplace=True)
    x1 = xd + attention(qkv, b, t, c) @ dev("proj").T
    y = x1 + d.gated_ffn(d.layer_norm(x1, dev("n2"), dev("n2b")), dev("wg"), dev("wu"), dev("wd"))

    P = {k: v.double() for k, v in p.items()}
    n1 = norm_oracle(x, p["n1"], p["n1b"], 1e-5)[0]
    q, k, v = (n1 @ P["qkv"].T).split(c, -1)
    full = pos.expand(2, b, t)
    q, k = (rotary_oracle(s[:, :, None], inv, full, "half", 1.0, False)[0][:, :, 0] for s in (q, k))
    o = torch.softmax(q @ k.transpose(1, 2) / c ** 0.5, -1) @ v
    r1 = x.double() + o @ P["proj"].T
    n2 = norm_oracle(r1, p["n2"], p["n2b"], 1e-5)[0]
    gate, up = n2 @ P["wg"].T, n2 @ P["wu"].T
    want = r1 + (act_oracle("silu", gate)[0] * up) @ P["wd"].T
    close(y, want, 2e-5 * want.abs().max(), "block")  # fp32 throughout: some 300 half steps of the largest value


def test_training_step_of_a_norm_and_ffn_sublayer():
    """y = x + ffn(norm(x)): the backward calls strung together give the gradients of autograd on the same formula in 64 bits."""
    g = torch.Generator().manual_seed(8)
    m, c, hidden = 150, 48, 100
    x, dy, p = rand(g, m, c), rand(g, m, c), block_params(g, c, hidden)
    dev = lambda n: p[n].to(DEV)  # noqa: E731
    xd, dyd = x.to(DEV), dy.to(DEV)
    n, mu, rs = d.layer_norm(xd, dev("n2"), dev("n2b"), return_stats=True)
    f, saved = d.gated_ffn(n, dev("wg"), dev("wu"), dev("wd"), save=True)
    dn, dwg, dwu, dwd, *_ = d.gated_ffn_backward(dyd, n, dev("wg"), dev("wu"), dev("wd"), saved)
    dx, dw, db = d.layer_norm_backward(dn, xd, dev("n2"), mu, rs)
    leaves = [t.double().requires_grad_() for t in (x, p["n2"], p["n2b"], p["wg"], p["wu"], p["wd"])]
    xr, w, b, wg, wu, wd = leaves
    z = (xr - xr.mean(-1, keepdim=True)) * (xr.var(-1, unbiased=False, keepdim=True) + 1e-5).rsqrt() * w + b
    gate = z @ wg.T
    (((gate * torch.sigmoid(gate) * (z @ wu.T)) @ wd.T + xr) * dy.double()).sum().backward()
    for got, leaf, name in zip((dx + dyd, dw, db, dwg, dwu, dwd), leaves, ("dx", "dw", "db", "wg", "wu", "wd")):
        close(got, leaf.grad, 1e-5 * leaf.grad.abs().max(), name)


def _calls(g, rows):
    """One call of each operator as closures over its inputs: (inputs, function of the inputs)."""
    c, f = 64, 136
    x, dy = rand(g, rows, c, dtype=torch.bfloat16).to(DEV), rand(g, rows, c, dtype=torch.bfloat16).to(DEV)
    w = rand(g, c, dtype=torch.bfloat16).to(DEV)
    ws = [rand(g, f, c, dtype=torch.bfloat16, scale=0.1).to(DEV), rand(g, f, c, dtype=torch.bfloat16, scale=0.1).to(DEV),
          rand(g, c, f, dtype=torch.bfloat16, scale=0.1).to(DEV)]
    inv = d.rotary_frequencies(16)[0].to(DEV)
    pos = torch.arange(rows, device=DEV)

    def run():
        y, mu, rs = d.layer_norm(x, w, return_stats=True)
        q = d.apply_rotary(y.view(1, rows, 4, 16), None, inv, pos)[0]
        z, saved = d.gated_ffn(q.view(rows, c), *ws, save=True)
        return (y, q, z) + d.layer_norm_backward(dy, x, w, mu, rs)[:2] + d.gated_ffn_backward(dy, q.view(rows, c), *ws, saved)[:4]
    return (x, dy, w), run


@pytest.mark.parametrize("rows", [3, 200])
def test_operators_under_graph_capture(rows):
    """Two captured graphs, replayed in turn on new inputs with eager calls in between, against the eager results."""
    g = torch.Generator().manual_seed(rows)
    made = [_calls(g, rows) for _ in range(2)]
    side = torch.cuda.Stream()
    graphs = []
    for inputs, run in made:
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run()
        graphs.append((graph, out))
    for turn in range(3):
        for (inputs, run), (graph, out) in zip(made, graphs):
            for t in inputs:
                t.copy_(torch.randn(t.shape, generator=g).to(t.dtype))
            want = run()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(out, want):
                assert torch.equal(a, b), turn


def test_operators_on_two_streams_at_once():
    """Calls that overlap on two streams (workspaces of their own) give the bits of calls one after the other."""
    g = torch.Generator().manual_seed(77)
    made = [_calls(g, 300), _calls(g, 1000)]
    want = [run() for _, run in made]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        got = []
        for (_, run), s in zip(made, streams):
            with torch.cuda.stream(s):
                got.append(run())
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(p, q) for p, q in zip(a, b))


# ------------------------------------------------------------------ rows and sizes where a kernel's last piece, tile or step is not whole

def _norm_bounds(x, w, b, dy, dt):
    """(name, value, bound) of y, dx, dw, db; the bounds are those of test_layer_norm_forward_and_backward."""
    y, z, _, rstd, gz, dx, dw, db = norm_oracle(x, w, b, 1e-5, dy)
    e = 64 * 2.0 ** -24
    xa = x.double().abs()
    ez = e * ((xa + xa.mean(-1, keepdim=True)) * rstd[:, None] + 1 + z.abs())
    span = rstd[:, None] * (gz.abs() + gz.abs().mean(-1, keepdim=True) + z.abs() * (gz * z).abs().mean(-1, keepdim=True))
    drift = rstd[:, None] * (ez * (gz * z).abs().mean(-1, keepdim=True) + z.abs() * (gz.abs() * ez).mean(-1, keepdim=True))
    ga = dy.double().abs()
    tiny = 1e-7 * (dt == torch.float16)
    return (("y", y, HALF[dt] * y.abs() + ez * w.double().abs() + e * b.double().abs() + tiny),
            ("dx", dx, HALF[dt] * dx.abs() + 2 * e * span + 2 * drift + tiny),
            ("dw", dw, HALF[w.dtype] * dw.abs() + (ga * (ez + e * z.abs())).sum(0) + tiny), ("db", db, HALF[w.dtype] * db.abs() + e * ga.sum(0) + tiny))


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("width", [3, 4, 9, 15, 33, 127, 511, 1001, 1032, 4097, 5000, 12289, 16385, 32769])
def test_layer_norm_rows_between_others(width, dtype):
    """Rows of any width at any element of a wider array whose other elements are NaN, parameters off 16-byte boundaries: nothing beside a
    row is read into its results, and a row behind the last one is not written."""
    dt = DTYPES[dtype]
    g = torch.Generator().manual_seed(width + 1)
    rows = 41 if width < 6000 else 6
    x, dy = rand(g, rows, width, dtype=dt, scale=1.5, shift=0.5), rand(g, rows, width, dtype=dt)
    w, b = rand(g, width, dtype=dt, scale=0.2, shift=1.0), rand(g, width, dtype=dt)
    nan = float("nan")
    flat = torch.full((rows + 1, width + 5), nan, dtype=dt, device=DEV)
    gflat = torch.full((rows, width + 3), nan, dtype=dt, device=DEV)
    wb = torch.full((2, width + 1), nan, dtype=dt, device=DEV)
    xd, dyd, wd, bd = flat[:rows, 1:1 + width], gflat[:, 3:], wb[0, 1:], wb[1, :width]
    for view, t in ((xd, x), (dyd, dy), (wd, w), (bd, b)):
        view.copy_(t)
    y, mu, rs = d.layer_norm(xd, wd, bd, return_stats=True)
    got = (y, *d.layer_norm_backward(dyd, xd, wd, mu, rs))
    for (name, want, tol), t in zip(_norm_bounds(x, w, b, dy, dt), got):
        close(t, want, tol, f"{name} {rows}x{width}")
    # the library's own entry point, into the middle of an array: what lies around the rows stays
    out = torch.full((rows + 2, width), 7.0, dtype=dt, device=DEV)
    code = {"fp32": 0, "bf16": 1, "fp16": 2}[dtype]
    _lib.check(_lib.lib().dm_layer_norm(xd.data_ptr(), xd.stride(0), wd.data_ptr(), bd.data_ptr(), code, out[1].data_ptr(), None, None, rows, width,
                                        1e-5, code, torch.cuda.current_stream().cuda_stream))
    assert torch.equal(out[1:-1], y) and (out[0] == 7).all() and (out[-1] == 7).all()


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("size", [(5000, 72, 88, 40), (300, 1100, 1544, 1100), (9, 600, 1200, 600), (520, 136, 2056, 24), (2100, 24, 16, 8), (70, 4100, 24, 520)],
                         ids=lambda s: "x".join(map(str, s)))
def test_gated_ffn_long_and_ragged_ranges(size, dtype):
    """Long sums of no whole steps, whole or dealt among several workgroups, with every bias' gradient; bounds as in
    test_gated_ffn_forward_and_backward."""
    m, dd, f, n = size
    dt = DTYPES[dtype]
    g = torch.Generator().manual_seed(m + n)
    x, dy, w, b = ffn_case(g, m, dd, f, n, dt, True)
    res, exact, rounded = ffn_oracle(x, dy, w, b, "silu")
    xd, dyd, wd, bd = x.to(DEV), dy.to(DEV), [t.to(DEV) for t in w], [t.to(DEV) for t in b]
    y, saved = d.gated_ffn(xd, *wd, *bd, save=True)
    got = (y, *d.gated_ffn_backward(dyd, xd, *wd, saved, bias=True))
    e = 2.0 ** -24 * (32 + max(dd, f, n, m) / 8)
    for name, t in zip(("y", "dx", "dw_gate", "dw_up", "dw_down", "db_gate", "db_up", "db_down"), got):
        close(t, res[name], HALF[dt] * res[name].abs() + e * exact[name] + (HALF[dt] * 1.01 * rounded[name] if dt != torch.float32 else 0), f"{name} {size}")


def test_rotary_of_one_tensor_as_query_and_key():
    g = torch.Generator().manual_seed(4)
    x = rand(g, 1, 5, 3, 16).to(DEV)
    inv = d.rotary_frequencies(16)[0].to(DEV)
    q, k = d.apply_rotary(x, x, inv)
    assert torch.equal(q, k) and torch.equal(q, d.apply_rotary(x, None, inv)[0])
    with pytest.raises(RuntimeError, match="share no elements"):
        d.apply_rotary(x, x, inv, inplace=True)


def test_ffn_of_one_weight_for_both_projections():
    """The same tensor twice among the inputs, and the gradient's tensor as the input itself."""
    g = torch.Generator().manual_seed(6)
    for rows in (3, 80):
        x, w, wd = rand(g, rows, 32).to(DEV), rand(g, 48, 32, scale=0.2).to(DEV), rand(g, 32, 48, scale=0.2).to(DEV)
        y, saved = d.gated_ffn(x, w, w, wd, save=True)
        assert torch.equal(y, d.gated_ffn(x, w, w.clone(), wd))
        a, b = d.gated_ffn_backward(x, x, w, w, wd, saved), d.gated_ffn_backward(x.clone(), x, w, w.clone(), wd, saved)
        assert all(torch.equal(p, q) for p, q in zip(a[:4], b[:4]))


@pytest.mark.parametrize("size", [(6, 5, 7, 3), (20, 3, 40, 5), (20, 40, 3, 5), (37, 515, 130, 129), (64, 63, 33, 1), (2, 2, 2, 2), (4, 517, 1031, 9)],
                         ids=lambda s: "x".join(map(str, s)))
def test_gated_ffn_few_fp32_rows_of_odd_widths(size):
    """Rows whose last piece is moved back, and rows of less than a piece; inputs between NaN.  Bounds as in
    test_gated_ffn_forward_and_backward."""
    m, dd, f, n = size
    g = torch.Generator().manual_seed(m * dd)
    x, dy, w, b = ffn_case(g, m, dd, f, n, torch.float32, True)
    res, exact, _ = ffn_oracle(x, dy, w, b, "gelu")
    wide = torch.full((m, dd + 3), float("nan"), device=DEV)
    wide[:, 2:2 + dd] = x.to(DEV)
    xd, dyd, wd, bd = wide[:, 2:2 + dd], dy.to(DEV), [t.to(DEV) for t in w], [t.to(DEV) for t in b]
    y, saved = d.gated_ffn(xd, *wd, *bd, activation="gelu", save=True)
    got = (y, *d.gated_ffn_backward(dyd, xd, *wd, saved, activation="gelu", bias=True))
    e = 2.0 ** -24 * (32 + max(size) / 8)
    for name, t in zip(("y", "dx", "dw_gate", "dw_up", "dw_down", "db_gate", "db_up", "db_down"), got):
        close(t, res[name], 2.0 ** -24 * res[name].abs() + e * exact[name], f"{name} {size}")


@pytest.mark.parametrize("size", [(90, 40, 56, 24), (90, 33, 57, 21), (1500, 64, 300, 64)], ids=lambda s: "x".join(map(str, s)))
def test_gated_ffn_backward_of_some_gradients(size):
    """The library's entry point asked for one projection's gradient, or one bias of two: what both together give, to fp32 rounding; what
    was not asked for is not written."""
    m, dd, f, n = size
    g = torch.Generator().manual_seed(m + dd)
    x, dy, w, b = ffn_case(g, m, dd, f, n, torch.float32, True)
    xd, dyd, wd, bd = x.to(DEV), dy.to(DEV), [t.to(DEV) for t in w], [t.to(DEV) for t in b]
    _, saved = d.gated_ffn(xd, *wd, *bd, save=True)
    full = dict(zip(("dx", "dwg", "dwu", "dwd", "dbg", "dbu", "dbd"), d.gated_ffn_backward(dyd, xd, *wd, saved, bias=True)))
    exact = ffn_oracle(x, dy, w, b, "silu")[1]
    bound = {"dx": "dx", "dwg": "dw_gate", "dwu": "dw_up", "dwd": "dw_down", "dbg": "db_gate", "dbu": "db_up", "dbd": "db_down"}
    L = _lib.lib()
    nbytes = L.dm_gated_ffn_backward_workspace_bytes(m, dd, f, n, 0)
    e = 2 * 2.0 ** -24 * (32 + max(size) / 8)  # both sides within the bound of test_gated_ffn_forward_and_backward
    for asked in (("dwg",), ("dwu", "dbu"), ("dwg", "dwu", "dbu"), ("dwg", "dwu", "dbg"), ("dx", "dwd"), ("dwd", "dbd"), ("dwg", "dbg", "dwd")):
        out = {k: torch.full_like(t, 3.0) for k, t in full.items()}
        ws = torch.empty(nbytes, dtype=torch.uint8, device=DEV)
        p = {k: t.data_ptr() if k in asked else None for k, t in out.items()}
        _lib.check(L.dm_gated_ffn_backward(dyd.data_ptr(), n, xd.data_ptr(), dd, wd[0].data_ptr(), wd[1].data_ptr(), wd[2].data_ptr(), saved.data_ptr(),
                                           p["dx"], p["dwg"], p["dwu"], p["dwd"], p["dbg"], p["dbu"], p["dbd"], m, dd, f, n, 0, 0, ws.data_ptr(), nbytes,
                                           torch.cuda.current_stream().cuda_stream))
        for k, t in out.items():
            if k in asked:
                close(t, full[k].cpu().double(), 2.0 ** -23 * full[k].cpu().double().abs() + e * exact[bound[k]], f"{k} of {asked}")
            else:
                assert (t == 3).all(), (k, asked)


def test_operators_on_nothing():
    """Batches, tokens and heads of no elements, one vector without a leading dimension, gradients and weights as views."""
    inv = d.rotary_frequencies(8)[0].to(DEV)
    for shape in ((2, 0, 3, 8), (0, 5, 3, 8), (2, 3, 0, 8)):
        x = torch.empty(shape, device=DEV)
        for inplace in (False, True):
            q, k = d.apply_rotary(x, x.clone(), inv, torch.zeros(shape[:2], dtype=torch.int32, device=DEV), inplace=inplace)
            assert q.shape == k.shape == shape
    g = torch.Generator().manual_seed(9)
    w, wd = rand(g, 4, 8).to(DEV), rand(g, 8, 4).to(DEV)
    for shape in ((3, 0, 8), (8,)):
        x = rand(g, *shape).to(DEV)
        n, mu, rs = d.layer_norm(x, return_stats=True)
        y, saved = d.gated_ffn(x, w, w, wd, save=True)
        assert n.shape == y.shape == shape and mu.shape == shape[:-1]
        assert d.layer_norm_backward(y, x, None, mu, rs)[0].shape == shape and d.gated_ffn_backward(y, x, w, w, wd, saved)[0].shape == shape
    x = rand(g, 70, 16, dtype=torch.bfloat16).to(DEV)
    ws = [rand(g, 16, 24).to(DEV, torch.bfloat16).t(), rand(g, 24, 32).to(DEV, torch.bfloat16)[:, ::2], rand(g, 16, 24).to(DEV, torch.bfloat16)]
    dy = torch.ones(1, 1, device=DEV, dtype=torch.bfloat16).expand(70, 16)
    saved = d.gated_ffn(x, *ws, save=True)[1]
    a, b = d.gated_ffn_backward(dy, x, *ws, saved), d.gated_ffn_backward(dy.contiguous(), x, *[t.contiguous() for t in ws], saved)
    assert all(torch.equal(p, q) for p, q in zip(a[:4], b[:4]))
