"""Transformer-block operators (GPU): every tile and split of the gated block's products, layer norms of many rows, rotary calls whose
threads walk several heads; against the formulas in 64 bits (oracles and bounds of test_gpu_transformer.py)."""
import pytest
import torch

import diffusion_model_amd as d
from diffusion_model_amd import _lib
from test_gpu_transformer import DEV, DTYPES, HALF, _norm_bounds, close, ffn_case, ffn_oracle, norm_oracle, rand, rotary_oracle

pytestmark = pytest.mark.gpu
NAMES = ("y", "dx", "dw_gate", "dw_up", "dw_down", "db_gate", "db_up", "db_down")
TILES = {"256x256": 0, "128x128": 1, "64x128": 2}
COLUMNS = 3


class plan:
    """The tiled products of the block with one tile and k ranges of `splits` parts."""

    def __init__(self, tile, splits):
        self.args = TILES.get(tile, tile), splits

    def __enter__(self):
        _lib.check(_lib.lib().dm_debug_ffn_plan(*self.args))

    def __exit__(self, *_):
        _lib.check(_lib.lib().dm_debug_ffn_plan(-1, 1))


def step(x, dy, w, b, act):
    y, saved = d.gated_ffn(x, *w, *b, activation=act, save=True)
    return (y, *d.gated_ffn_backward(dy, x, *w, saved, activation=act, bias=True))


def ffn_bounds(x, dy, w, b, act, dt):
    """(name, value, bound).  fp32 sums of K terms: at most K/8 + 32 half steps of the absolute sums.  16-bit types round h, u act'(g),
    act(g), dg and du, each by half a step, before they are multiplied: two roundings of dg and du, one of h."""
    res, exact, _ = ffn_oracle(x, dy, w, b, act)
    m, dd = x.shape
    f, n = w[0].shape[0], w[2].shape[0]
    e = 2.0 ** -24 * (32 + max(dd, f, n, m) / 8)
    X, DY, (wg, wu, wd) = x.double(), dy.double(), [t.double() for t in w]
    bg, bu, _ = [0.0 if t is None else t.double() for t in b]
    g, u = X @ wg.T + bg, X @ wu.T + bu
    a, da = {"relu": lambda v: (v.clamp_min(0), (v > 0).double()), "silu": lambda v: (v * torch.sigmoid(v), torch.sigmoid(v) * (1 + v * torch.sigmoid(-v)))}[act](g)
    dh = DY @ wd
    h, dg, du = a * u, dh * u * da, dh * a
    half = HALF[dt] if dt != torch.float32 else 0.0
    hr, dgr, dur = half * h.abs(), 2 * half * dg.abs(), 2 * half * du.abs()
    if act == "relu":  # at the kink an error of g decides between the two slopes
        near = g.abs() <= e * (X.abs() @ wg.abs().T + abs(bg))
        dgr = dgr + near * (dh * u).abs()
    rounded = {"y": hr @ wd.abs().T, "dx": dgr @ wg.abs() + dur @ wu.abs(), "dw_gate": dgr.T @ X.abs(), "dw_up": dur.T @ X.abs(),
               "dw_down": DY.abs().T @ hr, "db_gate": dgr.sum(0), "db_up": dur.sum(0), "db_down": torch.zeros(n, dtype=torch.float64)}
    tiny = 1e-6 if dt == torch.float16 else 0.0  # of fp16 values below its normal range, half a step of 2^-24 each
    return [(k, res[k], HALF[dt] * res[k].abs() + e * exact[k] + 1.01 * rounded[k] + tiny) for k in NAMES]


# rows, width, hidden, out: several tiles of every size with a rest, in whole 16-byte pieces and off them; long sums over the rows, the
# width and the hidden values
SIZES = [(700, 264, 312, 280), (613, 259, 301, 277), (2100, 136, 152, 136), (300, 1304, 328, 520)]


@pytest.mark.parametrize("splits", [1, 2, 5])
@pytest.mark.parametrize("tile", list(TILES))
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_every_tile_and_split(size, dtype, tile, splits):
    m, dd, f, n = size
    dt = DTYPES[dtype]
    act = "relu" if (m + splits) % 2 else "silu"
    g = torch.Generator().manual_seed(m + f)
    x, dy, w, b = ffn_case(g, m, dd, f, n, dt, True)
    args = x.to(DEV), dy.to(DEV), [t.to(DEV) for t in w], [t.to(DEV) for t in b]
    with plan(tile, splits):
        got = step(*args, act)
        again = step(*args, act)
    for (name, want, tol), t, t2 in zip(ffn_bounds(x, dy, w, b, act, dt), got, again):
        close(t, want, tol, f"{name} {size} {dtype} {act} {tile} in {splits}")
        assert torch.equal(t, t2), name


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("rows", [2, 40, 150])
def test_relu_of_16_bit_rows(rows, dtype):
    dt = DTYPES[dtype]
    g = torch.Generator().manual_seed(rows)
    x, dy, w, b = ffn_case(g, rows, 72, 120, 56, dt, True)
    got = step(x.to(DEV), dy.to(DEV), [t.to(DEV) for t in w], [t.to(DEV) for t in b], "relu")
    for (name, want, tol), t in zip(ffn_bounds(x, dy, w, b, "relu", dt), got):
        close(t, want, tol, f"{name} {rows} {dtype}")


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_strided_rows_of_every_path(dtype):
    """Rows inside wider arrays give the bits of contiguous ones: few rows and many, x and the output's gradient."""
    dt = DTYPES[dtype]
    for rows in (2, 20, 64, 300):
        g = torch.Generator().manual_seed(rows)
        x, dy, w, b = ffn_case(g, rows, 48, 72, 40, dt, True)
        w, b = [t.to(DEV) for t in w], [t.to(DEV) for t in b]
        want = step(x.to(DEV), dy.to(DEV), w, b, "silu")
        for off in (0, 3, 8):
            wide = torch.full((rows, 64), float("nan"), dtype=dt, device=DEV)
            pad = torch.full((rows, 56), float("nan"), dtype=dt, device=DEV)
            wide[:, off:off + 48], pad[:, off:off + 40] = x.to(DEV), dy.to(DEV)
            for name, p, q in zip(NAMES, want, step(wide[:, off:off + 48], pad[:, off:off + 40], w, b, "silu")):
                assert torch.equal(p, q), (rows, off, name)


# ------------------------------------------------------------------ layer norm, many rows

# shapes of the kernels in every type: 16, 64, 256, 512 and 1024 threads a row, one to eight pieces each, whole pieces and not
MANY = [(5003, 100), (4101, 250), (3001, 300), (3007, 520), (5000, 1000), (1100, 1030), (2101, 1504), (1029, 2050), (1301, 4095), (1025, 4096),
        (1100, 6001), (1061, 12289)]


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("rows,width", MANY, ids=lambda v: str(v))
def test_layer_norm_of_many_rows(rows, width, dtype):
    """Every block walks several rows in the backward pass, and the forward pass takes its kernels for many rows.  Bounds as in
    test_layer_norm_forward_and_backward; a column's sum has at most rows / 256 + 4 + 16 + 16 additions on end."""
    dt = DTYPES[dtype]
    g = torch.Generator().manual_seed(rows + width)
    x, dy = rand(g, rows, width, dtype=dt, scale=1.5, shift=0.5), rand(g, rows, width, dtype=dt)
    w, b = rand(g, width, dtype=dt, scale=0.2, shift=1.0), rand(g, width, dtype=dt)
    xd, dyd, wd = x.to(DEV), dy.to(DEV), w.to(DEV)
    y, mu, rs = d.layer_norm(xd, wd, b.to(DEV), return_stats=True)
    got = (y, *d.layer_norm_backward(dyd, xd, wd, mu, rs))
    for (name, want, tol), t in zip(_norm_bounds(x, w, b, dy, dt), got):
        close(t, want, tol, f"{name} {rows}x{width}")
    _, _, mean, rstd = norm_oracle(x, w, b, 1e-5)
    xa = x.double().abs().mean(-1)
    e = 64 * 2.0 ** -24
    em = e * xa * rstd
    close(mu, mean, e * xa, "mean")
    close(rs, rstd, rstd * (e + em + em * em), "rstd")


# ------------------------------------------------------------------ rotary: several heads per thread

# (tokens, heads, kv_heads, head_dim, rotary_dim): a thread walks 2, 4 or 8 heads; head counts that no group divides, groups that hold
# the last query heads and the first key heads; one element at a time (33 and 9 pairs) and whole vectors
WALKS = [(1400, 9, 2, 66, 66), (2700, 9, 2, 66, 66), (4100, 9, 2, 66, 66), (8000, 5, 1, 66, 66), (4000, 5, 1, 66, 66), (8200, 9, 2, 64, 64),
         (16500, 9, 2, 64, 48), (3300, 13, 6, 40, 18)]


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("walk", WALKS, ids=lambda s: "x".join(map(str, s)))
def test_rotary_of_several_heads_per_thread(walk, layout, dtype):
    t, h, hk, dd, rd = walk
    dt = DTYPES[dtype]
    g = torch.Generator().manual_seed(t + h)
    qkv = rand(g, 1, t, (h + 2 * hk) * dd, dtype=dt)
    inv, _ = d.rotary_frequencies(rd)
    pos = torch.randint(0, 10 ** 6, (1, t), generator=g)
    qd = qkv.to(DEV)
    views = lambda a: (a[..., :h * dd].unflatten(-1, (h, dd)), a[..., h * dd:(h + hk) * dd].unflatten(-1, (hk, dd)))  # noqa: E731
    got = d.apply_rotary(*views(qd), inv.to(DEV), pos.to(DEV), layout=layout, scale=1.1)
    e = 6 * 2.0 ** -24 + 4 * 10 ** 6 * 2.0 ** -52  # as in test_rotary
    for x, y in zip(views(qkv), got):
        want, mag = rotary_oracle(x, inv, pos[None], layout, 1.1, False)
        close(y, want, HALF[dt] * want.abs() + e * mag, f"{walk}")
        assert torch.equal(y[..., rd:].cpu(), x[..., rd:])
    d.apply_rotary(*views(qd), inv.to(DEV), pos.to(DEV), layout=layout, scale=1.1, inplace=True)
    for x, y in zip(views(qd), got):
        assert torch.equal(x, y)
    assert torch.equal(qd[..., (h + hk) * dd:].cpu(), qkv[..., (h + hk) * dd:])


@pytest.mark.parametrize("size", [(40000, 256, 320, 256), (3000, 700, 1500, 700)], ids=lambda s: "x".join(map(str, s)))
def test_fp32_steps_are_as_exact_as_fp32_products(size):
    """Every result's error against 64 bits, over its elements, beside that of the same formula in fp32 products and sums: twice it at most.
    (Errors of one sign in dh would add up in the bias' gradients over the rows.)"""
    m, dd, f, n = size
    g = torch.Generator(device=DEV).manual_seed(5)
    mk = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    x, dy, w = mk(m, dd), mk(m, n), [mk(f, dd) * dd ** -0.5, mk(f, dd) * dd ** -0.5, mk(n, f) * f ** -0.5]
    b = [0.1 * mk(f), 0.1 * mk(f), 0.1 * mk(n)]
    got = step(x, dy, w, b, "silu")

    def formula(t):
        X, DY, wg, wu, wd, bg, bu, bd = [v.to(t) for v in (x, dy, *w, *b)]
        gate, up = X @ wg.T + bg, X @ wu.T + bu
        s = torch.sigmoid(gate)
        h, dh = gate * s * up, DY @ wd
        dg, du = dh * up * s * (1 + gate * torch.sigmoid(-gate)), dh * gate * s
        return h @ wd.T + bd, dg @ wg + du @ wu, dg.T @ X, du.T @ X, DY.T @ h, dg.sum(0), du.sum(0), DY.sum(0)
    for name, t, plain, want in zip(NAMES, got, formula(torch.float32), formula(torch.float64)):
        err, ref = ((v.double() - want).norm() / want.norm() for v in (t, plain))
        print(size, name, "%.2e %.2e" % (err, ref))
        assert err <= 2 * ref, (name, err, ref)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_one_row_has_any_stride(dtype):
    """The library's entry points with one row: the distance to a next row, which is not there, does not matter."""
    dt, code = DTYPES[dtype], {"fp32": 0, "bf16": 1}[dtype]
    g = torch.Generator().manual_seed(2)
    x, dy, w, _ = ffn_case(g, 1, 64, 136, 72, dt, False)
    xd, dyd, wd = x.to(DEV), dy.to(DEV), [t.to(DEV) for t in w]
    y, saved = d.gated_ffn(xd, *wd, save="compact")  # (what the entry points take without DM_FFN_KEEP_F32)
    want = d.gated_ffn_backward(dyd, xd, *wd, saved, bias=True)
    L = _lib.lib()
    nbytes = L.dm_gated_ffn_backward_workspace_bytes(1, 64, 136, 72, code)
    fbytes = L.dm_gated_ffn_workspace_bytes(1, 64, 136, 72, code, 0)
    stream = torch.cuda.current_stream().cuda_stream
    for stride in (0, 8, 1, 1 << 22):
        got = [torch.full_like(t, 3.0) for t in want]
        ws = torch.empty(nbytes + fbytes, dtype=torch.uint8, device=DEV)
        _lib.check(L.dm_gated_ffn_backward(dyd.data_ptr(), stride, xd.data_ptr(), stride, *(t.data_ptr() for t in wd), saved.data_ptr(),
                                           *(t.data_ptr() for t in got), 1, 64, 136, 72, 0, code, ws.data_ptr(), nbytes, stream))
        for name, p, q in zip(NAMES[1:], got, want):
            assert torch.equal(p, q), (stride, name)
        out = torch.full_like(y, 3.0)
        _lib.check(L.dm_gated_ffn(xd.data_ptr(), stride, *(t.data_ptr() for t in wd), None, None, None, out.data_ptr(), None, 1, 64, 136, 72, 0, code,
                                  ws.data_ptr(), fbytes, stream))
        assert torch.equal(out, y), stride


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("splits", [1, 3])
@pytest.mark.parametrize("rows", [3, 70])
def test_infinities_of_odd_widths_stay_infinities(rows, splits, dtype):
    """16-bit rows whose hidden width is no whole number of pieces: an infinite element among positive numbers gives infinities, not NaN."""
    dt = DTYPES[dtype]
    g = torch.Generator().manual_seed(1)
    pos = lambda *s: (torch.rand(*s, generator=g) * 0.1 + 0.1).to(dt).to(DEV)  # noqa: E731
    dd, f, n = 400, 205, 403
    x, dy, w = pos(rows, dd), pos(rows, n), [pos(f, dd), pos(f, dd), pos(n, f)]
    w[2] = w[2] * 0.1
    clean = d.gated_ffn(x, *w, activation="relu")
    xi, dyi = x.clone(), dy.clone()
    xi[1, 5], dyi[2, 7] = float("inf"), float("inf")
    keep = torch.arange(rows, device=DEV)
    with plan("128x128", splits):
        y = d.gated_ffn(xi, *w, activation="relu")
        assert (y[1] == float("inf")).all() and torch.equal(y[keep != 1], d.gated_ffn(x, *w, activation="relu")[keep != 1]) and clean.isfinite().all()
        _, saved = d.gated_ffn(x, *w, activation="relu", save=True)
        dx, dwg, dwu, dwd = d.gated_ffn_backward(dyi, x, *w, saved, activation="relu")[:4]
    assert (dx[2] == float("inf")).all() and dx[keep != 2].isfinite().all()
    assert (dwg == float("inf")).all() and (dwu == float("inf")).all()
    assert (dwd[7] == float("inf")).all() and dwd[:7].isfinite().all()


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("rows", [3, 30, 150])
def test_sigmoid_slope_of_large_gates(rows, dtype):
    """s (1 - s) where 1 - s is far below s: relative to the slope itself."""
    dt = DTYPES[dtype]
    g = torch.Generator().manual_seed(rows)
    x, dy, w, b = ffn_case(g, rows, 8, 40, 24, dt, True)
    b[0] = torch.linspace(9.0, 14.0 if dt != torch.float16 else 10.5, 40).to(dt)
    b[1] = torch.full((40,), 64.0).to(dt)
    w[0] = w[0] * 0.125
    got = step(x.to(DEV), dy.to(DEV), [t.to(DEV) for t in w], [t.to(DEV) for t in b], "sigmoid")
    X, DY, (wg, wu, wd) = x.double(), dy.double(), [t.double() for t in w]
    gate, up = X @ wg.T + b[0].double(), X @ wu.T + b[1].double()
    dh = DY @ wd
    dg = dh * up * torch.sigmoid(gate) * torch.sigmoid(-gate)
    # g is of order 14 and a sum of 9 terms: 9 half steps of 16 move the slope by 2^-17; the exponential and the reciprocal of 16-bit types
    # 2^-18, half a step of u and of dh (24 terms of their absolute sum); then two roundings of 16-bit types
    rel = 2.0 ** -16 + (2 * HALF[dt] if dt != torch.float32 else 0.0)
    err = rel * dg.abs() + 32 * 2.0 ** -24 * (DY.abs() @ wd.abs()) * (dg / dh).abs()
    tiny = 2.0 ** -25 * (2 + dh.abs()) if dt == torch.float16 else 0.0  # half a step of fp16 numbers below the normal ones, of u act'(g) and dg
    close(got[5], dg.sum(0), HALF[dt] * dg.sum(0).abs() + (err + tiny).sum(0) + (2.0 ** -25 if dt == torch.float16 else 0.0), "db_gate")
    close(got[2], dg.T @ X, HALF[dt] * (dg.T @ X).abs() + (err + tiny).T @ X.abs() + (2.0 ** -25 if dt == torch.float16 else 0.0), "dw_gate")


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh", "relu", "sigmoid"])
@pytest.mark.parametrize("rows", [2, 30, 150])
def test_slopes_of_huge_gates(rows, act, dtype):
    """Gates of 1e6 to 1e20 either way: act(g) is g or 0 (sigmoid: 1 or 0), the slope 1 or 0 (sigmoid: 0)."""
    dt = DTYPES[dtype]
    g = torch.Generator().manual_seed(rows)
    x, dy, w, b = ffn_case(g, rows, 16, 24, 8, dt, True)
    size = torch.tensor([1e6, -1e6, 1e10, -1e10, 1e13, -1e13, 1e15, -1e15, 1e18, -1e18, 1e20, -1e20]).to(dt)
    b[0] = size.repeat(2)
    w[2] = (w[2].float() * (1e-12 if act != "sigmoid" else 1.0)).to(dt)
    got = step(x.to(DEV), dy.to(DEV), [t.to(DEV) for t in w], [t.to(DEV) for t in b], act)
    up = x.double() @ w[1].double().T + b[1].double()
    ua = x.double().abs() @ w[1].double().abs().T + b[1].double().abs()
    dh, dha = dy.double() @ w[2].double(), dy.double().abs() @ w[2].double().abs()
    slope = (b[0] > 0).double() if act != "sigmoid" else torch.zeros(24, dtype=torch.float64)
    dg, bound = dh * up * slope, (dha * ua * slope)
    # two roundings of 16-bit types, 32 half steps for the two sums; the sum over the rows
    err = (32 * 2.0 ** -24 + (2 * HALF[dt] if dt != torch.float32 else 0.0)) * bound
    close(got[5], dg.sum(0), HALF[dt] * dg.sum(0).abs() + err.sum(0) + rows * 2.0 ** -24 * bound.sum(0), "db_gate")
    assert all(t.isfinite().all() for t in got)


@pytest.mark.parametrize("dtype,ptype", [("fp32", "fp32"), ("bf16", "bf16"), ("fp16", "fp32")])
def test_layer_norm_backward_of_a_bias_without_weight(dtype, ptype):
    dt, pt = DTYPES[dtype], DTYPES[ptype]
    g = torch.Generator().manual_seed(3)
    for rows, width in ((37, 100), (300, 1001), (0, 24), (5, 3), (2, 40000)):
        x, dy, b = rand(g, rows, width, dtype=dt), rand(g, rows, width, dtype=dt), rand(g, width, dtype=pt)
        _, mu, rs = d.layer_norm(x.to(DEV), None, b.to(DEV), return_stats=True)
        dx, dw, db = d.layer_norm_backward(dy.to(DEV), x.to(DEV), None, mu, rs, bias=b.to(DEV))
        assert dw is None and db.dtype == pt and db.shape == (width,)
        want = dy.double().sum(0)
        close(db, want, HALF[pt] * want.abs() + 64 * 2.0 ** -24 * dy.double().abs().sum(0), "db")
        assert torch.equal(dx, d.layer_norm_backward(dy.to(DEV), x.to(DEV), None, mu, rs)[0])
        w = torch.ones(width, dtype=pt, device=DEV)
        assert torch.equal(d.layer_norm_backward(dy.to(DEV), x.to(DEV), w, mu, rs, bias=b.to(DEV))[2], db)
    with pytest.raises(RuntimeError, match="bias"):
        d.layer_norm_backward(dy.to(DEV), x.to(DEV), None, mu, rs, bias=b.to(DEV)[:-1])


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("rows", [1, 2])
@pytest.mark.parametrize("size", [(512, 1400, 264), (72, 33, 17)], ids=lambda s: "x".join(map(str, s)))
def test_single_tokens_round_once(size, rows, dtype):
    """Of one or two rows nothing but the result is rounded to 16 bits, with or without what a backward pass needs."""
    dt = DTYPES[dtype]
    dd, f, n = size
    g = torch.Generator().manual_seed(rows + f)
    x, dy, w, b = ffn_case(g, rows, dd, f, n, dt, True)
    res, exact, _ = ffn_oracle(x, dy, w, b, "gelu")
    xd, w, b = x.to(DEV), [t.to(DEV) for t in w], [t.to(DEV) for t in b]
    y = d.gated_ffn(xd, *w, *b, activation="gelu")
    e = 2.0 ** -24 * (32 + max(dd, f, n) / 8)
    close(y, res["y"], HALF[dt] * res["y"].abs() + e * exact["y"] + (2.0 ** -25 if dt == torch.float16 else 0.0), "y")
    assert torch.equal(y, d.gated_ffn(xd, *w, *b, activation="gelu", save=True)[0])


@pytest.mark.parametrize("size", [(1, 64, 256, 64), (3, 40, 24, 56), (6, 5, 7, 3), (17, 100, 130, 100), (20, 40, 8, 5), (37, 515, 130, 129), (64, 63, 33, 1),
                                  (2, 4, 4, 1), (33, 1030, 1100, 260), (64, 300, 2000, 1027), (48, 4, 5000, 4)], ids=lambda s: "x".join(map(str, s)))
def test_few_fp32_rows_without_planes(size):
    """The backward pass that reads fp32 weights as they lie, at sizes where it is not chosen too: widths off its pieces, blocks of 16 rows with a
    rest, split sums, rows inside wider arrays."""
    m, dd, f, n = size
    g = torch.Generator().manual_seed(m + f)
    x, dy, w, b = ffn_case(g, m, dd, f, n, torch.float32, True)
    wide, pad = torch.full((m, dd + 3), float("nan"), device=DEV), torch.full((m, n + 5), float("nan"), device=DEV)
    wide[:, 2:2 + dd], pad[:, 4:4 + n] = x.to(DEV), dy.to(DEV)
    args = wide[:, 2:2 + dd], pad[:, 4:4 + n], [t.to(DEV) for t in w], [t.to(DEV) for t in b], "silu"
    with plan(COLUMNS, 1):
        got, again = step(*args), step(*args)
    for (name, want, tol), t, t2 in zip(ffn_bounds(x, dy, w, b, "silu", torch.float32), got, again):
        close(t, want, tol, f"{name} {size}")
        assert torch.equal(t, t2), name


@pytest.mark.parametrize("rows", [1, 22, 23])
def test_few_fp32_rows_of_large_weights(rows):
    """Both sides of the rows up to which 8 million elements of each weight are read as they lie."""
    g = torch.Generator().manual_seed(rows)
    x, dy, w, b = ffn_case(g, rows, 1999, 3999, 2010, torch.float32, True)
    got = step(x.to(DEV), dy.to(DEV), [t.to(DEV) for t in w], [t.to(DEV) for t in b], "silu")
    for (name, want, tol), t in zip(ffn_bounds(x, dy, w, b, "silu", torch.float32), got):
        close(t, want, tol, f"{name} {rows}")


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("rows,splits", [(1, 1), (4, 1), (70, 1), (70, 3), (300, 1)])
@pytest.mark.parametrize("size", [(40, 136, 72), (33, 131, 70)], ids=lambda s: "x".join(map(str, s)))
def test_gradients_of_the_hidden_values_round_once(size, rows, splits, dtype):
    """The biases' gradients where one row alone has a gradient are its dg and du: fp32 values rounded once.  The compact form rounds
    u act'(g) and act(g) as well: twice."""
    dt = DTYPES[dtype]
    dd, f, n = size
    g = torch.Generator().manual_seed(rows + f)
    x, dy, w, b = ffn_case(g, rows, dd, f, n, dt, True)
    dy = dy * (torch.arange(rows)[:, None] == rows // 2)
    res, exact, _ = ffn_oracle(x, dy, w, b, "silu")
    e = 2.0 ** -24 * (32 + max(dd, f, n) / 8)
    xd, dyd, w, b = x.to(DEV), dy.to(DEV), [t.to(DEV) for t in w], [t.to(DEV) for t in b]
    for tile in TILES:
        with plan(tile, splits):
            for save, roundings in ((True, 1), ("compact", 2)):
                y, saved = d.gated_ffn(xd, *w, *b, save=save)
                got = dict(zip(NAMES[1:], d.gated_ffn_backward(dyd, xd, *w, saved, bias=True)))
                for name in ("db_gate", "db_up"):
                    tol = roundings * 1.004 * HALF[dt] * res[name].abs() + e * exact[name] + (2.0 ** -24 if dt == torch.float16 else 0)
                    close(got[name], res[name], tol, f"{name} {save} {tile}")
                assert torch.equal(y, d.gated_ffn(xd, *w, *b))


def test_what_a_forward_pass_keeps():
    x, w, wd = torch.ones(6, 16, dtype=torch.bfloat16, device=DEV), torch.ones(24, 16, dtype=torch.bfloat16, device=DEV), torch.ones(8, 24, dtype=torch.bfloat16, device=DEV)
    full, compact = d.gated_ffn(x, w, w, wd, save=True)[1], d.gated_ffn(x, w, w, wd, save="compact")[1]
    assert full.numel() == 6 * 24 * 10 and compact.numel() == 6 * 24 * 6
    with pytest.raises(ValueError, match="save"):
        d.gated_ffn(x, w, w, wd, save="small")
    with pytest.raises(RuntimeError, match="saved"):
        d.gated_ffn_backward(torch.ones_like(x[:, :8]), x, w, w, wd, full[:-1])
    # hidden gradients of half whose slope alone is beyond the type: fp32 keeps it
    h = lambda *s: torch.full(s, 1.0, dtype=torch.float16, device=DEV)  # noqa: E731
    x, wg, wu, wd, dy = h(80, 8), h(8, 8) * 2.0 ** -13, h(8, 8) * 2.0 ** 14, h(8, 8) * 2.0 ** -10, h(80, 8) * 2.0 ** -3
    y, saved = d.gated_ffn(x, wg, wu, wd, activation="relu", save=True)  # g = 2^-10, u = 2^17, h = 2^7, dh = 2^-10, dg = 2^7, du = 2^-20
    dx, dwg, dwu, dwd = d.gated_ffn_backward(dy, x, wg, wu, wd, saved, activation="relu")[:4]
    assert (y == 1).all() and (dwg == 80 * 2.0 ** 7).all() and (dwd == 80 * 2.0 ** 4).all() and (dwu - 80 * 2.0 ** -20).abs().max() <= 2.0 ** -25
    want = 2.0 ** -3 + 2.0 ** -3  # 8 x dg 2^-13 + 8 x du 2^14
    assert (dx.double() - want).abs().max() <= 2.0 ** -11 * want


def test_layer_norm_refuses_parameters_of_two_types():
    x, w, b = torch.ones(3, 8, dtype=torch.bfloat16, device=DEV), torch.ones(8, dtype=torch.bfloat16, device=DEV), torch.ones(8, device=DEV)
    for p, q in ((w, b), (b, w)):
        with pytest.raises(RuntimeError, match="bias must be of type"):
            d.layer_norm(x, p, q)
    for p in (w.half(), b.double()):
        with pytest.raises(RuntimeError, match="weight must be"):
            d.layer_norm(x, p)
    _, mu, rs = d.layer_norm(x, b, b, return_stats=True)
    with pytest.raises(RuntimeError, match="bias must be of type"):
        d.layer_norm_backward(x, x, b, mu, rs, bias=w)
