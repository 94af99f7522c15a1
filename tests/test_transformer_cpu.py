"""Transformer-block operators without a GPU: refusals of the C entry points and of the Python functions, workspace sizes, and the
rotary frequency tables."""
import ctypes as C
import math

import pytest
import torch

import diffusion_model_amd as d
from diffusion_model_amd import _lib

P = C.c_void_p(1 << 20)  # a pointer that no refused call may read
ODD = C.c_void_p((1 << 20) + 8)


def refused(rc, word):
    msg = _lib.lib().dm_last_error().decode()
    assert rc != 0 and word in msg, (rc, msg)


def test_layer_norm_refusals():
    L = _lib.lib()
    ok = dict(x=P, xs=64, w=P, b=P, pt=1, y=P, mean=None, rstd=None, M=4, C=64, eps=1e-5, dt=1)

    def call(**kw):
        a = {**ok, **kw}
        return L.dm_layer_norm(a["x"], a["xs"], a["w"], a["b"], a["pt"], a["y"], a["mean"], a["rstd"], a["M"], a["C"], a["eps"], a["dt"], None)
    refused(call(x=None), "null")
    refused(call(y=None), "null")
    refused(call(dt=7), "dtype")
    refused(call(pt=2), "parameters")
    refused(call(C=0), "width")
    refused(call(M=-1), "rows")
    refused(call(xs=63), "stride")
    refused(call(eps=-1.0), "eps")
    refused(call(eps=float("nan")), "eps")
    assert call(M=0, x=None) == 0
    need = L.dm_layer_norm_backward_workspace_bytes(5000, 64)
    assert need > 0 and L.dm_layer_norm_backward_workspace_bytes(0, 64) == 0

    def back(dys=64, dy=P, dw=P, ws=P, n=need):
        return L.dm_layer_norm_backward(dy, dys, P, 64, P, 1, P, P, P, dw, P, 5000, 64, 1, ws, n, None)
    refused(back(dy=None), "null")
    refused(back(dys=10), "stride")
    refused(back(n=need - 1), "workspace")
    refused(back(ws=None), "workspace")


def test_rotary_refusals():
    L = _lib.lib()

    def tensor(heads=4, out=1 << 20, strides=(512, 64, 16)):
        t = _lib.RotaryTensor()
        t.in_, t.out, t.heads = 1 << 20, out, heads
        for i in range(3):
            t.in_stride[i], t.out_stride[i] = (512, 64, 16)[i], strides[i]
        return t

    def call(q=None, k=None, pos=P, ps=(0, 8, 1), axes=1, inv=P, B=2, T=8, hd=16, rd=16, dt=0):
        q = q or tensor()
        return L.dm_rotary(C.byref(q), C.byref(k) if k else None, pos, (C.c_int64 * 3)(*ps) if ps else None, axes, inv, B, T, hd, rd, 0, 1.0, 0, dt, None)
    refused(call(dt=3), "dtype")
    refused(call(rd=18), "rotary_dim")
    refused(call(rd=7), "rotary_dim")
    refused(call(axes=3), "axes")
    refused(call(axes=0), "axes")
    refused(call(axes=2, pos=None), "positions")
    refused(call(ps=None), "strides")
    refused(call(inv=None), "null")
    refused(call(T=-1), "sizes")
    refused(call(q=tensor(heads=-1)), "heads")
    refused(call(q=tensor(out=0)), "null")
    refused(call(q=tensor(strides=(512, 64, 32))), "in place")
    refused(call(k=tensor(strides=(512, 128, 16))), "in place")
    assert L.dm_rotary(None, None, None, None, 1, P, 1, 1, 16, 16, 0, 1.0, 0, 0, None) != 0
    assert call(B=0) == 0 and call(T=0) == 0 and call(q=tensor(heads=0)) == 0


def test_gated_ffn_refusals():
    L = _lib.lib()
    need = L.dm_gated_ffn_workspace_bytes(100, 64, 128, 64, 1, 0)
    assert need >= 100 * 128 * 2
    assert L.dm_gated_ffn_workspace_bytes(100, 64, 128, 64, 0, 0) >= 3 * 2 * (100 * 64 + 3 * 64 * 128 + 100 * 128)  # three planes of every operand
    assert L.dm_gated_ffn_saved_bytes(100, 129, 1) == 3 * 100 * 136 * 2 and L.dm_gated_ffn_saved_bytes(0, 129, 1) == 0
    assert L.dm_gated_ffn_workspace_bytes(0, 64, 128, 64, 1, 0) == 0 and L.dm_gated_ffn_workspace_bytes(10, 0, 128, 64, 1, 0) == 0
    ok = dict(x=P, xs=64, wg=P, wu=P, wd=P, y=P, saved=None, M=100, D=64, F=128, N=64, act=0, dt=1, ws=P, n=need)

    def call(**kw):
        a = {**ok, **kw}
        return L.dm_gated_ffn(a["x"], a["xs"], a["wg"], a["wu"], a["wd"], None, None, None, a["y"], a["saved"], a["M"], a["D"], a["F"], a["N"], a["act"],
                              a["dt"], a["ws"], a["n"], None)
    for name in ("x", "wg", "wu", "wd", "y"):
        refused(call(**{name: None}), "null")
    for name in ("x", "wg", "wu", "wd", "saved"):
        refused(call(**{name: ODD}), "16")
    refused(call(xs=68), "16")
    refused(call(xs=56), "stride")
    refused(call(xs=1 << 22), "stride")
    refused(call(dt=5), "dtype")
    refused(call(act=5), "activation")
    refused(call(act=-1), "activation")
    refused(call(D=0), "widths")
    refused(call(F=(1 << 20) + 1), "widths")
    refused(call(M=-3), "rows")
    refused(call(n=need - 1), "workspace")
    refused(call(ws=None), "workspace")
    assert call(M=0) == 0
    need_b = L.dm_gated_ffn_backward_workspace_bytes(100, 64, 128, 64, 1)

    def back(dy=P, dys=64, saved=P, n=need_b, dw=P, db=None):
        return L.dm_gated_ffn_backward(dy, dys, P, 64, P, P, P, saved, P, dw, P, P, db, None, None, 100, 64, 128, 64, 0, 1, P, n, None)
    refused(back(dy=None), "null")
    refused(back(dy=ODD), "16")
    refused(back(dys=63), "stride")
    refused(back(saved=None), "saved")
    refused(back(n=need_b - 1), "workspace")
    refused(back(dw=None, db=P), "weight's")


def test_functions_need_the_gpu():
    x = torch.zeros(3, 8)
    inv = d.rotary_frequencies(8)[0]
    for call in (lambda: d.layer_norm(x), lambda: d.layer_norm_backward(x, x, None, x[:, 0], x[:, 0]),
                 lambda: d.apply_rotary(x.view(1, 3, 1, 8), None, inv), lambda: d.gated_ffn(x, x, x, x.T),
                 lambda: d.gated_ffn_backward(x, x, x, x, x.T, None)):
        with pytest.raises(RuntimeError, match="GPU"):
            call()


def test_rotary_frequencies():
    inv, scale = d.rotary_frequencies(128)
    assert inv.dtype == torch.float64 and inv.shape == (64,) and scale == 1.0
    assert inv[0] == 1.0 and abs(inv[-1].item() - 10000.0 ** (-126 / 128)) < 1e-18
    two, _ = d.rotary_frequencies(64, axes=2)
    assert torch.equal(two[:16], two[16:]) and torch.equal(two[:16], d.rotary_frequencies(32)[0])
    lin, _ = d.rotary_frequencies(128, scaling="linear", factor=4.0)
    assert torch.allclose(lin * 4, inv, rtol=1e-15, atol=0)
    ntk, _ = d.rotary_frequencies(128, scaling="ntk", factor=4.0)  # the fastest pair stays, the slowest is divided by the factor
    assert ntk[0] == 1.0 and abs(ntk[-1] * 4 / inv[-1] - 1) < 1e-12 and (ntk[1:] < inv[1:]).all()
    yarn, scale = d.rotary_frequencies(128, scaling="yarn", factor=8.0, original_length=4096)
    assert abs(scale - (0.1 * math.log(8.0) + 1)) < 1e-15
    turns = inv * 4096 / (2 * math.pi)
    assert torch.equal(yarn[turns > 40], inv[turns > 40]) and torch.allclose(yarn[turns < 0.8] * 8, inv[turns < 0.8], rtol=1e-15)
    assert ((yarn <= inv) & (yarn >= inv / 8 * (1 - 1e-15))).all() and (yarn[1:] < yarn[:-1]).all()
    assert d.rotary_frequencies(0)[0].numel() == 0 and d.rotary_frequencies(2, scaling="ntk", factor=2.0)[0][0] == 1.0
    for bad in (dict(rotary_dim=7), dict(rotary_dim=8, axes=3), dict(rotary_dim=8, axes=0), dict(rotary_dim=8, base=0.0),
                dict(rotary_dim=8, factor=0.0), dict(rotary_dim=8, scaling="cubic"), dict(rotary_dim=8, scaling="yarn", factor=2.0)):
        with pytest.raises(ValueError):
            d.rotary_frequencies(**bad)


@pytest.mark.parametrize("dim,base,length,factor", [(128, 10000.0, 131072, 4.0), (128, 10000.0, 65536, 4.0), (8, 10000.0, 8192, 16.0),
                                                     (64, 500.0, 100000, 8.0), (128, 10000.0, 4096, 8.0), (128, 10000.0, 10 ** 11, 2.0)])
def test_yarn_blends_every_pair_that_turns_more_than_once(dim, base, length, factor):
    """A pair is divided whole only from where pairs turn less than once over the trained length, also where that lies behind the last one."""
    pairs = dim // 2
    inv, _ = d.rotary_frequencies(dim, base=base)
    yarn, _ = d.rotary_frequencies(dim, base=base, scaling="yarn", factor=factor, original_length=length)
    turns = inv * length / (2 * math.pi)

    def pair(n):  # base^(-i / pairs) length = 2 pi n
        return pairs * math.log(length / (2 * math.pi * n)) / math.log(base)
    first, last = max(math.floor(pair(32)), 0), min(math.ceil(pair(1)), dim - 1)
    for i in range(pairs):
        part = min(max((i - first) / (last - first), 0.0), 1.0) if last > first else 0.0
        want = inv[i].item() * ((1 - part) + part / factor)
        assert abs(yarn[i].item() - want) <= 4e-16 * want, (i, turns[i].item())
        if turns[i] > 1:
            assert yarn[i] > inv[i] / factor * (1 + 1e-12), i


def test_gated_ffn_forms_of_what_is_kept_and_plans():
    L = _lib.lib()
    keep = 256  # DM_FFN_KEEP_F32
    for dtype, plain, kept in ((0, 14, 14), (1, 6, 10), (2, 6, 10)):
        assert L.dm_gated_ffn_saved_bytes(7, 33, dtype) == 7 * 40 * plain and L.dm_gated_ffn_saved_bytes(7, 33, dtype | keep) == 7 * 40 * kept
    assert L.dm_gated_ffn_saved_bytes(7, 33, 3 | keep) == 0
    need = L.dm_gated_ffn_workspace_bytes(100, 64, 128, 64, 1, 1)
    for act in (5 | keep, -1, 512):
        refused(L.dm_gated_ffn(P, 64, P, P, P, None, None, None, P, P, 100, 64, 128, 64, act, 1, P, need, None), "activation")
    for tile, splits in ((4, 1), (-2, 1), (0, 0), (0, 65)):
        refused(L.dm_debug_ffn_plan(tile, splits), "plan")
    assert L.dm_debug_ffn_plan(0, 4) == 0 and L.dm_gated_ffn_workspace_bytes(100, 4096, 128, 64, 1, 0) > need and L.dm_debug_ffn_plan(-1, 1) == 0
    assert L.dm_gated_ffn_workspace_bytes(100, 64, 128, 64, 1, 1) == need
