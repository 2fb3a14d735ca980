"""Host-side checks of the optimizer and 4-bit entry points (nothing is launched), and the oracles they are tested against."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from oracle import mxfp4 as OM
from oracle import optim as OO

P = C.c_void_p(1 << 20)       # a pointer that is never followed: every call below is refused before a launch


def _refused(lib, rc, text):
    assert rc < 0 and text.encode() in lib.cfd_last_error(), lib.cfd_last_error()


def test_grad_norm_refuses(lib):
    n = (C.c_int64 * 2)(10, -1)
    g = (C.c_void_p * 2)(1 << 20, 1 << 20)
    _refused(lib, lib.cfd_grad_norm_workspace_bytes(n, 2), "negative")
    _refused(lib, lib.cfd_grad_norm(g, n, 2, 0, 1.0, P, P, None), "negative")
    n[1] = 5
    assert lib.cfd_grad_norm_workspace_bytes(n, 2) >= 16
    _refused(lib, lib.cfd_grad_norm(g, n, 2, 2, 1.0, P, P, None), "dtype")
    _refused(lib, lib.cfd_grad_norm(g, n, 2, 0, 0.0, P, P, None), "max_norm")
    _refused(lib, lib.cfd_grad_norm(g, n, 2, 0, 1.0, None, P, None), "bad arguments")
    g[1] = None
    _refused(lib, lib.cfd_grad_norm(g, n, 2, 0, 1.0, P, P, None), "NULL")


def test_adamw_refuses(lib):
    from cfd_amd._lib import AdamwDesc, AdamwTensor
    t = (AdamwTensor * 1)()
    t[0].p = t[0].g = 1 << 20
    t[0].n = 10
    good = dict(p_dtype=0, g_dtype=0, state_bits=8, seed=0, lr=1e-3, eps=1e-7, beta1=0.9, beta2=0.999)

    def call(text, m=P, ms=P, **kw):
        d = AdamwDesc(**{**good, **kw})
        _refused(lib, lib.cfd_adamw_step(t, 1, C.byref(d), m, P, ms, ms, P, None, None, P, None), text)

    call("bad arguments", m=None)
    call("state_bits", state_bits=4)
    call("state_bits", ms=None)
    call("dtype", p_dtype=3)
    call("beta", beta1=1.0)
    call("beta", beta2=float("nan"))
    call("beta", eps=-1.0)
    call("aligned", m=C.c_void_p((1 << 20) + 4))
    t[0].state_offset = 100
    call("256")
    t[0].state_offset = 0
    t[0].copy = 1 << 20
    call("copy", p_dtype=1)
    t[0].copy, t[0].n = None, -1
    call("negative")


def test_mxfp4_refuses(lib):
    from cfd_amd._lib import Mxfp4DenseDesc
    q = lib.cfd_mxfp4_quantize
    _refused(lib, q(P, 8, 2, 4, 8, P, P, None, None, None), "dtype")
    _refused(lib, q(P, 7, 0, 4, 8, P, P, None, None, None), "bad arguments")
    _refused(lib, q(P, 8, 0, 4, 0, P, P, None, None, None), "columns")
    _refused(lib, q(P, 8, 0, -1, 8, P, P, None, None, None), "rows")
    _refused(lib, q(P, 8, 0, 4, 8, None, None, None, None, None), "orientation")
    _refused(lib, q(P, 8, 0, 4, 8, P, None, None, None, None), "orientation")
    _refused(lib, q(P, 8, 0, 4, 8, C.c_void_p(24), P, None, None, None), "aligned")
    _refused(lib, q(P, 8, 0, 1 << 23, 8, P, P, P, P, None), "columns")
    _refused(lib, lib.cfd_mxfp4_dequantize(P, P, 4, 8, P, 7, 0, None), "bad arguments")
    _refused(lib, lib.cfd_mxfp4_dense_workspace_bytes(1, 1, 0, 0), "columns")
    assert lib.cfd_mxfp4_scale_pitch(1) == 16 and lib.cfd_mxfp4_scale_pitch(512) == 16 and lib.cfd_mxfp4_scale_pitch(513) == 32
    good = dict(x_kind=2, out_dtype=0, act=0, leaky_slope=0.2, m=4, n=4, k=64, ldx=0, ldy=4)

    def call(text, x=P, xs=P, w=P, y=P, **kw):
        d = Mxfp4DenseDesc(**{**good, **kw})
        _refused(lib, lib.cfd_mxfp4_dense(C.byref(d), x, xs, w, P, None, y, None, None), text)

    call("x_kind", x_kind=3)
    call("out_dtype", out_dtype=2)
    call("activation", act=4)
    call("bad arguments", ldy=3)
    call("bad arguments", y=None)
    call("bad activations", xs=None)
    call("bad activations", x_kind=0, ldx=63)
    call("aligned", w=C.c_void_p(8))
    call("aligned", x=C.c_void_p(8))
    call("workspace", m=64, n=64, k=1 << 20, ldy=64)
    call("rows", m=-1)


def test_wrappers_refuse_host_tensors():
    from cfd_amd import _lib, ops, trainer
    x = torch.zeros(4, 32)
    q = ops.Mxfp4(torch.zeros(4, 16, dtype=torch.uint8), torch.zeros(4, 16, dtype=torch.uint8), 32)
    for call in (lambda: ops.grad_norm([x], 1.0), lambda: trainer.AdamW([x]), lambda: ops.mxfp4_quantize(x),
                 lambda: ops.mxfp4_dequantize(q), lambda: ops.mxfp4_dense(x, q), lambda: ops.mxfp4_from_parts(q.codes, q.scales[:, :1], 32)):
        with pytest.raises(_lib.CfdError):
            call()


def test_oracle_fp4_is_the_nearest_value():
    """every code's value maps to itself; any other value to a nearest one; a block keeps its sign and its zeros"""
    x = np.linspace(-7, 7, 32 * 50).reshape(50, 32)
    x[:, 0] = 6.5                                  # scale 1
    v = OM.round_trip(x)
    best = np.abs(x[..., None] - np.concatenate([OM.GRID, -OM.GRID])).min(-1)
    assert np.array_equal(np.abs(v - x), best)
    g = np.concatenate([OM.GRID, -OM.GRID, OM.GRID, -OM.GRID])[None]
    for e in (-100, 0, 90):
        assert np.array_equal(OM.round_trip(g * 2.0 ** e), g * 2.0 ** e)
    assert OM.quantize(np.zeros((1, 5)))[1].tolist() == [[0]]


def test_oracle_state_encoding_brackets_the_value():
    """the two values stochastic rounding may store are neighbours around x, and their mean over the draws is x"""
    r = np.random.default_rng(0)
    x = np.abs(r.standard_normal(256)) * 10.0 ** r.uniform(-3, 0, 256)
    for enc, digits in ((OO.encode_m, 3), (OO.encode_v, 2)):
        lo, s = enc(x, np.zeros(256))
        hi, _ = enc(x, np.full(256, 65535.0))
        lo, hi = lo * s, hi * s
        assert (lo <= x * (1 + 2.0 ** -24)).all() and (hi >= x * (1 - 2.0 ** -10)).all()
        assert (hi - lo <= np.maximum(x * 2.0 ** -digits, s * 2.0 ** -9)).all()
        mean = np.mean([enc(x, np.full(256, u))[0] for u in range(0, 65536, 256)], 0) * s
        assert np.abs(mean - x).max() <= 2.0 ** -7 * np.maximum(x, s).max()


def test_oracle_adamw_published_first_step():
    p, m, v = OO.adamw(10.0, 3.0, 0.0, 0.0, 1, 0.1, 0.9, 0.999, 1e-7, 0.0)
    assert abs(p - 9.9) < 1e-6 and math.isclose(float(m), 0.3) and math.isclose(float(v), 0.009)
    assert OO.grad_norm([[3.0], [4.0]], 1.0) == (5.0, 0.2)


def test_mxfp4_plan_reaches_every_way_of_sharing(lib):
    """the products that the GPU tests compute exactly are divided as their lists say: one, two and four waves on a weight tile, with
    one round over the K groups and several, whole and ragged, in one slice of K and in many; both 4-bit tiles with and without slices"""
    from tests import test_mxfp4_sums_gpu as T
    seen = set()
    for m, n, k, kind, how in T.FLOAT:
        rows, slices, groups, waves = T.plan(lib, m, n, k, kind)
        total = -(-k // 512)
        last = total - (slices - 1) * groups
        assert (waves, -(-groups // waves), bool(groups % waves or last % waves), slices) == how, (m, n, k, kind)
        seen |= {(waves, "rounds", groups > waves), (waves, "ragged", how[2]), (waves, "slices", slices > 1), (kind, waves)}
    assert {(w, "rounds", True) for w in (1, 2, 4)} | {(w, "rounds", False) for w in (2, 4)} <= seen
    assert {(w, "ragged", r) for w in (2, 4) for r in (True, False)} <= seen
    assert {(t, w) for t in ("fp32", "bf16") for w in (1, 2, 4)} | {(4, "slices", False), (4, "slices", True)} <= seen
    four = [T.plan(lib, m, n, k, "fp4") for m, n, k, _ in T.FOUR]
    assert [(rows, groups, slices) for rows, slices, groups, _ in four] == [how for *_, how in T.FOUR]
    assert {(rows, slices > 1) for rows, slices, *_ in four} == {(r, s) for r in (64, 256) for s in (True, False)}
    assert lib.cfd_mxfp4_dense_plan(4, 4, 0, 2, None) < 0 and lib.cfd_mxfp4_dense_plan(4, 4, 64, 3, (C.c_int * 4)()) < 0
    _refused(lib, lib.cfd_mxfp4_dense_plan(0, 4, 64, 2, (C.c_int * 4)()), "bad arguments")


def test_an_output_over_an_operand_is_seen():
    """_apart on views of one buffer: between the rows of an output or behind it is beside it, one byte inside is over it"""
    from cfd_amd import ops
    buf = torch.zeros(6, 64)
    flat, raw = buf.view(-1), buf.view(-1).view(torch.uint8)
    out = buf[:, :24]
    assert ops._apart(out, None, buf[2, 24:48], flat[24:64], flat[5 * 64 + 24:], torch.zeros(24), raw[96:256].view(10, 16))
    for t in (buf[2, 23:47], buf[2, 40:].contiguous().set_(flat[150:220]), flat[:1], flat[5 * 64 + 23:], flat[60:65], raw[95:111], raw[96:257], buf):
        assert not ops._apart(out, None, t), t.shape
    assert ops._apart(buf[:1, :24], flat[24:]) and not ops._apart(buf[:1, :24], flat[23:])
    assert ops._apart(buf[:0], buf) and ops._apart(buf[:, :0], buf)
    half = torch.zeros(4, 10, dtype=torch.bfloat16)
    assert not ops._apart(half[:, :3], half.view(-1)[32:33]) and ops._apart(half[:, :3], half.view(-1)[33:40])


def test_what_stochastic_rounding_cuts():
    """over all 65536 draws a stored value is low by 0 to 2^-16 of its code's spacing in the mean, never high"""
    x = np.abs(np.random.default_rng(1).standard_normal(256)) * 10.0 ** np.random.default_rng(2).uniform(-3, 0, 256)
    for enc in (OO.encode_m, OO.encode_v):
        lo, s = enc(x, np.zeros(256))
        hi, _ = enc(x, np.full(256, 65535.0))
        total = np.zeros(256)
        for u in range(0, 65536, 4096):
            q, _ = enc(np.tile(x, 4096), np.repeat(np.arange(u, u + 4096.0), 256))
            total += q.reshape(4096, 256).sum(0)
        low = (x - total / 65536 * s) / ((hi - lo) * s)
        assert (hi > lo).all() and low.min() >= -1e-9 and low.max() <= 2.0 ** -16


def test_adamw_refuses_a_slow_beta_in_8_bits(lib):
    """past 0.9999 what an 8-bit state's rounding cuts is no longer small beside a step's movement"""
    from cfd_amd._lib import AdamwDesc, AdamwTensor
    t = (AdamwTensor * 1)()
    t[0].p = t[0].g = 1 << 20
    t[0].n = 10
    good = dict(p_dtype=0, g_dtype=0, state_bits=8, seed=0, lr=1e-3, eps=1e-7, beta1=0.9, beta2=0.999)
    for kw in (dict(beta1=0.99991), dict(beta2=0.99999)):
        d = AdamwDesc(**{**good, **kw})
        _refused(lib, lib.cfd_adamw_step(t, 1, C.byref(d), P, P, P, P, P, None, None, P, None), "0.9999")
