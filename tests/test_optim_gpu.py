"""Gradient norm and AdamW over tensor lists on the GPU against the 64-bit formulas.

Tolerances: one fp32 operation is off by at most 2^-24 of its result.  The state's recursion is three operations an entry
(compared exactly with single fp32 operations); a parameter takes two roundings of its own and about eight in its update,
whose terms are bounded by alpha (|m| + |g|) / (sqrt(v) + eps); storing bf16 adds 2^-8 of the value."""
import math

import numpy as np
import pytest
import torch

from oracle import optim as O

pytestmark = pytest.mark.gpu
SIZES = [1, 3, 0, 255, 256, 257, 4096, 4097, 10001]
HYPER = dict(lr=3e-3, beta_1=0.9, beta_2=0.999, epsilon=1e-7, seed=77)


def _views(sizes, dtype, seed, scale=1.0):
    """slices of one buffer: odd offsets, element alignment only"""
    flat = torch.randn(sum(sizes) + 1, generator=torch.Generator().manual_seed(seed)) * scale
    return list(torch.split(flat.to(dtype).cuda()[1:], sizes))


def _f64(t):
    return t.detach().float().cpu().numpy().astype(np.float64)


def _state(opt):
    """(m, v) of every tensor as the values they stand for"""
    out = []
    for k, p in enumerate(opt.params):
        lo, n = opt.offsets[k], O.padded(p.numel())
        mv = []
        for x, s in ((opt.m, opt.m_scale), (opt.v, opt.v_scale)):
            val = _f64(x[lo:lo + n])
            if s is not None:
                val = val * np.repeat(_f64(s[lo // 256:(lo + n) // 256]), 256)
            mv.append(val)
        out.append(mv)
    return out


def _check_step(opt, grads, scale, lr, wd):
    """runs one step and compares parameters, copies and state with the oracle"""
    t = int(opt.t) + 1
    before, p0, g0 = _state(opt), [_f64(p) for p in opt.params], [_f64(g) for g in grads]
    gs = None if scale is None else torch.full((1,), scale, device="cuda")
    opt.step(grads, gs)
    assert int(opt.t) == t
    s = 1.0 if scale is None else float(np.float32(scale))
    total = O.padded(max(opt.offsets) + 1) + 20000
    um, uv = O.draws(total, t, opt.seed)
    a = O.alpha(lr, opt.b1, opt.b2, t)
    for k, p in enumerate(opt.params):
        n = p.numel()
        if n == 0:
            continue
        m0, v0 = before[k]
        g = np.zeros(O.padded(n))
        g[:n] = g0[k].reshape(-1)
        p64, m64, v64 = O.adamw(p0[k].reshape(-1), g[:n], m0[:n], v0[:n], t, lr, opt.b1, opt.b2, opt.eps, wd[k], s)
        tol = 2.0 ** -23 * (2 * np.abs(p64) + 8 * a * (np.abs(m64) + np.abs(g[:n] * s)) / (np.sqrt(v64) + opt.eps)) + 1e-38
        if p.dtype == torch.bfloat16:
            tol = tol + 2.0 ** -8 * np.abs(p64)
        got = _f64(p).reshape(-1)
        assert (np.abs(got - p64) <= tol).all(), (k, n, np.abs(got - p64).max())
        if opt.copies is not None:
            assert torch.equal(opt.copies[k], p.to(torch.bfloat16))
        m32, v32 = O.state32(g, m0, v0, opt.b1, opt.b2, s)
        assert np.all(np.abs(m32[:n] - m64) <= 2.0 ** -22 * (np.abs(m64) + np.abs(g[:n] * s)) + 1e-38)
        m1, v1 = _state(opt)[k]
        if opt.state_bits == 32:
            assert np.array_equal(m1[:n], m32[:n].astype(np.float64)) and np.array_equal(v1[:n], v32[:n].astype(np.float64))
        else:
            lo = opt.offsets[k]
            for got, x, u, enc in ((m1, m32, um, O.encode_m), (v1, v32, uv, O.encode_v)):
                q, sc = enc(x, u[lo:lo + len(x)])
                assert np.array_equal(got, q * np.repeat(sc, 256))
        assert not m1[n:].any() and not v1[n:].any()        # the padding stays zero


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("pdt,gdt,copy", [(torch.float32, torch.float32, False), (torch.float32, torch.float32, True),
                                          (torch.float32, torch.bfloat16, True), (torch.bfloat16, torch.bfloat16, False),
                                          (torch.bfloat16, torch.float32, False)])
def test_adamw_steps(bits, pdt, gdt, copy):
    from cfd_amd import trainer
    params = _views(SIZES, pdt, 1, 0.05)
    wd = [0.0 if n < 100 else 0.02 for n in SIZES]
    copies = [torch.zeros(n, dtype=torch.bfloat16, device="cuda") for n in SIZES] if copy else None
    opt = trainer.AdamW(params, weight_decay=wd, state_bits=bits, copies=copies, **HYPER)
    for i, scale in enumerate((None, 0.5, 1.0, 1e-3)):
        grads = _views(SIZES, gdt, 10 + i, 10.0 ** -i)
        _check_step(opt, grads, scale, HYPER["lr"], wd)


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_many_tensors_and_large_magnitudes(bits):
    """more tensors than one launch takes; gradients from 1e-30 to 1e15 in one block"""
    from cfd_amd import trainer
    sizes = [(37 * i) % 300 for i in range(150)]
    params = _views(sizes, torch.float32, 3)
    opt = trainer.AdamW(params, weight_decay=0.0, state_bits=bits, **HYPER)
    for i in range(2):
        grads = [g * 10.0 ** torch.linspace(-30, 15, max(g.numel(), 1), device="cuda")[:g.numel()] for g in _views(sizes, torch.float32, 20 + i)]
        _check_step(opt, grads, None, HYPER["lr"], [0.0] * len(sizes))


def test_adamw_first_step_moves_by_the_learning_rate():
    from cfd_amd import trainer
    for bits in (32, 8):
        p = torch.full((1000,), 10.0, device="cuda")
        trainer.AdamW([p], lr=0.1, weight_decay=0.0, state_bits=bits).step([torch.full_like(p, 3.0)])
        assert float((p - 9.9).abs().max()) < 2e-6


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_adamw_skips_a_step_that_is_not_finite(bits, bad):
    from cfd_amd import ops, trainer
    p = _views([5, 1000], torch.float32, 4)
    opt = trainer.AdamW(p, state_bits=bits, **HYPER)
    g = _views([5, 1000], torch.float32, 5)
    opt.step(g)
    keep = [x.clone() for x in p] + [opt.m.view(torch.uint8).clone(), opt.v.view(torch.uint8).clone()]
    g[1][700] = bad
    n = ops.grad_norm(g, 1.0)
    assert math.isnan(float(n[1]))
    opt.step(g, n[1:])
    now = list(p) + [opt.m.view(torch.uint8), opt.v.view(torch.uint8)]
    assert int(opt.t) == 1 and all(torch.equal(a, b) for a, b in zip(keep, now))


def test_adamw8_infinity_stays_in_its_block():
    from cfd_amd import trainer
    p = torch.ones(1024, device="cuda")
    opt = trainer.AdamW([p], state_bits=8, **HYPER)
    g = torch.ones(1024, device="cuda")
    g[300] = float("inf")
    opt.step([g])
    opt.step([torch.ones(1024, device="cuda")])
    bad = torch.isnan(p)
    assert bad[256:512].all() and not bad[:256].any() and not bad[512:].any()


def test_adamw8_rounding_is_unbiased():
    """the mean of n stored values is within 5 standard errors of the value: a stored value is one of two neighbours a step
    apart, so its standard deviation is at most half a step (16 rounding bits: a bias of 2^-16 steps at most)"""
    from cfd_amd import trainer
    n = 1 << 16
    p = torch.zeros(n, device="cuda")
    opt = trainer.AdamW([p], state_bits=8, lr=0.0, weight_decay=0.0, seed=5)
    g = torch.full((n,), 0.77, device="cuda")
    g[::256] = 3.1                                       # the block's maximum: the others lie inside the code range
    opt.step([g])
    m1, v1 = O.state32(np.float32(0.77), 0.0, 0.0, 0.9, 0.999)
    pick = torch.arange(n, device="cuda") % 256 != 0
    for got, s, want in ((opt.m, opt.m_scale, float(m1)), (opt.v, opt.v_scale, float(v1))):
        val = (got.float() * s.repeat_interleave(256))[pick].double()
        lo, hi = float(val.min()), float(val.max())
        assert lo <= want <= hi and (hi - lo) <= want / 4    # two neighbours: at most 2^-2 (e5m2) apart relatively
        assert abs(float(val.mean()) - want) <= 5 * (hi - lo) / 2 / math.sqrt(n) + (hi - lo) * 2.0 ** -15


def test_adamw_in_a_captured_graph():
    """replays advance t, read the scale and the rate from the device, and equal eager steps bit for bit"""
    from cfd_amd import ops, trainer
    sizes = [1, 777, 5000]
    def build():
        return trainer.AdamW(_views(sizes, torch.float32, 6), lr=torch.full((1,), 1e-2, device="cuda"), state_bits=8, weight_decay=0.01, seed=3)
    a, b = build(), build()
    grads = _views(sizes, torch.float32, 7)
    norm = torch.zeros(2, device="cuda")
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):                          # warm-up outside the capture, on the optimizer that is compared
        ops.grad_norm(grads, 0.5, out=norm)
        a.step(grads, norm[1:])
    torch.cuda.current_stream().wait_stream(st)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.grad_norm(grads, 0.5, out=norm)
        a.step(grads, norm[1:])
    b.step(grads, ops.grad_norm(grads, 0.5)[1:])
    for i in range(4):
        for g in grads:
            g.mul_(1.0 + i).add_(0.01)
        a.lr.fill_(1e-2 / (i + 1)), b.lr.fill_(1e-2 / (i + 1))
        graph.replay()
        torch.cuda.synchronize()
        b.step(grads, ops.grad_norm(grads, 0.5)[1:])
        assert int(a.t) == int(b.t) == i + 2
        assert all(torch.equal(x, y) for x, y in zip(a.params, b.params))
        assert torch.equal(a.m.view(torch.uint8), b.m.view(torch.uint8)) and torch.equal(a.v_scale, b.v_scale)


def test_adamw_on_another_stream_and_repeated_runs_agree():
    from cfd_amd import trainer
    sizes = [999, 100_003]
    got = []
    for k in range(2):
        p = _views(sizes, torch.float32, 8)
        opt = trainer.AdamW(p, state_bits=8, **HYPER)
        st = torch.cuda.Stream() if k else torch.cuda.current_stream()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            for i in range(3):
                opt.step(_views(sizes, torch.bfloat16, 30 + i))
        torch.cuda.synchronize()
        got.append([x.clone() for x in p] + [opt.m.view(torch.uint8).clone(), opt.v.view(torch.uint8).clone()])
    assert all(torch.equal(a, b) for a, b in zip(*got))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("sizes", [[1], [0, 5], [4096], [4097, 1, 0, 33], [(13 * i) % 70 for i in range(200)], [9_000_001]])
def test_grad_norm(sizes, dtype):
    """fp64 sums rounded once: 2^-24, twice that with the division's own rounding"""
    from cfd_amd import ops
    g = _views(sizes, dtype, 40)
    for max_norm in (0.3, 1e9):
        n, s = O.grad_norm([_f64(x) for x in g], max_norm)
        got = ops.grad_norm(g, max_norm).double().cpu().numpy()
        assert abs(got[0] - n) <= 2.0 ** -23 * n and abs(got[1] - s) <= 2.0 ** -23 * s
    assert torch.equal(ops.grad_norm(g, 0.3), ops.grad_norm(g, 0.3))


def test_grad_norm_extremes():
    from cfd_amd import ops
    z = torch.zeros(100, device="cuda")
    assert ops.grad_norm([z], 1.0).tolist() == [0.0, 1.0]
    assert ops.grad_norm([z[:0]], 1.0).tolist() == [0.0, 1.0]
    big = torch.full((3,), 1e38, device="cuda")           # squares past fp32
    n = ops.grad_norm([big], 1.0).double().tolist()
    assert abs(n[0] - math.sqrt(3) * 1e38) <= 2e-7 * n[0]
    tiny = torch.full((4,), 1e-30, device="cuda")         # squares under fp32
    assert abs(float(ops.grad_norm(tiny, 1.0)[0]) - 2e-30) <= 1e-36
    z[50] = float("inf")
    n = ops.grad_norm([z, big], 1.0).tolist()
    assert n[0] == float("inf") and math.isnan(n[1])


def test_tensors_past_32_bits():
    """a tensor of more than 2^31 elements: norm over all of it, and its last elements step like a short tensor's (first step: the
    parameters do not depend on how the state is rounded)"""
    from cfd_amd import ops, trainer
    n = (1 << 31) + 777
    p, g = torch.zeros(n, dtype=torch.bfloat16, device="cuda"), torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    tail = torch.randn(5000, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    p[-5000:], g[-5000:] = 0.5, tail
    want = float(tail.double().square().sum().sqrt())
    assert abs(float(ops.grad_norm([g], 1.0)[0]) - want) <= 2.0 ** -23 * want
    q = torch.full((5000,), 0.5, dtype=torch.bfloat16, device="cuda")
    a, b = trainer.AdamW([p], state_bits=8, **HYPER), trainer.AdamW([q], state_bits=8, **HYPER)
    a.step([g]), b.step([tail])
    assert torch.equal(p[-5000:], q) and not p[:-5000].any()
    lo = n - 4096
    m = a.m[lo // 256 * 256:].float() * a.m_scale[lo // 256:].repeat_interleave(256)
    want = 0.1 * g[lo // 256 * 256:].float()
    m = m[:want.numel()]
    assert (m - want).abs().max() <= want.abs().max() / 8      # a code step apart at most


def test_only_empty_tensors():
    from cfd_amd import trainer
    for bits in (32, 8):
        e = torch.zeros(0, device="cuda")
        opt = trainer.AdamW([e], state_bits=bits)
        opt.step([e.clone()])
        assert int(opt.t) == 1


def test_refusals():
    from cfd_amd import _lib, ops, trainer
    c = lambda *s, dt=torch.float32: torch.zeros(*s, dtype=dt, device="cuda")  # noqa: E731
    bad = _lib.CfdError
    for grads in ([], [c(4), c(4, dt=torch.bfloat16)], [c(4, dt=torch.float64)], [c(4, 4).t()[1:]], [torch.zeros(4)]):
        with pytest.raises(bad):
            ops.grad_norm(grads, 1.0)
    for m in (0.0, -1.0, float("nan")):
        with pytest.raises(bad):
            ops.grad_norm([c(4)], m)
    p = c(8)
    for kw in (dict(state_bits=16), dict(beta_1=1.0), dict(beta_2=-0.1), dict(epsilon=-1.0), dict(weight_decay=[0.1, 0.2]),
               dict(copies=[c(7, dt=torch.bfloat16)]), dict(lr=torch.zeros(1))):
        with pytest.raises(ValueError):
            trainer.AdamW([p], **kw)
    with pytest.raises(ValueError):
        trainer.AdamW([])
    with pytest.raises(ValueError):
        trainer.AdamW([p, p])                             # the same tensor twice
    with pytest.raises(ValueError):
        trainer.AdamW([p[:5], p[4:]])
    with pytest.raises(ValueError):
        trainer.AdamW([c(8, dt=torch.bfloat16)], copies=[c(8, dt=torch.bfloat16)])
    with pytest.raises(bad):
        trainer.AdamW([c(4, 4).t()])
    opt = trainer.AdamW([p])
    for g in ([], [c(7)], [c(8), c(8)]):
        with pytest.raises(ValueError):
            opt.step(g)
    with pytest.raises(bad):
        opt.step([c(8, dt=torch.float16)])
    for s in (c(2), torch.zeros(1), c(1, dt=torch.float64)):
        with pytest.raises(ValueError):
            opt.step([c(8)], s)
    p.data = c(8)
    with pytest.raises(RuntimeError):
        opt.step([c(8)])
    assert int(opt.t) == 0


@pytest.mark.parametrize("bits", [32, 8])
def test_refuses_a_replaced_state(bits):
    """a checkpoint is copied into the state; another tensor in its place, or a learning rate that the kernel cannot read, is refused"""
    from cfd_amd import trainer
    for name in ("m", "v", "t") + (("m_scale", "v_scale") if bits == 8 else ()):
        opt = trainer.AdamW([torch.zeros(300, device="cuda")], state_bits=bits)
        setattr(opt, name, getattr(opt, name).clone())
        with pytest.raises(RuntimeError):
            opt.step([torch.ones(300, device="cuda")])
    opt = trainer.AdamW([torch.zeros(300, device="cuda")], state_bits=bits)
    for lr in (torch.zeros(1), torch.zeros(1, dtype=torch.float64, device="cuda"), torch.zeros(2, device="cuda")):
        opt.lr = lr
        with pytest.raises(ValueError):
            opt.step([torch.ones(300, device="cuda")])
    assert int(opt.t) == 0


def test_regressor_step_on_its_parameter_store():
    """the regressor's own forward and backward, its parameters and gradients as views of the flat buffers, clipped AdamW with an 8-bit
    state writing master and compute copy, then the trained wide layer in 4 bits beside the bf16 one"""
    from oracle import mxfp4 as OM
    from cfd_amd import nets, ops, trainer
    net = nets.CnnRegressor((16, 64, 1), dtype=torch.bfloat16, seed=5)
    P = net.params
    P.enable_training()
    names = [n for n, s in P.specs.items() if s.kind != "stat"]
    wd = [0.004 if n.endswith("kernel") else 0.0 for n in names]
    opt = trainer.AdamW([P.m(n) for n in names], copies=[P.c(n) for n in names], weight_decay=wd, state_bits=8, **HYPER)
    gen = torch.Generator().manual_seed(2)
    x, target = torch.randn(4, 16, 64, 1, generator=gen).cuda(), torch.randn(4, 1, generator=gen).cuda()
    for step in range(3):
        P.zero_grad()
        y = net.forward(x, training=True, seed=step)
        dy, loss = torch.empty_like(y), torch.zeros(1, device="cuda")
        ops.field_loss(y, target, ops.MSE, loss, dout=dy)
        net.backward(dy, x, seed=step)
        grads = [P.g(n) for n in names]
        norm = ops.grad_norm(grads, 0.1)
        want = O.grad_norm([_f64(g) for g in grads], 0.1)
        assert abs(float(norm[0]) - want[0]) <= 2.0 ** -23 * want[0]
        _check_step(opt, grads, float(norm[1]), HYPER["lr"], wd)
        P.refresh_transposed()
    feats = torch.relu(torch.randn(3, P.c("fc1.kernel").shape[1], generator=gen)).to(torch.bfloat16).cuda()
    w4 = ops.mxfp4_quantize(P.c("fc1.kernel"))
    y4 = ops.mxfp4_dense(feats, w4, bias=P.m("fc1.bias"), act=ops.ACT_RELU, out_dtype=torch.float32)
    w64 = OM.round_trip(_f64(P.c("fc1.kernel")))
    ref = np.maximum(_f64(feats) @ w64.T + _f64(P.m("fc1.bias")), 0)
    mag = _f64(feats) @ np.abs(w64).T + 1.0
    assert (np.abs(_f64(y4) - ref) <= (w64.shape[1] / 32 + 64) * 2.0 ** -23 * mag).all()
    y16 = ops.conv_forward(feats, P.c("fc1.kernel"), P.m("fc1.bias"), ops.DENSE, 256, act=ops.ACT_RELU, out_dtype=torch.float32)
    # the two layers differ by what the weights lost, and by fp32 sums
    off = _f64(feats) @ np.abs(w64 - _f64(P.c("fc1.kernel"))).T
    assert (np.abs(_f64(y4) - _f64(y16)) <= off * 1.01 + 8192 / 32 * 2.0 ** -23 * mag).all()
