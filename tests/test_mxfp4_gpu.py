"""4-bit microscaled matrices and the Dense layer on them, on the GPU, against the 64-bit restatement.

Quantisation and decoding are exact.  A product of decoded values is exact in fp32, so an output is off by its sum alone: at
most one fp32 rounding (2^-24 of the sum of magnitudes; matrix instructions may truncate: 2^-23) for every addition on the
way -- K / 32 of them per element and chain, plus slices and the epilogue -- and 2^-8 of the value where it is stored as bf16."""
import numpy as np
import pytest
import torch

from oracle import mxfp4 as O

pytestmark = pytest.mark.gpu


def _np(t):
    return t.detach().float().cpu().numpy().astype(np.float64)


def _rnd(r, c, seed, dtype=torch.float32, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(r, c, generator=g) * torch.exp(spread * torch.randn(r, 1, generator=g))
    x[torch.rand(r, c, generator=g) < 0.05] = 0.0
    return x.to(dtype)


def _same(q, x):
    """an Mxfp4 matrix holds exactly the oracle's codes and scales of x (R, C), zeros behind them"""
    codes, scales = O.quantize(_np(x))
    assert q.shape == tuple(x.shape)
    assert np.array_equal(q.codes.cpu().numpy(), O.pack(codes))
    got = q.scales.cpu().numpy()
    assert np.array_equal(got[:, :scales.shape[1]], scales) and not got[:, scales.shape[1]:].any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(1, 1), (1, 31), (3, 32), (5, 33), (1, 4096), (130, 70), (257, 1000), (64, 4100), (1000, 7), (33, 513)])
def test_quantize(shape, dtype):
    from cfd_amd import ops
    x = _rnd(*shape, 1, dtype).cuda()
    _same(ops.mxfp4_quantize(x), x)
    q, t = ops.mxfp4_quantize_both(x)
    _same(q, x)
    _same(t, x.t())
    _same(ops.mxfp4_quantize(x, transpose=True), x.t())
    wide = torch.full((shape[0], shape[1] + 5), float("nan"), dtype=dtype, device="cuda")      # a slice of a wider buffer
    wide[:, 3:3 + shape[1]] = x
    q, t = ops.mxfp4_quantize_both(wide[:, 3:3 + shape[1]])
    _same(q, x)
    _same(t, x.t())
    _same(ops.mxfp4_quantize(wide[:, 3:3 + shape[1]]), x)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(128, 128), (128, 640), (400, 384), (256, 512), (640, 128)])
def test_quantize_both_in_whole_tiles(shape, dtype):
    """matrices that end with a 128-column tile: scales behind the last block are zero, a NaN stays in its two blocks"""
    from cfd_amd import ops
    x = _rnd(*shape, 2, dtype).cuda()
    x[127, 127] = float("nan")
    q, t = ops.mxfp4_quantize_both(x)
    _same(q, x)
    _same(t, x.t())


def test_quantize_special_blocks():
    from cfd_amd import ops
    rows = []
    top = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 6.999, 0.249, 0.251, 4.999, 5.001, -5.0, -0.0])
    for e in (-126, -40, 0, 3, 100, 124):                      # ties and borders at several scales
        for biggest in (4.0, 6.0, 7.0, 7.0000005):
            rows.append(torch.cat([top.clamp(-biggest, biggest), torch.full((15,), 0.3), torch.tensor([biggest])]) * 2.0 ** e)
    rows.append(torch.zeros(32))
    rows.append(torch.full((32,), -0.0))
    rows.append(torch.full((32,), 1e-45))                      # subnormal blocks
    rows.append(torch.linspace(-1.1e-38, 1.1e-38, 32))
    rows.append(torch.full((32,), 3.4028234663852886e38))
    x = torch.stack(rows).float()
    for bad in (float("inf"), -float("inf"), float("nan")):
        b = torch.arange(32.0)
        b[7] = bad
        x = torch.cat([x, b[None]])
    x = x.cuda()
    _same(ops.mxfp4_quantize(x), x)
    _same(ops.mxfp4_quantize(x.t().contiguous(), transpose=True), x)
    got = ops.mxfp4_dequantize(ops.mxfp4_quantize(x)).cpu().double().numpy()
    with np.errstate(over="ignore"):
        want = O.round_trip(_np(x)).astype(np.float32).astype(np.float64)
    assert np.array_equal(got, want, equal_nan=True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_dequantize_every_code_and_scale(dtype):
    from cfd_amd import ops
    codes = np.tile(np.arange(16, dtype=np.uint8), (256, 2))
    scales = np.arange(256, dtype=np.uint8)[:, None]
    q = ops.mxfp4_from_parts(torch.from_numpy(O.pack(codes)).cuda(), torch.from_numpy(scales).cuda(), 32)
    want = torch.from_numpy(O.values(codes, scales, 32)).to(dtype)
    got = ops.mxfp4_dequantize(q, dtype).cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got.double(), posinf=1e300, neginf=-1e300), torch.nan_to_num(want.double(), posinf=1e300, neginf=-1e300))
    odd = ops.mxfp4_quantize(_rnd(7, 45, 3).cuda())
    buf = torch.full((7, 50), 9.0, dtype=dtype, device="cuda")
    ops.mxfp4_dequantize(odd, out=buf[:, 2:47])
    assert (buf[:, :2] == 9).all() and (buf[:, 47:] == 9).all()
    assert torch.equal(buf[:, 2:47], ops.mxfp4_dequantize(odd, dtype))


def _act(z, act):
    return {0: z, 1: np.where(z > 0, z, 0.2 * z), 2: np.maximum(z, 0), 3: 1 / (1 + np.exp(-z))}[act]


def _close(y, x64, w64, bias, act):
    z = x64 @ w64.T + (0 if bias is None else _np(bias))
    mag = np.abs(x64) @ np.abs(w64).T + (0 if bias is None else np.abs(_np(bias)))
    k = x64.shape[1]
    tol = (3 * k / 32 + 64) * 2.0 ** -23 * mag + 1e-37
    if act == 3:
        tol = tol + 1e-6
    want = _act(z, act)
    if y.dtype == torch.bfloat16:
        tol = tol * 1.01 + 2.0 ** -8 * np.abs(want)
    assert (np.abs(_np(y) - want) <= tol).all(), float((np.abs(_np(y) - want) / tol).max())


SHAPES = [(1, 1, 32), (1, 1, 1), (5, 3, 31), (16, 16, 128), (64, 64, 256), (65, 63, 257), (100, 130, 1000), (17, 200, 4100),
          (128, 256, 16384), (300, 70, 96), (513, 260, 520), (1, 128, 256), (260, 1, 300), (256, 256, 512), (700, 1030, 2080)]
#: the 256 x 256 tiles: whole and ragged, odd columns (16-bit stores), a K that ends inside a group, slices of K
LARGE = [(1800, 1700, 100), (2048, 1536, 512), (1999, 1537, 515), (260, 250, 65536)]


@pytest.mark.parametrize("m,n,k", SHAPES + LARGE)
def test_dense_four_bit_operands(m, n, k):
    from cfd_amd import ops
    x, w = _rnd(m, k, 11, spread=1.0).cuda(), _rnd(n, k, 12, spread=1.0).cuda()
    bias = torch.randn(n, generator=torch.Generator().manual_seed(13)).cuda()
    xq, wq = ops.mxfp4_quantize(x), ops.mxfp4_quantize(w)
    x64, w64 = O.round_trip(_np(x)), O.round_trip(_np(w))
    _close(ops.mxfp4_dense(xq, wq), x64, w64, None, 0)
    for act in (0, 1, 2, 3):
        _close(ops.mxfp4_dense(xq, wq, bias=bias, act=act, out_dtype=torch.bfloat16), x64, w64, bias, act)
    buf = torch.full((m, n + 7), 5.0, device="cuda")
    ops.mxfp4_dense(xq, wq, bias=bias, act=2, out=buf[:, 3:3 + n])
    _close(buf[:, 3:3 + n], x64, w64, bias, 2)
    assert (buf[:, :3] == 5).all() and (buf[:, 3 + n:] == 5).all()
    again = ops.mxfp4_dense(xq, wq)
    assert torch.equal(again, ops.mxfp4_dense(xq, wq))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,n,k", SHAPES + [(2, 256, 65536), (33, 40, 777)])
def test_dense_float_activations(m, n, k, dtype):
    from cfd_amd import ops
    x, w = _rnd(m, k, 21, dtype, 1.0).cuda(), _rnd(n, k, 22, spread=1.0).cuda()
    bias = torch.randn(n, generator=torch.Generator().manual_seed(23)).cuda()
    wq = ops.mxfp4_quantize(w)
    w64 = O.round_trip(_np(w))
    y = ops.mxfp4_dense(x, wq, out_dtype=torch.float32)
    _close(y, _np(x), w64, None, 0)
    assert ops.mxfp4_dense(x, wq).dtype == dtype
    for act in (0, 1, 2, 3):
        _close(ops.mxfp4_dense(x, wq, bias=bias, act=act, out_dtype=torch.bfloat16), _np(x), w64, bias, act)
    wide = torch.full((m, k + 3), float("nan"), dtype=dtype, device="cuda")
    wide[:, 1:1 + k] = x
    assert torch.equal(ops.mxfp4_dense(wide[:, 1:1 + k], wq, out_dtype=torch.float32), y)


@pytest.mark.parametrize("m,n,k,dtype", [(48, 60, 300000, torch.bfloat16), (16, 100, 140000, torch.float32), (16, 1030, 17000, torch.float32),
                                         (1, 1030, 17000, torch.float32), (1, 40000, 9000, torch.float32), (49, 200, 5000, torch.bfloat16),
                                         (2, 1030, 2040, torch.float32), (5, 300, 1000, torch.float32), (16, 70, 900, torch.bfloat16), (6, 70, 1900, torch.bfloat16)])
def test_dense_float_activations_shared_between_waves(m, n, k, dtype):
    """one, two and four waves on a weight tile, one and several K groups each, and rows in more than one tile"""
    from cfd_amd import ops
    x, w = _rnd(m, k, 91, dtype, 0.5).cuda(), ops.mxfp4_quantize(_rnd(n, k, 92, spread=0.5).cuda())
    w64 = _np(ops.mxfp4_dequantize(w))
    y = ops.mxfp4_dense(x, w, out_dtype=torch.float32)
    _close(y, _np(x), w64, None, 0)
    assert torch.equal(y, ops.mxfp4_dense(x, w, out_dtype=torch.float32))


def test_dense_float_activations_at_the_ends_of_the_range():
    """activations that a bf16 rounding would push to infinity, infinities and NaN: only the rows that hold them change"""
    from cfd_amd import ops
    w = torch.ones(20, 64, device="cuda")
    x = torch.zeros(5, 64, device="cuda")
    x[0, 3] = 3.4028234663852886e38
    x[1, 3] = float("inf")
    x[2, 3] = float("nan")
    x[3, 3] = 1.0 + 2.0 ** -23
    y = ops.mxfp4_dense(x, ops.mxfp4_quantize(w))
    assert (y[0] == x[0, 3]).all() and (y[1] == float("inf")).all() and torch.isnan(y[2]).all()
    assert (y[3] == x[3, 3]).all() and (y[4] == 0).all()


def test_dense_nan_blocks_reach_their_row_or_column_only():
    from cfd_amd import ops
    for x_four in (True, False):
        x, w = _rnd(70, 600, 31, spread=0.0).cuda(), _rnd(90, 600, 32, spread=0.0).cuda()
        x[5, 599] = float("nan")
        w[80, 0] = float("inf")
        y = ops.mxfp4_dense(ops.mxfp4_quantize(x) if x_four else x, ops.mxfp4_quantize(w))
        bad = torch.isnan(y)
        want = torch.zeros_like(bad)
        want[5], want[:, 80] = True, True
        assert torch.equal(bad, want)


@pytest.mark.parametrize("m,n,k", [(20, 70, 608), (1750, 1720, 96)])
def test_dense_scales_at_the_ends_of_their_range(m, n, k):
    """2^127 on one operand and 2^-127 on the other: the product is of order one, whichever side's values are subnormal"""
    from cfd_amd import ops
    r = np.random.default_rng(7)
    cx, cw = r.integers(0, 16, (m, k), dtype=np.uint8), r.integers(0, 16, (n, k), dtype=np.uint8)
    for bx, bw in ((254, 0), (0, 254), (127, 127)):
        sx, sw = np.full((m, (k + 31) // 32), bx, np.uint8), np.full((n, (k + 31) // 32), bw, np.uint8)
        xq, wq = (ops.mxfp4_from_parts(torch.from_numpy(O.pack(c)).cuda(), torch.from_numpy(s).cuda(), k) for c, s in ((cx, sx), (cw, sw)))
        _close(ops.mxfp4_dense(xq, wq), O.values(cx, sx, k), O.values(cw, sw, k), None, 0)
    sw = np.zeros((n, (k + 31) // 32), np.uint8)
    wq = ops.mxfp4_from_parts(torch.from_numpy(O.pack(cw)).cuda(), torch.from_numpy(sw).cuda(), k)
    x = (torch.randn(20, k, generator=torch.Generator().manual_seed(8)) * 2.0 ** 124).cuda()
    for t in (x, x.bfloat16()):
        _close(ops.mxfp4_dense(t, wq, out_dtype=torch.float32), _np(t), O.values(cw, sw, k), None, 0)


def test_dense_output_beside_its_activations():
    """columns of one buffer: the output's next to the activations' is a concat in place, over them is refused"""
    from cfd_amd import _lib, ops
    w = ops.mxfp4_quantize(_rnd(24, 40, 71, spread=0.0).cuda())
    buf = torch.zeros(6, 64, device="cuda")
    buf[:, :40] = _rnd(6, 40, 72, spread=0.0).cuda()
    want = ops.mxfp4_dense(buf[:, :40].contiguous(), w)
    kept = buf[:, :40].clone()
    ops.mxfp4_dense(buf[:, :40], w, out=buf[:, 40:])
    assert torch.equal(buf[:, 40:], want) and torch.equal(buf[:, :40], kept)
    for out in (buf[:, 39:63], buf[:, :24], buf.view(-1)[:144].view(6, 24)):
        with pytest.raises(_lib.CfdError):
            ops.mxfp4_dense(buf[:, :40], w, out=out)


@pytest.mark.parametrize("m,n,k", [(65, 63, 257), (3, 129, 600), (1999, 1537, 515), (260, 250, 65536), (2048, 1536, 512)])
def test_nothing_behind_the_last_row_is_written(m, n, k):
    from cfd_amd import _lib, ops
    lib, st = _lib.load(), torch.cuda.current_stream().cuda_stream
    x, w = _rnd(m, k, 81, spread=0.5).cuda(), ops.mxfp4_quantize(_rnd(n, k, 82, spread=0.5).cuda())
    xq = ops.mxfp4_quantize(x)
    for dtype in (torch.float32, torch.bfloat16):
        for a in (xq, x[:40]):
            rows = a.shape[0]
            buf = torch.full((rows + 3, n + n % 2), 5.0, dtype=dtype, device="cuda")
            ops.mxfp4_dense(a, w, out=buf[:rows, :n])
            assert torch.equal(buf[:rows, :n], ops.mxfp4_dense(a, w, out_dtype=dtype))
            assert (buf[rows:] == 5).all() and (buf[:, n:] == 5).all()
        buf = torch.full((m + 2, k), 5.0, dtype=dtype, device="cuda")
        ops.mxfp4_dequantize(xq, out=buf[:m])
        assert (buf[m:] == 5).all()
        xd = x.to(dtype)
        q, t = ops.mxfp4_quantize_both(xd)
        ends = []
        for part in (q.codes, q.scales, t.codes, t.scales):       # each array with 4 KiB behind it
            ends.append(torch.full((part.numel() + 4096,), 77, dtype=torch.uint8, device="cuda"))
        for ptrs in ([e.data_ptr() for e in ends], [ends[0].data_ptr(), ends[1].data_ptr(), None, None], [None, None, ends[2].data_ptr(), ends[3].data_ptr()]):
            _lib.check(lib.cfd_mxfp4_quantize(xd.data_ptr(), k, ops._DT[dtype], m, k, *ptrs, st), "cfd_mxfp4_quantize")
            for e, part, p in zip(ends, (q.codes, q.scales, t.codes, t.scales), ptrs):
                if p is not None:
                    assert torch.equal(e[:part.numel()], part.view(-1))
                assert (e[part.numel():] == 77).all()


def test_empty():
    from cfd_amd import ops
    w = ops.mxfp4_quantize(torch.ones(4, 40, device="cuda"))
    e = torch.zeros(0, 40, device="cuda")
    assert ops.mxfp4_dense(e, w).shape == (0, 4) and ops.mxfp4_dense(ops.mxfp4_quantize(e), w).shape == (0, 4)
    assert ops.mxfp4_dense(torch.ones(3, 40, device="cuda"), ops.mxfp4_quantize(e)).shape == (3, 0)
    assert ops.mxfp4_dequantize(ops.mxfp4_quantize(e)).shape == (0, 40)


def test_from_parts_clears_what_lies_past_the_columns():
    from cfd_amd import ops
    codes = torch.randint(0, 256, (6, 32), dtype=torch.uint8, generator=torch.Generator().manual_seed(1)).cuda()
    scales = torch.full((6, 2), 127, dtype=torch.uint8, device="cuda")
    for cols in (64, 63, 50, 33):
        q = ops.mxfp4_from_parts(codes, scales, cols)
        v = O.values(O.unpack(codes.cpu().numpy()), scales.cpu().numpy(), cols)
        assert np.array_equal(_np(ops.mxfp4_dequantize(q)), v)
        assert not O.unpack(q.codes.cpu().numpy())[:, cols:].any()


def test_gradients_of_dense_against_differences():
    """y = x w^T on what the 4-bit operands hold is linear in each: <dy, y(x + h) - y(x)> = <dx, h> exactly in 64 bits; the kernel's
    gradients equal the formula's on the quantised dy within the product's tolerance"""
    from cfd_amd import ops
    m, n, k = 96, 160, 224
    x, w, dy = _rnd(m, k, 41, spread=0.5).cuda(), _rnd(n, k, 42, spread=0.5).cuda(), _rnd(m, n, 43, spread=0.5).cuda()
    (xq, xt), (wq, wt), (dq, dt) = (ops.mxfp4_quantize_both(t) for t in (x, w, dy))
    dx, dw = ops.mxfp4_dense(dq, wt), ops.mxfp4_dense(dt, xt)
    dy_r, dy_c, w_c, x_c = O.round_trip(_np(dy)), O.round_trip(_np(dy).T), O.round_trip(_np(w).T), O.round_trip(_np(x).T)
    _close(dx, dy_r, w_c, None, 0)
    _close(dw, dy_c, x_c, None, 0)
    h = np.random.default_rng(0).standard_normal((m, k))
    f = lambda a: float((dy_r * (a @ w_c)).sum())  # noqa: E731
    base = O.round_trip(_np(x))
    num = (f(base + h) - f(base - h)) / 2
    assert abs(num - float((_np(dx) * h).sum())) <= 1e-5 * float((np.abs(_np(dx)) * np.abs(h)).sum())


@pytest.mark.parametrize("x_four", [True, False])
def test_dense_in_a_captured_graph(x_four):
    """two graphs of one layer, replayed in turn with eager calls between: each equals the eager result"""
    from cfd_amd import ops
    w = ops.mxfp4_quantize(_rnd(256, 8192, 51, spread=0.5).cuda())
    xs = [_rnd(m, 8192, 52, spread=0.5).cuda() for m in (3, 40)]
    call = lambda x: ops.mxfp4_dense(ops.mxfp4_quantize(x) if x_four else x, w, act=1)  # noqa: E731
    graphs, outs = [], []
    for x in xs:
        call(x)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(x))
        graphs.append(g)
    for i in range(4):
        for x in xs:
            x.mul_(0.5).add_(0.1 * i)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for x, y in zip(xs, outs):
            assert torch.equal(y, call(x))


def test_train_a_wide_dense_head():
    """the operators together, as a training program uses them: 4-bit products forward and backward, clipped AdamW with
    an 8-bit state, then the trained weights served in 4 bits.  Every stage is checked against the 64-bit formulas on its own inputs."""
    from oracle import optim as OP
    from cfd_amd import ops, trainer
    m, n, k = 48, 64, 2048
    gen = torch.Generator().manual_seed(61)
    w = (torch.randn(n, k, generator=gen) / k ** 0.5).cuda()
    bias = torch.zeros(n, device="cuda")
    x, target = torch.relu(torch.randn(m, k, generator=gen)).cuda(), torch.randn(m, n, generator=gen).cuda()
    opt = trainer.AdamW([w, bias], lr=1e-3, weight_decay=[0.01, 0.0], state_bits=8, seed=9)
    for step in range(4):
        (xq, xt), wq = ops.mxfp4_quantize_both(x), ops.mxfp4_quantize(w)
        y = ops.mxfp4_dense(xq, wq, bias=bias)
        _close(y, O.round_trip(_np(x)), O.round_trip(_np(w)), bias, 0)
        dy = (y - target) * (2.0 / y.numel())
        dw, db = ops.mxfp4_dense(ops.mxfp4_quantize(dy, transpose=True), xt), torch.zeros(n, device="cuda")
        ops.colsum(dy, db)
        _close(dw, O.round_trip(_np(dy).T), O.round_trip(_np(x).T), None, 0)
        norm = ops.grad_norm([dw, db], 0.05)
        want = OP.grad_norm([_np(dw), _np(db)], 0.05)
        assert abs(float(norm[0]) - want[0]) <= 2.0 ** -23 * want[0]
        before = [_np(t) for t in (w, bias)]
        opt.step([dw, db], norm[1:])
        if step == 0:            # zero state: the first step moves each weight by lr at most, towards minus its gradient
            for t, b, g, wd in zip((w, bias), before, (dw, db), (0.01, 0.0)):
                p64, _, _ = OP.adamw(b, _np(g), 0 * b, 0 * b, 1, 1e-3, 0.9, 0.999, 1e-7, wd, float(norm[1]))
                assert np.abs(_np(t) - p64).max() <= 2.0 ** -21 * (np.abs(p64).max() + 1e-3)
    served = ops.mxfp4_dense(x[:1], ops.mxfp4_quantize(w), bias=bias, act=ops.ACT_RELU)
    _close(served, _np(x[:1]), O.round_trip(_np(w)), bias, 2)


def test_matrices_past_32_bits():
    """more than 2^32 bytes of codes and 2^33 values: the last rows are quantised, decoded and multiplied like a short matrix's"""
    from cfd_amd import ops
    rows, k = 66000, 131072
    x = torch.empty(rows, k, dtype=torch.bfloat16, device="cuda").normal_(generator=torch.Generator(device="cuda").manual_seed(1))
    q, last = ops.mxfp4_quantize(x), ops.mxfp4_quantize(x[-100:])
    assert q.codes.numel() > 1 << 32
    assert torch.equal(q.codes[-100:], last.codes) and torch.equal(q.scales[-100:], last.scales)
    a = torch.relu(x[:3]).float()
    del x
    y, z = ops.mxfp4_dense(a, q), ops.mxfp4_dense(a, last)
    tol = 64 * 2.0 ** -23 * k ** 0.5 * float(z.abs().max())     # (the K slices differ: other orders of the same fp32 sums)
    assert (y[:, -100:] - z).abs().max() <= tol
    aq = ops.mxfp4_quantize(a)
    assert (ops.mxfp4_dense(aq, q)[:, -100:] - ops.mxfp4_dense(aq, last)).abs().max() <= tol
    a4 = ops.mxfp4_quantize(a.repeat(100, 1))                   # 300 rows: the 256 x 256 tiles
    assert (ops.mxfp4_dense(a4, q)[:3, -100:] - ops.mxfp4_dense(aq, last)).abs().max() <= tol
    del y, z
    v = ops.mxfp4_dequantize(q, torch.bfloat16)
    assert torch.equal(v[-100:], ops.mxfp4_dequantize(last, torch.bfloat16))


def test_refusals():
    from cfd_amd import _lib, ops
    bad = pytest.raises(_lib.CfdError)
    c = lambda *s, dt=torch.float32: torch.zeros(*s, dtype=dt, device="cuda")  # noqa: E731
    for x in (c(4), c(2, 3, 4), c(2, 3, dt=torch.float16), c(4, 0), c(8, 8).t(), c(8)[None].expand(3, 8), torch.zeros(2, 3)):
        with bad:
            ops.mxfp4_quantize(x)
    with bad:
        ops.mxfp4_quantize(c(0, 4), transpose=True)
    q = ops.mxfp4_quantize(c(4, 40))
    for args in ((q, ops.mxfp4_quantize(c(3, 41))), (c(4, 41), q), (c(4, 40, dt=torch.float16), q), (c(4, 40), c(3, 40)),
                 (torch.zeros(4, 40), q), (q, ops.Mxfp4(q.codes[:, :16], q.scales, 40)), (q, ops.Mxfp4(q.codes, q.scales[:, :2], 40)),
                 (q, ops.Mxfp4(q.codes.cpu(), q.scales.cpu(), 40))):
        with bad:
            ops.mxfp4_dense(*args)
    for kw in (dict(bias=c(3)), dict(bias=c(4, dt=torch.bfloat16)), dict(out=c(4, 5)), dict(out=c(4, 4, dt=torch.bfloat16), out_dtype=torch.float32),
               dict(out=c(4, 4).t()[:, :4].t().t()), dict(out_dtype=torch.float16), dict(act=7)):
        with bad:
            ops.mxfp4_dense(q, q, **kw)
    with bad:
        ops.mxfp4_dequantize(q, out=c(4, 41))
    with bad:
        ops.mxfp4_dequantize(q, torch.float16)
    with bad:
        ops.mxfp4_from_parts(q.codes, q.scales, 40)
    for cols in (0, -5, 1 << 23):
        with bad:
            ops.mxfp4_from_parts(q.codes, q.scales[:, :2], cols)
