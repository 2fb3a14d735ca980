"""4-bit matrices and the Dense layer on them where values, views and types meet their ends."""
import pytest
import torch

from tests.test_mxfp4_gpu import O, _np, _same

pytestmark = pytest.mark.gpu


def test_quantize_special_blocks_bf16():
    """ties and borders at several scales, subnormals, zeros, infinities and NaN: bf16 blocks are examined as they lie in memory,
    on ragged tiles and on whole ones"""
    from cfd_amd import ops
    rows = []
    top = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 6.96875, 0.2490234375, 0.251953125, 4.96875, 5.03125, -5.0, -0.0])
    for e in (-126, -40, 0, 3, 100, 124):
        for biggest in (4.0, 6.0, 7.0, 7.03125):                # (7.03125: the next one over 7)
            rows.append(torch.cat([top.clamp(-biggest, biggest), torch.full((15,), 0.30078125), torch.tensor([biggest])]) * 2.0 ** e)
    rows += [torch.zeros(32), torch.full((32,), -0.0), torch.full((32,), 2.0 ** -133), torch.linspace(-1.1e-38, 1.1e-38, 32),
             torch.full((32,), 3.3895313892515355e38)]
    for bad in (float("inf"), -float("inf"), float("nan")):
        rows.append(torch.arange(32.0))
        rows[-1][7] = bad
    x = torch.stack(rows).to(torch.bfloat16).cuda()
    assert int((x[26] != 0).sum()) == 32                        # (2^-133 is bf16's smallest subnormal)
    tile = torch.cat([x.roll(5 * i, 0) for i in range(4)], 1).repeat(8, 1)[:256]      # 256 x 128: two whole tiles
    for a in (x, tile, tile[:129], torch.cat([tile, tile[:, :40]], 1)):
        q, t = ops.mxfp4_quantize_both(a)
        _same(q, a), _same(t, a.t())
        _same(ops.mxfp4_quantize(a), a)
        _same(ops.mxfp4_quantize(a, transpose=True), a.t())
        _same(ops.mxfp4_quantize(a.t().contiguous(), transpose=True), a)
    v = torch.from_numpy(O.round_trip(_np(x))).to(torch.bfloat16)
    assert torch.equal(torch.nan_to_num(ops.mxfp4_dequantize(ops.mxfp4_quantize(x), torch.bfloat16).cpu()), torch.nan_to_num(v))


@pytest.mark.parametrize("m,n,k,x_four", [(5, 20, 64, False), (2, 30, 40000, False), (20, 30, 64, True), (8, 8, 40000, True),
                                          (1800, 1700, 96, True), (260, 250, 65536, True)])
def test_activations_of_infinite_sums(m, n, k, x_four):
    """ReLU of a sum of -infinity is 0, of NaN is NaN, in every epilogue: tiles of 16, 64 and 256 rows, with and without slices of K"""
    from cfd_amd import ops
    x, w = torch.zeros(m, k, device="cuda"), torch.zeros(n, k, device="cuda")
    if x_four:                 # products of 2^254
        x[:, 3] = 2.0 ** 127 * torch.tensor([1.0, -1.0], device="cuda").repeat(m)[:m]
        x[m - 1, 3] = float("nan")
        w[:, 3] = 2.0 ** 127 * torch.tensor([1.0, -1.0, 0.0], device="cuda").repeat(n)[:n]
    else:
        x[:, 3] = torch.tensor([float("inf"), -float("inf"), 1.0, float("nan")], device="cuda").repeat(m)[:m]
        w[:, 3] = torch.tensor([1.0, -1.0, 0.0], device="cuda").repeat(n)[:n]
    z = x[:, 3, None] * w[None, :, 3]
    assert torch.isinf(z).any() and (z == -float("inf")).any()
    a, b = ops.mxfp4_quantize(x) if x_four else x, ops.mxfp4_quantize(w)
    bias = torch.ones(n, device="cuda")
    for out_dtype in (torch.float32, torch.bfloat16):
        for act, want in ((ops.ACT_RELU, torch.relu(z + 1)), (ops.ACT_LEAKY, torch.nn.functional.leaky_relu(z + 1, 0.2)),
                          (ops.ACT_NONE, z + 1), (ops.ACT_SIGMOID, torch.sigmoid(z + 1))):
            y = ops.mxfp4_dense(a, b, bias=bias, act=act, out_dtype=out_dtype).float()
            tol = 2.0 ** -8 if out_dtype == torch.bfloat16 else 2.0 ** -20
            same = (y == want) | (torch.isnan(y) & torch.isnan(want)) | ((y - want).abs() <= tol)     # (|finite values| <= 2)
            assert same.all(), (out_dtype, act, y[~same][:4], want[~same][:4])
    y = ops.mxfp4_dense(a, b, act=ops.ACT_RELU)                                                       # no bias
    assert torch.equal(torch.isnan(y), torch.isnan(z)) and torch.equal(torch.nan_to_num(y), torch.nan_to_num(torch.relu(z)))


@pytest.mark.parametrize("cols", [64, 63, 33])
def test_from_parts_keeps_a_copy(cols):
    """the matrix does not follow its parts, whether or not its last block is whole"""
    from cfd_amd import ops
    codes = torch.randint(0, 256, (6, 32), dtype=torch.uint8, generator=torch.Generator().manual_seed(1)).cuda()
    scales = torch.full((6, 2), 127, dtype=torch.uint8, device="cuda")
    q = ops.mxfp4_from_parts(codes, scales, cols)
    want = ops.mxfp4_dequantize(q)
    codes.fill_(0x77), scales.fill_(120)
    assert torch.equal(ops.mxfp4_dequantize(q), want)


def test_an_output_over_an_operand_is_refused():
    """a tile would read a bias, codes or scales that another has written; beside them, in one buffer, is allowed"""
    from cfd_amd import _lib, ops
    n, k = 24, 40
    wq, x = ops.mxfp4_quantize(torch.randn(n, k, generator=torch.Generator().manual_seed(1)).cuda()), torch.ones(6, k, device="cuda")
    buf = torch.zeros(6, 64, device="cuda")
    bias = torch.arange(float(n), device="cuda")
    out = buf[:, :n]
    for a in (x, ops.mxfp4_quantize(x)):
        for over in (buf[2, :n], buf[5, 20:44], buf[0, n - 1:2 * n - 1], buf.view(-1)):
            with pytest.raises(_lib.CfdError):
                ops.mxfp4_dense(a, wq, bias=over, out=out)
        assert not buf.any()
        buf[3, n:2 * n] = bias
        assert torch.equal(ops.mxfp4_dense(a, wq, bias=buf[3, n:2 * n], out=out), ops.mxfp4_dense(a, wq, bias=bias))
        buf.zero_()
    # a 4-bit matrix inside the output's bytes: its codes or its scales alone, on either side and in the decoding
    room = torch.zeros(64 * 64, device="cuda").view(torch.uint8)
    q = ops.mxfp4_quantize(torch.ones(n, k, device="cuda"))
    for name in ("codes", "scales"):
        part = getattr(q, name)
        inside = room[:part.numel()].view(part.shape)
        inside.copy_(part)
        over = q._replace(**{name: inside})
        y = room.view(torch.float32)
        for call in (lambda: ops.mxfp4_dense(x, over, out=y[:6 * n].view(6, n)), lambda: ops.mxfp4_dense(over, over, out=y[:n * n].view(n, n)),
                     lambda: ops.mxfp4_dense(over, q, out=y[:n * n].view(n, n)), lambda: ops.mxfp4_dequantize(over, out=y[:n * k].view(n, k))):
            with pytest.raises(_lib.CfdError):
                call()
        assert torch.equal(inside, part)
