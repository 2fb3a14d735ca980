"""The 4-bit Dense layer on operands whose every partial sum is a whole number of units under 2^24: fp32 holds each of them in
whatever order they are added, so the output has to EQUAL the 64-bit sum.  A K group that is left out, taken twice or put
beside another one's scales shows at any length."""
import ctypes as C

import pytest
import torch

pytestmark = pytest.mark.gpu

#: m, n, k, activations, (waves on a weight tile, rounds over its K groups, is a round ragged, slices of K)
FLOAT = [(1, 28672, 8192, "fp32", (4, 4, False, 1)),
         (1, 28672, 9000, "fp32", (4, 5, True, 1)),
         (1, 16384, 17000, "fp32", (4, 5, True, 2)),
         (3, 20000, 12000, "bf16", (4, 6, False, 1)),
         (1, 256, 262144, "fp32", (4, 1, False, 128)),
         (9, 1030, 8200, "bf16", (4, 1, True, 17)),
         (64, 60, 262144, "fp32", (2, 2, False, 128)),      # four waves' activations would not fit the LDS
         (64, 128, 262144, "fp32", (2, 2, False, 128)),
         (33, 128, 200000, "fp32", (2, 2, True, 131)),
         (64, 100, 262144, "bf16", (2, 1, False, 256)),
         (100, 100, 262144, "bf16", (2, 2, False, 128)),
         (64, 256, 262144, "bf16", (1, 2, False, 256)),
         (64, 256, 262144, "fp32", (1, 4, False, 128)),
         (1, 40000, 9000, "fp32", (1, 6, False, 3))]
#: m, n, k, (tile rows, groups of the longest slice, slices of K); the 64-row tiles' four waves take groups in turn
FOUR = [(128, 256, 262144, (64, 16, 32)),
        (64, 64, 9000, (64, 5, 4)),
        (100, 1000, 20000, (64, 5, 8)),
        (700, 1030, 2080, (64, 5, 1)),
        (260, 250, 65536, (256, 4, 32)),
        (2000, 2000, 40000, (256, 20, 4)),
        (1800, 1700, 1100, (256, 3, 1)),
        (64, 262144, 256, (64, 1, 1)),                      # dx and dw of a 262144 -> 256 layer on 64 and 65 rows
        (256, 262144, 65, (256, 1, 1))]
KINDS = {"fp32": 0, "bf16": 1, "fp4": 2}


def plan(lib, m, n, k, kind):
    """(tile rows, slices of K, K groups a slice, waves that take them in turn)"""
    p = (C.c_int * 4)()
    assert lib.cfd_mxfp4_dense_plan(m, n, k, KINDS[kind], p) == 0
    return tuple(p)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _fp4(rows, k, seed):
    """random codes with scales of 1 and 2 -> (4-bit matrix, its values in fp64): multiples of a half up to 12"""
    from cfd_amd import ops
    g, nb = _gen(seed), (k + 31) // 32
    c = torch.randint(0, 16, (rows, 32 * nb), generator=g, device="cuda", dtype=torch.uint8)
    s = torch.randint(127, 129, (rows, nb), generator=g, device="cuda", dtype=torch.uint8)
    q = ops.mxfp4_from_parts(c[:, 0::2] | (c[:, 1::2] << 4), s, k)
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device="cuda")
    v = torch.cat([grid, -grid])[c.int()].view(rows, nb, 32) * (s.double() - 126)[..., None]      # (1 or 2: 2^(byte - 127))
    return q, v.view(rows, -1)[:, :k]


def _want(x, w, bias, unit):
    """fp64 sums and the check that fp32 holds every partial one"""
    assert float((x.abs() @ w.abs().t()).max() + bias.abs().max()) < 2.0 ** 24 * unit
    return x @ w.t() + bias.double()


@pytest.mark.parametrize("m,n,k,dtype,how", FLOAT)
def test_float_activations(m, n, k, dtype, how):
    from cfd_amd import ops
    w, w64 = _fp4(n, k, 1)
    g = _gen(2)
    x = torch.randint(-3, 4, (m, k), generator=g, device="cuda").float()
    if dtype == "fp32":      # a few values that only three bf16 terms hold
        x[:, torch.randint(0, k, (6,), generator=g, device="cuda")] = 66003.0
    x = x.to(torch.bfloat16 if dtype == "bf16" else torch.float32)
    bias = torch.randint(-9, 10, (n,), generator=g, device="cuda").float()
    want = _want(x.double(), w64, bias, 0.5)
    assert torch.equal(ops.mxfp4_dense(x, w, bias=bias, out_dtype=torch.float32).double(), want)
    assert torch.equal(ops.mxfp4_dense(x, w, bias=bias, act=ops.ACT_RELU, out_dtype=torch.float32).double(), want.clamp(min=0))


@pytest.mark.parametrize("m,n,k,how", FOUR)
def test_four_bit_operands(m, n, k, how):
    from cfd_amd import ops
    (x, x64), (w, w64) = _fp4(m, k, 3), _fp4(n, k, 4)
    bias = torch.randint(-9, 10, (n,), generator=_gen(5), device="cuda").float()
    want = _want(x64, w64, bias, 0.25)
    assert torch.equal(ops.mxfp4_dense(x, w, bias=bias).double(), want)
    y16 = ops.mxfp4_dense(x, w, bias=bias, act=ops.ACT_RELU, out_dtype=torch.bfloat16)
    assert torch.equal(y16, want.clamp(min=0).float().to(torch.bfloat16))     # (exact in fp32: one rounding)
