"""The 4-bit rows and their product through the C ABI against numpy in float64.

Quantisation scales by powers of two and rounds once, so codes, scales and fp32 values are equal bit for bit. A product of two
4-bit numbers is exact in fp32; a sum of K of them in any order is off by at most K * 2^-23 of the sum of magnitudes (each
addition by half a step, 2^-24, or by a whole one where the matrix cores cut), and by nothing where every partial sum is
a whole number below 2^24; an output of fewer bits is rounded once more, by half its step."""
import numpy as np
import pytest
import torch

import mx4_ref as R
from mignon_ai_amd import (MignonError, mx4_dequantize, mx4_dequantize_device, mx4_gemm, mx4_gemm_device, mx4_quantize,
                           mx4_quantize_device)

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _x(M, K, seed, kind="normal"):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((M, K)).astype(np.float32) * np.exp(rng.standard_normal(K)).astype(np.float32)
    if kind == "edges":  # borders between the values, their neighbours, signed zeros, subnormals, the largest numbers
        e = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.999, 0.0], np.float32)
        x = e[rng.integers(0, len(e), (M, K))] * rng.choice([-1, 1], (M, K)).astype(np.float32)
        x = np.nextafter(x, x + rng.integers(-1, 2, (M, K)).astype(np.float32), dtype=np.float32)
        for m in range(M):
            x[m] = np.ldexp(x[m], rng.integers(-149, 125))
    return x


def _device4(M, K):
    return (torch.full((M, R.padded(K) // 2), 255, dtype=torch.uint8, device="cuda"),
            torch.full((M, R.padded(K) // 32), 255, dtype=torch.uint8, device="cuda"))


@pytest.mark.parametrize("kind", ["normal", "edges"])
@pytest.mark.parametrize("M,K", [(1, 1), (3, 31), (2, 32), (5, 33), (4, 129), (7, 384), (1, 4096), (300, 130), (3, 2176)])
def test_quantize_is_exact(M, K, kind):
    x = _x(M, K, M * 1000 + K, kind)
    codes, scales = mx4_quantize(x)
    want = R.quantize(x)
    assert np.array_equal(scales, want[1])
    assert np.array_equal(codes, want[0])
    y = mx4_dequantize(codes, scales, K)
    assert np.array_equal(y, R.values(*want)[:, :K])


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("offset,extra", [(0, 0), (0, 3), (1, 0), (8, 24)])
def test_quantize_types_strides_and_alignment(t, offset, extra):
    """Rows at any element offset and stride; what lies between the rows of the result is left as it was."""
    M, K = 37, 200
    flat = torch.from_numpy(_x(1, M * (K + extra) + offset, 5)).cuda().to(t).flatten()
    x = flat[offset:].view(M, K + extra)[:, :K]
    codes, scales = _device4(M, K)
    mx4_quantize_device(x, codes, scales)
    want = R.quantize(x.float().cpu().numpy())
    assert np.array_equal(codes.cpu().numpy(), want[0]) and np.array_equal(scales.cpu().numpy(), want[1])
    out = torch.full_like(flat, 77.0)
    y = out[offset:].view(M, K + extra)[:, :K]
    mx4_dequantize_device(codes, scales, y)
    assert torch.equal(y.cpu(), torch.from_numpy(R.values(*want)[:, :K]).to(t))
    out[offset:].view(M, K + extra)[:, :K] = 77.0
    assert bool((out == 77.0).all())


def test_nan_and_infinity_take_their_block():
    x = _x(4, 160, 9)
    x[0, 3], x[1, 40], x[2, 159] = np.nan, np.inf, -np.inf
    codes, scales = mx4_quantize(x)
    want = R.quantize(x)
    assert np.array_equal(scales, want[1]) and np.count_nonzero(scales == 255) == 3
    y = mx4_dequantize(codes, scales, 160)
    assert np.array_equal(y, R.values(*want)[:, :160], equal_nan=True)
    W = _x(6, 160, 10)
    C = mx4_gemm(codes, scales, *mx4_quantize(W))
    assert np.isnan(C[:3]).all() and np.isfinite(C[3]).all()


def test_rows_beyond_32_bit_offsets():
    """Codes of more than 2^32 bytes: the last rows go to and come from their place."""
    M, K = (1 << 22) + 5, 2048
    x = torch.zeros((M, K), dtype=torch.bfloat16, device="cuda")
    x[-2:] = torch.from_numpy(_x(2, K, 3)).cuda().to(x.dtype)
    codes, scales = _device4(M, K)
    assert codes.numel() > 1 << 32
    mx4_quantize_device(x, codes, scales)
    want = R.quantize(x[-2:].float().cpu().numpy())
    assert np.array_equal(codes[-2:].cpu().numpy(), want[0]) and np.array_equal(scales[-2:].cpu().numpy(), want[1])
    assert int(codes[:-2].max()) == 0 and int(scales[:-2].max()) == 0
    x.fill_(7.0)
    mx4_dequantize_device(codes, scales, x)
    assert np.array_equal(x[-2:].float().cpu().numpy(), R.values(*want).astype(np.float32)) and float(x[:-2].abs().max()) == 0
    W = torch.from_numpy(_x(3, K, 4)).cuda()
    wc, ws = _device4(3, K)
    mx4_quantize_device(W, wc, ws)
    C = torch.full((M, 3), 5.0, device="cuda")
    mx4_gemm_device(codes, scales, wc, ws, C)
    exact = R.values(*want) @ R.values(wc.cpu().numpy(), ws.cpu().numpy()).T
    assert np.allclose(C[-2:].cpu().numpy(), exact, rtol=1e-4, atol=1e-4) and float(C[:-2].abs().max()) == 0


# one row, a few, odd numbers of rows and channels around the kernels' tiles, one step of K and many
SHAPES = [(1, 1, 1), (1, 384, 8192), (3, 100, 17), (16, 128, 16), (17, 130, 33), (40, 4096, 70), (63, 640, 129), (64, 256, 64),
          (128, 128, 128), (129, 1152, 255), (256, 512, 256), (300, 384, 1000), (515, 900, 384), (1001, 1152, 512),
          (2048, 256, 2048), (2049, 384, 2050), (4, 8192, 4096), (33, 33, 3000)]


def _operands(M, K, N, seed):
    return R.quantize(_x(M, K, seed)), R.quantize(_x(N, K, seed + 1))


@pytest.mark.parametrize("M,K,N", SHAPES)
@pytest.mark.parametrize("t", TYPES)
def test_product(M, K, N, t):
    (A, As), (W, Ws) = _operands(M, K, N, M + K + N)
    C = torch.full((M + 1, N), 9.0, dtype=t, device="cuda")
    mx4_gemm_device(*(torch.from_numpy(a).cuda() for a in (A, As, W, Ws)), C[:M])
    a, w = R.values(A, As), R.values(W, Ws)
    want, size = a @ w.T, np.abs(a) @ np.abs(w).T
    tol = K * 2.0 ** -23 * size + torch.finfo(t).eps / 2 * np.abs(want) + (2.0 ** -25 if t == torch.float16 else 0)
    assert (np.abs(C[:M].double().cpu().numpy() - want) <= tol).all()
    assert bool((C[M] == 9.0).all())


@pytest.mark.parametrize("M,K,N", [(1, 640, 40), (50, 1000, 70), (200, 2000, 300), (520, 384, 600)])
def test_product_of_whole_numbers_is_exact(M, K, N):
    """Scales of one and partial sums below 2^24 in quarters: every addition is exact, whatever the order."""
    rng = np.random.default_rng(K)
    Kp = R.padded(K)
    A, W = (rng.integers(0, 256, (r, Kp // 2)).astype(np.uint8) for r in (M, N))
    s = lambda r: np.full((r, Kp // 32), 127, np.uint8)  # noqa: E731
    C = mx4_gemm(A, s(M), W, s(N))
    assert np.array_equal(C.astype(np.float64), R.values(A, s(M)) @ R.values(W, s(N)).T)


def test_product_scales_of_every_block():
    """Each block's scale is its own: powers of two from 2^-30 to 2^30 over blocks of ones give exact sums of each alone."""
    K, M, N = 640, 20, 24
    one = np.full((M, K // 2), 0x22, np.uint8)
    for blk in range(K // 32):
        As, Ws = np.zeros((M, K // 32), np.uint8), np.full((N, K // 32), 127, np.uint8)
        As[:, blk] = 97 + 3 * np.arange(M)
        Ws[:, blk] = 110 + np.arange(N)
        C = mx4_gemm(one, As, np.full((N, K // 2), 0x22, np.uint8), Ws)
        want = 32 * np.ldexp(1.0, As[:, blk].astype(int)[:, None] + Ws[:, blk].astype(int) - 254)
        assert np.allclose(C, want, rtol=2.0 ** -20)  # the other blocks add 2^-127 each


def test_another_stream_and_a_captured_graph():
    """Quantise, product and back on a side stream, then captured and replayed on new inputs: each replay equals the eager
    results."""
    M, K, N = 70, 300, 200
    w, ws = (torch.from_numpy(a).cuda() for a in R.quantize(_x(N, K, 1)))
    x = torch.from_numpy(_x(M, K, 2)).cuda()
    codes, scales = _device4(M, K)
    C, y = torch.empty((M, N), device="cuda"), torch.empty((M, K), device="cuda")

    def step():
        mx4_quantize_device(x, codes, scales)
        mx4_gemm_device(codes, scales, w, ws, C)
        mx4_dequantize_device(codes, scales, y)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for seed in (3, 4, 5):
        x.copy_(torch.from_numpy(_x(M, K, seed)))
        C.fill_(-1)
        g.replay()
        torch.cuda.synchronize()
        got = C.clone(), y.clone()
        step()
        assert torch.equal(got[0], C) and torch.equal(got[1], y)
        assert np.array_equal(y.cpu().numpy(), R.rounded(np.pad(_x(M, K, seed), ((0, 0), (0, 20))))[:, :K])


def test_refusals():
    x = torch.zeros((4, 64), device="cuda")
    codes, scales = _device4(4, 64)
    for bad in (lambda: mx4_quantize_device(x.cpu(), codes, scales), lambda: mx4_quantize_device(x.double(), codes, scales),
                lambda: mx4_quantize_device(x.t(), codes, scales), lambda: mx4_quantize_device(x, codes[:3], scales[:3]),
                lambda: mx4_quantize_device(x, codes[:, :32], scales), lambda: mx4_quantize_device(x, codes, scales.cpu()),
                lambda: mx4_gemm_device(codes, scales, *_device4(3, 200), torch.empty((4, 3), device="cuda")),
                lambda: mx4_gemm_device(codes, scales, codes, scales, torch.empty((4, 5), device="cuda")),
                lambda: mx4_gemm_device(codes, scales, codes, scales, torch.empty((4, 8), device="cuda")[:, ::2]),
                lambda: mx4_dequantize_device(codes, scales, torch.empty((4, 129), device="cuda"))):
        with pytest.raises(MignonError):
            bad()
    flat = torch.zeros(4 * 64 + 16, dtype=torch.uint8, device="cuda")
    with pytest.raises(MignonError, match="misaligned"):
        mx4_quantize_device(x, flat[1:257].view(4, 64), scales)


@pytest.mark.parametrize("M,K,N", [(3600, 128, 3700), (3841, 384, 3712), (3700, 640, 3601), (3600, 1000, 3704), (3585, 1025, 3590),
                                   (1001, 1152, 1024), (1000, 128, 1030), (1030, 384, 1004), (2050, 896, 2056), (2048, 128, 2052)])
@pytest.mark.parametrize("t", TYPES)
def test_product_of_large_matrices(M, K, N, t):
    """Tiles of every size with whole and cut edges, odd and even numbers of steps, and outputs of every alignment."""
    (A, As), (W, Ws) = _operands(M, K, N, M + K + N)
    C = torch.full((M + 1, N), 9.0, dtype=t, device="cuda")
    mx4_gemm_device(*(torch.from_numpy(a).cuda() for a in (A, As, W, Ws)), C[:M])
    a, w = (torch.from_numpy(R.values(*x)).cuda() for x in ((A, As), (W, Ws)))
    want, size = a @ w.T, a.abs() @ w.abs().T
    tol = K * 2.0 ** -23 * size + torch.finfo(t).eps / 2 * want.abs() + (2.0 ** -25 if t == torch.float16 else 0)
    assert bool(((C[:M].double() - want).abs() <= tol).all())
    assert bool((C[M] == 9.0).all())
