"""How moe_fp8_linear sums within a block, on activations whose groups hold one
element far above the others: 16-bit results of wide batches bit for bit as far
as fp32 additions allow against the e4m3 instruction in 64 bits
(fp8_reference.e4m3_instruction), and with MOE_SUMS_F32 as close to the exact
product as fp32 sums are."""
import pytest

import moe_ffn

torch = pytest.importorskip("torch")
import fp8_reference as R  # noqa: E402

DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
gpu = pytest.mark.gpu


def same(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


def test_set_sums_arguments():
    lib = moe_ffn.library()
    assert lib.moe_fp8_linear_set_sums(None, moe_ffn.SUMS_F32) == 1
    assert (moe_ffn.SUMS_AUTO, moe_ffn.SUMS_F32) == (0, 1)


def outliers(n, k, g):
    """Rows with one element in each group of 128 a hundred to a thousand times
    the others, and every fourth row without."""
    x = torch.randn((n, k), generator=g, device=DEV)
    factor = torch.exp2(6.6 + 3.4 * torch.rand((n, R.blocks(k)), generator=g, device=DEV))
    factor[3::4] = 1.0
    at = torch.randint(0, 128, (n, R.blocks(k)), generator=g, device=DEV) + 128 * torch.arange(R.blocks(k), device=DEV)
    at = at.clamp_max(k - 1)
    return x.scatter(1, at, x.gather(1, at) * factor)


def sample(n, count, g):
    """Indices of about `count` of n, the ends among them."""
    if n <= count:
        return torch.arange(n, device=DEV)
    return torch.unique(torch.cat([torch.tensor([0, n - 1], device=DEV), torch.randint(0, n, (count - 2,), generator=g, device=DEV)]))


# One at least for each tile of 16-bit results, and for each that fp32 sums
# take; the last one's 105,000 results are few enough for fp32 sums in any case.
SHAPES = [(672, 300, 1500), (352, 1000, 900), (672, 1020, 1000), (352, 1300, 1500), (672, 1300, 1400), (352, 2047, 1500),
          (160, 2000, 1700), (672, 3000, 2100), (352, 4000, 4090), (96, 5500, 70), (8192, 5000, 70),
          (8192, 1500, 70)]


@gpu
@pytest.mark.parametrize("K,M,N", SHAPES)
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_outlier_rows(K, M, N, dtype):
    g = R.generator(K + M + N)
    codes, scales = R.random_matrix(M, K, g)
    # Some subnormal and some of the largest codes, which random values leave out.
    some = torch.rand((M, K), generator=g, device=DEV)
    codes = codes.view(torch.uint8)
    codes[some < 0.05] &= 0x87
    codes[some > 0.99] |= 0x7e
    codes[(codes & 0x7f) == 0x7f] = 0x7e
    x = outliers(N, K, g).to(BF16)
    qc, qs = R.quantise(x)
    rows, cols = sample(N, 64, g), sample(M, 400, g)
    args = qc[rows], qs[rows], codes[cols], scales, cols // 128
    exact = R.rows(qc[rows], qs[rows]) @ (R.codes_to_values(codes[cols]) * R.spread(scales[cols // 128], 1, K)).T
    magnitude = R.rows(qc[rows], qs[rows]).abs() @ (R.codes_to_values(codes[cols]) * R.spread(scales[cols // 128], 1, K)).abs().T
    half, tiny = R.half_step(dtype), 2.0 ** -25 if dtype == F16 else 0.0

    lin = moe_ffn.MoeFp8Linear(K, M, codes, scales, max_columns=N)
    y = lin.forward(qc, qs, dtype=dtype)
    assert same(lin.apply(x, dtype=dtype)[0], y)
    few = M * N <= 327680
    ref, tol = (exact, (128 + R.blocks(K) + 2) * 2.0 ** -23 * magnitude) if few else R.e4m3_instruction(*args)
    off = (y[rows][:, cols].double() - ref).abs()
    tol = tol + half * (ref.abs() + tol) + tiny
    assert bool((off <= tol).all()), float((off / tol).max())
    # Seven of eight may lose 2^-13 of the largest, 2^-10 beside a subnormal code.
    assert bool(((ref - exact).abs() <= 7 * 2.0 ** -10 * magnitude).all())
    assert float((ref - exact).norm() / exact.norm()) <= 2e-4

    lin.set_sums(moe_ffn.SUMS_F32)
    z = lin.forward(qc, qs, dtype=dtype)
    assert same(lin.apply(x, dtype=dtype)[0], z)
    tol = (128 + R.blocks(K) + 2) * 2.0 ** -23 * magnitude
    tol = tol + half * (exact.abs() + tol) + tiny
    off = (z[rows][:, cols].double() - exact).abs()
    assert bool((off <= tol).all()), float((off / tol).max())
    # The fp32 result has the same sums; only the tiles' shares of K differ.
    f = lin.forward(qc, qs, dtype=F32)[rows][:, cols].double()
    assert bool(((f - exact).abs() <= (128 + R.blocks(K) + 2) * 2.0 ** -23 * magnitude + 2.0 ** -24 * exact.abs()).all())
    lin.set_sums(moe_ffn.SUMS_AUTO)
    assert same(lin.forward(qc, qs, dtype=dtype), y)
    for bad in (2, -1):
        with pytest.raises(moe_ffn.MoeError):
            lin.set_sums(bad)
    lin.close()


@gpu
def test_strided_results_of_fp32_sums_and_a_captured_call():
    """16-bit rows inside a wider tensor, and a call that keeps the sums it was
    captured with."""
    K, M, N = 352, 2101, 1501
    g = R.generator(5)
    codes, scales = R.random_matrix(M, K, g)
    qc, qs = R.quantise(outliers(N, K, g))
    lin = moe_ffn.MoeFp8Linear(K, M, codes, scales, sums=moe_ffn.SUMS_F32)
    want = lin.forward(qc, qs, dtype=BF16)
    out = torch.full((N + 1, M + 6), 7.0, dtype=BF16, device=DEV)
    y = out[:N, 1:1 + M]
    lin.forward(qc, qs, y=y)
    assert same(y, want)
    y.fill_(7.0)
    assert bool((out == 7.0).all())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lin.forward(qc, qs, y=y)
    lin.set_sums(moe_ffn.SUMS_AUTO)
    other = lin.forward(qc, qs, dtype=BF16)
    assert not same(other, want)
    for _ in range(3):
        y.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert same(y, want)
        assert same(lin.forward(qc, qs, dtype=BF16), other)
    lin.close()
