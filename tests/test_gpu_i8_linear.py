"""moe_quantize_i8 and moe_i8_linear_* against the formats and products in 64
bits (i8_reference.py): codes and scales bit for bit, products within the
roundings that they make."""
import pytest

import moe_ffn

torch = pytest.importorskip("torch")
import i8_reference as R  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(scope="module", autouse=True)
def gpu_ready():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    yield
    torch.cuda.synchronize()


def flag(e):
    return int(e.cpu()[0])


# ------------------------------------------------------------- quantiser ---
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n,k,extra", [(1, 1, 0), (1, 64, 0), (3, 129, 0), (5, 512, 0), (6, 1000, 1), (5, 2047, 0), (7, 2560, 8),
                                       (33, 640, 3), (300, 2048, 0), (9, 4100, 0), (2, 8192, 4), (2, 16383, 0), (70, 16384, 0)])
def test_quantise_bits(dtype, n, k, extra):
    g = R.generator(n * 1000 + k)
    x = (torch.randn((n, k + extra), generator=g, device=DEV) * torch.exp2(torch.randint(-9, 9, (n, k + extra), generator=g, device=DEV).float())).to(dtype)[:, :k]
    codes, scales, e = moe_ffn.quantize_i8(x)
    want, ws = R.quantise(x)
    assert flag(e) == 0
    assert torch.equal(scales, ws) and torch.equal(codes, want)


def test_quantise_rounds_to_even():
    """Every midpoint between neighbouring codes, and both fp32 neighbours of
    it, in rows whose factor is exactly 1 (one element is 127)."""
    mid = torch.arange(0, 127, dtype=torch.float32) + 0.5
    v = torch.cat([mid, torch.nextafter(mid, torch.zeros(())), torch.nextafter(mid, torch.full((), 1e9))])
    x = torch.cat([torch.full((1,), 127.0), v, -v])[None].to(DEV)
    codes, scales, e = moe_ffn.quantize_i8(x)
    want, ws = R.quantise(x)
    assert float(scales[0]) == 1.0 and torch.equal(scales, ws) and torch.equal(codes, want) and flag(e) == 0
    assert int(codes[0, 1]) == 0 and int(codes[0, 2]) == 2   # 0.5 and 1.5


@pytest.mark.parametrize("k", [300, 2048, 5000])
def test_quantise_special_rows(k):
    x = torch.zeros((8, k), device=DEV)
    x[1, 5] = 2.0 ** -149                       # below the scale's floor: rounds to 0
    x[2, 128:] = 2.0 ** -101
    x[3, 7] = 3.4e38
    x[4, k - 1] = float("inf")
    x[5, 3] = float("nan")
    x[5, 200] = 1.0
    x[6, 0] = -float("inf")
    x[7, :] = -0.0
    codes, scales, e = moe_ffn.quantize_i8(x)
    assert flag(e) == 1
    bad, good = [4, 5, 6], [0, 1, 2, 3, 7]
    assert not codes[bad].any() and not scales[bad].any()
    want, ws = R.quantise(x[good])
    assert torch.equal(codes[good], want) and torch.equal(scales[good], ws)


def test_quantise_leaves_other_rows_alone():
    """Codes and scales behind the rows, and an error word already set."""
    x = torch.randn((3, 96), device=DEV)
    codes = torch.full((5, 96), 77, dtype=torch.int8, device=DEV)
    scales = torch.full((5,), 7.0, device=DEV)
    e = torch.full((1,), 2, dtype=torch.int32, device=DEV)
    moe_ffn.quantize_i8(x, codes[:3], scales[:3], e)
    assert bool((codes[3:] == 77).all()) and bool((scales[3:] == 7.0).all()) and flag(e) == 2


# ---------------------------------------------------------------- linear ---
def make(k, m, seed=1, columns=0):
    codes, scales = R.weights(1, m, k, seed)
    return moe_ffn.MoeI8Linear(k, m, codes[0], scales[0], max_columns=columns), codes[0], scales[0]


SIZES = [(32, 1, 1), (64, 16, 1), (96, 17, 3), (2048, 64, 1), (160, 100, 15), (2080, 1000, 16), (1024, 130, 17), (352, 257, 40),
         (640, 2560, 64), (2048, 48, 65), (96, 2047, 100), (512, 300, 333), (2080, 1000, 333), (16384, 33, 5), (16384, 16, 130),
         (128, 4099, 700), (2048, 2048, 1032), (256, 8192, 900), (64, 520, 5000), (192, 3001, 2100), (320, 4096, 4100), (640, 2560, 700), (352, 2100, 330),
         (160, 4001, 2700), (8192, 2, 2), (8192, 100, 3), (16384, 40, 1), (4064, 33, 4)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("k,m,n", SIZES)
def test_forward_and_apply(dtype, k, m, n):
    matrix, codes, scales = make(k, m, k + m, n)
    x = torch.randn((n, k), generator=R.generator(n), device=DEV).to(dtype)
    q, s = R.quantise(x)
    # f16's range: results stay below 60000.
    ref = R.product(q, s, codes, scales)
    if dtype == F16 and float(ref.abs().max()) > 6e4:
        x = (x / 64).to(dtype)
        q, s = R.quantise(x)
        ref = R.product(q, s, codes, scales)
    y = matrix.forward(q, s, dtype=dtype)
    R.close(y, ref, dtype)
    z, e = matrix.apply(x)
    assert flag(e) == 0 and torch.equal(z, y)   # the same sums, the same bits


def test_codes_at_their_ends_sum_exactly():
    """The largest sums there are: 16,384 products of -128 and -128, or 127."""
    k, m, n = 16384, 48, 40
    codes = torch.full((m, k), -128, dtype=torch.int8, device=DEV)
    codes[1] = 127
    matrix = moe_ffn.MoeI8Linear(k, m, codes, torch.ones(m, device=DEV))
    x = torch.full((n, k), -128, dtype=torch.int8, device=DEV)
    x[1] = 127
    y = matrix.forward(x, torch.ones(n, device=DEV))
    assert torch.equal(y.double(), R.sums(x, codes).float().double())


# 64 x 16, 64 x 32 in stages of four chunks and of two, 64 x 64, 64 x 128, 128 x 128, 256 x 256
TILES = [(1000, 40), (1000, 300), (16999, 21), (8970, 40), (10230, 70), (16641, 33), (40960, 129)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("k", [32, 96, 416])
@pytest.mark.parametrize("m,n", TILES)
def test_every_tile(dtype, k, m, n):
    """Every tile on short rows, whose last stage is cut."""
    codes, scales = R.weights(1, m, k, m + k)
    q, s = R.quantise(0.1 * torch.randn((n, k), generator=R.generator(n), device=DEV))
    matrix = moe_ffn.MoeI8Linear(k, m, codes[0], scales[0])
    y = torch.full((n + 1, m), 7.0, dtype=dtype, device=DEV)
    matrix.forward(q, s, y[:n])
    R.close(y[:n], R.product(q, s, codes[0], scales[0]), dtype)
    assert bool((y[n] == 7.0).all())


@pytest.mark.parametrize("n", [2, 50, 700])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strided_rows(dtype, n):
    """y's rows further apart than they are long and not on 16 bytes: what lies
    between them stays; x's rows strided as well."""
    k, m = 160, 77
    matrix, codes, scales = make(k, m, 5, n)
    wide = torch.randn((n, k + 3), device=DEV).to(dtype)
    x = wide[:, 1:k + 1]
    out = torch.full((n, m + 6), 9.0, dtype=dtype, device=DEV)
    y = out[:, 3:m + 3]
    e = torch.zeros(1, dtype=torch.int32, device=DEV)
    matrix.apply(x, y, e)
    q, s = R.quantise(x)
    R.close(y, R.product(q, s, codes, scales), dtype)
    assert bool((out[:, :3] == 9.0).all()) and bool((out[:, m + 3:] == 9.0).all())


@pytest.mark.parametrize("n", [1, 20, 300])
def test_apply_in_place(n):
    matrix, codes, scales = make(256, 256, 6, n)
    x = torch.randn((n, 256), device=DEV)
    q, s = R.quantise(x)
    ref = matrix.forward(q, s)
    y, _ = matrix.apply(x, x)
    assert y.data_ptr() == x.data_ptr() and torch.equal(x, ref)


@pytest.mark.parametrize("n", [3, 100])
def test_nonfinite_rows(n):
    """A row with a NaN or infinity counts as zeros and flags; the others are as
    without it."""
    matrix, codes, scales = make(512, 96, 7, n)
    x = torch.randn((n, 512), device=DEV, dtype=BF16)
    clean, e = matrix.apply(x)
    x[1, 300] = float("nan")
    y, e = matrix.apply(x)
    assert flag(e) == 1 and not y[1].any()
    keep = torch.arange(n, device=DEV) != 1
    assert torch.equal(y[keep], clean[keep])


def test_host_weights_and_bytes():
    codes, scales = R.weights(1, 70, 96, 8)
    a = moe_ffn.MoeI8Linear(96, 70, codes[0], scales[0])
    b = moe_ffn.MoeI8Linear(96, 70, codes[0].cpu().numpy(), scales[0].cpu().numpy())
    q, s = R.quantise(torch.randn((20, 96), device=DEV))
    assert a.weight_bytes() == 70 * 100
    assert torch.equal(a.forward(q, s), b.forward(q, s))


def test_refusals():
    matrix, codes, scales = make(64, 32, 9, 8)
    x = torch.zeros((9, 64), device=DEV)
    e = torch.zeros(1, dtype=torch.int32, device=DEV)
    with pytest.raises(moe_ffn.MoeError):
        matrix.apply(x)                                                    # more columns than the workspace has
    q, s = R.quantise(x)
    for args, exc in (((q.to(torch.uint8), s), TypeError), ((q[:, :32], s), ValueError), ((q, s[:8]), ValueError),
                      ((q, s.double()), TypeError), ((q.cpu(), s.cpu()), ValueError)):
        with pytest.raises(exc):
            matrix.forward(*args)
    with pytest.raises(TypeError):
        matrix.forward(q, s, torch.zeros((9, 32), dtype=torch.float64, device=DEV))
    with pytest.raises(ValueError):
        matrix.forward(q, s, torch.zeros((9, 31), device=DEV))
    with pytest.raises(moe_ffn.MoeError):
        matrix.forward(q[:0], s[:0])                                       # no rows
    for bad, exc in ((x.double(), TypeError), (x.t(), ValueError)):
        with pytest.raises(exc):
            moe_ffn.quantize_i8(bad)
    call = matrix.bind_apply(x[:8], torch.zeros((8, 32), device=DEV), e)
    matrix.close()
    with pytest.raises(moe_ffn.MoeError):
        call()


def test_graph_replay():
    """apply captured, replayed on new inputs with eager work between."""
    matrix, codes, scales = make(2048, 640, 10, 40)
    x, y = torch.zeros((40, 2048), device=DEV, dtype=BF16), torch.zeros((40, 640), device=DEV, dtype=BF16)
    e = torch.zeros(1, dtype=torch.int32, device=DEV)
    call = None
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        call = matrix.bind_apply(x, y, e)
        call()
    for seed in range(4):
        x.copy_(torch.randn(x.shape, generator=R.generator(seed), device=DEV).to(BF16))
        graph.replay()
        torch.cuda.synchronize()
        q, s = R.quantise(x)
        R.close(y, R.product(q, s, codes, scales), BF16)
        eager, _ = matrix.apply(x)
        assert torch.equal(y, eager)


def test_forwards_of_one_handle_overlap():
    matrix, codes, scales = make(2048, 2048, 11)
    inputs = [R.quantise(torch.randn((300, 2048), generator=R.generator(i), device=DEV)) for i in range(2)]
    want = [matrix.forward(*q) for q in inputs]
    outs = [torch.zeros_like(w) for w in want]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        for q, y, st in zip(inputs, outs, streams):
            matrix.forward(*q, y=y, stream=st)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))


@pytest.mark.parametrize("n", [9, 300])
def test_results_past_32_bits(n):
    """Rows of y that begin beyond 2^31 elements."""
    matrix, codes, scales = make(96, 40, 12, n)
    stride = (1 << 32) // n + 40
    wide = torch.empty(stride * n, dtype=BF16, device=DEV)
    y = wide.as_strided((n, 40), (stride, 1), 5)
    x = torch.randn((n, 96), generator=R.generator(2), device=DEV).to(BF16)
    e = torch.zeros(1, dtype=torch.int32, device=DEV)
    matrix.apply(x, y, e)
    q, s = R.quantise(x)
    R.close(y, R.product(q, s, codes, scales), BF16)


def test_rows_on_a_stream_of_their_own():
    x = torch.randn((300, 1000), device=DEV)
    want = moe_ffn.quantize_i8(x)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    got = moe_ffn.quantize_i8(x, stream=side)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
