"""moe_quantize_e4m3 and moe_fp8_linear_* against the formats and products in
64 bits (fp8_reference.py): codes and scales bit for bit, products within
bounds that follow from the additions and roundings they make."""
import pytest

import moe_ffn

torch = pytest.importorskip("torch")
import fp8_reference as R  # noqa: E402

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


def same(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


# ------------------------------------------------------------- quantiser ---
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n,k,extra", [(1, 1, 0), (1, 128, 0), (3, 129, 0), (5, 2047, 0), (7, 2560, 8), (33, 640, 3),
                                       (300, 2048, 0), (2, 16384, 0)])
def test_quantise_bits(dtype, n, k, extra):
    g = R.generator(n * 1000 + k)
    x = (torch.randn((n, k + extra), generator=g, device=DEV) * torch.exp2(torch.randint(-9, 9, (n, k + extra), generator=g, device=DEV).float())).to(dtype)[:, :k]
    codes, scales, e = moe_ffn.quantize_e4m3(x)
    want, ws = R.quantise(x)
    assert flag(e) == 0
    assert same(scales, ws)
    assert torch.equal(codes.view(torch.uint8), want)


def test_quantise_rounds_to_even_at_every_boundary():
    """Every midpoint between neighbouring codes, and both fp32 neighbours of
    it, in groups whose scale is exactly 1 (one element is 448)."""
    t = R.e4m3_table()[:0x7f]
    mid = ((t[1:] + t[:-1]) / 2).float()
    v = torch.cat([t.float(), mid, torch.nextafter(mid, torch.zeros(())), torch.nextafter(mid, torch.full((), 1e9))])
    v = torch.cat([v, -v])
    v = torch.nn.functional.pad(v, (0, -v.numel() % 127)).view(-1, 127)
    x = torch.cat([torch.full((v.shape[0], 1), 448.0), v], dim=1).to(DEV)
    codes, scales, e = moe_ffn.quantize_e4m3(x)
    want, ws = R.quantise(x)
    assert bool((scales == 1).all()) and same(scales, ws) and torch.equal(codes.view(torch.uint8), want)


def test_quantise_special_rows():
    x = torch.zeros((8, 256), device=DEV)
    x[1, 5] = 2.0 ** -149                       # below the scale's floor: rounds to 0
    x[2, 128:] = 2.0 ** -101
    x[3, 7] = 3.4e38
    x[4, 130] = float("inf")
    x[5, 3] = float("nan")
    x[5, 200] = 1.0
    x[6, 0] = -float("inf")
    x[7, :] = -0.0
    codes, scales, e = moe_ffn.quantize_e4m3(x)
    assert flag(e) == 1
    c = codes.view(torch.uint8)
    for row, group in ((4, 1), (5, 0), (6, 0)):
        assert bool((c[row, group * 128:(group + 1) * 128] == 0).all()) and float(scales[row, group]) == 0.0
    finite = torch.nan_to_num(x, nan=0.0, posinf=0.0, neginf=0.0)
    want, ws = R.quantise(finite)
    keep = torch.tensor([[r, g] for r in range(8) for g in range(2) if (r, g) not in ((4, 1), (5, 0), (6, 0))], device=DEV)
    assert torch.equal(scales[keep[:, 0], keep[:, 1]], ws[keep[:, 0], keep[:, 1]])
    assert torch.equal(c.view(8, 2, 128)[keep[:, 0], keep[:, 1]], want.view(8, 2, 128)[keep[:, 0], keep[:, 1]])


# -------------------------------------------------------------- products ---
def check(y, codes_x, scales_x, w, dtype, wide):
    x = R.rows(codes_x, scales_x)
    ref = x @ w.T
    tol = R.linear_tolerance(x, w, ref, dtype, wide)
    bad = (y.double() - ref).abs() > tol
    assert not bool(bad.any()), (int(bad.sum()), float(((y.double() - ref).abs() / tol).max()))
    if ref.norm() > 0:   # the error of the sums over many outputs, beside the rounding of y
        rel = float((y.double() - ref).norm() / ref.norm())
        assert rel <= (1e-4 if wide and dtype != F32 else 1e-6) + R.half_step(dtype)


# Every kernel: few columns (one and two column tiles, one to four row tiles), and each of the
# tiles that wide batches take as they grow, for 16-bit and for fp32 results
# (64 x 32 and 32 x 48 whose waves share K, 64 x 64 in groups of waves, up to 256 x 256); rows and columns that end inside
# a tile, blocks cut short, one to 128 blocks a row, and numbers of blocks that
# the groups do not share evenly.
SHAPES = [(32, 1, 1), (96, 17, 3), (160, 130, 16), (1056, 100, 14), (8192, 4200, 1), (2048, 33, 16), (2048, 512, 1), (2048, 2048, 17), (1056, 300, 33), (16384, 48, 5),
          (640, 2560, 65), (352, 8200, 20), (288, 8210, 50), (3200, 77, 1500), (8192, 1500, 70), (2048, 5000, 66), (2080, 1000, 333), (128, 40, 700), (512, 2047, 1500), (8192, 200, 130),
          (1056, 1500, 1300), (64, 2100, 1100), (320, 2100, 1100), (192, 3000, 2100), (128, 4100, 4000), (416, 4000, 4090), (1024, 4000, 4090),
          (160, 1500, 300), (1056, 1000, 900), (96, 1000, 900), (16384, 700, 1111), (416, 1020, 1000), (256, 2040, 2000),
          (352, 4000, 4090), (64, 4090, 4000)]


@pytest.mark.parametrize("K,M,N", SHAPES)
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_forward_and_apply(K, M, N, dtype):
    g = R.generator(K + 3 * M + 7 * N)
    codes, scales = R.random_matrix(M, K, g)
    w = R.matrix(codes, scales)
    x = torch.randn((N, K), generator=g, device=DEV).to(dtype)
    qc, qs = R.quantise(x)
    lin = moe_ffn.MoeFp8Linear(K, M, codes, scales, max_columns=N)
    assert lin.weight_bytes() == M * K + 4 * scales.numel()
    y = lin.forward(qc, qs, dtype=dtype)
    check(y, qc, qs, w, dtype, N > 64)
    z, e = lin.apply(x)
    assert z.dtype == dtype and flag(e) == 0
    check(z, qc, qs, w, dtype, N > 64)
    assert same(y, z)   # the same products in the same order, wherever the columns are quantised
    lin.close()


@pytest.mark.parametrize("N", [1, 9, 40, 200])
@pytest.mark.parametrize("x_type,y_type", [(BF16, F32), (F32, BF16), (F16, F32)])
def test_strided_and_mixed_types(N, x_type, y_type):
    """Rows of x and y inside wider tensors, at starts that no vector load
    fits; what lies between the rows stays as it was."""
    K, M = 352, 77
    g = R.generator(N)
    codes, scales = R.random_matrix(M, K, g)
    w = R.matrix(codes, scales)
    wide = torch.randn((N, K + 5), generator=g, device=DEV).to(x_type)
    x = wide[:, 3:3 + K]
    qc, qs = R.quantise(x)
    lin = moe_ffn.MoeFp8Linear(K, M, codes.view(torch.uint8), scales, max_columns=N)
    out = torch.full((N + 1, M + 9), 7.0, dtype=y_type, device=DEV)
    e = torch.zeros(1, dtype=torch.int32, device=DEV)
    lin.apply(x, y=out[:N, 2:2 + M], error=e)
    check(out[:N, 2:2 + M], qc, qs, w, y_type, N > 64)
    out[:N, 2:2 + M] = 7.0
    assert bool((out == 7.0).all()) and flag(e) == 0
    lin.close()


@pytest.mark.parametrize("N", [3, 16, 17, 100])
def test_apply_in_place(N):
    K = 256
    g = R.generator(N)
    codes, scales = R.random_matrix(K, K, g)
    x = torch.randn((N, K), generator=g, device=DEV)
    lin = moe_ffn.MoeFp8Linear(K, K, codes, scales, max_columns=N)
    want, _ = lin.apply(x)
    lin.apply(x, y=x)
    assert same(x, want)
    lin.close()


def test_weights_from_host_equal_weights_from_device():
    K, M, N = 288, 130, 20
    g = R.generator(5)
    codes, scales = R.random_matrix(M, K, g)
    x = torch.randn((N, K), generator=g, device=DEV)
    a = moe_ffn.MoeFp8Linear(K, M, codes, scales, max_columns=N)
    b = moe_ffn.MoeFp8Linear(K, M, codes.view(torch.uint8).cpu().numpy(), scales.cpu().numpy(), max_columns=N)
    assert same(a.apply(x)[0], b.apply(x)[0])
    a.close()
    b.close()


@pytest.mark.parametrize("N", [2, 50, 300])
def test_every_code_and_nan(N):
    """A matrix of all 256 codes: NaN weights make exactly their rows NaN, and
    a NaN in one column's codes exactly that column."""
    K, M = 256, 48
    g = R.generator(9)
    codes = torch.randint(0, 256, (M, K), generator=g, device=DEV, dtype=torch.uint8)
    codes[codes & 127 == 127] = 5
    scales = torch.full((1, 2), 0.01, device=DEV)
    codes[7, 200] = 0x7f
    codes[41, 3] = 0xff
    x = torch.randn((N, K), generator=g, device=DEV)
    qc, qs = R.quantise(x)
    qc[1, 130] = 0x7f
    lin = moe_ffn.MoeFp8Linear(K, M, codes, scales)
    for dtype in (F32, BF16):
        y = lin.forward(qc, qs, dtype=dtype)
        nan = torch.zeros((N, M), dtype=torch.bool, device=DEV)
        nan[:, 7] = nan[:, 41] = True
        nan[1] = True
        assert torch.equal(y.isnan(), nan)
        rows, cols = [i for i in range(N) if i != 1], [i for i in range(M) if i not in (7, 41)]
        check(y[rows][:, cols], qc[rows], qs[rows], R.matrix(codes, scales)[cols], dtype, N > 64)
    lin.close()


@pytest.mark.parametrize("N", [4, 40])
def test_nonfinite_activations(N):
    """A group with an infinity or NaN counts as zeros and raises bit 1."""
    K, M = 384, 96
    g = R.generator(11)
    codes, scales = R.random_matrix(M, K, g)
    x = torch.randn((N, K), generator=g, device=DEV)
    clean = x.clone()
    clean[2, 128:256] = 0
    clean[N - 1, 256:] = 0
    x[2, 130] = float("inf")
    x[N - 1, 383] = float("nan")
    lin = moe_ffn.MoeFp8Linear(K, M, codes, scales, max_columns=N)
    y, e = lin.apply(x)
    z, f = lin.apply(clean)
    assert flag(e) == 1 and flag(f) == 0
    assert same(y, z)
    lin.close()


def test_stream_and_graph_replay():
    """Two captured calls on one handle and other work between the replays, on
    a stream of their own."""
    K, M = 512, 300
    g = R.generator(13)
    codes, scales = R.random_matrix(M, K, g)
    lin = moe_ffn.MoeFp8Linear(K, M, codes, scales, max_columns=128)
    small, big = (torch.randn((n, K), generator=g, device=DEV).to(BF16) for n in (5, 128))
    ys, yb = torch.empty((5, M), dtype=BF16, device=DEV), torch.empty((128, M), dtype=BF16, device=DEV)
    e = torch.zeros(1, dtype=torch.int32, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        lin.apply(small, y=ys, error=e)
        lin.apply(big, y=yb, error=e)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lin.apply(small, y=ys, error=e)
        lin.apply(big, y=yb, error=e)
    for i in range(4):
        small.normal_(generator=g)
        big.normal_(generator=g)
        want_s, want_b = lin.apply(small)[0], lin.apply(big)[0]
        ys.zero_()
        yb.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert same(ys, want_s) and same(yb, want_b), i
    assert flag(e) == 0
    lin.close()


def test_refusals():
    K, M = 64, 32
    g = R.generator(17)
    codes, scales = R.random_matrix(M, K, g)
    lin = moe_ffn.MoeFp8Linear(K, M, codes, scales, max_columns=4)
    x = torch.zeros((4, K), device=DEV)
    with pytest.raises(TypeError):
        lin.apply(x.double())
    with pytest.raises(ValueError):
        lin.apply(x[:, :32])
    with pytest.raises(ValueError):
        lin.apply(x.t().contiguous().t())
    with pytest.raises(ValueError):
        lin.apply(torch.zeros((1, K), device=DEV).expand(4, K))
    with pytest.raises(moe_ffn.MoeError) as ex:
        lin.apply(torch.zeros((5, K), device=DEV))   # past max_columns
    assert ex.value.status == 1
    with pytest.raises(moe_ffn.MoeError):
        lin.apply(torch.zeros((0, K), device=DEV))
    with pytest.raises(ValueError):
        lin.apply(x, y=torch.zeros((4, M + 1), device=DEV))
    with pytest.raises(ValueError):
        lin.apply(x.cpu())
    qc, qs, _ = moe_ffn.quantize_e4m3(x)
    with pytest.raises(ValueError):
        lin.forward(qc, qs[:, :0])
    with pytest.raises(TypeError):
        lin.forward(qc.float(), qs)
    raw = torch.zeros(4 * K + 8, dtype=torch.uint8, device=DEV)
    with pytest.raises(moe_ffn.MoeError):   # codes must start on 16 bytes
        lin.forward(raw[8:].view(4, K), qs)
    with pytest.raises(ValueError):
        moe_ffn.MoeFp8Linear(K, M, codes, scales.expand(2, 1).contiguous())
    lin.close()


@pytest.mark.parametrize("N", [1, 20, 100, 2000])
def test_matrix_past_32_bits(N):
    """The largest matrix: its codes and its tiles pass 2^32 bytes."""
    K, M = 16384, 262144
    g = R.generator(19)
    codes = torch.empty((M, K), dtype=torch.uint8, device=DEV)
    codes.random_(generator=g).bitwise_and_(0xBF)   # below 2: no NaN
    scales = torch.rand((M // 128, K // 128), generator=g, device=DEV) * 0.02
    lin = moe_ffn.MoeFp8Linear(K, M, codes, scales)
    x = torch.randn((N, K), generator=g, device=DEV)
    qc, qs = R.quantise(x)
    y = lin.forward(qc, qs, dtype=BF16)
    cols = torch.cat([torch.arange(40, device=DEV), M // 2 + torch.arange(40, device=DEV), M - 1 - torch.arange(120, device=DEV)])
    rows = torch.unique(torch.tensor([0, N // 3, N - 1], device=DEV))
    w = R.codes_to_values(codes[cols]) * R.spread(scales[cols // 128], 1, K)
    check(y[rows][:, cols], qc[rows], qs[rows], w, BF16, N > 64)
    assert bool(y.isfinite().all())
    lin.close()


def test_rows_past_32_bits():
    """65,536 rows of x and of y inside a buffer of more than 2^32 elements."""
    K, M, N = 32, 40, 65536
    g = R.generator(23)
    codes, scales = R.random_matrix(M, K, g)
    buf = torch.full((N, 65700), 3.0, dtype=BF16, device=DEV)
    x, y = buf[:, 7:7 + K], buf[:, 65600:65600 + M]
    x.normal_(generator=g)
    qc, qs = R.quantise(x)
    lin = moe_ffn.MoeFp8Linear(K, M, codes, scales, max_columns=N)
    got = moe_ffn.quantize_e4m3(x)
    assert torch.equal(got[0].view(torch.uint8), qc) and torch.equal(got[1], qs) and flag(got[2]) == 0
    e = torch.zeros(1, dtype=torch.int32, device=DEV)
    lin.apply(x, y=y, error=e)
    check(y, qc, qs, R.matrix(codes, scales), BF16, True)
    assert flag(e) == 0 and bool((buf[:, :7] == 3).all()) and bool((buf[:, 7 + K:65600] == 3).all())
    lin.close()


def test_bound_calls_keep_the_matrix():
    """A bound call outlives the caller's last reference to the handle, and
    raises once the handle is closed."""
    K, M = 128, 64
    g = R.generator(29)
    codes, scales = R.random_matrix(M, K, g)
    x = torch.randn((3, K), generator=g, device=DEV)
    y, e = torch.empty((3, M), device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    lin = moe_ffn.MoeFp8Linear(K, M, codes, scales, max_columns=3)
    want, _ = lin.apply(x)
    call = lin.bind_apply(x, y, e)
    del lin
    call()
    assert same(y, want)
    lin = moe_ffn.MoeFp8Linear(K, M, codes, scales)
    call = lin.bind_forward(*moe_ffn.quantize_e4m3(x)[:2], y)
    lin.close()
    with pytest.raises(moe_ffn.MoeError):
        call()


# The tiles of test_forward_and_apply's wider shapes, with a last row tile of few rows.
@pytest.mark.parametrize("K,M,N", [(160, 1501, 300), (1056, 1001, 900), (512, 2047, 1500), (64, 2101, 1100), (192, 3003, 2100),
                                   (352, 4090, 4090)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strided_rows_of_wide_batches(K, M, N, dtype):
    """Rows of x and y inside wider tensors at odd starts: the results of
    contiguous ones, and nothing between them touched."""
    g = R.generator(K + M)
    codes, scales = R.random_matrix(M, K, g)
    x = torch.randn((N, K + 5), generator=g, device=DEV).to(dtype)[:, 3:3 + K]
    lin = moe_ffn.MoeFp8Linear(K, M, codes, scales, max_columns=N)
    want, e = lin.apply(x.contiguous())
    out = torch.full((N + 1, M + 6), 7.0, dtype=dtype, device=DEV)
    y = out[:N, 1:1 + M]
    lin.apply(x, y=y, error=e)
    assert same(y, want) and flag(e) == 0
    y.fill_(7.0)
    assert bool((out == 7.0).all())
    lin.forward(*R.quantise(x), y=y)
    assert same(y, want)
    y.fill_(7.0)
    assert bool((out == 7.0).all())
    lin.close()


def test_overlapping_forwards_of_one_handle():
    K, M = 1024, 1000
    g = R.generator(31)
    codes, scales = R.random_matrix(M, K, g)
    lin = moe_ffn.MoeFp8Linear(K, M, codes, scales)
    rows = [R.quantise(torch.randn((n, K), generator=g, device=DEV)) for n in (7, 900)]
    want = [lin.forward(*r, dtype=BF16) for r in rows]
    streams = [torch.cuda.Stream() for _ in rows]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for r, s in zip(rows, streams):
            with torch.cuda.stream(s):
                got.append(lin.forward(*r, dtype=BF16))
    torch.cuda.synchronize()
    assert all(same(y, want[i % 2]) for i, y in enumerate(got))
    lin.close()


@pytest.mark.parametrize("K,M,N", [(640, 4090, 4090), (896, 1500, 1500), (1056, 600, 900), (2048, 512, 16), (512, 1000, 60)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_scales_at_any_start(K, M, N, dtype):
    """Scales of the rows one element behind a 16-byte boundary, and rows of
    scales of which not every four lie within a row."""
    g = R.generator(K + N)
    codes, scales = R.random_matrix(M, K, g)
    qc, qs = R.quantise(torch.randn((N, K), generator=g, device=DEV))
    lin = moe_ffn.MoeFp8Linear(K, M, codes, scales)
    want = lin.forward(qc, qs, dtype=dtype)
    moved = torch.full((qs.numel() + 2,), float("nan"), device=DEV)
    moved[1:-1] = qs.flatten()
    assert same(lin.forward(qc, moved[1:-1].view_as(qs), dtype=dtype), want)
    check(want, qc, qs, R.matrix(codes, scales), dtype, N > 64)
    lin.close()
