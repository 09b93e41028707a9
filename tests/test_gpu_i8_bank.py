"""moe_i8_bank_*: products of rows grouped by expert against 64 bits, over
ragged, empty and bad groups."""
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


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def check(bank, codes, scales, sizes, dtype, gather=None, seed=0, lead=0, extra=0, zero_rows=()):
    """A product with groups of the given sizes that begin at row `lead`, `extra`
    rows behind the last; gather: number of x's rows."""
    rows = sum(sizes)
    total = lead + rows + extra
    offsets = [lead]
    for n in sizes:
        offsets.append(offsets[-1] + n)
    g = R.generator(seed)
    x = 0.05 * torch.randn((gather or max(total, 1), bank.K), generator=g, device=DEV)
    q, s = R.quantise(x)
    index = torch.randint(0, gather, (total,), generator=g, device=DEV).to(torch.int32) if gather else None
    y = torch.full((max(total, 1), bank.M), 5.0, dtype=dtype, device=DEV)
    if total:
        _, e = bank.forward(q, s, ints(offsets), y, index=index)
        assert flag(e) == 0
    at = index.long() if gather else torch.arange(total, device=DEV)
    for i, n in enumerate(sizes):
        if n:
            r = at[offsets[i]:offsets[i + 1]]
            R.close(y[offsets[i]:offsets[i + 1]], R.product(q[r], s[r], codes[i], scales[i]), dtype)
    assert bool((y[:lead] == 5.0).all()) and bool((y[lead + rows:] == 5.0).all())
    return y


RAGGED = [[1], [0, 0, 1], [3, 0, 1, 16, 17, 0], [64, 65, 1, 0, 63, 15], [200, 1, 0, 129, 128, 127], [0, 0, 700, 0], [5] * 33,
          [0] * 60 + [40] + [0] * 10, [130, 257, 64, 1]]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("case", range(len(RAGGED)))
def test_ragged(dtype, case):
    sizes = RAGGED[case]
    k, m = [(96, 70), (64, 128), (2080, 100), (256, 1000)][case % 4]
    codes, scales = R.weights(len(sizes), m, k, case)
    bank = moe_ffn.MoeI8Bank(len(sizes), k, m, codes, scales)
    check(bank, codes, scales, sizes, dtype, seed=case)
    check(bank, codes, scales, sizes, dtype, gather=max(1, sum(sizes) // 3), seed=case + 50)


# Every tile: 64 x 16, 64 x 32 in stages of four chunks and of two, 128 x 64, 256 x 128.
TILES = [(4, 96, 1000, 50), (4, 416, 1000, 400), (64, 1088, 1000, 500), (8, 416, 1000, 600), (8, 96, 1000, 600), (4, 96, 4000, 900),
         (4, 416, 4001, 1000)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("experts,k,m,rows", TILES)
def test_every_tile(dtype, experts, k, m, rows):
    codes, scales = R.weights(experts, m, k, rows)
    bank = moe_ffn.MoeI8Bank(experts, k, m, codes, scales)
    g = torch.Generator().manual_seed(rows + k)
    share = torch.rand(experts, generator=g) ** 2
    share[1] = 0.0
    sizes = [int(v) for v in (share / share.sum() * rows).floor()]
    sizes[0] += rows - sum(sizes)
    check(bank, codes, scales, sizes, dtype, seed=k, lead=3, extra=5)
    check(bank, codes, scales, sizes, dtype, gather=77, seed=k)


def test_rows_outside_the_groups_stay():
    codes, scales = R.weights(3, 80, 64, 1)
    bank = moe_ffn.MoeI8Bank(3, 64, 80, codes, scales)
    for lead, extra in ((0, 9), (7, 0), (5, 130)):
        check(bank, codes, scales, [10, 0, 21], BF16, lead=lead, extra=extra)
        check(bank, codes, scales, [10, 0, 21], F32, gather=6, lead=lead, extra=extra)
    check(bank, codes, scales, [0, 0, 0], F32, extra=20)


@pytest.mark.parametrize("experts", [1, 63, 64, 65, 512, 4096])
def test_numbers_of_experts(experts):
    codes, scales = R.weights(experts, 17, 32, experts)
    bank = moe_ffn.MoeI8Bank(experts, 32, 17, codes, scales)
    g = torch.Generator().manual_seed(experts)
    sizes = [0] * experts
    for e in torch.randint(0, experts, (150,), generator=g).tolist():
        sizes[e] += 1
    sizes[experts - 1] += 3
    sizes[0] += 20
    check(bank, codes, scales, sizes, F32, seed=experts)


def test_same_row_many_times():
    """One row of x for every row of every group."""
    codes, scales = R.weights(4, 96, 128, 3)
    bank = moe_ffn.MoeI8Bank(4, 128, 96, codes, scales)
    q, s = R.quantise(torch.randn((1, 128), device=DEV))
    y, e = bank.forward(q, s, ints([0, 1, 40, 40, 200]), index=torch.zeros(200, dtype=torch.int32, device=DEV))
    assert flag(e) == 0
    for i, (a, b) in enumerate(((0, 1), (1, 40), (40, 40), (40, 200))):
        assert bool((y[a:b] == y[a:a + 1]).all())
        if b > a:
            R.close(y[a:b], R.product(q, s, codes[i], scales[i]).expand(b - a, 96), F32)


def test_bad_offsets_flag():
    """Decreasing offsets and offsets outside the rows: flagged, nothing written
    outside, and the groups that are as they should be are right."""
    codes, scales = R.weights(3, 40, 64, 4)
    bank = moe_ffn.MoeI8Bank(3, 64, 40, codes, scales)
    q, s = R.quantise(torch.randn((100, 64), device=DEV))
    for offsets, right in (([0, 30, 20, 20], [(0, 0, 30)]), ([0, 30, 60, 101], [(0, 0, 30), (1, 30, 60), (2, 60, 100)]),
                           ([-5, 30, 60, 70], [(0, 0, 30), (1, 30, 60), (2, 60, 70)]),
                           ([0, -2147483648, 2147483647, 5], [])):
        out = torch.full((102, 40), 3.0, device=DEV)
        y = out[1:101]
        _, e = bank.forward(q, s, ints(offsets), y)
        assert flag(e) == 1, offsets
        for g, a, b in right:
            R.close(y[a:b], R.product(q[a:b], s[a:b], codes[g], scales[g]), F32)
        assert bool((out[0] == 3.0).all()) and bool((out[101] == 3.0).all())


def test_offsets_that_go_back_and_forth():
    """Offsets of which every other one decreases: no row is computed for two
    groups, so that the work stays that of the rows."""
    for experts, rows in ((6, 1000), (4096, 270000), (1025, 300)):
        codes, scales = R.weights(experts, 17, 32, 12)
        bank = moe_ffn.MoeI8Bank(experts, 32, 17, codes, scales)
        q, s = R.quantise(torch.randn((rows, 32), generator=R.generator(experts), device=DEV))
        offsets = torch.zeros(experts + 1, dtype=torch.int32, device=DEV)
        offsets[1::2] = rows
        y, e = bank.forward(q, s, offsets)
        assert flag(e) == 1
        R.close(y, R.product(q, s, codes[0], scales[0]), F32)


def test_bad_index_gives_zero_rows():
    codes, scales = R.weights(2, 130, 96, 5)
    bank = moe_ffn.MoeI8Bank(2, 96, 130, codes, scales)
    q, s = R.quantise(torch.randn((10, 96), device=DEV))
    index = torch.arange(90, dtype=torch.int32, device=DEV) % 10
    bad = {3: -1, 40: 10, 88: 2147483647, 89: -2147483648}
    for r, v in bad.items():
        index[r] = v
    for dtype in (F32, BF16):
        y, e = bank.forward(q, s, ints([0, 45, 90]), index=index, dtype=dtype)
        assert flag(e) == 1
        good = torch.tensor([r for r in range(90) if r not in bad], device=DEV)
        assert not y[list(bad)].any()
        at = index[good].long()
        ref = torch.where((good < 45)[:, None], R.product(q[at], s[at], codes[0], scales[0]),
                          R.product(q[at], s[at], codes[1], scales[1]))
        R.close(y[good], ref, dtype)


@pytest.mark.parametrize("dtype", [F32, F16])
def test_strided_rows_of_y(dtype):
    codes, scales = R.weights(3, 50, 160, 6)
    bank = moe_ffn.MoeI8Bank(3, 160, 50, codes, scales)
    q, s = R.quantise(0.1 * torch.randn((70, 160), device=DEV))
    out = torch.full((70, 57), 2.0, dtype=dtype, device=DEV)
    bank.forward(q, s, ints([0, 20, 20, 70]), out[:, 3:53])
    for e, a, b in ((0, 0, 20), (2, 20, 70)):
        R.close(out[a:b, 3:53], R.product(q[a:b], s[a:b], codes[e], scales[e]), dtype)
    assert bool((out[:, :3] == 2.0).all()) and bool((out[:, 53:] == 2.0).all())


def test_refusals():
    codes, scales = R.weights(2, 32, 64, 7)
    bank = moe_ffn.MoeI8Bank(2, 64, 32, codes, scales)
    q, s = R.quantise(torch.randn((10, 64), device=DEV))
    offsets, e = ints([0, 5, 10]), ints([0])
    y = torch.zeros((10, 32), device=DEV)
    with pytest.raises(ValueError):
        bank.bind_forward(q, s, offsets, torch.zeros((11, 32), device=DEV), e)          # more rows than x has
    with pytest.raises(ValueError):
        bank.bind_forward(q, s, offsets[:2], y, e)
    with pytest.raises(TypeError):
        bank.bind_forward(q, s, offsets.long(), y, e)
    with pytest.raises(ValueError):
        bank.bind_forward(q, s, offsets, y, e, index=ints([0] * 9))
    with pytest.raises(ValueError):
        bank.bind_forward(q[:, :32], s, offsets, y, e)
    with pytest.raises(ValueError):
        bank.bind_forward(q, s[:9], offsets, y, e)
    with pytest.raises(ValueError):
        bank.bind_forward(q, s, offsets, y[0], e)
    with pytest.raises(moe_ffn.MoeError):
        bank.bind_forward(q, s, offsets, y[:0], e)()
    call = bank.bind_forward(q, s, offsets, y, e)
    bank.close()
    with pytest.raises(moe_ffn.MoeError):
        call()


def test_graph_replay_with_new_groups():
    """One captured call serves any grouping of the same number of rows."""
    codes, scales = R.weights(8, 200, 256, 8)
    bank = moe_ffn.MoeI8Bank(8, 256, 200, codes, scales)
    q, s = torch.zeros((300, 256), dtype=torch.int8, device=DEV), torch.zeros(300, device=DEV)
    offsets, e, y = ints([0] * 9), ints([0]), torch.zeros((300, 200), device=DEV, dtype=BF16)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        bank.bind_forward(q, s, offsets, y, e)()
    for seed in range(4):
        g = R.generator(seed)
        a, b = R.quantise(torch.randn((300, 256), generator=g, device=DEV))
        cuts = torch.randint(0, 301, (7,), generator=g, device=DEV).sort().values
        q.copy_(a)
        s.copy_(b)
        offsets[1:8] = cuts.to(torch.int32)
        offsets[8] = 300
        graph.replay()
        torch.cuda.synchronize()
        bounds = offsets.tolist()
        for i in range(8):
            lo, hi = bounds[i], bounds[i + 1]
            if hi > lo:
                R.close(y[lo:hi], R.product(q[lo:hi], s[lo:hi], codes[i], scales[i]), BF16)
        eager, _ = bank.forward(q, s, offsets, dtype=BF16)
        assert torch.equal(eager, y) and flag(e) == 0


def test_many_experts_with_many_rows_each():
    """The largest table of groups beside the largest tile."""
    experts, k, m = 4096, 32, 17
    codes, scales = R.weights(experts, m, k, 9)
    bank = moe_ffn.MoeI8Bank(experts, k, m, codes, scales)
    g = R.generator(9)
    sizes = 66 + torch.randint(0, 12, (experts,), generator=g, device=DEV)
    sizes[100:300] = 0
    sizes[7], sizes[4095] = 900, 8000
    offsets = torch.zeros(experts + 1, dtype=torch.int32, device=DEV)
    offsets[1:] = sizes.cumsum(0)
    rows = int(offsets[-1])
    assert rows // experts > 64
    q, s = R.quantise(torch.randn((rows, k), generator=g, device=DEV))
    y, e = bank.forward(q, s, offsets)
    assert flag(e) == 0
    owner = torch.repeat_interleave(torch.arange(experts, device=DEV), sizes)
    for at in range(0, rows, 20000):
        o = owner[at:at + 20000]
        ref = (codes[o].double() * q[at:at + 20000].double()[:, None]).sum(2) * s[at:at + 20000].double()[:, None] * scales[o].double()
        R.close(y[at:at + 20000], ref, F32)


def test_rows_past_32_bits():
    """x's codes beyond 2^32 bytes and y's rows beyond 2^31 elements."""
    k, m, rows = 16384, 16, 270000
    codes, scales = R.weights(3, m, k, 10)
    bank = moe_ffn.MoeI8Bank(3, k, m, codes, scales)
    q = torch.zeros((rows, k), dtype=torch.int8, device=DEV)
    s = torch.ones(rows, device=DEV)
    some = torch.tensor([0, 1, 129999, 130000, 262143, 262144, 262145, 269999], device=DEV)
    q[some] = torch.randint(-127, 128, (8, k), generator=R.generator(1), device=DEV).to(torch.int8)
    wide = torch.empty((rows, 10000), dtype=BF16, device=DEV)
    y = wide[:, 9000:9016]
    _, e = bank.forward(q, s, ints([0, 130000, 130000, rows]), y)
    assert flag(e) == 0
    for r in some.tolist():
        i = 0 if r < 130000 else 2
        R.close(y[r:r + 1], R.product(q[r:r + 1], s[r:r + 1], codes[i], scales[i]), BF16)
    assert not y[2:129999].any() and not y[262146:269999].any()


def test_calls_of_one_bank_overlap():
    codes, scales = R.weights(16, 512, 1024, 11)
    bank = moe_ffn.MoeI8Bank(16, 1024, 512, codes, scales)
    calls = []
    for i in range(2):
        q, s = R.quantise(torch.randn((900, 1024), generator=R.generator(i), device=DEV))
        cuts = torch.randint(0, 901, (15,), generator=R.generator(i), device=DEV).sort().values.to(torch.int32)
        offsets = torch.cat([ints([0]), cuts, ints([900])])
        want, _ = bank.forward(q, s, offsets)
        calls.append((q, s, offsets, want, torch.zeros_like(want), torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(5):
        for q, s, offsets, _, y, st in calls:
            bank.forward(q, s, offsets, y=y, stream=st)
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) for _, _, _, want, y, _ in calls)
