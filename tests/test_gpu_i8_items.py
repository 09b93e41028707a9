"""int8 products in which a workgroup takes several tiles one after the other, whole
ones (every result stored) and ragged ones in turn, on rows from one to several
stages long: the next tile's operands are on their way while results are
written."""
import pytest

import moe_ffn

torch = pytest.importorskip("torch")
import i8_reference as R  # noqa: E402
from test_gpu_i8_layer import Case, flag  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [F32, BF16, F16]


@pytest.fixture(scope="module", autouse=True)
def gpu_ready():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    yield
    torch.cuda.synchronize()


def up(a, b):
    return (a + b - 1) // b


# m, n, tile, workgroups: 64 x 32, 128 x 128 and 256 x 256 tiles, at most 3, 2 and 1 workgroups a CU.
LINEAR = [(60000, 32, (64, 32), 768), (60010, 21, (64, 32), 768), (70000, 128, (128, 128), 512), (70001, 100, (128, 128), 512),
          (8192, 4200, (256, 256), 256), (8200, 4352, (256, 256), 256)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("k", [32, 96, 160, 416])
@pytest.mark.parametrize("m,n,tile,workgroups", LINEAR)
def test_linear(dtype, k, m, n, tile, workgroups):
    assert up(m, tile[0]) * up(n, tile[1]) > workgroups
    codes, scales = R.weights(1, m, k, m + k)
    q, s = R.quantise(0.1 * torch.randn((n, k), generator=R.generator(n), device=DEV))
    matrix = moe_ffn.MoeI8Linear(k, m, codes[0], scales[0])
    y = torch.full((n + 1, m), 7.0, dtype=dtype, device=DEV)
    matrix.forward(q, s, y[:n])
    for at in range(0, n, 1024):
        part = slice(at, min(n, at + 1024))
        R.close(y[part], R.product(q[part], s[part], codes[0], scales[0]), dtype)
    assert bool((y[n] == 7.0).all())


MANY = [512, 384, 640, 130, 0, 512, 1, 517]                        # whole and ragged tiles of 128 rows
EVEN = [64] * 12 + [63, 65, 128, 0, 1, 127] + [64] * 14            # of 64
FEW = [0, 32] * 10 + [0] * 30 + [31, 33, 0, 1] * 3                 # of 32
RARE = [0] * 300 + [16] * 10 + [15, 17, 1] + [0] * 187 + [16, 14]  # of 16
# sizes, m, the length of x's rows, tile, workgroups
BANK = [(MANY, 8192, (32, 96, 416, 1056), (256, 128), 256), (EVEN, 4100, (32, 96, 416), (128, 64), 512),
        (FEW, 4096, (1088, 1632), (64, 32), 768), (RARE, 8192, (32, 320, 1056), (64, 16), 512)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sizes,m,k,tile,workgroups", [(s, m, k, t, w) for s, m, ks, t, w in BANK for k in ks])
def test_bank(dtype, sizes, m, k, tile, workgroups):
    assert sum(up(n, tile[1]) for n in sizes) * up(m, tile[0]) > workgroups
    experts, rows = len(sizes), sum(sizes)
    codes, scales = R.weights(experts, m, k, m + k)
    bank = moe_ffn.MoeI8Bank(experts, k, m, codes, scales)
    q, s = R.quantise(0.05 * torch.randn((rows, k), generator=R.generator(k), device=DEV))
    offsets = torch.tensor([0] + sizes, device=DEV).cumsum(0).to(torch.int32)
    index = torch.randint(0, rows, (rows,), generator=R.generator(k + 1), device=DEV).to(torch.int32)
    for gather in (None, index):
        y = torch.full((rows + 1, m), 5.0, dtype=dtype, device=DEV)
        _, e = bank.forward(q, s, offsets, y[:rows], index=gather)
        assert flag(e) == 0 and bool((y[rows] == 5.0).all())
        at, bounds = torch.arange(rows, device=DEV) if gather is None else gather.long(), offsets.tolist()
        for i in range(experts):
            r = at[bounds[i]:bounds[i + 1]]
            if len(r):
                R.close(y[bounds[i]:bounds[i + 1]], R.product(q[r], s[r], codes[i], scales[i]), dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("h", [32, 96, 416])
def test_layer_wide_middle(dtype, h):
    """Gate and up by 256 x 128 tiles, of which the shared expert's are whole."""
    assert up(8192, 256) * (up(768, 128) + 8) > 256
    Case(768, h, 4096, 8, 2, True, seed=h).check(dtype, gate=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,experts,k,spread,rows,tile,workgroups",
                         [(1280, 40, 2, 40, 64, (128, 64), 512), (64, 256, 8, 16, 32, (128, 32), 256)])
def test_layer_even_groups(dtype, tokens, experts, k, spread, rows, tile, workgroups):
    """Groups of exactly a tile's rows."""
    for h in (32, 160):
        c = Case(tokens, h, 2080, experts, k, False, seed=tokens)
        t, r = torch.arange(tokens, device=DEV)[:, None], torch.arange(k, device=DEV)[None]
        c.ids = ((t * k + r) % spread).to(torch.int32).contiguous()
        assert torch.bincount(c.ids.reshape(-1).long(), minlength=experts).tolist() == [rows] * spread + [0] * (experts - spread)
        assert spread * up(2 * 2112, tile[0]) > workgroups
        c.check(dtype)
