"""A token's result from moe_i8_layer_forward: the same bits whatever its batch, and
in a 16-bit type the fp32 result rounded once; moe_i8_linear_apply the same where
it takes one launch and where it takes two."""
import pytest

import moe_ffn

torch = pytest.importorskip("torch")
import i8_reference as R  # noqa: E402
from test_gpu_i8_layer import Case, flag  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(scope="module", autouse=True)
def gpu_ready():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    yield
    torch.cuda.synchronize()


# Few and many experts, so that down and the sum take one launch or three up to 64 tokens.
SHAPES = [(320, 96, 24, 10), (2048, 512, 64, 10), (4096, 2048, 8, 2)]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("h,i,experts,k", SHAPES)
@pytest.mark.parametrize("n", [1, 32, 33, 63, 64, 65, 130, 700])
def test_sixteen_bits_are_the_fp32_result_rounded(dtype, h, i, experts, k, n):
    """x is exact in fp32, so its codes, and all up to the sum, are those of the
    fp32 call: y differs from it by its own rounding alone."""
    c = Case(n, h, i, experts, k, True, seed=n)
    x = c.x.to(dtype)
    y, e = c.layer.forward(x, c.ids, c.w, shared_gate=c.gate)
    full, f = c.layer.forward(x.float(), c.ids, c.w, shared_gate=c.gate)
    assert flag(e) == 0 and flag(f) == 0
    assert torch.equal(y, full.to(dtype))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("h,i,experts,k", SHAPES)
def test_same_bits_in_every_batch(dtype, h, i, experts, k):
    c = Case(300, h, i, experts, k, True, seed=36)
    x = c.x.to(dtype)
    whole, e = c.layer.forward(x, c.ids, c.w, shared_gate=c.gate)
    assert flag(e) == 0
    for n in (1, 16, 33, 64, 65, 100):
        part, e = c.layer.forward(x[:n], c.ids[:n], c.w[:n], shared_gate=c.gate[:n])
        assert flag(e) == 0 and torch.equal(part, whole[:n]), n


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("k,m", [(512, 16384), (512, 16385), (2048, 8192), (2048, 8193), (32, 40001), (8192, 8192)])
def test_few_rows_in_one_launch_or_two(dtype, k, m):
    """Both sides of the numbers of outputs and rows up to which the product's kernel
    quantises x itself, with a row that is not finite."""
    codes, scales = R.weights(1, m, k, m + k)
    matrix = moe_ffn.MoeI8Linear(k, m, codes[0], scales[0] / 64, max_columns=17)
    for n in (1, 2, 4, 5, 8, 9, 16, 17):
        x = torch.randn((n, k), generator=R.generator(n), device=DEV).to(dtype)
        q, s = R.quantise(x)
        y, e = matrix.apply(x)
        assert flag(e) == 0 and torch.equal(y, matrix.forward(q, s, dtype=dtype)), n
        R.close(y, R.product(q, s, codes[0], scales[0] / 64), dtype)
        x[n - 1, 17] = float("nan")
        z, e = matrix.apply(x)
        assert flag(e) == 1 and not z[n - 1].any() and torch.equal(z[:n - 1], y[:n - 1]), n
