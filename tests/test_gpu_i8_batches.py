"""A token's result from moe_i8_layer_forward: the same bits whatever its batch, and
in a 16-bit type the fp32 result rounded once."""
import pytest

import moe_ffn

torch = pytest.importorskip("torch")
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
