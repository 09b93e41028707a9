"""int8 operators at the ends of their ranges: the most experts and routes a layer
takes, its widest rows either way, and gathered rows up to 2^31 bytes of codes."""
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


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("tokens", [1, 5, 40, 64, 65, 300, 2100])
@pytest.mark.parametrize("experts,shared", [(4095, True), (4096, False)])
def test_most_experts(dtype, tokens, experts, shared):
    Case(tokens, 64, 32, experts, 32, shared, seed=tokens).check(dtype, gate=shared)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("tokens", [1, 33, 64, 200])
@pytest.mark.parametrize("h,i", [(16384, 32), (32, 16384), (16352, 96), (96, 16352)])
def test_widest_rows(dtype, tokens, h, i):
    Case(tokens, h, i, 4, 3, True, seed=tokens + h).check(dtype, gate=True)


def test_gathered_rows_up_to_two_gib():
    k, m, x_rows = 16384, 40, 1 << 17
    codes, scales = R.weights(2, m, k, 13)
    bank = moe_ffn.MoeI8Bank(2, k, m, codes, scales)
    q = torch.zeros((x_rows, k), dtype=torch.int8, device=DEV)
    s = torch.ones(x_rows, device=DEV)
    some = torch.tensor([0, 1, 65535, 65536, x_rows - 2, x_rows - 1], device=DEV)
    q[some] = torch.randint(-127, 128, (6, k), generator=R.generator(2), device=DEV).to(torch.int8)
    s[some] = torch.rand(6, generator=R.generator(3), device=DEV) + 0.5
    index = some.to(torch.int32).repeat(30)
    for rows in (6, 90, 180):
        offsets = torch.tensor([0, rows // 3, rows], dtype=torch.int32, device=DEV)
        y, e = bank.forward(q, s, offsets, index=index[:rows])
        assert flag(e) == 0
        for g, (a, b) in enumerate(((0, rows // 3), (rows // 3, rows))):
            r = index[a:b].long()
            R.close(y[a:b], R.product(q[r], s[r], codes[g], scales[g]), F32)
