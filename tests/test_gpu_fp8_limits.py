"""The e4m3 layer and linear at the ends of their ranges: weights and gates that
are not finite, and scales so far apart that a product of two that do not belong
together overflows."""
import pytest

import moe_ffn

torch = pytest.importorskip("torch")
import fp8_reference as R  # noqa: E402
from test_gpu_fp8_layer import BF16, DEV, F32, Bank, check, flag, routes, same  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def gpu_ready():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    yield
    torch.cuda.synchronize()


@pytest.mark.parametrize("gated", [False, True])
def test_weights_and_gates_out_of_range(gated):
    """A nonfinite weight leaves its token the shared expert alone, a negative
    one counts as it is, a nonfinite gate makes its token's row 0; the other
    tokens' results do not change."""
    g = R.generator(41)
    E, k, T = 6, 3, 5
    bank = Bank(128, 64, E, True, g)
    layer = bank.layer(k, T)
    x = torch.randn((T, 128), generator=g, device=DEV)
    ids, w = routes(T, E, k, g)
    gate = torch.randn(T, generator=g, device=DEV) if gated else None
    clean, e = layer.forward(x, ids, w, shared_gate=gate)
    assert flag(e) == 0
    for value in (float("nan"), float("inf"), -float("inf")):
        v = w.clone()
        v[1, 2] = value
        y, e = layer.forward(x, ids, v, shared_gate=gate)
        none = w.clone()
        none[1] = 0.0
        assert flag(e) == 1 and same(y[[0, 2, 3, 4]], clean[[0, 2, 3, 4]])
        check(y, x, ids, none, bank, gate)
        if gated:
            b = gate.clone()
            b[3] = value
            y, e = layer.forward(x, ids, w, shared_gate=b)
            assert flag(e) == 1 and bool((y[3] == 0).all()) and same(y[[0, 1, 2, 4]], clean[[0, 1, 2, 4]])
    v = w.clone()
    v[2, 0] = -1.5
    y, e = layer.forward(x, ids, v, shared_gate=gate)
    assert flag(e) == 1
    check(y, x, ids, v, bank, gate)
    layer.close()
