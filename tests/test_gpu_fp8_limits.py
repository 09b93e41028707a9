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


# Seven blocks a row: two groups of waves share them unevenly, and the last
# group's step past the end meets an earlier block's scale (16-bit results of
# 64 x 64 tiles, whose form with half as many waves takes 1,300 x 1,500); four
# groups and two for fp32 results; a single group and canonical rows for more.
@pytest.mark.parametrize("M,N", [(1000, 900), (1300, 1500), (2000, 1700), (2047, 1500)])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("K", [640, 672, 896])
def test_scales_of_other_blocks_do_not_meet(K, M, N, dtype):
    g = R.generator(43)
    nb = R.blocks(K)
    codes, scales = R.random_matrix(M, K, g)
    qc, qs = R.quantise(torch.randn((N, K), generator=g, device=DEV))
    want = moe_ffn.MoeFp8Linear(K, M, codes, scales).forward(qc, qs, dtype=dtype)
    for b in range(nb - 1):   # block b's rows are scaled up and its matrix down, the last block's the other way round
        up, down = torch.ones(nb, device=DEV), torch.ones(nb, device=DEV)
        up[b], down[b] = 2.0 ** 110, 2.0 ** -110
        up[nb - 1], down[nb - 1] = 2.0 ** -60, 2.0 ** 60
        lin = moe_ffn.MoeFp8Linear(K, M, codes, scales * down)
        assert same(lin.forward(qc, (qs * up).contiguous(), dtype=dtype), want), b
        lin.close()
