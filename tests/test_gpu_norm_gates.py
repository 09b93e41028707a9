"""moe_block_norm's sigmoid gates over all of their range: steps of a quarter
past where the exponential overflows and vanishes, every bf16 and fp16 value,
infinities and NaN, in each form of gate and on rows of one and of two groups of
elements a thread."""
import pytest

import moe_ffn

torch = pytest.importorskip("torch")
import fp8_reference as R  # noqa: E402
from test_gpu_norm import BF16, DEV, F16, F32, U, flag, make, reference  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def gpu_ready():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    yield
    torch.cuda.synchronize()


QUARTERS = torch.cat([torch.arange(-1200, 1201) / 4.0, torch.tensor([float("inf"), -float("inf")])])


def check(norm, residual, block, gate):
    """h and n within reference()'s bounds, which hold for results in fp32's
    normal range, and what comes on top below it: a sigmoid under 2^-126 may
    count as 0, which changes b by up to 2^-126 of itself; and an operation
    whose result is subnormal rounds by up to half of fp32's last step there,
    2^-150, however small it is.  Before h those are the norm after the block
    (two products), the gate's product and the sum: 4 x 2^-150 with factors of
    at most 2 behind them here; on the way to n, h's error and one product of
    its own are multiplied by 1 / s and the weight."""
    got = norm(residual, block=block, gate=gate)
    hv, dh, nv, dn = reference(norm, residual, block, gate)
    b = block.double()
    if norm.post_weight is not None:
        b = b / (b.square().mean(dim=1, keepdim=True) + norm.eps).sqrt() * (norm.weight_offset + norm.post_weight.double())
    lost = 2.0 ** -126 * b.abs() + 8 * 2.0 ** -150
    s = (hv.square().mean(dim=1, keepdim=True) + norm.eps).sqrt()
    tiny = {F32: 2.0 ** -150, BF16: 2.0 ** -134, F16: 2.0 ** -25}   # half of the smallest subnormal
    for name, value, tol in (("residual", hv, dh + lost), ("out", nv, dn + (lost / s + 2.0 ** -150) * (norm.weight_offset + norm.pre_weight.double()).abs())):
        assert bool(value.isfinite().all())
        tol = tol + R.half_step(got[name].dtype) * (value.abs() + tol) + tiny[got[name].dtype]
        off = (got[name].double() - value).abs().nan_to_num(nan=float("inf"))
        bad = off > tol
        assert not bool(bad.any()), (name, bad.nonzero()[:4].tolist(), off[bad][:4].tolist(), tol[bad][:4].tolist())
    assert flag(got["error"]) == 0


@pytest.mark.parametrize("h", [96, 2047, 8200])
@pytest.mark.parametrize("zero", [False, True])
def test_token_gates(h, zero):
    g = R.generator(h)
    n = QUARTERS.numel()
    norm = make(g, h, gate_sigmoid=True)
    block = torch.randn((n, h), generator=g, device=DEV)
    residual = torch.zeros_like(block) if zero else torch.randn((n, h), generator=g, device=DEV)
    check(norm, residual, block, QUARTERS.to(DEV)[:, None].contiguous())


@pytest.mark.parametrize("h", [2403, 9001])
@pytest.mark.parametrize("form", ["channel", "element"])
@pytest.mark.parametrize("post", [True, False])
def test_channel_and_element_gates(h, form, post):
    g = R.generator(h)
    norm = make(g, h, post=post, gate_sigmoid=True)
    for dtype in (F32, BF16, F16):
        block = torch.randn((3, h), generator=g, device=DEV).to(dtype)
        gate = QUARTERS.repeat(-(-h // QUARTERS.numel()))[:h].to(DEV)
        gate = gate.contiguous() if form == "channel" else gate.repeat(3, 1).to(dtype)
        for residual in (torch.zeros((3, h), device=DEV), torch.randn((3, h), generator=g, device=DEV)):
            check(norm, residual, block, gate)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("h", [2048, 16384])
def test_every_16_bit_gate(dtype, h):
    g = R.generator(h)
    gate = torch.arange(65536, device=DEV).to(torch.int32).to(torch.int16).view(dtype).view(-1, h)
    gate = torch.where(gate.isnan(), torch.ones_like(gate), gate)
    norm = make(g, h, gate_sigmoid=True)
    block = torch.randn(gate.shape, generator=g, device=DEV).to(dtype)
    check(norm, torch.zeros(gate.shape, device=DEV), block, gate)


@pytest.mark.parametrize("h", [640, 8200])
def test_nan_gates_stay_in_their_rows(h):
    g = R.generator(h)
    norm = make(g, h, gate_sigmoid=True)
    residual, block = (torch.randn((4, h), generator=g, device=DEV) for _ in range(2))
    gate = torch.randn((4, h), generator=g, device=DEV)
    want = norm(residual, block=block, gate=gate)
    gate[2, 7] = float("nan")
    got = norm(residual, block=block, gate=gate)
    nan = torch.zeros((4, h), dtype=torch.bool, device=DEV)
    nan[2, 7] = True
    assert torch.equal(got["residual"].isnan(), nan)
    assert bool(got["out"][2].isnan().all())
    for k in ("residual", "out"):
        assert torch.equal(got[k][[0, 1, 3]], want[k][[0, 1, 3]])


@pytest.mark.parametrize("h", [640, 8200])
def test_rows_whose_squares_overflow(h):
    """Finite rows of 10^20: the sum is what it is, its norm 0, as are its
    quantised rows, without a flag; other rows are not touched."""
    g = R.generator(h)
    norm = make(g, h, post=False)
    x, block = (torch.randn((3, h), generator=g, device=DEV) for _ in range(2))
    outputs = ("residual", "out", "e4m3")
    want = norm(x, block=block, outputs=outputs)
    x[1] *= 1e20
    got = norm(x, block=block, outputs=outputs)
    assert bool(got["residual"][1].isfinite().all()) and flag(got["error"]) == 0
    assert bool((got["out"][1] == 0).all()) and bool((got["codes"].view(torch.uint8)[1] & 0x7f == 0).all())
    for k in outputs[:2] + ("scales",):
        assert torch.equal(got[k][[0, 2]], want[k][[0, 2]])
