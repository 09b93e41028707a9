"""The int8 calls with an explicit stream= that make their own outputs, while the
current stream is busy and its pending work writes memory that has been freed:
results and flags, copied on the given stream before the current one is through,
are those of the same call on the current stream."""
import pytest

import moe_ffn

torch = pytest.importorskip("torch")
import i8_reference as R  # noqa: E402
from test_gpu_streams import tensors  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16 = torch.float32, torch.bfloat16
H, I, E, K = 256, 128, 32, 4


@pytest.fixture(scope="module", autouse=True)
def gpu_ready():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    yield
    torch.cuda.synchronize()


def calls(n):
    """name -> callable(stream) on n rows, with a NaN row, a bad id, an index outside
    the rows and offsets that decrease where the call takes them."""
    g = R.generator(n)
    x = torch.randn((n, H), generator=g, device=DEV)
    q, s = R.quantise(x)
    nan = x.clone()
    nan[3, 7] = float("nan")
    ids = torch.rand((n, E), generator=g, device=DEV).topk(K, dim=1).indices.to(torch.int32).contiguous()
    ids[2, 1] = -3
    w = torch.softmax(torch.randn((n, K), generator=g, device=DEV), dim=1).contiguous()
    gate, up, down = R.weights(E, I, H, 1), R.weights(E, I, H, 2), R.weights(E, H, I, 3)
    linear = moe_ffn.MoeI8Linear(H, I, gate[0][0], gate[1][0], max_columns=n)
    bank = moe_ffn.MoeI8Bank(E, H, I, *gate)
    layer = moe_ffn.MoeI8Layer(H, I, E, K, False, n, gate, up, down)
    offsets = (torch.arange(E + 1, device=DEV) * n // E).to(torch.int32)
    back = offsets.clone()
    back[E // 2] = 0
    index = torch.arange(n, device=DEV, dtype=torch.int32)
    index[1] = n
    return {
        "quantize": (lambda st: moe_ffn.quantize_i8(nan, stream=st), True),
        "forward": (lambda st: linear.forward(q, s, stream=st), False),
        "apply": (lambda st: linear.apply(nan, stream=st), True),
        "bank": (lambda st: bank.forward(q, s, back, stream=st), True),
        "bank_index": (lambda st: bank.forward(q, s, offsets, index=index, dtype=BF16, stream=st), True),
        "layer": (lambda st: layer.forward(x, ids, w, stream=st), True),
    }


@pytest.mark.parametrize("n", [9, 300])
def test_outputs_belong_to_the_given_stream(n):
    side, busy = torch.cuda.Stream(), {}
    load = torch.randn((8192, 8192), device=DEV, dtype=BF16)
    load @ load
    for name, (call, flagged) in calls(n).items():
        want = [t.clone() for t in tensors(call(None))]
        if flagged:
            assert any(t.dtype == torch.int32 and t.shape == (1,) and int(t[0]) != 0 for t in want), name
        call(side)            # the side stream has memory of its own from here on
        copies = [torch.zeros_like(t) for t in want]
        torch.cuda.synchronize()
        for _ in range(40):   # some tens of milliseconds
            load @ load
        # Freed at once, written when the products are through.
        for t in want:
            for _ in range(3):
                torch.empty_like(t).view(torch.uint8).fill_(0x5a)
        got = tensors(call(side))
        with torch.cuda.stream(side):
            for t, c in zip(got, copies):
                c.copy_(t)
        side.synchronize()
        busy[name] = not torch.cuda.current_stream().query()
        torch.cuda.synchronize()
        for a, b in zip(copies, want):
            assert torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8)), name
    assert all(busy.values()), busy   # no call waited for the current stream
