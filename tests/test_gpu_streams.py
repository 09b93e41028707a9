"""Calls with an explicit stream= that make their own outputs, while the current
stream is busy and its pending work writes memory that has been freed: results
and flags are those of the same call on the current stream."""
import pytest

import moe_ffn
import numpy as np
import workloads as W

torch = pytest.importorskip("torch")
import fp8_reference as R  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16 = torch.float32, torch.bfloat16
H, I, E, K, N = 256, 128, 32, 4, 9


@pytest.fixture(scope="module", autouse=True)
def gpu_ready():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    yield
    torch.cuda.synchronize()


def tensors(out):
    if isinstance(out, torch.Tensor):
        return [out]
    if isinstance(out, dict):
        out = out.values()
    return [t for t in out if t is not None]


def calls():
    """name -> callable(stream): every call that makes outputs of its own, on
    inputs that raise a flag where the call has one."""
    g = R.generator(1)
    rng = np.random.default_rng(1)
    x = torch.randn((N, H), generator=g, device=DEV)
    x[3, 7] = float("nan")
    ok = torch.randn((N, H), generator=g, device=DEV)
    ids = torch.rand((N, E), generator=g, device=DEV).topk(K, dim=1).indices.to(torch.int32).contiguous()
    bad = ids.clone()
    bad[2, 1] = -3
    w = torch.softmax(torch.randn((N, K), generator=g, device=DEV), dim=1).contiguous()
    layer = moe_ffn.MoeLayer(H, I, E, K, True, N, synthetic_seed=2)
    linear = moe_ffn.MoeLinear(moe_ffn.TYPE_Q4_0, H, I, W.q4_blocks(I * H // 32, rng).reshape(-1), max_columns=N)
    matrices = lambda n, rows, cols: tuple(torch.stack(t) for t in zip(*[R.random_matrix(rows, cols, g) for _ in range(n)]))  # noqa: E731
    bank = [(c.view(torch.uint8), s) for c, s in (matrices(E, I, H), matrices(E, I, H), matrices(E, H, I))]
    fp8 = moe_ffn.MoeFp8Layer(H, I, E, K, False, N, *bank)
    fp8_linear = moe_ffn.MoeFp8Linear(H, I, *R.random_matrix(I, H, g), max_columns=N)
    norm = moe_ffn.BlockNorm(H, pre_weight=torch.ones(H, device=DEV))
    q8, _ = moe_ffn.quantize_q8_1(ok)
    mq, _ = moe_ffn.quantize_q8_1(torch.randn((N, I), generator=g, device=DEV))
    codes, scales, _ = moe_ffn.quantize_e4m3(ok)
    logits = torch.randn((N, E), generator=g, device=DEV)
    logits[5, 2] = float("nan")
    parts = torch.randn((N, K, H), generator=g, device=DEV)
    parts[4, 1, 9] = float("inf")
    torch.cuda.synchronize()
    return {
        "quantize_e4m3": lambda s: moe_ffn.quantize_e4m3(x, stream=s),
        "fp8_linear_forward": lambda s: fp8_linear.forward(codes, scales, stream=s),
        "fp8_linear_apply": lambda s: fp8_linear.apply(x, stream=s),
        "fp8_layer": lambda s: fp8.forward(ok, bad, w, stream=s),
        "norm": lambda s: norm(x, outputs=("residual", "out", "q8", "e4m3"), stream=s),
        "quantize_q8_1": lambda s: moe_ffn.quantize_q8_1(x, stream=s),
        "linear_forward_q8": lambda s: linear.forward_q8(q8, N, stream=s),
        "linear_apply": lambda s: linear.apply(x, stream=s),
        "layer": lambda s: layer.forward(x, ids, w, stream=s),
        "layer_q8": lambda s: layer.forward_q8(q8, bad, w, stream=s),
        "router": lambda s: moe_ffn.router_select(logits, top_k=K, probabilities=True, stream=s),
        "combine": lambda s: moe_ffn.combine(parts, w, stream=s),
        "groups": lambda s: {k: layer.group_routes(bad, w, stream=s)[k] for k in ("counts", "offsets", "error")},
        "gate_up": lambda s: layer.expert_gate_up(1, q8, N, dots=True, stream=s),
        "down": lambda s: layer.expert_down(1, mq, N, dots=True, stream=s),
        "expf": lambda s: moe_ffn.expf_device(ok, stream=s),
    }


FLAGGED = ("quantize_e4m3", "fp8_linear_apply", "fp8_layer", "norm", "quantize_q8_1", "linear_apply", "layer", "layer_q8",
           "router", "combine", "groups")


def test_outputs_belong_to_the_given_stream():
    side, busy = torch.cuda.Stream(), []
    load = torch.randn((8192, 8192), device=DEV, dtype=BF16)
    load @ load
    for name, call in calls().items():
        want = [t.clone() for t in tensors(call(None))]
        if name in FLAGGED:
            assert any(t.dtype == torch.int32 and t.shape == (1,) and int(t[0]) != 0 for t in want), name
        call(side)            # the side stream has memory of its own from here on
        torch.cuda.synchronize()
        for _ in range(12):   # some milliseconds
            load @ load
        # Freed at once, written when the products are through.
        for t in want:
            for _ in range(3):
                torch.empty_like(t).view(torch.uint8).fill_(0x5a)
        got = tensors(call(side))
        side.synchronize()
        busy.append(not torch.cuda.current_stream().query())
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8)), name
    assert any(busy)   # the calls on the side stream did not wait
