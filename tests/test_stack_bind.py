"""What MoeStack.bind makes and refuses, without a GPU: the handles are empty
shells of their classes and no run is made."""
import pytest

import moe_ffn

torch = pytest.importorskip("torch")

H, E, K = 64, 32, 4
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def shell(kind, **attributes):
    m = object.__new__(kind)
    m.__dict__.update(dict(H=H, E=E, k=K, K=H, M=H, max_tokens=64, max_columns=64, device=0, handle=None), **attributes)
    return m


def norm(final=True, hidden=H):
    return shell(moe_ffn.BlockNorm, hidden=hidden, pre_weight=torch.ones(hidden) if final else None)


def q4(n=2):
    return [shell(moe_ffn.MoeLayer) for _ in range(n)]


def fp8(n=2):
    return [shell(moe_ffn.MoeFp8Layer) for _ in range(n)]


def routes(n):
    return torch.zeros((n, K), dtype=torch.int32), torch.zeros((n, K))


@pytest.mark.parametrize("layers", [q4(3), fp8(3)])
def test_fewer_batches_take_the_first_layers(layers):
    S = moe_ffn.MoeStack(layers, routers=[shell(moe_ffn.MoeLinear) for _ in layers])
    S.bind([torch.zeros((5, H)), torch.zeros((2, H))])
    assert [tuple(y.shape) for y in S.outputs()] == [(5, H), (2, H)] and len(S.steps) == 2
