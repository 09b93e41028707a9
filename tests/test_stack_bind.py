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


@pytest.mark.parametrize("kind", [BF16, F16])
def test_16_bit_rows_of_q4_handles_are_refused(kind):
    x = torch.zeros((3, H), dtype=kind)
    linears = lambda t: [shell(t) for _ in range(2)]  # noqa: E731
    q, e = moe_ffn.MoeLinear, moe_ffn.MoeFp8Linear
    norms = [norm() for _ in range(3)]
    ids, w = routes(3)
    for layers, projections, routers, bad in ((q4(), None, None, True), (q4(), linears(e), None, True),
                                              (fp8(), linears(q), None, True), (fp8(), linears(e), linears(q), True),
                                              (fp8(1) + q4(1), None, linears(e), True),
                                              (fp8(), linears(e), linears(e), False), (fp8(), None, None, False)):
        for stream in (None, norms):
            S = moe_ffn.MoeStack(layers, projections, routers, norms=stream)
            args = ([x] if stream else [x, x], [ids] * 2, [w] * 2)
            if bad:
                with pytest.raises(TypeError, match="float32"):
                    S.bind(*args)
                assert not hasattr(S, "steps")   # nothing half bound
            else:
                S.bind(*args)
                assert all(st["y"].dtype == kind for st in S.steps)
            S.bind([t.float() for t in args[0]], *args[1:])   # as fp32 rows they are taken
            assert all(st["y"].dtype == F32 for st in S.steps)


def test_dtype_and_stream():
    """16-bit blocks may run on an fp32 stream, not the other way round."""
    ids, w = routes(3)
    S = moe_ffn.MoeStack(fp8(), norms=[norm() for _ in range(3)])
    S.bind([torch.zeros((3, H))], [ids] * 2, [w] * 2, dtype=BF16)
    assert S.residual.dtype == F32 and S.steps[0]["y"].dtype == S.last["out"].dtype == BF16
    for x, dtype in ((BF16, F32), (BF16, F16)):
        with pytest.raises(TypeError):
            S.bind([torch.zeros((3, H), dtype=x)], [ids] * 2, [w] * 2, dtype=dtype)
    with pytest.raises(TypeError):
        moe_ffn.MoeStack(q4(), norms=[norm() for _ in range(3)]).bind([torch.zeros((3, H))], [ids] * 2, [w] * 2, dtype=BF16)


def test_rows_of_norms():
    """Only the rows that a layer reads are made: e4m3 rows alone for an e4m3
    projection."""
    ids, w = routes(3)
    norms = [norm() for _ in range(3)]
    S = moe_ffn.MoeStack(fp8(), [shell(moe_ffn.MoeFp8Linear) for _ in range(2)], norms=norms)
    S.bind([torch.zeros((3, H))], [ids] * 2, [w] * 2)
    assert all("x" not in st and set(st["norm"]) == {"codes", "scales"} for st in S.steps)
    S = moe_ffn.MoeStack(q4(), norms=norms)
    S.bind([torch.zeros((3, H))], [ids] * 2, [w] * 2)
    assert all(set(st["norm"]) == {"out", "q8"} for st in S.steps)


def test_norms_that_do_not_fit():
    with pytest.raises(ValueError):
        moe_ffn.MoeStack([], norms=[norm()])
    with pytest.raises(ValueError):
        moe_ffn.MoeStack(fp8(1), norms=[norm(), norm(hidden=32)])
    with pytest.raises(ValueError):
        moe_ffn.MoeStack(fp8(1), norms=[norm(final=False), norm()])
    ids, w = routes(3)
    with pytest.raises(ValueError):
        moe_ffn.MoeStack(fp8(1), norms=[norm(), norm()]).bind([torch.zeros((3, H))] * 2, [ids], [w])


def test_batches_past_the_handles_are_refused():
    """A batch larger than a layer's, a projection's or a router's capacity, and
    rows of another width, before anything runs."""
    ids, w = routes(9)
    small = dict(max_tokens=8, max_columns=8)
    linears = lambda **a: [shell(moe_ffn.MoeFp8Linear, **a)]  # noqa: E731
    for layers, projections, routers in (([shell(moe_ffn.MoeFp8Layer, **small)], None, None),
                                         ([shell(moe_ffn.MoeLayer, **small)], None, None),
                                         (fp8(1), linears(**small), None), (fp8(1), None, linears(**small)),
                                         (fp8(1), [shell(moe_ffn.MoeLinear, **small)], None)):
        S = moe_ffn.MoeStack(layers, projections, routers)
        with pytest.raises(ValueError):
            S.bind([torch.zeros((9, H))], [ids], [w])
        S.bind([torch.zeros((8, H))], [ids[:8]], [w[:8]])
        with pytest.raises(ValueError):
            S.bind([torch.zeros((8, H + 1))], [ids[:8]], [w[:8]])
        with pytest.raises(ValueError):
            S.bind([torch.zeros((0, H))], [ids[:0]], [w[:0]])
    # A projection that takes the norm's e4m3 rows needs no workspace.
    S = moe_ffn.MoeStack(fp8(1), linears(max_columns=0), norms=[norm(), norm()])
    S.bind([torch.zeros((9, H))], [ids], [w])
