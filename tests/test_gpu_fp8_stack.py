"""MoeStack with norms, on e4m3 and on Q4 handles: the operators in a run, as
a model's blocks use them.  Each stage is compared with its formula in 64 bits
on the inputs that the run itself gave it, and a captured run with the eager
one, replay for replay."""
import numpy as np
import pytest

import moe_ffn
import workloads as W

torch = pytest.importorskip("torch")
import fp8_reference as R  # noqa: E402
from test_gpu_fp8_layer import Bank, Values  # noqa: E402
from test_gpu_norm import near, reference  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16 = torch.float32, torch.bfloat16
H, I, E, K, LAYERS = 256, 128, 32, 4, 3


@pytest.fixture(scope="module", autouse=True)
def gpu_ready():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    yield
    torch.cuda.synchronize()


def same(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


def norms(g, final):
    w = lambda: 0.1 * torch.randn(H, generator=g, device=DEV)  # noqa: E731
    out = [moe_ffn.BlockNorm(H, pre_weight=w(), weight_offset=1.0)]
    for l in range(LAYERS):
        last = l == LAYERS - 1
        out.append(moe_ffn.BlockNorm(H, pre_weight=None if last and not final else w(), post_weight=w(), weight_offset=1.0,
                                     residual_scale=0.9, block_scale=0.5))
    return out


def linear_near(y, x, w, bound_dtype=None):
    ref = x @ w.T
    tol = R.linear_tolerance(x, w, ref, y.dtype, False)
    assert bool(((y.double() - ref).abs() <= tol).all())


@pytest.mark.parametrize("n,final,dtype", [(1, True, BF16), (11, False, BF16), (64, True, F32)])
def test_fp8_stack(n, final, dtype):
    g = R.generator(n)
    banks = [Bank(H, I, E, True, g) for _ in range(LAYERS)]
    layers = [b.layer(K, n) for b in banks]
    pw, rw = ([R.random_matrix(m, H, g) for _ in range(LAYERS)] for m in (H, E))
    projections = [moe_ffn.MoeFp8Linear(H, H, *w, max_columns=n) for w in pw]
    routers = [moe_ffn.MoeFp8Linear(H, E, *w, max_columns=n) for w in rw]
    ns = norms(g, final)
    x = torch.randn((n, H), generator=g, device=DEV).to(F32 if n == 11 else dtype)   # also an fp32 stream of 16-bit blocks
    S = moe_ffn.MoeStack(layers, projections, routers, norms=ns)
    S.bind([x], dtype=dtype)
    seen = []

    def keep(l, outputs, stream, norm=S._norm):   # the stream before and after each norm
        before = (S.x if l <= 1 else S.residual).clone()
        norm(l, outputs, stream)
        seen.append((before, S.residual.clone()))
    S._norm = keep
    S.run()
    torch.cuda.synchronize()
    del S._norm
    assert int(S.error.cpu()[0]) == 0
    for l, st in enumerate(S.steps):
        before, after = seen[l]
        block = S.steps[l - 1]["y"] if l else None
        hv, dh, nv, dn = reference(ns[l], before, block, None)
        if l:
            near(after, hv, dh, l)
        v, slack = R.quantise_with_slack(nv, dn)
        assert bool(((R.rows(st["codes"], st["scales"]) - v).abs() <= slack + 2.0 ** -24 * v.abs()).all())
        linear_near(st["h"], R.rows(st["codes"], st["scales"]), R.matrix(*pw[l]))
        linear_near(st["logits"], R.rows(*R.quantise(st["h"])), R.matrix(*rw[l]))
        ids, w, _, _ = moe_ffn.router_select(st["logits"], top_k=K)
        assert torch.equal(ids, st["ids"]) and same(w, st["w"])
        ref, tol = R.layer(st["h"], ids, w, Values(banks[l]), banks[l].values(E))
        near(st["y"], ref, tol, l)
    hv, dh, nv, dn = reference(ns[-1], seen[-1][0], S.steps[-1]["y"], None)
    outs = S.outputs()
    near(outs[0], hv, dh, "stream")
    assert len(outs) == 1 + final
    if final:
        near(outs[1], nv, dn, "final")
    eager = [o.clone() for o in outs]
    S.capture()
    for i in range(3):
        for o in outs:
            o.zero_()
        S.replay()
        torch.cuda.synchronize()
        assert all(same(a, b) for a, b in zip(outs, eager)), i
        layers[0].forward(S.steps[0]["h"], S.steps[0]["ids"], S.steps[0]["w"])   # eager work between
    S.graph = None
    for m in layers + projections + routers:
        m.close()


@pytest.mark.parametrize("n,projected", [(3, False), (40, False), (3, True)])
def test_q4_stack(n, projected):
    """Q4 layers take the norm's Q8_1 rows, or a Q4 projection of its values:
    the same bits as the operators one by one."""
    g = R.generator(n)
    rng = np.random.default_rng(n)
    layers = [moe_ffn.MoeLayer(H, I, E, K, True, n, synthetic_seed=50 + l) for l in range(LAYERS)]
    q4 = lambda m: moe_ffn.MoeLinear(moe_ffn.TYPE_Q4_0, H, m, W.q4_blocks(m * H // 32, rng).reshape(-1), max_columns=n)  # noqa: E731
    routers = [q4(E) for _ in range(LAYERS)]
    projections = [q4(H) for _ in range(LAYERS)] if projected else None
    ns = norms(g, True)
    x = torch.randn((n, H), generator=g, device=DEV)
    S = moe_ffn.MoeStack(layers, projections, routers, norms=ns)
    S.bind([x])
    S.run()
    res, block = x, None
    for l, L in enumerate(layers):
        got = ns[l](res, block=block)
        res, h = (got["residual"], got["out"]) if l else (res, got["out"])
        if projected:
            h, _ = projections[l].apply(h)
        ids, w, _, _ = moe_ffn.router_select(routers[l].apply(h)[0], top_k=K)
        block, _ = L.forward(h, ids, w)
        assert same(block, S.steps[l]["y"])
    got = ns[-1](res, block=block)
    assert same(got["residual"], S.outputs()[0]) and same(got["out"], S.outputs()[1])
    assert int(S.error.cpu()[0]) == 0
    for m in layers + routers + (projections or []):
        m.close()


def test_fp8_stack_without_norms():
    """Each layer on its own batch, e4m3 and Q4 handles side by side."""
    g = R.generator(77)
    bank = Bank(H, I, E, False, g)
    layers = [bank.layer(K, 5), moe_ffn.MoeLayer(H, I, E, K, True, 9, synthetic_seed=3)]
    rw = [R.random_matrix(E, H, g) for _ in layers]
    routers = [moe_ffn.MoeFp8Linear(H, E, *w, max_columns=9) for w in rw]
    xs = [torch.randn((5, H), generator=g, device=DEV).to(BF16), torch.randn((9, H), generator=g, device=DEV)]
    S = moe_ffn.MoeStack(layers, routers=routers)
    S.bind(xs)
    S.run()
    torch.cuda.synchronize()
    for L, r, x, st in zip(layers, routers, xs, S.steps):
        logits = r.apply(x, dtype=F32)[0]
        ids, w, _, _ = moe_ffn.router_select(logits, top_k=K)
        assert same(logits, st["logits"]) and torch.equal(ids, st["ids"])
        assert same(L.forward(x, ids, w)[0], st["y"])
    with pytest.raises(ValueError):
        moe_ffn.MoeStack(layers, norms=norms(g, True))   # two layers take three norms
    for m in layers + routers:
        m.close()
