"""moe_i8_layer_* against the layer in 64 bits (i8_reference.py)."""
import numpy as np
import pytest

import moe_ffn

torch = pytest.importorskip("torch")
import i8_reference as R  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(scope="module", autouse=True)
def gpu_ready():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    yield
    torch.cuda.synchronize()


def flag(e):
    return int(e.cpu()[0])


def matrices(count, rows, cols, seed):
    g = R.generator(seed)
    codes = torch.randn((count, rows, cols), generator=g, device=DEV).mul_(32.0).round_().clamp_(-128, 127).to(torch.int8)
    return codes, (0.6 / 32 / cols ** 0.5) * (0.5 + torch.rand((count, rows), generator=g, device=DEV))


class Case:
    def __init__(self, tokens, h, i, experts, k, shared, seed=0, capacity=None):
        self.bank = [matrices(experts, i, h, seed + 1), matrices(experts, i, h, seed + 2), matrices(experts, h, i, seed + 3)]
        self.shared = [tuple(t[0] for t in matrices(1, *s, seed + 4)) for s in ((i, h), (i, h), (h, i))] if shared else None
        self.layer = moe_ffn.MoeI8Layer(h, i, experts, k, shared, capacity or tokens, *self.bank, shared=self.shared)
        self.k = k
        g = R.generator(seed + 5)
        self.x = torch.randn((tokens, h), generator=g, device=DEV)
        self.ids = torch.rand((tokens, experts), generator=g, device=DEV).topk(k, dim=1).indices.to(torch.int32).contiguous()
        self.w = torch.softmax(torch.randn((tokens, k), generator=g, device=DEV), dim=1).contiguous()
        self.gate = torch.randn(tokens, generator=g, device=DEV) if shared else None

    def check(self, dtype, gate=False):
        x = self.x.to(dtype)
        y, e = self.layer.forward(x, self.ids, self.w, shared_gate=self.gate if gate else None)
        assert flag(e) == 0
        ref = R.layer(x, self.bank, self.shared, self.ids, self.w, self.gate if gate else None)
        bound = R.layer_bound(*ref, self.k, dtype)
        d = (y.double() - ref[0]).abs()
        assert bool((d <= bound).all()), float((d / bound).max())
        return y


SHAPES = [(1, 64, 32, 4, 1, False), (1, 2048, 512, 64, 10, True), (3, 96, 64, 5, 5, True), (8, 2048, 512, 64, 10, True),
          (5, 2560, 640, 32, 10, True), (17, 160, 96, 40, 3, False), (64, 1056, 352, 16, 4, True), (65, 256, 32, 8, 2, True),
          (130, 2048, 512, 8, 2, True), (300, 512, 160, 24, 10, False), (1032, 256, 128, 64, 10, True), (700, 320, 1056, 3, 2, True)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape", SHAPES)
def test_layer(dtype, shape):
    c = Case(*shape, seed=sum(shape))
    c.check(dtype)
    if c.shared:
        c.check(dtype, gate=True)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape", [(40, 160, 512, 64, 4, True), (600, 160, 512, 16, 4, True), (1000, 160, 544, 16, 4, False),
                                   (1000, 2048, 160, 16, 4, True), (100, 512, 1056, 64, 4, True)])
def test_every_tile(dtype, shape):
    """The tiles of the grouped products that the shapes above do not reach."""
    Case(*shape, seed=34).check(dtype, gate=shape[5])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_shared_experts_of_a_small_batch(dtype):
    """Few tokens whose experts are read once for all of them: the same bits for a
    token as in a batch in which its experts are its own."""
    c = Case(64, 4096, 2048, 8, 2, True, seed=35)
    y = c.check(dtype, gate=True)
    for n in (1, 4, 33):
        part, e = c.layer.forward(c.x[:n].to(dtype), c.ids[:n], c.w[:n], shared_gate=c.gate[:n])
        assert flag(e) == 0 and torch.equal(part, y[:n])


def test_one_handle_takes_batches_of_all_sizes():
    """Rows and routes of an earlier, larger batch change nothing."""
    big = Case(600, 256, 64, 16, 4, True, seed=3)
    big.check(F32)
    for n in (1, 9, 64, 66, 257):
        c = Case(n, 256, 64, 16, 4, True, seed=3, capacity=600)
        want, e = c.layer.forward(c.x, c.ids, c.w)
        got, e = big.layer.forward(c.x, c.ids, c.w)
        assert flag(e) == 0 and torch.equal(want, got)
    big.check(F32)


def test_one_expert_takes_all():
    for n in (20, 200):
        c = Case(n, 128, 64, 6, 1, False, seed=n)
        c.ids.fill_(4)
        c.check(BF16)


@pytest.mark.parametrize("n", [6, 40, 300])
def test_bad_routes(n):
    """Bad and repeated ids are dropped and flagged, the rest of the sum stays."""
    c = Case(n, 256, 96, 12, 4, True, seed=n)
    good, e = c.layer.forward(c.x, c.ids, c.w)
    ids, w = c.ids.clone(), c.w.clone()
    ids[1, 2], ids[2, 0], ids[3, 3], ids[4, 1] = 12, -1, ids[3, 0], -2147483648
    y, e = c.layer.forward(c.x, ids, w)
    assert flag(e) == 1
    w2 = w.clone()
    w2[1, 2] = w2[2, 0] = w2[3, 3] = w2[4, 1] = 0.0     # the dropped routes
    ref = R.layer(c.x, c.bank, c.shared, c.ids, w2, None)
    assert bool(((y.double() - ref[0]).abs() <= R.layer_bound(*ref, 4, F32)).all())
    keep = torch.tensor([i for i in range(n) if i not in (1, 2, 3, 4)], device=DEV)
    assert torch.equal(y[keep], good[keep])
    # every route of a token bad: the shared expert is left
    ids[0] = -7
    y, e = c.layer.forward(c.x, ids, w)
    ref = R.layer(c.x[:1], c.bank, c.shared, c.ids[:1, :0], c.w[:1, :0], None)
    assert flag(e) == 1 and bool(((y[:1].double() - ref[0]).abs() <= R.layer_bound(*ref, 4, F32)).all())


@pytest.mark.parametrize("n", [4, 100])
def test_nonfinite_values(n):
    c = Case(n, 256, 96, 12, 4, True, seed=9)
    good, _ = c.layer.forward(c.x, c.ids, c.w, shared_gate=c.gate)
    keep = torch.tensor([i for i in range(n) if i != 2], device=DEV)
    alone = R.layer(c.x[2:3], c.bank, c.shared, c.ids[2:3, :0], c.w[2:3, :0], c.gate[2:3])
    x = c.x.clone()
    x[2, 17] = float("inf")                         # the token counts as zeros
    y, e = c.layer.forward(x, c.ids, c.w, shared_gate=c.gate)
    assert flag(e) == 1 and not y[2].any() and torch.equal(y[keep], good[keep])
    w = c.w.clone()
    w[2, 1] = float("nan")                          # gives up the routed sum
    y, e = c.layer.forward(c.x, c.ids, w, shared_gate=c.gate)
    assert flag(e) == 1 and torch.equal(y[keep], good[keep])
    assert bool(((y[2:3].double() - alone[0]).abs() <= R.layer_bound(*alone, 4, F32)).all())
    gate = c.gate.clone()
    gate[2] = float("nan")                          # gives up the token
    y, e = c.layer.forward(c.x, c.ids, c.w, shared_gate=gate)
    assert flag(e) == 1 and not y[2].any() and torch.equal(y[keep], good[keep])
    w = c.w.clone()
    w[2, 0] = -0.25                                 # flagged, and stays in the sum
    y, e = c.layer.forward(c.x, c.ids, w, shared_gate=c.gate)
    ref = R.layer(c.x, c.bank, c.shared, c.ids, w, c.gate)
    assert flag(e) == 1 and bool(((y.double() - ref[0]).abs() <= R.layer_bound(*ref, 4, F32)).all())


def test_nonfinite_weight_scales():
    """A nonfinite scale gives up what it reaches: its elements of the outputs of
    the tokens that its expert has, or its part of the middle."""
    for n in (4, 100):
        c = Case(n, 256, 96, 12, 4, True, seed=10)
        good, _ = c.layer.forward(c.x, c.ids, c.w)
        e0 = int(c.ids[0, 0])
        hit = (c.ids == e0).any(dim=1)
        down = c.bank[2][1].clone()
        down[e0, 33] = float("inf")
        layer = moe_ffn.MoeI8Layer(256, 96, 12, 4, True, n, c.bank[0], c.bank[1], (c.bank[2][0], down), shared=c.shared)
        y, e = layer.forward(c.x, c.ids, c.w)
        assert flag(e) & 1 and bool(torch.isfinite(y).all())
        other = torch.arange(256, device=DEV) != 33
        assert torch.equal(y[:, other], good[:, other]) and torch.equal(y[~hit], good[~hit])
        gate = c.bank[0][1].clone()
        gate[e0, 5] = float("nan")
        layer = moe_ffn.MoeI8Layer(256, 96, 12, 4, True, n, (c.bank[0][0], gate), c.bank[1], c.bank[2], shared=c.shared)
        y, e = layer.forward(c.x, c.ids, c.w)
        assert flag(e) & 1 and bool(torch.isfinite(y).all()) and torch.equal(y[~hit], good[~hit])


@pytest.mark.parametrize("down,up", [(120, -60), (-120, 40), (100, -60), (-95, 40)])
def test_scales_at_the_ends_of_their_range(down, up):
    """Scales of the down matrices, or of one expert's, far from 1: bf16 results
    within the bound, and as the fp32 ones where fp16 cannot hold an output on the
    way."""
    n = 100
    c = Case(n, 256, 96, 12, 4, True, seed=33)
    x = c.x.to(BF16)
    some = torch.zeros((12, 1), device=DEV)
    some[3] = 1.0
    for d in (torch.ones_like(some), some):
        bank = [c.bank[0], (c.bank[1][0], c.bank[1][1] * 2.0 ** (up * d)), (c.bank[2][0], c.bank[2][1] * 2.0 ** (down * d))]
        layer = moe_ffn.MoeI8Layer(256, 96, 12, 4, True, n, *bank, shared=c.shared)
        y, e = layer.forward(x, c.ids, c.w)
        full, f = layer.forward(x.float(), c.ids, c.w)
        assert flag(e) == 0 and flag(f) == 0
        ref = R.layer(x, bank, c.shared, c.ids, c.w, None)
        assert bool(((y.double() - ref[0]).abs() <= R.layer_bound(*ref, 4, BF16)).all())
        assert bool(((full.double() - ref[0]).abs() <= R.layer_bound(*ref, 4, F32)).all())
        if abs(down) == 120:
            assert torch.equal(y, full.to(BF16))


def test_host_weights():
    c = Case(12, 96, 64, 6, 2, True, seed=11)
    host = lambda m: tuple(np.ascontiguousarray(t.cpu().numpy()) for t in m)  # noqa: E731
    layer = moe_ffn.MoeI8Layer(96, 64, 6, 2, True, 12, *[host(m) for m in c.bank], shared=[host(m) for m in c.shared])
    a, _ = c.layer.forward(c.x, c.ids, c.w)
    b, _ = layer.forward(c.x, c.ids, c.w)
    assert torch.equal(a, b)


@pytest.mark.parametrize("n", [4, 200])
def test_graph_replay(n):
    c = Case(n, 512, 128, 16, 4, True, seed=12)
    x, ids, w = torch.zeros_like(c.x), torch.zeros_like(c.ids), torch.zeros_like(c.w)
    ids.copy_(c.ids)
    y, e = torch.zeros_like(x), torch.zeros(1, dtype=torch.int32, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.layer.bind_forward(x, ids, w, y, e, shared_gate=c.gate)()
    for seed in range(4):
        g = R.generator(seed)
        x.copy_(torch.randn(x.shape, generator=g, device=DEV))
        ids.copy_(torch.rand((n, 16), generator=g, device=DEV).topk(4, dim=1).indices)
        w.copy_(torch.softmax(torch.randn(w.shape, generator=g, device=DEV), dim=1))
        graph.replay()
        torch.cuda.synchronize()
        eager, flags = c.layer.forward(x, ids, w, shared_gate=c.gate)
        assert torch.equal(eager, y) and flag(e) == 0 and flag(flags) == 0


def test_same_bits_every_time():
    c = Case(500, 512, 256, 32, 8, True, seed=13)
    first, _ = c.layer.forward(c.x, c.ids, c.w)
    for _ in range(5):
        assert torch.equal(first, c.layer.forward(c.x, c.ids, c.w)[0])


def test_refusals():
    c = Case(4, 64, 32, 4, 2, True, seed=14)
    with pytest.raises(ValueError):
        c.layer.forward(torch.zeros((5, 64), device=DEV), c.ids, c.w)       # more tokens than the layer has room for
    with pytest.raises(TypeError):
        c.layer.forward(c.x.double(), c.ids, c.w)
    with pytest.raises(ValueError):
        c.layer.forward(c.x, c.ids[:3], c.w)
    with pytest.raises(TypeError):
        c.layer.forward(c.x, c.ids.long(), c.w)
    with pytest.raises(ValueError):
        c.layer.forward(c.x, c.ids, c.w, y=torch.zeros((4, 96), device=DEV)[:, :64])
    e = torch.zeros(1, dtype=torch.int32, device=DEV)
    call = c.layer.bind_forward(c.x, c.ids, c.w, torch.zeros_like(c.x), e)
    c.layer.close()
    with pytest.raises(moe_ffn.MoeError):
        call()


@pytest.mark.parametrize("n", [3, 150])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_stack(dtype, n):
    """int8 layers, projections and routers in a MoeStack, with norms between the
    layers: the steps one by one, and as a replayed graph."""
    h, i, experts, k, depth = 256, 96, 32, 4, 3
    cases = [Case(n, h, i, experts, k, True, seed=20 + l) for l in range(depth)]
    projections, routers, norms = [], [], []
    for l in range(depth):
        pc, ps = matrices(1, h, h, 40 + l)
        rc, rs = matrices(1, experts, h, 50 + l)
        projections.append(moe_ffn.MoeI8Linear(h, h, pc[0], ps[0], max_columns=n))
        routers.append(moe_ffn.MoeI8Linear(h, experts, rc[0], rs[0], max_columns=n))
    for l in range(depth + 1):
        g = R.generator(60 + l)
        norms.append(moe_ffn.BlockNorm(h, pre_weight=torch.rand(h, generator=g, device=DEV)))
    stack = moe_ffn.MoeStack([c.layer for c in cases], projections, routers, norms)
    x = cases[0].x.to(dtype)
    stack.bind([x])
    stack.run()
    eager = [t.clone() for t in stack.outputs()]
    residual, normed = x, norms[0](x, outputs=("out",))["out"]
    for l in range(depth):
        p, _ = projections[l].apply(normed)
        logits, _ = routers[l].apply(p, dtype=F32)
        ids, w, _, _ = moe_ffn.router_select(logits, top_k=k)
        y, _ = cases[l].layer.forward(p, ids, w)
        out = norms[l + 1](residual, block=y)
        residual, normed = out["residual"], out["out"]
    assert torch.equal(eager[0], residual) and torch.equal(eager[1], normed) and flag(stack.error) == 0
    stack.capture()
    for _ in range(3):
        stack.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(stack.outputs(), eager))


@pytest.mark.parametrize("tokens,k", [(65536, 32), (40000, 3)])
def test_largest_batches(tokens, k):
    """Rows, routes and groups at the ends of their ranges; the first and last
    tokens against 64 bits, and the rest against the same tokens in a batch of
    their own."""
    c = Case(tokens, 32, 32, 40, k, True, seed=30)
    y, e = c.layer.forward(c.x, c.ids, c.w, shared_gate=c.gate)
    assert flag(e) == 0
    for part in (slice(0, 300), slice(tokens // 2 - 50, tokens // 2 + 50), slice(tokens - 300, tokens)):
        ref = R.layer(c.x[part], c.bank, c.shared, c.ids[part], c.w[part], c.gate[part])
        assert bool(((y[part].double() - ref[0]).abs() <= R.layer_bound(*ref, k, F32)).all())
        again, _ = c.layer.forward(c.x[part], c.ids[part], c.w[part], shared_gate=c.gate[part])
        assert torch.equal(again, y[part])


@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 63, 64, 65, 204, 205])
def test_limits_between_kernels(n):
    """Either side of the sizes at which other kernels take over: the same bits
    for a token whatever its batch (fp32)."""
    c = Case(210, 320, 96, 24, 10, True, seed=31)
    whole, e = c.layer.forward(c.x, c.ids, c.w, shared_gate=c.gate)
    part, f = c.layer.forward(c.x[:n], c.ids[:n], c.w[:n], shared_gate=c.gate[:n])
    assert flag(e) == 0 and flag(f) == 0
    ref = R.layer(c.x[:n], c.bank, c.shared, c.ids[:n], c.w[:n], c.gate[:n])
    assert bool(((part.double() - ref[0]).abs() <= R.layer_bound(*ref, 10, F32)).all())
    assert torch.equal(whole[:n], part)


@pytest.mark.parametrize("n", [5, 300])
def test_on_a_stream_of_its_own(n):
    c = Case(n, 256, 96, 12, 4, True, seed=32)
    want, _ = c.layer.forward(c.x, c.ids, c.w)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    got, e = c.layer.forward(c.x, c.ids, c.w, stream=side)
    side.synchronize()
    assert torch.equal(got, want) and flag(e) == 0
