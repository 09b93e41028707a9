"""moe_fp8_layer_* against the layer in 64 bits (fp8_reference.py), with
tolerances that follow from the additions and roundings on the way: fp32 sums,
and a whole step of the middle's e4m3 codes only where its value lies within
those sums' error of a rounding boundary."""
import pytest

import moe_ffn

torch = pytest.importorskip("torch")
import fp8_reference as R  # noqa: E402

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


def same(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


class Bank:
    """Random e4m3 experts, as a handle takes them and in float64."""

    def __init__(self, H, I, E, shared, g):
        self.H, self.I, self.E = H, I, E
        self.parts = []
        for rows, cols in ((I, H), (I, H), (H, I)):
            codes, scales = zip(*[R.random_matrix(rows, cols, g) for _ in range(E + shared)])
            self.parts.append((torch.stack([c.view(torch.uint8) for c in codes]), torch.stack(scales)))
        self.shared = [(c[E], s[E]) for c, s in self.parts] if shared else None
        self.experts = [(c[:E], s[:E]) for c, s in self.parts]

    def values(self, e):
        return tuple(R.matrix(c[e], s[e]) for c, s in self.parts)

    def layer(self, k, tokens):
        return moe_ffn.MoeFp8Layer(self.H, self.I, self.E, k, self.shared is not None, tokens, *self.experts,
                                   shared=self.shared)


class Values:
    """experts[e] in float64, made when first asked for."""

    def __init__(self, bank):
        self.bank, self.got = bank, {}

    def __len__(self):
        return self.bank.E

    def __getitem__(self, e):
        return self.got.setdefault(e, self.bank.values(e))


def routes(n, E, k, g):
    ids = torch.rand((n, E), generator=g, device=DEV).topk(k, dim=1).indices.to(torch.int32).contiguous()
    return ids, torch.softmax(torch.randn((n, k), generator=g, device=DEV), dim=1).contiguous()


def check(y, x, ids, w, bank, gate):
    ref, tol = R.layer(x, ids, w, Values(bank), bank.values(bank.E) if bank.shared else None, gate)
    tol = tol + R.half_step(y.dtype) * (ref.abs() + tol) + (2.0 ** -25 if y.dtype == F16 else 0.0)
    off = (y.double() - ref).abs()
    assert bool((off <= tol).all()), float((off / tol).max())
    if ref.norm() > 0:   # few codes change: the result as a whole is close
        assert float((y.double() - ref).norm() / ref.norm()) <= 2e-3 + R.half_step(y.dtype)


# One token to 64; one expert that every token shares (four column groups) to
# 512; hidden and intermediate sizes whose last blocks are cut, of one block
# and of 128 (which gate/up takes in pieces); 1 to 32 routes a token.
CASES = [(1, 64, 32, 4, 2, True), (1, 2048, 512, 64, 10, True), (3, 96, 160, 8, 8, False), (64, 128, 96, 1, 1, True),
         (64, 256, 352, 5, 2, False), (17, 416, 64, 40, 32, True), (33, 640, 288, 16, 3, True), (2, 16384, 32, 3, 1, True),
         (9, 32, 16384, 3, 2, False), (20, 4128, 128, 6, 6, True), (8, 2048, 512, 512, 10, True), (5, 2560, 640, 48, 10, True),
         (64, 4096, 64, 40, 32, True)]


@pytest.mark.parametrize("T,H,I,E,k,shared", CASES)
def test_layer(T, H, I, E, k, shared):
    g = R.generator(T * 100 + E)
    bank = Bank(H, I, E, shared, g)
    layer = bank.layer(k, T)
    for dtype in (F32, BF16, F16):
        x = torch.randn((T, H), generator=g, device=DEV).to(dtype)
        ids, w = routes(T, E, k, g)
        gate = torch.randn(T, generator=g, device=DEV) if dtype != F16 else None
        y, e = layer.forward(x, ids, w, shared_gate=gate)
        assert y.dtype == dtype and flag(e) == 0
        check(y, x, ids, w, bank, gate)
        again, _ = layer.forward(x, ids, w, shared_gate=gate)
        assert same(y, again)
    layer.close()


def test_batch_of_one_equals_its_rows_in_a_batch():
    """A token's result does not depend on the batch it comes in."""
    g = R.generator(3)
    bank = Bank(384, 192, 12, True, g)
    layer = bank.layer(4, 20)
    x = torch.randn((20, 384), generator=g, device=DEV)
    ids, w = routes(20, 12, 4, g)
    y, _ = layer.forward(x, ids, w)
    for t in (0, 7, 19):
        one, _ = layer.forward(x[t:t + 1].contiguous(), ids[t:t + 1].contiguous(), w[t:t + 1].contiguous())
        assert same(one[0], y[t])
    layer.close()


def test_bad_routes():
    """Bad ids and repeats are dropped and flagged; a token all of whose routes
    are bad gets the shared expert alone; weights out of range are flagged."""
    g = R.generator(4)
    E, k, T = 6, 3, 7
    bank = Bank(128, 64, E, True, g)
    layer = bank.layer(k, T)
    x = torch.randn((T, 128), generator=g, device=DEV)
    good, w = routes(T, E, k, g)
    for change in ("negative", "large", "repeat", "all", "weight", "nan"):
        ids, v, want_w = good.clone(), w.clone(), w.clone()
        if change == "negative":
            ids[2, 1] = -5
        elif change == "large":
            ids[0, 0] = E
            ids[6, 2] = 2 ** 31 - 1
        elif change == "repeat":
            ids[3, 2] = ids[3, 0]
            ids[4, 1] = ids[4, 0]
        elif change == "all":
            ids[5] = -1
        elif change == "weight":
            v[1, 1] = want_w[1, 1] = -0.5
        else:
            v[1, 0], want_w[1, 0] = float("nan"), 0.0
        y, e = layer.forward(x, ids, v)
        assert flag(e) == 1, change
        if change == "nan":   # the token's routed sum is given up, its shared expert stays
            want_w[1] = 0.0
        check(y, x, ids, want_w, bank, None)
    layer.close()
    bare = Bank(128, 64, E, False, g)
    layer = bare.layer(k, T)
    ids = good.clone()
    ids[5] = E + 1
    y, e = layer.forward(x, ids, w)
    assert flag(e) == 1 and bool((y[5] == 0).all())
    check(y, x, ids, w, bare, None)
    layer.close()


def test_nonfinite_input():
    """A group with an infinity or NaN counts as zeros and is flagged, also
    where none of the token's routes is good."""
    g = R.generator(5)
    bank = Bank(384, 96, 5, False, g)
    layer = bank.layer(2, 6)
    x = torch.randn((6, 384), generator=g, device=DEV)
    ids, w = routes(6, 5, 2, g)
    clean, dirty = x.clone(), x.clone()
    clean[1, :128] = 0
    clean[4, 256:] = 0
    dirty[1, 3] = float("nan")
    dirty[4, 300] = -float("inf")
    a, e = layer.forward(dirty, ids, w)
    b, f = layer.forward(clean, ids, w)
    assert flag(e) == 1 and flag(f) == 0 and same(a, b)
    ids[1] = -1
    x = clean.clone()
    x[1, 200] = float("inf")
    assert flag(layer.forward(x, ids, w)[1]) == 1
    layer.close()


def test_zero_rows_and_untouched_tail():
    g = R.generator(6)
    bank = Bank(256, 128, 4, True, g)
    layer = bank.layer(2, 8)
    x = torch.randn((8, 256), generator=g, device=DEV)
    x[3] = 0
    ids, w = routes(8, 4, 2, g)
    out = torch.full((9, 256), 5.0, device=DEV)
    e = torch.zeros(1, dtype=torch.int32, device=DEV)
    layer.forward(x, ids, w, y=out[:8], error=e)
    assert bool((out[3] == 0).all()) and bool((out[8] == 5).all()) and flag(e) == 0
    check(out[:8], x, ids, w, bank, None)
    layer.close()


def test_weights_from_host():
    g = R.generator(7)
    bank = Bank(160, 96, 3, True, g)
    host = lambda pairs: [(c.cpu().numpy(), s.cpu().numpy()) for c, s in pairs]  # noqa: E731
    a = bank.layer(2, 4)
    b = moe_ffn.MoeFp8Layer(160, 96, 3, 2, True, 4, *host(bank.experts), shared=host(bank.shared))
    x = torch.randn((4, 160), generator=g, device=DEV)
    ids, w = routes(4, 3, 2, g)
    assert same(a.forward(x, ids, w)[0], b.forward(x, ids, w)[0])
    a.close()
    b.close()


def test_two_layers_on_two_streams_and_a_graph():
    g = R.generator(8)
    banks = [Bank(512, 128, 10, True, g) for _ in range(2)]
    layers = [b.layer(4, 16) for b in banks]
    x = torch.randn((16, 512), generator=g, device=DEV).to(BF16)
    ids, w = routes(16, 10, 4, g)
    want = [l.forward(x, ids, w)[0] for l in layers]
    streams = [torch.cuda.Stream() for _ in layers]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for l, s in zip(layers, streams):
            with torch.cuda.stream(s):
                got.append(l.forward(x, ids, w)[0])
    torch.cuda.synchronize()
    assert all(same(y, want[i % 2]) for i, y in enumerate(got))
    y, e = torch.empty_like(x), torch.zeros(1, dtype=torch.int32, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layers[0].forward(x, ids, w, y=y, error=e)
    for _ in range(3):
        x.normal_(generator=g)
        eager, _ = layers[0].forward(x, ids, w)
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert same(y, eager) and flag(e) == 0
    for l in layers:
        l.close()


def test_refusals():
    g = R.generator(9)
    bank = Bank(64, 32, 4, True, g)
    layer = bank.layer(2, 4)
    x = torch.zeros((4, 64), device=DEV)
    ids, w = routes(4, 4, 2, g)
    with pytest.raises(ValueError):
        layer.forward(torch.zeros((5, 64), device=DEV), *routes(5, 4, 2, g))
    with pytest.raises(ValueError):
        layer.forward(x[:0], ids[:0], w[:0])
    with pytest.raises(TypeError):
        layer.forward(x.double(), ids, w)
    with pytest.raises(TypeError):
        layer.forward(x, ids.long(), w)
    with pytest.raises(TypeError):
        layer.forward(x, ids, w, y=torch.empty((4, 64), dtype=BF16, device=DEV))
    with pytest.raises(ValueError):
        layer.forward(x, ids[:, :1], w[:, :1])
    raw = torch.zeros(4 * 64 + 1, device=DEV)
    with pytest.raises(moe_ffn.MoeError) as ex:   # x must start on 16 bytes
        layer.forward(raw[1:].view(4, 64), ids, w)
    assert ex.value.status == 1
    with pytest.raises(ValueError):
        moe_ffn.MoeFp8Layer(64, 32, 4, 2, True, 4, *bank.experts)
    with pytest.raises(ValueError):
        moe_ffn.MoeFp8Layer(64, 32, 5, 2, True, 4, *bank.experts, shared=bank.shared)
    with pytest.raises(moe_ffn.MoeError):
        moe_ffn.MoeFp8Layer(64, 32, 4, 2, True, 65, *bank.experts, shared=bank.shared)
    layer.close()


def test_bank_past_32_bits():
    """Matrices of 17 GB a kind, which also take more than one launch to lay
    out: every expert's tiles are where the products look for them."""
    H, I, E, k, T = 2048, 2080, 4096, 4, 5
    if torch.cuda.mem_get_info()[0] < 80 << 30:
        pytest.skip("needs 80 GiB of free device memory")
    g = R.generator(10)
    codes = torch.empty((E, I, H), dtype=torch.uint8, device=DEV)
    codes.random_(generator=g).bitwise_and_(0xBF)   # below 2: no NaN
    parts = [(codes, torch.rand((E, 17, 16), generator=g, device=DEV) * 0.02) for _ in range(2)]
    parts.append((codes.view(E, H, I), torch.rand((E, 16, 17), generator=g, device=DEV) * 0.02))
    layer = moe_ffn.MoeFp8Layer(H, I, E, k, False, T, *parts)
    x = torch.randn((T, H), generator=g, device=DEV).to(BF16)
    ids, w = routes(T, E, k, g)
    ids[0] = torch.tensor([E - 1, 0, E // 2, E - 2], device=DEV)
    ids[1] = torch.tensor([4032, 4033, 1024, 1023], device=DEV)

    class Experts:
        def __len__(self):
            return E

        def __getitem__(self, e):
            return tuple(R.matrix(c[e], s[e]) for c, s in parts)

    y, e = layer.forward(x, ids, w)
    ref, tol = R.layer(x, ids, w, Experts())
    tol = tol + R.half_step(BF16) * (ref.abs() + tol)
    assert flag(e) == 0 and bool(((y.double() - ref).abs() <= tol).all())
    layer.close()


def test_bound_call_keeps_the_layer():
    g = R.generator(12)
    bank = Bank(64, 32, 4, True, g)
    layer = bank.layer(2, 3)
    x = torch.randn((3, 64), generator=g, device=DEV)
    ids, w = routes(3, 4, 2, g)
    y, e = torch.empty_like(x), torch.zeros(1, dtype=torch.int32, device=DEV)
    want, _ = layer.forward(x, ids, w)
    call = layer.bind_forward(x, ids, w, y, e)
    del layer
    call()
    assert same(y, want)
    layer = bank.layer(2, 3)
    call = layer.bind_forward(x, ids, w, y, e)
    layer.close()
    with pytest.raises(moe_ffn.MoeError):
        call()
