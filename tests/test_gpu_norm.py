"""moe_block_norm against its formulas in 64 bits, with bounds that follow from
the fp32 operations on the way; its Q8_1 and e4m3 rows against the framework's
quantisers, bit for bit."""
import pytest

import moe_ffn

torch = pytest.importorskip("torch")
import fp8_reference as R  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U = 2.0 ** -24


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


def reference(norm, residual, block, gate):
    """(h, dh, n, dn): values and bounds of a fp32 evaluation, float64.  A sum
    of squares passes through at most 16 + 6 + 16 additions (elements of a
    thread, lanes, waves), each off by U of a sum of positive terms; mean, eps,
    root and quotient add 4 U; a product or quotient U each; a sigmoid is within
    8 U (exponential and reciprocal 2 U each, the sum, the argument)."""
    sums = 40 * U
    r = residual.double() * norm.residual_scale
    h, dh = r, U * r.abs()
    if block is not None:
        b = block.double()
        rel = 0.0
        if norm.post_weight is not None:
            b = b / (b.square().mean(dim=1, keepdim=True) + norm.eps).sqrt()
            b = b * (norm.weight_offset + norm.post_weight.double())
            rel = sums / 2 + 8 * U
        if gate is not None:
            g = gate.double()
            b = b * (torch.sigmoid(g) if norm.gate_sigmoid else g)
            rel = rel + 10 * U
        b = b * norm.block_scale
        h = r + b
        dh = b.abs() * (rel + 2 * U) + U * r.abs() + U * h.abs()
    if norm.pre_weight is None:
        return h, dh, None, None
    s = (h.square().mean(dim=1, keepdim=True) + norm.eps).sqrt()
    w = norm.weight_offset + norm.pre_weight.double()
    n = h / s * w
    # ms off by 2 |h| dh on average; the root halves it
    rel = (2 * h.abs() * dh + dh.square()).mean(dim=1, keepdim=True) / s.square() / 2 + sums / 2 + 8 * U
    return h, dh, n, n.abs() * rel + (dh / s * w.abs()) * (1 + rel)


def near(got, ref, tol, what):
    tiny = 2.0 ** -25 if got.dtype == F16 else 2.0 ** -149
    tol = tol + R.half_step(got.dtype) * (ref.abs() + tol) + tiny
    off = (got.double() - ref).abs()
    assert bool((off <= tol).all()), (what, float((off / tol).max()))


def make(g, hidden, post=True, pre=True, **kw):
    w = lambda: 0.1 * torch.randn(hidden, generator=g, device=DEV)  # noqa: E731
    return moe_ffn.BlockNorm(hidden, pre_weight=w() if pre else None, post_weight=w() if post else None, **kw)


def gates(form, n, h, dtype, g):
    shape = {"none": None, "token": (n, 1), "channel": (h,), "element": (n, h)}[form]
    if shape is None:
        return None
    return torch.randn(shape, generator=g, device=DEV).to(dtype if form == "element" else F32)


# One row to more than a grid holds; one channel to 16384, odd, of one wave, of
# two elements' groups a thread; every gate, with and without the norm after.
CASES = [(1, 2048, True, "none"), (1, 1, True, "element"), (3, 7, False, "channel"), (5, 8, True, "token"),
         (2, 512, False, "none"), (9, 520, True, "channel"), (4, 1000, True, "element"), (3, 2047, True, "token"),
         (17, 2560, False, "element"), (2, 8192, True, "none"), (3, 8200, True, "channel"), (2, 16384, True, "element"),
         (4999, 640, True, "token"), (4999, 96, False, "none")]


@pytest.mark.parametrize("n,h,post,form", CASES)
@pytest.mark.parametrize("dtype,rtype", [(F32, F32), (BF16, BF16), (BF16, F32), (F16, F16), (F16, F32)])
def test_values(n, h, post, form, dtype, rtype):
    g = R.generator(n * 7 + h)
    norm = make(g, h, post=post, weight_offset=1.0, residual_scale=0.75, block_scale=1.5, gate_sigmoid=n % 2 == 1)
    block = (torch.randn((n, h), generator=g, device=DEV) * 3).to(dtype)
    residual = torch.randn((n, h), generator=g, device=DEV).to(rtype)
    gate = gates(form, n, h, dtype, g)
    got = norm(residual, block=block, gate=gate)
    hv, dh, nv, dn = reference(norm, residual, block, gate)
    assert got["residual"].dtype == rtype and got["out"].dtype == dtype and flag(got["error"]) == 0
    near(got["residual"], hv, dh, "residual")
    near(got["out"], nv, dn, "out")


@pytest.mark.parametrize("n,h", [(1, 2048), (3, 33), (700, 1024), (2, 16384)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_first_and_last_form(n, h, dtype):
    """The norm before a first block (no block), and after a last one (no norm
    of the sum)."""
    g = R.generator(h)
    x = torch.randn((n, h), generator=g, device=DEV).to(dtype)
    first = make(g, h, post=False, weight_offset=0.0)
    got = first(x, outputs=("out",))
    _, _, nv, dn = reference(first, x, None, None)
    near(got["out"], nv, dn, "out")
    last = make(g, h, pre=False)
    got = last(x, block=x * 2, outputs=("residual",))
    hv, dh, _, _ = reference(last, x, x * 2, None)
    near(got["residual"], hv, dh, "residual")


@pytest.mark.parametrize("n,h", [(1, 32), (3, 96), (5, 2048), (300, 640), (2, 2560), (3, 16384)])
def test_quantised_rows_are_the_quantisers(n, h):
    g = R.generator(h + 1)
    norm = make(g, h)
    residual, block = (torch.randn((n, h), generator=g, device=DEV) for _ in range(2))
    got = norm(residual, block=block, outputs=("residual", "out", "q8", "e4m3"))
    q8, e = moe_ffn.quantize_q8_1(got["out"])
    codes, scales, f = moe_ffn.quantize_e4m3(got["out"])
    assert flag(e) == flag(f) == flag(got["error"]) == 0
    assert same(got["q8"], q8) and same(got["codes"], codes) and same(got["scales"], scales)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("h", [1000, 2047, 640])
def test_e4m3_rows_of_16_bit_blocks(dtype, h):
    """The rows are of the fp32 norm, not of its 16-bit rounding, and a group
    that the row's end cuts short is of the elements that are there."""
    g = R.generator(h)
    norm = make(g, h)
    residual, block = (torch.randn((40, h), generator=g, device=DEV).to(dtype) for _ in range(2))
    got = norm(residual, block=block, outputs=("e4m3",))
    _, _, nv, dn = reference(norm, residual, block, None)
    v, slack = R.quantise_with_slack(nv, dn)
    off = (R.rows(got["codes"], got["scales"]) - v).abs()
    assert bool((off <= slack + U * v.abs()).all())


def test_strides_and_in_place():
    """Rows inside wider tensors at starts no vector load fits; the sum written
    over the residual and the norm over the block."""
    n, h = 6, 200
    g = R.generator(2)
    norm = make(g, h, weight_offset=1.0)
    wide = [torch.randn((n, h + 11), generator=g, device=DEV).to(BF16) for _ in range(3)]
    residual, block, gate = (w[:, 3:3 + h] for w in wide)
    want = norm(residual, block=block, gate=gate, outputs=("residual", "out", "e4m3"))
    dense = norm(residual.contiguous(), block=block.contiguous(), gate=gate.contiguous(), outputs=("residual", "out", "e4m3"))
    for k in ("residual", "out", "codes", "scales"):
        assert same(want[k], dense[k]), k
    edges = [w.clone() for w in wide]
    norm.bind(residual, block=block, gate=gate, residual_out=residual, out=block)()
    assert same(residual, want["residual"]) and same(block, want["out"])
    for w, before in zip(wide[:2], edges[:2]):
        assert same(w[:, :3], before[:, :3]) and same(w[:, 3 + h:], before[:, 3 + h:])


def test_special_rows():
    """Zero rows stay zero; a row with an infinity or NaN is its own affair; its
    quantised groups are flagged and zero."""
    n, h = 5, 384
    g = R.generator(3)
    norm = make(g, h)
    residual, block = (torch.randn((n, h), generator=g, device=DEV) for _ in range(2))
    residual[1] = 0
    block[1] = 0
    block[2, 5] = float("nan")
    residual[3, 300] = float("inf")
    got = norm(residual, block=block, outputs=("residual", "out", "q8", "e4m3"))
    assert flag(got["error"]) & 1
    assert bool((got["out"][1] == 0).all()) and bool((got["residual"][1] == 0).all())
    assert bool(got["out"][2].isnan().all()) and bool((got["codes"][2].view(torch.uint8) == 0).all())
    assert bool((got["scales"][2] == 0).all()) and bool((got["q8"][2] == 0).all())
    assert bool((got["residual"][3].isinf() == (torch.arange(h, device=DEV) == 300)).all())
    keep = [0, 4]
    clean = norm(residual[keep], block=block[keep], outputs=("residual", "out", "q8", "e4m3"))
    assert flag(clean["error"]) == 0
    for k in ("residual", "out", "q8", "codes", "scales"):
        assert same(got[k][keep], clean[k]), k


def test_graph_replay():
    n, h = 40, 2048
    g = R.generator(4)
    norm = make(g, h)
    residual, block = (torch.randn((n, h), generator=g, device=DEV).to(BF16) for _ in range(2))
    out, res = torch.empty_like(block), torch.empty_like(residual)
    norm.bind(residual, block=block, residual_out=res, out=out)()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm.bind(residual, block=block, residual_out=res, out=out)()
    for _ in range(3):
        residual.normal_(generator=g)
        want = norm(residual, block=block)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert same(out, want["out"]) and same(res, want["residual"])


def test_refusals():
    g = R.generator(5)
    norm = make(g, 64)
    x = torch.zeros((2, 64), device=DEV)
    out = torch.zeros_like(x)
    for kw in (dict(block=x[:, :32]), dict(block=x[:1]), dict(gate=torch.zeros(64, device=DEV)), dict(out=out[:1]),
               dict(block=x, gate=torch.zeros(3, device=DEV)), dict(codes=torch.zeros((2, 64), dtype=torch.uint8, device=DEV)),
               dict(), dict(block=x.cpu())):
        with pytest.raises(ValueError):
            norm.bind(x, **{"out": out, **kw} if kw else kw)
    for kw in (dict(block=x.double()), dict(block=x, gate=torch.zeros((2, 64), dtype=BF16, device=DEV)),
               dict(block=x.to(BF16), out=out), dict(block=x, residual_out=out.to(BF16))):
        with pytest.raises(TypeError):
            norm.bind(x, **{"out": out, **kw})
    with pytest.raises(TypeError):   # a 16-bit residual of another type than the block's
        norm.bind(x.to(BF16), block=x.to(F16), out=out.to(F16))
    with pytest.raises(ValueError):
        make(g, 64, pre=False).bind(x, block=x, out=out)
    with pytest.raises(ValueError):
        make(g, 50)(torch.zeros((2, 50), device=DEV), outputs=("q8",))
    with pytest.raises(ValueError):
        moe_ffn.BlockNorm(64)
    with pytest.raises(ValueError):
        make(g, 64, eps=0.0)
    with pytest.raises(moe_ffn.MoeError):
        norm.bind(x[:0], out=out[:0])()


def test_rows_past_32_bits():
    """65,536 rows of residual, block and outputs inside a buffer of more than
    2^32 elements."""
    n, h = 65536, 96
    g = R.generator(6)
    norm = make(g, h)
    buf = torch.full((n, 65700), 3.0, dtype=BF16, device=DEV)
    residual, block = buf[:, 65600:65600 + h], buf[:, 5:5 + h]
    residual.normal_(generator=g)
    block.normal_(generator=g)
    want = norm(residual.contiguous(), block=block.contiguous())
    norm.bind(residual, block=block, residual_out=residual, out=block)()
    assert same(residual, want["residual"]) and same(block, want["out"])
    assert bool((buf[:, 5 + h:65600] == 3).all()) and bool((buf[:, 65600 + h:] == 3).all())


def test_bound_call_keeps_the_weights():
    n, h = 3, 256
    g = R.generator(7)
    norm = make(g, h)
    x = torch.randn((n, h), generator=g, device=DEV)
    want = norm(x, block=x)["out"]
    out = torch.empty_like(x)
    call = norm.bind(x, block=x, out=out)
    del norm
    other = [torch.full((h,), 9.0, device=DEV) for _ in range(64)]   # would take the weights' memory
    call()
    assert same(out, want) and len(other) == 64
