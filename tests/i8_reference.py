"""Restatement of the 8-bit integer formats and operators for the tests: codes
and scales of x as the format defines them (fp32 operations, each rounded on its
own), everything else in 64 bits."""
import torch

EPS = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}   # half a step, relative
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}   # a subnormal's step


def generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def quantise(x):
    """(codes int8, scales fp32) of finite rows.  Divisions of fp32 numbers in 64
    bits, rounded, are the correctly rounded fp32 quotients."""
    v = x.float()
    a = v.abs().amax(dim=1).clamp_min(2.0 ** -100).double()
    return (v * (127.0 / a).float()[:, None]).round().to(torch.int8), (a / 127.0).float()


def weights(count, rows, cols, seed):
    """int8 matrices over the whole range of codes, -128 among them, with scales
    over two powers of ten."""
    g = generator(seed)
    codes = torch.randint(-128, 128, (count, rows, cols), generator=g, device="cuda", dtype=torch.int32).to(torch.int8)
    scales = 1e-3 * torch.exp(4.6 * torch.rand((count, rows), generator=g, device="cuda"))
    return codes, scales


def sums(x, w):
    """The whole-number sums, in 64 bits."""
    return x.double() @ w.double().T


def product(x, sx, w, sw):
    return sums(x, w) * sx.double()[:, None] * sw.double()


def product_bound(ref, dtype):
    """|y - ref| of a product: the sum made fp32, the product of the scales, their
    product (2^-24 each, and second-order terms), y's own rounding."""
    return ref.abs() * (3.01 * 2.0 ** -24 + EPS[dtype] * (1 + 2.0 ** -20)) + TINY[dtype]


def close(y, ref, dtype):
    assert y.dtype == dtype
    d = (y.double() - ref).abs()
    assert bool((d <= product_bound(ref, dtype)).all()), float((d / product_bound(ref, dtype)).max())


def middle(x, sx, gate, up):
    """(SiLU(g) u in 64 bits, a bound of a kernel's error in it).  g and u have
    three roundings; SiLU turns g's relative error into at most 1 + |g| times
    that; its sigmoid is within 8 half ulps, and three products follow."""
    g, u = product(x, sx, *gate), product(x, sx, *up)
    m = g * torch.sigmoid(g) * u
    return m, m.abs() * ((3.01 * g.abs() + 18) * 2.0 ** -24) + u.abs() * 2.0 ** -120


def expert(x, sx, gate, up, down):
    """(One expert's output in 64 bits, a bound of what its middle row's codes may
    change, half a step of the smallest fp16 numbers in which an output may be held
    on the way to a bf16 sum: 2^-25 sx 2^-p with 2^-p < 2 I max |sw|).

    A code may be the neighbour of the exact one where the middle's error reaches
    the border between the two."""
    m, err = middle(x, sx, gate, up)
    a = m.abs().amax(dim=1, keepdim=True).clamp_min(2.0 ** -100)
    rel = (err / a).amax(dim=1, keepdim=True) + 2.0 ** -22     # of the scale
    v = m * (127 / a)
    far = 127 / a * err + v.abs() * rel
    codes, s = torch.round(v), (a / 127)[:, 0]
    near = ((v - torch.floor(v) - 0.5).abs() <= far).double()
    c = product(codes, s, *down)
    slack = product(near, s, down[0].double().abs(), down[1].abs()) + c.abs() * rel
    return c, slack, (2.0 ** -24 * m.shape[1] * float(down[1].abs().max())) * s[:, None]


def layer(x, bank, shared, ids, w, gate):
    """(y in 64 bits, sum of the magnitudes that it adds up, sum of the half steps,
    sum of the codes' bounds)."""
    q, s = quantise(x)
    n, k = ids.shape
    y = torch.zeros((n, x.shape[1]), dtype=torch.float64, device=x.device)
    size, slack = torch.zeros_like(y), torch.zeros_like(y)
    steps = torch.zeros((n, 1), dtype=torch.float64, device=x.device)

    def add(t, f, args):
        c, more, step = expert(*args)
        y.index_add_(0, t, f * c)
        size.index_add_(0, t, (f * c).abs())
        slack.index_add_(0, t, f.abs() * more)
        steps.index_add_(0, t, f.abs() * step)
    for e in torch.unique(ids).tolist():
        t, r = torch.nonzero(ids == e, as_tuple=True)
        add(t, w[t, r].double()[:, None], (q[t], s[t], *[(codes[e], scales[e]) for codes, scales in bank]))
    if shared is not None:
        f = torch.ones((n, 1), dtype=torch.float64, device=x.device) if gate is None else torch.sigmoid(gate.double())[:, None]
        add(torch.arange(n, device=x.device), f, (q, s, *shared))
    return y, size, steps, slack


def layer_bound(y, size, steps, slack, k, dtype):
    """A contribution has three roundings of its own, one of its weight and up to
    five in its gate's sigmoid; each of k + 1 sums has one.  Where y is bf16 the
    contributions may have been fp16, each rounded by 2^-11 of itself or half a
    step."""
    e = size * ((k + 11) * 2.0 ** -24) + slack
    if dtype == torch.bfloat16:
        e = e + size * (2.0 ** -11 + 2.0 ** -22) + steps
    return e + (y.abs() + e) * EPS[dtype] * (1 + 2.0 ** -10) + TINY[dtype]
