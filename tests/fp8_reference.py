"""The 8-bit floating point formats and products in 64 bits, for the tests.

Codes and scales are part of the format and are formed as it defines them
(each operation correctly rounded to fp32); everything after them is float64.
"""
import torch

GROUP = 128


def e4m3_table():
    """The value of each code, float64 (OCP E4M3FN: 0x7f and 0xff are NaN)."""
    c = torch.arange(256)
    e, m = (c >> 3) & 15, (c & 7).double()
    v = torch.where(e > 0, (1 + m / 8) * torch.exp2(e.double() - 7), m * 2.0 ** -9)
    v = torch.where(c >= 128, -v, v)
    v[0x7f] = v[0xff] = float("nan")
    return v


def codes_to_values(codes):
    return e4m3_table().to(codes.device)[codes.view(torch.uint8).long()]


def blocks(n):
    return -(-n // GROUP)


def spread(scales, dim, size):
    """A scale per 128 along `dim` -> one per element."""
    return scales.double().repeat_interleave(GROUP, dim=dim).narrow(dim, 0, size)


def matrix(codes, scales):
    rows, cols = codes.shape
    return codes_to_values(codes) * spread(spread(scales, 0, rows), 1, cols)


def rows(codes, scales):
    return codes_to_values(codes) * spread(scales, 1, codes.shape[1])


def quantise(x):
    """Finite rows -> (codes uint8, scales float32), nearest even."""
    n, k = x.shape
    x = x.float()
    v = torch.nn.functional.pad(x, (0, blocks(k) * GROUP - k)).view(n, -1, GROUP)
    a = v.abs().amax(dim=2).clamp_min(2.0 ** -100).double()
    s, r = (a / 448).float(), (448 / a).float()
    t = (v * r[..., None]).double()            # one fp32 multiplication
    e = torch.frexp(t.abs().clamp_min(2.0 ** -20)).exponent.double()
    step = torch.exp2((e - 4).clamp_min(-9.0))
    q = (torch.round(t.abs() / step) * step).clamp_max(448.0)
    mag = torch.searchsorted(e4m3_table()[:0x7f].contiguous().to(x.device), q.contiguous())
    codes = (mag + 128 * (torch.signbit(t)).long()).to(torch.uint8)
    return codes.view(n, -1)[:, :k].contiguous(), s


def random_matrix(m, k, g, device="cuda"):
    """Codes of values about N(0, 0.02) and their scales."""
    codes = (torch.randn((m, k), generator=g, device=device) * 110).clamp(-448, 448).to(torch.float8_e4m3fn)
    scales = (0.02 / 110) * (0.5 + torch.rand((blocks(m), blocks(k)), generator=g, device=device))
    return codes, scales


def generator(seed, device="cuda"):
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    return g


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def product_bounds(x, w, nb):
    """(sum of |x w| over K, sum over the blocks of the largest |x w|), per
    output, for rows x and matrix w in float64."""
    total = x.abs() @ w.abs().T
    peak = torch.zeros_like(total)
    for b in range(nb):
        xs, ws = x[:, b * GROUP:(b + 1) * GROUP].abs(), w[:, b * GROUP:(b + 1) * GROUP].abs()
        for n0 in range(0, x.shape[0], 64):
            part = torch.zeros((min(64, x.shape[0] - n0), w.shape[0]), dtype=torch.float64, device=x.device)
            for k in range(xs.shape[1]):
                part = torch.maximum(part, xs[n0:n0 + 64, k, None] * ws[None, :, k])
            peak[n0:n0 + 64] += part
    return total, peak


def linear_tolerance(x, w, y, dtype, wide):
    """How far a product may be from y (float64), by arithmetic: within a block
    the matrix instruction adds 128 products, and the accumulator adds one term
    per block, each addition off by at most 2^-23 of the sum of magnitudes
    (truncation included), the two scale products by 2 half steps; then y's own
    rounding, half a step (fp16: at least half its smallest subnormal).  `wide`: 16-bit
    results of more than 64 columns come from the e4m3 instruction, in which
    each of a block's 128 products may lose up to 2^-13 of the largest."""
    nb = blocks(x.shape[1])
    if wide and dtype != torch.float32:
        total, peak = product_bounds(x, w, nb)
        extra = 128 * 2.0 ** -13 * peak
    else:
        total, extra = x.abs() @ w.abs().T, 0.0
    tol = (128 + nb + 2) * 2.0 ** -23 * total + extra
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    return tol + half_step(dtype) * (y.abs() + tol) + tiny


def quantise_with_slack(m, slack):
    """Rows m (float64) as e4m3 values, and how far each may be from what a
    kernel gives whose m is off by up to `slack`: one step where the scaled
    value lies within the slack of a rounding boundary, else the slack of the
    scale alone."""
    codes, s = quantise(m)
    v = rows(codes, s)
    n, k = m.shape
    pad = lambda t: torch.nn.functional.pad(t, (0, blocks(k) * GROUP - k)).view(n, -1, GROUP)  # noqa: E731
    a = pad(m.abs()).amax(dim=2).clamp_min(2.0 ** -100)
    rel = spread(pad(slack).amax(dim=2) / a + 2.0 ** -22, 1, k)      # of the scale
    sd = spread(s, 1, k)
    t, dt = m / sd, slack / sd + (m / sd).abs() * rel
    # The two values next to t: a kernel's code may be any between the
    # roundings of t - dt and t + dt.
    r = lambda z: _round(z.clamp(-448, 448))  # noqa: E731
    spread_ = torch.maximum((r(t + dt) - v / sd).abs(), (r(t - dt) - v / sd).abs())
    return v, spread_ * sd + v.abs() * rel


def _round(t):
    e = torch.frexp(t.abs().clamp_min(2.0 ** -20)).exponent.double()
    step = torch.exp2((e - 4).clamp_min(-9.0))
    return torch.round(t / step) * step


def expert(x, gate, up, down):
    """(output, tolerance) of one expert for rows x (e4m3 values), float64:
    the tolerance is that of fp32 sums, carried through SiLU(g) u (slope of
    SiLU at most 1.1) and the rounding of the middle."""
    g, u = x @ gate.T, x @ up.T
    dg, du = (linear_tolerance(x, w, y, torch.float32, False) for w, y in ((gate, g), (up, u)))
    silu = g * torch.sigmoid(g)
    m = silu * u
    dm = 1.1 * dg * (u.abs() + du) + silu.abs() * du + 8 * 2.0 ** -24 * m.abs()
    v, dv = quantise_with_slack(m, dm)
    y = v @ down.T
    return y, dv @ down.abs().T + linear_tolerance(v, down, y, torch.float32, False)


def layer(x, ids, weights, experts, shared=None, gate=None):
    """(output, tolerance) of a layer, float64; routes with a bad id or a
    repeated one are dropped.  experts[e] = (gate, up, down) in float64."""
    codes, s = quantise(x)
    q = rows(codes, s)
    n, k = ids.shape
    y = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(y)
    size = torch.zeros_like(y)
    use = {}
    for t, row in enumerate(ids.tolist()):
        for r, e in enumerate(row):
            if 0 <= e < len(experts) and e not in row[:r]:
                use.setdefault(e, []).append((t, r))
    for e, where in use.items():
        t, r = (torch.tensor(i, device=q.device) for i in zip(*where))
        out, d = expert(q[t], *experts[e])
        w = weights[t, r].double()[:, None]
        y.index_add_(0, t, w * out)
        tol.index_add_(0, t, w.abs() * d)
        size.index_add_(0, t, (w * out).abs())
    if shared is not None:
        out, d = expert(q, *shared)
        w = torch.ones(n, device=q.device).double() if gate is None else torch.sigmoid(gate.double())
        y += w[:, None] * out
        tol += w[:, None] * (d + 4 * 2.0 ** -24 * out.abs())
        size += (w[:, None] * out).abs()
    return y, tol + (k + 3) * 2.0 ** -24 * size


# ------------------------------------------------- the e4m3 instruction ---
def _exponents(codes):
    """The power of two of each code, -6 for subnormal ones."""
    e = (codes.view(torch.uint8).long() >> 3) & 15
    return torch.where(e > 0, e - 7, -6).double()


def e4m3_instruction(xc, xs, wc, ws, block_rows):
    """(y, tolerance): products of e4m3 rows xc (scales xs) and matrix rows wc
    (scales ws, of the blocks of rows `block_rows`) as the e4m3 matrix
    instruction sums them, float64.  Of eight neighbouring products, with 2^e
    the largest power of two among them, each keeps what lies at or above 2^(e -
    13), toward zero; those sums are exact (18 bits).  What is left is fp32: 16
    sums of eight added within a block and one term a block, each addition off
    by at most 2^-23 of the magnitudes, and two products with scales (half of that
    each)."""
    n, k = xc.shape
    nb = blocks(k)
    y = torch.zeros((n, wc.shape[0]), dtype=torch.float64, device=xc.device)
    size = torch.zeros_like(y)
    xv, wv, xe, we = codes_to_values(xc), codes_to_values(wc), _exponents(xc), _exponents(wc)
    sw = ws[block_rows].double()
    for k0 in range(0, k, 8):
        at = slice(k0, min(k, k0 + 8))
        p = xv[:, None, at] * wv[None, :, at]
        e = torch.where(p == 0, -100.0, xe[:, None, at] + we[None, :, at]).amax(dim=2, keepdim=True)
        grid = torch.exp2(e - 13)
        part = (torch.trunc(p / grid) * grid).sum(dim=2)
        s = xs.double()[:, k0 // GROUP, None] * sw[None, :, k0 // GROUP]
        y += part * s
        size += part.abs() * s
    return y, (16 + nb + 2) * 2.0 ** -23 * size
