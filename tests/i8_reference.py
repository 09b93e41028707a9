"""Restatement of the 8-bit integer formats and operators for the tests: codes,
scales and middle rows as the formats define them (fp32 operations, each rounded
on its own), everything after them in 64 bits."""
import numpy as np
import torch

import moe_ffn

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
    """fp32 SiLU(g) u with every operation rounded as the kernels round it."""
    def rows(w):
        s = sx.float()[:, None].cpu() * w[1].float().cpu()
        return sums(x, w[0]).cpu().float() * s
    g, u = rows(gate), rows(up)
    e = torch.from_numpy(moe_ffn.expf_host((-g).numpy().astype(np.float32)))
    return ((g / (1.0 + e)) * u).to(x.device)


def expert(x, sx, gate, up, down):
    """One expert's output in 64 bits, from its middle row's codes."""
    m, sm = quantise(middle(x, sx, gate, up))
    return product(m, sm, *down)


def half_step(x, sx, gate, up, down):
    """Half a step of the smallest fp16 numbers in which an expert's output may be
    held on the way to a bf16 sum: 2^-25 sx 2^-p with 2^-p < 2 I max |sw|."""
    _, sm = quantise(middle(x, sx, gate, up))
    return (2.0 ** -24 * up[0].shape[0] * float(down[1].abs().max())) * sm.double()[:, None]


def layer(x, bank, shared, ids, w, gate):
    """(y in 64 bits, sum of the magnitudes that it adds up, sum of their half steps)."""
    q, s = quantise(x)
    n, k = ids.shape
    y = torch.zeros((n, x.shape[1]), dtype=torch.float64, device=x.device)
    size, steps = torch.zeros_like(y), torch.zeros((n, 1), dtype=torch.float64, device=x.device)
    for e in torch.unique(ids).tolist():
        t, r = torch.nonzero(ids == e, as_tuple=True)
        args = (q[t], s[t], *[(codes[e], scales[e]) for codes, scales in bank])
        f = w[t, r].double()[:, None]
        c = f * expert(*args)
        y.index_add_(0, t, c)
        size.index_add_(0, t, c.abs())
        steps.index_add_(0, t, f.abs() * half_step(*args))
    if shared is not None:
        f = 1.0 if gate is None else torch.sigmoid(gate.double())[:, None]
        c = f * expert(q, s, *shared)
        y, size, steps = y + c, size + c.abs(), steps + f * half_step(q, s, *shared)
    return y, size, steps


def layer_bound(y, size, k, dtype, steps=0.0):
    """A contribution has three roundings of its own, one of its weight and up to
    five in its gate's sigmoid; each of k + 1 sums has one.  Where y is bf16 the
    contributions may have been fp16, each rounded by 2^-11 of itself or half a
    step."""
    half = size * (2.0 ** -11 + 2.0 ** -22) + steps if dtype == torch.bfloat16 else 0.0
    return size * ((k + 11) * 2.0 ** -24) + half + (y.abs() + half) * EPS[dtype] * (1 + 2.0 ** -10) + TINY[dtype]
