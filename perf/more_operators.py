"""Measured cases of the 8-bit integer operators: int8 matrices with a scale per
output channel, int8 activations with a scale per token.

Four operators, each in its plain form (elementary torch operations in 32 bits)
and, where `own` is true, through the framework's entry points:

  rows     x -> int8 codes and one fp32 scale per row
  linear   y = W x, with x quantised by the call itself (apply) or before it
           (forward)
  grouped  the same product with a bank of matrices, rows grouped by expert at
           offsets that only the device knows
  layer    a mixture-of-experts layer of such matrices, from routes to the
           weighted sum with the shared expert

A row x with a = max(max |x|, 2^-100) has the scale s = a / 127 and the codes
rint(x * r) with r = 127 / a: each of the three operations rounded to fp32.
Codes of a row against codes of a matrix row sum to a whole number, which both
scales multiply.
"""
import importlib.util
import math
import os
import sys

import torch

own = False

TOP_K, EXPERTS = 10, 512
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _package():
    """The binding of the tree the program runs in (its folder's name is no
    Python identifier)."""
    if "moe_ffn" not in sys.modules:
        path = os.path.join(os.getcwd(), "gfx906-qwen3.8fn_amd", "moe_ffn.py")
        spec = importlib.util.spec_from_file_location("moe_ffn", path)
        module = importlib.util.module_from_spec(spec)
        sys.modules["moe_ffn"] = module
        spec.loader.exec_module(module)
    return sys.modules["moe_ffn"]


# ----------------------------------------------------------------- cases ---
def _rows(rows, width, type_="bf16"):
    return {"kind": "rows", "rows": rows, "input": width, "type": type_}


def _linear(inputs, outputs, columns, type_="bf16", codes=False):
    return {"kind": "linear", "input": inputs, "output": outputs, "columns": columns, "type": type_, "codes": codes}


def _grouped(tokens, inputs, outputs, type_="bf16", s=0.0, gather=True):
    return {"kind": "grouped", "tokens": tokens, "input": inputs, "output": outputs, "type": type_, "s": s, "gather": gather}


def _layer(tokens, hidden=2048, intermediate=512, type_="bf16", s=0.0, gate=False):
    return {"kind": "layer", "tokens": tokens, "hidden": hidden, "intermediate": intermediate, "type": type_, "s": s,
            "gate": gate}


def listed():
    return [
        # A decode batch's rows before its projections: latency only.
        dict(_rows(8, 2048), name="rows_decode_8"),
        # A 16K prompt's rows before a wide projection.
        dict(_rows(16384, 8192), name="rows_prefill_16384"),
        # One decode token through a hidden-size projection: latency only.
        dict(_linear(2048, 2048, 1), name="linear_decode_1"),
        # A small prompt's rows, quantised before, on a matrix of a size that no tile divides.
        dict(_linear(2080, 1000, 333, "f16", codes=True), name="linear_ragged_333"),
        # Decode tokens beside a prefill chunk, from and to fp32 as the Q4 path has them.
        dict(_linear(2048, 2048, 1032, "f32"), name="linear_mixed_1032"),
        # A long prompt through a wide projection: the largest work here.
        dict(_linear(8192, 8192, 8192), name="linear_prefill_8192"),
        # A decode batch's expert rows (eight tokens, top-10), gathered from the tokens.
        dict(_grouped(8, 2048, 1024), name="grouped_decode_8"),
        # Decode tokens beside a prefill chunk on the checkpoint's own expert shape, a few experts popular.
        dict(_grouped(1032, 2560, 640, "f32", s=1.3), name="grouped_mixed_1032"),
        # A 16K prompt's expert rows as a shard receives them, down to the hidden size.
        dict(_grouped(16384, 512, 2048, gather=False), name="grouped_prefill_16384"),
        # A decode batch of eight, the benchmark's headline shape.
        dict(_layer(8, gate=True), name="layer_decode_8"),
        # Decode tokens beside a prefill chunk, as one layer of the benchmark's stack.
        dict(_layer(1032, type_="f16", s=1.3, gate=True), name="layer_mixed_1032"),
        # A 4K prompt, the benchmark's prefill shape.
        dict(_layer(4096, s=1.1), name="layer_prefill_4096"),
    ]


def _spread(rng, lo, hi):
    """A whole number, evenly over the logarithm of lo..hi."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


LINEAR_SHAPES = [(2048, 2048), (2048, 512), (512, 2048), (2560, 640), (640, 2560), (2560, 2560), (1024, 4096),
                 (2048, 8192), (8192, 2048), (8192, 8192), (2080, 1000), (96, 2047)]
EXPERT_SHAPES = [(2048, 512), (2048, 512), (2560, 640), (1056, 352)]


def draw(rng):
    kind = rng.choice(["rows", "linear", "linear", "grouped", "layer", "layer"])
    type_ = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind == "rows":
        width = 32 * _spread(rng, 1, 512) if rng.random() < 0.7 else _spread(rng, 1, 16384)
        return _rows(_spread(rng, 1, 16000), width, type_)
    if kind == "linear":
        inputs, outputs = rng.choice(LINEAR_SHAPES)
        if rng.random() < 0.4:
            inputs, outputs = 32 * _spread(rng, 1, 256), _spread(rng, 1, 8192)
        return _linear(inputs, outputs, _spread(rng, 1, 8000), type_, codes=rng.random() < 0.4)
    hidden, intermediate = rng.choice(EXPERT_SHAPES)
    s = rng.choice([0.0, 1.1, 1.3])
    if kind == "grouped":
        shape = rng.choice([(hidden, 2 * intermediate), (hidden, intermediate), (intermediate, hidden), (hidden, 1000)])
        return _grouped(_spread(rng, 1, 8000), *shape, type_, s, rng.random() < 0.5)
    return _layer(_spread(rng, 1, 6000), hidden, intermediate, rng.choice(["bf16", "f16"]), s, rng.random() < 0.5)


# ---------------------------------------------------------------- inputs ---
def _generator(seed, stream):
    g = torch.Generator(device="cuda")
    g.manual_seed((int(seed) * 1000003 + stream * 7919 + 41) % (1 << 62))
    return g


def _matrices(count, rows, cols, g):
    """`count` matrices as a checkpoint holds them: int8 codes [count][rows]
    [cols] of values about N(0, 0.02) and a scale per output channel."""
    codes = torch.empty((count, rows, cols), dtype=torch.int8, device="cuda")
    for i in range(0, count, 64):   # the fp32 values of 64 experts at a time
        part = codes[i:i + 64]
        part.copy_(torch.randn(part.shape, generator=g, device="cuda").mul_(32.0).round_().clamp_(-127.0, 127.0))
    scales = (0.02 / 32.0) * (0.75 + 0.5 * torch.rand((count, rows), generator=g, device="cuda"))
    return codes, scales


def _activations(rows, width, type_, g):
    return torch.randn((rows, width), generator=g, device="cuda").to(TYPES[type_])


def _routes(c, g):
    """(ids, weights): top-10 by Gumbel keys, strongest first."""
    n = c["tokens"]
    logp = torch.zeros(EXPERTS, device="cuda", dtype=torch.float64)
    if c["s"]:
        perm = torch.randperm(EXPERTS, generator=g, device="cuda")
        logp[perm] = -c["s"] * torch.log(torch.arange(1, EXPERTS + 1, device="cuda", dtype=torch.float64))
    u = torch.rand((n, EXPERTS), generator=g, device="cuda", dtype=torch.float64).clamp_(1e-12, 1 - 1e-12)
    ids = (logp - torch.log(-torch.log(u))).topk(TOP_K, dim=1).indices.to(torch.int32).contiguous()
    return ids, torch.softmax(torch.randn((n, TOP_K), generator=g, device="cuda"), dim=1).contiguous()


def _linear_inputs(c, seed):
    g = _generator(seed, 1)
    codes, scales = _matrices(1, c["output"], c["input"], g)
    return codes[0], scales[0], _activations(c["columns"], c["input"], c["type"], g)


def _grouped_inputs(c, seed):
    """(codes, scales, x, index, offsets): the tokens' routes sorted by expert;
    without gather the rows themselves lie in that order."""
    g = _generator(seed, 2)
    codes, scales = _matrices(EXPERTS, c["output"], c["input"], g)
    ids, _ = _routes(c, g)
    order = torch.argsort(ids.reshape(-1).long(), stable=True)
    offsets = torch.zeros(EXPERTS + 1, dtype=torch.int32, device="cuda")
    offsets[1:] = torch.bincount(ids.reshape(-1).long(), minlength=EXPERTS).cumsum(0)
    rows = c["tokens"] if c["gather"] else c["tokens"] * TOP_K
    x = _activations(rows, c["input"], "bf16", g)
    return codes, scales, x, (order // TOP_K).to(torch.int32) if c["gather"] else None, offsets


def _layer_inputs(c, seed):
    g = _generator(seed, 3)
    h, i = c["hidden"], c["intermediate"]
    bank = [_matrices(EXPERTS, i, h, g), _matrices(EXPERTS, i, h, g), _matrices(EXPERTS, h, i, g)]
    shared = [tuple(t[0] for t in _matrices(1, *shape, g)) for shape in ((i, h), (i, h), (h, i))]
    x = _activations(c["tokens"], h, c["type"], g)
    ids, weights = _routes(c, g)
    gate = torch.randn(c["tokens"], generator=g, device="cuda") if c["gate"] else None
    return bank, shared, x, ids, weights, gate


def prepare(case, seed):
    kind, state = case["kind"], {"case": dict(case)}
    type_ = TYPES[case["type"]]
    error = torch.zeros(1, dtype=torch.int32, device="cuda")
    if kind == "rows":
        x = _activations(case["rows"], case["input"], case["type"], _generator(seed, 0))
        state.update(x=x)
        if own:
            out = [torch.empty(x.shape, dtype=torch.int8, device="cuda"), torch.empty(x.shape[0], device="cuda")]
            state.update(call=_package().bind_quantize_i8(x, *out, error), out=out)
    elif kind == "linear":
        codes, scales, x = _linear_inputs(case, seed)
        if case["codes"]:
            x = _quantise(x)
        state.update(weight=(codes, scales), x=x)
        if own:
            y = torch.empty((case["columns"], case["output"]), dtype=type_, device="cuda")
            matrix = _package().MoeI8Linear(case["input"], case["output"], codes, scales,
                                            max_columns=0 if case["codes"] else case["columns"])
            call = matrix.bind_forward(*x, y) if case["codes"] else matrix.bind_apply(x, y, error)
            state.update(handle=matrix, call=call, out=y, weight=None)
    elif kind == "grouped":
        codes, scales, x, index, offsets = _grouped_inputs(case, seed)
        x = _quantise(x)
        state.update(bank=(codes, scales), x=x, index=index, offsets=offsets)
        if own:
            y = torch.empty((case["tokens"] * TOP_K, case["output"]), dtype=type_, device="cuda")
            bank = _package().MoeI8Bank(EXPERTS, case["input"], case["output"], codes, scales)
            state.update(handle=bank, call=bank.bind_forward(*x, offsets, y, error, index=index), out=y, bank=None)
    else:
        bank, shared, x, ids, weights, gate = _layer_inputs(case, seed)
        state.update(bank=bank, shared=shared, x=x, ids=ids, weights=weights, gate=gate)
        if own:
            y = torch.empty_like(x)
            layer = _package().MoeI8Layer(case["hidden"], case["intermediate"], EXPERTS, TOP_K, True, case["tokens"],
                                          *bank, shared=shared)
            call = layer.bind_forward(x, ids, weights, y, error, shared_gate=gate)
            state.update(handle=layer, call=call, out=y, bank=None, shared=None)
    state["error"] = error
    return state


# ------------------------------------------------------------------ runs ---
BLOCK = 64   # rows of one expert that the plain form multiplies at once


def _quantise(x):
    """Rows -> (int8 codes, fp32 scale of each): divisions in 64 bits and
    rounded, which is the correctly rounded fp32 quotient."""
    v = x.float()
    a = v.abs().amax(dim=1).clamp_min(2.0 ** -100).double()
    return (v * (127.0 / a).float()[:, None]).round().to(torch.int8), (a / 127.0).float()


def _product(codes, scales, weight):
    w, sw = weight
    return (codes.float() @ w.float().T) * scales[:, None] * sw


def _blocks(offsets, rows):
    """Blocks of up to 64 rows of one expert: (expert of each block, its rows
    [blocks][64], which of them there are).  As many blocks as there can be."""
    count = rows // BLOCK + min(EXPERTS, rows)
    per = (offsets[1:] - offsets[:-1] + BLOCK - 1).long() // BLOCK
    first = torch.cumsum(per, 0)
    b = torch.arange(count, device=offsets.device)
    expert = torch.searchsorted(first, b, right=True).clamp_max(EXPERTS - 1)
    row = offsets[expert].long() + (b - (first - per)[expert]) * BLOCK
    row = row[:, None] + torch.arange(BLOCK, device=offsets.device)
    there = (row < offsets[expert + 1][:, None]) & (b < first[-1])[:, None]
    return expert, torch.where(there, row, rows), there


def _grouped_product(x, index, blocks, bank, rows):
    """Row i: x's row index[i] (or i) times its expert's matrix, fp32."""
    (codes, scales), (w, sw), (expert, row, there) = x, bank, blocks
    source = row.clamp_max(rows - 1)
    if index is not None:
        source = index.long()[source]
    right = codes[source].float().transpose(1, 2).contiguous()            # [block][input][64]
    y = torch.bmm(w[expert].float(), right).transpose(1, 2) * scales[source][..., None] * sw[expert][:, None]
    out = torch.zeros((rows + 1, w.shape[1]), device=y.device)
    out[row.reshape(-1)] = y.reshape(-1, w.shape[1])                      # those that are not there: a row past the end
    return out[:rows]


def _silu_mul(g, u):
    return g / (1.0 + torch.exp(-g)) * u


def _plain_layer(state):
    x, ids, weights, gate = state["x"], state["ids"], state["weights"], state["gate"]
    n, k = ids.shape
    flat = ids.reshape(-1).long()
    order = torch.argsort(flat, stable=True)
    offsets = torch.zeros(EXPERTS + 1, dtype=torch.long, device=x.device)
    offsets[1:] = (flat[:, None] == torch.arange(EXPERTS, device=x.device)).sum(0).cumsum(0)
    blocks = _blocks(offsets, n * k)
    q, token = _quantise(x), order // k
    gate_bank, up_bank, down_bank = state["bank"]
    middle = _silu_mul(_grouped_product(q, token, blocks, gate_bank, n * k), _grouped_product(q, token, blocks, up_bank, n * k))
    c = torch.empty((n * k, x.shape[1]), device=x.device)
    c[order] = _grouped_product(_quantise(middle), None, blocks, down_bank, n * k)
    y = (c.view(n, k, -1) * weights[..., None]).sum(dim=1)
    sg, su, sd = state["shared"]
    shared = _product(*_quantise(_silu_mul(_product(*q, sg), _product(*q, su))), sd)
    if gate is not None:
        shared = shared / (1.0 + torch.exp(-gate))[:, None]
    return (y + shared).to(x.dtype)


def run(state):
    if own:
        state["call"]()
        return state["out"]
    c = state["case"]
    if c["kind"] == "rows":
        return list(_quantise(state["x"]))
    if c["kind"] == "linear":
        x = state["x"] if c["codes"] else _quantise(state["x"])
        return _product(*x, state["weight"]).to(TYPES[c["type"]])
    if c["kind"] == "grouped":
        rows = c["tokens"] * TOP_K
        y = _grouped_product(state["x"], state["index"], _blocks(state["offsets"], rows), state["bank"], rows)
        return y.to(TYPES[c["type"]])
    return _plain_layer(state)


# ------------------------------------------------------------------ work ---
SIZE = {"f32": 4.0, "bf16": 2.0, "f16": 2.0}


def _touched(c):
    """Experts that a batch reaches, on average: expert i is among a token's
    ten with probability 1 - exp(-r p_i), r such that they add up to ten."""
    p = [(i + 1.0) ** -c["s"] for i in range(EXPERTS)]
    lo, hi = 0.0, 1e9
    for _ in range(80):
        r = (lo + hi) / 2
        lo, hi = (r, hi) if sum(1 - math.exp(-r * q) for q in p) < TOP_K else (lo, r)
    return sum(1 - math.exp(-lo * q * c["tokens"]) for q in p)


def work(case):
    size = SIZE[case["type"]]
    if case["kind"] == "rows":
        n, k = case["rows"], case["input"]
        return {"bytes": n * k * (size + 1) + 4.0 * n, "flops": 3.0 * n * k}
    if case["kind"] == "linear":
        k, m, n = case["input"], case["output"], case["columns"]
        x = n * (k + 4.0) if case["codes"] else n * k * size
        return {"bytes": m * (k + 4.0) + x + n * m * size, "flops": 2.0 * n * m * k}
    if case["kind"] == "grouped":
        k, m, rows = case["input"], case["output"], case["tokens"] * TOP_K
        x = case["tokens"] * (k + 4.0) + 4.0 * rows if case["gather"] else rows * (k + 4.0)
        return {"bytes": _touched(case) * m * (k + 4.0) + x + rows * m * size + 4.0 * EXPERTS, "flops": 2.0 * rows * m * k}
    n, h, i = case["tokens"], case["hidden"], case["intermediate"]
    expert = 3.0 * h * i + 4.0 * (2 * i + h)
    return {"bytes": (_touched(case) + 1) * expert + 2 * n * h * size + n * TOP_K * 8.0,
            "flops": 6.0 * h * i * n * (TOP_K + 1)}


# ----------------------------------------------------------------- exact ---
def _codes64(x):
    """The codes and scales of the rows of x, in 64 bits.  The format forms
    them in fp32, so x, the factor and the product are rounded to fp32."""
    x = x.float()
    a = torch.maximum(x.abs().max(dim=1).values, torch.tensor(2.0 ** -100, device=x.device)).double()
    r = (127.0 / a).float().double()
    v = (x.double() * r[:, None]).float().double()
    low = torch.floor(v)
    up = (v - low > 0.5) | ((v - low == 0.5) & (torch.remainder(low, 2.0) == 1.0))
    return torch.where(up, low + 1.0, low), (a / 127.0).float().double()


def _dot64(x, w):
    """x w^T of whole numbers up to 128, exact: sums of 1,024 products stay below
    2^24, where fp32 holds every whole number, and meet in 64 bits."""
    y = torch.zeros((x.shape[0], w.shape[0]), dtype=torch.float64, device=x.device)
    for at in range(0, x.shape[1], 1024):
        y += x[:, at:at + 1024].float() @ w[:, at:at + 1024].float().T
    return y


def _linear64(x, w):
    return _dot64(x[0], w[0]) * x[1][:, None] * w[1].double()


def _expert64(x, matrices):
    """One expert's output for quantised rows x."""
    g, u = _linear64(x, matrices[0]), _linear64(x, matrices[1])
    return _linear64(_codes64(g * torch.sigmoid(g) * u), matrices[2])


def _layer64(c, seed):
    bank, shared, x, ids, weights, gate = _layer_inputs(c, seed)
    q, s = _codes64(x)
    w = weights.double()
    y = _expert64((q, s), shared)
    if gate is not None:
        y = y * torch.sigmoid(gate.double())[:, None]
    for e in torch.unique(ids).tolist():
        t, r = torch.nonzero(ids == e, as_tuple=True)
        y[t] += w[t, r][:, None] * _expert64((q[t], s[t]), [(codes[e], scales[e]) for codes, scales in bank])
    return y


def _grouped64(c, seed):
    codes, scales, x, index, offsets = _grouped_inputs(c, seed)
    q, s = _codes64(x)
    at = index.long() if index is not None else torch.arange(q.shape[0], device=q.device)
    y = torch.zeros((at.shape[0], c["output"]), dtype=torch.float64, device=q.device)
    bounds = offsets.tolist()
    for e in range(EXPERTS):
        rows = at[bounds[e]:bounds[e + 1]]
        y[bounds[e]:bounds[e + 1]] = _linear64((q[rows], s[rows]), (codes[e], scales[e]))
    return y


def exact(case, seed):
    if case["kind"] == "layer":
        return _layer64(case, seed)
    if case["kind"] == "grouped":
        return _grouped64(case, seed)
    if case["kind"] == "linear":
        codes, scales, x = _linear_inputs(case, seed)
        return _linear64(_codes64(x), (codes, scales))
    x = _activations(case["rows"], case["input"], case["type"], _generator(seed, 0)).double()
    return [None, x.abs().amax(dim=1).clamp_min(2.0 ** -100) / 127.0]   # the codes are whole numbers
