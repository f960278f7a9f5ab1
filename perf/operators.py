"""The microscaled (MX) operators as a user's program calls them: rows and weights in 8 or 4 bits
with a power-of-two scale for every 32 values, the norm that gives such rows, and the products
that take them -- with their plain forms in torch operations, their work and their exact results.

A row of K values is divided into blocks of 32; the scale of a block is the smallest power of two
with which its largest magnitude does not pass the format's largest value (6 for the 4-bit e2m1,
448 for the 8-bit e4m3).  Stored rows are padded with zeros to a multiple of 128 values; byte j of
a 4-bit row holds value 2j in its low nibble; a scale is stored as its exponent plus 127.
"""

import math

import torch

own = False

BLOCK, PAD = 32, 128
LARGEST = {4: 6.0, 8: 448.0}
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
HEAD_DIM = 128
EPS = 1e-6


def listed():
    return [
        # a layer's gate projection, laid out in 4 bits when a model is loaded
        {"name": "quantize_weight_mlp", "op": "quantize", "rows": 5632, "k": 2048, "bits": 4, "f32": False},
        # SwiGLU rows of a long prompt, in 8 bits for the down projection
        {"name": "quantize_rows_prompt", "op": "quantize", "rows": 8192, "k": 5632, "bits": 8, "f32": False},
        # eight sequences' rows between two projections of a decode step
        {"name": "norm_step", "op": "norm", "rows": 8, "k": 2048, "add": True, "final": False},
        # the same for every row of a long prompt
        {"name": "norm_prompt", "op": "norm", "rows": 8192, "k": 2048, "add": True, "final": False},
        # the last layer of a loop (final norm in the chain) over the active rows of a narrower model, ragged blocks
        {"name": "norm_final_ragged", "op": "norm", "rows": 2051, "k": 1000, "add": True, "final": True},
        # decode at batch one: input norm, then q, k and v with the rotary embedding
        {"name": "gemv_qkv_1", "op": "gemv", "kind": "rope", "chain": True, "rows": 1, "k": 2048, "n": 2048, "f32": False},
        # decode of eight sequences: the gate and up projections
        {"name": "gemv_swiglu_8", "op": "gemv", "kind": "swiglu", "chain": False, "rows": 8, "k": 2048, "n": 5632, "f32": False},
        # the attention's f32 rows through the output projection, added to what an earlier loop gave
        {"name": "gemv_add_3", "op": "gemv", "kind": "add", "chain": False, "rows": 3, "k": 2048, "n": 2048, "f32": True},
        # the vocabulary's logits of one token
        {"name": "gemv_head_1", "op": "gemv", "kind": "f32", "chain": False, "rows": 1, "k": 2048, "n": 49152, "f32": False},
        # a decode step of more sequences than the GEMV takes: the gate projection
        {"name": "matmul_batch_32", "op": "matmul", "rows": 32, "k": 2048, "n": 5632, "f32": False},
        # active rows of a late loop on odd sizes, f32 results
        {"name": "matmul_ragged", "op": "matmul", "rows": 819, "k": 1000, "n": 1111, "f32": True},
        # the gate projection of a long prompt
        {"name": "matmul_prompt", "op": "matmul", "rows": 8192, "k": 2048, "n": 5632, "f32": False},
    ]


def _between(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["quantize", "norm", "gemv", "gemv", "matmul", "matmul"])
    if op == "quantize":
        k = _between(rng, 1, 8192)
        return {"op": op, "rows": _between(rng, 1, max(1, 40_000_000 // k)), "k": k, "bits": rng.choice([4, 8]), "f32": rng.random() < 0.5}
    if op == "norm":
        k = 8 * _between(rng, 8, 1024)
        add = rng.random() < 0.8
        return {"op": op, "rows": _between(rng, 1, max(1, 16_000_000 // k)), "k": k, "add": add, "final": rng.random() < 0.3}
    if op == "gemv":
        kind = rng.choice(["plain", "f32", "add", "swiglu", "rope"])
        chain = kind in ("plain", "swiglu", "rope") and rng.random() < 0.4
        k = 8 * _between(rng, 8, 512 if chain else 1024)
        n = HEAD_DIM * _between(rng, 1, 32) if kind == "rope" else _between(rng, 64, 10_000_000 // max(k, 200))
        return {"op": op, "kind": kind, "chain": chain, "rows": rng.randint(1, 8), "k": k, "n": n, "f32": not chain and rng.random() < 0.5}
    k = _between(rng, 32, 6000)
    n = _between(rng, 16, 8192)
    return {"op": op, "rows": _between(rng, 1, max(1, min(8192, 90_000_000_000 // (k * n)))), "k": k, "n": n, "f32": rng.random() < 0.3}


# ---------------------------------------------------------------------------- plain forms
def _blocks(x):
    """Rows padded with zeros to whole blocks, as [rows, blocks, 32]."""
    pad = -x.shape[1] % BLOCK
    return torch.nn.functional.pad(x, (0, pad)).view(x.shape[0], -1, BLOCK)


def _exponents(b, bits):
    """The blocks' scale exponents: largest magnitude <= LARGEST * 2**e, e as small as it gets."""
    m, e = torch.frexp(b.abs().amax(2))
    top, te = math.frexp(LARGEST[bits])
    return (torch.where(m == 0, -126, e - te + (m > top))).clamp(min=-126)


def _to_grid(v, bits):
    """The format's value that is nearest to v, ties to the even one."""
    least, mant = (0, 1) if bits == 4 else (-6, 3)
    _, e = torch.frexp(v)
    step = torch.ldexp(torch.ones_like(v), (e - 1).clamp(min=least) - mant)
    return torch.round(v / step) * step


def _quantized(x, bits):
    """(values in the format [rows, K to whole blocks], exponents [rows, blocks])."""
    b = _blocks(x)
    e = _exponents(b, bits)
    return _to_grid(torch.ldexp(b, -e[..., None]), bits).view(x.shape[0], -1), e


def _values(q, e, k):
    return torch.ldexp(q.view(q.shape[0], -1, BLOCK), e[..., None]).view(q.shape[0], -1)[:, :k]


def _stored(x, bits):
    """x [rows, K] f32 as its bytes: (codes u8, scales u8), rows padded to 128 values."""
    rows, k = x.shape
    q, e = _quantized(x, bits)
    kp = -(-k // PAD) * PAD
    q = torch.nn.functional.pad(q, (0, kp - q.shape[1]))
    scales = torch.nn.functional.pad(e + 127, (0, kp // BLOCK - e.shape[1]), value=1).to(torch.uint8)
    if bits == 8:
        return q.to(torch.float8_e4m3fn).view(torch.uint8), scales
    code = (torch.bucketize(q.abs(), torch.tensor(E2M1, device=x.device)) + 8 * (q < 0)).to(torch.uint8)
    return code[:, 0::2] | code[:, 1::2] << 4, scales


def _of_stored(codes, scales, bits, k):
    """The f32 values of stored rows."""
    if bits == 8:
        v = codes.view(torch.float8_e4m3fn).float()
    else:
        table = torch.tensor(E2M1 + [-v for v in E2M1], device=codes.device)
        v = table[torch.stack((codes & 15, codes >> 4), 2).view(codes.shape[0], -1).long()]
    return _values(v, scales.int() - 127, k)


def _norm(x, w):
    """w * x / sqrt(mean(x^2) + eps) in 64 bits (the result is rounded to few bits next)."""
    x = x.double()
    return w.double() * x * torch.rsqrt(x.square().mean(1, keepdim=True) + EPS)


def _chain(s):
    """h = r (+ norm(x)), through the final norm where there is one; rounded to bf16."""
    h = s["r"].double()
    if s["x"] is not None:
        h = h + _norm(s["x"], s["w_a"])
    if s["w_f"] is not None:
        h = _norm(h, s["w_f"])
    return h.to(torch.bfloat16)


def _epilogue(s, ys):
    """The GEMV's outputs from its products ys, in ys's type; the caller rounds them."""
    kind = s["case"]["kind"]
    if kind == "add":
        return [ys[0] + s["addend"].to(ys[0].dtype)]
    if kind == "swiglu":
        return [ys[0] * torch.sigmoid(ys[0]) * ys[1]]
    if kind == "rope":
        cos, sin = (t[:, None].to(ys[0].dtype) for t in s["rope"])
        turned = []
        for y in ys[:2]:
            y = y.view(y.shape[0], -1, HEAD_DIM)
            other = torch.cat((-y[..., HEAD_DIM // 2:], y[..., :HEAD_DIM // 2]), 2)
            turned.append((y * cos + other * sin).flatten(1))
        return [*turned, ys[2]]
    return ys


def _plain(s):
    case = s["case"]
    op, k = case["op"], case["k"]
    if op == "quantize":
        return _values(*_quantized(s["x"].float(), case["bits"]), k).to(torch.bfloat16)
    if op == "norm":
        h = _chain(s)
        return [h, _values(*_quantized(_norm(h, s["w_b"]), 8), k).to(torch.bfloat16)]
    if op == "gemv":
        out, x = [], s["x"]
        if case["chain"]:
            h = _chain(s)
            out, x = [h], _norm(h, s["w_b"])
        x = x.to(torch.bfloat16).float()  # (the operator's rows are bf16)
        ys = _epilogue(s, [x @ _of_stored(*w, 4, k).t() for w in s["weights"]])
        return out + [y.to(torch.float32 if case["kind"] == "f32" else torch.bfloat16) for y in ys]
    y = _of_stored(*s["x"], 8, k) @ _of_stored(*s["weight"], 4, k).t()
    return y if case["f32"] else y.to(torch.bfloat16)


# ---------------------------------------------------------------------------- inputs
def _rows(gen, rows, k, dtype, spread=1.0):
    """Activations: normal, channels of unequal size, a few far ones, some blocks of zeros."""
    x = torch.randn(rows, k, generator=gen, device="cuda") * spread
    x = x * torch.exp(torch.randn(k, generator=gen, device="cuda"))
    x = torch.where(torch.rand(rows, k, generator=gen, device="cuda") < 1e-4, 30 * x, x)
    zero = torch.rand(rows, -(-k // BLOCK), generator=gen, device="cuda") < 1e-3
    return torch.where(zero.repeat_interleave(BLOCK, 1)[:, :k], 0.0, x).to(dtype)


def _gain(gen, k):
    return (1 + 0.2 * torch.randn(k, generator=gen, device="cuda")).to(torch.bfloat16)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rows, k, op = case["rows"], case["k"], case["op"]
    s = {"case": case, "x": None, "r": None, "w_a": None, "w_f": None, "w_b": None}
    if op == "quantize":
        if case["bits"] == 4:  # a weight matrix
            x = 0.02 * torch.randn(rows, k, generator=gen, device="cuda")
            s["x"] = x if case["f32"] else x.to(torch.bfloat16)
        else:
            s["x"] = _rows(gen, rows, k, torch.float32 if case["f32"] else torch.bfloat16)
        return s
    chain = op == "norm" or (op == "gemv" and case["chain"])
    if chain:
        s["r"] = _rows(gen, rows, k, torch.bfloat16)
        s["w_b"] = _gain(gen, k)
        if case.get("add", True):
            s["x"], s["w_a"] = _rows(gen, rows, k, torch.bfloat16, 0.3), _gain(gen, k)
        if case.get("final"):
            s["w_f"] = _gain(gen, k)
    if op == "gemv":
        if not chain:
            s["x"] = _rows(gen, rows, k, torch.float32 if case["f32"] else torch.bfloat16)
        count = {"swiglu": 2, "rope": 3}.get(case["kind"], 1)
        s["weights"] = [_stored(0.02 * torch.randn(case["n"], k, generator=gen, device="cuda"), 4) for _ in range(count)]
        if case["kind"] == "add":
            s["addend"] = torch.randn(rows, case["n"], generator=gen, device="cuda").to(torch.bfloat16)
        if case["kind"] == "rope":
            at = torch.randint(0, 32768, (rows, 1), generator=gen, device="cuda").double()
            f = at * 10000.0 ** (-torch.arange(0, HEAD_DIM, 2, device="cuda", dtype=torch.float64) / HEAD_DIM)
            f = torch.cat((f, f), 1)
            s["rope"] = (f.cos().to(torch.bfloat16), f.sin().to(torch.bfloat16))
    if op == "matmul":
        s["x"] = _stored(_rows(gen, rows, k, torch.bfloat16).float(), 8)
        s["weight"] = _stored(0.02 * torch.randn(case["n"], k, generator=gen, device="cuda"), 4)
    return s


def run(state):
    if not own:
        return _plain(state)
    from flashloop_amd import kernels as K

    s, case = state, state["case"]
    op, k = case["op"], case["k"]
    if op == "quantize":
        return K.mx_dequantize(K.mx_quantize(s["x"], case["bits"]))
    if op == "norm":
        h, z = K.norm_chain_mx(s["r"], x=s["x"], w_a=s["w_a"], w_f=s["w_f"], w_b=s["w_b"], eps=EPS)
        return [h, K.mx_dequantize(z)]
    if op == "gemv":
        weights = [K.MXTensor(*w, cols=k, bits=4) for w in s["weights"]]
        kind = case["kind"]
        epilogue = {"plain": K.EPI_PLAIN, "f32": K.EPI_F32, "add": K.EPI_ADD, "swiglu": K.EPI_SWIGLU, "rope": K.EPI_ROPE}[kind]
        more = {"addend": s.get("addend"), "rope": s.get("rope"), "head_dim": HEAD_DIM}
        if case["chain"]:
            h, y = K.mx_gemv_chain(s["r"], weights, x=s["x"], w_a=s["w_a"], w_f=s["w_f"], w_b=s["w_b"], eps=EPS,
                                   epilogue=epilogue, **more)
            return [h, *(y if kind == "rope" else [y])]
        y = K.mx_gemv(s["x"], weights, epilogue=epilogue, **more)
        return list(y) if kind == "rope" else [y]
    x = K.MXTensor(*s["x"], cols=k, bits=8)
    w = K.MXTensor(*s["weight"], cols=k, bits=4)
    return K.mx_matmul(x, w, out_dtype=torch.float32 if case["f32"] else torch.bfloat16)


def work(case):
    rows, k, op = case["rows"], case["k"], case["op"]
    kp = -(-k // PAD) * PAD

    def stored(r, bits):
        return r * (kp * bits // 8 + kp // BLOCK)

    if op == "quantize":  # read the rows, write their bytes and the values that they stand for
        return {"bytes": rows * k * (4 if case["f32"] else 2) + stored(rows, case["bits"]) + 2 * rows * k, "flops": 4 * rows * k}
    if op == "norm":
        gains = 1 + int(case["add"]) + int(case["final"])
        return {"bytes": 2 * rows * k * (2 + int(case["add"])) + 2 * k * gains + stored(rows, 8) + 2 * rows * k,
                "flops": 6 * rows * k * gains}
    n = case["n"]
    if op == "gemv":
        mats, outs = {"swiglu": (2, 1), "rope": (3, 3)}.get(case["kind"], (1, 1))
        io = 4 if case["f32"] else 2
        if case["chain"]:
            io = 6
        more = {"add": 2 * rows * n, "rope": 4 * rows * HEAD_DIM}.get(case["kind"], 0)
        return {"bytes": mats * stored(n, 4) + rows * k * io + outs * rows * n * (4 if case["kind"] == "f32" else 2) + more,
                "flops": 2 * rows * k * n * mats}
    return {"bytes": stored(rows, 8) + stored(n, 4) + rows * n * (4 if case["f32"] else 2), "flops": 2 * rows * k * n}


# ---------------------------------------------------------------------------- 64-bit results
def _exact_values(codes, scales, bits, k):
    """Stored rows in 64 bits, from the fields of each code: sign, exponent, fraction."""
    if bits == 4:
        c = torch.empty(codes.shape[0], 2 * codes.shape[1], dtype=torch.int64, device=codes.device)
        c[:, 0::2], c[:, 1::2] = codes.long() % 16, codes.long() // 16
        sign, ex, fr, bias, fb = c // 8, c // 2 % 4, c % 2, 1, 1
    else:
        c = codes.long()
        sign, ex, fr, bias, fb = c // 128, c // 8 % 16, c % 8, 7, 3
    scale = scales.double().sub(127).exp2().repeat_interleave(BLOCK, 1)
    mag = (fr.double() / 2**fb + (ex > 0)) * (ex.clamp(min=1) - bias).double().exp2()
    return ((1 - 2 * sign) * mag * scale)[:, :k]


def _exact_quantized(x, bits):
    """x in 64 bits, each block's values replaced by the nearest of the format's, ties to the even code."""
    grid = torch.tensor([(f / 2 + (e > 0)) * 2.0 ** max(e - 1, 0) for e in range(4) for f in range(2)] if bits == 4 else
                        [(f / 8 + (e > 0)) * 2.0 ** (max(e, 1) - 7) for e in range(16) for f in range(8)][:127],
                        dtype=torch.float64, device=x.device)
    middle = (grid[1:] + grid[:-1]) / 2
    rows, k = x.shape
    out = torch.zeros(rows, -(-k // BLOCK) * BLOCK, dtype=torch.float64, device=x.device)
    out[:, :k] = x
    b = out.view(rows, -1, BLOCK)
    peak = b.abs().max(2, keepdim=True).values
    e = torch.log2((peak / grid[-1]).clamp(min=2.0**-126)).ceil()
    e = torch.where(peak > grid[-1] * e.exp2(), e + 1, torch.where(peak <= grid[-1] * (e - 1).exp2(), e - 1, e)).clamp(min=-126)
    v = b / e.exp2()
    below = torch.bucketize(v.abs(), middle)  # the first code whose upper border is not under v
    on_border = (below < len(middle)) & (middle[below.clamp(max=len(middle) - 1)] == v.abs())
    code = torch.where(on_border & (below % 2 == 1), below + 1, below)
    return (torch.sign(v) * grid[code] * e.exp2()).view(rows, -1)[:, :k]


def exact(case, seed):
    s = prepare(case, seed)
    op, k = case["op"], case["k"]
    if op == "quantize":
        return _exact_quantized(s["x"].double(), case["bits"])

    def normed(v, w):
        return v * w.double() / (v.pow(2).sum(1, keepdim=True) / k + EPS).sqrt()

    h = None
    if s["r"] is not None:
        h = s["r"].double()
        if s["x"] is not None:
            h = h + normed(s["x"].double(), s["w_a"])
        if s["w_f"] is not None:
            h = normed(h, s["w_f"])
    if op == "norm":
        return [h, _exact_quantized(normed(h.to(torch.bfloat16).double(), s["w_b"]), 8)]
    if op == "gemv":
        x = normed(h.to(torch.bfloat16).double(), s["w_b"]) if case["chain"] else s["x"].double()
        x = x.to(torch.bfloat16).double()  # the operator's rows are bf16
        ys = [x @ _exact_values(*w, 4, k).t().contiguous() for w in s["weights"]]
        kind = case["kind"]
        if kind == "add":
            ys = [ys[0] + s["addend"].double()]
        elif kind == "swiglu":
            ys = [ys[0] / (1 + torch.exp(-ys[0])) * ys[1]]
        elif kind == "rope":
            c, n = (t.double().repeat(1, case["n"] // HEAD_DIM) for t in s["rope"])
            half = HEAD_DIM // 2
            at = torch.arange(case["n"], device=x.device)
            first = at % HEAD_DIM < half
            pair = torch.where(first, at + half, at - half)
            ys = [y * c + torch.where(first, -y[:, pair], y[:, pair]) * n for y in ys[:2]] + [ys[2]]
        return ([h] if case["chain"] else []) + ys
    return _exact_values(*s["x"], 8, k) @ _exact_values(*s["weight"], 4, k).t().contiguous()
