"""The cases on which the low-bit operators (``prime_amd.lowbit``) are measured, and their plain forms.

Five operators, in the order a training or decoding step meets them:

  norm        rms_norm_quantize / add_rms_norm_quantize: root-mean-square norm of a row, after the
              residual's addition if there is one, as 8-bit codes (int8 or e4m3) with one scale a row
  norm_grad   rms_norm_quantize_backward: the gradients of its input and of its weight
  round_trip  quantize_4bit, then dequantize_4bit of what it gave: weights as 4-bit codes with a
              scale per group of 32, 64 or 128, and the weights those codes stand for
  widen       dequantize_4bit alone, before a library product over many rows
  matvec      matvec_4bit: products of one to 64 rows with such weights; the rows in floating point,
              or 8-bit codes with a scale each as the norm gives them

The sizes are the hidden and feed-forward widths of the 1B model whose buckets bench.py quantizes
(2048 and 5632), and powers of two, multiples and odd neighbours around them.
"""
import math

import torch

own = False

HIDDEN, FFN = 2048, 5632
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "int8": torch.int8, "e4m3": torch.float8_e4m3fn}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4, "int8": 1, "e4m3": 1}
EPS = 1e-6
MOST_ROWS = 16384
MOST_ACTIVATIONS = 16384 * 4096 * 2    # bytes of the largest norm's rows
MOST_WEIGHTS = 4 * FFN * 8192          # elements of the largest weight, but for the output head's
TOP = {"int8": 127.0, "e4m3": 448.0}


def listed():
    return [
        # one new token of the 1B model between two blocks: latency alone
        {"name": "norm_token", "op": "norm", "rows": 1, "dim": HIDDEN, "dtype": "bf16", "weight": "fp32", "residual": True, "codes": "int8"},
        # a ragged batch with an odd width in full precision, for an fp8 product
        {"name": "norm_odd_fp8", "op": "norm", "rows": 733, "dim": 1999, "dtype": "fp32", "weight": "fp32", "residual": False, "codes": "e4m3"},
        # a training batch, or a long prompt: bandwidth
        {"name": "norm_batch", "op": "norm", "rows": 16384, "dim": 4096, "dtype": "bf16", "weight": "bf16", "residual": True, "codes": "int8"},
        # the first norm of a model has no gradient of a sum to take along; few rows, so little to hide behind
        {"name": "norm_grad_few", "op": "norm_grad", "rows": 77, "dim": HIDDEN, "dtype": "fp32", "weight": "fp32", "grad_hidden": False},
        # the same training batch on its way back
        {"name": "norm_grad_batch", "op": "norm_grad", "rows": 16384, "dim": 4096, "dtype": "bf16", "weight": "fp32", "grad_hidden": True},
        # one square matrix of the outer copy, fp32 as the outer step keeps it
        {"name": "round_trip_square", "op": "round_trip", "n": HIDDEN, "k": HIDDEN, "dtype": "fp32", "group": 32, "scale": "fp32"},
        # a large feed-forward matrix
        {"name": "round_trip_large", "op": "round_trip", "n": 4 * FFN, "k": 8192, "dtype": "bf16", "group": 128, "scale": "bf16"},
        # a feed-forward matrix whose rows end inside a group
        {"name": "widen_ragged", "op": "widen", "n": FFN, "k": 2024, "dtype": "fp16", "group": 64, "scale": "bf16"},
        # one new token through a square matrix: latency
        {"name": "matvec_token", "op": "matvec", "rows": 1, "n": HIDDEN, "k": HIDDEN, "x": "bf16", "group": 128, "scale": "bf16", "out": "bf16"},
        # one new token against a large vocabulary, from the norm's codes, logits in 32 bits
        {"name": "matvec_head_int8", "op": "matvec", "rows": 1, "n": 128000, "k": 8192, "x": "int8", "group": 128, "scale": "bf16", "out": "fp32"},
        # a few sequences decoded together; odd sizes, small groups
        {"name": "matvec_few_odd", "op": "matvec", "rows": 7, "n": 2 * FFN - 1, "k": FFN - 28, "x": "fp16", "group": 32, "scale": "fp32", "out": "fp16"},
        # a full decoding batch
        {"name": "matvec_batch", "op": "matvec", "rows": 64, "n": 4 * FFN, "k": 8192, "x": "bf16", "group": 64, "scale": "bf16", "out": "bf16"},
    ]


def spread(rng, low, high):
    """A whole number between two, spread over its logarithm; a multiple of 64 every other time where there is one."""
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if v >= 128 and rng.random() < 0.5:
        v = v // 64 * 64
    return max(low, min(high, v))


def draw(rng):
    op = rng.choice(["norm", "norm", "norm_grad", "round_trip", "widen", "matvec", "matvec", "matvec"])
    if op in ("norm", "norm_grad"):
        dim = spread(rng, 48, 16384)
        dtype = rng.choice(["bf16", "fp16", "fp32"])
        c = {"op": op, "rows": spread(rng, 1, min(MOST_ROWS, MOST_ACTIVATIONS // (dim * BYTES[dtype]))), "dim": dim, "dtype": dtype}
        c["weight"] = rng.choice(["fp32", dtype])
        if op == "norm":
            return {**c, "residual": rng.random() < 0.6, "codes": rng.choice(["int8", "e4m3"])}
        return {**c, "grad_hidden": rng.random() < 0.6}
    group, scale = rng.choice([32, 64, 128]), rng.choice(["bf16", "fp32"])
    k = spread(rng, 48, 16384)
    if op in ("round_trip", "widen"):
        dtype = rng.choice(["bf16", "fp16", "fp32"])
        return {"op": op, "n": spread(rng, 16, min(65536, 2 * MOST_WEIGHTS // (k * BYTES[dtype]))), "k": k, "dtype": dtype, "group": group, "scale": scale}
    n = spread(rng, 16, min(65536, MOST_WEIGHTS // k))
    x = rng.choice(["bf16", "fp16", "fp32", "int8"])
    return {"op": op, "rows": 1 if rng.random() < 0.4 else spread(rng, 1, 64), "n": n, "k": k, "x": x, "group": group, "scale": scale,
            "out": rng.choice(["bf16", "fp32"]) if x == "int8" else x}


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def activations(rows, dim):
        # hidden states: a few channels run many times larger than the rest
        channel = torch.exp(0.3 * normal(dim)) * torch.where(torch.rand(dim, generator=g, device="cuda") < 0.005, 12.0, 1.0)
        return normal(rows, dim) * channel

    state, op = dict(case), case["op"]
    if op in ("norm", "norm_grad"):
        dtype = DTYPES[case["dtype"]]
        state["w"] = (1.0 + 0.15 * normal(case["dim"])).to(DTYPES[case["weight"]])
        x = activations(case["rows"], case["dim"])
        if op == "norm":
            state["x"] = (0.4 * x if case["residual"] else x).to(dtype)
            state["r"] = activations(case["rows"], case["dim"]).to(dtype) if case["residual"] else None
        else:
            state["h"] = x.to(dtype)
            state["inv"] = (state["h"].double().square().mean(-1) + EPS).rsqrt().float()
            state["dy"] = (1e-3 * normal(case["rows"], case["dim"])).to(dtype)
            state["dh"] = (1e-3 * normal(case["rows"], case["dim"])).to(dtype) if case["grad_hidden"] else None
        return state
    n, k, group = case["n"], case["k"], case["group"]
    groups = -(-k // group)
    if op == "round_trip":
        state["weight"] = (0.02 * normal(n, k)).to(DTYPES[case["dtype"]])
        return state
    # 4-bit codes of normal weights (the largest of a group is 7), low nibble first; what lies behind a row's end is zero
    codes = torch.randn(n, groups * group, generator=g, device="cuda", dtype=torch.float16).mul_(2.6).round_().clamp_(-7, 7).to(torch.int8)
    codes[:, k:] = 0
    state["packed"] = ((codes[:, 0::2] & 15) | (codes[:, 1::2] << 4)).view(torch.uint8)
    state["scales"] = (0.01 * torch.exp(0.2 * normal(n, groups))).to(DTYPES[case["scale"]])
    if op == "matvec":
        x = activations(case["rows"], k)
        state["xs"] = None
        if case["x"] == "int8":
            top = x.abs().amax(-1, keepdim=True)
            state["xs"] = (top / 127).reshape(-1).contiguous()
            x = (x / top * 127).round()
        state["x_in"] = x.to(DTYPES[case["x"]])
    return state


def to_e4m3(t):
    """The nearest e4m3 value (ties to even) of each of ``t``, |t| <= 448, in ``t``'s own type."""
    step = torch.ldexp(torch.ones_like(t), torch.frexp(t)[1].clamp_min(-5) - 4)
    return torch.round(t / step) * step


def plain_norm(x, r, w, codes):
    h = x if r is None else (x.float() + r.float()).to(x.dtype)      # the stream as it is stored: what later blocks see
    z = h.float() * w.float()
    s = (z.abs().amax(-1).double() / TOP[codes]).float()
    # next to a border between two codes 32 bits are not enough
    t = z.double() / torch.where(s > 0, s, 1.0).double()[:, None]
    q = torch.round(t).clamp(-127, 127).to(torch.int8) if codes == "int8" else to_e4m3(t.clamp(-448, 448)).float().to(torch.float8_e4m3fn)
    inv = (h.double().square().mean(-1) + EPS).rsqrt()
    out = {"codes": q, "scales": (s.double() * inv).float(), "inv_rms": inv.float()}
    return out if r is None else {**out, "hidden": h}


def plain_norm_grad(dy, h, w, inv, dh):
    g, hf, i = dy.float(), h.float(), inv[:, None]
    u = g * w.float()
    dx = i * (u - hf * (i * i) * (u * hf).mean(-1, keepdim=True))
    if dh is not None:
        dx = dx + dh.float()
    return {"grad_x": dx.to(h.dtype), "grad_weight": (g * hf * i).sum(0).to(w.dtype)}


def plain_quantize(weight, group, scale):
    n, k = weight.shape
    groups = -(-k // group)
    w = torch.nn.functional.pad(weight.float(), (0, groups * group - k)).view(n, groups, group)
    s = (w.abs().amax(-1).double() / 7).float().to(DTYPES[scale])
    t = w.double() / torch.where(s > 0, s, 1.0).double()[..., None]      # next to a border 32 bits are not enough
    q = torch.round(t).clamp(-7, 7).to(torch.int8).view(n, groups * group)
    return ((q[:, 0::2] & 15) | (q[:, 1::2] << 4)).view(torch.uint8), s


def plain_widen(packed, scales, k):
    n, groups = scales.shape
    low, high = packed.bitwise_left_shift(4).view(torch.int8) >> 4, packed.view(torch.int8) >> 4
    q = torch.stack((low, high), -1).view(n, groups, -1).float()
    return q.mul_(scales.float()[..., None]).view(n, -1)[:, :k]


def plain_matvec(x, xs, packed, scales, out):
    y = x.float() @ plain_widen(packed, scales, x.shape[1]).T
    return (y if xs is None else y * xs[:, None]).to(DTYPES[out])


def run(s):
    op = s["op"]
    if own:
        from prime_amd import lowbit

        if op == "norm":
            dtype = DTYPES[s["codes"]]
            if s["residual"]:
                codes, scales, hidden, inv = lowbit.add_rms_norm_quantize(s["x"], s["r"], s["w"], EPS, dtype)
                return {"codes": codes, "scales": scales, "hidden": hidden, "inv_rms": inv}
            codes, scales, inv = lowbit.rms_norm_quantize(s["x"], s["w"], EPS, dtype)
            return {"codes": codes, "scales": scales, "inv_rms": inv}
        if op == "norm_grad":
            grad_x, grad_weight = lowbit.rms_norm_quantize_backward(s["dy"], s["h"], s["w"], s["inv"], s["dh"])
            return {"grad_x": grad_x, "grad_weight": grad_weight}
        if op == "round_trip":
            packed, scales = lowbit.quantize_4bit(s["weight"], s["group"], DTYPES[s["scale"]])
            return {"values": lowbit.dequantize_4bit(packed, scales, s["k"], DTYPES[s["dtype"]]), "scales": scales}
        if op == "widen":
            return lowbit.dequantize_4bit(s["packed"], s["scales"], s["k"], DTYPES[s["dtype"]])
        return lowbit.matvec_4bit(s["x_in"], s["packed"], s["scales"], s["xs"], DTYPES[s["out"]])
    if op == "norm":
        return plain_norm(s["x"], s["r"], s["w"], s["codes"])
    if op == "norm_grad":
        return plain_norm_grad(s["dy"], s["h"], s["w"], s["inv"], s["dh"])
    if op == "round_trip":
        packed, scales = plain_quantize(s["weight"], s["group"], s["scale"])
        return {"values": plain_widen(packed, scales, s["k"]).to(DTYPES[s["dtype"]]), "scales": scales}
    if op == "widen":
        return plain_widen(s["packed"], s["scales"], s["k"]).to(DTYPES[s["dtype"]])
    return plain_matvec(s["x_in"], s["xs"], s["packed"], s["scales"], s["out"])


def work(case):
    op = case["op"]
    if op in ("norm", "norm_grad"):
        b, rows, dim = BYTES[case["dtype"]], case["rows"], case["dim"]
        weight = dim * BYTES[case["weight"]]
        if op == "norm":
            # x (and the residual) in, codes (and the sum) out, two statistics a row
            return {"bytes": rows * dim * (b * (3 if case["residual"] else 1) + 1) + weight + 8 * rows, "flops": 6 * rows * dim}
        # the gradient and the row (and the sum's gradient) in, one gradient out
        return {"bytes": rows * dim * b * (4 if case["grad_hidden"] else 3) + 2 * weight + 4 * rows, "flops": 11 * rows * dim}
    n, k, groups = case["n"], case["k"], -(-case["k"] // case["group"])
    codes, scales = n * groups * case["group"] // 2, n * groups * BYTES[case["scale"]]
    if op == "round_trip":
        # two calls: the codes and scales of the first are written, and read by the second
        return {"bytes": 2 * n * k * BYTES[case["dtype"]] + 2 * (codes + scales), "flops": 4 * n * k}
    if op == "widen":
        return {"bytes": codes + scales + n * k * BYTES[case["dtype"]], "flops": n * k}
    rows = case["rows"]
    x = rows * k * BYTES[case["x"]] + (4 * rows if case["x"] == "int8" else 0)
    return {"bytes": codes + scales + x + rows * n * BYTES[case["out"]], "flops": 2 * rows * n * k}


def exact(case, seed):
    """The definitions once more, in float64 and by other steps. Roundings that belong to an operator's definition (the stored
    sum, the 32-bit product and scale that codes are taken from, the stored group scale) are kept."""
    s = prepare(case, seed)
    op = case["op"]
    f64 = torch.float64
    if op == "norm":
        h = s["x"].to(f64) if s["r"] is None else s["x"].to(f64).add(s["r"].to(f64)).to(torch.float32).to(s["x"].dtype).to(f64)
        z = (h * s["w"].to(f64)).to(torch.float32).to(f64)
        unit = (torch.maximum(z.max(1).values, -z.min(1).values) / TOP[case["codes"]]).to(torch.float32).to(f64)
        rms = torch.sqrt(torch.einsum("td,td->t", h, h) / case["dim"] + EPS)
        codes = None
        if case["codes"] == "e4m3":
            t = z / unit.clamp_min(1e-300).unsqueeze(1)
            m, e = torch.frexp(t.abs())                                   # t = m 2^e, 1/2 <= m < 1: four bits of m are kept
            keep = torch.pow(torch.full_like(t, 2.0), (e - 4).clamp_min(-9).to(f64))
            n = t.abs() / keep
            low = torch.floor(n)
            up = (n - low > 0.5) | ((n - low == 0.5) & (low.remainder(2) == 1))
            codes = torch.copysign((low + up.to(f64)) * keep, t)
        return {"codes": codes, "scales": unit / rms, "inv_rms": 1 / rms, **({} if s["r"] is None else {"hidden": h})}
    if op == "norm_grad":
        h, w, dy, inv = s["h"].to(f64), s["w"].to(f64), s["dy"].to(f64), s["inv"].to(f64)
        n = h * inv.unsqueeze(1)                                          # the normalised row
        u = dy * w
        dx = inv.unsqueeze(1) * (u - n * ((u * n).sum(1, keepdim=True) / case["dim"]))
        if s["dh"] is not None:
            dx = dx + s["dh"].to(f64)
        return {"grad_x": dx, "grad_weight": torch.einsum("td,td->d", dy, n)}

    def weights(codes, scales):
        return codes * scales.to(f64).repeat_interleave(case["group"], 1)

    if op == "round_trip":
        n, k, group = case["n"], case["k"], case["group"]
        values, scales = torch.empty(n, k, dtype=f64, device="cuda"), []
        for a in range(0, n, 4096):
            w = s["weight"][a:a + 4096].to(f64)
            parts = []
            for b in range(0, k, group):
                unit = (w[:, b:b + group].abs().max(1).values / 7).to(torch.float32).to(DTYPES[case["scale"]])
                t = w[:, b:b + group] / unit.to(f64).clamp_min(1e-300).unsqueeze(1)
                low = torch.floor(t)
                up = (t - low > 0.5) | ((t - low == 0.5) & (low.remainder(2) == 1))
                values[a:a + 4096, b:b + group] = (low + up.to(f64)).clamp(-7, 7) * unit.to(f64).unsqueeze(1)
                parts.append(unit)
            scales.append(torch.stack(parts, 1))
        return {"values": values, "scales": torch.cat(scales)}

    def codes_of(packed):
        b = packed.to(torch.int16)
        both = torch.empty(packed.shape[0], 2 * packed.shape[1], dtype=f64, device="cuda")
        both[:, 0::2] = ((b % 16 + 8) % 16 - 8).to(f64)
        both[:, 1::2] = ((b // 16 + 8) % 16 - 8).to(f64)
        return both

    k, parts = case["k"], []
    for a in range(0, case["n"], 8192):
        w = weights(codes_of(s["packed"][a:a + 8192]), s["scales"][a:a + 8192])[:, :k]
        parts.append(w if op == "widen" else (s["x_in"].to(f64) if s["xs"] is None else s["x_in"].to(f64) * s["xs"].to(f64).unsqueeze(1)) @ w.T)
    return torch.cat(parts, 0 if op == "widen" else 1)
