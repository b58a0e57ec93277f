"""Cases, inputs and plain forms of the 8-bit training and serving operators.

Four operators that work together when the DiT is trained or sampled in 8 bits:

  quantize  ``ops.fp8_quantize``: e4m3 values with one power-of-two scale for each block of
            128 (1 x 128 along a row, 1 x 128 along a column, or 128 x 128 for weights)
  linear    ``ops.fp8_matmul``: act(x W^T + b) of a bf16 activation and a block-quantised
            weight, the activation quantised within the call
  train     ``quant.fp8_linear``: the same product under autograd, with dx, dW and db from
            block-quantised gradients
  adamw     ``ops.adamw_multi_``: AdamW over many tensors at once, moments in fp32 or in 8 bits
            with one power-of-two scale for each 128 elements and stochastic rounding

Formats.  A block scale is the smallest 2^k (k from -126) with max|x| / 2^k within the
format's largest value, kept as the byte k + 127; non-finite elements do not count for the
maximum and are stored as NaN.  Scales of a matrix [R, K] lie in chunks of 128 rows x 4
blocks, chunk [r / 128][k / 512] holding [r % 32][r % 128 / 32][k / 128 % 4]; bytes of rows
and blocks outside the matrix are zero.  Values are padded with zeros to a multiple of 128
columns.  First moments are e4m3; second moments are the sign-less top byte of an IEEE half
(5 exponent bits, 3 mantissa bits, 255 = NaN), where a positive value is never stored as 0.
"""
import math

import torch

own = False

BLOCK = 128
E4M3_TOP = 448.0          # largest e4m3 value,  0.875  * 2^9
LR, BETA1, BETA2, EPS, DECAY, CLIP = 1e-4, 0.9, 0.999, 1e-8, 0.01, 0.75


def listed():
    return [
        # the text context of one sample as a GEMM operand: a few microseconds, launch latency counts
        {"name": "quantize_text_rows", "op": "quantize", "rows": 512, "cols": 4096, "dtype": "bfloat16",
         "block_rows": 1, "layout": "rows", "strided": False},
        # gradient of FFN-up of the 14B model on one of four SSP ranks, for dX (rows) and dW (columns)
        {"name": "quantize_grad_both", "op": "quantize", "rows": 20160, "cols": 13824, "dtype": "bfloat16",
         "block_rows": 1, "layout": "both", "strided": False},
        # fp32 master weight of a 1.3B FFN layer, for the forward and the dX product
        {"name": "quantize_weight", "op": "quantize", "rows": 8960, "cols": 1536, "dtype": "float32",
         "block_rows": 128, "layout": "both", "strided": False},
        # time projection of the 14B model at batch 1: one row against a 157 MB weight
        {"name": "linear_time_1row", "op": "linear", "rows": 1, "in": 5120, "out": 30720, "act": "", "bias": True,
         "out_dtype": "bfloat16", "strided": False},
        # text embedding: one prompt of 512 tokens
        {"name": "linear_text", "op": "linear", "rows": 512, "in": 4096, "out": 5120, "act": "gelu_tanh",
         "bias": True, "out_dtype": "bfloat16", "strided": False},
        # output head over an odd number of tokens: a narrow product
        {"name": "linear_head_odd", "op": "linear", "rows": 20161, "in": 5120, "out": 64, "act": "", "bias": True,
         "out_dtype": "float32", "strided": False},
        # FFN-up of the 14B model at 81 frames of 768 x 1280 (80640 tokens), the largest product of sampling
        {"name": "linear_ffn_up", "op": "linear", "rows": 80640, "in": 5120, "out": 13824, "act": "gelu_tanh",
         "bias": True, "out_dtype": "bfloat16", "strided": False},
        # FFN-up training step of the 1.3B model, 33 frames of 480 x 832, fp32 master weight on one GPU
        {"name": "train_1_3b", "op": "train", "rows": 14040, "in": 1536, "out": 8960, "wdtype": "float32",
         "bias": True},
        # the same layer of the 14B model on one of four SSP ranks, bf16 weight as FSDP gathers it
        {"name": "train_14b", "op": "train", "rows": 20160, "in": 5120, "out": 13824, "wdtype": "bfloat16",
         "bias": True},
        # the tiny two-layer configuration: 60 small tensors, launch latency counts
        {"name": "adamw32_tiny", "op": "adamw", "bits": 32, "tensors": 60, "elements": 2600000,
         "gdtype": "float32"},
        # rank-64 LoRA factors of the 1.3B model: 600 tensors
        {"name": "adamw8_lora", "op": "adamw", "bits": 8, "tensors": 600, "elements": 87000000,
         "gdtype": "bfloat16"},
        # the 1.3B model's shard on one of eight FSDP ranks
        {"name": "adamw8_shard", "op": "adamw", "bits": 8, "tensors": 820, "elements": 177000000,
         "gdtype": "float32"},
    ]


def _log(rng, lo, hi):
    """A size between lo and hi, even over its logarithm; half of them multiples of 16."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5 and hi >= 32:
        n = min(hi // 16 * 16, (n + 15) // 16 * 16)
    return max(lo, min(hi, n))


def draw(rng):
    op = rng.choice(["quantize", "linear", "train", "adamw"])
    if op == "quantize":
        block = rng.choice([1, 1, 128])
        return {"op": op, "rows": _log(rng, 1, 20160), "cols": _log(rng, 64, 13824),
                "dtype": rng.choice(["bfloat16", "float16", "float32"]), "block_rows": block,
                "layout": rng.choice(["rows", "cols", "both"]), "strided": rng.random() < 0.3}
    if op == "linear":
        return {"op": op, "rows": _log(rng, 1, 80640), "in": _log(rng, 64, 5120), "out": _log(rng, 16, 13824),
                "act": rng.choice(["", "gelu_tanh"]), "bias": rng.random() < 0.7,
                "out_dtype": rng.choice(["bfloat16", "float32"]), "strided": rng.random() < 0.3}
    if op == "train":
        return {"op": op, "rows": _log(rng, 64, 20160), "in": _log(rng, 64, 5120), "out": _log(rng, 64, 13824),
                "wdtype": rng.choice(["float32", "bfloat16"]), "bias": rng.random() < 0.7}
    elements = _log(rng, 100000, 177000000)
    return {"op": op, "bits": rng.choice([8, 8, 32]), "tensors": min(_log(rng, 1, 1200), elements // 1024),
            "elements": elements, "gdtype": rng.choice(["float32", "bfloat16"])}


# ---------------------------------------------------------------------------- 8-bit formats

def _pow2(e):
    """2^e as fp32 for an int32 tensor -126 <= e <= 127."""
    return ((e + 127) << 23).view(torch.float32)


def _scale_exp(amax, frac, shift):
    """Smallest k >= -126 with amax <= frac * 2^(shift + k), as int32."""
    f, e = torch.frexp(amax)
    return torch.where(amax > 0, e.int() - shift + (f > frac).int(), -126).clamp_(min=-126)


def _blocks(x):
    """fp32 [R, Kp / 128, 128] of a matrix padded with zeros to a multiple of 128 columns."""
    pad = -x.shape[1] % BLOCK
    x = x.float()
    if pad:
        x = torch.cat([x, x.new_zeros(x.shape[0], pad)], 1)
    return x.view(x.shape[0], -1, BLOCK)


def _pack(b, rows, kblocks):
    """Scale bytes [rows, kblocks] in chunks of 128 rows x 4 blocks."""
    rt, kg = -(-rows // 128), -(-kblocks // 4)
    full = torch.zeros(rt * 128, kg * 4, dtype=torch.uint8, device=b.device)
    full[:rows, :kblocks] = b
    return full.view(rt, 4, 32, kg, 4).permute(0, 3, 2, 1, 4).contiguous()


def _unpack(p, rows, kblocks):
    rt, kg = p.shape[:2]
    return p.permute(0, 3, 2, 1, 4).reshape(rt * 128, kg * 4)[:rows, :kblocks]


def _quantize(x, block_rows):
    """(e4m3 values [R, Kp], packed scale bytes) of a matrix, in fp32."""
    xb = _blocks(x)
    rows, kblocks = xb.shape[:2]
    amax = xb.abs().masked_fill(~torch.isfinite(xb), 0.0).amax(2)
    if block_rows > 1:
        pad = -rows % block_rows
        amax = torch.cat([amax, amax.new_zeros(pad, kblocks)], 0) if pad else amax
        amax = amax.view(-1, block_rows, kblocks).amax(1).repeat_interleave(block_rows, 0)[:rows]
    k = _scale_exp(amax, 0.875, 9)
    q = (xb * _pow2(-k)[:, :, None]).to(torch.float8_e4m3fn).view(rows, -1)
    return q, _pack((k + 127).to(torch.uint8), rows, kblocks)


def _dequantize(q, scale):
    rows, kp = q.shape
    k = _unpack(scale, rows, kp // BLOCK).int() - 127
    return (q.float().view(rows, -1, BLOCK) * _pow2(k)[:, :, None]).view(rows, kp)


def _gelu_tanh(x):
    return 0.5 * x * (1 + torch.tanh(0.7978845608028654 * (x + 0.044715 * x * x * x)))


# stochastic rounding: element i of tensor t takes 32 bits mixed from i and a key of (seed, t);
# the multipliers are the first bits of the fractional parts of sqrt 2, sqrt 3 and sqrt 5
_MIX1, _MIX2, _MIX3 = 0x6A09E667, 0xBB67AE85, 0x3C6EF373
_U32 = 0xFFFFFFFF


def _mix(x):
    """32 mixed bits of an int64 tensor of values below 2^32."""
    x = (x ^ (x >> 16)) * _MIX1 & _U32
    x = (x ^ (x >> 15)) * _MIX2 & _U32
    return x ^ (x >> 16)


def _random_bits(seed, tensor_id, block):
    """int32 [blocks, 128]: bits of element 128 * block + j of its tensor."""
    key = _mix((tensor_id * _MIX3 + seed) & _U32)
    i = block[:, None] * BLOCK + torch.arange(BLOCK, device=block.device)
    return _mix((i + key[:, None]) & _U32)


def _encode_m(m, bits16):
    """e4m3 codes [blocks, 128] and scale bytes of first moments, stochastically rounded."""
    fin = torch.isfinite(m)
    k = _scale_exp(m.abs().masked_fill(~fin, 0.0).amax(1), 0.875, 9)
    y = m * _pow2(-k)[:, None]
    a = y.abs().masked_fill(~fin, 0.0)
    small = a < 2.0 ** -6
    t = torch.where(small, a + 2.0 ** -6, a).view(torch.int32) + (bits16 << 4)
    code = (t >> 20) - torch.where(small, 968, 960)
    code = torch.where(fin, code, 127) + torch.signbit(y).int() * 128
    return code.to(torch.uint8).view(torch.float8_e4m3fn), (k + 127).to(torch.uint8)


def _encode_v(v, bits16):
    """Codes (top byte of a half) and scale bytes of second moments, stochastically rounded."""
    fin = torch.isfinite(v)
    a = v.masked_fill(~fin, 0.0)
    k = _scale_exp(a.amax(1), 0.9375, 16)
    a = a * _pow2(-k)[:, None]
    small = a < 2.0 ** -14
    t = torch.where(small, a + 2.0 ** -14, a).view(torch.int32) + (bits16 << 4)
    code = (t >> 20) - torch.where(small, 904, 896)
    code = torch.maximum(code, (v > 0).int())
    return torch.where(fin, code, 255).to(torch.uint8), (k + 127).to(torch.uint8)


def _decode_m(q, scale):
    return q.float() * _pow2(scale.int() - 127)[:, None]


def _decode_v(q, scale):
    return (q.to(torch.int16) << 7).view(torch.float16).float() * _pow2(scale.int() - 127)[:, None]


# ---------------------------------------------------------------------------- inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _activation(rows, cols, dtype, strided, g):
    """Normal values with a few strong channels, optionally as columns of a wider buffer."""
    width = cols + 256 if strided else cols
    x = torch.randn(rows, width, generator=g, device="cuda")
    gain = torch.exp(0.7 * torch.randn(width, generator=g, device="cuda"))
    x = (x * gain).to(getattr(torch, dtype))
    return x[:, 128:128 + cols] if strided else x


def _gradient(rows, cols, g):
    size = torch.exp(1.5 * torch.randn(rows, 1, generator=g, device="cuda"))
    return (1e-4 * size * torch.randn(rows, cols, generator=g, device="cuda")).bfloat16()


def _sizes(case):
    """Tensor sizes: every third one a vector of a 64th part, the rest share what is left."""
    n, total = case["tensors"], case["elements"]
    mean = total // n
    small = [max(1, mean // 64 + i % 3) if i % 3 == 2 else 0 for i in range(n)]
    big = sum(s == 0 for s in small)
    share = (total - sum(small)) // big
    return [s or share - i % 5 for i, s in enumerate(small)]


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    if op == "quantize":
        return {"case": case, "x": _activation(case["rows"], case["cols"], case["dtype"], case["strided"], g)}
    if op in ("linear", "train"):
        rows, k, n = case["rows"], case["in"], case["out"]
        w = torch.randn(n, k, generator=g, device="cuda") * (1.0 / math.sqrt(k))
        bias = 0.1 * torch.randn(n, generator=g, device="cuda") if case["bias"] else None
        s = {"case": case, "bias": bias}
        if op == "linear":
            s["x"] = _activation(rows, k, "bfloat16", case["strided"], g)
            # a served weight is quantised once, when it is loaded
            s["wq"], s["wscale"] = _quantize(w, BLOCK)
        else:
            s["x"] = _activation(rows, k, "bfloat16", False, g).requires_grad_(True)
            s["w"] = w.to(getattr(torch, case["wdtype"])).requires_grad_(True)
            if bias is not None:
                bias.requires_grad_(True)
            s["dy"] = _gradient(rows, n, g)
        return s
    # one flat buffer for each of p, g, m, v; each tensor starts on a block of 128
    sizes = _sizes(case)
    nblk = [-(-n // BLOCK) for n in sizes]
    starts = [0]
    for b in nblk:
        starts.append(starts[-1] + b * BLOCK)
    flat = starts[-1]
    tensor_id = torch.repeat_interleave(torch.arange(len(sizes), device="cuda"), torch.tensor(nblk, device="cuda"))
    first = torch.tensor(starts[:-1], device="cuda") // BLOCK
    block = torch.arange(flat // BLOCK, device="cuda") - first[tensor_id]
    inside = (block[:, None] * BLOCK + torch.arange(BLOCK, device="cuda")) \
        < torch.tensor(sizes, device="cuda")[tensor_id][:, None]
    size = 1e-4 * torch.exp(2.0 * torch.randn(len(sizes), generator=g, device="cuda"))[tensor_id][:, None]

    def noise():
        return torch.randn(flat // BLOCK, BLOCK, generator=g, device="cuda") * inside
    p = 0.02 * noise()
    grad = (size * noise()).to(getattr(torch, case["gdtype"]))
    m = 0.3 * size * noise()
    v = (size * noise()).square_()
    s = {"case": case, "sizes": sizes, "starts": starts, "nblk": nblk, "p": p.view(-1), "g": grad.view(-1),
         "seed": seed & 0xFFFFFF, "tensor_id": tensor_id, "block": block, "step": 100}
    if case["bits"] == 32:
        s["m"], s["v"] = m.view(-1), v.view(-1)
    else:
        half = torch.full_like(m, 0x8000, dtype=torch.int32)
        (mq, s["mscale"]), (vq, s["vscale"]) = _encode_m(m, half), _encode_v(v, half)
        s["m"], s["v"] = mq.view(-1), vq.view(-1)
    # the optimizer's lists of tensors, as it keeps them between steps

    def tensors(flat_t, per=1):
        return [flat_t[o // per:o // per + (n if per == 1 else -(-n // per))] for o, n in zip(starts, sizes)]
    s["lists"] = [tensors(s["p"]), tensors(s["g"]), tensors(s["m"]), tensors(s["v"])]
    if case["bits"] == 8:
        s["lists"] += [tensors(s["mscale"], BLOCK), tensors(s["vscale"], BLOCK)]
    return s


# ---------------------------------------------------------------------------- one pass

def run(s):
    return _RUN[s["case"]["op"]](s)


def _run_quantize(s):
    c, x = s["case"], s["x"]
    if own:
        from osp_next_b200 import ops
        out = ops.fp8_quantize(x, block_rows=c["block_rows"], layout=c["layout"])
        out = out if c["layout"] == "both" else (out,)
        return [(t.data, t.scale) for t in out]
    sides = {"rows": [x], "cols": [x.t()], "both": [x, x.t()]}[c["layout"]]
    return [_quantize(t, c["block_rows"]) for t in sides]


def _run_linear(s):
    c, x = s["case"], s["x"]
    out_dtype = getattr(torch, c["out_dtype"])
    if own:
        from osp_next_b200 import ops
        w = ops.Fp8Tensor(s["wq"], s["wscale"], c["out"], c["in"], BLOCK)
        return ops.fp8_matmul(x, w, bias=s["bias"], act=c["act"] or None, out_dtype=out_dtype)
    y = _dequantize(*_quantize(x, 1)) @ _dequantize(s["wq"], s["wscale"]).t()
    y = y if s["bias"] is None else y + s["bias"]
    return (_gelu_tanh(y) if c["act"] else y).to(out_dtype)


def _run_train(s):
    c, x, w, bias, dy = s["case"], s["x"], s["w"], s["bias"], s["dy"]
    if own:
        from osp_next_b200.quant import fp8_linear
        y = fp8_linear(x, w, bias)
        grads = torch.autograd.grad(y, [x, w] + ([] if bias is None else [bias]), dy)
        return [y.detach(), *grads]
    with torch.no_grad():
        n, k = c["out"], c["in"]
        wq = _dequantize(*_quantize(w, BLOCK))
        y = _dequantize(*_quantize(x, 1)) @ wq.t()
        y = y if bias is None else y + bias
        dx = _dequantize(*_quantize(dy, 1))[:, :n] @ wq[:, :k]
        dw = _dequantize(*_quantize(dy.t(), 1)) @ _dequantize(*_quantize(x.t(), 1)).t()
        out = [y.bfloat16(), dx.to(x.dtype), dw.to(w.dtype)]
        return out if bias is None else out + [dy.float().sum(0)]


def _run_adamw(s):
    c = s["case"]
    s["step"] += 1
    step = s["step"]
    if own:
        from osp_next_b200 import ops
        ops.adamw_multi_(*s["lists"], lr=LR, beta1=BETA1, beta2=BETA2, eps=EPS, weight_decay=DECAY, step=step,
                         grad_scale=CLIP, seed=s["seed"] + step)
    else:
        p = s["p"].view(-1, BLOCK)
        g = s["g"].view(-1, BLOCK).float() * CLIP
        m, v = s["m"].view(-1, BLOCK), s["v"].view(-1, BLOCK)
        if c["bits"] == 8:
            m, v = _decode_m(m, s["mscale"]), _decode_v(v, s["vscale"])
        m = m * BETA1 + g * (1 - BETA1)
        v = v * BETA2 + (g * g) * (1 - BETA2)
        den = torch.sqrt(v) / torch.full_like(v, math.sqrt(1 - BETA2 ** step)) + EPS
        p.copy_(p * (1 - LR * DECAY) - LR / (1 - BETA1 ** step) * (m / den))
        if c["bits"] == 8:
            bits = _random_bits(s["seed"] + step, s["tensor_id"], s["block"])
            m, ms = _encode_m(m, (bits & 0xFFFF).int())
            v, vs = _encode_v(v, (bits >> 16).int())
            s["mscale"].copy_(ms)
            s["vscale"].copy_(vs)
        s["m"].copy_(m.view(-1))
        s["v"].copy_(v.view(-1))
    out = [s["p"], s["m"], s["v"]]
    return out + [s["mscale"], s["vscale"]] if c["bits"] == 8 else out


_RUN = {"quantize": _run_quantize, "linear": _run_linear, "train": _run_train, "adamw": _run_adamw}


def work(case):
    op = case["op"]
    size = {"bfloat16": 2, "float16": 2, "float32": 4}
    if op == "quantize":
        n = case["rows"] * case["cols"]
        sides = 2 if case["layout"] == "both" else 1
        return {"bytes": n * size[case["dtype"]] + sides * n * (1 + 1 / 128), "flops": 2 * n * sides}
    if op in ("linear", "train"):
        m, k, n = case["rows"], case["in"], case["out"]
        if op == "linear":
            return {"bytes": 2 * m * k + n * k * (1 + 1 / 128) + 4 * n * case["bias"] + m * n * size[case["out_dtype"]],
                    "flops": 2 * m * n * k}
        w = size[case["wdtype"]]
        # x, w, dy read; y, dx, dw (and db) written
        return {"bytes": 2 * (2 * m * k + 2 * m * n) + 2 * w * n * k + 8 * n * case["bias"], "flops": 6 * m * n * k}
    n = sum(_sizes(case))
    state = 4 * (1 + 1 / 128) if case["bits"] == 8 else 16
    return {"bytes": n * (8 + size[case["gdtype"]] + state), "flops": 15 * n}


# ---------------------------------------------------------------------------- 64 bits

def _two_to(k):
    """2^k in 64 bits, exactly, for whole numbers -1022 <= k <= 1023."""
    return ((k.long() + 1023) << 52).view(torch.float64)


def _exact_values(x, block_rows=1):
    """(values in units of their scale, scales) of a matrix in 64 bits, [R, K] each."""
    x = x.detach().double()
    rows, cols = x.shape
    rp, cp = -(-rows // block_rows) * block_rows, -(-cols // BLOCK) * BLOCK
    full = torch.zeros(rp, cp, dtype=torch.float64, device=x.device)
    full[:rows, :cols] = x
    tiles = full.view(rp // block_rows, block_rows, cp // BLOCK, BLOCK)
    top = tiles.abs().amax((1, 3), keepdim=True)
    k = torch.ceil(torch.log2(top / E4M3_TOP)).clamp(min=-126.0)
    k = torch.where(top > E4M3_TOP * _two_to(k), k + 1, torch.where(top <= E4M3_TOP * _two_to(k - 1), k - 1, k))
    scale = _two_to(k.clamp(min=-126.0))
    y = tiles / scale
    _, e = torch.frexp(y.abs().clamp(min=2.0 ** -6))
    step = _two_to(e - 4)
    q = torch.round(y / step) * step
    return q.reshape(rp, cp)[:rows], scale.expand_as(tiles).reshape(rp, cp)[:rows]


def _exact_product(a, b):
    return (a[0] * a[1]) @ (b[0] * b[1]).t()


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "quantize":
        x, b = s["x"], case["block_rows"]
        sides = {"rows": [x], "cols": [x.t()], "both": [x, x.t()]}[case["layout"]]
        return [(_exact_values(t, b)[0], None) for t in sides]
    if op == "linear":
        rows, kp = s["wq"].shape
        e = s["wscale"].permute(0, 3, 2, 1, 4).reshape(s["wscale"].shape[0] * 128, -1)[:rows, :kp // BLOCK]
        w = (s["wq"].double(), _two_to(e.long() - 127).repeat_interleave(BLOCK, 1))
        y = _exact_product(_exact_values(s["x"]), w)
        y = y if s["bias"] is None else y + s["bias"].double()
        if case["act"]:
            y = y / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))
        return y
    if op == "train":
        x, w, dy = s["x"].detach(), s["w"].detach(), s["dy"]
        wq = _exact_values(w, BLOCK)
        y = _exact_product(_exact_values(x), wq)
        y = y if s["bias"] is None else y + s["bias"].detach().double()
        wt = tuple(t[:, :case["in"]].t() for t in wq)
        dx = _exact_product(tuple(t[:, :case["out"]] for t in _exact_values(dy)), wt)
        dw = _exact_product(_exact_values(dy.t()), _exact_values(x.t()))
        return [y, dx, dw] + ([] if s["bias"] is None else [dy.double().sum(0)])
    step = s["step"] + 1
    g = s["g"].double() * CLIP
    if case["bits"] == 8:
        m = s["m"].double().view(-1, BLOCK) * _two_to(s["mscale"].long() - 127)[:, None]
        c = s["v"].long().view(-1, BLOCK)
        v = torch.where(c < 8, c * 2.0 ** -17, (8 + c % 8) * _two_to(c // 8 - 18)) \
            * _two_to(s["vscale"].long() - 127)[:, None]
        m, v = m.view(-1), v.view(-1)
    else:
        m, v = s["m"].double(), s["v"].double()
    m = BETA1 * m + (1 - BETA1) * g
    v = BETA2 * v + (1 - BETA2) * g * g
    mhat, vhat = m / (1 - BETA1 ** step), v / (1 - BETA2 ** step)
    p = s["p"].double()
    p = p - LR * DECAY * p - LR * mhat / (vhat.sqrt() + EPS)
    # the rounded moments depend on the random bits: held to the plain form alone
    return [p, None, None, None, None] if case["bits"] == 8 else [p, m, v]
