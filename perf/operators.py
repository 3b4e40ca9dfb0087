"""Cases for the 8-bit floating point product and the mixture-of-experts layer.

Three operators, each in two forms.  ``own`` false: elementary torch
operations in 32 bits (64 for router logits), rounded once at the end.
``own`` true: the calls a user makes of this package.

* pack: fp32 / bf16 / fp16 [rows x cols] -> e4m3 codes with one fp32 scale
  per 1 x 128 (activations) or 128 x 128 (weights) block:
  scale = fp32(amax / 448), code = e4m3(fp32(x / scale)), ties to even;
  a block whose scale is 0 has codes 0.
* linear: y = q(x) . W^T (+ bias), W packed in 128 x 128 blocks, x packed in
  1 x 128 blocks within the call.
* moe: softmax router with top_k of the experts (ties to the lowest index,
  weights normalised to sum 1), then
  y = sum_j p_j * W_down[e_j] . (silu(W_gate[e_j] . x) * (W_up[e_j] . x)),
  the experts' weights packed in a block format or in e4m3 blocks.
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
#: elements and bytes of a block
BLOCKS = {"Q8_0": (32, 34), "Q4_0": (32, 18), "Q2_K": (256, 84), "Q3_K": (256, 110), "Q4_K": (256, 144),
          "Q5_K": (256, 176), "Q6_K": (256, 210)}
F8_MAX = 448.0


def _up(n, m):
    return -(-n // m)


# ---------------------------------------------------------------- cases

def listed():
    return [
        # a decode batch's activations before a projection: launch latency
        {"name": "pack act 16x4096", "op": "pack", "rows": 16, "cols": 4096, "block_rows": 1, "dtype": "bf16"},
        # a prompt's activations with a ragged hidden size
        {"name": "pack act 2500x8200", "op": "pack", "rows": 2500, "cols": 8200, "block_rows": 1, "dtype": "fp16"},
        # loading the largest weight of the low-bit workload
        {"name": "pack weight 28672x8192", "op": "pack", "rows": 28672, "cols": 8192, "block_rows": 128,
         "dtype": "fp32"},
        # one generated token through an attention projection
        {"name": "linear 1x4096x4096", "op": "linear", "tokens": 1, "out": 4096, "cols": 4096, "dtype": "bf16",
         "bias": False},
        # a few sequences decoding together, fp32 activations as the rest of this package has them
        {"name": "linear 7x11008x4096", "op": "linear", "tokens": 7, "out": 11008, "cols": 4096, "dtype": "fp32",
         "bias": True},
        # a larger decode batch through the down projection
        {"name": "linear 64x4096x11008", "op": "linear", "tokens": 64, "out": 4096, "cols": 11008, "dtype": "fp16",
         "bias": False},
        # a prompt of odd length and a ragged width
        {"name": "linear 509x4100x4000", "op": "linear", "tokens": 509, "out": 4100, "cols": 4000, "dtype": "bf16",
         "bias": True},
        # a long prompt through the largest weight
        {"name": "linear 4096x28672x8192", "op": "linear", "tokens": 4096, "out": 28672, "cols": 8192,
         "dtype": "bf16", "bias": False},
        # one generated token, many small experts
        {"name": "moe 1 token Q4_K", "op": "moe", "tokens": 1, "experts": 64, "top_k": 8, "hidden": 2048,
         "ffn": 1408, "fmt": "Q4_K", "fmt_down": "Q6_K", "dtype": "bf16"},
        # a few tokens, few large experts of the MLP block's shapes and formats
        {"name": "moe 4 tokens large", "op": "moe", "tokens": 4, "experts": 8, "top_k": 2, "hidden": 4096,
         "ffn": 11008, "fmt": "Q4_K", "fmt_down": "Q6_K", "dtype": "fp32"},
        # a decode batch at odd sizes in the low-bit formats
        {"name": "moe 33 tokens ragged", "op": "moe", "tokens": 33, "experts": 32, "top_k": 4, "hidden": 4000,
         "ffn": 1000, "fmt": "Q3_K", "fmt_down": "Q5_K", "dtype": "fp16"},
        # a decode batch with experts in 8-bit floating point
        {"name": "moe 16 tokens F8", "op": "moe", "tokens": 16, "experts": 16, "top_k": 4, "hidden": 4096,
         "ffn": 1408, "fmt": "F8", "fmt_down": "F8", "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["pack", "linear", "linear", "moe", "moe"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    if op == "pack":
        rows = _log(rng, 1, 16384)
        cols = _log(rng, 64, min(16384, max(64, 120_000_000 // rows)))
        return {"op": op, "rows": rows, "cols": cols, "block_rows": rng.choice([1, 128]), "dtype": dtype}
    if op == "linear":
        out, cols = _log(rng, 100, 16384), _log(rng, 100, 12000)
        if rng.random() < 0.5:  # half of the widths are whole blocks, as most models have them
            out, cols = _up(out, 128) * 128, _up(cols, 128) * 128
        return {"op": op, "tokens": _log(rng, 1, 4096), "out": out, "cols": cols, "dtype": dtype,
                "bias": rng.random() < 0.5}
    fmt = rng.choice(sorted(BLOCKS) + ["F8"])
    down = "F8" if fmt == "F8" else rng.choice(sorted(BLOCKS))
    experts = _log(rng, 4, 64)
    hidden = _log(rng, 256, 4096)
    ffn = _log(rng, 128, max(256, min(8192, 160_000_000 // (experts * hidden))))
    if fmt == "F8":
        ffn, hidden = _up(ffn, 128) * 128, _up(hidden, 128) * 128
    elif rng.random() < 0.5:
        ffn, hidden = _up(ffn, 256) * 256, _up(hidden, 256) * 256
    return {"op": op, "tokens": _log(rng, 1, 64), "experts": experts, "top_k": rng.randint(1, min(8, experts)),
            "hidden": hidden, "ffn": ffn, "fmt": fmt, "fmt_down": down, "dtype": dtype}


# ---------------------------------------------------------------- inputs

def _activations(gen, rows, cols, dtype):
    """N(0, 1) with one channel in a hundred twenty times larger, as hidden states have them."""
    x = torch.randn(rows, cols, generator=gen, device="cuda")
    big = torch.rand(cols, generator=gen, device="cuda") < 0.01
    return (x * torch.where(big, 20.0, 1.0)).to(dtype)


def _packed(gen, rows, cols, fmt, std):
    """Packed rows whose values have mean 0 and about the standard deviation `std`: uniform codes and sub-block
    scales, block scales that vary, minimums that centre the asymmetric formats."""
    be, bb = BLOCKS[fmt]
    n = rows * _up(cols, be)
    b = torch.randint(0, 256, (n, bb), generator=gen, device="cuda", dtype=torch.uint8)
    # rms of (sub-block scale * code), the ratio dmin / d, and where d (and dmin) stand
    rms, ratio, at = {"Q8_0": (73.9, 0, 0), "Q4_0": (4.65, 0, 0), "Q2_K": (14.0, 1.5, 0), "Q3_K": (42.3, 0, 108),
                      "Q4_K": (230.0, 7.5, 0), "Q5_K": (460.0, 15.5, 0), "Q6_K": (1367.0, 0, 208)}[fmt]
    # a block scale below 2^-14 (subnormal in fp16) is 0 by the formats' definition: stay above it
    d = max(std / rms, 1.3e-4) * (0.5 + torch.rand(n, 1, generator=gen, device="cuda"))
    b[:, at:at + 2] = d.half().view(torch.uint8)
    if ratio:
        b[:, 2:4] = (d * ratio).half().view(torch.uint8)
    return b.view(-1)


def _f8_weight(gen, rows, cols, std):
    """Codes [rows x cols rounded up to 16] and scales of N(0, std^2) weights, one scale per 128 x 128 block."""
    w = torch.randn(rows, cols, generator=gen, device="cuda") * std
    codes, scales = _pack_plain(w, 128)
    data = torch.zeros(rows, _up(cols, 16) * 16, device="cuda", dtype=torch.uint8)
    data[:, :cols] = codes.view(torch.uint8)
    return data.view(torch.float8_e4m3fn), scales


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "pack":
        if case["block_rows"] == 1:
            return {"case": case, "x": _activations(gen, case["rows"], case["cols"], dtype)}
        return {"case": case, "x": (torch.randn(case["rows"], case["cols"], generator=gen, device="cuda") * 0.02)
                .to(dtype)}
    if case["op"] == "linear":
        s = {"case": case, "x": _activations(gen, case["tokens"], case["cols"], dtype)}
        s["w"], s["w_scales"] = _f8_weight(gen, case["out"], case["cols"], 0.02)
        s["bias"] = torch.randn(case["out"], generator=gen, device="cuda") if case["bias"] else None
        return s
    e, h, f = case["experts"], case["hidden"], case["ffn"]
    s = {"case": case, "x": torch.randn(case["tokens"], h, generator=gen, device="cuda").to(dtype),
         "router": torch.randn(e, h, generator=gen, device="cuda") / math.sqrt(h)}
    for name, rows, cols, fmt in (("gate", e * f, h, case["fmt"]), ("up", e * f, h, case["fmt"]),
                                  ("down", e * h, f, case["fmt_down"])):
        if fmt == "F8":
            s[name], s[name + "_scales"] = _f8_weight(gen, rows, cols, 1 / math.sqrt(cols))
        else:
            s[name], s[name + "_scales"] = _packed(gen, rows, cols, fmt, 1 / math.sqrt(cols)), None
    return s


# ---------------------------------------------------------------- the operators' passes

def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    import axon_b200 as ax

    c = s["case"]
    if c["op"] == "pack":
        q = ax.quantize_f8(ax.F8Tensor.empty(c["rows"], c["cols"], c["block_rows"]), s["x"])
        return {"codes": q.data[:, :c["cols"]], "scales": q.scales}
    if c["op"] == "linear":
        w = ax.F8Tensor(s["w"], s["w_scales"], (c["out"], c["cols"]), 128)
        return ax.linear_f8(s["x"], w, bias=s["bias"])
    w = {}
    for name, rows, cols, fmt in (("gate", c["ffn"], c["hidden"], c["fmt"]), ("up", c["ffn"], c["hidden"], c["fmt"]),
                                  ("down", c["hidden"], c["ffn"], c["fmt_down"])):
        shape = (c["experts"] * rows, cols)
        w[name] = (ax.F8Tensor(s[name], s[name + "_scales"], shape, 128) if fmt == "F8"
                   else ax.QTensor(s[name], shape, ax.QuantFormat[fmt]))
    y, ids, weights = ax.moe_q(s["x"], s["router"], w["gate"], w["up"], w["down"], c["top_k"])
    return {"y": y, "ids": ids, "weights": weights}


def _pack_plain(x, block_rows):
    """e4m3 codes [rows x cols] and scales of a matrix, in 32 bits."""
    rows, cols = x.shape
    nr, nc = _up(rows, block_rows), _up(cols, 128)
    x = torch.nn.functional.pad(x.float(), (0, nc * 128 - cols, 0, nr * block_rows - rows))
    x = x.view(nr, block_rows, nc, 128)
    scales = x.abs().amax(dim=(1, 3))
    scales = scales / torch.full_like(scales, F8_MAX)  # by a tensor: by a number it would be a product with 1 / 448
    q = x / scales[:, None, :, None]
    q = torch.where(scales[:, None, :, None] == 0, 0.0, q).clamp(-F8_MAX, F8_MAX)
    q = q.to(torch.float8_e4m3fn).view(torch.uint8).view(nr * block_rows, nc * 128)[:rows, :cols]
    return q.contiguous().view(torch.float8_e4m3fn), scales


def _unpack_f8(codes, scales, block_rows, cols):
    """fp32 values of e4m3 blocks; `codes` may have padding columns."""
    rows = codes.shape[0]
    s = scales.repeat_interleave(block_rows, 0)[:rows].repeat_interleave(128, 1)[:, :cols]
    return codes[:, :cols].float() * s


def _k4_plain(b):
    """6-bit scales and minimums [..., 8] of the 12 scale bytes of Q4_K and Q5_K."""
    lo, mid, hi = b[..., 0:4], b[..., 4:8], b[..., 8:12]
    sc = torch.cat([lo & 63, (hi & 15) | ((lo >> 6) << 4)], -1)
    m = torch.cat([mid & 63, (hi >> 4) | ((mid >> 6) << 4)], -1)
    return sc.float(), m.float()


def _unpack_plain(b, fmt):
    """fp32 values [..., blocks * elements] of packed blocks [..., blocks, bytes]."""
    lead = b.shape[:-2]

    def half(at):  # subnormal scales are 0
        d = b[..., at:at + 2].contiguous().view(torch.float16).float()
        return torch.where(d.abs() < 2.0 ** -14, 0.0, d)

    two = torch.arange(0, 8, 2, device=b.device, dtype=torch.uint8).view(4, 1)
    if fmt == "Q8_0":
        v = b[..., 2:].contiguous().view(torch.int8).float() * half(0)
    elif fmt == "Q4_0":
        q = torch.stack([b[..., 2:] & 15, b[..., 2:] >> 4], -1).flatten(-2)
        v = (q.float() - 8) * half(0)
    elif fmt == "Q2_K":
        q = (b[..., 20:84].unflatten(-1, (2, 1, 32)) >> two) & 3
        sc = b[..., 4:20].unflatten(-1, (2, 4, 2)).repeat_interleave(16, -1)
        d, dmin = half(0)[..., None, None], half(2)[..., None, None]
        v = (d * (sc & 15).float()) * q.float() - dmin * (sc >> 4).float()
    elif fmt == "Q3_K":
        q = (b[..., 32:96].unflatten(-1, (2, 1, 32)) >> two) & 3
        bit = torch.arange(8, device=b.device, dtype=torch.uint8).view(2, 4, 1)
        h = (b[..., None, None, 0:32] >> bit) & 1
        s = b[..., 96:108]
        low = torch.cat([s[..., 0:8] & 15, s[..., 0:8] >> 4], -1)
        sc = low | (((s[..., None, 8:12] >> two) & 3) << 4).flatten(-2)
        sc = (sc.float() - 32).unflatten(-1, (2, 4, 2)).repeat_interleave(16, -1)
        v = (half(108)[..., None, None] * sc) * (q.float() - 4 + 4 * h.float())
    elif fmt in ("Q4_K", "Q5_K"):
        qs = b[..., -128:].unflatten(-1, (4, 1, 32))
        q = torch.cat([qs & 15, qs >> 4], -2).flatten(-3, -2)
        if fmt == "Q5_K":
            bit = torch.arange(8, device=b.device, dtype=torch.uint8).view(8, 1)
            q = q | (((b[..., None, 16:48] >> bit) & 1) << 4)
        sc, m = _k4_plain(b[..., 4:16])
        v = (half(0) * sc)[..., None] * q.float() - (half(2) * m)[..., None]
    else:  # Q6_K
        ql, qh = b[..., 0:128].unflatten(-1, (2, 2, 32)), b[..., 128:192].unflatten(-1, (2, 1, 32))
        q = torch.cat([ql & 15, ql >> 4], -2) | (((qh >> two) & 3) << 4)
        sc = b[..., 192:208].contiguous().view(torch.int8).float().unflatten(-1, (2, 4, 2)).repeat_interleave(16, -1)
        v = (half(208)[..., None, None] * sc) * (q.float() - 32)
    return v.reshape(*lead, -1)


def _experts_plain(s, name, rows, cols, fmt, pick):
    """fp32 weights [experts picked x rows x cols]; pick None: all of them."""
    e = s["case"]["experts"]
    if fmt == "F8":
        nc = _up(cols, 128)
        codes, scales = s[name].view(e, rows, -1)[..., :cols], s[name + "_scales"].view(e, rows // 128, nc)
        if pick is not None:
            codes, scales = codes.view(torch.uint8)[pick].view(torch.float8_e4m3fn), scales[pick]
        return codes.float() * scales.repeat_interleave(128, 1).repeat_interleave(128, 2)[..., :cols]
    be, bb = BLOCKS[fmt]
    b = s[name].view(e, rows, _up(cols, be), bb)
    return _unpack_plain(b if pick is None else b[pick], fmt)[..., :cols]


def _moe_plain(s):
    c, x = s["case"], s["x"]
    k, h, f = c["top_k"], c["hidden"], c["ffn"]
    p = torch.softmax(x.double() @ s["router"].double().T, -1)
    top, ids = torch.sort(p, dim=-1, descending=True, stable=True)  # ties go to the lowest index
    top, ids = top[:, :k], ids[:, :k]
    weights = (top / top.sum(-1, keepdim=True)).float()
    few = x.shape[0] * k < c["experts"]
    pick = ids.reshape(-1) if few else None
    gate, up = (_experts_plain(s, n, f, h, c["fmt"], pick) for n in ("gate", "up"))
    down = _experts_plain(s, "down", h, f, c["fmt_down"], pick)
    x32 = x.float()
    if few:  # one weight matrix for each token's choice
        xs = x32.repeat_interleave(k, 0)[..., None]
        g, u = torch.bmm(gate, xs), torch.bmm(up, xs)
        z = torch.bmm(down, g / (1 + torch.exp(-g)) * u).view(x.shape[0], k, h)
        y = (z * weights[..., None]).sum(1)
    else:  # every expert for every token, weighted by 0 where it was not chosen
        g, u = torch.matmul(x32, gate.transpose(1, 2)), torch.matmul(x32, up.transpose(1, 2))
        share = torch.zeros(x.shape[0], c["experts"], device=x.device).scatter_add_(1, ids, weights)
        z = g / (1 + torch.exp(-g)) * u * share.T[..., None]
        y = torch.bmm(z, down.transpose(1, 2)).sum(0)
    return {"y": y.to(x.dtype), "ids": ids.int(), "weights": weights}


def _run_plain(s):
    c = s["case"]
    if c["op"] == "pack":
        codes, scales = _pack_plain(s["x"], c["block_rows"])
        return {"codes": codes, "scales": scales}
    if c["op"] == "linear":
        codes, scales = _pack_plain(s["x"], 1)
        x = _unpack_f8(codes, scales, 1, c["cols"])
        y = x @ _unpack_f8(s["w"], s["w_scales"], 128, c["cols"]).T
        return (y if s["bias"] is None else y + s["bias"]).to(s["x"].dtype)
    return _moe_plain(s)


# ---------------------------------------------------------------- what a pass cannot do without

def _weight_bytes(rows, cols, fmt):
    if fmt == "F8":
        return rows * cols + 4 * _up(rows, 128) * _up(cols, 128)
    be, bb = BLOCKS[fmt]
    return rows * _up(cols, be) * bb


def work(case):
    size = {"fp32": 4, "bf16": 2, "fp16": 2}[case["dtype"]]
    if case["op"] == "pack":
        n = case["rows"] * case["cols"]
        return {"bytes": n * size + n + 4 * _up(case["rows"], case["block_rows"]) * _up(case["cols"], 128),
                "flops": 3 * n}
    if case["op"] == "linear":
        t, m, k = case["tokens"], case["out"], case["cols"]
        return {"bytes": _weight_bytes(m, k, "F8") + size * t * (m + k) + (4 * m if case["bias"] else 0),
                "flops": 2 * t * m * k}
    t, e, k, h, f = (case[n] for n in ("tokens", "experts", "top_k", "hidden", "ffn"))
    used = e * (1 - (1 - k / e) ** t)  # experts that some token chose, where each is as likely as another
    per = 2 * _weight_bytes(f, h, case["fmt"]) + _weight_bytes(h, f, case["fmt_down"])
    return {"bytes": used * per + 4 * e * h + 2 * size * t * h + 8 * t * k, "flops": 6 * t * k * h * f + 2 * t * e * h}


# ---------------------------------------------------------------- 64 bits

def _e4m3_exact(r):
    """The e4m3 value nearest to r (ties to even), as float64: steps of 2^(e-3) for r in [2^e, 2^(e+1)), of 2^-9 below 2^-6."""
    a = r.double().abs()
    e = torch.frexp(a.clamp(min=2.0 ** -6))[1].long() - 1
    step = ((e - 3 + 1023) << 52).view(torch.float64)  # 2^(e - 3) by its bits
    return torch.copysign((torch.round(a / step) * step).clamp(max=F8_MAX), r.double())


def _pack_exact(x, block_rows):
    """Code values [rows x cols] and scales, each in float64; scale and quotient are 32-bit roundings by definition.
    In bands of rows, so that a large matrix fits."""
    rows, cols = x.shape
    group = torch.arange(cols, device=x.device) // 128
    codes, scales = [], []
    band = max(128, (1 << 25) // max(cols, 1) // 128 * 128)
    for at in range(0, rows, band):
        v = x[at:at + band].float()
        big = torch.zeros(v.shape[0], _up(cols, 128), device=x.device)
        big = big.scatter_reduce(1, group.expand_as(v), v.abs(), "amax")
        if block_rows > 1:
            row = torch.arange(v.shape[0], device=x.device) // block_rows
            n = _up(v.shape[0], block_rows)
            big = torch.zeros(n, big.shape[1], device=x.device).scatter_reduce(0, row[:, None].expand_as(big), big,
                                                                               "amax")
        s = (big.double() / F8_MAX).float()
        each = (s if block_rows == 1 else s[row])[:, group].double()
        r = torch.where(each == 0, 0.0, v.double() / each).float()
        codes.append(_e4m3_exact(r).float())  # a code's value is exact in 32 bits
        scales.append(s.double())
    return torch.cat(codes), torch.cat(scales)


def _half_exact(b, at):
    bits = b[..., at].int() | (b[..., at + 1].int() << 8)
    return torch.where(bits & 0x7C00 == 0, 0, bits).short().view(torch.float16).double()  # subnormals are 0


def _unpack_exact(b, fmt):
    """float64 values of packed blocks, element by element from the format's definition."""
    be, _ = BLOCKS[fmt]
    e = torch.arange(be, device=b.device)
    i = b.short()
    if fmt == "Q8_0":
        q = i[..., 2:]
        return (torch.where(q > 127, q - 256, q).double() * _half_exact(b, 0)[..., None]).flatten(-2)
    if fmt == "Q4_0":
        q = (i[..., 2 + e // 2] >> (4 * (e % 2))) & 15
        return ((q - 8).double() * _half_exact(b, 0)[..., None]).flatten(-2)
    n, l = e // 128, e % 32
    j, run = (e // 32) % 4, e // 16
    if fmt == "Q2_K":
        q = (i[..., 20 + 32 * n + l] >> (2 * j)) & 3
        sc = i[..., 4 + run]
        v = _half_exact(b, 0)[..., None] * ((sc & 15) * q).double() - _half_exact(b, 2)[..., None] * (sc >> 4).double()
    elif fmt == "Q3_K":
        q = ((i[..., 32 + 32 * n + l] >> (2 * j)) & 3) + 4 * ((i[..., l] >> (e // 32)) & 1) - 4
        sc = ((i[..., 96 + run % 8] >> (4 * (run // 8))) & 15) + 16 * ((i[..., 104 + run % 4] >> (2 * (run // 4))) & 3)
        v = _half_exact(b, 108)[..., None] * ((sc - 32) * q).double()
    elif fmt in ("Q4_K", "Q5_K"):
        g = e // 32
        q = (i[..., (16 if fmt == "Q4_K" else 48) + 32 * (g // 2) + l] >> (4 * (g % 2))) & 15
        if fmt == "Q5_K":
            q = q + 16 * ((i[..., 16 + l] >> g) & 1)
        low = g < 4
        first, second, third = i[..., 4 + g % 4], i[..., 8 + g % 4], i[..., 12 + g % 4]
        sc = torch.where(low, first & 63, (third & 15) + 16 * (first >> 6))
        m = torch.where(low, second & 63, (third >> 4) + 16 * (second >> 6))
        v = _half_exact(b, 0)[..., None] * (sc * q).double() - _half_exact(b, 2)[..., None] * m.double()
    else:
        low = (i[..., 64 * n + 32 * (j % 2) + l] >> (4 * (j // 2))) & 15
        q = low + 16 * ((i[..., 128 + 32 * n + l] >> (2 * j)) & 3) - 32
        sc = i[..., 192 + run]
        v = _half_exact(b, 208)[..., None] * torch.where(sc > 127, sc - 256, sc).double() * q.double()
    return v.flatten(-2)


def _expert_exact(s, name, rows, cols, fmt, e):
    if fmt == "F8":
        codes = s[name][e * rows:(e + 1) * rows, :cols].double()
        at = torch.arange(e * rows, (e + 1) * rows, device=codes.device) // 128
        return codes * s[name + "_scales"].double()[at][:, torch.arange(cols, device=codes.device) // 128]
    be, bb = BLOCKS[fmt]
    b = s[name].view(s["case"]["experts"], rows, _up(cols, be), bb)[e]
    return _unpack_exact(b, fmt)[:, :cols]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "pack":
        codes, scales = _pack_exact(s["x"], case["block_rows"])
        return {"codes": codes, "scales": scales}
    x = s["x"].double()
    if case["op"] == "linear":
        codes, scales = _pack_exact(s["x"], 1)
        x = codes.double() * scales.repeat_interleave(128, 1)[:, :case["cols"]]
        w = s["w"][:, :case["cols"]].double()
        w *= s["w_scales"].double().repeat_interleave(128, 0)[:w.shape[0]].repeat_interleave(128, 1)[:, :w.shape[1]]
        y = torch.matmul(x, w.T)
        return y if s["bias"] is None else y + s["bias"].double()
    k, h, f = case["top_k"], case["hidden"], case["ffn"]
    logits = torch.matmul(x, s["router"].double().T)
    ids = torch.argsort(logits, dim=1, descending=True, stable=True)[:, :k]
    chosen = torch.gather(logits, 1, ids)
    w = torch.exp(chosen - chosen[:, :1])
    w = w / w.sum(1, keepdim=True)  # the other experts' exponentials cancel
    y = torch.zeros(x.shape[0], h, dtype=torch.float64, device=x.device)
    for e in torch.unique(ids).tolist():
        t, j = torch.nonzero(ids == e, as_tuple=True)
        g = x[t] @ _expert_exact(s, "gate", f, h, case["fmt"], e).T
        u = x[t] @ _expert_exact(s, "up", f, h, case["fmt"], e).T
        z = (g * torch.sigmoid(g) * u) @ _expert_exact(s, "down", h, f, case["fmt_down"], e).T
        y.index_add_(0, t, z * w[t, j][:, None])
    return {"y": y, "ids": ids.int(), "weights": w}
