"""What is timed of the operators behind a LoRA trained and served on a 4-bit base: block-scaled 4-bit numbers and their products, rotary
positions and counter-based dropout, through the public entry points of kiln_b200.ops, next to their plain forms.

The sizes are those of a DiT with 2048 channels (16 heads of 128), an MLP of 8192 and a text context of 1024 channels, over 1 to 4096 tokens
(rotary positions also over longer sequences), and odd ones around them.

Kinds of case:
  quant    a matrix to 4 bits and back: what loading a weight does, and what the gradient of a projection reads
  linear   16-bit activations to 4 bits, times a 4-bit weight, one epilogue
  mlp      both products of an MLP; the hidden activations leave the first product as GELU in 4 bits
  dx       the gradient of a 4-bit projection's input
  rope     rotary positions of q and k, or (inverse) the gradients of that
  dropout  dropout of an activation and of its gradient by the same mask, with or without a sum into a residual

4-bit matrices are held as kb_quant4 lays them out: two codes to a byte, the even column in the low half, rows padded to 32 columns;
the scales in pieces of 512 bytes for 128 rows x 4 blocks, row r at byte 16 (r % 32) + 4 (r / 32 % 4), pieces of a row block side by side.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
BLOCK = {"mx4": 32, "nv4": 16}
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # one token through a projection: modulation vectors, a latency chain
        {"name": "linear_1x8192x2048_nv4", "kind": "linear", "tokens": 1, "out": 8192, "in": 2048, "dtype": "f16", "fmt": "nv4", "epi": "f16"},
        # the K projection of a short prompt
        {"name": "linear_77x2048x1024_mx4", "kind": "linear", "tokens": 77, "out": 2048, "in": 1024, "dtype": "bf16", "fmt": "mx4", "epi": "f16"},
        # a projection of a token count that no tile divides, fp32 out
        {"name": "linear_1000x2048x2048_nv4_f32", "kind": "linear", "tokens": 1000, "out": 2048, "in": 2048, "dtype": "f32", "fmt": "nv4", "epi": "f32"},
        # the MLP of a block at 1024x1024: the largest call
        {"name": "mlp_4096_nv4", "kind": "mlp", "tokens": 4096, "out": 8192, "in": 2048, "dtype": "f16", "fmt": "nv4"},
        # a training step's gradient through a projection at 512x512
        {"name": "dx_1024x2048x2048_nv4", "kind": "dx", "tokens": 1024, "out": 2048, "in": 2048, "fmt": "nv4"},
        # through the up-projection at 768x1152
        {"name": "dx_3456x8192x2048_mx4", "kind": "dx", "tokens": 3456, "out": 8192, "in": 2048, "fmt": "mx4"},
        # activations of 512x768
        {"name": "quant_1536x2048_nv4_f16", "kind": "quant", "rows": 1536, "cols": 2048, "dtype": "f16", "fmt": "nv4", "exp": 0},
        # loading the up-projection's weight
        {"name": "quant_8192x2048_mx4_f32", "kind": "quant", "rows": 8192, "cols": 2048, "dtype": "f32", "fmt": "mx4", "exp": 0},
        # q and k of 512x768, three position axes
        {"name": "rope_1536_half_axes_f32", "kind": "rope", "tokens": 1536, "batch": 1, "hq": 16, "hk": 16, "dim": 128, "rot": 128, "layout": "half",
         "axes": 3, "dtype": "f32", "scaling": "none", "start": 0, "inverse": False},
        # gradients of a long sequence far into a stretched context: interleaved pairs in part of the head, few k heads
        {"name": "rope_8190_interleaved_part_bf16", "kind": "rope", "tokens": 4095, "batch": 2, "hq": 16, "hk": 4, "dim": 128, "rot": 96,
         "layout": "interleaved", "axes": 1, "dtype": "bf16", "scaling": "parts", "start": 100000, "inverse": True},
        # the input of a LoRA's down-projection at 512x768
        {"name": "dropout_1536x2048_f16", "kind": "dropout", "rows": 1536, "cols": 2048, "dtype": "f16", "p": 0.1, "resid": False},
        # the hidden activations of an MLP at 1024x1024, added to a residual
        {"name": "dropout_4096x8192_bf16_resid", "kind": "dropout", "rows": 4096, "cols": 8192, "dtype": "bf16", "p": 0.05, "resid": True},
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["linear", "linear", "linear", "mlp", "dx", "quant", "rope", "rope", "dropout"])
    fmt = rng.choice(["mx4", "nv4"])
    c = {"kind": kind}
    if kind == "linear":
        c.update(tokens=spread(1, 4096), out=spread(64, 8192), dtype=rng.choice(list(DTYPES)), fmt=fmt, epi=rng.choice(["f16", "f32", "gelu16"]))
        c["in"] = min(spread(64, 8192), 4096 * 8192 * 2048 // (c["tokens"] * c["out"]))     # no more work than one product of the largest listed case
    elif kind == "mlp":
        c.update(tokens=spread(16, 4096), out=8 * spread(64, 1024), dtype=rng.choice(list(DTYPES)), fmt=fmt)
        c["in"] = spread(128, 2048)
    elif kind == "dx":
        c.update(tokens=spread(64, 4096), out=64 * spread(2, 128), fmt=fmt)
        c["in"] = 8 * spread(32, 256)
    elif kind == "quant":
        c.update(rows=spread(1, 8192), cols=spread(32, 8192), dtype=rng.choice(list(DTYPES)), fmt=fmt, exp=rng.choice([0, -4, -9]) if fmt == "nv4" else 0)
    elif kind == "rope":
        dim = 8 * rng.randint(4, 32)
        rot = rng.choice([dim, dim, 2 * rng.randint(1, dim // 2)])
        hq = spread(1, 16)
        c.update(tokens=spread(1, 4096), batch=rng.choice([1, 1, 2, 3]), hq=hq, hk=rng.randint(1, hq), dim=dim, rot=rot,
                 layout=rng.choice(["half", "interleaved"]), axes=rng.choice([1, 1, 3]), dtype=rng.choice(list(DTYPES)),
                 scaling=rng.choice(["none", "linear", "base", "parts"]), start=rng.choice([0, 0, spread(100, 1000000)]), inverse=rng.random() < 0.4)
    else:
        c.update(rows=spread(1, 4096), cols=spread(16, 8192), dtype=rng.choice(list(DTYPES)), p=rng.choice([0.0, 0.05, 0.1, 0.5]),
                 resid=rng.random() < 0.4)
    return c


# ---------------------------------------------------------------- plain forms, in 32 bits
def _fit(x, block):
    """[rows, cols] -> [rows, blocks, block], zeros behind the last column."""
    rows, cols = x.shape
    n = -(-cols // block)
    y = torch.zeros(rows, n * block, dtype=torch.float32, device=x.device)
    y[:, :cols] = x
    return y.view(rows, n, block)


def _pow2(e):
    """2^e as the bits of a 32-bit number, exact (pow need not be); e from -126 to 127."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _quantise(x, fmt, exp=0):
    """Codes 0 to 15 [rows, blocks, block] and the scales [rows, blocks] (32-bit numbers, 2^exp left out)."""
    y = _fit(x, BLOCK[fmt]) * 2.0 ** -exp
    a = y.abs()
    top = a.amax(2)
    if fmt == "mx4":
        s = _pow2(torch.clamp(torch.frexp(top)[1] - 3, min=-126))   # frexp: top = m 2^e, m in [0.5, 1)
    else:
        t = top / torch.full_like(top, 6.0)          # a quotient, not a product with a rounded 1/6: scales next to a border
        step = _pow2(torch.clamp(torch.frexp(t)[1] - 1, min=-6) - 3)
        s = torch.clamp(torch.round(t / step) * step, 2.0 ** -9, 448.0)
    v = a / s[:, :, None]
    code = ((v > 0.25).int() + (v >= 0.75).int() + (v > 1.25).int() + (v >= 1.75).int() + (v > 2.5).int() + (v >= 3.5).int() + (v > 5.0).int())
    return code + 8 * torch.signbit(y).int(), s


def _values(code, s, exp, cols):
    """The matrix that codes and scales stand for, fp32."""
    mag = torch.tensor(E2M1, device=code.device)[(code & 7).long()]
    v = torch.where(code >= 8, -mag, mag) * s[:, :, None] * 2.0 ** exp
    return v.reshape(code.shape[0], -1)[:, :cols]


def _through4(x, fmt, exp=0):
    code, s = _quantise(x.float(), fmt, exp)
    return _values(code, s, exp, x.shape[1])


def _pack(code, s, fmt):
    """The bytes that kb_quant4 writes: codes [rows, 16 ceil(cols / 32)] and scales."""
    rows, n, block = code.shape
    c = code.reshape(rows, n * block)
    wide = torch.zeros(rows, -(-n * block // 32) * 32, dtype=torch.int32, device=c.device)
    wide[:, :n * block] = c
    packed = (wide[:, 0::2] | (wide[:, 1::2] << 4)).to(torch.uint8)
    if fmt == "mx4":
        byte = torch.frexp(s)[1] - 1 + 127
    else:
        e = torch.frexp(s)[1] - 1
        m = torch.where(e >= -6, torch.round(s * _pow2(3 - e)) - 8, torch.round(s * 512.0))
        byte = torch.where(e >= -6, (e + 7) * 8 + m.int(), m.int())
    rb, kb = -(-rows // 128), -(-n // 4)
    full = torch.zeros(rb * 128, kb * 4, dtype=torch.uint8, device=c.device)
    full[:rows, :n] = byte.to(torch.uint8)
    scales = full.view(rb, 4, 32, kb, 4).permute(0, 3, 2, 1, 4).contiguous().view(-1)     # [row block][piece][r % 32][r / 32][block]
    return packed, scales


def _unpack(packed, scales, rows, cols, fmt, exp):
    """The matrix that the bytes stand for, fp32."""
    block = BLOCK[fmt]
    n = -(-cols // block)
    code = torch.stack([packed & 15, packed >> 4], 2).view(rows, -1)[:, :n * block].int().view(rows, n, block)
    rb, kb = -(-rows // 128), -(-n // 4)
    byte = scales.view(rb, kb, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(rb * 128, kb * 4)[:rows, :n].int()
    if fmt == "mx4":
        s = _pow2(torch.clamp(byte - 127, min=-126))
    else:
        e, m = byte >> 3, (byte & 7).float()
        s = torch.where(e > 0, (1.0 + m / 8.0) * _pow2(e - 7), m / 512.0)
    return _values(code, s, exp, cols)


def _gelu(v):
    return 0.5 * v * (1.0 + torch.erf(v * math.sqrt(0.5)))


def _freqs(c):
    """Radians per position of every pair, in 64 bits, and the axis whose position turns it. The contexts are stretched by 4 from 4096."""
    n = c["rot"] // 2
    i = np.arange(n, dtype=np.float64)
    base, by, trained = 10000.0, 4.0, 4096.0
    if c["scaling"] == "base":
        base *= by ** (c["rot"] / max(c["rot"] - 2.0, 1.0))
    f = base ** (-2.0 * i / c["rot"])
    if c["scaling"] == "linear":
        f = f / by
    elif c["scaling"] == "parts":
        turns = trained * f / (2.0 * math.pi)                        # fast pairs keep their pace, slow ones are stretched, between 1 and 32 turns a mixture
        keep = np.clip((turns - 1.0) / (32.0 - 1.0), 0.0, 1.0)
        f = f * keep + f / by * (1.0 - keep)
    axis = (np.arange(n) * c["axes"] // max(n, 1)).astype(np.int32)
    return f, axis, (0.1 * math.log(by) + 1.0 if c["scaling"] == "parts" else 1.0)


def _rotate(x, heads, c, cos, sin):
    x = x.float().view(x.shape[0], heads, c["dim"])
    rot, n = c["rot"], c["rot"] // 2
    y = x.clone()
    cos, sin = cos[:, None, :], sin[:, None, :]
    if c["layout"] == "half":
        a, b = x[..., :n], x[..., n:rot]
        y[..., :n], y[..., n:rot] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y[..., 0:rot:2], y[..., 1:rot:2] = a * cos - b * sin, b * cos + a * sin
    return y.view(x.shape[0], -1)


def _mul_hi_lo(a, x):
    """Both halves of a 32-bit constant times 32-bit numbers held in int64."""
    lo, hi = a * (x & 0xffff), a * (x >> 16)
    return (hi + (lo >> 16)) >> 16, (lo + ((hi & 0xffff) << 16)) & 0xffffffff


def _philox(c0, c1, c2, c3, k0, k1):
    """Philox4x32 with ten rounds (Salmon et al., 2011) on int64 tensors that hold 32-bit words."""
    for _ in range(10):
        h0, l0 = _mul_hi_lo(0xD2511F53, c0)
        h1, l1 = _mul_hi_lo(0xCD9E8D57, c2)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & 0xffffffff, (k1 + 0xBB67AE85) & 0xffffffff
    return c0, c1, c2, c3


def _keep(rows, cols, p, rng):
    """The mask: of a row's columns 8 g to 8 g + 7 the 16-bit halves of one Philox block, low half first."""
    dev = rng.device
    g = torch.arange(-(-cols // 8), dtype=torch.int64, device=dev)[None, :].expand(rows, -1)
    r = torch.arange(rows, dtype=torch.int64, device=dev)[:, None].expand_as(g)
    w = _philox(g, r, (rng[1] & 0xffffffff).expand_as(g), ((rng[1] >> 32) & 0xffffffff).expand_as(g), rng[0] & 0xffffffff, (rng[0] >> 32) & 0xffffffff)
    halves = torch.stack([w[0] & 0xffff, w[0] >> 16, w[1] & 0xffff, w[1] >> 16, w[2] & 0xffff, w[2] >> 16, w[3] & 0xffff, w[3] >> 16], 2)
    return halves.reshape(rows, -1)[:, :cols] >= int(math.floor(65536.0 * p + 0.5))


def _dropped(x, keep, p):
    t = int(math.floor(65536.0 * p + 0.5))
    return torch.where(keep, x.float() * (65536.0 / (65536 - t)), torch.zeros((), device=x.device))


# ---------------------------------------------------------------- cases
def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")
    st = {"case": c}

    def weight(name, n, k):
        """Normal weights of a trained projection's size, in 4 bits (nv4: with the power of two that brings their scales into range)."""
        exp = -9 if c["fmt"] == "nv4" else 0
        code, s = _quantise(randn(n, k) / math.sqrt(k), c["fmt"], exp)
        st[name] = _pack(code, s, c["fmt"]) + (n, k, c["fmt"], exp)

    kind = c["kind"]
    if kind in ("linear", "mlp"):
        # normalised activations: most channels near 1, a few outlying ones
        x = randn(c["tokens"], c["in"]) * (1.0 + 4.0 * (torch.rand(c["in"], generator=gen, device="cuda") < 0.01))
        st["x"] = x.to(DTYPES[c["dtype"]])
        weight("w", c["out"], c["in"])
        if kind == "mlp":
            weight("w2", c["in"], c["out"])
    elif kind == "dx":
        st["dy"] = randn(c["tokens"], c["out"]).half()
        weight("w", c["out"], c["in"])
    elif kind == "quant":
        st["x"] = (randn(c["rows"], c["cols"]) * 2.0 ** c["exp"]).to(DTYPES[c["dtype"]])
    elif kind == "rope":
        rows = c["batch"] * c["tokens"]
        st["q"] = randn(rows, c["hq"] * c["dim"]).to(DTYPES[c["dtype"]])
        st["k"] = randn(rows, c["hk"] * c["dim"]).to(DTYPES[c["dtype"]])
        t = torch.arange(c["tokens"], device="cuda", dtype=torch.int32)
        if c["axes"] == 3:                                            # frame, row, column of a patch grid
            wide = max(1, int(math.sqrt(c["tokens"])))
            st["pos"] = torch.stack([torch.zeros_like(t), t // wide, t % wide], 1) + c["start"]
        else:
            st["pos"] = t[:, None] + c["start"]
        st["freq"], st["axis"], st["amplitude"] = _freqs(c)
    else:
        st["x"] = randn(c["rows"], c["cols"]).to(DTYPES[c["dtype"]])
        st["dy"] = randn(c["rows"], c["cols"]).to(DTYPES[c["dtype"]])
        st["resid"] = randn(c["rows"], c["cols"]).to(DTYPES[c["dtype"]]) if c["resid"] else None
        st["rng"] = torch.randint(-2 ** 62, 2 ** 62, (2,), generator=gen, device="cuda")     # seed and offset of a training step
    return st


def _run_own(st):
    from kiln_b200 import ops
    c = st["case"]
    kind = c["kind"]
    FMT = {"mx4": ops.MX4, "nv4": ops.NV4}

    def weight(name):
        packed, scales, n, k, fmt, exp = st[name]
        return ops.Quant4(packed, scales, n, k, FMT[fmt], exp)

    if kind == "quant":
        q = ops.quant4(st["x"], FMT[c["fmt"]], exp=c["exp"])
        return ops.dequant4(torch.empty(c["rows"], c["cols"], device="cuda"), q)
    if kind == "linear":
        x4 = ops.quant4(st["x"], FMT[c["fmt"]])
        epi = {"f16": ops.EPI_F16, "f32": ops.EPI_F32, "gelu16": ops.EPI_GELU16}[c["epi"]]
        out = ops.padded_empty(c["tokens"], c["out"], torch.float32 if c["epi"] == "f32" else torch.float16, "cuda")
        return ops.linear4(out, x4, weight("w"), epi)
    if kind == "mlp":
        x4 = ops.quant4(st["x"], FMT[c["fmt"]])
        h4 = ops.quant4_empty(c["tokens"], c["out"], FMT[c["fmt"]], "cuda")
        ops.linear4(h4, x4, weight("w"), ops.EPI_GELU4)
        out = ops.padded_empty(c["tokens"], c["in"], torch.float16, "cuda")
        return ops.linear4(out, h4, weight("w2"), ops.EPI_F16)
    if kind == "dx":
        return ops.linear4_dx(torch.empty(c["tokens"], c["in"], device="cuda", dtype=torch.float16), st["dy"], weight("w"))
    if kind == "rope":
        outs = [torch.empty_like(st["q"]), torch.empty_like(st["k"])]
        layout = ops.ROPE_HALF if c["layout"] == "half" else ops.ROPE_INTERLEAVED
        return ops.rope(outs, [st["q"], st["k"]], [c["hq"], c["hk"]], c["dim"], st["pos"], st["freq"], st["axis"], layout=layout,
                        amplitude=st["amplitude"], inverse=c["inverse"])
    y = ops.dropout(torch.empty_like(st["x"]), st["x"], st["rng"], c["p"], resid=st["resid"])
    dx = ops.dropout(torch.empty_like(st["x"]), st["dy"], st["rng"], c["p"])
    return [y, dx]


def run(state):
    st = state
    if own:
        return _run_own(st)
    c = st["case"]
    kind = c["kind"]
    if kind == "quant":
        return _through4(st["x"], c["fmt"], c["exp"])
    if kind == "linear":
        y = _through4(st["x"], c["fmt"]) @ _unpack(*st["w"]).t()
        return y if c["epi"] == "f32" else (_gelu(y) if c["epi"] == "gelu16" else y).half()
    if kind == "mlp":
        h = _gelu(_through4(st["x"], c["fmt"]) @ _unpack(*st["w"]).t())
        return (_through4(h, c["fmt"]) @ _unpack(*st["w2"]).t()).half()
    if kind == "dx":
        return (st["dy"].float() @ _unpack(*st["w"])).half()
    if kind == "rope":
        pos = st["pos"].repeat(c["batch"], 1).double()[:, torch.from_numpy(st["axis"]).to("cuda").long()]
        t = pos * torch.from_numpy(st["freq"]).to("cuda") * (-1.0 if c["inverse"] else 1.0)      # far positions turn many times: the angle in 64 bits
        cos, sin = (torch.cos(t) * st["amplitude"]).float(), (torch.sin(t) * st["amplitude"]).float()
        return [_rotate(st["q"], c["hq"], c, cos, sin).to(st["q"].dtype), _rotate(st["k"], c["hk"], c, cos, sin).to(st["k"].dtype)]
    keep = _keep(c["rows"], c["cols"], c["p"], st["rng"])
    y = _dropped(st["x"], keep, c["p"])
    if st["resid"] is not None:
        y = y + st["resid"].float()
    return [y.to(st["x"].dtype), _dropped(st["dy"], keep, c["p"]).to(st["x"].dtype)]


def work(case):
    c = case
    kind = c["kind"]
    size = {"f16": 2, "bf16": 2, "f32": 4}
    four = lambda r, k: r * k * (0.5 + 1.0 / BLOCK[c["fmt"]])       # bytes of a 4-bit matrix
    if kind == "quant":
        n = c["rows"] * c["cols"]
        return {"bytes": n * (size[c["dtype"]] + 4) + 2 * four(c["rows"], c["cols"]), "flops": 4 * n}
    if kind == "rope":
        n = c["batch"] * c["tokens"] * (c["hq"] + c["hk"]) * c["dim"]
        return {"bytes": 2 * n * size[c["dtype"]] + 4 * c["axes"] * c["tokens"], "flops": 3 * n * c["rot"] // c["dim"]}
    if kind == "dropout":
        n = c["rows"] * c["cols"]
        return {"bytes": n * size[c["dtype"]] * (5 if c["resid"] else 4), "flops": 4 * n}
    m, n, k = c["tokens"], c["out"], c["in"]
    if kind == "dx":
        return {"bytes": 2 * m * (n + k) + four(n, k), "flops": 2 * m * n * k}
    if kind == "mlp":
        return {"bytes": m * k * (size[c["dtype"]] + 2) + 2 * four(n, k), "flops": 4 * m * n * k}
    return {"bytes": m * k * size[c["dtype"]] + four(n, k) + m * n * (4 if c["epi"] == "f32" else 2), "flops": 2 * m * n * k}


# ---------------------------------------------------------------- the definition in 64 bits
def _nearest4(x, fmt, exp):
    """Every element replaced by the nearest value that its block of 4-bit numbers can hold, 64 bits."""
    block = BLOCK[fmt]
    rows, cols = x.shape
    pad = -cols % block
    y = torch.cat([x.double(), torch.zeros(rows, pad, dtype=torch.float64, device=x.device)], 1) * 2.0 ** -exp
    y = y.view(rows, -1, block)
    top = y.abs().max(dim=2, keepdim=True).values
    two = lambda e: ((e.long() + 1023) << 52).view(torch.float64)                # 2^e
    floor2 = lambda v: (torch.clamp(v, min=2.0 ** -140).view(torch.int64) >> 52) - 1023
    if fmt == "mx4":
        s = two(torch.clamp(floor2(top) - 2, min=-127))
    else:
        want = top / torch.full_like(top, 6)         # a quotient: ties stay ties
        e = torch.clamp(floor2(want), min=-6)
        s = torch.clamp(torch.round(want * two(3 - e)) * two(e - 3), 2.0 ** -9, 448.0)
    v = torch.clamp(y.abs() / s, max=6.0)
    step = torch.where(v < 2, 0.5, torch.where(v < 4, 1.0, 2.0))
    v = torch.round(v / step) * step
    return (torch.where(y < 0, -v, v) * s * 2.0 ** exp).view(rows, -1)[:, :cols]


def _held(w):
    """What a packed weight stands for, 64 bits, byte by byte from the layout's description."""
    packed, scales, n, k, fmt, exp = w
    p, s = packed.cpu().numpy(), scales.cpu().numpy()
    r, j = np.arange(n)[:, None], np.arange(k)[None, :]
    byte = p[r, j // 2]
    code = np.where(j % 2 == 0, byte & 15, byte >> 4).astype(np.int64)
    b = j // BLOCK[fmt]
    pieces = -(-(-(-k // BLOCK[fmt])) // 4)
    sb = s[((r // 128) * pieces + b // 4) * 512 + (r % 32) * 16 + (r // 32 % 4) * 4 + b % 4].astype(np.int64)
    if fmt == "mx4":
        scale = 2.0 ** (sb - 127.0)
    else:
        scale = np.where(sb >= 8, (8 + sb % 8) * 2.0 ** (sb // 8 - 10.0), sb * 2.0 ** -9)
    v = np.array(E2M1)[code % 8] * scale * 2.0 ** exp
    return torch.from_numpy(np.where(code >= 8, -v, v)).to(packed.device)


def _words(rows, cols, seed, offset):
    """The 16-bit number behind every element, from 64-bit integers."""
    m32 = np.uint64(0xffffffff)
    g = -(-cols // 8)
    c0 = np.tile(np.arange(g, dtype=np.uint64), rows)
    c1 = np.repeat(np.arange(rows, dtype=np.uint64), g)
    c2, c3 = np.full_like(c0, offset & 0xffffffff), np.full_like(c0, offset >> 32)
    k = [seed & 0xffffffff, seed >> 32]
    for _ in range(10):
        p0, p1 = np.uint64(0xD2511F53) * c0, np.uint64(0xCD9E8D57) * c2
        c0, c1, c2, c3 = (p1 >> np.uint64(32)) ^ c1 ^ np.uint64(k[0]), p1 & m32, (p0 >> np.uint64(32)) ^ c3 ^ np.uint64(k[1]), p0 & m32
        k = [(k[0] + 0x9E3779B9) % 2 ** 32, (k[1] + 0xBB67AE85) % 2 ** 32]
    words = np.stack([c0, c1, c2, c3], 1).astype("<u4")
    return words.view("<u2").reshape(rows, 8 * g)[:, :cols]


def exact(case, seed):
    c = case
    st = prepare(c, seed)
    kind = c["kind"]
    gelu = lambda v: v * torch.special.ndtr(v)
    if kind == "quant":
        return _nearest4(st["x"], c["fmt"], c["exp"])
    if kind in ("linear", "mlp"):
        y = _nearest4(st["x"], c["fmt"], 0) @ _held(st["w"]).T
        if kind == "mlp":
            return _nearest4(gelu(y), c["fmt"], 0) @ _held(st["w2"]).T
        return gelu(y) if c["epi"] == "gelu16" else y
    if kind == "dx":
        return st["dy"].double() @ _held(st["w"])
    if kind == "rope":
        pos = st["pos"].cpu().numpy().astype(np.float64)[:, st["axis"]]
        z = np.exp((-1j if c["inverse"] else 1j) * pos * st["freq"]) * st["amplitude"]
        z = torch.from_numpy(np.tile(z, (c["batch"], 1))).to("cuda")[:, None, :]
        outs = []
        for x, heads in ((st["q"], c["hq"]), (st["k"], c["hk"])):
            x = x.double().view(x.shape[0], heads, c["dim"])
            turned, rest = x[..., :c["rot"]], x[..., c["rot"]:]
            if c["layout"] == "half":
                w = torch.complex(*turned.reshape(*turned.shape[:2], 2, -1).unbind(2)) * z
                turned = torch.cat([w.real, w.imag], 2)
            else:
                w = torch.complex(*turned.reshape(*turned.shape[:2], -1, 2).unbind(3)) * z
                turned = torch.view_as_real(w).reshape(turned.shape)
            outs.append(torch.cat([turned, rest], 2).reshape(x.shape[0], -1))
        return outs
    sd, off = (int(v) % 2 ** 64 for v in st["rng"].cpu())
    t = int(math.floor(65536.0 * c["p"] + 0.5))
    keep = torch.from_numpy(_words(c["rows"], c["cols"], sd, off).astype(np.int32)).to("cuda") >= t
    y, dx = (torch.where(keep, v.double() * (65536 / (65536 - t)), 0.0) for v in (st["x"], st["dy"]))
    return [y + st["resid"].double() if c["resid"] else y, dx]
