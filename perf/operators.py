"""What the framework's microscaled 4-bit (MXFP4) operators are measured on: a
list of cases, a generator of more of the same ranges, and the operators in
their plain form.

  listed()              the cases
  draw(rng)             one more case of the same ranges
  prepare(case, seed)   inputs on the GPU; for the framework's operators also the
                        uploaded weights and, for decode, the captured graph
  run(state)            one pass: the plain form, or (own) the framework's calls
  work(case)            bytes and operations a pass cannot do without
  exact(case, seed)     the same outputs in 64 bits

Operators (op):
  quantize    rows of fp32 into MXFP4 blocks, and the values they stand for
  matvec      W x for one token, W in MXFP4, several layers
  matmul      X W^T for many tokens, X in fp32
  matmul_q    the same with X quantised to MXFP4 in the call
  experts     router, top-k and the selected experts' FFN, experts in MXFP4,
              several tokens one after the other

An MXFP4 block holds 32 elements in 17 bytes: a scale byte e (2^(e - 127)) and
16 bytes of 4-bit codes, element i in the low and element 16 + i in the high
half of byte i.  A code is a sign and one of 0, .5, 1, 1.5, 2, 3, 4, 6.
Weights are blocks of trained weights' size (about 0.03, the blocks' scales a
few powers of two apart); activations are normal with a few channels ten times
larger, as after a norm in a trained model.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

BLOCK, BYTES = 32, 17
MAGNITUDES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


# ------------------------------------------------------------------- the cases
def listed():
    return [
        # one token's activations before a 4-bit product, called eagerly
        {"name": "quantize_token", "op": "quantize", "rows": 1, "cols": 2816},
        # the weights of one layer, quantised on the device after a load
        {"name": "quantize_weights", "op": "quantize", "rows": 9728, "cols": 4096},
        # an attention or FFN projection of a decode step, 16 layers of it
        {"name": "matvec_square", "op": "matvec", "rows": 4096, "cols": 4096, "layers": 16},
        # a projection of a small model: rows of 28 blocks, sizes no powers of two
        {"name": "matvec_ragged", "op": "matvec", "rows": 4865, "cols": 896, "layers": 12},
        # the output head of a 262,144-word vocabulary, once a token
        {"name": "matvec_head", "op": "matvec", "rows": 262144, "cols": 2816, "layers": 1},
        # several sequences' decode step together, or a short speculative run
        {"name": "matmul_batch", "op": "matmul", "tokens": 7, "rows": 4096, "cols": 4096},
        # an ordinary prompt, of odd length, through an FFN's up projection
        {"name": "matmul_prompt", "op": "matmul", "tokens": 509, "rows": 4864, "cols": 2816},
        # a long prompt's batch of tokens
        {"name": "matmul_long", "op": "matmul", "tokens": 4096, "rows": 8192, "cols": 4096},
        # a prompt with 4-bit activations
        {"name": "matmul_q_prompt", "op": "matmul_q", "tokens": 1024, "rows": 4096, "cols": 4096},
        # a long prompt with 4-bit activations, odd sizes
        {"name": "matmul_q_long", "op": "matmul_q", "tokens": 4095, "rows": 7001, "cols": 2816},
        # decode of the 128-expert, top-8 layer
        {"name": "experts_decode", "op": "experts", "tokens": 8, "experts": 128, "d_model": 2048, "d_expert": 768,
         "k": 8, "act": "silu", "norm_topk": True},
        # decode of a layer of fewer, larger experts whose width is no power of two
        {"name": "experts_wide", "op": "experts", "tokens": 6, "experts": 32, "d_model": 2816, "d_expert": 2112,
         "k": 4, "act": "gelu", "norm_topk": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cols(rng, lo, hi):
    """A whole number of blocks, over its logarithm."""
    return min(hi, max(lo, BLOCK * int(round(_log(rng, lo, hi) / BLOCK))))


def draw(rng):
    op = rng.choice(["quantize", "matvec", "matvec", "matvec", "matmul", "matmul", "matmul", "matmul_q", "matmul_q",
                     "experts", "experts"])
    if op == "quantize":
        cols = _cols(rng, 32, 16384)
        return {"op": op, "rows": min(_log(rng, 1, 20000), 39_000_000 // cols), "cols": cols}
    if op == "matvec":
        cols = _cols(rng, 256, 16384)
        rows = min(_log(rng, 64, 160000), 600_000_000 // cols)
        return {"op": op, "rows": rows, "cols": cols, "layers": max(1, min(16, 200_000_000 // (rows * cols)))}
    if op in ("matmul", "matmul_q"):
        return {"op": op, "tokens": _log(rng, 2, 4096), "rows": _log(rng, 200, 8192), "cols": _cols(rng, 256, 4096)}
    experts, k = rng.choice([8, 32, 60, 128]), rng.choice([1, 2, 4, 6, 8])
    d, f = BLOCK * rng.randint(24, 90), BLOCK * rng.randint(8, 2200 // BLOCK if experts < 60 else 32)
    return {"op": op, "tokens": min(rng.randint(1, 8), max(1, 600_000_000 // (3 * d * f * k))), "experts": experts,
            "d_model": d, "d_expert": f, "k": k, "act": rng.choice(["silu", "gelu"]), "norm_topk": rng.random() < 0.6}


# ------------------------------------------------------------------- the inputs
def _gen(seed, what):
    g = torch.Generator(device="cuda")
    g.manual_seed((int(seed) * 1_000_003 + what) & 0x7FFFFFFF)
    return g


def _activations(g, rows, n):
    x = torch.randn(rows, n, generator=g, device="cuda")
    big = torch.rand(n, generator=g, device="cuda") < 0.004
    return torch.where(big, x * 10.0, x).contiguous()


def _blocks(g, rows, cols):
    """uint8 [rows, cols / 32 * 17]: blocks of weights of about 0.03."""
    b = torch.randint(0, 256, (rows, cols // BLOCK, BYTES), generator=g, device="cuda", dtype=torch.uint8)
    b[..., 0] = torch.randint(119, 123, (rows, cols // BLOCK), generator=g, device="cuda", dtype=torch.uint8)
    return b.view(rows, -1)


def _inputs(case, seed):
    op, g, gx = case["op"], _gen(seed, 1), _gen(seed, 2)
    if op == "quantize":
        return {"x": _activations(gx, case["rows"], case["cols"])}
    if op == "matvec":
        n, r, c = case["layers"], case["rows"], case["cols"]
        return {"w": _blocks(g, n * r, c).view(n, r, -1), "x": _activations(gx, n, c)}
    if op in ("matmul", "matmul_q"):
        return {"w": _blocks(g, case["rows"], case["cols"]), "x": _activations(gx, case["tokens"], case["cols"])}
    e, d, f = case["experts"], case["d_model"], case["d_expert"]
    return {"router": torch.randn(e, d, generator=g, device="cuda") * 0.02, "gu": _blocks(g, e * 2 * f, d).view(e, 2 * f, -1),
            "dn": _blocks(g, e * d, f).view(e, d, -1), "x": _activations(gx, case["tokens"], d)}


class State:
    """What a program has in hand before the call."""

    def __init__(self, case, inputs):
        self.case, self.v = case, inputs
        self.handles = None  # the framework's side of it


def prepare(case, seed):
    s = State(case, _inputs(case, seed))
    if own:  # the weights uploaded once, the outputs' memory, a decode loop's graph
        s.handles = _Handles(case, s.v)
    torch.cuda.synchronize()
    return s


# ------------------------------------------------------------------- the framework's calls
_context = []


def _framework():
    """(package, context) of this repository."""
    if not _context:
        root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        sys.path.insert(0, os.path.join(root, "llmtoy-zig_amd"))
        import llmtoy_amd as lt
        _context.append((lt, lt.Context(0)))
    return _context[0]


class _Handles:
    """Uploaded weights, output buffers and the calls of one pass; gives the
    weights back."""

    def __init__(self, case, v):
        self.lt, self.ctx = _framework()
        self.tensors, self.graph = [], None
        op, x = case["op"], v["x"]
        mx, ctx = self.lt.ggml.MXFP4, self.ctx
        if op == "quantize":
            t = self.keep(ctx.create(mx, case["rows"], case["cols"]))
            self.out = torch.zeros_like(x)

            def once():
                ctx.quantize(t, x)
                ctx.dequantize(self.out, t)
        elif op == "matvec":
            n, r, c = case["layers"], case["rows"], case["cols"]
            self.out = torch.zeros(n, r, device="cuda")
            io = [(self.upload(v["w"][i], mx, r, c), x[i], self.out[i]) for i in range(n)]

            def once():
                for w, xi, oi in io:
                    ctx.quant_matvec(oi, w, xi)
        elif op in ("matmul", "matmul_q"):
            w = self.upload(v["w"], mx, case["rows"], case["cols"])
            self.out = torch.zeros(case["tokens"], case["rows"], device="cuda")
            if op == "matmul":
                def once():
                    ctx.quant_matmul(self.out, w, x)
            else:
                xq = self.keep(ctx.create(mx, case["tokens"], case["cols"]))

                def once():
                    ctx.quantize(xq, x)
                    ctx.quant_matmul(self.out, w, xq)
        else:
            n, e, d, f, k = case["tokens"], case["experts"], case["d_model"], case["d_expert"], case["k"]
            router = self.upload(v["router"].view(torch.uint8), self.lt.ggml.F32, e, d)
            gu, dn = self.upload(v["gu"], mx, 2 * f, d, e), self.upload(v["dn"], mx, d, f, e)
            out = torch.zeros(n, d, device="cuda")
            ids = torch.zeros(n, k, dtype=torch.int32, device="cuda")
            p = torch.zeros(n, k, device="cuda")
            self.out = {"ids": ids, "weights": p, "out": out}
            act = self.lt.ACT_SILU if case["act"] == "silu" else self.lt.ACT_GELU_TANH
            io = [(out[i], x[i], ids[i], p[i]) for i in range(n)]

            def once():
                for oi, xi, ii, pi in io:
                    ctx.moe_forward(oi, xi, router, gu, dn, k, f, act=act, norm_topk=case["norm_topk"], out_ids=ii,
                                    out_w=pi)
        self.once = once
        if op in ("matvec", "experts"):  # a decode loop replays its calls from a graph
            torch.cuda.synchronize()
            once()  # sizes the context's scratch
            ctx.sync()
            from llmtoy_amd import hip
            self.graph = hip.Graph(ctx.stream, once)

    def keep(self, t):
        self.tensors.append(t)
        return t

    def upload(self, blocks, kind, rows, cols, n_experts=1):
        return self.keep(self.ctx.upload(blocks.cpu().numpy(), kind, rows, cols, n_experts))

    def __del__(self):
        torch.cuda.synchronize()
        if self.graph is not None:
            self.graph.destroy()
        for t in self.tensors:
            t.free()


# ------------------------------------------------------------------- the plain form
def _decode(b, cols):
    """fp32 [..., cols] of MXFP4 block bytes."""
    b = b.view(*b.shape[:-1], cols // BLOCK, BYTES)
    table = torch.tensor(MAGNITUDES + [-m for m in MAGNITUDES], device=b.device)
    q = b[..., 1:].int()
    v = table[torch.cat([q & 15, q >> 4], -1)]
    v = torch.ldexp(v, b[..., :1].int() - 127)  # (scales of normal numbers: a product with a power of two)
    return v.view(*b.shape[:-2], cols)


def _quantized(x):
    """The values that the MXFP4 blocks of x's rows stand for, fp32."""
    v = x.view(*x.shape[:-1], -1, BLOCK)
    top = torch.frexp(v.abs().amax(-1, keepdim=True)).exponent - 3  # floor(log2) - 2
    m = torch.ldexp(v.abs(), -top)
    step = torch.where(m < 2, 0.5, torch.where(m < 4, 1.0, 2.0))
    m = (torch.round(m / step) * step).clamp(max=6.0)
    return torch.copysign(torch.ldexp(m, top), v).view(x.shape)


def _activate(case, g):
    if case["act"] == "silu":
        return g / (1 + torch.exp(-g))
    return 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g * g * g)))


def _experts(case, v):
    x, f, d, k = v["x"], case["d_expert"], case["d_model"], case["k"]
    logits = x.double() @ v["router"].double().T  # next to a border between two experts 32 bits would not do
    order = torch.sort(logits, dim=-1, descending=True, stable=True).indices
    ids = order[:, :k]
    p = torch.exp(logits - logits.amax(-1, keepdim=True))
    sel = p.gather(-1, ids)
    w = (sel / (sel if case["norm_topk"] else p).sum(-1, keepdim=True)).float()
    gu = _decode(v["gu"][ids], d) @ x[:, None, :, None]
    h = _activate(case, gu[..., :f, :]) * gu[..., f:, :]
    y = (_decode(v["dn"][ids], f) @ h).squeeze(-1)
    return {"ids": ids.int(), "weights": w, "out": (w.unsqueeze(-1) * y).sum(1)}


def _plain(case, v):
    op, x = case["op"], v["x"]
    if op == "quantize":
        return _quantized(x)
    if op == "matvec":
        return (_decode(v["w"], case["cols"]) @ x.unsqueeze(-1)).squeeze(-1)
    if op == "matmul":
        return x @ _decode(v["w"], case["cols"]).T
    if op == "matmul_q":
        return _quantized(x) @ _decode(v["w"], case["cols"]).T
    return _experts(case, v)


def run(state):
    if not own:
        return _plain(state.case, state.v)
    h = state.handles
    if h.graph is not None:
        h.graph.launch()
    else:
        h.once()
    return h.out


# ------------------------------------------------------------------- what a pass needs
def _weight_bytes(rows, cols):
    return rows * (cols // BLOCK) * BYTES


def work(case):
    op = case["op"]
    if op == "quantize":
        n = case["rows"] * case["cols"]
        return {"bytes": 8 * n, "flops": 4 * n}
    if op == "matvec":
        r, c = case["rows"], case["cols"]
        return {"bytes": case["layers"] * (_weight_bytes(r, c) + 4 * (r + c)), "flops": case["layers"] * 2 * r * c}
    if op in ("matmul", "matmul_q"):
        t, r, c = case["tokens"], case["rows"], case["cols"]
        return {"bytes": _weight_bytes(r, c) + 4 * t * (r + c), "flops": 2 * t * r * c}
    t, e, d, f, k = case["tokens"], case["experts"], case["d_model"], case["d_expert"], case["k"]
    return {"bytes": t * (k * (_weight_bytes(2 * f, d) + _weight_bytes(d, f)) + 4 * e * d + 8 * d),
            "flops": t * (6 * k * d * f + 2 * e * d)}


# ------------------------------------------------------------------- the same in 64 bits
def _decode64(b, cols):
    """float64 [rows, cols]: the format's definition, sign * 2^(e - 127) * (0 or 1).m, by bits."""
    b = b.reshape(-1, BYTES)
    q = torch.stack([b[:, 1:] & 15, b[:, 1:] >> 4], 1).reshape(-1, BLOCK).double()
    sign = torch.where(q >= 8, -1.0, 1.0).double()
    q = q - 8 * (q >= 8)
    man, ex = q % 2, torch.floor(q / 2)
    v = torch.where(ex == 0, 0.5 * man, (1 + 0.5 * man) * 2.0 ** (ex - 1))
    return (sign * v * 2.0 ** (b[:, :1].double() - 127)).view(-1, cols)


def _quantized64(x):
    """The nearest of the eight magnitudes, a tie to the even one."""
    v = x.double().reshape(-1, BLOCK)
    a = v.abs()
    unit = 2.0 ** (torch.floor(torch.log2(a.amax(1, keepdim=True))) - 2)
    code = torch.zeros_like(a)
    for i in range(7):  # past the middle of two neighbours; at the middle itself only to an even code
        middle = (MAGNITUDES[i] + MAGNITUDES[i + 1]) / 2 * unit
        code += (a >= middle) if i % 2 else (a > middle)
    mags = torch.tensor(MAGNITUDES, device=x.device, dtype=torch.float64)
    return (torch.sign(v) * mags[code.long()] * unit).view(x.shape)


def _act64(case, g):
    if case["act"] == "silu":
        return g * torch.sigmoid(g)
    return g * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3))


def exact(case, seed):
    op, v = case["op"], _inputs(case, seed)
    x = v["x"].double()
    if op == "quantize":
        return _quantized64(v["x"])
    if op == "matvec":
        part = max(1, 50_000_000 // case["cols"])
        return torch.stack([torch.cat([_decode64(p, case["cols"]) @ x[i] for p in v["w"][i].split(part)])
                            for i in range(case["layers"])])
    if op in ("matmul", "matmul_q"):
        return (x if op == "matmul" else _quantized64(v["x"])) @ _decode64(v["w"], case["cols"]).T
    d, f = case["d_model"], case["d_expert"]
    logits = x @ v["router"].double().T
    p = logits.softmax(-1)
    w, ids = p.topk(case["k"], -1)
    if case["norm_topk"]:
        w = w / w.sum(-1, keepdim=True)
    out = torch.zeros_like(x)
    for t in range(case["tokens"]):
        for s, e in enumerate(ids[t].tolist()):
            gate_up = _decode64(v["gu"][e], d) @ x[t]
            out[t] += w[t, s] * (_decode64(v["dn"][e], f) @ (_act64(case, gate_up[:f]) * gate_up[f:]))
    return {"ids": None, "weights": w, "out": out}
