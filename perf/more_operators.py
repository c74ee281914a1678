"""What the framework's attention operators are measured on: a list of cases,
a generator of more of the same ranges, and the operators in their plain form.

  listed()              the cases
  draw(rng)             one more case of the same ranges
  prepare(case, seed)   inputs on the GPU; for the framework's operators also the
                        filled caches and, for decode, the captured graph
  run(state)            one pass: the plain form, or (own) the framework's calls
  work(case)            bytes and operations a pass cannot do without
  exact(case, seed)     the same outputs in 64 bits

Operators (op):
  rope        RMS norms of queries and keys for each head, then the position
              rotation
  plan        block tables, slot maps and the batch's layout from the lengths of
              the requests and a list of free blocks
  append      keys and values into a cache of 8-bit blocks, and the values that
              the blocks touched stand for
  attention   queries over such a cache

A cache block holds 32 tokens of a sequence.  For each block and head, keys and
values each have one scale, s = max |x| / 127 over the block's tokens so far,
and a code round(x / s) an element (a tie to the even one).  The tokens of a
batch lie one sequence after the other; a sequence's tokens in the batch are its
last ones; a query sees the keys of its own position and before, of the last
`window` positions where that is not 0.

Queries and keys are normal with a few channels larger, as after a norm in a
trained model; block tables are permutations, as after a while of serving.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

BLOCK = 32
NONE = -1


# ------------------------------------------------------------------- the cases
def listed():
    return [
        # one token's queries and keys, 16 layers of a decode step
        {"name": "rope_token", "op": "rope", "tokens": 1, "heads": 32, "kv_heads": 4, "head_dim": 128, "n_rot": 128,
         "base": 1e6, "style": "neox", "fused": True, "far": 40000, "layers": 16},
        # a long prompt, read out of the fused projection; half of each head is rotated
        {"name": "rope_prompt", "op": "rope", "tokens": 4095, "heads": 16, "kv_heads": 8, "head_dim": 256, "n_rot": 128,
         "base": 1e4, "style": "pairs", "fused": True, "far": 1000000, "layers": 1},
        # a decode step of a few requests
        {"name": "plan_few", "op": "plan", "seqs": 8, "new": 1, "rest": 1, "context": 2000, "room": 8, "table": 256},
        # a step of many requests: some prompts, mostly single tokens, some rows idle
        {"name": "plan_many", "op": "plan", "seqs": 2000, "new": 600, "rest": 9, "context": 30000, "room": 65536,
         "table": 1024},
        # one token of 16 requests, 8 layers of a decode step
        {"name": "append_token", "op": "append", "seqs": 16, "new": 1, "rest": 1, "open": True, "kv_heads": 8,
         "head_dim": 128, "layers": 8},
        # two prompts of odd length
        {"name": "append_prompt", "op": "append", "seqs": 2, "new": 4095, "rest": 701, "open": False, "kv_heads": 8,
         "head_dim": 128, "layers": 1},
        # decode of a small model at an ordinary length (14 heads over 2), 12 layers
        {"name": "attention_token", "op": "attention", "seqs": 1, "new": 1, "rest": 1, "context": 1500, "heads": 14,
         "kv_heads": 2, "head_dim": 64, "window": 0, "layers": 12},
        # one request's decode over a long context
        {"name": "attention_long", "op": "attention", "seqs": 1, "new": 1, "rest": 1, "context": 131072, "heads": 32,
         "kv_heads": 4, "head_dim": 128, "window": 0, "layers": 1},
        # a batch of requests of very different lengths
        {"name": "attention_batch", "op": "attention", "seqs": 48, "new": 1, "rest": 1, "context": 8191, "heads": 32,
         "kv_heads": 4, "head_dim": 128, "window": 0, "layers": 1},
        # a layer with a sliding window, three tokens a request (one drawn, two proposed)
        {"name": "attention_window", "op": "attention", "seqs": 12, "new": 3, "rest": 3, "context": 5000, "heads": 16,
         "kv_heads": 8, "head_dim": 256, "window": 1024, "layers": 4},
        # a prompt of odd length
        {"name": "attention_prompt", "op": "attention", "seqs": 1, "new": 4095, "rest": 1, "context": 4095, "heads": 32,
         "kv_heads": 4, "head_dim": 128, "window": 0, "layers": 1},
        # a part of a long prompt beside other requests' tokens, wide heads
        {"name": "attention_mixed", "op": "attention", "seqs": 7, "new": 389, "rest": 1, "context": 9000, "heads": 16,
         "kv_heads": 2, "head_dim": 512, "window": 0, "layers": 1},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "rope", "plan", "append", "append", "attention", "attention", "attention", "attention",
                     "attention"])
    d = rng.choice([64, 96, 128, 128, 192, 256, 512])
    kv = rng.choice([1, 2, 4, 8])
    if op == "rope":
        heads = kv * rng.choice([1, 2, 3, 7, 8])
        tokens = max(1, min(_log(rng, 1, 8192), 25_000_000 // ((heads + kv) * d)))
        return {"op": op, "tokens": tokens, "heads": heads, "kv_heads": kv, "head_dim": d,
                "n_rot": rng.choice([d, d, d // 2, d // 4]), "base": rng.choice([1e4, 5e5, 1e6]),
                "style": rng.choice(["neox", "pairs"]), "fused": rng.random() < 0.5, "far": _log(rng, 10000, 1000000),
                "layers": 8 if tokens < 64 else 1}
    if op == "plan":
        seqs = _log(rng, 1, 2000)
        new, rest, context = _log(rng, 1, 600), rng.randint(1, 9), _log(rng, 700, 30000)
        return {"op": op, "seqs": seqs, "new": new, "rest": rest, "context": context,
                "room": min(65536, seqs * max(new, rest) + rng.randint(0, 40)), "table": -(-context // BLOCK) + 24}
    if op == "append":
        seqs = _log(rng, 1, 64)
        if rng.random() < 0.5:
            new, rest, opened = rng.randint(1, 4), rng.randint(1, 3), True
        else:
            new, rest, opened = _log(rng, 33, 4096), rng.randint(1, 60), False
        most = max(1, 8_000_000 // (kv * d))
        new, rest = min(new, most), min(rest, max(1, most // seqs))
        return {"op": op, "seqs": seqs, "new": new, "rest": rest, "open": opened, "kv_heads": kv, "head_dim": d,
                "layers": 4 if seqs * new < 100 else 1}
    group = rng.choice([1, 2, 4, 7, 8, 16])
    if kv * group > 32:
        group = 32 // kv
    heads, kind = kv * group, rng.choice(["token", "batch", "prompt", "chunk"])
    most = 60_000_000 // (kv * d)  # tokens of all caches
    if kind == "token":
        seqs, new, context = 1, rng.randint(1, 4), min(_log(rng, 64, 131072), most)
    elif kind == "batch":
        seqs = rng.randint(2, 64)
        new, context = rng.randint(1, 3), min(_log(rng, 64, 8192), most // seqs)
    else:
        seqs = 1 if kind == "prompt" else rng.randint(1, 6)
        context = min(_log(rng, 64, 4096), most // seqs)
        new = context if kind == "prompt" else min(context, _log(rng, 16, 512))
        while seqs * new * context * heads * d > 30_000_000_000:
            new, context = new // 2 + 1, max(new // 2 + 1, context * 3 // 4)
    rest = new if kind in ("token", "batch") else 1
    return {"op": op, "seqs": seqs, "new": new, "rest": rest, "context": max(context, new), "heads": heads,
            "kv_heads": kv, "head_dim": d, "window": rng.choice([0, 0, 0, 100, 1024]),
            "layers": 4 if kind == "token" and context < 10000 else 1}


# ------------------------------------------------------------------- the inputs
def _gen(seed, what):
    g = torch.Generator(device="cuda")
    g.manual_seed((int(seed) * 1_000_003 + what) & 0x7FFFFFFF)
    return g


def _normal(g, *shape, large=0.0):
    """Normal values; a share `large` of the last axis' channels four times larger."""
    x = torch.randn(*shape, generator=g, device="cuda")
    if large:
        x *= 1 + 3 * (torch.rand(shape[-1], generator=g, device="cuda") < large)
    return x


def _share(i):
    """A number in [0, 1) for each sequence, spread evenly, the first one's 0."""
    return np.modf(np.asarray(i) * 0.6180339887498949)[0]


def _lengths(case):
    """(tokens before the step, new tokens) of each sequence, int64 numpy."""
    i = np.arange(case["seqs"])
    if case["op"] == "append":
        new = np.where(i == 0, case["new"], 1 + (i * 7) % case["rest"])
        if case["open"]:  # inside a block that earlier tokens began
            return 320 + np.floor(_share(i + 1) * (BLOCK + 1 - new)).astype(np.int64), new
        return BLOCK * (i % 5), new
    if case["op"] == "plan":
        new = np.where(i % 7 == 3, 0, np.where(i % 97 == 0, case["new"], 1 + (i * 5) % case["rest"]))
        return np.floor(_share(i + 1) * (case["context"] - new)).astype(np.int64), new
    new = np.where(i == 0, case["new"], case["rest"])
    total = np.maximum(new, np.floor(case["context"] * (1 - 0.95 * _share(i))).astype(np.int64))
    return total - new, new


def _i32(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()


def _layout(case, seed, extra):
    """Where the sequences' blocks and the batch's tokens lie."""
    past, new = _lengths(case)
    total = past + new
    blocks = -(-total // BLOCK)
    width = int(blocks.max())
    pool = int(blocks.sum()) + extra
    order = np.random.RandomState((int(seed) * 31 + 7) & 0x7FFFFFFF).permutation(pool)
    table = np.full((case["seqs"], width), NONE, np.int64)
    first = np.concatenate([[0], np.cumsum(blocks)])
    for i in range(case["seqs"]):
        table[i, :blocks[i]] = order[first[i]:first[i + 1]]
    return {"past": past, "new": new, "total": total, "table": table, "pool": pool,
            "start": np.concatenate([[0], np.cumsum(new)])}


def _tokens(begin, end):
    """(sequence, position) of the positions begin[i] .. end[i] - 1 of every sequence i."""
    n = end - begin
    seq = np.repeat(np.arange(len(n)), n)
    return seq, np.arange(n.sum()) - np.repeat(np.cumsum(n) - n, n) + np.repeat(begin, n)


def _inputs(case, seed):
    op, g = case["op"], _gen(seed, 1)
    if op == "rope":
        t, h, kv, d, n = case["tokens"], case["heads"], case["kv_heads"], case["head_dim"], case["layers"]
        x = _normal(g, n, t, (h + (2 if case["fused"] else 1) * kv) * d)  # (fused: the values lie behind)
        w = [1 + 0.3 * torch.randn(n, d, generator=g, device="cuda") for _ in range(2)]
        pos = torch.randint(0, case["far"], (1,), generator=g, device="cuda", dtype=torch.int32)
        return {"x": x, "wq": w[0], "wk": w[1], "pos": pos + torch.arange(t, device="cuda", dtype=torch.int32)}
    if op == "plan":
        past, new = _lengths(case)
        need = int((-(-(past + new) // BLOCK)).sum())
        r = np.random.RandomState((int(seed) * 31 + 7) & 0x7FFFFFFF)
        order, held = r.permutation(need + 50), -(-past // BLOCK)
        table = np.full((case["seqs"], case["table"]), NONE, np.int64)
        table[np.arange(case["table"]) < held[:, None]] = order[:held.sum()]
        return {"past": _i32(past), "new": _i32(new), "table": _i32(table), "free": _i32(order[held.sum():]),
                "used": _i32([int(r.randint(0, 40))])}
    at = _layout(case, seed, 16)
    kv, d, n = case["kv_heads"], case["head_dim"], case["layers"]
    v = {"at": at, "table": _i32(at["table"]), "len": _i32(at["total"]), "start": _i32(at["start"])}
    # keys and values: of the blocks that the batch touches, or of all that the cache holds
    begin = at["past"] // BLOCK * BLOCK if op == "append" else np.zeros_like(at["past"])
    seq, pos = _tokens(begin, at["total"])
    v["seq"], v["pos"] = seq, pos
    v["slot"] = _i32(at["table"][seq, pos // BLOCK] * BLOCK + pos % BLOCK)
    v["k"], v["v"] = _normal(g, n, len(seq), kv, d, large=0.03), _normal(g, n, len(seq), kv, d)
    if op == "attention":
        v["q"] = 1.5 * _normal(g, n, int(at["new"].sum()), case["heads"], d)
    return v


class State:
    """What a program has in hand before the call."""

    def __init__(self, case, inputs):
        self.case, self.v = case, inputs
        self.handles = None  # the framework's side of it


def prepare(case, seed):
    s = State(case, _inputs(case, seed))
    if own:  # filled caches, the outputs' memory, a decode loop's graph
        s.handles = _Handles(case, s.v)
    elif case["op"] == "attention":  # the cache in a plain layout
        s.v.update(_plain_cache(case, s.v))
    if case["op"] == "attention":
        del s.v["k"], s.v["v"]
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
    """Caches, output buffers and the calls of one pass; gives the caches back."""

    def __init__(self, case, v):
        self.lt, self.ctx = _framework()
        self.owned, self.graph, self.caches = [], None, []
        {"rope": self.rope, "plan": self.plan, "append": self.append, "attention": self.attention}[case["op"]](case, v)
        # a decode loop replays its calls from a graph
        if case.get("layers", 1) > 1 or case["op"] == "attention" and int(v["at"]["new"].max()) < 4:
            torch.cuda.synchronize()
            self.once()  # sizes the context's scratch
            self.ctx.sync()
            from llmtoy_amd import hip
            self.graph = hip.Graph(self.ctx.stream, self.once)

    def rope(self, case, v):
        ctx, lt = self.ctx, self.lt
        t, h, kv, d, n = case["tokens"], case["heads"], case["kv_heads"], case["head_dim"], case["layers"]
        plan = self.keep(ctx.rope(d, n_rot=case["n_rot"], base=case["base"],
                                  style=lt.ROPE_NEOX if case["style"] == "neox" else lt.ROPE_PAIRS))
        x = v["x"]
        q, k = x[..., :h * d].unflatten(-1, (h, d)), x[..., h * d:(h + kv) * d].unflatten(-1, (kv, d))
        q_out, k_out = torch.zeros(n, t, h, d, device="cuda"), torch.zeros(n, t, kv, d, device="cuda")
        self.out = {"q": q_out, "k": k_out}
        io = [(q_out[i], k_out[i], q[i], k[i], v["wq"][i], v["wk"][i]) for i in range(n)]

        def once():
            for a in io:
                ctx.qk_norm_rope(*a, v["pos"], plan, eps=1e-6)
        self.once = once

    def plan(self, case, v):
        ctx, n, t = self.ctx, case["seqs"], case["room"]
        new = lambda *s: torch.zeros(*s, device="cuda", dtype=torch.int32)  # noqa: E731
        table = v["table"].clone()
        batch = self.lt.KvBatch(new(n + 1), new(n), table, t)
        pos, slot, used = new(t), new(t), new(1)
        self.out = {"table": table, "len": batch.len, "start": batch.start, "pos": pos, "slot": slot, "used": used}

        def once():
            ctx.kv_plan(batch, v["past"], v["new"], v["free"], v["used"], used, pos, slot)
        self.once = once

    def filled(self, case, v, seq, pos, upto, k, w):
        """A cache for each layer holding the tokens (seq, pos) of which there are upto[i] in sequence i."""
        at, lt = v["at"], self.lt
        table = v["table"]
        n_new = np.bincount(seq, minlength=case["seqs"])
        batch = lt.KvBatch(_i32(np.concatenate([[0], np.cumsum(n_new)])), _i32(upto), table, max(1, len(seq)))
        torch.cuda.synchronize()
        for i in range(case["layers"]):
            c = self.keep(self.ctx.kv_cache(at["pool"], case["kv_heads"], case["head_dim"], case["seqs"]))
            if len(seq):
                c.append(k[i], w[i], batch)
            self.caches.append(c)
        self.ctx.sync()

    def append(self, case, v):
        at, n = v["at"], case["layers"]
        old = v["pos"] < at["past"][v["seq"]]
        io = {}
        for name in ("k", "v"):
            io["old" + name] = v[name][:, torch.from_numpy(old).cuda()].contiguous()
            io[name] = v[name][:, torch.from_numpy(~old).cuda()].contiguous()
        self.filled(case, v, v["seq"][old], v["pos"][old], at["past"], io["oldk"], io["oldv"])
        batch = self.lt.KvBatch(v["start"], v["len"], v["table"], int(at["new"].sum()), max_new=int(at["new"].max()))
        self.out = {"k": torch.zeros_like(v["k"]), "v": torch.zeros_like(v["v"])}

        def once():
            for i in range(n):
                self.caches[i].append(io["k"][i], io["v"][i], batch)
                self.caches[i].read(self.out["k"][i], self.out["v"][i], v["slot"])
        self.once = once

    def attention(self, case, v):
        at, ctx, n = v["at"], self.ctx, case["layers"]
        self.filled(case, v, v["seq"], v["pos"], at["total"], v["k"], v["v"])
        batch = self.lt.KvBatch(v["start"], v["len"], v["table"], int(at["new"].sum()), max_new=int(at["new"].max()))
        out = torch.zeros_like(v["q"])
        self.out = out
        q, scale = v["q"], 1 / math.sqrt(case["head_dim"])

        def once():
            for i in range(n):
                ctx.attention(out[i], q[i], self.caches[i], batch, scale=scale, window=case["window"])
        self.once = once

    def keep(self, t):
        self.owned.append(t)
        return t

    def __del__(self):
        torch.cuda.synchronize()
        if self.graph is not None:
            self.graph.destroy()
        for t in self.owned:
            t.free()


# ------------------------------------------------------------------- the plain form
def _rms(x, w):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w[:, None, None]


def _rotate(case, x, cos, sin):
    """x [n, t, h, d]; cos, sin [t, 1, n_rot / 2]."""
    n = case["n_rot"]
    r = x[..., :n]
    if case["style"] == "neox":
        a, b = r[..., :n // 2], r[..., n // 2:]
        r = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    else:
        a, b = r[..., 0::2], r[..., 1::2]
        r = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    return torch.cat([r, x[..., n:]], -1)


def _plain_rope(case, v):
    h, kv, d, n = case["heads"], case["kv_heads"], case["head_dim"], case["n_rot"]
    x = v["x"]
    i = torch.arange(n // 2, device=x.device, dtype=torch.float64)
    angle = v["pos"].double()[:, None, None] * case["base"] ** (-2 * i / n)  # (far positions: 64 bits)
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    q, k = x[..., :h * d].unflatten(-1, (h, d)), x[..., h * d:(h + kv) * d].unflatten(-1, (kv, d))
    return {"q": _rotate(case, _rms(q, v["wq"]), cos, sin), "k": _rotate(case, _rms(k, v["wk"]), cos, sin)}


def _plain_plan(case, v):
    past, new, table, free = v["past"].long(), v["new"].long(), v["table"], v["free"]
    total = past + new
    first, last = (past + BLOCK - 1) // BLOCK, (total + BLOCK - 1) // BLOCK
    ends = v["used"] + torch.cumsum(last - first, 0)
    col = torch.arange(case["table"], device=past.device)
    fresh = (col >= first[:, None]) & (col < last[:, None])
    served = (ends <= len(free)) & (last <= case["table"])
    pick = (ends - (last - first))[:, None] + col - first[:, None]
    table = torch.where(fresh, torch.where(served[:, None], free[pick.clamp(0, len(free) - 1)], NONE), table)
    start = torch.cat([torch.zeros_like(ends[:1]), torch.cumsum(new, 0)])
    t = torch.arange(case["room"], device=past.device)
    seq = torch.searchsorted(start, t, right=True) - 1
    inside = seq < case["seqs"]
    seq = seq.clamp(max=case["seqs"] - 1)
    pos = torch.where(inside, past[seq] + t - start[seq], 0)
    block = table[seq, (pos // BLOCK).clamp(max=case["table"] - 1)]
    slot = torch.where(inside & (block != NONE), block * BLOCK + pos % BLOCK, NONE)
    used = torch.where(served, ends, v["used"]).amax(0, keepdim=True)
    return {"table": table, "len": total.int(), "start": start.int(), "pos": pos.int(), "slot": slot.int(),
            "used": used.int()}


def _codes(x):
    """Codes (as whole numbers in 32 bits) and scales of x [..., 32, d], scale [..., 1, 1]."""
    s = (x.abs().amax((-2, -1), keepdim=True).double() / 127).float()
    c = torch.round(x.double() / torch.where(s > 0, s, 1).double()).clamp(-127, 127)  # (next to a tie: 64 bits)
    return c.float(), s


def _in_blocks(case, v, x):
    """x [n, tokens, kv, d] in the blocks that hold them, [n, blocks, kv, 32, d], zeros where no token is; and the
    place of each token there."""
    key = v["seq"] * (1 << 32) + v["pos"] // BLOCK
    which = torch.from_numpy(np.unique(key, return_inverse=True)[1] * BLOCK + v["pos"] % BLOCK).to(x.device)
    room = torch.zeros(x.shape[0], (int(which.max()) // BLOCK + 1) * BLOCK, *x.shape[2:], device=x.device)
    room[:, which] = x
    return room.unflatten(1, (-1, BLOCK)).transpose(2, 3), which


def _plain_append(case, v):
    out = {}
    for name in ("k", "v"):
        x, which = _in_blocks(case, v, v[name])
        c, s = _codes(x)
        out[name] = (c * s).transpose(2, 3).flatten(1, 2)[:, which]
    return out


def _plain_cache(case, v):
    at, got = v["at"], {}
    first = torch.from_numpy(np.flatnonzero(v["pos"] % BLOCK == 0))
    block = torch.from_numpy(at["table"][v["seq"], v["pos"] // BLOCK]).to(v["k"].device)[first]
    for name in ("k", "v"):
        c, s = _codes(_in_blocks(case, v, v[name])[0])
        codes = torch.zeros(case["layers"], at["pool"], *c.shape[2:], dtype=torch.int8, device=c.device)
        scales = torch.zeros(case["layers"], at["pool"], *s.shape[2:], device=c.device)
        codes[:, block], scales[:, block] = c.to(torch.int8), s
        got[name + "c"], got[name + "s"] = codes, scales
    return got


def _plain_attention(case, v):
    at, q = v["at"], v["q"]
    n, b, kv, d = case["layers"], case["seqs"], case["kv_heads"], case["head_dim"]
    group, most = case["heads"] // kv, int(at["new"].max())
    table = v["table"].long().clamp(min=0)

    def values(name):  # [n, b, kv, length, d]
        x = v[name + "c"][:, table].float() * v[name + "s"][:, table]
        return x.transpose(2, 3).flatten(3, 4)

    start, total = v["start"].long(), v["len"].long()
    j = torch.arange(most, device=q.device)
    new = start[1:] - start[:-1]
    inside = j < new[:, None]
    rows = (start[:-1, None] + j).clamp(max=q.shape[1] - 1)
    x = q[:, rows].unflatten(3, (kv, group)).permute(0, 1, 3, 2, 4, 5).flatten(3, 4)  # [n, b, kv, most * group, d]
    s = (x @ values("k").transpose(-1, -2)).mul_(1 / math.sqrt(d))
    pos = (total - new)[:, None] + j
    key = torch.arange(s.shape[-1], device=q.device)
    seen = (key <= pos[..., None]) & (inside[..., None] | (key == 0))
    if case["window"]:
        seen &= (key > pos[..., None] - case["window"]) | ~inside[..., None]
    seen = seen.repeat_interleave(group, 1)[:, None]
    s.masked_fill_(~seen, -math.inf)
    s = s.sub_(s.amax(-1, keepdim=True)).exp_()
    o = (s @ values("v")).div_(s.sum(-1, keepdim=True))
    o = o.unflatten(3, (most, group)).permute(0, 1, 3, 2, 4, 5).flatten(3, 4)  # [n, b, most, heads, d]
    return o.flatten(1, 2)[:, inside.flatten()]


def _plain(case, v):
    return {"rope": _plain_rope, "plan": _plain_plan, "append": _plain_append,
            "attention": _plain_attention}[case["op"]](case, v)


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
def _visible(case):
    """(pairs of a query position and a key that it sees, keys that a sequence's queries see), over the sequences."""
    past, new = _lengths(case)
    window = case["window"] or 1 << 40
    pairs = keys = 0
    for p, m in zip(past.tolist(), new.tolist()):
        pos = np.arange(p, p + m)
        pairs += int(np.minimum(pos + 1, window).sum())
        keys += p + m - max(0, p - window + 1)
    return pairs, keys


def work(case):
    op = case["op"]
    if op == "rope":
        n = case["layers"] * case["tokens"] * (case["heads"] + case["kv_heads"]) * case["head_dim"]
        return {"bytes": 8 * n + 4 * case["tokens"], "flops": 8 * n}
    if op == "plan":
        past, new = _lengths(case)
        blocks = int((-(-(past + new) // BLOCK) + past // -BLOCK).sum())
        return {"bytes": 4 * (4 * case["seqs"] + 2 * blocks + 2 * case["room"]), "flops": 8 * (case["seqs"] + case["room"])}
    kv, d, n = case["kv_heads"], case["head_dim"], case["layers"]
    past, new = _lengths(case)
    if op == "append":
        touched = int((past + new - past // BLOCK * BLOCK).sum())
        # read: the blocks' tokens; written: codes, scales and the values they stand for
        return {"bytes": n * 2 * kv * (touched * d * 9 + touched // BLOCK * 4), "flops": n * 2 * kv * touched * d * 5}
    pairs, keys = _visible(case)
    return {"bytes": n * (2 * kv * keys * d + keys // BLOCK * kv * 8 + 8 * int(new.sum()) * case["heads"] * d),
            "flops": n * 4 * pairs * case["heads"] * d}


# ------------------------------------------------------------------- the same in 64 bits
def _exact_rope(case, v):
    h, kv, d, n = case["heads"], case["kv_heads"], case["head_dim"], case["n_rot"]
    x = v["x"].double().unflatten(-1, (-1, d))
    turn = torch.tensor([case["base"] ** (-2 * i / n) for i in range(n // 2)], dtype=torch.float64, device=x.device)
    z = torch.polar(torch.ones_like(turn), v["pos"].double()[:, None] * turn)[None, :, None]  # e^(i angle)

    def one(x, w):
        x = x / (x.pow(2).sum(-1, keepdim=True) / d + 1e-6).sqrt() * w.double()[:, None, None]
        r = x[..., :n]
        pairs = r.unflatten(-1, (2, n // 2)).transpose(-1, -2) if case["style"] == "neox" else r.unflatten(-1, (n // 2, 2))
        y = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * z)
        y = y.transpose(-1, -2) if case["style"] == "neox" else y
        return torch.cat([y.flatten(-2), x[..., n:]], -1)
    return {"q": one(x[..., :h, :], v["wq"]), "k": one(x[..., h:h + kv, :], v["wk"])}


def _exact_values(x):
    """What the 8-bit blocks of x [tokens, kv, d] (whole blocks from the first token on) stand for."""
    got = []
    for part in x.split(BLOCK):
        s = (part.abs().amax((0, 2)).double() / 127).float().double()[None, :, None]  # (the scale is held in 32 bits)
        u = part.double() / torch.where(s == 0, 1, s)
        low = torch.floor(u)
        up = (u - low > 0.5) | ((u - low == 0.5) & (low % 2 != 0))
        got.append((low + up) * s)
    return torch.cat(got)


def _exact_cache(case, v, layer):
    """[(keys, values)] of each sequence in 64 bits."""
    got = []
    for i in range(case["seqs"]):
        at = torch.from_numpy(np.flatnonzero(v["seq"] == i)).to(v["k"].device)
        got.append((_exact_values(v["k"][layer, at]), _exact_values(v["v"][layer, at])))
    return got


def _exact_attention(case, v):
    past, new = _lengths(case)
    group, window = case["heads"] // case["kv_heads"], case["window"] or 1 << 40
    out = torch.zeros_like(v["q"], dtype=torch.float64)
    for layer in range(case["layers"]):
        at = 0
        for i, (k, w) in enumerate(_exact_cache(case, v, layer)):
            m = int(new[i])
            low = max(0, int(past[i]) - window + 1)
            key = torch.arange(low, int(past[i]) + m, device=k.device)
            for h in range(case["heads"]):
                for a in range(0, m, 1024):
                    pos = torch.arange(int(past[i]) + a, int(past[i]) + min(m, a + 1024), device=k.device)[:, None]
                    rows = slice(at + a, at + min(m, a + 1024))
                    s = v["q"][layer, rows, h].double() @ k[low:, h // group].T / math.sqrt(case["head_dim"])
                    s = torch.where((key <= pos) & (pos - key < window), s, -math.inf)
                    out[layer, rows, h] = torch.softmax(s, -1) @ w[low:, h // group]
            at += m
    return out


def exact(case, seed):
    v = _inputs(case, seed)
    if case["op"] == "rope":
        return _exact_rope(case, v)
    if case["op"] == "append":
        caches = [_exact_cache(case, v, layer) for layer in range(case["layers"])]
        return {"k": torch.stack([torch.cat([k for k, _ in c]) for c in caches]),
                "v": torch.stack([torch.cat([w for _, w in c]) for c in caches])}
    if case["op"] == "attention":
        return _exact_attention(case, v)
    return None
