"""The paged-cache operators as measured work: queries and keys normalised per head and
rotated into the cache, a cache held in 8 or 4 bits (written, read back, attended by
decode steps and prompt chunks), and attention for a tree of drafted tokens.

Each case is a dict of plain values. prepare() makes what a serving program holds before
the call (pools of pages, block tables, lengths, the fused projection's output), run()
makes one pass: with `own` the framework's calls, without it the same operator in
elementary torch operations."""
import math
import os
import sys

import torch

own = False

BASE = 1e6
EPS = 1e-6
DT = {"bf16": torch.bfloat16, "f16": torch.float16}


def _framework():
    """The package (its directory's name has dashes, so it is registered by hand)."""
    name = "mlx_server_runtime_b200"
    if name not in sys.modules:
        import importlib.util
        at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                          "mlx-server-runtime_b200")
        spec = importlib.util.spec_from_file_location(
            name, os.path.join(at, "__init__.py"), submodule_search_locations=[at])
        mod = importlib.util.module_from_spec(spec)
        sys.modules[name] = mod
        spec.loader.exec_module(mod)
    import importlib
    return importlib.import_module(name + ".attention")


# --------------------------------------------------------------------------------------
# cases

def _heads(hq, hkv, hd):
    return {"hq": hq, "hkv": hkv, "hd": hd}


QWEN = _heads(28, 4, 128)     # the decoder configuration of this repository
SMALL = _heads(8, 2, 64)      # its small test configuration
WIDE = _heads(16, 2, 128)     # eight query heads to a key head


def listed():
    return [
        # a decode step of eight sequences: eight new tokens are normalised, rotated, appended
        {"name": "append step", "op": "append", "dtype": "bf16", **QWEN, "page": 16,
         "tokens": 8},
        # the prompts of a batch, some rows of it padding without a slot
        {"name": "append prompts", "op": "append", "dtype": "bf16", **QWEN, "page": 16,
         "tokens": 8190},
        # a small model's decode step into a 4-bit cache, the new rows read back
        {"name": "write 4 bits step", "op": "write", "dtype": "f16", **SMALL, "page": 8,
         "tokens": 5, "bits": 4, "gs": 32},
        # a prompt batch into an 8-bit cache, read back (a prefix handed to another worker)
        {"name": "write 8 bits prompts", "op": "write", "dtype": "bf16", **QWEN, "page": 16,
         "tokens": 8190, "bits": 8, "gs": 64},
        # one user's chat turn: a single sequence, latency counts
        {"name": "decode one", "op": "decode", "dtype": "bf16", **QWEN, "page": 16, "bits": 4,
         "gs": 64, "batch": 1, "kv": 641},
        # an ordinary batch of decode steps, 8-bit cache, one group to a row
        {"name": "decode batch", "op": "decode", "dtype": "f16", **WIDE, "page": 32, "bits": 8,
         "gs": 128, "batch": 16, "kv": 4097},
        # a full server: many long sequences, what the 4-bit cache is for
        {"name": "decode long", "op": "decode", "dtype": "bf16", **QWEN, "page": 16, "bits": 4,
         "gs": 64, "batch": 32, "kv": 16384},
        # eight drafted tokens checked for one user over a 16-bit cache
        {"name": "tree one", "op": "tree", "dtype": "bf16", **QWEN, "page": 16, "bits": 16,
         "gs": 0, "batch": 1, "nodes": 8, "kv": 600},
        # a batch's drafted trees over a 4-bit cache
        {"name": "tree 4 bits", "op": "tree", "dtype": "bf16", **QWEN, "page": 16, "bits": 4,
         "gs": 64, "batch": 8, "nodes": 31, "kv": 4100},
        # the largest trees over long 16-bit sequences
        {"name": "tree long", "op": "tree", "dtype": "bf16", **QWEN, "page": 16, "bits": 16,
         "gs": 0, "batch": 16, "nodes": 64, "kv": 8192},
        # prompt chunks of a small model over an 8-bit cache
        {"name": "chunk small", "op": "chunk", "dtype": "f16", **SMALL, "page": 16, "bits": 8,
         "gs": 32, "batch": 4, "tokens": 100, "kv": 333},
        # two long prompts' next chunks over a 4-bit cache
        {"name": "chunk long", "op": "chunk", "dtype": "bf16", **QWEN, "page": 16, "bits": 4,
         "gs": 64, "batch": 2, "tokens": 2048, "kv": 8200},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["append", "write", "decode", "tree", "chunk"])
    hkv = rng.choice([1, 2, 4, 8])
    hd = rng.choice([64, 128, 128])
    c = {"op": op, "dtype": rng.choice(["bf16", "f16"]),
         **_heads(hkv * rng.randint(1, 32 // hkv if hkv > 4 else 8), hkv, hd),
         "page": rng.choice([8, 16, 16, 32])}
    if op != "append":
        c["bits"] = rng.choice([4, 8])
        c["gs"] = rng.choice([32, 64] if hd == 64 else [32, 64, 128])
    if op == "append":
        c["tokens"] = _log(rng, 1, 8192 * 36 // max(36, c["hq"] + 2 * hkv))
    elif op == "write":
        # whole prompts in 8 bits, decode steps in either
        c["tokens"] = _log(rng, 1, 8192 * 36 // max(36, c["hq"] + 2 * hkv)
                           if c["bits"] == 8 else 64)
    elif op == "decode":
        c["batch"] = _log(rng, 1, 64)
        c["kv"] = _log(rng, 1, min(32768, 32 * 16384 * 16 // (c["batch"] * hkv * c["bits"])))
    elif op == "tree":
        if rng.random() < 0.5:
            c["bits"], c["gs"] = 16, 0
        c["batch"] = _log(rng, 1, 16)
        c["nodes"] = _log(rng, 1, 64)
        c["kv"] = c["nodes"] + _log(rng, 1, min(16384, 16 * 8192 * 4 // (c["batch"] * max(4, hkv)))
                                    - c["nodes"])
    else:
        c["batch"] = _log(rng, 1, 4)
        c["tokens"] = _log(rng, 1, 2048)
        c["kv"] = c["tokens"] + _log(rng, 1, min(16384, 18_000_000 // (c["batch"] * c["tokens"]))
                                     - min(c["tokens"], 1024))
    return c


def _lens(case):
    """Cached keys of each sequence after the step, ragged down to a quarter of the longest."""
    B, kv = case["batch"], case["kv"]
    low = {"tree": case.get("nodes", 1), "chunk": case.get("tokens", 1)}.get(case["op"], 1)
    return [max(min(low, kv), kv - (3 * kv * b) // (4 * B)) for b in range(B)]


def _news(case):
    """New tokens of each sequence: one, its tree's nodes, or its chunk."""
    if case["op"] == "decode":
        return [1] * case["batch"]
    n = case["nodes"] if case["op"] == "tree" else case["tokens"]
    return [max(1, n - b) if case["op"] == "tree" else max(1, n - (n * b) // (2 * case["batch"]))
            for b in range(case["batch"])]


def _row_bytes(case):
    bits, hd = case.get("bits", 16), case["hd"]
    return hd * 2 if bits == 16 else hd * bits // 8 + hd // case["gs"] * 4


def work(case):
    hq, hkv, hd = case["hq"], case["hkv"], case["hd"]
    if case["op"] in ("append", "write"):
        T = case["tokens"]
        b = T * ((hq + 2 * hkv) * hd * 2 + 8 + hq * hd * 2)       # projections, q
        b += T * 2 * hkv * _row_bytes(case)                       # rows written
        if case["op"] == "write":
            b += T * 2 * hkv * (_row_bytes(case) + hd * 2)        # and read back
        return {"bytes": b, "flops": T * (hq + hkv) * hd * 7}
    lens, news = _lens(case), _news(case)
    b = sum(lens) * 2 * hkv * _row_bytes(case) + 2 * sum(news) * hq * hd * 2
    if case["op"] == "tree":
        b += 8 * sum(news)
        pairs = sum(n * (L - n) + n * (1 + int(math.log2(n))) for n, L in zip(news, lens))
    else:
        pairs = sum(n * (L - n) + n * (n + 1) // 2 for n, L in zip(news, lens))
    return {"bytes": b, "flops": 4 * hd * hq * pairs}


# --------------------------------------------------------------------------------------
# inputs

def _quantize(x, gs, bits):
    """Affine group quantisation of the rows of x (values of a 16-bit type): codes packed
    from the low bits of int32 words up, scales and biases in x's type. The rule is the
    framework's quantize: 32-bit arithmetic, the end of larger magnitude kept exactly."""
    v = x.float().unflatten(-1, (-1, gs))
    hi, lo = v.amax(-1, keepdim=True), v.amin(-1, keepdim=True)
    n = float(2 ** bits - 1)
    neg = lo.abs() > hi.abs()
    s = ((hi - lo) / n).clamp_min(1e-7)
    s = torch.where(neg, s, -s)
    edge = torch.where(neg, lo, hi)
    q0 = torch.round(edge / s)
    s = torch.where(q0 != 0, edge / q0, s)
    b = torch.where(q0 != 0, edge, torch.zeros_like(edge))
    q = torch.round((v - b) / s).clamp_(0, n).to(torch.int32).flatten(-2)
    per = 32 // bits
    shift = torch.arange(per, device=x.device, dtype=torch.int32) * bits
    words = (q.unflatten(-1, (-1, per)) << shift).sum(-1, dtype=torch.int32)
    return words, s.squeeze(-1).to(x.dtype), b.squeeze(-1).to(x.dtype)


def _values(words, s, b, gs, bits):
    """What the cache stands for: s * q + b, rounded once to its type."""
    per = 32 // bits
    shift = torch.arange(per, device=words.device, dtype=torch.int32) * bits
    q = ((words.unsqueeze(-1) >> shift) & (2 ** bits - 1)).flatten(-2)
    # a code times a 16-bit scale is exact in 32 bits; the sum is taken in 64 before its one rounding
    v = q.unflatten(-1, (-1, gs)).float() * s.float().unsqueeze(-1)
    v = (v.double() + b.double().unsqueeze(-1)).float()
    return v.flatten(-2).to(s.dtype)


class _Pool:
    """One pool of pages, 16-bit or in codes, with the framework's view of it for `own`."""

    def __init__(self, x, gs, bits):
        self.gs, self.bits = gs, bits
        if bits == 16:
            self.x = x
        else:
            self.words, self.s, self.b = _quantize(x, gs, bits)
        self.cache = None
        if own:
            if bits == 16:
                self.cache = self.x
            else:
                self.cache = _framework().QuantizedKV(self.words.view(torch.uint32), self.s,
                                                      self.b, gs, bits)

    def rows(self, at):
        """The values of the pool's rows `at` (page * page_size + offset)."""
        if self.bits == 16:
            return self.x.flatten(0, 1)[at]
        return _values(self.words.flatten(0, 1)[at], self.s.flatten(0, 1)[at],
                       self.b.flatten(0, 1)[at], self.gs, self.bits)

    def put(self, at, x):
        if self.bits == 16:
            self.x.flatten(0, 1)[at] = x
        else:
            w, s, b = _quantize(x, self.gs, self.bits)
            self.words.flatten(0, 1)[at] = w
            self.s.flatten(0, 1)[at] = s
            self.b.flatten(0, 1)[at] = b


def _tree(rng, n):
    """Ancestor masks of a random tree: each node continues an earlier one, or starts anew."""
    masks = []
    for i in range(n):
        p = rng.randint(max(-1, i - 8), i - 1)
        masks.append((masks[p] if p >= 0 else 0) | (1 << i))
    return [m - (1 << 64) if m >> 63 else m for m in masks]


def prepare(case, seed):
    import random
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    dt = DT[case["dtype"]]
    hq, hkv, hd, page = case["hq"], case["hkv"], case["hd"], case["page"]
    bits, gs = case.get("bits", 16), case.get("gs", 0)
    st = {"op": case["op"], "hq": hq, "hkv": hkv, "hd": hd, "page": page}

    def normal(*shape):
        return torch.randn(*shape, device=dev, generator=g)

    # keys vary from channel to channel, values less
    kc = torch.exp(0.4 * normal(hkv, hd))
    if case["op"] in ("append", "write"):
        T = case["tokens"]
        pages = -(-T // page) + 2
        st["qkv"] = (normal(T, (hq + 2 * hkv) * hd) * 1.5).to(dt)
        st["q_norm"] = (1 + 0.2 * normal(hd)).to(dt)
        st["k_norm"] = (1 + 0.2 * normal(hd)).to(dt)
        st["positions"] = torch.randint(0, 131072, (T,), device=dev, generator=g,
                                        dtype=torch.int32)
        slots = torch.randperm(pages * page, device=dev, generator=g)[:T].to(torch.int32)
        if T > 16:
            slots[-3:] = -1     # the batch's padding has no place in the cache
        st["slots"] = slots
        st["k"] = _Pool(torch.zeros(pages, page, hkv, hd, device=dev, dtype=dt), gs, bits)
        st["v"] = _Pool(torch.zeros(pages, page, hkv, hd, device=dev, dtype=dt), gs, bits)
        return st
    lens, news = _lens(case), _news(case)
    news = [min(n, L) for n, L in zip(news, lens)]
    blocks = [-(-L // page) for L in lens]
    pages = sum(blocks) + 3
    perm = torch.randperm(pages, device=dev, generator=g).to(torch.int32)
    table = torch.zeros(len(lens), max(blocks), dtype=torch.int32, device=dev)
    at = 0
    for b, nb in enumerate(blocks):
        table[b, :nb] = perm[at:at + nb]
        at += nb
    st["k"] = _Pool((normal(pages, page, hkv, hd) * kc).to(dt), gs, bits)
    st["v"] = _Pool(normal(pages, page, hkv, hd).to(dt), gs, bits)
    st["table"] = table
    st["lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
    st["max_kv"] = max(lens)
    cu = [0]
    for n in news:
        cu.append(cu[-1] + n)
    st["cu"] = torch.tensor(cu, dtype=torch.int32, device=dev)
    st["max_q"] = max(news)
    st["q"] = normal(cu[-1], hq, hd).to(dt)
    st["scale"] = hd ** -0.5
    if case["op"] == "tree":
        rng = random.Random(seed)
        st["mask"] = torch.tensor([m for n in news for m in _tree(rng, n)], dtype=torch.int64,
                                  device=dev)
    return st


# --------------------------------------------------------------------------------------
# one pass

def _rotated(x, w, positions, hd, dt):
    """Per-head norm and rotation of x [T, heads, hd], rounded to the end's type. Angles in
    64 bits: positions are far."""
    i = torch.arange(hd // 2, device=x.device, dtype=torch.float64)
    angle = positions.double()[:, None] * torch.pow(BASE, -2.0 * i / hd)
    cos, sin = torch.cos(angle).to(x.dtype)[:, None], torch.sin(angle).to(x.dtype)[:, None]
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.to(x.dtype)
    a, b = y[..., :hd // 2], y[..., hd // 2:]
    return torch.cat([a * cos - b * sin, a * sin + b * cos], -1).to(dt)


def _append(st):
    hq, hkv, hd = st["hq"], st["hkv"], st["hd"]
    qkv = st["qkv"]
    # a key next to a border between two codes is decided in 64 bits
    wide = qkv.float() if st["k"].bits == 16 else qkv.double()
    wide = wide.unflatten(-1, (-1, hd))
    q = _rotated(wide[:, :hq], st["q_norm"], st["positions"], hd, qkv.dtype)
    k = _rotated(wide[:, hq:hq + hkv], st["k_norm"], st["positions"], hd, qkv.dtype)
    v = qkv.unflatten(-1, (-1, hd))[:, hq + hkv:]
    live = st["slots"] >= 0
    at = st["slots"].long()[live]
    st["k"].put(at, k[live])
    st["v"].put(at, v[live])
    return q


def _read(pool, slots):
    return torch.where((slots >= 0)[:, None, None], pool.rows(slots.long().clamp_min(0)), 0)


def _attend(st):
    """Attention of every sequence's new tokens over its pages, padded to the longest."""
    hkv, hd, page = st["hkv"], st["hd"], st["page"]
    dev = st["q"].device
    L, n = st["max_kv"], st["max_q"]
    pos = torch.arange(L, device=dev)
    rows = st["table"].long()[:, pos // page] * page + pos % page            # [B, L]
    k, v = st["k"].rows(rows).float(), st["v"].rows(rows).float()            # [B, L, hkv, hd]
    cu, lens = st["cu"].long(), st["lens"].long()
    i = torch.arange(n, device=dev)
    new = cu[1:] - cu[:-1]
    at = (cu[:-1, None] + i).clamp_max(cu[-1] - 1)                           # [B, n]
    q = st["q"].float()[at].unflatten(2, (hkv, -1))                          # [B, n, hkv, G, hd]
    s = torch.einsum("bnhgd,blhd->bhgnl", q, k) * st["scale"]
    j = pos[None] - (lens - new)[:, None]                                    # key's place in the new ones
    if "mask" in st:
        bit = (st["mask"][at][:, :, None] >> j[:, None].clamp(0, 63)) & 1
        seen = (j[:, None] < 0) | ((j[:, None] < 64) & (bit == 1))
    else:
        seen = j[:, None] <= i[None, :, None]
    seen = seen & (pos[None, None] < lens[:, None, None])                    # [B, n, L]
    s = s.masked_fill_(~seen[:, None, None], float("-inf"))
    m = s.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)
    p = torch.exp_(s.sub_(m))
    o = torch.einsum("bhgnl,blhd->bnhgd", p, v)
    den = p.sum(-1).permute(0, 3, 1, 2)[..., None]
    o = torch.where(den > 0, o / den, 0.0).flatten(2, 3)                     # [B, n, hq, hd]
    return o[i[None] < new[:, None]].to(st["q"].dtype)


def run(st):
    op = st["op"]
    if own:
        A = _framework()
        k, v = st["k"].cache, st["v"].cache
        if op in ("append", "write"):
            q = A.rope_kv_append(st["qkv"], st["positions"], st["slots"], k, v, st["hq"],
                                 st["hkv"], st["hd"], BASE, q_norm=st["q_norm"],
                                 k_norm=st["k_norm"], eps=EPS)
            if op == "append":
                return {"q": q, "k": k, "v": v}
            rk, rv = A.kv_cache_read(k, v, st["slots"])
            return {"q": q, "k": rk, "v": rv}
        if op == "decode":
            return A.paged_attention_decode(st["q"], k, v, st["table"], st["lens"], st["max_kv"],
                                            st["scale"])
        if op == "tree":
            return A.paged_attention_tree(st["q"], st["cu"], st["max_q"], k, v, st["table"],
                                          st["lens"], st["max_kv"], st["mask"], st["scale"])
        return A.paged_attention_prefill(st["q"], st["cu"], st["max_q"], k, v, st["table"],
                                         st["lens"], st["scale"])
    if op == "append":
        q = _append(st)
        return {"q": q, "k": st["k"].x, "v": st["v"].x}
    if op == "write":
        q = _append(st)
        return {"q": q, "k": _read(st["k"], st["slots"]), "v": _read(st["v"], st["slots"])}
    return _attend(st)


# --------------------------------------------------------------------------------------
# the operators' definitions in 64 bits

def _exact_heads(x, w, positions):
    """Norm and rotation as a product of complex numbers."""
    x = x.double()
    hd = x.shape[-1]
    y = x / torch.sqrt(x.square().sum(-1, keepdim=True) / hd + EPS) * w.double()
    z = torch.complex(y[..., :hd // 2].contiguous(), y[..., hd // 2:].contiguous())
    e = torch.arange(0, hd, 2, device=x.device, dtype=torch.float64) / hd
    turn = positions.double()[:, None] * torch.exp(-e * math.log(BASE))
    z = z * torch.polar(torch.ones_like(turn), turn)[:, None]
    return torch.cat([z.real, z.imag], -1)


def _exact_stored(x, gs, bits):
    """The value each element of the rows x (in the cache's type) is stored as. The codes
    follow the quantisation rule in its own 32-bit arithmetic; the value is s * q + b."""
    T, h, hd = x.shape
    v = x.float().reshape(T, h, hd // gs, gs)
    top, bottom = v.max(3).values, v.min(3).values
    levels = 2 ** bits - 1
    step = torch.maximum((top - bottom) / levels, torch.full_like(top, 1e-7))
    below = bottom.abs() > top.abs()
    step = step * torch.where(below, 1.0, -1.0)
    end = torch.where(below, bottom, top)
    k = torch.round(end / step)
    zero = k == 0
    step = torch.where(zero, step, end / torch.where(zero, torch.ones_like(k), k))
    off = end * (~zero)
    code = torch.round((v - off[..., None]) / step[..., None]).clamp(0, levels).double()
    s, b = step.to(x.dtype).double(), off.to(x.dtype).double()
    return (s[..., None] * code + b[..., None]).reshape(T, h, hd)


def exact(case, seed):
    global own
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    hq, hkv, hd = st["hq"], st["hkv"], st["hd"]
    if case["op"] in ("append", "write"):
        x = st["qkv"].reshape(case["tokens"], -1, hd)
        q = _exact_heads(x[:, :hq], st["q_norm"], st["positions"])
        k = _exact_heads(x[:, hq:hq + hkv], st["k_norm"], st["positions"])
        v = x[:, hq + hkv:]
        live = (st["slots"] >= 0).nonzero().flatten()
        if case["op"] == "append":
            kc, vc = st["k"].x.double(), st["v"].x.double()
            at = st["slots"][live].long()
            kc.reshape(-1, hkv, hd)[at] = k[live]
            vc.reshape(-1, hkv, hd)[at] = v[live].double()
            return {"q": q, "k": kc, "v": vc}
        outs = []
        for y in (k.to(x.dtype), v):
            o = torch.zeros(y.shape, dtype=torch.float64, device=y.device)
            o[live] = _exact_stored(y[live], case["gs"], case["bits"])
            outs.append(o)
        return {"q": q, "k": outs[0], "v": outs[1]}
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=st["q"].device)
    cu, page = st["cu"].tolist(), st["page"]
    for b, L in enumerate(st["lens"].tolist()):
        n = cu[b + 1] - cu[b]
        t = torch.arange(L, device=out.device)
        at = st["table"][b].long()[t.div(page, rounding_mode="floor")] * page + t.remainder(page)
        k, v = st["k"].rows(at).double(), st["v"].rows(at).double()
        first = L - n
        if case["op"] == "tree":
            m = st["mask"][cu[b]:cu[b + 1]].tolist()
            tail = torch.tensor([[m[i] >> j & 1 for j in range(n)] for i in range(n)],
                                dtype=torch.bool, device=out.device)
        else:
            tail = torch.ones(n, n, dtype=torch.bool, device=out.device).tril()
        hidden = torch.cat([torch.zeros(n, first, dtype=torch.bool, device=out.device), ~tail], 1)
        for h in range(hq):
            q = st["q"][cu[b]:cu[b + 1], h].double()
            s = (q @ k[:, h // (hq // hkv)].T) * st["scale"]
            p = torch.softmax(s.masked_fill(hidden, -math.inf), -1)
            out[cu[b]:cu[b + 1], h] = p @ v[:, h // (hq // hkv)]
    return out
