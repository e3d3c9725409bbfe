"""The operators of a full attention layer and of a step's answer, as timed cases: plain torch,
and the library's kernels.

  linear  y = act(x w^T + bias) [* (x up^T + up_bias)] + residual over Q8_0 matrices, repacked or as
          the model file has them (aotx_q8_linear)
  norm    RMSNorm of fp32 rows into the fp16 rows that a product takes (aotx_norm_rows)
  append  head norm and rotary turn of a product's q, k and v rows; q into rows, k and v into the
          paged cache (aotx_kv_append)
  adjust  penalties for repeated tokens, biases and grammar masks on logits (aotx_logits_adjust)

Matrix sizes are those of the 8B shape (4096 wide, 32 / 8 heads of 128, FFN 14336, vocabulary 128256)
and ragged ones drawn around them, up to 64 slots and prompts of 8192 rows. Inputs come from the
seed alone: weights N(0, 1/k), so that sums are about 1, activations and rows N(0, 1), logits
N(0, 2), token lists that repeat themselves as texts do.
"""
import math
import struct
import zlib

import torch

own = False

EPS = 1e-6
SLOTS, PAGES_EACH, PAGE_BYTES, PAGE_HEADER, BLOCK = 64, 640, 2 << 20, 256, 16
SPLIT, ADJACENT = 0, 1
ACTS = ["none", "silu", "gelu", "gelu_tanh", "relu"]
MOST = 2048 * 4096 * 2 * 14336      # products of the largest case


def listed():
    return [
        # one agent's token through the attention's output matrix into the residual stream
        _linear("linear_o_1", 1, 4096, 4096, resid=True),
        # eight agents' q, k and v with their bias, over weights left as the model file has them
        _linear("linear_qkv_file_8", 8, 6144, 4096, bias=True, packed=False),
        # 32 agents through the gated feed-forward unit
        _linear("linear_gate_32", 32, 14336, 4096, gated=True, act="silu", half=True),
        # a ragged piece of a prompt through a small projection with odd sizes, rows of a wider buffer
        _linear("linear_ragged_147", 147, 1001, 2080, act="gelu", bias=True, half=True, pad=24),
        # four prompt chunks of 512 at once through the gated unit
        _linear("linear_gate_2048", 2048, 14336, 4096, gated=True, act="silu", half=True),
        # decode rows of 64 agents before a product
        {"name": "norm_64", "kind": "norm", "tokens": 64, "width": 4096},
        # the rows of a long document
        {"name": "norm_8192", "kind": "norm", "tokens": 8192, "width": 4096},
        # one agent's next token: launch and latency
        _append("append_1", 1, 1, 1, at=1000, layers=32),
        # the next token of 64 agents, with head norms
        _append("append_64", 64, 1, 1, at=2000, layers=32, norm=True, pairs=SPLIT),
        # a long document, positions stretched by factors
        _append("append_8192", 1, 8192, 8192, at=0, layers=2, factor=True),
        # one agent's answer under a grammar that allows few tokens
        _adjust("adjust_1", 1, 128256, 2000, allow=0.01),
        # a whole step of 64 agents: penalties over long texts, biases, grammars for some
        _adjust("adjust_64", 64, 128256, 8000, allow=0.5, biases=64),
    ]


def _linear(name, m, n, k, gated=False, act="none", bias=False, resid=False, half=False, packed=True, pad=0):
    return {"name": name, "kind": "linear", "m": m, "n": n, "k": k, "gated": gated, "act": act, "bias": bias,
            "resid": resid, "half": half, "packed": packed, "pad": pad}


def _append(name, seqs, lo, hi, at, layers, heads=32, kv_heads=8, dim=128, rope_dim=None, pairs=ADJACENT, axes=1,
            norm=False, factor=False, gain=1.0, theta=5e5):
    return {"name": name, "kind": "append", "seqs": seqs, "lo": lo, "hi": hi, "at": at, "layers": layers,
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "rope_dim": rope_dim or dim, "pairs": pairs,
            "axes": axes, "norm": norm, "factor": factor, "gain": gain, "theta": theta}


def _adjust(name, rows, vocab, length, allow=1.0, biases=0, penalties=True, window=256):
    return {"name": name, "kind": "adjust", "rows": rows, "vocab": vocab, "length": length, "allow": allow,
            "biases": biases, "penalties": penalties, "window": window}


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choices(["linear", "norm", "append", "adjust"], [5, 1, 3, 3])[0]
    if kind == "linear":
        n, k, gated = _log(rng, 60, 16384), 32 * _log(rng, 8, 448), rng.random() < 0.4
        case = _linear(None, _log(rng, 1, min(2048, MOST // (n * k * (1 + gated)))), n, k, gated,
                       rng.choice(ACTS), rng.random() < 0.5, rng.random() < 0.4, rng.random() < 0.5, rng.random() < 0.6,
                       rng.choice([0, 0, 8, 136]))
    elif kind == "norm":
        width = 8 * _log(rng, 8, 2048)
        case = {"kind": kind, "tokens": _log(rng, 1, 8192 * 4096 // max(4096, width)), "width": width}
    elif kind == "append":
        kv, dim, seqs = rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 128]), _log(rng, 1, 64)
        lo, hi = sorted(_log(rng, 1, 8192 // seqs) for _ in range(2))
        case = _append(None, seqs, lo, hi, _log(rng, 1, 8192 - hi) if hi < 8192 else 0, rng.choice([1, 2, 4]),
                       kv * rng.choice([1, 2, 4]), kv, dim, rng.choice([dim // 4, dim // 2, dim, dim]),
                       rng.choice([SPLIT, ADJACENT]), rng.choice([1, 1, 3]), rng.random() < 0.5, rng.random() < 0.4,
                       rng.choice([1.0, 1.0, 1.2]), rng.choice([1e4, 5e5, 1e6]))
    else:
        case = _adjust(None, _log(rng, 1, 64), _log(rng, 2000, 152064), _log(rng, 1, 8192),
                       rng.choice([1.0, 0.5, 0.02]), rng.choice([0, 0, 1, 40, 300]), rng.random() < 0.8,
                       rng.choice([0, 64, 1024]))
    case.pop("name", None)
    return case


# ---- inputs -------------------------------------------------------------------------------

def _gen(*seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(zlib.crc32(repr(seed).encode()))
    return g


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _q8(g, n, k, packed):
    """A Q8_0 matrix of N(0, 1/k): rows of k / 32 blocks (fp16 scale, 32 quants), or repacked: 16 rows by 128
    columns at a time, [n/16][k/128][halves of a block's quants][block of four][row][16] bytes of quant + 128,
    then [n/16][k/128][block of four][row] scales; what fills up the last ones is zero."""
    w = torch.randn(n, k // 32, 32, generator=g, device="cuda") * k ** -0.5
    d = w.abs().amax(-1) / 127
    q = torch.round(w / d[..., None]).to(torch.int8)
    d = d.half()
    del w
    if not packed:
        return torch.cat([d.view(torch.uint8).view(n, k // 32, 2), q.view(torch.uint8)], -1).flatten()
    t, quads = -(-n // 16), -(-k // 128)
    full = torch.zeros(t * 16, quads * 4, 32, dtype=torch.int8, device="cuda")
    full[:n, :k // 32] = q
    scale = torch.zeros(t * 16, quads * 4, dtype=torch.float16, device="cuda")
    scale[:n, :k // 32] = d
    q = (full.view(torch.uint8) ^ 128).view(t, 16, quads, 4, 2, 16).permute(0, 2, 4, 3, 1, 5)
    return torch.cat([q.flatten(), scale.view(t, 16, quads, 4).permute(0, 2, 3, 1).contiguous().view(torch.uint8).flatten()])


def _lengths(case):
    """Row counts of the case's sequences, the same for every seed: `hi` first, then spread."""
    lo, hi, n = case["lo"], case["hi"], case["seqs"]
    return [hi - (hi - lo) * ((7 * i) % n) // max(1, n - 1) if n > 1 else hi for i in range(n)]


def _block_bytes(case):
    return 2 * case["kv_heads"] * BLOCK * case["dim"] * 2


def _prepare_append(s, case, g):
    lens = _lengths(case)
    seqs, h, kv, d = case["seqs"], case["heads"], case["kv_heads"], case["dim"]
    s["tokens"] = tokens = sum(lens)
    s["width"] = (h + 2 * kv) * d
    s["qkv"] = torch.randn(tokens, s["width"], generator=g, device="cuda")
    s["offset"] = _ints([sum(lens[:i]) for i in range(seqs + 1)])
    slots = torch.randperm(SLOTS, generator=g, device="cuda")[:seqs].tolist()
    first = [case["at"] - min(case["at"], 3 * i) for i in range(seqs)]
    s["agent"], s["pos"] = _ints(slots), _ints(first)
    s["layer"] = case["layers"] // 2
    # the pages that the call's rows stand in, in mixed order as a pool hands them out
    per = (PAGE_BYTES - PAGE_HEADER) // _block_bytes(case)
    need = [(slot, i) for slot, p, n in zip(slots, first, lens)
            for i in range((p // BLOCK * case["layers"] + s["layer"]) // per,
                           ((p + n - 1) // BLOCK * case["layers"] + s["layer"]) // per + 1)]
    s["pool"] = torch.randn(len(need), PAGE_BYTES // 2, generator=g, device="cuda").half()
    order = torch.randperm(len(need), generator=g, device="cuda")
    at = torch.tensor(need, device="cuda")
    s["page"] = torch.zeros(SLOTS, PAGES_EACH, dtype=torch.int64, device="cuda")
    s["page"][at[:, 0], at[:, 1]] = s["pool"].data_ptr() + order * PAGE_BYTES
    half = case["rope_dim"] // 2
    for name in ("q_norm", "k_norm"):
        s[name] = 1 + 0.1 * torch.randn(d, generator=g, device="cuda") if case["norm"] else None
    s["factor"] = 1 + 7 * torch.rand(half, generator=g, device="cuda") if case["factor"] else None
    s["span"] = [half - 2 * (half // 3), half // 3, half // 3] if case["axes"] == 3 else [half]
    s["place"] = None
    if case["axes"] == 3:            # a text with images: time, height and width
        run = torch.arange(tokens, device="cuda") + case["at"]
        s["place"] = torch.stack([run, run - run % 48 + run // 8 % 48, run // 2], 1).int().contiguous()
    s["q"] = torch.zeros(tokens, h * d, dtype=torch.float16, device="cuda")
    s["row_pos"], s["row_agent"] = (torch.zeros(tokens, dtype=torch.int32, device="cuda") for _ in range(2))


def _prepare_adjust(s, case, g):
    rows, vocab, length = case["rows"], case["vocab"], case["length"]
    s["logits"] = 2 * torch.randn(rows, vocab, generator=g, device="cuda")
    s["out"] = torch.zeros_like(s["logits"])
    slots = torch.randperm(SLOTS, generator=g, device="cuda")[:rows]
    s["agent"] = slots.int()
    # texts: most tokens come from few words
    u = torch.rand(SLOTS, length, generator=g, device="cuda")
    s["list"] = (vocab * u ** 6).int().clamp_(0, vocab - 1)
    s["length"] = (length * (0.5 + 0.5 * torch.rand(SLOTS, generator=g, device="cuda"))).int()
    sample = [struct.pack("<fIfffIff48x", 0.8, 40, 0.9, 0.0, 1.05 + 0.05 * (i % 5), case["window"],
                          0.1 * ((i + 1) % 4), 0.02 * ((i + 1) % 7)) for i in range(rows)]
    s["sample"] = torch.frombuffer(bytearray(b"".join(sample)), dtype=torch.int32).view(rows, 20).cuda() if case["penalties"] else None
    n = min(case["biases"], vocab)
    s["bias_at"] = _ints([n * i for i in range(rows + 1)]) if n else None
    pick = torch.rand(rows, vocab, generator=g, device="cuda").topk(n, 1).indices if n else None
    s["bias_token"] = pick.int().contiguous() if n else None
    s["bias"] = 5 * torch.randn(rows, n, generator=g, device="cuda") if n else None
    s["words"] = words = (vocab + 31) // 32
    s["masks"] = masks = 8 if case["allow"] < 1 else 0
    s["mask"] = s["mask_of"] = None
    if masks:
        bits = torch.rand(masks, words, 32, generator=g, device="cuda") < case["allow"]
        word = (bits.long() << torch.arange(32, device="cuda")).sum(-1)
        s["mask"] = torch.where(word >= 1 << 31, word - (1 << 32), word).int()
        # rows share the masks of grammar states; some rows have no grammar
        s["mask_of"] = _ints([(3 * i) % (masks + 2) for i in range(rows)])


def prepare(case, seed):
    g = _gen(sorted(case.items(), key=str), seed)
    s = {"case": case}
    if case["kind"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        s["w"] = _q8(g, n, k, case["packed"])
        s["up"] = _q8(g, n, k, case["packed"]) if case["gated"] else None
        s["x"] = torch.randn(m, k + case["pad"], generator=g, device="cuda").half()
        s["bias"] = torch.randn(n, generator=g, device="cuda") if case["bias"] else None
        s["up_bias"] = torch.randn(n, generator=g, device="cuda") if case["bias"] and case["gated"] else None
        s["resid"] = 3 * torch.randn(m, n, generator=g, device="cuda") if case["resid"] else None
        s["y"] = torch.zeros(m, n, dtype=torch.float16 if case["half"] else torch.float32, device="cuda")
    elif case["kind"] == "norm":
        t, w = case["tokens"], case["width"]
        s["x"] = torch.randn(t, w, generator=g, device="cuda") * (0.1 + 10 * torch.rand(t, 1, generator=g, device="cuda"))
        s["w"] = 1 + 0.1 * torch.randn(w, generator=g, device="cuda")
        s["out"] = torch.zeros(t, w, dtype=torch.float16, device="cuda")
    elif case["kind"] == "append":
        _prepare_append(s, case, g)
    else:
        _prepare_adjust(s, case, g)
    s["at"] = {k: v.data_ptr() for k, v in s.items() if isinstance(v, torch.Tensor)}
    return s


# ---- plain forms --------------------------------------------------------------------------

def _weights(data, n, k, packed):
    """half(quant * scale) of a matrix as fp32 [n][k]."""
    if not packed:
        b = data.view(n, k // 32, 34)
        d, q = b[..., :2].contiguous().view(torch.float16), b[..., 2:].contiguous().view(torch.int8)
        return (q.float() * d.float()).half().float().view(n, k)
    t, quads = -(-n // 16), -(-k // 128)
    split = t * quads * 2048
    q = (data[:split] ^ 128).view(torch.int8).view(t, quads, 2, 4, 16, 16).permute(0, 4, 1, 3, 2, 5)
    d = data[split:].view(torch.float16).view(t, quads, 4, 16).permute(0, 3, 1, 2)
    w = (q.float() * d.float()[..., None, None]).half().float()
    return w.reshape(t * 16, quads * 128)[:n, :k]


def _act(x, act):
    if act == "silu":
        return x / (1 + torch.exp(-x))
    if act == "gelu":
        return 0.5 * x * (1 + torch.erf(x * 0.5 ** 0.5))
    if act == "gelu_tanh":
        return 0.5 * x * (1 + torch.tanh((2 / math.pi) ** 0.5 * (x + 0.044715 * x * x * x)))
    return torch.clamp(x, min=0) if act == "relu" else x


def _plain_linear(s):
    c = s["case"]
    x = s["x"][:, :c["k"]].float()
    y = x @ _weights(s["w"], c["n"], c["k"], c["packed"]).T
    y = _act(y + s["bias"] if c["bias"] else y, c["act"])
    if c["gated"]:
        up = x @ _weights(s["up"], c["n"], c["k"], c["packed"]).T
        y = y * (up + s["up_bias"] if c["bias"] else up)
    s["y"].copy_(y + s["resid"] if c["resid"] else y)
    return s["y"]


def _plain_norm(s):
    x = s["x"]
    s["out"].copy_(x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * s["w"])
    return s["out"]


def _rows(s):
    """Slot and cache position of every row."""
    lens = (s["offset"][1:] - s["offset"][:-1]).long()
    seq = torch.repeat_interleave(torch.arange(len(lens), device="cuda"), lens, output_size=s["tokens"])
    at = s["pos"].long()[seq] + torch.arange(s["tokens"], device="cuda") - s["offset"].long()[seq]
    return s["agent"].long()[seq], at


def _axes(s):
    return torch.repeat_interleave(torch.arange(len(s["span"]), device="cuda"), torch.tensor(s["span"], device="cuda"),
                                   output_size=sum(s["span"]))


def _places(s, pos):
    """Index of position `pos` of K head 0 in the pool's halves, for every row."""
    c = s["case"]
    slot, at = pos
    per = (PAGE_BYTES - PAGE_HEADER) // _block_bytes(c)
    block = at // BLOCK * c["layers"] + s["layer"]
    byte = s["page"][slot, block // per] - s["pool"].data_ptr() + PAGE_HEADER + block % per * _block_bytes(c)
    return byte // 2 + at % BLOCK * c["dim"]


def _plain_append(s):
    c = s["case"]
    h, kv, d, r = c["heads"], c["kv_heads"], c["dim"], c["rope_dim"]
    slot, at = _rows(s)
    i = torch.arange(r // 2, dtype=torch.float64, device="cuda")
    place = at[:, None] if s["place"] is None else s["place"].long()
    angle = place[:, _axes(s)].double() * torch.exp(-2 * i / r * math.log(c["theta"]))
    if s["factor"] is not None:
        angle = angle / s["factor"].double()
    cos, sin = (c["gain"] * torch.cos(angle)).float()[:, None], (c["gain"] * torch.sin(angle)).float()[:, None]
    x = s["qkv"].view(-1, h + 2 * kv, d)

    def turn(x, norm):
        if norm is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * norm
        a, b = (x[..., :r // 2], x[..., r // 2:r]) if c["pairs"] == SPLIT else (x[..., 0:r:2], x[..., 1:r:2])
        a, b = a * cos - b * sin, a * sin + b * cos
        turned = torch.cat([a, b], -1) if c["pairs"] == SPLIT else torch.stack([a, b], -1).flatten(-2)
        return torch.cat([turned, x[..., r:]], -1)

    s["q"].copy_(turn(x[:, :h], s["q_norm"]).reshape(s["q"].shape))
    k, v = turn(x[:, h:h + kv], s["k_norm"]), x[:, h + kv:]
    head = torch.arange(2 * kv, device="cuda") * BLOCK * d
    to = (_places(s, (slot, at))[:, None, None] + head[:, None] + torch.arange(d, device="cuda"))
    s["pool"].view(-1)[to] = torch.cat([k, v], 1).half()
    s["row_pos"].copy_(at)
    s["row_agent"].copy_(slot)
    return s["q"], s["pool"], s["row_pos"], s["row_agent"]


def _plain_adjust(s):
    c = s["case"]
    rows, vocab = c["rows"], c["vocab"]
    z = s["logits"]
    if s["sample"] is not None:
        f = s["sample"].view(torch.float32)
        repeat, presence, frequency, window = f[:, 4:5], f[:, 6:7], f[:, 7:8], s["sample"][:, 5:6]
        token, length = s["list"][s["agent"].long()].long(), s["length"][s["agent"].long()][:, None]
        place = torch.arange(c["length"], device="cuda")
        token = torch.where(place < length, token, vocab)
        count = torch.zeros(rows, vocab + 1, device="cuda").scatter_add_(1, token, torch.ones_like(token, dtype=torch.float32))[:, :vocab]
        recent = torch.zeros(rows, vocab + 1, dtype=torch.bool, device="cuda")
        recent = recent.scatter_(1, torch.where(place >= length - window, token, vocab), True)[:, :vocab]
        z = z - torch.where(count > 0, presence + frequency * count, 0)
        z = torch.where(recent, torch.where(z > 0, z / repeat, z * repeat), z)
    if s["bias"] is not None:
        z = z + torch.zeros_like(z).scatter_(1, s["bias_token"].long(), s["bias"])
    if s["mask"] is not None:
        bits = (s["mask"][..., None] >> torch.arange(32, dtype=torch.int32, device="cuda") & 1).bool().view(s["masks"], -1)[:, :vocab]
        of = s["mask_of"].long()
        allowed = bits[torch.clamp(of, max=s["masks"] - 1)] | (of >= s["masks"])[:, None]
        z = torch.where(allowed, z, float("-inf"))
    s["out"].copy_(z)
    return s["out"]


# ---- the library's kernels ------------------------------------------------------------------

def _own(s):
    import aotx_amd as A
    lib, c, at = A.lib(), s["case"], s["at"]
    get, stream = at.get, torch.cuda.current_stream().cuda_stream
    kind = c["kind"]
    if kind == "linear":
        if "how" not in s:                                               # kept for the passes after
            need = lib.aotx_q8_linear_work(c["n"], c["k"], c["m"], int(c["gated"]))
            s["work"] = torch.zeros(need, dtype=torch.uint8, device="cuda")
            s["how"] = A.LinearHow(w=at["w"], up=get("up"), bias=get("bias"), up_bias=get("up_bias"), resid=get("resid"),
                                   n=c["n"], k=c["k"], ldx=c["k"] + c["pad"], ldy=c["n"], ldr=c["n"],
                                   act=ACTS.index(c["act"]), out=int(c["half"]), packed=int(c["packed"]))
        rc = lib.aotx_q8_linear(s["how"], at["x"], c["m"], at["y"], s["work"].data_ptr(), s["work"].numel(), stream)
        got = s["y"]
    elif kind == "norm":
        rc = lib.aotx_norm_rows(at["x"], c["width"], at["w"], c["tokens"], c["width"], EPS, at["out"], stream)
        got = s["out"]
    elif kind == "append":
        if "how" not in s:
            s["how"] = A.RopeHow(theta=c["theta"], eps=EPS, rope_dim=c["rope_dim"], pairs=c["pairs"], axes=c["axes"],
                                 order=A.AOTX_ROPE_AXES_RUNS, span=(A.u32 * 4)(*s["span"]))
        rc = lib.aotx_kv_append(at["qkv"], s["width"], get("q_norm"), get("k_norm"), s["how"], get("factor"), c["gain"],
                                get("place"), at["offset"], at["pos"], at["agent"], c["seqs"], s["tokens"], c["heads"],
                                c["kv_heads"], c["dim"], s["layer"], c["layers"], at["page"], at["q"], at["row_pos"],
                                at["row_agent"], stream)
        got = s["q"], s["pool"], s["row_pos"], s["row_agent"]
    else:
        if "how" not in s:
            s["how"] = A.AdjustHow(sample=get("sample"), agent=at["agent"], list=at["list"], length=at["length"],
                                   lists=SLOTS, list_stride=c["length"], bias_at=get("bias_at"), bias_token=get("bias_token"),
                                   bias=get("bias"), biases=s["bias"].numel() if "bias" in at else 0, mask=get("mask"),
                                   mask_of=get("mask_of"), masks=s["masks"], mask_stride=s["words"])
        rc = lib.aotx_logits_adjust(s["how"], at["logits"], c["vocab"], c["rows"], c["vocab"], at["out"], c["vocab"], stream)
        got = s["out"]
    A.check(rc, kind)
    return got


def run(state):
    if own:
        return _own(state)
    return {"linear": _plain_linear, "norm": _plain_norm, "append": _plain_append,
            "adjust": _plain_adjust}[state["case"]["kind"]](state)


# ---- what a pass has to move, and its outputs in 64 bits ------------------------------------

def work(case):
    kind = case["kind"]
    if kind == "linear":
        m, n, k, mats = case["m"], case["n"], case["k"], 1 + case["gated"]
        return {"bytes": mats * n * k // 32 * 34 + 2 * m * k + m * n * (2 if case["half"] else 4)
                + (4 * m * n if case["resid"] else 0) + (4 * n * mats if case["bias"] else 0), "flops": 2 * m * n * k * mats}
    if kind == "norm":
        return {"bytes": 6 * case["tokens"] * case["width"] + 4 * case["width"], "flops": 4 * case["tokens"] * case["width"]}
    if kind == "append":
        t = sum(_lengths(case))
        n = t * (case["heads"] + 2 * case["kv_heads"]) * case["dim"]
        return {"bytes": 6 * n + 8 * t + (12 * t if case["axes"] == 3 else 0), "flops": 6 * n}
    rows, vocab = case["rows"], case["vocab"]
    return {"bytes": rows * (8 * vocab + (3 * case["length"] if case["penalties"] else 0) + 8 * case["biases"])
            + (min(rows, 8) * vocab // 8 if case["allow"] < 1 else 0), "flops": 4 * rows * vocab}


def _exact_linear(s):
    c = s["case"]
    n, k = c["n"], c["k"]

    def matrix(data):
        """Block by block, from the layout's description."""
        if not c["packed"]:
            raw = data.view(n, k // 32, 34)
            scale = raw[:, :, 0:2].clone().view(torch.float16)[..., 0]
            quant = raw[:, :, 2:].clone().view(torch.int8)
        else:
            quads, tiles = (k + 127) // 128, (n + 15) // 16
            row, block = torch.arange(n, device="cuda")[:, None], torch.arange(k // 32, device="cuda")
            unit = (row // 16 * quads + block // 4) * 64 + 16 * (block % 4) + row % 16
            scale = data[tiles * quads * 2048:].clone().view(torch.float16)[unit]
            first = unit // 64 * 2048 + unit % 64 * 16
            byte = torch.arange(32, device="cuda")
            quant = data[first[..., None] + byte // 16 * 1024 + byte % 16].double() - 128
        return (quant.double() * scale.double()[..., None]).to(torch.float16).double().reshape(n, k)

    x = s["x"][:, :k].double()
    y = torch.nn.functional.linear(x, matrix(s["w"]), s["bias"].double() if c["bias"] else None)
    if c["act"] == "silu":
        y = y * torch.sigmoid(y)
    elif c["act"] == "gelu":
        y = y * torch.special.ndtr(y)
    elif c["act"] == "gelu_tanh":
        y = y * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3))
    elif c["act"] == "relu":
        y = torch.maximum(y, torch.zeros_like(y))
    if c["gated"]:
        y = y * torch.nn.functional.linear(x, matrix(s["up"]), s["up_bias"].double() if c["bias"] else None)
    return y + s["resid"].double() if c["resid"] else y


def _exact_append(s):
    c = s["case"]
    h, kv, d, r = c["heads"], c["kv_heads"], c["dim"], c["rope_dim"]
    slots, firsts, begins = s["agent"].tolist(), s["pos"].tolist(), s["offset"].tolist()
    at = torch.cat([torch.arange(p, p + e - b) for p, b, e in zip(firsts, begins, begins[1:])]).cuda()
    slot = torch.cat([torch.full((e - b,), a) for a, b, e in zip(slots, begins, begins[1:])]).cuda()
    freq = torch.tensor([c["theta"] ** (-2.0 * i / r) for i in range(r // 2)], dtype=torch.float64, device="cuda")
    if s["factor"] is not None:
        freq = freq / s["factor"].double()
    turn = at.double()[:, None] * freq
    if s["place"] is not None:
        axis = torch.tensor([j for j, n in enumerate(s["span"]) for _ in range(n)], device="cuda")
        turn = s["place"].double()[:, axis] * freq
    turn = torch.polar(torch.full_like(turn, c["gain"]), turn)[:, None]
    x = s["qkv"].double().view(-1, h + 2 * kv, d)

    def one(y, norm):
        if norm is not None:
            y = y / (y.square().mean(-1, keepdim=True) + EPS).sqrt() * norm.double()
        y = y.clone()
        low, high = (y[..., :r // 2], y[..., r // 2:r]) if c["pairs"] == SPLIT else (y[..., 0:r:2], y[..., 1:r:2])
        z = torch.complex(low.contiguous(), high.contiguous()) * turn
        low.copy_(z.real)
        high.copy_(z.imag)
        return y

    new = torch.cat([one(x[:, h:h + kv], s["k_norm"]), x[:, h + kv:]], 1)
    pool = s["pool"].double()
    base, per = s["pool"].data_ptr(), (PAGE_BYTES - PAGE_HEADER) // _block_bytes(c)
    block = torch.div(at, BLOCK, rounding_mode="floor") * c["layers"] + s["layer"]
    page = torch.div(s["page"][slot, torch.div(block, per, rounding_mode="floor")] - base, PAGE_BYTES, rounding_mode="floor")
    for j in range(2 * kv):
        first = (PAGE_HEADER + block % per * _block_bytes(c)) // 2 + (j * BLOCK + at % BLOCK) * d
        pool[page[:, None], first[:, None] + torch.arange(d, device="cuda")] = new[:, j]
    return one(x[:, :h], s["q_norm"]).reshape(len(at), -1), pool, None, None


def _exact_adjust(s):
    c = s["case"]
    vocab, got = c["vocab"], []
    for r in range(c["rows"]):
        z = s["logits"][r].double()
        if s["sample"] is not None:
            how = s["sample"][r]
            repeat, presence, frequency = (how.view(torch.float32)[i].double() for i in (4, 6, 7))
            a = int(s["agent"][r])
            text = s["list"][a, :int(s["length"][a])].long()
            count = torch.bincount(text, minlength=vocab).double()
            z = torch.where(count > 0, z - presence - frequency * count, z)
            late = text[max(0, len(text) - int(how[5])):].unique()
            z[late] = torch.where(z[late] > 0, z[late] / repeat, z[late] * repeat)
        if s["bias"] is not None:
            z[s["bias_token"][r].long()] += s["bias"][r].double()
        if s["mask"] is not None and int(s["mask_of"][r]) < s["masks"]:
            t = torch.arange(vocab, device="cuda")
            z[(s["mask"][int(s["mask_of"][r])][t // 32] >> (t % 32).int()) & 1 == 0] = -math.inf
        got.append(z)
    return torch.stack(got)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "linear":
        return _exact_linear(s)
    if case["kind"] == "norm":
        x = s["x"].double()
        return x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * s["w"].double()
    return _exact_append(s) if case["kind"] == "append" else _exact_adjust(s)
