"""The operators of hybrid models' layers, as timed cases: plain torch, and the library's kernels.

A hybrid model has linear layers, which keep a matrix per head instead of a cache, beside full
attention layers whose rows carry several positions (time, height, width):

  linear layer  product -> conv -> step or chunk -> norm -> product
  full layer    product -> rope -> page write -> paged attention -> product

  conv    short causal convolution with SiLU over a product's fp32 rows, into fp16 rows
          (aotx_delta_conv)
  step    gated delta rule, one token of each slot: the state of every head is read, decayed,
          corrected and written (aotx_delta_step)
  chunk   the same rule over sequences of any length (aotx_delta_chunk)
  norm    RMSNorm of every head's output times its SiLU gate (aotx_norm_gate)
  rope    head norm and rotary turn of q and k by the positions of one to four axes, fp32 rows of
          a product into fp16 rows (aotx_rope_axes)

Sizes are generic: 16 key heads and 32 value heads of 128 (8192 channels of q, k and v), the 32 / 8
heads of 128 that the attention kernels run, up to 64 slots, prompt chunks of 512 and long prompts.
Inputs come from the seed alone. Activations behind the convolution are silu(N(0, 1)), so keys lean
the same way; decay rates and time steps are those that such layers start from (rates of 1 to 16,
steps of 0.001 to 0.1); states are N(0, 0.1).
"""
import math
import zlib

import torch

own = False

CHUNK = 64            # rows that the plain form of `chunk` takes at once
EPS = 1e-6
SPLIT, ADJACENT = 0, 1


def listed():
    return [
        # one agent's next token: launches and latency
        {"name": "step_1", "kind": "step", "slots": 1, "key_heads": 16, "heads": 32, "dim": 128},
        # all 64 slots of the runtime decode one token each
        {"name": "step_64", "kind": "step", "slots": 64, "key_heads": 16, "heads": 32, "dim": 128},
        # the last piece of a chat prompt, shorter than a chunk's rows
        {"name": "chunk_40", "kind": "chunk", "seqs": 1, "lo": 40, "hi": 40, "fresh": False,
         "key_heads": 16, "heads": 32, "dim": 128},
        # one prompt chunk of the runtime's largest pass, after cached tokens
        {"name": "chunk_512", "kind": "chunk", "seqs": 1, "lo": 512, "hi": 512, "fresh": False,
         "key_heads": 16, "heads": 32, "dim": 128},
        # a long document from its beginning
        {"name": "chunk_8192", "kind": "chunk", "seqs": 1, "lo": 8192, "hi": 8192, "fresh": True,
         "key_heads": 16, "heads": 32, "dim": 128},
        # prompts of different agents and lengths in one pass, small heads
        {"name": "chunk_ragged_24", "kind": "chunk", "seqs": 24, "lo": 1, "hi": 700, "fresh": False,
         "key_heads": 8, "heads": 8, "dim": 64},
        # the next token of 64 agents through the convolution
        {"name": "conv_step_64", "kind": "conv", "seqs": 64, "lo": 1, "hi": 1, "fresh": False,
         "channels": 8192, "width": 4, "bias": False},
        # a long document through the convolution
        {"name": "conv_8192", "kind": "conv", "seqs": 1, "lo": 8192, "hi": 8192, "fresh": True,
         "channels": 8192, "width": 4, "bias": False},
        # decode rows of 64 agents
        {"name": "norm_64", "kind": "norm", "tokens": 64, "heads": 32, "dim": 128},
        # the rows of a long document
        {"name": "norm_8192", "kind": "norm", "tokens": 8192, "heads": 32, "dim": 128},
        # decode rows of 64 agents: head norms, half of each head turned, its pairs dealt to three axes in turn
        {"name": "rope_64", "kind": "rope", "tokens": 64, "heads": 32, "kv_heads": 8, "dim": 128,
         "rope_dim": 64, "axes": 3, "order": 1, "pairs": SPLIT, "norm": True, "factor": False, "theta": 1e7},
        # the rows of a document with images
        {"name": "rope_8192", "kind": "rope", "tokens": 8192, "heads": 32, "kv_heads": 8, "dim": 128,
         "rope_dim": 128, "axes": 3, "order": 0, "pairs": SPLIT, "norm": True, "factor": False, "theta": 1e6},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choices(["step", "chunk", "conv", "norm", "rope"], [3, 5, 2, 2, 3])[0]
    key_heads = rng.choice([1, 2, 4, 8, 16])
    heads, dim = key_heads * rng.choice([1, 1, 2, 3]), rng.choice([64, 128, 128])
    heads = min(heads, key_heads * max(1, 32 // key_heads))
    if kind == "step":
        return {"kind": kind, "slots": _log(rng, 1, 64), "key_heads": key_heads, "heads": heads, "dim": dim}
    if kind == "chunk":
        seqs = _log(rng, 1, 32)
        lo, hi = sorted(_log(rng, 1, 8192 // seqs) for _ in range(2))
        return {"kind": kind, "seqs": seqs, "lo": lo, "hi": hi, "fresh": rng.random() < 0.5,
                "key_heads": key_heads, "heads": heads, "dim": dim}
    if kind == "conv":
        seqs = _log(rng, 1, 64)
        lo, hi = sorted(_log(rng, 1, 7900 // seqs) for _ in range(2))
        return {"kind": kind, "seqs": seqs, "lo": lo, "hi": hi, "fresh": rng.random() < 0.5,
                "channels": 4 * _log(rng, 8, 2048), "width": rng.choice([2, 3, 4]), "bias": rng.random() < 0.5}
    if kind == "norm":
        dim = rng.choice([64, 128, 256, 8 * _log(rng, 2, 1024)])
        heads = rng.choice([1, 2, 8, 32]) if dim <= 256 else 1
        return {"kind": kind, "tokens": _log(rng, 1, 8192 * 4096 // max(4096, heads * dim)), "heads": heads, "dim": dim}
    kv = rng.choice([1, 2, 4, 8])
    return {"kind": kind, "tokens": _log(rng, 1, 8192), "heads": kv * rng.choice([1, 2, 4]), "kv_heads": kv,
            "dim": dim, "rope_dim": rng.choice([dim // 4, dim // 2, dim]), "axes": rng.randint(1, 4),
            "order": rng.choice([0, 1]), "pairs": rng.choice([SPLIT, ADJACENT]), "norm": rng.random() < 0.5,
            "factor": rng.random() < 0.3, "theta": rng.choice([1e4, 5e5, 1e6, 1e7])}


# ---- inputs -------------------------------------------------------------------------------

def _gen(*seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(zlib.crc32(repr(seed).encode()))
    return g


def _lengths(case):
    """Row counts of the case's sequences, the same for every seed: `hi` first, then spread."""
    lo, hi, n = case["lo"], case["hi"], case["seqs"]
    return [hi - (hi - lo) * ((7 * i) % n) // max(1, n - 1) if n > 1 else hi for i in range(n)]


def _spans(case):
    """Pairs per axis: as even as they come, the first axis has the rest."""
    pairs, axes = case["rope_dim"] // 2, case["axes"]
    spans = [pairs // axes] * axes
    spans[0] += pairs - sum(spans)
    return spans


def _axis_of(case):
    """The axis of every pair: runs of pairs one axis after another (order 0), or turn by turn."""
    spans, axes = _spans(case), case["axes"]
    if case["order"] == 0:
        return [j for j in range(axes) for _ in range(spans[j])]
    return [i % axes if i < axes * spans[i % axes] else 0 for i in range(sum(spans))]


def prepare(case, seed):
    g = _gen(sorted(case.items(), key=str), seed)
    kind = case["kind"]
    s = {"case": case}

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device="cuda") * scale

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    if kind in ("step", "chunk", "conv"):
        lens = [1] * case["slots"] if kind == "step" else _lengths(case)
        n = len(lens)
        s["lens"] = lens
        s["tokens"] = tokens = sum(lens)
        s["offset"] = ints([sum(lens[:i]) for i in range(n + 1)])
        s["held"] = held = min(64, n + 2)                                # slots that keep a state
        s["slots"] = torch.randperm(held, generator=g, device="cuda")[:n].tolist()
        s["agent"] = ints(s["slots"])
        s["first"] = [0 if kind != "step" and case["fresh"] else 100 + 3 * i for i in range(n)]
        s["pos"] = ints(s["first"])
    if kind in ("step", "chunk"):
        heads, keys, d = case["heads"], case["key_heads"], case["dim"]
        s["width"] = width = (2 * keys + heads) * d
        x = normal(tokens, width)
        s["qkv"] = (x / (1 + torch.exp(-x))).half()
        s["a"], s["b"] = normal(tokens, heads), normal(tokens, heads)
        s["decay"] = -(1 + 15 * torch.rand(heads, generator=g, device="cuda"))
        steps = torch.exp(math.log(1e-3) + math.log(100.0) * torch.rand(heads, generator=g, device="cuda"))
        s["dt"] = steps + torch.log(-torch.expm1(-steps))
        s["state"] = normal(held, heads, d, d, scale=0.1)
        s["out"] = torch.zeros(tokens, heads * d, dtype=torch.float16, device="cuda")
    elif kind == "conv":
        c, w = case["channels"], case["width"]
        s["x"] = normal(tokens, c)
        s["w"] = normal(c, w, scale=w ** -0.5)
        s["bias"] = normal(c, scale=0.1) if case["bias"] else None
        s["state"] = normal(held, w - 1, c)
        s["out"] = torch.zeros(tokens, c, dtype=torch.float16, device="cuda")
    elif kind == "norm":
        t, h, d = case["tokens"], case["heads"], case["dim"]
        s["x"] = normal(t, h * d, scale=0.3).half()
        s["z"] = normal(t, h * d)
        s["w"] = 1 + normal(d, scale=0.1)
        s["out"] = torch.zeros(t, h * d, dtype=torch.float16, device="cuda")
    else:
        t, h, kv, d = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
        s["width"] = (h + 2 * kv) * d
        s["qkv"] = normal(t, s["width"])
        s["q_norm"] = 1 + normal(d, scale=0.1) if case["norm"] else None
        s["k_norm"] = 1 + normal(d, scale=0.1) if case["norm"] else None
        s["factor"] = 1 + 7 * torch.rand(case["rope_dim"] // 2, generator=g, device="cuda") if case["factor"] else None
        # rows of a text with images: time runs on, height and width within an image's patches
        at = torch.arange(t, device="cuda") + 1000 * (1 + seed % 7)
        s["place"] = torch.stack([at, at - at % 48 + at // 8 % 48, at - at % 48 + at % 48, at // 2][:case["axes"]], 1).int().contiguous()
        for name, n in (("q", h), ("k", kv), ("v", kv)):
            s[name] = torch.zeros(t, n * d, dtype=torch.float16, device="cuda")
    s["at"] = {k: v.data_ptr() for k, v in s.items() if isinstance(v, torch.Tensor)}
    return s


# ---- plain forms --------------------------------------------------------------------------

def _silu(x):
    return x / (1 + torch.exp(-x))


def _gates(s):
    """(log decay, beta) of every row and head."""
    x = s["a"] + s["dt"]
    soft = torch.clamp(x, min=0) + torch.log1p(torch.exp(-torch.abs(x)))
    return s["decay"] * soft, 1 / (1 + torch.exp(-s["b"]))


def _heads(s):
    """Unit q and k rows and v rows per value head, fp32 [tokens][heads][d]."""
    c = s["case"]
    heads, keys, d = c["heads"], c["key_heads"], c["dim"]
    x = s["qkv"].float()
    q, k, v = x[:, :keys * d], x[:, keys * d:2 * keys * d], x[:, 2 * keys * d:]
    q, k = (y.reshape(-1, keys, d) for y in (q, k))
    q = q / torch.sqrt((q * q).sum(-1, keepdim=True) + EPS) / math.sqrt(d)
    k = k / torch.sqrt((k * k).sum(-1, keepdim=True) + EPS)
    of = torch.arange(heads, device=x.device) // (heads // keys)
    return q[:, of], k[:, of], v.reshape(-1, heads, d)


def _start(s):
    """The states of the call's sequences: zeros where the sequence begins at position 0."""
    keep = (s["pos"] != 0).float()
    return s["state"][s["agent"].long()] * keep.view(-1, *[1] * (s["state"].dim() - 1))


def _plain_step(s):
    q, k, v = _heads(s)
    g, beta = _gates(s)
    state = _start(s) * torch.exp(g)[..., None, None]
    u = beta[..., None] * (v - (state * k[..., None]).sum(-2))
    state = state + k[..., None] * u[..., None, :]
    s["out"].copy_((state * q[..., None]).sum(-2).reshape(s["out"].shape))
    s["state"][s["agent"].long()] = state
    return s["out"], s["state"]


def _plain_chunk(s):
    c = s["case"]
    n, h, d = c["seqs"], c["heads"], c["dim"]
    chunks = max(1, -(-max(s["lens"]) // CHUNK))
    rows = torch.arange(chunks * CHUNK, device="cuda")
    lens = (s["offset"][1:] - s["offset"][:-1]).long()
    live = rows < lens[:, None]                                          # [seqs][rows]
    at = torch.where(live, s["offset"][:-1, None].long() + rows, 0)

    def lay(x):                                                          # -> [seqs][heads][chunks][64][...]
        x = x[at] * live.view(*live.shape, *[1] * (x.dim() - 1))
        x = x.view(n, chunks, CHUNK, h, *x.shape[3:])
        return x.movedim(3, 1).contiguous()

    q, k, v = (lay(x) for x in _heads(s))
    g, beta = (lay(x) for x in _gates(s))
    total = torch.cumsum(g, -1)
    low = torch.ones(CHUNK, CHUNK, device="cuda").tril(-1).bool()
    fade = torch.exp(torch.where(low | torch.eye(CHUNK, device="cuda").bool(), total[..., :, None] - total[..., None, :], float("-inf")))
    m = torch.where(low, beta[..., None] * (k @ k.transpose(-1, -2).contiguous()) * fade, 0)
    t = torch.diag_embed(beta)
    for i in range(1, CHUNK):                                            # rows of (1 + m)^-1 diag(beta)
        t[..., i, :] -= (m[..., i, :i, None] * t[..., :i, :]).sum(-2)
    p = (q @ k.transpose(-1, -2).contiguous()) * fade
    state = _start(s)
    out = torch.empty_like(v)
    for i in range(chunks):                                              # each starts from the last one's state
        e = torch.exp(total[:, :, i])[..., None]
        u = t[:, :, i] @ (v[:, :, i] - e * (k[:, :, i] @ state))
        out[:, :, i] = e * (q[:, :, i] @ state) + p[:, :, i] @ u
        last = total[:, :, i, -1:, None]
        kept = k[:, :, i] * torch.exp(last - total[:, :, i][..., None])
        state = torch.exp(last) * state + kept.transpose(-1, -2).contiguous() @ u
    s["out"].copy_(out.movedim(1, 3).reshape(n, chunks * CHUNK, h * d)[live])
    s["state"][s["agent"].long()] = state
    return s["out"], s["state"]


def _plain_conv(s):
    c, w = s["case"]["channels"], s["case"]["width"]
    lens = (s["offset"][1:] - s["offset"][:-1]).long()
    seq = torch.repeat_interleave(torch.arange(len(s["lens"]), device="cuda"), lens, output_size=s["tokens"])
    # rows of every sequence behind the w - 1 rows that its slot keeps
    full = torch.empty(s["tokens"] + (w - 1) * len(s["lens"]), c, device="cuda")
    begin = s["offset"][:-1].long() + (w - 1) * torch.arange(len(s["lens"]), device="cuda")
    for j in range(w - 1):
        full[begin + j] = _start(s)[:, j]
    row = torch.arange(s["tokens"], device="cuda") + (w - 1) * (seq + 1)
    full[row] = s["x"]
    y = s["bias"] if s["bias"] is not None else torch.zeros(c, device="cuda")
    for j in range(w):
        y = y + full[row - (w - 1) + j] * s["w"][:, j]
    s["out"].copy_(_silu(y))
    for j in range(w - 1):
        s["state"][s["agent"].long(), j] = full[begin + lens + j]
    return s["out"], s["state"]


def _plain_norm(s):
    h, d = s["case"]["heads"], s["case"]["dim"]
    x = s["x"].float().view(-1, h, d)
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * s["w"]
    s["out"].copy_(y.view(-1, h * d) * _silu(s["z"]))
    return s["out"]


def _turn(x, norm, s, cos, sin):
    """Head norm and turn of [tokens][heads][d]."""
    r, split = s["case"]["rope_dim"], s["case"]["pairs"] == SPLIT
    if norm is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * norm
    a, b = (x[..., :r // 2], x[..., r // 2:r]) if split else (x[..., 0:r:2], x[..., 1:r:2])
    a, b = a * cos - b * sin, a * sin + b * cos
    turned = torch.cat([a, b], -1) if split else torch.stack([a, b], -1).flatten(-2)
    return torch.cat([turned, x[..., r:]], -1)


def _plain_rope(s):
    c = s["case"]
    h, kv, d, r = c["heads"], c["kv_heads"], c["dim"], c["rope_dim"]
    i = torch.arange(r // 2, dtype=torch.float64, device="cuda")
    angle = s["place"][:, torch.tensor(_axis_of(c), device="cuda")].double() * torch.exp(-2 * i / r * math.log(c["theta"]))
    if s["factor"] is not None:
        angle = angle / s["factor"].double()
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    x = s["qkv"].view(-1, h + 2 * kv, d)
    s["q"].copy_(_turn(x[:, :h], s["q_norm"], s, cos, sin).reshape(s["q"].shape))
    s["k"].copy_(_turn(x[:, h:h + kv], s["k_norm"], s, cos, sin).reshape(s["k"].shape))
    s["v"].copy_(x[:, h + kv:].reshape(s["v"].shape))
    return s["q"], s["k"], s["v"]


# ---- the library's kernels ------------------------------------------------------------------

def _own(s):
    import aotx_amd as A
    lib, c, at = A.lib(), s["case"], s["at"]
    get, stream = at.get, torch.cuda.current_stream().cuda_stream
    kind = c["kind"]
    if kind == "step":
        rc = lib.aotx_delta_step(at["qkv"], s["width"], at["a"], at["b"], c["heads"], at["decay"], at["dt"],
                                 at["pos"], at["agent"], s["tokens"], c["key_heads"], c["heads"], c["dim"], EPS,
                                 at["state"], s["held"], at["out"], stream)
        got = s["out"], s["state"]
    elif kind == "chunk":
        if "work" not in s:                                              # kept for the passes after
            need = lib.aotx_delta_work(s["tokens"], c["seqs"], c["heads"], c["dim"])
            s["work"] = torch.empty(need, dtype=torch.uint8, device="cuda")
        rc = lib.aotx_delta_chunk(at["qkv"], s["width"], at["a"], at["b"], c["heads"], at["decay"], at["dt"],
                                  at["offset"], at["pos"], at["agent"], c["seqs"], s["tokens"], c["key_heads"],
                                  c["heads"], c["dim"], EPS, at["state"], s["held"], s["work"].data_ptr(), s["work"].numel(),
                                  at["out"], stream)
        got = s["out"], s["state"]
    elif kind == "conv":
        rc = lib.aotx_delta_conv(at["x"], c["channels"], at["w"], get("bias"), at["offset"], at["pos"], at["agent"],
                                 c["seqs"], s["tokens"], c["channels"], c["width"], at["state"], s["held"], at["out"], stream)
        got = s["out"], s["state"]
    elif kind == "norm":
        rc = lib.aotx_norm_gate(at["x"], at["z"], c["heads"] * c["dim"], at["w"], c["tokens"], c["heads"], c["dim"],
                                EPS, at["out"], stream)
        got = s["out"]
    else:
        how = A.RopeHow(theta=c["theta"], eps=EPS, rope_dim=c["rope_dim"], pairs=c["pairs"], axes=c["axes"],
                        order=c["order"], span=(A.u32 * 4)(*_spans(c)))
        rc = lib.aotx_rope_axes(at["qkv"], s["width"], get("q_norm"), get("k_norm"), how, get("factor"), at["place"],
                                c["tokens"], c["heads"], c["kv_heads"], c["dim"], at["q"], at["k"], at["v"], stream)
        got = s["q"], s["k"], s["v"]
    A.check(rc, kind)
    return got


def run(state):
    if own:
        return _own(state)
    return {"step": _plain_step, "chunk": _plain_chunk, "conv": _plain_conv, "norm": _plain_norm,
            "rope": _plain_rope}[state["case"]["kind"]](state)


# ---- what a pass has to move, and its outputs in 64 bits ------------------------------------

def work(case):
    kind = case["kind"]
    if kind in ("step", "chunk"):
        heads, keys, d = case["heads"], case["key_heads"], case["dim"]
        lens = [1] * case["slots"] if kind == "step" else _lengths(case)
        t = sum(lens)
        states = heads * d * d * 4 * len(lens) * (1 if kind == "chunk" and case["fresh"] else 2)
        return {"bytes": t * ((2 * keys + 2 * heads) * d * 2 + 8 * heads) + states, "flops": 6 * t * heads * d * d}
    if kind == "conv":
        c, w, lens = case["channels"], case["width"], _lengths(case)
        kept = (w - 1) * c * 4 * len(lens) * (1 if case["fresh"] else 2)
        return {"bytes": sum(lens) * c * 6 + kept + c * w * 4, "flops": sum(lens) * c * (2 * w + 4)}
    if kind == "norm":
        n = case["tokens"] * case["heads"] * case["dim"]
        return {"bytes": 8 * n + 4 * case["dim"], "flops": 9 * n}
    n = case["tokens"] * (case["heads"] + 2 * case["kv_heads"]) * case["dim"]
    return {"bytes": 6 * n + 4 * case["axes"] * case["tokens"], "flops": 6 * n}


def _exact_delta(s):
    """Token by token, every sequence's row t at once."""
    c = s["case"]
    heads, keys, d = c["heads"], c["key_heads"], c["dim"]
    x = s["qkv"].double()
    group = heads // keys
    q = x[:, :keys * d].view(-1, keys, 1, d).expand(-1, keys, group, d).reshape(-1, heads, d)
    k = x[:, keys * d:2 * keys * d].view(-1, keys, 1, d).expand(-1, keys, group, d).reshape(-1, heads, d)
    v = x[:, 2 * keys * d:].view(-1, heads, d)
    q = q * (q.square().sum(-1, keepdim=True) + EPS).rsqrt() * d ** -0.5
    k = k * (k.square().sum(-1, keepdim=True) + EPS).rsqrt()
    fade = torch.exp(s["decay"].double() * torch.logaddexp(s["a"].double() + s["dt"].double(), torch.zeros((), dtype=torch.float64, device="cuda")))
    beta = torch.sigmoid(s["b"].double())
    state = s["state"].double()
    out = torch.zeros(s["tokens"], heads, d, dtype=torch.float64, device="cuda")
    begins = [sum(s["lens"][:i]) for i in range(len(s["lens"]))]
    for i, (slot, first) in enumerate(zip(s["slots"], s["first"])):
        if first == 0 and s["lens"][i] > 0:
            state[slot] = 0
    order = sorted(range(len(begins)), key=lambda i: -s["lens"][i])      # the longest first
    slots = torch.tensor([s["slots"][i] for i in order], device="cuda")
    begin = torch.tensor([begins[i] for i in order], device="cuda")
    held = state[slots]
    for t in range(max(s["lens"])):
        live = sum(1 for n in s["lens"] if n > t)
        at = begin[:live] + t
        now = held[:live]
        now *= fade[at][..., None, None]
        u = beta[at][..., None] * (v[at] - torch.matmul(k[at][..., None, :], now)[..., 0, :])
        now += k[at][..., None] * u[..., None, :]
        out[at] = torch.matmul(q[at][..., None, :], now)[..., 0, :]
    state[slots] = held
    return out.view(s["tokens"], heads * d), state


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind in ("step", "chunk"):
        return _exact_delta(s)
    if kind == "conv":
        w, state = case["width"], s["state"].double()
        out, begin = [], 0
        for slot, first, n in zip(s["slots"], s["first"], s["lens"]):
            before = state[slot] if first else torch.zeros_like(state[slot])
            x = torch.cat([before, s["x"][begin:begin + n].double()])
            y = (x.unfold(0, w, 1) * s["w"].double()).sum(-1)
            y = y + s["bias"].double() if s["bias"] is not None else y
            out.append(y * torch.sigmoid(y))
            state[slot] = x[n:]
            begin += n
        return torch.cat(out), state
    if kind == "norm":
        x = s["x"].double().view(case["tokens"], case["heads"], case["dim"])
        y = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * s["w"].double()
        z = s["z"].double()
        return y.view(z.shape) * z * torch.sigmoid(z)
    h, kv, d, r = case["heads"], case["kv_heads"], case["dim"], case["rope_dim"]
    x = s["qkv"].double().view(-1, h + 2 * kv, d)
    freq = torch.tensor([case["theta"] ** (-2.0 * i / r) for i in range(r // 2)], dtype=torch.float64, device="cuda")
    if s["factor"] is not None:
        freq = freq / s["factor"].double()
    where = torch.tensor(_axis_of(case), device="cuda")
    turn = s["place"].double()[:, where] * freq
    turn = torch.polar(torch.ones_like(turn), turn)[:, None]

    def one(y, norm):
        if norm is not None:
            y = y / (y.square().mean(-1, keepdim=True) + EPS).sqrt() * norm.double()
        low, high = (y[..., :r // 2], y[..., r // 2:r]) if case["pairs"] == SPLIT else (y[..., 0:r:2], y[..., 1:r:2])
        z = torch.complex(low.contiguous(), high.contiguous()) * turn
        y = y.clone()
        if case["pairs"] == SPLIT:
            y[..., :r // 2], y[..., r // 2:r] = z.real, z.imag
        else:
            y[..., 0:r:2], y[..., 1:r:2] = z.real, z.imag
        return y.reshape(y.shape[0], -1)

    return one(x[:, :h], s["q_norm"]), one(x[:, h:h + kv], s["k_norm"]), x[:, h + kv:].reshape(-1, kv * d)
