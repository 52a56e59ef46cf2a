"""Timing cases of the operators that stand around the Dense, attention and recurrent layers in a training step: the word
embedding and its gradient, the norms before and after a block with the block's gate and residual scale, and the AdamW
step over all tensors of a network with states in 32 or in 8 bits.

With ``own`` false ``run`` computes an operator in elementary torch operations, with ``own`` true through the package's
entry points on the same device memory.

Definitions
  embedding   y[t] = scale * W[id[t]];  dW[v] = scale * sum of dy[t] over the tokens t with id[t] = v.  An id outside
              [0, vocabulary) is no token: a row of zeros, no gradient.
  block norm  u = x + residual_scale * act(gate) * N_post(y);  h = N_pre(u)  (u as it is stored);
              N(z) = (z - mean) * rstd * weight + bias  (layer), z * rstd * weight  (rms), z  (none).
  AdamW       m' = b1 m + (1 - b1) g;  v' = b2 v + (1 - b2) g g;
              p' = p (1 - lr wd) - lr / (1 - b1^t) * m' / (sqrt(v') / sqrt(1 - b2^t) + eps).
              States in 8 bits: blocks of 256 elements of one tensor, m as e4m3 and v as e5m2 times a power of two per
              block (2^(code - 127), code = max(e - 7, 1) for m and max(e - 14, 1) for v with e the biased exponent of
              the block's largest magnitude), rounded up or down at random with 16 bits each of a Philox4x32-10 word
              (key: seed; counter: element / 4 low, high, tensor, step; word: element % 4; low half m, high half v);
              a positive v is never stored as zero.
"""
import math

import torch

own = False

BLOCK = 256
BETA1, BETA2, EPS, DECAY, RATE = 0.9, 0.999, 1e-8, 0.1, 1e-3
NORM_EPS = 1e-5
_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "i32": torch.int32, "i64": torch.int64}
_BYTES = {"f32": 4, "bf16": 2, "i32": 4, "i64": 8}


# ---------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------
def listed():
    emb, norm = "embedding", "block norm"
    return [
        # one new token for each of a batch of sequences that are being generated
        dict(name="embed 64x1024", op=emb, backward=False, tokens=64, vocabulary=32000, dim=1024, ids="i32", table="bf16", out="bf16", pad=False),
        # a training batch of 32 sequences of 1024 tokens, fp32 table into bf16 activations
        dict(name="embed 32768x2048", op=emb, backward=False, tokens=32768, vocabulary=50000, dim=2048, ids="i64", table="f32", out="bf16", pad=True),
        # a word-level text classifier as the reference trains it: float ids, a small odd vocabulary
        dict(name="embed grad 4000x100", op=emb, backward=True, tokens=4000, vocabulary=5003, dim=100, ids="f32", table="f32", out="f32", pad=True),
        # the gradient of the training batch above, half the width and twice the tokens
        dict(name="embed grad 65536x1024", op=emb, backward=True, tokens=65536, vocabulary=50000, dim=1024, ids="i64", table="f32", out="bf16", pad=True),
        # generation: the join between two blocks for a handful of rows
        dict(name="norm 8x4096", op=norm, backward=False, rows=8, dim=4096, pre="rms", post="rms", gate="vector", group=0, act="none", bias=False, stream="bf16", block="bf16", train=False),
        # a pre-norm layer on the rows of an odd width
        dict(name="norm 1000x1001", op=norm, backward=False, rows=1000, dim=1001, pre="layer", post="none", gate="none", group=0, act="none", bias=True, stream="f32", block="f32", train=True),
        # a training step's join: fp32 residual stream, bf16 blocks, one gate row per sequence
        dict(name="norm 16384x2048", op=norm, backward=False, rows=16384, dim=2048, pre="layer", post="layer", gate="group", group=1024, act="sigmoid", bias=True, stream="f32", block="bf16", train=True),
        # the backward pass of a small model in fp32
        dict(name="norm grad 2048x512", op=norm, backward=True, rows=2048, dim=512, pre="layer", post="none", gate="vector", group=0, act="none", bias=True, stream="f32", block="f32", train=True),
        # the backward pass of a large one
        dict(name="norm grad 16384x4096", op=norm, backward=True, rows=16384, dim=4096, pre="rms", post="rms", gate="group", group=1, act="sigmoid", bias=False, stream="f32", block="bf16", train=True),
        # the LSTM layer of the recurrent benchmark (256 -> 512)
        dict(name="adamw lstm", op="adamw", layers=1, width=512, vocabulary=0, shape="lstm", bits=32, grad="f32", copy=False),
        # a transformer of 12 blocks of width 896 with its embedding, bf16 copies of the weights for the next step
        dict(name="adamw 12x896", op="adamw", layers=12, width=896, vocabulary=30000, shape="blocks", bits=32, grad="f32", copy=True),
        # a larger one whose states only fit in 8 bits
        dict(name="adamw8 24x1024", op="adamw", layers=24, width=1024, vocabulary=50000, shape="blocks", bits=8, grad="bf16", copy=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.randrange(6)
    two = ("f32", "bf16")
    if kind < 2:
        tokens, dim = _log(rng, 1, 65536), _log(rng, 16, 4096)
        dim = dim // 8 * 8 if rng.random() < 0.75 else dim
        vocabulary = min(_log(rng, 50, 130000), 100_000_000 // max(dim, 1))
        return dict(op="embedding", backward=kind == 1, tokens=min(tokens, 64_000_000 // dim), vocabulary=vocabulary, dim=dim,
                    ids=rng.choice(("i32", "i64", "f32")), table="f32" if kind == 1 else rng.choice(two), out=rng.choice(two), pad=rng.random() < 0.5)
    if kind < 4:
        dim = _log(rng, 32, 8192)
        dim = dim // 8 * 8 if rng.random() < 0.75 else dim
        rows = min(_log(rng, 1, 32768), 64_000_000 // dim)
        pre, post = rng.choice(("rms", "layer")), rng.choice(("none", "rms", "layer"))
        gate = rng.choice(("none", "vector", "group"))
        group = 0 if gate != "group" else rng.choice((1, max(1, rows // 8)))
        stream = rng.choice(two)
        return dict(op="block norm", backward=kind == 3, rows=rows, dim=dim, pre=pre, post=post, gate=gate, group=group,
                    act=rng.choice(("none", "sigmoid", "tanh")) if gate != "none" else "none", bias=rng.random() < 0.5,
                    stream=stream, block="bf16" if stream == "bf16" else rng.choice(two), train=True)
    width = _log(rng, 64, 960) // 4 * 4 + rng.choice((0, 0, 1))
    return dict(op="adamw", layers=rng.randint(1, 12), width=width, vocabulary=_log(rng, 10, 50000), shape=rng.choice(("blocks", "lstm")),
                bits=32 if kind == 4 else 8, grad=rng.choice(two), copy=rng.random() < 0.5)


def _shapes(c):
    """The tensors of an AdamW case: (shape, decayed) of every parameter."""
    w, out = c["width"], []
    if c["vocabulary"]:
        out.append(((c["vocabulary"], w), True))
    for _ in range(c["layers"]):
        if c["shape"] == "lstm":
            out += [((4 * w, w // 2), True), ((4 * w, w), True), ((4 * w,), False), ((4 * w,), False)]
        else:
            out += [((w, w), True)] * 4 + [((w,), False)] * 4 + [((4 * w, w), True), ((4 * w,), False), ((w, 4 * w), True), ((w,), False)]
            out += [((w,), False)] * 4
    return out


def _offsets(c):
    """Where each tensor starts in the parameter space (multiples of 256 elements), and the size of the space."""
    at, total = [], 0
    for shape, decayed in _shapes(c):
        n = math.prod(shape)
        at.append((total, n, decayed))
        total += -(-n // BLOCK) * BLOCK
    return at, total


def work(case):
    c = case
    if c["op"] == "embedding":
        t, v, d = c["tokens"], c["vocabulary"], c["dim"]
        ids = t * _BYTES[c["ids"]]
        if c["backward"]:
            return {"bytes": ids + t * d * _BYTES[c["out"]] + 4 * v * d, "flops": t * d + v * d}
        return {"bytes": ids + min(t, v) * d * _BYTES[c["table"]] + t * d * _BYTES[c["out"]], "flops": t * d}
    if c["op"] == "block norm":
        r, d, s, b = c["rows"], c["dim"], _BYTES[c["stream"]], _BYTES[c["block"]]
        joined = c["post"] != "none" or c["gate"] != "none"
        gate = 0 if c["gate"] == "none" else 4 * d if c["gate"] == "vector" else -(-r // c["group"]) * d * b
        weights = 4 * d * ((1 if c["pre"] != "none" else 0) + (1 if c["post"] != "none" else 0)) * (2 if c["bias"] else 1)
        stats = 8 * r * (1 + (c["post"] != "none")) if c["train"] else 0
        if c["backward"]:
            moved = r * d * (3 * s + b + (2 * b if joined else 0))
            return {"bytes": moved + 2 * gate + 2 * weights + stats, "flops": 30 * r * d}
        moved = r * d * ((2 * s + 2 * b) if joined else s + b)
        return {"bytes": moved + gate + weights + stats, "flops": 16 * r * d}
    n = sum(math.prod(shape) for shape, _ in _shapes(c))
    state = 16 if c["bits"] == 32 else 4 + 4 / BLOCK
    return {"bytes": n * (8 + _BYTES[c["grad"]] + state + (2 if c["copy"] else 0)), "flops": 16 * n}


# ---------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, sigma=1.0, mean=0.0, type="f32"):
        return torch.randn(*shape, device="cuda", generator=gen).mul_(sigma).add_(mean).to(_TYPES[type])

    if c["op"] == "embedding":
        t, v, d = c["tokens"], c["vocabulary"], c["dim"]
        # word frequencies fall off as 1 / rank
        ids = (torch.rand(t, device="cuda", generator=gen, dtype=torch.float64) * math.log(v + 1)).exp().sub(1).long().clamp(0, v - 1)
        if c["pad"]:  # the ends of the batch's short sequences
            ids[t - t // 16:] = -1
        s = {"case": c, "scale": math.sqrt(d), "ids": ids.to(_TYPES[c["ids"]])}
        if c["backward"]:
            s["dy"] = normal(t, d, sigma=0.01, type=c["out"])
            s["dw"] = torch.empty(v, d, device="cuda")
        else:
            s["w"] = normal(v, d, sigma=1 / math.sqrt(d), type=c["table"])
            s["y"] = torch.empty(t, d, device="cuda", dtype=_TYPES[c["out"]])
        return s
    if c["op"] == "block norm":
        r, d = c["rows"], c["dim"]
        joined = c["post"] != "none" or c["gate"] != "none"
        s = {"case": c, "scale": 0.7, "joined": joined, "x": normal(r, d, sigma=2.0, mean=0.1, type=c["stream"])}
        if joined:
            s["y"] = normal(r, d, sigma=0.5, type=c["block"])
        if c["gate"] == "vector":
            s["gate"] = normal(d, sigma=0.3, mean=0.5)
        elif c["gate"] == "group":
            s["gate"] = normal(-(-r // c["group"]), d, type=c["block"])
        for which in ("pre", "post"):
            if c[which] != "none":
                s[which + "_weight"] = normal(d, sigma=0.1, mean=1.0)
                if c["bias"] and c[which] == "layer":
                    s[which + "_bias"] = normal(d, sigma=0.1)
        if c["backward"]:
            s["u"] = s.pop("x")
            s["du"] = normal(r, d, sigma=0.01, type=c["stream"])
            s["dh"] = normal(r, d, sigma=0.01, type=c["block"])
            s["pre_stats"] = _statistics(s["u"], c["pre"])
            if c["post"] != "none":
                s["post_stats"] = _statistics(s["y"], c["post"])
        return s
    at, total = _offsets(c)
    s = {"case": c, "at": at, "step": 100, "seed": seed}
    real = torch.zeros(total, device="cuda")
    decay = torch.zeros(total // BLOCK, device="cuda")
    for off, n, decayed in at:
        real[off:off + n] = 1
        if decayed:
            decay[off // BLOCK:-(-(off + n) // BLOCK)] = DECAY
    s["decay"] = decay
    s["p"] = normal(total, sigma=0.02).mul_(real)
    # gradients whose size differs from one run of 256 elements to the next, some elements without any
    size = torch.exp(normal(total // BLOCK, sigma=1.5, mean=-7.0)).repeat_interleave(BLOCK)
    drop = torch.rand(total, device="cuda", generator=gen) < 0.02
    s["g"] = (normal(total) * size).mul_(real).masked_fill_(drop, 0).to(_TYPES[c["grad"]])
    m = (normal(total) * size * 0.3).mul_(real)
    v = (normal(total).square_().mul_(0.5).add_(0.5) * size.square()).mul_(real)
    del size, drop, real
    if c["bits"] == 32:
        s["m"], s["v"] = m, v
    else:
        s["m"], s["m_code"] = _nearest8(m, 7, torch.float8_e4m3fn)
        s["v"], s["v_code"] = _nearest8(v, 14, torch.float8_e5m2)
    del m, v
    if c["copy"]:
        s["copy"] = s["p"].to(torch.bfloat16)
    if c["bits"] == 8:  # which tensor an element belongs to, and which quarter of four of it: what the random words go by
        s["tensor"] = torch.zeros(total // BLOCK, device="cuda", dtype=torch.int32)
        s["first"] = torch.zeros(total // BLOCK, device="cuda", dtype=torch.int32)
        for k, (off, n, _) in enumerate(at):
            b0, b1 = off // BLOCK, -(-(off + n) // BLOCK)
            s["tensor"][b0:b1] = k
            s["first"][b0:b1] = torch.arange(b1 - b0, device="cuda", dtype=torch.int32)
    return s


def _statistics(z, kind):
    z = z.double()
    mean = z.mean(1) if kind == "layer" else torch.zeros_like(z[:, 0])
    var = (z - mean[:, None]).square().mean(1)
    return torch.stack((mean, (var + NORM_EPS).rsqrt()), 1).float()


def _power(e):
    """2^e in 32 bits, exactly (-126 <= e <= 127)."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _nearest8(x, room, type):
    """8-bit states as an earlier step left them (here rounded to nearest): the values, and the code of each block's power of two."""
    blocks = x.view(-1, BLOCK)
    code = ((blocks.abs().amax(1).view(torch.int32) >> 23) - room).clamp_(min=1)
    return (blocks * _power(127 - code)[:, None]).to(type).view(-1), code.to(torch.uint8)


# ---------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------
def run(state):
    c = state["case"]
    if c["op"] == "embedding":
        return _embedding_own(state) if own else _embedding_plain(state)
    if c["op"] == "block norm":
        if c["backward"]:
            return _norm_backward_own(state) if own else _norm_backward_plain(state)
        return _norm_forward_own(state) if own else _norm_forward_plain(state)
    state["step"] += 1
    return _adamw_own(state) if own else _adamw_plain(state)


# -- the plain forms ------------------------------------------------------------------------------------------------
def _embedding_plain(s):
    c = s["case"]
    ids = s["ids"].long()
    valid = (ids >= 0) & (ids < c["vocabulary"])
    factor = valid.float().mul_(s["scale"])[:, None]
    ids = ids.masked_fill(~valid, 0)
    if c["backward"]:
        return torch.zeros_like(s["dw"]).index_add_(0, ids, s["dy"].float() * factor)
    return (s["w"][ids].float() * factor).to(s["y"].dtype)


def _act(gate, act):
    return torch.sigmoid(gate) if act == "sigmoid" else torch.tanh(gate) if act == "tanh" else gate


def _act_slope(q, act):
    return q * (1 - q) if act == "sigmoid" else 1 - q * q if act == "tanh" else torch.ones_like(q)


def _gate_rows(s):
    """The gate of every row, as (rows, dim) or a vector."""
    c = s["case"]
    g = s["gate"].float()
    return g if c["gate"] == "vector" or c["group"] == 1 else g.repeat_interleave(c["group"], 0)[: c["rows"]]


def _norm_plain(z, kind, weight, bias):
    """The normed rows and (mean, 1 / deviation) of each."""
    if kind == "layer":
        mean = z.mean(1, keepdim=True)
        z = z - mean
        rstd = (z.square().mean(1, keepdim=True) + NORM_EPS).rsqrt()
    else:
        mean = torch.zeros_like(z[:, :1])
        rstd = (z.square().mean(1, keepdim=True) + NORM_EPS).rsqrt()
    n = z * rstd * weight
    return (n if bias is None else n + bias), torch.cat((mean, rstd), 1)


def _norm_forward_plain(s):
    c, out = s["case"], {}
    u = s["x"]
    if s["joined"]:
        n = s["y"].float()
        if c["post"] != "none":
            n, out["post_stats"] = _norm_plain(n, c["post"], s["post_weight"], s.get("post_bias"))
        if c["gate"] != "none":
            n = n * _act(_gate_rows(s), c["act"])
        u = out["u"] = (s["x"].float() + s["scale"] * n).to(s["x"].dtype)
    h, out["pre_stats"] = _norm_plain(u.float(), c["pre"], s["pre_weight"], s.get("pre_bias"))
    out["h"] = h.to(_TYPES[c["block"]])
    if not c["train"]:
        out.pop("pre_stats"), out.pop("post_stats", None)
    return out


def _norm_slope(z, stats, kind, weight, dn):
    """(dz, z normed) for n = N(z), given dn."""
    mean, rstd = stats[:, :1], stats[:, 1:]
    z = (z - mean) * rstd
    a = dn * weight
    da = a - z * (a * z).mean(1, keepdim=True)
    if kind == "layer":
        da = da - a.mean(1, keepdim=True)
    return da * rstd, z


def _norm_backward_plain(s):
    c, out = s["case"], {}
    dh = s["dh"].float()
    dx, z = _norm_slope(s["u"].float(), s["pre_stats"], c["pre"], s["pre_weight"], dh)
    out["d_pre_weight"] = (dh * z).sum(0)
    if "pre_bias" in s:
        out["d_pre_bias"] = dh.sum(0)
    dx = dx + s["du"].float()
    out["dx"] = dx.to(s["u"].dtype)
    if not s["joined"]:
        return out
    t, y = dx * s["scale"], s["y"].float()
    z = (y - s["post_stats"][:, :1]) * s["post_stats"][:, 1:] if c["post"] != "none" else y
    if c["gate"] != "none":
        q = _act(_gate_rows(s), c["act"])
        n = z
        if c["post"] != "none":
            n = z * s["post_weight"]
            n = n + s["post_bias"] if "post_bias" in s else n
        dq = t * n * _act_slope(q, c["act"])
        if c["gate"] == "vector":
            out["d_gate"] = dq.sum(0)
        else:
            if c["group"] > 1:
                short = -c["rows"] % c["group"]
                dq = torch.cat((dq, dq.new_zeros(short, c["dim"]))) if short else dq
                dq = dq.view(-1, c["group"], c["dim"]).sum(1)
            out["d_gate"] = dq.to(s["gate"].dtype)
        t = t * q
    if c["post"] != "none":
        out["d_post_weight"] = (t * z).sum(0)
        if "post_bias" in s:
            out["d_post_bias"] = t.sum(0)
        t, _ = _norm_slope(y, s["post_stats"], c["post"], s["post_weight"], t)
    out["dy"] = t.to(s["y"].dtype)
    return out


def _philox(counter, key):
    """Four 32-bit words (in int64) per counter of four of them: ten rounds."""
    a, b, c, d = counter
    k0, k1 = key
    for _ in range(10):
        x, y = a * 0xD2511F53, c * 0xCD9E8D57
        a, b, c, d = ((y >> 32) & 0xFFFFFFFF) ^ b ^ k0, y & 0xFFFFFFFF, ((x >> 32) & 0xFFFFFFFF) ^ d ^ k1, x & 0xFFFFFFFF
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return a, b, c, d


def _words(s):
    quad = s["first"].long()[:, None] * (BLOCK // 4) + torch.arange(BLOCK // 4, device="cuda")
    tensor = s["tensor"].long()[:, None].expand_as(quad)
    counter = (quad, torch.zeros_like(quad), tensor, torch.full_like(quad, s["step"]))
    return torch.stack(_philox(counter, (s["seed"] & 0xFFFFFFFF, s["seed"] >> 32)), 2).view(-1, BLOCK)


def _store8(x, room, mantissa, lowest, random, type):
    """x (blocks of 256) rounded at random to `type` times a power of two per block: (values, code)."""
    code = ((x.abs().amax(1).view(torch.int32) >> 23) - room).clamp_(min=1)
    t = x * _power(127 - code)[:, None]
    e = ((t.abs().view(torch.int32) >> 23) - 127).clamp_(min=lowest)
    whole = (t.abs() * _power(23 - e)).to(torch.int32)
    k = (whole + (random << (7 - mantissa))) >> (23 - mantissa)
    if type == torch.float8_e5m2:
        k = torch.where((k == 0) & (x > 0), 1, k)
    return (k.float() * _power(e - mantissa)).copysign_(t).to(type).view(-1), code.to(torch.uint8)


def _adamw_plain(s):
    c, p, g = s["case"], s["p"], s["g"].float()
    if c["bits"] == 32:
        m, v = s["m"], s["v"]
    else:
        m = (s["m"].float().view(-1, BLOCK) * _power(s["m_code"].int() - 127)[:, None]).view(-1)
        v = (s["v"].float().view(-1, BLOCK) * _power(s["v_code"].int() - 127)[:, None]).view(-1)
    m.mul_(BETA1).add_(g * (1 - BETA1))
    v.mul_(BETA2).add_((g * g).mul_(1 - BETA2))
    p.view(-1, BLOCK).mul_((1 - RATE * s["decay"])[:, None])
    p.sub_(m / (v.sqrt().mul_(1 / math.sqrt(1 - BETA2 ** s["step"])).add_(EPS)) * (RATE / (1 - BETA1 ** s["step"])))
    if c["bits"] == 8:
        words = _words(s)
        m, s["m_code"] = _store8(m.view(-1, BLOCK), 7, 3, -6, (words & 0xFFFF).int(), torch.float8_e4m3fn)
        v, s["v_code"] = _store8(v.view(-1, BLOCK), 14, 2, -14, (words >> 16).int(), torch.float8_e5m2)
        s["m"], s["v"] = m, v
    if c["copy"]:
        s["copy"].copy_(p)
    return _adamw_out(s)


def _adamw_out(s):
    return {k: s[k] for k in ("p", "m", "v", "m_code", "v_code", "copy") if k in s}


# -- the package ------------------------------------------------------------------------------------------------------
def _tensor(t, shape=None):
    """The package's tensor on the memory of a torch tensor."""
    from sharpnet_amd import GPUTensor
    names = {torch.float32: "float32", torch.bfloat16: "bfloat16", torch.int32: "int32", torch.int64: "int64"}
    return GPUTensor.FromPointer(shape or list(t.shape), t.data_ptr(), names.get(t.dtype, "uint8"), owner=t)


def _held(s):
    """What a program that uses the package holds from step to step: its tensors and its layer."""
    if "held" not in s:
        from sharpnet_amd import embedding, normalization, optimizer
        c = s["case"]
        if c["op"] == "adamw":
            parts = []
            for off, n, _ in s["at"]:
                nb = -(-n // BLOCK)
                part = {k: _tensor(s[k][off:off + n]) for k in ("p", "g", "m", "v", "copy") if k in s}
                part.update({k: _tensor(s[k][off // BLOCK:off // BLOCK + nb]) for k in ("m_code", "v_code") if k in s})
                parts.append(part)
            states = [[q[k] for k in ("m", "v", "m_code", "v_code") if k in q] for q in parts]
            s["held"] = optimizer.AdamW([q["p"] for q in parts], [q["g"] for q in parts], learningRate=RATE, beta1=BETA1, beta2=BETA2,
                                        epsilon=EPS, weightDecay=[DECAY if decayed else 0.0 for _, _, decayed in s["at"]], stateBits=c["bits"],
                                        seed=s["seed"], states=states, copies=[q["copy"] for q in parts] if "copy" in s else None, step=s["step"] - 1)
        elif c["op"] == "embedding":
            s["held"] = {k: _tensor(v) for k, v in s.items() if isinstance(v, torch.Tensor)}
            s["layer"] = embedding.WordEmbedding(c["vocabulary"], c["dim"], scale=s["scale"])
        else:
            s["layer"] = normalization.BlockNorm(c["dim"], preNorm=c["pre"], postNorm=c["post"], residualScale=s["scale"], gateActivation=c["act"], epsilon=NORM_EPS)
            like = torch.empty_like
            if c["backward"]:
                s["out"] = {"dx": like(s["u"])}
                s["out"].update({"d_" + k: like(s[k]) for k in ("pre_weight", "pre_bias", "post_weight", "post_bias", "gate") if k in s})
                if s["joined"]:
                    s["out"]["dy"] = like(s["y"])
            else:
                s["out"] = {"h": torch.empty(c["rows"], c["dim"], device="cuda", dtype=_TYPES[c["block"]])}
                if s["joined"]:
                    s["out"]["u"] = like(s["x"])
                if c["train"]:
                    s["out"].update({k + "_stats": torch.empty(c["rows"], 2, device="cuda") for k in ("pre", "post") if c[k] != "none"})
            s["held"] = {k: _tensor(v) for k, v in list(s.items()) + list(s["out"].items()) if isinstance(v, torch.Tensor)}
    return s["held"]


def _embedding_own(s):
    t = _held(s)
    if s["case"]["backward"]:
        s["layer"].BackwardPropagation(t["dw"], t["ids"], t["dy"])
        return s["dw"]
    s["layer"].ForwardPropagation(t["y"], t["ids"], t["w"])
    return s["y"]


def _norm_forward_own(s):
    t = _held(s).get
    s["layer"].ForwardPropagation(t("x"), t("h"), y=t("y"), u=t("u"), gate=t("gate"), gateRows=s["case"]["group"], preWeight=t("pre_weight"), preBias=t("pre_bias"),
                                  postWeight=t("post_weight"), postBias=t("post_bias"), preStatistics=t("pre_stats"), postStatistics=t("post_stats"))
    return s["out"]


def _norm_backward_own(s):
    t = _held(s).get
    s["layer"].BackwardPropagation(t("dx"), t("u"), t("dh"), du=t("du"), y=t("y"), dy=t("dy"), gate=t("gate"), dGate=t("d_gate"), gateRows=s["case"]["group"],
                                   preWeight=t("pre_weight"), preStatistics=t("pre_stats"), dPreWeight=t("d_pre_weight"), dPreBias=t("d_pre_bias"),
                                   postWeight=t("post_weight"), postBias=t("post_bias"), postStatistics=t("post_stats"), dPostWeight=t("d_post_weight"), dPostBias=t("d_post_bias"))
    return s["out"]


def _adamw_own(s):
    _held(s).Step()
    return _adamw_out(s)


# ---------------------------------------------------------------------------------------------------------------
# 64 bits
# ---------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    c = case
    if c["op"] == "embedding":
        return _embedding_exact(s)
    if c["op"] == "block norm":
        return _norm_backward_exact(s) if c["backward"] else _norm_forward_exact(s)
    s["step"] += 1
    return _adamw_exact(s)


def _embedding_exact(s):
    c = s["case"]
    ids = s["ids"].double()
    keep = torch.nonzero((ids >= 0) & (ids < c["vocabulary"])).view(-1)
    ids = ids[keep].long()
    if c["backward"]:
        dw = torch.zeros(c["vocabulary"], c["dim"], device="cuda", dtype=torch.float64)
        return dw.index_add_(0, ids, s["dy"][keep].double()).mul_(s["scale"])
    y = torch.zeros(c["tokens"], c["dim"], device="cuda", dtype=torch.float64)
    y[keep] = s["scale"] * s["w"].double()[ids]
    return y


def _exact_gate(s):
    """act(gate) of every row and its derivative, in 64 bits."""
    c = s["case"]
    g = s["gate"].double()
    if c["gate"] == "group":
        g = g[torch.arange(c["rows"], device="cuda") // c["group"]]
    if c["act"] == "sigmoid":
        e = torch.exp(-g)
        return 1 / (1 + e), e / (1 + e) ** 2
    if c["act"] == "tanh":
        return torch.tanh(g), 1 / torch.cosh(g) ** 2
    return g, torch.ones_like(g)


def _norm_forward_exact(s):
    c, out = s["case"], {}

    def norm(z, which):
        mu = z.mean(dim=1) if c[which] == "layer" else z.new_zeros(z.shape[0])
        sigma = torch.sqrt(((z - mu[:, None]) ** 2).mean(dim=1) + NORM_EPS)
        if c["train"]:
            out[which + "_stats"] = torch.stack((mu, 1 / sigma), dim=1)
        r = (z - mu[:, None]) / sigma[:, None] * s[which + "_weight"].double()
        return r + s[which + "_bias"].double() if which + "_bias" in s else r

    u = s["x"].double()
    if s["joined"]:
        n = norm(s["y"].double(), "post") if c["post"] != "none" else s["y"].double()
        if c["gate"] != "none":
            n = _exact_gate(s)[0] * n
        out["u"] = u + s["scale"] * n
        u = out["u"].to(s["x"].dtype).double()  # the norm reads the stream as it is stored
    out["h"] = norm(u, "pre")
    return out


def _norm_backward_exact(s):
    c, out = s["case"], {}

    def back(z, which, dn):
        mu, r = s[which + "_stats"].double().unbind(1)
        hat = (z - mu[:, None]) * r[:, None]
        out["d_%s_weight" % which] = (dn * hat).sum(dim=0)
        if which + "_bias" in s:
            out["d_%s_bias" % which] = dn.sum(dim=0)
        w = dn * s[which + "_weight"].double()
        inner = (w * hat).sum(dim=1, keepdim=True) / c["dim"]
        level = w.sum(dim=1, keepdim=True) / c["dim"] if c[which] == "layer" else 0.0
        return r[:, None] * (w - level - hat * inner), hat

    dx = s["du"].double() + back(s["u"].double(), "pre", s["dh"].double())[0]
    out["dx"] = dx
    if not s["joined"]:
        return out
    y, dn = s["y"].double(), s["scale"] * dx
    if c["gate"] != "none":
        n = y
        if c["post"] != "none":
            mu, r = s["post_stats"].double().unbind(1)
            n = (y - mu[:, None]) * r[:, None] * s["post_weight"].double()
            if "post_bias" in s:
                n = n + s["post_bias"].double()
        q, slope = _exact_gate(s)
        each = slope * n * dn
        rows = torch.arange(c["rows"], device="cuda") // c["group"] if c["gate"] == "group" else torch.zeros(c["rows"], device="cuda", dtype=torch.long)
        d_gate = torch.zeros(s["gate"].numel() // c["dim"], c["dim"], device="cuda", dtype=torch.float64).index_add_(0, rows, each)
        out["d_gate"] = d_gate.view(s["gate"].shape)
        dn = dn * q
    out["dy"] = back(y, "post", dn)[0] if c["post"] != "none" else dn
    return out


def _adamw_exact(s):
    c = s["case"]
    g = s["g"].double()
    two = lambda e: ((e.long() + 1023) << 52).view(torch.float64)  # noqa: E731
    per = lambda code: two(code.long() - 127).repeat_interleave(BLOCK)  # noqa: E731
    floor_log2 = lambda x: (x.view(torch.int64) >> 52) - 1023  # noqa: E731
    m0, v0 = s["m"].float().double(), s["v"].float().double()
    if c["bits"] == 8:
        m0, v0 = m0 * per(s["m_code"]), v0 * per(s["v_code"])
    m = BETA1 * m0 + (1 - BETA1) * g
    v = BETA2 * v0 + (1 - BETA2) * g * g
    del m0, v0, g
    rate = m / (1 - BETA1 ** s["step"]) / (torch.sqrt(v / (1 - BETA2 ** s["step"])) + EPS)
    p = s["p"].double() * (1 - RATE * s["decay"].double().repeat_interleave(BLOCK)) - RATE * rate
    del rate
    out = {"p": p}
    if c["copy"]:
        out["copy"] = p
    if c["bits"] == 32:
        out.update(m=m, v=v)
        return out
    out.update(m_code=None, v_code=None)  # whole numbers
    quad = s["first"].long().repeat_interleave(BLOCK // 4) * (BLOCK // 4) + torch.arange(BLOCK // 4, device="cuda").repeat(s["first"].numel())
    lo32 = 0xFFFFFFFF
    state = [quad, torch.zeros_like(quad), s["tensor"].long().repeat_interleave(BLOCK // 4), torch.full_like(quad, s["step"])]
    for r in range(10):
        left, right = state[0] * 0xD2511F53, state[2] * 0xCD9E8D57
        keys = (s["seed"] + r * 0x9E3779B9) & lo32, ((s["seed"] >> 32) + r * 0xBB67AE85) & lo32
        state = [((right >> 32) & lo32) ^ state[1] ^ keys[0], right & lo32, ((left >> 32) & lo32) ^ state[3] ^ keys[1], left & lo32]
    words = torch.stack(state, dim=1).view(-1)
    del state, quad, left, right
    for name, z, room, bits, lowest, chance in (("m", m, 7, 3, -6, words & 0xFFFF), ("v", v, 14, 2, -14, words >> 16)):
        top = z.abs().view(-1, BLOCK).amax(dim=1)
        unit = two(torch.clamp(floor_log2(top) - room, min=-126)).repeat_interleave(BLOCK)
        a = z.abs() / unit
        step = two(torch.clamp(floor_log2(a), min=lowest) - bits)
        k = torch.floor(a / step + chance.double() / 65536)
        if name == "v":
            k = torch.where((k == 0) & (a > 0), torch.ones_like(k), k)
        out[name] = torch.sign(z) * k * step
    return out
