"""Cases of the row operators of quantised transformer serving: per-row
quantisation, the dense product with its epilogue, the products grouped by
expert and the log probabilities at the end.  `run` computes a case either in
plain torch operations (own = False) or through dlq_amd.ops (own = True).

Codes: "s8" is int8, "f8" is e4m3 held as uint8 (the library's own form).
"""
import math

import torch

own = False

F8 = torch.float8_e4m3fn
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # -- quantise: activations on their way into a product
        # a prompt's hidden states, bf16, into int8
        dict(name="quant_s8_prompt", op="quant", type="s8", x="bf16", rows=8192, cols=8192, ld=8192),
        # a served batch's rows, fp32, odd width, padded rows for the product behind it
        dict(name="quant_f8_batch", op="quant", type="f8", x="f32", rows=257, cols=5001, ld=5008),
        # -- linear: the dense layers
        # one new token through an output projection: bias, residual stream added
        dict(name="linear_s8_token", op="linear", type="s8", M=1, N=4096, K=4096, pad=0, act="none", bias=True,
             residual=True, out="bf16"),
        # a decode batch through an up projection
        dict(name="linear_f8_decode", op="linear", type="f8", M=32, N=12288, K=4096, pad=0, act="silu", bias=False,
             residual=False, out="bf16"),
        # a long prompt through a square layer
        dict(name="linear_s8_prompt", op="linear", type="s8", M=8192, N=8192, K=8192, pad=0, act="gelu", bias=True,
             residual=False, out="bf16"),
        # a ragged prompt: no size a multiple of a tile, rows cut from a wider buffer
        dict(name="linear_f8_ragged", op="linear", type="f8", M=1003, N=5000, K=2736, pad=48, act="gelu_tanh",
             bias=True, residual=True, out="bf16"),
        # odd everything: a classifier head, fp32 logits
        dict(name="linear_s8_odd", op="linear", type="s8", M=77, N=1001, K=1531, pad=0, act="none", bias=True,
             residual=False, out="f32"),
        # -- grouped: the experts' products over rows sorted by expert
        # a decode batch spread thin over many experts, some without a row
        dict(name="grouped_s8_decode", op="grouped", type="s8", T=64, E=64, N=1536, K=2048, behind=0, act="silu",
             bias=False, residual=False, out="bf16"),
        # a prompt over few large experts, padding rows behind the last expert's
        dict(name="grouped_f8_prompt", op="grouped", type="f8", T=16384, E=8, N=4096, K=4096, behind=100,
             act="gelu_tanh", bias=True, residual=False, out="bf16"),
        # -- logprobs: what the model answered with
        # four sequences' next token with twenty alternatives, odd vocabulary
        dict(name="logprobs_f32_decode", op="logprobs", x="f32", rows=4, K=100003, top=20, masked=0.0),
        # a prompt's tokens scored, bf16 logits, part of the vocabulary masked out
        dict(name="logprobs_bf16_prompt", op="logprobs", x="bf16", rows=2048, K=65536, top=5, masked=0.25),
        # a router: few classes, many rows, the experts taken are the alternatives
        dict(name="logprobs_f32_router", op="logprobs", x="f32", rows=4096, K=64, top=8, masked=0.0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _size(rng, lo, hi):
    """A size spread over its logarithm: as drawn (odd ones among them) or a multiple of 16."""
    n = _log(rng, lo, hi)
    return n if rng.random() < 0.4 else max(16, n // 16 * 16)


def draw(rng):
    op = rng.choice(["quant", "linear", "linear", "grouped", "grouped", "logprobs", "logprobs"])
    act = rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"])
    if op == "quant":
        rows, cols = _log(rng, 1, 16384), _size(rng, 16, 16384)
        rows = min(rows, (1 << 26) // cols)
        return dict(op=op, type=rng.choice(["s8", "f8"]), x=rng.choice(["f32", "bf16"]), rows=rows, cols=cols,
                    ld=cols + rng.choice([0, 0, 1, 16]))
    t = rng.choice(["s8", "f8"])
    out = "bf16" if t == "f8" else rng.choice(["bf16", "f32"])
    if op == "linear":
        M, N, K = _log(rng, 1, 8192), _size(rng, 16, 16384), _size(rng, 16, 16384)
        N = min(N, (1 << 27) // K)
        M = min(M, (1 << 38) // (N * K))
        return dict(op=op, type=t, M=M, N=N, K=K, pad=rng.choice([0, 0, 7, 16, 64]), act=act,
                    bias=rng.random() < 0.5, residual=rng.random() < 0.5, out=out)
    if op == "grouped":
        T, E = _log(rng, 1, 16384), _log(rng, 2, 128)
        N, K = _size(rng, 32, 4096), _size(rng, 32, 4096)
        E = max(2, min(E, (1 << 27) // (N * K)))
        return dict(op=op, type=t, T=T, E=E, N=N, K=K, behind=rng.choice([0, 0, 1, 37]), act=act,
                    bias=rng.random() < 0.5, residual=rng.random() < 0.5, out=out)
    K = _log(rng, 8, 262144)
    rows = min(_log(rng, 1, 8192), (1 << 27) // K)
    return dict(op="logprobs", x=rng.choice(["f32", "bf16"]), rows=rows, K=K,
                top=min(K, rng.choice([0, 1, 5, 20, 64])), masked=rng.choice([0.0, 0.1, 0.6]))


# --------------------------------------------------------------- the inputs

def _codes(g, t, *shape):
    """Codes of a normally distributed tensor quantised at its largest value."""
    x = torch.randn(shape, generator=g, device="cuda")
    if t == "s8":
        return (x * 32.0).round_().clamp_(-127, 127).to(torch.int8)
    return (x * 112.0).clamp_(-448, 448).to(F8).view(torch.uint8)


def _counts(E, T, seed):
    """Rows per expert: some experts popular, some without a row; sums to T."""
    g = torch.Generator().manual_seed(seed)
    p = torch.rand(E, generator=g).clamp_(min=0.05)
    p[torch.rand(E, generator=g) < 0.15] = 0.0
    if not p.any():
        p[0] = 1.0
    return torch.bincount(torch.multinomial(p, T, replacement=True, generator=g), minlength=E)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    c = dict(case)
    if c["op"] == "quant":
        x = torch.randn(c["rows"], c["cols"], generator=g, device="cuda")
        x *= torch.exp(torch.randn(c["rows"], 1, generator=g, device="cuda"))
        return c | {"x": x.to(DT[c["x"]])}
    if c["op"] == "logprobs":
        rows, K = c["rows"], c["K"]
        x = torch.randn(rows, K, generator=g, device="cuda") * 2.5
        if c["masked"]:
            x.masked_fill_(torch.rand(rows, K, generator=g, device="cuda") < c["masked"], -math.inf)
        tokens = torch.randint(0, K, (rows,), generator=g, device="cuda", dtype=torch.int32)
        tokens[torch.rand(rows, generator=g, device="cuda") < 0.1] = -1  # padding: no token given
        return c | {"logits": x.to(DT[c["x"]]), "tokens": tokens}
    N, K, t = c["N"], c["K"], c["type"]
    if c["op"] == "linear":
        M, E = c["M"], 1
        x = _codes(g, t, M, K + c["pad"])[:, :K]
    else:
        E = c["E"]
        counts = _counts(E, c["T"], seed)
        M = c["T"] + c["behind"]
        x = _codes(g, t, M, K)
        first = torch.zeros(E + 1, dtype=torch.int64)
        first[1:] = counts.cumsum(0)
        c["offsets"] = first.to(torch.int32).cuda()
        c["most"] = int(counts.max())
        c["expert"] = torch.repeat_interleave(torch.arange(E), counts).cuda()
    c["x"] = x
    shape = (E,) if c["op"] == "grouped" else ()
    c["w"] = _codes(g, t, *shape, N, K)
    one = 1.0 / 32 if t == "s8" else 1.0 / 112
    c["x_scale"] = torch.exp(0.3 * torch.randn(M, generator=g, device="cuda")) * one
    c["w_scale"] = torch.exp(0.3 * torch.randn(*shape, N, generator=g, device="cuda")) * (one / K ** 0.5)
    c["b"] = torch.randn(*shape, N, generator=g, device="cuda") * 0.5 if c["bias"] else None
    c["r"] = torch.randn(M, N, generator=g, device="cuda").to(DT[c["out"]]) if c["residual"] else None
    if c["op"] == "grouped":
        c["y"] = torch.randn(M, N, generator=g, device="cuda").to(DT[c["out"]])  # a buffer in use
    return c


# ----------------------------------------------------------- the plain forms

def _values(codes):
    return codes.float() if codes.dtype == torch.int8 else codes.view(F8).float()


def _act(v, act):
    if act == "relu":
        return v.clamp(min=0.0)
    if act == "gelu":
        return 0.5 * v * (1.0 + torch.erf(v * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * v * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (v + 0.044715 * v * v * v)))
    if act == "silu":
        return v / (1.0 + torch.exp(-v))
    return v


def _plain_quant(s):
    most = 127.0 if s["type"] == "s8" else 448.0
    x = s["x"].float()
    top = x.abs().amax(1, keepdim=True)
    none = top < 2.0 ** -100
    scale = torch.where(none, 1.0, top / torch.full_like(top, most))
    v = torch.where(none, 0.0, x * (torch.ones_like(scale) / scale)).clamp(-most, most)
    q = v.round().to(torch.int8) if s["type"] == "s8" else (v + 0.0).to(F8)
    out = torch.zeros(x.shape[0], s["ld"], dtype=torch.uint8, device="cuda").view(q.dtype)
    out[:, :s["cols"]] = q
    return {"q": out, "scale": scale[:, 0]}


def _plain_linear(s):
    v = _values(s["x"]) @ _values(s["w"]).T * (s["x_scale"][:, None] * s["w_scale"])
    if s["b"] is not None:
        v = v + s["b"]
    v = _act(v, s["act"])
    if s["r"] is not None:
        v = v + s["r"].float()
    return v.to(DT[s["out"]])


def _plain_grouped(s):
    # rows into a block of equal height for each expert, one batched product, rows back out
    E, K, T, most, e = s["E"], s["K"], s["T"], s["most"], s["expert"]
    at = torch.arange(T, device="cuda") - s["offsets"].long()[e]
    blocks = torch.zeros(E, most, K, device="cuda")
    blocks[e, at] = _values(s["x"][:T])
    v = torch.bmm(_values(s["w"]), blocks.transpose(1, 2).contiguous())[e, :, at]
    v = v * (s["x_scale"][:T, None] * s["w_scale"][e])
    if s["b"] is not None:
        v = v + s["b"][e]
    v = _act(v, s["act"])
    if s["r"] is not None:
        v = v + s["r"][:T].float()
    s["y"][:T] = v.to(DT[s["out"]])
    return s["y"]


def _plain_logprobs(s):
    x, tokens, K, k = s["logits"].float(), s["tokens"].long(), s["K"], s["top"]
    m = x.amax(1, keepdim=True)
    m = torch.where(torch.isinf(m), 0.0, m)
    d = x - m
    e = torch.exp(d)
    z = e.sum(1)
    lz = torch.log(z)
    entropy = torch.where(z > 0, lz - torch.where(e > 0, e * d, 0.0).sum(1) / z, 0.0)
    given = d.gather(1, tokens.clamp(min=0)[:, None])[:, 0]
    logprob = torch.where(tokens < 0, 0.0, torch.where(torch.isinf(given), given, given - lz))
    out = {"logprob": logprob, "entropy": entropy}
    if k:
        bits = (x + 0.0).view(torch.int32)
        order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()  # as the values are ordered
        key = order * (1 << 32) + (K - 1 - torch.arange(K, device="cuda"))  # ties: the lowest index
        idx = K - 1 - (key.topk(k, 1).values & 0xFFFFFFFF)
        t = d.gather(1, idx)
        out |= {"top_idx": idx.to(torch.int32), "top_logprob": torch.where(torch.isinf(t), t, t - lz[:, None])}
    return out


def run(s):
    if not own:
        return {"quant": _plain_quant, "linear": _plain_linear, "grouped": _plain_grouped,
                "logprobs": _plain_logprobs}[s["op"]](s)
    from dlq_amd import ops
    if s["op"] == "quant":
        f = ops.quantize_rows_dyn_s8 if s["type"] == "s8" else ops.quantize_rows_dyn_f8
        q, scale = f(s["x"], ld=s["ld"])
        return {"q": q if s["type"] == "s8" else q.view(F8), "scale": scale}
    if s["op"] == "linear":
        f = ops.linear_act_s8 if s["type"] == "s8" else ops.linear_act_f8
        return f(s["x"], s["w"], s["x_scale"], s["w_scale"], bias=s["b"], act=s["act"], residual=s["r"],
                 out_dtype=DT[s["out"]])
    if s["op"] == "grouped":
        f = ops.linear_grouped_s8 if s["type"] == "s8" else ops.linear_grouped_f8
        return f(s["x"], s["offsets"], s["w"], s["x_scale"], s["w_scale"], bias=s["b"], act=s["act"],
                 residual=s["r"], out=s["y"])
    r = ops.logprobs(s["logits"], s["tokens"], top=s["top"])
    out = {"logprob": r.logprob, "entropy": r.entropy}
    if s["top"]:
        out |= {"top_idx": r.top_idx, "top_logprob": r.top_logprob}
    return out


# ----------------------------------------------------------------- the work

def work(case):
    c = case
    if c["op"] == "quant":
        n = c["rows"] * c["cols"]
        return {"bytes": n * DT[c["x"]].itemsize + c["rows"] * (c["ld"] + 4), "flops": 2 * n}
    if c["op"] == "logprobs":
        n = c["rows"] * c["K"]
        return {"bytes": n * DT[c["x"]].itemsize + c["rows"] * (12 + 8 * c["top"]), "flops": 4 * n}
    M, E = (c["M"], 1) if c["op"] == "linear" else (c["T"], min(c["E"], c["T"]))
    N, K, o = c["N"], c["K"], DT[c["out"]].itemsize
    b = M * K + E * N * K + M * N * o * (2 if c["residual"] else 1) + 4 * M + 4 * E * N * (2 if c["bias"] else 1)
    return {"bytes": b, "flops": 2 * M * N * K}


# ------------------------------------------------------ the answer in 64 bits

def _epilogue64(s, acc, xs, ws, b, r):
    v = acc * xs.double()[:, None] * ws.double()
    if b is not None:
        v += b.double()
    if s["act"] == "relu":
        v = torch.relu(v)
    elif s["act"] == "gelu":
        v = torch.special.ndtr(v) * v
    elif s["act"] == "gelu_tanh":
        v = v * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (v + 0.044715 * v ** 3))
    elif s["act"] == "silu":
        v = v * torch.sigmoid(v)
    return v if r is None else v + r.double()


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "quant":
        most = 127.0 if s["type"] == "s8" else 448.0
        x = s["x"].double()
        scale = x.abs().amax(1) / most
        if s["type"] == "s8":
            return {"q": None, "scale": scale}  # whole numbers
        q = torch.zeros(x.shape[0], s["ld"], dtype=torch.float64, device="cuda")
        q[:, :s["cols"]] = (x / scale[:, None]).float().clamp(-448, 448).to(F8).double()
        return {"q": q, "scale": scale}
    if s["op"] == "logprobs":
        x = s["logits"].double()
        lp = x - torch.logsumexp(x, 1, keepdim=True)
        none = torch.isneginf(x).all(1)
        lp[none] = -math.inf
        tokens = s["tokens"].long()
        logprob = lp.gather(1, tokens.clamp(min=0)[:, None])[:, 0]
        out = {"logprob": logprob.masked_fill(tokens < 0, 0.0), "entropy": torch.special.entr(lp.exp()).sum(1)}
        if s["top"]:
            out |= {"top_idx": None, "top_logprob": lp.sort(1, descending=True).values[:, :s["top"]].contiguous()}
        return out
    x = (s["x"].double() if s["type"] == "s8" else s["x"].view(F8).double())
    w = (s["w"].double() if s["type"] == "s8" else s["w"].view(F8).double())
    if s["op"] == "linear":
        return _epilogue64(s, x @ w.T, s["x_scale"], s["w_scale"], s["b"], s["r"])
    y, at = s["y"].double(), s["offsets"].tolist()
    for e in range(s["E"]):
        lo, hi = at[e], at[e + 1]
        if lo < hi:
            y[lo:hi] = _epilogue64(s, x[lo:hi] @ w[e].T, s["x_scale"][lo:hi], s["w_scale"][e],
                                   None if s["b"] is None else s["b"][e], None if s["r"] is None else s["r"][lo:hi])
    return y
