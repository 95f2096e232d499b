"""Cases of the language-model row operators: what is measured, and their plain forms.

The operators are the path of an 8-bit linear layer and its two ends: the root-mean-square norm
with the residual's addition and its backward pass, the e4m3 quantiser of weights and gradients,
the product of e4m3 operands with one scale per 128 elements of K, and the log probabilities of
given tokens with entropy, the best alternatives and the gradient.

``run`` takes what ``prepare`` gives.  With ``own`` false it computes the plain form in elementary
torch operations in 32 bits; with ``own`` true it makes the calls of the library's device object
(mag_b200.Device), writing into the buffers that a user's program keeps.
"""
import math
import os
import sys

import torch

own = False

EPS = 1e-6
E4M3_MAX = 448.0
#: The smallest largest magnitude that a group's scale is formed from: below it the group is zeros.
E4M3_TINY = 2.0 ** -100

_device = None


def _dev():
    """The library's device object, made at the first call."""
    global _device
    if _device is None:
        root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        sys.path.insert(0, os.path.join(root, "magnetron-pre-oss-release-old_b200"))
        import mag_b200
        _device = mag_b200.Device()
    return _device


def _up(n, a=128):
    return -(-n // a) * a


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # eight sequences that each take one more token: one norm of a 4096-wide model, latency
        {"name": "norm_8x4096", "op": "norm", "rows": 8, "cols": 4096},
        # a prompt batch of 8192 tokens in an 8192-wide model
        {"name": "norm_8192x8192", "op": "norm", "rows": 8192, "cols": 8192},
        # training, a ragged batch and a width that is no multiple of 128
        {"name": "norm_backward_4099x5000", "op": "norm_backward", "rows": 4099, "cols": 5000},
        # a weight stored as the framework's product reads it ([K][N]), laid out once for the 8-bit product
        {"name": "quantize_weight_8192x4096", "op": "quantize", "rows": 8192, "cols": 4096, "block": True, "transpose": True},
        # a gradient turned for the weight's gradient, tokens along the groups, ragged
        {"name": "quantize_turned_2500x4100", "op": "quantize", "rows": 2500, "cols": 4100, "block": False, "transpose": True},
        # four tokens through a square layer
        {"name": "product_4x4096x4096", "op": "product", "m": 4, "k": 4096, "n": 4096, "block": True},
        # a batch of decoded tokens, or a short ragged prompt, through a wide layer
        {"name": "product_100x4096x14336", "op": "product", "m": 100, "k": 4096, "n": 14336, "block": True},
        # a prompt batch through a large square layer
        {"name": "product_8192x8192x8192", "op": "product", "m": 8192, "k": 8192, "n": 8192, "block": True},
        # a weight's gradient: both operands scaled along the tokens, ragged
        {"name": "product_rows_4100x2500x4000", "op": "product", "m": 4100, "k": 2500, "n": 4000, "block": False},
        # four sampled tokens over a large vocabulary, with their best alternatives: latency
        {"name": "logprobs_4x131072", "op": "logprobs", "rows": 4, "cols": 131072, "top": 20},
        # scoring a batch of answers over a vocabulary that is no multiple of four
        {"name": "logprobs_4095x100003", "op": "logprobs", "rows": 4095, "cols": 100003, "top": 8},
        # the loss's gradient over a vocabulary in padded rows
        {"name": "logprobs_backward_2048x65600", "op": "logprobs_backward", "rows": 2048, "cols": 65600},
    ]


def _log_between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "norm_backward", "quantize", "product", "product", "logprobs", "logprobs_backward"])
    if op in ("norm", "norm_backward"):
        return {"op": op, "rows": _log_between(rng, 1, 8192), "cols": _log_between(rng, 100, 8192)}
    if op == "quantize":
        return {"op": op, "rows": _log_between(rng, 1, 8192), "cols": _log_between(rng, 100, 8192),
                "block": rng.random() < 0.5, "transpose": rng.random() < 0.5}
    if op == "product":
        return {"op": op, "m": _log_between(rng, 1, 8192), "k": _log_between(rng, 200, 8192),
                "n": _log_between(rng, 200, 8192), "block": rng.random() < 0.6}
    if op == "logprobs":
        return {"op": op, "rows": _log_between(rng, 1, 2048), "cols": _log_between(rng, 1000, 160000),
                "top": rng.choice([0, 1, 5, 20, 32])}
    return {"op": op, "rows": _log_between(rng, 1, 1024), "cols": _log_between(rng, 1000, 100000)}


def work(case):
    op = case["op"]
    if op == "product":
        m, k, n = case["m"], case["k"], case["n"]
        g = _up(k) // 128
        scales = m * g + (_up(n) // 128 if case["block"] else n) * g
        return {"bytes": m * k + n * k + 4 * m * n + 4 * scales, "flops": 2 * m * n * k}
    r, c = case["rows"], case["cols"]
    if op == "norm":  # x, residual and weight in; sum, 8-bit rows, scales and reciprocal roots out
        return {"bytes": 13 * r * c + 4 * c + 4 * r * (_up(c) // 128) + 4 * r, "flops": 8 * r * c}
    if op == "norm_backward":  # dy, sum and the residual's gradient in; dx out
        return {"bytes": 16 * r * c + 8 * c + 4 * r, "flops": 10 * r * c}
    if op == "quantize":
        a, b = (c, r) if case["transpose"] else (r, c)
        groups = (_up(a) // 128 if case["block"] else a) * (_up(b) // 128)
        return {"bytes": 5 * r * c + 4 * groups, "flops": 3 * r * c}
    if op == "logprobs":
        return {"bytes": 4 * r * c + (16 + 8 * case["top"]) * r, "flops": 8 * r * c}
    return {"bytes": 8 * r * c + 20 * r, "flops": 8 * r * c}


# ---------------------------------------------------------------- inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def _operand(g, rows, cols, block):
    """An e4m3 operand as a user keeps it: rows of a multiple of 128 bytes, zero past cols, and its scales."""
    v = _normal(g, rows, cols).mul_(110.0).clamp_(-E4M3_MAX, E4M3_MAX)
    q = torch.zeros(rows, _up(cols), dtype=torch.uint8, device="cuda")
    q[:, :cols] = v.to(torch.float8_e4m3fn).view(torch.uint8)
    n = _up(rows) // 128 if block else rows
    s = torch.exp(_normal(g, n, _up(cols) // 128) * 0.3) * (0.02 / 110.0)
    return q, s


def prepare(case, seed):
    if own and torch.cuda.current_stream().cuda_stream != _dev().stream:
        # The memory is torch's: from here on torch works on the library's stream, as in a program that has both, so
        # that a call follows what torch still writes and torch's next work follows the call.
        stream = torch.cuda.ExternalStream(_dev().stream, device=f"cuda:{_dev().ordinal}")
        stream.wait_stream(torch.cuda.current_stream())
        torch.cuda.set_stream(stream)
    g = _generator(seed)
    op = case["op"]
    s = dict(case)

    def empty(*shape, dtype=torch.float32):
        return torch.empty(*shape, dtype=dtype, device="cuda")

    if op == "product":
        m, k, n = case["m"], case["k"], case["n"]
        s["xq"], s["xs"] = _operand(g, m, k, False)
        s["yq"], s["ys"] = _operand(g, n, k, case["block"])
        s["r"] = empty(m, n)
        return s
    r, c = case["rows"], case["cols"]
    if op == "norm":
        # a residual stream: some columns are far larger than the others
        s["x"], s["res"] = _normal(g, r, c), _normal(g, r, c) * torch.exp(_normal(g, c) * 0.8)
        s["w"] = 1.0 + 0.2 * _normal(g, c)
        s["h"], s["q_scale"], s["rstd"] = empty(r, c), empty(r, _up(c) // 128), empty(r)
        s["q"] = empty(r, _up(c), dtype=torch.float8_e4m3fn)
        s["q_cols"] = s["q"][:, :c]  # without the padding of each row
    elif op == "norm_backward":
        s["h"], s["dy"], s["dh"] = _normal(g, r, c) * torch.exp(_normal(g, c) * 0.8), _normal(g, r, c) * 1e-2, _normal(g, r, c) * 1e-2
        s["w"] = 1.0 + 0.2 * _normal(g, c)
        s["rstd"] = 1.0 / (s["h"].double().square().mean(1) + EPS).sqrt()
        s["rstd"] = s["rstd"].float()
        s["dx"], s["dw"] = empty(r, c), empty(c)
    elif op == "quantize":
        s["x"] = _normal(g, r, c) * torch.exp(_normal(g, r, 1)) * 0.02
        a, b = (c, r) if case["transpose"] else (r, c)
        s["q"] = empty(a, _up(b), dtype=torch.float8_e4m3fn)
        s["q_cols"] = s["q"][:, :b]
        s["q_scale"] = empty(_up(a) // 128 if case["block"] else a, _up(b) // 128)
    else:
        # logits: a bell of width 2.5 and a few likely tokens in each row
        s["x"] = _normal(g, r, c).mul_(2.5)
        like = torch.randint(0, c, (r, 8), device="cuda", generator=g)
        s["x"].scatter_add_(1, like, 6.0 + 4.0 * _normal(g, r, 8).abs())
        s["id"] = torch.where(torch.rand(r, device="cuda", generator=g) < 0.7, like[:, 0],
                              torch.randint(0, c, (r,), device="cuda", generator=g)).to(torch.int32)
        if op == "logprobs":
            s["logp"], s["lse"], s["entropy"] = empty(r), empty(r), empty(r)
            s["top_logp"], s["top_id"] = empty(r, case["top"]), empty(r, case["top"], dtype=torch.int32)
        else:
            x = s["x"]
            lse, ent = [], []
            for i in range(0, r, 256):  # as the forward pass left them
                b = x[i:i + 256].double()
                z = torch.logsumexp(b, 1)
                lse.append(z.float())
                ent.append((z - (torch.exp(b - z[:, None]) * b).sum(1)).float())
            s["lse"], s["entropy"] = torch.cat(lse), torch.cat(ent)
            s["g_logp"], s["g_entropy"] = _normal(g, r) / r, _normal(g, r) * (0.01 / r)
            s["dx"] = empty(r, c)
    return s


# ---------------------------------------------------------------- the calls
def run(state):
    return (_own if own else _plain)(state)


def _own(s):
    d, op = _dev(), s["op"]
    if op == "norm":
        r, c = s["rows"], s["cols"]
        d.rmsnorm_rows(r, c, s["x"].data_ptr(), s["w"].data_ptr(), EPS, residual=s["res"].data_ptr(),
                       h=s["h"].data_ptr(), q=s["q"].data_ptr(), q_scale=s["q_scale"].data_ptr(),
                       rstd=s["rstd"].data_ptr())
        return {"h": s["h"], "q": s["q_cols"], "q_scale": s["q_scale"], "rstd": s["rstd"]}
    if op == "norm_backward":
        d.rmsnorm_rows_backward(s["rows"], s["cols"], s["dx"].data_ptr(), s["dw"].data_ptr(), s["dy"].data_ptr(),
                                s["h"].data_ptr(), s["w"].data_ptr(), s["rstd"].data_ptr(), dh=s["dh"].data_ptr())
        return {"dx": s["dx"], "dw": s["dw"]}
    if op == "quantize":
        d.quantize_e4m3(s["rows"], s["cols"], s["x"].data_ptr(), s["q"].data_ptr(), s["q_scale"].data_ptr(),
                        block=s["block"], transpose=s["transpose"])
        return {"q": s["q_cols"], "q_scale": s["q_scale"]}
    if op == "product":
        d.matmul_e4m3(s["m"], s["k"], s["n"], s["r"].data_ptr(), s["xq"].data_ptr(), s["xs"].data_ptr(),
                      s["yq"].data_ptr(), s["ys"].data_ptr(), y_block=s["block"])
        return {"r": s["r"]}
    if op == "logprobs":
        d.token_logprobs(s["rows"], s["cols"], s["x"].data_ptr(), s["id"].data_ptr(), logp=s["logp"].data_ptr(),
                         lse=s["lse"].data_ptr(), entropy=s["entropy"].data_ptr(), top=s["top"],
                         top_logp=s["top_logp"].data_ptr(), top_id=s["top_id"].data_ptr())
        return {n: s[n] for n in ("logp", "lse", "entropy", "top_logp", "top_id")}
    d.token_logprobs_backward(s["rows"], s["cols"], s["dx"].data_ptr(), s["x"].data_ptr(), s["id"].data_ptr(),
                              s["lse"].data_ptr(), s["entropy"].data_ptr(), s["g_logp"].data_ptr(),
                              s["g_entropy"].data_ptr())
    return {"dx": s["dx"]}


# ---------------------------------------------------------------- plain forms
def _plain_quantize(x, block):
    """Rows of x as e4m3 with one scale per 128 columns (and per 128 rows): values and scales."""
    r, c = x.shape
    p = torch.nn.functional.pad(x, (0, _up(c) - c, 0, _up(r) - r if block else 0))
    t = p.view(p.shape[0] // 128 if block else r, 128 if block else 1, _up(c) // 128, 128)
    scale = t.abs().amax((1, 3)).clamp(min=E4M3_TINY) / E4M3_MAX
    q = (t / scale[:, None, :, None]).to(torch.float8_e4m3fn).view(p.shape)
    return q.view(torch.uint8)[:r, :c].view(torch.float8_e4m3fn), scale


def _plain_scaled(q, scale, cols, block):
    """The f32 values that an e4m3 operand stands for."""
    rows = q.shape[0]
    s = scale.repeat_interleave(128, 0)[:rows] if block else scale
    return (q.view(torch.float8_e4m3fn).float().view(rows, -1, 128) * s[:, :, None]).view(rows, -1)[:, :cols]


def _plain(s):
    op = s["op"]
    if op == "norm":
        h = s["x"] + s["res"]
        rstd = torch.rsqrt(h.square().mean(1) + EPS)
        q, scale = _plain_quantize(h * rstd[:, None] * s["w"], False)
        return {"h": h, "q": q, "q_scale": scale, "rstd": rstd}
    if op == "norm_backward":
        h, rstd = s["h"], s["rstd"][:, None]
        u = s["dy"] * s["w"]
        c = rstd * rstd * (u * h).mean(1, keepdim=True)
        return {"dx": s["dh"] + rstd * (u - h * c), "dw": (s["dy"] * h * rstd).sum(0)}
    if op == "quantize":
        x = s["x"].t().contiguous() if s["transpose"] else s["x"]
        q, scale = _plain_quantize(x, s["block"])
        return {"q": q, "q_scale": scale}
    if op == "product":
        x = _plain_scaled(s["xq"], s["xs"], s["k"], False)
        return {"r": x @ _plain_scaled(s["yq"], s["ys"], s["k"], s["block"]).t()}
    x, rows = s["x"], torch.arange(s["rows"], device="cuda")
    if op == "logprobs":
        m = x.amax(1, keepdim=True)
        e = torch.exp(x - m)
        total = e.sum(1)
        lse = m[:, 0] + torch.log(total)
        entropy = torch.log(total) - (e * (x - m)).sum(1) / total
        # ties go to the lowest index: whole numbers in the order of (value, -index) are chosen from
        bits = (x + 0.0).view(torch.int32)
        key = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long() << 32
        key += torch.arange(s["cols"] - 1, -1, -1, device="cuda")
        ids = s["cols"] - 1 - (torch.topk(key, s["top"], 1).values & 0xFFFFFFFF)
        return {"logp": x[rows, s["id"].long()] - lse, "lse": lse, "entropy": entropy,
                "top_logp": x.gather(1, ids) - lse[:, None], "top_id": ids.to(torch.int32)}
    logp = x - s["lse"][:, None]
    p = torch.exp(logp)
    dx = -p * (s["g_logp"][:, None] + s["g_entropy"][:, None] * (logp + s["entropy"][:, None]))
    dx[rows, s["id"].long()] += s["g_logp"]
    return {"dx": dx}


# ---------------------------------------------------------------- in 64 bits
def _exact_e4m3(v):
    """v rounded to the nearest e4m3 value, ties to even: 3 bits after the leading one, steps of 2^-9 below 2^-6."""
    _, e = torch.frexp(v)
    step = torch.ldexp(torch.ones_like(v), (e - 4).clamp(min=-9))
    return (torch.round(v / step) * step).clamp(-E4M3_MAX, E4M3_MAX)


def _exact_groups(y, block):
    r, c = y.shape
    n, g = (_up(r) // 128 if block else r), _up(c) // 128
    top = torch.zeros(n, g, dtype=torch.float64, device="cuda")
    row = torch.arange(r, device="cuda") // (128 if block else 1)
    for j in range(g):
        top[:, j].index_reduce_(0, row, y[:, 128 * j:128 * (j + 1)].abs().amax(1), "amax")
    scale = top.clamp(min=E4M3_TINY) / E4M3_MAX
    q = torch.empty_like(y)
    for j in range(g):
        q[:, 128 * j:128 * (j + 1)] = _exact_e4m3(y[:, 128 * j:128 * (j + 1)] / scale[row, j, None])
    return q, scale


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        h = s["x"].double() + s["res"].double()
        root = ((h * h).sum(1) / case["cols"] + EPS).sqrt()
        q, scale = _exact_groups(h / root[:, None] * s["w"].double(), False)
        return {"h": h, "q": q, "q_scale": scale, "rstd": 1.0 / root}
    if op == "norm_backward":
        h, dy, w, rstd = (s[n].double() for n in ("h", "dy", "w", "rstd"))
        n = h * rstd[:, None]  # the normalised rows: their gradient loses its part along n
        along = (dy * w * n).sum(1) / case["cols"]
        return {"dx": s["dh"].double() + rstd[:, None] * (dy * w - n * along[:, None]), "dw": (dy * n).sum(0)}
    if op == "quantize":
        x = s["x"].double()
        q, scale = _exact_groups(x.t().contiguous() if case["transpose"] else x, case["block"])
        return {"q": q, "q_scale": scale}
    if op == "product":
        r = torch.zeros(case["m"], case["n"], dtype=torch.float64, device="cuda")
        nb = torch.arange(case["n"], device="cuda") // (128 if case["block"] else 1)
        for j in range(s["xs"].shape[1]):
            x = s["xq"][:, 128 * j:128 * (j + 1)].contiguous().view(torch.float8_e4m3fn).double()
            y = s["yq"][:, 128 * j:128 * (j + 1)].contiguous().view(torch.float8_e4m3fn).double()
            r += (x * s["xs"][:, j, None].double()) @ (y * s["ys"][nb, j, None].double()).t()
        return {"r": r}
    if op == "logprobs":
        outs = {n: [] for n in ("logp", "lse", "entropy", "top_logp")}
        k = case["top"]
        for i in range(0, case["rows"], 256):
            x = s["x"][i:i + 256].double()
            lse = torch.logsumexp(x, 1)
            p = torch.exp(x - lse[:, None])
            outs["logp"].append(x.gather(1, s["id"][i:i + 256, None].long())[:, 0] - lse)
            outs["lse"].append(lse)
            outs["entropy"].append(-(p * (x - lse[:, None])).sum(1))
            outs["top_logp"].append(torch.topk(x, k, 1).values - lse[:, None])
        # the ids are whole numbers: they have to be equal, and have no value in 64 bits
        return {**{n: torch.cat(v) for n, v in outs.items()}, "top_id": None}
    out = torch.empty(case["rows"], case["cols"], dtype=torch.float64, device="cuda")
    for i in range(0, case["rows"], 256):
        x, one = s["x"][i:i + 256].double(), slice(i, i + 256)
        logp = x - s["lse"][one, None].double()
        p = torch.exp(logp)
        hot = torch.zeros_like(p).scatter_(1, s["id"][one, None].long(), 1.0)
        out[one] = s["g_logp"][one, None].double() * (hot - p) - s["g_entropy"][one, None].double() * p * (
            logp + s["entropy"][one, None].double())
    return {"dx": out}
