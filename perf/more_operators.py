"""Cases of the attention operators over an 8-bit paged cache: what is measured, and their plain forms.

The operators are the path between the product that makes queries, keys and values and the product that takes
attention's output: the norm of each head with the position's rotation and its backward pass, the cache's write
(keys normed and rotated, keys and values to e4m3 with one scale per token and head, the queries in the same
pass) and read, and attention of new tokens over the cache's pages.

``run`` takes what ``prepare`` gives.  With ``own`` false it computes the plain form in elementary torch
operations in 32 bits; with ``own`` true it makes the calls of the library's device object (mag_b200.Device),
writing into the buffers that a user's program keeps.
"""
import math
import os
import random
import sys

import torch

own = False

EPS = 1e-6
E4M3_MAX = 448.0
#: The smallest largest magnitude that a row's scale is formed from: below it the row is zeros.
E4M3_TINY = 2.0 ** -100

_device = None


def _library():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    path = os.path.join(root, "magnetron-pre-oss-release-old_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import mag_b200
    return mag_b200


def _dev():
    """The library's device object, made at the first call."""
    global _device
    if _device is None:
        _device = _library().Device()
    return _device


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # five tokens of a small fine-tuning step, a fifth of whose width is rotated in neighbouring pairs
        {"name": "heads_5x12x80", "op": "heads", "rows": 5, "heads": 12, "dim": 80, "rot": 16, "pairs": True, "norm": True},
        # the queries of a training batch of 8191 tokens, the whole head rotated
        {"name": "heads_8191x32x128", "op": "heads", "rows": 8191, "heads": 32, "dim": 128, "rot": 128, "pairs": False, "norm": True},
        # the keys' gradient of a ragged batch, half of each head rotated
        {"name": "heads_backward_777x8x64", "op": "heads_backward", "rows": 777, "heads": 8, "dim": 64, "rot": 32, "pairs": False, "norm": True},
        # the queries' gradient of a training batch
        {"name": "heads_backward_8191x32x128", "op": "heads_backward", "rows": 8191, "heads": 32, "dim": 128, "rot": 128, "pairs": False, "norm": True},
        # eight sequences that each take one more token: latency
        {"name": "write_8_of_32+8x128", "op": "write", "rows": 8, "q_heads": 32, "heads": 8, "dim": 128, "page": 16, "rot": 128, "pairs": False, "norm": True},
        # a prompt batch of 8191 tokens without norms
        {"name": "write_8191_of_40+8x128", "op": "write", "rows": 8191, "q_heads": 40, "heads": 8, "dim": 128, "page": 64, "rot": 128, "pairs": False, "norm": False},
        # a short prefix taken out of the cache
        {"name": "read_300x2x96", "op": "read", "rows": 300, "heads": 2, "dim": 96, "page": 16},
        # a long conversation taken out of the cache
        {"name": "read_65000x8x128", "op": "read", "rows": 65000, "heads": 8, "dim": 128, "page": 64},
        # four sequences of different lengths that each take one more token: latency
        {"name": "decode_4x2000", "op": "attention", "seqs": 4, "new": 1, "length": 2000, "q_heads": 32, "heads": 8, "dim": 128, "page": 16, "window": 0},
        # a full server: 64 sequences of up to 16000 tokens
        {"name": "decode_64x16000", "op": "attention", "seqs": 64, "new": 1, "length": 16000, "q_heads": 32, "heads": 8, "dim": 128, "page": 64, "window": 0},
        # chunks of up to 300 new tokens of three long documents, five queries to a key, an odd head
        {"name": "chunk_3x300_20000", "op": "attention", "seqs": 3, "new": 300, "length": 20000, "q_heads": 20, "heads": 4, "dim": 96, "page": 32, "window": 0},
        # four prompts of different lengths, up to 4100 tokens, from the first token on
        {"name": "prompt_4x4100", "op": "attention", "seqs": 4, "new": 4100, "length": 4100, "q_heads": 32, "heads": 8, "dim": 128, "page": 128, "window": 0},
    ]


def _log_between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["heads", "heads_backward", "write", "read", "attention", "attention", "attention"])
    dim = rng.choice([64, 80, 96, 112, 128, 128])
    page = rng.choice([16, 32, 64, 128])
    if op == "read":
        return {"op": op, "rows": _log_between(rng, 1, 65000), "heads": rng.randint(1, 8), "dim": dim, "page": page}
    if op != "attention":
        c = {"op": op, "rows": _log_between(rng, 1, 8191), "heads": rng.randint(1, 32) if op != "write" else rng.randint(1, 8), "dim": dim}
        if op == "write":
            c.update(q_heads=c["heads"] * rng.randint(1, 5), page=page)
        c.update(rot=rng.choice([dim, dim, dim // 16 * 8, 16]), pairs=rng.random() < 0.4, norm=rng.random() < 0.7)
        return c
    heads, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 5, 7, 8, 8, 12, 16])
    c = {"op": op, "seqs": _log_between(rng, 1, 64), "new": 1, "length": _log_between(rng, 1, 40000),
         "q_heads": heads * group, "heads": heads, "dim": dim, "page": page, "window": 0}
    if rng.random() < 0.6:  # several new tokens
        c["seqs"] = _log_between(rng, 1, 16)
        c["new"] = _log_between(rng, 2, 4100)
        c["length"] = max(c["new"], c["length"])
    if rng.random() < 0.25:
        c["window"] = _log_between(rng, 16, 8192)
    full = {k.get("name"): work(k) for k in listed()}
    while True:  # no more than the largest listed cases
        w = work(c)
        if w["bytes"] <= full["decode_64x16000"]["bytes"] and w["flops"] <= full["prompt_4x4100"]["flops"] \
                and c["seqs"] * c["new"] * c["q_heads"] <= 16400 * 32 and c["seqs"] * c["length"] * c["heads"] <= 64 * 16000 * 8 \
                and c["seqs"] * c["new"] * c["length"] * c["q_heads"] <= 4 * 4100 * 4100 * 32:
            return c
        if c["seqs"] > 1:
            c["seqs"] = max(1, c["seqs"] // 2)
        else:
            c["new"] = max(1, c["new"] // 2)
            c["length"] = max(c["new"], c["length"] // 2)


def _sequences(case):
    """New tokens and cached tokens (the new ones among them) of each sequence: the case's own, the same for every seed."""
    r = random.Random(1000003 * case["seqs"] + 1009 * case["length"] + case["new"])
    out = []
    for i in range(case["seqs"]):
        share = 1.0 if i == 0 else r.uniform(0.25, 1.0)
        new = max(1, round(case["new"] * share))
        length = new if case["length"] == case["new"] else max(new, round(case["length"] * (1.0 if i == 0 else r.uniform(0.25, 1.0))))
        out.append((new, length))
    return out


def _seen(new, length, window):
    """Pairs of a new token and a cached one that it sees, and the cached tokens that any sees."""
    lo = [max(0, length - new + i + 1 - window) if window else 0 for i in range(new)]
    return sum(length - new + i + 1 - lo[i] for i in range(new)), length - lo[0]


def work(case):
    op = case["op"]
    if op == "attention":
        group, d = case["q_heads"] // case["heads"], case["dim"]
        pairs = keys = rows = 0
        for new, length in _sequences(case):
            p, k = _seen(new, length, case["window"])
            pairs, keys, rows = pairs + p, keys + k, rows + new
        return {"bytes": keys * case["heads"] * (2 * d + 8) + rows * case["q_heads"] * (8 * d + 4),
                "flops": 4 * d * pairs * case["heads"] * group}
    n = case["rows"] * case["heads"] * case["dim"]
    if op == "read":
        return {"bytes": 2 * 5 * n + 8 * case["rows"] * case["heads"] + 4 * case["rows"], "flops": 2 * n}
    if op == "write":
        q = case["rows"] * case["q_heads"] * case["dim"]
        return {"bytes": 8 * q + 2 * 5 * n + 8 * case["rows"] * case["heads"] + 8 * case["rows"], "flops": 8 * (q + 2 * n)}
    stat = 4 * case["rows"] * case["heads"] if case["norm"] else 0
    if op == "heads":
        return {"bytes": 8 * n + stat + 4 * case["rows"], "flops": 8 * n}
    return {"bytes": (12 if case["norm"] else 8) * n + stat + 4 * case["rows"], "flops": 14 * n}


# ---------------------------------------------------------------- inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def _frequencies(rot):
    """Angles a position turns each pair by: f32, slower from pair to pair."""
    return torch.tensor([500000.0 ** (-2.0 * i / max(rot, 1)) for i in range(rot // 2)], dtype=torch.float32, device="cuda")


def _cache(g, pages, heads, page, dim):
    """A cache in use: e4m3 values of rows in which some columns are larger, and each row's scale."""
    out = []
    for kind in range(2):
        q = torch.empty(pages, heads, page, dim, dtype=torch.float8_e4m3fn, device="cuda")
        step = max(1, (1 << 26) // (heads * page * dim))
        for i in range(0, pages, step):
            v = _normal(g, min(step, pages - i), heads, page, dim).mul_(110.0).clamp_(-E4M3_MAX, E4M3_MAX)
            q[i:i + step] = v.to(torch.float8_e4m3fn)
        out += [q, torch.exp(_normal(g, pages, heads, page) * 0.3) * (1.0 / 110.0)]
    return out


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

    def whole(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    h, d = case["heads"], case["dim"]
    if op == "attention":
        page, seqs = case["page"], _sequences(case)
        s["sequences"] = seqs
        need = [-(-length // page) for _, length in seqs]
        pages = sum(need) + 3
        order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
        s["table"] = torch.full((len(seqs), max(need)), -1, dtype=torch.int32, device="cuda")
        at = 0
        for i, n in enumerate(need):
            s["table"][i, :n] = order[at:at + n]
            at += n
        s["start"] = whole([sum(n for n, _ in seqs[:i]) for i in range(len(seqs) + 1)])
        s["lengths"] = whole([length for _, length in seqs])
        s["rows"] = sum(n for n, _ in seqs)
        s["k"], s["k_scale"], s["v"], s["v_scale"] = _cache(g, pages, h, page, d)
        # queries of logits a few wide
        s["q"] = _normal(g, s["rows"], case["q_heads"], d) * torch.exp(_normal(g, s["rows"], case["q_heads"], 1) * 0.4)
        s["scale"] = 1.5 / math.sqrt(d)
        s["out"], s["lse"] = empty(s["rows"], case["q_heads"], d), empty(s["rows"], case["q_heads"])
    else:
        r = case["rows"]
        if op in ("write", "read"):
            page = case["page"]
            pages = -(-r // page) + 2
            # slots as sequences leave them: whole pages in any order, the tokens within them in theirs
            order = torch.randperm(pages, device="cuda", generator=g)
            token = torch.arange(r, device="cuda")
            s["slot"] = (order[token // page] * page + token % page).to(torch.int32)
            s["k"], s["k_scale"], s["v"], s["v_scale"] = _cache(g, pages, h, page, d)
        if op == "read":
            s["k_out"], s["v_out"] = empty(r, h, d), empty(r, h, d)
        else:
            s["pos"] = torch.randint(0, 131072, (r,), device="cuda", generator=g).to(torch.int32)
            s["freq"] = _frequencies(case["rot"])
            wide = torch.exp(_normal(g, d) * 0.5)
            if op == "write":
                qh = case["q_heads"]
                # one row of a fused projection: queries, keys, values
                s["qkv"] = _normal(g, r, qh + 2 * h, d) * wide
                s["q_in"], s["k_in"], s["v_in"] = s["qkv"][:, :qh], s["qkv"][:, qh:qh + h], s["qkv"][:, qh + h:]
                s["q_w"], s["k_w"] = ((1.0 + 0.2 * _normal(g, d)) if case["norm"] else None for _ in range(2))
                s["q_out"] = empty(r, qh, d)
            else:
                s["x"] = _normal(g, r, h, d) * wide
                s["w"] = 1.0 + 0.2 * _normal(g, d) if case["norm"] else None
                if op == "heads":
                    s["y"], s["rstd"] = empty(r, h, d), empty(r, h) if case["norm"] else None
                else:
                    s["dy"] = _normal(g, r, h, d) * 1e-2
                    s["rstd"] = (1.0 / (s["x"].double().square().mean(2) + EPS).sqrt()).float() if case["norm"] else None
                    s["dx"], s["dw"] = empty(r, h, d), empty(d) if case["norm"] else None
    if own:
        mb = _library()
        if "k_scale" in s:
            s["cache"] = mb.KvCache(s["k"].data_ptr(), s["v"].data_ptr(), s["k_scale"].data_ptr(), s["v_scale"].data_ptr(),
                                    pages, h, d, case["page"])
        if "pos" in s:
            s["rotation"] = mb.Rotation(s["pos"].data_ptr(), s["freq"].data_ptr(), case["rot"], interleaved=case["pairs"])
    return s


# ---------------------------------------------------------------- the calls
def run(state):
    return (_own if own else _plain)(state)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _own(s):
    dev, op = _dev(), s["op"]
    if op == "heads":
        dev.rotate_heads(s["rows"], s["heads"], s["dim"], s["y"].data_ptr(), s["x"].data_ptr(), w=_ptr(s["w"]), eps=EPS,
                         rstd=_ptr(s["rstd"]), rotation=s["rotation"])
        return {"y": s["y"], "rstd": s["rstd"]} if s["norm"] else {"y": s["y"]}
    if op == "heads_backward":
        if not s["norm"]:
            dev.rotate_heads_backward(s["rows"], s["heads"], s["dim"], s["dx"].data_ptr(), None, s["dy"].data_ptr(),
                                      rotation=s["rotation"])
            return {"dx": s["dx"]}
        dev.rotate_heads_backward(s["rows"], s["heads"], s["dim"], s["dx"].data_ptr(), s["dw"].data_ptr(), s["dy"].data_ptr(),
                                  x=s["x"].data_ptr(), w=s["w"].data_ptr(), rstd=s["rstd"].data_ptr(), rotation=s["rotation"])
        return {"dx": s["dx"], "dw": s["dw"]}
    if op == "write":
        row = (s["q_heads"] + 2 * s["heads"]) * s["dim"]
        dev.kv_write(s["cache"], s["rows"], s["slot"].data_ptr(), s["k_in"].data_ptr(), s["v_in"].data_ptr(), k_w=_ptr(s["k_w"]),
                     q=s["q_in"].data_ptr(), q_out=s["q_out"].data_ptr(), q_heads=s["q_heads"], q_w=_ptr(s["q_w"]), eps=EPS,
                     rotation=s["rotation"], k_stride=row, v_stride=row, q_stride=row)
        return {n: s[n] for n in ("q_out", "k", "k_scale", "v", "v_scale")}
    if op == "read":
        dev.kv_read(s["cache"], s["rows"], s["slot"].data_ptr(), k=s["k_out"].data_ptr(), v=s["v_out"].data_ptr())
        return {"k_out": s["k_out"], "v_out": s["v_out"]}
    dev.attention_paged(s["cache"], s["rows"], s["q_heads"], s["out"].data_ptr(), s["q"].data_ptr(), s["table"].data_ptr(),
                        s["start"].data_ptr(), s["lengths"].data_ptr(), s["seqs"], s["table"].shape[1], max_new=s["new"],
                        scale=s["scale"], window=s["window"], lse=s["lse"].data_ptr())
    return {"out": s["out"], "lse": s["lse"]}


# ---------------------------------------------------------------- plain forms
def _plain_turn(v, s, back=False):
    """v [rows][heads][dim] turned by each row's position, or turned back."""
    rot = s["rot"]
    # the angle in 64 bits: a far position times an f32 frequency loses the turn's fraction in 32
    a = s["pos"].double()[:, None] * s["freq"].double()
    c, n = torch.cos(a).float()[:, None, :], torch.sin(a).float()[:, None, :]
    if back:
        n = -n
    p = v[..., :rot]
    x, y = (p[..., 0::2], p[..., 1::2]) if s["pairs"] else (p[..., :rot // 2], p[..., rot // 2:])
    u, w = x * c - y * n, y * c + x * n
    turned = torch.stack((u, w), -1).flatten(-2) if s["pairs"] else torch.cat((u, w), -1)
    return torch.cat((turned, v[..., rot:]), -1)


def _plain_norm(x, w):
    rstd = torch.rsqrt(x.square().mean(-1) + EPS)
    return x * rstd[..., None] * w, rstd


def _plain_e4m3(v):
    """Each row of v as e4m3 values and its scale."""
    scale = v.abs().amax(-1).clamp(min=E4M3_TINY) / E4M3_MAX
    return (v / scale[..., None]).to(torch.float8_e4m3fn), scale


def _plain_attention(s):
    page, h, d, group = s["page"], s["heads"], s["dim"], s["q_heads"] // s["heads"]
    out, lse = torch.empty_like(s["q"]), torch.empty(s["rows"], s["q_heads"], device="cuda")
    row = 0
    for i, (new, length) in enumerate(s["sequences"]):
        ids = s["table"][i, :-(-length // page)].long()

        def rows(q, scale):  # [heads][length][dim]
            v = q.view(torch.uint8)[ids].view(torch.float8_e4m3fn).float() * scale[ids][..., None]
            return v.transpose(0, 1).reshape(h, -1, d)[:, :length]

        k, v = rows(s["k"], s["k_scale"]), rows(s["v"], s["v_scale"])
        key = torch.arange(length, device="cuda")
        step = max(1, (1 << 29) // (s["q_heads"] * length))
        for a in range(0, new, step):
            b = min(new, a + step)
            q = s["q"][row + a:row + b].view(b - a, h, group, d).permute(1, 0, 2, 3).reshape(h, -1, d)
            x = (q @ k.transpose(1, 2) * s["scale"]).view(h, b - a, group, length)
            pos = torch.arange(length - new + a, length - new + b, device="cuda")[:, None]
            hidden = key > pos
            if s["window"]:
                hidden |= key <= pos - s["window"]
            x.masked_fill_(hidden[None, :, None, :], -math.inf)
            m = x.amax(-1, keepdim=True)
            e = torch.exp(x - m)
            total = e.sum(-1)
            o = (e.view(h, -1, length) @ v).view(h, b - a, group, d) / total[..., None]
            out[row + a:row + b] = o.permute(1, 0, 2, 3).reshape(b - a, -1, d)
            lse[row + a:row + b] = (m[..., 0] + torch.log(total)).permute(1, 0, 2).reshape(b - a, -1)
        row += new
    return {"out": out, "lse": lse}


def _plain(s):
    op = s["op"]
    if op == "attention":
        return _plain_attention(s)
    if op == "read":
        page, slot = s["page"], s["slot"].long()

        def rows(q, scale):
            at = slot // page, slice(None), slot % page
            return q.view(torch.uint8)[at].view(torch.float8_e4m3fn).float() * scale[at][..., None]

        return {"k_out": rows(s["k"], s["k_scale"]), "v_out": rows(s["v"], s["v_scale"])}
    if op == "write":
        q, k, v = s["q_in"], s["k_in"], s["v_in"]
        if s["norm"]:
            q, k = _plain_norm(q, s["q_w"])[0], _plain_norm(k, s["k_w"])[0]
        page, slot = s["page"], s["slot"].long()
        at = slot // page, slice(None), slot % page
        for name, x in (("k", _plain_turn(k, s)), ("v", v)):
            e, scale = _plain_e4m3(x)
            s[name].view(torch.uint8)[at] = e.view(torch.uint8)
            s[name + "_scale"][at] = scale
        return {"q_out": _plain_turn(q, s), **{n: s[n] for n in ("k", "k_scale", "v", "v_scale")}}
    if op == "heads":
        if not s["norm"]:
            return {"y": _plain_turn(s["x"], s)}
        v, rstd = _plain_norm(s["x"], s["w"])
        return {"y": _plain_turn(v, s), "rstd": rstd}
    u = _plain_turn(s["dy"], s, back=True)
    if not s["norm"]:
        return {"dx": u}
    x, rstd = s["x"], s["rstd"][..., None]
    g = u * s["w"]
    return {"dx": rstd * (g - x * (rstd * rstd * (g * x).mean(-1, keepdim=True))), "dw": (u * x * rstd).sum((0, 1))}


# ---------------------------------------------------------------- in 64 bits
def _exact_e4m3(v):
    """v rounded to the nearest e4m3 value, ties to even: 3 bits after the leading one, steps of 2^-9 below 2^-6."""
    _, e = torch.frexp(v)
    step = torch.ldexp(torch.ones_like(v), (e - 4).clamp(min=-9))
    return (torch.round(v / step) * step).clamp(-E4M3_MAX, E4M3_MAX)


def _exact_turns(s, sign):
    """cos + i sin of every row's angles, as complex numbers, one for each pair."""
    a = s["freq"].double()[None, :] * s["pos"].double()[:, None] * sign
    return torch.polar(torch.ones_like(a), a)[:, None, :]


def _exact_turn(v, s, sign=1.0):
    half, out = s["rot"] // 2, v.clone()
    first = slice(0, s["rot"], 2) if s["pairs"] else slice(0, half)
    second = slice(1, s["rot"], 2) if s["pairs"] else slice(half, s["rot"])
    z = torch.complex(v[:, :, first].contiguous(), v[:, :, second].contiguous()) * _exact_turns(s, sign)
    out[:, :, first], out[:, :, second] = z.real, z.imag
    return out


def _exact_unit(x, w):
    root = ((x * x).sum(-1) / x.shape[-1] + EPS).sqrt()
    return x / root[..., None] * w.double(), 1.0 / root


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    h, d = case["heads"], case["dim"]
    if op == "heads":
        v, rstd = s["x"].double(), None
        if case["norm"]:
            v, rstd = _exact_unit(v, s["w"])
        y = {"y": _exact_turn(v, s)}
        return {**y, "rstd": rstd} if case["norm"] else y
    if op == "heads_backward":
        u = _exact_turn(s["dy"].double(), s, -1.0)
        if not case["norm"]:
            return {"dx": u}
        rstd = s["rstd"].double()[..., None]
        n = s["x"].double() * rstd
        along = torch.einsum("rhd,rhd,d->rh", u, n, s["w"].double())[..., None] / d
        return {"dx": rstd * (u * s["w"].double() - n * along), "dw": torch.einsum("rhd,rhd->d", u, n)}
    if op == "read":
        out = {}
        flat = (s["slot"].long() // case["page"])[:, None] * (h * case["page"]) + torch.arange(h, device="cuda") * case["page"] \
            + (s["slot"].long() % case["page"])[:, None]
        for n in ("k", "v"):
            out[n + "_out"] = s[n].view(torch.uint8).view(-1, d)[flat].view(torch.float8_e4m3fn).double() \
                * s[n + "_scale"].view(-1)[flat].double()[..., None]
        return out
    if op == "write":
        q, k, v = (s[n].double() for n in ("q_in", "k_in", "v_in"))
        if case["norm"]:
            q, k = _exact_unit(q, s["q_w"])[0], _exact_unit(k, s["k_w"])[0]
        out = {"q_out": _exact_turn(q, s)}
        flat = (s["slot"].long() // case["page"])[:, None] * (h * case["page"]) + torch.arange(h, device="cuda") * case["page"] \
            + (s["slot"].long() % case["page"])[:, None]
        for n, x in (("k", _exact_turn(k, s)), ("v", v)):
            scale = x.abs().amax(-1).clamp(min=E4M3_TINY) / E4M3_MAX
            values, scales = s[n].double().view(-1, d), s[n + "_scale"].double().view(-1)
            values[flat.view(-1)] = _exact_e4m3(x / scale[..., None]).view(-1, d)
            scales[flat.view(-1)] = scale.view(-1)
            out[n], out[n + "_scale"] = values.view(s[n].shape), scales.view(s[n + "_scale"].shape)
        return {n: out[n] for n in ("q_out", "k", "k_scale", "v", "v_scale")}
    group, page = case["q_heads"] // h, case["page"]
    out = torch.empty(s["rows"], case["q_heads"], d, dtype=torch.float64, device="cuda")
    lse = torch.empty(s["rows"], case["q_heads"], dtype=torch.float64, device="cuda")
    first = 0
    for i, (new, length) in enumerate(s["sequences"]):
        at = torch.arange(length, device="cuda")
        slot_page, slot_row = s["table"][i].long()[at // page], at % page
        for head in range(h):
            k, v = (s[n].view(torch.uint8)[slot_page, head, slot_row].view(torch.float8_e4m3fn).double()
                    * s[n + "_scale"][slot_page, head, slot_row].double()[:, None] for n in ("k", "v"))
            for g in range(head * group, (head + 1) * group):
                step = max(1, (1 << 27) // length)
                for a in range(0, new, step):
                    rows = slice(first + a, first + min(new, a + step))
                    x = torch.mm(s["q"][rows, g].double() * s["scale"], k.t())
                    back = (length - new + a + torch.arange(x.shape[0], device="cuda"))[:, None] - at[None, :]
                    seen = (back >= 0) & (back < case["window"]) if case["window"] else back >= 0
                    x = torch.where(seen, x, torch.full_like(x, -math.inf))
                    z = torch.logsumexp(x, 1)
                    out[rows, g] = torch.mm(torch.exp(x - z[:, None]), v)
                    lse[rows, g] = z
        first += new
    return {"out": out, "lse": lse}
