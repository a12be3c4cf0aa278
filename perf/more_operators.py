"""Positions in a decoder's attention, and prompts that continue from its cache: what they are timed on.

A case is a dict of plain values; `op` names what one pass does:

  rotate  a packed batch's projection: each query and key head normed (where `norm` is true) and
          rotated by its token's position, the values as they are
  train   the same and its backward: the result, the projection's gradient and, with a norm, the
          gradients of its two weights
  append  new tokens of sequences that are in a paged cache already: their keys normed, rotated and
          written with the values, their queries normed and rotated for the attention that follows;
          the cache as it is then, or of an 8-bit one the new rows read back
  chunk   attention of those queries over the cache: each new token to its sequence up to itself

`lengths` are the sequences' new tokens as a text, "a,b,c", or "a*n" for n sequences of a; `context`
what each has in the cache before them.  Query, key and value heads are column blocks of one
projection [tokens, (heads + 2 kv_heads) * dh].

The norm of a head x is x / sqrt(mean(x^2) + eps) * weight.  The rotation takes the first `dims`
columns, angle i of dims / 2 being position * base^(-2 i / dims) in 64 bits: layout "halves" turns
columns (i, dims / 2 + i), "pairs" (2 i, 2 i + 1), (a, b) -> (a cos - b sin, a sin + b cos).  A
position is a token's place in its sequence, the cached ones included.

A cache of format "int8" holds a byte a value and a float32 scale for each token and head: scale =
max|x| / 127, code = round(x / scale) + 128, both in float32 with ties to even; the values' codes of
four neighbouring slots lie together.  Everything else is float32, the framework's only floating type.
"""
from __future__ import annotations

import ctypes
import math

import torch

own = False
EPS = 1e-6

# ---------------------------------------------------------------------------
# The cases
# ---------------------------------------------------------------------------


def listed():
    return [
        # A short turn of one conversation: latency.
        {"name": "rotate_64", "op": "rotate", "lengths": "64", "heads": 8, "kv_heads": 8, "dh": 64,
         "dims": 64, "layout": "halves", "base": 10000.0, "norm": False},
        # A server's batch of prompts of all lengths; half of each head is rotated.
        {"name": "rotate_packed", "op": "rotate",
         "lengths": "777,1,256,1290,64,333,17,512,96,131,640,5,901", "heads": 16, "kv_heads": 4,
         "dh": 64, "dims": 32, "layout": "pairs", "base": 10000.0, "norm": True},
        # A training batch of the encoder block's sizes.
        {"name": "train_256", "op": "train", "lengths": "256*16", "heads": 8, "kv_heads": 8, "dh": 64,
         "dims": 64, "layout": "halves", "base": 10000.0, "norm": True},
        # Packed training documents of odd lengths, half of each head rotated.
        {"name": "train_ragged", "op": "train", "lengths": "1001,37,555,1,723,289,130", "heads": 10,
         "kv_heads": 2, "dh": 80, "dims": 40, "layout": "halves", "base": 10000.0, "norm": False},
        # Long-context training.
        {"name": "train_4096", "op": "train", "lengths": "4096*4", "heads": 16, "kv_heads": 8, "dh": 128,
         "dims": 128, "layout": "halves", "base": 1000000.0, "norm": True},
        # A busy server's next tokens over an 8-bit cache, requests of all ages.
        {"name": "append_step", "op": "append", "lengths": "1*40",
         "context": "5000,1,777,2048,64*8,1290,333,4097,12,901*5,2500,640*9,3333,100*6,1777,0", "heads": 32,
         "kv_heads": 8, "dh": 128, "dims": 128, "layout": "halves", "base": 1000000.0, "norm": True,
         "format": "int8", "page": 64},
        # A batch of prompts, some of them continued.
        {"name": "append_prompts", "op": "append", "lengths": "2048*8,1531*5,4099", "context": "0*6,8192*3,513*5",
         "heads": 16, "kv_heads": 8, "dh": 128, "dims": 128, "layout": "pairs", "base": 500000.0, "norm": False,
         "format": "f32", "page": 64},
        # A few tokens at once after a short conversation: latency.
        {"name": "chunk_small", "op": "chunk", "lengths": "7", "context": "333", "heads": 8, "kv_heads": 8,
         "dh": 64, "format": "f32", "page": 16},
        # A server's mixed batch over an 8-bit cache: pieces of prompts beside single tokens.
        {"name": "chunk_mixed", "op": "chunk", "lengths": "512,1*24,77,256,0,5,129",
         "context": "1500,5000,1,777,2048*4,64*5,1290,333,4097,12,901*5,2500,640*3,0,7000,300,2222",
         "heads": 32, "kv_heads": 8, "dh": 128, "format": "int8", "page": 64},
        # The next piece of one long prompt.
        {"name": "chunk_512", "op": "chunk", "lengths": "512", "context": "8192", "heads": 32, "kv_heads": 8,
         "dh": 128, "format": "f32", "page": 64},
        # A question to one very long document, one key head.
        {"name": "chunk_long", "op": "chunk", "lengths": "16", "context": "131056", "heads": 8, "kv_heads": 1,
         "dh": 128, "format": "f32", "page": 64},
        # Large pieces of several prompts: the matrix cores' own.
        {"name": "chunk_large", "op": "chunk", "lengths": "2048*4", "context": "6144,0,16384,2000", "heads": 16,
         "kv_heads": 2, "dh": 128, "format": "f32", "page": 128},
    ]


def _lengths(text):
    out = []
    for part in text.split(","):
        n, _, times = part.partition("*")
        out += [int(n)] * int(times or 1)
    return out


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _several(rng, count, lo, hi):
    """`count` lengths: alike in a quarter of the draws, else all over."""
    if rng.random() < 0.25:
        return "%d*%d" % (_log(rng, lo, hi), count)
    return ",".join(str(_log(rng, lo, hi)) for _ in range(count))


def draw(rng):
    op = rng.choice(["rotate", "train", "train", "append", "append", "chunk", "chunk", "chunk", "chunk"])
    dh = rng.choice([32, 40, 64, 64, 80, 96, 128, 128])
    kv = rng.choice([1, 2, 4, 8])
    while True:
        group = rng.choice([1, 2, 4, 5, 8])
        if kv * group > 32:
            continue
        case = {"op": op, "heads": kv * group, "kv_heads": kv, "dh": dh}
        width = (case["heads"] + 2 * kv) * dh
        if op != "chunk":
            case["dims"] = rng.choice([dh, dh, dh, dh // 16 * 8, 8])
            case["layout"] = rng.choice(["halves", "halves", "pairs"])
            case["base"] = rng.choice([10000.0, 500000.0, 1000000.0])
            case["norm"] = rng.random() < 0.6
        if op in ("rotate", "train"):
            case["lengths"] = _several(rng, _log(rng, 1, 24), 1, 6000)
            if sum(_lengths(case["lengths"])) * width <= 16384 * 4096:
                return case
            continue
        case["format"] = rng.choice(["f32", "int8"])
        case["page"] = rng.choice([16, 32, 64, 128, 256])
        n = _log(rng, 1, 48)
        case["lengths"] = _several(rng, n, 1, 2048)
        case["context"] = _several(rng, n, 1, 32768)
        new, old = _lengths(case["lengths"]), _lengths(case["context"])
        total = [a + b for a, b in zip(new, old)]
        if n * max(total) * kv * dh > 1 << 28:
            continue
        if op == "append":
            if sum(new) * width <= 28138 * 4096:
                return case
        elif sum(a * b for a, b in zip(new, total)) * case["heads"] * dh <= 2048 * 30000 * 16 * 128:
            return case


# ---------------------------------------------------------------------------
# What a user's program holds
# ---------------------------------------------------------------------------


def _normal(gen, *shape, scale=1.0):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * scale


def _quantise(x):
    """Codes (0..255) and scales of x along its last axis."""
    top = x.abs().amax(-1)
    scale = top / torch.full_like(top, 127.0)  # by a tensor: by a number, torch multiplies by 1 / 127
    step = torch.where(scale > 0, scale, torch.ones_like(scale))
    return (x / step[..., None]).round().clamp(-127, 127).add(128).to(torch.uint8), scale


def _empty_cache(case, pages):
    hk, ps, d = case["kv_heads"], case["page"], case["dh"]
    if case["format"] == "f32":
        return {n: torch.zeros(pages, hk, ps, d, device="cuda") for n in ("k", "v")}
    return {"k": torch.full((pages, hk, ps, d), 128, dtype=torch.uint8, device="cuda"),
            "v": torch.full((pages, hk, ps // 4, d, 4), 128, dtype=torch.uint8, device="cuda"),
            "ks": torch.zeros(pages, hk, ps, device="cuda"),
            "vs": torch.zeros(pages, hk, ps, device="cuda")}


def _filled_cache(case, pages, gen):
    """A cache whose every slot holds a token."""
    hk, ps, d = case["kv_heads"], case["page"], case["dh"]
    if case["format"] == "f32":
        return {n: _normal(gen, pages, hk, ps, d) for n in ("k", "v")}
    out = {}
    for n in ("k", "v"):
        codes, scale = _quantise(_normal(gen, pages, hk, ps, d))
        if n == "v":
            codes = codes.reshape(pages, hk, ps // 4, 4, d).transpose(3, 4).contiguous()
        out[n], out[n + "s"] = codes, scale
    return out


def _table(case, lens, gen):
    """Each sequence's pages, scattered over the cache, and how many the cache has."""
    ps = case["page"]
    need = [-(-n // ps) for n in lens]
    pages = sum(need)
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.zeros(len(lens), max(need), dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    return table, pages


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    new, op, d, H, hk = _lengths(case["lengths"]), case["op"], case["dh"], case["heads"], case["kv_heads"]
    T, W = sum(new), (H + 2 * hk) * d
    s = {"case": case, "new": new, "plan": {}}
    rows = torch.tensor(new, device="cuda")
    s["seq"] = torch.repeat_interleave(torch.arange(len(new), device="cuda"), rows)
    s["pos"] = torch.arange(T, device="cuda") - (rows.cumsum(0) - rows)[s["seq"]]
    if op != "chunk":
        s["x"] = _normal(gen, T, W)
        if case["norm"]:
            s["wq"], s["wk"] = (1.0 + _normal(gen, d, scale=0.2) for _ in range(2))
        i = torch.arange(case["dims"] // 2, dtype=torch.float64)
        s["freqs"] = case["base"] ** (-2.0 * i / case["dims"])  # on the host
        s["turn"] = s["freqs"].cuda()
    if op in ("rotate", "train"):
        s["y"] = torch.zeros(T, W, device="cuda")
        if op == "train":
            s["dy"], s["dx"] = _normal(gen, T, W, scale=1e-2), torch.zeros(T, W, device="cuda")
            if case["norm"]:
                s["dwq"], s["dwk"] = (torch.zeros(d, device="cuda") for _ in range(2))
        return s
    s["total"] = [a + b for a, b in zip(new, _lengths(case["context"]))]
    s["table"], pages = _table(case, s["total"], gen)
    s["ends"] = torch.tensor(s["total"], dtype=torch.int32, device="cuda")
    s["pos"] = s["pos"] + (s["ends"] - rows)[s["seq"]]
    if op == "append":
        s["cache"] = _empty_cache(case, pages)
        s["q"] = torch.zeros(T, H * d, device="cuda")
        if case["format"] == "int8":
            s["back"] = torch.zeros(2, T, hk * d, device="cuda")
    else:
        s["cache"] = _filled_cache(case, pages, gen)
        s["q"], s["out"] = _normal(gen, T, H * d), torch.zeros(T, H * d, device="cuda")
    return s


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------


def _plain_angles(s):
    a = s["pos"].double()[:, None] * s["turn"]
    return a.cos()[:, None], a.sin()[:, None]


def _plain_turn(x, cos, sin, layout, back=False):
    """x [T, heads, d] with its first columns turned, or turned back."""
    n = 2 * cos.shape[-1]
    if back:
        sin = -sin
    if layout == "halves":
        a, b = x[..., :n // 2], x[..., n // 2:n]
        y = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    else:
        a, b = x[..., 0:n:2], x[..., 1:n:2]
        y = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).reshape(*x.shape[:-1], n)
    return torch.cat([y, x[..., n:]], -1)


def _plain_heads(s, kind):
    """The projection's heads [T, heads, d] in that type, and the cosines and sines in it."""
    case = s["case"]
    cos, sin = _plain_angles(s)
    return s["x"].to(kind).reshape(s["x"].shape[0], -1, case["dh"]), cos.to(kind), sin.to(kind)


def _plain_forward(s, kind=torch.float32):
    """Normed and rotated heads [T, heads, d], rounded at the end, the values as they are."""
    case = s["case"]
    H, hk = case["heads"], case["kv_heads"]
    x, cos, sin = _plain_heads(s, kind)
    y = x[:, :H + hk]
    if case["norm"]:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS)
        y = torch.cat([y[:, :H] * s["wq"].to(kind), y[:, H:] * s["wk"].to(kind)], 1)
    y = _plain_turn(y, cos, sin, case["layout"])
    return torch.cat([y, x[:, H + hk:]], 1).float()


def _plain_rotate(s):
    s["y"].copy_(_plain_forward(s).reshape(s["y"].shape))
    return {"y": s["y"]}


def _plain_train(s):
    case = s["case"]
    H, hk, d = case["heads"], case["kv_heads"], case["dh"]
    out = _plain_rotate(s)
    x, cos, sin = _plain_heads(s, torch.float32)
    g = s["dy"].reshape(x.shape)
    v = g[:, H + hk:]
    g = _plain_turn(g[:, :H + hk], cos, sin, case["layout"], back=True)
    if case["norm"]:
        x = x[:, :H + hk]
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        x = x * r
        dw = g * x
        s["dwq"].copy_(dw[:, :H].sum((0, 1), dtype=torch.float64))
        s["dwk"].copy_(dw[:, H:].sum((0, 1), dtype=torch.float64))
        g = torch.cat([g[:, :H] * s["wq"], g[:, H:] * s["wk"]], 1)
        g = r * (g - x * (g * x).mean(-1, keepdim=True))
        out.update(dwq=s["dwq"], dwk=s["dwk"])
    s["dx"].copy_(torch.cat([g, v], 1).reshape(s["dx"].shape))
    return {**out, "dx": s["dx"]}


def _plain_append(s):
    """In 64 bits for an 8-bit cache, whose codes have borders."""
    case, c = s["case"], s["cache"]
    H, hk, ps = case["heads"], case["kv_heads"], case["page"]
    x = _plain_forward(s, torch.float64 if case["format"] == "int8" else torch.float32)
    s["q"].copy_(x[:, :H].reshape(s["q"].shape))
    k, v = x[:, H:H + hk], x[:, H + hk:]
    page, slot = s["table"][s["seq"], s["pos"] // ps].long(), s["pos"] % ps
    if case["format"] == "f32":
        c["k"][page, :, slot], c["v"][page, :, slot] = k, v
        return {"q": s["q"], "k": c["k"], "v": c["v"]}
    c["k"][page, :, slot], c["ks"][page, :, slot] = _quantise(k)
    c["v"][page, :, slot // 4, :, slot % 4], c["vs"][page, :, slot] = _quantise(v)
    for i, n in enumerate(("k", "v")):
        codes = c[n][page, :, slot] if n == "k" else c[n][page, :, slot // 4, :, slot % 4]
        x = (codes.float() - 128.0) * c[n + "s"][page, :, slot][..., None]
        s["back"][i].copy_(x.reshape(s["back"][i].shape))
    return {"q": s["q"], "k": s["back"][0], "v": s["back"][1]}


def _plain_pages(case, c, n, pages):
    """The named pages' keys or values as floats [Hk, tokens, d]."""
    x = c[n][pages]
    if case["format"] == "int8":
        if n == "v":
            x = x.transpose(-2, -1).reshape(*x.shape[:2], case["page"], case["dh"])
        x = (x.float() - 128.0) * c[n + "s"][pages][..., None]
    return x.transpose(0, 1).reshape(case["kv_heads"], -1, case["dh"])


def _plain_chunk(s):
    case, at = s["case"], 0
    H, hk, d, ps = case["heads"], case["kv_heads"], case["dh"], case["page"]
    for i, (n, total) in enumerate(zip(s["new"], s["total"])):
        if n == 0:
            continue
        pages = s["table"][i, :-(-total // ps)].long()
        k, v = (_plain_pages(case, s["cache"], x, pages)[:, None, :total] for x in ("k", "v"))
        q = s["q"][at:at + n].reshape(n, hk, H // hk, d).permute(1, 2, 0, 3)
        x = q @ k.transpose(2, 3) * (1.0 / math.sqrt(d))
        x = x.masked_fill(torch.ones(n, total, dtype=torch.bool, device="cuda").triu(total - n + 1), -math.inf)
        p = torch.exp(x - x.amax(-1, keepdim=True))
        p = p / p.sum(-1, keepdim=True)
        s["out"][at:at + n] = (p @ v).permute(2, 0, 1, 3).reshape(n, H * d)
        at += n
    return {"out": s["out"]}


_ctx = None


def _plan(s):
    """What a user's program makes once for a batch: the context, the packed lengths, the rotation and
    the cache's description."""
    global _ctx
    import numrs_amd as nr
    if _ctx is None:
        _ctx = nr.Context(0)
    p, case = s["plan"], s["case"]
    if not p:
        p["lib"] = nr.load()
        p["seqs"] = nr.PackedSequences(s["new"], ctx=_ctx)
        if "freqs" in s:
            p["rotary"] = nr.Rotary(case["dh"], case["dims"], layout=case["layout"], freqs=s["freqs"].tolist())
        if "cache" in s:
            c = s["cache"]
            at = lambda n: c[n].data_ptr() if n in c else None  # noqa: E731
            p["cache"] = nr.KVPages(at("k"), at("v"), at("ks"), at("vs"), c["k"].shape[0],
                                    case["page"], case["kv_heads"], case["dh"],
                                    nr.KV_F32 if case["format"] == "f32" else nr.KV_INT8)
    return p


def _check(rc):
    if rc != 0:
        import numrs_amd as nr
        raise nr.HipError(rc, nr.load().numrs_hip_last_error(_ctx.handle).decode())


def _weights(s):
    return (s["wq"].data_ptr(), s["wk"].data_ptr()) if "wq" in s else (None, None)


def _own_rotate(s):
    p, case = _plan(s), s["case"]
    H, hk, d, W = case["heads"], case["kv_heads"], case["dh"], s["x"].shape[1]
    lib, h, seqs, rot = p["lib"], _ctx.handle, p["seqs"].handle, ctypes.byref(p["rotary"].spec)
    wq, wk = _weights(s)
    x, y = s["x"].data_ptr(), s["y"].data_ptr()
    _check(lib.numrs_hip_qk_rotary_forward(h, seqs, None, x, W, wq, wk, EPS, rot, y, W, H, hk, d))
    out = {"y": s["y"]}
    if case["op"] == "train":
        dwq, dwk = (s["dwq"].data_ptr(), s["dwk"].data_ptr()) if case["norm"] else (None, None)
        _check(lib.numrs_hip_qk_rotary_backward(h, seqs, None, x, W, wq, wk, EPS, rot, s["dy"].data_ptr(), W,
                                                s["dx"].data_ptr(), W, dwq, dwk, H, hk, d, 0))
        if case["norm"]:
            out.update(dwq=s["dwq"], dwk=s["dwk"])
        out["dx"] = s["dx"]
    return out


def _own_append(s):
    p, case = _plan(s), s["case"]
    H, hk, d = case["heads"], case["kv_heads"], case["dh"]
    lib, h, seqs, cache = p["lib"], _ctx.handle, p["seqs"].handle, ctypes.byref(p["cache"])
    wq, wk = _weights(s)
    table, ends, most = s["table"].data_ptr(), s["ends"].data_ptr(), s["table"].shape[1]
    _check(lib.numrs_hip_kv_cache_append(h, cache, seqs, s["x"].data_ptr(), s["x"].shape[1], wq, wk, EPS,
                                         ctypes.byref(p["rotary"].spec), s["q"].data_ptr(), H * d, H, table, most,
                                         ends))
    if case["format"] == "f32":
        return {"q": s["q"], "k": s["cache"]["k"], "v": s["cache"]["v"]}
    _check(lib.numrs_hip_kv_cache_read(h, cache, seqs, s["back"][0].data_ptr(), s["back"][1].data_ptr(), hk * d,
                                       table, most, ends))
    return {"q": s["q"], "k": s["back"][0], "v": s["back"][1]}


def _own_chunk(s):
    p, case = _plan(s), s["case"]
    H, w = case["heads"], case["heads"] * case["dh"]
    _check(p["lib"].numrs_hip_attention_paged_chunk(
        _ctx.handle, ctypes.byref(p["cache"]), p["seqs"].handle, s["q"].data_ptr(), w, H, s["table"].data_ptr(),
        s["table"].shape[1], s["ends"].data_ptr(), s["out"].data_ptr(), w))
    return {"out": s["out"]}


def run(s):
    op = s["case"]["op"]
    if own:
        return {"rotate": _own_rotate, "train": _own_rotate, "append": _own_append, "chunk": _own_chunk}[op](s)
    return {"rotate": _plain_rotate, "train": _plain_train, "append": _plain_append, "chunk": _plain_chunk}[op](s)


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------


def work(case):
    new, op, d, H, hk = _lengths(case["lengths"]), case["op"], case["dh"], case["heads"], case["kv_heads"]
    T, q, kv = sum(new), H * d, hk * d
    if op == "rotate":
        return {"bytes": 4 * T * 2 * (q + 2 * kv), "flops": 8 * T * (q + kv)}
    if op == "train":  # x, y, dy, dx
        return {"bytes": 4 * T * 4 * (q + 2 * kv), "flops": 24 * T * (q + kv)}
    token = 2 * hk * (4 * d if case["format"] == "f32" else d + 4)  # a cached token
    if op == "append":
        n = 4 * T * (2 * q + 2 * kv) + T * token
        if case["format"] == "int8":  # and back
            n += T * token + 4 * T * 2 * kv
        return {"bytes": n, "flops": T * (8 * (q + kv) + 6 * kv)}
    total = [a + b for a, b in zip(new, _lengths(case["context"]))]
    cached = sum(t for n, t in zip(new, total) if n)
    pairs = sum(n * t - n * (n - 1) // 2 for n, t in zip(new, total))
    return {"bytes": cached * token + 4 * T * 2 * q, "flops": 4 * pairs * q}


# ---------------------------------------------------------------------------
# The same in 64 bits
# ---------------------------------------------------------------------------


def _exact_positions(case):
    before = _lengths(case["context"]) if "context" in case else [0] * len(_lengths(case["lengths"]))
    return [b + j for n, b in zip(_lengths(case["lengths"]), before) for j in range(n)]


def _exact_matrix(case):
    """Columns that turn together, and the unit complex number of each token and angle."""
    n = case["dims"]
    i = torch.arange(n // 2, dtype=torch.float64, device="cuda")
    angle = torch.outer(torch.tensor(_exact_positions(case), dtype=torch.float64, device="cuda"),
                        torch.pow(torch.tensor(case["base"], dtype=torch.float64, device="cuda"), -2 * i / n))
    first = torch.arange(n // 2, device="cuda") * (1 if case["layout"] == "halves" else 2)
    return first, first + (n // 2 if case["layout"] == "halves" else 1), torch.polar(torch.ones_like(angle), angle)


def _exact_rotated(x, first, second, unit):
    z = torch.complex(x[:, first], x[:, second]) * unit
    out = x.clone()
    out[:, first], out[:, second] = z.real, z.imag
    return out


def _exact_heads(case, s, grads):
    H, hk, d = case["heads"], case["kv_heads"], case["dh"]
    first, second, unit = _exact_matrix(case)
    y, dx = s["x"].double(), s["dy"].double() if grads else None
    dw = [torch.zeros(d, dtype=torch.float64, device="cuda") for _ in range(2)]
    for h in range(H + hk):
        cols = slice(h * d, h * d + d)
        x = s["x"][:, cols].double()
        w = s["wq" if h < H else "wk"].double() if case["norm"] else None
        rms = (x.square().sum(1, keepdim=True) / d + EPS).sqrt() if case["norm"] else None
        y[:, cols] = _exact_rotated(x / rms * w if case["norm"] else x, first, second, unit)
        if not grads:
            continue
        g = _exact_rotated(s["dy"][:, cols].double(), first, second, unit.conj())
        if case["norm"]:
            dw[h >= H] += (g * x / rms).sum(0)
            g = g * w
            g = g / rms - x * (g * x).sum(1, keepdim=True) / (d * rms ** 3)
        dx[:, cols] = g
    return y, dx, dw


def _exact_quantised(x):
    """What the cache stands for: the rows and the quotients are rounded to float32 as the format says."""
    x = x.float().double()
    top = x.abs().max(dim=-1, keepdim=True).values
    scale = (top / 127).float().double()
    code = torch.round((x / scale.clamp_min(1e-300)).float().double())
    return torch.clamp(code, -127, 127) * scale


def _exact_append(case, s):
    H, hk, d, ps = case["heads"], case["kv_heads"], case["dh"], case["page"]
    y, _, _ = _exact_heads(case, s, False)
    out = {"q": y[:, :H * d]}
    for i, name in enumerate(("k", "v")):
        x = y[:, (H + i * hk) * d:(H + (i + 1) * hk) * d].reshape(-1, hk, d)
        if case["format"] == "int8":
            out[name] = _exact_quantised(x).reshape(-1, hk * d)
            continue
        # the cache was zeros before
        pages, at = torch.zeros(s["cache"]["k"].shape, dtype=torch.float64, device="cuda"), 0
        for j, (n, total) in enumerate(zip(s["new"], s["total"])):
            where = torch.arange(total - n, total, device="cuda")
            pages[s["table"][j].long()[where // ps], :, where % ps] = x[at:at + n]
            at += n
        out[name] = pages
    return out


def _exact_chunk(case, s):
    H, hk, d, ps = case["heads"], case["kv_heads"], case["dh"], case["page"]
    c, outs, at = s["cache"], [], 0
    for i, (n, total) in enumerate(zip(s["new"], s["total"])):
        if n == 0:
            continue
        pages = s["table"][i, :-(-total // ps)].long()
        kv = {}
        for name in ("k", "v"):
            t = c[name][pages]
            if case["format"] == "int8":
                if name == "v":
                    t = t.permute(0, 1, 2, 4, 3).reshape(len(pages), hk, ps, d)
                t = (t.double() - 128) * c[name + "s"][pages].double().unsqueeze(-1)
            kv[name] = t.double().permute(1, 0, 2, 3).reshape(hk, -1, d)[:, :total]
        seen = torch.arange(total, device="cuda") <= torch.arange(total - n, total, device="cuda")[:, None]
        out = torch.zeros(n, H * d, dtype=torch.float64, device="cuda")
        for h in range(H):
            g, cols = h // (H // hk), slice(h * d, h * d + d)
            w = s["q"][at:at + n, cols].double().matmul(kv["k"][g].T) / d ** 0.5
            out[:, cols] = torch.where(seen, w, -torch.inf).softmax(1).matmul(kv["v"][g])
        outs.append(out)
        at += n
    return {"out": torch.cat(outs)}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "chunk":
        return _exact_chunk(case, s)
    if case["op"] == "append":
        return _exact_append(case, s)
    y, dx, dw = _exact_heads(case, s, case["op"] == "train")
    out = {"y": y}
    if case["op"] == "train":
        if case["norm"]:
            out.update(dwq=dw[0], dwk=dw[1])
        out["dx"] = dx
    return out
