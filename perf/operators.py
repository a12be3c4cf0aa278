"""Decoder attention over packed sequences and a paged key-value cache, and what it is timed on.

A case is a dict of plain values; `op` names what one pass does:

  prompt  causal attention with grouped heads over a packed batch of prompts (forward)
  train   the same forward and its backward: the output, dq, dk and dv
  step    one decoding step: every request's new key and value go into the cache, then its
          query attends to all of its cached tokens
  cache   a packed batch's keys and values written into the cache, then read back

`lengths` are the sequences' tokens as a text, "a,b,c", or "a*n" for n sequences of a. q, k and v
are column blocks of one projection [tokens, (heads + 2 kv_heads) * dh]. A cache of format "int8"
holds a byte a value and a float32 scale for each token and head: scale = max|x| / 127, code =
round(x / scale) + 128, both in float32 with ties to even; the values' codes of four neighbouring
slots lie together.  Everything else is float32, the framework's only floating type.
"""
from __future__ import annotations

import ctypes
import math

import torch

own = False

# ---------------------------------------------------------------------------
# The cases
# ---------------------------------------------------------------------------


def listed():
    return [
        # A short turn of one conversation: latency.
        {"name": "prompt_64", "op": "prompt", "lengths": "64", "heads": 8, "kv_heads": 8, "dh": 64},
        # A server's batch of prompts of all lengths, a single token among them.
        {"name": "prompt_packed", "op": "prompt",
         "lengths": "777,1,256,1290,64,333,17,512,96,131,640,5,901", "heads": 16, "kv_heads": 4,
         "dh": 64},
        # One long document.
        {"name": "prompt_8192", "op": "prompt", "lengths": "8192", "heads": 16, "kv_heads": 4,
         "dh": 128},
        # A training batch of the encoder block's sizes, causal.
        {"name": "train_256", "op": "train", "lengths": "256*16", "heads": 8, "kv_heads": 8,
         "dh": 64},
        # Packed training documents: no length is a multiple of anything.
        {"name": "train_ragged", "op": "train", "lengths": "1001,37,555,1,723,289,130", "heads": 10,
         "kv_heads": 2, "dh": 80},
        # Long-context training.
        {"name": "train_4096", "op": "train", "lengths": "4096*2", "heads": 16, "kv_heads": 4,
         "dh": 128},
        # One conversation's next token.
        {"name": "step_1", "op": "step", "lengths": "333", "heads": 8, "kv_heads": 8, "dh": 64,
         "format": "f32", "page": 16},
        # A busy server: requests of all ages over an 8-bit cache.
        {"name": "step_ragged", "op": "step",
         "lengths": "5000,1,777,2048,64*8,1290,333,4097,12,901*5,2500,640*9,3333,100*6,1777", "heads": 32,
         "kv_heads": 8, "dh": 128, "format": "int8", "page": 64},
        # A single very long conversation, one key head.
        {"name": "step_long", "op": "step", "lengths": "131072", "heads": 8, "kv_heads": 1, "dh": 128,
         "format": "f32", "page": 64},
        # Many long conversations: the whole chip reads the cache.
        {"name": "step_large", "op": "step", "lengths": "6000*64,8000*32", "heads": 32, "kv_heads": 8,
         "dh": 128, "format": "f32", "page": 64},
        # A small prompt into an exact cache, and back.
        {"name": "cache_small", "op": "cache", "lengths": "100,45,300,7", "kv_heads": 8, "dh": 64,
         "format": "f32", "page": 16},
        # A batch of prompts into an 8-bit cache, and back.
        {"name": "cache_prompts", "op": "cache", "lengths": "2048*8,1531*5,4099", "kv_heads": 8,
         "dh": 128, "format": "int8", "page": 64},
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
    """`count` lengths around one of their own: alike in half of the draws, else all over."""
    if rng.random() < 0.25:
        return "%d*%d" % (_log(rng, lo, hi), count)
    return ",".join(str(_log(rng, lo, hi)) for _ in range(count))


def draw(rng):
    op = rng.choice(["prompt", "prompt", "train", "train", "step", "step", "step", "cache"])
    dh = rng.choice([32, 40, 64, 64, 80, 96, 128, 128])
    kv = rng.choice([1, 2, 4, 8])
    while True:
        group = rng.choice([1, 2, 4, 5, 8])
        if kv * group > 32:
            continue
        case = {"op": op, "heads": kv * group, "kv_heads": kv, "dh": dh}
        if op in ("prompt", "train"):
            case["lengths"] = _several(rng, _log(rng, 1, 24), 1, 6000)
            pairs = sum(n * n for n in _lengths(case["lengths"]))
            if pairs * case["heads"] * dh <= 4096 * 4096 * 2 * 16 * 128:
                return case
            continue
        case["format"] = rng.choice(["f32", "int8", "int8"])
        case["page"] = rng.choice([16, 32, 64, 128, 256])
        if op == "step":
            case["lengths"] = _several(rng, _log(rng, 1, 128), 1, 32768)
            most = 640000 * 8 * 128
        else:
            del case["heads"]
            case["lengths"] = _several(rng, _log(rng, 1, 64), 1, 8192)
            most = 28138 * 8 * 128
        lens = _lengths(case["lengths"])
        if sum(lens) * kv * dh <= most and len(lens) * max(lens) * kv * dh <= 1 << 30:
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
    lens, op, d, hk = _lengths(case["lengths"]), case["op"], case["dh"], case["kv_heads"]
    s = {"case": case, "lens": lens, "plan": {}}
    if op in ("prompt", "train"):
        H, T = case["heads"], sum(lens)
        s["qkv"], s["out"] = _normal(gen, T, (H + 2 * hk) * d), torch.zeros(T, H * d, device="cuda")
        if op == "train":
            s["g"] = _normal(gen, T, H * d, scale=1e-2)
            s["stats"] = torch.zeros(T, H, 2, device="cuda")
            s["dqkv"] = torch.zeros_like(s["qkv"])
        return s
    s["table"], pages = _table(case, lens, gen)
    s["ends"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    s["new"] = [1] * len(lens) if op == "step" else lens
    T = sum(s["new"])
    # each new row's sequence and its place among the sequence's new rows
    rows = torch.tensor(s["new"], device="cuda")
    s["seq"] = torch.repeat_interleave(torch.arange(len(lens), device="cuda"), rows)
    s["row"] = torch.arange(T, device="cuda") - (rows.cumsum(0) - rows)[s["seq"]]
    if op == "step":
        H = case["heads"]
        s["cache"] = _filled_cache(case, pages, gen)
        s["qkv"], s["out"] = _normal(gen, T, (H + 2 * hk) * d), torch.zeros(T, H * d, device="cuda")
    else:
        s["cache"] = _empty_cache(case, pages)
        s["qkv"] = _normal(gen, T, 2 * hk * d)
        s["back"] = torch.zeros(2, T, hk * d, device="cuda")
    return s


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------


def _plain_sequence(q, k, v, g):
    """Causal attention of one sequence: q [H, L, d], k and v [Hk, L, d]; with g its gradients."""
    (H, L, d), hk = q.shape, k.shape[0]
    q = q.reshape(hk, H // hk, L, d)
    k, v = k[:, None], v[:, None]
    s = q @ k.transpose(2, 3) * (1.0 / math.sqrt(d))
    s = s.masked_fill(torch.ones(L, L, dtype=torch.bool, device=q.device).triu(1), -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    out = p @ v
    if g is None:
        return out.reshape(H, L, d), None
    g = g.reshape(out.shape)
    dv = (p.transpose(2, 3) @ g).sum(1)
    ds = p * (g @ v.transpose(2, 3) - (g * out).sum(-1, keepdim=True)) * (1.0 / math.sqrt(d))
    dq = (ds @ k).reshape(H, L, d)
    return out.reshape(H, L, d), (dq, (ds.transpose(2, 3) @ q).sum(1), dv)


def _plain_attention(s):
    case = s["case"]
    H, hk, d, at = case["heads"], case["kv_heads"], case["dh"], 0
    heads = lambda t: t.reshape(t.shape[0], -1, d).transpose(0, 1)  # noqa: E731
    flat = lambda t: t.transpose(0, 1).reshape(t.shape[1], -1)  # noqa: E731
    for n in s["lens"]:
        x = s["qkv"][at:at + n]
        q, k, v = (heads(t).contiguous() for t in x.split([H * d, hk * d, hk * d], 1))
        g = heads(s["g"][at:at + n]).contiguous() if case["op"] == "train" else None
        out, grads = _plain_sequence(q, k, v, g)
        s["out"][at:at + n] = flat(out)
        if grads:
            s["dqkv"][at:at + n] = torch.cat([flat(t) for t in grads], 1)
        at += n
    return {k: s[k] for k in (("out", "dqkv") if case["op"] == "train" else ("out",))}


def _plain_slots(s):
    """Page and slot of each new row."""
    ps, rows = s["case"]["page"], torch.tensor(s["new"], device="cuda")
    pos = (s["ends"] - rows)[s["seq"]] + s["row"]
    return s["table"][s["seq"], pos // ps].long(), pos % ps


def _plain_write(s, k, v):
    case, c = s["case"], s["cache"]
    page, slot = _plain_slots(s)
    k, v = (t.reshape(t.shape[0], case["kv_heads"], case["dh"]) for t in (k, v))
    if case["format"] == "f32":
        c["k"][page, :, slot], c["v"][page, :, slot] = k, v
        return
    c["k"][page, :, slot], c["ks"][page, :, slot] = _quantise(k)
    c["v"][page, :, slot // 4, :, slot % 4], c["vs"][page, :, slot] = _quantise(v)


def _plain_pages(case, c, n, pages):
    """The named pages' keys or values as floats [..., Hk, page, d]."""
    x = c[n][pages]
    if case["format"] == "f32":
        return x
    if n == "v":
        x = x.transpose(-2, -1).reshape(*x.shape[:-3], case["page"], case["dh"])
    return (x.float() - 128.0) * c[n + "s"][pages][..., None]


def _plain_step(s):
    case = s["case"]
    H, hk, d, ps = case["heads"], case["kv_heads"], case["dh"], case["page"]
    q, k, v = s["qkv"].split([H * d, hk * d, hk * d], 1)
    _plain_write(s, k, v)
    n, most = s["table"].shape
    table = s["table"].long()
    k, v = (_plain_pages(case, s["cache"], x, table).transpose(1, 2).reshape(n, hk, most * ps, d)
            for x in ("k", "v"))
    x = q.reshape(n, hk, H // hk, d) @ k.transpose(2, 3) * (1.0 / math.sqrt(d))
    gone = torch.arange(most * ps, device="cuda") >= s["ends"][:, None]
    x = x.masked_fill(gone[:, None, None], -math.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    s["out"].copy_((p @ v).reshape(n, H * d))
    return {"out": s["out"]}


def _plain_cache(s):
    case = s["case"]
    k, v = s["qkv"].chunk(2, 1)
    _plain_write(s, k, v)
    page, slot = _plain_slots(s)
    for i, n in enumerate(("k", "v")):
        c = s["cache"]
        if case["format"] == "f32":
            x = c[n][page, :, slot]
        else:
            codes = c[n][page, :, slot] if n == "k" else c[n][page, :, slot // 4, :, slot % 4]
            x = (codes.float() - 128.0) * c[n + "s"][page, :, slot][..., None]
        s["back"][i].copy_(x.reshape(s["back"][i].shape))
    return {"k": s["back"][0], "v": s["back"][1]}


_ctx = None


def _plan(s):
    """What a user's program makes once for a batch: the context, the packed lengths, the cache's
    description."""
    global _ctx
    import numrs_amd as nr
    if _ctx is None:
        _ctx = nr.Context(0)
    p, case = s["plan"], s["case"]
    if not p:
        p["lib"] = nr.load()
        p["seqs"] = nr.PackedSequences(s.get("new", s["lens"]), ctx=_ctx)
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


def _own_attention(s):
    p, case = _plan(s), s["case"]
    H, hk, d = case["heads"], case["kv_heads"], case["dh"]
    lib, h, seqs, ld = p["lib"], _ctx.handle, p["seqs"].handle, (H + 2 * hk) * d
    q, out = s["qkv"].data_ptr(), s["out"].data_ptr()
    k, v = q + 4 * H * d, q + 4 * (H + hk) * d
    stats = s["stats"].data_ptr() if case["op"] == "train" else None
    _check(lib.numrs_hip_attention_packed_forward(h, seqs, q, ld, k, v, ld, out, H * d, stats, H,
                                                  hk, d))
    if case["op"] == "prompt":
        return {"out": s["out"]}
    dq = s["dqkv"].data_ptr()
    dk, dv = dq + 4 * H * d, dq + 4 * (H + hk) * d
    _check(lib.numrs_hip_attention_packed_backward(h, seqs, q, ld, k, v, ld, out, s["g"].data_ptr(),
                                                   H * d, stats, dq, dk, dv, H, hk, d, 0))
    return {"out": s["out"], "dqkv": s["dqkv"]}


def _own_step(s):
    p, case = _plan(s), s["case"]
    H, hk, d = case["heads"], case["kv_heads"], case["dh"]
    lib, h, ld = p["lib"], _ctx.handle, (H + 2 * hk) * d
    q, cache = s["qkv"].data_ptr(), ctypes.byref(p["cache"])
    table, ends, most = s["table"].data_ptr(), s["ends"].data_ptr(), s["table"].shape[1]
    _check(lib.numrs_hip_kv_cache_write(h, cache, p["seqs"].handle, q + 4 * H * d,
                                        q + 4 * (H + hk) * d, ld, table, most, ends))
    _check(lib.numrs_hip_attention_paged(h, cache, q, ld, H, table, most, ends, len(s["lens"]),
                                         s["out"].data_ptr(), H * d))
    return {"out": s["out"]}


def _own_cache(s):
    p, case = _plan(s), s["case"]
    w = case["kv_heads"] * case["dh"]
    lib, h, seqs = p["lib"], _ctx.handle, p["seqs"].handle
    k, cache = s["qkv"].data_ptr(), ctypes.byref(p["cache"])
    table, ends, most = s["table"].data_ptr(), s["ends"].data_ptr(), s["table"].shape[1]
    _check(lib.numrs_hip_kv_cache_write(h, cache, seqs, k, k + 4 * w, 2 * w, table, most, ends))
    _check(lib.numrs_hip_kv_cache_read(h, cache, seqs, s["back"][0].data_ptr(),
                                       s["back"][1].data_ptr(), w, table, most, ends))
    return {"k": s["back"][0], "v": s["back"][1]}


def run(s):
    op = s["case"]["op"]
    if op in ("prompt", "train"):
        return _own_attention(s) if own else _plain_attention(s)
    if op == "step":
        return _own_step(s) if own else _plain_step(s)
    return _own_cache(s) if own else _plain_cache(s)


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------


def work(case):
    lens, op, d, hk = _lengths(case["lengths"]), case["op"], case["dh"], case["kv_heads"]
    T = sum(lens)
    if op in ("prompt", "train"):
        H, pairs = case["heads"], sum(n * (n + 1) // 2 for n in lens)
        if op == "prompt":
            return {"bytes": 4 * T * d * (2 * H + 2 * hk), "flops": 4 * d * H * pairs}
        # q, k, v, out, the output's gradient, dq, dk, dv
        return {"bytes": 4 * T * d * (4 * H + 4 * hk), "flops": 14 * d * H * pairs}
    token = 2 * hk * (4 * d if case["format"] == "f32" else d + 4)  # a cached token
    if op == "step":
        H, n = case["heads"], len(lens)
        return {"bytes": T * token + n * 4 * d * (2 * H + 2 * hk), "flops": 4 * d * H * T}
    return {"bytes": 2 * T * token + 4 * T * 4 * hk * d, "flops": 6 * T * hk * d}


# ---------------------------------------------------------------------------
# The same in 64 bits
# ---------------------------------------------------------------------------


def _exact_quantised(x):
    """What the cache stands for: the quotients are rounded to float32 as the format says."""
    top = x.abs().max(dim=-1, keepdim=True).values
    scale = (top / 127).float().double()
    code = torch.round((x / scale.clamp_min(1e-300)).float().double())
    return torch.clamp(code, -127, 127) * scale


def _exact_attention(case, s):
    H, hk, d, lens = case["heads"], case["kv_heads"], case["dh"], s["lens"]
    train, outs, grads, at = case["op"] == "train", [], [], 0
    for n in lens:
        x = s["qkv"][at:at + n].double()
        out = torch.zeros(n, H * d, dtype=torch.float64, device="cuda")
        dx = torch.zeros_like(x)
        mask = torch.arange(n, device="cuda")[:, None] >= torch.arange(n, device="cuda")
        for h in range(H):
            g = h // (H // hk)
            cq = slice(h * d, h * d + d)
            ck = slice((H + g) * d, (H + g) * d + d)
            cv = slice((H + hk + g) * d, (H + hk + g) * d + d)
            q, k, v = x[:, cq], x[:, ck], x[:, cv]
            w = torch.where(mask, q.matmul(k.T) / d ** 0.5, -torch.inf).softmax(1)
            out[:, cq] = w.matmul(v)
            if train:
                go = s["g"][at:at + n, cq].double()
                dw = go.matmul(v.T)
                dz = w * (dw - (w * dw).sum(1, keepdim=True)) / d ** 0.5
                dx[:, cq] = dz.matmul(k)
                dx[:, ck] += dz.T.matmul(q)
                dx[:, cv] += w.T.matmul(go)
        outs.append(out)
        grads.append(dx)
        at += n
    return {"out": torch.cat(outs), **({"dqkv": torch.cat(grads)} if train else {})}


def _exact_step(case, s):
    H, hk, d, ps = case["heads"], case["kv_heads"], case["dh"], case["page"]
    c, outs = s["cache"], []
    for i, n in enumerate(s["lens"]):
        pages = s["table"][i, :-(-n // ps)].long()
        x = s["qkv"][i].double()
        new = {"k": x[H * d:(H + hk) * d].reshape(hk, d), "v": x[(H + hk) * d:].reshape(hk, d)}
        kv = {}
        for name in ("k", "v"):
            t = c[name][pages]
            if case["format"] == "int8":
                if name == "v":
                    t = t.permute(0, 1, 2, 4, 3).reshape(len(pages), hk, ps, d)
                t = (t.double() - 128) * c[name + "s"][pages].double().unsqueeze(-1)
                new[name] = _exact_quantised(new[name])
            t = t.double().permute(1, 0, 2, 3).reshape(hk, -1, d)[:, :n].clone()
            t[:, n - 1] = new[name]
            kv[name] = t
        w = torch.bmm(x[:H * d].reshape(hk, H // hk, d), kv["k"].permute(0, 2, 1).contiguous())
        outs.append(torch.bmm((w / d ** 0.5).softmax(-1), kv["v"]).reshape(H * d))
    return {"out": torch.stack(outs)}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("prompt", "train"):
        return _exact_attention(case, s)
    if case["op"] == "step":
        return _exact_step(case, s)
    w = case["kv_heads"] * case["dh"]
    out = {}
    for i, name in enumerate(("k", "v")):
        x = s["qkv"][:, i * w:(i + 1) * w].double()
        if case["format"] == "int8":
            x = _exact_quantised(x.reshape(-1, case["dh"])).reshape(x.shape)
        out[name] = x
    return out
