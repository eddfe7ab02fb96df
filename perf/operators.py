"""The serving operators of the decode path, as cases that can be run and timed: the paged
key-value cache (append with rotary positions, attention of one new token), the residual RMS norm
with 8-bit output, and the logits processor.

Every case has a plain form (elementary torch operations in 32 bits) and, with `own` set, the
calls a program makes of the framework's kernels.  `exact` restates the definitions in 64 bits.
"""
import math

import torch

own = False

DEV = "cuda"
BF16, F32, I8 = torch.bfloat16, torch.float32, torch.int8


# ------------------------------------------------------------------------------------- cases
def listed():
    return [
        # Gemma-3-1B's global layer, one stream at its 4,096 context: a call where latency counts
        dict(name="attention one stream", op="attention", b=1, hq=4, hkv=1, d=256, page=64, longest=4096,
             ragged=False, kv="bf16", window=0, lse=False),
        # its sliding-window layers, 64 streams
        dict(name="attention window 512", op="attention", b=64, hq=4, hkv=1, d=256, page=64, longest=4096,
             ragged=False, kv="bf16", window=512, lse=False),
        # opt-125m heads (no sharing), 32 streams of every length up to its 2,048 positions, one still
        # empty; the log-sum-exp is kept to join with another part of the context
        dict(name="attention 12 heads ragged", op="attention", b=32, hq=12, hkv=12, d=64, page=64, longest=2048,
             ragged=True, kv="bf16", window=0, lse=True),
        # a server's full batch: shared heads, small pages, every length up to 8k
        dict(name="attention 64 streams ragged", op="attention", b=64, hq=32, hkv=8, d=128, page=16, longest=8192,
             ragged=True, kv="bf16", window=0, lse=False),
        # few streams with long documents, 8-bit cache
        dict(name="attention 64k int8", op="attention", b=4, hq=32, hkv=8, d=128, page=64, longest=65536,
             ragged=False, kv="int8", window=0, lse=False),
        # one decode step's keys and values of 64 streams
        dict(name="append 64 streams", op="append", t=64, streams=64, hq=32, hkv=8, d=128, page=16, rot=128,
             interleaved=False, src="bf16", kv="bf16", start=1000),
        # a batch of prompts, straight from an int8 product's f32 output
        dict(name="append prompts", op="append", t=8192, streams=4, hq=32, hkv=8, d=128, page=16, rot=128,
             interleaved=False, src="f32", kv="bf16", start=0),
        # a prompt of odd length into an 8-bit cache, Gemma-3-1B heads
        dict(name="append prompt int8", op="append", t=2003, streams=1, hq=4, hkv=1, d=256, page=64, rot=256,
             interleaved=False, src="bf16", kv="int8", start=0),
        # Gemma-3-1B's hidden size at 64 streams
        dict(name="norm 64 rows", op="norm", m=64, d=1152, x="bf16", res="bf16", unit_offset=True),
        # a batch of prompts
        dict(name="norm 8192 rows", op="norm", m=8192, d=4096, x="bf16", res="bf16", unit_offset=False),
        # opt-125m's vocabulary, one stream, 32 prompt and 128 generated tokens
        dict(name="logits one stream", op="logits", b=1, v=50272, src="f32", prompt=32, generated=128, biases=8,
             grammar=False),
        # Gemma-3-1B's vocabulary, 64 streams with a grammar
        dict(name="logits 64 streams", op="logits", b=64, v=262144, src="f32", prompt=3000, generated=1000,
             biases=300, grammar=True),
    ]


MOST_BYTES = 1.05e9          # no drawn case reads and writes more than the largest listed one


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "append", "norm", "logits"])
    if op == "attention":
        d, hkv, g = rng.choice([64, 128, 256]), _log(rng, 1, 12), rng.choice([1, 2, 3, 4, 5, 7, 8, 12, 16])
        c = dict(op=op, b=_log(rng, 1, 128), hq=hkv * g, hkv=hkv, d=d, page=rng.choice([8, 16, 24, 32, 64, 128]),
                 longest=_log(rng, 1, 65536), ragged=rng.random() < 0.7, kv=rng.choice(["bf16", "int8"]),
                 window=_log(rng, 1, 4096) if rng.random() < 0.3 else 0, lse=rng.random() < 0.5)
        # the whole cache, of which a window reads a part, bounds the case
        while _attention_bytes(dict(c, window=0)) > MOST_BYTES or (c["longest"] * c["b"] * hkv * d > 2.2e8):
            c["longest"] = max(1, c["longest"] * 2 // 3)
        return c
    if op == "append":
        d, hkv, g = rng.choice([64, 128, 256]), _log(rng, 1, 12), rng.choice([1, 2, 3, 4, 7, 8])
        streams = _log(rng, 1, 128)
        c = dict(op=op, t=streams * _log(rng, 1, 2000), streams=streams, hq=hkv * g, hkv=hkv, d=d,
                 page=rng.choice([8, 16, 24, 32, 64]), rot=rng.choice([d, d, d // 2, d // 4]),
                 interleaved=rng.random() < 0.3, src=rng.choice(["bf16", "f32"]), kv=rng.choice(["bf16", "int8"]),
                 start=_log(rng, 1, 30000))
        while work(c)["bytes"] > 4e8:
            c["t"] = max(streams, c["t"] // streams // 2 * streams)
        return c
    if op == "norm":
        c = dict(op=op, m=_log(rng, 1, 16384), d=_log(rng, 64, 16384), x=rng.choice(["bf16", "f32"]),
                 res=rng.choice(["bf16", "f32"]), unit_offset=rng.random() < 0.5)
        c["d"] += 0 if rng.random() < 0.3 else -c["d"] % 128           # mostly what the int8 products take
        while work(c)["bytes"] > 6e8:
            c["m"] = max(1, c["m"] // 2)
        return c
    return dict(op=op, b=_log(rng, 1, 128), v=_log(rng, 1000, 262144), src=rng.choice(["bf16", "f32"]),
                prompt=_log(rng, 1, 8192), generated=_log(rng, 1, 4096), biases=_log(rng, 1, 300),
                grammar=rng.random() < 0.5)


def _lens(c):
    """The streams' lengths: all alike, or spread evenly from none at all to the longest."""
    if not c["ragged"] or c["b"] == 1:
        return [c["longest"]] * c["b"]
    return [c["longest"] * i // (c["b"] - 1) for i in range(c["b"])]


def _attention_bytes(c):
    kept = sum(min(n, c["window"] or n) for n in _lens(c))
    row = c["hkv"] * (c["d"] * (2 if c["kv"] == "bf16" else 1) + (4 if c["kv"] == "int8" else 0))
    return 2 * kept * row + 2 * c["b"] * c["hq"] * c["d"] * 2 + kept // c["page"] * 4 + c["b"] * (4 + 4 * c["hq"] * c["lse"])


def work(c):
    if c["op"] == "attention":
        kept = sum(min(n, c["window"] or n) for n in _lens(c))
        return {"bytes": _attention_bytes(c), "flops": 4 * kept * c["hq"] * c["d"]}
    if c["op"] == "append":
        t, heads, d = c["t"], c["hq"] + 2 * c["hkv"], c["d"]
        kv = 2 if c["kv"] == "bf16" else 1
        positions = c["t"] // c["streams"]
        return {"bytes": t * heads * d * (2 if c["src"] == "bf16" else 4) + t * c["hq"] * d * 2
                + 2 * t * c["hkv"] * (d * kv + (4 if kv == 1 else 0)) + positions * c["rot"] * 4 + t * 12,
                "flops": t * (c["hq"] + c["hkv"]) * c["rot"] * 3}
    if c["op"] == "norm":
        x, r = (2 if c[k] == "bf16" else 4 for k in ("x", "res"))
        return {"bytes": c["m"] * c["d"] * (x + 2 * r + 1) + c["m"] * 4 + c["d"] * 4, "flops": 7 * c["m"] * c["d"]}
    b, v = c["b"], c["v"]
    return {"bytes": b * v * ((4 if c["src"] == "f32" else 2) + 4) + (b * ((v + 31) // 32) * 4 if c["grammar"] else 0)
            + b * ((c["prompt"] + c["generated"]) * 4 + c["biases"] * 8 + 28), "flops": b * v}


# ----------------------------------------------------------------------------------- inputs
def _rng(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _normal(g, *shape, dtype=F32, std=1.0):
    return (torch.randn(*shape, generator=g, device=DEV, dtype=F32) * std).to(dtype)


def _ints(g, lo, hi, *shape, dtype=torch.int32):
    return torch.randint(lo, hi, shape, generator=g, device=DEV, dtype=dtype)


def _type(name):
    return BF16 if name == "bf16" else F32


def _rope_table(n, rot, theta=10000.0):
    """[n][rot]: the cosines of a position's rot / 2 angles, then their sines (computed in 64 bits)."""
    inv = theta ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=DEV) / rot)
    a = torch.arange(n, dtype=torch.float64, device=DEV)[:, None] * inv
    return torch.cat([a.cos(), a.sin()], 1).float()


def _inputs(c, seed):
    g = _rng(seed)
    if c["op"] == "attention":
        b, hkv, d, ps = c["b"], c["hkv"], c["d"], c["page"]
        order = torch.randperm(b, generator=g, device=DEV)
        lens = torch.tensor(_lens(c), dtype=torch.int32, device=DEV)[order]
        width = max(1, -(-c["longest"] // ps))
        pages = (lens + ps - 1) // ps
        n_pages = sum(-(-n // ps) for n in _lens(c)) + 1
        ids = torch.randperm(n_pages, generator=g, device=DEV).int()
        first = torch.cumsum(pages, 0) - pages
        col = torch.arange(width, device=DEV)
        # a stream's entries past its own pages are left at -1
        table = torch.where(col[None] < pages[:, None], ids[(first[:, None] + col[None]).clamp_max(n_pages - 1)], -1)
        s = dict(q=_normal(g, b, c["hq"], d, dtype=BF16, std=1.5), lens=lens, table=table.int().contiguous())
        shape = (n_pages, hkv, ps, d)
        if c["kv"] == "bf16":
            s["k"] = torch.empty(shape, device=DEV, dtype=BF16).normal_(generator=g)
            s["v"] = torch.empty(shape, device=DEV, dtype=BF16).normal_(generator=g)
        else:
            s["k"], s["v"] = (torch.randint(-127, 128, shape, generator=g, device=DEV, dtype=I8) for _ in "kv")
            s["k_scale"], s["v_scale"] = (torch.rand(shape[:3], generator=g, device=DEV) * 0.02 + 0.005 for _ in "kv")
        return s
    if c["op"] == "append":
        t, streams, ps, d = c["t"], c["streams"], c["page"], c["d"]
        each = t // streams
        qkv = _normal(g, t, (c["hq"] + 2 * c["hkv"]) * d, dtype=_type(c["src"]))
        # the pages that these positions lie in, with one more; the rest of the streams' pages is not held here
        first, last = c["start"] // ps, (c["start"] + each - 1) // ps
        n_pages = streams * (last - first + 1) + 1
        ids = torch.randperm(n_pages, generator=g, device=DEV).int()
        table = torch.full((streams, last + 1), -1, dtype=torch.int32, device=DEV)
        table[:, first:] = ids[: n_pages - 1].view(streams, last - first + 1)
        s = dict(qkv=qkv, table=table, rope=_rope_table(c["start"] + each, c["rot"]),
                 seq=torch.arange(streams, dtype=torch.int32, device=DEV).repeat_interleave(each),
                 pos=(c["start"] + torch.arange(each, dtype=torch.int32, device=DEV)).repeat(streams))
        shape = (n_pages, c["hkv"], ps, d)
        if c["kv"] == "bf16":
            s["k"], s["v"] = (torch.zeros(shape, dtype=BF16, device=DEV) for _ in "kv")
        else:
            s["k"], s["v"] = (torch.zeros(shape, dtype=I8, device=DEV) for _ in "kv")
            s["k_scale"], s["v_scale"] = (torch.zeros(shape[:3], device=DEV) for _ in "kv")
        return s
    if c["op"] == "norm":
        return dict(x=_normal(g, c["m"], c["d"], dtype=_type(c["x"])),
                    res=_normal(g, c["m"], c["d"], dtype=_type(c["res"]), std=4.0),
                    w=_normal(g, c["d"], std=0.2) + (0.0 if c["unit_offset"] else 1.0))
    b, v, n = c["b"], c["v"], c["prompt"] + c["generated"]
    # a text's tokens come in very unequal numbers, a few of them often
    hist = (v * torch.rand(b * n, generator=g, device=DEV) ** 4).int().clamp_max(v - 1)
    s = dict(logits=_normal(g, b, v, dtype=_type(c["src"]), std=3.0), hist=hist,
             hist_start=torch.arange(0, b * n + 1, n, dtype=torch.int32, device=DEV),
             n_prompt=torch.full((b,), c["prompt"], dtype=torch.int32, device=DEV),
             repetition=torch.rand(b, generator=g, device=DEV) * 0.5 + 0.8,
             frequency=torch.rand(b, generator=g, device=DEV) * 0.5,
             presence=torch.rand(b, generator=g, device=DEV) - 0.3,
             bias_ids=torch.cat([torch.randperm(v, generator=g, device=DEV)[: c["biases"]] for _ in range(b)]).int(),
             bias=_normal(g, b * min(v, c["biases"]), std=4.0),
             bias_start=torch.arange(0, b * min(v, c["biases"]) + 1, min(v, c["biases"]), dtype=torch.int32, device=DEV))
    if c["grammar"]:
        s["mask"] = torch.randint(-2**31, 2**31, (b, (v + 31) // 32), generator=g, device=DEV, dtype=torch.int64).int()
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    c = case
    if c["op"] == "append":
        hq, hkv, d, t = c["hq"], c["hkv"], c["d"], c["t"]
        q, k, v = s["qkv"].split([hq * d, hkv * d, hkv * d], 1)
        s.update(q_in=q.view(t, hq, d), k_in=k.view(t, hkv, d), v_in=v.view(t, hkv, d))
    if own:
        import xdna_engine_b200 as X
        s["X"] = X
        if c["op"] in ("attention", "append"):
            s["cache"] = X.PagedCache(X.Device(0), s["k"], s["v"], s.get("k_scale"), s.get("v_scale"),
                                      max_seqs=c.get("b") or c["streams"])
        # the buffers that a decode loop keeps
        if c["op"] == "attention":
            s["out"] = torch.empty(c["b"], c["hq"], c["d"], dtype=BF16, device=DEV)
            s["lse"] = torch.empty(c["b"], c["hq"], device=DEV) if c["lse"] else None
        elif c["op"] == "append":
            s["out"] = torch.empty(c["t"], c["hq"], c["d"], dtype=BF16, device=DEV)
        elif c["op"] == "norm":
            s["q8"] = torch.empty(c["m"], c["d"], dtype=I8, device=DEV)
            s["scale"] = torch.empty(c["m"], device=DEV)
            s["res_out"] = torch.empty_like(s["res"])
        else:
            s["out"] = torch.empty(c["b"], c["v"], device=DEV)
            s["ids"] = torch.empty(c["b"], dtype=torch.int64, device=DEV)
    return s


# -------------------------------------------------------------------------------- one pass
def _paged(pool, scale, table):
    """The streams' rows [b][hkv][n][d] in 32 bits."""
    t = table.clamp_min(0)
    x = pool[t].float()                                   # [b][pages][hkv][page][d]
    if scale is not None:
        x = x * scale[t][..., None]
    b, p, h, ps, d = x.shape
    return x.transpose(1, 2).reshape(b, h, p * ps, d)


def _attention(s):
    c = s["case"]
    b, hq, hkv, d = c["b"], c["hq"], c["hkv"], c["d"]
    k, v = (_paged(s[x], s.get(x + "_scale"), s["table"]) for x in "kv")
    q = s["q"].float().view(b, hkv, hq // hkv, d)
    pos = torch.arange(k.shape[2], device=DEV)
    live = pos[None] < s["lens"][:, None]
    if c["window"]:
        live &= pos[None] >= s["lens"][:, None] - c["window"]
    sc = (q @ k.transpose(2, 3)) * d ** -0.5
    sc = sc.masked_fill(~live[:, None, None], -math.inf)
    m = sc.amax(-1, keepdim=True)
    p = torch.exp(sc - m.clamp_min(-3e38))
    l = p.sum(-1, keepdim=True)
    o = torch.where(l > 0, (p @ v) / l, 0.0).view(b, hq, d).to(BF16)
    if not c["lse"]:
        return {"out": o}
    return {"out": o, "lse": (m + torch.log(l)).view(b, hq)}


def _rotate(x, cs, rot, interleaved):
    cos, sin = cs[:, None, : rot // 2], cs[:, None, rot // 2:]
    if interleaved:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
    else:
        a, b = x[..., : rot // 2], x[..., rot // 2: rot]
    u, w = a * cos - b * sin, b * cos + a * sin
    y = torch.stack([u, w], -1).flatten(-2) if interleaved else torch.cat([u, w], -1)
    return torch.cat([y, x[..., rot:]], -1)


def _quantise(x):
    """Rows to whole numbers of 8 bits and a scale, the greatest magnitude at 127."""
    top = x.abs().amax(-1, keepdim=True)
    q = torch.round(x * torch.where(top > 0, 127.0 / top, 0.0))
    return q, torch.where(top > 0, top / 127.0, 1.0)[..., 0]


def _append(s):
    c = s["case"]
    cs = s["rope"][s["pos"]]
    q = _rotate(s["q_in"].float(), cs, c["rot"], c["interleaved"]).to(BF16)
    k, v = _rotate(s["k_in"].float(), cs, c["rot"], c["interleaved"]), s["v_in"].float()
    page, at = s["table"][s["seq"], s["pos"] // c["page"]], s["pos"] % c["page"]
    if c["kv"] == "bf16":
        s["k"][page, :, at] = k.to(BF16)
        s["v"][page, :, at] = v.to(BF16)
    else:
        for name, x in (("k", k), ("v", v)):
            whole, scale = _quantise(x)
            s[name][page, :, at] = whole.to(I8)
            s[name + "_scale"][page, :, at] = scale
    return _appended(s, q)


def _appended(s, q):
    """The rotated queries and the pool: an 8-bit one as the values that it stands for."""
    if s["case"]["kv"] == "bf16":
        return {"q": q, "k": s["k"], "v": s["v"]}
    return {"q": q, "k": s["k"] * s["k_scale"][..., None], "v": s["v"] * s["v_scale"][..., None]}


def _norm(s):
    c = s["case"]
    r = s["x"].float() + s["res"].float()
    inv = torch.rsqrt((r * r).mean(-1, keepdim=True) + 1e-6)
    # whole numbers do not depend on the row's own factor `inv`, only the scale does
    whole, scale = _quantise(r * (s["w"] + 1.0 if c["unit_offset"] else s["w"]))
    scale = scale * inv[:, 0]
    return {"y": whole * scale[:, None], "scale": scale, "res": r.to(_type(c["res"]))}


def _logits(s):
    c = s["case"]
    b, v = c["b"], c["v"]
    x = s["logits"].float()
    n = c["prompt"] + c["generated"]
    h = s["hist"].view(b, n).long()
    one = torch.ones((), device=DEV).expand(b, n)
    seen = torch.zeros(b, v, device=DEV).scatter_add_(1, h, one) > 0
    count = torch.zeros(b, v, device=DEV).scatter_add_(1, h[:, c["prompt"]:], one[:, c["prompt"]:])
    rep = s["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
    x = x - count * s["frequency"][:, None]
    x = x - torch.where(count > 0, s["presence"][:, None], 0.0)
    x = x.scatter_add(1, s["bias_ids"].view(b, -1).long(), s["bias"].view(b, -1))
    if c["grammar"]:
        bit = torch.arange(32, device=DEV, dtype=torch.int32)
        allowed = ((s["mask"][..., None] >> bit) & 1).view(b, -1)[:, :v] != 0
        x = x.masked_fill(~allowed, -math.inf)
    top = x.amax(1, keepdim=True)
    at = torch.where(x == top, torch.arange(v, device=DEV), v).amin(1)
    return {"logits": x, "ids": torch.where(top[:, 0] > -math.inf, at, -1)}


def run(s):
    c = s["case"]
    op = c["op"]
    if not own:
        return {"attention": _attention, "append": _append, "norm": _norm, "logits": _logits}[op](s)
    if op == "attention":
        s["cache"].attend(s["q"], s["table"], s["lens"], window=c["window"], out=s["out"], lse=s["lse"])
        return {"out": s["out"], "lse": s["lse"]} if c["lse"] else {"out": s["out"]}
    if op == "append":
        s["cache"].append(s["q_in"], s["k_in"], s["v_in"], s["seq"], s["pos"], s["table"], rope=s["rope"],
                          interleaved=c["interleaved"], q_out=s["out"])
        return _appended(s, s["out"])
    if op == "norm":
        s["X"].rmsnorm_residual_i8(s["x"], s["w"], residual=s["res"], eps=1e-6, unit_offset=c["unit_offset"],
                                   q8=s["q8"], scale=s["scale"], residual_out=s["res_out"])
        return {"y": s["q8"] * s["scale"][:, None], "scale": s["scale"], "res": s["res_out"]}
    s["X"].process_logits(s["logits"], history=s["hist"], history_start=s["hist_start"], n_prompt=s["n_prompt"],
                          repetition=s["repetition"], frequency=s["frequency"], presence=s["presence"],
                          bias_ids=s["bias_ids"], bias=s["bias"], bias_start=s["bias_start"], mask=s.get("mask"),
                          out=s["out"], ids=s["ids"])
    return {"logits": s["out"], "ids": s["ids"]}


# ------------------------------------------------------------------------- 64-bit definitions
def exact(case, seed):
    """Stream by stream and row by row from the definitions, in 64 bits."""
    c, s = case, _inputs(case, seed)
    f64 = torch.float64
    if c["op"] == "attention":
        outs, lses = [], []
        group = c["hq"] // c["hkv"]
        for i, n in enumerate(s["lens"].tolist()):
            lo = max(0, n - c["window"]) if c["window"] else 0
            if n == lo:
                outs.append(torch.zeros(c["hq"], c["d"], dtype=f64, device=DEV))
                lses.append(torch.full((c["hq"],), -math.inf, dtype=f64, device=DEV))
                continue
            at = torch.arange(lo, n, device=DEV)
            page, off = s["table"][i, at // c["page"]].long(), at % c["page"]
            heads, parts = [], []
            for h in range(c["hkv"]):
                k, v = s["k"][page, h, off].to(f64), s["v"][page, h, off].to(f64)
                if c["kv"] == "int8":
                    k = k * s["k_scale"][page, h, off].to(f64)[:, None]
                    v = v * s["v_scale"][page, h, off].to(f64)[:, None]
                a = s["q"][i, h * group:(h + 1) * group].to(f64) @ k.T / math.sqrt(c["d"])
                heads.append(torch.softmax(a, 1) @ v)
                parts.append(torch.logsumexp(a, 1))
            outs.append(torch.cat(heads))
            lses.append(torch.cat(parts))
        return {"out": torch.stack(outs), "lse": torch.stack(lses)} if c["lse"] else {"out": torch.stack(outs)}
    if c["op"] == "append":
        hq, hkv, d, rot = c["hq"], c["hkv"], c["d"], c["rot"]
        x = s["qkv"].to(f64).view(c["t"], hq + 2 * hkv, d)
        cs = s["rope"][s["pos"].long()].to(f64)
        turn = torch.complex(cs[:, : rot // 2], cs[:, rot // 2:])[:, None]
        i = torch.arange(rot // 2, device=DEV)
        first, second = (2 * i, 2 * i + 1) if c["interleaved"] else (i, i + rot // 2)
        y = x[:, : hq + hkv]
        z = torch.complex(y[..., first], y[..., second]) * turn
        y = y.clone()
        y[..., first], y[..., second] = z.real, z.imag
        page, at = s["table"][s["seq"].long(), s["pos"].long() // c["page"]].long(), s["pos"].long() % c["page"]
        out = {"q": y[:, :hq]}
        for name, rows in (("k", y[:, hq:]), ("v", x[:, hq + hkv:])):
            if c["kv"] == "int8":
                step = rows.abs().amax(-1, keepdim=True) / 127
                rows = torch.round(rows / step) * step
            pool = torch.zeros(s[name].shape, dtype=f64, device=DEV)
            pool[page, :, at] = rows
            out[name] = pool
        return out
    if c["op"] == "norm":
        r = s["x"].to(f64) + s["res"].to(f64)
        y = r / torch.sqrt(r.square().sum(1, keepdim=True) / c["d"] + 1e-6)
        y = y * (1 + s["w"].to(f64) if c["unit_offset"] else s["w"].to(f64))
        step = y.abs().amax(1) / 127
        return {"y": torch.round(y / step[:, None]) * step[:, None], "scale": step, "res": r}
    rows = []
    n = c["prompt"] + c["generated"]
    for i in range(c["b"]):
        x = s["logits"][i].to(f64)
        h = s["hist"][i * n:(i + 1) * n].long()
        seen = torch.bincount(h, minlength=c["v"]) > 0
        count = torch.bincount(h[c["prompt"]:], minlength=c["v"]).to(f64)
        rep = s["repetition"][i].to(f64)
        x = torch.where(seen & (x > 0), x / rep, torch.where(seen, x * rep, x))
        x = x - count * s["frequency"][i].to(f64) - (count > 0) * s["presence"][i].to(f64)
        m = min(c["v"], c["biases"])
        x[s["bias_ids"][i * m:(i + 1) * m].long()] += s["bias"][i * m:(i + 1) * m].to(f64)
        if c["grammar"]:
            j = torch.arange(c["v"], device=DEV)
            x[((s["mask"][i].long() & 0xFFFFFFFF)[j // 32] >> (j % 32)) & 1 == 0] = -math.inf
        rows.append(x)
    return {"logits": torch.stack(rows), "ids": None}
