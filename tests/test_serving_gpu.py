"""The serving ops (paged cache, residual RMS norm with int8 rows, logits) on the GPU against plain
implementations in 64 bits of the definitions in include/xdna_b200.h.

Tolerances come from the arithmetic the header states, not from observed errors:
* attention: the output is rounded once to bf16 (8 significant bits: 2^-8 of its value).  Before that, a score of D
  products accumulated in f32 is off by at most D 2^-23 sum|q_i k_i| scale (2^-23: the tensor core
  may truncate), which scales its weight by exp of that; a weight kept to 16 bits of mantissa adds
  2^-16, hardware exponentials and the joins 2^-19, and f32 sums over n terms n 2^-23.  All of these
  scale sum p|v| / sum p.
* append: the rotation's products and sums are f32 (2^-22 (|a| + |b|)), bf16 rounding 2^-8;
  int8 rows lie within half a step, and 127 steps of f32 rounding.
* norm: the mean of D squares in f32 is off by at most D 2^-24, its root by half of that.
* logits: every step is one f32 operation that numpy repeats bit for bit."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

BF16, F32, F64, I8, I32 = torch.bfloat16, torch.float32, torch.float64, torch.int8, torch.int32


@pytest.fixture(scope="module")
def X():
    import xdna_engine_b200 as X
    from xdna_engine_b200 import _build
    _build.build()
    return X


@pytest.fixture(scope="module")
def dev(X):
    d = X.Device(0)
    yield d
    d.close()


def rng(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


# ------------------------------------------------------------------------------- attention
def make_pool(g, kv, lens, hkv, page, d, layers=1, layout="hnd"):
    """Pools whose rows past the streams' lengths hold NaN (bf16) or wild scales (int8), and a block
    table whose unused entries are out of range."""
    n_pages = sum(-(-max(n, 0) // page) for n in lens) + 3
    width = max(1, max(-(-n // page) for n in lens))
    ids = torch.randperm(n_pages, generator=g, device="cuda").int()
    table = torch.full((len(lens), width), 2**31 - 1, dtype=I32, device="cuda")
    used = torch.zeros(n_pages, page, dtype=torch.bool, device="cuda")
    at = 0
    for b, n in enumerate(lens):
        p = -(-max(n, 0) // page)
        table[b, :p] = ids[at:at + p]
        for j in range(p):
            used[int(ids[at + j]), : min(page, n - j * page)] = True
        at += p
    shape = (layers, n_pages, hkv, page, d)

    def lay(t):
        if layout == "nhd":                # [page][slot][head][c]
            return t.transpose(2, 3).contiguous().transpose(2, 3)
        return t

    keep = used[None, :, None, :, None]
    if kv == "bf16":
        k, v = (torch.randn(shape, generator=g, device="cuda") for _ in "kv")
        k, v = (lay(torch.where(keep, t, math.nan).to(BF16)) for t in (k, v))
        return dict(k=k, v=v, k_scale=None, v_scale=None, table=table)
    k, v = (lay(torch.randint(-127, 128, shape, generator=g, device="cuda", dtype=I8)) for _ in "kv")
    ks, vs = (torch.where(keep[..., 0], torch.rand(shape[:4], generator=g, device="cuda") * 0.02 + 1e-3, math.nan)
              for _ in "kv")
    return dict(k=k, v=v, k_scale=ks.contiguous(), v_scale=vs.contiguous(), table=table)


def attention_64(q, p, lens, scale, window, layer=0):
    """(out, lse, bound of |out - exact|, bound of |lse - exact|) from the definition in 64 bits."""
    hkv, page = p["k"].shape[2], p["k"].shape[3]
    hq, d = q.shape[1:]
    res = []
    for b, n in enumerate(lens):
        lo = max(0, n - window) if window else 0
        if n <= lo:
            z = torch.zeros(hq, d, dtype=F64, device="cuda")
            res.append((z, z[:, 0] - math.inf, z, z[:, 0]))
            continue
        pos = torch.arange(lo, n, device="cuda")
        pg, at = p["table"][b, pos // page].long(), pos % page
        rows = []
        for h in range(hq):
            hk = h // (hq // hkv)
            k, v = p["k"][layer, pg, hk, at].to(F64), p["v"][layer, pg, hk, at].to(F64)
            if p["k_scale"] is not None:
                k = k * p["k_scale"][layer, pg, hk, at].to(F64)[:, None]
                v = v * p["v_scale"][layer, pg, hk, at].to(F64)[:, None]
            qh = q[b, h].to(F64)
            s = k @ qh * scale
            w = torch.softmax(s, 0)
            o = w @ v
            ds = float((k.abs() @ qh.abs()).max()) * scale * (d + 4) * 2.0**-23
            rel = 2 * ds + 2.0**-16 + 2.0**-19 + (n - lo) * 2.0**-23
            lse = torch.logsumexp(s, 0)
            rows.append((o, lse, o.abs() * 1.01 * 2.0**-8 + rel * (w @ v.abs()) + 1e-30,
                         ds + (n - lo + 64) * 2.0**-23 + lse.abs() * 2.0**-22 + 2.0**-19))
        res.append(tuple(torch.stack(x) for x in zip(*rows)))
    return tuple(torch.stack(x) for x in zip(*res))


def check_attention(got, lse, want):
    o, l, bo, bl = want
    assert torch.isfinite(got.float()).all()
    far = (got.to(F64) - o).abs() - bo
    assert float(far.max()) <= 0, float(far.max())
    if lse is not None:
        none = torch.isinf(l)
        assert torch.equal(torch.isinf(lse), none) and bool((lse[none] < 0).all())
        far = (lse.to(F64) - l).abs()[~none] - bl[~none]
        assert not far.numel() or float(far.max()) <= 0, float(far.max())


HEADS = [(1, 1), (4, 1), (12, 12), (32, 8), (6, 2), (16, 1), (40, 2), (14, 2)]


@pytest.mark.parametrize("kv", ["bf16", "int8"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("hq,hkv", HEADS)
def test_attention_heads(X, dev, hq, hkv, d, kv):
    g = rng(hq * 1000 + d)
    lens = [0, 1, 2, 15, 16, 17, 63, 64, 65, 130, 301]
    p = make_pool(g, kv, lens, hkv, 16, d)
    q = torch.randn(len(lens), hq, d, generator=g, device="cuda").mul(1.5).to(BF16)
    c = X.PagedCache(dev, p["k"], p["v"], p["k_scale"], p["v_scale"], max_seqs=len(lens))
    lse = torch.full((len(lens), hq), math.nan, device="cuda")
    out = c.attend(q, p["table"], torch.tensor(lens, dtype=I32, device="cuda"), lse=lse)
    c.check()
    check_attention(out, lse, attention_64(q, p, lens, d ** -0.5, 0))
    assert not out[0].any()


@pytest.mark.parametrize("kv", ["bf16", "int8"])
@pytest.mark.parametrize("page", [1, 7, 8, 24, 64, 100, 4096])
@pytest.mark.parametrize("window", [0, 1, 16, 50, 513])
def test_attention_pages_and_windows(X, dev, page, window, kv):
    g = rng(page * 7 + window)
    lens = [3, 600, 0, 99, 1025]
    p = make_pool(g, kv, lens, 2, page, 64, layers=2)
    q = torch.randn(len(lens), 8, 64, generator=g, device="cuda").to(BF16)
    c = X.PagedCache(dev, p["k"], p["v"], p["k_scale"], p["v_scale"], max_seqs=16)
    lse = torch.empty(len(lens), 8, device="cuda")
    out = c.attend(q, p["table"], torch.tensor(lens, dtype=I32, device="cuda"), scale=0.2, window=window, layer=1,
                   lse=lse)
    c.check()
    check_attention(out, lse, attention_64(q, p, lens, 0.2, window, layer=1))


@pytest.mark.parametrize("kv", ["bf16", "int8"])
@pytest.mark.parametrize("d,hq,hkv,lens", [(64, 8, 1, [20000]), (128, 8, 8, [9000, 12, 4097]),
                                           (256, 4, 1, [33333]), (128, 32, 8, [1] * 150 + [7000] + [33] * 100),
                                           (64, 4, 4, [300] * 400), (128, 16, 1, [5000] * 3)])
def test_attention_long_and_many(X, dev, d, hq, hkv, lens, kv):
    g = rng(d + len(lens))
    p = make_pool(g, kv, lens, hkv, 16, d)
    q = torch.randn(len(lens), hq, d, generator=g, device="cuda").to(BF16)
    c = X.PagedCache(dev, p["k"], p["v"], p["k_scale"], p["v_scale"], max_seqs=len(lens))
    lse = torch.empty(len(lens), hq, device="cuda")
    t = torch.tensor(lens, dtype=I32, device="cuda")
    out = c.attend(q, p["table"], t, lse=lse)
    c.check()
    few = sorted({0, len(lens) // 3, lens.index(max(lens)), len(lens) - 1})
    sub = dict(p, table=p["table"][few])
    check_attention(out[few], lse[few], attention_64(q[few], sub, [lens[i] for i in few], d ** -0.5, 0))
    again = c.attend(q, p["table"], t)
    assert torch.equal(out, again)                       # the join's order does not vary


def test_attention_strides(X, dev):
    """Pools as [page][slot][head][c] and as K | V in one buffer; q as rows of a wider product."""
    g = rng(5)
    lens = [77, 300]
    t = torch.tensor(lens, dtype=I32, device="cuda")
    p = make_pool(g, "bf16", lens, 2, 16, 128, layout="nhd")
    wide = torch.randn(2, 1024 + 64, generator=g, device="cuda").to(BF16)
    q = wide[:, 64:64 + 8 * 128].view(2, 8, 128)
    want = attention_64(q, p, lens, 128 ** -0.5, 0)
    c = X.PagedCache(dev, p["k"][0], p["v"][0])
    check_attention(c.attend(q, p["table"], t), None, want)
    both = torch.stack([p["k"][0].contiguous(), p["v"][0].contiguous()], 1)
    c = X.PagedCache(dev, both[:, 0], both[:, 1])
    table = torch.full((2, 40), -7, dtype=I32, device="cuda")
    table[:, : p["table"].shape[1]] = p["table"]
    check_attention(c.attend(q, table[:, : p["table"].shape[1]], t), None, want)
    c.check()


def test_attention_negative_and_spiked(X, dev):
    """A negative length counts as none; scores of +-1e4 and equal maxima stay exact softmaxes."""
    g = rng(6)
    lens = [40, 64]
    p = make_pool(g, "bf16", lens, 1, 16, 64)
    t = torch.tensor([-1, 64], dtype=I32, device="cuda")
    q = torch.randn(2, 4, 64, generator=g, device="cuda").mul(400.0).to(BF16)
    c = X.PagedCache(dev, p["k"], p["v"])
    lse = torch.empty(2, 4, device="cuda")
    out = c.attend(q, p["table"], t, lse=lse)
    check_attention(out, lse, attention_64(q, p, [0, 64], 0.125, 0))
    q.zero_()
    out = c.attend(q, p["table"], t)
    check_attention(out, None, attention_64(q, p, [0, 64], 0.125, 0))
    # a NaN among the live keys makes that stream's result NaN and no other's
    p["k"][0, int(p["table"][1, 2]), 0, 5] = math.nan
    t = torch.tensor(lens, dtype=I32, device="cuda")
    q = torch.randn(2, 4, 64, generator=g, device="cuda").to(BF16)
    out = c.attend(q, p["table"], t)
    assert torch.isnan(out[1].float()).all() and torch.isfinite(out[0].float()).all()


def test_int8_rows_keep_a_nan(X, dev):
    """A NaN in an appended row, or a NaN scale of a live key or value, shows in the result; in the rows
    past a stream's length it does not."""
    g = rng(13)
    pools = [torch.zeros(4, 1, 16, 64, dtype=I8, device="cuda") for _ in "kv"]
    scales = [torch.full((4, 1, 16), math.nan, device="cuda") for _ in "kv"]
    c = X.PagedCache(dev, *pools, *scales)
    table = torch.tensor([[0], [1]], dtype=I32, device="cuda")
    pos = torch.arange(8, dtype=I32, device="cuda")
    for stream in (0, 1):
        k, v = (torch.randn(8, 1, 64, generator=g, device="cuda") for _ in "kv")
        if stream:
            v[5, 0, 7] = math.nan
        c.append(None, k, v, torch.full_like(pos, stream), pos, table)
    q = torch.randn(2, 4, 64, generator=g, device="cuda").to(BF16)
    out = c.attend(q, table, torch.tensor([8, 8], dtype=I32, device="cuda")).float()
    assert torch.isfinite(out[0]).all() and torch.isnan(out[1]).all()
    out = c.attend(q, table, torch.tensor([8, 5], dtype=I32, device="cuda")).float()
    assert torch.isfinite(out).all()
    scales[0][0, 0, 3] = math.nan
    out = c.attend(q, table, torch.tensor([8, 5], dtype=I32, device="cuda")).float()
    assert torch.isnan(out[0]).all() and torch.isfinite(out[1]).all()
    c.check()


def test_attention_past_32_bits(X, dev):
    """Pages whose elements lie past 2^31 in the pool."""
    g = rng(7)
    d, hkv, page = 128, 8, 64
    n_pages = 2**31 // (d * hkv * page) + 40
    pool = torch.empty(n_pages, hkv, page, d, dtype=BF16, device="cuda")
    lens = [130, 640]
    ids = torch.tensor([[n_pages - 1, n_pages - 7, n_pages - 3] + [-1] * 7,
                        [n_pages - 20 + i for i in range(9)] + [0]], dtype=I32, device="cuda")
    for i in ids.flatten().tolist():
        if i >= 0:
            pool[i] = torch.randn(hkv, page, d, generator=g, device="cuda").to(BF16)
    q = torch.randn(2, 16, d, generator=g, device="cuda").to(BF16)
    c = X.PagedCache(dev, pool, pool)
    out = c.attend(q, ids, torch.tensor(lens, dtype=I32, device="cuda"))
    p = dict(k=pool[None], v=pool[None], k_scale=None, v_scale=None, table=ids)
    check_attention(out, None, attention_64(q, p, lens, d ** -0.5, 0))
    new = torch.randn(1, hkv, d, generator=g, device="cuda").to(BF16)
    c.append(None, new, new, None, torch.tensor([129], dtype=I32, device="cuda"), ids[:1])
    assert torch.equal(pool[n_pages - 3, :, 1], new[0])
    c.check()


def test_attention_bad_pages_are_reported(X, dev):
    """A page outside the pool is left out of the softmax and reported; other streams are unharmed."""
    g = rng(8)
    lens = [100, 100]
    p = make_pool(g, "bf16", lens, 2, 16, 64)
    t = torch.tensor(lens, dtype=I32, device="cuda")
    q = torch.randn(2, 4, 64, generator=g, device="cuda").to(BF16)
    c = X.PagedCache(dev, p["k"], p["v"])
    want = attention_64(q, p, lens, 0.125, 0)
    for bad in (-1, p["k"].shape[1], 2**31 - 1):
        table = p["table"].clone()
        table[0, 2] = bad
        out = c.attend(q, table, t)
        with pytest.raises(X.XdnaError, match="page id"):
            c.check()
        check_attention(out[1:], None, tuple(w[1:] for w in want))
        assert torch.isfinite(out.float()).all()
    lse = torch.empty(2, 4, device="cuda")
    out = c.attend(q, torch.stack([torch.full_like(p["table"][0], -3), p["table"][1]]), t, lse=lse)
    with pytest.raises(X.XdnaError, match="page id"):
        c.check()
    assert not out[0].any() and bool((lse[0] == -math.inf).all())          # nothing left: zeros
    check_attention(out[1:], lse[1:], tuple(w[1:] for w in want))
    out = c.attend(q, p["table"], torch.tensor([100, 113], dtype=I32, device="cuda"))
    with pytest.raises(X.XdnaError, match="position"):
        c.check()
    check_attention(out[:1], None, tuple(w[:1] for w in want))
    c.check()


def test_attention_streams_and_graphs(X, dev):
    """On a stream of its own, behind work still running there, and replayed from a graph with
    new lengths and tables in place."""
    g = rng(9)
    lens = [700, 30, 2000]
    p = make_pool(g, "bf16", lens, 2, 16, 128)
    c = X.PagedCache(dev, p["k"], p["v"])
    q = torch.randn(3, 8, 128, generator=g, device="cuda").to(BF16)
    want = attention_64(q, p, lens, 128 ** -0.5, 0)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    late, out = torch.zeros_like(q), torch.empty_like(q)
    t = torch.zeros(3, dtype=I32, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        big = torch.randn(4096, 4096, device="cuda")
        for _ in range(8):
            big = big @ big * 1e-2
        late.copy_(q)
        t.copy_(torch.tensor(lens, dtype=I32))
        c.attend(late, p["table"], t, out=out)
    s.synchronize()
    check_attention(out, None, want)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        c.attend(late, p["table"], t, out=out)
    for cut in (0, 3, 30):
        now = [max(0, n - cut) for n in lens]
        t.copy_(torch.tensor(now, dtype=I32))
        gr.replay()
        torch.cuda.synchronize()
        check_attention(out, None, attention_64(q, p, now, 128 ** -0.5, 0))


# ----------------------------------------------------------------------------------- append
def rotated_64(x, pos, table, rot, interleaved):
    """Rotation in 64 bits, and |a| + |b| of each component's pair."""
    cs = table[pos.long()].to(F64)[:, None]
    cos, sin = cs[..., : rot // 2], cs[..., rot // 2:]
    y = x.to(F64).clone()
    m = y.abs()
    i = torch.arange(rot // 2, device="cuda")
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
    u, w = y[..., a].clone(), y[..., b].clone()
    y[..., a], y[..., b] = u * cos - w * sin, w * cos + u * sin
    m[..., a] = m[..., b] = u.abs() + w.abs()
    return y, m


@pytest.mark.parametrize("kv", ["bf16", "int8"])
@pytest.mark.parametrize("src", [BF16, F32])
@pytest.mark.parametrize("d,rot,interleaved", [(64, 64, False), (64, 16, True), (128, 128, False), (128, 128, True),
                                               (128, 48, False), (256, 256, False), (256, 64, True), (128, 0, False)])
@pytest.mark.parametrize("hq,hkv", [(1, 1), (6, 2), (7, 7)])
def test_append(X, dev, hq, hkv, d, rot, interleaved, src, kv):
    g = rng(d + rot + hq)
    n, page, streams, layers = 53, 7, 3, 2
    qkv = torch.randn(n, (hq + 2 * hkv) * d, generator=g, device="cuda").to(src)
    qkv[5] = 0                                           # a zero row: scale 1
    q, k, v = (t.view(n, -1, d) for t in qkv.split([hq * d, hkv * d, hkv * d], 1))
    seq = torch.randint(0, streams, (n,), generator=g, device="cuda", dtype=I32)
    pos = torch.randperm(200, generator=g, device="cuda")[:n].int()
    pos[11] = -1
    table = torch.randperm(streams * 29, generator=g, device="cuda").int().view(streams, 29)
    shape = (layers, streams * 29, hkv, page, d)
    if kv == "bf16":
        pk, pv = (torch.randn(shape, generator=g, device="cuda").to(BF16) for _ in "kv")
        ks = vs = None
    else:
        pk, pv = (torch.randint(-127, 128, shape, generator=g, device="cuda", dtype=I8) for _ in "kv")
        ks, vs = (torch.rand(shape[:4], generator=g, device="cuda") for _ in "kv")
    before = [None if t is None else t.clone() for t in (pk, pv, ks, vs)]
    rope = X.rope_table(200, rot) if rot else None
    c = X.PagedCache(dev, pk, pv, ks, vs)
    got = c.append(q, k, v, seq, pos, table, rope=rope, interleaved=interleaved, layer=1)
    c.check()
    live = pos >= 0
    q64, qm = rotated_64(q, pos.clamp_min(0), rope, rot, interleaved) if rot else (q.to(F64), q.to(F64).abs())
    k64, km = rotated_64(k, pos.clamp_min(0), rope, rot, interleaved) if rot else (k.to(F64), k.to(F64).abs())
    assert not got[~live].any()
    far = (got.to(F64) - q64).abs() - (q64.abs() * 1.01 * 2.0**-8 + qm * 2.0**-22)
    assert float(far[live].max()) <= 0
    pg = table[seq.long(), (pos.clamp_min(0) // page).long()].long()[live]
    at = (pos % page).long()[live]
    for pool, sc, x, m, old, old_sc in ((pk, ks, k64, km, before[0], before[2]),
                                        (pv, vs, v.to(F64), v.to(F64).abs(), before[1], before[3])):
        x, m, rows = x[live], m[live], pool[1, pg, :, at]
        if kv == "bf16":
            far = (rows.to(F64) - x).abs() - (x.abs() * 1.01 * 2.0**-8 + m * 2.0**-22)
        else:
            step = sc[1, pg, :, at].to(F64)
            top = x.abs().amax(-1)
            assert float(((step - torch.where(top > 0, top / 127, 1.0)).abs() - m.amax(-1) * 2.0**-22).max()) <= 0
            assert int(rows.abs().max()) <= 127
            far = (rows.to(F64) * step[..., None] - x).abs() - step[..., None] * (0.5 + 2.0**-14) - m * 2.0**-22
            old_sc[1, pg, :, at] = sc[1, pg, :, at]
            assert torch.equal(sc, old_sc)
        assert float(far.max()) <= 0
        old[1, pg, :, at] = pool[1, pg, :, at]
        assert torch.equal(pool.view(torch.int16 if kv == "bf16" else I8),
                           old.view(torch.int16 if kv == "bf16" else I8))          # nothing else was written


def test_append_one_token_of_any_stride(X, dev):
    """A single token's strides say nothing: x[None] of a transposed product is taken."""
    g = rng(12)
    pool = torch.zeros(2, 2, 16, 64, dtype=BF16, device="cuda")
    c = X.PagedCache(dev, pool, pool.clone())
    k = torch.randn(2, 64, generator=g, device="cuda").to(BF16)
    odd = k.as_strided((1, 2, 64), (1, 64, 1))
    c.append(odd, odd, odd, None, torch.tensor([3], dtype=I32, device="cuda"), torch.tensor([[1]], dtype=I32, device="cuda"))
    c.check()
    assert torch.equal(pool[1, :, 3], k) and int((pool != 0).any(-1).sum()) == 2


def test_append_bad_inputs_are_reported(X, dev):
    """Rows with a page, position or stream out of range are skipped and reported."""
    g = rng(3)
    k = torch.randn(4, 2, 64, generator=g, device="cuda").to(BF16)
    pool = torch.zeros(6, 2, 8, 64, dtype=BF16, device="cuda")
    c = X.PagedCache(dev, pool, pool.clone())
    table = torch.tensor([[0, 1], [6, -1]], dtype=I32, device="cuda")
    i32 = lambda *x: torch.tensor(x, dtype=I32, device="cuda")  # noqa: E731
    cases = [(i32(0, 0, 1, 0), i32(0, 1, 0, 9), None, "page id"), (i32(0, 0, 0, 0), i32(0, 1, 16, 9), None, "position"),
             (i32(0, 0, 2, 0), i32(0, 1, 0, 9), None, "stream"), (i32(0, 0, -1, 0), i32(0, 1, 0, 9), None, "stream"),
             (i32(0, 0, 0, 0), i32(0, 1, 12, 9), X.rope_table(12, 64), "position")]
    for seq, pos, rope, what in cases:
        pool.zero_()
        c.append(k, k, k, seq, pos, table, rope=rope)
        with pytest.raises(X.XdnaError, match=what):
            c.check()
        assert int((pool != 0).any(-1).any(1).sum()) == 3
    c.check()


# ------------------------------------------------------------------------------------- norm
@pytest.mark.parametrize("x_type", [BF16, F32])
@pytest.mark.parametrize("res_type", [BF16, F32, None])
@pytest.mark.parametrize("m,d", [(1, 1), (3, 7), (1, 1152), (5, 64), (2, 768), (300, 1000), (4, 1024), (7, 4096),
                                 (2, 4097), (3, 8192), (2, 16384), (2, 16383)])
@pytest.mark.parametrize("unit", [False, True])
def test_norm(X, m, d, x_type, res_type, unit):
    g = rng(m * d)
    x = torch.randn(m, d + 8, generator=g, device="cuda").to(x_type)[:, :d]
    res = None if res_type is None else torch.randn(m, d, generator=g, device="cuda").mul(3).to(res_type)
    w = torch.randn(d, generator=g, device="cuda")
    if m > 2:
        x[1] = 0
        if res is not None:
            res[1] = 0
    y = torch.empty(m, d, dtype=BF16, device="cuda")
    q8, scale, out = X.rmsnorm_residual_i8(x, w, residual=res, eps=1e-5, unit_offset=unit, y=y)
    r = x.to(F64) if res is None else x.to(F64) + res.to(F64)
    want = r / torch.sqrt((r * r).mean(1, keepdim=True) + 1e-5) * (w.to(F64) + unit)
    slack = d * 2.0**-24 + 2.0**-20
    if res is not None:
        assert out.dtype is res_type
        assert torch.equal(out, (x.float() + res.float()).to(res_type))
    else:
        assert out is None
    wide = want.abs() * slack + (want.abs() + (want / (w.to(F64) + unit)).abs()) * 2.0**-22   # w + 1 rounds too
    assert float(((y.to(F64) - want).abs() - want.abs() * 1.01 * 2.0**-8 - wide).max()) <= 0
    top = want.abs().amax(1)
    assert float(((scale.to(F64) - torch.where(top > 0, top / 127, 1.0)).abs() - wide.amax(1)).max()) <= 0
    far = (q8.to(F64) * scale.to(F64)[:, None] - want).abs() - scale.to(F64)[:, None] * (0.5 + 2.0**-14) - wide
    assert float(far.max()) <= 0
    # in place, and without the int8 rows
    if res is not None:
        keep = res.clone()
        a, b, same = X.rmsnorm_residual_i8(x, w, residual=keep, eps=1e-5, unit_offset=unit, residual_out=keep)
        assert same is keep and torch.equal(keep, out) and torch.equal(a, q8) and torch.equal(b, scale)
    only = torch.empty_like(y)
    none = X.rmsnorm_residual_i8(x, w, residual=res, eps=1e-5, unit_offset=unit, y=only, quantize=False)
    assert none[0] is None and none[1] is None and torch.equal(only, y)


def test_norm_feeds_the_int8_product(X):
    """The rows and scales are xdna_gemm_i8's A operand with one row per clip."""
    g = rng(4)
    m, d, n = 130, 256, 512
    x = torch.randn(m, d, generator=g, device="cuda").to(BF16)
    q8, scale, _ = X.rmsnorm_residual_i8(x, torch.ones(d, device="cuda"))
    wq = torch.randint(-127, 128, (n, d), generator=g, device="cuda", dtype=I8)
    ws = torch.rand(n, generator=g, device="cuda") * 1e-2
    out = torch.empty(m, n, device="cuda")
    L = X.lib()
    assert L.xdna_gemm_i8(q8.data_ptr(), wq.data_ptr(), scale.data_ptr(), 1, ws.data_ptr(), None, 0, None, 1.0,
                          out.data_ptr(), None, m, n, d, torch.cuda.current_stream().cuda_stream) == 0
    want = (q8.to(F64) @ wq.to(F64).T) * scale.to(F64)[:, None] * ws.to(F64)
    torch.cuda.synchronize()
    assert L.xdna_gemm_check() == 0
    assert float(((out.to(F64) - want).abs() - want.abs() * 2.0**-21).max()) <= 0


# ----------------------------------------------------------------------------------- logits
def logits_plain(x, hist, n_prompt, rep, freq, pres, biases, mask):
    """Row by row in numpy f32, one rounded operation at a time."""
    y = x.astype(np.float32).copy()
    ids = []
    for b in range(y.shape[0]):
        v = y.shape[1]
        if hist is not None:
            h = np.asarray(hist[b])
            ok = (h >= 0) & (h < v)
            seen = np.bincount(h[ok], minlength=v) > 0
            np_ = 0 if n_prompt is None else n_prompt[b]
            cnt = np.bincount(h[np_:][ok[np_:]], minlength=v).astype(np.float32)
            if rep is not None:
                y[b] = np.where(seen, np.where(y[b] > 0, y[b] / rep[b], y[b] * rep[b]), y[b])
            if freq is not None:
                y[b] = np.where(cnt > 0, y[b] - cnt * freq[b], y[b])
            if pres is not None:
                y[b] = np.where(cnt > 0, y[b] - pres[b], y[b])
        if biases is not None:
            last = dict(biases[b])
            for i, val in last.items():
                if 0 <= i < v:
                    y[b, i] = np.float32(y[b, i] + np.float32(val))
        if mask is not None:
            bits = (mask[b][np.arange(v) // 32].view(np.uint32) >> (np.arange(v, dtype=np.uint32) % 32)) & 1
            y[b] = np.where(bits != 0, y[b], np.float32(-np.inf))
        z = np.where(np.isnan(y[b]), np.float32(-np.inf), y[b])
        ids.append(int(np.argmax(z)) if z.max() > -np.inf else -1)
    return y, np.array(ids, np.int64)


@pytest.mark.parametrize("src", [F32, BF16])
@pytest.mark.parametrize("b,v", [(1, 1), (3, 31), (2, 33), (5, 1000), (1, 4096), (2, 4097), (3, 50272), (2, 151937),
                                 (2, 262144)])
@pytest.mark.parametrize("what", ["all", "history", "bias", "mask", "none"])
def test_logits(X, b, v, src, what):
    r = np.random.default_rng(b * v)
    x = (r.standard_normal((b, v)) * 3).astype(np.float32)
    x.flat[:: max(1, x.size // 50)] = 0.0
    x = torch.from_numpy(x).cuda().to(src)
    kw, pl = {}, dict(hist=None, n_prompt=None, rep=None, freq=None, pres=None, biases=None, mask=None)
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    if what in ("all", "history"):
        hist = [(v * r.random(n) ** 3).astype(np.int32) for n in r.integers(0, 3000, b)]
        hist[0] = np.concatenate([hist[0], np.array([-1, v, 2**31 - 1, -2**31, 0, 0], np.int32)])
        npr = np.array([r.integers(0, len(h) + 1) for h in hist], np.int32)
        pl.update(hist=hist, n_prompt=npr, rep=(r.random(b) + 0.6).astype(np.float32),
                  freq=r.random(b).astype(np.float32), pres=(r.random(b) - 0.3).astype(np.float32))
        kw.update(history=dev(np.concatenate(hist)), history_start=dev(np.cumsum([0] + [len(h) for h in hist]).astype(np.int32)),
                  n_prompt=dev(npr), repetition=dev(pl["rep"]), frequency=dev(pl["freq"]), presence=dev(pl["pres"]))
    if what in ("all", "bias"):
        pl["biases"] = [[(int(r.integers(-1, v + 1)), float(np.float32(r.standard_normal() * 5)))
                         for _ in range(r.integers(0, 40))] for _ in range(b)]
        flat = [e for row in pl["biases"] for e in row]
        kw.update(bias_ids=dev(np.array([e[0] for e in flat] + [0], np.int32)),
                  bias=dev(np.array([e[1] for e in flat] + [9], np.float32)),
                  bias_start=dev(np.cumsum([0] + [len(row) for row in pl["biases"]]).astype(np.int32)))
    if what in ("all", "mask"):
        m = r.integers(0, 2**32, (b, (v + 31) // 32), dtype=np.uint64).astype(np.uint32).view(np.int32)
        m[-1] = 0                                        # a row whose mask leaves nothing
        pl["mask"] = m
        kw["mask"] = dev(m)
    want, ids = logits_plain(x.float().cpu().numpy(), **pl)
    out, got = X.process_logits(x, **kw)
    assert np.array_equal(out.cpu().numpy().view(np.uint32), want.view(np.uint32))
    assert np.array_equal(got.cpu().numpy(), ids)
    if src is F32:
        out2, got2 = X.process_logits(x, **kw, out=x)    # in place
        assert out2 is x and torch.equal(x, out) and torch.equal(got, got2)


@pytest.mark.parametrize("src", [F32, BF16])
@pytest.mark.parametrize("b,v", [(40, 70001), (20, 100000)])
def test_logits_long_histories(X, b, v, src):
    """Many long rows (their histories are sorted by chunk first), one of them empty, one of a single token."""
    r = np.random.default_rng(b)
    x = torch.from_numpy((r.standard_normal((b, v)) * 3).astype(np.float32)).cuda().to(src)
    hist = [(v * r.random(n) ** 3).astype(np.int32) for n in r.integers(0, 12000, b)]
    hist[3], hist[4] = hist[3][:0], np.full(9000, v - 1, np.int32)
    hist[5] = np.concatenate([hist[5], np.array([-1, v, 2**31 - 1, -2**31, 0, 0], np.int32)])
    npr = np.array([r.integers(0, len(h) + 1) for h in hist], np.int32)
    rep, freq, pres = ((r.random(b) + 0.6).astype(np.float32) for _ in range(3))
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    want, ids = logits_plain(x.float().cpu().numpy(), hist, npr, rep, freq, pres, None, None)
    out, got = X.process_logits(x, history=dev(np.concatenate(hist)),
                                history_start=dev(np.cumsum([0] + [len(h) for h in hist]).astype(np.int32)),
                                n_prompt=dev(npr), repetition=dev(rep), frequency=dev(freq), presence=dev(pres))
    assert np.array_equal(out.cpu().numpy().view(np.uint32), want.view(np.uint32))
    assert np.array_equal(got.cpu().numpy(), ids)


def test_logits_ties_and_odd_values(X):
    """Equal maxima go to the lowest id, across the whole row; NaN is never chosen and a masked NaN or
    infinity becomes -inf; +inf wins; -0 and 0 are equal."""
    v = 50273
    x = torch.zeros(6, v, device="cuda")
    x[0, [40000, 123, 50272]] = 7.0
    x[1] = -0.0
    x[1, 30000] = 0.0
    x[2, 17] = math.nan
    x[2, 20000] = 1.0
    x[3] = -math.inf
    x[4] = math.nan
    x[5, 5] = math.inf
    x[5, 3] = math.nan
    mask = torch.full((6, (v + 31) // 32), -1, dtype=I32, device="cuda")
    out, ids = X.process_logits(x)
    assert ids.tolist() == [123, 0, 20000, -1, -1, 5]
    mask[5, 0] = ~((1 << 5) | (1 << 3))
    out, ids = X.process_logits(x, mask=mask)
    assert ids.tolist() == [123, 0, 20000, -1, -1, 0]
    assert bool((out[5, [3, 5]] == -math.inf).all())


def test_logits_strides(X):
    g = rng(11)
    wide = torch.randn(3, 5000, generator=g, device="cuda")
    x = wide[:, 3:4004]
    keep = wide.clone()
    big = torch.full((3, 4099), 5.0, device="cuda")
    out, ids = X.process_logits(x, out=big[:, 1:4002])
    assert torch.equal(out, x) and torch.equal(ids, x.argmax(1)) and torch.equal(wide, keep)
    assert bool((big[:, 0] == 5).all()) and bool((big[:, 4002:] == 5).all())


# --------------------------------------------------------------------------------- refusals
def test_refusals(X, dev):
    z = lambda *s, t=BF16: torch.zeros(*s, dtype=t, device="cuda")  # noqa: E731
    pool = z(4, 2, 16, 64)
    with pytest.raises(ValueError):
        X.PagedCache(dev, pool, z(4, 2, 16, 128))
    with pytest.raises(ValueError):
        X.PagedCache(dev, pool.float(), pool.float())
    with pytest.raises(ValueError):
        X.PagedCache(dev, z(4, 2, 16, 64, t=I8), z(4, 2, 16, 64, t=I8))
    with pytest.raises(ValueError):
        X.PagedCache(dev, pool.cpu(), pool.cpu())
    with pytest.raises(X.XdnaError, match="head_dim"):
        X.PagedCache(dev, z(4, 2, 16, 80), z(4, 2, 16, 80))
    with pytest.raises(X.XdnaError, match="aligned"):
        X.PagedCache(dev, z(4 * 2 * 16 * 64 + 4)[4:].view(4, 2, 16, 64), z(4 * 2 * 16 * 64 + 4)[4:].view(4, 2, 16, 64))
    over = z(4096)
    with pytest.raises(X.XdnaError, match="overlap"):
        X.PagedCache(dev, over.as_strided((4, 2, 4, 64), (128, 64, 64, 1)), over.as_strided((4, 2, 4, 64), (128, 64, 64, 1)))
    with pytest.raises(X.XdnaError):
        X.PagedCache(dev, pool, pool.clone(), max_seqs=0)
    c = X.PagedCache(dev, pool, pool.clone(), max_seqs=3)
    table, lens = z(3, 2, t=I32), z(3, t=I32)
    q = z(3, 4, 64)
    assert c.attend(q, table, lens).shape == (3, 4, 64)
    for bad in (dict(q=q.float()), dict(q=z(3, 4, 128)), dict(q=z(2, 4, 64)), dict(seq_lens=lens.long()),
                dict(block_table=table.long()), dict(block_table=z(2, 2, t=I32)), dict(out=z(3, 4, 64, t=F32)),
                dict(lse=z(3, 5, t=F32)), dict(q=z(3, 64, 4).transpose(1, 2)), dict(q=q.cpu())):
        with pytest.raises(ValueError):
            c.attend(**{**dict(q=q, block_table=table, seq_lens=lens), **bad})
    for bad, what in ((dict(q=z(3, 3, 64)), "multiple"), (dict(layer=1), "layer"), (dict(layer=-1), "layer"),
                      (dict(window=-1), "window"), (dict(scale=0.0), "scale"), (dict(scale=math.nan), "scale"),
                      (dict(q=z(3, 260)[:, 4:].view(3, 4, 64)), "aligned"),
                      (dict(q=z(4, 4, 64), block_table=z(4, 2, t=I32), seq_lens=z(4, t=I32)), "max_seqs")):
        with pytest.raises(X.XdnaError, match=what):
            c.attend(**{**dict(q=q, block_table=table, seq_lens=lens), **bad})
    one = q.data_ptr()
    assert X.lib().xdna_paged_attention(c.handle, 0, one, 256, 4, one, 3, 1 << 26, 1 << 26, one, 0.125, 0, one, None, None) == -1
    assert "2^29" in X.last_error()
    k, pos = z(3, 2, 64), z(3, t=I32)
    good = dict(q=q, k=k, v=k, tok_seq=None, tok_pos=pos, block_table=table)
    for bad in (dict(k=k.float()), dict(k=z(3, 3, 64)), dict(q=z(2, 4, 64)), dict(tok_pos=pos.long()),
                dict(tok_seq=z(2, t=I32)), dict(rope=z(4, 64)), dict(q_out=z(3, 4, 64, t=F32))):
        with pytest.raises(ValueError):
            c.append(**{**good, **bad})
    for bad, what in ((dict(rope=z(4, 24, t=F32)), "rot_dim"), (dict(rope=z(4, 128, t=F32)), "rot_dim"),
                      (dict(block_table=z(2, 2, t=I32)), "tok_seq"), (dict(layer=7), "layer")):
        with pytest.raises(X.XdnaError, match=what):
            c.append(**{**good, **bad})
    x, w = z(3, 64), z(64, t=F32)
    for bad in (dict(x=z(3, 64, t=torch.float16)), dict(gamma=w.to(BF16)), dict(gamma=z(65, t=F32)),
                dict(residual=z(3, 65)), dict(residual=x, residual_out=z(3, 64, t=F32)), dict(residual_out=x),
                dict(q8=z(3, 64)), dict(y=z(3, 64, t=F32)), dict(quantize=False, q8=z(3, 64, t=I8)),
                dict(x=z(64, 3).T)):
        with pytest.raises(ValueError):
            X.rmsnorm_residual_i8(**{**dict(x=x, gamma=w), **bad})
    for bad, what in ((dict(x=z(1, 16385), gamma=z(16385, t=F32)), "16384"), (dict(eps=-1.0), "eps"),
                      (dict(quantize=False), "no output")):
        with pytest.raises(X.XdnaError, match=what):
            X.rmsnorm_residual_i8(**{**dict(x=x, gamma=w), **bad})
    lg = z(3, 100, t=F32)
    for bad in (dict(logits=lg.long()), dict(out=z(3, 100)), dict(ids=z(3, t=I32)), dict(mask=z(3, 3, t=I32)),
                dict(history=z(5, t=torch.int64), history_start=z(4, t=I32))):
        with pytest.raises(ValueError):
            X.process_logits(**{**dict(logits=lg), **bad})
    for bad, what in ((dict(repetition=z(3, t=F32)), "history"), (dict(history=z(5, t=I32)), "together"),
                      (dict(bias=z(5, t=F32)), "together")):
        with pytest.raises(X.XdnaError, match=what):
            X.process_logits(**{**dict(logits=lg), **bad})
