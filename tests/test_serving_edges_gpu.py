"""Edges of the serving ops: what a call meets at the ends of its ranges, against definitions in 64 bits.

Tolerances are derived where they are used."""
import math

import pytest

torch = pytest.importorskip("torch")
from test_serving_gpu import attention_64, check_attention, make_pool  # noqa: E402

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


def i32(x):
    return torch.tensor(x, dtype=I32, device="cuda")


# ------------------------------------------------------------------------------- attention
@pytest.mark.parametrize("d,hq,hkv", [(64, 32, 8), (128, 32, 8), (256, 8, 8), (128, 32, 2)])
def test_attention_weights_are_f32(X, dev, d, hq, hkv):
    """bf16 pools: the weights keep the 24 bits of f32.

    Two keys, of values 0 and v, and scores below 1 with one product each that is not 0: o = v p / (1 + p).  In
    units of 2^-24 p is off by 8 (scale log2 e, its constant, the product and the difference, for both scores) and 4
    (the hardware exponential), the sum, 1 / sum and the last product by 1 each and the accumulated terms by 6: 21, below
    2^-19.  So the output is the bf16 nearest to something within 2^-19 of o.  Weights of 16 bits are off by
    up to 2^-18 and miss that in some of these 2 million places."""
    g = rng(d + hkv)
    n = 2**21 // (hq * d)
    k, v = (torch.zeros(n, hkv, 16, d, dtype=BF16, device="cuda") for _ in "kv")
    k[:, :, :2, 0] = torch.rand(n, hkv, 2, generator=g, device="cuda").mul(2).sub(1).to(BF16)
    v[:, :, 1] = torch.randn(n, hkv, d, generator=g, device="cuda").to(BF16)
    q = torch.randn(n, hq, d, generator=g, device="cuda").to(BF16)
    q[..., 0] = 0.5 + 0.5 * torch.rand(n, hq, generator=g, device="cuda").to(BF16)
    c = X.PagedCache(dev, k, v, max_seqs=n)
    out = c.attend(q, torch.arange(n, dtype=I32, device="cuda")[:, None], torch.full((n,), 2, dtype=I32, device="cuda"),
                   scale=1.0)
    c.check()
    s = k[:, :, :2, 0].to(F64).repeat_interleave(hq // hkv, 1) * q[..., :1].to(F64)
    o = torch.softmax(s, -1)[..., 1:] * v[:, :, 1].to(F64).repeat_interleave(hq // hkv, 1)
    ends = [(o * (1 + e)).float().to(BF16) for e in (-2.0**-19, 2.0**-19)]       # f32 first: 2^-24 more
    lo, hi = torch.minimum(*ends), torch.maximum(*ends)
    assert int(((out < lo) | (out > hi)).sum()) == 0


@pytest.mark.parametrize("d,slots,kv", [(256, 2**23, "bf16"), (128, 2**24, "bf16"), (256, 2**24, "int8"), (256, 2**23 + 48, "bf16")])
def test_attention_past_32_bits_within_a_page(X, dev, d, slots, kv):
    """Rows whose bytes lie past 2^31 in their page: a contiguous cache of one page.  A page of zeros whose last
    301 rows count; without a window every row does, at weight 1."""
    g = rng(d + slots % 97)
    n, window = slots - 5, 301
    pool = torch.zeros(1, 1, slots, d, dtype=BF16 if kv == "bf16" else I8, device="cuda")
    scales = [None, None] if kv == "bf16" else [torch.full((1, 1, slots), 2.0**-5 * (i + 1), device="cuda") for i in range(2)]
    rows = torch.randn(window, d, generator=g, device="cuda") if kv == "bf16" else \
        torch.randint(-127, 128, (window, d), generator=g, device="cuda")
    pool[0, 0, n - window:n] = rows.to(pool.dtype)
    c = X.PagedCache(dev, pool, pool, *scales)
    q = torch.randn(1, 4, d, generator=g, device="cuda").to(BF16)
    table, lens = i32([[0]]), i32([n])
    live = pool[0, 0, n - window:n].to(F64)
    k, v = (live, live) if kv == "bf16" else (live / 32, live / 16)
    s = q[0].to(F64) @ k.T * d ** -0.5
    o = torch.softmax(s, 1) @ v
    # the scores' f32 sums, 2^-23 of sum|q k| each, and their weights' share; bf16 outputs
    ds = float((q[0].to(F64).abs() @ k.abs().T).max()) * d ** -0.5 * (d + 4) * 2.0**-23
    rel = 2 * ds + 2.0**-16 + window * 2.0**-23
    out = c.attend(q, table, lens, window=window)
    c.check()
    bound = o.abs() * 1.01 * 2.0**-8 + rel * (torch.softmax(s, 1) @ v.abs())
    assert float(((out[0].to(F64) - o).abs() - bound).max()) <= 0
    lse = torch.empty(1, 4, device="cuda")
    c.attend(q.zero_(), table, lens, lse=lse)
    c.check()
    # a sum of n ones: every part of it is a whole number below 2^24, exact
    assert float((lse.to(F64) - math.log(n)).abs().max()) <= 2.0**-19 + math.log(n) * 2.0**-22


@pytest.mark.parametrize("d,hkv,n", [(64, 1, 40000), (128, 2, 70000), (256, 1, 33000)])
def test_int8_values_of_scale_zero(X, dev, d, hkv, n):
    """Value rows of scale 0 give zeros and leave the log-sum-exp alone."""
    g = rng(n)
    p = make_pool(g, "int8", [n, 50], hkv, 16, d)
    p["k_scale"] = p["k_scale"].nan_to_num(0.0)
    p["v_scale"] = torch.zeros_like(p["v_scale"])
    q = torch.randn(2, 4 * hkv, d, generator=g, device="cuda").mul(0.1).to(BF16)
    c = X.PagedCache(dev, p["k"], p["v"], p["k_scale"], p["v_scale"])
    lse = torch.empty(2, 4 * hkv, device="cuda")
    out = c.attend(q, p["table"], i32([n, 50]), lse=lse)
    c.check()
    check_attention(out, lse, attention_64(q, p, [n, 50], d ** -0.5, 0))
    assert not out.any()


@pytest.mark.parametrize("v_scale", [1e-30, 1e-12, 1.0, 1e6])
@pytest.mark.parametrize("d,hq,hkv", [(64, 4, 1), (128, 32, 2), (256, 16, 2)])
def test_int8_values_of_any_scale(X, dev, d, hq, hkv, v_scale):
    """The same bounds hold whatever the values' scales are, and as scores climb through a stream."""
    g = rng(d)
    lens = [700, 3, 1500]
    p = make_pool(g, "int8", lens, hkv, 16, d)
    p["v_scale"] *= v_scale
    climb = torch.linspace(1, 8, p["k"].shape[1], device="cuda")
    p["k_scale"] *= climb[None, :, None, None]
    q = torch.randn(3, hq, d, generator=g, device="cuda").to(BF16)
    c = X.PagedCache(dev, p["k"], p["v"], p["k_scale"], p["v_scale"])
    lse = torch.empty(3, hq, device="cuda")
    out = c.attend(q, p["table"], i32(lens), lse=lse)
    c.check()
    check_attention(out, lse, attention_64(q, p, lens, d ** -0.5, 0))


@pytest.mark.parametrize("at", [0, 100, 299])
@pytest.mark.parametrize("gap", [0, 12, 20, 40, 80])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_int8_zero_value_row_that_dominates(X, dev, d, gap, at):
    """A key whose value row is zero, of scale 1 as append leaves it, `gap` above the others' scores: their values
    still come out to bf16's rounding."""
    g = rng(d + gap + at)
    p = make_pool(g, "int8", [300], 1, 16, d)
    p["k"][..., 1:] = 0
    p["k"][..., 0].clamp_(-64, 64)
    p["k_scale"] = torch.full_like(p["k_scale"], 1 / 64)
    p["v_scale"] = torch.where(p["v_scale"].isnan(), 1.0, p["v_scale"])
    page, slot = int(p["table"][0, at // 16]), at % 16
    p["k"][0, page, 0, slot, 0] = 127
    p["k_scale"][0, page, 0, slot] = (1 + gap) / 127
    p["v"][0, page, 0, slot] = 0
    p["v_scale"][0, page, 0, slot] = 1.0
    q = torch.zeros(1, 4, d, dtype=BF16, device="cuda")
    q[..., 0] = 1.0
    c = X.PagedCache(dev, p["k"], p["v"], p["k_scale"], p["v_scale"])
    lse = torch.empty(1, 4, device="cuda")
    out = c.attend(q, p["table"], i32([300]), scale=1.0, lse=lse)
    c.check()
    check_attention(out, lse, attention_64(q, p, [300], 1.0, 0))


@pytest.mark.parametrize("kv", ["bf16", "int8"])
@pytest.mark.parametrize("d,hq,hkv", [(64, 8, 8), (128, 32, 8), (256, 8, 8), (64, 64, 4), (128, 64, 4), (256, 64, 4)])
@pytest.mark.parametrize("b,window", [(64, 0), (150, 0), (150, 300000)])
def test_attention_wide_tables(X, dev, d, hq, hkv, b, window, kv):
    """A table of a million positions a stream, whose tiles need 64 bits to be shared out, gives the bits that a
    narrow one gives: its CTAs and their shares are the same."""
    g = rng(b + d)
    lens = [(i * 37) % 1800 for i in range(b)]
    p = make_pool(g, kv, lens, hkv, 16, d)
    q = torch.randn(b, hq, d, generator=g, device="cuda").to(BF16)
    c = X.PagedCache(dev, p["k"], p["v"], p["k_scale"], p["v_scale"], max_seqs=b)
    wide = torch.full((b, 65536), -5, dtype=I32, device="cuda")
    wide[:, : p["table"].shape[1]] = p["table"]
    res = []
    for table in (p["table"], wide):
        lse = torch.empty(b, hq, device="cuda")
        out = c.attend(q, table, i32(lens), lse=lse, window=window)
        c.check()
        res.append((out, lse))
    assert torch.equal(res[0][0].view(torch.int16), res[1][0].view(torch.int16)) and torch.equal(res[0][1], res[1][1])
    few = [0, 1, b // 2, b - 1, max(range(b), key=lambda i: lens[i])]
    check_attention(out[few], lse[few], attention_64(q[few], dict(p, table=p["table"][few]), [lens[i] for i in few],
                                                     d ** -0.5, 0))


@pytest.mark.parametrize("kv", ["bf16", "int8"])
@pytest.mark.parametrize("d", [128, 256])
@pytest.mark.parametrize("page", [7, 24])
@pytest.mark.parametrize("window", [0, 50])
def test_attention_pages_that_cut_steps(X, dev, d, page, window, kv):
    """Pages that are not whole steps of 16 keys, at the head sizes that lay their shared memory out otherwise."""
    g = rng(d + page)
    lens = [0, 5, 600, 99, 1025, 16, 1]
    p = make_pool(g, kv, lens, 2, page, d)
    for hq in (8, 32):
        q = torch.randn(len(lens), hq, d, generator=g, device="cuda").to(BF16)
        c = X.PagedCache(dev, p["k"], p["v"], p["k_scale"], p["v_scale"])
        lse = torch.empty(len(lens), hq, device="cuda")
        out = c.attend(q, p["table"], i32(lens), window=window, lse=lse)
        c.check()
        check_attention(out, lse, attention_64(q, p, lens, d ** -0.5, window))


def test_attention_every_stream_as_alone(X, dev):
    """A batch's streams each give what they give in a call of their own, to the joins' f32 rounding: the same parts
    in other shares, 2^-19 of the sums, and one rounding to bf16 on either side."""
    g = rng(77)
    lens = [1] * 150 + [7000] + [33] * 100 + [300] * 49
    p = make_pool(g, "bf16", lens, 8, 16, 128)
    q = torch.randn(len(lens), 32, 128, generator=g, device="cuda").to(BF16)
    c = X.PagedCache(dev, p["k"], p["v"], max_seqs=len(lens))
    out = c.attend(q, p["table"], i32(lens)).float()
    top = 0.0
    for i, n in enumerate(lens):
        one = c.attend(q[i:i + 1], p["table"][i:i + 1, :-(-n // 16)], i32([n]))[0].float()
        top = max(top, float(((out[i] - one).abs() - one.abs() * 2.0**-7 - 2.0**-17).max()))
    c.check()
    assert top <= 0


# --------------------------------------------------------------------------------- streams
def busy(stream, ms=20):
    """Keep `stream` at work for some milliseconds."""
    with torch.cuda.stream(stream):
        torch.cuda._sleep(int(ms * 1.9e6))


@pytest.mark.parametrize("b,v", [(3, 100003), (2, 262144)])
def test_a_given_streams_workspace_is_its_own(X, b, v):
    """process_logits on a stream that is still at work: what the current stream allocates and writes
    meanwhile is neither the call's workspace nor its outputs."""
    g = rng(v)
    side = torch.cuda.Stream()
    x = torch.randn(b, v, generator=g, device="cuda")
    torch.cuda.synchronize()
    for size in (X.lib().xdna_logits_workspace(b, v), b * v * 4, b * 8):
        busy(side)
        out, ids = X.process_logits(x, stream=side.cuda_stream)
        mine = [torch.full((size,), 0xff, dtype=torch.uint8, device="cuda") for _ in range(4)]
        torch.cuda.synchronize()
        assert all(bool((m == 0xff).all()) for m in mine)
        assert torch.equal(out, x) and torch.equal(ids, x.argmax(1))


def test_a_given_streams_outputs_are_its_own(X, dev):
    """Outputs that a call on a given stream allocates are not memory that the current stream's earlier work
    still writes; the default stream (0) may be named too."""
    g = rng(21)
    side = torch.cuda.Stream()
    m, d = 64, 1024
    x, w = torch.randn(m, d, generator=g, device="cuda").to(BF16), torch.ones(d, device="cuda")
    res = torch.randn(m, d, generator=g, device="cuda")
    pool = torch.randn(m, 2, 16, 64, generator=g, device="cuda").to(BF16)
    c = X.PagedCache(dev, pool, pool.clone())
    q, k = (torch.randn(m, h, 64, generator=g, device="cuda").to(BF16) for h in (8, 2))
    at, table = torch.full((m,), 15, dtype=I32, device="cuda"), torch.arange(m, dtype=I32, device="cuda")[:, None]
    lg = torch.randn(m, 2000, generator=g, device="cuda")
    calls = [lambda **s: X.rmsnorm_residual_i8(x, w, residual=res, **s),
             lambda **s: c.append(q, k, k, None, at, table, **s),
             lambda **s: c.attend(q, table, at, **s),
             lambda **s: X.process_logits(lg, **s)]
    flat = lambda t: [t] if torch.is_tensor(t) else [y for y in t if y is not None]  # noqa: E731
    for call in calls:
        want = flat(call())
        torch.cuda.synchronize()
        busy(torch.cuda.current_stream())
        for t in want:                                    # freed at once, written late
            torch.empty_like(t).fill_(7)
        late = flat(call(stream=side.cuda_stream))
        again = flat(call(stream=0))
        torch.cuda.synchronize()
        for a, b, e in zip(late, again, want):
            assert torch.equal(a, e) and torch.equal(b, e)


# ------------------------------------------------------------------------------------- norm
@pytest.mark.parametrize("x_type,res_type", [(BF16, BF16), (F32, None), (BF16, F32)])
@pytest.mark.parametrize("d", [40, 1152, 4096, 5120, 16384, 37, 865, 2434, 10001])
def test_norm_keeps_what_is_not_finite(X, d, x_type, res_type):
    """Rows with one NaN, of nothing but NaN, of zeros and one NaN, with an infinity, and a NaN in gamma: not a
    finite row in any output; the rows beside them are what they are alone."""
    g = rng(d)
    m = 9
    x = torch.randn(m, d, generator=g, device="cuda").to(x_type)
    res = None if res_type is None else torch.randn(m, d, generator=g, device="cuda").to(res_type)
    w = torch.randn(d, generator=g, device="cuda")
    good = [0, 2, 4, 6, 8]
    alone = [t[good] for t in (X.rmsnorm_residual_i8(x, w, residual=res)[:2])]
    x[1, d // 3] = math.nan
    x[3] = math.nan
    x[5] = 0
    x[7, d - 1] = -math.inf
    if res is not None:
        res[5] = 0
    x[5, d // 2] = math.nan
    y = torch.empty(m, d, dtype=BF16, device="cuda")
    q8, scale, _ = X.rmsnorm_residual_i8(x, w, residual=res, y=y)
    values = q8 * scale[:, None]
    assert torch.isnan(scale[[1, 3, 5, 7]]).all() and torch.isnan(values[[1, 3, 5, 7]]).all()
    assert torch.isnan(y[[1, 3, 5]].float()).all() and torch.isnan(y[7, d - 1].float())
    assert torch.equal(q8[good], alone[0]) and torch.equal(scale[good], alone[1])
    w[d - 2] = math.nan
    q8, scale, _ = X.rmsnorm_residual_i8(x[good], w, residual=None if res is None else res[good])
    assert torch.isnan(scale).all()


# ----------------------------------------------------------------------------------- logits
@pytest.mark.parametrize("v", [70, 5000, 100003])
def test_logits_offsets_are_held_within_the_lists(X, v):
    """Starts that fall, lie below 0 or past the lists, down to -2^31 and up to 2^31 - 1: as if they were held to [0,
    length], with no entries where a row's end lies before its start."""
    big = 2**31 - 1
    g = rng(v)
    starts = [5, -big - 1, 3, big, -3, 2, 9, 9, 8, -big - 1, big]
    b = len(starts) - 1
    x = torch.randn(b, v, generator=g, device="cuda")
    ids = torch.randperm(70, generator=g, device="cuda")[:8].int()
    add = torch.randn(8, generator=g, device="cuda")
    want = x.clone()
    for r in range(b):
        lo, hi = max(0, starts[r]), min(8, starts[r + 1])
        for j in range(lo, hi):
            want[r, int(ids[j])] += add[j]
    out, best = X.process_logits(x, bias_ids=ids, bias=add, bias_start=i32(starts))
    assert torch.equal(out, want) and torch.equal(best, want.argmax(1))
    minus = torch.linspace(0.5, 2, b, device="cuda")
    want = x.clone()
    for r in range(b):
        lo, hi = max(0, starts[r]), min(8, starts[r + 1])
        for j in range(lo, hi):
            want[r, int(ids[j])] -= minus[r]
    out, best = X.process_logits(x, history=ids, history_start=i32(starts), presence=minus)
    assert torch.equal(out, want) and torch.equal(best, want.argmax(1))


@pytest.mark.parametrize("v", [50, 100003])
def test_logits_empty_lists(X, v):
    """A step whose rows have no tokens yet, or no biases: lists of no entries are lists."""
    g = rng(v)
    x = torch.randn(3, v, generator=g, device="cuda")
    none, start = torch.empty(0, dtype=I32, device="cuda"), i32([0] * 4)
    one = torch.ones(3, device="cuda")
    both = dict(history=none, history_start=start, n_prompt=i32([0, 0, 0]), repetition=one * 2, frequency=one, presence=one)
    bias = dict(bias_ids=none, bias=none.float(), bias_start=start)
    for kw in (both, bias, {**both, **bias}):
        out, ids = X.process_logits(x, **kw)
        assert torch.equal(out, x) and torch.equal(ids, x.argmax(1))
    with pytest.raises(X.XdnaError, match="together"):
        X.process_logits(x, history_start=start)


# --------------------------------------------------------------------------------- refusals
def test_shapes_of_the_same_size_are_refused(X, dev):
    """A tensor of the right size whose dimensions lie in another order."""
    z = lambda *s, t=BF16: torch.zeros(*s, dtype=t, device="cuda")  # noqa: E731
    pool, scale = z(4, 2, 16, 64, t=I8), z(4, 2, 16, t=F32)
    nhd = z(4, 16, 2, 64, t=I8).transpose(1, 2)
    for kw in (dict(k=nhd, v=nhd, k_scale=z(4, 16, 2, t=F32), v_scale=z(4, 16, 2, t=F32)),
               dict(k=pool, v=pool, k_scale=scale, v_scale=z(4, 16, 2, t=F32)),
               dict(k=pool, v=pool, k_scale=scale[None], v_scale=scale[None])):
        with pytest.raises(ValueError, match="_scale"):
            X.PagedCache(dev, **kw)
    c = X.PagedCache(dev, nhd, nhd, scale, scale)
    q, table, lens = z(3, 4, 64), z(3, 2, t=I32), z(3, t=I32)
    for bad in (dict(out=z(4, 3, 64)), dict(lse=z(4, 3, t=F32))):
        with pytest.raises(ValueError, match=next(iter(bad))):
            c.attend(q, table, lens, **bad)
    with pytest.raises(ValueError, match="q_out"):
        c.append(q, z(3, 2, 64), z(3, 2, 64), None, lens, table, q_out=z(4, 3, 64))
    x, w = z(3, 64), z(64, t=F32)
    for bad in (dict(q8=z(64, 3, t=I8)), dict(y=z(64, 3))):
        with pytest.raises(ValueError, match=next(iter(bad))):
            X.rmsnorm_residual_i8(x, w, **bad)
    with pytest.raises(ValueError, match="mask"):
        X.process_logits(z(3, 100, t=F32), mask=z(4, 3, t=I32))


def test_pointers_off_their_elements(X, dev):
    """The cache's C entries refuse 4-byte arrays that lie off 4 bytes, before anything is enqueued."""
    z = lambda *s, t=BF16: torch.zeros(*s, dtype=t, device="cuda")  # noqa: E731
    pool = z(4, 2, 16, 64)
    c = X.PagedCache(dev, pool, pool.clone())
    L, one = X.lib(), z(4096).data_ptr()
    attend = dict(c=c.handle, layer=0, q=one, qs=256, hq=4, table=one, n=3, width=2, ts=2, lens=one, scale=0.125, window=0,
                  out=one, lse=one, st=None)
    for name in ("table", "lens", "lse"):
        assert L.xdna_paged_attention(*{**attend, name: one + 2}.values()) == -1 and "aligned" in X.last_error(), name
    append = dict(c=c.handle, layer=0, n=0, hq=4, f=0, q=one, qs=256, k=one, ks=128, v=one, vs=128, seq=one, pos=one, table=one,
                  ns=3, width=2, ts=2, rope=None, rows=0, rot=0, inter=0, out=one, st=None)
    assert L.xdna_paged_append(*append.values()) == 0
    for name in ("seq", "pos", "table"):
        assert L.xdna_paged_append(*{**append, name: one + 2}.values()) == -1 and "aligned" in X.last_error(), name
