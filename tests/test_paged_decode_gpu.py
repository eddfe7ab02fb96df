"""examples/paged_decode.py, the serving ops run together as a decoder: its logits against the same
network in 64 bits, whole prompts against single steps, and streams that come and go.

Tolerance of the logits: the reference repeats the int8 rounding of the norms (and of an int8
cache), which leaves the bf16 roundings: of rotated q, cached k and v, attention's output, the
projection, norm 2, the feed-forward's hidden and its output, 8 to a layer, each of 2^-8 / sqrt(3) at
most in the root mean square (0.23%), and a few int8 values that fall on the other side (one step in 127
of few).  Two layers and the head: sqrt(18) 0.23% = 1%; 3% allows for their gain through the layers."""
import importlib.util
import os

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

HERE = os.path.dirname(os.path.abspath(__file__))
F64 = torch.float64


@pytest.fixture(scope="module")
def E():
    from xdna_engine_b200 import _build
    _build.build()
    spec = importlib.util.spec_from_file_location("paged_decode", os.path.join(HERE, "..", "examples", "paged_decode.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


@pytest.fixture(scope="module")
def dev(E):
    d = E.X.Device(0)
    yield d
    d.close()


def rounded(x):
    """Rows to int8 and back."""
    step = x.abs().amax(-1, keepdim=True) / 127
    return torch.round(x / step) * step


def network_64(cfg, w, tokens, kv):
    """Logits of every position of one stream."""
    n, hd, hq, hk = len(tokens), cfg.head_dim, cfg.n_q_heads, cfg.n_kv_heads

    def norm(h, g):
        return h / torch.sqrt(h.square().mean(1, keepdim=True) + cfg.eps) * g.to(F64)

    def turn(x):
        a = torch.arange(n, dtype=F64, device="cuda")[:, None] * cfg.theta ** (-torch.arange(0, hd, 2, dtype=F64, device="cuda") / hd)
        z = torch.complex(x[..., : hd // 2], x[..., hd // 2:]) * torch.polar(torch.ones_like(a), a)[:, None]
        return torch.cat([z.real, z.imag], -1)

    h = w["embed"][torch.tensor(tokens, device="cuda")].to(F64)
    for ly in w["layers"]:
        qkv = rounded(norm(h, ly["norm1"])) @ (ly["wqkv"].to(F64) * ly["wqkv_scale"].to(F64)[:, None]).T
        q, k, v = (t.view(n, -1, hd) for t in qkv.split([hq * hd, hk * hd, hk * hd], 1))
        q, k = turn(q), turn(k)
        if kv == "int8":
            k, v = rounded(k), rounded(v)
        k, v = (t.repeat_interleave(hq // hk, 1) for t in (k, v))
        s = torch.einsum("ihd,jhd->hij", q, k) * hd ** -0.5
        s = s.masked_fill(torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1), -torch.inf)
        ctx = torch.einsum("hij,jhd->ihd", torch.softmax(s, -1), v).reshape(n, hq * hd)
        h = h + ctx @ ly["wo"].to(F64).T
        y = norm(h, ly["norm2"])
        u = y @ ly["w1"].to(F64).T
        h = h + (0.5 * u * (1 + torch.erf(u / 2 ** 0.5))) @ ly["w2"].to(F64).T
    return norm(h, w["norm"]) @ w["head"].to(F64).T


@pytest.mark.parametrize("kv", ["bf16", "int8"])
@pytest.mark.parametrize("n,page", [(1, 16), (37, 16), (300, 16), (75, 7)])
def test_prompt_and_steps(E, dev, n, page, kv):
    cfg = E.Config(n_layers=2)
    w = E.make_weights(cfg, seed=n)
    g = torch.Generator().manual_seed(n)
    tokens = torch.randint(0, cfg.vocab, (n,), generator=g).tolist()
    want = network_64(cfg, w, tokens, kv)
    pages = -(-n // page) + 2
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    table = i32([torch.randperm(pages, generator=g).tolist()])
    model = E.PagedDecoder(dev, cfg, w, pages, page_size=page, kv=kv)
    whole = model.logits(torch.tensor(tokens, device="cuda"), i32([0] * n), i32(list(range(n))), table)
    model.check()
    assert float((whole.to(F64) - want).norm() / want.norm()) < 0.03
    # one token at a time into a cache of its own
    model = E.PagedDecoder(dev, cfg, w, pages, page_size=page, kv=kv)
    for p in range(min(n, 40)):
        one = model.logits(torch.tensor(tokens[p:p + 1], device="cuda"), i32([0]), i32([p]), table)
        assert float((one[0].to(F64) - want[p]).norm() / want[p].norm()) < 0.03
    model.check()


def test_streams_come_and_go(E, dev):
    """Each stream's tokens are the choices that the 64-bit network would make of its own tokens, up to ties within
    the logits' tolerance, whatever shares the batch with it; pages return to the pool."""
    cfg = E.Config(n_layers=2)
    w = E.make_weights(cfg, seed=3)
    model = E.PagedDecoder(dev, cfg, w, 64, kv="bf16")
    server = E.Server(model, 64, width=32)
    g = torch.Generator().manual_seed(4)
    prompts = {i: torch.randint(0, cfg.vocab, (n,), generator=g).tolist() for i, n in enumerate((5, 70, 33, 1))}
    got = {}
    for i in (0, 1, 2):
        server.admit(i, prompts[i])
    for step in range(12):
        if step == 5:
            got[1] = server.release(1)
            server.admit(3, prompts[3])
        server.step()
    for i in list(server.streams):
        got[i] = server.release(i)
    model.check()
    assert sorted(server.free) == list(range(64)) and sorted(got) == [0, 1, 2, 3]
    for i, new in got.items():
        tokens = prompts[i] + new
        want = network_64(cfg, w, tokens[:-1], "bf16")
        for k, t in enumerate(new):
            x = want[len(prompts[i]) - 1 + k].clone()
            seen = torch.tensor(sorted(set(tokens[: len(prompts[i]) + k])), device="cuda")
            x[seen] = torch.where(x[seen] > 0, x[seen] / 1.1, x[seen] * 1.1)
            assert float(x.max() - x[t]) <= 0.03 * 6 * float(x.std()), (i, k)
