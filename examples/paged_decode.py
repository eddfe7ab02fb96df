"""A decoder served with continuous batching from a paged key-value cache, on the op-level entries.

    python examples/paged_decode.py            # on a B200

One layer of the step, for any number of tokens of any streams:

    rmsnorm_residual_i8   h += x; int8 rows of norm(h)          the residual addition of the layer before
    xdna_gemm_i8          q | k | v in f32                      rows_per_clip 1: a scale per token
    PagedCache.append     rotate, write k and v into pages
    PagedCache.attend     one query per token over its stream's pages
    xdna_gemm_bf16        output projection
    rmsnorm_residual_i8   h += x; norm(h) in bf16
    xdna_ffn_fused_bf16   the feed-forward's two products

and at the end the LM head and process_logits: penalties, biases, grammar mask, the next token.  A
prompt goes through the same step: its tokens are appended together, max_tokens of them to a call, and token i
attends over the first i + 1 positions as a stream of that length with the same pages.
"""
import dataclasses
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import xdna_engine_b200 as X  # noqa: E402


@dataclasses.dataclass
class Config:
    n_layers: int = 4
    d_model: int = 512
    n_q_heads: int = 8
    n_kv_heads: int = 2
    head_dim: int = 64
    ffn: int = 1024
    vocab: int = 4096
    eps: float = 1e-6
    theta: float = 10000.0
    max_positions: int = 2048


def make_weights(cfg, seed, device="cuda"):
    """Random weights as the products take them: [out, in], int8 rows with scales for q | k | v, bf16 else."""
    g = torch.Generator(device=device)
    g.manual_seed(seed)

    def normal(*shape, std=0.05):
        return torch.randn(*shape, generator=g, device=device) * std

    def bf16(*shape, std=0.05):
        return normal(*shape, std=std).bfloat16()

    heads = cfg.n_q_heads + 2 * cfg.n_kv_heads
    layers = []
    for _ in range(cfg.n_layers):
        w = normal(heads * cfg.head_dim, cfg.d_model)
        scale = w.abs().amax(1) / 127
        layers.append(dict(norm1=1 + normal(cfg.d_model, std=0.1), norm2=1 + normal(cfg.d_model, std=0.1),
                           wqkv=torch.round(w / scale[:, None]).to(torch.int8), wqkv_scale=scale,
                           wo=bf16(cfg.d_model, cfg.n_q_heads * cfg.head_dim),
                           w1=bf16(cfg.ffn, cfg.d_model), w2=bf16(cfg.d_model, cfg.ffn)))
    return dict(embed=bf16(cfg.vocab, cfg.d_model, std=1.0), layers=layers, norm=1 + normal(cfg.d_model, std=0.1),
                head=bf16(cfg.vocab, cfg.d_model))


def _call(rc):
    if rc:
        raise X.XdnaError(X.last_error())


class PagedDecoder:
    """The model over a pool of pages; what stream owns which pages is the caller's business."""

    def __init__(self, device, cfg, weights, n_pages, page_size=16, kv="bf16", max_tokens=512):
        self.cfg, self.w, self.dev, self.max_tokens = cfg, weights, f"cuda:{device.ordinal}", max_tokens
        shape = (cfg.n_layers, n_pages, cfg.n_kv_heads, page_size, cfg.head_dim)
        pools = [torch.zeros(shape, dtype=torch.bfloat16 if kv == "bf16" else torch.int8, device=self.dev) for _ in "kv"]
        scales = [None, None] if kv == "bf16" else [torch.ones(shape[:4], device=self.dev) for _ in "kv"]
        self.cache = X.PagedCache(device, *pools, *scales, max_seqs=max_tokens)
        self.rope = X.rope_table(cfg.max_positions, cfg.head_dim, cfg.theta, device=self.dev)

    def logits(self, tokens, streams, positions, table, rows=None):
        """bf16 logits of the given tokens: tokens int64 [n], token i at positions[i] of streams[i] (int32),
        table int32 [n_streams, width].  rows: the tokens whose logits are wanted (all)."""
        cfg, L, n = self.cfg, X.lib(), tokens.numel()
        st = torch.cuda.current_stream().cuda_stream
        bf16, f32 = torch.bfloat16, torch.float32
        new = lambda *s, t=bf16: torch.empty(*s, dtype=t, device=self.dev)  # noqa: E731
        d, hq, hk, hd = cfg.d_model, cfg.n_q_heads, cfg.n_kv_heads, cfg.head_dim
        h = self.w["embed"][tokens].float()                       # the residual stream
        own_table, lens = table[streams.long()], positions + 1    # a query is a stream of its own length
        x = torch.zeros_like(h, dtype=bf16)
        for i, ly in enumerate(self.w["layers"]):
            q8, scale, h = X.rmsnorm_residual_i8(x, ly["norm1"], residual=h, eps=cfg.eps, residual_out=h)
            qkv = new(n, (hq + 2 * hk) * hd, t=f32)
            _call(L.xdna_gemm_i8(q8.data_ptr(), ly["wqkv"].data_ptr(), scale.data_ptr(), 1, ly["wqkv_scale"].data_ptr(), None,
                                 0, None, 1.0, qkv.data_ptr(), None, n, qkv.shape[1], d, st))
            q, k, v = (t.view(n, -1, hd) for t in qkv.split([hq * hd, hk * hd, hk * hd], 1))
            q = self.cache.append(q, k, v, streams, positions, table, rope=self.rope, layer=i)
            ctx = self.cache.attend(q, own_table, lens, layer=i)
            o = new(n, d)
            _call(L.xdna_gemm_bf16(ctx.data_ptr(), ly["wo"].data_ptr(), None, None, o.data_ptr(), n, d, hq * hd, 0, st))
            y = new(n, d)
            X.rmsnorm_residual_i8(o, ly["norm2"], residual=h, eps=cfg.eps, residual_out=h, y=y, quantize=False)
            x = new(n, d)
            _call(L.xdna_ffn_fused_bf16(y.data_ptr(), ly["w1"].data_ptr(), None, 1, ly["w2"].data_ptr(), None, None,
                                        x.data_ptr(), None, n, d, cfg.ffn, d, st))
        y = new(n, d)
        X.rmsnorm_residual_i8(x, self.w["norm"], residual=h, eps=cfg.eps, residual_out=h, y=y, quantize=False)
        if rows is not None:
            y = y[rows].contiguous()
        out = new(y.shape[0], cfg.vocab)
        _call(L.xdna_gemm_bf16(y.data_ptr(), self.w["head"].data_ptr(), None, None, out.data_ptr(), y.shape[0], cfg.vocab, d,
                               0, st))
        return out

    def check(self):
        """Report what the kernels met on the device (page ids out of the pool, bounded waits that ran out)."""
        self.cache.check()
        _call(X.lib().xdna_gemm_check())
        _call(X.lib().xdna_ffn_fused_check())


class Server:
    """Streams that come and go: pages are handed out as they grow and taken back when they end."""

    def __init__(self, model, n_pages, page_size=16, width=128, repetition=1.1):
        self.model, self.page_size, self.width, self.repetition = model, page_size, width, repetition
        self.free, self.streams = list(range(n_pages)), {}

    def _grow(self, s, length):
        while len(s["pages"]) * self.page_size < length:
            s["pages"].append(self.free.pop())

    def _table(self, group):
        t = torch.full((len(group), self.width), -1, dtype=torch.int32)
        for i, s in enumerate(group):
            t[i, : len(s["pages"])] = torch.tensor(s["pages"], dtype=torch.int32)
        return t.to(self.model.dev)

    def _next(self, logits, group):
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=self.model.dev)  # noqa: E731
        starts = [0]
        for s in group:
            starts.append(starts[-1] + len(s["tokens"]))
        rep = torch.full((len(group),), self.repetition, device=self.model.dev)
        _, ids = X.process_logits(logits, history=i32([t for s in group for t in s["tokens"]]), history_start=i32(starts),
                                  n_prompt=i32([s["prompt"] for s in group]), repetition=rep)
        for s, t in zip(group, ids.tolist()):
            s["tokens"].append(t)

    def admit(self, name, prompt):
        """Run a prompt and choose the first token after it."""
        n, dev = len(prompt), self.model.dev
        if name in self.streams or n == 0 or -(-n // self.page_size) > min(self.width, len(self.free)):
            raise ValueError(f"a stream {name!r} of {n} tokens: known already, empty, or too long for the free pages")
        s = self.streams[name] = dict(tokens=list(prompt), prompt=n, pages=[])
        self._grow(s, n)
        table = self._table([s])
        for at in range(0, n, self.model.max_tokens):
            piece = torch.tensor(prompt[at:at + self.model.max_tokens], device=dev)
            k = piece.numel()
            out = self.model.logits(piece, torch.zeros(k, dtype=torch.int32, device=dev),
                                    torch.arange(at, at + k, dtype=torch.int32, device=dev), table,
                                    rows=torch.tensor([k - 1], device=dev))
        self._next(out, [s])

    def step(self):
        """One token for every stream, at its own position."""
        group, dev = list(self.streams.values()), self.model.dev
        if not group:
            return
        pos = [len(s["tokens"]) - 1 for s in group]
        for s, p in zip(group, pos):
            self._grow(s, p + 1)
        out = self.model.logits(torch.tensor([s["tokens"][-1] for s in group], device=dev),
                                torch.arange(len(group), dtype=torch.int32, device=dev),
                                torch.tensor(pos, dtype=torch.int32, device=dev), self._table(group))
        self._next(out, group)

    def release(self, name):
        """The stream's tokens; its pages go back."""
        s = self.streams.pop(name)
        self.free += s["pages"]
        return s["tokens"][s["prompt"]:]


def main():
    cfg = Config()
    dev = X.Device(0)
    n_pages = 256
    model = PagedDecoder(dev, cfg, make_weights(cfg, seed=0), n_pages, kv="int8")
    server = Server(model, n_pages)
    g = torch.Generator().manual_seed(1)
    for i, n in enumerate((5, 40, 17)):
        server.admit(f"stream {i}", torch.randint(0, cfg.vocab, (n,), generator=g).tolist())
    for step in range(24):
        if step == 8:
            print("stream 1:", server.release("stream 1"))
            server.admit("stream 3", torch.randint(0, cfg.vocab, (64,), generator=g).tolist())
        server.step()
    for name in list(server.streams):
        print(f"{name}:", server.release(name))
    model.check()


if __name__ == "__main__":
    main()
