"""The serving ops over torch tensors: a decoder's step between its int8 / bf16 products.

PagedCache (append with rotary positions, attention of one new token), rmsnorm_residual_i8 and
process_logits call the xdna_paged_*, xdna_rmsnorm_residual_i8 and xdna_logits_process entries of
the C ABI on the tensors' memory.  All of them are asynchronous on `stream` (a raw cudaStream_t;
None: torch's current stream of the tensors' device, so that torch's own ordering holds), and
leave every tensor where it is: a tensor of the wrong type, shape, layout or device is refused with
ValueError before anything is enqueued, and what the C ABI refuses raises XdnaError.

With a `stream` given, what a call allocates (a workspace, outputs that were not passed in) is memory of
that stream, which torch gives out again only behind that stream's work.  To order the inputs before the
call and the outputs after it, and to keep the inputs until the stream has read them, is then the caller's.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import XdnaError, _check, last_error, lib

__all__ = ["PagedCache", "process_logits", "rmsnorm_residual_i8", "rope_table"]



class _PagedConfig(C.Structure):
    _fields_ = [(n, C.c_int) for n in ("kv_type", "n_layers", "n_pages", "page_size", "n_kv_heads", "head_dim",
                                       "max_seqs")] + \
               [("k", C.c_void_p), ("v", C.c_void_p)] + \
               [(n, C.c_int64) for n in ("stride_layer", "stride_page", "stride_head", "stride_slot")] + \
               [("k_scale", C.c_void_p), ("v_scale", C.c_void_p)]


def _declare(L):
    vp, i, i64, f = C.c_void_p, C.c_int, C.c_int64, C.c_float
    L.xdna_paged_cache_create.argtypes = [vp, vp]
    L.xdna_paged_cache_create.restype = vp
    L.xdna_paged_cache_free.argtypes = [vp]
    L.xdna_paged_append.argtypes = [vp, i, i, i, i, vp, i64, vp, i64, vp, i64, vp, vp, vp, i, i, i64, vp, i, i, i,
                                    vp, vp]
    L.xdna_paged_append.restype = i
    L.xdna_paged_attention.argtypes = [vp, i, vp, i64, i, vp, i, i, i64, vp, f, i, vp, vp, vp]
    L.xdna_paged_attention.restype = i
    L.xdna_paged_cache_check.argtypes = [vp, vp]
    L.xdna_paged_cache_check.restype = i
    L.xdna_rmsnorm_residual_i8.argtypes = [vp, i, i64, vp, i, i64, vp, i, f, i, i, vp, vp, vp, vp, vp]
    L.xdna_rmsnorm_residual_i8.restype = i
    L.xdna_logits_process.argtypes = [vp, i, i64, i, i, vp, i, vp, vp, vp, vp, vp, vp, vp, i, vp, vp, i64,
                                      vp, i64, vp, vp, vp]
    L.xdna_logits_process.restype = i
    L.xdna_logits_workspace.argtypes = [i, i]
    L.xdna_logits_workspace.restype = C.c_size_t
    return L


_L = None


def _lib():
    global _L
    if _L is None:
        _L = _declare(lib())
    return _L


# These run in front of every launch, and a small launch is bound by them: plain attribute reads, and no
# message is formatted unless it is raised.
def _dense(t, dtype, shape, dev, name):
    """The address of a contiguous tensor of this type and shape on device dev (None: NULL)."""
    if t is None:
        return None
    if t.dtype is not dtype or t.shape != shape or t.get_device() != dev or not t.is_contiguous():
        raise ValueError(f"{name}: want a contiguous {dtype} tensor {tuple(shape)} on GPU {dev}, got {t.dtype} "
                         f"{tuple(t.shape)} on {t.device}, strides {t.stride()}")
    return t.data_ptr()


def _flat(t, dtype, n, dev, name):
    """The address of a contiguous tensor of n elements, a list of any shape, of this type on device dev (None: NULL)."""
    if t is None:
        return None
    if t.dtype is not dtype or t.numel() != n or t.get_device() != dev or not t.is_contiguous():
        raise ValueError(f"{name}: want a contiguous {dtype} tensor of {n} elements on GPU {dev}, got {t.dtype} "
                         f"{tuple(t.shape)} on {t.device}, strides {t.stride()}")
    return t.data_ptr()


def _list(t, start, dtype, n, dev, name):
    """As _flat, for a list whose rows begin at `start`: torch's address of an empty tensor is 0, which is no list at
    all, so that of `start`, where nothing is read, stands for it."""
    return _flat(t, dtype, n, dev, name) or (None if t is None or start is None else start.data_ptr())


def _heads(x, dtype, n, d, dev, name):
    """(heads, token stride) of an [n, heads, d] tensor with contiguous heads."""
    shape, s = x.shape, x.stride()
    if (len(shape) != 3 or x.dtype is not dtype or shape[0] != n or shape[2] != d or s[2] != 1
            or (s[1] != d and shape[1] != 1) or x.get_device() != dev):
        raise ValueError(f"{name}: want {dtype} [{n}, heads, {d}] with contiguous heads on GPU {dev}, got {x.dtype} "
                         f"{tuple(shape)} on {x.device}, strides {s}")
    return shape[1], s[0] if n > 1 else shape[1] * d


def _table(t, dev):
    """(rows, width, row stride) of a block table."""
    shape, s = t.shape, t.stride()
    if len(shape) != 2 or t.dtype is not torch.int32 or (s[1] != 1 and shape[1] != 1) or t.get_device() != dev:
        raise ValueError(f"block_table: want int32 [n_seqs, width] with contiguous rows on GPU {dev}, got {t.dtype} "
                         f"{tuple(shape)} on {t.device}, strides {s}")
    return shape[0], shape[1], s[0]


def _rows(x, m, d, dev, name):
    """Row stride of a bf16 or f32 [m, d] tensor with contiguous rows."""
    shape, s = x.shape, x.stride()
    if (len(shape) != 2 or shape[0] != m or shape[1] != d or (x.dtype is not torch.bfloat16 and x.dtype is not torch.float32)
            or (s[1] != 1 and d > 1) or x.get_device() != dev):
        raise ValueError(f"{name}: want bf16 or f32 [{m}, {d}] with contiguous rows on GPU {dev}, got {x.dtype} "
                         f"{tuple(shape)} on {x.device}, strides {s}")
    return s[0] if m > 1 else d


# the raw stream and the current device without building objects (2 us of a small call), where torch has that
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
    (lambda index: torch.cuda.current_stream(index).cuda_stream)

_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _new(shape, dtype, device, stream, strides=None):
    """An uninitialised tensor for a call on `stream` (None: the current one; 0 and 1: the default one)."""
    if stream is not None:
        of = torch.cuda.ExternalStream(stream, device=device) if stream > 1 else torch.cuda.default_stream(device)
        with torch.cuda.stream(of):
            return _new(shape, dtype, device, None, strides)
    if strides is not None:
        return torch.empty_strided(shape, strides, dtype=dtype, device=device)
    return torch.empty(shape, dtype=dtype, device=device)


def rope_table(n_positions, rot_dim, theta=10000.0, device="cuda"):
    """The rotary table that PagedCache.append takes: [n_positions][rot_dim] f32, a position's
    rot_dim / 2 cosines, then its sines, of angles position * theta^(-2 i / rot_dim) in 64 bits."""
    inv = float(theta) ** (-torch.arange(0, rot_dim, 2, dtype=torch.float64, device=device) / rot_dim)
    a = torch.arange(n_positions, dtype=torch.float64, device=device)[:, None] * inv
    return torch.cat([a.cos(), a.sin()], 1).float()


class PagedCache:
    """A paged key-value cache over the caller's pools k and v: tensors [n_pages, n_kv_heads,
    page_size, head_dim] (or with a leading [n_layers]), bf16, or int8 with k_scale and v_scale
    f32 of the same shape without head_dim, contiguous, not negative.  k and v may be strided views of one kind (the
    last dimension contiguous).  The pools are kept alive by this object.  Calls on one object run in
    one stream at a time."""

    def __init__(self, device, k, v, k_scale=None, v_scale=None, max_seqs=256):
        if k.dim() not in (4, 5) or k.shape != v.shape or k.stride() != v.stride() or k.dtype is not v.dtype:
            raise ValueError("k and v: want 4 or 5 dimensions and the same shape, strides and type")
        if k.dtype is not torch.bfloat16 and k.dtype is not torch.int8:
            raise ValueError(f"k: want bf16 or int8, got {k.dtype}")
        dev = device.ordinal
        if k.get_device() != dev or v.get_device() != dev:
            raise ValueError(f"k and v are not on device {dev}")
        if k.stride(-1) != 1:
            raise ValueError("k: the last dimension is not contiguous")
        i8 = k.dtype is torch.int8
        if i8 != (k_scale is not None) or i8 != (v_scale is not None):
            raise ValueError("int8 pools, and only they, have scales")
        five = k if k.dim() == 5 else k[None]
        c = _PagedConfig(int(i8), five.shape[0], five.shape[1], five.shape[3], five.shape[2], five.shape[4], max_seqs,
                         k.data_ptr(), v.data_ptr(), *five.stride()[:4],
                         _dense(k_scale, torch.float32, k.shape[:-1], dev, "k_scale"),
                         _dense(v_scale, torch.float32, k.shape[:-1], dev, "v_scale"))
        self.handle = None
        h = _lib().xdna_paged_cache_create(device.handle, C.byref(c))
        if not h:
            raise XdnaError(last_error())
        self.handle, self._keep = h, (k, v, k_scale, v_scale)
        self.device, self.dev, self.n_kv_heads, self.head_dim = k.device, dev, five.shape[2], five.shape[4]

    def append(self, q, k, v, tok_seq, tok_pos, block_table, rope=None, interleaved=False, layer=0, q_out=None,
               stream=None):
        """Write the rotated keys and the values of len(tok_pos) tokens into the pools and return
        their rotated queries (q_out, bf16 [n, n_q_heads, head_dim]; None for q None).  q, k, v
        [n, heads, head_dim], all bf16 or all f32, heads contiguous, tokens at any stride; tok_seq
        (None: token t is stream t) and tok_pos int32 [n], block_table int32 [n_seqs, width], rope as
        rope_table makes it (None: no rotation)."""
        dev, d, n, src = self.dev, self.head_dim, tok_pos.shape[0], k.dtype
        if src is not torch.bfloat16 and src is not torch.float32:
            raise ValueError(f"k: want bf16 or f32, got {src}")
        kh, ks = _heads(k, src, n, d, dev, "k")
        vh, vs = _heads(v, src, n, d, dev, "v")
        if kh != self.n_kv_heads or vh != kh:
            raise ValueError(f"k and v: want {self.n_kv_heads} heads, got {kh} and {vh}")
        hq = qs = rows = rot = 0
        if q is not None:
            hq, qs = _heads(q, src, n, d, dev, "q")
            if q_out is None:
                q_out = _new((n, hq, d), torch.bfloat16, self.device, stream)
        if rope is not None:
            rows, rot = rope.shape
        n_seqs, width, ts = _table(block_table, dev)
        if n == 0:
            return q_out
        if (_L or _lib()).xdna_paged_append(
                self.handle, layer, n, hq, src is torch.float32, None if q is None else q.data_ptr(), qs, k.data_ptr(),
                ks, v.data_ptr(), vs, _flat(tok_seq, torch.int32, n, dev, "tok_seq"),
                _flat(tok_pos, torch.int32, n, dev, "tok_pos"), block_table.data_ptr(), n_seqs, width, ts,
                _dense(rope, torch.float32, (rows, rot), dev, "rope"), rows, rot, interleaved,
                None if q is None else _dense(q_out, torch.bfloat16, (n, hq, d), dev, "q_out"),
                _raw_stream(dev) if stream is None else stream):
            raise XdnaError(last_error())
        return q_out

    def attend(self, q, block_table, seq_lens, scale=None, window=0, layer=0, out=None, lse=None, stream=None):
        """Attention of one new token per stream, q bf16 [n_seqs, n_q_heads, head_dim], over the last
        `window` (0: all) of its seq_lens[b] positions; scale None: head_dim ** -0.5.  Returns out
        (bf16, as q); lse (f32 [n_seqs, n_q_heads]) is filled when given."""
        dev, d, n = self.dev, self.head_dim, seq_lens.shape[0]
        hq, qs = _heads(q, torch.bfloat16, n, d, dev, "q")
        n_seqs, width, ts = _table(block_table, dev)
        if n_seqs != n:
            raise ValueError(f"block_table: want {n} rows, got {n_seqs}")
        if out is None:
            out = _new((n, hq, d), torch.bfloat16, self.device, stream)
        if n == 0:
            return out
        if (_L or _lib()).xdna_paged_attention(
                self.handle, layer, q.data_ptr(), qs, hq, block_table.data_ptr(), n, width, ts,
                _flat(seq_lens, torch.int32, n, dev, "seq_lens"), d ** -0.5 if scale is None else scale, window,
                _dense(out, torch.bfloat16, (n, hq, d), dev, "out"), _dense(lse, torch.float32, (n, hq), dev, "lse"),
                _raw_stream(dev) if stream is None else stream):
            raise XdnaError(last_error())
        return out

    def check(self, stream=None):
        """Wait for the stream and raise XdnaError for page ids, positions or streams out of range
        that calls since the last check met."""
        _check(_lib().xdna_paged_cache_check(self.handle, _raw_stream(self.dev) if stream is None else stream))

    def close(self):
        if getattr(self, "handle", None):
            _lib().xdna_paged_cache_free(self.handle)
            self.handle = self._keep = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def rmsnorm_residual_i8(x, gamma, residual=None, eps=1e-6, unit_offset=False, q8=None, scale=None, residual_out=None,
                        y=None, quantize=True, stream=None):
    """r = x + residual; y = r / sqrt(mean(r^2) + eps) * gamma (gamma + 1 with unit_offset), as int8
    rows with scales (y = q8 * scale).  x and residual bf16 or f32 [m, d].  Returns (q8, scale,
    residual_out): residual_out holds r in residual's type (None without a residual); a given buffer is
    used, residual itself among them.  `y` (bf16 [m, d]) also takes the unquantised norm;
    quantize=False leaves q8 and scale out (None)."""
    dev = x.get_device()
    if dev < 0 or x.dim() != 2:
        raise ValueError(f"x: want [m, d] on a GPU, got {tuple(x.shape)} on {x.device}")
    if dev != _current_device():
        with torch.cuda.device(dev):
            return rmsnorm_residual_i8(x, gamma, residual, eps, unit_offset, q8, scale, residual_out, y, quantize, stream)
    m, d = x.shape
    xs = _rows(x, m, d, dev, "x")
    rs = 0
    res_f32 = False
    if residual is not None:
        rs = _rows(residual, m, d, dev, "residual")
        res_f32 = residual.dtype is torch.float32
        if residual_out is None:
            residual_out = _new((m, d), residual.dtype, x.device, stream, (rs, 1))
        elif residual_out is not residual and (
                residual_out.dtype is not residual.dtype or _rows(residual_out, m, d, dev, "residual_out") != rs):
            raise ValueError("residual_out: want the type and row stride of residual")
    elif residual_out is not None:
        raise ValueError("residual_out without a residual")
    if quantize:
        if q8 is None:
            q8 = _new((m, d), torch.int8, x.device, stream)
        if scale is None:
            scale = _new((m,), torch.float32, x.device, stream)
    elif q8 is not None or scale is not None:
        raise ValueError("q8 or scale with quantize=False")
    if m == 0:
        return q8, scale, residual_out
    if (_L or _lib()).xdna_rmsnorm_residual_i8(
            x.data_ptr(), x.dtype is torch.float32, xs, None if residual is None else residual.data_ptr(), res_f32, rs,
            _flat(gamma, torch.float32, d, dev, "gamma"), unit_offset, eps, m, d,
            None if residual_out is None else residual_out.data_ptr(), _dense(y, torch.bfloat16, (m, d), dev, "y"),
            _dense(q8, torch.int8, (m, d), dev, "q8"), _flat(scale, torch.float32, m, dev, "scale"),
            _raw_stream(dev) if stream is None else stream):
        raise XdnaError(last_error())
    return q8, scale, residual_out


def process_logits(logits, history=None, history_start=None, n_prompt=None, repetition=None, frequency=None,
                   presence=None, bias_ids=None, bias=None, bias_start=None, mask=None, out=None, ids=None,
                   stream=None):
    """Penalties, biases and mask on logits [b, v] (bf16 or f32), in the order of
    xdna_logits_process; returns (out f32 [b, v], ids int64 [b]: the greedy next token, -1 where the
    mask leaves none).  history int32 [total] with history_start int32 [b + 1]; n_prompt int32 [b];
    repetition, frequency, presence f32 [b]; bias_ids int32, bias f32 [entries] with bias_start int32
    [b + 1]; mask int32 [b, (v + 31) / 32], bit set: allowed.  out may be logits (f32)."""
    dev = logits.get_device()
    if dev < 0 or logits.dim() != 2:
        raise ValueError(f"logits: want [b, v] on a GPU, got {tuple(logits.shape)} on {logits.device}")
    if dev != _current_device():
        with torch.cuda.device(dev):
            return process_logits(logits, history, history_start, n_prompt, repetition, frequency, presence, bias_ids,
                                  bias, bias_start, mask, out, ids, stream)
    b, v = logits.shape
    i32, f32 = torch.int32, torch.float32
    ls = _rows(logits, b, v, dev, "logits")
    if out is None:
        out = _new((b, v), f32, logits.device, stream)
    os_ = _rows(out, b, v, dev, "out")
    if out.dtype is not f32:
        raise ValueError(f"out: want f32, got {out.dtype}")
    if ids is None:
        ids = _new((b,), torch.int64, logits.device, stream)
    if b == 0:
        return out, ids
    L = _L or _lib()
    # rows of several clusters of CTAs need room for their chunks' choices
    work = _new((L.xdna_logits_workspace(b, v),), torch.uint8, logits.device, stream) if v > 60000 else None
    n = 0 if history is None else history.numel()
    e = 0 if bias is None else bias.numel()
    words = (v + 31) // 32
    if L.xdna_logits_process(
            logits.data_ptr(), logits.dtype is f32, ls, b, v, _list(history, history_start, i32, n, dev, "history"), n,
            _flat(history_start, i32, b + 1, dev, "history_start"), _flat(n_prompt, i32, b, dev, "n_prompt"),
            _flat(repetition, f32, b, dev, "repetition"), _flat(frequency, f32, b, dev, "frequency"),
            _flat(presence, f32, b, dev, "presence"), _list(bias_ids, bias_start, i32, e, dev, "bias_ids"),
            _list(bias, bias_start, f32, e, dev, "bias"), e, _flat(bias_start, i32, b + 1, dev, "bias_start"),
            _dense(mask, i32, (b, words), dev, "mask"), words, out.data_ptr(), os_, _flat(ids, torch.int64, b, dev, "ids"),
            None if work is None else work.data_ptr(), _raw_stream(dev) if stream is None else stream):
        raise XdnaError(last_error())
    return out, ids
