// paged_cache.cu -- the paged key-value cache of the serving ops: append with rotary positions,
// and attention of one new token per stream over it (xdna_paged_*, include/xdna_b200.h).
#include <cuda_runtime.h>
#include <cuda_bf16.h>

#include <cstdint>
#include <new>
#include <string>

#include "../../include/xdna_b200.h"
#include "ptx.cuh"

namespace xdna {
void set_last_error_message(const std::string &m);
}
using xdna::set_last_error_message;

// what a call met in its device inputs (the handle's status word)
enum : unsigned { kBadPage = 1, kBadPosition = 2, kBadStream = 4 };

struct XdnaPagedCache {
    int ordinal = 0;
    XdnaPagedCacheConfig cfg{};
    unsigned *status = nullptr;
};

namespace {

bool ck(cudaError_t e, const char *what) {
    if (e == cudaSuccess) return true;
    set_last_error_message(std::string(what) + ": " + cudaGetErrorString(e));
    return false;
}
int fail(const std::string &m) {
    set_last_error_message(m);
    return -1;
}
bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// a call on a cache leaves the caller's current device as it was
struct OnDevice {
    int before = -1, want;
    bool ok = false;
    explicit OnDevice(int ordinal) : want(ordinal) {
        ok = cudaGetDevice(&before) == cudaSuccess && (before == want || cudaSetDevice(want) == cudaSuccess);
    }
    ~OnDevice() {
        if (ok && before != want) cudaSetDevice(before);
    }
};

// pool geometry, passed by value to the kernels (k, v already at the call's layer)
struct Pool {
    void *k, *v;
    float *ks, *vs;                       // int8 scales [page][head][slot] of the layer
    int64_t sp, sh, ss;                   // page, head, slot strides in elements
    int n_pages, page_size, n_kv_heads;
};

struct Table {
    const int32_t *ids;
    int64_t stride;
    int n_seqs, width;
};

// ------------------------------------------------------------------------------- append
struct AppendArgs {
    Pool pool;
    Table table;
    const void *q, *k, *v;
    int64_t q_stride, k_stride, v_stride;
    const int32_t *seq, *pos;
    const float *rope;
    int n_tokens, n_q_heads, rope_rows, rot, interleaved;
    __nv_bfloat16 *q_out;
    unsigned *status;
};

__device__ __forceinline__ void load8(const float *p, float (&x)[8]) {
    const float4 a = reinterpret_cast<const float4 *>(p)[0], b = reinterpret_cast<const float4 *>(p)[1];
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
__device__ __forceinline__ void load8(const __nv_bfloat16 *p, float (&x)[8]) {
    const uint4 a = *reinterpret_cast<const uint4 *>(p);
    const uint32_t u[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        x[2 * i] = xdna::bf16lo(u[i]);
        x[2 * i + 1] = xdna::bf16hi(u[i]);
    }
}
__device__ __forceinline__ void store8(__nv_bfloat16 *p, const float (&x)[8]) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; i++) u[i] = xdna::bf16bits(x[2 * i]) | (xdna::bf16bits(x[2 * i + 1]) << 16);
    *reinterpret_cast<uint4 *>(p) = make_uint4(u[0], u[1], u[2], u[3]);
}
__device__ __forceinline__ uint32_t whole8(float x, float inv) {
    return (uint32_t)(max(-127, min(127, __float2int_rn(__fmul_rn(x, inv))))) & 0xffu;
}
__device__ __forceinline__ void store8(int8_t *p, const float (&x)[8], float inv) {
    uint32_t u[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; i++) u[i / 4] |= whole8(x[i], inv) << (8 * (i % 4));
    *reinterpret_cast<uint2 *>(p) = make_uint2(u[0], u[1]);
}

// One lane per 16 components of a row (a token's head): the two 8-component chunks whose pairs turn
// together, so that a lane holds both halves of its pairs; a row's D / 16 lanes lie side by side in
// a warp, which gives the int8 row's maximum by shuffles.
template <int D, typename Src, bool I8>
__global__ void __launch_bounds__(256) append_kernel(const AppendArgs a) {
    constexpr int L = D / 16;
    const int heads = (a.q ? a.n_q_heads : 0) + 2 * a.pool.n_kv_heads, first_k = heads - 2 * a.pool.n_kv_heads;
    const int64_t item = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) / L;
    const int lane = threadIdx.x % L;
    const bool live = item < (int64_t)a.n_tokens * heads;
    const int t = live ? (int)(item / heads) : 0, hh = live ? (int)(item % heads) : 0;
    const int kind = hh < first_k ? 0 : hh < first_k + a.pool.n_kv_heads ? 1 : 2;
    const int h = kind == 0 ? hh : (hh - first_k) % a.pool.n_kv_heads;

    const int pos = a.pos[t];
    bool skip = pos < 0;
    unsigned bad = 0;
    int page = 0, slot = 0;
    if (live && !skip) {
        if (a.rope && pos >= a.rope_rows) bad |= kBadPosition;
        if (kind) {
            const int s = a.seq ? a.seq[t] : t;
            const int col = pos / a.pool.page_size;
            slot = pos % a.pool.page_size;
            if (s < 0 || s >= a.table.n_seqs) bad |= kBadStream;
            else if (col >= a.table.width) bad |= kBadPosition;
            else {
                page = a.table.ids[(int64_t)s * a.table.stride + col];
                if (page < 0 || page >= a.pool.n_pages) bad |= kBadPage;
            }
        }
        if (bad) {
            if (lane == 0) atomicOr(a.status, bad);
            skip = true;
        }
    }

    const bool turned = kind < 2 && lane * 16 < a.rot;
    const int c0 = turned && !a.interleaved ? lane : 2 * lane;
    const int c1 = turned && !a.interleaved ? lane + a.rot / 16 : 2 * lane + 1;
    float x[8], y[8];
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = y[i] = 0.0f;
    if (live && !skip) {
        const Src *src = static_cast<const Src *>(kind == 0 ? a.q : kind == 1 ? a.k : a.v) +
                         t * (kind == 0 ? a.q_stride : kind == 1 ? a.k_stride : a.v_stride) + h * D;
        load8(src + 8 * c0, x);
        load8(src + 8 * c1, y);
        if (turned) {
            const float *r = a.rope + (int64_t)pos * a.rot + 8 * lane;
            float cs[8], sn[8];
            load8(r, cs);
            load8(r + a.rot / 2, sn);
            auto turn = [](float &u, float &w, float c, float s) {
                const float p = __fsub_rn(__fmul_rn(u, c), __fmul_rn(w, s));
                w = __fadd_rn(__fmul_rn(w, c), __fmul_rn(u, s));
                u = p;
            };
            if (a.interleaved) {
#pragma unroll
                for (int i = 0; i < 4; i++) turn(x[2 * i], x[2 * i + 1], cs[i], sn[i]);
#pragma unroll
                for (int i = 0; i < 4; i++) turn(y[2 * i], y[2 * i + 1], cs[4 + i], sn[4 + i]);
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++) turn(x[i], y[i], cs[i], sn[i]);
            }
        }
    }
    if (kind == 0) {
        if (live) {
            __nv_bfloat16 *o = a.q_out + ((int64_t)t * a.n_q_heads + h) * D;
            store8(o + 8 * c0, x);
            store8(o + 8 * c1, y);
        }
        if (!I8) return;                   // int8: the row's lanes all reach the shuffles below
    }
    if constexpr (I8) {
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) top = fmaxf(top, fmaxf(fabsf(x[i]), fabsf(y[i])));
#pragma unroll
        for (int o = 1; o < L; o *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        if (kind == 0 || !live || skip) return;
        // below 127 / FLT_MAX the factor would be infinite: such a row counts as zero
        const bool zero = !(top > 3.8e-37f);
        const float inv = zero ? 0.0f : __fmul_rn(__frcp_rn(top), 127.0f);
        const int64_t row = ((int64_t)page * a.pool.n_kv_heads + h) * a.pool.page_size + slot;
        int8_t *o = static_cast<int8_t *>(kind == 1 ? a.pool.k : a.pool.v) + page * a.pool.sp + h * a.pool.sh +
                    slot * a.pool.ss;
        store8(o + 8 * c0, x, inv);
        store8(o + 8 * c1, y, inv);
        if (lane == 0) (kind == 1 ? a.pool.ks : a.pool.vs)[row] = zero ? 1.0f : __fdiv_rn(top, 127.0f);
    } else {
        if (!live || skip) return;
        __nv_bfloat16 *o = static_cast<__nv_bfloat16 *>(kind == 1 ? a.pool.k : a.pool.v) + page * a.pool.sp +
                           h * a.pool.sh + slot * a.pool.ss;
        store8(o + 8 * c0, x);
        store8(o + 8 * c1, y);
    }
}

// ---------------------------------------------------------------------------- attention
struct AttnArgs {
    Pool pool;
    Table table;
    const __nv_bfloat16 *q;
    int64_t q_stride;
    const int32_t *lens;
    int n_q_heads, window;
    float scale;
    __nv_bfloat16 *out;
    float *lse;
    unsigned *status;
};

// One CTA per (stream, query head); its 4 warps take every 4th key, a lane D / 32 components.
template <int D, bool I8>
__global__ void __launch_bounds__(128) attention_kernel(const AttnArgs a) {
    constexpr int E = D / 32;
    const int h = blockIdx.x, b = blockIdx.y, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int hk = h / (a.n_q_heads / a.pool.n_kv_heads);
    int n = max(0, a.lens[b]);
    if (n > (int64_t)a.table.width * a.pool.page_size) {
        n = a.table.width * a.pool.page_size;
        if (threadIdx.x == 0) atomicOr(a.status, kBadPosition);
    }
    const int lo = a.window && n > a.window ? n - a.window : 0;
    float q[E], o[E], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int e = 0; e < E; e++) {
        q[e] = __bfloat162float(a.q[b * a.q_stride + h * D + lane * E + e]);
        o[e] = 0.0f;
    }
    for (int j = lo + warp; j < n; j += 4) {
        const int page = a.table.ids[(int64_t)b * a.table.stride + j / a.pool.page_size], slot = j % a.pool.page_size;
        if (page < 0 || page >= a.pool.n_pages) {
            if (lane == 0) atomicOr(a.status, kBadPage);
            continue;
        }
        const int64_t at = page * a.pool.sp + hk * a.pool.sh + slot * a.pool.ss + lane * E;
        const int64_t row = ((int64_t)page * a.pool.n_kv_heads + hk) * a.pool.page_size + slot;
        float s = 0.0f, v[E];
#pragma unroll
        for (int e = 0; e < E; e++) {
            if constexpr (I8) {
                s = fmaf(q[e], (float)static_cast<const int8_t *>(a.pool.k)[at + e], s);
                v[e] = __fmul_rn((float)static_cast<const int8_t *>(a.pool.v)[at + e], a.pool.vs[row]);
            } else {
                s = fmaf(q[e], __bfloat162float(static_cast<const __nv_bfloat16 *>(a.pool.k)[at + e]), s);
                v[e] = __bfloat162float(static_cast<const __nv_bfloat16 *>(a.pool.v)[at + e]);
            }
        }
#pragma unroll
        for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
        if constexpr (I8) s *= a.pool.ks[row];
        s *= a.scale;
        const float mn = fmaxf(m, s), corr = m == mn ? 1.0f : expf(m - mn), p = expf(s - mn);
        l = fmaf(l, corr, p);
#pragma unroll
        for (int e = 0; e < E; e++) o[e] = fmaf(o[e], corr, p * v[e]);
        m = mn;
    }
    __shared__ float sm[4], sl[4], so[4][D];
    if (lane == 0) { sm[warp] = m; sl[warp] = l; }
#pragma unroll
    for (int e = 0; e < E; e++) so[warp][lane * E + e] = o[e];
    __syncthreads();
    const float top = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
    float w[4], sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        w[i] = sl[i] == 0.0f ? 0.0f : expf(sm[i] - top);
        sum = fmaf(sl[i], w[i], sum);
    }
    const bool none = sm[0] == -INFINITY && sl[0] == 0.0f && sl[1] == 0.0f && sl[2] == 0.0f && sl[3] == 0.0f;
    for (int c = threadIdx.x; c < D; c += 128) {
        float acc = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; i++) acc = fmaf(so[i][c], w[i], acc);
        a.out[((int64_t)b * a.n_q_heads + h) * D + c] = __float2bfloat16_rn(none ? 0.0f : acc / sum);
    }
    if (a.lse && threadIdx.x == 0) a.lse[(int64_t)b * a.n_q_heads + h] = none ? -INFINITY : top + logf(sum);
}

Pool pool_of(const XdnaPagedCache *c, int layer) {
    const auto &g = c->cfg;
    const size_t es = g.kv_type ? 1 : 2;
    const int64_t rows = (int64_t)g.n_pages * g.n_kv_heads * g.page_size;
    Pool p{};
    p.k = static_cast<char *>(g.k) + layer * g.stride_layer * es;
    p.v = static_cast<char *>(g.v) + layer * g.stride_layer * es;
    if (g.kv_type) {
        p.ks = g.k_scale + layer * rows;
        p.vs = g.v_scale + layer * rows;
    }
    p.sp = g.stride_page;
    p.sh = g.stride_head;
    p.ss = g.stride_slot;
    p.n_pages = g.n_pages;
    p.page_size = g.page_size;
    p.n_kv_heads = g.n_kv_heads;
    return p;
}

// NULL, or what is wrong with a call's block table
const char *table_fault(const int32_t *table, int n_seqs, int width, int64_t stride) {
    if (!table) return "null block table";
    if (n_seqs < 1 || width < 1) return "empty block table";
    if (n_seqs > 1 && stride < width) return "table_stride below table_width";
    return nullptr;
}

}  // namespace

extern "C" {

XdnaPagedCache *xdna_paged_cache_create(XdnaDevice *dev, const XdnaPagedCacheConfig *cfg) {
    const std::string me = "xdna_paged_cache_create: ";
    auto refuse = [&](const char *m) -> XdnaPagedCache * {
        set_last_error_message(me + m);
        return nullptr;
    };
    if (!dev || !cfg || !cfg->k || !cfg->v) return refuse("null pointer");
    XdnaPagedCacheConfig g = *cfg;
    if (g.kv_type != 0 && g.kv_type != 1) return refuse("kv_type not 0 (bf16) or 1 (int8)");
    if (g.head_dim != 64 && g.head_dim != 128 && g.head_dim != 256) return refuse("head_dim not 64, 128 or 256");
    if (g.n_layers < 1 || g.n_pages < 1 || g.page_size < 1 || g.n_kv_heads < 1 || g.max_seqs < 1)
        return refuse("n_layers, n_pages, page_size, n_kv_heads and max_seqs must be at least 1");
    if (g.n_kv_heads > 1024 || g.max_seqs > 65535) return refuse("more than 1024 K/V heads or 65535 streams");
    if (g.kv_type && (!g.k_scale || !g.v_scale)) return refuse("int8 pools need k_scale and v_scale");
    if (!g.stride_page && !g.stride_head && !g.stride_slot) {
        g.stride_slot = g.head_dim;
        g.stride_head = g.stride_slot * g.page_size;
        g.stride_page = g.stride_head * g.n_kv_heads;
        if (!g.stride_layer) g.stride_layer = g.stride_page * g.n_pages;
    }
    const int64_t unit = g.kv_type ? 16 : 8;
    const int64_t st[4] = {g.stride_layer, g.stride_page, g.stride_head, g.stride_slot};
    const int ext[4] = {g.n_layers, g.n_pages, g.n_kv_heads, g.page_size};
    if (!aligned16(g.k) || !aligned16(g.v)) return refuse("pools not 16-byte aligned");
    for (int i = 0; i < 4; i++)
        if (ext[i] > 1 && (st[i] < g.head_dim || st[i] % unit))
            return refuse("a stride below head_dim or not a multiple of 16 bytes");
    // rows of different (layer, page, head, slot) may not overlap: from the smallest stride up, each
    // must pass what the smaller ones span
    bool used[4] = {false, false, false, false};
    int64_t span = g.head_dim;
    for (int n = 0; n < 4; n++) {
        int at = -1;
        for (int i = 0; i < 4; i++)
            if (!used[i] && ext[i] > 1 && (at < 0 || st[i] < st[at])) at = i;
        if (at < 0) break;
        if (st[at] < span) return refuse("strides let rows overlap");
        span = st[at] * (ext[at] - 1) + span;
        used[at] = true;
    }
    auto *c = new (std::nothrow) XdnaPagedCache();
    if (!c) return refuse("out of host memory");
    c->ordinal = xdna_device_ordinal(dev);
    c->cfg = g;
    OnDevice on(c->ordinal);
    if (!on.ok || !ck(cudaMalloc(&c->status, sizeof(unsigned)), "xdna_paged_cache_create") ||
        !ck(cudaMemset(c->status, 0, sizeof(unsigned)), "xdna_paged_cache_create") ||
        !ck(cudaDeviceSynchronize(), "xdna_paged_cache_create")) {
        xdna_paged_cache_free(c);
        return nullptr;
    }
    return c;
}

void xdna_paged_cache_free(XdnaPagedCache *c) {
    if (!c) return;
    {
        OnDevice on(c->ordinal);
        cudaFree(c->status);
    }
    delete c;
}

int xdna_paged_append(XdnaPagedCache *c, int layer, int n_tokens, int n_q_heads, int src_f32, const void *q,
                      int64_t q_stride, const void *k, int64_t k_stride, const void *v, int64_t v_stride,
                      const int32_t *tok_seq, const int32_t *tok_pos, const int32_t *block_table, int n_seqs,
                      int table_width, int64_t table_stride, const float *rope, int rope_rows, int rot_dim,
                      int interleaved, uint16_t *q_out, void *stream) {
    const std::string me = "xdna_paged_append: ";
    if (!c || !k || !v || !tok_pos || (!q != !q_out)) return fail(me + "null pointer");
    const auto &g = c->cfg;
    if (layer < 0 || layer >= g.n_layers) return fail(me + "layer out of range");
    if (n_tokens < 0 || (q && (n_q_heads < 1 || n_q_heads > 65535))) return fail(me + "bad n_tokens or n_q_heads");
    if (const char *w = table_fault(block_table, n_seqs, table_width, table_stride)) return fail(me + w);
    if (!tok_seq && n_tokens > n_seqs) return fail(me + "more tokens than streams and no tok_seq");
    if (rot_dim < 0 || rot_dim > g.head_dim || rot_dim % 16 || (rot_dim > 0) != (rope != nullptr) ||
        (rope && rope_rows < 1))
        return fail(me + "rot_dim not a multiple of 16 up to head_dim, or rope table missing or empty");
    const int64_t unit = src_f32 ? 4 : 8;
    if (k_stride < (int64_t)g.n_kv_heads * g.head_dim || v_stride < (int64_t)g.n_kv_heads * g.head_dim ||
        (q && q_stride < (int64_t)n_q_heads * g.head_dim))
        return fail(me + "a token stride below its heads' width");
    if (k_stride % unit || v_stride % unit || (q && q_stride % unit) || !aligned16(q) || !aligned16(k) ||
        !aligned16(v) || !aligned16(q_out) || !aligned16(rope))
        return fail(me + "rows not 16-byte aligned");
    if (n_tokens == 0) return 0;
    OnDevice on(c->ordinal);
    if (!on.ok) return fail(me + "cannot select the cache's device");
    AppendArgs a{};
    a.pool = pool_of(c, layer);
    a.table = {block_table, table_stride, n_seqs, table_width};
    a.q = q; a.k = k; a.v = v;
    a.q_stride = q_stride; a.k_stride = k_stride; a.v_stride = v_stride;
    a.seq = tok_seq; a.pos = tok_pos;
    a.rope = rope; a.rope_rows = rope_rows; a.rot = rot_dim; a.interleaved = interleaved;
    a.n_tokens = n_tokens; a.n_q_heads = q ? n_q_heads : 0;
    a.q_out = reinterpret_cast<__nv_bfloat16 *>(q_out);
    a.status = c->status;
    const int64_t lanes = (int64_t)n_tokens * (a.n_q_heads + 2 * g.n_kv_heads) * (g.head_dim / 16);
    const int64_t blocks = (lanes + 255) / 256;
    if (blocks > 0x7fffffff) return fail(me + "too many tokens for one call");
    auto st = static_cast<cudaStream_t>(stream);
    auto go = [&](auto d) {
        constexpr int D = decltype(d)::value;
        if (g.kv_type) {
            if (src_f32) append_kernel<D, float, true><<<(unsigned)blocks, 256, 0, st>>>(a);
            else append_kernel<D, __nv_bfloat16, true><<<(unsigned)blocks, 256, 0, st>>>(a);
        } else {
            if (src_f32) append_kernel<D, float, false><<<(unsigned)blocks, 256, 0, st>>>(a);
            else append_kernel<D, __nv_bfloat16, false><<<(unsigned)blocks, 256, 0, st>>>(a);
        }
    };
    if (g.head_dim == 64) go(std::integral_constant<int, 64>{});
    else if (g.head_dim == 128) go(std::integral_constant<int, 128>{});
    else go(std::integral_constant<int, 256>{});
    return ck(cudaGetLastError(), "xdna_paged_append") ? 0 : -1;
}

int xdna_paged_attention(XdnaPagedCache *c, int layer, const uint16_t *q, int64_t q_stride, int n_q_heads,
                         const int32_t *block_table, int n_seqs, int table_width, int64_t table_stride,
                         const int32_t *seq_lens, float scale, int window, uint16_t *out, float *lse, void *stream) {
    const std::string me = "xdna_paged_attention: ";
    if (!c || !q || !seq_lens || !out) return fail(me + "null pointer");
    const auto &g = c->cfg;
    if (layer < 0 || layer >= g.n_layers) return fail(me + "layer out of range");
    if (const char *w = table_fault(block_table, n_seqs, table_width, table_stride)) return fail(me + w);
    if (n_seqs > g.max_seqs) return fail(me + "more streams than the cache's max_seqs");
    if (n_q_heads < 1 || n_q_heads > 65535 || n_q_heads % g.n_kv_heads)
        return fail(me + "n_q_heads not a multiple of the cache's K/V heads");
    if ((int64_t)table_width * g.page_size > 0x40000000) return fail(me + "more than 2^30 positions in a table row");
    if (window < 0 || !(scale > 0.0f)) return fail(me + "negative window or scale not above 0");
    if (q_stride < (int64_t)n_q_heads * g.head_dim || q_stride % 8 || !aligned16(q) || !aligned16(out))
        return fail(me + "q_stride below the heads' width, or rows not 16-byte aligned");
    OnDevice on(c->ordinal);
    if (!on.ok) return fail(me + "cannot select the cache's device");
    AttnArgs a{};
    a.pool = pool_of(c, layer);
    a.table = {block_table, table_stride, n_seqs, table_width};
    a.q = reinterpret_cast<const __nv_bfloat16 *>(q);
    a.q_stride = q_stride;
    a.lens = seq_lens;
    a.n_q_heads = n_q_heads;
    a.window = window;
    a.scale = scale;
    a.out = reinterpret_cast<__nv_bfloat16 *>(out);
    a.lse = lse;
    a.status = c->status;
    auto st = static_cast<cudaStream_t>(stream);
    const dim3 grid(n_q_heads, n_seqs);
    auto go = [&](auto d) {
        constexpr int D = decltype(d)::value;
        if (g.kv_type) attention_kernel<D, true><<<grid, 128, 0, st>>>(a);
        else attention_kernel<D, false><<<grid, 128, 0, st>>>(a);
    };
    if (g.head_dim == 64) go(std::integral_constant<int, 64>{});
    else if (g.head_dim == 128) go(std::integral_constant<int, 128>{});
    else go(std::integral_constant<int, 256>{});
    return ck(cudaGetLastError(), "xdna_paged_attention") ? 0 : -1;
}

int xdna_paged_cache_check(XdnaPagedCache *c, void *stream) {
    if (!c) return fail("xdna_paged_cache_check: null cache");
    OnDevice on(c->ordinal);
    if (!on.ok) return fail("xdna_paged_cache_check: cannot select the cache's device");
    auto st = static_cast<cudaStream_t>(stream);
    unsigned got = 0;
    if (!ck(cudaMemcpyAsync(&got, c->status, sizeof(got), cudaMemcpyDeviceToHost, st), "xdna_paged_cache_check") ||
        !ck(cudaMemsetAsync(c->status, 0, sizeof(got), st), "xdna_paged_cache_check") ||
        !ck(cudaStreamSynchronize(st), "xdna_paged_cache_check"))
        return -1;
    if (!got) return 0;
    std::string m = "xdna_paged_cache_check:";
    if (got & kBadPage) m += " a page id outside the pool;";
    if (got & kBadPosition) m += " a position past the block table or the rope rows;";
    if (got & kBadStream) m += " a stream index outside the block table;";
    m.back() = '.';
    return fail(m);
}

}  // extern "C"
