// paged_cache.cu -- the paged key-value cache of the serving ops: append with rotary positions,
// and attention of one new token per stream over it (xdna_paged_*, include/xdna_b200.h).
#include <cuda_runtime.h>
#include <cuda_bf16.h>

#include <algorithm>
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
    int sms = 0;
    unsigned *status = nullptr;
    // parts of units that several CTAs share, see the attention kernel; split grows with the units
    // (streams x K/V heads x head groups) that max_seqs allows: at most kMaxGroups groups a head
    float *part_o = nullptr;
    float2 *part_ml = nullptr;
    int2 *split = nullptr;
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
//
// For each stream b and K/V head, with the G query heads that share it:
//   s_j = scale q.k_j,  m = max s_j,  l = sum exp(s_j - m),  o = sum exp(s_j - m) v_j / l
// over the stream's live keys.  Every key and value is read once: 2 n D elements for 4 n G D
// operations, at most G (bf16) or 2 G (int8) operations a byte, so HBM bounds it.
//
// Work split.  A unit is (stream, K/V head, group of up to 8 NT query heads); its keys are cut into
// tiles of 16 keys per warp.  All units' tiles, laid end to end, are dealt to the CTAs in equal
// contiguous shares, whatever the streams' lengths; a CTA walks its share unit by unit.  A unit
// that lies in one CTA is written at once; one that a share's border cuts leaves its
// (max, sum, unnormalised o) in the workspace, and join_kernel adds the parts in CTA order.
//
// Inside a CTA each warp runs alone: its own ring of cp.async stages (16 keys' K and V rows), its own
// running maximum and sum, no barrier until the unit's end, where the warps' parts are added.
// S^T = K q^T and o^T += V^T p^T are m16n8k16 products with the keys (the components) in the 16-row
// operand, so that 8 query heads fill the 8 columns and fewer heads waste nothing but columns.
// The weights p are used as two bf16 terms (16 bits), which keeps the output's error that of its own
// rounding.  Keys past the end, before the window or on a bad page are zero-filled in shared
// memory and masked: what lies in the pool there is not read.
constexpr int kWarps = 4, kStep = 16, kTileKeys = kWarps * kStep;

struct AttnArgs {
    Pool pool;
    Table table;
    const __nv_bfloat16 *q;
    int64_t q_stride;
    const int32_t *lens;
    int n_q_heads, group, n_groups, window, page_shift;   // group: query heads per K/V head
    float scale;                                          // times log2(e)
    __nv_bfloat16 *out;
    float *lse;
    unsigned *status;
    float *part_o;                                        // [2 * grid][8 NT][D]
    float2 *part_ml;                                      // [2 * grid][8 NT]
    int2 *split;                                          // per unit: first part's CTA, parts (0: none)
};

template <int D, bool I8, int NT>
struct AttnShape {
    static constexpr int kRowBytes = D * (I8 ? 1 : 2);
    static constexpr int kRows = 2 * kStep * kRowBytes;                  // K and V of a step
    static constexpr int kStages = kRows >= 8192 ? 3 : kRows >= 4096 ? 4 : 6;
    static constexpr int kStage = kRows + (I8 ? 128 : 0) + 16;           // + scales, + live mask
    static constexpr int kHeads = 8 * NT;
    static constexpr int kJoinRow = 68;                                  // 64 components, padded
    static constexpr int kJoin = kWarps * kHeads * kJoinRow * 4;
    static constexpr int kQRow = D + 8;
    static constexpr int kQ = D == 256 && NT == 2 ? kHeads * kQRow * 2 : 0;  // q in shared memory, see below
    static constexpr int kRing = kWarps * kStages * kStage;              // the join reuses it
    static constexpr int kSmem = kRing + kQ;
    static constexpr int kCtas = kSmem > 112 * 1024 ? 1 : kSmem > 74 * 1024 ? 2 : 3;
    static_assert(kJoin <= kRing, "join");
};

__device__ __forceinline__ void cp_async16_or_zero(uint32_t dst, const void *src, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async4_or_zero(uint32_t dst, const void *src, bool live) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(live ? 4 : 0) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// two of a word's int8 bytes (picked by `sel`) to bf16 pairs, exactly: with v's sign bit s and low
// bits w, v = (128 + w) - (128 + 128 s), and 0x4300 | w, 0x4300 | 128 s are those bf16 numbers
__device__ __forceinline__ uint32_t bf16x2_of_i8(uint32_t word, uint32_t sel) {
    const uint32_t u = __byte_perm(word, 0x43434343u, sel);
    const uint32_t lo = u & 0xff7fff7fu, hi = u & 0xff80ff80u;
    __nv_bfloat162 a, b;
    a = *reinterpret_cast<const __nv_bfloat162 *>(&lo);
    b = *reinterpret_cast<const __nv_bfloat162 *>(&hi);
    const __nv_bfloat162 d = __hsub2(a, b);
    return *reinterpret_cast<const uint32_t *>(&d);
}
// (x, y) as the bf16 pair nearest and the pair of what that leaves
__device__ __forceinline__ void split_bf16x2(float x, float y, uint32_t &hi, uint32_t &lo) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    hi = *reinterpret_cast<const uint32_t *>(&h);
    const __nv_bfloat162 r = __floats2bfloat162_rn(x - xdna::bf16lo(hi), y - xdna::bf16hi(hi));
    lo = *reinterpret_cast<const uint32_t *>(&r);
}

// live keys of stream b: [first, first + count)
__device__ __forceinline__ int2 live_keys(const AttnArgs &a, int b) {
    const int n = min(max(0, a.lens[b]), a.table.width * a.pool.page_size);
    const int first = a.window && n > a.window ? n - a.window : 0;
    return make_int2(first, n - first);
}
__device__ __forceinline__ int tiles_of(int keys) { return (keys + kTileKeys - 1) / kTileKeys; }

template <int D, bool I8, int NT>
__global__ void __launch_bounds__(128, (AttnShape<D, I8, NT>::kCtas)) attention_kernel(const AttnArgs a) {
    using S = AttnShape<D, I8, NT>;
    constexpr int kChunks = S::kRowBytes / 16, kRowsPerCopy = 32 / kChunks < 1 ? 1 : 32 / kChunks;
    constexpr int kMt = D / 16;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ int scan[kWarps], where[4];
    __shared__ float join_m[kWarps][S::kHeads], join_l[kWarps][S::kHeads];
    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, g = lane / 4, j = lane % 4;
    unsigned char *ring = smem + warp * S::kStages * S::kStage;
    const uint32_t ring_u = xdna::smem_u32(ring);
    float *join_o = reinterpret_cast<float *>(smem);
    __nv_bfloat16 *q_s = reinterpret_cast<__nv_bfloat16 *>(smem + S::kRing);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    // ---- this CTA's share: tiles [share0, share1) of all units laid end to end
    const int units_per_stream = a.pool.n_kv_heads * a.n_groups, B = a.table.n_seqs;
    auto block_scan = [&](int x, int &total) {            // inclusive, over the 128 threads
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const int y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        __syncthreads();
        if (lane == 31) scan[warp] = x;
        __syncthreads();
        total = 0;
#pragma unroll
        for (int w = 0; w < kWarps; w++) {
            if (w < warp) x += scan[w];
            total += scan[w];
        }
        return x;
    };
    int64_t total = 0;
    int mine = 0, upto = 0;
    for (int b0 = 0; b0 < B; b0 += 128) {
        mine = b0 + tid < B ? tiles_of(live_keys(a, b0 + tid).y) : 0;
        int sum;
        upto = block_scan(mine, sum);
        total += sum;
    }
    total *= units_per_stream;
    // no share is empty, so that a unit's parts lie in consecutive CTAs
    const int ctas = (int)min((int64_t)gridDim.x, total);
    if ((int)blockIdx.x >= ctas) return;
    const int64_t share0 = total * blockIdx.x / ctas, share1 = total * (blockIdx.x + 1) / ctas;
    int64_t before = 0;                                   // tiles of one head of the streams before b0
    for (int b0 = 0; b0 < B; b0 += 128) {
        int sum;
        if (B > 128) {
            mine = b0 + tid < B ? tiles_of(live_keys(a, b0 + tid).y) : 0;
            upto = block_scan(mine, sum);
        } else {
            sum = 0x7fffffff;
        }
        if ((before + sum) * units_per_stream > share0) {
            const int64_t from = (before + upto - mine) * units_per_stream;
            if (mine && from <= share0 && share0 < from + (int64_t)mine * units_per_stream) {
                where[0] = b0 + tid;
                where[1] = (int)((share0 - from) / mine);
                where[2] = (int)((share0 - from) % mine);
            }
            break;
        }
        before += sum;
    }
    __syncthreads();
    int b = where[0], unit = where[1], t0 = where[2];
    int2 live = live_keys(a, b);
    int tiles = tiles_of(live.y);
    if (tid == 0 && a.lens[b] > a.table.width * a.pool.page_size) atomicOr(a.status, kBadPosition);

    for (int64_t at = share0; at < share1;) {
        const int t1 = (int)min((int64_t)tiles, t0 + (share1 - at));
        const int hk = unit / a.n_groups, h0 = hk * a.group + (unit % a.n_groups) * S::kHeads;
        const int heads = min(S::kHeads, a.group - (unit % a.n_groups) * S::kHeads);
        const unsigned char *kb = static_cast<const unsigned char *>(a.pool.k) + hk * a.pool.sh * (I8 ? 1 : 2);
        const unsigned char *vb = static_cast<const unsigned char *>(a.pool.v) + hk * a.pool.sh * (I8 ? 1 : 2);
        const int32_t *ids = a.table.ids + b * a.table.stride;
        const int end = live.x + live.y;

        // ---- q of the unit's heads as the products' 8-column operand: pair (2j, 2j + 1) and (2j + 8,
        // 2j + 9) of each 16 components; an int8 row's words hold 4 components in order, so there the
        // pairs are (4j, 4j + 1) and (4j + 2, 4j + 3), in K and q alike
        uint32_t qf[S::kQ ? 1 : NT][S::kQ ? 1 : kMt][2];
        const __nv_bfloat16 *q = a.q + b * a.q_stride + (int64_t)h0 * D;
        if constexpr (S::kQ) {                            // 64 registers of q beside 128 of o would spill
            __syncthreads();
            for (int i = tid; i < S::kHeads * D / 2; i += 128)
                reinterpret_cast<uint32_t *>(q_s)[i / (D / 2) * (S::kQRow / 2) + i % (D / 2)] =
                    i / (D / 2) < heads ? reinterpret_cast<const uint32_t *>(q)[i] : 0u;
            __syncthreads();
        } else {
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int c = 0; c < kMt; c++) {
                    const int h = nt * 8 + g, e0 = 16 * c + (I8 ? 4 * j : 2 * j), e1 = e0 + (I8 ? 2 : 8);
                    qf[nt][c][0] = h < heads ? *reinterpret_cast<const uint32_t *>(q + h * D + e0) : 0u;
                    qf[nt][c][1] = h < heads ? *reinterpret_cast<const uint32_t *>(q + h * D + e1) : 0u;
                }
        }

        float o[NT][kMt][4], m[NT][2], ms[NT][2], l[NT][2];   // ms: m, or 0 while there is no maximum
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
#pragma unroll
            for (int c = 0; c < kMt; c++)
#pragma unroll
                for (int i = 0; i < 4; i++) o[nt][c][i] = 0.0f;
#pragma unroll
            for (int i = 0; i < 2; i++) m[nt][i] = -INFINITY, ms[nt][i] = l[nt][i] = 0.0f;
        }

        // ---- the ring: lane r (and r + 16) looks up key r's page a step ahead of its copy
        auto key_of = [&](int t) { return live.x + (t * kWarps + warp) * kStep + (lane & 15); };
        auto page_of = [&](int t) {
            const int pos = key_of(t);
            if (t >= t1 || pos >= end) return -1;
            return ids[a.page_shift >= 0 ? pos >> a.page_shift : pos / a.pool.page_size];
        };
        auto issue = [&](int stage, int t, int page) {
            const int pos = key_of(t);
            bool ok = t < t1 && pos < end;
            if (ok && (unsigned)page >= (unsigned)a.pool.n_pages) {
                atomicOr(a.status, kBadPage);
                ok = false;
            }
            const int slot = a.page_shift >= 0 ? pos & ((1 << a.page_shift) - 1) : pos % a.pool.page_size;
            const int64_t row = ok ? (page * a.pool.sp + slot * a.pool.ss) * (I8 ? 1 : 2) : -1;
            const unsigned mask = __ballot_sync(0xffffffffu, ok) & 0xffffu;
            const uint32_t base = ring_u + stage * S::kStage;
            if (lane == 0) *reinterpret_cast<unsigned *>(ring + stage * S::kStage + S::kStage - 16) = mask;
#pragma unroll
            for (int i = 0; i < kStep / kRowsPerCopy; i++) {
                const int r = i * kRowsPerCopy + (kChunks < 32 ? lane / kChunks : 0), c = lane % kChunks;
                const int64_t off = __shfl_sync(0xffffffffu, row, r);
                const uint32_t dst = base + r * S::kRowBytes + ((c ^ (kChunks >= 8 ? r & 7 : (r >> 1) & 3)) * 16);
                const int64_t from = off < 0 ? 0 : off + c * 16;
                cp_async16_or_zero(dst, kb + from, off >= 0);
                cp_async16_or_zero(dst + kStep * S::kRowBytes, vb + from, off >= 0);
            }
            if constexpr (I8) {
                const int64_t r = ok ? ((int64_t)page * a.pool.n_kv_heads + hk) * a.pool.page_size + slot : 0;
                cp_async4_or_zero(base + S::kRows + lane * 4, (lane < 16 ? a.pool.ks : a.pool.vs) + r, ok);
            }
        };
        int page = page_of(t0);
#pragma unroll
        for (int i = 0; i < S::kStages - 1; i++) {
            const int next = page_of(t0 + i + 1);
            if (t0 + i < t1) issue(i, t0 + i, page);
            xdna::cp_async_commit();
            page = next;
        }
        int stage = 0;
        for (int t = t0; t < t1; t++) {
            xdna::cp_async_wait_group<S::kStages - 2>();
            __syncwarp();
            const int last = stage == 0 ? S::kStages - 1 : stage - 1;
            const int next = page_of(t + S::kStages);
            if (t + S::kStages - 1 < t1) issue(last, t + S::kStages - 1, page);
            xdna::cp_async_commit();
            page = next;

            const uint32_t ks = ring_u + stage * S::kStage, vs = ks + kStep * S::kRowBytes;
            const unsigned char *tail = ring + stage * S::kStage + S::kRows;
            const unsigned mask = *reinterpret_cast<const unsigned *>(tail + (I8 ? 128 : 0));
            if (mask) {
                // ---- S^T: keys g, g + 8 by heads 2j, 2j + 1
                float s[NT][2][4];
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int i = 0; i < 4; i++) s[nt][0][i] = s[nt][1][i] = 0.0f;
                const int r = lane & 15, sw = kChunks >= 8 ? r & 7 : (r >> 1) & 3;
                auto q_of = [&](int nt, int c, int i) -> uint32_t {
                    if constexpr (S::kQ)
                        return *reinterpret_cast<const uint32_t *>(
                            q_s + (nt * 8 + g) * S::kQRow + 16 * c + (I8 ? 4 * j + 2 * i : 2 * j + 8 * i));
                    else
                        return qf[nt][c][i];
                };
                if constexpr (!I8) {
#pragma unroll
                    for (int c = 0; c < kMt; c++) {
                        uint32_t k[4];
                        ldsm4(k, ks + r * S::kRowBytes + (((2 * c + (lane >> 4)) ^ sw) * 16));
#pragma unroll
                        for (int nt = 0; nt < NT; nt++)
                            mma_bf16(s[nt][c & 1], k[0], k[1], k[2], k[3], q_of(nt, c, 0), q_of(nt, c, 1));
                    }
                } else {
#pragma unroll
                    for (int c = 0; c < kMt; c += 2) {
                        uint32_t k[4];
                        ldsm4(k, ks + r * S::kRowBytes + (((c + (lane >> 4)) ^ sw) * 16));
#pragma unroll
                        for (int x = 0; x < 2; x++) {
                            const uint32_t a0 = bf16x2_of_i8(k[2 * x], 0x4140), a2 = bf16x2_of_i8(k[2 * x], 0x4342);
                            const uint32_t a1 = bf16x2_of_i8(k[2 * x + 1], 0x4140), a3 = bf16x2_of_i8(k[2 * x + 1], 0x4342);
#pragma unroll
                            for (int nt = 0; nt < NT; nt++)
                                mma_bf16(s[nt][x], a0, a1, a2, a3, q_of(nt, c + x, 0), q_of(nt, c + x, 1));
                        }
                    }
                }
                // ---- running maximum and weights
                const bool ok0 = (mask >> g) & 1, ok1 = (mask >> (g + 8)) & 1;
                float f0 = a.scale, f1 = a.scale, v0 = 1.0f, v1 = 1.0f;
                if constexpr (I8) {
                    const float *sc = reinterpret_cast<const float *>(tail);
                    f0 *= sc[g]; f1 *= sc[g + 8];
                    v0 = sc[16 + g]; v1 = sc[24 + g];
                }
                bool up = false;
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        s[nt][0][i] = ok0 ? (s[nt][0][i] + s[nt][1][i]) * f0 : -INFINITY;
                        s[nt][0][2 + i] = ok1 ? (s[nt][0][2 + i] + s[nt][1][2 + i]) * f1 : -INFINITY;
                        up |= fmaxf(s[nt][0][i], s[nt][0][2 + i]) > m[nt][i];
                    }
                if (__any_sync(0xffffffffu, up)) {
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
                        float corr[2];
#pragma unroll
                        for (int i = 0; i < 2; i++) {
                            float top = fmaxf(m[nt][i], fmaxf(s[nt][0][i], s[nt][0][2 + i]));
#pragma unroll
                            for (int x = 4; x < 32; x *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
                            corr[i] = top == m[nt][i] ? 1.0f : exp2_approx(m[nt][i] - top);
                            m[nt][i] = top;
                            ms[nt][i] = top == -INFINITY ? 0.0f : top;
                            l[nt][i] *= corr[i];
                        }
#pragma unroll
                        for (int c = 0; c < kMt; c++) {
                            o[nt][c][0] *= corr[0]; o[nt][c][1] *= corr[1];
                            o[nt][c][2] *= corr[0]; o[nt][c][3] *= corr[1];
                        }
                    }
                }
                uint32_t ph[NT][2], pl[NT][2];
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    float p[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        p[i] = exp2_approx(s[nt][0][i] - ms[nt][i & 1]);
                        l[nt][i & 1] += p[i];
                        if constexpr (I8) p[i] *= i < 2 ? v0 : v1;
                    }
                    split_bf16x2(p[0], p[1], ph[nt][0], pl[nt][0]);
                    split_bf16x2(p[2], p[3], ph[nt][1], pl[nt][1]);
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        ph[nt][i] = transpose8x8(ph[nt][i]);
                        pl[nt][i] = transpose8x8(pl[nt][i]);
                    }
                }
                // ---- o^T += V^T p^T; an int8 word's bytes are components (2g, 2g + 1) of two keys: the
                // product's rows g and g + 8 stand for these there
                if constexpr (!I8) {
                    const int rv = (lane & 7) + (lane >> 4) * 8, swv = kChunks >= 8 ? rv & 7 : (rv >> 1) & 3;
#pragma unroll
                    for (int c = 0; c < kMt; c++) {
                        uint32_t v[4];
                        ldsm4_trans(v, vs + rv * S::kRowBytes + (((2 * c + ((lane >> 3) & 1)) ^ swv) * 16));
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) {
                            mma_bf16(o[nt][c], v[0], v[1], v[2], v[3], ph[nt][0], ph[nt][1]);
                            mma_bf16(o[nt][c], v[0], v[1], v[2], v[3], pl[nt][0], pl[nt][1]);
                        }
                    }
                } else {
#pragma unroll
                    for (int c = 0; c < kMt; c += 2) {
                        uint32_t v[4];
                        ldsm4_trans(v, vs + r * S::kRowBytes + (((c + (lane >> 4)) ^ sw) * 16));
#pragma unroll
                        for (int x = 0; x < 2; x++) {
                            const uint32_t a0 = bf16x2_of_i8(v[2 * x], 0x4240), a1 = bf16x2_of_i8(v[2 * x], 0x4341);
                            const uint32_t a2 = bf16x2_of_i8(v[2 * x + 1], 0x4240), a3 = bf16x2_of_i8(v[2 * x + 1], 0x4341);
#pragma unroll
                            for (int nt = 0; nt < NT; nt++) {
                                mma_bf16(o[nt][c + x], a0, a1, a2, a3, ph[nt][0], ph[nt][1]);
                                mma_bf16(o[nt][c + x], a0, a1, a2, a3, pl[nt][0], pl[nt][1]);
                            }
                        }
                    }
                }
            }
            __syncwarp();
            stage = stage + 1 == S::kStages ? 0 : stage + 1;
        }
        xdna::cp_async_wait_all();

        // ---- the warps' parts into one
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
#pragma unroll
                for (int x = 4; x < 32; x *= 2) l[nt][i] += __shfl_xor_sync(0xffffffffu, l[nt][i], x);
                if (g == 0) {
                    join_m[warp][nt * 8 + 2 * j + i] = m[nt][i];
                    join_l[warp][nt * 8 + 2 * j + i] = l[nt][i];
                }
            }
        __syncthreads();
        float fac[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int h = nt * 8 + 2 * j + i;
                float top = join_m[0][h];
#pragma unroll
                for (int w = 1; w < kWarps; w++) top = fmaxf(top, join_m[w][h]);
                fac[nt][i] = m[nt][i] == top ? 1.0f : exp2_approx(m[nt][i] - top);
            }
        const bool whole = t0 == 0 && t1 == tiles;
        const int slot = 2 * blockIdx.x + (t0 == 0);
#pragma unroll
        for (int d0 = 0; d0 < D; d0 += 64) {
            if (d0) __syncthreads();
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int c = 0; c < 4; c++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int comp = 16 * c + (I8 ? 2 * g + (i >> 1) : g + 8 * (i >> 1));
                        join_o[(warp * S::kHeads + nt * 8 + 2 * j + (i & 1)) * S::kJoinRow + comp] =
                            o[nt][d0 / 16 + c][i] * fac[nt][i & 1];
                    }
            __syncthreads();
            for (int x = tid; x < heads * 16; x += 128) {
                const int h = x / 16, c = x % 16 * 4;
                float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int w = 0; w < kWarps; w++) {
                    const float4 y = *reinterpret_cast<const float4 *>(&join_o[(w * S::kHeads + h) * S::kJoinRow + c]);
                    sum.x += y.x; sum.y += y.y; sum.z += y.z; sum.w += y.w;
                }
                if (whole) {
                    float top = join_m[0][h], den = 0.0f;
#pragma unroll
                    for (int w = 1; w < kWarps; w++) top = fmaxf(top, join_m[w][h]);
#pragma unroll
                    for (int w = 0; w < kWarps; w++)
                        den += join_l[w][h] * (join_m[w][h] == top ? 1.0f : exp2_approx(join_m[w][h] - top));
                    const float inv = 1.0f / den;
                    const __nv_bfloat162 lo = __floats2bfloat162_rn(sum.x * inv, sum.y * inv),
                                         hi = __floats2bfloat162_rn(sum.z * inv, sum.w * inv);
                    *reinterpret_cast<uint2 *>(a.out + ((int64_t)b * a.n_q_heads + h0 + h) * D + d0 + c) =
                        make_uint2(*reinterpret_cast<const uint32_t *>(&lo), *reinterpret_cast<const uint32_t *>(&hi));
                } else {
                    *reinterpret_cast<float4 *>(a.part_o + ((int64_t)slot * S::kHeads + h) * D + d0 + c) = sum;
                }
            }
        }
        if (tid < heads) {
            float top = join_m[0][tid], den = 0.0f;
#pragma unroll
            for (int w = 1; w < kWarps; w++) top = fmaxf(top, join_m[w][tid]);
#pragma unroll
            for (int w = 0; w < kWarps; w++)
                den += join_l[w][tid] * (join_m[w][tid] == top ? 1.0f : exp2_approx(join_m[w][tid] - top));
            if (!whole) a.part_ml[slot * S::kHeads + tid] = make_float2(top, den);
            else if (a.lse) a.lse[(int64_t)b * a.n_q_heads + h0 + tid] = (top + log2f(den)) * 0.69314718f;
        }
        if (t0 == 0 && tid == 0) {                        // which CTAs hold the unit's parts
            int2 *sp = a.split + (int64_t)b * units_per_stream + unit;
            if (whole) {
                *sp = make_int2(0, 0);
            } else {
                const int64_t stop = at + tiles - 1;      // the unit's last tile lies in share `to`
                const int64_t to = ((stop + 1) * ctas - 1) / total;
                *sp = make_int2(blockIdx.x, (int)to - (int)blockIdx.x + 1);
            }
        }
        __syncthreads();
        at += t1 - t0;
        t0 = 0;
        if (at < share1 && ++unit == units_per_stream) {
            unit = 0;
            do {
                if (++b == B) return;
                live = live_keys(a, b);
            } while (live.y == 0);
            tiles = tiles_of(live.y);
            if (tid == 0 && a.lens[b] > a.table.width * a.pool.page_size) atomicOr(a.status, kBadPosition);
        }
    }
}

// One CTA per unit and head: a stream of no keys gets zeros; a unit cut among CTAs gets the sum of its
// parts, taken at the largest of their maxima, in CTA order.
template <int D>
__global__ void __launch_bounds__(256) join_kernel(const AttnArgs a, int unit_heads) {
    constexpr int kCols = D / 4, kRowsAtOnce = 256 / kCols;
    __shared__ float red[8], dens[8], weight[1024];
    __shared__ float4 sums[256];
    const int units = a.pool.n_kv_heads * a.n_groups, b = blockIdx.x / units, unit = blockIdx.x % units;
    const int first = (unit % a.n_groups) * unit_heads, h = blockIdx.y, tid = threadIdx.x;
    if (first + h >= a.group) return;
    const int head = unit / a.n_groups * a.group + first + h;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    __nv_bfloat16 *out = a.out + ((int64_t)b * a.n_q_heads + head) * D;
    if (live_keys(a, b).y == 0) {
        if (tid < D / 2) reinterpret_cast<uint32_t *>(out)[tid] = 0u;
        if (a.lse && tid == 0) a.lse[(int64_t)b * a.n_q_heads + head] = -INFINITY;
        return;
    }
    const int2 sp = a.split[blockIdx.x];
    if (sp.y == 0) return;
    // part 0 is its CTA's last unit (slot 1), the others begin their CTAs' shares (slot 0)
    auto slot = [&](int i) { return 2 * (sp.x + i) + (i == 0); };
    float top = -INFINITY;
    for (int i = tid; i < sp.y; i += 256) top = fmaxf(top, a.part_ml[slot(i) * unit_heads + h].x);
#pragma unroll
    for (int x = 16; x; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
    if (tid % 32 == 0) red[tid / 32] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; w++) top = fmaxf(top, red[w]);
    float den = 0.0f;
    for (int i = tid; i < sp.y; i += 256) {
        const float2 ml = a.part_ml[slot(i) * unit_heads + h];
        weight[i] = ml.x == top ? 1.0f : exp2_approx(ml.x - top);
        den = fmaf(ml.y, weight[i], den);
    }
#pragma unroll
    for (int x = 16; x; x >>= 1) den += __shfl_xor_sync(0xffffffffu, den, x);
    if (tid % 32 == 0) dens[tid / 32] = den;
    __syncthreads();
    const int col = tid % kCols, row = tid / kCols;
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
    for (int i = row; i < sp.y; i += kRowsAtOnce) {
        const float4 y = *reinterpret_cast<const float4 *>(a.part_o + ((int64_t)slot(i) * unit_heads + h) * D + col * 4);
        const float w = weight[i];
        sum.x = fmaf(y.x, w, sum.x); sum.y = fmaf(y.y, w, sum.y);
        sum.z = fmaf(y.z, w, sum.z); sum.w = fmaf(y.w, w, sum.w);
    }
    sums[tid] = sum;
    __syncthreads();
    if (row) return;
    den = 0.0f;
#pragma unroll
    for (int w = 0; w < 8; w++) den += dens[w];
#pragma unroll
    for (int r = 1; r < kRowsAtOnce; r++) {
        const float4 y = sums[r * kCols + col];
        sum.x += y.x; sum.y += y.y; sum.z += y.z; sum.w += y.w;
    }
    const float inv = 1.0f / den;
    const __nv_bfloat162 lo = __floats2bfloat162_rn(sum.x * inv, sum.y * inv),
                         hi = __floats2bfloat162_rn(sum.z * inv, sum.w * inv);
    reinterpret_cast<uint2 *>(out)[col] =
        make_uint2(*reinterpret_cast<const uint32_t *>(&lo), *reinterpret_cast<const uint32_t *>(&hi));
    if (a.lse && tid == 0) a.lse[(int64_t)b * a.n_q_heads + head] = (top + log2f(den)) * 0.69314718f;
}

// Workspace of a cache's attention calls, whatever their heads: two parts for every CTA of the largest
// grid, and a split entry per unit
constexpr int kMaxCtasPerSm = 3, kMaxUnitHeads = 16, kMaxGroups = 8;

template <int D, bool I8, int NT>
bool allow_smem() {
    return ck(cudaFuncSetAttribute(attention_kernel<D, I8, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                   AttnShape<D, I8, NT>::kSmem),
              "xdna_paged_cache_create");
}
template <int D>
bool allow_smem() {
    return allow_smem<D, false, 1>() && allow_smem<D, false, 2>() && allow_smem<D, true, 1>() && allow_smem<D, true, 2>();
}

template <int D, bool I8, int NT>
cudaError_t launch_attention(AttnArgs a, int sms, cudaStream_t st) {
    using S = AttnShape<D, I8, NT>;
    static_assert(S::kCtas <= kMaxCtasPerSm && S::kHeads <= kMaxUnitHeads, "workspace");
    a.n_groups = (a.group + S::kHeads - 1) / S::kHeads;
    const int64_t units = (int64_t)a.table.n_seqs * a.pool.n_kv_heads * a.n_groups;
    int64_t keys = (int64_t)a.table.width * a.pool.page_size;
    if (a.window) keys = std::min<int64_t>(keys, a.window);
    const int64_t tiles = units * ((keys + kTileKeys - 1) / kTileKeys);
    const int grid = (int)std::min<int64_t>((int64_t)sms * S::kCtas, tiles);
    attention_kernel<D, I8, NT><<<grid, 128, S::kSmem, st>>>(a);
    if (cudaError_t e = cudaGetLastError()) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)units, std::min(a.group, S::kHeads));
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    cudaLaunchAttribute early{};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &early;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, join_kernel<D>, a, (int)S::kHeads);
}
template <int D>
cudaError_t launch_attention(const AttnArgs &a, bool i8, int sms, cudaStream_t st) {
    if (a.group <= 8) return i8 ? launch_attention<D, true, 1>(a, sms, st) : launch_attention<D, false, 1>(a, sms, st);
    return i8 ? launch_attention<D, true, 2>(a, sms, st) : launch_attention<D, false, 2>(a, sms, st);
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
    if (!on.ok || !ck(cudaDeviceGetAttribute(&c->sms, cudaDevAttrMultiProcessorCount, c->ordinal), "xdna_paged_cache_create") ||
        !(g.head_dim == 64 ? allow_smem<64>() : g.head_dim == 128 ? allow_smem<128>() : allow_smem<256>()) ||
        !ck(cudaMalloc(&c->part_o, (size_t)c->sms * kMaxCtasPerSm * 2 * kMaxUnitHeads * g.head_dim * sizeof(float)),
            "xdna_paged_cache_create") ||
        !ck(cudaMalloc(&c->part_ml, (size_t)c->sms * kMaxCtasPerSm * 2 * kMaxUnitHeads * sizeof(float2)),
            "xdna_paged_cache_create") ||
        !ck(cudaMalloc(&c->split, (size_t)g.max_seqs * g.n_kv_heads * kMaxGroups * sizeof(int2)),
            "xdna_paged_cache_create") ||
        !ck(cudaMalloc(&c->status, sizeof(unsigned)), "xdna_paged_cache_create") ||
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
        cudaFree(c->part_o);
        cudaFree(c->part_ml);
        cudaFree(c->split);
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
    if (n_q_heads / g.n_kv_heads > kMaxUnitHeads * kMaxGroups) return fail(me + "more than 128 query heads per K/V head");
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
    a.scale = scale * 1.44269504f;
    a.out = reinterpret_cast<__nv_bfloat16 *>(out);
    a.lse = lse;
    a.status = c->status;
    a.group = n_q_heads / g.n_kv_heads;
    a.page_shift = g.page_size & (g.page_size - 1) ? -1 : __builtin_ctz(g.page_size);
    a.part_o = c->part_o;
    a.part_ml = c->part_ml;
    a.split = c->split;
    auto st = static_cast<cudaStream_t>(stream);
    const bool i8 = g.kv_type != 0;
    const cudaError_t e = g.head_dim == 64    ? launch_attention<64>(a, i8, c->sms, st)
                          : g.head_dim == 128 ? launch_attention<128>(a, i8, c->sms, st)
                                              : launch_attention<256>(a, i8, c->sms, st);
    return ck(e, "xdna_paged_attention") ? 0 : -1;
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
