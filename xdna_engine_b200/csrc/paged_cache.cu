// paged_cache.cu -- the paged key-value cache of the serving ops: append with rotary positions,
// and attention of one new token per stream over it (xdna_paged_*, include/xdna_b200.h).
#include <cuda_runtime.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cstdint>
#include <new>
#include <string>
#include <type_traits>

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
    // parts of units that several CTAs share and counts of those that are there, see the attention kernel
    float *part_o = nullptr;
    float2 *part_ml = nullptr;
    int *arrived = nullptr;
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
// the pointers that lie off their elements' boundary (NULL does not)
template <typename... P>
bool off_elements(size_t bytes, P... p) {
    return ((reinterpret_cast<uintptr_t>(p) % bytes) | ...) != 0;
}

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
    int n_tokens, n_q_heads, rope_rows, rot, interleaved, page_shift;
    __nv_bfloat16 *q_out;
    unsigned *status;
};

// values that are read once pass L1 by, which holds the rotary rows that all heads of a token read
__device__ __forceinline__ void load8_rope(const float *p, float (&x)[8]) {
    const float4 a = __ldg(reinterpret_cast<const float4 *>(p)), b = __ldg(reinterpret_cast<const float4 *>(p) + 1);
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
__device__ __forceinline__ void load8(const float *p, float (&x)[8]) {
    const float4 a = __ldcs(reinterpret_cast<const float4 *>(p)), b = __ldcs(reinterpret_cast<const float4 *>(p) + 1);
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
__device__ __forceinline__ void load8(const __nv_bfloat16 *p, float (&x)[8]) {
    const uint4 a = __ldcs(reinterpret_cast<const uint4 *>(p));
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
    for (int i = 0; i < 4; i++) {
        const __nv_bfloat162 two = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
        u[i] = *reinterpret_cast<const uint32_t *>(&two);
    }
    *reinterpret_cast<uint4 *>(p) = make_uint4(u[0], u[1], u[2], u[3]);
}
// x inv + 1.5 2^23 rounds x inv to a whole number, half to even, whose low byte is the int8
__device__ __forceinline__ void store8(int8_t *p, const float (&x)[8], float inv) {
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; i++) w[i] = __float_as_uint(__fadd_rn(__fmul_rn(x[i], inv), 12582912.0f));
    *reinterpret_cast<uint2 *>(p) =
        make_uint2(__byte_perm(__byte_perm(w[0], w[1], 0x0040), __byte_perm(w[2], w[3], 0x0040), 0x5410),
                   __byte_perm(__byte_perm(w[4], w[5], 0x0040), __byte_perm(w[6], w[7], 0x0040), 0x5410));
}

// One lane per 16 components of a row (a token's head): the two 8-component chunks whose pairs turn
// together, so that a lane holds both halves of its pairs; a row's D / 16 lanes lie side by side in
// a warp, which gives the int8 row's maximum by shuffles.  4 or 2 bytes in and 2 or 1 out per element, so
// HBM bounds it; a token's rotary row comes from L1 for all its heads but the first.  Measured: 8192 tokens
// of 32/8 heads x 128, f32 in, 52.7 us (5.8 TB/s; several heads to a lane, with the rotary row kept in
// registers: 60 us); 2003 tokens of 4/1 x 256 into int8 5.0 us; 64 tokens 2.7 us.  Six CTAs an SM leave 40
// registers a thread and spill 20 to 32 bytes.
template <int D, typename Src, bool I8>
__global__ void __launch_bounds__(256, 6) append_kernel(const AppendArgs a) {
    constexpr int L = D / 16;
    const int heads = (a.q ? a.n_q_heads : 0) + 2 * a.pool.n_kv_heads, first_k = heads - 2 * a.pool.n_kv_heads;
    const unsigned item = blockIdx.x * (256 / L) + threadIdx.x / L;   // n_tokens * heads are below 2^31
    const int lane = threadIdx.x % L;
    const bool live = item < (unsigned)a.n_tokens * heads;
    const int t = live ? item / heads : 0, hh = live ? item - t * heads : 0;
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
            const int col = a.page_shift >= 0 ? pos >> a.page_shift : pos / a.pool.page_size;
            slot = pos - col * a.pool.page_size;
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
            load8_rope(r, cs);
            load8_rope(r + a.rot / 2, sn);
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
        // magnitudes ordered as bits, so that a NaN is the largest and makes the row's scale NaN
        unsigned bits = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) bits = max(bits, max(__float_as_uint(fabsf(x[i])), __float_as_uint(fabsf(y[i]))));
#pragma unroll
        for (int o = 1; o < L; o *= 2) bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, o));
        if (kind == 0 || !live || skip) return;
        const float top = __uint_as_float(bits);
        // below 127 / FLT_MAX the factor would be infinite: such a row counts as zero
        const bool zero = top <= 3.8e-37f;
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
// over the stream's live keys.  Up to 16 heads a group, every key and value is read once (of more, once for each 16):
// 2 n D elements for 4 n G D operations, at most 16 (bf16) or 32 (int8) operations a byte, so HBM bounds it.
//
// Work split.  A unit is (stream, K/V head, group of up to 8 NT query heads); its keys are cut into
// tiles of 16 keys per warp.  All units' tiles, laid end to end, are dealt to the CTAs in equal
// contiguous shares, whatever the streams' lengths; a CTA walks its share unit by unit.  A unit's end
// counts as kEndCost tiles, since its work there costs so much (32 ragged streams of 12 heads x 64, up
// to 2k: 32.2 us at 0, 29.5 at 1, 27.4 at 2, 27.2 at 3; 28.0 now at 2).  A unit
// that lies in one CTA is written at once; of one that shares' borders cut, each CTA leaves its
// (max, sum, unnormalised o) in the workspace, and the last of every 16 neighbours to do so adds
// theirs, in CTA order whoever is last, until one is left: no CTA waits, no second launch.  A fence, an
// atomic and a part's way through L2 take about 3 us, as long as some 4 tiles: a small call gets
// fewer CTAs, so that a unit has no more than 16 parts, or equally many CTAs a unit.
//
// Inside a CTA each warp runs alone: its own ring of cp.async stages (16 keys' K and V rows), which
// runs on over the share's units without a break, its own running maximum and sum, no barrier
// until a unit's end, where the warps' parts are added.  S^T = K q^T and o^T += V^T p^T are m16n8k16
// products with the keys (the components) in the 16-row operand, so that 8 query heads fill the 8
// columns and fewer heads waste nothing but columns.  The weights p are used as three bf16 terms, which
// hold all of an f32 (of two terms, 17 bits, the output comes to the other bf16 neighbour four times as often as
// of an f32 sum; one stream of 4k takes 0.4 us less with them, larger calls the same).  Keys past the end,
// before the window or on a bad page are zero-filled in shared memory and masked: what lies in the pool there is not read.
//
// int8 pools: a value's scale goes into its key's weight, p v_scale in f32.  V's whole numbers become bf16, the only
// 16-bit type that holds such weights whatever they are: as fp16 (4 x 64k 99 us, now 116) those 2^39 below the
// largest vanish, be its value row zero or not.  K's become fp16, in 5/4 instructions a pair to bf16's 17/4, and q is
// scaled for that by a power of two per head to fp16's upper range: components of q down to 2^-30 of the
// head's largest are exact, the others off by 2^-38 of it at most.
//
// Measured back to back: 64 streams of 0 to 8k, 32/8 heads x 128, pages of 16, 182 us (5.9 TB/s, 90 % of a copy);
// 4 x 64k in int8 117 us (4.7 TB/s; 137 us in calls of a second and more, under lower clocks), bound by its
// instructions: 60 % of the issue slots with 3 warps a scheduler; 32 streams of 0 to 2k, 12 heads x 64, 28.0 us; one
// stream of 4k, 4/1 x 256, 13.4 us, a chain of waits.
constexpr int kWarps = 4, kStep = 16, kTileKeys = kWarps * kStep;

struct AttnArgs {
    Pool pool;
    Table table;
    const __nv_bfloat16 *q;
    int64_t q_stride;
    const int32_t *lens;
    int n_q_heads, group, n_groups, window, page_shift;   // group: query heads per K/V head
    int whole_steps, dense_steps;                         // a page holds whole steps of 16 keys; their rows lie side by side
    float scale;                                          // times log2(e)
    __nv_bfloat16 *out;
    float *lse;
    unsigned *status;
    float *part_o;                                        // [2 * grid][8 NT][D]
    float2 *part_ml;                                      // [2 * grid][8 NT]
    int *arrived;                                         // [kJoinLevels][2 * grid], zero between calls
};
constexpr int kMaxCtasPerSm = 3, kMaxUnitHeads = 16, kMaxGroups = 8;
constexpr int kJoinWays = 16, kJoinLevels = 3;            // 16^3 parts

template <int D, bool I8, int NT>
struct AttnShape {
    // bf16 rows of 256 are halved between two warps, which both work on a step's 16 keys and exchange their parts
    // of the scores: one CTA's ring fills the SM, and 4 warps are one to a scheduler (one stream of 4k
    // 13.1 us so, 12.4 us with pairs; 53 streams to 5.8k 39.8 and 37.3 us)
    static constexpr int kPair = D == 256 && !I8 ? 2 : 1, kPart = D / kPair;   // components to a warp
    static constexpr int kThreads = 32 * kWarps * kPair;
    static constexpr int kRowBytes = kPart * (I8 ? 1 : 2);
    static constexpr int kRows = 2 * kStep * kRowBytes;                  // K and V of a step
    static constexpr int kStages = kRows >= 8192 ? 3 : kRows >= 4096 ? 4 : 6;
    static constexpr int kStage = kRows + (I8 ? 128 : 0) + 16;           // + scales, + live mask
    static constexpr int kHeads = 8 * NT;
    static constexpr int kEndCost = 2, kApartTiles = 4;
    static constexpr int kRing = kWarps * kPair * kStages * kStage;
    static constexpr int kJoinCols = 32, kJoinRow = kJoinCols + 4;
    static constexpr int kJoin = kWarps * kPair * kHeads * kJoinRow * 4;
    static_assert(kPair == 1 || kJoin >= 2 * kWarps * kPair * 32 * NT * 16, "a pair's scores, twice, lie there too");
    static constexpr int kQRow = D + 8;
    static constexpr int kQ = kHeads * kQRow * 2 + kHeads * 4;           // q, and an int8 pool's factors
    static constexpr bool kQInRegs = !(kPart == 256 && NT == 2);             // 64 registers of q beside 128 of o would not fit (without, int8 still spills 164 bytes)
    static constexpr int kSmem = kRing + kJoin + kQ;
    static_assert(kSmem + 2048 <= 227 * 1024, "shared memory");
    static constexpr int kCtas = 3 * (kSmem + 1800) <= 228 * 1024 ? 3 : 2 * (kSmem + 1800) <= 228 * 1024 ? 2 : 1;
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
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// bytes sel of a word of int8 + 128 (the word with its sign bits flipped) as an fp16 pair, exactly:
// 0x6400 | u is 1024 + u
__device__ __forceinline__ uint32_t f16x2_of_u8(uint32_t word, uint32_t sel) {
    const uint32_t u = __byte_perm(word, 0x64646464u, sel), off = 0x64806480u;   // 1024 + 128
    const __half2 d = __hsub2(*reinterpret_cast<const __half2 *>(&u), *reinterpret_cast<const __half2 *>(&off));
    return *reinterpret_cast<const uint32_t *>(&d);
}
// the low bytes of a word's halves, signed, as a bf16 pair, exactly.  With u = x + 128, 0x4300 | u is 128 + u up to
// 255 and 2 u from 256, of which x = f / 2 - 128 - max(128 - f / 2, 0)
__device__ __forceinline__ uint32_t bf16x2_of_s8(uint32_t word) {
    const uint32_t f = (word & 0x00ff00ffu) ^ 0x43804380u;
    uint32_t r, y;
    asm("{.reg .b32 half, back;\n\tmov.b32 half, 0x3f003f00;\n\tmov.b32 back, 0xbf00bf00;\n\t"
        "fma.rn.relu.bf16x2 %0, %2, back, %3;\n\tfma.rn.bf16x2 %1, %2, half, %4;\n\t}" : "=&r"(r), "=r"(y) : "r"(f), "r"(0x43004300u), "r"(0xc300c300u));
    const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162 *>(&y), *reinterpret_cast<const __nv_bfloat162 *>(&r));
    return *reinterpret_cast<const uint32_t *>(&d);
}
// (x, y) as bf16 pairs, each the nearest to what the ones before it leave
template <int N>
__device__ __forceinline__ void split_pair(float x, float y, uint32_t (&t)[N]) {
#pragma unroll
    for (int n = 0; n < N; n++) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
        t[n] = *reinterpret_cast<const uint32_t *>(&h);
        x -= xdna::bf16lo(t[n]);
        y -= xdna::bf16hi(t[n]);
    }
}

// live keys of a stream of n tokens: [x, y); tiles are laid from `first`: with whole steps to a page, from
// the step that holds x, so that no step crosses a page
struct Live {
    int x, y, first, tiles;
};
__device__ __forceinline__ Live live_keys(const AttnArgs &a, int n) {
    Live k;
    k.y = min(max(0, n), a.table.width * a.pool.page_size);
    k.x = a.window && k.y > a.window ? k.y - a.window : 0;
    k.first = a.whole_steps ? k.x & -kStep : k.x;
    k.tiles = (k.y - k.first + kTileKeys - 1) / kTileKeys;
    return k;
}

template <int D, bool I8, int NT, bool kSmall>
__global__ void __launch_bounds__((AttnShape<D, I8, NT>::kThreads), (AttnShape<D, I8, NT>::kCtas)) attention_kernel(const AttnArgs a) {
    using S = AttnShape<D, I8, NT>;
    constexpr int kChunks = S::kRowBytes / 16, kRowsPerCopy = kChunks >= 32 ? 1 : 32 / kChunks, kCopies = kStep / kRowsPerCopy;
    constexpr int kMt = S::kPart / 16, kElem = I8 ? 1 : 2, kThreads = S::kThreads;
    constexpr int kTerms = 3;                             // bf16 terms of a weight
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ float join_m[kWarps][S::kHeads], join_l[kWarps][S::kHeads];
    __shared__ int last;
    // warp: which 16 keys of a tile; half: which of a pair's two
    const int tid = threadIdx.x, any_warp = tid / 32, warp = any_warp / S::kPair, half = any_warp % S::kPair;
    const int lane = tid % 32, g = lane / 4, j = lane % 4;
    unsigned char *ring = smem + any_warp * S::kStages * S::kStage;
    const uint32_t ring_u = xdna::smem_u32(ring);
    float *join_o = reinterpret_cast<float *>(smem + S::kRing);
    uint16_t *q_s = reinterpret_cast<uint16_t *>(smem + S::kRing + S::kJoin);
    float *q_inv = reinterpret_cast<float *>(q_s + S::kHeads * S::kQRow);
    [[maybe_unused]] float *swap = reinterpret_cast<float *>(smem + S::kRing);   // pairs' scores, between joins
    // ---- streams of no keys, once the CTA is through
    auto empty_streams = [&]() {
        for (int b = blockIdx.x; b < a.table.n_seqs; b += gridDim.x) {
            const int n = a.lens[b];
            if (n > a.table.width * a.pool.page_size && tid == 0) atomicOr(a.status, kBadPosition);
            if (n > 0) continue;
            uint4 *out = reinterpret_cast<uint4 *>(a.out + (int64_t)b * a.n_q_heads * D);
            for (int i = tid; i < a.n_q_heads * (D / 8); i += kThreads) out[i] = make_uint4(0, 0, 0, 0);
            if (a.lse)
                for (int i = tid; i < a.n_q_heads; i += kThreads) a.lse[(int64_t)b * a.n_q_heads + i] = -INFINITY;
        }
    };

    // ---- this CTA's share: [share0, share1) of all units' tiles and ends laid end to end.  Every warp works
    // it out for itself, 128 streams at a time, 4 to a lane.
    const int units_per_stream = a.pool.n_kv_heads * a.n_groups, B = a.table.n_seqs;
    int tiles4[4], mine = 0, upto = 0;                    // of a lane's streams, their sum, the sum up to them
    int some = 0, some_upto = 0;                          // the same for how many have any
    auto count128 = [&](int b0) {
        mine = some = 0;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int b = b0 + lane * 4 + k;
            tiles4[k] = b < B ? live_keys(a, a.lens[b]).tiles : 0;
            mine += tiles4[k];
            some += tiles4[k] != 0;
        }
        upto = mine;
        some_upto = some;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const int y = __shfl_up_sync(0xffffffffu, upto, o), z = __shfl_up_sync(0xffffffffu, some_upto, o);
            if (lane >= o) {
                upto += y;
                some_upto += z;
            }
        }
    };
    using Int = std::conditional_t<kSmall, int, int64_t>;  // total * ctas fits
    Int total = 0, live_units = 0;
    int longest = 0;
    for (int b0 = 0; b0 < B; b0 += 128) {
        count128(b0);
        total += __shfl_sync(0xffffffffu, upto, 31);
        live_units += __shfl_sync(0xffffffffu, some_upto, 31);
        longest = max(longest, __reduce_max_sync(0xffffffffu, max(max(tiles4[0], tiles4[1]), max(tiles4[2], tiles4[3]))));
    }
    total *= units_per_stream;
    live_units *= units_per_stream;
    if (total == 0) {
        empty_streams();
        return;
    }
    // Short units, one CTA to each: its own steps take less than a join would (6 streams x 3 heads x 64 of 2
    // tiles 5.8 us, in parts 7.7, of 4 tiles 7.0 and 7.8; 32 x 5 x 128 of 3 tiles 9.0 and 8.7; beyond, 6 x 3 of up
    // to 10 tiles 12.6 us so, 8.4 in parts).  Else no
    // share is empty, so that a unit's parts lie in consecutive CTAs (one may hold an end alone): up to 64
    // tiles a unit, no more CTAs than make 16 parts of the longest (one unit of 32 tiles 10.9 us, else 12.3; of 64
    // 13.4 and 12.5, 16 such units 13.9 and 16.3; past the border, 16 units of 65 tiles 16.4 us, within the rule 14.2,
    // but one of 65 12.4 and 14.6, of 128 12.3 and 19.0); units of one length and few tiles, as many CTAs to each, whose
    // parts then all have an end (64 units of 8 tiles 14.3 us, else 15.7; 160 of 8 15.1 and 18.5)
    const bool apart = live_units <= (Int)gridDim.x && longest <= S::kApartTiles;
    Int want = min((Int)gridDim.x, total);
    if (longest <= 4 * kJoinWays) want = min(want, total * kJoinWays / longest);
    const bool even = live_units < want && total < 8 * want && (Int)longest * live_units == total;
    if (even) want = want / live_units * live_units;
    const int ctas = (int)(apart ? live_units : want), end_cost = even ? 0 : S::kEndCost;
    if ((int)blockIdx.x >= ctas) {
        empty_streams();
        return;
    }
    total += live_units * end_cost;
    const Int share0 = apart ? (Int)blockIdx.x : total * (Int)blockIdx.x / ctas;
    const Int share1 = apart ? share0 + 1 : total * (Int)(blockIdx.x + 1) / ctas;
    int at_b = 0, at_unit = 0, at_tile = 0;
    Int before = 0;                                       // what the streams before b0 come to
    for (int b0 = 0; b0 < B; b0 += 128) {
        if (B > 128) count128(b0);
        // what a lane's streams come to, of one unit each: in tiles and ends, or in units
        const Int own = apart ? (Int)some : mine + (Int)some * end_cost;
        const Int upto_own = apart ? (Int)some_upto : upto + (Int)some_upto * end_cost;
        const Int sum = __shfl_sync(0xffffffffu, upto_own, 31);
        if (before + sum * units_per_stream > share0) {
            Int from = before + (upto_own - own) * units_per_stream;
            const bool here = own && from <= share0 && share0 < from + own * units_per_stream;
            auto unit_of = [&](int q) { return tiles4[q] == 0 ? 0 : apart ? 1 : tiles4[q] + end_cost; };
            int k = 0, n = max(1, unit_of(0));
#pragma unroll
            for (int q = 0; q < 3; q++) {
                const Int next = from + (Int)unit_of(q) * units_per_stream;
                if (k == q && share0 >= next) {
                    from = next;
                    k = q + 1;
                    n = max(1, unit_of(q + 1));
                }
            }
            const Int off = here ? share0 - from : 0;
            const int unit = (int)(off / n), tile = (int)(off - (Int)unit * n);
            const int owner = __ffs(__ballot_sync(0xffffffffu, here)) - 1;
            at_b = __shfl_sync(0xffffffffu, b0 + lane * 4 + k, owner);
            at_unit = __shfl_sync(0xffffffffu, unit, owner);
            at_tile = __shfl_sync(0xffffffffu, tile, owner);
            break;
        }
        before += sum * units_per_stream;
    }

    // ---- a place in the share: a unit of a stream, and a tile of its keys
    struct Place {
        int b, unit, t;
        Live live;
    };
    auto next_unit = [&](Place &p) {                      // only within the share: there is one
        p.t = 0;
        if (++p.unit == units_per_stream) {
            p.unit = 0;
            do {
                if (++p.b >= B) { p.b = B - 1; return; }
                p.live = live_keys(a, a.lens[p.b]);
            } while (p.live.tiles == 0);
        }
    };
    Place at{at_b, at_unit, at_tile, live_keys(a, a.lens[at_b])}, ahead = at;
    int left = apart ? at.live.tiles : (int)(share1 - share0), unfetched = left;
    Int unit_at = share0 - at.t;                          // where the unit begins
    auto pass_end = [&](Place &p, int &rest) {            // from a unit's last tile to the next unit, if the share goes on
        rest -= end_cost;
        if (rest > 0) next_unit(p);
    };
    if (at.t >= at.live.tiles) {                          // the share begins in a unit's end
        unit_at += at.live.tiles + end_cost;
        left -= (int)(unit_at - share0) - end_cost;
        pass_end(at, left);
        if (left <= 0) {
            empty_streams();
            return;
        }
        ahead = at;
        unfetched = left;
    }

    // ---- the ring.  issue() copies the step of the place `ahead`, whose page (that of its key r in lanes r
    // and r + 16, where steps do not lie whole in pages) look_up() fetched a step before, and moves on.
    int ahead_hk = ahead.unit / a.n_groups;
    auto look_up = [&](int t, int row) {
        const int key = ahead.live.first + (t * kWarps + warp) * kStep + row;
        return t < ahead.live.tiles && key < ahead.live.y
                   ? a.table.ids[ahead.b * a.table.stride + (a.page_shift >= 0 ? key >> a.page_shift : key / a.pool.page_size)]
                   : -1;
    };
    const int own_row = a.whole_steps ? 0 : lane & 15;
    const int lane_row = lane / kChunks, lane_chunk = lane % kChunks;
    auto swizzled = [](int r, int chunk) { return r * S::kRowBytes + ((chunk ^ (kChunks >= 8 ? r & 7 : (r >> 1) & 3)) * 16); };
    const int64_t kv = static_cast<const unsigned char *>(a.pool.v) - static_cast<const unsigned char *>(a.pool.k);
    auto issue = [&](int stage, int page) {
        if (unfetched <= 0) return;
        const uint32_t base = ring_u + stage * S::kStage;
        const int pos = ahead.live.first + (ahead.t * kWarps + warp) * kStep;
        const unsigned char *kb = static_cast<const unsigned char *>(a.pool.k) + ahead_hk * a.pool.sh * kElem + half * S::kRowBytes;
        unsigned mask = 0xffffu;
        if (a.dense_steps && pos >= ahead.live.x && pos + kStep <= ahead.live.y && (unsigned)page < (unsigned)a.pool.n_pages) {
            // 16 whole rows side by side
            const int slot = a.page_shift >= 0 ? pos & ((1 << a.page_shift) - 1) : pos % a.pool.page_size;
            const unsigned char *at = kb + page * a.pool.sp * kElem + (int64_t)(slot + lane_row) * (D * kElem) + lane_chunk * 16;
#pragma unroll
            for (int i = 0; i < kCopies; i++) {
                const uint32_t dst = base + swizzled(i * kRowsPerCopy + lane_row, lane_chunk);
                cp_async16_or_zero(dst, at + i * kRowsPerCopy * D * kElem, true);
                cp_async16_or_zero(dst + kStep * S::kRowBytes, at + kv + i * kRowsPerCopy * D * kElem, true);
            }
            if constexpr (I8) {                           // lanes 0-15 the keys' scales, 16-31 the values'
                const int64_t r = ((int64_t)page * a.pool.n_kv_heads + ahead_hk) * a.pool.page_size + slot + (lane & 15);
                cp_async4_or_zero(base + S::kRows + lane * 4, (lane < 16 ? a.pool.ks : a.pool.vs) + r, true);
            }
        } else {                                          // row by row: lane r looks after row r
            const int row = lane & 15, key = pos + row, from = a.whole_steps ? pos : key;
            const int slot = (a.page_shift >= 0 ? from & ((1 << a.page_shift) - 1) : from % a.pool.page_size) + key - from;
            bool ok = key >= ahead.live.x && key < ahead.live.y;
            if (ok && (unsigned)page >= (unsigned)a.pool.n_pages) {
                atomicOr(a.status, kBadPage);
                ok = false;
            }
            mask = __ballot_sync(0xffffffffu, ok) & 0xffffu;
            const int64_t off = ok ? page * a.pool.sp * kElem + slot * a.pool.ss * kElem : -1;
#pragma unroll 1
            for (int r = lane_row; r < kStep; r += kRowsPerCopy) {
                const int64_t at = __shfl_sync(0xffffffffu, off, r);
                const unsigned char *src = kb + (at < 0 ? 0 : at + lane_chunk * 16);
                const uint32_t dst = base + swizzled(r, lane_chunk);
                cp_async16_or_zero(dst, src, at >= 0);
                cp_async16_or_zero(dst + kStep * S::kRowBytes, src + kv, at >= 0);
            }
            if constexpr (I8) {
                const int64_t r = ok ? ((int64_t)page * a.pool.n_kv_heads + ahead_hk) * a.pool.page_size + slot : 0;
                cp_async4_or_zero(base + S::kRows + lane * 4, (lane < 16 ? a.pool.ks : a.pool.vs) + r, ok);
            }
        }
        if (lane == 0) *reinterpret_cast<unsigned *>(ring + stage * S::kStage + S::kStage - 16) = mask;
        unfetched--;
        if (++ahead.t == ahead.live.tiles) {
            pass_end(ahead, unfetched);
            ahead_hk = ahead.unit / a.n_groups;
        }
    };

    // ---- q: a warp takes every 4th (8th) head, a lane D / 32 components, from global memory to registers
    // (load_q), to 16 bits in shared memory (store_q), from there as the products' 8-column operand:
    // pair (2j, 2j + 1) and (2j + 8, 2j + 9) of each 16 components; an int8 row's words hold 4 components
    // in order, so there the pairs are (4j, 4j + 1) and (4j + 2, 4j + 3), in K and q alike
    constexpr int kQWords = D / 64, kQWarps = kWarps * S::kPair;
    uint32_t q_in[S::kHeads / kQWarps][kQWords];
    uint32_t qf[S::kQInRegs ? NT : 1][S::kQInRegs ? kMt : 1][2];
    auto load_q = [&](const Place &p) {
        const int first = p.unit % a.n_groups * S::kHeads;
        const __nv_bfloat16 *q = a.q + p.b * a.q_stride + (int64_t)(p.unit / a.n_groups * a.group + first) * D;
#pragma unroll
        for (int i = 0; i < S::kHeads / kQWarps; i++)
#pragma unroll
            for (int w = 0; w < kQWords; w++)
                q_in[i][w] = first + any_warp + kQWarps * i < a.group
                                 ? reinterpret_cast<const uint32_t *>(q + (any_warp + kQWarps * i) * D)[lane * kQWords + w]
                                 : 0u;
    };
    auto store_q = [&]() {
#pragma unroll
        for (int i = 0; i < S::kHeads / kQWarps; i++) {
            const int h = any_warp + kQWarps * i;
            if constexpr (I8) {
                float top = 0.0f;
#pragma unroll
                for (int w = 0; w < kQWords; w++)
                    top = fmaxf(top, fmaxf(fabsf(xdna::bf16lo(q_in[i][w])), fabsf(xdna::bf16hi(q_in[i][w]))));
#pragma unroll
                for (int x = 16; x; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
                // the largest to [2^13, 2^14), as far as the factor's own exponent reaches
                const int e = max(1, min(253, 267 - (__float_as_int(top) >> 23)));
                const float f = __int_as_float(e << 23);
                if (lane == 0) q_inv[h] = __int_as_float((254 - e) << 23);
#pragma unroll
                for (int w = 0; w < kQWords; w++) {
                    const __half2 v = __floats2half2_rn(xdna::bf16lo(q_in[i][w]) * f, xdna::bf16hi(q_in[i][w]) * f);
                    q_in[i][w] = *reinterpret_cast<const uint32_t *>(&v);
                }
            }
#pragma unroll
            for (int w = 0; w < kQWords; w++)
                reinterpret_cast<uint32_t *>(q_s + h * S::kQRow)[lane * kQWords + w] = q_in[i][w];
        }
    };
    auto q_word = [&](int nt, int c, int i) -> uint32_t {
        return *reinterpret_cast<const uint32_t *>(q_s + (nt * 8 + g) * S::kQRow + half * S::kPart + 16 * c + (I8 ? 4 * j + 2 * i : 2 * j + 8 * i));
    };
    float q_back[NT][2];                                  // an int8 pool's factors of heads 2j, 2j + 1
    auto take_q = [&]() {
        if constexpr (S::kQInRegs) {
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int c = 0; c < kMt; c++) {
                    qf[nt][c][0] = q_word(nt, c, 0);
                    qf[nt][c][1] = q_word(nt, c, 1);
                }
        }
        if constexpr (I8) {
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int i = 0; i < 2; i++) q_back[nt][i] = q_inv[nt * 8 + 2 * j + i] * a.scale;
        }
    };
    load_q(at);
    const int same_unit = a.whole_steps ? min(32, ahead.live.tiles - ahead.t) : 0;
    const int first_pages = look_up(ahead.t + lane, 0);   // lane i: the first unit's step i
#pragma unroll 1
    for (int i = 0; i < S::kStages - 1; i++) {
        const int page = __shfl_sync(0xffffffffu, first_pages, i);
        issue(i, i < same_unit ? page : look_up(ahead.t, own_row));
        xdna::cp_async_commit();
    }
    int page = look_up(ahead.t, own_row);
    store_q();
    __syncthreads();
    take_q();

    int stage = 0;
    [[maybe_unused]] int turn = 0;
    for (;;) {
        const int run = min(at.live.tiles - at.t, left);  // tiles of this unit
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
        for (int t = 0; t < run; t++) {
            xdna::cp_async_wait_group<S::kStages - 2>();
            __syncwarp();
            issue(stage == 0 ? S::kStages - 1 : stage - 1, page);
            xdna::cp_async_commit();
            page = look_up(ahead.t, own_row);

            const uint32_t ks = ring_u + stage * S::kStage, vs = ks + kStep * S::kRowBytes;
            const unsigned char *tail = ring + stage * S::kStage + S::kRows;
            const unsigned mask = *reinterpret_cast<const unsigned *>(tail + (I8 ? 128 : 0));
            if (S::kPair == 2 || mask) {                  // a pair's warps meet in every step
                // ---- S^T: keys g, g + 8 by heads 2j, 2j + 1
                float s[NT][2][4];
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int i = 0; i < 4; i++) s[nt][0][i] = s[nt][1][i] = 0.0f;
                const int r = lane & 15, sw = kChunks >= 8 ? r & 7 : (r >> 1) & 3;
                auto q_of = [&](int nt, int c, int i) -> uint32_t {
                    if constexpr (S::kQInRegs) return qf[nt][c][i];
                    else return q_word(nt, c, i);
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
                        for (int x = 0; x < 4; x++) k[x] ^= 0x80808080u;
#pragma unroll
                        for (int x = 0; x < 2; x++) {
                            const uint32_t a0 = f16x2_of_u8(k[2 * x], 0x4140), a2 = f16x2_of_u8(k[2 * x], 0x4342);
                            const uint32_t a1 = f16x2_of_u8(k[2 * x + 1], 0x4140), a3 = f16x2_of_u8(k[2 * x + 1], 0x4342);
#pragma unroll
                            for (int nt = 0; nt < NT; nt++)
                                mma_f16(s[nt][x], a0, a1, a2, a3, q_of(nt, c + x, 0), q_of(nt, c + x, 1));
                        }
                    }
                }
                if constexpr (S::kPair == 2) {            // the other half's part of the scores
                    float4 *mine = reinterpret_cast<float4 *>(swap) + ((turn * kWarps + warp) * 2 + half) * 32 * NT + lane;
                    const float4 *other = reinterpret_cast<const float4 *>(swap) + ((turn * kWarps + warp) * 2 + 1 - half) * 32 * NT + lane;
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
                        mine[nt * 32] = make_float4(s[nt][0][0] + s[nt][1][0], s[nt][0][1] + s[nt][1][1],
                                                    s[nt][0][2] + s[nt][1][2], s[nt][0][3] + s[nt][1][3]);
                    xdna::named_bar(1 + warp, 64);
                    turn ^= 1;
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {     // in one order for both, so that both get the same
                        const float4 x = half ? other[nt * 32] : mine[nt * 32], y = half ? mine[nt * 32] : other[nt * 32];
                        s[nt][0][0] = x.x; s[nt][0][1] = x.y; s[nt][0][2] = x.z; s[nt][0][3] = x.w;
                        s[nt][1][0] = y.x; s[nt][1][1] = y.y; s[nt][1][2] = y.z; s[nt][1][3] = y.w;
                    }
                }
                // ---- running maximum and weights
                const bool ok0 = (mask >> g) & 1, ok1 = (mask >> (g + 8)) & 1;
                float f0 = a.scale, f1 = a.scale, v0 = 0.0f, v1 = 0.0f;
                if constexpr (I8) {
                    const float *sc = reinterpret_cast<const float *>(tail);
                    f0 = sc[g]; f1 = sc[g + 8];
                    v0 = sc[16 + g]; v1 = sc[24 + g];
                }
                bool up = false;
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        float x = (s[nt][0][i] + s[nt][1][i]) * (i < 2 ? f0 : f1);
                        if constexpr (I8) x *= q_back[nt][i & 1];
                        x = (i < 2 ? ok0 : ok1) ? x : -INFINITY;
                        s[nt][0][i] = x;
                        up |= x > m[nt][i & 1];
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
                uint32_t pt[NT][2][kTerms];
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    float p[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        p[i] = exp2_approx(s[nt][0][i] - ms[nt][i & 1]);
                        l[nt][i & 1] += p[i];
                        if constexpr (I8) p[i] *= i < 2 ? v0 : v1;
                    }
                    split_pair(p[0], p[1], pt[nt][0]);
                    split_pair(p[2], p[3], pt[nt][1]);
#pragma unroll
                    for (int x = 0; x < kTerms; x++) {
                        pt[nt][0][x] = transpose8x8(pt[nt][0][x]);
                        pt[nt][1][x] = transpose8x8(pt[nt][1][x]);
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
#pragma unroll
                            for (int x = 0; x < kTerms; x++)
                                mma_bf16(o[nt][c], v[0], v[1], v[2], v[3], pt[nt][0][x], pt[nt][1][x]);
                        }
                    }
                } else {
#pragma unroll
                    for (int c = 0; c < kMt; c += 2) {
                        uint32_t v[4];
                        ldsm4_trans(v, vs + r * S::kRowBytes + (((c + (lane >> 4)) ^ sw) * 16));
#pragma unroll
                        for (int x = 0; x < 2; x++) {
                            const uint32_t a0 = bf16x2_of_s8(v[2 * x]), a1 = bf16x2_of_s8(v[2 * x] >> 8);
                            const uint32_t a2 = bf16x2_of_s8(v[2 * x + 1]), a3 = bf16x2_of_s8(v[2 * x + 1] >> 8);
#pragma unroll
                            for (int nt = 0; nt < NT; nt++) {
#pragma unroll
                                for (int y = 0; y < kTerms; y++)
                                    mma_bf16(o[nt][c + x], a0, a1, a2, a3, pt[nt][0][y], pt[nt][1][y]);
                            }
                        }
                    }
                }
            }
            __syncwarp();
            stage = stage + 1 == S::kStages ? 0 : stage + 1;
        }

        // ---- the unit's end: the warps' parts into one, the next unit's q on its way meanwhile
        const Place done = at;
        const Int begin = unit_at;
        left -= run;
        if (left > 0) {                                   // else the unit may go on in the next share
            unit_at += at.live.tiles + end_cost;
            pass_end(at, left);
        }
        if (left > 0) load_q(at);
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
#pragma unroll
                for (int x = 4; x < 32; x *= 2) l[nt][i] += __shfl_xor_sync(0xffffffffu, l[nt][i], x);
                if (g == 0 && half == 0) {
                    join_m[warp][nt * 8 + 2 * j + i] = m[nt][i];
                    join_l[warp][nt * 8 + 2 * j + i] = l[nt][i];
                }
            }
        if (left <= 0) xdna::cp_async_wait_all();
        __syncthreads();
        if (left > 0) store_q();
        const int hk = done.unit / a.n_groups, h0 = hk * a.group + (done.unit % a.n_groups) * S::kHeads;
        const int heads = min(S::kHeads, a.group - (done.unit % a.n_groups) * S::kHeads);
        const bool whole = done.t == 0 && run == done.live.tiles;
        const int slot = 2 * blockIdx.x + (done.t == 0);
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
        auto of_warps = [&](int h, float &top, float &den) {
            top = join_m[0][h];
            den = 0.0f;
#pragma unroll
            for (int w = 1; w < kWarps; w++) top = fmaxf(top, join_m[w][h]);
#pragma unroll
            for (int w = 0; w < kWarps; w++)
                den += join_l[w][h] * (join_m[w][h] == top ? 1.0f : exp2_approx(join_m[w][h] - top));
        };
        auto join_warps = [&](auto columns) {             // that many components of each part at a time
            constexpr int kCols = decltype(columns)::value, kRow = kCols + 4, kLine = S::kPair * kCols / 4;
#pragma unroll
            for (int d0 = 0; d0 < S::kPart; d0 += kCols) {
                if (d0) __syncthreads();
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int c = 0; c < kCols / 16; c++)
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const int comp = 16 * c + (I8 ? 2 * g + (i >> 1) : g + 8 * (i >> 1));
                            join_o[(any_warp * S::kHeads + nt * 8 + 2 * j + (i & 1)) * kRow + comp] =
                                o[nt][d0 / 16 + c][i] * fac[nt][i & 1];
                        }
                __syncthreads();
                for (int x = tid; x < heads * kLine; x += kThreads) {
                    const int h = x / kLine, part = x % kLine / (kCols / 4), c = x % (kCols / 4) * 4;
                    const int to = part * S::kPart + d0 + c;
                    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                    for (int w = 0; w < kWarps; w++) {
                        const float4 y = *reinterpret_cast<const float4 *>(&join_o[((w * S::kPair + part) * S::kHeads + h) * kRow + c]);
                        sum.x += y.x; sum.y += y.y; sum.z += y.z; sum.w += y.w;
                    }
                    if (whole) {
                        float top, den;
                        of_warps(h, top, den);
                        const float inv = den == 0.0f ? 0.0f : 1.0f / den;
                        const __nv_bfloat162 lo = __floats2bfloat162_rn(sum.x * inv, sum.y * inv),
                                             hi = __floats2bfloat162_rn(sum.z * inv, sum.w * inv);
                        *reinterpret_cast<uint2 *>(a.out + ((int64_t)done.b * a.n_q_heads + h0 + h) * D + to) =
                            make_uint2(*reinterpret_cast<const uint32_t *>(&lo), *reinterpret_cast<const uint32_t *>(&hi));
                    } else {
                        *reinterpret_cast<float4 *>(a.part_o + ((int64_t)slot * S::kHeads + h) * D + to) = sum;
                    }
                }
            }
        };
        if (left > 0) {
            join_warps(std::integral_constant<int, S::kJoinCols>{});
        } else {                                          // the ring is free: all at once
            join_o = reinterpret_cast<float *>(smem);
            join_warps(std::integral_constant<int, S::kPart>{});
        }
        if (tid < heads) {
            float top, den;
            of_warps(tid, top, den);
            if (!whole) a.part_ml[slot * S::kHeads + tid] = make_float2(top, den);
            else if (a.lse) a.lse[(int64_t)done.b * a.n_q_heads + h0 + tid] = (top + log2f(den)) * 0.69314718f;
        }
        if (!whole) {
            // ---- parts: a unit's tiles [begin, begin + tiles) lie in the shares of CTAs first .. first + parts - 1
            __threadfence();
            __syncthreads();
            const int first = (int)(((begin + 1) * ctas - 1) / total);
            const int parts = (int)(((begin + done.live.tiles) * ctas - 1) / total) - first + 1;
            for (int level = 0, n = parts, i = blockIdx.x - first, stride = 1; level < kJoinLevels; level++) {
                const int group = i / kJoinWays, size = min(kJoinWays, n - group * kJoinWays);
                auto slot_of = [&](int k) {                   // a CTA's first unit is in its slot 0, unless it begins there
                    const int part = (group * kJoinWays + k) * stride;
                    return 2 * (first + part) + (part == 0);
                };
                if (size > 1) {
                    if (tid == 0) {
                        int *count = a.arrived + level * 2 * gridDim.x + slot_of(0);
                        last = atomicAdd(count, 1) == size - 1;
                        if (last) *count = 0;
                    }
                    __syncthreads();
                    if (!last) break;
                    __threadfence();
                    const bool final = n <= kJoinWays;
                    // kThreads / heads threads a head: the weights once, then their columns
                    const int per_head = kThreads / heads, h = tid / per_head;
                    if (h < heads) {
                        const int64_t hop = (int64_t)2 * stride * S::kHeads;    // from part to part, in rows
                        const int64_t row0 = (int64_t)slot_of(0) * S::kHeads + h, row1 = (int64_t)slot_of(1) * S::kHeads + h - hop;
                        float2 ml[kJoinWays];
                        constexpr int kUnder = S::kCtas < 3 && NT == 1 ? 16 : 8;   // loads under way, as registers allow
                        float4 y[kUnder];
                        auto load = [&](int k0, int c) {
#pragma unroll
                            for (int k = 0; k < kUnder; k++)
                                y[k] = k0 + k < size ? __ldcg(reinterpret_cast<const float4 *>(
                                                           a.part_o + (k0 + k ? row1 + (k0 + k) * hop : row0) * D + c))
                                                     : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        };
#pragma unroll
                        for (int k = 0; k < kJoinWays; k++)
                            ml[k] = k < size ? __ldcg(a.part_ml + (k ? row1 + k * hop : row0)) : make_float2(-INFINITY, 0.0f);
                        int c = tid % per_head * 4;
                        if (c < D) load(0, c);
                        float top = ml[0].x, den = 0.0f;
#pragma unroll
                        for (int k = 1; k < kJoinWays; k++) top = fmaxf(top, ml[k].x);
#pragma unroll
                        for (int k = 0; k < kJoinWays; k++) {
                            ml[k].x = ml[k].x == top ? 1.0f : exp2_approx(ml[k].x - top);
                            if (k < size) den = fmaf(ml[k].y, ml[k].x, den);
                        }
                        const float inv = den == 0.0f ? 0.0f : 1.0f / den;
#pragma unroll 1
                        for (; c < D; c += per_head * 4) {
                            float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                            for (int k = 0; k < kJoinWays; k++) {
                                if (k == kUnder) {
                                    if (size <= kUnder) break;
                                    load(kUnder, c);
                                }
                                if (k < size) {
                                    sum.x = fmaf(y[k % kUnder].x, ml[k].x, sum.x); sum.y = fmaf(y[k % kUnder].y, ml[k].x, sum.y);
                                    sum.z = fmaf(y[k % kUnder].z, ml[k].x, sum.z); sum.w = fmaf(y[k % kUnder].w, ml[k].x, sum.w);
                                }
                            }
                            if (final) {
                                const __nv_bfloat162 lo = __floats2bfloat162_rn(sum.x * inv, sum.y * inv),
                                                     hi = __floats2bfloat162_rn(sum.z * inv, sum.w * inv);
                                *reinterpret_cast<uint2 *>(a.out + ((int64_t)done.b * a.n_q_heads + h0 + h) * D + c) = make_uint2(
                                    *reinterpret_cast<const uint32_t *>(&lo), *reinterpret_cast<const uint32_t *>(&hi));
                            } else {                          // in place of the group's first part: this thread alone reads it
                                *reinterpret_cast<float4 *>(a.part_o + row0 * D + c) = sum;
                            }
                            if (c + per_head * 4 < D) load(0, c + per_head * 4);
                        }
                        if (tid % per_head == 0) {
                            if (!final) join_m[0][h] = top, join_l[0][h] = den;
                            else if (a.lse) a.lse[(int64_t)done.b * a.n_q_heads + h0 + h] = (top + log2f(den)) * 0.69314718f;
                        }
                    }
                    if (final) break;
                    __syncthreads();
                    // the new maximum and sum after all threads have read the old
                    if (tid < heads) a.part_ml[slot_of(0) * S::kHeads + tid] = make_float2(join_m[0][tid], join_l[0][tid]);
                    __threadfence();
                    __syncthreads();
                }
                i = group;
                n = (n + kJoinWays - 1) / kJoinWays;
                stride *= kJoinWays;
            }
        }
        if (left <= 0) break;
        __syncthreads();
        take_q();
    }

    empty_streams();
}

template <int D, bool I8, int NT>
bool allow_smem() {
    return ck(cudaFuncSetAttribute(attention_kernel<D, I8, NT, true>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                   AttnShape<D, I8, NT>::kSmem),
              "xdna_paged_cache_create") &&
           ck(cudaFuncSetAttribute(attention_kernel<D, I8, NT, false>, cudaFuncAttributeMaxDynamicSharedMemorySize,
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
    const int64_t tiles = units * ((keys + kStep - 1 + kTileKeys - 1) / kTileKeys + S::kEndCost);
    const int grid = (int)std::min<int64_t>((int64_t)sms * S::kCtas, tiles);
    if ((tiles + 8) * (grid + 8) < 0x7fffffff) attention_kernel<D, I8, NT, true><<<grid, S::kThreads, S::kSmem, st>>>(a);
    else attention_kernel<D, I8, NT, false><<<grid, S::kThreads, S::kSmem, st>>>(a);
    return cudaGetLastError();
}
template <int D>
cudaError_t launch_attention(const AttnArgs &a, bool i8, int sms, cudaStream_t st) {
    // up to 16 heads to a unit: 32 x 8k, 64/4 heads x 128 takes 103 us, as two units of 8 that read K and V twice 176
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

// log2 of a page size that is a power of two, else -1
int shift_of(int page_size) { return page_size & (page_size - 1) ? -1 : __builtin_ctz(page_size); }

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
    if (off_elements(4, g.k_scale, g.v_scale)) return refuse("scales not aligned to their elements");
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
        !ck(cudaMalloc(&c->arrived, (size_t)c->sms * kMaxCtasPerSm * 2 * kJoinLevels * sizeof(int)),
            "xdna_paged_cache_create") ||
        !ck(cudaMemset(c->arrived, 0, (size_t)c->sms * kMaxCtasPerSm * 2 * kJoinLevels * sizeof(int)),
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
        cudaFree(c->arrived);
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
    if (off_elements(4, tok_seq, tok_pos, block_table)) return fail(me + "a pointer not aligned to its elements");
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
    a.page_shift = shift_of(g.page_size);
    const int64_t rows = (int64_t)n_tokens * (a.n_q_heads + 2 * g.n_kv_heads), at_once = 4096 / g.head_dim;
    if (rows > 0x7fff0000) return fail(me + "more than 2^31 rows in one call");
    const int64_t blocks = (rows + at_once - 1) / at_once;
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
    // 128 streams' tiles are summed in 32 bits, and so is a CTA's share
    if ((int64_t)table_width * g.page_size > 0x20000000) return fail(me + "more than 2^29 positions in a table row");
    if ((double)n_seqs * n_q_heads * table_width * g.page_size > 1e13) return fail(me + "more than 10^13 positions of all heads");
    if (window < 0 || !(scale > 0.0f)) return fail(me + "negative window or scale not above 0");
    if (q_stride < (int64_t)n_q_heads * g.head_dim || q_stride % 8 || !aligned16(q) || !aligned16(out))
        return fail(me + "q_stride below the heads' width, or rows not 16-byte aligned");
    if (off_elements(4, block_table, seq_lens, lse)) return fail(me + "a pointer not aligned to its elements");
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
    a.page_shift = shift_of(g.page_size);
    a.whole_steps = g.page_size % kStep == 0;
    a.dense_steps = a.whole_steps && g.stride_slot == g.head_dim;
    a.part_o = c->part_o;
    a.part_ml = c->part_ml;
    a.arrived = c->arrived;
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
