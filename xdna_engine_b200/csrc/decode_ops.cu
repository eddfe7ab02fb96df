// decode_ops.cu -- the serving ops on both sides of a decoder layer's products
// (include/xdna_b200.h): the residual RMS norm with int8 rows, and the logits processor.
#include <cuda_runtime.h>
#include <cuda_bf16.h>

#include <algorithm>
#include <atomic>
#include <cstdint>
#include <string>

#include "../../include/xdna_b200.h"
#include "ptx.cuh"

namespace xdna {
void set_last_error_message(const std::string &m);
}
using xdna::set_last_error_message;

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

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }

// ----------------------------------------------------------------- residual RMS norm, int8
struct NormArgs {
    const void *x, *res;
    int64_t x_stride, res_stride;
    const float *gamma;
    int unit_offset, M, D;
    float eps;
    void *res_out;
    __nv_bfloat16 *y;
    int8_t *q8;
    float *scale;
};

// N elements of a row as they lie in memory (8: one or two 16-byte loads), and as f32
template <typename T, int N>
struct Piece;
template <>
struct Piece<float, 8> {
    float4 a, b;
    __device__ void load(const float *p) {
        a = __ldcs(reinterpret_cast<const float4 *>(p));
        b = __ldcs(reinterpret_cast<const float4 *>(p) + 1);
    }
    __device__ float operator[](int k) const { return k == 0 ? a.x : k == 1 ? a.y : k == 2 ? a.z : k == 3 ? a.w : k == 4 ? b.x : k == 5 ? b.y : k == 6 ? b.z : b.w; }
};
template <>
struct Piece<__nv_bfloat16, 8> {
    uint4 a;
    __device__ void load(const __nv_bfloat16 *p) { a = __ldcs(reinterpret_cast<const uint4 *>(p)); }
    __device__ float operator[](int k) const {
        const uint32_t u = k < 2 ? a.x : k < 4 ? a.y : k < 6 ? a.z : a.w;
        return k % 2 ? xdna::bf16hi(u) : xdna::bf16lo(u);
    }
};
template <>
struct Piece<float, 1> {
    float a;
    __device__ void load(const float *p) { a = __ldcs(p); }
    __device__ float operator[](int) const { return a; }
};
template <>
struct Piece<__nv_bfloat16, 1> {
    __nv_bfloat16 a;
    __device__ void load(const __nv_bfloat16 *p) { a = *p; }
    __device__ float operator[](int) const { return __bfloat162float(a); }
};
template <int N>
__device__ __forceinline__ void store_n(float *p, const float (&v)[N]) {
    if constexpr (N == 8) {
        reinterpret_cast<float4 *>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4 *>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        *p = v[0];
    }
}
template <int N>
__device__ __forceinline__ void store_n(__nv_bfloat16 *p, const float (&v)[N]) {
    if constexpr (N == 8) {
        uint32_t u[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const __nv_bfloat162 two = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
            u[i] = *reinterpret_cast<const uint32_t *>(&two);
        }
        *reinterpret_cast<uint4 *>(p) = make_uint4(u[0], u[1], u[2], u[3]);
    } else {
        *p = __float2bfloat16_rn(v[0]);
    }
}

// A CTA takes every gridDim.x-th row, one pass over it: a thread keeps P pieces of N elements in
// registers, so that x and the residual are read once (7 bytes an element with bf16 in and out: HBM
// bounds it).  The sum of squares and max|r g| need one joint reduction, since the row's factor 1 / rms
// scales both y and its maximum and drops out of the whole numbers.  kAhead: gamma stays in registers and
// the next row's loads pass under the reduction and the outputs; without it (wide rows, whose
// threads have no registers left) other CTAs of the SM do that.  N = 8 where every row is 16-byte
// aligned, else N = 1.  Measured: 8192 x 4096 bf16 47.3 us, 5.0 TB/s (kAhead off: 50.6); 64 x 1152
// 2.3 us; 4592 rows of 865, f32 and bf16 (N = 1) 16.5 us, 2.2 TB/s, bound by its 2- and 4-byte accesses.
template <typename X, typename R, int N, int P, int kThreads, bool kAhead>
__global__ void __launch_bounds__(kThreads) rmsnorm_kernel(const NormArgs a) {
    __shared__ float2 red[2][kThreads / 32];              // alternating, so that a row needs one barrier
    const int threads = blockDim.x, warps = threads / 32, lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    auto place = [&](int p) { return (p * threads + (int)threadIdx.x) * N; };
    Piece<X, N> x[kAhead ? P : 1];
    Piece<R, N> res[kAhead ? P : 1];
    auto load = [&](int64_t row, int p, int to) {
        if (place(p) >= a.D) return;
        x[to].load(static_cast<const X *>(a.x) + row * a.x_stride + place(p));
        if (a.res) res[to].load(static_cast<const R *>(a.res) + row * a.res_stride + place(p));
    };
    float g[kAhead ? P : 1][N];
    auto load_gamma = [&](int p, float (&w)[N]) {
        if constexpr (N == 8) {
            const float4 lo = __ldg(reinterpret_cast<const float4 *>(a.gamma + place(p))),
                         hi = __ldg(reinterpret_cast<const float4 *>(a.gamma + place(p)) + 1);
            w[0] = lo.x; w[1] = lo.y; w[2] = lo.z; w[3] = lo.w;
            w[4] = hi.x; w[5] = hi.y; w[6] = hi.z; w[7] = hi.w;
        } else {
            w[0] = __ldg(a.gamma + place(p));
        }
        if (a.unit_offset)
#pragma unroll
            for (int k = 0; k < N; k++) w[k] = __fadd_rn(w[k], 1.0f);
    };
    if constexpr (kAhead) {
#pragma unroll
        for (int p = 0; p < P; p++) load(blockIdx.x, p, p);
#pragma unroll
        for (int p = 0; p < P; p++)
            if (place(p) < a.D) load_gamma(p, g[p]);
    }
    int phase = 0;
    for (int64_t row = blockIdx.x; row < a.M; row += gridDim.x, phase ^= 1) {
        float r[P][N], sum = 0.0f;
        unsigned bits = 0;                                // magnitudes ordered as bits: a NaN is the largest and makes the scale NaN
#pragma unroll
        for (int p = 0; p < P; p++) {
            if (place(p) >= a.D) break;
            if (!kAhead) load(row, p, 0);
            const int at = kAhead ? p : 0;
#pragma unroll
            for (int k = 0; k < N; k++) r[p][k] = a.res ? __fadd_rn(x[at][k], res[at][k]) : x[at][k];
        }
        if (kAhead && row + gridDim.x < a.M) {
#pragma unroll
            for (int p = 0; p < P; p++) load(row + gridDim.x, p, kAhead ? p : 0);
        }
#pragma unroll
        for (int p = 0; p < P; p++) {
            if (place(p) >= a.D) break;
            if (a.res_out) store_n(static_cast<R *>(a.res_out) + row * a.res_stride + place(p), r[p]);
            float w[N];
            if constexpr (!kAhead) load_gamma(p, w);
#pragma unroll
            for (int k = 0; k < N; k++) {
                sum = fmaf(r[p][k], r[p][k], sum);
                r[p][k] = __fmul_rn(r[p][k], kAhead ? g[p][k] : w[k]);
                bits = max(bits, __float_as_uint(fabsf(r[p][k])));
            }
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        bits = __reduce_max_sync(0xffffffffu, bits);
        if (lane == 0) red[phase][warp] = make_float2(sum, __uint_as_float(bits));
        __syncthreads();
        if constexpr (kThreads <= 256) {
            sum = red[phase][0].x;
            for (int w = 1; w < warps; w++) {
                sum += red[phase][w].x;
                bits = max(bits, __float_as_uint(red[phase][w].y));
            }
            bits = max(bits, __float_as_uint(red[phase][0].y));
        } else {
            const float2 part = lane < warps ? red[phase][lane] : make_float2(0.0f, 0.0f);
            sum = part.x;
#pragma unroll
            for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            bits = __reduce_max_sync(0xffffffffu, __float_as_uint(part.y));
        }
        const float top = __uint_as_float(bits);
        const float inv = rsqrtf(__fdiv_rn(sum, (float)a.D) + a.eps);
        // below 127 / FLT_MAX the factor would be infinite: such a row counts as zero
        const bool zero = top <= 3.8e-37f;
        const float to8 = zero ? 0.0f : __fmul_rn(__frcp_rn(top), 127.0f);
#pragma unroll
        for (int p = 0; p < P; p++) {
            if (place(p) >= a.D) break;
            if (a.q8) {
                // x + 1.5 2^23 rounds x to a whole number, half to even, whose low byte is the int8
                uint32_t w[N];
#pragma unroll
                for (int k = 0; k < N; k++) w[k] = __float_as_uint(__fadd_rn(__fmul_rn(r[p][k], to8), 12582912.0f));
                int8_t *q = a.q8 + row * a.D + place(p);
                if constexpr (N == 8)
                    *reinterpret_cast<uint2 *>(q) =
                        make_uint2(__byte_perm(__byte_perm(w[0], w[1], 0x0040), __byte_perm(w[2], w[3], 0x0040), 0x5410),
                                   __byte_perm(__byte_perm(w[4], w[5], 0x0040), __byte_perm(w[6], w[7], 0x0040), 0x5410));
                else
                    *q = (int8_t)w[0];
            }
            if (a.y) {
                float y[N];
#pragma unroll
                for (int k = 0; k < N; k++) y[k] = r[p][k] * inv;
                store_n(a.y + row * a.D + place(p), y);
            }
        }
        if (a.scale && threadIdx.x == 0) a.scale[row] = zero ? 1.0f : __fmul_rn(__fdiv_rn(top, 127.0f), inv);
    }
}

template <typename X, typename R, int N, int P, int kThreads, bool kAhead>
cudaError_t launch_norm(const NormArgs &a, int sms, cudaStream_t st) {
    const int pieces = (a.D + N - 1) / N, threads = std::max(32, ((pieces + P - 1) / P + 31) / 32 * 32);
    // as many CTAs as fit (64 to 80 registers a thread), and a row more to each
    const int64_t grid = kAhead ? std::min<int64_t>(a.M, (int64_t)sms * std::max(1, std::min(16, 768 / threads))) : a.M;
    rmsnorm_kernel<X, R, N, P, kThreads, kAhead><<<(unsigned)grid, threads, 0, st>>>(a);
    return cudaGetLastError();
}
template <typename X, typename R>
cudaError_t launch_norm(const NormArgs &a, bool wide, int sms, cudaStream_t st) {
    if (wide) {
        // one piece to a thread up to 256 of them, then two (4096: 46.6 us; one to 512 threads 53.8, four 67.5)
        if (a.D <= 2048) return launch_norm<X, R, 8, 1, 256, true>(a, sms, st);
        if (a.D <= 4096) return launch_norm<X, R, 8, 2, 256, true>(a, sms, st);
        return launch_norm<X, R, 8, 2, 1024, false>(a, sms, st);
    }
    // 31 x 2434: 3.6 us with 4 elements to each of 1024 threads, 9.6 us with 16, which spill
    if (a.D <= 1024) return launch_norm<X, R, 1, 4, 256, true>(a, sms, st);
    if (a.D <= 4096) return launch_norm<X, R, 1, 4, 1024, false>(a, sms, st);
    return launch_norm<X, R, 1, 16, 1024, false>(a, sms, st);
}

// ---------------------------------------------------------------------------------- logits
struct LogitsArgs {
    const void *logits;
    int64_t stride, out_stride, mask_stride;
    int V, n_hist, n_bias;
    const int32_t *hist, *hist_start, *n_prompt;
    const float *rep, *freq, *pres;
    const int32_t *bias_ids, *bias_start;
    const float *bias;
    const uint32_t *mask;
    float *out;
    int64_t *ids;
    unsigned long long *best;                             // [B][chunks] where the chunks do not meet in a cluster
};

// a float's bits as an unsigned that orders alike (-0 as 0); -inf and NaN: 0, below every other
__device__ __forceinline__ unsigned ordered(float x) {
    const unsigned u = __float_as_uint(x == 0.0f ? 0.0f : x);
    return x > -INFINITY ? (u & 0x80000000u ? ~u : u | 0x80000000u) : 0u;
}
// a value and its id as one number: larger for the larger value, of equals for the lower id; 0: none
__device__ __forceinline__ unsigned long long choice(unsigned key, int id) {
    return key ? ((unsigned long long)key << 32) | (0xffffffffu - (unsigned)id) : 0ull;
}

// One CTA per row and chunk of 512 P W ids; 4 + 4 bytes an id in f32, so HBM bounds it as long as an id
// costs few instructions.
// * A thread takes P pieces of W ids.  W = 4: one 16-byte access, with chunks laid from the row's
//   preceding 16-byte boundary where rows start off one; W = 1 where logits and out lie differently.
// * Logits, mask bits and list entries are loaded into registers before they are needed, so that
//   their latencies pass together; every chunk of a row scans the row's lists.
// * The chunk's counts and bias entries lie in shared memory (integer atomics, so in any order), with a
//   bit per touched id.  The touched ids' penalties and biases are worked out first, from the
//   bits, and their results put where the counts were; then every id is taken from its register or
//   from there, masked, stored and compared.
// * The best ids of a row's chunks meet in a cluster (kCluster: the row's CTAs are one), whose first
//   CTA writes the row's, or in the workspace, from which choose_kernel takes it.
// Measured: 64 x 262144 f32 with a history of 4000, 300 biases and a mask 48.7 us (2.8 TB/s); without any of
// these 20.7 us (6.5 TB/s).  The lists cost three barriers in the 5.5 us that a CTA lives.
constexpr int kLogitsThreads = 512, kLogitsWarps = kLogitsThreads / 32, kMaxCluster = 8;

template <int W>
__device__ __forceinline__ void load_ids(const float *x, float *y) {
    if (W == 4) {
        const float4 v = __ldcs(reinterpret_cast<const float4 *>(x));
        y[0] = v.x; y[1] = v.y; y[2] = v.z; y[3] = v.w;
    } else {
        y[0] = *x;
    }
}
template <int W>
__device__ __forceinline__ void load_ids(const __nv_bfloat16 *x, float *y) {
    if (W == 4) {
        const uint2 v = __ldcs(reinterpret_cast<const uint2 *>(x));
        y[0] = xdna::bf16lo(v.x); y[1] = xdna::bf16hi(v.x); y[2] = xdna::bf16lo(v.y); y[3] = xdna::bf16hi(v.y);
    } else {
        y[0] = __bfloat162float(*x);
    }
}

template <typename T, int P, int W, bool kCluster>
__global__ void __launch_bounds__(kLogitsThreads, 2) logits_kernel(const LogitsArgs a) {
    constexpr int kChunk = kLogitsThreads * P * W, kAhead = 8, kBits = P * W;   // kBits: touched bits a thread works out
    constexpr unsigned kPiece = (1u << W) - 1;
    extern __shared__ __align__(16) unsigned smem[];
    // bit i: place i is in the history (any: in the history or the bias list)
    __shared__ unsigned seen[kChunk / 32], any[kChunk / 32];
    __shared__ unsigned key_of[kLogitsWarps], id_of[kLogitsWarps];
    __shared__ unsigned long long of_rank[kMaxCluster];
    unsigned *count = smem;                               // generated occurrences, then the touched ids' results
    int *entry = reinterpret_cast<int *>(smem + kChunk);  // 1 + the id's last bias entry
    const int64_t b = blockIdx.y;
    const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
    if constexpr (kCluster) asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");
    // the chunk's place i is id first + i, live for lo <= i < hi
    const int shift = W == 4 ? (int)((reinterpret_cast<uintptr_t>(a.out + b * a.out_stride) / 4) % 4) : 0;
    const int first = blockIdx.x * kChunk - shift, lo = max(0, -first), hi = min(kChunk, a.V - first);
    const bool full = lo == 0 && hi == kChunk;
    const T *x = static_cast<const T *>(a.logits) + b * a.stride + first;
    float *out = a.out + b * a.out_stride + first;
    auto place_of = [&](int p) { return (p * kLogitsThreads + tid) * W; };
    const bool lists = a.hist || a.bias;
    int h0 = 0, h1 = 0, gen = 0, e0 = 0, e1 = 0;
    float rep = 1.0f, freq = 0.0f, pres = 0.0f;
    if (lists) {                                          // the lists' ids wait for these: first of all
        h0 = a.hist ? a.hist_start[b] : 0;
        h1 = a.hist ? a.hist_start[b + 1] : 0;
        gen = a.n_prompt ? a.n_prompt[b] : 0;
        e0 = a.bias ? a.bias_start[b] : 0;
        e1 = a.bias ? a.bias_start[b + 1] : 0;
        rep = a.rep ? a.rep[b] : 1.0f;
        freq = a.freq ? a.freq[b] : 0.0f;
        pres = a.pres ? a.pres[b] : 0.0f;
    }
    float y[P][W];
    unsigned allowed = 0xffffffffu;                       // bit p W + w
    const uint32_t *mask = a.mask ? a.mask + b * a.mask_stride : nullptr;
    if (full) {
#pragma unroll
        for (int p = 0; p < P; p++) load_ids<W>(x + place_of(p), y[p]);
    } else {
#pragma unroll
        for (int p = 0; p < P; p++)
#pragma unroll
            for (int w = 0; w < W; w++) {
                const int i = place_of(p) + w;
                y[p][w] = i >= lo && i < hi ? to_f32(x[i]) : -INFINITY;
            }
    }
    const bool whole_words = mask && full && shift == 0;
    unsigned word[P];
    if (whole_words) {
#pragma unroll
        for (int p = 0; p < P; p++) word[p] = mask[(first + place_of(p)) / 32];
    } else if (mask) {
        allowed = 0;
#pragma unroll
        for (int p = 0; p < P; p++)
#pragma unroll
            for (int w = 0; w < W; w++) {
                const int i = place_of(p) + w;
                if (i >= lo && i < hi) allowed |= ((mask[(first + i) / 32] >> ((first + i) % 32)) & 1u) << (p * W + w);
            }
    }
    if (lists) {
        h0 = max(0, h0);
        h1 = min(a.n_hist, h1);
        gen = min(max(0, gen), 0x7fffffff - h0) + h0;
        e0 = max(0, e0);
        e1 = max(e0, min(a.n_bias, e1));                  // so that e1 - e0 does not wrap
        int biased = e1 - e0 > tid ? a.bias_ids[e0 + tid] : -1;
        int ids[kAhead];
        auto ahead = [&](int j0) {
#pragma unroll
            for (int k = 0; k < kAhead; k++) ids[k] = h1 - j0 > k * kLogitsThreads + tid ? a.hist[j0 + k * kLogitsThreads + tid] : -1;
        };
        if (h0 < h1) ahead(h0);
        uint4 *zero = reinterpret_cast<uint4 *>(smem) + tid;
#pragma unroll
        for (int i = 0; i < kChunk / 4 / kLogitsThreads; i++) zero[i * kLogitsThreads] = make_uint4(0, 0, 0, 0);
        if (a.bias) {
#pragma unroll
            for (int i = 0; i < kChunk / 4 / kLogitsThreads; i++) zero[kChunk / 4 + i * kLogitsThreads] = make_uint4(0, 0, 0, 0);
        }
        if (tid < kChunk / 32) seen[tid] = any[tid] = 0;
        __syncthreads();
        // an id of the chunk: id_lo <= id < id_lo + span, as unsigned, which leaves negative ids out
        const unsigned id_lo = (unsigned)(first + lo), span = (unsigned)max(0, hi - lo);
        for (int j0 = h0; j0 < h1;) {
#pragma unroll
            for (int k = 0; k < kAhead; k++) {
                if ((unsigned)ids[k] - id_lo < span) {
                    const int i = ids[k] - first;
                    atomicOr(&seen[i / 32], 1u << (i % 32));
                    if (j0 + k * kLogitsThreads + tid >= gen) atomicAdd(&count[i], 1u);
                }
            }
            if (h1 - j0 <= kAhead * kLogitsThreads) break;
            j0 += kAhead * kLogitsThreads;
            ahead(j0);
        }
        for (int j = tid; j < e1 - e0;) {
            if ((unsigned)biased - id_lo < span) {
                const int i = biased - first;
                atomicOr(&any[i / 32], 1u << (i % 32));
                atomicMax(&entry[i], j + 1);
            }
            if (e1 - e0 - j <= kLogitsThreads) break;
            j += kLogitsThreads;
            biased = a.bias_ids[e0 + j];
        }
        __syncthreads();
        // ---- touched ids: a thread works out kBits neighbouring places
        const int from = tid * kBits;
        const unsigned in_hist = (seen[from / 32] >> (from % 32)) & ((1u << kBits) - 1);
        for (unsigned left = in_hist | ((any[from / 32] >> (from % 32)) & ((1u << kBits) - 1)); left; left &= left - 1) {
            const int k = __ffs(left) - 1, i = from + k;
            float z = to_f32(x[i]);
            if (a.rep && ((in_hist >> k) & 1u)) z = z > 0.0f ? __fdiv_rn(z, rep) : __fmul_rn(z, rep);
            const unsigned n = count[i];
            if (n) z = __fsub_rn(__fsub_rn(z, __fmul_rn((float)n, freq)), pres);
            if (a.bias && entry[i]) z = __fadd_rn(z, a.bias[e0 + entry[i] - 1]);
            count[i] = __float_as_uint(z);
        }
        __syncthreads();
    }
    // ---- every id
    if (whole_words) {
        allowed = 0;
#pragma unroll
        for (int p = 0; p < P; p++) allowed |= ((word[p] >> (place_of(p) % 32)) & kPiece) << (p * W);
    }
    float top = -INFINITY;
#pragma unroll
    for (int p = 0; p < P; p++) {
        const int i = place_of(p);
        if (lists) {
            const unsigned hit = ((seen[i / 32] | any[i / 32]) >> (i % 32)) & kPiece;
            if (hit) {
                float z[W];
                if constexpr (W == 4) {
                    const float4 v = *reinterpret_cast<const float4 *>(count + i);
                    z[0] = v.x; z[1] = v.y; z[2] = v.z; z[3] = v.w;
                } else {
                    z[0] = __uint_as_float(count[i]);
                }
#pragma unroll
                for (int w = 0; w < W; w++) y[p][w] = (hit >> w) & 1u ? z[w] : y[p][w];
            }
        }
#pragma unroll
        for (int w = 0; w < W; w++) {
            if (!((allowed >> (p * W + w)) & 1u)) y[p][w] = -INFINITY;
            top = fmaxf(top, y[p][w]);
        }
        if (W == 4 && full) {
            *reinterpret_cast<float4 *>(out + i) = make_float4(y[p][0], y[p][1 % W], y[p][2 % W], y[p][3 % W]);
        } else {
#pragma unroll
            for (int w = 0; w < W; w++)
                if (i + w >= lo && i + w < hi) out[i + w] = y[p][w];
        }
    }
    // ---- the chunk's choice: the largest value of all, then the lowest place that has it
    unsigned long long best = 0;
    if (a.ids) {
        const unsigned key = __reduce_max_sync(0xffffffffu, ordered(top));
        int at = 0x7fffffff;
        if (ordered(top) == key) {
#pragma unroll
            for (int p = P - 1; p >= 0; p--)
#pragma unroll
                for (int w = W - 1; w >= 0; w--)
                    if (y[p][w] == top) at = place_of(p) + w;
        }
        at = __reduce_min_sync(0xffffffffu, at);
        if (lane == 0) {
            key_of[warp] = key;
            id_of[warp] = key ? (unsigned)(first + at) : 0xffffffffu;
        }
        __syncthreads();
        if (warp == 0) {
            const unsigned mine = lane < kLogitsWarps ? key_of[lane] : 0u;
            const unsigned all = __reduce_max_sync(0xffffffffu, mine);
            const unsigned id = __reduce_min_sync(0xffffffffu, lane < kLogitsWarps && mine == all ? id_of[lane] : 0xffffffffu);
            best = choice(all, (int)id);
        }
    }
    if constexpr (kCluster) {
        // every CTA of the cluster has started (the barrier's first phase): the first one's memory is
        // there; its second phase says that all have written
        const unsigned rank = blockIdx.x;
        asm volatile("barrier.cluster.wait;" ::: "memory");
        if (tid == 0) {
            uint32_t to;
            asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(to) : "r"(xdna::smem_u32(&of_rank[rank])));
            asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(to), "l"(best) : "memory");
        }
        asm volatile("barrier.cluster.arrive.release;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
        if (rank || tid || !a.ids) return;
        for (unsigned r = 1; r < gridDim.x; r++) best = max(best, of_rank[r]);
        a.ids[b] = best ? (int64_t)(0xffffffffu - (unsigned)best) : -1;
    } else if (a.ids && tid == 0) {
        a.best[b * gridDim.x + blockIdx.x] = best;
    }
}

// one warp per row: the best of its chunks
__global__ void __launch_bounds__(128) choose_kernel(const unsigned long long *best, int chunks, int B, int64_t *ids) {
    const int64_t b = blockIdx.x * 4 + threadIdx.x / 32;
    const int lane = threadIdx.x % 32;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (b >= B) return;
    unsigned long long k = 0;
    for (int c = lane; c < chunks; c += 32) {
        const unsigned long long other = best[b * chunks + c];
        k = other > k ? other : k;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) k = max(k, __shfl_xor_sync(0xffffffffu, k, o));
    if (lane == 0) ids[b] = k ? (int64_t)(0xffffffffu - (unsigned)k) : -1;
}

// ids per thread: with 4, a chunk of 2048 ids, 25 CTAs for a row of 50k; with 16, 8192
constexpr int kFewPerThread = 4, kManyPerThread = 16;
constexpr int chunks_of(int64_t ids, int per_thread) {
    return (int)((ids + kLogitsThreads * per_thread - 1) / (kLogitsThreads * per_thread));
}

template <typename T, int P, int W, bool kCluster>
cudaError_t launch_logits(const LogitsArgs &a, int B, int64_t places, cudaStream_t st) {
    const int chunks = chunks_of(places, P * W);
    const size_t smem = a.hist || a.bias ? (size_t)kLogitsThreads * P * W * 4 * (a.bias ? 2 : 1) : 0;
    if (smem > 40 * 1024) {
        static std::atomic<uint64_t> allowed{0};          // the devices (of the first 64) on which it has been raised
        int dev = 0;
        if (cudaError_t e = cudaGetDevice(&dev)) return e;
        if (dev > 63 || !(allowed.load() >> dev & 1)) {
            if (cudaError_t e = cudaFuncSetAttribute(logits_kernel<T, P, W, kCluster>,
                                                     cudaFuncAttributeMaxDynamicSharedMemorySize, kLogitsThreads * P * W * 8))
                return e;
            if (dev <= 63) allowed.fetch_or(1ull << dev);
        }
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(chunks, B);
    cfg.blockDim = dim3(kLogitsThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr{};
    cfg.attrs = &attr;
    if (kCluster) {
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim = {(unsigned)chunks, 1, 1};
        cfg.numAttrs = 1;
    }
    if (cudaError_t e = cudaLaunchKernelEx(&cfg, logits_kernel<T, P, W, kCluster>, a)) return e;
    if (kCluster || !a.ids) return cudaSuccess;
    cfg.gridDim = dim3((B + 3) / 4);
    cfg.blockDim = dim3(128);
    cfg.dynamicSmemBytes = 0;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, choose_kernel, (const unsigned long long *)a.best, chunks, B, a.ids);
}
template <typename T, int E, bool kCluster>
cudaError_t launch_logits(const LogitsArgs &a, int B, bool wide, int64_t places, cudaStream_t st) {
    return wide ? launch_logits<T, E / 4, 4, kCluster>(a, B, places, st) : launch_logits<T, E, 1, kCluster>(a, B, a.V, st);
}

// A row of up to 8 chunks is one cluster, small chunks first: one launch (1 x 50272: 5.5 us on the GPU, 10 us
// submitted from Python; chunks of 2048 and choose_kernel: 4.9 and 13 us).  A longer one takes the large
// chunks, or the small ones while the large fill less than half of the GPU (2 x 262144: 5.3 us small, 6.0
// large; 4 x 262144: 7.5 and 6.2).
template <typename T>
cudaError_t launch_logits(const LogitsArgs &a, int B, cudaStream_t st) {
    // wide accesses need logits and out of a row to lie alike against 4 elements; rows that start off
    // such a boundary take up to 3 places before their first id
    const uintptr_t x = reinterpret_cast<uintptr_t>(a.logits) / sizeof(T), o = reinterpret_cast<uintptr_t>(a.out) / 4;
    const bool wide = (x - o) % 4 == 0 && (B == 1 || (a.stride - a.out_stride) % 4 == 0);
    const int64_t places = (int64_t)a.V + (o % 4 || (B > 1 && a.out_stride % 4) ? 3 : 0);
    const int few = chunks_of(places, kFewPerThread), many = chunks_of(places, kManyPerThread);
    if (few <= kMaxCluster) return launch_logits<T, kFewPerThread, true>(a, B, wide, places, st);
    if (many <= kMaxCluster) return launch_logits<T, kManyPerThread, true>(a, B, wide, places, st);
    if ((int64_t)B * many < 80) return launch_logits<T, kFewPerThread, false>(a, B, wide, places, st);
    return launch_logits<T, kManyPerThread, false>(a, B, wide, places, st);
}

}  // namespace

extern "C" {

int xdna_rmsnorm_residual_i8(const void *x, int x_f32, int64_t x_stride, const void *residual, int res_f32,
                             int64_t res_stride, const float *gamma, int unit_offset, float eps, int M, int D,
                             void *residual_out, uint16_t *y_bf16, int8_t *q8, float *scale, void *stream) {
    const std::string me = "xdna_rmsnorm_residual_i8: ";
    if (!x || !gamma) return fail(me + "null pointer");
    if (!q8 != !scale) return fail(me + "q8 and scale go together");
    if (!residual_out && !y_bf16 && !q8) return fail(me + "no output");
    if (M < 0 || D < 1 || D > 16384) return fail(me + "negative M, or D outside 1..16384");
    if (x_stride < D || ((residual || residual_out) && res_stride < D)) return fail(me + "a row stride below D");
    if (!(eps >= 0.0f)) return fail(me + "negative eps");
    if (off_elements(x_f32 ? 4 : 2, x) || off_elements(res_f32 ? 4 : 2, residual, residual_out) ||
        off_elements(4, gamma, scale) || off_elements(2, y_bf16))
        return fail(me + "a pointer not aligned to its elements");
    if (M == 0) return 0;
    NormArgs a{x, residual, x_stride, res_stride, gamma, unit_offset, M, D, eps, residual_out,
               reinterpret_cast<__nv_bfloat16 *>(y_bf16), q8, scale};
    auto st = static_cast<cudaStream_t>(stream);
    int dev = 0, sms = 0;
    if (!ck(cudaGetDevice(&dev), "xdna_rmsnorm_residual_i8") ||
        !ck(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev), "xdna_rmsnorm_residual_i8"))
        return -1;
    const int xe = x_f32 ? 4 : 8, re = res_f32 ? 4 : 8;    // elements of 16 bytes
    const bool wide = D % 8 == 0 && x_stride % xe == 0 && (!(residual || residual_out) || res_stride % re == 0) &&
                      aligned16(x) && aligned16(gamma) && aligned16(residual) && aligned16(residual_out) && aligned16(y_bf16) &&
                      reinterpret_cast<uintptr_t>(q8) % 8 == 0;
    const cudaError_t e = x_f32 ? (res_f32 ? launch_norm<float, float>(a, wide, sms, st)
                                           : launch_norm<float, __nv_bfloat16>(a, wide, sms, st))
                                : (res_f32 ? launch_norm<__nv_bfloat16, float>(a, wide, sms, st)
                                           : launch_norm<__nv_bfloat16, __nv_bfloat16>(a, wide, sms, st));
    return ck(e, "xdna_rmsnorm_residual_i8") ? 0 : -1;
}

size_t xdna_logits_workspace(int B, int V) {
    if (B < 1 || V < 1 || chunks_of((int64_t)V + 3, kManyPerThread) <= kMaxCluster) return 0;
    return (size_t)B * chunks_of((int64_t)V + 3, kFewPerThread) * 8;
}
int xdna_logits_process(const void *logits, int src_f32, int64_t logits_stride, int B, int V,
                        const int32_t *history, int n_history, const int32_t *history_start,
                        const int32_t *n_prompt, const float *repetition, const float *frequency,
                        const float *presence, const int32_t *bias_ids, const float *bias, int n_biases,
                        const int32_t *bias_start,
                        const uint32_t *mask, int64_t mask_stride, float *out, int64_t out_stride, int64_t *ids,
                        void *workspace, void *stream) {
    const std::string me = "xdna_logits_process: ";
    if (!logits || !out) return fail(me + "null pointer");
    if (n_history < 0 || n_biases < 0) return fail(me + "negative n_history or n_biases");
    if (B < 0 || V < 1) return fail(me + "negative B or empty V");
    if (!history != !history_start) return fail(me + "history and history_start go together");
    if (!history && (n_prompt || repetition || frequency || presence)) return fail(me + "a penalty without a history");
    if (!bias != !bias_ids || !bias != !bias_start) return fail(me + "bias, bias_ids and bias_start go together");
    if (B > 1 && (logits_stride < V || out_stride < V)) return fail(me + "a row stride below V");
    if (mask && B > 1 && mask_stride < (V + 31) / 32) return fail(me + "mask_stride below (V + 31) / 32");
    if (out == logits && (!src_f32 || (B > 1 && out_stride != logits_stride)))
        return fail(me + "out on bf16 logits, or on logits of another stride");
    if (B > 65535) return fail(me + "more than 65535 rows");
    if (off_elements(src_f32 ? 4 : 2, logits) || off_elements(8, ids) ||
        off_elements(4, out, history, history_start, n_prompt, repetition, frequency, presence, bias_ids, bias, bias_start, mask))
        return fail(me + "a pointer not aligned to its elements");
    if (ids && xdna_logits_workspace(B, V) && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 8))
        return fail(me + "ids need a workspace, 8-byte aligned");
    if (B == 0) return 0;
    LogitsArgs a{logits, logits_stride, out_stride, mask_stride, V, n_history, n_biases, history, history_start, n_prompt,
                 repetition, frequency, presence, bias_ids, bias_start, bias, mask, out,
                 ids, static_cast<unsigned long long *>(workspace)};
    auto st = static_cast<cudaStream_t>(stream);
    const cudaError_t e = src_f32 ? launch_logits<float>(a, B, st) : launch_logits<__nv_bfloat16>(a, B, st);
    return ck(e, "xdna_logits_process") ? 0 : -1;
}

}  // extern "C"
