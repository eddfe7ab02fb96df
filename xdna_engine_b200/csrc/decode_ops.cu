// decode_ops.cu -- the serving ops on both sides of a decoder layer's products
// (include/xdna_b200.h): the residual RMS norm with int8 rows, and the logits processor.
#include <cuda_runtime.h>
#include <cuda_bf16.h>

#include <algorithm>
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

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }

// ----------------------------------------------------------------- residual RMS norm, int8
struct NormArgs {
    const void *x, *res;
    int64_t x_stride, res_stride;
    const float *gamma;
    int unit_offset, D;
    float eps;
    void *res_out;
    __nv_bfloat16 *y;
    int8_t *q8;
    float *scale;
};

// N elements of a row as f32 (8: one or two 16-byte loads)
template <int N>
__device__ __forceinline__ void load_n(const float *p, float (&v)[N]) {
    if constexpr (N == 8) {
        const float4 a = __ldcs(reinterpret_cast<const float4 *>(p)), b = __ldcs(reinterpret_cast<const float4 *>(p) + 1);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
        v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
        v[0] = __ldcs(p);
    }
}
template <int N>
__device__ __forceinline__ void load_n(const __nv_bfloat16 *p, float (&v)[N]) {
    if constexpr (N == 8) {
        const uint4 a = __ldcs(reinterpret_cast<const uint4 *>(p));
        const uint32_t u[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            v[2 * i] = xdna::bf16lo(u[i]);
            v[2 * i + 1] = xdna::bf16hi(u[i]);
        }
    } else {
        v[0] = __bfloat162float(*p);
    }
}
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
        for (int i = 0; i < 4; i++) u[i] = xdna::bf16bits(v[2 * i]) | (xdna::bf16bits(v[2 * i + 1]) << 16);
        *reinterpret_cast<uint4 *>(p) = make_uint4(u[0], u[1], u[2], u[3]);
    } else {
        *p = __float2bfloat16_rn(v[0]);
    }
}

// One CTA per row, one pass: a thread keeps P pieces of N elements in registers, so that x and the
// residual are read once (7 bytes an element with bf16 in and out: HBM bounds it); the sum of squares and
// max|r g| need one joint reduction, since the row's factor 1 / rms scales both y and its maximum and
// drops out of the whole numbers.  N = 8 where every row is 16-byte aligned, else N = 1.
template <typename X, typename R, int N, int P>
__global__ void __launch_bounds__(1024) rmsnorm_kernel(const NormArgs a) {
    __shared__ float red[2][32];
    const int64_t row = blockIdx.x;
    const X *x = static_cast<const X *>(a.x) + row * a.x_stride;
    const R *res = a.res ? static_cast<const R *>(a.res) + row * a.res_stride : nullptr;
    const int threads = blockDim.x, lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    float r[P][N];
#pragma unroll
    for (int p = 0; p < P; p++) {
        const int i = (p * threads + threadIdx.x) * N;
        if (i < a.D) {
            load_n(x + i, r[p]);
            if (res) {
                float y[N];
                load_n(res + i, y);
#pragma unroll
                for (int k = 0; k < N; k++) r[p][k] = __fadd_rn(r[p][k], y[k]);
            }
        } else {
#pragma unroll
            for (int k = 0; k < N; k++) r[p][k] = 0.0f;
        }
    }
    float sum = 0.0f, top = 0.0f;
#pragma unroll
    for (int p = 0; p < P; p++) {
        const int i = (p * threads + threadIdx.x) * N;
        if (i >= a.D) break;
        if (a.res_out) store_n(static_cast<R *>(a.res_out) + row * a.res_stride + i, r[p]);
        float w[N];
        if constexpr (N == 8) {
            const float4 lo = __ldg(reinterpret_cast<const float4 *>(a.gamma + i)),
                         hi = __ldg(reinterpret_cast<const float4 *>(a.gamma + i) + 1);
            w[0] = lo.x; w[1] = lo.y; w[2] = lo.z; w[3] = lo.w;
            w[4] = hi.x; w[5] = hi.y; w[6] = hi.z; w[7] = hi.w;
        } else {
            w[0] = __ldg(a.gamma + i);
        }
#pragma unroll
        for (int k = 0; k < N; k++) {
            const float g = a.unit_offset ? __fadd_rn(w[k], 1.0f) : w[k];
            sum = fmaf(r[p][k], r[p][k], sum);
            r[p][k] = __fmul_rn(r[p][k], g);
            top = fmaxf(top, fabsf(r[p][k]));
        }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        sum += __shfl_xor_sync(0xffffffffu, sum, o);
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    }
    if (lane == 0) {
        red[0][warp] = sum;
        red[1][warp] = top;
    }
    __syncthreads();
    sum = lane < threads / 32 ? red[0][lane] : 0.0f;
    top = lane < threads / 32 ? red[1][lane] : 0.0f;
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        sum += __shfl_xor_sync(0xffffffffu, sum, o);
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    }
    const float inv = rsqrtf(__fdiv_rn(sum, (float)a.D) + a.eps);
    // below 127 / FLT_MAX the factor would be infinite: such a row counts as zero
    const bool zero = !(top > 3.8e-37f);
    const float to8 = zero ? 0.0f : __fmul_rn(__frcp_rn(top), 127.0f);
#pragma unroll
    for (int p = 0; p < P; p++) {
        const int i = (p * threads + threadIdx.x) * N;
        if (i >= a.D) break;
        if (a.q8) {
            uint32_t w[N == 8 ? 2 : 1] = {};
#pragma unroll
            for (int k = 0; k < N; k++)
                w[k / 4] |= ((uint32_t)max(-127, min(127, __float2int_rn(__fmul_rn(r[p][k], to8)))) & 0xffu) << (8 * (k % 4));
            if constexpr (N == 8) *reinterpret_cast<uint2 *>(a.q8 + row * a.D + i) = make_uint2(w[0], w[1]);
            else a.q8[row * a.D + i] = (int8_t)w[0];
        }
        if (a.y) {
            float y[N];
#pragma unroll
            for (int k = 0; k < N; k++) y[k] = r[p][k] * inv;
            store_n(a.y + row * a.D + i, y);
        }
    }
    if (a.scale && threadIdx.x == 0) a.scale[row] = zero ? 1.0f : __fmul_rn(__fdiv_rn(top, 127.0f), inv);
}

// threads and pieces: enough threads that a thread keeps one piece, up to 256 of them; then up to 4
// pieces of 8 (16 of 1), which 512 (1024) threads cover D = 16384 with
template <typename X, typename R>
cudaError_t launch_norm(const NormArgs &a, int M, bool wide, cudaStream_t st) {
    const int pieces = wide ? a.D / 8 : a.D;
    auto threads = [&](int p) { return std::max(32, ((pieces + p - 1) / p + 31) / 32 * 32); };
    if (wide) {
        if (pieces <= 256) rmsnorm_kernel<X, R, 8, 1><<<M, threads(1), 0, st>>>(a);
        else if (pieces <= 512) rmsnorm_kernel<X, R, 8, 2><<<M, threads(2), 0, st>>>(a);
        else rmsnorm_kernel<X, R, 8, 4><<<M, threads(4), 0, st>>>(a);
    } else {
        if (pieces <= 1024) rmsnorm_kernel<X, R, 1, 4><<<M, threads(4), 0, st>>>(a);
        else rmsnorm_kernel<X, R, 1, 16><<<M, threads(16), 0, st>>>(a);
    }
    return cudaGetLastError();
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
    unsigned long long *best;                             // [B][chunks], NULL: no id wanted
};

// x with its id as one number that is larger for the larger x, of equals for the lower id; 0: none
__device__ __forceinline__ unsigned long long choice(float x, int id) {
    const unsigned u = __float_as_uint(x == 0.0f ? 0.0f : x);
    const unsigned key = u & 0x80000000u ? ~u : u | 0x80000000u;
    return x > -INFINITY ? ((unsigned long long)key << 32) | (0xffffffffu - (unsigned)id) : 0ull;
}
__device__ __forceinline__ unsigned long long largest(unsigned long long k) {
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const unsigned long long other = __shfl_xor_sync(0xffffffffu, k, o);
        k = other > k ? other : k;
    }
    return k;
}

// One CTA per row and chunk of 512 E ids.  A logit is read once into a register before anything else, so
// that its latency passes under the counting: the chunk's counts and bias entries are built in
// shared memory from the row's history and bias list (integer atomics, so in any order), which every
// chunk of the row scans.  4 + 4 bytes an id in f32: HBM bounds it.  The chunk's best id goes to the
// workspace, from which choose_kernel takes the row's.
constexpr int kLogitsThreads = 512;
template <typename T, int E>
__global__ void __launch_bounds__(kLogitsThreads) logits_kernel(const LogitsArgs a) {
    constexpr int kChunk = kLogitsThreads * E;
    extern __shared__ unsigned smem[];
    __shared__ unsigned long long red[kLogitsThreads / 32];
    unsigned *count = smem;                               // generated occurrences; bit 31: seen at all
    int *entry = reinterpret_cast<int *>(smem + (a.hist ? kChunk : 0));   // 1 + the id's last bias entry
    const int64_t b = blockIdx.y;
    const int tid = threadIdx.x, v0 = blockIdx.x * kChunk, nv = min(kChunk, a.V - v0);
    const T *x = static_cast<const T *>(a.logits) + b * a.stride + v0;
    float y[E];
#pragma unroll
    for (int e = 0; e < E; e++) {
        const int i = e * kLogitsThreads + tid;
        y[e] = i < nv ? to_f32(x[i]) : -INFINITY;
    }
    const int h0 = a.hist ? max(0, a.hist_start[b]) : 0, h1 = a.hist ? min(a.n_hist, a.hist_start[b + 1]) : 0;
    const int64_t gen = (int64_t)h0 + (a.n_prompt ? a.n_prompt[b] : 0);
    const int e0 = a.bias ? max(0, a.bias_start[b]) : 0, e1 = a.bias ? min(a.n_bias, a.bias_start[b + 1]) : 0;
    if (a.hist || a.bias) {
        const int words = kChunk * ((a.hist ? 1 : 0) + (a.bias ? 1 : 0));
        for (int i = tid; i < words / 4; i += kLogitsThreads) reinterpret_cast<uint4 *>(smem)[i] = make_uint4(0, 0, 0, 0);
        __syncthreads();
        for (int j = h0 + tid; j < h1; j += kLogitsThreads) {
            const unsigned i = (unsigned)a.hist[j] - (unsigned)v0;
            if (i < (unsigned)nv) {
                atomicOr(&count[i], 0x80000000u);
                if (j >= gen) atomicAdd(&count[i], 1u);
            }
        }
        for (int j = e0 + tid; j < e1; j += kLogitsThreads) {
            const unsigned i = (unsigned)a.bias_ids[j] - (unsigned)v0;
            if (i < (unsigned)nv) atomicMax(&entry[i], j - e0 + 1);
        }
        __syncthreads();
    }
    const float rep = a.rep ? a.rep[b] : 1.0f, freq = a.freq ? a.freq[b] : 0.0f, pres = a.pres ? a.pres[b] : 0.0f;
    float *out = a.out + b * a.out_stride + v0;
    float best = -INFINITY;
    int at = 0;
#pragma unroll
    for (int e = 0; e < E; e++) {
        const int i = e * kLogitsThreads + tid;
        if (i >= nv) break;
        const unsigned n = a.hist ? count[i] : 0u;
        if (n) {
            const unsigned g = n & 0x7fffffffu;
            if (a.rep) y[e] = y[e] > 0.0f ? __fdiv_rn(y[e], rep) : __fmul_rn(y[e], rep);
            if (g) y[e] = __fsub_rn(__fsub_rn(y[e], __fmul_rn((float)g, freq)), pres);
        }
        if (a.bias && entry[i]) y[e] = __fadd_rn(y[e], a.bias[e0 + entry[i] - 1]);
        // a warp's 32 ids share a word
        if (a.mask && !((a.mask[b * a.mask_stride + (v0 + i) / 32] >> (tid % 32)) & 1u)) y[e] = -INFINITY;
        out[i] = y[e];
        if (y[e] > best) {                                // ids ascend: of equals the first stays
            best = y[e];
            at = v0 + i;
        }
    }
    if (!a.best) return;
    unsigned long long k = largest(choice(best, at));
    if (tid % 32 == 0) red[tid / 32] = k;
    __syncthreads();
    if (tid >= 32) return;
    k = largest(tid < kLogitsThreads / 32 ? red[tid] : 0ull);
    if (tid == 0) a.best[b * gridDim.x + blockIdx.x] = k;
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
    k = largest(k);
    if (lane == 0) ids[b] = k ? (int64_t)(0xffffffffu - (unsigned)k) : -1;
}

constexpr int kFewestPerThread = 4, kMostPerThread = 16;

template <typename T, int E>
cudaError_t launch_logits(const LogitsArgs &a, int B, int64_t *ids, cudaStream_t st) {
    constexpr int kChunk = kLogitsThreads * E;
    const int chunks = (a.V + kChunk - 1) / kChunk;
    const size_t smem = (size_t)kChunk * 4 * ((a.hist ? 1 : 0) + (a.bias ? 1 : 0));
    if (smem > 48 * 1024)
        if (cudaError_t e = cudaFuncSetAttribute(logits_kernel<T, E>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem))
            return e;
    logits_kernel<T, E><<<dim3(chunks, B), kLogitsThreads, smem, st>>>(a);
    if (cudaError_t e = cudaGetLastError()) return e;
    if (!ids) return cudaSuccess;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((B + 3) / 4);
    cfg.blockDim = dim3(128);
    cfg.stream = st;
    cudaLaunchAttribute early{};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &early;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, choose_kernel, (const unsigned long long *)a.best, chunks, B, ids);
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
    if (M == 0) return 0;
    NormArgs a{x, residual, x_stride, res_stride, gamma, unit_offset, D, eps, residual_out,
               reinterpret_cast<__nv_bfloat16 *>(y_bf16), q8, scale};
    auto st = static_cast<cudaStream_t>(stream);
    const int xe = x_f32 ? 4 : 8, re = res_f32 ? 4 : 8;    // elements of 16 bytes
    const bool wide = D % 8 == 0 && x_stride % xe == 0 && (!(residual || residual_out) || res_stride % re == 0) &&
                      aligned16(x) && aligned16(gamma) && aligned16(residual) && aligned16(residual_out) && aligned16(y_bf16) &&
                      reinterpret_cast<uintptr_t>(q8) % 8 == 0;
    const cudaError_t e = x_f32 ? (res_f32 ? launch_norm<float, float>(a, M, wide, st)
                                           : launch_norm<float, __nv_bfloat16>(a, M, wide, st))
                                : (res_f32 ? launch_norm<__nv_bfloat16, float>(a, M, wide, st)
                                           : launch_norm<__nv_bfloat16, __nv_bfloat16>(a, M, wide, st));
    return ck(e, "xdna_rmsnorm_residual_i8") ? 0 : -1;
}

size_t xdna_logits_workspace(int B, int V) {
    constexpr int kChunk = kLogitsThreads * kFewestPerThread;
    return B > 0 && V > 0 ? (size_t)B * (((size_t)V + kChunk - 1) / kChunk) * 8 : 0;
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
    if (ids && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 8)) return fail(me + "ids need a workspace, 8-byte aligned");
    if (B == 0) return 0;
    LogitsArgs a{logits, logits_stride, out_stride, mask_stride, V, n_history, n_biases, history, history_start, n_prompt,
                 repetition, frequency, presence, bias_ids, bias_start, bias, mask, out,
                 ids ? static_cast<unsigned long long *>(workspace) : nullptr};
    auto st = static_cast<cudaStream_t>(stream);
    // few rows: smaller chunks, until there is one for every SM
    const bool few = (int64_t)B * ((V + 8191) / 8192) < 148;
    const cudaError_t e =
        src_f32 ? (few ? launch_logits<float, kFewestPerThread>(a, B, ids, st) : launch_logits<float, kMostPerThread>(a, B, ids, st))
                : (few ? launch_logits<__nv_bfloat16, kFewestPerThread>(a, B, ids, st) : launch_logits<__nv_bfloat16, kMostPerThread>(a, B, ids, st));
    return ck(e, "xdna_logits_process") ? 0 : -1;
}

}  // extern "C"
