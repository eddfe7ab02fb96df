// decode_ops.cu -- the serving ops on both sides of a decoder layer's products
// (include/xdna_b200.h): the residual RMS norm with int8 rows, and the logits processor.
#include <cuda_runtime.h>
#include <cuda_bf16.h>

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

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void from_f32(float x, float *p) { *p = x; }
__device__ __forceinline__ void from_f32(float x, __nv_bfloat16 *p) { *p = __float2bfloat16_rn(x); }

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

template <typename X, typename R>
__global__ void __launch_bounds__(256) rmsnorm_kernel(const NormArgs a) {
    __shared__ float red[2][8];
    const int64_t row = blockIdx.x;
    const X *x = static_cast<const X *>(a.x) + row * a.x_stride;
    const R *res = a.res ? static_cast<const R *>(a.res) + row * a.res_stride : nullptr;
    float sum = 0.0f, top = 0.0f;
    for (int i = threadIdx.x; i < a.D; i += 256) {
        const float r = res ? __fadd_rn(to_f32(x[i]), to_f32(res[i])) : to_f32(x[i]);
        const float g = a.unit_offset ? __fadd_rn(a.gamma[i], 1.0f) : a.gamma[i];
        sum = fmaf(r, r, sum);
        top = fmaxf(top, fabsf(__fmul_rn(r, g)));
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        sum += __shfl_xor_sync(0xffffffffu, sum, o);
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    }
    if (threadIdx.x % 32 == 0) {
        red[0][threadIdx.x / 32] = sum;
        red[1][threadIdx.x / 32] = top;
    }
    __syncthreads();
    sum = 0.0f;
#pragma unroll
    for (int w = 0; w < 8; w++) {
        sum += red[0][w];
        top = fmaxf(top, red[1][w]);
    }
    const float inv = rsqrtf(__fdiv_rn(sum, (float)a.D) + a.eps);
    const bool zero = !(top > 3.8e-37f);
    const float to8 = zero ? 0.0f : __fmul_rn(__frcp_rn(top), 127.0f);
    for (int i = threadIdx.x; i < a.D; i += 256) {
        const float r = res ? __fadd_rn(to_f32(x[i]), to_f32(res[i])) : to_f32(x[i]);
        const float g = a.unit_offset ? __fadd_rn(a.gamma[i], 1.0f) : a.gamma[i];
        const float t = __fmul_rn(r, g);
        if (a.res_out) from_f32(r, static_cast<R *>(a.res_out) + row * a.res_stride + i);
        if (a.y) a.y[row * a.D + i] = __float2bfloat16_rn(t * inv);
        if (a.q8) a.q8[row * a.D + i] = (int8_t)max(-127, min(127, __float2int_rn(__fmul_rn(t, to8))));
    }
    if (a.scale && threadIdx.x == 0) a.scale[row] = zero ? 1.0f : __fmul_rn(__fdiv_rn(top, 127.0f), inv);
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
};

constexpr int kVocabChunk = 4096;            // ids whose counts and bias entries lie in shared memory

// one CTA per row
template <typename T>
__global__ void __launch_bounds__(512) logits_kernel(const LogitsArgs a) {
    __shared__ unsigned count[kVocabChunk];  // generated occurrences; bit 31: seen at all
    __shared__ int entry[kVocabChunk];       // 1 + the last bias entry of the id
    __shared__ unsigned long long best;
    const int64_t b = blockIdx.x;
    const int tid = threadIdx.x;
    const int h0 = a.hist ? max(0, a.hist_start[b]) : 0, h1 = a.hist ? min(a.n_hist, a.hist_start[b + 1]) : 0;
    const int64_t gen = (int64_t)h0 + (a.n_prompt ? a.n_prompt[b] : 0);
    const int e0 = a.bias ? max(0, a.bias_start[b]) : 0, e1 = a.bias ? min(a.n_bias, a.bias_start[b + 1]) : 0;
    const float rep = a.rep ? a.rep[b] : 1.0f, freq = a.freq ? a.freq[b] : 0.0f, pres = a.pres ? a.pres[b] : 0.0f;
    const T *x = static_cast<const T *>(a.logits) + b * a.stride;
    if (tid == 0) best = 0;
    unsigned long long mine = 0;
    for (int v0 = 0; v0 < a.V; v0 += kVocabChunk) {
        const int nv = min(kVocabChunk, a.V - v0);
        __syncthreads();
        for (int i = tid; i < nv; i += 512) count[i] = 0, entry[i] = 0;
        __syncthreads();
        for (int j = h0 + tid; j < h1; j += 512) {
            const int i = a.hist[j] - v0;
            if (i >= 0 && i < nv) {
                atomicOr(&count[i], 0x80000000u);
                if (j >= gen) atomicAdd(&count[i], 1u);
            }
        }
        for (int j = e0 + tid; j < e1; j += 512) {
            const int i = a.bias_ids[j] - v0;
            if (i >= 0 && i < nv) atomicMax(&entry[i], j - e0 + 1);
        }
        __syncthreads();
        for (int i = tid; i < nv; i += 512) {
            float y = to_f32(x[v0 + i]);
            const unsigned n = count[i];
            if (n) {
                const unsigned g = n & 0x7fffffffu;
                if (a.rep) y = y > 0.0f ? __fdiv_rn(y, rep) : __fmul_rn(y, rep);
                if (g) y = __fsub_rn(__fsub_rn(y, __fmul_rn((float)g, freq)), pres);
            }
            if (entry[i]) y = __fadd_rn(y, a.bias[e0 + entry[i] - 1]);
            if (a.mask && !((a.mask[b * a.mask_stride + (v0 + i) / 32] >> ((v0 + i) % 32)) & 1u)) y = -INFINITY;
            a.out[b * a.out_stride + v0 + i] = y;
            if (y > -INFINITY) {             // ordered bits, then the lower id
                const unsigned u = __float_as_uint(y == 0.0f ? 0.0f : y);
                const unsigned key = u & 0x80000000u ? ~u : u | 0x80000000u;
                mine = max(mine, ((unsigned long long)key << 32) | (0xffffffffu - (unsigned)(v0 + i)));
            }
        }
    }
    if (mine) atomicMax(&best, mine);
    __syncthreads();
    if (a.ids && tid == 0) a.ids[b] = best ? (int64_t)(0xffffffffu - (unsigned)best) : -1;
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
    if (x_f32 && res_f32) rmsnorm_kernel<float, float><<<M, 256, 0, st>>>(a);
    else if (x_f32) rmsnorm_kernel<float, __nv_bfloat16><<<M, 256, 0, st>>>(a);
    else if (res_f32) rmsnorm_kernel<__nv_bfloat16, float><<<M, 256, 0, st>>>(a);
    else rmsnorm_kernel<__nv_bfloat16, __nv_bfloat16><<<M, 256, 0, st>>>(a);
    return ck(cudaGetLastError(), "xdna_rmsnorm_residual_i8") ? 0 : -1;
}

int xdna_logits_process(const void *logits, int src_f32, int64_t logits_stride, int B, int V,
                        const int32_t *history, int n_history, const int32_t *history_start,
                        const int32_t *n_prompt, const float *repetition, const float *frequency,
                        const float *presence, const int32_t *bias_ids, const float *bias, int n_biases,
                        const int32_t *bias_start,
                        const uint32_t *mask, int64_t mask_stride, float *out, int64_t out_stride, int64_t *ids,
                        void *stream) {
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
    if (B == 0) return 0;
    LogitsArgs a{logits, logits_stride, out_stride, mask_stride, V, n_history, n_biases, history, history_start, n_prompt, repetition,
                 frequency, presence, bias_ids, bias_start, bias, mask, out, ids};
    auto st = static_cast<cudaStream_t>(stream);
    if (src_f32) logits_kernel<float><<<B, 512, 0, st>>>(a);
    else logits_kernel<__nv_bfloat16><<<B, 512, 0, st>>>(a);
    return ck(cudaGetLastError(), "xdna_logits_process") ? 0 : -1;
}

}  // extern "C"
