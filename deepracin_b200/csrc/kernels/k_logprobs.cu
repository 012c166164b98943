/*
 * Scoring of a network's outputs: for each row v of `len` logits at temperature 1 / s
 *
 *   lse = log sum_i exp(s v_i),  log p_i = s v_i - lse,  H = -sum_i p_i log p_i = log S - (1 / S) sum_i e_i d_i
 *
 * with d_i = s (v_i - max v), e_i = exp(d_i), S = sum e_i; the log probabilities of given labels, and the k largest logits
 * with their log probabilities.  The order of the alternatives is total: by value (NaN above everything), equal ones by
 * ascending index; a value and its index are compared as one 64-bit key.
 */
#include <math.h>
#include <stdio.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "k_common.cuh"

#define LP_THREADS 512
#define LP_KMAX 32

template <typename T> __device__ __forceinline__ float lp_load(const T *p);
template <> __device__ __forceinline__ float lp_load(const float *p) { return *p; }
template <> __device__ __forceinline__ float lp_load(const __nv_bfloat16 *p) { return __bfloat162float(*p); }
template <> __device__ __forceinline__ float lp_load(const __half *p) { return __half2float(*p); }

/* float -> uint32 with the order of the values: -inf lowest, +inf below the NaNs, which all map to one value; -0 equals +0 */
__device__ __forceinline__ uint32_t lp_order(float v)
{
    const uint32_t u = __float_as_uint(v + 0.0f);
    if ((u & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float lp_value(uint32_t o) { return o == 0xffffffffu ? __uint_as_float(0x7fffffffu) : __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o); }
__device__ __forceinline__ unsigned long long lp_key(float v, uint32_t i) { return ((unsigned long long)lp_order(v) << 32) | (0xffffffffu - i); }

__device__ __forceinline__ unsigned long long lp_block_max(unsigned long long v, unsigned long long *red)
{
    for (int o = 16; o > 0; o >>= 1) {
        const unsigned long long t = __shfl_xor_sync(0xffffffffu, v, o);
        v = t > v ? t : v;
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    for (int i = 0; i < LP_THREADS / 32; i++) v = red[i] > v ? red[i] : v;
    return v;
}
__device__ __forceinline__ float lp_block_sum(float v, float *red)
{
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.0f;
    for (int i = 0; i < LP_THREADS / 32; i++) v += red[i];
    return v;
}

template <typename T>
__global__ void __launch_bounds__(LP_THREADS) k_logprobs(const T *__restrict__ logits, size_t ld, int len, float s, const int *__restrict__ labels, int m,
                                                         float *__restrict__ logprob, float *__restrict__ entropy, int k,
                                                         float *__restrict__ top_logprob, int *__restrict__ top_index)
{
    __shared__ unsigned long long red[LP_THREADS / 32];
    __shared__ float fred[LP_THREADS / 32];
    drk_dep_wait();
    drk_dep_trigger();
    const size_t row = blockIdx.x;
    const T *v = logits + row * ld;
    unsigned long long best = 0;
    for (int i = threadIdx.x; i < len; i += LP_THREADS) {
        const unsigned long long key = lp_key(lp_load(v + i), (uint32_t)i);
        best = key > best ? key : best;
    }
    best = lp_block_max(best, red);
    const float mx = lp_value((uint32_t)(best >> 32));
    const float base = mx == -INFINITY ? 0.0f : mx;     /* a row with nothing left: every d_i is -inf */
    float S = 0.0f, t = 0.0f;
    for (int i = threadIdx.x; i < len; i += LP_THREADS) {
        const float d = (lp_load(v + i) - base) * s, e = expf(d);
        S += e;
        if (e != 0.0f) t += e * d;
    }
    S = lp_block_sum(S, fred);
    t = lp_block_sum(t, fred);
    const bool none = mx == -INFINITY;
    const float ls = logf(S);
    if (entropy && threadIdx.x == 0) entropy[row] = none ? 0.0f : ls - t / S;
    for (int j = threadIdx.x; j < m; j += LP_THREADS) {
        const int l = labels[row * m + j];
        logprob[row * m + j] = l < 0 ? 0.0f : l >= len ? __uint_as_float(0x7fffffffu) : none ? -INFINITY : (lp_load(v + l) - base) * s - ls;
    }
    for (int j = 0; j < k; j++) {
        if (threadIdx.x == 0) {
            top_logprob[row * k + j] = none ? -INFINITY : (lp_value((uint32_t)(best >> 32)) - base) * s - ls;
            top_index[row * k + j] = (int)(0xffffffffu - (uint32_t)best);
        }
        unsigned long long next = 0;
        for (int i = threadIdx.x; i < len; i += LP_THREADS) {
            const unsigned long long key = lp_key(lp_load(v + i), (uint32_t)i);
            if (key < best && key > next) next = key;
        }
        best = lp_block_max(next, red);
    }
}

static int lp_refuse(const char *why)
{
    fprintf(stderr, "dRk_logprobs: %s\n", why);
    return -1;
}

template <typename T>
static cudaError_t lp_launch(cudaStream_t st, const void *logits, size_t ld, int n, int len, float scale, const int *labels, int m, float *logprob,
                             float *entropy, int k, float *top_logprob, int *top_index)
{
    return drk_launch_dep(k_logprobs<T>, dim3((unsigned)n), dim3(LP_THREADS), 0, st, (const T *)logits, ld, len, scale, labels, m, logprob, entropy, k,
                          top_logprob, top_index);
}

extern "C" int dRk_logprobs(dRk_stream stream, const void *logits, int type, long long ld, int n, int len, float scale, const int *labels, int m,
                            float *logprob, float *entropy, int k, float *top_logprob, int *top_index)
{
    const int size = type == DRK_F32 ? 4 : type == DRK_BF16 || type == DRK_F16 ? 2 : 0;
    if (!size) return lp_refuse("unknown element type");
    if (n < 1 || len < 1) return lp_refuse("needs at least one row and one logit");
    if (n > 1 && ld < len) return lp_refuse("rows overlap (ld < len)");
    if (m < 0 || k < 0 || k > LP_KMAX || k > len) return lp_refuse("number of labels below 0, or of alternatives outside 0..min(32, len)");
    if (!logits || (m > 0 && (!labels || !logprob)) || (k > 0 && (!top_logprob || !top_index))) return lp_refuse("null pointer");
    if (!(scale > 0.0f) || isinf(scale)) return lp_refuse("scale (1 / temperature) must be positive and finite");
    if ((uintptr_t)logits % size || (uintptr_t)labels % 4 || (uintptr_t)logprob % 4 || (uintptr_t)entropy % 4 || (uintptr_t)top_logprob % 4 || (uintptr_t)top_index % 4)
        return lp_refuse("pointer not aligned to its element type");
    const int dev = drk_stream_device("dRk_logprobs", stream, -1);
    if (dev < 0) return dev;
    cudaStream_t st = drk_stream(stream);
    const size_t pitch = n > 1 ? (size_t)ld : 0;
    const cudaError_t e = type == DRK_F32    ? lp_launch<float>(st, logits, pitch, n, len, scale, labels, m, logprob, entropy, k, top_logprob, top_index)
                          : type == DRK_BF16 ? lp_launch<__nv_bfloat16>(st, logits, pitch, n, len, scale, labels, m, logprob, entropy, k, top_logprob, top_index)
                                             : lp_launch<__half>(st, logits, pitch, n, len, scale, labels, m, logprob, entropy, k, top_logprob, top_index);
    return drk_launched(e);
}
