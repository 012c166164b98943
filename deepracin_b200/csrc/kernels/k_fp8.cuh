/* What the translation units of the 8-bit fully connected layer share: sizes, element types, and the launchers of its products. */
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include "k_common.cuh"

#define FP8_BLOCK 128                                   /* values under one scale, rows of a packed block, bytes of its rows */
#define FP8_BLOCK_BYTES (FP8_BLOCK * FP8_BLOCK)
#define FP8_MAX 448.0f
#define FP8_FLOOR 0x1p-96f      /* smallest block maximum a scale is made from: 448 / A stays finite */

static inline int fp8_blocks(int n) { return (int)(((long long)n + FP8_BLOCK - 1) / FP8_BLOCK); }

template <typename T> __device__ __forceinline__ T fp8_store(float v);
template <> __device__ __forceinline__ float fp8_store<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 fp8_store<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half fp8_store<__half>(float v) { return __float2half_rn(v); }
template <typename W> __device__ __forceinline__ W fp8_store2(float a, float b);
template <> __device__ __forceinline__ __nv_bfloat162 fp8_store2<__nv_bfloat162>(float a, float b) { return __floats2bfloat162_rn(a, b); }
template <> __device__ __forceinline__ __half2 fp8_store2<__half2>(float a, float b) { return __floats2half2_rn(a, b); }

/* ReLU that lets NaN pass (a comparison with NaN is false) */
__device__ __forceinline__ float fp8_act(float v, int act)
{
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(v), "f"(act ? 0.0f : -INFINITY));
    return r;
}

struct Fp8Params {
    const void *in;
    size_t ldi;
    int in_type, Nin, vec;              /* vec: rows of `in` start on 16-byte boundaries */
    const float *sx, *scales, *bias;    /* sx [kb][n], scales [ob][kb] */
    void *out;
    size_t ldo;
    int out_type, n, Nout, kb, ob, act;
    int *status;
};

/* which product a layer's shape runs on, and its tensor maps */
struct Fp8Tensor {
    CUtensorMap mapW, mapX;
    int pairs, mtiles, ntiles;          /* k_fp8_pair: pairs of CTAs, tiles of 256 rows and of 256 outputs; pairs = 0: k_fp8_swap */
    int nt;                             /* rows per tile of k_fp8_swap */
    int fuse;                           /* 1: k_fp8_swap rounds the input itself, no launch in front */
    int stages;                         /* K blocks of the largest share: no more stages than that */
    int split;                          /* CTAs of a cluster that share a tile's K blocks */
};

int drk_fp8_tensor_plan(Fp8Tensor *t, const Fp8Params *p, const void *codes, const void *q, int sms);
int drk_fp8_tensor_launch(cudaStream_t st, const Fp8Tensor *t, const Fp8Params *p);
