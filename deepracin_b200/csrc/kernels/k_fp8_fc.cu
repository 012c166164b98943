/*
 * Fully connected layer with operands in 8-bit floating point (e4m3), a scale for each block of 128:
 *
 *   out[r][o] = act(bias[o] + sum_b sx[b][r] * sw[o / 128][b] * sum_{k in block b} qx[r][k] * qw[o][k])
 *
 * Weights carry one float scale per 128 x 128 block, each row of the input one per block of 128 values, taken when the
 * layer runs: A = max(largest |x| of the block, 2^-96), qx = e4m3(x * (448 / A)), sx = A / 448 (all in 32 bits, codes
 * rounded to nearest even).  The sums of a block and over the blocks are held in 32 bits.
 *
 * Packed weights: [ceil(Nout/128)][ceil(Nin/128)] blocks of 128 rows (outputs) x 128 bytes (inputs), zero behind the edges,
 * then their scales as floats in the same order.  A block is one contiguous 16 KiB run, so a weight stream reads DRAM in order.
 */
#include <math.h>
#include <stdio.h>
#include <stdlib.h>
#include "k_fp8.cuh"


template <typename T> __device__ __forceinline__ float fp8_load(const T *p);
template <> __device__ __forceinline__ float fp8_load(const float *p) { return *p; }
template <> __device__ __forceinline__ float fp8_load(const __nv_bfloat16 *p) { return __bfloat162float(*p); }
template <> __device__ __forceinline__ float fp8_load(const __half *p) { return __half2float(*p); }
__device__ __forceinline__ float fp8_decode(unsigned char c) { return __half2float(__half(__nv_cvt_fp8_to_halfraw(c, __NV_E4M3))); }

/* the largest magnitude of eight values, NaN aside, two at a time in 16 bits */
template <typename T> __device__ __forceinline__ float fp8_largest(const uint4 *raw);
template <> __device__ __forceinline__ float fp8_largest<float>(const uint4 *raw)
{
    const float *v = reinterpret_cast<const float *>(raw);
    float a = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; j++) a = fmaxf(a, fabsf(v[j]));
    return a;
}
__device__ __forceinline__ uint32_t fp8_max2(uint32_t a, uint32_t b, __nv_bfloat16) { uint32_t r; asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b)); return r; }
__device__ __forceinline__ uint32_t fp8_max2(uint32_t a, uint32_t b, __half) { uint32_t r; asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b)); return r; }
template <typename T> __device__ __forceinline__ float fp8_largest(const uint4 *raw)
{
    const uint32_t m = 0x7fff7fffu;
    const uint32_t r = fp8_max2(fp8_max2(raw->x & m, raw->y & m, T()), fp8_max2(raw->z & m, raw->w & m, T()), T());
    const T *two = reinterpret_cast<const T *>(&r);
    return fmaxf(fp8_load(two), fp8_load(two + 1));
}

/* ------------------------------------------------------------------ activations
 * A team of 16 / G lanes owns a block of 128 values of one row, G times 8 per lane.  Bound by HBM (reads sizeof(T), writes one byte
 * a value; 4096 x 8192: fp32 28 us, 26 at the copy rate; bf16 17.4 us, 15) when G = 2; with G = 1 a warp issues nearly twice as
 * much per value (bf16 21.6 us), G = 4 is no faster and twice as slow off 16-byte boundaries.  Few blocks: G = 1, more warps.
 * q: [block][n rows][128], sx: [block][n rows]. */
template <typename T, int G>
__global__ void __launch_bounds__(256) k_fp8_quantize_rows(const T *__restrict__ in, size_t ldi, unsigned char *__restrict__ q, float *__restrict__ sx,
                                                           int n, int Nin, int kb, int vec)
{
    drk_dep_wait();
    drk_dep_trigger();
    constexpr int W = sizeof(T) / 2;        /* 16-byte loads of 8 values */
    constexpr int LANES = 16 / G, TEAMS = 32 / LANES;
    const int sub = threadIdx.x % LANES;
    const unsigned total = (unsigned)n * (unsigned)kb, teams = gridDim.x * (blockDim.x / LANES);
    /* whole warps stay in the loop: their teams shuffle together */
    unsigned i0 = (blockIdx.x * (blockDim.x / 32) + (threadIdx.x >> 5)) * TEAMS;
    const unsigned first = i0 + (threadIdx.x & 31) / LANES, drow = teams / (unsigned)kb, dblk = teams - drow * (unsigned)kb;
    unsigned row = first / (unsigned)kb, blk = first - row * (unsigned)kb;
    for (; i0 < total; i0 += teams) {
        const bool here = row < (unsigned)n;
        uint4 raw[G][W];
        float a = FP8_FLOOR;
#pragma unroll
        for (int g = 0; g < G; g++) {
            const int k0 = (int)blk * FP8_BLOCK + (g * LANES + sub) * 8;
            const T *src = in + row * ldi + k0;
#pragma unroll
            for (int j = 0; j < W; j++) raw[g][j] = make_uint4(0u, 0u, 0u, 0u);
            if (here && vec && k0 + 8 <= Nin) {
#pragma unroll
                for (int j = 0; j < W; j++) raw[g][j] = __ldg(reinterpret_cast<const uint4 *>(src) + j);
            } else if (here) {
                T *one = reinterpret_cast<T *>(raw[g]);
#pragma unroll
                for (int j = 0; j < 8; j++) if (k0 + j < Nin) one[j] = src[j];
            }
        }
#pragma unroll
        for (int g = 0; g < G; g++) a = fmaxf(a, fp8_largest<T>(raw[g]));
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
        const float inv = __fdiv_rn(FP8_MAX, a), scale = __fdiv_rn(a, FP8_MAX);
        const size_t at = (size_t)blk * n + row;
#pragma unroll
        for (int g = 0; g < G; g++) {
            float v[8];
            uint32_t c[2];
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = fp8_load(reinterpret_cast<const T *>(raw[g]) + j) * inv;
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(v[4 * j], v[4 * j + 1]), __NV_SATFINITE, __NV_E4M3);
                const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(v[4 * j + 2], v[4 * j + 3]), __NV_SATFINITE, __NV_E4M3);
                c[j] = lo | (hi << 16);
            }
            if (here) *reinterpret_cast<uint2 *>(q + at * FP8_BLOCK + (g * LANES + sub) * 8) = make_uint2(c[0], c[1]);
        }
        if (here && sub == 0) sx[at] = scale;
        row += drow;
        blk += dblk;
        if (blk >= (unsigned)kb) { blk -= kb; row++; }
    }
}

/* Many 32-bit rows off 16-byte boundaries: a warp per block, value j * 32 + lane, so that single loads and stores are contiguous;
 * four blocks under way, a lane divides for one of them.  4096 x 8191: 34 us, 47 us with single loads in the kernel above; in 16
 * bits, where a warp's load is 64 bytes, 40 against 29 us. */
__global__ void __launch_bounds__(256) k_fp8_quantize_unaligned(const float *__restrict__ in, size_t ldi, unsigned char *__restrict__ q, float *__restrict__ sx,
                                                                int n, int Nin, int kb)
{
    drk_dep_wait();
    drk_dep_trigger();
    constexpr int U = 4;
    const int lane = threadIdx.x & 31;
    const unsigned total = (unsigned)n * (unsigned)kb, warps = gridDim.x * (blockDim.x / 32), drow = warps / (unsigned)kb, dblk = warps - drow * (unsigned)kb;
    unsigned i0 = blockIdx.x * (blockDim.x / 32) + (threadIdx.x >> 5);
    unsigned row = i0 / (unsigned)kb, blk = i0 - row * (unsigned)kb;
    for (; i0 < total; i0 += U * warps) {
        float v[U][4], a[U];
        unsigned rows[U], blks[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            rows[u] = row; blks[u] = blk;
            const int k0 = (int)blk * FP8_BLOCK + lane;
            const float *src = in + row * ldi + k0;
#pragma unroll
            for (int j = 0; j < 4; j++) v[u][j] = row < (unsigned)n && k0 + j * 32 < Nin ? src[j * 32] : 0.0f;
            row += drow;
            blk += dblk;
            if (blk >= (unsigned)kb) { blk -= kb; row++; }
        }
#pragma unroll
        for (int u = 0; u < U; u++) a[u] = fmaxf(fmaxf(fmaxf(FP8_FLOOR, fabsf(v[u][0])), fabsf(v[u][1])), fmaxf(fabsf(v[u][2]), fabsf(v[u][3])));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
#pragma unroll
            for (int u = 0; u < U; u++) a[u] = fmaxf(a[u], __shfl_xor_sync(0xffffffffu, a[u], o));
        float b = a[0];
#pragma unroll
        for (int u = 1; u < U; u++) b = lane % U == u ? a[u] : b;
        const float bi = __fdiv_rn(FP8_MAX, b), bs = __fdiv_rn(b, FP8_MAX);
#pragma unroll
        for (int u = 0; u < U; u++) {
            const float inv = __shfl_sync(0xffffffffu, bi, u);
            if (rows[u] >= (unsigned)n) continue;
            const size_t at = (size_t)blks[u] * n + rows[u];
            unsigned char *to = q + at * FP8_BLOCK + lane;
#pragma unroll
            for (int j = 0; j < 4; j += 2) {
                const uint32_t two = __nv_cvt_float2_to_fp8x2(make_float2(v[u][j] * inv, v[u][j + 1] * inv), __NV_SATFINITE, __NV_E4M3);
                to[j * 32] = (unsigned char)two;
                to[j * 32 + 32] = (unsigned char)(two >> 8);
            }
            if (lane == u) sx[at] = bs;
        }
    }
}

/* ------------------------------------------------------------------ weights
 * The layer's kernel reads packed weights by TMA before it waits for the launch in front, so what writes them ends with this. */
__device__ __forceinline__ void fp8_publish() { asm volatile("fence.proxy.async;\n\tfence.acq_rel.gpu;" ::: "memory"); }

/*
 * One CTA per 128 x 128 block of w [Nin][Nout]: the block goes through shared memory, once for its largest magnitude and
 * once transposed into codes. */
__global__ void __launch_bounds__(256) k_fp8_pack_weights(const float *__restrict__ w, unsigned char *__restrict__ codes, float *__restrict__ scales,
                                                          int Nin, int Nout, int kb)
{
    __shared__ float tile[32][FP8_BLOCK + 1];
    __shared__ float red[8];
    const int b = blockIdx.x % kb, ob = blockIdx.x / kb;
    float a = FP8_FLOOR;
    for (int i = threadIdx.x; i < FP8_BLOCK_BYTES; i += 256) {
        const int k = b * FP8_BLOCK + i / FP8_BLOCK, o = ob * FP8_BLOCK + i % FP8_BLOCK;
        if (k < Nin && o < Nout) a = fmaxf(a, fabsf(w[(size_t)k * Nout + o]));
    }
    for (int s = 16; s > 0; s >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, s));
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = a;
    __syncthreads();
    for (int s = 0; s < 8; s++) a = fmaxf(a, red[s]);
    const float inv = __fdiv_rn(FP8_MAX, a);
    for (int k0 = 0; k0 < FP8_BLOCK; k0 += 32) {
        __syncthreads();
        for (int i = threadIdx.x; i < 32 * FP8_BLOCK; i += 256) {
            const int k = b * FP8_BLOCK + k0 + i / FP8_BLOCK, o = ob * FP8_BLOCK + i % FP8_BLOCK;
            tile[i / FP8_BLOCK][i % FP8_BLOCK] = k < Nin && o < Nout ? w[(size_t)k * Nout + o] * inv : 0.0f;
        }
        __syncthreads();
        for (int i = threadIdx.x; i < 32 * FP8_BLOCK / 4; i += 256) {
            const int o = i / 8, k = (i % 8) * 4;
            const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(tile[k][o], tile[k + 1][o]), __NV_SATFINITE, __NV_E4M3);
            const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(tile[k + 2][o], tile[k + 3][o]), __NV_SATFINITE, __NV_E4M3);
            *reinterpret_cast<uint32_t *>(codes + (size_t)blockIdx.x * FP8_BLOCK_BYTES + o * FP8_BLOCK + k0 + k) = lo | (hi << 16);
        }
    }
    if (threadIdx.x == 0) scales[blockIdx.x] = __fdiv_rn(a, FP8_MAX);
    fp8_publish();
}

__global__ void __launch_bounds__(256) k_fp8_pack_codes(const unsigned char *__restrict__ src, size_t ldw, const float *__restrict__ src_scales,
                                                        unsigned char *__restrict__ codes, float *__restrict__ scales, int Nin, int Nout, int kb)
{
    const int b = blockIdx.x % kb, ob = blockIdx.x / kb;
    for (int i = threadIdx.x; i < FP8_BLOCK_BYTES; i += 256) {
        const int o = ob * FP8_BLOCK + i / FP8_BLOCK, k = b * FP8_BLOCK + i % FP8_BLOCK;
        codes[(size_t)blockIdx.x * FP8_BLOCK_BYTES + i] = o < Nout && k < Nin ? src[(size_t)o * ldw + k] : 0;
    }
    if (threadIdx.x == 0) scales[blockIdx.x] = src_scales[blockIdx.x];
    fp8_publish();
}

__global__ void __launch_bounds__(256) k_fp8_unpack_weights(const unsigned char *__restrict__ codes, const float *__restrict__ scales, float *__restrict__ w,
                                                            int Nin, int Nout, int kb)
{
    const int b = blockIdx.x % kb, ob = blockIdx.x / kb;
    const float s = scales[blockIdx.x];
    for (int i = threadIdx.x; i < FP8_BLOCK_BYTES; i += 256) {
        const int k = b * FP8_BLOCK + i / FP8_BLOCK, o = ob * FP8_BLOCK + i % FP8_BLOCK;
        if (k < Nin && o < Nout)
            w[(size_t)k * Nout + o] = fp8_decode(codes[(size_t)blockIdx.x * FP8_BLOCK_BYTES + (size_t)(i % FP8_BLOCK) * FP8_BLOCK + i / FP8_BLOCK]) * s;
    }
}

/* ------------------------------------------------------------------ host side */
struct dRk_Fp8FcPlan {
    int dev;
    unsigned char *q;                   /* rounded input and its scales, in the caller's scratch */
    float *sx;
    Fp8Params p;
    Fp8Tensor t;
};

static int fp8_type_size(int type) { return type == DRK_F32 ? 4 : type == DRK_BF16 || type == DRK_F16 ? 2 : 0; }

static int fp8_refuse(const char *who, const char *why)
{
    fprintf(stderr, "%s: %s\n", who, why);
    return -1;
}

/* block numbers are grid indices and rows of a tensor map: both fit 31 bits */
extern "C" int dRk_fp8_fc_supported(int n, int Nin, int Nout)
{
    if (n < 1 || Nin < 1 || Nout < 1) return 0;
    const size_t wb = (size_t)fp8_blocks(Nin) * fp8_blocks(Nout), xr = (size_t)fp8_blocks(Nin) * n;
    return wb * FP8_BLOCK < (1ull << 31) && xr < (1ull << 31) && (size_t)fp8_blocks(n) * 2 * fp8_blocks(Nout) * 2 < (1ull << 31);
}

extern "C" size_t dRk_fp8_fc_packed_bytes(int Nin, int Nout)
{
    if (!dRk_fp8_fc_supported(1, Nin, Nout)) return 0;
    return (size_t)fp8_blocks(Nin) * fp8_blocks(Nout) * (FP8_BLOCK_BYTES + sizeof(float));
}

extern "C" size_t dRk_fp8_fc_scratch_bytes(int n, int Nin, int Nout)
{
    if (!dRk_fp8_fc_supported(n, Nin, Nout)) return 0;
    return (size_t)fp8_blocks(Nin) * n * (FP8_BLOCK + sizeof(float));
}

static int fp8_pack_checks(const char *who, const void *src, const void *packed, int Nin, int Nout)
{
    if (!src || !packed) return fp8_refuse(who, "null pointer");
    if (!dRk_fp8_fc_supported(1, Nin, Nout)) return fp8_refuse(who, "sizes outside the supported range");
    if ((uintptr_t)packed % 16) return fp8_refuse(who, "the packed weights must start on a 16-byte boundary");
    return 0;
}

extern "C" int dRk_fp8_fc_pack_weights(dRk_stream stream, const float *w, void *packed, int Nin, int Nout)
{
    const char *who = "dRk_fp8_fc_pack_weights";
    if (fp8_pack_checks(who, w, packed, Nin, Nout)) return -1;
    const int dev = drk_stream_device(who, stream, -1);
    if (dev < 0) return dev;
    const int kb = fp8_blocks(Nin), blocks = kb * fp8_blocks(Nout);
    unsigned char *codes = (unsigned char *)packed;
    k_fp8_pack_weights<<<blocks, 256, 0, drk_stream(stream)>>>(w, codes, (float *)(codes + (size_t)blocks * FP8_BLOCK_BYTES), Nin, Nout, kb);
    return drk_launched(cudaGetLastError());
}

extern "C" int dRk_fp8_fc_pack_codes(dRk_stream stream, const unsigned char *src, long long ldw, const float *scales, void *packed, int Nin, int Nout)
{
    const char *who = "dRk_fp8_fc_pack_codes";
    if (fp8_pack_checks(who, src, packed, Nin, Nout)) return -1;
    if (!scales) return fp8_refuse(who, "null pointer");
    if (ldw < Nin) return fp8_refuse(who, "rows of codes overlap (ldw < Nin)");
    const int dev = drk_stream_device(who, stream, -1);
    if (dev < 0) return dev;
    const int kb = fp8_blocks(Nin), blocks = kb * fp8_blocks(Nout);
    unsigned char *codes = (unsigned char *)packed;
    k_fp8_pack_codes<<<blocks, 256, 0, drk_stream(stream)>>>(src, (size_t)ldw, scales, codes, (float *)(codes + (size_t)blocks * FP8_BLOCK_BYTES), Nin, Nout, kb);
    return drk_launched(cudaGetLastError());
}

extern "C" int dRk_fp8_fc_unpack_weights(dRk_stream stream, const void *packed, float *w, int Nin, int Nout)
{
    const char *who = "dRk_fp8_fc_unpack_weights";
    if (fp8_pack_checks(who, w, packed, Nin, Nout)) return -1;
    const int dev = drk_stream_device(who, stream, -1);
    if (dev < 0) return dev;
    const int kb = fp8_blocks(Nin), blocks = kb * fp8_blocks(Nout);
    const unsigned char *codes = (const unsigned char *)packed;
    k_fp8_unpack_weights<<<blocks, 256, 0, drk_stream(stream)>>>(codes, (const float *)(codes + (size_t)blocks * FP8_BLOCK_BYTES), w, Nin, Nout, kb);
    return drk_launched(cudaGetLastError());
}

extern "C" dRk_Fp8FcPlan *dRk_fp8_fc_plan(const void *in, int in_type, long long ldi, const void *packed, const float *bias, void *out, int out_type,
                                          long long ldo, void *scratch, int n, int Nin, int Nout, int act, int *status)
{
    const char *who = "dRk_fp8_fc_plan";
    const int isz = fp8_type_size(in_type), osz = fp8_type_size(out_type);
    if (!in || !packed || !out || !scratch) { fp8_refuse(who, "null pointer"); return NULL; }
    if (!isz || !osz) { fp8_refuse(who, "unknown element type"); return NULL; }
    if (!dRk_fp8_fc_supported(n, Nin, Nout)) { fp8_refuse(who, "sizes outside the supported range"); return NULL; }
    if (n > 1 && (ldi < Nin || ldo < Nout)) { fp8_refuse(who, "rows overlap (ldi < Nin or ldo < Nout)"); return NULL; }
    if (ldi < 0 || ldo < 0) { fp8_refuse(who, "negative row pitch"); return NULL; }
    if (act != 0 && act != 1) { fp8_refuse(who, "activation must be 0 (linear) or 1 (ReLU)"); return NULL; }
    if ((uintptr_t)in % isz || (uintptr_t)out % osz || (uintptr_t)bias % 4) { fp8_refuse(who, "pointer not aligned to its element type"); return NULL; }
    if ((uintptr_t)packed % 16 || (uintptr_t)scratch % 16) { fp8_refuse(who, "packed weights and scratch must start on a 16-byte boundary"); return NULL; }
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) { (void)cudaGetLastError(); fp8_refuse(who, "no CUDA device"); return NULL; }
    dRk_Fp8FcPlan *p = (dRk_Fp8FcPlan *)calloc(1, sizeof(*p));
    if (!p) { fp8_refuse(who, "out of host memory"); return NULL; }
    p->dev = dev;
    p->p.in = in;
    p->p.ldi = (size_t)ldi;
    p->p.in_type = in_type;
    p->p.Nin = Nin;
    p->p.vec = (uintptr_t)in % 16 == 0 && (n == 1 || (size_t)ldi * isz % 16 == 0);
    const int kb = fp8_blocks(Nin), ob = fp8_blocks(Nout);
    const unsigned char *codes = (const unsigned char *)packed;
    p->q = (unsigned char *)scratch;
    p->sx = (float *)(p->q + (size_t)kb * n * FP8_BLOCK);
    p->p.sx = p->sx;
    p->p.scales = (const float *)(codes + (size_t)kb * ob * FP8_BLOCK_BYTES);
    p->p.bias = bias;
    p->p.out = out;
    p->p.ldo = (size_t)ldo;
    p->p.out_type = out_type;
    p->p.n = n; p->p.Nout = Nout; p->p.kb = kb; p->p.ob = ob; p->p.act = act;
    p->p.status = status;
    int sms = 148;
    if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || drk_fp8_tensor_plan(&p->t, &p->p, codes, p->q, sms)) {
        (void)cudaGetLastError();
        fp8_refuse(who, "tensor maps could not be made");
        free(p);
        return NULL;
    }
    return p;
}

template <typename T> static int fp8_quantize(const dRk_Fp8FcPlan *p, cudaStream_t st)
{
    /* many: more blocks than half warps find a place for (eight CTAs on an SM) */
    const size_t blocks = (size_t)p->p.n * p->p.kb;
    const bool many = blocks > 16 * 148 * 8;
    if (sizeof(T) == 4 && many && !p->p.vec)
        return drk_launched(drk_launch_dep(k_fp8_quantize_unaligned, dim3(drk_blocks(blocks, 8, 148u * 8u)), dim3(256), 0, st, (const float *)p->p.in, p->p.ldi, p->q,
                                           p->sx, p->p.n, p->p.Nin, p->p.kb));
    return drk_launched(drk_launch_dep(many ? k_fp8_quantize_rows<T, 2> : k_fp8_quantize_rows<T, 1>, dim3(drk_blocks(blocks, many ? 32 : 16, 148u * 8u)), dim3(256), 0, st,
                                       (const T *)p->p.in, p->p.ldi, p->q, p->sx, p->p.n, p->p.Nin, p->p.kb, p->p.vec));
}

extern "C" int dRk_fp8_fc_run(dRk_stream stream, dRk_Fp8FcPlan *p)
{
    if (!p) return fp8_refuse("dRk_fp8_fc_run", "no plan");
    const int dev = drk_stream_device("dRk_fp8_fc_run", stream, p->dev);
    if (dev < 0) return dev;
    cudaStream_t st = drk_stream(stream);
    if (!p->t.fuse) {
        const int type = p->p.in_type, rc = type == DRK_F32 ? fp8_quantize<float>(p, st) : type == DRK_BF16 ? fp8_quantize<__nv_bfloat16>(p, st) : fp8_quantize<__half>(p, st);
        if (rc) return rc;
    }
    return drk_fp8_tensor_launch(st, &p->t, &p->p);
}

extern "C" void dRk_fp8_fc_free(dRk_Fp8FcPlan *p) { free(p); }
