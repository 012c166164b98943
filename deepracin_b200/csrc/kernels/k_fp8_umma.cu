/*
 * Products of the 8-bit fully connected layer on the tensor cores: tcgen05.mma kind::f8f6f4 (e4m3 x e4m3, FP32 accumulate).
 *
 * A float scale per block of 128 inputs means that the tensor core may sum no further than one block: its accumulator is read
 * back after every 128 inputs (four MMAs of K = 32), multiplied by sx * sw and added to the running sum in registers.
 */
#include <stdlib.h>
#include <string.h>
#include "k_fp8.cuh"
#include "k_umma.cuh"

__device__ __forceinline__ void umma_f8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
/* instruction descriptor: D = F32, A = B = e4m3, both K-major, M = m, N = n */
__host__ __device__ constexpr uint32_t make_idesc_f8(int m, int n) { return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24); }

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16])
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 "
                 "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(taddr) : "memory");
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
/* two FP32 FMAs in one instruction */
__device__ __forceinline__ void ffma2(unsigned long long &acc, unsigned long long a, uint32_t b0, uint32_t b1)
{
    asm("{\n\t.reg .b64 b;\n\tmov.b64 b, {%2, %3};\n\tfma.rn.f32x2 %0, %1, b, %0;\n\t}" : "+l"(acc) : "l"(a), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t cluster_rank() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ void cluster_sync()
{
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float ld_cluster(uint32_t saddr, uint32_t rank)
{
    float v;
    asm volatile("{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %1, %2;\n\tld.shared::cluster.f32 %0, [a];\n\t}" : "=f"(v) : "r"(saddr), "r"(rank) : "memory");
    return v;
}
__device__ __forceinline__ void fp8_put(const Fp8Params &p, size_t r, int o, float v)
{
    v = fp8_act(v, p.act);
    const size_t at = r * p.ldo + o;
    if (p.out_type == DRK_F32) static_cast<float *>(p.out)[at] = v;
    else if (p.out_type == DRK_BF16) static_cast<__nv_bfloat16 *>(p.out)[at] = fp8_store<__nv_bfloat16>(v);
    else static_cast<__half *>(p.out)[at] = fp8_store<__half>(v);
}

/*
 * Few rows: the weights are on the M side (a packed block of 128 outputs x 128 inputs per stage, the only large operand), NT
 * rows of the input on the N side.  A cluster of `split` CTAs shares the K blocks of one tile and adds its sums through
 * distributed shared memory, in the order of the ranks.  Warp 0 issues TMA, warp 1 the MMAs, warps 2-5 own the 128 outputs (one
 * per lane) and hold NT running sums each; block i's accumulator is one of SLOTS in TMEM.
 */
template <int NT> struct SwapCfg {
    static constexpr int B_BYTES = NT * FP8_BLOCK;
    static constexpr int STAGE_BYTES = FP8_BLOCK_BYTES + B_BYTES;
    static constexpr int STAGES = NT == 16 ? 6 : NT == 32 ? 5 : NT == 64 ? 4 : 6;
    static constexpr int SLOTS = NT <= 64 ? 4 : 2;
    static constexpr int TMEM_COLS = SLOTS * NT < 32 ? 32 : SLOTS * NT;
    static constexpr int CTAS = NT <= 64 ? 2 : 1;               /* resident per SM */
    static constexpr int SMEM = 1024 + STAGES * STAGE_BYTES + 4 * 2 * NT * 4 + 256;
};

template <int NT>
__global__ void __launch_bounds__(192, SwapCfg<NT>::CTAS)
k_fp8_swap(const __grid_constant__ CUtensorMap mapW, const __grid_constant__ CUtensorMap mapX, const Fp8Params p, int split)
{
    using C = SwapCfg<NT>;
    extern __shared__ char smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    char *gen = smem_raw + (base - smem_u32(smem_raw));
    float *factors = reinterpret_cast<float *>(gen + C::STAGES * C::STAGE_BYTES);       /* [4 warps][2][NT] */
    char *tail = reinterpret_cast<char *>(factors + 4 * 2 * NT);
    const uint32_t bars = smem_u32(tail);
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(tail + 8 * (2 * C::STAGES + 2 * C::SLOTS + 1));
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    auto full_bar = [&](int s) { return bars + 8u * s; };
    auto empty_bar = [&](int s) { return bars + 8u * (C::STAGES + s); };
    auto tfull_bar = [&](int a) { return bars + 8u * (2 * C::STAGES + a); };
    auto tempty_bar = [&](int a) { return bars + 8u * (2 * C::STAGES + C::SLOTS + a); };
    const uint32_t drain_bar = bars + 8u * (2 * C::STAGES + 2 * C::SLOTS);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int s = 0; s < C::STAGES; s++) { mbar_init(full_bar(s), 1); mbar_init(empty_bar(s), 1); }
        for (int a = 0; a < C::SLOTS; a++) { mbar_init(tfull_bar(a), 1); mbar_init(tempty_bar(a), 4); }
        mbar_init(drain_bar, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) tmem_alloc(smem_u32(tmem_slot), C::TMEM_COLS);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    const int tile = blockIdx.x / split, rank = blockIdx.x - tile * split;
    const int ot = tile % p.ob, r0 = (tile / p.ob) * NT;
    const int b0 = (int)((long long)p.kb * rank / split), b1 = (int)((long long)p.kb * (rank + 1) / split);
    unsigned long long acc[NT / 2];
#pragma unroll
    for (int j = 0; j < NT / 2; j++) acc[j] = 0ull;

    if (warp == 0) {
        if (lane == 0) {
            int pre = 0;
            /* weights do not depend on the launch in front (the rounding of the input): the first blocks are on their way before it ends */
            for (; pre < C::STAGES && b0 + pre < b1; pre++) {
                mbar_expect_tx(full_bar(pre), C::STAGE_BYTES);
                tma_load_2d(base + pre * C::STAGE_BYTES, &mapW, 0, (ot * p.kb + b0 + pre) * FP8_BLOCK, full_bar(pre));
            }
            drk_dep_wait();
            int stage = 0, issued = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int b = b0; b < b1; b++) {
                const uint32_t sw = base + stage * C::STAGE_BYTES;
                if (issued >= pre) {
                    if (!mbar_wait(empty_bar(stage), phase ^ 1u, abort_flag, p.status, 31)) { ok = false; break; }
                    mbar_expect_tx(full_bar(stage), C::STAGE_BYTES);
                    tma_load_2d(sw, &mapW, 0, (ot * p.kb + b) * FP8_BLOCK, full_bar(stage));
                }
                tma_load_2d(sw + FP8_BLOCK_BYTES, &mapX, 0, b * p.n + r0, full_bar(stage));
                issued++;
                if (++stage == C::STAGES) { stage = 0; phase ^= 1u; }
            }
            if (!ok) {      /* no copy may land after the exit */
                const int pending = issued < C::STAGES ? issued : C::STAGES;
                for (int i = 0; i < pending; i++) {
                    if (--stage < 0) { stage = C::STAGES - 1; phase ^= 1u; }
                    const long long t0 = clock64();
                    while (!mbar_try(full_bar(stage), phase) && clock64() - t0 < WAIT_CYCLES) { }
                }
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            constexpr uint32_t idesc = make_idesc_f8(128, NT);
            int stage = 0, slot = 0;
            uint32_t phase = 0, sphase = 0;
            bool ok = true;
            for (int b = b0; b < b1; b++) {
                if (!mbar_wait(tempty_bar(slot), sphase ^ 1u, abort_flag, p.status, 32) ||
                    !mbar_wait(full_bar(stage), phase, abort_flag, p.status, 33)) { ok = false; break; }
                tc_fence_after();
                const uint32_t sw = base + stage * C::STAGE_BYTES;
                const uint64_t adesc = make_smem_desc(sw), bdesc = make_smem_desc(sw + FP8_BLOCK_BYTES);
#pragma unroll
                for (int j = 0; j < 4; j++)     /* 32 inputs each, 32 bytes further inside the swizzled row */
                    umma_f8(tmem_base + (uint32_t)(slot * NT), adesc + (uint64_t)(j * 2), bdesc + (uint64_t)(j * 2), idesc, j ? 1u : 0u);
                umma_commit(empty_bar(stage));
                umma_commit(tfull_bar(slot));
                if (++stage == C::STAGES) { stage = 0; phase ^= 1u; }
                if (++slot == C::SLOTS) { slot = 0; sphase ^= 1u; }
            }
            if (!ok) umma_drain(drain_bar);
        }
    } else {
        const int quarter = warp & 3;
        float *mine = factors + quarter * 2 * NT;
        constexpr int PER = (NT + 31) / 32;
        float next[PER];
        drk_dep_wait();     /* sx is written by the launch in front */
        auto fetch = [&](int b) {
            const float s = __ldg(p.scales + (size_t)ot * p.kb + b);
#pragma unroll
            for (int j = 0; j < PER; j++) {
                const int r = j * 32 + lane;
                next[j] = r < NT && r0 + r < p.n ? __ldg(p.sx + (size_t)b * p.n + r0 + r) * s : 0.0f;
            }
        };
        if (b0 < b1) fetch(b0);
        int slot = 0, flip = 0;
        uint32_t sphase = 0;
        for (int b = b0; b < b1; b++) {
            float *f = mine + flip * NT;
#pragma unroll
            for (int j = 0; j < PER; j++) if (j * 32 + lane < NT) f[j * 32 + lane] = next[j];
            __syncwarp();
            if (b + 1 < b1) fetch(b + 1);
            if (!mbar_wait_warp(tfull_bar(slot), sphase, abort_flag, p.status, 34)) break;
            tc_fence_after();
            const uint32_t taddr = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(slot * NT);
#pragma unroll
            for (int c0 = 0; c0 < NT; c0 += 16) {
                uint32_t r[16];
                tmem_ld16(taddr + (uint32_t)c0, r);
#pragma unroll
                for (int j = 0; j < 16; j += 4) {
                    const ulonglong2 g = *reinterpret_cast<const ulonglong2 *>(f + c0 + j);
                    ffma2(acc[(c0 + j) / 2], g.x, r[j], r[j + 1]);
                    ffma2(acc[(c0 + j) / 2 + 1], g.y, r[j + 2], r[j + 3]);
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(tempty_bar(slot));
            flip ^= 1;
            if (++slot == C::SLOTS) { slot = 0; sphase ^= 1u; }
        }
    }
    drk_dep_trigger();

    /* every role is done: the stages hold the sums now, [NT rows][128 outputs] */
    tc_fence_before();
    __syncthreads();
    if (warp == 1) tmem_dealloc(tmem_base, C::TMEM_COLS);
    float *part = reinterpret_cast<float *>(gen);
    const int ol = (warp & 3) * 32 + lane, o = ot * FP8_BLOCK + ol;
    if (split == 1) {
        if (warp >= 2 && o < p.Nout) {
            const float bias = p.bias ? __ldg(p.bias + o) : 0.0f;
#pragma unroll
            for (int j = 0; j < NT; j++) {
                const float v = __uint_as_float((uint32_t)(j & 1 ? acc[j / 2] >> 32 : acc[j / 2]));
                if (r0 + j < p.n) fp8_put(p, (size_t)r0 + j, o, v + bias);
            }
        }
        return;
    }
    if (warp >= 2)
#pragma unroll
        for (int j = 0; j < NT; j++)
            if (r0 + j < p.n) part[j * FP8_BLOCK + ol] = __uint_as_float((uint32_t)(j & 1 ? acc[j / 2] >> 32 : acc[j / 2]));
    cluster_sync();
    if (warp >= 2) {
        const float bias = p.bias && o < p.Nout ? __ldg(p.bias + o) : 0.0f;
        for (int j = rank; j < NT && r0 + j < p.n; j += split) {
            const uint32_t at = smem_u32(part + j * FP8_BLOCK + ol);
            float v = 0.0f;
            for (int s = 0; s < split; s++) v += ld_cluster(at, (uint32_t)s);
            if (o < p.Nout) fp8_put(p, (size_t)r0 + j, o, v + bias);
        }
    }
    cluster_sync();     /* the other CTAs read this one's sums until here */
}

/* ------------------------------------------------------------------ host side */
typedef CUresult (*PFN_encodeTiled)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                                    const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

/* rows of 128 bytes back to back, fetched box_rows at a time into 128-byte-swizzled shared memory; rows behind the end read as zero */
static int encode_rows(CUtensorMap *map, const void *base, size_t rows, int box_rows)
{
    void *fn = NULL;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) {
        (void)cudaGetLastError();
        return -1;
    }
    const cuuint64_t dims[2] = {FP8_BLOCK, (cuuint64_t)rows}, strides[1] = {FP8_BLOCK};
    const cuuint32_t box[2] = {FP8_BLOCK, (cuuint32_t)box_rows}, es[2] = {1, 1};
    return ((PFN_encodeTiled)fn)(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                 CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS ? 0 : -1;
}

int drk_fp8_tensor_plan(Fp8Tensor *t, const Fp8Params *p, const void *codes, const void *q, int sms)
{
    t->nt = p->n <= 16 ? 16 : p->n <= 32 ? 32 : p->n <= 64 ? 64 : 128;
    const int tiles = p->ob * ((p->n + t->nt - 1) / t->nt);
    t->split = 1;
    while (t->split < 8 && tiles * t->split < sms && t->split * 4 <= p->kb) t->split *= 2;
    /* the attribute holds for the current device, which is the plan's */
    const cudaError_t e = t->nt == 16   ? cudaFuncSetAttribute(k_fp8_swap<16>, cudaFuncAttributeMaxDynamicSharedMemorySize, SwapCfg<16>::SMEM)
                          : t->nt == 32 ? cudaFuncSetAttribute(k_fp8_swap<32>, cudaFuncAttributeMaxDynamicSharedMemorySize, SwapCfg<32>::SMEM)
                          : t->nt == 64 ? cudaFuncSetAttribute(k_fp8_swap<64>, cudaFuncAttributeMaxDynamicSharedMemorySize, SwapCfg<64>::SMEM)
                                        : cudaFuncSetAttribute(k_fp8_swap<128>, cudaFuncAttributeMaxDynamicSharedMemorySize, SwapCfg<128>::SMEM);
    if (e != cudaSuccess) return -1;
    if (encode_rows(&t->mapW, codes, (size_t)p->ob * p->kb * FP8_BLOCK, FP8_BLOCK)) return -1;
    return encode_rows(&t->mapX, q, (size_t)p->kb * p->n, t->nt);
}

template <int NT> static int swap_launch(cudaStream_t st, const Fp8Tensor *t, const Fp8Params *p)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(p->ob * ((p->n + NT - 1) / NT) * t->split));
    cfg.blockDim = dim3(192);
    cfg.dynamicSmemBytes = SwapCfg<NT>::SMEM;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)t->split;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = drk_dep_launch_enabled() ? 2 : 1;
    return drk_launched(cudaLaunchKernelEx(&cfg, k_fp8_swap<NT>, t->mapW, t->mapX, *p, t->split));
}

int drk_fp8_tensor_launch(cudaStream_t st, const Fp8Tensor *t, const Fp8Params *p)
{
    return t->nt == 16 ? swap_launch<16>(st, t, p) : t->nt == 32 ? swap_launch<32>(st, t, p) : t->nt == 64 ? swap_launch<64>(st, t, p) : swap_launch<128>(st, t, p);
}
