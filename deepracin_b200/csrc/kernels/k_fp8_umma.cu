/*
 * Products of the 8-bit fully connected layer on the tensor cores: tcgen05.mma kind::f8f6f4 (e4m3 x e4m3, FP32 accumulate).
 *
 * A float scale per block of 128 inputs means that the tensor core may sum no further than one block: its accumulator is read
 * back after every 128 inputs (four MMAs of K = 32), multiplied by sx * sw and added to the running sum in registers.
 */
#include <stdlib.h>
#include <string.h>
#include <type_traits>
#include "k_fp8.cuh"
#include "k_umma.cuh"

__device__ __forceinline__ void umma_f8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
/* instruction descriptor: D = F32, A = B = e4m3, both K-major, M = m, N = n */
__host__ __device__ constexpr uint32_t make_idesc_f8(int m, int n) { return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24); }

/* One statement loads and waits: with a wait of its own that names the registers as its operands, the compiler copied them, and
 * k_fp8_pair's additions took three times as long. */
__device__ __forceinline__ void tmem_ld_wait(uint32_t taddr, uint32_t (&r)[16])
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 "
                 "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
                 "tcgen05.wait::ld.sync.aligned;"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_ld_wait(uint32_t taddr, uint32_t (&r)[32])
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
                 "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
                 "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\t"
                 "tcgen05.wait::ld.sync.aligned;"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
                   "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
                   "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_ld_wait(uint32_t taddr, uint32_t (&r)[64])
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x64.b32 "
                 "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
                 "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, "
                 "%32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, "
                 "%48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%64];\n\t"
                 "tcgen05.wait::ld.sync.aligned;"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
                   "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
                   "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]),
                   "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]),
                   "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]),
                   "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]),
                   "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
                 : "r"(taddr) : "memory");
}
/* Loads ahead of their use.  They stay where they are written (the compiler would move plain ones down to the use), and callers
 * clamp addresses instead of skipping a load, and use a register again instead of handing its value on: a copy of a loaded value
 * waits for the load, be it at the end of a branch or of a loop's pass.  ld_ahead is for what this launch or the one in front
 * writes, ld_const for weights' scales. */
__device__ __forceinline__ float ld_ahead(const float *p)
{
    float v;
    asm volatile("ld.global.cg.f32 %0, [%1];" : "=f"(v) : "l"(p));
    return v;
}
__device__ __forceinline__ float ld_const(const float *p)
{
    float v;
    asm volatile("ld.global.nc.f32 %0, [%1];" : "=f"(v) : "l"(p));
    return v;
}
/* two FP32 FMAs in one instruction */
__device__ __forceinline__ void ffma2(unsigned long long &acc, unsigned long long a, uint32_t b0, uint32_t b1)
{
    asm("{\n\t.reg .b64 b;\n\tmov.b64 b, {%2, %3};\n\tfma.rn.f32x2 %0, %1, b, %0;\n\t}" : "+l"(acc) : "l"(a), "r"(b0), "r"(b1));
}
__device__ __forceinline__ bool elect_one()
{
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one != 0;
}
/* whether a phase is over, without waiting for it (try_wait suspends the thread for a while) */
__device__ __forceinline__ uint32_t mbar_test(uint32_t bar, uint32_t parity)
{
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok;
}
__device__ __forceinline__ uint32_t cluster_rank() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ void cluster_sync()
{
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait()
{
    __syncwarp();
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
/* where saddr lies in the shared memory of the cluster's CTA `rank` */
__device__ __forceinline__ uint32_t cluster_addr(uint32_t saddr, uint32_t rank)
{
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(saddr), "r"(rank));
    return a;
}
__device__ __forceinline__ void st_cluster(uint32_t cluster_addr, float v)
{
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(cluster_addr), "f"(v) : "memory");
}

/* a wait of a whole warp that holds many registers: no call inside, which would have them saved around it */
__device__ __forceinline__ bool mbar_wait_warp_inline(uint32_t bar, uint32_t parity, volatile int *abort_flag, int *status, int code)
{
    bool ok = mbar_try(bar, parity);
    if (!__all_sync(0xffffffffu, ok)) {
        const long long t0 = clock64();
        while (!ok && !*abort_flag) {
            ok = mbar_try(bar, parity);
            if (!ok && clock64() - t0 > WAIT_CYCLES) {
                *abort_flag = 1;
                if (status) atomicExch(status, code);
            }
        }
    }
    return __all_sync(0xffffffffu, ok);
}

/* the same for one thread */
__device__ __forceinline__ bool mbar_wait1(uint32_t bar, uint32_t parity, volatile int *abort_flag, int *status, int code)
{
    if (mbar_try(bar, parity)) return true;     /* reading the clock costs as much as half an MMA: not on this way */
    const long long t0 = clock64();
    while (!mbar_try(bar, parity)) {
        if (*abort_flag) return false;
        if (clock64() - t0 > WAIT_CYCLES) { *abort_flag = 1; if (status) atomicExch(status, code); return false; }
    }
    return true;
}
/*
 * Few rows: the weights are on the M side (a packed block of 128 outputs x 128 inputs per stage, the only large operand), NT
 * rows of the input on the N side.  A cluster of `split` CTAs shares the K blocks of one tile; each sends its sums of a row to
 * the CTA that owns the row (distributed shared memory), which adds them in the order of the ranks.  Warp 0 issues TMA, warp 1
 * the MMAs; two groups of four warps own the 128 outputs, one per lane, and add the blocks times sx * sw to NT sums each, taking
 * turns (what a block costs them beside the additions -- the wait, the factors -- is 350 of 600 clocks); with NT = 128 each has
 * half of the rows instead.  A block's accumulator is one of SLOTS in TMEM.  The weights do not depend on the launch in front:
 * their first blocks are on the way before it ends.
 *
 * Bound by the weights' way from HBM behind 4 us of launch, first loads and exchange: 1 x 25088 -> 4096 fp32 19.8 us (15.7 at the
 * copy rate), 1 x 4096 -> 4096 6.1 us (2.6); with 64 rows by the sums of a block too, and the rounding's launch: 64 x 25088 -> 4096
 * 24.5 us (16.8), 64 x 4096 -> 1000 7.8 us; with NT = 128 by the sums, 0.6 us a block, and 5 us of start and end, where code runs
 * once and costs its way from the L2 (4000 x 256 -> 256 bf16: 8.0 us with the rounding, 15.7 us when an unsplit tile's results
 * went through the inbox row by row).
 *
 * FUSE (the bytes of an input value; at most FUSE_ROWS rows): four more warps round the input themselves, a block each in turn,
 * straight into the swizzled operand tile; what takes two launches takes one.
 */
#define FUSE_ROWS 4
template <int NT, int FUSE> struct SwapCfg {
    static constexpr int B_BYTES = NT * FP8_BLOCK;
    static constexpr int STAGE_BYTES = FP8_BLOCK_BYTES + B_BYTES;
    static constexpr int STAGES = NT == 16 ? 10 : NT == 32 ? 9 : NT == 64 ? 6 : 4;       /* at most: fewer for a short share */
    static constexpr int SLOTS = NT <= 64 ? 4 : 2;
    static constexpr int TMEM_COLS = SLOTS * NT;
    static constexpr int GROUPS = NT <= 64 ? 2 : 1;             /* of summing warps that take turns */
    static constexpr int COLS = GROUPS == 2 ? NT : NT / 2;      /* sums per lane */
    static constexpr int THREADS = 32 * (2 + 8 + (FUSE ? 4 : 0));
    /* factors: a pair of slots per summing warp, or, written by the rounding warps, one per block that is under way: a stage is
       filled again when its MMAs are done, and those wait for the accumulator of SLOTS blocks before */
    static constexpr int RING = STAGES + SLOTS, FACTORS = FUSE ? RING * NT : 8 * 2 * COLS;
    static constexpr int INBOX = GROUPS * NT * FP8_BLOCK;       /* floats: sums of the rows this CTA owns, from every group of every CTA */
    static constexpr int smem(int stages) { return 1024 + stages * STAGE_BYTES + INBOX * 4 + FACTORS * 4 + 256; }
};

__device__ __forceinline__ float2 fp8_two(uint32_t w, int type)
{
    return type == DRK_BF16 ? make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)) : __half22float2(*reinterpret_cast<const __half2 *>(&w));
}
/* four values of a row from k on, zero behind Nin */
__device__ __forceinline__ float4 fp8_load4(const Fp8Params &p, int r, int k)
{
    float e[4];
    const size_t at = (size_t)r * p.ldi + k;
#pragma unroll
    for (int j = 0; j < 4; j++)
        e[j] = k + j >= p.Nin        ? 0.0f
               : p.in_type == DRK_F32  ? static_cast<const float *>(p.in)[at + j]
               : p.in_type == DRK_BF16 ? __bfloat162float(static_cast<const __nv_bfloat16 *>(p.in)[at + j])
                                       : __half2float(static_cast<const __half *>(p.in)[at + j]);
    return make_float4(e[0], e[1], e[2], e[3]);
}

template <int NT, int FUSE>
__global__ void __launch_bounds__((SwapCfg<NT, FUSE>::THREADS), 1)
k_fp8_swap(const __grid_constant__ CUtensorMap mapW, const __grid_constant__ CUtensorMap mapX, const __grid_constant__ Fp8Params p, int split, int stages)
{
    using C = SwapCfg<NT, FUSE>;
    extern __shared__ char smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    char *gen = smem_raw + (base - smem_u32(smem_raw));
    float *inbox = reinterpret_cast<float *>(gen + stages * C::STAGE_BYTES);
    float *factors = inbox + C::INBOX;
    char *tail = reinterpret_cast<char *>(factors + C::FACTORS);
    const uint32_t bars = smem_u32(tail);
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(tail + 8 * (2 * C::STAGES + 2 * C::SLOTS + 1));
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    auto full_bar = [&](int s) { return bars + 8u * s; };
    auto empty_bar = [&](int s) { return bars + 8u * (C::STAGES + s); };
    auto tfull_bar = [&](int a) { return bars + 8u * (2 * C::STAGES + a); };
    auto tempty_bar = [&](int a) { return bars + 8u * (2 * C::STAGES + C::SLOTS + a); };
    const uint32_t drain_bar = bars + 8u * (2 * C::STAGES + 2 * C::SLOTS);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    const int tile = blockIdx.x / split, rank = blockIdx.x - tile * split;
    const int ot = tile % p.ob, r0 = (tile / p.ob) * NT;
    const int b0 = (int)((long long)p.kb * rank / split), b1 = (int)((long long)p.kb * (rank + 1) / split);
    constexpr uint32_t TX = FUSE ? FP8_BLOCK_BYTES : C::STAGE_BYTES;
    if (split > 1) cluster_arrive();    /* waited for before the first store into another CTA: it runs by then */
    int pre = 0;        /* blocks whose weights are on the way before the launch in front has ended */

    if (threadIdx.x == 0) {
        for (int s = 0; s < C::STAGES; s++) { mbar_init(full_bar(s), FUSE ? 2 : 1); mbar_init(empty_bar(s), 1); }
        for (int a = 0; a < C::SLOTS; a++) { mbar_init(tfull_bar(a), 1); mbar_init(tempty_bar(a), 8 / C::GROUPS); }
        mbar_init(drain_bar, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;\n\tfence.proxy.async.shared::cta;" ::: "memory");
        for (; pre < stages && b0 + pre < b1; pre++) {
            mbar_expect_tx(full_bar(pre), TX);
            tma_load_2d(base + pre * C::STAGE_BYTES, &mapW, 0, (ot * p.kb + b0 + pre) * FP8_BLOCK, full_bar(pre));
        }
    }
    /* No TMEM before the launch in front has ended: its CTAs may still ask for theirs on this SM, and would wait for ours */
    if (warp == 1) {
        drk_dep_wait();
        tmem_alloc(smem_u32(tmem_slot), C::TMEM_COLS);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    float acc[C::COLS];
#pragma unroll
    for (int j = 0; j < C::COLS; j++) acc[j] = 0.0f;

    if (warp == 0) {
        if (lane == 0) {
            drk_dep_wait();
            int stage = 0, issued = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int b = b0; b < b1; b++) {
                const uint32_t sw = base + stage * C::STAGE_BYTES;
                if (issued >= pre) {
                    if (!mbar_wait1(empty_bar(stage), phase ^ 1u, abort_flag, p.status, 31)) { ok = false; break; }
                    mbar_expect_tx(full_bar(stage), TX);
                    tma_load_2d(sw, &mapW, 0, (ot * p.kb + b) * FP8_BLOCK, full_bar(stage));
                }
                if (!FUSE) tma_load_2d(sw + FP8_BLOCK_BYTES, &mapX, 0, b * p.n + r0, full_bar(stage));
                issued++;
                if (++stage == stages) { stage = 0; phase ^= 1u; }
            }
            if (!ok) {      /* no copy may land after the exit */
                const int pending = issued < stages ? issued : stages;
                for (int i = 0; i < pending; i++) {
                    if (--stage < 0) { stage = stages - 1; phase ^= 1u; }
                    const long long t0 = clock64();
                    while (!mbar_try(full_bar(stage), phase) && clock64() - t0 < WAIT_CYCLES) { }
                }
            }
        }
    } else if (warp == 1) {
        constexpr uint32_t idesc = make_idesc_f8(128, NT);
        int stage = 0, slot = 0;
        uint32_t phase = 0, sphase = 0;
        bool ok = true;
        for (int b = b0; b < b1; b++) {
            const bool full = mbar_try(full_bar(stage), phase), room = mbar_try(tempty_bar(slot), sphase ^ 1u);
            if (!__all_sync(0xffffffffu, full && room) &&
                (!mbar_wait_warp_inline(full_bar(stage), phase, abort_flag, p.status, 33) ||
                 !mbar_wait_warp_inline(tempty_bar(slot), sphase ^ 1u, abort_flag, p.status, 32))) { ok = false; break; }
            tc_fence_after();
            if (elect_one()) {
                const uint32_t sw = base + stage * C::STAGE_BYTES;
                const uint64_t adesc = make_smem_desc(sw), bdesc = make_smem_desc(sw + FP8_BLOCK_BYTES);
#pragma unroll
                for (int j = 0; j < 4; j++)     /* 32 inputs each, 32 bytes further inside the swizzled row */
                    umma_f8(tmem_base + (uint32_t)(slot * NT), adesc + (uint64_t)(j * 2), bdesc + (uint64_t)(j * 2), idesc, j ? 1u : 0u);
                umma_commit(empty_bar(stage));
                umma_commit(tfull_bar(slot));
            }
            __syncwarp();
            if (++stage == stages) { stage = 0; phase ^= 1u; }
            if (++slot == C::SLOTS) { slot = 0; sphase ^= 1u; }
        }
        if (!ok && elect_one()) umma_drain(drain_bar);
        __syncwarp();
    } else if (warp < 10) {
        const int quarter = warp & 3, part = (warp - 2) >> 2, c0 = C::GROUPS == 2 ? 0 : part * C::COLS;
        float *mine = factors + (warp - 2) * 2 * C::COLS;
        constexpr int PER = (C::COLS + 31) / 32;
        const float *swp = p.scales + (size_t)ot * p.kb;
        drk_dep_wait();     /* sx is written by the launch in front; the rows in p.out may still be read by it */
        const int first = b0 + (C::GROUPS == 2 ? part : 0), last = b1 - 1;      /* this group's first block */
        /* factors of this group's block and of its next one; rows behind the last stand for the last (they are not stored) */
        const float *sxp[PER];
        float x[PER], x1[PER], sw = 0.0f, sw1 = 0.0f;
        auto fetch = [&](int b, float (&to)[PER]) {
#pragma unroll
            for (int j = 0; j < PER; j++) to[j] = ld_ahead(sxp[j] + (size_t)min(b, last) * p.n);
            return ld_const(swp + min(b, last));
        };
        if (!FUSE) {
#pragma unroll
            for (int j = 0; j < PER; j++) sxp[j] = p.sx + min(r0 + c0 + j * 32 + lane, p.n - 1);
            sw = fetch(first, x);
            sw1 = fetch(first + C::GROUPS, x1);
        }
        int slot = C::GROUPS == 2 ? part : 0, flip = 0;
        uint32_t sphase = 0;
        for (int b = first; b < b1; b += C::GROUPS) {
            const float *f = factors + ((b - b0) % C::RING) * NT + c0;
            if (!FUSE) {
                float *g = mine + flip * C::COLS;
#pragma unroll
                for (int j = 0; j < PER; j++) if (j * 32 + lane < C::COLS) g[j * 32 + lane] = x[j] * sw;
                __syncwarp();
                f = g;
                flip ^= 1;
            }
            if (!mbar_wait_warp_inline(tfull_bar(slot), sphase, abort_flag, p.status, 34)) break;
            tc_fence_after();
            const uint32_t taddr = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(slot * NT + c0);
            constexpr int STEP = C::COLS < 32 ? 16 : 32;
#pragma unroll
            for (int c = 0; c < C::COLS; c += STEP) {
                uint32_t r[STEP];
                tmem_ld_wait(taddr + (uint32_t)c, r);
                if (c + STEP >= C::COLS) {      /* the accumulator is in registers */
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(tempty_bar(slot));
                }
#pragma unroll
                for (int j = 0; j < STEP; j += 4) {
                    const float4 g = *reinterpret_cast<const float4 *>(f + c + j);
                    acc[c + j] = fmaf(g.x, __uint_as_float(r[j]), acc[c + j]);
                    acc[c + j + 1] = fmaf(g.y, __uint_as_float(r[j + 1]), acc[c + j + 1]);
                    acc[c + j + 2] = fmaf(g.z, __uint_as_float(r[j + 2]), acc[c + j + 2]);
                    acc[c + j + 3] = fmaf(g.w, __uint_as_float(r[j + 3]), acc[c + j + 3]);
                }
            }
            if (!FUSE) {
#pragma unroll
                for (int j = 0; j < PER; j++) x[j] = x1[j];
                sw = sw1;
                sw1 = fetch(b + 2 * C::GROUPS, x1);
            }
            slot += C::GROUPS;
            if (slot >= C::SLOTS) { slot -= C::SLOTS; sphase ^= 1u; }
        }
    } else if (FUSE) {
        /* warp w rounds the blocks w, w + 4, ...: a row's 128 values are four per lane */
        using Raw = typename std::conditional<FUSE == 4, uint4, uint2>::type;
        const float *swp = p.scales + (size_t)ot * p.kb;
        const int first = b0 + warp - 10, last = b1 - 1;
        drk_dep_wait();
        auto rounding = [&](auto fast) {
            constexpr bool FAST = decltype(fast)::value;    /* whole vectors: the next block's are on their way while one is rounded */
            const char *row[FUSE_ROWS] = {};
            Raw raw[FUSE_ROWS];
            float sw = 0.0f;
            auto fetch = [&](int b, int r) {
                const char *at = row[r] + (size_t)min(min(b, last) * FP8_BLOCK + lane * 4, p.Nin - 4) * FUSE;
                if constexpr (FUSE == 4) asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(raw[r].x), "=r"(raw[r].y), "=r"(raw[r].z), "=r"(raw[r].w) : "l"(at));
                else asm volatile("ld.global.v2.u32 {%0, %1}, [%2];" : "=r"(raw[r].x), "=r"(raw[r].y) : "l"(at));
            };
            if (FAST) {
#pragma unroll
                for (int r = 0; r < FUSE_ROWS; r++) { row[r] = static_cast<const char *>(p.in) + (size_t)min(r, p.n - 1) * p.ldi * FUSE; fetch(first, r); }
            }
            sw = ld_const(swp + min(first, last));
            for (int b = first; b < b1; b += 4) {
                const int i = b - b0, stage = i % stages;
                if (i >= stages && !mbar_wait_warp_inline(empty_bar(stage), ((uint32_t)(i / stages) & 1u) ^ 1u, abort_flag, p.status, 35)) break;
                char *tile_x = gen + stage * C::STAGE_BYTES + FP8_BLOCK_BYTES;
                float *f = factors + (i % C::RING) * NT;
#pragma unroll
                for (int r = 0; r < FUSE_ROWS; r++) {
                    float4 v;
                    if constexpr (FAST) {
                        if constexpr (FUSE == 4) v = make_float4(__uint_as_float(raw[r].x), __uint_as_float(raw[r].y), __uint_as_float(raw[r].z), __uint_as_float(raw[r].w));
                        else {
                            const float2 lo = fp8_two(raw[r].x, p.in_type), hi = fp8_two(raw[r].y, p.in_type);
                            v = make_float4(lo.x, lo.y, hi.x, hi.y);
                        }
                        if (b * FP8_BLOCK + lane * 4 >= p.Nin) v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        fetch(b + 4, r);
                    }
                    if (r >= p.n) continue;
                    if constexpr (!FAST) v = fp8_load4(p, r, b * FP8_BLOCK + lane * 4);
                    float a = fmaxf(fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))), FP8_FLOOR);
                    a = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(a)));      /* positive floats compare as whole numbers */
                    const float inv = __fdiv_rn(FP8_MAX, a);
                    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(v.x * inv, v.y * inv), __NV_SATFINITE, __NV_E4M3);
                    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(v.z * inv, v.w * inv), __NV_SATFINITE, __NV_E4M3);
                    *reinterpret_cast<uint32_t *>(tile_x + r * FP8_BLOCK + ((((lane >> 2) ^ (r & 7)) << 4) | ((lane & 3) << 2))) = lo | (hi << 16);
                    if (lane == 0) f[r] = __fdiv_rn(a, FP8_MAX) * sw;
                }
                sw = ld_const(swp + min(b + 4, last));
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(full_bar(stage));
            }
        };
        if (p.vec && p.Nin % 4 == 0) rounding(std::true_type{});
        else rounding(std::false_type{});
    }
    drk_dep_trigger();

    tc_fence_before();
    __syncthreads();
    if (split > 1) cluster_wait();
    /* row j of the tile belongs to CTA j % split, a power of two of up to eight; inbox [source][row / split][128 outputs] */
    const bool summing = warp >= 2 && warp < 10;
    const int part = (warp - 2) >> 2, ol = (warp & 3) * 32 + lane, o = ot * FP8_BLOCK + ol;
    const int c0 = C::GROUPS == 2 ? 0 : part * C::COLS, lg = 31 - __clz(split), own = NT >> lg, sources = C::GROUPS * split;
    const float bias = summing && p.bias && o < p.Nout ? __ldg(p.bias + o) : 0.0f;
    /* one source: its sums are the result */
    const bool alone = C::GROUPS == 1 && split == 1;
    if (summing && alone && o < p.Nout) {
        auto put = [&](auto *out) {
            out += (size_t)(r0 + c0) * p.ldo + o;
            const int left = p.n - r0 - c0;
#pragma unroll
            for (int j = 0; j < C::COLS; j++) {
                if (j < left) *out = fp8_store<std::remove_pointer_t<decltype(out)>>(fp8_act(acc[j] + bias, p.act));
                out += p.ldo;
            }
        };
        if (p.out_type == DRK_F32) put(static_cast<float *>(p.out));
        else if (p.out_type == DRK_BF16) put(static_cast<__nv_bfloat16 *>(p.out));
        else put(static_cast<__half *>(p.out));
    }
    if (summing && !alone) {
        const uint32_t to = smem_u32(inbox + (C::GROUPS * rank + (C::GROUPS == 2 ? part : 0)) * own * FP8_BLOCK + ol);
        if (NT == 16) {         /* row by row, as there may be one */
#pragma unroll
            for (int j = 0; j < C::COLS; j++) {
                if (r0 + j >= p.n) break;
                st_cluster(cluster_addr(to + (uint32_t)(j >> lg) * (FP8_BLOCK * 4), (uint32_t)(j & (split - 1))), acc[j]);
            }
        } else {                /* eight addresses that move on together: what runs once is paid by its length */
            uint32_t at[8];
#pragma unroll
            for (int k = 0; k < 8; k++) at[k] = cluster_addr(to + (uint32_t)((c0 + k) >> lg) * (FP8_BLOCK * 4), (uint32_t)(k & (split - 1)));
            const uint32_t step = (uint32_t)(8 >> lg) * (FP8_BLOCK * 4);
#pragma unroll
            for (int j0 = 0; j0 < C::COLS; j0 += 8) {
                if (r0 + c0 + j0 >= p.n) break;
#pragma unroll
                for (int k = 0; k < 8; k++) { st_cluster(at[k], acc[j0 + k]); at[k] += step; }
            }
        }
    }
    __syncwarp();
    if (split > 1) cluster_arrive();
    if (warp == 1) tmem_dealloc(tmem_base, C::TMEM_COLS);
    if (split > 1) cluster_wait();
    else __syncthreads();
    constexpr int ROWS = NT == 16 ? 1 : 4;
    /* rows in fours, whose reads and stores do not wait for one another; up to 16 rows one by one (1 x 4096 -> 4096: 6.1 instead of 6.4 us) */
    if (summing && !alone && o < p.Nout)
        for (int q0 = part; q0 < own && r0 + q0 * split + rank < p.n; q0 += 2 * ROWS) {
            float sum[ROWS];
#pragma unroll
            for (int u = 0; u < ROWS; u++) sum[u] = 0.0f;
            for (int s = 0; s < sources; s++)
#pragma unroll
                for (int u = 0; u < ROWS; u++) sum[u] += inbox[(s * own + min(q0 + 2 * u, own - 1)) * FP8_BLOCK + ol];
            size_t at[ROWS];
            bool here[ROWS];
#pragma unroll
            for (int u = 0; u < ROWS; u++) {
                const int q = q0 + 2 * u, r = r0 + q * split + rank;
                here[u] = q < own && r < p.n;
                at[u] = (size_t)r * p.ldo + o;
                sum[u] = fp8_act(sum[u] + bias, p.act);
            }
            if (p.out_type == DRK_F32) {
#pragma unroll
                for (int u = 0; u < ROWS; u++) if (here[u]) static_cast<float *>(p.out)[at[u]] = sum[u];
            } else if (p.out_type == DRK_BF16) {
#pragma unroll
                for (int u = 0; u < ROWS; u++) if (here[u]) static_cast<__nv_bfloat16 *>(p.out)[at[u]] = fp8_store<__nv_bfloat16>(sum[u]);
            } else {
#pragma unroll
                for (int u = 0; u < ROWS; u++) if (here[u]) static_cast<__half *>(p.out)[at[u]] = fp8_store<__half>(sum[u]);
            }
        }
}

/*
 * Many rows: a pair of CTAs (cta_group::2) computes 256 rows x 256 outputs, persistent over the tiles.  Per 128 inputs each CTA
 * fetches its 128 rows of the input and 64 rows of each of the tile's two weight blocks (32 KiB a stage; a single CTA's tile of
 * 128 x 256 would fetch 48), counted on the leader's barriers.  Two warps of the leader issue, one for each weight block (M = 256,
 * N = 128, four MMAs of K = 32), into one of two accumulators per block; the commits tell both CTAs.  Warps 4-11 own 32 rows and
 * one weight block each: they read the accumulator, hand its slot back, and add it times sx * sw to 128 sums per lane.  Warp 3
 * makes the factors sx * sw of a block and leaves them in shared memory.
 *
 * What bounds it: the way issue -> commit -> read -> hand back -> issue, 700 to 900 clocks a block with two accumulators under
 * way, where the MMAs take 512; 8 us of start (registers, TMEM, barriers of two CTAs, first loads: 3) and of a tile's results
 * (10000 clocks each when every chunk had code of its own, bank conflicts and its bias to wait for); in a long run the board's
 * power (half of it spent on copies and at rest, a third on the MMAs).  With the rounding of the input, 4096 x 8192 -> 8192 bf16:
 * 249 us alone, 292 us back to back (980 W, 1.43 GHz), copies and MMAs without the sums 207 us; 1000 x 4096 -> 4096 23.1 us.
 * Measured on the way there (back to back): factors read by the summing warps themselves 341 us (the instructions that ran once
 * in four blocks stalled each time, those of a loop unrolled by two or four missed the instruction cache: 384 us), scalar FMAs
 * 337 us, one issuing warp 328 us, sixteen summing warps 409 us, 8 row tiles walked together instead of 16 321 us, these against
 * 316 us; a cluster-scope release on the hand-back (a memory barrier) and registers copied after a separate wait cost 100 us and
 * more each, and so do a few registers more in the results' code (335 us: the sums are spilled), or sums staged in fours, which
 * wants them in aligned registers (338 us).
 */
struct PairCfg {
    static constexpr int STAGE_BYTES = 2 * FP8_BLOCK_BYTES;
    static constexpr int STAGES = 6;
    static constexpr int RING = 8;                              /* blocks whose factors are kept: STAGES + 2, see there */
    static constexpr int SMEM = 1024 + STAGES * STAGE_BYTES + 8 * 32 * 16 * 4 + RING * 256 * 4 + 8 * FP8_BLOCK * 4 + 256;
    static constexpr int GROUP = 16;                             /* row tiles that are walked together before the next outputs */
};

__device__ __forceinline__ void umma_f8_pair(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
/* both CTAs' barriers at this address are arrived at once all MMAs issued so far have completed */
__device__ __forceinline__ void umma_commit_pair(uint32_t bar)
{
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((uint16_t)3) : "memory");
}
/* a copy into this CTA's shared memory that is counted on a barrier of the pair's leader */
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap *map, int c0, int c1, uint32_t cluster_bar)
{
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(cluster_bar) : "memory");
}
__device__ __forceinline__ uint32_t leader_addr(uint32_t saddr) { uint32_t a; asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(saddr)); return a; }
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t cluster_bar)
{
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}

__global__ void __launch_bounds__(384, 1)
k_fp8_pair(const __grid_constant__ CUtensorMap mapW, const __grid_constant__ CUtensorMap mapX, const __grid_constant__ Fp8Params p, int mtiles, int ntiles)
{
    using C = PairCfg;
    extern __shared__ char smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    char *gen = smem_raw + (base - smem_u32(smem_raw));
    float *stage_out = reinterpret_cast<float *>(gen + C::STAGES * C::STAGE_BYTES);
    float *ring = stage_out + 8 * 32 * 16;          /* sx * sw [RING][weight block][128 rows] */
    float *bias_of = ring + C::RING * 256;          /* [summing warp][128 outputs] */
    char *tail = reinterpret_cast<char *>(bias_of + 8 * FP8_BLOCK);
    const uint32_t bars = smem_u32(tail);
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(tail + 8 * (2 * C::STAGES + 10));
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    auto full_bar = [&](int s) { return bars + 8u * s; };
    auto empty_bar = [&](int s) { return bars + 8u * (C::STAGES + s); };
    auto tfull_bar = [&](int a) { return bars + 8u * (2 * C::STAGES + a); };
    auto tempty_bar = [&](int a) { return bars + 8u * (2 * C::STAGES + 4 + a); };
    const uint32_t drain_bar = bars + 8u * (2 * C::STAGES + 8);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)cluster_rank();
    const bool leader = rank == 0;

    if (threadIdx.x == 0) {
        for (int s = 0; s < C::STAGES; s++) { mbar_init(full_bar(s), 3); mbar_init(empty_bar(s), 2); }
        for (int a = 0; a < 4; a++) { mbar_init(tfull_bar(a), 1); mbar_init(tempty_bar(a), 8); }
        for (int h = 0; h < 2; h++) mbar_init(drain_bar + 8u * h, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {    /* shared memory leaves no room for another CTA with TMEM on this SM: nobody waits for this one's */
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();     /* the partner's barriers are ready, and its TMEM */
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    const int tiles = mtiles * ntiles, pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    /* tile t -> row tile, output tile: GROUP row tiles by all output tiles at a time, so that the tiles in flight share both operands */
    auto place = [&](int t, int &mt, int &nt) {
        const int per = C::GROUP * ntiles, g = t / per, left = t - g * per;
        const int rows = min(C::GROUP, mtiles - g * C::GROUP);
        nt = left / rows;
        mt = g * C::GROUP + left - nt * rows;
    };

    /* registers: 384 threads x 168 at launch = 128 x 56 + 256 x 224 */
    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        if (warp == 0) {
            if (lane == 0) {
                const uint32_t leader_full = leader_addr(full_bar(0));
                int pre = 0, mt, nt;
                /* this CTA's 64 rows of the two weight blocks of a tile: the pair's MMA over N = 128 takes half of B from each CTA */
                auto load_w = [&](uint32_t dst, int ntile, int b, uint32_t bar) {
                    for (int h = 0; h < 2; h++)
                        tma_load_2d_pair(dst + h * (FP8_BLOCK_BYTES / 2), &mapW, 0,
                                         ((2 * ntile + h) * p.kb + b) * FP8_BLOCK + rank * 64, bar);
                };
                if (pair < tiles) {
                    place(pair, mt, nt);
                    for (; pre < C::STAGES && pre < p.kb; pre++) {      /* weights first, as in k_fp8_swap */
                        if (leader) mbar_expect_tx(full_bar(pre), 2 * C::STAGE_BYTES);
                        load_w(base + pre * C::STAGE_BYTES + FP8_BLOCK_BYTES, nt, pre, leader_full + 8u * pre);
                    }
                }
                drk_dep_wait();
                int stage = 0;
                uint32_t phase = 0;
                long long issued = 0;
                bool ok = true;
                for (int t = pair; t < tiles && ok; t += pairs) {
                    place(t, mt, nt);
                    for (int b = 0; b < p.kb; b++) {
                        const uint32_t sa = base + stage * C::STAGE_BYTES, bar = leader_full + 8u * stage;
                        if (issued >= pre) {
                            if (!mbar_wait1(empty_bar(stage), phase ^ 1u, abort_flag, p.status, 41)) { ok = false; break; }
                            if (leader) mbar_expect_tx(full_bar(stage), 2 * C::STAGE_BYTES);
                            load_w(sa + FP8_BLOCK_BYTES, nt, b, bar);
                        }
                        tma_load_2d_pair(sa, &mapX, 0, b * p.n + mt * 256 + rank * 128, bar);
                        issued++;
                        if (++stage == C::STAGES) { stage = 0; phase ^= 1u; }
                    }
                }
                if (!ok && leader) {        /* no copy may land after the exit: the leader's barriers count both CTAs' */
                    const long long pending = issued < C::STAGES ? issued : C::STAGES;
                    for (long long i = 0; i < pending; i++) {
                        if (--stage < 0) { stage = C::STAGES - 1; phase ^= 1u; }
                        const long long t0 = clock64();
                        while (!mbar_try(full_bar(stage), phase) && clock64() - t0 < WAIT_CYCLES) { }
                    }
                }
            }
        } else if (warp < 3 && leader) {
            /* Two issuers, one for each weight block of a tile: what one spends on its two waits, the other's MMAs cover.  The whole
               warp walks the loop and one elected lane issues, so that the descriptors live in uniform registers. */
            constexpr uint32_t idesc = make_idesc_f8(256, 128);
            const int h = warp - 1;
            int stage = 0, slot = 0;
            uint32_t phase = 0, sphase = 0;
            bool ok = true;
            for (int t = pair; t < tiles && ok; t += pairs)
                for (int b = 0; b < p.kb; b++) {
                    const bool full = mbar_try(full_bar(stage), phase), room = mbar_try(tempty_bar(2 * h + slot), sphase ^ 1u);
                    if (!__all_sync(0xffffffffu, full && room) &&
                        (!mbar_wait_warp_inline(full_bar(stage), phase, abort_flag, p.status, 43) ||
                         !mbar_wait_warp_inline(tempty_bar(2 * h + slot), sphase ^ 1u, abort_flag, p.status, 42))) { ok = false; break; }
                    tc_fence_after();
                    if (elect_one()) {
                        const uint32_t sa = base + stage * C::STAGE_BYTES;
                        const uint64_t adesc = make_smem_desc(sa), bdesc = make_smem_desc(sa + FP8_BLOCK_BYTES + h * (FP8_BLOCK_BYTES / 2));
#pragma unroll
                        for (int j = 0; j < 4; j++)
                            umma_f8_pair(tmem_base + (uint32_t)(slot * 256 + h * 128), adesc + (uint64_t)(j * 2), bdesc + (uint64_t)(j * 2), idesc, j ? 1u : 0u);
                        umma_commit_pair(tfull_bar(2 * h + slot));
                        umma_commit_pair(empty_bar(stage));
                    }
                    __syncwarp();
                    if (++stage == C::STAGES) { stage = 0; phase ^= 1u; }
                    slot ^= 1;
                    if (!slot) sphase ^= 1u;
                }
            if (!ok && elect_one()) {       /* what was issued may still run */
                asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(drain_bar + 8u * h) : "memory");
                const long long t0 = clock64();
                while (!mbar_try(drain_bar + 8u * h, 0) && clock64() - t0 < WAIT_CYCLES) { }
            }
        } else if (warp == 3) {
            /* The factors of a block, for the summing warps: on the leader's barrier of the block's stage like its operands, so that the
               accumulator is there only after them.  A ring's slot is free when the stage is: its MMAs waited for the accumulator
               of two blocks before, which was read after the factors. */
            const uint32_t leader_full = leader_addr(full_bar(0));
            int stage = 0, slot = 0;
            uint32_t phase = 0;
            bool ok = true;
            drk_dep_wait();
            for (int t = pair; t < tiles && ok; t += pairs) {
                int mt, nt;
                place(t, mt, nt);
                const int last = p.kb - 1;
                const float *sw0 = p.scales + (size_t)(2 * nt) * p.kb, *sw1 = sw0 + (2 * nt + 1 < p.ob ? p.kb : 0);
                const float *sx[4];
#pragma unroll
                for (int q = 0; q < 4; q++) sx[q] = p.sx + min(mt * 256 + rank * 128 + q * 32 + lane, p.n - 1);
                float x[2][4], w0[2], w1[2];
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const int b = min(u, last);
#pragma unroll
                    for (int q = 0; q < 4; q++) x[u][q] = ld_ahead(sx[q] + (size_t)b * p.n);
                    w0[u] = ld_const(sw0 + b);
                    w1[u] = ld_const(sw1 + b);
                }
                for (int b4 = 0; b4 < p.kb && ok; b4 += 2)
#pragma unroll
                    for (int u = 0; u < 2; u++) {
                        if (b4 + u >= p.kb) break;
                        if (!mbar_wait_warp_inline(empty_bar(stage), phase ^ 1u, abort_flag, p.status, 45)) { ok = false; break; }
                        float *f = ring + slot * 256 + lane;
#pragma unroll
                        for (int q = 0; q < 4; q++) { f[q * 32] = x[u][q] * w0[u]; f[128 + q * 32] = x[u][q] * w1[u]; }
                        __syncwarp();
                        if (lane == 0) mbar_arrive_cluster(leader_full + 8u * stage);
                        const int b = min(b4 + u + 2, last);
#pragma unroll
                        for (int q = 0; q < 4; q++) x[u][q] = ld_ahead(sx[q] + (size_t)b * p.n);
                        w0[u] = ld_const(sw0 + b);
                        w1[u] = ld_const(sw1 + b);
                        if (++stage == C::STAGES) { stage = 0; phase ^= 1u; }
                        if (++slot == C::RING) slot = 0;
                    }
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
        const int quarter = warp & 3, half = (warp - 4) >> 2;       /* this warp's rows and its weight block of the tile's two */
        const uint32_t lane_base = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(half * 128);
        const uint32_t tempty0 = leader_addr(tempty_bar(0));
        float *stg = stage_out + (warp - 4) * 32 * 16;
        float4 *bias128 = reinterpret_cast<float4 *>(bias_of + (warp - 4) * FP8_BLOCK);
        const float *factor = ring + half * 128 + quarter * 32 + lane;
        const int osize = p.out_type == DRK_F32 ? 4 : 2;
        const bool vec = (reinterpret_cast<uintptr_t>(p.out) % 16 == 0) && (p.ldo * osize % 16 == 0);
        /* an accumulator is in registers: its slot may be written again */
        auto release = [&](int a) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(tempty0 + 8u * a);
        };
        /* this lane's four of the bias of a tile's outputs: asked for while the tile in front is written */
        auto bias4 = [&](int t) {
            int mt, nt;
            place(t, mt, nt);
            const int o = (2 * nt + half) * FP8_BLOCK + lane * 4;
            float b[4];
#pragma unroll
            for (int e = 0; e < 4; e++) b[e] = p.bias && o + e < p.Nout ? __ldg(p.bias + o + e) : 0.0f;
            return make_float4(b[0], b[1], b[2], b[3]);
        };
        if (pair < tiles) bias128[lane] = bias4(pair);
        drk_dep_wait();
        int slot = 0, at_ring = 0;
        uint32_t sphase = 0;
        bool ok = true;
        for (int t = pair; t < tiles && ok; t += pairs) {
            int mt, nt;
            place(t, mt, nt);
            const int row0 = mt * 256 + rank * 128 + quarter * 32;
            const int ot = 2 * nt + half;
            unsigned long long acc[64];
#pragma unroll
            for (int j = 0; j < 64; j++) acc[j] = 0ull;
            uint32_t ready = mbar_test(tfull_bar(2 * half + slot), sphase);
            for (int b = 0; b < p.kb; b++) {
                const uint32_t at = lane_base + (uint32_t)(slot * 256), a = 2 * half + slot;
                if (!__all_sync(0xffffffffu, ready) && !mbar_wait_warp_inline(tfull_bar(a), sphase, abort_flag, p.status, 44)) { ok = false; break; }
                tc_fence_after();
                const float f = factor[at_ring];
                unsigned long long ff;
                asm("mov.b64 %0, {%1, %1};" : "=l"(ff) : "f"(f));
                at_ring = (at_ring + 256) & (C::RING * 256 - 1);
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    uint32_t r[64];
                    tmem_ld_wait(at + 64u * c, r);
                    if (c == 1) {
                        release(a);
                        slot ^= 1;
                        if (!slot) sphase ^= 1u;
                        ready = mbar_test(tfull_bar(2 * half + slot), sphase);
                    }
#pragma unroll
                    for (int j = 0; j < 64; j += 2) ffma2(acc[32 * c + j / 2], ff, r[j], r[j + 1]);
                }
            }
            if (!ok) break;
            /* 32 rows x 16 outputs at a time through shared memory, the eight pairs of a row exchanged by its number so that
               neither side meets a bank twice; four lanes then store a row's run.  A loop, as code that runs once a tile costs its
               way from the L2. */
            const int cl = (lane & 3) * 4, o0 = ot * FP8_BLOCK + cl;
            auto stage16 = [&](auto chunk) {
#pragma unroll
                for (int j = 0; j < 8; j++)
                    reinterpret_cast<unsigned long long *>(stg)[lane * 8 + (j ^ (lane >> 1 & 7))] = acc[decltype(chunk)::value * 8 + j];
            };
            /* 16-bit results are rounded first and leave 32 outputs at a time */
            auto out16 = [&](auto two) {
                using W = decltype(two);
                auto stage32 = [&](auto chunk) {
                    constexpr int c = decltype(chunk)::value;
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const float4 b = bias128[c * 8 + j];
                        const unsigned long long lo = acc[c * 16 + 2 * j], hi = acc[c * 16 + 2 * j + 1];
                        const W w0 = fp8_store2<W>(fp8_act(__uint_as_float((uint32_t)lo) + b.x, p.act), fp8_act(__uint_as_float((uint32_t)(lo >> 32)) + b.y, p.act));
                        const W w1 = fp8_store2<W>(fp8_act(__uint_as_float((uint32_t)hi) + b.z, p.act), fp8_act(__uint_as_float((uint32_t)(hi >> 32)) + b.w, p.act));
                        reinterpret_cast<uint2 *>(stg)[lane * 8 + (j ^ (lane >> 1 & 7))] = make_uint2(reinterpret_cast<const uint32_t &>(w0), reinterpret_cast<const uint32_t &>(w1));
                    }
                };
                const int left = p.n - row0 - (lane >> 2);
                char *to = static_cast<char *>(p.out) + ((size_t)(row0 + (lane >> 2)) * p.ldo + ot * FP8_BLOCK + (lane & 3) * 8) * 2;
                const size_t down = (size_t)p.ldo * 16;
#pragma unroll 1
                for (int c = 0; c < 4; c++, to += 64) {
                    __syncwarp();
                    if (c == 0) stage32(std::integral_constant<int, 0>{});
                    else if (c == 1) stage32(std::integral_constant<int, 1>{});
                    else if (c == 2) stage32(std::integral_constant<int, 2>{});
                    else stage32(std::integral_constant<int, 3>{});
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int rr = i * 8 + (lane >> 2);
                        uint4 w = reinterpret_cast<const uint4 *>(stg)[rr * 4 + ((lane & 3) ^ (rr >> 2 & 3))];
                        if (rr >> 1 & 1) w = make_uint4(w.z, w.w, w.x, w.y);
                        if (i * 8 < left) *reinterpret_cast<uint4 *>(to + i * down) = w;
                    }
                }
            };
            const float4 next_bias = bias4(min(t + pairs, tiles - 1));
            if (vec && p.out_type != DRK_F32 && (ot + 1) * FP8_BLOCK <= p.Nout) {
                if (p.out_type == DRK_BF16) out16(__nv_bfloat162());
                else out16(__half2());
            } else
#pragma unroll 1
            for (int c = 0; c < 8; c++) {
                const int o = o0 + c * 16;
                __syncwarp();
                switch (c) {
                case 0: stage16(std::integral_constant<int, 0>{}); break;
                case 1: stage16(std::integral_constant<int, 1>{}); break;
                case 2: stage16(std::integral_constant<int, 2>{}); break;
                case 3: stage16(std::integral_constant<int, 3>{}); break;
                case 4: stage16(std::integral_constant<int, 4>{}); break;
                case 5: stage16(std::integral_constant<int, 5>{}); break;
                case 6: stage16(std::integral_constant<int, 6>{}); break;
                default: stage16(std::integral_constant<int, 7>{}); break;
                }
                __syncwarp();
                if (!vec || ot * FP8_BLOCK + c * 16 + 16 > p.Nout) {     /* two rows of sixteen at a time (459 x 128 -> 13522 fp16: 17.6 us, 37 us in single values of four lanes' runs) */
                    const int col = lane & 15, oc = ot * FP8_BLOCK + c * 16 + col;
                    const float b = reinterpret_cast<const float *>(bias128)[c * 16 + col];
                    char *to = static_cast<char *>(p.out) + ((size_t)(row0 + (lane >> 4)) * p.ldo + oc) * osize;
                    int rr = lane >> 4;
                    if (oc < p.Nout)
#pragma unroll 4
                    for (; rr < min(32, p.n - row0); rr += 2) {
                        const float w = fp8_act(stg[rr * 16 + ((col >> 1) ^ (rr >> 1 & 7)) * 2 + (col & 1)] + b, p.act);
                        if (p.out_type == DRK_F32) *reinterpret_cast<float *>(to) = w;
                        else if (p.out_type == DRK_BF16) *reinterpret_cast<__nv_bfloat16 *>(to) = fp8_store<__nv_bfloat16>(w);
                        else *reinterpret_cast<__half *>(to) = fp8_store<__half>(w);
                        to += (size_t)p.ldo * 2 * osize;
                    }
                    continue;
                }
                const float4 bias = bias128[c * 4 + (lane & 3)];
                float v[4][4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int rr = i * 8 + (lane >> 2);
                    float4 w = reinterpret_cast<const float4 *>(stg)[rr * 4 + ((lane & 3) ^ (rr >> 2 & 3))];
                    if (rr >> 1 & 1) w = make_float4(w.z, w.w, w.x, w.y);
                    v[i][0] = fp8_act(w.x + bias.x, p.act); v[i][1] = fp8_act(w.y + bias.y, p.act);
                    v[i][2] = fp8_act(w.z + bias.z, p.act); v[i][3] = fp8_act(w.w + bias.w, p.act);
                }
                const int left = p.n - row0 - (lane >> 2);      /* rows i * 8 below it exist */
                const size_t at0 = (size_t)(row0 + (lane >> 2)) * p.ldo + o;
                if (p.out_type == DRK_F32) {
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (i * 8 < left) *reinterpret_cast<float4 *>(static_cast<float *>(p.out) + at0 + (size_t)(i * 8) * p.ldo) = make_float4(v[i][0], v[i][1], v[i][2], v[i][3]);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        uint2 w;
                        if (p.out_type == DRK_BF16) {
                            const __nv_bfloat162 lo = __floats2bfloat162_rn(v[i][0], v[i][1]), hi = __floats2bfloat162_rn(v[i][2], v[i][3]);
                            w = make_uint2(*reinterpret_cast<const uint32_t *>(&lo), *reinterpret_cast<const uint32_t *>(&hi));
                        } else {
                            const __half2 lo = __floats2half2_rn(v[i][0], v[i][1]), hi = __floats2half2_rn(v[i][2], v[i][3]);
                            w = make_uint2(*reinterpret_cast<const uint32_t *>(&lo), *reinterpret_cast<const uint32_t *>(&hi));
                        }
                        if (i * 8 < left) *reinterpret_cast<uint2 *>(static_cast<char *>(p.out) + (at0 + (size_t)(i * 8) * p.ldo) * 2) = w;
                    }
                }
            }
            __syncwarp();
            bias128[lane] = next_bias;
        }
    }
    drk_dep_trigger();

    tc_fence_before();
    __syncthreads();
    cluster_sync();     /* neither CTA leaves while the other may still signal it or multiply into its TMEM */
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512) : "memory");
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

/* how many clusters of `split` CTAs that have an SM to themselves run at once: fewer than sms / split, as a cluster stays inside one
 * of the GPU's groups of SMs (33 of four, 15 of eight) */
static int swap_clusters(int split, int sms)
{
    if (split == 1) return sms;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)split);
    cfg.blockDim = dim3(SwapCfg<16, 0>::THREADS);
    cfg.dynamicSmemBytes = SwapCfg<16, 0>::smem(SwapCfg<16, 0>::STAGES);
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)split;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaFuncSetAttribute(k_fp8_swap<16, 0>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)cfg.dynamicSmemBytes) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&n, k_fp8_swap<16, 0>, &cfg) != cudaSuccess) {
        (void)cudaGetLastError();
        return sms / split * 3 / 4;
    }
    return n < sms / split ? n : sms / split;
}

/* shares of a tile's blocks in k_fp8_swap<nt>: as many as still run at once, one on an SM (64 x 4096 -> 2304: 18 clusters of eight,
 * of which 15 fit, 14.3 us, of four 9.3 us); returns the rounds */
static long long swap_split(Fp8Tensor *t, const Fp8Params *p, int nt, int sms)
{
    const long long tiles = (long long)p->ob * ((p->n + nt - 1) / nt);
    int at_once = sms;
    t->nt = nt;
    t->split = 1;
    while (t->split < 8 && t->split * 4 <= p->kb && tiles * t->split * 2 <= sms) {
        const int clusters = swap_clusters(t->split * 2, sms);
        if (tiles > clusters) break;
        t->split *= 2;
        at_once = clusters;
    }
    t->stages = (p->kb + t->split - 1) / t->split;
    return (tiles + at_once - 1) / at_once;
}

int drk_fp8_tensor_plan(Fp8Tensor *t, const Fp8Params *p, const void *codes, const void *q, int sms)
{
    t->mtiles = (p->n + 255) / 256;
    t->ntiles = (p->ob + 1) / 2;
    t->pairs = 0;
    if (p->n <= 64) swap_split(t, p, p->n <= 16 ? 16 : p->n <= 32 ? 32 : 64, sms);
    else {
        /* In units of 0.05 us a block of 128 inputs takes a CTA of k_fp8_swap<64> 5, one of k_fp8_swap<128> 9, and a pair of
           k_fp8_pair, on four times the latter's tile, 8; a round adds 30, 16 and 20, and the pair starts 10 later (fitted on 399
           shapes, 0.5 % worse than the best of the three in each.  In this order, 4096 -> 3200: 17.7, 22.5 and 20.7 us for 300
           rows; 18560 -> 1792: 31.0, 45.0 and 61.4; 4096 -> 7680, 700 rows: 74.0, 59.6 and 36.5). */
        const long long ptiles = (long long)t->mtiles * t->ntiles, prounds = (ptiles + sms / 2 - 1) / (sms / 2);
        long long rounds = swap_split(t, p, 64, sms);
        const long long cost64 = rounds * (5 * t->stages + 30);
        rounds = swap_split(t, p, 128, sms);
        const long long cost128 = rounds * (9 * t->stages + 16), paired = prounds * (8 * p->kb + 20) + 10;
        if (paired <= cost128 && paired <= cost64) t->pairs = (int)(ptiles < sms / 2 ? ptiles : sms / 2);
        else if (cost64 < cost128) swap_split(t, p, 64, sms);
    }
    /* rounding inside the product's kernel costs nothing while its four warps keep up with the weights: 16-bit rows, one row, or a
       short share (25088 -> 4096, fp32: one row 19.8 against 22.2 us, two rows 23.8 against 22.4; 4096 -> 4096, four rows 7.6
       against 8.2) */
    t->fuse = !t->pairs && p->n <= FUSE_ROWS && (p->in_type != DRK_F32 || p->n == 1 || p->n * t->stages <= 64);
    /* the attribute holds for the current device, which is the plan's */
    const cudaFuncAttribute dyn = cudaFuncAttributeMaxDynamicSharedMemorySize;
    const cudaError_t e = t->pairs      ? cudaFuncSetAttribute(k_fp8_pair, dyn, PairCfg::SMEM)
                          : t->fuse     ? (p->in_type == DRK_F32 ? cudaFuncSetAttribute(k_fp8_swap<16, 4>, dyn, SwapCfg<16, 4>::smem(SwapCfg<16, 4>::STAGES))
                                                                 : cudaFuncSetAttribute(k_fp8_swap<16, 2>, dyn, SwapCfg<16, 2>::smem(SwapCfg<16, 2>::STAGES)))
                          : t->nt == 16 ? cudaFuncSetAttribute(k_fp8_swap<16, 0>, dyn, SwapCfg<16, 0>::smem(SwapCfg<16, 0>::STAGES))
                          : t->nt == 32 ? cudaFuncSetAttribute(k_fp8_swap<32, 0>, dyn, SwapCfg<32, 0>::smem(SwapCfg<32, 0>::STAGES))
                          : t->nt == 64 ? cudaFuncSetAttribute(k_fp8_swap<64, 0>, dyn, SwapCfg<64, 0>::smem(SwapCfg<64, 0>::STAGES))
                                        : cudaFuncSetAttribute(k_fp8_swap<128, 0>, dyn, SwapCfg<128, 0>::smem(SwapCfg<128, 0>::STAGES));
    if (e != cudaSuccess) return -1;
    if (encode_rows(&t->mapW, codes, (size_t)p->ob * p->kb * FP8_BLOCK, t->pairs ? 64 : FP8_BLOCK)) return -1;
    return encode_rows(&t->mapX, q, (size_t)p->kb * p->n, t->nt);
}

template <typename... KArgs, typename... Args>
static int cluster_launch(void (*kernel)(KArgs...), unsigned grid, unsigned block, unsigned cluster, size_t smem, cudaStream_t st, Args &&...args)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = drk_dep_launch_enabled() ? 2 : 1;
    return drk_launched(cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...));
}

template <int NT, int FUSE> static int swap_launch(cudaStream_t st, const Fp8Tensor *t, const Fp8Params *p)
{
    using C = SwapCfg<NT, FUSE>;
    const int stages = t->stages > C::STAGES ? C::STAGES : t->stages;
    return cluster_launch(k_fp8_swap<NT, FUSE>, (unsigned)(p->ob * ((p->n + NT - 1) / NT) * t->split), C::THREADS, t->split, C::smem(stages), st, t->mapW,
                          t->mapX, *p, t->split, stages);
}

int drk_fp8_tensor_launch(cudaStream_t st, const Fp8Tensor *t, const Fp8Params *p)
{
    if (t->pairs) return cluster_launch(k_fp8_pair, 2u * t->pairs, 384, 2, PairCfg::SMEM, st, t->mapW, t->mapX, *p, t->mtiles, t->ntiles);
    if (t->fuse) return (p->in_type == DRK_F32 ? swap_launch<16, 4>(st, t, p) : swap_launch<16, 2>(st, t, p));
    return t->nt == 16   ? swap_launch<16, 0>(st, t, p)
           : t->nt == 32 ? swap_launch<32, 0>(st, t, p)
           : t->nt == 64 ? swap_launch<64, 0>(st, t, p)
                         : swap_launch<128, 0>(st, t, p);
}
