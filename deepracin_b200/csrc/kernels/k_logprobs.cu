/*
 * Scoring of a network's outputs: for each row v of `len` logits at temperature 1 / s
 *
 *   lse = log sum_i exp(s v_i),  log p_i = s v_i - lse,  H = -sum_i p_i log p_i = log S - T / S
 *
 * with d_i = s (v_i - max v), e_i = exp(d_i), S = sum e_i, T = sum e_i d_i; the log probabilities of given labels, and the k
 * largest logits with their log probabilities.  The order of the alternatives is total: by value (NaN above everything), equal
 * ones by ascending index; a value and its index are compared as one 64-bit key, so results do not depend on any timing.
 *
 * One pass over the row: each thread holds a running maximum, S and T, rescaled when its maximum grows (d falls by D, so
 * S -> 2^-D S and T -> 2^-D (T - D S); exponents are kept in base 2), and writes down the maximum of every slot of its share.
 * The k-th largest of the maxima of 64 groups of threads bounds the k-th largest value from below, so only slots whose maximum
 * reaches it are read again (for 131072 normal logits and k = 20 about 30 of 2048 slots), and what reaches it is ranked by
 * counting.  Few rows are split over a cluster of CTAs, which join through distributed shared memory: one launch, no workspace.
 * A row that fits a warp's registers is taken by one warp (k_logprobs_short).
 *
 * Bound by HBM in 32 bits (2048 x 131072: 158 us without alternatives = 6.8 TB/s, 166 us with five, 175 us with twenty); in 16 bits
 * and in rows of some thousands by what the CTAs of an SM issue and wait for between two rows' loads (2048 x 131072 bf16: 88, 94
 * and 102 us, 82 us at the copy rate; 4096 x 8192 fp32: 28, 37 and 39 us, 20 us); below that by the chain of a launch, one round
 * of loads and the selection's barriers (1 x 131072 bf16: 4.3 and 8.0 us with twenty).  CTAs of 512 threads took 192 us for
 * 2048 x 131072.  Not kept: maxima of parts of four neighbouring threads, 64 contiguous bytes each (3 us saved at k = 5 in rows of
 * 8192, 2 us lost at k = 20); the second reading in batches of four loads (39.2 instead of 37.3 us for 4096 x 8192); prefetches
 * into the L2 for 32-bit rows (1 to 3 us slower); d as one FMA, x c - m c, saved nothing and left a row of one value off zero.
 */
#include <math.h>
#include <stdio.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "k_common.cuh"

#define LP_KMAX 32
#define LP_LN2 0.693147181f
#define LP_NT 256           /* threads of a CTA, four of which share an SM */
#define LP_SPLIT 8          /* CTAs that share a row at most */
#define LP_U 4              /* 16-byte loads a thread has under way, twice (the next batch is requested before this one is used) */
#define LP_SLOTS 16         /* parts of a thread's share whose maxima are kept */
#define LP_GROUPS 64
#define LP_CAND 1024        /* values and slots that a selection may look at; more: a narrower bound, then one pass per alternative */
#define LP_ITEMS 1024
#define LP_WU 8             /* 16-byte loads of a lane that a warp's row may take: 1024 values in 32 bits, 2048 in 16 */
#define LP_WNT 128          /* threads of a CTA whose warps have a row each */
#define LP_WCAND 288        /* values that a warp ranks */
#define LP_LOW (-200.0f)    /* 2^-200 is zero in 32 bits: exponents are not held below it, so that no 0 * inf appears */

struct LpParams {
    const void *logits;
    size_t ld;
    int len, m, k, split;
    float scale;
    const int *labels;
    float *logprob, *entropy, *top_logprob;
    int *top_index;
};

/* the larger one, NaN if either is */
__device__ __forceinline__ float lp_max_nan(float a, float b) { float r; asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }

/* a 16-byte load of each type; max2: the larger of packed values, last: the larger of what a word holds */
template <typename T> struct LpType;
template <> struct LpType<float> {
    static constexpr int V = 4;
    static constexpr uint32_t FILL = 0xff800000u;
    static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) { uint32_t r; asm("max.NaN.f32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b)); return r; }
    static __device__ __forceinline__ float last(uint32_t a) { return __uint_as_float(a); }
    static __device__ __forceinline__ float one(const float *p) { return *p; }
    static __device__ __forceinline__ void unpack(uint4 w, float *v)
    {
        v[0] = __uint_as_float(w.x); v[1] = __uint_as_float(w.y); v[2] = __uint_as_float(w.z); v[3] = __uint_as_float(w.w);
    }
};
template <> struct LpType<__nv_bfloat16> {
    static constexpr int V = 8;
    static constexpr uint32_t FILL = 0xff80ff80u;
    static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) { uint32_t r; asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b)); return r; }
    static __device__ __forceinline__ float last(uint32_t a) { return lp_max_nan(__uint_as_float(a << 16), __uint_as_float(a & 0xffff0000u)); }
    static __device__ __forceinline__ float one(const __nv_bfloat16 *p) { return __bfloat162float(*p); }
    static __device__ __forceinline__ void unpack(uint4 w, float *v)
    {
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int j = 0; j < 4; j++) { v[2 * j] = __uint_as_float(u[j] << 16); v[2 * j + 1] = __uint_as_float(u[j] & 0xffff0000u); }
    }
};
template <> struct LpType<__half> {
    static constexpr int V = 8;
    static constexpr uint32_t FILL = 0xfc00fc00u;
    static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) { uint32_t r; asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b)); return r; }
    static __device__ __forceinline__ float last(uint32_t a)
    {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&a));
        return lp_max_nan(f.x, f.y);
    }
    static __device__ __forceinline__ float one(const __half *p) { return __half2float(*p); }
    static __device__ __forceinline__ void unpack(uint4 w, float *v)
    {
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&u[j]));
            v[2 * j] = f.x; v[2 * j + 1] = f.y;
        }
    }
};

/* float -> uint32 with the order of the values: -inf lowest, +inf below the NaNs, which all map to one value; -0 equals +0.
 * 0 stands below every value: nothing there. */
__device__ __forceinline__ uint32_t lp_order(float v)
{
    const uint32_t u = __float_as_uint(v + 0.0f);
    if ((u & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float lp_value(uint32_t o) { return o == 0xffffffffu ? __uint_as_float(0x7fffffffu) : __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o); }
__device__ __forceinline__ unsigned long long lp_key(uint32_t order, uint32_t i) { return ((unsigned long long)order << 32) | (0xffffffffu - i); }
__device__ __forceinline__ float lp_exp2(float x) { float r; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x)); return r; }

/* stores into the shared memory of the cluster's CTA 0 */
__device__ __forceinline__ void lp_st_first(uint32_t saddr, float v)
{
    asm volatile("{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %0, 0;\n\tst.shared::cluster.f32 [a], %1;\n\t}" ::"r"(saddr), "f"(v) : "memory");
}
__device__ __forceinline__ void lp_st_first(uint32_t saddr, unsigned long long v)
{
    asm volatile("{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %0, 0;\n\tst.shared::cluster.u64 [a], %1;\n\t}" ::"r"(saddr), "l"(v) : "memory");
}
__device__ __forceinline__ void lp_cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void lp_cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

/* how many of n keys are larger */
__device__ __forceinline__ int lp_rank(const unsigned long long *keys, int n, unsigned long long key)
{
    int r = 0;
#pragma unroll 4
    for (int j = 0; j < n; j += 2) {
        const ulonglong2 y = *reinterpret_cast<const ulonglong2 *>(keys + j);
        r += (y.x > key) + (j + 1 < n && y.y > key);
    }
    return r;
}

/* S and T of a few values below the maximum m, two at a time; d is held above LP_LOW, NaN too */
template <bool PACKED> struct LpSums {
    const float m, c;
    float s0 = 0.0f, s1 = 0.0f, t0 = 0.0f, t1 = 0.0f;
    __device__ __forceinline__ LpSums(float m, float c) : m(m), c(c) {}
    __device__ __forceinline__ void add(float x0, float x1)
    {
        const float d0 = fmaxf((x0 - m) * c, LP_LOW), d1 = fmaxf((x1 - m) * c, LP_LOW);
        const float e0 = lp_exp2(d0), e1 = lp_exp2(d1);
        s0 += e0; s1 += e1;
        t0 = fmaf(e0, d0, t0); t1 = fmaf(e1, d1, t1);
    }
    __device__ __forceinline__ void join(float &S, float &T) const { S += s0 + s1; T += t0 + t1; }
};
/* the same operations on pairs of registers: 2048 x 131072 bf16 106 instead of 110 us; in 32 bits the pairs that the loads leave
 * cost more than they save (1000 x 32000: 33.6 instead of 30.8 us) */
template <> struct LpSums<true> {
    unsigned long long m, c, s = 0, t = 0;
    __device__ __forceinline__ LpSums(float m_, float c_)
    {
        asm("mov.b64 %0, {%1, %1};" : "=l"(m) : "f"(-m_));
        asm("mov.b64 %0, {%1, %1};" : "=l"(c) : "f"(c_));
    }
    __device__ __forceinline__ void add(float x0, float x1)
    {
        float d0, d1;
        asm("{\n\t.reg .b64 x;\n\tmov.b64 x, {%2, %3};\n\tadd.rn.f32x2 x, x, %4;\n\tmul.rn.f32x2 x, x, %5;\n\tmov.b64 {%0, %1}, x;\n\t}"
            : "=f"(d0), "=f"(d1) : "f"(x0), "f"(x1), "l"(m), "l"(c));
        d0 = fmaxf(d0, LP_LOW); d1 = fmaxf(d1, LP_LOW);
        const float e0 = lp_exp2(d0), e1 = lp_exp2(d1);
        asm("{\n\t.reg .b64 e, d;\n\tmov.b64 e, {%2, %3};\n\tmov.b64 d, {%4, %5};\n\tadd.rn.f32x2 %0, %0, e;\n\tfma.rn.f32x2 %1, e, d, %1;\n\t}"
            : "+l"(s), "+l"(t) : "f"(e0), "f"(e1), "f"(d0), "f"(d1));
    }
    __device__ __forceinline__ void join(float &S, float &T) const
    {
        float a, b;
        asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(s));
        S += a + b;
        asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(t));
        T += a + b;
    }
};

/* S and T after the maximum grew by D (in base 2, times the scale) */
__device__ __forceinline__ void lp_rescale(float D, float &S, float &T)
{
    if (S > 0.0f) {
        D = fminf(D, -LP_LOW);
        const float f = lp_exp2(-D);
        T = f * (T - D * S);
        S *= f;
    }
}

/* what a row's largest value, its sum and the order of its largest value (NaN included) make of a logit */
struct LpScore {
    float M, S, scale, logS;
    bool none, bad;
    __device__ __forceinline__ LpScore(const LpParams &p, float M, float S, uint32_t O) :
        M(M), S(S), scale(p.scale), logS(logf(S)), none(M == -INFINITY && O == lp_order(-INFINITY)), bad(O >= lp_order(INFINITY)) {}
    __device__ __forceinline__ float operator()(float x) const
    {
        return bad ? __uint_as_float(0x7fffffffu) : none || x == -INFINITY ? -INFINITY : (x - M) * scale - logS;
    }
    __device__ __forceinline__ float entropy(float E) const { return bad ? __uint_as_float(0x7fffffffu) : none ? 0.0f : logS - E / S * LP_LN2; }
};

/*
 * Short rows: a warp holds one in registers, so the maximum is known before the sum and no barrier is needed.  The k-th largest
 * of the lanes' maxima bounds the k-th largest value; vectors that reach it are read again and ranked as above, the places of
 * both found by ballots.  Bound by the issue of a row's instructions, 20000 x 1000 fp32: 15.5 us without alternatives, 25 us with
 * five, 31 us with twenty (12 us at the copy rate); a CTA of 128 threads a row took 65, 109 and 117 us, its barriers and single
 * warps' steps a row's whole time.  1 x 1000: 2.0, 3.0 and 3.2 us.
 */
template <typename T, int U>
__global__ void __launch_bounds__(LP_WNT) k_logprobs_short(const LpParams p, const int n)
{
    using Y = LpType<T>;
    constexpr int V = Y::V;
    __shared__ __align__(16) unsigned long long cands[LP_WNT / 32][LP_WCAND + 2], lists[LP_WNT / 32][LP_KMAX];
    __shared__ __align__(16) uint32_t lanes[LP_WNT / 32][64];
    __shared__ uint16_t items[LP_WNT / 32][32 * U];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const size_t row = (size_t)blockIdx.x * (LP_WNT / 32) + warp;
    drk_dep_wait();     /* no trigger: see k_logprobs (2000 x 1000 fp32, k = 20: 6.9 instead of 5.7 us) */
    if (row >= (size_t)n) return;
    const T *v = static_cast<const T *>(p.logits) + row * p.ld;
    const int head = min(p.len, (int)((16 - (uintptr_t)v % 16) % 16 / sizeof(T)));
    const int nvec = (p.len - head) / V, singles = p.len - nvec * V;
    const uint4 *vec = reinterpret_cast<const uint4 *>(v + head);
    const float c = p.scale * 1.44269504f;
    const int single = lane < head ? lane : nvec * V + lane;
    uint4 x[U];
#pragma unroll
    for (int u = 0; u < U; u++) x[u] = u * 32 + lane < nvec ? __ldg(vec + u * 32 + lane) : make_uint4(Y::FILL, Y::FILL, Y::FILL, Y::FILL);
    float alone = lane < singles ? Y::one(v + single) : -INFINITY;
    int label = -1;
    float labelled = 0.0f;
    if (lane < p.m) {
        label = p.labels[row * p.m + lane];
        if (label >= 0 && label < p.len) labelled = Y::one(v + label);
    }
    unsigned long long *cand = cands[warp], *list = lists[warp];
    list[lane] = 0;

    float vm[U], mine = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; u++) {
        vm[u] = Y::last(Y::max2(Y::max2(x[u].x, x[u].y), Y::max2(x[u].z, x[u].w)));
        mine = lp_max_nan(mine, vm[u]);
    }
    const uint32_t own = max(lane < nvec ? lp_order(mine) : 0u, lane < singles ? lp_order(alone) : 0u);
    const uint32_t O = __reduce_max_sync(0xffffffffu, own);
    float M = fmaxf(mine, alone);           /* the largest that is a number */
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    float S = 0.0f, E = 0.0f;
    {
        const float d = fmaxf((alone - M) * c, LP_LOW), e = lp_exp2(d);
        S += e;
        E = fmaf(e, d, E);
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        float y[V], s = 0.0f, t = 0.0f;
        Y::unpack(x[u], y);
#pragma unroll
        for (int j = 0; j < V; j++) {
            const float d = fmaxf((y[j] - M) * c, LP_LOW), e = lp_exp2(d);
            s += e;
            t = fmaf(e, d, t);
        }
        S += s;
        E += t;
    }
    for (int o = 16; o > 0; o >>= 1) { S += __shfl_xor_sync(0xffffffffu, S, o); E += __shfl_xor_sync(0xffffffffu, E, o); }

    if (p.k > 0) {
        uint32_t border;
        if (p.k <= 24) {
            lanes[warp][lane] = own;
            __syncwarp();
            int r = 0;
#pragma unroll
            for (int j = 0; j < 32; j += 4) {
                const uint4 y = *reinterpret_cast<const uint4 *>(&lanes[warp][j]);
                r += (y.x > own || (y.x == own && j < lane)) + (y.y > own || (y.y == own && j + 1 < lane)) + (y.z > own || (y.z == own && j + 2 < lane)) +
                     (y.w > own || (y.w == own && j + 3 < lane));
            }
            border = __shfl_sync(0xffffffffu, own, __ffs(__ballot_sync(0xffffffffu, r == p.k - 1)) - 1);
        } else {
            /* two parts of a lane's share: the k-th largest of 64 maxima, which 44 values are expected to reach at k = 32 (130 reach
               the least of 32, and at times more than a warp ranks: 20000 x 1000 fp32, k = 32: 50 instead of 125 us, k = 28: 48
               instead of 49; at k = 24 42 instead of 38) */
            float a0 = -INFINITY, a1 = -INFINITY;
#pragma unroll
            for (int u = 0; u < U; u += 2) { a0 = lp_max_nan(a0, vm[u]); a1 = lp_max_nan(a1, vm[u + 1]); }
            const uint32_t g0 = max(lane < nvec ? lp_order(a0) : 0u, lane < singles ? lp_order(alone) : 0u), g1 = 32 + lane < nvec ? lp_order(a1) : 0u;
            lanes[warp][lane] = g0;
            lanes[warp][32 + lane] = g1;
            __syncwarp();
            int r0 = 0, r1 = 0;
#pragma unroll 4
            for (int j = 0; j < 64; j++) {
                const uint32_t y = lanes[warp][j];
                r0 += y > g0 || (y == g0 && j < lane);
                r1 += y > g1 || (y == g1 && j < 32 + lane);
            }
            const uint32_t mine0 = __ballot_sync(0xffffffffu, r0 == p.k - 1), mine1 = __ballot_sync(0xffffffffu, r1 == p.k - 1);
            border = __shfl_sync(0xffffffffu, mine0 ? g0 : g1, __ffs(mine0 | mine1) - 1);
        }
        const float low = lp_value(border);         /* NaN where everything counts */
        const uint32_t before = (1u << lane) - 1;
        int count = 0, found = 0;
        auto offer = [&](bool here, float a, int i) {       /* by the whole warp */
            here = here && !(a < low);
            const uint32_t all = __ballot_sync(0xffffffffu, here);
            const int at = count + __popc(all & before);
            if (here && at < LP_WCAND) cand[at] = lp_key(lp_order(a), (uint32_t)i);
            count += __popc(all);
        };
        if (singles > 0) offer(lane < singles, alone, single);
#pragma unroll
        for (int u = 0; u < U; u++) {
            const bool here = u * 32 + lane < nvec && !(vm[u] < low);
            const uint32_t all = __ballot_sync(0xffffffffu, here);
            if (here) items[warp][found + __popc(all & before)] = (uint16_t)(u * 32 + lane);
            found += __popc(all);
        }
        __syncwarp();
        for (int w = lane; w - lane < found; w += 32) {
            const int i = w < found ? items[warp][w] : 0;
            float y[V];
            Y::unpack(__ldg(vec + i), y);
#pragma unroll
            for (int j = 0; j < V; j++) offer(w < found, y[j], head + i * V + j);
        }
        __syncwarp();
        if (count <= LP_WCAND) {
            for (int i = lane; i < count; i += 32) {
                const unsigned long long key = cand[i];
                const int at = lp_rank(cand, count, key);
                if (at < p.k) list[at] = key;
            }
        } else {
            /* many values equal to the bound: one pass over the row for each alternative */
            unsigned long long limit = ~0ull;
            for (int a = 0; a < p.k; a++) {
                unsigned long long best = 0;
                auto look_at = [&](float z, int i) {
                    const unsigned long long key = lp_key(lp_order(z), (uint32_t)i);
                    if (key <= limit && key > best) best = key;
                };
                if (lane < singles) look_at(alone, single);
                for (int i = lane; i < nvec; i += 32) {
                    float y[V];
                    Y::unpack(__ldg(vec + i), y);
#pragma unroll
                    for (int j = 0; j < V; j++) look_at(y[j], head + i * V + j);
                }
                for (int o = 16; o > 0; o >>= 1) {
                    const unsigned long long y = __shfl_xor_sync(0xffffffffu, best, o);
                    best = y > best ? y : best;
                }
                if (lane == 0) list[a] = best;
                limit = best ? best - 1 : 0;
            }
        }
        __syncwarp();
    }

    const LpScore score(p, M, S, O);
    if (p.entropy && lane == 0) p.entropy[row] = score.entropy(E);
    for (int j = lane; j < p.m; j += 32) {
        if (j != lane) {
            label = p.labels[row * p.m + j];
            if (label >= 0 && label < p.len) labelled = Y::one(v + label);
        }
        p.logprob[row * p.m + j] = label < 0 ? 0.0f : label >= p.len ? __uint_as_float(0x7fffffffu) : score(labelled);
    }
    if (lane < p.k) {
        const unsigned long long key = list[lane];
        p.top_logprob[row * p.k + lane] = score(lp_value((uint32_t)(key >> 32)));
        p.top_index[row * p.k + lane] = (int)(0xffffffffu - (uint32_t)key);
    }
}

template <typename T, int NT>
__global__ void __launch_bounds__(NT, 1024 / NT) k_logprobs(const LpParams p)
{
    using Y = LpType<T>;
    constexpr int V = Y::V, WARPS = NT / 32, PER_GROUP = NT / LP_GROUPS;
    __shared__ float smax[LP_SLOTS][NT];
    __shared__ __align__(16) unsigned long long cand[LP_CAND + 2];
    __shared__ __align__(16) unsigned long long all[LP_SPLIT * LP_KMAX];    /* the alternatives of the cluster's CTAs, k each */
    __shared__ float stats[LP_SPLIT][4];    /* their maxima, S, T and the orders of their largest values (NaN included) */
    __shared__ uint32_t items[LP_ITEMS];
    __shared__ unsigned long long group_key[LP_GROUPS], list[LP_KMAX], red[WARPS], bound;
    __shared__ __align__(16) uint32_t group[LP_GROUPS];
    __shared__ float fred[4][WARPS];
    __shared__ int n_items, n_cand;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (p.split > 1) lp_cluster_arrive();   /* waited for before the first store into another CTA: it runs by then */
    /* The next launch may begin when this one's CTAs end (no trigger before): CTAs that waited beside these would take the places of
       their own launch's others and leave it crowded on few SMs (77 x 50001 f16 12.5 instead of 9.2 us, 300 x 32000 fp32 15.6
       instead of 13.1; without dependent launches 11.1 and 14.8). */
    drk_dep_wait();
    const size_t row = blockIdx.x / p.split;
    const int rank = (int)(blockIdx.x - row * p.split);
    const T *v = static_cast<const T *>(p.logits) + row * p.ld;
    /* single values up to the first 16-byte boundary and behind the last one, vectors between them; the cluster shares the vectors */
    const int head = min(p.len, (int)((16 - (uintptr_t)v % 16) % 16 / sizeof(T)));
    const int nvec = (p.len - head) / V, singles = rank == 0 ? p.len - nvec * V : 0;
    const int v0 = (int)((long long)nvec * rank / p.split), count = (int)((long long)nvec * (rank + 1) / p.split) - v0;
    const uint4 *vec = reinterpret_cast<const uint4 *>(v + head) + v0;
    const int first = head + v0 * V;        /* index of the share's first value */
    auto single_index = [&](int i) { return i < head ? i : nvec * V + i; };
    const float c = p.scale * 1.44269504f;
    /* the first label's logit is asked for now and used at the end */
    int label = -1;
    float labelled = 0.0f;
    if (rank == 0 && tid < p.m) {
        label = p.labels[row * p.m + tid];
        if (label >= 0 && label < p.len) labelled = Y::one(v + label);
    }

    float m = -INFINITY, RS = 0.0f, RT = 0.0f, mine = -INFINITY;
    const int batches = (count + NT * LP_U - 1) / (NT * LP_U), few = max(1, (batches + 7) / 8);
    /* slots of up to four batches: eight; longer ones are cut again, as they are read again (2048 x 131072: 177 us with sixteen,
       187 with eight; 4000 x 8192 bf16: 34 us with eight, 37 with sixteen) */
    const int per_slot = few <= 4 ? few : max(4, (batches + LP_SLOTS - 1) / LP_SLOTS), slots = (batches + per_slot - 1) / per_slot;
    uint4 next[LP_U];
    auto fetch = [&](int b) {
#pragma unroll
        for (int u = 0; u < LP_U; u++) {
            const int i = (b * LP_U + u) * NT + tid;
            next[u] = i < count ? __ldg(vec + i) : make_uint4(Y::FILL, Y::FILL, Y::FILL, Y::FILL);
        }
    };
    /* 16-bit rows, whose sums leave a CTA less time for its loads, are also asked into the L2 one batch further ahead */
    auto ahead = [&](int from, int to) {
        const int a = from * NT * LP_U, z = min(count, to * NT * LP_U);
        if (sizeof(T) == 2 && tid == 0 && a < z) asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(vec + a), "r"((z - a) * 16) : "memory");
    };
    ahead(1, 2);
    if (batches > 0) fetch(0);
    for (int slot = 0; slot < slots; slot++) {
        float sm = -INFINITY;
        for (int b = slot * per_slot; b < min(batches, (slot + 1) * per_slot); b++) {
            uint4 now[LP_U];
#pragma unroll
            for (int u = 0; u < LP_U; u++) now[u] = next[u];
            if (b + 1 < batches) fetch(b + 1);
            ahead(b + 2, b + 3);
            uint32_t w2 = Y::max2(now[0].x, now[0].y);
            w2 = Y::max2(w2, Y::max2(now[0].z, now[0].w));
#pragma unroll
            for (int u = 1; u < LP_U; u++) w2 = Y::max2(w2, Y::max2(Y::max2(now[u].x, now[u].y), Y::max2(now[u].z, now[u].w)));
            const float bm = Y::last(w2);
            sm = lp_max_nan(sm, bm);
            if (bm > m) {
                lp_rescale((bm - m) * c, RS, RT);
                m = bm;
            }
            /* a batch is summed by itself: a long row adds len / (threads x 16 or 32) of them, not its values, to one sum */
            LpSums<sizeof(T) == 2> sums(m, c);
#pragma unroll
            for (int u = 0; u < LP_U; u++) {
                float x[V];
                Y::unpack(now[u], x);
#pragma unroll
                for (int j = 0; j < V; j += 2) sums.add(x[j], x[j + 1]);
            }
            sums.join(RS, RT);
        }
        smax[slot][tid] = sm;
        mine = lp_max_nan(mine, sm);
    }
    uint32_t own_single = 0;                /* order of the single value this thread looks at */
    if (tid < singles) {
        const float x = Y::one(v + single_index(tid));
        own_single = lp_order(x);
        if (x > m) {
            lp_rescale((x - m) * c, RS, RT);
            m = x;
        }
        const float d = fmaxf((x - m) * c, LP_LOW), e = lp_exp2(d);
        RS += e;
        RT = fmaf(e, d, RT);
    }
    const uint32_t own = tid < count ? lp_order(mine) : 0;      /* order of the largest of this thread's vectors */

    /* the CTA's maximum, S and T */
    float M = m, S = 0.0f, E = 0.0f;
    uint32_t O = __reduce_max_sync(0xffffffffu, max(own, own_single));
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    if (lane == 0) { fred[0][warp] = M; fred[1][warp] = __uint_as_float(O); }
    /* the largest of each group of threads, for the bound below */
    uint32_t g = own;
#pragma unroll
    for (int o = 1; o < PER_GROUP; o <<= 1) g = max(g, __shfl_xor_sync(0xffffffffu, g, o));
    if (tid % PER_GROUP == 0) group[tid / PER_GROUP] = g;
    if (tid == 0) { n_items = 0; n_cand = 0; bound = 0; }
    if (tid < LP_KMAX) list[tid] = 0;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WARPS; w++) { M = fmaxf(M, fred[0][w]); O = max(O, __float_as_uint(fred[1][w])); }
    lp_rescale((M - m) * c, RS, RT);
    for (int o = 16; o > 0; o >>= 1) { RS += __shfl_xor_sync(0xffffffffu, RS, o); RT += __shfl_xor_sync(0xffffffffu, RT, o); }
    if (lane == 0) { fred[2][warp] = RS; fred[3][warp] = RT; }
    /* the k-th largest group */
    if (p.k > 0 && tid < LP_GROUPS) {
        const uint32_t x = group[tid];
        int r = 0;
#pragma unroll
        for (int j = 0; j < LP_GROUPS; j += 4) {
            const uint4 y = *reinterpret_cast<const uint4 *>(group + j);
            r += (y.x > x || (y.x == x && j < tid)) + (y.y > x || (y.y == x && j + 1 < tid)) + (y.z > x || (y.z == x && j + 2 < tid)) +
                 (y.w > x || (y.w == x && j + 3 < tid));
        }
        if (r == p.k - 1) bound = (unsigned long long)x << 32;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WARPS; w++) { S += fred[2][w]; E += fred[3][w]; }

    if (p.k > 0) {
        /* Looks at every value whose key is at least `bound`; false if they or their slots are too many.  A slot's first index
           bounds the keys of its values that are equal to its maximum. */
        auto collect = [&]() {
            const uint32_t border = (uint32_t)(bound >> 32);
            const float low = lp_value(border);         /* NaN where everything counts: x < low is false then */
            auto offer = [&](uint32_t order, int i) {
                const unsigned long long key = lp_key(order, (uint32_t)i);
                if (key >= bound) {
                    const int at = atomicAdd(&n_cand, 1);
                    if (at < LP_CAND) cand[at] = key;
                }
            };
            if (tid < singles) offer(own_single, single_index(tid));
            if (own >= border && own > 0)
                for (int s = 0; s < slots; s++)
                    if (lp_key(lp_order(smax[s][tid]), (uint32_t)(first + (s * per_slot * LP_U * NT + tid) * V)) >= bound) {
                        const int at = atomicAdd(&n_items, 1);
                        if (at < LP_ITEMS) items[at] = (uint32_t)tid | ((uint32_t)s << 16);
                    }
            __syncthreads();
            if (n_items > LP_ITEMS) return false;
            const int each = per_slot * LP_U;
            for (int w = tid; w < n_items * each; w += NT) {
                const uint32_t it = items[w / each];
                const int i = ((int)(it >> 16) * each + w % each) * NT + (int)(it & 0xffffu);
                if (i >= count) continue;
                float x[V];
                Y::unpack(__ldg(vec + i), x);
#pragma unroll
                for (int j = 0; j < V; j++) if (!(x[j] < low)) offer(lp_order(x[j]), first + i * V + j);
            }
            __syncthreads();
            return n_cand <= LP_CAND;
        };
        bool ok = collect();
        if (!ok) {
            /* Many values equal to the bound (a row of one value, for instance): the same bound on keys, which differ by their
               index.  A thread's largest stands first in the first slot that has it. */
            unsigned long long key = 0;
            if (own > 0) {
                int s = 0;
                while (s < slots - 1 && lp_order(smax[s][tid]) != own) s++;
                for (int w = 0; w < per_slot * LP_U && key == 0; w++) {
                    const int i = (s * per_slot * LP_U + w) * NT + tid;
                    if (i >= count) break;
                    float x[V];
                    Y::unpack(__ldg(vec + i), x);
                    for (int j = V - 1; j >= 0; j--) if (lp_order(x[j]) == own) key = lp_key(own, (uint32_t)(first + i * V + j));
                }
            }
#pragma unroll
            for (int o = 1; o < PER_GROUP; o <<= 1) {
                const unsigned long long y = __shfl_xor_sync(0xffffffffu, key, o);
                key = y > key ? y : key;
            }
            __syncthreads();
            if (tid % PER_GROUP == 0) group_key[tid / PER_GROUP] = key;
            if (tid == 0) { n_items = 0; n_cand = 0; }
            __syncthreads();
            if (tid < LP_GROUPS) {
                const unsigned long long x = group_key[tid];
                int r = 0;
                for (int j = 0; j < LP_GROUPS; j++) r += group_key[j] > x || (group_key[j] == x && j < tid);
                if (r == p.k - 1) bound = x;
            }
            __syncthreads();
            ok = collect();
        }
        if (ok) {
            const int n = n_cand;
            for (int i = tid; i < n; i += NT) {
                const unsigned long long key = cand[i];
                const int r = lp_rank(cand, n, key);
                if (r < p.k) list[r] = key;
            }
        } else {
            /* the largest values crowd in few threads' shares: one pass over the row for each alternative */
            unsigned long long limit = ~0ull;
            for (int r = 0; r < p.k; r++) {
                unsigned long long best = 0;
                for (int i = tid; i < count; i += NT) {
                    float x[V];
                    Y::unpack(__ldg(vec + i), x);
#pragma unroll
                    for (int j = 0; j < V; j++) {
                        const unsigned long long key = lp_key(lp_order(x[j]), (uint32_t)(first + i * V + j));
                        if (key <= limit && key > best) best = key;
                    }
                }
                if (tid < singles) {
                    const unsigned long long key = lp_key(own_single, (uint32_t)single_index(tid));
                    if (key <= limit && key > best) best = key;
                }
                for (int o = 16; o > 0; o >>= 1) {
                    const unsigned long long y = __shfl_xor_sync(0xffffffffu, best, o);
                    best = y > best ? y : best;
                }
                __syncthreads();
                if (lane == 0) red[warp] = best;
                __syncthreads();
                for (int w = 0; w < WARPS; w++) best = red[w] > best ? red[w] : best;
                if (tid == 0) list[r] = best;
                limit = best ? best - 1 : 0;
            }
        }
    }
    __syncthreads();

    if (p.split > 1) {
        __syncwarp();
        lp_cluster_wait();
        if (tid < p.k) lp_st_first((uint32_t)__cvta_generic_to_shared(all + rank * p.k + tid), list[tid]);
        if (tid < 4) lp_st_first((uint32_t)__cvta_generic_to_shared(&stats[rank][tid]), tid == 0 ? M : tid == 1 ? S : tid == 2 ? E : __uint_as_float(O));
        __syncwarp();
        lp_cluster_arrive();
        if (rank != 0) return;
        lp_cluster_wait();
        S = E = 0.0f;
#pragma unroll
        for (int r = 0; r < LP_SPLIT; r++)
            if (r < p.split) { M = fmaxf(M, stats[r][0]); O = max(O, __float_as_uint(stats[r][3])); }
#pragma unroll
        for (int r = 0; r < LP_SPLIT; r++)
            if (r < p.split) {
                float s = stats[r][1], t = stats[r][2];
                lp_rescale((M - stats[r][0]) * c, s, t);
                S += s;
                E += t;
            }
        for (int i = tid; i < p.split * p.k; i += NT) {
            const unsigned long long key = all[i];
            const int r = lp_rank(all, p.split * p.k, key);
            if (key != 0 && r < p.k) list[r] = key;
        }
        __syncthreads();
    }

    const LpScore score(p, M, S, O);
    if (p.entropy && tid == 0) p.entropy[row] = score.entropy(E);
    for (int j = tid; j < p.m; j += NT) {
        if (j != tid) {
            label = p.labels[row * p.m + j];
            if (label >= 0 && label < p.len) labelled = Y::one(v + label);
        }
        p.logprob[row * p.m + j] = label < 0 ? 0.0f : label >= p.len ? __uint_as_float(0x7fffffffu) : score(labelled);
    }
    for (int j = tid; j < p.k; j += NT) {
        const unsigned long long key = list[j];
        p.top_logprob[row * p.k + j] = score(lp_value((uint32_t)(key >> 32)));
        p.top_index[row * p.k + j] = (int)(0xffffffffu - (uint32_t)key);
    }
}

template <typename T, int U> static int lp_launch_short(cudaStream_t st, const LpParams &p, int n)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((n + LP_WNT / 32 - 1) / (LP_WNT / 32)));
    cfg.blockDim = dim3(LP_WNT);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = drk_dep_launch_enabled() ? 1 : 0;
    return drk_launched(cudaLaunchKernelEx(&cfg, k_logprobs_short<T, U>, p, n));
}

static int lp_refuse(const char *why)
{
    fprintf(stderr, "dRk_logprobs: %s\n", why);
    return -1;
}

template <typename T, int NT> static int lp_launch(cudaStream_t st, const LpParams &p, int n)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)n * (unsigned)p.split);
    cfg.blockDim = dim3(NT);
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    int na = 0;
    if (p.split > 1) {
        attr[na].id = cudaLaunchAttributeClusterDimension;
        attr[na].val.clusterDim.x = (unsigned)p.split;
        attr[na].val.clusterDim.y = attr[na].val.clusterDim.z = 1;
        na++;
    }
    if (drk_dep_launch_enabled()) {
        attr[na].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[na].val.programmaticStreamSerializationAllowed = 1;
        na++;
    }
    cfg.attrs = attr;
    cfg.numAttrs = na;
    return drk_launched(cudaLaunchKernelEx(&cfg, k_logprobs<T, NT>, p));
}

/* A row is split over up to eight CTAs while that leaves at most two on each of 148 SMs and a load for each thread of a share.
 * Four would fit, but then the next launch finds no place to start in while this one ends: 148 x 32000 bf16 with 20 alternatives
 * takes 7.6 us unsplit, 8.3 us in twos, 12 to 14 us in threes and fours; 100 x 131072 fp32 27, 19, and 18 us.
 * CTAs of 128 threads, eight on an SM, when the rows do not all find a place in fours of 256 (4096 x 8192 fp32: 39 instead of
 * 54 us, 1000 x 32000 28 instead of 31; but 592 x 131072, 61 instead of 51), in 16 bits, where more threads than loads are
 * missing, when they fill six places of eight (131072 bf16: 700 rows 53 instead of 40 us, 1100 rows 59 both, 2000 rows 96 instead
 * of 98; 32000 f16: 700 rows 21.0 instead of 19.4, 900 rows 22.0 instead of 22.5, 2000 rows 36.6 instead of 40.3); or when a
 * share is a few of their batches (300 x 8192 fp32: 6.8 instead of 8.7 us; 1 x 131072 bf16 in eight shares of four batches: 9.7
 * instead of 8.0 us). */
template <typename T> static int lp_run(cudaStream_t st, LpParams &p, int n)
{
    constexpr int V = LpType<T>::V;
    if (p.len <= 32 * LP_WU * V) return lp_launch_short<T, LP_WU>(st, p, n);
    if (p.len <= 64 * LP_WU * V) return lp_launch_short<T, 2 * LP_WU>(st, p, n);
    const int room = 2 * 148 / n, most = p.len / (LP_NT * V);
    p.split = room < most ? room : most;
    p.split = p.split < 1 ? 1 : p.split > LP_SPLIT ? LP_SPLIT : p.split;
    return n > (sizeof(T) == 2 ? 6 : 4) * 148 || p.len / p.split <= (p.split > 1 ? 2 : 4) * 128 * LP_U * V ? lp_launch<T, 128>(st, p, n) : lp_launch<T, LP_NT>(st, p, n);
}

extern "C" int dRk_logprobs(dRk_stream stream, const void *logits, int type, long long ld, int n, int len, float scale, const int *labels, int m,
                            float *logprob, float *entropy, int k, float *top_logprob, int *top_index)
{
    const int size = type == DRK_F32 ? 4 : type == DRK_BF16 || type == DRK_F16 ? 2 : 0;
    if (!size) return lp_refuse("unknown element type");
    if (n < 1 || len < 1) return lp_refuse("needs at least one row and one logit");
    if (n > 1 << 28 || len > 1 << 30) return lp_refuse("more than 2^28 rows or 2^30 logits");
    if (n > 1 && ld < len) return lp_refuse("rows overlap (ld < len)");
    if (m < 0 || k < 0 || k > LP_KMAX || k > len) return lp_refuse("number of labels below 0, or of alternatives outside 0..min(32, len)");
    if (!logits || (m > 0 && (!labels || !logprob)) || (k > 0 && (!top_logprob || !top_index))) return lp_refuse("null pointer");
    if (!(scale > 0.0f) || !(scale <= 0x1p120f)) return lp_refuse("scale (1 / temperature) must be positive and at most 2^120");
    if ((uintptr_t)logits % size || (uintptr_t)labels % 4 || (uintptr_t)logprob % 4 || (uintptr_t)entropy % 4 || (uintptr_t)top_logprob % 4 || (uintptr_t)top_index % 4)
        return lp_refuse("pointer not aligned to its element type");
    const int dev = drk_stream_device("dRk_logprobs", stream, -1);
    if (dev < 0) return dev;
    LpParams p = {};
    p.logits = logits;
    p.ld = n > 1 ? (size_t)ld : 0;
    p.len = len; p.m = m; p.k = k; p.split = 1;
    p.scale = scale;
    p.labels = labels;
    p.logprob = logprob; p.entropy = entropy;
    p.top_logprob = top_logprob; p.top_index = top_index;
    cudaStream_t st = drk_stream(stream);
    return type == DRK_F32 ? lp_run<float>(st, p, n) : type == DRK_BF16 ? lp_run<__nv_bfloat16>(st, p, n) : lp_run<__half>(st, p, n);
}
