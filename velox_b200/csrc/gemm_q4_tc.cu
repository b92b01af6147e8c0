// The products with matrices held in four bits (q4.cuh) for more than a few rows, on the fifth-generation tensor cores:
// out[M,N] = x[M,K] W^T (+ bias), and out[M,N] = act(x Wg^T) * (x Wu^T).
//
// The operands are turned, out^T = W x^T: 128 rows of W on the M side of tcgen05.mma, n rows of x as its columns.  W is the instruction's A
// operand, and A may lie in tensor memory: a lane is a row, a column two neighbouring k.  So a thread makes 64 k of its own row
// from 32 bytes of codes in registers and stores them with one tcgen05.st; W as bfloat16 exists in tensor memory only.
// Gated, gate and up rows of a feature are the same lane's in two accumulators, and the epilogue joins them without an exchange.
//
// Warps of a block:
//   warp 0       producer: x (128-byte swizzle), codes, scales and offsets of a step of 128 k by TMA; W's first stages are asked for before the
//                wait for the kernel launched before this one (if the caller says that W is ready);
//   warp 1       tensor memory; issues the products;
//   warps 2-17   four groups of four that make W's values, half a step each: two groups every other step, gated two gate and two up of every
//                step; into places for four steps (gated two) in tensor memory;
//   warps 18-25  epilogue.
// K may be cut into `splits` runs, one to each block of a cluster, whose float32 sums are added in ascending order through distributed
// shared memory: the same result on every run.
// A run's sum stays in one float32 accumulator, which the tensor core cuts towards zero at every 16 k: a float32 result's error grows with the
// run (root mean square, relative: 6.7e-7 at 1,024 k, 2e-6 at 2,560, 1.2e-5 at 12,288, as of the dense products on tcgen05).  A bfloat16
// result does not show it (1.7e-3), and for logits it is little beside the rounding of x; fresh accumulators every few steps, added in registers, would have the
// epilogue read the accumulators as often.
// Every wait on an mbarrier is bounded; a block whose wait runs out records a code in the caller's error word and writes NaN, the other roles run
// out of their own, all meet, free their tensor memory and return.
//
// Tensor memory is taken before the wait for the kernel before and before the next one is let in (gemm_turned.cu says why that is safe).  A block
// takes all of it, and so much shared memory that no other block that takes some fits beside it, whatever stream that one is on: two clusters
// whose blocks waited for each other's tensor memory on two SMs would wait for good, as a cluster gives none back before its blocks have met.
#include "q4.cuh"
#include "tcgen05_pair.cuh"

#define QT_TEAMS 4           // groups of four warps that make W's values
#define QT_MAKERS 2          // their first warp
#define QT_EPILOGUE (QT_MAKERS + 4 * QT_TEAMS)   // ... and the epilogue's
#define QT_THREADS (32 * (QT_EPILOGUE + 8))
#define QT_K 128             // k of a step
#define QT_PLACES_AT 256     // W's values in tensor memory: 256 columns behind the accumulators
#define QT_MAX_STAGES 8
#define QT_ROOM (224 * 1024) // shared memory for stages
#define QT_LEAST (160 * 1024)   // ... at least: the smallest ring beside tensor memory, of a turned product with two blocks an SM, is 84 KB
#define QT_CODES 8192        // bytes of a stage: codes of 128 rows by 128 k
#define QT_AFFINE 2048       // ... room for their scales and offsets (512, 1024, 2048 for groups of 128, 64, 32)
#define QT_MOST_K (1 << 24)  // depth up to which a tile takes well under the second that its epilogue waits for (131,072 steps of up to 0.93 us)
#define QT_ERR_PRODUCER 10
#define QT_ERR_MMA 11
#define QT_ERR_EPILOGUE 12
#define QT_ERR_VALUES 13

struct QtShape {
    int n;             // rows of x in a tile
    int splits;        // runs of k
    int steps;         // steps of a run
    int stages;
};
struct QtMaps { CUtensorMap x, codes[2], affine[2]; };

__device__ __forceinline__ void qt_st16(unsigned taddr, const unsigned (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};\n"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void qt_ld16(unsigned taddr, unsigned (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
          "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr) : "memory");
}
// (What is waited for takes microseconds; this many polls take a good part of a second at least.)
__device__ __forceinline__ bool qt_wait(unsigned bar, unsigned parity) { return tc_warp_wait(bar, parity, 1 << 20); }
__device__ __forceinline__ uint2 qt_lds8(unsigned addr) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];\n" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ unsigned qt_lds4(unsigned addr) {
    unsigned v;
    asm volatile("ld.shared.u32 %0, [%1];\n" : "=r"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float qt_ld_cluster(unsigned addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];\n" : "=f"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void qt_arrive(unsigned bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(bar) : "memory");
}
// z / (1 + exp(-z)) by the hardware's 2^x and 1 / x (a few 2^-23 each; the result is rounded to bfloat16, 2^-8).
__device__ __forceinline__ float qt_silu(float z) {
    float e, d;
    asm("ex2.approx.f32 %0, %1;\n" : "=f"(e) : "f"(z * -1.4426950408889634f));
    asm("rcp.approx.f32 %0, %1;\n" : "=f"(d) : "f"(1.f + e));
    return z * d;
}
// Four products of 16 k: A in tensor memory (8 columns each), B in a swizzled K-major tile.
__device__ __forceinline__ void qt_mma_64(unsigned d, unsigned a, unsigned b_lo, unsigned idesc, unsigned add) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
        asm volatile("{\n .reg .pred p;\n .reg .b64 b;\n setp.ne.b32 p, %4, 0;\n mov.b64 b, {%2, %5};\n"
                     " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n}\n"
                     ::"r"(d), "r"(a + 8 * k), "r"(b_lo + 2 * k), "r"(idesc), "r"(k ? 1u : add), "r"(TC_DESC_HI) : "memory");
}

// 32 codes of a row to 16 pairs of values.
template <bool SMALL>
__device__ __forceinline__ void qt_values(uint2 first, uint2 second, unsigned affine, unsigned (&w)[16]) {
    const unsigned scale = SMALL ? q4_raised(q4_scale(affine)) : q4_scale(affine), offset = q4_offset(affine);
    const unsigned words[4] = {first.x, first.y, second.x, second.y};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        unsigned v[4];
        q4_values<SMALL>(words[i], scale, offset, v);
        w[4 * i] = v[0]; w[4 * i + 1] = v[1]; w[4 * i + 2] = v[2]; w[4 * i + 3] = v[3];
    }
}

template <bool GATED, typename TO>
__global__ void __launch_bounds__(QT_THREADS, 1)
gemm_q4_tc_kernel(const __grid_constant__ QtMaps maps, const float* __restrict__ bias, TO* __restrict__ C, int M, int N, int blocks, int ldc, int act,
                  int group, int w_ready, const QtShape sh, int* __restrict__ error) {
    constexpr int MATS = GATED ? 2 : 1, PLACES = GATED ? 2 : 4;   // (places: steps whose values there is room for)
    // A step's products begin when its values are there: gated, half by half, so that the groups that make the two halves do not go in
    // step with each other, all making values and all waiting.  (Plain, the groups take turns at steps.)
    constexpr int PARTS = GATED ? 2 : 1;
    extern __shared__ unsigned char qt_raw[];
    __shared__ __align__(8) unsigned long long full_bar[QT_MAX_STAGES], empty_bar[QT_MAX_STAGES], w_full[PLACES * PARTS], w_empty[PLACES * PARTS], acc_full[2], acc_empty[2];
    __shared__ unsigned tmem_s;
    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int split = sh.splits > 1 ? (int)tp_cluster_rank() : 0;
    const int group_shift = group == 32 ? 5 : (group == 64 ? 6 : 7);
    const unsigned affine_row = (QT_K >> group_shift) * 64u;      // bytes of 16 rows' scales and offsets of a step
    const unsigned x_room = (unsigned)sh.n * (QT_K * 2), stage_bytes = x_room + MATS * (QT_CODES + QT_AFFINE);
    const unsigned tiles = (tc_smem_u32(qt_raw) + 1023) & ~1023u;
    const int step0 = split * sh.steps, steps = min((blocks + 1) / 2 - step0, sh.steps);   // of this block's run
    const int xt = (M + sh.n - 1) / sh.n, total = (N + 127) / 128 * xt;
    const int me = (int)blockIdx.x / sh.splits, teams = (int)gridDim.x / sh.splits;
    const int my_tiles = (total - me + teams - 1) / teams;
    const int buffers = 2 * MATS * sh.n <= QT_PLACES_AT ? 2 : 1;   // accumulators: two where there is room, so that a tile's epilogue runs under the next one's products
    // (once a tile: divisions.  Once a load they were most of the producer's time.)  Tiles that are worked on at the same time share rows of W.
    struct Tile { int w0, m0; };
    auto tile_of = [&](int ti) {
        const int i = me + ti * teams, row = i / xt;
        return Tile{row * 128, (i - row * xt) * sh.n};
    };
    if (threadIdx.x == 0) {
        for (int s = 0; s < sh.stages; ++s) {
            tc_mbar_init(tc_smem_u32(&full_bar[s]), 1);    // the producer, with the bytes
            // the commit of the products that read the stage's x; plain, the warps that make W's values too (see there)
            tc_mbar_init(tc_smem_u32(&empty_bar[s]), GATED ? 1 : 1 + 4 * QT_TEAMS);
        }
        for (int p = 0; p < PLACES * PARTS; ++p) {
            tc_mbar_init(tc_smem_u32(&w_full[p]), 8);   // the warps that fill it
            tc_mbar_init(tc_smem_u32(&w_empty[p]), 1);  // the commit of the products that read it
        }
        for (int b = 0; b < 2; ++b) {
            tc_mbar_init(tc_smem_u32(&acc_full[b]), 1);
            tc_mbar_init(tc_smem_u32(&acc_empty[b]), 8);   // the epilogue's warps
        }
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(tc_smem_u32(&tmem_s)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
    __syncwarp();
    asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
    const unsigned tmem = tmem_s;

    auto load = [&](const Tile& tile, int step, int s, bool of_w, bool of_x) {
        const unsigned bar = tc_smem_u32(&full_bar[s]), st = tiles + (unsigned)s * stage_bytes;
        const int k = (step0 + step) * QT_K;
        if (of_w) {
            tc_mbar_expect_tx(bar, x_room + MATS * (QT_CODES + 8 * affine_row));
#pragma unroll
            for (int i = 0; i < MATS; ++i) {
                const unsigned at = st + x_room + i * (QT_CODES + QT_AFFINE);
                tc_tma_load_2d(at, &maps.codes[i], k * 2, tile.w0 >> 4, bar);
                tc_tma_load_2d(at + QT_CODES, &maps.affine[i], (k >> group_shift) * 16, tile.w0 >> 4, bar);
            }
        }
        if (of_x) {
            tc_tma_load_2d(st, &maps.x, k, tile.m0, bar);
            tc_tma_load_2d(st + x_room / 2, &maps.x, k + TC_BK, tile.m0, bar);
        }
    };
    const Tile tile0 = tile_of(0);
    const int ahead = w_ready ? min(sh.stages, steps) : 0;   // stages whose W is asked for before the wait
    if (warp == 0)
        for (int i = 0; i < ahead; ++i)
            if (tc_elect()) load(tile0, i, i, true, false);
    pdl_wait();
    if (warp == 0)
        for (int i = 0; i < ahead; ++i)
            if (tc_elect()) load(tile0, i, i, false, true);
    __syncwarp();
    pdl_trigger();

    if (warp == 0) {
        int s = ahead == sh.stages ? 0 : ahead;
        unsigned phase = ahead == sh.stages ? 0 : 1;   // (the first time round a stage is free: the phase before the first has ended)
        for (int ti = 0; ti < my_tiles; ++ti) {
            const Tile tile = tile_of(ti);
            for (int i = ti ? 0 : ahead; i < steps; ++i) {
                if (!qt_wait(tc_smem_u32(&empty_bar[s]), phase)) {
                    if (lane == 0) atomicExch(error, QT_ERR_PRODUCER);
                    ti = my_tiles;
                    break;
                }
                if (tc_elect()) load(tile, i, s, true, true);
                if (++s == sh.stages) { s = 0; phase ^= 1; }
            }
        }
    } else if (warp == 1) {
        int s = 0, place = 0;
        unsigned phase = 0, place_phase = 0;
        bool ok = true;
        // float32 accumulator, bfloat16 operands, both K-major, N = n, M = 128
        const unsigned idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((unsigned)(sh.n >> 3) << 17) | (8u << 24);
        const unsigned x_half = x_room >> 5;   // (in a descriptor's units)
        for (int ti = 0; ok && ti < my_tiles; ++ti) {
            const int buf = buffers == 2 ? ti & 1 : 0, use = buffers == 2 ? ti >> 1 : ti;
            const unsigned d = tmem + (unsigned)(buf * MATS * sh.n);
            ok = !use || qt_wait(tc_smem_u32(&acc_empty[buf]), (unsigned)((use - 1) & 1));
            for (int i = 0; ok && i < steps; ++i) {
                ok = qt_wait(tc_smem_u32(&full_bar[s]), phase);
                const unsigned xd = tc_desc_lo(tiles + (unsigned)s * stage_bytes), a = tmem + QT_PLACES_AT + (unsigned)(place * MATS * 64);
#pragma unroll
                for (int part = 0; part < PARTS; ++part) {
                    ok = ok && qt_wait(tc_smem_u32(&w_full[place * PARTS + part]), place_phase);
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
                    if (tc_elect()) {
#pragma unroll
                        for (int h = part; h < (PARTS == 2 ? part + 1 : 2); ++h)
#pragma unroll
                            for (int m = 0; m < MATS; ++m)
                                qt_mma_64(d + (unsigned)(m * sh.n), a + m * 64 + h * 32, xd + h * x_half, idesc, h ? 1u : (unsigned)(i > 0));
                        tc_commit(tc_smem_u32(&w_empty[place * PARTS + part]));
                        if (part == PARTS - 1) tc_commit(tc_smem_u32(&empty_bar[s]));
                    }
                }
                if (!ok) break;
                if (++place == PLACES) { place = 0; place_phase ^= 1; }
                if (++s == sh.stages) { s = 0; phase ^= 1; }
            }
            if (ok && tc_elect()) tc_commit(tc_smem_u32(&acc_full[buf]));
        }
        if (!ok && lane == 0) atomicExch(error, QT_ERR_MMA);
    } else if (warp < QT_EPILOGUE) {
        constexpr int STRIDE = GATED ? 1 : 2;   // steps that a group goes on by
        const int team = (warp - QT_MAKERS) >> 2, quarter = warp & 3, row = quarter * 32 + lane;
        const int mat = GATED ? team & 1 : 0, part = GATED ? team >> 1 : team & 1;   // which half of a step
        const unsigned w_at = tiles + x_room + mat * (QT_CODES + QT_AFFINE);
        const unsigned codes_at = w_at + (row >> 4) * 1024 + part * 512 + (row & 7) * 16 + (row >> 3 & 1) * 8;
        const unsigned affine_at = w_at + QT_CODES + (row >> 4) * affine_row + (part * 64 >> group_shift) * 64 + (row & 7) * 8 + (row >> 3 & 1) * 4;
        const unsigned second = group == 32 ? 64 : 0;   // (of 64 k the second half's group)
        const unsigned lanes = tmem + QT_PLACES_AT + mat * 64 + part * 32 + ((unsigned)(quarter * 32) << 16);
        const int all = my_tiles * steps;
        int i = GATED ? 0 : team >> 1, place = i, seen = 0, s = 0;
        unsigned phase = 0, place_phase = 1;   // (the first time round a place is free)
        uint2 q[4];
        unsigned a0, a1, st = 0;
        // Step `want`'s codes, scales and offsets from its stage.  Every step's mbarrier is waited for, in order, that of the other groups'
        // steps too, and a stage is loaded again only when all have done so: who sees some of an mbarrier's phases only could take one for
        // another, or miss one.  (Gated, every group has a part in every step, and no step's products begin without it.)
        // `wait` false: only if it is there already.
        auto fetch = [&](int want, bool wait) {
            for (; seen <= want; ++seen) {
                const unsigned bar = tc_smem_u32(&full_bar[s]);
                if (!(wait ? qt_wait(bar, phase) : tc_warp_look(bar, phase))) return false;
                if (!GATED && lane == 0) qt_arrive(tc_smem_u32(&empty_bar[s]));
                st = (unsigned)s * stage_bytes;
                if (++s == sh.stages) { s = 0; phase ^= 1; }
            }
            a0 = qt_lds4(affine_at + st);
            a1 = qt_lds4(affine_at + st + second);
#pragma unroll
            for (int t = 0; t < 4; ++t) q[t] = qt_lds8(codes_at + st + t * 128);
            return true;
        };
        bool ok = i >= all || fetch(i, true);
        for (; ok && i < all; i += STRIDE) {
            // 32 k at a time: the first half's values are on their way to tensor memory while the second's are made
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const unsigned pair = h ? a1 : a0;
                unsigned w[16];
                if (__all_sync(0xffffffffu, q4_small(pair))) qt_values<true>(q[2 * h], q[2 * h + 1], pair, w);
                else qt_values<false>(q[2 * h], q[2 * h + 1], pair, w);
                if (h == 0) {
                    ok = qt_wait(tc_smem_u32(&w_empty[place * PARTS + (GATED ? part : 0)]), place_phase);
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
                }
                qt_st16(lanes + place * (MATS * 64) + h * 16, w);
            }
            if (!ok) break;
            // The next step's codes while the values are on their way, if they have come.  (Waited for only behind the arrival: the ring may
            // have no stage for them until this step's products have ended.)
            const bool last = i + STRIDE >= all, there = !last && fetch(i + STRIDE, false);
            asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory");
            asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
            __syncwarp();
            if (lane == 0) qt_arrive(tc_smem_u32(&w_full[place * PARTS + (GATED ? part : 0)]));
            if (!last && !there) ok = fetch(i + STRIDE, true);
            place += STRIDE;
            if (place >= PLACES) { place -= PLACES; place_phase ^= 1; }
        }
        if (!ok && lane == 0) atomicExch(error, QT_ERR_VALUES);
    } else {
        const int quarter = warp & 3, half = (warp - QT_EPILOGUE) >> 2;
        const int l = quarter * 32 + lane;   // this thread's row of the block's 128 rows of W
        const bool pairs = !((ldc | N) & 1) && !(reinterpret_cast<uintptr_t>(C) & 3);   // (an odd N's last row has no neighbour to be stored with)
        bool ok = true;
        for (int ti = 0; ti < my_tiles; ++ti) {
            const int buf = buffers == 2 ? ti & 1 : 0, use = buffers == 2 ? ti >> 1 : ti;
            if (ok) {
                ok = qt_wait(tc_smem_u32(&acc_full[buf]), (unsigned)(use & 1));
                if (!ok && lane == 0) atomicExch(error, QT_ERR_EPILOGUE);
            }
            asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
            const unsigned acc = tmem + (unsigned)(buf * MATS * sh.n) + ((unsigned)(quarter * 32) << 16);
            const Tile tile = tile_of(ti);
            const int m0 = tile.m0, width = min(sh.n, M - m0), row = tile.w0 + l;
            const float add = bias && row < N && sh.splits == 1 ? bias[row] : 0.f;
#pragma unroll 1
            for (int c0 = half * 16; c0 < width; c0 += 32) {
                unsigned r[MATS][16];
                if (ok) {
#pragma unroll
                    for (int i = 0; i < MATS; ++i) qt_ld16(acc + (unsigned)(i * sh.n + c0), r[i]);
                    asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
                } else {   // (a wait ran out, and the error word says so: NaN rather than what the memory held)
#pragma unroll
                    for (int i = 0; i < MATS; ++i)
#pragma unroll
                        for (int j = 0; j < 16; ++j) r[i][j] = 0x7fc00000u;
                }
                if (sh.splits > 1) {   // [matrix][n][128], in place of the stages
#pragma unroll
                    for (int i = 0; i < MATS; ++i)
#pragma unroll
                        for (int j = 0; j < 16; ++j)
                            asm volatile("st.shared.f32 [%0], %1;\n" ::"r"(tiles + (unsigned)(((i * sh.n + c0 + j) * 128 + l) * 4)), "f"(__uint_as_float(r[i][j])) : "memory");
                    continue;
                }
                float v[16];
                if (!GATED) {
#pragma unroll
                    for (int j = 0; j < 16; ++j) v[j] = __uint_as_float(r[0][j]) + add;
                } else if (act == VX_ACT_SILU) {
#pragma unroll
                    for (int j = 0; j < 16; ++j) v[j] = qt_silu(__uint_as_float(r[0][j])) * __uint_as_float(r[MATS - 1][j]);
                } else {
#pragma unroll
                    for (int j = 0; j < 16; ++j) v[j] = activation(__uint_as_float(r[0][j]), act) * __uint_as_float(r[MATS - 1][j]);
                }
                TO* to = C + (size_t)(m0 + c0) * ldc;
                if (sizeof(TO) == 2 && pairs) {
                    // of two columns the even lanes take the first, with their neighbour's row beside theirs
                    const bool odd = lane & 1;
#pragma unroll
                    for (int j = 0; j < 16; j += 2) {
                        const float o = __shfl_xor_sync(0xffffffffu, odd ? v[j] : v[j + 1], 1);
                        const int c = j + (odd ? 1 : 0);
                        if (row < N && c0 + c < width)
                            *reinterpret_cast<__nv_bfloat162*>(to + (size_t)c * ldc + (row & ~1)) = __floats2bfloat162_rn(odd ? o : v[j], odd ? v[j + 1] : o);
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        if (row < N && c0 + j < width) to[(size_t)j * ldc + row] = from_f32<TO>(v[j]);
                }
            }
            // the accumulator may be overwritten once the epilogue's warps have read it
            asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
            __syncwarp();
            if (lane == 0) qt_arrive(tc_smem_u32(&acc_empty[buf]));
        }
    }
    // All roles meet before the tensor memory goes back; with splits all blocks of the cluster, and all their sums are there.
    __syncwarp();
    asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
    if (sh.splits > 1) tp_cluster_sync();
    else __syncthreads();
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(512u) : "memory");
    }
    if (sh.splits > 1) {
        // each block adds its share of the columns, run after run
        const int w0 = tile0.w0, m0 = tile0.m0;
        const int width = min(sh.n, M - m0), c_end = min(width, (split + 1) * sh.n / sh.splits), c_beg = min(width, split * sh.n / sh.splits);
        for (int e = (int)threadIdx.x; e < (c_end - c_beg) * 128; e += QT_THREADS) {
            const int c = c_beg + (e >> 7), l = e & 127;
            if (w0 + l >= N) continue;
            float a = 0.f, b = 0.f;
            for (int p = 0; p < sh.splits; ++p) {
                a += qt_ld_cluster(tp_map_to_rank(tiles + (unsigned)((c * 128 + l) * 4), (unsigned)p));
                if (GATED) b += qt_ld_cluster(tp_map_to_rank(tiles + (unsigned)(((sh.n + c) * 128 + l) * 4), (unsigned)p));
            }
            C[(size_t)(m0 + c) * ldc + w0 + l] = from_f32<TO>(GATED ? activation(a, act) * b : a + (bias ? bias[w0 + l] : 0.f));
        }
        __syncwarp();
        tp_cluster_sync();   // (a block's sums are read until here)
    }
}

// ---- host side ----
// 32-bit words [rows, words], rows `words` apart, in boxes of 8 rows by `box` words.
static bool qt_make_map(CUtensorMap* map, const void* base, long long rows, long long words, int box) {
    tc_encode_fn enc = tc_encoder();
    if (!enc) return false;
    cuuint64_t dims[2] = {(cuuint64_t)words, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)words * 4};
    cuuint32_t boxes[2] = {(cuuint32_t)box, 8}, steps[2] = {1, 1};
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, const_cast<void*>(base), dims, strides, boxes, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <bool GATED, typename TO>
static int qt_launch(const QtMaps& maps, const float* bias, TO* C, int M, int N, int blocks, int ldc, int act, int group, int w_ready,
                     const QtShape& sh, size_t smem, int teams, int* error, cudaStream_t stream) {
    auto kernel = gemm_q4_tc_kernel<GATED, TO>;
    static bool configured[VX_MAX_DEVICES];
    if (int rc = vx_configure_smem(kernel, 226 * 1024, configured)) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(teams * sh.splits));
    cfg.blockDim = dim3(QT_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (vx_pdl_is_enabled() && ((vx_pdl_mask() >> VX_K_GEMM) & 1)) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (sh.splits > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = sh.splits;
        attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
        ++n;
    }
    cfg.attrs = attr;
    cfg.numAttrs = n;
    cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, maps, bias, C, M, N, blocks, ldc, act, group, w_ready, sh, error);
    if (e != cudaSuccess) return (int)e;
    VX_LAUNCH_CHECK();
    return VX_OK;
}

// With a tile's shape: n a multiple of 16 up to 256 (gated 128), splits up to 8.  The other arguments as in vx_gemm_q4.
extern "C" int vx_gemm_q4_tc_shape(const void* x, const void* codes, const void* affine, const void* codes1, const void* affine1, const float* bias,
                                   void* out, int M, int N, int K, int ldx, int ldo, int group, int act, int out_dtype, int w_ready, int n,
                                   int splits, int* error, cudaStream_t stream) {
    if (M <= 0 || N <= 0) return VX_OK;
    if (M > Q4_MOST || N > Q4_MOST || K > QT_MOST_K) return VX_ERR_LIMIT;
    const int mats = codes1 ? 2 : 1, blocks = (K + 63) / 64, steps = (blocks + 1) / 2;
    if (K <= 0 || !error || n < 16 || n > 256 / mats || (n & 15) || splits < 1 || splits > 8 || splits > steps) return VX_ERR_SHAPE;
    if ((group != 32 && group != 64 && group != 128) || K % group || ldx < K || ldo < N) return VX_ERR_SHAPE;
    if (codes1 && (!affine1 || bias || act < 0 || act > VX_ACT_LAST)) return VX_ERR_SHAPE;
    if (out_dtype != VX_BF16 && (out_dtype != VX_F32 || codes1)) return VX_ERR_DTYPE;
    if (ldx & 7 || (((uintptr_t)x) | ((uintptr_t)codes) | ((uintptr_t)affine) | ((uintptr_t)codes1) | ((uintptr_t)affine1)) & 15) return VX_ERR_ALIGN;
    static int sm_counts[VX_MAX_DEVICES];
    const int sms = vx_sm_count(sm_counts);
    const long long tiles = (long long)((N + 127) / 128) * ((M + n - 1) / n);
    if (tiles > 0x7fffff || (tiles / sms + 1) * steps > 0x7fffffff) return VX_ERR_LIMIT;   // (a block counts its steps in 31 bits)
    QtShape sh;
    sh.n = n;
    sh.steps = (steps + splits - 1) / splits;
    sh.splits = (steps + sh.steps - 1) / sh.steps;   // (no run is empty)
    const int stage = n * (QT_K * 2) + mats * (QT_CODES + QT_AFFINE), stages = QT_ROOM / stage;
    sh.stages = stages > QT_MAX_STAGES ? QT_MAX_STAGES : stages;
    size_t bytes = (size_t)sh.stages * stage;
    const size_t sums = (size_t)mats * n * 512;
    if (sh.splits > 1 && bytes < sums) bytes = sums;
    static_assert(QT_LEAST + 84 * 1024 > 228 * 1024, "no block that takes tensor memory fits beside one of these");
    if (bytes < QT_LEAST) bytes = QT_LEAST;
    QtMaps maps;
    const long long wt = (N + 15) / 16, words = (long long)blocks * Q4_BLOCK_WORDS, pairs = (long long)blocks * 64 / group * 16;
    const int box = QT_K / group * 16;
    if (!tc_make_map(&maps.x, x, M, K, ldx, n) || !qt_make_map(&maps.codes[0], codes, wt, words, 2 * Q4_BLOCK_WORDS) ||
        !qt_make_map(&maps.affine[0], affine, wt, pairs, box))
        return VX_ERR_DRIVER;
    maps.codes[1] = maps.codes[0];
    maps.affine[1] = maps.affine[0];
    if (codes1 && (!qt_make_map(&maps.codes[1], codes1, wt, words, 2 * Q4_BLOCK_WORDS) || !qt_make_map(&maps.affine[1], affine1, wt, pairs, box)))
        return VX_ERR_DRIVER;
    const int teams = sh.splits > 1 ? (int)tiles : (int)(tiles < sms ? tiles : sms);
#define QT_GO(G_, T_) qt_launch<G_, T_>(maps, bias, (T_*)out, M, N, blocks, ldo, act, group, w_ready, sh, bytes + 1024, teams, error, stream)
    if (out_dtype == VX_F32) return QT_GO(false, float);
    return codes1 ? QT_GO(true, bf16) : QT_GO(false, bf16);
#undef QT_GO
}

// Clusters of `blocks` blocks, each of which fills an SM, that run at once (a cluster lies within a group of SMs).
static int qt_clusters(int blocks, int sms) {
    static int cache[VX_MAX_DEVICES][9];
    const int dev = vx_current_device();
    if (dev < 0) return sms / blocks / 2;
    int& n = cache[dev][blocks];
    if (!n) {
        static bool configured[VX_MAX_DEVICES];
        auto kernel = gemm_q4_tc_kernel<false, bf16>;
        cudaLaunchAttribute attr;
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = blocks;
        attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)(blocks * sms));
        cfg.blockDim = dim3(QT_THREADS);
        cfg.dynamicSmemBytes = 222 * 1024;
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
        int found = 0;
        if (vx_configure_smem(kernel, 226 * 1024, configured) != VX_OK || cudaOccupancyMaxActiveClusters(&found, kernel, &cfg) != cudaSuccess || found <= 0) {
            cudaGetLastError();
            found = sms / blocks / 2;
        }
        n = found;
    }
    return n;
}

// The tile: rows of x (n) and runs of k, the least time by rounds of the SMs.  A step of 128 k takes 0.27 us + 2.1 ns a row of x (gated
// 0.55 + 3 ns), adding the runs' sums 1.2 us (four runs: 1.5) + 17 ns a row, and writing a tile 8 ns a row (gated 25), once, or in every
// round where there is room for one accumulator only; 4.5 us besides.  Measured and so, us, runs
// 1 / 2 / 4: 32 x 4096 x 4096 14.6, 10.6, 9.6 (15.3, 11.0, 9.7); 128 x 4096 x 4096 19.1, 15.4, 12.4 (21.7, 15.8, 12.9); 64 x 4096 x 12288 42.5,
// 25.5, 17.6 (43.3, 25.8, 17.2); gated 32 x 9728 x 2560 16.8, whole (17.4).  Three runs, or more clusters than run at once, make some wait
// for the others: 32 x 6144 x 4096 in two runs 11.8, in three 18.8.
struct QtPlan { int n, splits; };
static QtPlan qt_plan(int M, int N, int K, bool gated, int sms) {
    const int steps = (K + QT_K - 1) / QT_K, wtiles = (N + 127) / 128, most = gated ? 128 : 256;
    QtPlan best = {};
    double least = 0;
    for (int rows = most, last = 0; rows >= 16; rows -= 16) {
        const int xt = (M + rows - 1) / rows, n = ((M - 1) / xt + 16) & ~15;   // (as even as xt tiles can be)
        if (n == last) continue;
        last = n;
        const long long tiles = (long long)wtiles * ((M + n - 1) / n);
        const double step = gated ? 0.55 + 0.003 * n : 0.27 + 0.0021 * n;
        for (int splits = 1; splits <= 4; splits *= 2) {
            if (splits > 1 && (steps < 2 * splits || tiles > qt_clusters(splits, sms))) break;
            const long long rounds = splits > 1 ? 1 : (tiles + sms - 1) / sms;
            const double cost = (double)rounds * ((steps + splits - 1) / splits) * step + (splits == 1 ? 0 : (splits == 2 ? 1.2 : 1.5) + 0.017 * n) +
                                (gated ? 0.025 : 0.008) * n * (n * (gated ? 4 : 2) > QT_PLACES_AT ? rounds : 1);
            if (!best.n || cost < least) { best = QtPlan{n, splits}; least = cost; }
        }
    }
    return best;
}

// The product with that tile: the arguments as above.
extern "C" int vx_gemm_q4_tc(const void* x, const void* codes, const void* affine, const void* codes1, const void* affine1, const float* bias,
                             void* out, int M, int N, int K, int ldx, int ldo, int group, int act, int out_dtype, int w_ready, int* error,
                             cudaStream_t stream) {
    if (M <= 0 || N <= 0) return VX_OK;
    if (K <= 0) return VX_ERR_SHAPE;
    if (M > Q4_MOST || N > Q4_MOST || K > QT_MOST_K) return VX_ERR_LIMIT;
    static int sm_counts[VX_MAX_DEVICES];
    const QtPlan p = qt_plan(M, N, K, codes1 != nullptr, vx_sm_count(sm_counts));
    return vx_gemm_q4_tc_shape(x, codes, affine, codes1, affine1, bias, out, M, N, K, ldx, ldo, group, act, out_dtype, w_ready, p.n, p.splits, error,
                               stream);
}
