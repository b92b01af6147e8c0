// The products with matrices held in four bits (q4.cuh) for more than a few rows, on the fifth-generation tensor cores:
// out[M,N] = x[M,K] W^T (+ bias), and out[M,N] = act(x Wg^T) * (x Wu^T).
//
// The operands are turned, out^T = W x^T: 128 rows of W on the M side of tcgen05.mma, n rows of x as its columns.  W is the instruction's A
// operand, and A may lie in tensor memory: a lane is a row, a column two neighbouring k.  So a thread makes its own row's 64 k of a
// step from 32 bytes of codes in registers and stores them with one tcgen05.st; W as bfloat16 exists in tensor memory only.
// Gated, gate and up rows of a feature are the same lane's in two accumulators, and the epilogue joins them without an exchange.
//
// Warps of a block:
//   warp 0       producer: x (128-byte swizzle), codes, scales and offsets of 64 k a stage by TMA; W's first stages are asked for before the
//                wait for the kernel launched before this one (if the caller says that W is ready);
//   warp 1       tensor memory; issues the products;
//   warps 2-9    two groups of four that make W's values, step by step in turn (gated: one makes gate, the other up), into eight places in
//                tensor memory;
//   warps 10-17  epilogue.
// K may be cut into `splits` runs, one to each block of a cluster, whose float32 sums are added in ascending order through distributed
// shared memory: the same result on every run.
// Every wait on an mbarrier is bounded; a block whose wait runs out records a code in the caller's error word and writes NaN, the other roles run
// out of their own, all meet, free their tensor memory and return.
//
// Tensor memory is taken before the wait for the kernel before and before the next one is let in (gemm_turned.cu says why that is safe:
// every kernel that takes some after it lets the next one in fills an SM's shared memory, and so do these blocks all but).
#include "q4.cuh"
#include "tcgen05_pair.cuh"

#define QT_THREADS 576
#define QT_MAKERS 2          // first warp of those that make W's values
#define QT_EPILOGUE 10       // ... and of the epilogue's
#define QT_PLACES 8          // places for 64 k of W's values in tensor memory, 32 columns each, behind the accumulators
#define QT_PLACES_AT 256
#define QT_MAX_STAGES 12
#define QT_CODES 4096        // bytes of a stage: codes of 128 rows by 64 k
#define QT_AFFINE 1024       // ... room for their scales and offsets (512, or 1024 for groups of 32)
#define QT_ERR_PRODUCER 10
#define QT_ERR_MMA 11
#define QT_ERR_EPILOGUE 12
#define QT_ERR_VALUES 13

struct QtShape {
    int n;         // rows of x in a tile
    int splits;    // runs of k
    int kbs;       // steps of 64 k of a run
    int stages;
};
struct QtMaps { CUtensorMap x, codes[2], affine[2]; };

__device__ __forceinline__ void qt_st32(unsigned taddr, const unsigned (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};\n"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]),
        "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
    asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory");
}
__device__ __forceinline__ void qt_ld16(unsigned taddr, unsigned (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
          "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr) : "memory");
}
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
// Four products of 16 k: A in tensor memory (8 columns each), B in a swizzled K-major tile.
__device__ __forceinline__ void qt_mma_step(unsigned d, unsigned a, unsigned b_lo, unsigned idesc, unsigned add) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
        asm volatile("{\n .reg .pred p;\n .reg .b64 b;\n setp.ne.b32 p, %4, 0;\n mov.b64 b, {%2, %5};\n"
                     " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n}\n"
                     ::"r"(d), "r"(a + 8 * k), "r"(b_lo + 2 * k), "r"(idesc), "r"(k ? 1u : add), "r"(TC_DESC_HI) : "memory");
}

template <bool GATED, typename TO>
__global__ void __launch_bounds__(QT_THREADS, 1)
gemm_q4_tc_kernel(const __grid_constant__ QtMaps maps, const float* __restrict__ bias, TO* __restrict__ C, int M, int N, int blocks, int ldc, int act,
                  int group, int w_ready, const QtShape sh, int* __restrict__ error) {
    constexpr int MATS = GATED ? 2 : 1;
    extern __shared__ unsigned char qt_raw[];
    __shared__ __align__(8) unsigned long long full_bar[QT_MAX_STAGES], empty_bar[QT_MAX_STAGES], w_full[QT_PLACES], w_empty[QT_PLACES], acc_full, acc_empty;
    __shared__ unsigned tmem_s;
    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int split = sh.splits > 1 ? (int)tp_cluster_rank() : 0;
    const unsigned x_bytes = (unsigned)sh.n * (TC_BK * 2), w_bytes = QT_CODES + (group == 32 ? 1024u : 512u);   // (loaded, a matrix)
    const unsigned stage_bytes = x_bytes + MATS * (QT_CODES + QT_AFFINE);
    const unsigned tiles = (tc_smem_u32(qt_raw) + 1023) & ~1023u;
    const int kb0 = split * sh.kbs, nkb = min(blocks - kb0, sh.kbs);
    const int xt = (M + sh.n - 1) / sh.n, total = (N + 127) / 128 * xt;
    const int me = (int)blockIdx.x / sh.splits, teams = (int)gridDim.x / sh.splits;
    const int my_tiles = (total - me + teams - 1) / teams;
    // tiles that are worked on at the same time share rows of W
    auto w0_of = [&](int ti) { return (me + ti * teams) / xt * 128; };
    auto m0_of = [&](int ti) { return (me + ti * teams) % xt * sh.n; };
    if (threadIdx.x == 0) {
        for (int s = 0; s < sh.stages; ++s) {
            tc_mbar_init(tc_smem_u32(&full_bar[s]), 1);    // the producer, with the bytes
            tc_mbar_init(tc_smem_u32(&empty_bar[s]), 1);   // the commit of the products that read the stage's x
        }
        for (int p = 0; p < QT_PLACES; ++p) {
            tc_mbar_init(tc_smem_u32(&w_full[p]), 4);      // the four warps that fill it
            tc_mbar_init(tc_smem_u32(&w_empty[p]), 1);     // the commit of the products that read it
        }
        tc_mbar_init(tc_smem_u32(&acc_full), 1);
        tc_mbar_init(tc_smem_u32(&acc_empty), 8);          // the epilogue's warps
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

    auto load = [&](int ti, int kb, int s, bool of_w, bool of_x) {
        const unsigned bar = tc_smem_u32(&full_bar[s]), st = tiles + (unsigned)s * stage_bytes;
        if (of_w) {
            tc_mbar_expect_tx(bar, x_bytes + MATS * w_bytes);
#pragma unroll
            for (int i = 0; i < MATS; ++i) {
                const unsigned at = st + x_bytes + i * (QT_CODES + QT_AFFINE);
                tc_tma_load_2d(at, &maps.codes[i], (kb0 + kb) * Q4_BLOCK_WORDS, w0_of(ti) / 16, bar);
                tc_tma_load_2d(at + QT_CODES, &maps.affine[i], (kb0 + kb) * 64 / group * 16, w0_of(ti) / 16, bar);
            }
        }
        if (of_x) tc_tma_load_2d(st, &maps.x, (kb0 + kb) * TC_BK, m0_of(ti), bar);
    };
    const int ahead = w_ready ? min(sh.stages, nkb) : 0;   // stages whose W is asked for before the wait
    if (warp == 0)
        for (int kb = 0; kb < ahead; ++kb)
            if (tc_elect()) load(0, kb, kb, true, false);
    pdl_wait();
    if (warp == 0)
        for (int kb = 0; kb < ahead; ++kb)
            if (tc_elect()) load(0, kb, kb, false, true);
    __syncwarp();
    pdl_trigger();

    if (warp == 0) {
        int s = ahead == sh.stages ? 0 : ahead;
        unsigned phase = ahead == sh.stages ? 0 : 1;   // (the first time round a stage is free: the phase before the first has ended)
        for (int ti = 0; ti < my_tiles; ++ti)
            for (int kb = ti ? 0 : ahead; kb < nkb; ++kb) {
                if (!tc_warp_wait(tc_smem_u32(&empty_bar[s]), phase)) {
                    if (lane == 0) atomicExch(error, QT_ERR_PRODUCER);
                    ti = my_tiles;
                    break;
                }
                if (tc_elect()) load(ti, kb, s, true, true);
                if (++s == sh.stages) { s = 0; phase ^= 1; }
            }
    } else if (warp == 1) {
        // float32 accumulator, bfloat16 operands, both K-major, N = n, M = 128
        const unsigned idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((unsigned)(sh.n >> 3) << 17) | (8u << 24);
        int s = 0, place = 0;
        unsigned phase = 0, place_phase = 0;
        bool ok = true;
        for (int ti = 0; ok && ti < my_tiles; ++ti) {
            ok = !ti || tc_warp_wait(tc_smem_u32(&acc_empty), (unsigned)((ti - 1) & 1));
            asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
            for (int kb = 0; ok && kb < nkb; ++kb) {
                ok = tc_warp_wait(tc_smem_u32(&full_bar[s]), phase);
                const unsigned xd = tc_desc_lo(tiles + (unsigned)s * stage_bytes);
#pragma unroll
                for (int i = 0; i < MATS; ++i) {
                    ok = ok && tc_warp_wait(tc_smem_u32(&w_full[place]), place_phase);
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
                    if (tc_elect()) {
                        qt_mma_step(tmem + (unsigned)(i * sh.n), tmem + QT_PLACES_AT + place * 32, xd, idesc, kb > 0);
                        tc_commit(tc_smem_u32(&w_empty[place]));
                        if (i == MATS - 1) tc_commit(tc_smem_u32(&empty_bar[s]));
                    }
                    if (++place == QT_PLACES) { place = 0; place_phase ^= 1; }
                }
                if (++s == sh.stages) { s = 0; phase ^= 1; }
            }
            if (ok && tc_elect()) tc_commit(tc_smem_u32(&acc_full));
        }
        if (!ok && lane == 0) atomicExch(error, QT_ERR_MMA);
    } else if (warp < QT_EPILOGUE) {
        const int team = (warp - QT_MAKERS) >> 2, quarter = warp & 3, row = quarter * 32 + lane;
        const unsigned codes_at = x_bytes + (GATED ? team * (QT_CODES + QT_AFFINE) : 0) + (row >> 4) * 512 + (row & 7) * 16 + (row >> 3 & 1) * 8;
        const unsigned affine_at = x_bytes + (GATED ? team * (QT_CODES + QT_AFFINE) : 0) + QT_CODES + (row >> 4) * (group == 32 ? 128 : 64) +
                                   (row & 7) * 8 + (row >> 3 & 1) * 4;
        const unsigned second = group == 32 ? 64 : 0;   // (of 64 k the second half's group)
        const unsigned lanes = tmem + QT_PLACES_AT + ((unsigned)(quarter * 32) << 16);
        const int steps = my_tiles * nkb;
        int s = GATED ? 0 : team % sh.stages, place = team;
        unsigned phase = 0, place_phase = 1;   // (the first time round a place is free)
        for (int i = GATED ? 0 : team; i < steps; i += GATED ? 1 : 2) {
            if (!tc_warp_wait(tc_smem_u32(&full_bar[s]), phase)) {
                if (lane == 0) atomicExch(error, QT_ERR_VALUES);
                break;
            }
            const unsigned st = tiles + (unsigned)s * stage_bytes;
            const unsigned a0 = qt_lds4(st + affine_at), a1 = qt_lds4(st + affine_at + second);
            uint2 q[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) q[t] = qt_lds8(st + codes_at + t * 128);
            unsigned w[32];
            const unsigned s0 = q4_scale(a0), b0 = q4_offset(a0), s1 = q4_scale(a1), b1 = q4_offset(a1);
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                unsigned v[4];
                q4_values(q[t].x, t < 2 ? s0 : s1, t < 2 ? b0 : b1, v);
                w[8 * t] = v[0]; w[8 * t + 1] = v[1]; w[8 * t + 2] = v[2]; w[8 * t + 3] = v[3];
                q4_values(q[t].y, t < 2 ? s0 : s1, t < 2 ? b0 : b1, v);
                w[8 * t + 4] = v[0]; w[8 * t + 5] = v[1]; w[8 * t + 6] = v[2]; w[8 * t + 7] = v[3];
            }
            if (!tc_warp_wait(tc_smem_u32(&w_empty[place]), place_phase)) {
                if (lane == 0) atomicExch(error, QT_ERR_VALUES);
                break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
            qt_st32(lanes + place * 32, w);
            asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
            __syncwarp();
            if (lane == 0) qt_arrive(tc_smem_u32(&w_full[place]));
            place += 2;
            if (place >= QT_PLACES) { place -= QT_PLACES; place_phase ^= 1; }
            s += GATED ? 1 : 2;
            if (s >= sh.stages) { s -= sh.stages; phase ^= 1; }
        }
    } else {
        const int quarter = warp & 3, half = (warp - QT_EPILOGUE) >> 2;
        const int l = quarter * 32 + lane;   // this thread's row of the block's 128 rows of W
        const bool pairs = !(ldc & 1);
        bool ok = true;
        for (int ti = 0; ti < my_tiles; ++ti) {
            if (ok) {
                ok = tc_warp_wait(tc_smem_u32(&acc_full), (unsigned)(ti & 1));
                if (!ok && lane == 0) atomicExch(error, QT_ERR_EPILOGUE);
            }
            asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
            const unsigned acc = tmem + ((unsigned)(quarter * 32) << 16);
            const int w0 = w0_of(ti), m0 = m0_of(ti), width = min(sh.n, M - m0), row = w0 + l;
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
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const float a = __uint_as_float(r[0][j]);
                    v[j] = GATED ? activation(a, act) * __uint_as_float(r[MATS - 1][j]) : a + add;
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
            if (lane == 0) qt_arrive(tc_smem_u32(&acc_empty));
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
        const int w0 = w0_of(0), m0 = m0_of(0);
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

// With a tile's shape: n a multiple of 16 up to 256 (gated 128), splits up to 8.  The other arguments as in vx_gemm_q4, checked there.
extern "C" int vx_gemm_q4_tc_shape(const void* x, const void* codes, const void* affine, const void* codes1, const void* affine1, const float* bias,
                                   void* out, int M, int N, int K, int ldx, int ldo, int group, int act, int out_dtype, int w_ready, int n,
                                   int splits, int* error, cudaStream_t stream) {
    if (M <= 0 || N <= 0) return VX_OK;
    const int mats = codes1 ? 2 : 1, blocks = (K + 63) / 64;
    if (K <= 0 || !error || n < 16 || n > 256 / mats || (n & 15) || splits < 1 || splits > 8 || splits > blocks) return VX_ERR_SHAPE;
    if ((group != 32 && group != 64 && group != 128) || K % group || ldx < K || ldo < N) return VX_ERR_SHAPE;
    if (codes1 && (!affine1 || bias || act < 0 || act > VX_ACT_LAST)) return VX_ERR_SHAPE;
    if (out_dtype != VX_BF16 && (out_dtype != VX_F32 || codes1)) return VX_ERR_DTYPE;
    if (ldx & 7 || (((uintptr_t)x) | ((uintptr_t)codes) | ((uintptr_t)affine) | ((uintptr_t)codes1) | ((uintptr_t)affine1)) & 15) return VX_ERR_ALIGN;
    QtShape sh;
    sh.n = n;
    sh.kbs = (blocks + splits - 1) / splits;
    sh.splits = (blocks + sh.kbs - 1) / sh.kbs;   // (no run is empty)
    const int stage = n * (TC_BK * 2) + mats * (QT_CODES + QT_AFFINE), stages = 220 * 1024 / stage;
    sh.stages = stages > QT_MAX_STAGES ? QT_MAX_STAGES : stages;
    // An even number: plain, a group of makers then meets the same stages again and again, and sees every phase of their mbarriers.  (With
    // an odd one it would wait for a stage's phase whose predecessor only the other group has seen end.)
    sh.stages &= ~1;
    size_t bytes = (size_t)sh.stages * stage;
    const size_t sums = (size_t)mats * n * 512;
    if (sh.splits > 1 && bytes < sums) bytes = sums;
    if (bytes < 120 * 1024) bytes = 120 * 1024;   // (one block an SM: the tensor memory is one block's)
    if (bytes > 222 * 1024) return VX_ERR_SHAPE;
    QtMaps maps;
    const long long wt = (N + 15) / 16, words = (long long)blocks * Q4_BLOCK_WORDS, pairs = (long long)blocks * 64 / group * 16;
    const int box = group == 32 ? 32 : 16;
    if (words > 0xffffffffLL) return VX_ERR_LIMIT;
    if (!tc_make_map(&maps.x, x, M, K, ldx, n) || !qt_make_map(&maps.codes[0], codes, wt, words, Q4_BLOCK_WORDS) ||
        !qt_make_map(&maps.affine[0], affine, wt, pairs, box))
        return VX_ERR_DRIVER;
    maps.codes[1] = maps.codes[0];
    maps.affine[1] = maps.affine[0];
    if (codes1 && (!qt_make_map(&maps.codes[1], codes1, wt, words, Q4_BLOCK_WORDS) || !qt_make_map(&maps.affine[1], affine1, wt, pairs, box))) return VX_ERR_DRIVER;
    static int sm_counts[VX_MAX_DEVICES];
    const int sms = vx_sm_count(sm_counts);
    const long long tiles = (long long)((N + 127) / 128) * ((M + n - 1) / n);
    if (tiles > 0x7fffff) return VX_ERR_LIMIT;
    const int teams = sh.splits > 1 ? (int)tiles : (int)(tiles < sms ? tiles : sms);
#define QT_GO(G_, T_) qt_launch<G_, T_>(maps, bias, (T_*)out, M, N, blocks, ldo, act, group, w_ready, sh, bytes + 1024, teams, error, stream)
    if (out_dtype == VX_F32) return QT_GO(false, float);
    return codes1 ? QT_GO(true, bf16) : QT_GO(false, bf16);
#undef QT_GO
}

// The product with a tile that fits: the arguments as above.
extern "C" int vx_gemm_q4_tc(const void* x, const void* codes, const void* affine, const void* codes1, const void* affine1, const float* bias,
                             void* out, int M, int N, int K, int ldx, int ldo, int group, int act, int out_dtype, int w_ready, int* error,
                             cudaStream_t stream) {
    if (M <= 0 || N <= 0) return VX_OK;
    static int sm_counts[VX_MAX_DEVICES];
    const int sms = vx_sm_count(sm_counts), most = codes1 ? 128 : 256, blocks = (K + 63) / 64;
    const int xt = (M + most - 1) / most, n = ((M + xt - 1) / xt + 15) & ~15, tiles = (N + 127) / 128 * xt;
    int splits = sms / tiles;
    if (splits > blocks / 4) splits = blocks / 4;
    splits = splits < 1 ? 1 : (splits > 8 ? 8 : splits);
    return vx_gemm_q4_tc_shape(x, codes, affine, codes1, affine1, bias, out, M, N, K, ldx, ldo, group, act, out_dtype, w_ready, n, splits, error, stream);
}
