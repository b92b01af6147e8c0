// out[M,N] = x[M,K] W^T (+ bias) and out[M,N] = act(x Wg^T) * (x Wu^T) with matrices held in four bits (q4.cuh), for a few rows: the
// products of a decode step, whose floor is reading codes, scales and offsets once.
//
// As in the bfloat16 product of a few rows, out^T = W x^T on mma.sync.m16n8k16: 16 rows of W fill the instruction's 16-row side, 8 rows of x its
// 8-column side (NT such tiles of columns for up to 32 rows).  A block forms 16 rows of W at a time, or 32, for which x is read once (gated: 16
// gate rows and their up rows, so that both sums of a feature meet in it), over the whole of K: its warps have a run of code blocks each.  A
// warp's steps of four code blocks come by cp.async into a ring of its own, two ahead and across tiles; a lane's 16 bytes of a code block are its
// fragments of four products, which it makes bfloat16 in registers.  (Through registers alone the loads share what the warp waits on with
// those of x, and every block waited for memory.)  k is permuted the same way for x, of which a lane reads 32 neighbouring bytes of a
// row, a code block ahead, through L1.  The warps' sums are added in shared memory in warp order: the same result on every run, and a row's
// result does not depend on the rows beside it.  (A warp's sum is the tensor cores' float32, cut towards zero every 16 k: root mean square error of a
// float32 result, relative, 2e-7 at 2,560 k, 1.1e-6 at 12,288.)
//
// What bounds it: no unit alone.  Under the profiler 55 to 59 % of the issue slots are used, 48 to 51 % of the pipe for shifts and logic, 37 to 43 %
// of that for packed multiply-adds, and some 60 % of the copy rate.  A warp's chain of load, values and products is covered by 15 warps an SM only in part,
// every tile reads x again through L1, and some SMs have a tile more than others.  Eight weights take 15 instructions, a code block 87 to 94 for a
// warp.  us in a captured row of calls, and of the copy rate of 6,549 GB/s: gated 12288 x 4096 1 row 14.8, 58 %; gated 17408 x 5120 8 rows 25.3, 61 %;
// 151936 x 2560 4 rows to float32 48.7, 69 %; 4096 x 12288 1 row 9.0, 48 %.
#include "q4.cuh"

__device__ __forceinline__ unsigned q4_smem(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void q4_copy16(unsigned to, const char* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ uint4 q4_lds16(unsigned at) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
    return v;
}
__device__ __forceinline__ uint2 q4_lds8(unsigned at) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];\n" : "=r"(v.x), "=r"(v.y) : "r"(at));
    return v;
}
__device__ __forceinline__ uint4 q4_x16(const bf16* p) {
    uint4 v;
    asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ void q4_mma(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

struct Q4Pair { const unsigned *codes[2], *affine[2]; };   // the matrix, or gate and up

// What a block forms at a time: 16 rows of W; 32 rows (two tiles, for which x is read once); 16 gate rows and their up rows.
enum { Q4_ONE = 0, Q4_TWO = 1, Q4_GATED = 2 };
// A warp's step: BLOCKS code blocks, neighbours along K, with their scales and offsets; of both tiles where there are two.
template <int FORM, int GROUP, int BLOCKS> struct Q4Step {
    static constexpr int mats = FORM == Q4_ONE ? 1 : 2, codes = BLOCKS * 512, affine = BLOCKS * 64 * 64 / GROUP, bytes = codes + affine;
};

// A block's shared memory: the warps' rings, and their sums of a tile, in two buffers where these are small and leave room for PER_SM blocks
// on an SM (which has 228 KB, of which each block takes 1 KB more than its own).
template <int FORM, int GROUP, int NT, int WARPS, int BLOCKS, int DEPTH, int PER_SM> struct Q4Room {
    static constexpr int mats = Q4Step<FORM, GROUP, BLOCKS>::mats, ring = WARPS * DEPTH * mats * Q4Step<FORM, GROUP, BLOCKS>::bytes,
                         sums = mats * WARPS * 16 * (8 * NT + 1) * 4, share = 228 * 1024 / PER_SM - 1024,
                         buffers = NT <= 2 && ring + 2 * sums <= share ? 2 : 1, bytes = ring + buffers * sums;
    static constexpr bool fits = bytes <= share;
};

template <int FORM, typename TO, int GROUP, int NT, int WARPS, int BLOCKS, int DEPTH, int PER_SM>
__global__ void __launch_bounds__(WARPS * 32, PER_SM)
gemm_q4_kernel(const bf16* __restrict__ x, const Q4Pair w, const float* __restrict__ bias, TO* __restrict__ out, int M, int N, int K, int ldx,
               int ldo, int act, int blocks, int units, int w_ready) {
    typedef Q4Step<FORM, GROUP, BLOCKS> Step;
    constexpr bool GATED = FORM == Q4_GATED, TWO = FORM == Q4_TWO, BOTH = FORM != Q4_ONE;
    static_assert(BLOCKS * 64 % GROUP == 0, "a step holds whole groups");
    constexpr int MATS = Step::mats, SLOT = MATS * Step::bytes;
    extern __shared__ __align__(16) unsigned char q4_ring[];
    constexpr int RED = Q4Room<FORM, GROUP, NT, WARPS, BLOCKS, DEPTH, PER_SM>::buffers;
    typedef float Sums[MATS][WARPS][16][8 * NT + 1];
    Sums* red = reinterpret_cast<Sums*>(q4_ring + WARPS * DEPTH * SLOT);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, t = lane & 3;
    // the warp's code blocks of a tile: neighbours, as many for every warp as there can be (whole groups)
    constexpr int UNIT = GROUP == 128 ? 2 : 1;
    const int lo = warp * (blocks / UNIT) / WARPS * UNIT, mine = (warp + 1) * (blocks / UNIT) / WARPS * UNIT - lo;
    const int my_tiles = mine > 0 ? (units - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x : 0;
    const size_t tile_codes = (size_t)blocks * (Q4_BLOCK_WORDS * 4), tile_affine = (size_t)blocks * (64 * 64) / GROUP;
    const size_t unit_codes = tile_codes << TWO, unit_affine = tile_affine << TWO;
    const unsigned ring = q4_smem(q4_ring) + warp * (DEPTH * SLOT);
    // what is asked for next
    const char* ask_q = reinterpret_cast<const char*>(w.codes[0]) + blockIdx.x * unit_codes + (size_t)lo * 512 + lane * 16;
    const char* ask_a = reinterpret_cast<const char*>(w.affine[0]) + blockIdx.x * unit_affine + (size_t)lo * (64 * 64) / GROUP + lane * 16;
    // from a tile to its second: the up matrix's, or the next (of the matrix's last there may be none: then the first again, not written)
    ptrdiff_t up_q, up_a;
    const int tiles_of_w = (N + 15) / 16;
    auto second_of = [&](int unit) {
        if (GATED) {
            up_q = reinterpret_cast<const char*>(w.codes[1]) - reinterpret_cast<const char*>(w.codes[0]);
            up_a = reinterpret_cast<const char*>(w.affine[1]) - reinterpret_cast<const char*>(w.affine[0]);
        } else if (TWO) {
            const bool there = 2 * unit + 1 < tiles_of_w;
            up_q = there ? tile_codes : 0;
            up_a = there ? tile_affine : 0;
        }
    };
    int ask_unit = blockIdx.x;
    second_of(ask_unit);
    int ask_left = mine, ask_tiles = my_tiles;
    unsigned ask_at = ring + lane * 16;
    auto ask = [&]() {
        if (ask_tiles > 0) {
#pragma unroll
            for (int b = 0; b < BLOCKS; ++b)
                if (b < ask_left) {
                    q4_copy16(ask_at + b * 512, ask_q + b * 512);
                    if (BOTH) q4_copy16(ask_at + Step::bytes + b * 512, ask_q + up_q + b * 512);
                }
            if (lane * 16 < min(BLOCKS, ask_left) * (64 * 64 / GROUP)) {
                q4_copy16(ask_at + Step::codes, ask_a);
                if (BOTH) q4_copy16(ask_at + Step::bytes + Step::codes, ask_a + up_a);
            }
            ask_q += Step::codes;
            ask_a += Step::affine;
            ask_left -= BLOCKS;
            if (ask_left <= 0) {   // on to the next tile
                const int steps = (mine + BLOCKS - 1) / BLOCKS;
                ask_q += gridDim.x * unit_codes - (size_t)steps * Step::codes;
                ask_a += gridDim.x * unit_affine - (size_t)steps * Step::affine;
                ask_left = mine;
                --ask_tiles;
                if (TWO) second_of(ask_unit += gridDim.x);
            }
        }
        asm volatile("cp.async.commit_group;\n" ::: "memory");
        ask_at = ask_at == ring + lane * 16 + (DEPTH - 1) * SLOT ? ring + lane * 16 : ask_at + SLOT;
    };
    if (w_ready)
#pragma unroll 1
        for (int d = 0; d < DEPTH; ++d) ask();
    pdl_wait();
    pdl_trigger();
    if (!w_ready)
#pragma unroll 1
        for (int d = 0; d < DEPTH; ++d) ask();
    // Rows of x beyond the last are the last again: what comes of them is not written.
    const bf16* xr[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) xr[j] = x + (size_t)min(r + 8 * j, M - 1) * ldx + lo * 64 + t * 16;
    const bool cut = (K & 63) && lo + mine == blocks;   // the warp's last block reaches beyond K: x counts as 0 there (K is a multiple of the group)
    // block `at` from where the rows are; `last`: the tile's last block, from there
    auto fetch_x = [&](uint4 (&v)[NT][2], int at, int last) {
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            if (GROUP == 32 && cut && at == last && t >= 2) {
                v[j][0] = v[j][1] = make_uint4(0u, 0u, 0u, 0u);
            } else {
                v[j][0] = q4_x16(xr[j] + at * 64);
                v[j][1] = q4_x16(xr[j] + at * 64 + 8);
            }
        }
    };
    constexpr bool X_AHEAD = NT <= 2;   // x of the next block is asked for before a block's products (with four tiles of columns the registers are short)
    uint4 xn[NT][2];
    if (X_AHEAD && mine > 0) fetch_x(xn, 0, mine - 1);
    const unsigned own = (t * 8 + r) * 16, own_affine = Step::codes + r * 8 + (GROUP == 32 ? (t >> 1) * 64 : 0);
    unsigned at = ring;
    const int block_tiles = (units - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x;
    for (int ti = 0; ti < block_tiles; ++ti) {
        float acc[MATS][NT][4] = {};
#pragma unroll 1
        for (int left = mine; left > 0; left -= BLOCKS) {
            asm volatile("cp.async.wait_group %0;\n" ::"n"(DEPTH - 1) : "memory");
            __syncwarp();
            auto block = [&](int b) {
                uint4 xv[NT][2];
                if (X_AHEAD) {
#pragma unroll
                    for (int j = 0; j < NT; ++j) { xv[j][0] = xn[j][0]; xv[j][1] = xn[j][1]; }
                    // the next block's: of this step, the next, or the next tile's first
                    const bool more = b + 1 < BLOCKS && (left >= BLOCKS || b + 1 < left);
                    const int at = more ? b + 1 : (left > BLOCKS ? BLOCKS : left - mine);
                    fetch_x(xn, at, left - 1);
                } else {
                    fetch_x(xv, b, left - 1);
                }
#pragma unroll
                for (int i = 0; i < MATS; ++i) {
                    const uint4 q = q4_lds16(at + own + i * Step::bytes + b * 512);
                    const uint2 a = q4_lds8(at + own_affine + i * Step::bytes + (GROUP == 128 ? (b >> 1) * 64 : b * (64 * 64 / GROUP)));
                    const unsigned s0 = q4_scale(a.x), b0 = q4_offset(a.x), s1 = q4_scale(a.y), b1 = q4_offset(a.y);
#pragma unroll
                    for (int word = 0; word < 2; ++word) {
                        unsigned w0[4], w1[4];
                        q4_values<false>(word ? q.y : q.x, s0, b0, w0);
                        q4_values<false>(word ? q.w : q.z, s1, b1, w1);
#pragma unroll
                        for (int j = 0; j < NT; ++j) {
                            q4_mma(acc[i][j], w0[0], w1[0], w0[1], w1[1], xv[j][word].x, xv[j][word].y);
                            q4_mma(acc[i][j], w0[2], w1[2], w0[3], w1[3], xv[j][word].z, xv[j][word].w);
                        }
                    }
                }
            };
            // (A whole step has no branches between its blocks, whose loads can then go ahead of the products before.)
            if (left >= BLOCKS) {
#pragma unroll
                for (int b = 0; b < BLOCKS; ++b) block(b);
            } else {
#pragma unroll
                for (int b = 0; b < BLOCKS - 1; ++b)
                    if (b < left) block(b);
            }
            __syncwarp();   // (the lanes' copies below overwrite what all of them have read)
            ask();
            at = at == ring + (DEPTH - 1) * SLOT ? ring : at + SLOT;
#pragma unroll
            for (int j = 0; j < NT; ++j) xr[j] += BLOCKS * 64;
        }
#pragma unroll
        for (int j = 0; j < NT; ++j) xr[j] -= (mine + BLOCKS - 1) / BLOCKS * (BLOCKS * 64);
        // a lane holds out^T[row r (0, 1) and r + 8 (2, 3)][rows 2 t, 2 t + 1 of x]
        const int buf = ti & (RED - 1);
#pragma unroll
        for (int i = 0; i < MATS; ++i)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int m = 8 * n + 2 * t + (j & 1);
                    if (m < M) red[buf][i][warp][r + 8 * (j >> 1)][m] = acc[i][n][j];
                }
        __syncthreads();   // (with two buffers the sums that are read here are overwritten after the next of these)
        const int unit = blockIdx.x + ti * gridDim.x;
        constexpr int ROWS = TWO ? 32 : 16;
        for (int e = threadIdx.x; e < ROWS * M; e += WARPS * 32) {
            const int row = e % ROWS, m = e / ROWS, n = unit * ROWS + row;
            if (n < N) {
                float v = 0.f, up = 0.f;
#pragma unroll
                for (int i = 0; i < WARPS; ++i) {
                    v += red[buf][TWO ? row >> 4 : 0][i][row & 15][m];
                    if (GATED) up += red[buf][MATS - 1][i][row][m];
                }
                if (bias) v += bias[n];
                out[(size_t)m * ldo + n] = from_f32<TO>(GATED ? activation(v, act) * up : v);
            }
        }
        if (RED == 1) __syncthreads();
    }
    asm volatile("cp.async.wait_all;\n" ::: "memory");
}

static int q4_sms() {
    static int sms[VX_MAX_DEVICES];
    return vx_sm_count(sms);
}

template <int FORM, typename TO, int GROUP, int NT, int WARPS, int BLOCKS, int DEPTH, int PER_SM>
static int q4_go(const bf16* x, const Q4Pair& w, const float* bias, TO* out, int M, int N, int K, int ldx, int ldo, int act, int w_ready,
                 cudaStream_t stream) {
    typedef Q4Room<FORM, GROUP, NT, WARPS, BLOCKS, DEPTH, PER_SM> Room;
    static_assert(Room::fits, "a whole round of blocks is on the SMs at once");
    const int blocks = (K + 63) / 64, rows = FORM == Q4_TWO ? 32 : 16, units = (N + rows - 1) / rows, room = q4_sms() * PER_SM;
    auto kernel = gemm_q4_kernel<FORM, TO, GROUP, NT, WARPS, BLOCKS, DEPTH, PER_SM>;
    static bool configured[VX_MAX_DEVICES];
    if (int rc = vx_configure_smem(kernel, Room::bytes, configured)) return rc;
    VX_LAUNCH_K(VX_K_GEMM, kernel, (unsigned)(units < room ? units : room), WARPS * 32, Room::bytes, stream, x, w, bias, out, M, N, K, ldx, ldo, act, blocks,
                units, w_ready);
    VX_LAUNCH_CHECK();
    return VX_OK;
}

template <bool GATED, typename TO, int GROUP, int NT>
static int q4_launch(const bf16* x, const Q4Pair& w, const float* bias, TO* out, int M, int N, int K, int ldx, int ldo, int act,
                     int w_ready, cudaStream_t stream) {
    const int tiles = (N + 15) / 16, sms = q4_sms();
    // Eight warps a tile, two blocks an SM; three where that lets all tiles be worked on at once; two tiles at a time where there are more; and
    // four warps by four blocks where there are so many that a tile's end, which all of a block's warps wait for, counts more than a tile's length.
    // us, this way and the others: 1 row 4096 x 4096 4.2 (two tiles 4.3, three blocks 4.9); 6144 x 4096 5.3 (two blocks 6.6, two tiles 5.8); 8 rows 7168 x
    // 5120 two tiles 7.9 (one, three blocks 10.1); 4 rows 151936 x 2560 to float32 48.7 (eight warps 53.4, one tile 61.9).  Gated: 1 row 12288 x 4096 14.8
    // (four warps 16.1), 9728 x 2560 9.8 (10.0), 8 rows 17408 x 5120 four warps 25.3 (eight 26.7).
#define Q4_GO(F_, W_, P_) return q4_go<F_, TO, GROUP, NT, W_, 4, 2, P_>(x, w, bias, out, M, N, K, ldx, ldo, act, w_ready, stream)
    constexpr int BOTH = GATED ? Q4_GATED : Q4_TWO;
    constexpr int FOUR = Q4Room<BOTH, GROUP, NT, 4, 4, 2, 4>::fits ? 4 : 3;   // (17 to 32 rows in groups of 32: three blocks fit an SM)
    if (tiles > (GATED ? 6 : 16) * sms) Q4_GO(BOTH, 4, FOUR);
    if constexpr (!GATED) {
        if (tiles <= 2 * sms) Q4_GO(Q4_ONE, 8, 2);
        if (tiles <= 3 * sms) Q4_GO(Q4_ONE, 8, 3);
    }
    Q4_GO(BOTH, 8, 2);
#undef Q4_GO
}

// Rows up to which the kernel above is taken: 16, or 32 where the matrix is small.  us, this way and on tcgen05: 16 rows 4096 x 4096 6.2, 8.9; 4096 x
// 12288 13.4, 14.6; gated 12288 x 4096 21.3, 24.9; gated 17408 x 5120 31.4, 31.4; 151936 x 2560 to float32 66.6, 66.4; 32 rows 2048 x 2048 3.9, 7.0;
// 4096 x 4096 8.8, 9.5; 7168 x 5120 15.4, 13.5; gated 9728 x 2560 23.0, 16.8; 24 rows 4096 x 12288 18.8, 15.2.  At the limit, 6144 x 4096, the two are level
// at 24 rows (11.4, 11.4) and 32 rows lose (12.4, 11.5).
// (The only place that knows: whoever counts kernels with bounded waits asks here.)
extern "C" int vx_gemm_q4_few_rows(int N, int K, int gated) { return (long long)N * K * (gated ? 2 : 1) <= 26000000LL ? 32 : 16; }

extern "C" int vx_gemm_q4_tc(const void* x, const void* codes, const void* affine, const void* codes1, const void* affine1, const float* bias,
                             void* out, int M, int N, int K, int ldx, int ldo, int group, int act, int out_dtype, int w_ready, int* error,
                             cudaStream_t stream);

// One matrix (codes1 null), or gate (codes, affine) and up (codes1, affine1): out = act(gate) * up.  N rows each.  `w_ready`: the
// matrices are nothing that the kernel launched just before this one writes.
extern "C" int vx_gemm_q4(const void* x, const void* codes, const void* affine, const void* codes1, const void* affine1, const float* bias,
                          void* out, int M, int N, int K, int ldx, int ldo, int group, int act, int out_dtype, int w_ready,
                          int* error, cudaStream_t stream) {
    if (M <= 0 || N <= 0) return VX_OK;
    if (K <= 0 || (group != 32 && group != 64 && group != 128) || K % group || ldx < K || ldo < N) return VX_ERR_SHAPE;
    if (codes1 && (!affine1 || bias || act < 0 || act > VX_ACT_LAST)) return VX_ERR_SHAPE;
    if (ldx & 7 || (((uintptr_t)x) | ((uintptr_t)codes) | ((uintptr_t)affine) | ((uintptr_t)codes1) | ((uintptr_t)affine1)) & 15) return VX_ERR_ALIGN;
    if (M > Q4_MOST || N > Q4_MOST || K > Q4_MOST) return VX_ERR_LIMIT;
    if (M > vx_gemm_q4_few_rows(N, K, codes1 != nullptr))
        return vx_gemm_q4_tc(x, codes, affine, codes1, affine1, bias, out, M, N, K, ldx, ldo, group, act, out_dtype, w_ready, error, stream);
    const Q4Pair w = {{(const unsigned*)codes, (const unsigned*)codes1}, {(const unsigned*)affine, (const unsigned*)affine1}};
#define Q4_ROWS(G, T, GR, NT) q4_launch<G, T, GR, NT>((const bf16*)x, w, bias, (T*)out, M, N, K, ldx, ldo, act, w_ready, stream)
#define Q4_GROUP(G, T, GR) (M <= 8 ? Q4_ROWS(G, T, GR, 1) : (M <= 16 ? Q4_ROWS(G, T, GR, 2) : Q4_ROWS(G, T, GR, 4)))
#define Q4_CALL(G, T) (group == 32 ? Q4_GROUP(G, T, 32) : (group == 64 ? Q4_GROUP(G, T, 64) : Q4_GROUP(G, T, 128)))
    if (out_dtype == VX_BF16) return codes1 ? Q4_CALL(true, bf16) : Q4_CALL(false, bf16);
    if (out_dtype == VX_F32) return codes1 ? VX_ERR_DTYPE : Q4_CALL(false, float);
#undef Q4_CALL
#undef Q4_GROUP
#undef Q4_ROWS
    return VX_ERR_DTYPE;
}
