// out[M,N] = x[M,K] W^T (+ bias) and out[M,N] = act(x Wg^T) * (x Wu^T) with matrices held in four bits (q4.cuh), for a few rows: the
// products of a decode step, where the whole cost is reading codes, scales and offsets once.
//
// As in the bfloat16 product of a few rows, out^T = W x^T on mma.sync.m16n8k16: 16 rows of W fill the tile's 16-row side, up to 8 rows of x its
// 8-column side.  A block owns the 16 rows of one row of code blocks (gated: those of the gate's and those of the up matrix, so that
// both sums of a feature meet in it) and the whole of K; its warps take the 64-wide code blocks in turn.  A lane's 16 bytes of a code block are
// its fragments of four products; it makes them bfloat16 in registers and nothing passes through shared memory.  k is permuted
// the same way for x, of which a lane reads 32 neighbouring bytes of a row.  The warps' partial tiles are added in shared memory in warp
// order: the same result on every run, and a row's result does not depend on the rows beside it.
#include "q4.cuh"

__device__ __forceinline__ uint4 q4_stream16(const unsigned* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ uint2 q4_stream8(const unsigned* p) {
    uint2 v;
    asm volatile("ld.global.nc.v2.u32 {%0,%1}, [%2];\n" : "=r"(v.x), "=r"(v.y) : "l"(p));
    return v;
}
__device__ __forceinline__ void q4_mma(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

struct Q4Pair { const unsigned *codes[2], *affine[2]; };   // the matrix, or gate and up

template <bool GATED, typename TO, int WARPS, int UNROLL>
__global__ void __launch_bounds__(WARPS * 32)
gemm_q4_kernel(const bf16* __restrict__ x, const Q4Pair w, const float* __restrict__ bias, TO* __restrict__ out, int M, int N, int K, int ldx,
               int ldo, int act, int blocks, int groups, int group_shift, int w_ready) {
    constexpr int MATS = GATED ? 2 : 1;
    __shared__ float red[MATS][WARPS][16][9];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, t = lane & 3;
    const size_t tile = blockIdx.x;
    const int m0 = blockIdx.y * 8;
    const unsigned *codes[MATS], *affine[MATS];
#pragma unroll
    for (int i = 0; i < MATS; ++i) {
        codes[i] = w.codes[i] + tile * blocks * Q4_BLOCK_WORDS + (t * 8 + r) * 4;
        affine[i] = w.affine[i] + tile * groups * 16 + r * 2;
    }
    float acc[MATS][4] = {};
    uint4 q[MATS][UNROLL];
    uint2 a[MATS][UNROLL];
    int c = warp;
    auto ask = [&]() {
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int cu = c + u * WARPS;
            if (cu < blocks) {
#pragma unroll
                for (int i = 0; i < MATS; ++i) {
                    q[i][u] = q4_stream16(codes[i] + (size_t)cu * Q4_BLOCK_WORDS);
                    a[i][u] = q4_stream8(affine[i] + ((cu * 64 + t * 16) >> group_shift) * 16);
                }
            }
        }
    };
    if (w_ready) ask();
    pdl_wait();
    pdl_trigger();
    if (!w_ready) ask();
    const bool xok = m0 + r < M;
    const bf16* xr = x + (size_t)(xok ? m0 + r : 0) * ldx + t * 16;
    while (c < blocks) {
        uint4 xv[UNROLL][2];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int k = (c + u * WARPS) * 64;
            const bool ok = xok && k + t * 16 < K;
#pragma unroll
            for (int i = 0; i < 2; ++i) xv[u][i] = ok ? *reinterpret_cast<const uint4*>(xr + k + 8 * i) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            if (c + u * WARPS < blocks) {
#pragma unroll
                for (int i = 0; i < MATS; ++i) {
                    const unsigned s0 = q4_scale(a[i][u].x), b0 = q4_offset(a[i][u].x), s1 = q4_scale(a[i][u].y), b1 = q4_offset(a[i][u].y);
#pragma unroll
                    for (int word = 0; word < 2; ++word) {
                        unsigned w0[4], w1[4];
                        q4_values(word ? q[i][u].y : q[i][u].x, s0, b0, w0);
                        q4_values(word ? q[i][u].w : q[i][u].z, s1, b1, w1);
                        q4_mma(acc[i], w0[0], w1[0], w0[1], w1[1], xv[u][word].x, xv[u][word].y);
                        q4_mma(acc[i], w0[2], w1[2], w0[3], w1[3], xv[u][word].z, xv[u][word].w);
                    }
                }
            }
        }
        c += UNROLL * WARPS;
        ask();
    }
    // a lane holds out^T[row r (0, 1) and r + 8 (2, 3)][rows 2 t, 2 t + 1 of x]
#pragma unroll
    for (int i = 0; i < MATS; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) red[i][warp][r + 8 * (j >> 1)][2 * t + (j & 1)] = acc[i][j];
    __syncthreads();
    if (threadIdx.x < 128) {
        const int row = threadIdx.x & 15, m = threadIdx.x >> 4;
        const size_t n = tile * 16 + row;
        if (m0 + m < M && n < (size_t)N) {
            float v = 0.f, up = 0.f;
#pragma unroll
            for (int i = 0; i < WARPS; ++i) {
                v += red[0][i][row][m];
                if (GATED) up += red[MATS - 1][i][row][m];
            }
            if (bias) v += bias[n];
            out[(size_t)(m0 + m) * ldo + n] = from_f32<TO>(GATED ? activation(v, act) * up : v);
        }
    }
}

template <bool GATED, typename TO>
static int q4_launch(const bf16* x, const Q4Pair& w, const float* bias, TO* out, int M, int N, int K, int ldx, int ldo, int act, int group,
                     int w_ready, cudaStream_t stream) {
    const int blocks = (K + 63) / 64, groups = blocks * 64 / group, shift = group == 32 ? 5 : (group == 64 ? 6 : 7);
    const long long chunks = (M + 7LL) / 8;
    if (chunks > 65535) return VX_ERR_LIMIT;
    VX_LAUNCH_K(VX_K_GEMM, (gemm_q4_kernel<GATED, TO, 8, 4>), dim3((unsigned)((N + 15) / 16), (unsigned)chunks), 256, 0, stream, x, w, bias, out, M, N,
                K, ldx, ldo, act, blocks, groups, shift, w_ready);
    VX_LAUNCH_CHECK();
    return VX_OK;
}

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
    if (M > 8)
        return vx_gemm_q4_tc(x, codes, affine, codes1, affine1, bias, out, M, N, K, ldx, ldo, group, act, out_dtype, w_ready, error, stream);
    const Q4Pair w = {{(const unsigned*)codes, (const unsigned*)codes1}, {(const unsigned*)affine, (const unsigned*)affine1}};
#define Q4_CALL(G, T) q4_launch<G, T>((const bf16*)x, w, bias, (T*)out, M, N, K, ldx, ldo, act, group, w_ready, stream)
    if (out_dtype == VX_BF16) return codes1 ? Q4_CALL(true, bf16) : Q4_CALL(false, bf16);
    if (out_dtype == VX_F32) return codes1 ? VX_ERR_DTYPE : Q4_CALL(false, float);
#undef Q4_CALL
    return VX_ERR_DTYPE;
}
