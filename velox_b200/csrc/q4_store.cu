// Making a matrix in four bits from a bfloat16 or float32 one, and back.
//
//   lo = min, hi = max of a group;  s = bfloat16((hi - lo) / 15), b = bfloat16(lo);  q = min(max(round((w - b) / s), 0), 15), ties to the
//   even code; s = 0: q = 0.  All in float32, every operation rounded once.  A group that holds a value that is not finite, or whose
//   scale is not, gets s = b = NaN: what it stands for shows it, whatever is multiplied with it.
//
// A warp makes the blocks of 16 rows of one group (half a block for groups of 32 is made with its other half): lane 4 r + t holds rows r and
// r + 8, 16 k of each of a block, as the layout has them, so a row's 64 k are 128 or 256 neighbouring bytes read by four lanes, a group's
// extremes two or one exchanges away, and a block's 512 bytes are written at once.
// What bounds it: memory, both ways (q4.cuh: the layout).
#include "q4.cuh"

__device__ __forceinline__ void q4_load16(const float* p, bool ok, float (&w)[16]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float4 v = ok ? __ldcs(reinterpret_cast<const float4*>(p) + i) : make_float4(0.f, 0.f, 0.f, 0.f);
        w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
    }
}
__device__ __forceinline__ void q4_load16(const bf16* p, bool ok, float (&w)[16]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint4 v = ok ? __ldcs(reinterpret_cast<const uint4*>(p) + i) : make_uint4(0u, 0u, 0u, 0u);
        const unsigned u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            w[8 * i + 2 * j] = __uint_as_float(u[j] << 16);
            w[8 * i + 2 * j + 1] = __uint_as_float(u[j] & 0xffff0000u);
        }
    }
}

// BLOCKS: blocks of 64 k that a warp makes together (2 for groups of 128).  LANES: lanes that share a group (2, 4, 4).
template <typename TW, int GROUP>
__global__ void __launch_bounds__(256)
quantize_q4_kernel(const TW* __restrict__ W, unsigned* __restrict__ codes, unsigned* __restrict__ affine, int N, int K, long long ldw,
                   int blocks, int groups, long long units) {
    constexpr int BLOCKS = GROUP == 128 ? 2 : 1;
    const int lane = threadIdx.x & 31, r = lane >> 2, t = lane & 3;
    pdl_wait();
    pdl_trigger();
    const long long unit = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (unit >= units) return;
    const int per_tile = blocks / BLOCKS;
    const long long tile = unit / per_tile;
    const int c0 = (int)(unit - tile * per_tile) * BLOCKS;
    unsigned words[BLOCKS][4];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const long long row = tile * 16 + half * 8 + r;
        float w[BLOCKS][16];
        bool ok[BLOCKS], finite = true;
        float lo = INFINITY, hi = -INFINITY;
#pragma unroll
        for (int b = 0; b < BLOCKS; ++b) {
            const int k = (c0 + b) * 64 + t * 16;
            ok[b] = row < N && k < K;   // (K is a multiple of the group, so of 16)
            q4_load16(W + row * ldw + k, ok[b], w[b]);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                lo = fminf(lo, w[b][i]);
                hi = fmaxf(hi, w[b][i]);
                finite = finite && fabsf(w[b][i]) < INFINITY;
            }
        }
#pragma unroll
        for (int o = 1; o < (GROUP == 32 ? 2 : 4); o <<= 1) {
            lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
            hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
            const int other = __shfl_xor_sync(0xffffffffu, (int)finite, o);
            finite = finite && other;
        }
        bf16 s = __float2bfloat16_rn((hi - lo) / 15.f), b = __float2bfloat16_rn(lo);
        if (!finite || !(fabsf(__bfloat162float(s)) < INFINITY) || !(fabsf(__bfloat162float(b)) < INFINITY)) s = b = __ushort_as_bfloat16(0x7fc0);
        const float sf = __bfloat162float(s), bf = __bfloat162float(b);
#pragma unroll
        for (int blk = 0; blk < BLOCKS; ++blk)
#pragma unroll
            for (int word = 0; word < 2; ++word) {
                unsigned v = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float q = sf > 0.f ? fminf(fmaxf(rintf((w[blk][8 * word + i] - bf) / sf), 0.f), 15.f) : 0.f;
                    v |= (unsigned)q << (4 * (4 * (i & 1) + (i >> 1)));
                }
                words[blk][2 * half + word] = ok[blk] ? v : 0u;
            }
        if (t % (GROUP == 32 ? 2 : 4) == 0) {
            const int group = GROUP == 32 ? c0 * 2 + t / 2 : (GROUP == 64 ? c0 : c0 / 2);
            affine[(tile * groups + group) * 16 + r * 2 + half] =
                ok[0] ? (unsigned)__bfloat16_as_ushort(s) | (unsigned)__bfloat16_as_ushort(b) << 16 : 0u;
        }
    }
#pragma unroll
    for (int blk = 0; blk < BLOCKS; ++blk)
        reinterpret_cast<uint4*>(codes + (tile * blocks + c0 + blk) * Q4_BLOCK_WORDS)[t * 8 + r] =
            make_uint4(words[blk][0], words[blk][1], words[blk][2], words[blk][3]);
}

// A warp takes a block of 16 rows by 64 k back: lane 4 r + t writes 32 neighbouring bytes of rows r and r + 8.
__global__ void __launch_bounds__(256)
dequantize_q4_kernel(const unsigned* __restrict__ codes, const unsigned* __restrict__ affine, bf16* __restrict__ W, int N, int K, int group,
                     int blocks, int groups, long long units) {
    const int lane = threadIdx.x & 31, r = lane >> 2, t = lane & 3;
    pdl_wait();
    pdl_trigger();
    const long long unit = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (unit >= units) return;
    const long long tile = unit / blocks;
    const int c = (int)(unit - tile * blocks), k = c * 64 + t * 16;
    const uint4 v = __ldcs(reinterpret_cast<const uint4*>(codes + unit * Q4_BLOCK_WORDS) + t * 8 + r);
    const uint2 a = *reinterpret_cast<const uint2*>(affine + (tile * groups + k / group) * 16 + r * 2);
    const unsigned words[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const long long row = tile * 16 + half * 8 + r;
        const unsigned s = q4_scale(half ? a.y : a.x), b = q4_offset(half ? a.y : a.x);
        if (row < N && k < K) {
#pragma unroll
            for (int word = 0; word < 2; ++word) {
                unsigned w[4];
                q4_values(words[2 * half + word], s, b, w);
                __stcs(reinterpret_cast<uint4*>(W + row * K + k) + word, make_uint4(w[0], w[1], w[2], w[3]));
            }
        }
    }
}

static int q4_grid(long long units, unsigned* grid) {
    const long long n = (units + 7) / 8;
    if (n > 0x7fffffffLL) return VX_ERR_LIMIT;
    *grid = (unsigned)n;
    return VX_OK;
}

// W [N, K] with row stride ldw; codes [N / 16][K / 64][128] words, affine [N / 16][groups][16] words (rounded up as in q4.cuh).
extern "C" int vx_quantize_q4(const void* W, void* codes, void* affine, int N, int K, long long ldw, int group, int dtype, cudaStream_t stream) {
    if (N <= 0) return VX_OK;
    if (K <= 0 || (group != 32 && group != 64 && group != 128) || K % group || ldw < K) return VX_ERR_SHAPE;
    if (dtype != VX_F32 && dtype != VX_BF16) return VX_ERR_DTYPE;
    if ((((uintptr_t)W) | ((uintptr_t)codes) | ((uintptr_t)affine)) & 15 || (ldw * (dtype == VX_F32 ? 4 : 2)) & 15) return VX_ERR_ALIGN;
    const int blocks = (K + 63) / 64, groups = blocks * 64 / group;
    const long long units = (long long)((N + 15) / 16) * (group == 128 ? blocks / 2 : blocks);
    unsigned grid;
    if (int rc = q4_grid(units, &grid)) return rc;
#define Q4_GO(T, G)                                                                                                                     \
    VX_LAUNCH((quantize_q4_kernel<T, G>), grid, 256, 0, stream, (const T*)W, (unsigned*)codes, (unsigned*)affine, N, K, ldw, blocks, groups, \
              units)
    if (dtype == VX_BF16) {
        if (group == 32) Q4_GO(bf16, 32);
        else if (group == 64) Q4_GO(bf16, 64);
        else Q4_GO(bf16, 128);
    } else {
        if (group == 32) Q4_GO(float, 32);
        else if (group == 64) Q4_GO(float, 64);
        else Q4_GO(float, 128);
    }
#undef Q4_GO
    VX_LAUNCH_CHECK();
    return VX_OK;
}

// The bfloat16 matrix [N, K] (rows K apart) that codes and affine stand for.
extern "C" int vx_dequantize_q4(const void* codes, const void* affine, void* W, int N, int K, int group, cudaStream_t stream) {
    if (N <= 0) return VX_OK;
    if (K <= 0 || (group != 32 && group != 64 && group != 128) || K % group) return VX_ERR_SHAPE;
    if ((((uintptr_t)W) | ((uintptr_t)codes) | ((uintptr_t)affine)) & 15) return VX_ERR_ALIGN;
    const int blocks = (K + 63) / 64, groups = blocks * 64 / group;
    const long long units = (long long)((N + 15) / 16) * blocks;
    unsigned grid;
    if (int rc = q4_grid(units, &grid)) return rc;
    VX_LAUNCH(dequantize_q4_kernel, grid, 256, 0, stream, (const unsigned*)codes, (const unsigned*)affine, (bf16*)W, N, K, group, blocks, groups, units);
    VX_LAUNCH_CHECK();
    return VX_OK;
}
