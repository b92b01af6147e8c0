// Making a matrix in four bits from a bfloat16 or float32 one, and back.
//
//   lo = min, hi = max of a group;  s = bfloat16((hi - lo) / 15), b = bfloat16(lo);  q = min(max(round((w - b) / s), 0), 15), ties to the
//   even code; s = 0: q = 0.  All in float32, every operation rounded once.  A group that holds a value that is not finite, or whose
//   scale is not, gets s = b = NaN: what it stands for shows it, whatever is multiplied with it.
//
// A warp makes a block of 16 rows by 64 k (groups of 128: two): lane 4 r + t holds rows r and r + 8, 16 k of each of a block, as the layout has them,
// so a row's 64 k are 128 or 256 neighbouring bytes read by four lanes, a group's extremes two or one exchanges away, and a block's 512 bytes
// are written at once.
// What bounds them: from bfloat16 instructions (some nine an element), else memory.  12288 x 4096 in groups of 64, us of calls in a row and of the copy
// rate of 6,549 GB/s: from bfloat16 28.2, 70 % (33.6, 59 %, where every result goes to memory not written before); from float32 38.4, 91 %
// (41.2, 85 %); back 22.8, 87 %.
#include "q4.cuh"

// 16 neighbours of a row as they are stored: their extremes, whether all are finite, their values.
template <typename T> struct Q4Row;
template <> struct Q4Row<float> {
    float4 v[4];
    __device__ __forceinline__ void load(const float* p, bool ok) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = ok ? __ldcs(reinterpret_cast<const float4*>(p) + i) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    __device__ __forceinline__ float at(int i) const { return (&v[i >> 2].x)[i & 3]; }
    __device__ __forceinline__ void extremes(float& lo, float& hi, bool& finite) const {
        float zero = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            lo = fminf(lo, at(i));
            hi = fmaxf(hi, at(i));
            zero = fmaf(at(i), 0.f, zero);   // (NaN once a value is not finite)
        }
        finite = finite && zero == 0.f;
    }
};
template <> struct Q4Row<bf16> {
    unsigned v[8];
    __device__ __forceinline__ void load(const bf16* p, bool ok) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint4 u = ok ? __ldcs(reinterpret_cast<const uint4*>(p) + i) : make_uint4(0u, 0u, 0u, 0u);
            v[4 * i] = u.x; v[4 * i + 1] = u.y; v[4 * i + 2] = u.z; v[4 * i + 3] = u.w;
        }
    }
    __device__ __forceinline__ float at(int i) const { return __uint_as_float(i & 1 ? v[i >> 1] & 0xffff0000u : v[i >> 1] << 16); }
    __device__ __forceinline__ void extremes(float& lo, float& hi, bool& finite) const {   // two at a time
        unsigned l = v[0], h = v[0], zero = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (i) {
                asm("min.bf16x2 %0, %0, %1;\n" : "+r"(l) : "r"(v[i]));
                asm("max.bf16x2 %0, %0, %1;\n" : "+r"(h) : "r"(v[i]));
            }
            asm("fma.rn.bf16x2 %0, %1, %2, %0;\n" : "+r"(zero) : "r"(v[i]), "r"(0u));
        }
        lo = fminf(lo, fminf(__uint_as_float(l << 16), __uint_as_float(l & 0xffff0000u)));
        hi = fmaxf(hi, fmaxf(__uint_as_float(h << 16), __uint_as_float(h & 0xffff0000u)));
        finite = finite && (zero & 0x7fff7fffu) == 0u;
    }
};

// Eight codes of one word.  The quotient is a product with y = 1 / s and one correction by its exact remainder (Markstein's theorem: with y
// rounded correctly that gives the quotient rounded correctly, so ties are ties), a division only where a remainder could underflow, or where
// float32 values are so large that w - b can overflow although max - min does not (b is a float32 minimum rounded, maybe away from the values; of
// bfloat16 values it is the minimum itself): infinity divided by s is bounded by 15, its remainder would be NaN.
// (Dividing always, 12288 x 4096 bfloat16 in groups of 64 took 78 us; dividing where the plain product was within 1e-5 of half way, as some value of
// a word's 256 mostly was, 39.)  Rounding is the addition of 1.5 * 2^23: the code is the sum's low bits, and the sums, shifted, add up to the word
// and a constant.  Of bfloat16 values only the scale's own rounding takes a quotient beyond 15, to 15.06: no bounds are needed.
template <typename T>
__device__ __forceinline__ unsigned q4_codes(const Q4Row<T>& row, int first, float s, float b, float inverse) {
    constexpr unsigned MAGIC = 0x4b400000u;   // 1.5 * 2^23
    unsigned word = 0, sums = 0;
    if (s >= 1e-30f && (sizeof(T) == 2 || s <= 1e37f)) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int at = 4 * (4 * (i & 1) + (i >> 1));
            const float d = row.at(first + i) - b;
            float q = d * inverse;
            q = fmaf(fmaf(-q, s, d), inverse, q);
            if (sizeof(T) == 4) q = fminf(fmaxf(q, 0.f), 15.f);
            word += __float_as_uint(q + __uint_as_float(MAGIC)) << at;
            sums += MAGIC << at;
        }
        word -= sums;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float q = s > 0.f ? fminf(fmaxf(rintf((row.at(first + i) - b) / s), 0.f), 15.f) : 0.f;
            word |= (unsigned)q << (4 * (4 * (i & 1) + (i >> 1)));
        }
    }
    return word;
}

// BLOCKS: blocks of 64 k that a warp makes together (2 for groups of 128).
template <typename TW, int GROUP>
__global__ void __launch_bounds__(256)
quantize_q4_kernel(const TW* __restrict__ W, unsigned* __restrict__ codes, unsigned* __restrict__ affine, int N, int K, long long ldw,
                   int blocks, int groups) {
    constexpr int BLOCKS = GROUP == 128 ? 2 : 1;
    const int lane = threadIdx.x & 31, r = lane >> 2, t = lane & 3;
    pdl_wait();
    pdl_trigger();
    const long long tile = blockIdx.x;
    const int c0 = (int)(blockIdx.y * 8 + (threadIdx.x >> 5)) * BLOCKS;
    if (c0 >= blocks) return;
    Q4Row<TW> row[2][BLOCKS];
    bool ok[2][BLOCKS];
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int b = 0; b < BLOCKS; ++b) {
            const long long n = tile * 16 + half * 8 + r;
            const int k = (c0 + b) * 64 + t * 16;
            ok[half][b] = n < N && k < K;   // (K is a multiple of the group, so of 16)
            row[half][b].load(W + n * ldw + k, ok[half][b]);
        }
    unsigned words[BLOCKS][4];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        bool finite = true;
        float lo = INFINITY, hi = -INFINITY;
#pragma unroll
        for (int b = 0; b < BLOCKS; ++b) row[half][b].extremes(lo, hi, finite);
#pragma unroll
        for (int o = 1; o < (GROUP == 32 ? 2 : 4); o <<= 1) {
            lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
            hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
            const int other = __shfl_xor_sync(0xffffffffu, (int)finite, o);
            finite = finite && other;
        }
        bf16 s = __float2bfloat16_rn((hi - lo) / 15.f), b = __float2bfloat16_rn(lo);
        if (!finite || !(fabsf(__bfloat162float(s)) < INFINITY) || !(fabsf(__bfloat162float(b)) < INFINITY)) s = b = __ushort_as_bfloat16(0x7fc0);
        const float sf = __bfloat162float(s), bf = __bfloat162float(b), inverse = sf > 0.f ? 1.f / sf : 0.f;
        const bool some = sf > 0.f;   // (neither 0 nor NaN)
#pragma unroll
        for (int blk = 0; blk < BLOCKS; ++blk)
#pragma unroll
            for (int word = 0; word < 2; ++word)
                words[blk][2 * half + word] = ok[half][blk] && some ? q4_codes(row[half][blk], 8 * word, sf, bf, inverse) : 0u;
        if (t % (GROUP == 32 ? 2 : 4) == 0) {
            const int group = GROUP == 32 ? c0 * 2 + t / 2 : (GROUP == 64 ? c0 : c0 / 2);
            affine[(tile * groups + group) * 16 + r * 2 + half] =
                ok[half][0] ? (unsigned)__bfloat16_as_ushort(s) | (unsigned)__bfloat16_as_ushort(b) << 16 : 0u;
        }
    }
#pragma unroll
    for (int blk = 0; blk < BLOCKS; ++blk)
        __stcs(reinterpret_cast<uint4*>(codes + (tile * blocks + c0 + blk) * Q4_BLOCK_WORDS) + t * 8 + r,
               make_uint4(words[blk][0], words[blk][1], words[blk][2], words[blk][3]));
}

// A warp takes a block of 16 rows by 64 k back: lanes 4 r + t and their neighbours write 64 neighbouring bytes of rows r and r + 8.
__global__ void __launch_bounds__(256)
dequantize_q4_kernel(const unsigned* __restrict__ codes, const unsigned* __restrict__ affine, bf16* __restrict__ W, int N, int K, int group,
                     int blocks, int groups) {
    const int lane = threadIdx.x & 31, r = lane >> 2, t = lane & 3;
    pdl_wait();
    pdl_trigger();
    const long long tile = blockIdx.x;
    const int c = (int)(blockIdx.y * 8 + (threadIdx.x >> 5)), k = c * 64 + t * 16;
    if (c >= blocks) return;
    const uint4 v = __ldcs(reinterpret_cast<const uint4*>(codes + (tile * blocks + c) * Q4_BLOCK_WORDS) + t * 8 + r);
    const uint2 a = *reinterpret_cast<const uint2*>(affine + (tile * groups + k / group) * 16 + r * 2);
    const unsigned words[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const long long row = tile * 16 + half * 8 + r;
        const unsigned s = q4_scale(half ? a.y : a.x), b = q4_offset(half ? a.y : a.x);
        unsigned low[4], high[4], other[4];
        q4_values<false>(words[2 * half], s, b, low);
        q4_values<false>(words[2 * half + 1], s, b, high);
        // neighbours change 16 bytes, so that each of the two stores fills whole 32-byte sectors
        const bool odd = t & 1;
#pragma unroll
        for (int i = 0; i < 4; ++i) other[i] = __shfl_xor_sync(0xffffffffu, odd ? low[i] : high[i], 1);
        if (row < N && k < K) {   // (two neighbours are both within K or both beyond)
            uint4* to = reinterpret_cast<uint4*>(W + row * K + c * 64 + (t & 2) * 16) + (odd ? 1 : 0);
            __stcs(to, odd ? make_uint4(other[0], other[1], other[2], other[3]) : make_uint4(low[0], low[1], low[2], low[3]));
            __stcs(to + 2, odd ? make_uint4(high[0], high[1], high[2], high[3]) : make_uint4(other[0], other[1], other[2], other[3]));
        }
    }
}

// A block's eight warps lie along K.  (With units numbered through, a division of 64 bits a warp, 12288 x 4096 took a tenth longer.)
static int q4_grid(int N, int units, dim3* grid) {
    const int y = (units + 7) / 8;
    if (y > 65535) return VX_ERR_LIMIT;
    *grid = dim3((unsigned)((N + 15LL) / 16), (unsigned)y);
    return VX_OK;
}

// W [N, K] with row stride ldw; codes [N / 16][K / 64][128] words, affine [N / 16][groups][16] words (rounded up as in q4.cuh).
extern "C" int vx_quantize_q4(const void* W, void* codes, void* affine, int N, int K, long long ldw, int group, int dtype, cudaStream_t stream) {
    if (N <= 0) return VX_OK;
    if (K <= 0 || (group != 32 && group != 64 && group != 128) || K % group || ldw < K) return VX_ERR_SHAPE;
    if (N > Q4_MOST || K > Q4_MOST) return VX_ERR_LIMIT;
    if (dtype != VX_F32 && dtype != VX_BF16) return VX_ERR_DTYPE;
    if ((((uintptr_t)W) | ((uintptr_t)codes) | ((uintptr_t)affine)) & 15 || (ldw * (dtype == VX_F32 ? 4 : 2)) & 15) return VX_ERR_ALIGN;
    const int blocks = (K + 63) / 64, groups = blocks * 64 / group;
    dim3 grid;
    if (int rc = q4_grid(N, group == 128 ? blocks / 2 : blocks, &grid)) return rc;
#define Q4_GO(T, G)                                                                                                                     \
    VX_LAUNCH((quantize_q4_kernel<T, G>), grid, 256, 0, stream, (const T*)W, (unsigned*)codes, (unsigned*)affine, N, K, ldw, blocks, groups)
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
    if (N > Q4_MOST || K > Q4_MOST) return VX_ERR_LIMIT;
    if ((((uintptr_t)W) | ((uintptr_t)codes) | ((uintptr_t)affine)) & 15) return VX_ERR_ALIGN;
    const int blocks = (K + 63) / 64, groups = blocks * 64 / group;
    dim3 grid;
    if (int rc = q4_grid(N, blocks, &grid)) return rc;
    VX_LAUNCH(dequantize_q4_kernel, grid, 256, 0, stream, (const unsigned*)codes, (const unsigned*)affine, (bf16*)W, N, K, group, blocks, groups);
    VX_LAUNCH_CHECK();
    return VX_OK;
}
