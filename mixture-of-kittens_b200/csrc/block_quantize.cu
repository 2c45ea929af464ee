// bf16 [rows, cols] -> e4m3 codes and fp32 scales of blocks of 128 (block_scale.cuh): one scale per 128 columns of a row, or per
// 128 x 128, for the matrix as it is and / or for its transpose.  One block of threads takes a 128 x 128 tile, reads it once and
// writes both orientations, the transposed one through shared memory so that its rows leave in whole lines as well.  Bound by
// HBM: 2 bytes read and 1 byte written per element and orientation.  8192 x 7168: 28.7 us (6.1 TB/s), 41 us with the transpose (5.7
// TB/s), the same within 2 us for both forms of scales; with maxima in fp32, a shuffle for every row and step and reciprocals made by
// every thread for itself, scales per row took 42 and 61 us.
#include "block_scale.cuh"

namespace mok {
namespace {

constexpr int kTile = 128;

struct Quantize {
    const bf16* x;
    long long x_stride;
    long long rows;
    int cols;
    uint8_t *q, *qt;
    long long q_stride, qt_stride;
    float *scales, *scales_t;   // strides of the row (of the matrix concerned) and of the block along it
    long long s_row, s_block, st_row, st_block;
};

__device__ __forceinline__ uint32_t multiply_bf16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
// Two magnitudes at a time: the bits of bf16 without their sign, in integer order (infinities above the finite values, NaNs above
// those).  The scales' reciprocals are powers of two (or NaN) and so exact in bf16, as are the products (those below the normal
// range are far below half of e4m3's smallest step): the values are scaled in pairs too.
__device__ __forceinline__ uint32_t magnitude2(uint32_t v) { return v & 0x7FFF7FFFu; }
__device__ __forceinline__ uint32_t magnitude2(const uint4& v) {
    return __vmaxu2(__vmaxu2(magnitude2(v.x), magnitude2(v.y)), __vmaxu2(magnitude2(v.z), magnitude2(v.w)));
}
__device__ __forceinline__ uint32_t scale_code4(uint32_t a, uint32_t b, uint32_t inv_a, uint32_t inv_b) {
    const uint32_t p = multiply_bf16x2(a, inv_a), q = multiply_bf16x2(b, inv_b);
    return mxfp8_convert4(__uint_as_float(p << 16), __uint_as_float(p & 0xFFFF0000u), __uint_as_float(q << 16), __uint_as_float(q & 0xFFFF0000u));
}

// Thread (group, vec) holds rows [8 group, 8 group + 8) x columns [8 vec, 8 vec + 8) of the tile, as it was read: the 16 lanes of
// a half warp hold 8 whole row blocks.
template <bool SQUARE>
__global__ void __launch_bounds__(256, 4) block_quantize_kernel(const Quantize p) {
    __shared__ uint4 column_max[16][16];                      // [group][vec]
    __shared__ uint32_t column_inv[kTile / 2];                // of two columns each
    __shared__ __align__(16) uint8_t turned[kTile * kTile];   // [column][row], 8-byte units permuted (see below)
    __shared__ uint32_t warp_max[8];
    const int vec = threadIdx.x & 15, group = threadIdx.x >> 4;
    const long long row0 = static_cast<long long>(blockIdx.y) * kTile;
    const int col0 = blockIdx.x * kTile;
    const int col = col0 + vec * 8;
    const bool col_in = col < p.cols;
    uint4 v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const long long row = row0 + group * 8 + i;
        v[i] = col_in && row < p.rows ? *reinterpret_cast<const uint4*>(p.x + row * p.x_stride + col) : make_uint4(0, 0, 0, 0);
    }
    uint32_t inv_rows[8];   // twice the same reciprocal; SQUARE: eight times the same
    uint32_t inv_cols[4];   // reciprocals of two columns
    if (SQUARE) {
        uint32_t big = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) big = __vmaxu2(big, magnitude2(v[i]));
        big = __reduce_max_sync(0xffffffffu, max(big << 16, big & 0xFFFF0000u));
        if ((threadIdx.x & 31) == 0) warp_max[threadIdx.x >> 5] = big;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) big = max(big, warp_max[i]);
        float inv;
        const float scale = block_scale(big, inv);
        const uint32_t inv2 = __byte_perm(__float_as_uint(inv), 0, 0x3232);
#pragma unroll
        for (int i = 0; i < 8; ++i) inv_rows[i] = inv2;
#pragma unroll
        for (int i = 0; i < 4; ++i) inv_cols[i] = inv2;
        if (threadIdx.x == 0) {
            if (p.q != nullptr) p.scales[blockIdx.y * p.s_row + blockIdx.x * p.s_block] = scale;
            if (p.qt != nullptr) p.scales_t[blockIdx.x * p.st_row + blockIdx.y * p.st_block] = scale;
        }
    } else {
        if (p.q != nullptr) {
            // Eight maxima over 16 lanes with five exchanges: each sends the half of its rows that the other one keeps.  Every
            // lane ends with the row pair that its bits 3 and 2 name, and makes the scale of the one that bit 0 names.
            uint32_t pair[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t a = magnitude2(v[2 * i]), b = magnitude2(v[2 * i + 1]);
                pair[i] = __vmaxu2(__byte_perm(a, b, 0x5410), __byte_perm(a, b, 0x7632));
            }
            const bool high = vec & 8, middle = vec & 4;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t theirs = __shfl_xor_sync(0xffffffffu, high ? pair[i] : pair[2 + i], 8);
                pair[i] = __vmaxu2(high ? pair[2 + i] : pair[i], theirs);
            }
            uint32_t big = __vmaxu2(middle ? pair[1] : pair[0], __shfl_xor_sync(0xffffffffu, middle ? pair[0] : pair[1], 4));
            big = __vmaxu2(big, __shfl_xor_sync(0xffffffffu, big, 2));
            big = __vmaxu2(big, __shfl_xor_sync(0xffffffffu, big, 1));
            float inv;
            const float scale = block_scale((vec & 1) ? big & 0xFFFF0000u : big << 16, inv);
            const long long row = row0 + group * 8 + (vec >> 2) * 2 + (vec & 1);
            if ((vec & 2) == 0 && row < p.rows) p.scales[row * p.s_row + blockIdx.x * p.s_block] = scale;
            const uint32_t inv2 = __byte_perm(__float_as_uint(inv), 0, 0x3232);
#pragma unroll
            for (int i = 0; i < 8; ++i) inv_rows[i] = __shfl_sync(0xffffffffu, inv2, (i >> 1) * 4 + (i & 1), 16);
        }
        if (p.qt != nullptr) {
            uint4 big = make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                big.x = __vmaxu2(big.x, magnitude2(v[i].x));
                big.y = __vmaxu2(big.y, magnitude2(v[i].y));
                big.z = __vmaxu2(big.z, magnitude2(v[i].z));
                big.w = __vmaxu2(big.w, magnitude2(v[i].w));
            }
            column_max[group][vec] = big;
            __syncthreads();
            if (threadIdx.x < kTile / 2) {
                uint32_t m = 0;
#pragma unroll
                for (int g = 0; g < 16; ++g) m = __vmaxu2(m, reinterpret_cast<const uint32_t*>(column_max[g])[threadIdx.x]);
                float inv0, inv1;
                const float scale0 = block_scale(m << 16, inv0), scale1 = block_scale(m & 0xFFFF0000u, inv1);
                column_inv[threadIdx.x] = __byte_perm(__float_as_uint(inv0), __float_as_uint(inv1), 0x7632);
                const int c = col0 + threadIdx.x * 2;   // columns come in eights: both are inside or neither
                if (c < p.cols) {
                    p.scales_t[c * p.st_row + blockIdx.y * p.st_block] = scale0;
                    p.scales_t[(c + 1) * p.st_row + blockIdx.y * p.st_block] = scale1;
                }
            }
            __syncthreads();
            const uint4 w = *reinterpret_cast<const uint4*>(column_inv + vec * 4);
            inv_cols[0] = w.x; inv_cols[1] = w.y; inv_cols[2] = w.z; inv_cols[3] = w.w;
        }
    }
    if (p.q != nullptr) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const long long row = row0 + group * 8 + i;
            const uint32_t s = inv_rows[i];
            if (col_in && row < p.rows)
                *reinterpret_cast<uint2*>(p.q + row * p.q_stride + col) =
                    make_uint2(scale_code4(v[i].x, v[i].y, s, s), scale_code4(v[i].z, v[i].w, s, s));
        }
    }
    if (p.qt != nullptr) {
        // A column's 8-byte unit `group` goes to place group ^ (column / 8): the 32 lanes that store (two groups, 16 columns 8
        // apart) then use every bank twice instead of one bank sixteen times.
#pragma unroll
        for (int j = 0; j < 4; ++j) {   // two columns: pairs (even, odd) of eight rows become four codes of each column, twice
            uint32_t f[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                f[i] = multiply_bf16x2(j == 0 ? v[i].x : j == 1 ? v[i].y : j == 2 ? v[i].z : v[i].w, inv_cols[j]);
            auto low = [&](int i) { return __uint_as_float(f[i] << 16); };
            auto high = [&](int i) { return __uint_as_float(f[i] & 0xFFFF0000u); };
            uint8_t* to = turned + (vec * 8 + 2 * j) * kTile + ((group ^ vec) * 8);
            *reinterpret_cast<uint2*>(to) = make_uint2(mxfp8_convert4(low(0), low(1), low(2), low(3)), mxfp8_convert4(low(4), low(5), low(6), low(7)));
            *reinterpret_cast<uint2*>(to + kTile) =
                make_uint2(mxfp8_convert4(high(0), high(1), high(2), high(3)), mxfp8_convert4(high(4), high(5), high(6), high(7)));
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int c = i * 16 + (threadIdx.x >> 4), unit = threadIdx.x & 15;   // one column's 128 rows by half a warp
            const uint2 w = *reinterpret_cast<const uint2*>(turned + c * kTile + ((unit ^ (c >> 3)) * 8));
            const long long row = row0 + unit * 8;
            // rows behind the last are zero codes; the row stride of the output leaves room for whole units
            if (col0 + c < p.cols && row < p.rows) *reinterpret_cast<uint2*>(p.qt + (col0 + c) * p.qt_stride + row) = w;
        }
    }
}

}  // namespace
}  // namespace mok

extern "C" int mok_block_quantize(const void* x, int64_t x_stride, int64_t rows, int cols, int tile_rows, void* codes, int64_t codes_stride,
                                  float* scales, int64_t scale_row_stride, int64_t scale_block_stride, void* codes_t,
                                  int64_t codes_t_stride, float* scales_t, int64_t scale_t_row_stride, int64_t scale_t_block_stride,
                                  mok_stream_t stream) {
    using namespace mok;
    if (rows < 0 || cols < 0 || cols % 8 != 0 || (tile_rows != 1 && tile_rows != kTile)) return MOK_ERR_INVALID_ARGUMENT;
    if (rows > 65535LL * kTile) return MOK_ERR_TOO_LARGE;
    if (rows == 0 || cols == 0) return MOK_OK;
    if (!x || (!codes && !codes_t) || (codes == nullptr) != (scales == nullptr) || (codes_t == nullptr) != (scales_t == nullptr))
        return MOK_ERR_INVALID_ARGUMENT;
    if ((reinterpret_cast<uintptr_t>(x) & 15) != 0 || x_stride % 8 != 0 || x_stride < 0 || (reinterpret_cast<uintptr_t>(codes) & 7) != 0 ||
        (reinterpret_cast<uintptr_t>(codes_t) & 7) != 0)
        return MOK_ERR_INVALID_ARGUMENT;
    if (codes != nullptr && (codes_stride % 8 != 0 || codes_stride < cols)) return MOK_ERR_INVALID_ARGUMENT;
    if (codes_t != nullptr && (codes_t_stride % 8 != 0 || codes_t_stride < rows)) return MOK_ERR_INVALID_ARGUMENT;
    Quantize p{};
    p.x = static_cast<const bf16*>(x);
    p.x_stride = x_stride;
    p.rows = rows;
    p.cols = cols;
    p.q = static_cast<uint8_t*>(codes);
    p.q_stride = codes_stride;
    p.scales = scales;
    p.s_row = scale_row_stride;
    p.s_block = scale_block_stride;
    p.qt = static_cast<uint8_t*>(codes_t);
    p.qt_stride = codes_t_stride;
    p.scales_t = scales_t;
    p.st_row = scale_t_row_stride;
    p.st_block = scale_t_block_stride;
    const dim3 grid((cols + kTile - 1) / kTile, static_cast<unsigned>((rows + kTile - 1) / kTile));
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    if (tile_rows == 1) block_quantize_kernel<false><<<grid, 256, 0, s>>>(p);
    else block_quantize_kernel<true><<<grid, 256, 0, s>>>(p);
    MOK_LAUNCH_CHECK("block_quantize_kernel");
    return MOK_OK;
}
