// bf16 [rows, cols] -> e4m3 codes and fp32 scales of blocks of 128 (block_scale.cuh): one scale per 128 columns of a row, or per
// 128 x 128, for the matrix as it is and / or for its transpose.  One block of threads takes a 128 x 128 tile, reads it once and
// writes both orientations, the transposed one through shared memory so that its rows leave in whole lines as well.  Bound by
// HBM: 2 bytes read and 1 byte written per element and orientation.
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

// Thread (group, vec) holds rows [8 group, 8 group + 8) x columns [8 vec, 8 vec + 8) of the tile.
template <bool SQUARE>
__global__ void __launch_bounds__(256) block_quantize_kernel(const Quantize p) {
    __shared__ uint32_t column_max[16][kTile];
    __shared__ __align__(16) uint8_t turned[kTile * kTile];   // [column][row], 8-byte units permuted (see below)
    __shared__ uint32_t tile_max;
    const int vec = threadIdx.x & 15, group = threadIdx.x >> 4;
    const long long row0 = static_cast<long long>(blockIdx.y) * kTile;
    const int col0 = blockIdx.x * kTile;
    const int col = col0 + vec * 8;
    const bool col_in = col < p.cols;
    if (SQUARE && threadIdx.x == 0) tile_max = 0;
    uint4 v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const long long row = row0 + group * 8 + i;
        v[i] = col_in && row < p.rows ? *reinterpret_cast<const uint4*>(p.x + row * p.x_stride + col) : make_uint4(0, 0, 0, 0);
    }
    float inv_rows[8];   // SQUARE: the same value eight times
    float inv_cols[8];
    if (SQUARE) {
        uint32_t big = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            big = max(max(max(big, abs_bits_bf16x2(v[i].x)), max(abs_bits_bf16x2(v[i].y), abs_bits_bf16x2(v[i].z))), abs_bits_bf16x2(v[i].w));
        big = __reduce_max_sync(0xffffffffu, big);
        __syncthreads();
        if ((threadIdx.x & 31) == 0) atomicMax(&tile_max, big);
        __syncthreads();
        float inv;
        const float scale = block_scale(tile_max, inv);
#pragma unroll
        for (int i = 0; i < 8; ++i) inv_rows[i] = inv_cols[i] = inv;
        if (threadIdx.x == 0) {
            if (p.q != nullptr) p.scales[blockIdx.y * p.s_row + blockIdx.x * p.s_block] = scale;
            if (p.qt != nullptr) p.scales_t[blockIdx.x * p.st_row + blockIdx.y * p.st_block] = scale;
        }
    } else {
        if (p.q != nullptr) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                uint32_t big = max(max(abs_bits_bf16x2(v[i].x), abs_bits_bf16x2(v[i].y)), max(abs_bits_bf16x2(v[i].z), abs_bits_bf16x2(v[i].w)));
#pragma unroll
                for (int off = 8; off > 0; off >>= 1) big = max(big, __shfl_xor_sync(0xffffffffu, big, off));
                const float scale = block_scale(big, inv_rows[i]);
                const long long row = row0 + group * 8 + i;
                if (vec == 0 && row < p.rows) p.scales[row * p.s_row + blockIdx.x * p.s_block] = scale;
            }
        }
        if (p.qt != nullptr) {
            uint32_t big[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    big[2 * j] = max(big[2 * j], (w[j] << 16) & 0x7FFF0000u);
                    big[2 * j + 1] = max(big[2 * j + 1], w[j] & 0x7FFF0000u);
                }
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) column_max[group][vec * 8 + j] = big[j];
            __syncthreads();
            if (threadIdx.x < kTile) {
                uint32_t m = 0;
#pragma unroll
                for (int g = 0; g < 16; ++g) m = max(m, column_max[g][threadIdx.x]);
                column_max[0][threadIdx.x] = m;
                float inv;
                const float scale = block_scale(m, inv);
                if (col0 + static_cast<int>(threadIdx.x) < p.cols)
                    p.scales_t[(col0 + threadIdx.x) * p.st_row + blockIdx.y * p.st_block] = scale;
            }
            __syncthreads();
#pragma unroll
            for (int j = 0; j < 8; ++j) block_scale(column_max[0][vec * 8 + j], inv_cols[j]);
        }
    }
    if (p.q != nullptr) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float2 a = unpack_bf16x2(v[i].x), b = unpack_bf16x2(v[i].y), c = unpack_bf16x2(v[i].z), d = unpack_bf16x2(v[i].w);
            const float s = inv_rows[i];
            const long long row = row0 + group * 8 + i;
            if (col_in && row < p.rows)
                *reinterpret_cast<uint2*>(p.q + row * p.q_stride + col) =
                    make_uint2(mxfp8_convert4(a.x * s, a.y * s, b.x * s, b.y * s), mxfp8_convert4(c.x * s, c.y * s, d.x * s, d.y * s));
        }
    }
    if (p.qt != nullptr) {
        // A column's 8-byte unit `group` goes to place group ^ (column / 8): the 32 lanes that store (two groups, 16 columns 8
        // apart) then use every bank twice instead of one bank sixteen times.
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float f[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t w = j < 2 ? v[i].x : j < 4 ? v[i].y : j < 6 ? v[i].z : v[i].w;
                f[i] = __uint_as_float(j & 1 ? w & 0xFFFF0000u : w << 16) * inv_cols[j];
            }
            *reinterpret_cast<uint2*>(turned + (vec * 8 + j) * kTile + ((group ^ vec) * 8)) =
                make_uint2(mxfp8_convert4(f[0], f[1], f[2], f[3]), mxfp8_convert4(f[4], f[5], f[6], f[7]));
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
