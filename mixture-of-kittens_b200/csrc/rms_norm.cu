// Root-mean-square norm with the residual's addition: z = x + r in fp32, rho = (mean z^2 + eps)^-1/2, y = z rho w, as bf16
// and / or as e4m3 with a scale per 128 columns; hidden = bf16(z) is the next residual stream.  The norm is taken of z before
// it is rounded.  Backward, with z read back from `hidden`:
//   g = dy w,  dx = dr = rho (g - z rho^2 mean(g z)) + dhidden,  dw = sum over rows of dy z rho.
// Both are bound by HBM (by launch and latency for a few rows): every input is read once, into registers, and all sums are
// fp32.
#include "block_scale.cuh"

namespace mok {
namespace {

constexpr int kMaxHidden = 16384;   // 512 threads x 4 vectors of 8

struct NormForward {
    const bf16 *x, *residual;
    const void* weight;
    bf16 *hidden, *y;
    uint8_t* codes;
    float *scales, *inv_rms;
    long long x_stride, residual_stride, codes_stride, scale_row_stride, scale_block_stride, rows;
    int cols;
    float eps;
};

__device__ __forceinline__ void unpack8(const uint4& v, float (&f)[8]) {
    const float2 a = unpack_bf16x2(v.x), b = unpack_bf16x2(v.y), c = unpack_bf16x2(v.z), d = unpack_bf16x2(v.w);
    f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y; f[4] = c.x; f[5] = c.y; f[6] = d.x; f[7] = d.y;
}
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
    return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
}
template <bool W32>
__device__ __forceinline__ void load_weight(const void* w, int col, float (&f)[8]) {
    if (W32) {
        const float4 a = *reinterpret_cast<const float4*>(static_cast<const float*>(w) + col);
        const float4 b = *reinterpret_cast<const float4*>(static_cast<const float*>(w) + col + 4);
        f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
    } else {
        unpack8(*reinterpret_cast<const uint4*>(static_cast<const bf16*>(w) + col), f);
    }
}

// Sum over the block, the same value in every thread, in a fixed order.  `part` holds one float per warp; the caller alternates
// between two of them, so that one barrier per sum is enough.
__device__ __forceinline__ float block_sum(float v, float* part) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
    const int warps = blockDim.x >> 5;
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    float s = 0.0f;
    for (int i = 0; i < warps; ++i) s += part[i];
    return s;
}

// One row per block; a thread holds V vectors of 8 columns, so 16 adjacent lanes hold one block of 128.
template <int V, bool W32>
__global__ void __launch_bounds__(V < 4 ? 256 : 512) rms_norm_forward_kernel(const NormForward p) {
    __shared__ float part[32];
    const long long row = blockIdx.x;
    const int vectors = p.cols >> 3;
    const bf16* x = p.x + row * p.x_stride;
    const bf16* r = p.residual == nullptr ? nullptr : p.residual + row * p.residual_stride;
    float z[V][8];
    float sum = 0.0f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int i = v * blockDim.x + threadIdx.x;
        if (i < vectors) {
            unpack8(*reinterpret_cast<const uint4*>(x + i * 8), z[v]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) z[v][j] = 0.0f;
        }
    }
    if (r != nullptr) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int i = v * blockDim.x + threadIdx.x;
            if (i < vectors) {
                float f[8];
                unpack8(*reinterpret_cast<const uint4*>(r + i * 8), f);
#pragma unroll
                for (int j = 0; j < 8; ++j) z[v][j] += f[j];
                if (p.hidden != nullptr) *reinterpret_cast<uint4*>(p.hidden + row * p.cols + i * 8) = pack8(z[v]);
            }
        }
    }
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
        for (int j = 0; j < 8; ++j) sum = fmaf(z[v][j], z[v][j], sum);
    const float rho = __frsqrt_rn(__fdiv_rn(block_sum(sum, part), static_cast<float>(p.cols)) + p.eps);
    if (p.inv_rms != nullptr && threadIdx.x == 0) p.inv_rms[row] = rho;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int i = v * blockDim.x + threadIdx.x;
        const bool mine = i < vectors;
        float y[8];
        if (mine) {
            load_weight<W32>(p.weight, i * 8, y);
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = z[v][j] * rho * y[j];
            if (p.y != nullptr) *reinterpret_cast<uint4*>(p.y + row * p.cols + i * 8) = pack8(y);
        }
        if (p.codes != nullptr) {
            uint32_t big = 0;
            if (mine) {
#pragma unroll
                for (int j = 0; j < 8; ++j) big = max(big, abs_bits(y[j]));
            }
#pragma unroll
            for (int off = 8; off > 0; off >>= 1) big = max(big, __shfl_xor_sync(0xffffffffu, big, off));
            float inv;
            const float scale = block_scale(big, inv);
            if (mine) {
                uint2 q;
                q.x = mxfp8_convert4(y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv);
                q.y = mxfp8_convert4(y[4] * inv, y[5] * inv, y[6] * inv, y[7] * inv);
                *reinterpret_cast<uint2*>(p.codes + row * p.codes_stride + i * 8) = q;
                if ((i & 15) == 0) p.scales[row * p.scale_row_stride + (i >> 4) * p.scale_block_stride] = scale;
            }
        }
    }
}

struct NormBackward {
    const bf16 *d_y, *d_hidden, *z;
    const void* weight;
    const float* inv_rms;
    bf16* d_x;
    float* partials;   // [gridDim.x, cols]
    long long z_stride, rows;
    int cols;
};

// A block takes every gridDim.x-th row and keeps its share of the weight gradient in registers.
template <int V, bool W32>
__global__ void __launch_bounds__(V == 1 ? 256 : 512) rms_norm_backward_kernel(const NormBackward p) {
    __shared__ float part[2][32];
    const int vectors = p.cols >> 3;
    float dw[V][8];
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
        for (int j = 0; j < 8; ++j) dw[v][j] = 0.0f;
    int flip = 0;
    for (long long row = blockIdx.x; row < p.rows; row += gridDim.x, flip ^= 1) {
        const float rho = p.inv_rms[row];
        float z[V][8], g[V][8];
        float dot = 0.0f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int i = v * blockDim.x + threadIdx.x;
            if (i < vectors) {
                float w[8];
                unpack8(*reinterpret_cast<const uint4*>(p.z + row * p.z_stride + i * 8), z[v]);
                unpack8(*reinterpret_cast<const uint4*>(p.d_y + row * p.cols + i * 8), g[v]);
                load_weight<W32>(p.weight, i * 8, w);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    dw[v][j] = fmaf(g[v][j], z[v][j] * rho, dw[v][j]);
                    g[v][j] *= w[j];
                    dot = fmaf(g[v][j], z[v][j], dot);
                }
            }
        }
        const float c = rho * rho * __fdiv_rn(block_sum(dot, part[flip]), static_cast<float>(p.cols));
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int i = v * blockDim.x + threadIdx.x;
            if (i < vectors) {
                float d[8];
                if (p.d_hidden != nullptr) unpack8(*reinterpret_cast<const uint4*>(p.d_hidden + row * p.cols + i * 8), d);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float dx = rho * (g[v][j] - z[v][j] * c);
                    d[j] = p.d_hidden != nullptr ? dx + d[j] : dx;
                }
                *reinterpret_cast<uint4*>(p.d_x + row * p.cols + i * 8) = pack8(d);
            }
        }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int i = v * blockDim.x + threadIdx.x;
        if (i < vectors) {
            float4* out = reinterpret_cast<float4*>(p.partials + static_cast<long long>(blockIdx.x) * p.cols + i * 8);
            out[0] = make_float4(dw[v][0], dw[v][1], dw[v][2], dw[v][3]);
            out[1] = make_float4(dw[v][4], dw[v][5], dw[v][6], dw[v][7]);
        }
    }
}

// dw = sum of the blocks' shares, in block order: 32 columns x 8 phases a block.
template <bool W32>
__global__ void __launch_bounds__(256) rms_norm_weight_grad_kernel(const float* __restrict__ partials, int blocks, int cols, void* d_weight) {
    __shared__ float part[8][32];
    const int lane = threadIdx.x & 31, phase = threadIdx.x >> 5;
    const int col = blockIdx.x * 32 + lane;
    float s = 0.0f;
    if (col < cols)
        for (int b = phase; b < blocks; b += 8) s += partials[static_cast<long long>(b) * cols + col];
    part[phase][lane] = s;
    __syncthreads();
    if (phase == 0 && col < cols) {
        s = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) s += part[i][lane];
        if (W32) static_cast<float*>(d_weight)[col] = s;
        else static_cast<bf16*>(d_weight)[col] = __float2bfloat16(s);
    }
}

int backward_blocks(long long rows) {
    const long long most = 2LL * sm_count();
    return static_cast<int>(rows < most ? rows : most);
}

// Vectors of 8 columns per thread (1, 2 or 4) and threads for a row: vectors are added while the block is wider than `wide`.
void row_shape(int cols, int wide, int& v, int& threads) {
    const int vectors = cols / 8;
    v = 1;
    while (v < 4 && (vectors + v - 1) / v > (v == 1 ? 256 : wide)) v *= 2;
    threads = ((vectors + v - 1) / v + 31) / 32 * 32;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace mok

extern "C" int64_t mok_rms_norm_scratch_bytes(int64_t rows, int hidden) {
    if (rows <= 0 || hidden <= 0) return 0;
    return static_cast<int64_t>(mok::backward_blocks(rows)) * hidden * 4;
}

extern "C" int mok_rms_norm_forward(const void* x, int64_t x_stride, const void* residual, int64_t residual_stride, const void* weight,
                                    int weight_is_f32, int64_t rows, int hidden, float eps, void* hidden_out, void* y, void* codes,
                                    int64_t codes_stride, float* scales, int64_t scale_row_stride, int64_t scale_block_stride,
                                    float* inv_rms, mok_stream_t stream) {
    using namespace mok;
    if (rows < 0 || rows > 0x7fffffffLL || hidden <= 0 || hidden % 8 != 0) return MOK_ERR_INVALID_ARGUMENT;
    if (hidden > kMaxHidden) return MOK_ERR_TOO_LARGE;
    if (rows == 0) return MOK_OK;
    if (!x || !weight || (!y && !codes) || (codes == nullptr) != (scales == nullptr)) return MOK_ERR_INVALID_ARGUMENT;
    if (!aligned16(x) || !aligned16(residual) || !aligned16(weight) || !aligned16(hidden_out) || !aligned16(y) ||
        (reinterpret_cast<uintptr_t>(codes) & 7) != 0)
        return MOK_ERR_INVALID_ARGUMENT;
    if (x_stride % 8 != 0 || residual_stride % 8 != 0 || codes_stride % 8 != 0 || x_stride < 0 || residual_stride < 0)
        return MOK_ERR_INVALID_ARGUMENT;
    if (codes != nullptr && codes_stride < hidden) return MOK_ERR_INVALID_ARGUMENT;
    NormForward p{};
    p.x = static_cast<const bf16*>(x);
    p.residual = static_cast<const bf16*>(residual);
    p.weight = weight;
    p.hidden = static_cast<bf16*>(hidden_out);
    p.y = static_cast<bf16*>(y);
    p.codes = static_cast<uint8_t*>(codes);
    p.scales = scales;
    p.inv_rms = inv_rms;
    p.x_stride = x_stride;
    p.residual_stride = residual_stride;
    p.codes_stride = codes_stride;
    p.scale_row_stride = scale_row_stride;
    p.scale_block_stride = scale_block_stride;
    p.rows = rows;
    p.cols = hidden;
    p.eps = eps;
    int v, threads;
    row_shape(hidden, 256, v, threads);
    const int grid = static_cast<int>(rows);
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
#define MOK_NORM(V)                                                                      \
    do {                                                                                 \
        if (weight_is_f32) rms_norm_forward_kernel<V, true><<<grid, threads, 0, s>>>(p); \
        else rms_norm_forward_kernel<V, false><<<grid, threads, 0, s>>>(p);              \
    } while (0)
    if (v == 1) MOK_NORM(1);
    else if (v == 2) MOK_NORM(2);
    else MOK_NORM(4);
#undef MOK_NORM
    MOK_LAUNCH_CHECK("rms_norm_forward_kernel");
    return MOK_OK;
}

extern "C" int mok_rms_norm_backward(const void* d_y, const void* d_hidden, const void* z, int64_t z_stride, const void* weight,
                                     int weight_is_f32, const float* inv_rms, int64_t rows, int hidden, void* d_x, void* d_weight,
                                     float* scratch, mok_stream_t stream) {
    using namespace mok;
    if (rows <= 0 || rows > 0x7fffffffLL || hidden <= 0 || hidden % 8 != 0) return MOK_ERR_INVALID_ARGUMENT;
    if (hidden > kMaxHidden) return MOK_ERR_TOO_LARGE;
    if (!d_y || !z || !weight || !inv_rms || !d_x || !d_weight || !scratch) return MOK_ERR_INVALID_ARGUMENT;
    if (!aligned16(d_y) || !aligned16(d_hidden) || !aligned16(z) || !aligned16(weight) || !aligned16(d_x) || !aligned16(scratch) ||
        z_stride % 8 != 0 || z_stride < 0)
        return MOK_ERR_INVALID_ARGUMENT;
    NormBackward p{};
    p.d_y = static_cast<const bf16*>(d_y);
    p.d_hidden = static_cast<const bf16*>(d_hidden);
    p.z = static_cast<const bf16*>(z);
    p.weight = weight;
    p.inv_rms = inv_rms;
    p.d_x = static_cast<bf16*>(d_x);
    p.partials = scratch;
    p.z_stride = z_stride;
    p.rows = rows;
    p.cols = hidden;
    int v, threads;
    row_shape(hidden, 512, v, threads);
    const int grid = backward_blocks(rows);
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
#define MOK_NORM(V)                                                                       \
    do {                                                                                  \
        if (weight_is_f32) rms_norm_backward_kernel<V, true><<<grid, threads, 0, s>>>(p); \
        else rms_norm_backward_kernel<V, false><<<grid, threads, 0, s>>>(p);              \
    } while (0)
    if (v == 1) MOK_NORM(1);
    else if (v == 2) MOK_NORM(2);
    else MOK_NORM(4);
#undef MOK_NORM
    MOK_LAUNCH_CHECK("rms_norm_backward_kernel");
    if (weight_is_f32) rms_norm_weight_grad_kernel<true><<<(hidden + 31) / 32, 256, 0, s>>>(scratch, grid, hidden, d_weight);
    else rms_norm_weight_grad_kernel<false><<<(hidden + 31) / 32, 256, 0, s>>>(scratch, grid, hidden, d_weight);
    MOK_LAUNCH_CHECK("rms_norm_weight_grad_kernel");
    return MOK_OK;
}
