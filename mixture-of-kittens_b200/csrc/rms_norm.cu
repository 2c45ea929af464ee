// Root-mean-square norm with the residual's addition: z = x + r in fp32, rho = (mean z^2 + eps)^-1/2, y = z rho w, as bf16
// and / or as e4m3 with a scale per 128 columns; hidden = bf16(z) is the next residual stream.  The norm is taken of z before
// it is rounded.  Backward, with z read back from `hidden`:
//   g = dy w,  dx = dr = rho (g - z rho^2 mean(g z)) + dhidden,  dw = sum over rows of dy z rho.
// That z is off by 2^-8 of itself at most, which dw's terms take over: against 64 bits dw is off by 0.0024 of its norm, where its
// rounding to bf16 alone gives 0.0016 (dx: 0.0017 either way).  Exact sums would take x and r instead of one `hidden`, a fifth more
// bytes, and keep both from the forward on.
// Both are bound by HBM (by launch and latency for a few rows): every input is read once and all sums are fp32.  16384 x 7168 with
// a residual: forward 158 us, 5.9 TB/s; with 8-bit output instead 195 us; backward with d_hidden 172 us, 5.5 TB/s.  2048 columns:
// 45, 53 and 62 us.  One row: 4 us, which is the launch.
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
    double inv_cols;
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

// Sum over the block, the same value in every thread, in a fixed order.  `part` holds one value per warp; the caller alternates
// between two of them, so that one barrier per sum is enough.
template <class T>
__device__ __forceinline__ T block_sum(T v, T* part) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
    const int warps = blockDim.x >> 5;
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = (threadIdx.x & 31) < warps ? part[threadIdx.x & 31] : T(0);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
    return v;
}

// y / scale in fp32 is a few units off in its last place, which decides the code only where it comes that close to the middle
// between two codes: with 20 bits below e4m3's mantissa, one value in 130 000.  Those are made from 64 bits (in fp32, sums of 32
// squares of bf16 values come out 4e-8 too small on average, which alone turned one code of 5 million).  Codes below 2^-6 have
// their middles elsewhere; half a step there is 2^-18 of the largest value.
__device__ __forceinline__ uint32_t from_middle(float v) { return (__float_as_uint(v) - 0x7FFFCu) & 0xFFFFFu; }
constexpr uint32_t kNearMiddle = 8;
template <bool WIDE>
struct Sum {
    typedef float type;
};
template <>
struct Sum<true> {
    typedef double type;
};

// One row per block; a thread holds V vectors of 8 columns, so 16 adjacent lanes hold one block of 128.  With codes the bounds
// below ask for more blocks an SM than registers allow without spills, which all lie on the rare path: 16384 x 7168 in 195 us, 207
// with four blocks.  z kept in shared memory (225 us) and the rare values listed there for the block's end (221 us) took longer.
template <int V, int THREADS, bool W32, bool CODES>
__global__ void __launch_bounds__(THREADS, THREADS == 512 ? 2 : !CODES ? 1 : V == 4 ? 5 : V == 2 ? 6 : 7)
    rms_norm_forward_kernel(const NormForward p) {
    __shared__ typename Sum<CODES>::type part[32];   // codes: sums of eight squares are added in 64 bits
    const long long row = blockIdx.x;
    const int vectors = p.cols >> 3;
    const bf16* x = p.x + row * p.x_stride;
    const bf16* r = p.residual == nullptr ? nullptr : p.residual + row * p.residual_stride;
    float z[V][8];
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
    typename Sum<CODES>::type sum = 0;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        float eight = CODES ? 0.0f : static_cast<float>(sum);
#pragma unroll
        for (int j = 0; j < 8; ++j) eight = fmaf(z[v][j], z[v][j], eight);
        sum = CODES ? sum + eight : eight;
    }
    float rho;
    double mean = 0.0;
    const typename Sum<CODES>::type squares = block_sum<typename Sum<CODES>::type>(sum, part);
    if (CODES) {
        mean = squares * p.inv_cols + p.eps;
        rho = __frsqrt_rn(static_cast<float>(mean));
    } else {
        rho = __frsqrt_rn(__fdiv_rn(static_cast<float>(squares), static_cast<float>(p.cols)) + p.eps);
    }
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
            if (!CODES || p.y != nullptr) *reinterpret_cast<uint4*>(p.y + row * p.cols + i * 8) = pack8(y);
        }
        if (CODES) {
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
                uint32_t nearest = kNearMiddle;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    y[j] *= inv;
                    nearest = min(nearest, from_middle(y[j]));
                }
                if (nearest < kNearMiddle) {
                    float w[8];
                    load_weight<W32>(p.weight, i * 8, w);
                    const double r0 = rho, better = fma(0.5 * r0, fma(-mean * r0, r0, 1.0), r0);   // a Newton step
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (from_middle(y[j]) < kNearMiddle) y[j] = static_cast<float>(better * z[v][j] * w[j] * inv);
                }
                *reinterpret_cast<uint2*>(p.codes + row * p.codes_stride + i * 8) =
                    make_uint2(mxfp8_convert4(y[0], y[1], y[2], y[3]), mxfp8_convert4(y[4], y[5], y[6], y[7]));
                if ((i & 15) == 0) p.scales[row * p.scale_row_stride + (i >> 4) * p.scale_block_stride] = scale;
            }
        }
    }
}

// Eight weights of a thread's columns, as they are stored.
template <bool W32>
struct Weight8 {
    uint4 raw[W32 ? 2 : 1];
    __device__ __forceinline__ void load(const void* weight, int i, int vectors) {
#pragma unroll
        for (int k = 0; k < (W32 ? 2 : 1); ++k)
            raw[k] = i < vectors ? reinterpret_cast<const uint4*>(weight)[i * (W32 ? 2 : 1) + k] : make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ float at(int j) const {
        const uint4& q = raw[W32 ? j >> 2 : 0];
        const int k = W32 ? j & 3 : j >> 1;
        const uint32_t u = k == 0 ? q.x : k == 1 ? q.y : k == 2 ? q.z : q.w;
        return __uint_as_float(W32 ? u : (j & 1) ? (u & 0xFFFF0000u) : (u << 16));
    }
};

struct NormBackward {
    const bf16 *d_y, *d_hidden, *z;
    const void* weight;
    const float* inv_rms;
    bf16* d_x;
    float* partials;   // [gridDim.x, cols]
    long long z_stride, rows;
    int cols, stages;
};

// A block takes every gridDim.x-th row and keeps its share of the weight gradient in registers.  The rows to come are on their way to
// shared memory meanwhile (each thread copies, waits for and reads its own columns, so a row costs one barrier, that of its sum): with
// loads to registers, those of d_hidden behind the sum, a row was two trips to memory and 16384 x 7168 took 408 us.  Two blocks an SM
// fill each other's barriers (one of them with a ring of four rows 299 us, two with two rows 192 us, now 172 us).
template <int V, int THREADS, int BLOCKS, bool W32>
__global__ void __launch_bounds__(THREADS, BLOCKS) rms_norm_backward_kernel(const NormBackward p) {
    extern __shared__ __align__(16) uint8_t ring[];   // [stage][z, d_y, d_hidden][cols]
    __shared__ float part[2][32];
    const int vectors = p.cols >> 3;
    const long long row_bytes = p.cols * 2;
    const int inputs = p.d_hidden != nullptr ? 3 : 2;
    float dw[V][8];
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
        for (int j = 0; j < 8; ++j) dw[v][j] = 0.0f;
    allow_next_kernel();
    auto slot = [&](int stage, int input, int i) { return ring + (stage * inputs + input) * row_bytes + i * 16; };
    auto fetch = [&](long long row, int stage) {
        if (row < p.rows) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const int i = v * blockDim.x + threadIdx.x;
                if (i < vectors) {
                    copy16(smem_u32(slot(stage, 0, i)), p.z + row * p.z_stride + i * 8);
                    copy16(smem_u32(slot(stage, 1, i)), p.d_y + row * p.cols + i * 8);
                    if (inputs == 3) copy16(smem_u32(slot(stage, 2, i)), p.d_hidden + row * p.cols + i * 8);
                }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    for (int s = 0; s < p.stages - 1; ++s) fetch(blockIdx.x + static_cast<long long>(s) * gridDim.x, s);
    Weight8<W32> w[V];
#pragma unroll
    for (int v = 0; v < V; ++v) w[v].load(p.weight, v * blockDim.x + threadIdx.x, vectors);
    int flip = 0, stage = 0;
    float rho = p.inv_rms[blockIdx.x];
    for (long long row = blockIdx.x; row < p.rows; row += gridDim.x, flip ^= 1) {
        const float next_rho = row + gridDim.x < p.rows ? p.inv_rms[row + gridDim.x] : 0.0f;
        const int behind = stage == 0 ? p.stages - 1 : stage - 1;   // the stage of the row before, which this thread has read
        fetch(row + static_cast<long long>(p.stages - 1) * gridDim.x, behind);
        if (p.stages == 2) asm volatile("cp.async.wait_group 1;" ::: "memory");
        else if (p.stages == 3) asm volatile("cp.async.wait_group 2;" ::: "memory");
        else asm volatile("cp.async.wait_group 3;" ::: "memory");
        float dot = 0.0f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int i = v * blockDim.x + threadIdx.x;
            if (i < vectors) {
                float z[8], g[8];
                unpack8(*reinterpret_cast<const uint4*>(slot(stage, 0, i)), z);
                unpack8(*reinterpret_cast<const uint4*>(slot(stage, 1, i)), g);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    dw[v][j] = fmaf(g[j], z[j] * rho, dw[v][j]);
                    dot = fmaf(g[j] * w[v].at(j), z[j], dot);
                }
            }
        }
        const float c = rho * rho * __fdiv_rn(block_sum(dot, part[flip]), static_cast<float>(p.cols));
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int i = v * blockDim.x + threadIdx.x;
            if (i < vectors) {   // read again: kept in registers they would leave room for half the threads
                float z[8], g[8], d[8];
                unpack8(*reinterpret_cast<const uint4*>(slot(stage, 0, i)), z);
                unpack8(*reinterpret_cast<const uint4*>(slot(stage, 1, i)), g);
                if (inputs == 3) unpack8(*reinterpret_cast<const uint4*>(slot(stage, 2, i)), d);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float dx = rho * (g[j] * w[v].at(j) - z[j] * c);
                    d[j] = inputs == 3 ? dx + d[j] : dx;
                }
                *reinterpret_cast<uint4*>(p.d_x + row * p.cols + i * 8) = pack8(d);
            }
        }
        rho = next_rho;
        if (++stage == p.stages) stage = 0;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
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

// dw = sum of the blocks' shares in a fixed order: 32 columns x 32 phases a block.
template <bool W32>
__global__ void __launch_bounds__(1024) rms_norm_weight_grad_kernel(const float* __restrict__ partials, int blocks, int cols, void* d_weight) {
    __shared__ float part[32][33];
    const int lane = threadIdx.x & 31, phase = threadIdx.x >> 5;
    const int col = blockIdx.x * 32 + lane;
    float s = 0.0f;
    wait_previous_kernel();
    if (col < cols) {
#pragma unroll 8
        for (int b = phase; b < blocks; b += 32) s += partials[static_cast<long long>(b) * cols + col];
    }
    part[lane][phase] = s;
    __syncthreads();
    s = part[phase][lane];
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    const int out = blockIdx.x * 32 + phase;
    if (lane == 0 && out < cols) {
        if (W32) static_cast<float*>(d_weight)[out] = s;
        else static_cast<bf16*>(d_weight)[out] = __float2bfloat16(s);
    }
}

// Blocks of the backward: as many an SM as registers and rings of two rows leave room for.  16384 x 4096: two an SM 125 us, four 102 us.
int backward_blocks_per_sm(int cols) { return cols <= 4096 ? 4 : cols <= 8192 ? 2 : 1; }
int backward_blocks(long long rows, int cols) {
    const long long most = static_cast<long long>(backward_blocks_per_sm(cols)) * sm_count();
    return static_cast<int>(rows < most ? rows : most);
}

// Vectors of 8 columns per thread and threads for a row of the forward: vectors are added while the block is wider than 256.
void row_shape(int cols, int& v, int& threads) {
    const int vectors = cols / 8;
    v = 1;
    while (v < 4 && (vectors + v - 1) / v > 256) v *= 2;
    threads = ((vectors + v - 1) / v + 31) / 32 * 32;
}

template <int V, int THREADS, int BLOCKS, bool W32>
int launch_backward(const NormBackward& p, int grid, int threads, int smem, cudaStream_t stream) {
    static int ready[16] = {0};
    int dev = 0;
    MOK_CUDA_CHECK(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 16) return MOK_ERR_UNSUPPORTED;
    const auto rms_norm_backward = rms_norm_backward_kernel<V, THREADS, BLOCKS, W32>;
    if (ready[dev] == 0) {
        MOK_CUDA_CHECK(cudaFuncSetAttribute(rms_norm_backward, cudaFuncAttributeMaxDynamicSharedMemorySize, 224 * 1024));
        ready[dev] = 1;
    }
    rms_norm_backward<<<grid, threads, smem, stream>>>(p);
    MOK_LAUNCH_CHECK("rms_norm_backward_kernel");
    return MOK_OK;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace mok

extern "C" int64_t mok_rms_norm_scratch_bytes(int64_t rows, int hidden) {
    if (rows <= 0 || hidden <= 0) return 0;
    return static_cast<int64_t>(mok::backward_blocks(rows, hidden)) * hidden * 4;
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
    p.inv_cols = 1.0 / hidden;
    int v, threads;
    row_shape(hidden, v, threads);
    const int grid = static_cast<int>(rows);
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const bool w32 = weight_is_f32 != 0, with_codes = codes != nullptr;
    void (*kernel)(NormForward);
#define MOK_NORM(V, THREADS)                                                                                                     \
    kernel = with_codes ? w32 ? rms_norm_forward_kernel<V, THREADS, true, true> : rms_norm_forward_kernel<V, THREADS, false, true> \
                        : w32 ? rms_norm_forward_kernel<V, THREADS, true, false> : rms_norm_forward_kernel<V, THREADS, false, false>
    if (v == 1) MOK_NORM(1, 256);
    else if (v == 2) MOK_NORM(2, 256);
    else if (threads <= 256) MOK_NORM(4, 256);
    else MOK_NORM(4, 512);
#undef MOK_NORM
    kernel<<<grid, threads, 0, s>>>(p);
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
    const int vectors = hidden / 8, v = vectors <= 256 ? 1 : 2, threads = ((vectors + v - 1) / v + 31) / 32 * 32;
    const int row_bytes = (d_hidden != nullptr ? 3 : 2) * hidden * 2, room = (224 * 1024) / backward_blocks_per_sm(hidden) - 1024;
    p.stages = room / row_bytes > 4 ? 4 : room / row_bytes;   // 2 at 16384 columns
    const int grid = backward_blocks(rows, hidden), smem = p.stages * row_bytes;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    using Launch = int (*)(const NormBackward&, int, int, int, cudaStream_t);
    Launch launch;
    if (v == 1) launch = weight_is_f32 ? launch_backward<1, 256, 4, true> : launch_backward<1, 256, 4, false>;
    else if (threads <= 256) launch = weight_is_f32 ? launch_backward<2, 256, 4, true> : launch_backward<2, 256, 4, false>;
    else if (threads <= 512) launch = weight_is_f32 ? launch_backward<2, 512, 2, true> : launch_backward<2, 512, 2, false>;
    else launch = weight_is_f32 ? launch_backward<2, 1024, 1, true> : launch_backward<2, 1024, 1, false>;
    MOK_TRY(launch(p, grid, threads, smem, s));
    const dim3 columns((hidden + 31) / 32);
    const float* shares = scratch;
    if (weight_is_f32) return launch_early(rms_norm_weight_grad_kernel<true>, "rms_norm_weight_grad_kernel", columns, 1024, 0, s, shares, grid, hidden, d_weight);
    return launch_early(rms_norm_weight_grad_kernel<false>, "rms_norm_weight_grad_kernel", columns, 1024, 0, s, shares, grid, hidden, d_weight);
}
