// Products of weight rows with a few tokens, for kernels that are bound by reading the weights once: out[row, token] = sum over k
// of W[row, k] * x[token, k].
//
// A block has four producer warps and eight consumer warps.  The producers copy pieces of up to 32 weight rows and the rows of up
// to 32 tokens, kChunk elements of k at a time, into a ring of stages with cp.async (a warp's 32 x 16 bytes are one row of a chunk:
// any row count, stride and gather), and run ahead of the consumers as far as the ring reaches; about 100 KB in flight per SM is
// what HBM needs.  Bulk copies, one per row, were measured first: an SM issues about one in 60 clocks, so 512-byte rows came in at
// 1.4 - 1.8 TB/s and 1024-byte rows at 2.2 - 3.4 TB/s.  The consumers split k: a warp takes every eighth slice of a chunk, multiplies it with mma.sync (weights on the M
// side, tokens on the N side of 8) and keeps its own sums, which the eight warps add in a fixed order when a piece is done.
// tcgen05 would need 128 rows a tile, which leaves SMs idle at these sizes; the tensor work here is a few percent of the time.
//
// The order of k within a slice is free as long as both operands use the same one: lane (g, t) of an mma takes elements 8 t .. 8 t
// + 7 of rows g and g + 8, one 16-byte (8-byte in e4m3) shared-memory load per row, for two mma of K = 16.  Row pitches of 64 (32)
// bytes modulo 128 make these loads free of bank conflicts.
#pragma once

#include "mok_common.cuh"

namespace mok {
namespace stream {

constexpr int kConsumers = 8;                       // warps
constexpr int kConsumerThreads = kConsumers * 32;
constexpr int kProducers = 4;
constexpr int kProducerThreads = kProducers * 32;
constexpr int kThreads = kConsumerThreads + kProducerThreads;
constexpr int kPieceRows = 32;                      // weight rows of a piece: two m16 tiles
constexpr int kMaxStages = 8;

// W8 / X8: weights / tokens in e4m3 instead of bf16.
template <bool W8, bool X8>
struct Form {
    static constexpr int kChunk = W8 ? 512 : 256;               // elements of k per stage
    static constexpr int kRowBytes = kChunk * (W8 ? 1 : 2);     // 512
    static constexpr int kRowPitch = kRowBytes + (W8 ? 32 : 64);
    static constexpr int kTokenBytes = kChunk * (X8 ? 1 : 2);
    static constexpr int kTokenPitch = kTokenBytes + (X8 ? 32 : 64);
    static constexpr int kSlices = kChunk / 32 / kConsumers;    // slices of 32 per warp and chunk
    static constexpr int stage_bytes(int tokens) { return kPieceRows * kRowPitch + tokens * kTokenPitch; }
};

__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global.L2::256B [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// One arrival once every copy that this thread has issued so far is done.
__device__ __forceinline__ void arrive_when_copied(uint32_t bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void wait_copies() { asm volatile("cp.async.wait_all;" ::: "memory"); }
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void consumer_barrier() { asm volatile("bar.sync 1, %0;" ::"n"(kConsumerThreads) : "memory"); }
// The other kernels of a stream: let the next one begin, and wait for the one before to be done and visible.
__device__ __forceinline__ void allow_next_kernel() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_previous_kernel() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Ring state that producer and consumers walk alike.
struct Ring {
    uint32_t base, full, empty;   // shared addresses: stages, barriers
    int stage_bytes, stages;
    int stage = 0;
    uint32_t phase = 0;
    __device__ __forceinline__ void advance() {
        if (++stage == stages) {
            stage = 0;
            phase ^= 1u;
        }
    }
    __device__ __forceinline__ void init() const {   // one thread
        for (int s = 0; s < stages; ++s) {
            mbar_init(full + 8 * s, kProducerThreads);
            mbar_init(empty + 8 * s, kConsumers);
        }
        mbar_fence_init();
    }
};

// What a producer warp copies of a piece: every kProducers-th weight row and token row, as this lane's address in the row at k = 0
// (nullptr: no such row).  Found once per piece, so that a chunk costs its producers little more than the copies themselves: with
// addresses worked out chunk by chunk they were the bottleneck (1500 clocks a chunk, 2.2 TB/s).
template <int NT>
struct Feed {
    static constexpr int kWeights = kPieceRows / kProducers, kTokens = 8 * NT / kProducers;
    const uint8_t *weight[kWeights], *token[kTokens];
};
template <typename F, int NT>
__device__ __forceinline__ void copy_weights(uint32_t stage, const Feed<NT>& f, int k0, int len, int producer, int lane) {
    constexpr int kBytes = F::kRowBytes / F::kChunk;
    static_assert(F::kRowBytes == 512, "one copy of 16 bytes per lane");
    const long long at = static_cast<long long>(k0) * kBytes;
    const uint32_t dst = stage + producer * F::kRowPitch + lane * 16;
    if (lane * 16 < len * kBytes) {
#pragma unroll
        for (int j = 0; j < Feed<NT>::kWeights; ++j)
            if (f.weight[j] != nullptr) copy16(dst + j * kProducers * F::kRowPitch, f.weight[j] + at);
    }
}
template <typename F, int NT>
__device__ __forceinline__ void copy_tokens(uint32_t stage, const Feed<NT>& f, int k0, int len, int producer, int lane) {
    constexpr int kBytes = F::kTokenBytes / F::kChunk;
    const long long at = static_cast<long long>(k0) * kBytes;
    const uint32_t dst = stage + kPieceRows * F::kRowPitch + producer * F::kTokenPitch + lane * 16;
#pragma unroll
    for (int half = 0; half < F::kTokenBytes / 512; ++half)
        if (half * 512 + lane * 16 < len * kBytes) {
#pragma unroll
            for (int j = 0; j < Feed<NT>::kTokens; ++j)
                if (f.token[j] != nullptr) copy16(dst + j * kProducers * F::kTokenPitch + half * 512, f.token[j] + at + half * 512);
        }
}
// The producers' side of a piece from k0 on, chunk by chunk.  False: a wait ran out.
template <typename F, int NT>
__device__ __forceinline__ bool produce(Ring& ring, volatile int* abort_flag, uint32_t* status, const Feed<NT>& f, int k0, int k_total, int producer,
                                        int lane) {
    for (; k0 < k_total; k0 += F::kChunk) {
        if (!mbar_wait(ring.empty + 8 * ring.stage, ring.phase ^ 1u, abort_flag, status)) return false;
        const int len = min(F::kChunk, k_total - k0);
        const uint32_t stage = ring.base + ring.stage * ring.stage_bytes;
        copy_weights<F, NT>(stage, f, k0, len, producer, lane);
        copy_tokens<F, NT>(stage, f, k0, len, producer, lane);
        arrive_when_copied(ring.full + 8 * ring.stage);
        ring.advance();
    }
    return true;
}

// ---- consumer -----------------------------------------------------------------------------------------------------
__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t two_codes) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<uint16_t>(two_codes)));
    return h;
}
// Two of a word's four e4m3 codes as bf16: sign and the seven other bits moved to where bf16 has them read as the value times
// 2^-120 (subnormal codes land among bf16's subnormal numbers), and one exact multiplication puts that right.  A NaN code would
// read as +-480: nan_codes finds those.
__device__ __forceinline__ uint32_t e4m3x2_to_bf16x2(uint32_t word, uint32_t selector) {
    const uint32_t p = __byte_perm(word, 0, selector);   // code << 8 in each half
    const uint32_t v = ((p & 0x7F007F00u) >> 4) | (p & 0x80008000u);
    const uint32_t two_to_120 = 0x7B807B80u;
    const __nv_bfloat162 r = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&v), *reinterpret_cast<const __nv_bfloat162*>(&two_to_120));
    return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t nan_codes(uint32_t word) { return ((word & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u; }

// The first `count` (may be <= 0) of eight codes, the others zero.
__device__ __forceinline__ uint2 keep_codes(uint2 v, int count) {
    if (count < 8) v.y = count > 4 ? v.y & (0xFFFFFFFFu >> (8 * (8 - count))) : 0u;
    if (count < 4) v.x = count > 0 ? v.x & (0xFFFFFFFFu >> (8 * (4 - count))) : 0u;
    return v;
}

// Adds a warp's share of one stage to `acc`; `k_len` elements of the chunk are valid (a multiple of 32 unless X8).
// nan: per m tile the NaN codes met in rows g (bit 7 of each byte) and, in [1], rows g + 8.
template <bool W8, bool X8, int NT>
__device__ __forceinline__ void multiply(const uint8_t* stage, int k_len, int m_tiles, int n_tiles, int warp, int lane, float (&acc)[2][NT][4],
                                         uint32_t (&nan)[2][2]) {
    typedef Form<W8, X8> F;
    const int g = lane >> 2, t = lane & 3;
    const uint8_t* weights = stage + g * F::kRowPitch;
    const uint8_t* tokens = stage + kPieceRows * F::kRowPitch + g * F::kTokenPitch;
#pragma unroll
    for (int s = 0; s < F::kSlices; ++s) {
        const int k = (warp * F::kSlices + s) * 32 + 8 * t;   // of this lane
        if ((warp * F::kSlices + s) * 32 >= k_len) break;
        uint32_t b[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            if (n < n_tiles) {
                if (X8) {
                    const uint2 v = keep_codes(*reinterpret_cast<const uint2*>(tokens + n * 8 * F::kTokenPitch + k), k_len - k);
                    b[n][0] = e4m3x2_to_f16x2(v.x); b[n][1] = e4m3x2_to_f16x2(v.x >> 16);
                    b[n][2] = e4m3x2_to_f16x2(v.y); b[n][3] = e4m3x2_to_f16x2(v.y >> 16);
                } else {
                    const uint4 v = *reinterpret_cast<const uint4*>(tokens + n * 8 * F::kTokenPitch + k * 2);
                    b[n][0] = v.x; b[n][1] = v.y; b[n][2] = v.z; b[n][3] = v.w;
                }
            }
        }
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            if (m >= m_tiles) break;
            uint32_t lo[4], hi[4];
            if (W8) {
                uint2 l = *reinterpret_cast<const uint2*>(weights + (m * 16) * F::kRowPitch + k);
                uint2 h = *reinterpret_cast<const uint2*>(weights + (m * 16 + 8) * F::kRowPitch + k);
                if (X8) {
                    l = keep_codes(l, k_len - k);
                    h = keep_codes(h, k_len - k);
                    lo[0] = e4m3x2_to_f16x2(l.x); lo[1] = e4m3x2_to_f16x2(l.x >> 16);
                    lo[2] = e4m3x2_to_f16x2(l.y); lo[3] = e4m3x2_to_f16x2(l.y >> 16);
                    hi[0] = e4m3x2_to_f16x2(h.x); hi[1] = e4m3x2_to_f16x2(h.x >> 16);
                    hi[2] = e4m3x2_to_f16x2(h.y); hi[3] = e4m3x2_to_f16x2(h.y >> 16);
                } else {
                    lo[0] = e4m3x2_to_bf16x2(l.x, 0x1404); lo[1] = e4m3x2_to_bf16x2(l.x, 0x3424);
                    lo[2] = e4m3x2_to_bf16x2(l.y, 0x1404); lo[3] = e4m3x2_to_bf16x2(l.y, 0x3424);
                    hi[0] = e4m3x2_to_bf16x2(h.x, 0x1404); hi[1] = e4m3x2_to_bf16x2(h.x, 0x3424);
                    hi[2] = e4m3x2_to_bf16x2(h.y, 0x1404); hi[3] = e4m3x2_to_bf16x2(h.y, 0x3424);
                    nan[m][0] |= nan_codes(l.x) | nan_codes(l.y);
                    nan[m][1] |= nan_codes(h.x) | nan_codes(h.y);
                }
            } else {
                const uint4 l = *reinterpret_cast<const uint4*>(weights + (m * 16) * F::kRowPitch + k * 2);
                const uint4 h = *reinterpret_cast<const uint4*>(weights + (m * 16 + 8) * F::kRowPitch + k * 2);
                lo[0] = l.x; lo[1] = l.y; lo[2] = l.z; lo[3] = l.w;
                hi[0] = h.x; hi[1] = h.y; hi[2] = h.z; hi[3] = h.w;
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                if (n < n_tiles) {
                    if (X8) {
                        mma_f16(acc[m][n], lo[0], hi[0], lo[1], hi[1], b[n][0], b[n][1]);
                        mma_f16(acc[m][n], lo[2], hi[2], lo[3], hi[3], b[n][2], b[n][3]);
                    } else {
                        mma_bf16(acc[m][n], lo[0], hi[0], lo[1], hi[1], b[n][0], b[n][1]);
                        mma_bf16(acc[m][n], lo[2], hi[2], lo[3], hi[3], b[n][2], b[n][3]);
                    }
                }
            }
        }
    }
}

// Scales of a lane's rows (g and g + 8 of each m tile) and, X8, of its tokens (2 t and 2 t + 1 of each n tile), one per 128 of k.
template <bool W8, bool X8, int NT>
struct Scales {
    const float *lo[2], *hi[2], *x[NT][2];
    long long row_block, x_block;   // elements from one block of k to the next
    struct Values {
        float lo[2], hi[2], x[NT][2];
    };
    __device__ __forceinline__ void fetch(Values& v, int k, int n_tiles) const {
        const int block = k / 128;
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            v.lo[m] = __ldg(lo[m] + block * row_block);
            v.hi[m] = __ldg(hi[m] + block * row_block);
        }
        if (X8) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
                if (n < n_tiles) {
                    v.x[n][0] = __ldg(x[n][0] + block * x_block);
                    v.x[n][1] = __ldg(x[n][1] + block * x_block);
                }
        }
    }
};

// A consumer warp's part of one piece: its share of the sums over k_total.  All consumers wait for the same stages; one whose wait
// runs out goes on with what is there (every warp then meets the same barriers), and the status word tells.
template <bool W8, bool X8, int NT>
__device__ __forceinline__ void consume(Ring& ring, const uint8_t* stages, volatile int* abort_flag, uint32_t* status, int k_total, int m_tiles,
                                        int n_tiles, const Scales<W8, X8, NT>& scales, int warp, int lane, float (&acc)[2][NT][4]) {
    typedef Form<W8, X8> F;
    uint32_t nan[2][2] = {{0, 0}, {0, 0}};
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[m][n][i] = 0.0f;
    const int mine = warp * F::kSlices * 32;   // this warp's first k of a chunk; its slices lie in one block of 128
    typename Scales<W8, X8, NT>::Values now, next;
    if (W8) scales.fetch(now, min(mine, k_total - 1), n_tiles);
    for (int k0 = 0; k0 < k_total; k0 += F::kChunk) {
        if (W8 && k0 + F::kChunk < k_total) scales.fetch(next, min(k0 + F::kChunk + mine, k_total - 1), n_tiles);
        mbar_wait(ring.full + 8 * ring.stage, ring.phase, abort_flag, status);
        const uint8_t* stage = stages + ring.stage * ring.stage_bytes;
        const int len = min(F::kChunk, k_total - k0);
        if (W8) {
            float part[2][NT][4];
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) part[m][n][i] = 0.0f;
            multiply<W8, X8, NT>(stage, len, m_tiles, n_tiles, warp, lane, part, nan);
            if (mine < len) {
#pragma unroll
                for (int m = 0; m < 2; ++m)
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        const float x0 = X8 ? now.x[n][0] : 1.0f, x1 = X8 ? now.x[n][1] : 1.0f;
                        if (m < m_tiles && n < n_tiles) {
                            acc[m][n][0] = fmaf(part[m][n][0], X8 ? now.lo[m] * x0 : now.lo[m], acc[m][n][0]);
                            acc[m][n][1] = fmaf(part[m][n][1], X8 ? now.lo[m] * x1 : now.lo[m], acc[m][n][1]);
                            acc[m][n][2] = fmaf(part[m][n][2], X8 ? now.hi[m] * x0 : now.hi[m], acc[m][n][2]);
                            acc[m][n][3] = fmaf(part[m][n][3], X8 ? now.hi[m] * x1 : now.hi[m], acc[m][n][3]);
                        }
                    }
            }
            now = next;
        } else {
            multiply<W8, X8, NT>(stage, len, m_tiles, n_tiles, warp, lane, acc, nan);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(ring.empty + 8 * ring.stage);
        ring.advance();
    }
    if (W8 && !X8) {   // a NaN code makes its row NaN for every token; the lane that met it is one of four that hold the row
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t f = nan[m][h];
                f |= __shfl_xor_sync(0xffffffffu, f, 1);
                f |= __shfl_xor_sync(0xffffffffu, f, 2);
                if (f != 0)
#pragma unroll
                    for (int n = 0; n < NT; ++n) acc[m][n][2 * h] = acc[m][n][2 * h + 1] = __uint_as_float(0x7FC00000u);
            }
    }
}

// A warp's sums of a piece -> shared memory [warp][m][n][4][32]; sum_of reads the value of (row, token) from all eight.
template <int NT>
constexpr int scratch_floats() { return kConsumers * 2 * NT * 128; }

template <int NT>
__device__ __forceinline__ void store_sums(float* scratch, const float (&acc)[2][NT][4], int m_tiles, int n_tiles, int warp, int lane) {
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n)
            if (m < m_tiles && n < n_tiles)
#pragma unroll
                for (int r = 0; r < 4; ++r) scratch[((warp * 2 + m) * NT + n) * 128 + r * 32 + lane] = acc[m][n][r];
}
template <int NT>
__device__ __forceinline__ float sum_of(const float* scratch, int row, int token) {
    const float* at = scratch + ((row >> 4) * NT + (token >> 3)) * 128 + (((row >> 3) & 1) * 2 + (token & 1)) * 32 + (row & 7) * 4 + ((token & 7) >> 1);
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < kConsumers; ++w) s += at[w * 2 * NT * 128];
    return s;
}

}  // namespace stream
}  // namespace mok
