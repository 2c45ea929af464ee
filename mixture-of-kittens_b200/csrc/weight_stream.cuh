// Products of weight rows with a few tokens, for kernels that are bound by reading the weights once: out[row, token] = sum over k
// of W[row, k] * x[token, k].
//
// A block has four producer warps and eight consumer warps around a ring of stages.  A stage is a chunk of a piece: 16 weight rows
// and the rows of the tokens concerned, kChunk elements of k.  One producer warp fills it with cp.async (32 x 16 bytes lie in one
// row: any row count, stride and gather), one consumer warp multiplies it with mma.sync (weights on the M side, tokens on the N
// side of 8); chunks go round the producers and round the consumers in turn.  A last warp, the finisher, adds up the chunks' sums of
// a piece and does with them what the kernel is for, while the consumers are at the next piece.  Producers run ahead as far as the
// ring reaches: about 64 KB of weights in flight per block is what HBM needs.  tcgen05 would need 128 rows a tile, which leaves SMs
// idle at these sizes; the tensor work here is a few percent of the time.
//
// The barriers of a stage tell rounds apart by one bit, so nobody may be two rounds ahead of a barrier: the number of stages is a
// multiple of eight, so that a stage has one producer and one consumer, which have seen every round of it.
//
// What did not do: bulk copies, one per row (an SM issues one in about 60 clocks: 1.4 - 1.8 TB/s with rows of 512 bytes, 2.2 - 3.4
// with 1024); every consumer taking an eighth of every chunk (all eight pay the waits and addresses of each chunk, 350 instructions
// a warp for 21 KB of weights: 2.1 - 3.7 TB/s with experts of 768 rows); the last consumer of a piece as its finisher (178 instead of
// 147 us for the blocks whose experts have five tokens or more).
//
// The order of k within a slice of 32 is free as long as both operands use the same one: lane (g, t) of an mma takes elements 8 t ..
// 8 t + 7 of rows g and g + 8, one 16-byte (8-byte in e4m3) shared-memory load per row, for two mma of K = 16.  Row pitches of 64
// (32) bytes modulo 128 make these loads free of bank conflicts.
#pragma once

#include <cuda_fp16.h>

#include "mok_common.cuh"

namespace mok {
namespace stream {

constexpr int kConsumers = 8;                       // warps
constexpr int kConsumerThreads = kConsumers * 32;
constexpr int kProducers = 4;
constexpr int kFinisher = kConsumers + kProducers;  // warp
constexpr int kThreads = kConsumerThreads + kProducers * 32 + 32;
constexpr int kRows = 16;                           // weight rows of a piece
constexpr int kMaxStages = 16;
constexpr int kDeposits = 2;

// W8: weights in e4m3 instead of bf16, and tokens in f16 (every code is an f16 number, one conversion per pair; as bf16 it takes
// five operations a pair, all on the pipes of 64 lanes a clock, and 22 experts of 44 MB took 384 us instead of 351), or, X8, in
// e4m3 too.
template <bool W8, bool X8>
struct Form {
    static constexpr int kChunk = W8 ? 512 : 256;               // elements of k per stage
    static constexpr int kRowBytes = kChunk * (W8 ? 1 : 2);     // 512: one copy of 16 bytes per lane
    static constexpr int kRowPitch = kRowBytes + (W8 ? 32 : 64);
    static constexpr int kTokenBytes = kChunk * (X8 ? 1 : 2);
    static constexpr int kTokenPitch = kTokenBytes + (X8 ? 32 : 64);
    static constexpr int kBlocks = kChunk / 128;
    static constexpr int kScales = W8 ? 4 * kBlocks * kRows : 0;   // bytes; one per row and 128 of k, then X8 one per token
    // weight rows, their scales, token rows, their scales
    static constexpr int stage_bytes(int tokens) { return kRows * kRowPitch + kScales + tokens * (kTokenPitch + (X8 ? 4 * kBlocks : 0)); }
    static constexpr int kTokens = kRows * kRowPitch + kScales;
    __device__ static __forceinline__ int chunks(int k_total) { return (k_total + kChunk - 1) / kChunk; }
};

// One arrival once every copy that this thread has issued so far is done.
__device__ __forceinline__ void arrive_when_copied(uint32_t bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void wait_copies() { asm volatile("cp.async.wait_all;" ::: "memory"); }
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void consumer_barrier() { asm volatile("bar.sync 1, %0;" ::"n"(kConsumerThreads) : "memory"); }
struct Bars {
    uint64_t full[kMaxStages], empty[kMaxStages], routed;
    int count[kDeposits], done[kDeposits];   // deposits so far, pieces that were finished
    int abort_flag;
};

// The ring, and the place of a piece in the sequence of chunks that producers and consumers walk alike: its chunk 0 lies in stage
// `at` of round `round`.
struct Ring {
    uint32_t base, full, empty;   // shared addresses: stages, barriers
    int stage_bytes, stages;
    int at = 0, round = 0;
    __device__ __forceinline__ void next_piece(int chunks) {
        at += chunks;
        while (at >= stages) {
            at -= stages;
            ++round;
        }
    }
    // Stage and parity of chunk c.
    __device__ __forceinline__ int stage(int c, uint32_t& parity) const {
        int s = at + c, r = round;
        while (s >= stages) {
            s -= stages;
            ++r;
        }
        parity = r & 1;
        return s;
    }
};

__device__ __forceinline__ Ring set_up_ring(Bars& bars, const uint8_t* smem, int stage_bytes, int stages, int routed_arrivals) {
    Ring r;
    r.base = smem_u32(smem);
    r.full = smem_u32(bars.full);
    r.empty = smem_u32(bars.empty);
    r.stage_bytes = stage_bytes;
    r.stages = stages;
    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) {
            mbar_init(r.full + 8 * s, 32);
            mbar_init(r.empty + 8 * s, 1);
        }
        for (int d = 0; d < kDeposits; ++d) {
            bars.count[d] = bars.done[d] = 0;
        }
        mbar_init(smem_u32(&bars.routed), routed_arrivals);
        bars.abort_flag = 0;
        mbar_fence_init();
    }
    __syncthreads();
    return r;
}

// ---- producer -----------------------------------------------------------------------------------------------------
// Rows of a piece as a producer copies them.  Weights: rows 0 .. 7 from low and rows 8 .. 15 from high (this lane's 16 bytes at k = 0),
// row_bytes apart, `rows_low` and `rows_high` of them (the others stay as they are and are not used).  Tokens: lane j holds the address
// of row j.  Found once per piece: with addresses worked out chunk by chunk the producers were the bottleneck (1500 clocks a chunk,
// 2.2 TB/s), and with every lane holding all token addresses they were at 24 tokens.
struct Feed {
    const uint8_t *low, *high, *token;
    long long row_bytes;
    int rows_low, rows_high, tokens;
    // scales of this lane's row (lanes 0 .. 15; nullptr: none) and token, and the distance between blocks of k
    const float *scale, *token_scale;
    long long scale_stride, token_scale_stride;
};
// Consumers that fetched the scales themselves waited for them, some 600 clocks in every block of 128.
template <typename F, bool X8>
__device__ __forceinline__ void copy_scales(uint32_t stage, const Feed& f, int k0, int len, int token_cap, int lane) {
    const int block0 = k0 / 128, blocks = (len + 127) / 128;
#pragma unroll
    for (int b = 0; b < F::kBlocks; ++b) {
        if (b >= blocks) break;
        if (f.scale != nullptr) copy4(stage + kRows * F::kRowPitch + (lane * F::kBlocks + b) * 4, f.scale + (block0 + b) * f.scale_stride);
        if (X8 && f.token_scale != nullptr)
            copy4(stage + F::kTokens + token_cap * F::kTokenPitch + (lane * F::kBlocks + b) * 4, f.token_scale + (block0 + b) * f.token_scale_stride);
    }
}
template <typename F>
__device__ __forceinline__ void copy_weights(uint32_t stage, const Feed& f, int k0, int len, int lane) {
    constexpr int kBytes = F::kRowBytes / F::kChunk;
    static_assert(F::kRowBytes == 512, "");
    if (lane * 16 >= len * kBytes) return;
    const long long at = static_cast<long long>(k0) * kBytes;
    const uint8_t *low = f.low + at, *high = f.high + at;
    const uint32_t dst = stage + lane * 16;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if (i < f.rows_low) copy16(dst + i * F::kRowPitch, low);
        if (i < f.rows_high) copy16(dst + (8 + i) * F::kRowPitch, high);
        low += f.row_bytes;
        high += f.row_bytes;
    }
}
template <typename F>
__device__ __forceinline__ void copy_tokens(uint32_t stage, const Feed& f, int k0, int len, int lane) {
    constexpr int kBytes = F::kTokenBytes / F::kChunk;
    const int bytes = len * kBytes;
    uint32_t dst = stage + F::kTokens + lane * 16;
    const unsigned long long mine = reinterpret_cast<unsigned long long>(f.token) + static_cast<long long>(k0) * kBytes;
#pragma unroll 2
    for (int j = 0; j < f.tokens; ++j) {
        const uint8_t* row = reinterpret_cast<const uint8_t*>(__shfl_sync(0xffffffffu, mine, j)) + lane * 16;
#pragma unroll
        for (int part = 0; part < F::kTokenBytes; part += 512)
            if (part + lane * 16 < bytes) copy16(dst + part, row + part);
        dst += F::kTokenPitch;
    }
}
// A producer's chunks of a piece, from chunk `first` on: those whose number in the whole sequence is `producer` modulo kProducers.
// False: a wait ran out.
template <typename F, bool X8>
__device__ __forceinline__ bool produce(const Ring& ring, volatile int* abort_flag, uint32_t* status, const Feed& f, int first, int k_total,
                                        int token_cap, int lane) {
    for (int c = first; c * F::kChunk < k_total; c += kProducers) {
        uint32_t parity;
        const int s = ring.stage(c, parity);
        if (!mbar_wait(ring.empty + 8 * s, parity ^ 1u, abort_flag, status)) return false;
        const int k0 = c * F::kChunk, len = min(F::kChunk, k_total - k0);
        const uint32_t stage = ring.base + s * ring.stage_bytes;
        copy_weights<F>(stage, f, k0, len, lane);
        if (F::kScales) copy_scales<F, X8>(stage, f, k0, len, token_cap, lane);
        copy_tokens<F>(stage, f, k0, len, lane);
        arrive_when_copied(ring.full + 8 * s);
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
// The first `count` (may be <= 0) of eight codes, the others zero.
__device__ __forceinline__ uint2 keep_codes(uint2 v, int count) {
    if (count < 8) v.y = count > 4 ? v.y & (0xFFFFFFFFu >> (8 * (8 - count))) : 0u;
    if (count < 4) v.x = count > 0 ? v.x & (0xFFFFFFFFu >> (8 * (4 - count))) : 0u;
    return v;
}

template <int NT>
__device__ __forceinline__ void clear(float (&acc)[NT][4]) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[n][i] = 0.0f;
}

// acc += 32 elements of k from element `k` of a stage on (of this lane: k + 8 t .. k + 8 t + 7).  `left`: valid elements from k on
// (X8; the others hold multiples of 32).
template <bool W8, bool X8, int TILES, int NT>
__device__ __forceinline__ void multiply_slice(const uint8_t* weights, const uint8_t* tokens, int k, int left, int t, float (&acc)[NT][4]) {
    typedef Form<W8, X8> F;
    uint32_t lo[4], hi[4];
    if (W8) {
        uint2 l = *reinterpret_cast<const uint2*>(weights + k);
        uint2 h = *reinterpret_cast<const uint2*>(weights + 8 * F::kRowPitch + k);
        if (X8 && left < 32) {
            l = keep_codes(l, left - 8 * t);
            h = keep_codes(h, left - 8 * t);
        }
        lo[0] = e4m3x2_to_f16x2(l.x); lo[1] = e4m3x2_to_f16x2(l.x >> 16); lo[2] = e4m3x2_to_f16x2(l.y); lo[3] = e4m3x2_to_f16x2(l.y >> 16);
        hi[0] = e4m3x2_to_f16x2(h.x); hi[1] = e4m3x2_to_f16x2(h.x >> 16); hi[2] = e4m3x2_to_f16x2(h.y); hi[3] = e4m3x2_to_f16x2(h.y >> 16);
    } else {
        const uint4 l = *reinterpret_cast<const uint4*>(weights + k * 2);
        const uint4 h = *reinterpret_cast<const uint4*>(weights + 8 * F::kRowPitch + k * 2);
        lo[0] = l.x; lo[1] = l.y; lo[2] = l.z; lo[3] = l.w;
        hi[0] = h.x; hi[1] = h.y; hi[2] = h.z; hi[3] = h.w;
    }
#pragma unroll
    for (int n = 0; n < TILES; ++n) {
        uint32_t b[4];
        if (X8) {
            uint2 v = *reinterpret_cast<const uint2*>(tokens + n * 8 * F::kTokenPitch + k);
            if (left < 32) v = keep_codes(v, left - 8 * t);
            b[0] = e4m3x2_to_f16x2(v.x); b[1] = e4m3x2_to_f16x2(v.x >> 16); b[2] = e4m3x2_to_f16x2(v.y); b[3] = e4m3x2_to_f16x2(v.y >> 16);
            mma_f16(acc[n], lo[0], hi[0], lo[1], hi[1], b[0], b[1]);
            mma_f16(acc[n], lo[2], hi[2], lo[3], hi[3], b[2], b[3]);
        } else {
            const uint4 v = *reinterpret_cast<const uint4*>(tokens + n * 8 * F::kTokenPitch + k * 2);
            if (W8) {
                mma_f16(acc[n], lo[0], hi[0], lo[1], hi[1], v.x, v.y);
                mma_f16(acc[n], lo[2], hi[2], lo[3], hi[3], v.z, v.w);
            } else {
                mma_bf16(acc[n], lo[0], hi[0], lo[1], hi[1], v.x, v.y);
                mma_bf16(acc[n], lo[2], hi[2], lo[3], hi[3], v.z, v.w);
            }
        }
    }
}

// acc += a chunk, block of 128 by block.  Whole blocks are one run of code for a number of n tiles known to the compiler: with a
// condition on it in every slice nothing overlapped, 200 clocks a slice.
template <bool W8, bool X8, int TILES, int NT>
__device__ __forceinline__ void multiply_chunk(const uint8_t* weights, const uint8_t* tokens, const float* scales, const float* token_scales, int len,
                                               int t, float (&acc)[NT][4]) {
    typedef Form<W8, X8> F;
#pragma unroll 1
    for (int b = 0; b * 128 < len; ++b) {
        float part[NT][4];
        float(&to)[NT][4] = W8 ? part : acc;
        if (W8) clear(part);
        const int left = len - b * 128, k0 = b * 128 + 8 * t;
        if (left >= 128) {
#pragma unroll
            for (int k = 0; k < 128; k += 32) multiply_slice<W8, X8, TILES, NT>(weights, tokens, k0 + k, 32, t, to);
        } else {
#pragma unroll 1
            for (int k = 0; k < left; k += 32) multiply_slice<W8, X8, TILES, NT>(weights, tokens, k0 + k, left - k, t, to);
        }
        if (W8) {
            const float lo = scales[b], hi = scales[8 * F::kBlocks + b];
#pragma unroll
            for (int n = 0; n < TILES; ++n) {
                const float x0 = X8 ? token_scales[n * 8 * F::kBlocks + b] : 1.0f, x1 = X8 ? token_scales[(n * 8 + 1) * F::kBlocks + b] : 1.0f;
                acc[n][0] = fmaf(part[n][0], X8 ? lo * x0 : lo, acc[n][0]);
                acc[n][1] = fmaf(part[n][1], X8 ? lo * x1 : lo, acc[n][1]);
                acc[n][2] = fmaf(part[n][2], X8 ? hi * x0 : hi, acc[n][2]);
                acc[n][3] = fmaf(part[n][3], X8 ? hi * x1 : hi, acc[n][3]);
            }
        }
    }
}

// Waits for a chunk and adds its products to acc.  A wait that runs out is reported in the status word and the warp goes on with what
// is there, so that every warp still meets the same barriers.
template <bool W8, bool X8, int NT>
__device__ __forceinline__ void consume(const Ring& ring, const uint8_t* stages, volatile int* abort_flag, uint32_t* status, int c, int k_total, int tiles,
                                        int token_cap, int lane, float (&acc)[NT][4]) {
    typedef Form<W8, X8> F;
    const int g = lane >> 2, t = lane & 3;
    const int len = min(F::kChunk, k_total - c * F::kChunk);
    uint32_t parity;
    const int s = ring.stage(c, parity);
    mbar_wait(ring.full + 8 * s, parity, abort_flag, status);
    const uint8_t* stage = stages + s * ring.stage_bytes;
    const uint8_t* weights = stage + g * F::kRowPitch;
    const uint8_t* tokens = stage + F::kTokens + g * F::kTokenPitch;
    const float* scales = reinterpret_cast<const float*>(stage + kRows * F::kRowPitch) + g * F::kBlocks;
    const float* token_scales = reinterpret_cast<const float*>(stage + F::kTokens + token_cap * F::kTokenPitch) + 2 * t * F::kBlocks;
    if (NT == 1 || tiles == 1) multiply_chunk<W8, X8, 1, NT>(weights, tokens, scales, token_scales, len, t, acc);
    else if (NT == 2 || tiles == 2) multiply_chunk<W8, X8, NT < 2 ? NT : 2, NT>(weights, tokens, scales, token_scales, len, t, acc);
    else if (NT == 3 || tiles == 3) multiply_chunk<W8, X8, NT < 3 ? NT : 3, NT>(weights, tokens, scales, token_scales, len, t, acc);
    else multiply_chunk<W8, X8, NT, NT>(weights, tokens, scales, token_scales, len, t, acc);
    __syncwarp();
    if (lane == 0) mbar_arrive(ring.empty + 8 * s);
}

// ---- sums of a piece over the consumers -----------------------------------------------------------------------------
// Chunk c's sums go to slot c % 8 (whichever warp computed them), so the order of the final addition is that of k.  Two deposits in
// turn: consumers are at most two pieces ahead of the finisher.
template <int NT>
constexpr int deposit_floats() { return kDeposits * kConsumers * NT * 128; }

struct Deposit {
    float* scratch;
    int piece = 0;                     // pieces so far
    int expected0 = 0, expected1 = 0;  // finisher: deposits that make the pieces so far complete, of either
};
// Waits, with the limit of all pipeline waits, until a counter in shared memory has reached a value.  Not a barrier of one bit: a
// warp may have no part in many pieces and be far ahead.
__device__ __forceinline__ void wait_count(int* counter, int value, Bars& bars, uint32_t* status) {
    const long long start = clock64();
    while (*static_cast<volatile int*>(counter) < value && !*static_cast<volatile int*>(&bars.abort_flag)) {
        if (clock64() - start > kPipelineWaitCycles) {
            *static_cast<volatile int*>(&bars.abort_flag) = 1;
            if (status != nullptr) atomicOr(status, (uint32_t)MOK_STATUS_PIPELINE_TIMEOUT);
        }
    }
    __threadfence_block();
    __syncwarp();
}
template <int NT>
__device__ __forceinline__ void deposit(const Deposit& d, Bars& bars, uint32_t* status, const float (&acc)[NT][4], int slot, int tiles, int lane) {
    const int which = d.piece & 1;
    wait_count(&bars.done[which], d.piece >> 1, bars, status);
    float* at = d.scratch + (which * kConsumers + slot) * NT * 128 + lane;
#pragma unroll
    for (int n = 0; n < NT; ++n)
        if (n < tiles)
#pragma unroll
            for (int r = 0; r < 4; ++r) at[n * 128 + r * 32] = acc[n][r];
    __threadfence_block();
    __syncwarp();
    if (lane == 0) atomicAdd(&bars.count[which], 1);
}
// The finisher's side: every piece in order, `slots` deposits each.
__device__ __forceinline__ void collect(Deposit& d, Bars& bars, uint32_t* status, int slots) {
    const int which = d.piece & 1;
    (which ? d.expected1 : d.expected0) += slots;
    wait_count(&bars.count[which], which ? d.expected1 : d.expected0, bars, status);
}
__device__ __forceinline__ void collected(Deposit& d, Bars& bars, int lane) {
    __threadfence_block();
    __syncwarp();
    if (lane == 0) *static_cast<volatile int*>(&bars.done[d.piece & 1]) = (d.piece >> 1) + 1;
    ++d.piece;
}
template <int NT>
__device__ __forceinline__ float sum_of(const Deposit& d, int slots, int row, int token) {
    const float* at = d.scratch + ((d.piece & 1) * kConsumers * NT + (token >> 3)) * 128 + ((row >> 3) * 2 + (token & 1)) * 32 + (row & 7) * 4 + ((token & 7) >> 1);
    float v[kConsumers], s = 0.0f;
#pragma unroll
    for (int w = 0; w < kConsumers; ++w) v[w] = w < slots ? at[w * NT * 128] : 0.0f;
#pragma unroll
    for (int w = 0; w < kConsumers; ++w) s += v[w];
    return s;
}

}  // namespace stream
}  // namespace mok
