// Product of two matrices held in e4m3 with fp32 scales per block of 128:
//   D[m, n] = sum over blocks kb of sa[m, kb] * sb[n or n / 128, kb] * (sum over k in kb of a[m, k] * b[n, k]),  D in bf16.
//
// The scales are fp32 numbers of any value, so the tensor cores cannot apply them: every block of 128 along K is accumulated on
// its own in tensor memory (four tcgen05.mma of K = 32, kind::f8f6f4) and added, scaled, to fp32 registers.  CTA pairs own 256 x
// 256 tiles, each CTA stages 128 rows of A and 128 of B per block by TMA (32 KB, 4 stages); two 256-column accumulators, each with
// a thread that issues its MMAs, let the MMAs of one block run while eight epilogue warps scale the block before (a warp: 32 rows x
// 128 columns, 128 registers of sums).  Rows, columns and depth that are not multiples of the tile are zeros from TMA and are not
// stored.
//
// Bound by that scaling: about 950 clocks a block where the MMAs alone take 512, and 2300 more a tile for packing and storing.  8192 x
// 7168 x 7168 388 us (2.2 PFLOP/s), 8192 x 7168 x 2048 141 us (1.7), with a scale per column of B 4096 x 2048 x 4096 79 us.
//
// Few tiles (a short grid and a long K): the blocks along K are cut into `splits` shares, every share writes its fp32 sums, and
// a second kernel adds them in order.
#include "block_matmul.cuh"
#include "block_scale.cuh"
#include "gemm_tiles.cuh"
#include "ring_turn.cuh"

namespace mok {
namespace {

using namespace tiles;

constexpr int BK = 128;
constexpr int kStages = 4;
constexpr int kThreads = 384;                 // one warpgroup with the TMA producer and the MMA issuers, two of the epilogue
// Registers of the warpgroups: 384 threads start with 168 each; 128 * 40 + 256 * 232 = 384 * 168.
constexpr int kIssueRegisters = 40;
constexpr int kEpilogueRegisters = 232;
constexpr int kOperandBytes = 128 * BK;       // 16 KB
constexpr int kStageBytes = 2 * kOperandBytes;
constexpr int kGroup = 8;                     // m tiles that walk the columns together
constexpr int kBoxBytes = 32 * 128;           // output of an epilogue warp: two boxes of 32 rows x 64 columns

struct Layout {
    static constexpr int kPatch = kStages * kStageBytes;              // [8 warps][2 boxes]; 1024-byte aligned
    static constexpr int kScales = kPatch + 8 * 2 * kBoxBytes;        // [8 warps][2][128] fp32: column scales of a block
    static constexpr int kFull = kScales + 8 * 2 * 128 * 4;
    static constexpr int kEmpty = kFull + 8 * kStages;
    static constexpr int kAccEmpty = kEmpty + 8 * kStages;
    static constexpr int kTmemPtr = kAccEmpty + 16;
    static constexpr int kAbort = kTmemPtr + 4;
    static constexpr int kBytes = kAbort + 4;
};
static_assert(kEpiWarpBytes <= 2 * kBoxBytes, "the patch of outputs that TMA cannot address");
static_assert(Layout::kBytes + 1024 <= kMaxDynamicSmem, "shared memory");

struct Product {
    const float *sa, *sb;
    long long sa_row, sa_block, sb_row, sb_block;
    bf16* out;
    float* partial;          // [splits, rows, cols] when splits > 1
    long long out_stride;
    int rows, cols, k_blocks;
    int m_tiles, n_tiles, splits;
    int box_out;             // rows of out are 16-byte aligned: boxes leave by TMA
    uint32_t* status;
};

// Instruction descriptor for kind::f8f6f4, e4m3 x e4m3 -> fp32, both operands K-major: D format (1 = fp32) at 4, A / B formats
// (0 = e4m3) at 7 / 10, N >> 3 at 17, M >> 4 at 24.
__host__ __device__ constexpr uint32_t idesc_e4m3(int m, int n) {
    return (1u << 4) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}
__device__ __forceinline__ void umma_e4m3_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// A box of shared memory to the output, rows and columns beyond its end left out.
__device__ __forceinline__ void store_box(const CUtensorMap* map, uint32_t src, int col, int row) {
    asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4, %4}], [%1];"
                 ::"l"(reinterpret_cast<uint64_t>(map)), "r"(src), "r"(col), "r"(row), "r"(0)
                 : "memory");
}
// A value that a tensor-memory load brought: its use stays behind the wait for that load.
__device__ __forceinline__ float ordered(uint32_t v) {
    float f;
    asm volatile("mov.b32 %0, %1;" : "=f"(f) : "r"(v));
    return f;
}
// mbar_wait that polls instead of suspending the thread: the accumulators change hands once per block of K.
__device__ __forceinline__ bool mbar_poll(uint32_t bar, uint32_t parity, volatile int* abort_flag, uint32_t* status) {
    long long start = 0;
    for (uint32_t spin = 0;; ++spin) {
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok)
            : "r"(bar), "r"(parity)
            : "memory");
        if (ok) return true;
        if ((spin & 0x3FF) == 0x3FF) {
            if (*abort_flag) return false;
            if (start == 0) start = clock64();
            if (clock64() - start > kPipelineWaitCycles) {
                *abort_flag = 1;
                if (status != nullptr) atomicOr(status, (uint32_t)MOK_STATUS_PIPELINE_TIMEOUT);
                return false;
            }
        }
    }
}

// Arrival at the leader CTA's barrier that orders nothing but the tensor-memory loads before it (they are complete and fenced).  The
// usual release at cluster scope also waits for the scales on their way from L2: 8192 x 7168 x 7168 took 926 us instead of 524 then.
__device__ __forceinline__ void arrive_leader_relaxed(uint32_t bar) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar & kPairLeaderMask) : "memory");
}

struct Work {
    int m0, n0, split, kb0, kb1;
};
// Tile t: groups of kGroup m tiles walk the columns together (their A panels stay in L2), the shares of K innermost.
__device__ __forceinline__ Work decode(const Product& p, uint32_t t) {
    Work w;
    w.split = 0;
    w.kb0 = 0;
    w.kb1 = p.k_blocks;
    if (p.splits > 1) {   // k_blocks * splits < 2^31
        w.split = t % p.splits;
        t /= p.splits;
        w.kb0 = p.k_blocks * w.split / p.splits;
        w.kb1 = p.k_blocks * (w.split + 1) / p.splits;
    }
    const uint32_t per_group = kGroup * p.n_tiles;
    const uint32_t g = t / per_group, rem = t - g * per_group;
    const uint32_t width = min(kGroup, p.m_tiles - static_cast<int>(g) * kGroup);
    const uint32_t n = width == kGroup ? rem / kGroup : rem / width;
    w.m0 = (g * kGroup + rem - n * width) * BM;
    w.n0 = n * BN;
    return w;
}

// COLUMN_SCALES: sb holds one scale per column instead of one per 128.
template <bool COLUMN_SCALES>
__global__ void __launch_bounds__(kThreads, 1)
block_matmul_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_out,
                    const Product p) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
    const uint32_t bar_full = base + Layout::kFull, bar_empty = base + Layout::kEmpty;
    const uint32_t bar_acc_empty = base + Layout::kAccEmpty;
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(gen + Layout::kTmemPtr);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(gen + Layout::kAbort);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int cta = static_cast<int>(cluster_cta_rank());
    const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    const int tiles = p.m_tiles * p.n_tiles * p.splits;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(bar_full + 8 * s, 1);
            mbar_init(bar_empty + 8 * s, 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(bar_acc_empty + 8 * b, 16);   // eight epilogue warps of both CTAs
        }
        *abort_flag = 0;
        mbar_fence_init();
        tma_prefetch_desc(&map_a);
        tma_prefetch_desc(&map_b);
    }
    if (warp == 1) {
        tmem_alloc_pair(smem_u32(const_cast<uint32_t*>(tmem_slot)), TMEM_COLS);
        tmem_relinquish_pair();
    }
    tc_fence_before_sync();
    __syncthreads();
    cluster_sync_all();
    tc_fence_after_sync();
    const uint32_t tmem = *tmem_slot;
    allow_next_kernel();   // the kernel that adds the shares, if there is one, waits for this one

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kIssueRegisters));
        if (warp == 0) {
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int t = pair; t < tiles && ok; t += pairs) {
                const Work w = decode(p, t);
                for (int kb = w.kb0; kb < w.kb1; ++kb) {
                    ok = mbar_wait(bar_empty + 8 * stage, phase ^ 1u, abort_flag, p.status);
                    if (!ok) break;
                    if (lane == 0) {
                        const uint32_t full = bar_full + 8 * stage, dst = base + stage * kStageBytes;
                        if (cta == 0) mbar_expect_tx(full, 2 * kStageBytes);
                        tma_load_4d_pair(dst, &map_a, full & kPairLeaderMask, kb * BK, w.m0 + cta * BM_CTA, 0, 0);
                        tma_load_4d_pair(dst + kOperandBytes, &map_b, full & kPairLeaderMask, kb * BK, w.n0 + cta * BN_CTA, 0, 0);
                    }
                    __syncwarp();
                    if (++stage == kStages) { stage = 0; phase ^= 1u; }
                }
            }
        } else if (warp <= 2) {
            // Two issuers take the blocks in turn, one accumulator each: what one waits for (400 clocks a block, beside 560 in which it
            // hands over MMAs) is hidden behind the other's MMAs.  8192 x 7168 x 7168 444 -> 411 us.
            if (cta == 0 && lane == 0) {
                uint32_t blocks = 0;
                for (int t = pair; t < tiles; t += pairs) {
                    const Work w = decode(p, t);
                    blocks += w.kb1 - w.kb0;
                }
                const uint32_t buf = warp - 1;
                for (uint32_t block = buf; block < blocks; block += 2) {
                    const uint32_t stage = block % kStages, phase = (block / kStages) & 1u;
                    if (!mbar_poll(bar_full + 8 * stage, phase, abort_flag, p.status) ||
                        !mbar_poll(bar_acc_empty + 8 * buf, ((block >> 1) & 1u) ^ 1u, abort_flag, p.status))
                        break;
                    tc_fence_after_sync();
                    const uint32_t a = base + stage * kStageBytes;
                    const uint64_t a_desc = umma_smem_desc(a, 16, 1024), b_desc = umma_smem_desc(a + kOperandBytes, 16, 1024);
#pragma unroll
                    for (int k = 0; k < BK / 32; ++k)
                        umma_e4m3_pair(tmem + buf * BN, a_desc + k * 2u, b_desc + k * 2u, idesc_e4m3(BM, BN), k != 0 ? 1u : 0u);
                    umma_commit_pair(bar_empty + 8 * stage);
                }
            }
            __syncwarp();
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kEpilogueRegisters));
        const int quarter = warp & 3, half = (warp - 4) >> 2;
        float* col_scales = reinterpret_cast<float*>(gen + Layout::kScales) + (warp - 4) * 256;
        uint8_t* patch = gen + Layout::kPatch + (warp - 4) * 2 * kBoxBytes;
        const uint32_t accumulators = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + half * 128;
        // Scales of the next block, on their way.  COLUMN_SCALES: the lane fetches columns lane, lane + 32, ... of the warp's 128;
        // otherwise there is one for all of them.
        constexpr int kColumns = COLUMN_SCALES ? 4 : 1;
        const float *a_at = p.sa, *b_at[kColumns];
        float next_a, next_b[kColumns];
        auto load_scales = [&] {
            next_a = *a_at;
            a_at += p.sa_block;
#pragma unroll
            for (int j = 0; j < kColumns; ++j) {
                next_b[j] = *b_at[j];
                b_at[j] += p.sb_block;
            }
        };
        auto first_scales = [&](const Work& q) {
            a_at = p.sa + static_cast<long long>(min(q.m0 + cta * BM_CTA + quarter * 32 + lane, p.rows - 1)) * p.sa_row + q.kb0 * p.sa_block;
            const int col0 = q.n0 + half * 128;
#pragma unroll
            for (int j = 0; j < kColumns; ++j)
                b_at[j] = p.sb + static_cast<long long>(COLUMN_SCALES ? min(col0 + 32 * j + lane, p.cols - 1) : min(col0, p.cols - 1) / 128) * p.sb_row +
                          q.kb0 * p.sb_block;
            load_scales();
        };
        uint32_t block = 0;
        RingTurn<kStages> turn;
        Work w = decode(p, min(pair, tiles - 1));
        first_scales(w);
        for (int t = pair; t < tiles; t += pairs) {
            const int row0 = w.m0 + cta * BM_CTA + quarter * 32, row = row0 + lane;
            const int col0 = w.n0 + half * 128, split = w.split;
            float acc[128];
#pragma unroll
            for (int i = 0; i < 128; ++i) acc[i] = 0.0f;
            // 32 columns at a time, in single fp32 operations: with pairs of them (fma.rn.f32x2) three quarters of the columns took 610
            // clocks instead of 280.  Loads run while the columns before are added; the accumulator goes back to the MMAs when its last
            // columns are read.
            uint32_t v[2][32];
            for (int left = w.kb1 - w.kb0; left > 0; --left, ++block) {
                const uint32_t buf = block & 1u, taddr = accumulators + buf * BN;
                float scale = next_a;
                const float* cols = col_scales + buf * 128;
                if (COLUMN_SCALES) {
#pragma unroll
                    for (int j = 0; j < kColumns; ++j) col_scales[buf * 128 + 32 * j + lane] = next_b[j];
                    __syncwarp();   // two buffers: this one was read before the previous block's barrier
                } else {
                    scale *= next_b[0];
                }
                if (left > 1) load_scales();
                // the MMAs that read a stage are its block's
                if (!turn.next([&](uint32_t stage, uint32_t phase) { return mbar_poll(bar_empty + 8 * stage, phase, abort_flag, p.status); }))
                    break;
                tc_fence_after_sync();
                tmem_ld_32x32(taddr, v[0]);
                tmem_ld_32x32(taddr + 32, v[1]);
                tmem_ld_wait();
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    if (q == 2) {
                        tmem_ld_wait();
                        tc_fence_before_sync();
                        __syncwarp();
                        if (lane == 0) arrive_leader_relaxed(bar_acc_empty + 8 * buf);
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        float4 f = make_float4(scale, scale, scale, scale);
                        if (COLUMN_SCALES) {
                            const float4 cs = *reinterpret_cast<const float4*>(cols + q * 32 + 4 * i);
                            f.x *= cs.x; f.y *= cs.y; f.z *= cs.z; f.w *= cs.w;
                        }
                        acc[q * 32 + 4 * i] = fmaf(ordered(v[q & 1][4 * i]), f.x, acc[q * 32 + 4 * i]);
                        acc[q * 32 + 4 * i + 1] = fmaf(ordered(v[q & 1][4 * i + 1]), f.y, acc[q * 32 + 4 * i + 1]);
                        acc[q * 32 + 4 * i + 2] = fmaf(ordered(v[q & 1][4 * i + 2]), f.z, acc[q * 32 + 4 * i + 2]);
                        acc[q * 32 + 4 * i + 3] = fmaf(ordered(v[q & 1][4 * i + 3]), f.w, acc[q * 32 + 4 * i + 3]);
                    }
                    if (q < 2) tmem_ld_32x32(taddr + 64 + 32 * q, v[q]);
                }
            }
            if (t + pairs < tiles) {   // the next tile's scales arrive while this one is stored
                w = decode(p, t + pairs);
                first_scales(w);
            }
            if (!turn.ok) {   // a wait ran out (reported in the status word): this tile and the ones that follow are NaN
#pragma unroll
                for (int i = 0; i < 128; ++i) acc[i] = __uint_as_float(0x7FC00000u);
            }
            if (p.splits > 1) {
                // one row per lane, 16 bytes at a time; a line is filled by eight stores of one lane and merges in L2
                if (row < p.rows) {
                    float* out = p.partial + (static_cast<long long>(split) * p.rows + row) * p.cols;
                    const bool whole = (p.cols & 3) == 0;
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        uint32_t f[4];
                        f[0] = __float_as_uint(acc[4 * i]); f[1] = __float_as_uint(acc[4 * i + 1]); f[2] = __float_as_uint(acc[4 * i + 2]); f[3] = __float_as_uint(acc[4 * i + 3]);
                        const int col = col0 + 4 * i;
                        if (whole && col < p.cols) {
                            *reinterpret_cast<uint4*>(out + col) = make_uint4(f[0], f[1], f[2], f[3]);
                        } else {
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                if (col + j < p.cols) out[col + j] = __uint_as_float(f[j]);
                        }
                    }
                }
            } else if (p.box_out) {
                // The boxes leave while the next tile is on its way.
                if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");   // those of the tile before
                __syncwarp();
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    uint32_t f[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) f[j] = __float_as_uint(acc[i * 8 + j]);
                    *reinterpret_cast<uint4*>(patch + (i >> 3) * kBoxBytes + lane * 128 + (((i & 7) ^ (lane & 7)) << 4)) = pack8_bf16(f);
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) {
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        if (row0 < p.rows && col0 + 64 * h < p.cols) store_box(&map_out, smem_u32(patch) + h * kBoxBytes, col0 + 64 * h, row0);
                    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                }
            } else {
                const bool whole = (p.out_stride & 7) == 0 && (reinterpret_cast<uintptr_t>(p.out) & 15) == 0;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint4* mine = reinterpret_cast<uint4*>(patch + lane * kEpiRowPitch);
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        uint32_t f[8];
#pragma unroll
                        for (int j = 0; j < 8; ++j) f[j] = __float_as_uint(acc[h * 64 + i * 8 + j]);
                        mine[i] = pack8_bf16(f);
                    }
                    __syncwarp();
                    const int seg = lane & 7, col = col0 + h * 64 + seg * 8;
#pragma unroll
                    for (int it = 0; it < 8; ++it) {
                        const int r = it * 4 + (lane >> 3);
                        const uint4 q = *reinterpret_cast<const uint4*>(patch + r * kEpiRowPitch + seg * 16);
                        if (row0 + r >= p.rows || col >= p.cols) continue;
                        bf16* dst = p.out + static_cast<long long>(row0 + r) * p.out_stride + col;
                        if (whole && col + 8 <= p.cols) {
                            *reinterpret_cast<uint4*>(dst) = q;
                        } else {
                            const uint32_t word[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                            for (int j = 0; j < 8; ++j)
                                if (col + j < p.cols)
                                    reinterpret_cast<uint16_t*>(dst)[j] = static_cast<uint16_t>(j & 1 ? word[j >> 1] >> 16 : word[j >> 1]);
                        }
                    }
                    __syncwarp();
                }
            }
        }
        if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }

    if (*abort_flag) {
        for (int i = 0; i < 64; ++i) __nanosleep(2000);
    }
    tc_fence_before_sync();
    __syncthreads();
    cluster_sync_all();
    if (warp == 1) {
        tc_fence_after_sync();
        tmem_dealloc_pair(tmem, TMEM_COLS);
    }
}

// out = bf16(sum of the shares, in order).
__global__ void __launch_bounds__(256) sum_shares_kernel(const float* __restrict__ partial, int splits, long long count, int cols,
                                                         bf16* __restrict__ out, long long out_stride) {
    const long long i = (static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x) * 4;
    wait_previous_kernel();
    if (i >= count) return;
    if ((cols & 3) == 0) {
        float4 s = *reinterpret_cast<const float4*>(partial + i);
        for (int k = 1; k < splits; ++k) {
            const float4 v = *reinterpret_cast<const float4*>(partial + k * count + i);
            s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
        }
        const long long row = i / cols;
        bf16* dst = out + row * out_stride + (i - row * cols);
        if ((out_stride & 3) == 0 && (reinterpret_cast<uintptr_t>(out) & 7) == 0) {
            *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16x2(s.x, s.y), pack_bf16x2(s.z, s.w));
        } else {
            dst[0] = __float2bfloat16(s.x); dst[1] = __float2bfloat16(s.y);
            dst[2] = __float2bfloat16(s.z); dst[3] = __float2bfloat16(s.w);
        }
    } else {
        for (int j = 0; j < 4 && i + j < count; ++j) {
            float s = 0.0f;
            for (int k = 0; k < splits; ++k) s += partial[k * count + i + j];
            const long long row = (i + j) / cols;
            out[row * out_stride + (i + j - row * cols)] = __float2bfloat16(s);
        }
    }
}

int code_map(CUtensorMap* map, const void* base, long long stride, long long rows, int depth) {
    const cuuint64_t dims[4] = {static_cast<cuuint64_t>(depth), static_cast<cuuint64_t>(rows), 1, 1};
    const cuuint64_t strides[3] = {static_cast<cuuint64_t>(stride), static_cast<cuuint64_t>(stride * rows),
                                   static_cast<cuuint64_t>(stride * rows)};
    const cuuint32_t box[4] = {BK, 128, 1, 1};
    return encode_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

int div_up(long long a, int b) { return static_cast<int>((a + b - 1) / b); }

// Shares of K: enough to give every CTA pair a tile, each at least four blocks long, where that takes 16 blocks or more (0.4 us each)
// off the longest chain: writing, reading and adding the shares costs 6 us.  1000 x 1544 x 1808 has 28 tiles of 15 blocks and stays
// in one share (18.4 us; two shares took 4 us longer).
int shares(int tiles, int k_blocks) {
    const int pairs = sm_count() / 2;
    int s = pairs / tiles;
    if (s > k_blocks / 4) s = k_blocks / 4;
    return s < 2 || k_blocks - k_blocks / s < 16 ? 1 : s;
}

// Whether the streaming form is the faster one.  Its time grows with the rows, that of a tile does not; streaming against tiles, us:
//   rows                    8         16         24          with a scale per column    8         16         24
//   4096 x 7168     18.4/20.4  22.5/22.5  24.6/20.5                             20.5/24.6  22.5/24.5  24.6/24.6
//   7168 x 2048     14.3/18.4  16.4/18.4  18.4/18.4                             14.3/22.5  16.4/22.5  20.4/22.5
//   7168 x 16384    51.2/43.0  59.4/43.0  67.6/45.1                             51.2/63.5  59.4/61.5  67.6/63.5
bool few_rows(long long rows, int cols, int depth, int b_tile_rows) {
    return rows <= kFewRows && (b_tile_rows == 1 || rows * cols * depth <= 1LL << 29);
}

int plan_splits(long long rows, int cols, int depth) {
    if (few_rows(rows, cols, depth, 128)) return 1;
    return shares(div_up(rows, BM) * div_up(cols, BN), div_up(depth, BK));
}

}  // namespace
}  // namespace mok

extern "C" int64_t mok_block_matmul_scratch_bytes(int64_t rows, int cols, int depth) {
    if (rows <= 0 || rows > 0x7fffffffLL || cols <= 0 || depth <= 0) return 0;
    const int splits = mok::plan_splits(rows, cols, depth);
    return splits > 1 ? static_cast<int64_t>(splits) * rows * cols * 4 : 0;
}

extern "C" int mok_block_matmul(const void* a, int64_t a_stride, const float* a_scales, int64_t a_scale_row_stride,
                                int64_t a_scale_block_stride, const void* b, int64_t b_stride, const float* b_scales,
                                int64_t b_scale_row_stride, int64_t b_scale_block_stride, int b_tile_rows, int64_t rows, int cols,
                                int depth, void* out, int64_t out_stride, void* scratch, uint32_t* status, mok_stream_t stream) {
    using namespace mok;
    if (rows < 0 || cols <= 0 || depth <= 0 || (b_tile_rows != 1 && b_tile_rows != 128)) return MOK_ERR_INVALID_ARGUMENT;
    if (rows > (1 << 24) || cols > (1 << 24)) return MOK_ERR_TOO_LARGE;
    if (rows == 0) return MOK_OK;
    if (!a || !a_scales || !b || !b_scales || !out) return MOK_ERR_INVALID_ARGUMENT;
    if (((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) & 15) != 0 || a_stride % 16 != 0 || b_stride % 16 != 0 ||
        a_stride < depth || b_stride < depth || out_stride < cols)
        return MOK_ERR_INVALID_ARGUMENT;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    if (few_rows(rows, cols, depth, b_tile_rows)) {
        const BlockProduct few{static_cast<const uint8_t*>(a), static_cast<const uint8_t*>(b), a_stride, b_stride, a_scales, b_scales,
                               a_scale_row_stride, a_scale_block_stride, b_scale_row_stride, b_scale_block_stride, b_tile_rows,
                               static_cast<int>(rows), cols, depth, static_cast<bf16*>(out), out_stride, status};
        return launch_block_matmul_few(few, s);
    }
    Product p{};
    p.sa = a_scales;
    p.sa_row = a_scale_row_stride;
    p.sa_block = a_scale_block_stride;
    p.sb = b_scales;
    p.sb_row = b_scale_row_stride;
    p.sb_block = b_scale_block_stride;
    p.out = static_cast<bf16*>(out);
    p.out_stride = out_stride;
    p.rows = static_cast<int>(rows);
    p.cols = cols;
    p.k_blocks = div_up(depth, BK);
    p.m_tiles = div_up(rows, BM);
    p.n_tiles = div_up(cols, BN);
    p.splits = plan_splits(rows, cols, depth);
    p.partial = static_cast<float*>(scratch);
    p.status = status;
    if (p.splits > 1 && (scratch == nullptr || (reinterpret_cast<uintptr_t>(scratch) & 15) != 0)) return MOK_ERR_INVALID_ARGUMENT;
    if (static_cast<long long>(p.m_tiles) * p.n_tiles * p.splits > 0x7fffffffLL) return MOK_ERR_TOO_LARGE;
    CUtensorMap map_a, map_b, map_out{};
    MOK_TRY(code_map(&map_a, a, a_stride, rows, depth));
    MOK_TRY(code_map(&map_b, b, b_stride, cols, depth));
    p.box_out = p.splits == 1 && (reinterpret_cast<uintptr_t>(out) & 15) == 0 && out_stride % 8 == 0;
    if (p.box_out) {
        const cuuint64_t dims[4] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows), 1, 1};
        const cuuint64_t row_bytes = static_cast<cuuint64_t>(out_stride) * 2, strides[3] = {row_bytes, row_bytes * rows, row_bytes * rows};
        const cuuint32_t box[4] = {64, 32, 1, 1};
        MOK_TRY(encode_map(&map_out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, out, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B));
    }
    const int tiles = p.m_tiles * p.n_tiles * p.splits;
    if (b_tile_rows == 1) {
        static int resident[16] = {0};
        MOK_TRY(launch_pairs<kThreads>(block_matmul_kernel<true>, "block_matmul_kernel", resident, Layout::kBytes + 1024, tiles, s, map_a, map_b, map_out, p));
    } else {
        static int resident[16] = {0};
        MOK_TRY(launch_pairs<kThreads>(block_matmul_kernel<false>, "block_matmul_kernel", resident, Layout::kBytes + 1024, tiles, s, map_a, map_b, map_out, p));
    }
    if (p.splits > 1) {
        const long long count = rows * cols;
        MOK_TRY(launch_early(sum_shares_kernel, "sum_shares_kernel", dim3(static_cast<unsigned>((count + 1023) / 1024)), 256, 0, s,
                             static_cast<const float*>(p.partial), p.splits, count, cols, p.out, static_cast<long long>(out_stride)));
    }
    return MOK_OK;
}
