// The 8-bit block-scaled product for a few rows of A, which is the reading of B: B's rows are cut evenly, to the row, over the blocks and
// streamed as weight_stream.cuh describes, with A's rows on the N side of the mma.  Codes become f16, exactly; every block of 128 along k
// is summed on its own, scaled in fp32 and added.
#include "block_matmul.cuh"
#include "weight_stream.cuh"

namespace mok {
namespace {

using namespace stream;

typedef Form<true, true> F;

struct Few {
    BlockProduct p;
    int stage_bytes;
};

template <int NT>
__global__ void __launch_bounds__(kThreads, NT <= 2 ? 2 : 1) block_matmul_few_kernel(const Few f) {
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ Bars bars;
    const BlockProduct& p = f.p;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    Ring ring = set_up_ring(bars, smem, f.stage_bytes, kConsumers, 1);
    wait_previous_kernel();
    allow_next_kernel();
    Deposit sums;
    sums.scratch = reinterpret_cast<float*>(smem + kConsumers * f.stage_bytes);
    const int first = static_cast<int>(static_cast<long long>(p.cols) * blockIdx.x / gridDim.x);
    const int end = static_cast<int>(static_cast<long long>(p.cols) * (blockIdx.x + 1) / gridDim.x);
    const int pieces = (end - first + kRows - 1) / kRows;
    const int chunks = F::chunks(p.depth), slots = min(chunks, kConsumers), tiles = (p.rows + 7) >> 3;
    int turn = warp < kConsumers ? warp : warp - kConsumers;
    for (int i = 0; i < pieces; ++i) {
        const int row0 = first + (end - first) * i / pieces, count = first + (end - first) * (i + 1) / pieces - row0;
        if (warp == kFinisher) {
            collect(sums, bars, p.status, slots);
            const bool bad = bars.abort_flag != 0;
            for (int k = lane; k < kRows * p.rows; k += 32) {
                const int row = k & (kRows - 1), c = k / kRows;
                if (row < count)
                    p.out[c * p.out_stride + row0 + row] = __float2bfloat16(bad ? __uint_as_float(0x7FC00000u) : sum_of<NT>(sums, slots, row, c));
            }
            collected(sums, bars, lane);
        } else if (warp >= kConsumers) {
            Feed feed;
            feed.row_bytes = p.b_stride;
            feed.rows_low = count;
            feed.rows_high = count - 8;
            feed.low = p.b + row0 * p.b_stride + lane * 16;
            feed.high = feed.low + 8 * p.b_stride;
            feed.tokens = p.rows;
            feed.token = p.a + (lane < p.rows ? lane : 0) * p.a_stride;
            feed.scale = lane < count ? p.sb + (row0 + lane) / p.b_tile_rows * p.sb_row : nullptr;
            feed.scale_stride = p.sb_block;
            feed.token_scale = lane < p.rows ? p.sa + lane * p.sa_row : nullptr;
            feed.token_scale_stride = p.sa_block;
            if (!produce<F, true>(ring, &bars.abort_flag, p.status, feed, turn, p.depth, p.rows, lane)) break;
            turn = (turn - chunks) & (kProducers - 1);
            ring.next_piece(chunks);
        } else {
            const int slot = turn;
            if (slot < chunks) {
                float acc[NT][4];
                clear(acc);
                for (int c = slot; c < chunks; c += kConsumers)
                    consume<true, true, NT>(ring, smem, &bars.abort_flag, p.status, c, p.depth, tiles, p.rows, lane, acc);
                deposit<NT>(sums, bars, p.status, acc, slot, tiles, lane);
            }
            ++sums.piece;
            turn = (turn - chunks) & (kConsumers - 1);
            ring.next_piece(chunks);
        }
    }
    if (warp >= kConsumers && warp != kFinisher) wait_copies();
}

template <int NT>
int launch(const Few& f, cudaStream_t stream) {
    constexpr int kSmemPerSm = 228 * 1024, kSmemPerBlock = 227 * 1024, kStatic = 1024 + 384;
    static_assert(sizeof(Bars) <= 384 && kConsumers * F::stage_bytes(kFewRows) + 4 * deposit_floats<3>() <= kSmemPerBlock - kStatic, "");
    static int ready[16] = {0};
    int dev = 0;
    MOK_CUDA_CHECK(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 16) return MOK_ERR_UNSUPPORTED;
    if (ready[dev] == 0) {
        MOK_CUDA_CHECK(cudaFuncSetAttribute(block_matmul_few_kernel<NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemPerBlock - kStatic));
        MOK_CUDA_CHECK(cudaFuncSetAttribute(block_matmul_few_kernel<NT>, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));
        ready[dev] = 1;
    }
    const int smem = kConsumers * f.stage_bytes + 4 * deposit_floats<NT>();
    const int blocks = smem <= kSmemPerSm / 2 - kStatic ? 2 : 1;
    return launch_early(block_matmul_few_kernel<NT>, "block_matmul_few_kernel", dim3(blocks * sm_count()), kThreads, smem, stream, f);
}

}  // namespace

int launch_block_matmul_few(const BlockProduct& p, cudaStream_t stream) {
    Few f{p, F::stage_bytes(p.rows)};
    if (p.rows <= 8) return launch<1>(f, stream);
    if (p.rows <= 16) return launch<2>(f, stream);
    return launch<3>(f, stream);
}

}  // namespace mok
