// The whole MoE layer for a few tokens: out[t] = shared(x[t]) + sum over k of w[t, k] * expert(route[t, k])(x[t]), expert(x) =
// W_down (silu(W_gate x) * (W_up x)), in two kernels.  With a handful of tokens the layer is the reading of its experts' weights
// (3 H I elements each, once); padding every expert to 256 rows, staging and combining would cost more than that.
//
//   gate / up: the rows of all experts in use lie end to end and are cut evenly, to the row, over the SMs; a piece is 16 gate rows
//              and the same 16 up rows, so that a lane of the mma holds both and forms hidden = silu(gate) * up itself.
//   down:      every SM owns a slice of the output's columns and walks all experts, so a token's sum over its experts happens in
//              one place, in shared memory, in a fixed order: shared expert, then experts by number.  No atomics, no partial rows.
//
// The second kernel is launched while the first runs, next to it on each SM, fills its ring with down weights and waits for the
// hidden rows in hardware (programmatic dependent launch): no spinning, and nothing has to be co-resident for it to finish.
// Every block finds out by itself which experts are in use and by whom (at most 4096 routes, in shared memory); hidden rows are
// kept by route number, so the order in which that happens does not matter.
#include "swiglu_math.cuh"
#include "weight_stream.cuh"

namespace mok {
namespace {

using namespace stream;

constexpr int kMaxTokens = 256;
constexpr int kMaxTopk = 32;
constexpr int kMaxRoutes = 4096;

struct Decode {
    const bf16* x;
    long long x_stride;
    const int32_t* routes;
    const float* route_weights;
    const bf16 *shared_gate, *shared_up, *shared_down;
    const uint8_t *gate, *up, *down;
    const float *gate_scales, *up_scales, *down_scales;   // W8: [E, ceil(I / 128), ceil(H / 128)] and [E, ceil(H / 128), ceil(I / 128)]
    bf16 *hidden, *hidden_shared, *out;
    uint32_t* status;
    int tokens, hidden_size, intermediate, shared_intermediate, experts, first_expert, topk;
    int clamp;
    float limit;
    int stages, stage_bytes, token_cap;   // the ring; tokens of a stage
};

// Which experts are in use: active[i] and the range [begin[i], begin[i + 1]) of its routes in list.
struct Routing {
    int* counts;        // [experts], then the next free place of each
    uint16_t* active;   // [experts]
    uint16_t* begin;    // [experts + 1], 4096 at most
    uint16_t* list;     // [routes]
    float* weights;     // [routes], beside list (down kernel)
    int* num_active;
};
__host__ __device__ __forceinline__ int routing_bytes(int experts, int routes, bool weights) {
    return 16 + 4 * experts + (weights ? 4 * routes : 0) + 2 * (2 * experts + 1 + routes) + 16;
}
__device__ __forceinline__ Routing carve_routing(uint8_t* smem, int experts, int routes, bool weights) {
    Routing r;
    r.num_active = reinterpret_cast<int*>(smem);
    r.counts = reinterpret_cast<int*>(smem + 16);
    r.weights = reinterpret_cast<float*>(r.counts + experts);
    r.active = reinterpret_cast<uint16_t*>(r.weights + (weights ? routes : 0));
    r.begin = r.active + experts;
    r.list = r.begin + experts + 1;
    return r;
}

// The expert of route i on this rank if the route counts: -1 for other ranks' experts, and for an expert that the token named
// before (the first occurrence carries the sum of the weights).
__device__ __forceinline__ int local_expert(const Decode& p, int i) {
    const int route = p.routes[i];
    const uint32_t e = static_cast<uint32_t>(route) - static_cast<uint32_t>(p.first_expert);
    if (e >= static_cast<uint32_t>(p.experts)) return -1;
    for (int j = i / p.topk * p.topk; j < i; ++j)
        if (p.routes[j] == route) return -1;
    return static_cast<int>(e);
}
// All threads of the block.
template <bool WEIGHTS>
__device__ __forceinline__ void find_experts(const Decode& p, const Routing& r) {
    const int routes = p.tokens * p.topk;
    for (int e = threadIdx.x; e < p.experts; e += kThreads) r.counts[e] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < routes; i += kThreads) {
        const int e = local_expert(p, i);
        if (e >= 0) atomicAdd(&r.counts[e], 1);
    }
    __syncthreads();
    if (threadIdx.x < 32) {   // experts in use and their ranges, by number; counts becomes the first place of each
        const int lane = threadIdx.x;
        int used = 0, total = 0;
        for (int base = 0; base < p.experts; base += 32) {
            const int e = base + lane;
            const int c = e < p.experts ? r.counts[e] : 0;
            const uint32_t here = __ballot_sync(0xffffffffu, c > 0);
            int sum = c;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const int n = __shfl_up_sync(0xffffffffu, sum, off);
                if (lane >= off) sum += n;
            }
            if (c > 0) {
                const int at = used + __popc(here & ((1u << lane) - 1u));
                r.active[at] = static_cast<uint16_t>(e);
                r.begin[at] = static_cast<uint16_t>(total + sum - c);
                r.counts[e] = total + sum - c;
            }
            used += __popc(here);
            total += __shfl_sync(0xffffffffu, sum, 31);
        }
        if (lane == 0) {
            r.begin[used] = static_cast<uint16_t>(total);
            *r.num_active = used;
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < routes; i += kThreads) {
        const int e = local_expert(p, i);
        if (e < 0) continue;
        const int at = atomicAdd(&r.counts[e], 1);
        r.list[at] = static_cast<uint16_t>(i);
        if (WEIGHTS) {
            float w = p.route_weights[i];
            for (int j = i + 1; j < (i / p.topk + 1) * p.topk; ++j)
                if (p.routes[j] == p.routes[i]) w += p.route_weights[j];
            r.weights[at] = w;
        }
    }
    __syncthreads();
}

// A piece as both sides see it: rows [row, row + count) of an expert (-1: the shared one) times tokens [from, from + tokens) of
// its list.
struct Piece {
    int expert, row, count, from, tokens;
};

// Calls f for every piece of the gate / up kernel that belongs to this block, in order, until it returns false.
template <typename F>
__device__ __forceinline__ void for_gate_up_pieces(const Decode& p, const Routing& r, F&& f) {
    constexpr int kPairs = kPieceRows / 2;
    const long long b = blockIdx.x, n = gridDim.x;
    Piece q;
    if (p.shared_gate != nullptr) {
        const int end = static_cast<int>(p.shared_intermediate * (b + 1) / n);
        q.expert = -1;
        for (q.row = static_cast<int>(p.shared_intermediate * b / n); q.row < end; q.row += kPairs) {
            q.count = min(kPairs, end - q.row);
            for (q.from = 0; q.from < p.tokens; q.from += p.token_cap) {
                q.tokens = min(p.token_cap, p.tokens - q.from);
                if (!f(q)) return;
            }
        }
    }
    const long long rows = static_cast<long long>(*r.num_active) * p.intermediate;
    const long long end = rows * (b + 1) / n;
    for (long long at = rows * b / n; at < end;) {
        const int a = static_cast<int>(at / p.intermediate);
        q.expert = r.active[a];
        q.row = static_cast<int>(at - static_cast<long long>(a) * p.intermediate);
        q.count = static_cast<int>(min(static_cast<long long>(min(kPairs, p.intermediate - q.row)), end - at));
        for (q.from = r.begin[a]; q.from < r.begin[a + 1]; q.from += p.token_cap) {
            q.tokens = min(p.token_cap, r.begin[a + 1] - q.from);
            if (!f(q)) return;
        }
        at += q.count;
    }
}
// The same for the down kernel: this block's columns of the output, [first, end).
template <typename F>
__device__ __forceinline__ void for_down_pieces(const Decode& p, const Routing& r, int first, int end, F&& f) {
    const int active = *r.num_active;
    const int pieces = (end - first + kPieceRows - 1) / kPieceRows;
    Piece q;
    for (int a = p.shared_gate != nullptr ? -1 : 0; a < active; ++a) {
        q.expert = a < 0 ? -1 : r.active[a];
        const int from = a < 0 ? 0 : r.begin[a], to = a < 0 ? p.tokens : r.begin[a + 1];
        for (int i = 0; i < pieces; ++i) {
            q.row = first + (end - first) * i / pieces;
            q.count = first + (end - first) * (i + 1) / pieces - q.row;
            for (q.from = from; q.from < to; q.from += p.token_cap) {
                q.tokens = min(p.token_cap, to - q.from);
                if (!f(q)) return;
            }
        }
    }
}

struct Block {
    Ring ring;
    const uint8_t* stages;
    volatile int* abort_flag;
    float *scratch, *sums;   // sums: the down kernel's [tokens][columns of the block]
    Routing routing;
};
template <int NT>
__device__ __forceinline__ Block set_up(const Decode& p, uint8_t* smem, uint64_t* bars, int* abort_flag, int sums, bool weights) {
    Block b;
    b.stages = smem;
    b.ring.base = smem_u32(smem);
    b.ring.full = smem_u32(bars);
    b.ring.empty = smem_u32(bars + kMaxStages);
    b.ring.stage_bytes = p.stage_bytes;
    b.ring.stages = p.stages;
    b.abort_flag = abort_flag;
    b.scratch = reinterpret_cast<float*>(smem + p.stages * p.stage_bytes);
    b.sums = b.scratch + scratch_floats<NT>();
    b.routing = carve_routing(reinterpret_cast<uint8_t*>(b.sums + (sums + 3) / 4 * 4), p.experts, p.tokens * p.topk, weights);
    if (threadIdx.x == 0) {
        *abort_flag = 0;
        b.ring.init();
    }
    return b;
}

template <bool W8, int NT>
__device__ __forceinline__ void consume_gate_up(Ring& ring, const Block& b, const Decode& p, const Piece& q, int warp, int lane,
                                                float (&acc)[2][NT][4]) {
    Scales<W8, false, NT> s;
    if (W8) {
        const int blocks = (p.hidden_size + 127) / 128, row_blocks = (p.intermediate + 127) / 128;
        s.row_block = 1;
#pragma unroll
        for (int m = 0; m < 2; ++m) {   // m tile: eight gate rows and the same up rows
            const int row = min(q.row + m * 8 + (lane >> 2), p.intermediate - 1);
            const long long at = (static_cast<long long>(q.expert) * row_blocks + row / 128) * blocks;
            s.lo[m] = p.gate_scales + at;
            s.hi[m] = p.up_scales + at;
        }
    }
    consume<W8, false, NT>(ring, b.stages, b.abort_flag, p.status, p.hidden_size, (q.count + 7) / 8, (q.tokens + 7) / 8, s, warp, lane, acc);
}

template <bool W8, int NT>
__global__ void __launch_bounds__(kThreads, NT <= 2 ? 2 : 1) moe_gate_up_kernel(const Decode p) {
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ __align__(8) uint64_t bars[2 * kMaxStages];
    __shared__ int abort_flag;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    allow_next_kernel();
    Block b = set_up<NT>(p, smem, bars, &abort_flag, 0, false);
    find_experts<false>(p, b.routing);   // its barriers also publish the ring
    Ring ring = b.ring;
    if (warp >= kConsumers) {
        const int producer = warp - kConsumers;
        bool ok = true;
        for_gate_up_pieces(p, b.routing, [&](const Piece& q) {
            const bool shared = q.expert < 0, w8 = W8 && !shared;
            Feed<NT> f;
            const long long row_bytes = p.hidden_size * (w8 ? 1 : 2);
            const uint8_t* gate = shared ? reinterpret_cast<const uint8_t*>(p.shared_gate) : p.gate;
            const uint8_t* up = shared ? reinterpret_cast<const uint8_t*>(p.shared_up) : p.up;
            const long long at = ((shared ? 0 : static_cast<long long>(q.expert) * p.intermediate) + q.row) * row_bytes + lane * 16;
#pragma unroll
            for (int j = 0; j < Feed<NT>::kWeights; ++j) {   // m tile m of the piece: eight gate rows from 8 m on and the same up rows
                const int i = producer + j * kProducers, pair = (i >> 4) * 8 + (i & 7);
                f.weight[j] = pair < q.count ? (i & 8 ? up : gate) + at + pair * row_bytes : nullptr;
            }
#pragma unroll
            for (int j = 0; j < Feed<NT>::kTokens; ++j) {
                const int i = producer + j * kProducers;
                f.token[j] = nullptr;
                if (i < q.tokens) {
                    const int token = shared ? q.from + i : b.routing.list[q.from + i] / p.topk;
                    f.token[j] = reinterpret_cast<const uint8_t*>(p.x + token * p.x_stride) + lane * 16;
                }
            }
            if (w8) ok = produce<Form<W8, false>, NT>(ring, b.abort_flag, p.status, f, 0, p.hidden_size, producer, lane);
            else ok = produce<Form<false, false>, NT>(ring, b.abort_flag, p.status, f, 0, p.hidden_size, producer, lane);
            return ok;
        });
        wait_copies();
    } else {
        for_gate_up_pieces(p, b.routing, [&](const Piece& q) {
            float acc[2][NT][4];
            if (W8 && q.expert >= 0) consume_gate_up<W8, NT>(ring, b, p, q, warp, lane, acc);
            else consume_gate_up<false, NT>(ring, b, p, q, warp, lane, acc);
            store_sums<NT>(b.scratch, acc, (q.count + 7) / 8, (q.tokens + 7) / 8, warp, lane);
            consumer_barrier();
            for (int i = threadIdx.x; i < 16 * q.tokens; i += kConsumerThreads) {
                const int pair = i & 15, c = i >> 4;
                if (pair >= q.count) continue;
                const int row = (pair >> 3) * 16 + (pair & 7);
                float g = sum_of<NT>(b.scratch, row, c), u = sum_of<NT>(b.scratch, row + 8, c);
                if (p.clamp) {   // comparisons that let a NaN through
                    g = g > p.limit ? p.limit : g;
                    u = u > p.limit ? p.limit : u < -p.limit ? -p.limit : u;
                }
                const bf16 h = __float2bfloat16(g * sigmoid_fast(g) * u);
                if (q.expert < 0) p.hidden_shared[static_cast<long long>(q.from + c) * p.shared_intermediate + q.row + pair] = h;
                else p.hidden[static_cast<long long>(b.routing.list[q.from + c]) * p.intermediate + q.row + pair] = h;
            }
            consumer_barrier();
            return true;
        });
    }
}

template <bool W8, int NT>
__device__ __forceinline__ void consume_down(Ring& ring, const Block& b, const Decode& p, const Piece& q, int warp, int lane,
                                             float (&acc)[2][NT][4]) {
    Scales<W8, false, NT> s;
    const int depth = q.expert < 0 ? p.shared_intermediate : p.intermediate;
    if (W8) {
        const int blocks = (p.intermediate + 127) / 128, row_blocks = (p.hidden_size + 127) / 128;
        s.row_block = 1;
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            const int lo = min(q.row + m * 16 + (lane >> 2), p.hidden_size - 1), hi = min(lo + 8, p.hidden_size - 1);
            const long long at = static_cast<long long>(q.expert) * row_blocks;
            s.lo[m] = p.down_scales + (at + lo / 128) * blocks;
            s.hi[m] = p.down_scales + (at + hi / 128) * blocks;
        }
    }
    consume<W8, false, NT>(ring, b.stages, b.abort_flag, p.status, depth, (q.count + 15) / 16, (q.tokens + 7) / 8, s, warp, lane, acc);
}

template <bool W8, int NT>
__global__ void __launch_bounds__(kThreads, NT <= 2 ? 2 : 1) moe_down_kernel(const Decode p) {
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ __align__(8) uint64_t bars[2 * kMaxStages];
    __shared__ int abort_flag;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int first = static_cast<int>(static_cast<long long>(p.hidden_size) * blockIdx.x / gridDim.x);
    const int end = static_cast<int>(static_cast<long long>(p.hidden_size) * (blockIdx.x + 1) / gridDim.x);
    const int cols = end - first;
    Block b = set_up<NT>(p, smem, bars, &abort_flag, p.tokens * cols, true);
    for (int i = threadIdx.x; i < p.tokens * cols; i += kThreads) b.sums[i] = 0.0f;
    find_experts<true>(p, b.routing);
    Ring ring = b.ring;
    if (warp >= kConsumers) {
        const int producer = warp - kConsumers;
        // Until the gate / up kernel is done the stages of an empty ring get their weights only; the hidden rows follow.
        bool ok = true;
        int early = 0;   // stages that have their weights
        auto feed = [&](const Piece& q, Feed<NT>& f) {
            const bool shared = q.expert < 0;
            const int depth = shared ? p.shared_intermediate : p.intermediate;
            const long long row_bytes = depth * (W8 && !shared ? 1 : 2);
            const uint8_t* w = shared ? reinterpret_cast<const uint8_t*>(p.shared_down) : p.down;
            const bf16* h = shared ? p.hidden_shared : p.hidden;
            w += ((shared ? 0 : static_cast<long long>(q.expert) * p.hidden_size) + q.row) * row_bytes + lane * 16;
#pragma unroll
            for (int j = 0; j < Feed<NT>::kWeights; ++j) {
                const int i = producer + j * kProducers;
                f.weight[j] = i < q.count ? w + i * row_bytes : nullptr;
            }
#pragma unroll
            for (int j = 0; j < Feed<NT>::kTokens; ++j) {
                const int i = producer + j * kProducers;
                f.token[j] = nullptr;
                if (i < q.tokens) {
                    const long long row = shared ? q.from + i : b.routing.list[q.from + i];
                    f.token[j] = reinterpret_cast<const uint8_t*>(h + row * depth) + lane * 16;
                }
            }
            return depth;
        };
        auto run_early = [&](const Feed<NT>& f, int depth, auto form) {
            typedef decltype(form) F;
            for (int k0 = 0; k0 < depth && early < ring.stages; k0 += F::kChunk, ++early)
                copy_weights<F, NT>(ring.base + early * ring.stage_bytes, f, k0, min(F::kChunk, depth - k0), producer, lane);
        };
        for_down_pieces(p, b.routing, first, end, [&](const Piece& q) {
            Feed<NT> f;
            const int depth = feed(q, f);
            if (W8 && q.expert >= 0) run_early(f, depth, Form<W8, false>());
            else run_early(f, depth, Form<false, false>());
            return early < ring.stages;
        });
        wait_previous_kernel();
        auto run = [&](const Feed<NT>& f, int depth, auto form) {
            typedef decltype(form) F;
            int k0 = 0;
            for (; k0 < depth && early > 0; k0 += F::kChunk, --early) {
                copy_tokens<F, NT>(ring.base + ring.stage * ring.stage_bytes, f, k0, min(F::kChunk, depth - k0), producer, lane);
                arrive_when_copied(ring.full + 8 * ring.stage);
                ring.advance();
            }
            ok = produce<F, NT>(ring, b.abort_flag, p.status, f, k0, depth, producer, lane);
        };
        for_down_pieces(p, b.routing, first, end, [&](const Piece& q) {
            Feed<NT> f;
            const int depth = feed(q, f);
            if (W8 && q.expert >= 0) run(f, depth, Form<W8, false>());
            else run(f, depth, Form<false, false>());
            return ok;
        });
        wait_copies();
    } else {
        for_down_pieces(p, b.routing, first, end, [&](const Piece& q) {
            float acc[2][NT][4];
            if (W8 && q.expert >= 0) consume_down<W8, NT>(ring, b, p, q, warp, lane, acc);
            else consume_down<false, NT>(ring, b, p, q, warp, lane, acc);
            store_sums<NT>(b.scratch, acc, (q.count + 15) / 16, (q.tokens + 7) / 8, warp, lane);
            consumer_barrier();
            for (int i = threadIdx.x; i < 32 * q.tokens; i += kConsumerThreads) {
                const int row = i & 31, c = i >> 5;
                if (row >= q.count) continue;
                int token = q.from + c;
                float w = 1.0f;
                if (q.expert >= 0) {
                    w = b.routing.weights[token];
                    token = b.routing.list[token] / p.topk;
                }
                float* sum = b.sums + token * cols + q.row - first + row;   // one thread per (token, column): a token is listed once
                *sum = fmaf(w, sum_of<NT>(b.scratch, row, c), *sum);
            }
            consumer_barrier();
            return true;
        });
        wait_previous_kernel();   // its word on how it went
        const bool bad = p.status != nullptr && *reinterpret_cast<volatile uint32_t*>(p.status) != 0;
        for (int i = threadIdx.x; i < p.tokens * cols; i += kConsumerThreads) {
            const int token = i / cols;
            p.out[static_cast<long long>(token) * p.hidden_size + first + i - token * cols] =
                __float2bfloat16(bad ? __uint_as_float(0x7FC00000u) : b.sums[i]);
        }
    }
}

// ---------------------------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------------------------
constexpr int kSmemPerSm = 228 * 1024, kSmemPerBlock = 227 * 1024, kStatic = 1024 + 256;   // reserved per block + barriers

// Ring of a kernel whose other shared memory is `other` bytes: as many stages as leave room for the second kernel's block next to
// it on the SM, or, where that would be fewer than three, as many as fit at all.  0: does not fit.
int ring_stages(int stage, int other) {
    int n = (kSmemPerSm / 2 - kStatic - other) / stage;
    if (n < 3) n = (kSmemPerBlock - kStatic - other) / stage;
    return n < 2 ? 0 : n > kMaxStages ? kMaxStages : n;
}

template <typename Kernel>
int launch_decode(Kernel kernel, const char* name, const Decode& p, int smem, bool early, cudaStream_t stream) {
    MOK_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(sm_count());
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = early ? 1 : 0;
    const cudaError_t err = cudaLaunchKernelEx(&cfg, kernel, p);
    if (err != cudaSuccess) return fail_cuda(name, err);
    MOK_LAUNCH_CHECK(name);
    return MOK_OK;
}

template <bool W8, int NT>
int run_decode(Decode p, cudaStream_t stream) {
    p.token_cap = 8 * NT;
    p.stage_bytes = Form<false, false>::stage_bytes(p.token_cap);
    if (W8) p.stage_bytes = p.stage_bytes > Form<true, false>::stage_bytes(p.token_cap) ? p.stage_bytes : Form<true, false>::stage_bytes(p.token_cap);
    const int routes = p.tokens * p.topk, scratch = scratch_floats<NT>() * 4;
    const int cols = (p.hidden_size + sm_count() - 1) / sm_count();
    const int up = scratch + routing_bytes(p.experts, routes, false);
    const int down = scratch + (p.tokens * cols + 3) / 4 * 16 + routing_bytes(p.experts, routes, true);
    const int up_stages = ring_stages(p.stage_bytes, up), down_stages = ring_stages(p.stage_bytes, down);
    if (up_stages == 0 || down_stages == 0) return MOK_ERR_TOO_LARGE;
    p.stages = up_stages;
    MOK_TRY(launch_decode(moe_gate_up_kernel<W8, NT>, "moe_gate_up_kernel", p, up + up_stages * p.stage_bytes, false, stream));
    p.stages = down_stages;
    return launch_decode(moe_down_kernel<W8, NT>, "moe_down_kernel", p, down + down_stages * p.stage_bytes, true, stream);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace mok

extern "C" int64_t mok_moe_decode_scratch_bytes(int num_tokens, int topk, int intermediate, int shared_intermediate) {
    if (num_tokens <= 0 || topk <= 0 || intermediate <= 0 || shared_intermediate < 0) return 0;
    return 2 * (static_cast<int64_t>(num_tokens) * topk * intermediate + static_cast<int64_t>(num_tokens) * shared_intermediate);
}

extern "C" int mok_moe_decode(const void* x, int64_t x_stride, const int32_t* top_experts, const float* router_weights, int num_tokens,
                              int topk, int hidden, const void* w_shared_gate, const void* w_shared_up, const void* w_shared_down,
                              int shared_intermediate, const void* w_gate, const void* w_up, const void* w_down, const float* gate_scales,
                              const float* up_scales, const float* down_scales, int intermediate, int num_experts, int first_expert,
                              int has_limit, float limit, void* out, void* scratch, uint32_t* status, mok_stream_t stream) {
    using namespace mok;
    if (num_tokens <= 0 || topk <= 0 || hidden <= 0 || intermediate <= 0 || num_experts <= 0 || first_expert < 0 || hidden % 64 != 0 ||
        intermediate % 64 != 0 || shared_intermediate < 0 || shared_intermediate % 64 != 0)
        return MOK_ERR_INVALID_ARGUMENT;
    if (num_tokens > kMaxTokens || topk > kMaxTopk || num_tokens * topk > kMaxRoutes || num_experts > MOK_MAX_LOCAL_EXPERTS) return MOK_ERR_TOO_LARGE;
    const bool shared = w_shared_gate != nullptr, w8 = gate_scales != nullptr;
    if (!x || !top_experts || !router_weights || !w_gate || !w_up || !w_down || !out || !scratch) return MOK_ERR_INVALID_ARGUMENT;
    if ((w_shared_up != nullptr) != shared || (w_shared_down != nullptr) != shared || shared != (shared_intermediate > 0) ||
        (up_scales != nullptr) != w8 || (down_scales != nullptr) != w8)
        return MOK_ERR_INVALID_ARGUMENT;
    if (!aligned16(x) || !aligned16(w_gate) || !aligned16(w_up) || !aligned16(w_down) || !aligned16(w_shared_gate) || !aligned16(w_shared_up) ||
        !aligned16(w_shared_down) || !aligned16(scratch) || x_stride % 8 != 0 || x_stride < 0)
        return MOK_ERR_INVALID_ARGUMENT;
    Decode p{};
    p.x = static_cast<const bf16*>(x);
    p.x_stride = x_stride;
    p.routes = top_experts;
    p.route_weights = router_weights;
    p.shared_gate = static_cast<const bf16*>(w_shared_gate);
    p.shared_up = static_cast<const bf16*>(w_shared_up);
    p.shared_down = static_cast<const bf16*>(w_shared_down);
    p.gate = static_cast<const uint8_t*>(w_gate);
    p.up = static_cast<const uint8_t*>(w_up);
    p.down = static_cast<const uint8_t*>(w_down);
    p.gate_scales = gate_scales;
    p.up_scales = up_scales;
    p.down_scales = down_scales;
    p.hidden = static_cast<bf16*>(scratch);
    p.hidden_shared = p.hidden + static_cast<long long>(num_tokens) * topk * intermediate;
    p.out = static_cast<bf16*>(out);
    p.status = status;
    p.tokens = num_tokens;
    p.hidden_size = hidden;
    p.intermediate = intermediate;
    p.shared_intermediate = shared_intermediate;
    p.experts = num_experts;
    p.first_expert = first_expert;
    p.topk = topk;
    p.clamp = has_limit;
    p.limit = limit;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    if (w8) {
        if (num_tokens <= 8) return run_decode<true, 1>(p, s);
        if (num_tokens <= 16) return run_decode<true, 2>(p, s);
        return run_decode<true, 4>(p, s);
    }
    if (num_tokens <= 8) return run_decode<false, 1>(p, s);
    if (num_tokens <= 16) return run_decode<false, 2>(p, s);
    return run_decode<false, 4>(p, s);
}
