// The whole MoE layer for a few tokens: out[t] = shared(x[t]) + sum over k of w[t, k] * expert(route[t, k])(x[t]), expert(x) =
// W_down (silu(W_gate x) * (W_up x)), in two kernels (kWideFrom tokens and more: moe_decode_wide.cuh).  With a handful of tokens the
// layer is the reading of its experts' weights (3 H I elements each, once); padding every expert to 256 rows, staging and combining
// would cost more than that.
//
//   gate / up: the rows of all experts in use lie end to end and are cut evenly, to the row, over the SMs; a piece is 8 gate rows and
//              the same 8 up rows, so that hidden = silu(gate) * up is formed where the sums end up.
//   down:      every SM owns a slice of the output's columns and walks all experts, so a token's sum over its experts happens in
//              one place, in shared memory, in a fixed order: shared expert, then experts by number.  No atomics on values, no
//              partial rows.  One warp adds the experts' parts while the others are at the next experts: when the whole block met for
//              every expert, 2000 of 2500 clocks an expert were latency (hidden 2048, intermediate 768).
//
// The second kernel is launched while the first runs, takes an SM's place as soon as there is room, fills its ring with down weights
// and waits for the hidden rows in hardware (programmatic dependent launch): no spinning, and nothing has to be co-resident for it to
// finish.
// Every block finds out by itself which experts are in use and by whom, while its producers already copy the shared expert's
// weights; hidden rows are kept by route number, so the order in which that happens does not matter.
#include "row_slice.cuh"
#include "swiglu_math.cuh"
#include "weight_stream.cuh"

namespace mok {
namespace {

using namespace stream;

constexpr int kMaxTokens = 256;
constexpr int kMaxTopk = 32;
constexpr int kMaxRoutes = 4096;
constexpr int kPairs = kRows / 2;
constexpr int kNobody = 0xFFFF;

struct Decode {
    const bf16* x;
    long long x_stride;
    const int32_t* routes;
    const float* route_weights;
    const bf16 *shared_gate, *shared_up, *shared_down;
    const uint8_t *gate, *up, *down;
    const float *gate_scales, *up_scales, *down_scales;   // W8: [E, ceil(I / 128), ceil(H / 128)] and [E, ceil(H / 128), ceil(I / 128)]
    bf16 *hidden, *hidden_shared, *out;
    __half* x_half;                       // W8: tokens and, in place, hidden rows as f16 with a power of two per row
    float *x_scale, *hidden_scale;        // [tokens], [routes]
    float* parts;                         // wide form: [routes, then tokens for the shared expert][hidden_size]
    uint32_t* status;
    int tokens, hidden_size, intermediate, shared_intermediate, experts, first_expert, topk;
    int clamp;
    float limit;
    int stages, stage_bytes, token_cap;   // the ring; tokens of a stage
};

// Which experts are in use: active[i], and the range [begin[i], begin[i + 1]) of its routes in list (with their tokens and weights
// beside).  An expert that a token names more than once is listed once, with the sum of the weights.  passes[i]: how often the
// experts before i are read in all, when token_cap of their tokens fit a stage.
struct Routing {
    int* num_active;
    int* next;               // [experts] counts, then the next free place in list
    float* weights;          // [routes]
    uint16_t *expert;        // [routes] of this rank, or kNobody
    uint16_t *active, *begin, *passes, *list;   // [experts], [experts + 1], [experts + 1], [routes]
    uint8_t* token;          // [routes]
};
__host__ __device__ __forceinline__ int routing_bytes(int experts, int routes) {
    return 16 + 4 * experts + 4 * routes + 2 * (routes + 3 * experts + 2 + routes) + routes + 16;
}
__device__ __forceinline__ Routing carve_routing(uint8_t* smem, int experts, int routes) {
    Routing r;
    r.num_active = reinterpret_cast<int*>(smem);
    r.next = reinterpret_cast<int*>(smem + 16);
    r.weights = reinterpret_cast<float*>(r.next + experts);
    r.expert = reinterpret_cast<uint16_t*>(r.weights + routes);
    r.active = r.expert + routes;
    r.begin = r.active + experts;
    r.passes = r.begin + experts + 1;
    r.list = r.passes + experts + 1;
    r.token = reinterpret_cast<uint8_t*>(r.list + routes);
    return r;
}

// Up to 32 routes: one warp, in registers (the general form costs a single token 4 us, mostly instruction misses).
__device__ __forceinline__ void find_experts_of_few(const Decode& p, const Routing& r, int lane) {
    const int routes = p.tokens * p.topk, token = lane / p.topk;
    uint32_t e = kNobody;
    float w = 0.0f;
    if (lane < routes) {
        const uint32_t local = static_cast<uint32_t>(__ldcg(p.routes + lane)) - static_cast<uint32_t>(p.first_expert);
        if (local < static_cast<uint32_t>(p.experts)) e = local;
        w = __ldcg(p.route_weights + lane);
    }
    const uint32_t same = __match_any_sync(0xffffffffu, e == kNobody ? 0x80000000u | lane : e << 8 | token);   // token and expert
    const bool first = e != kNobody && (same & ((1u << lane) - 1u)) == 0;
    if (__any_sync(0xffffffffu, (same & (same - 1u)) != 0)) {
        float sum = 0.0f;
        for (int l = 0; l < routes; ++l) {
            const float other = __shfl_sync(0xffffffffu, w, l);
            if (same >> l & 1u) sum += other;
        }
        w = sum;
    }
    const uint32_t mates = __match_any_sync(0xffffffffu, first ? e : 0x80000000u | lane);
    const int mine = __popc(mates) | (__popc(mates) + p.token_cap - 1) / p.token_cap << 16;
    int rank = 0, before = 0, total = 0;
    const uint32_t leaders = __ballot_sync(0xffffffffu, first && (mates & ((1u << lane) - 1u)) == 0);
    for (uint32_t left = leaders; left != 0; left &= left - 1u) {
        const int l = __ffs(left) - 1;
        const uint32_t other = __shfl_sync(0xffffffffu, e, l);
        const int its = __shfl_sync(0xffffffffu, mine, l);
        total += its;
        if (other < e) {
            ++rank;
            before += its;
        }
    }
    if (first) {
        const int at = (before & 0xFFFF) + __popc(mates & ((1u << lane) - 1u));
        r.list[at] = static_cast<uint16_t>(lane);
        r.token[at] = static_cast<uint8_t>(token);
        r.weights[at] = w;
        r.active[rank] = static_cast<uint16_t>(e);   // by every route of the expert, alike
        r.begin[rank] = static_cast<uint16_t>(before & 0xFFFF);
        r.passes[rank] = static_cast<uint16_t>(before >> 16);
    }
    if (lane == 0) {
        r.begin[__popc(leaders)] = static_cast<uint16_t>(total & 0xFFFF);
        r.passes[__popc(leaders)] = static_cast<uint16_t>(total >> 16);
        *r.num_active = __popc(leaders);
    }
}

// The consumer threads of the block.
__device__ __forceinline__ void find_experts(const Decode& p, const Routing& r) {
    const int routes = p.tokens * p.topk;
    if (routes <= 32) {
        if (threadIdx.x < 32) find_experts_of_few(p, r, threadIdx.x);
        consumer_barrier();
        return;
    }
    for (int i = threadIdx.x; i < routes; i += kConsumerThreads) {
        const uint32_t e = static_cast<uint32_t>(__ldcg(p.routes + i)) - static_cast<uint32_t>(p.first_expert);
        r.expert[i] = static_cast<uint16_t>(e < static_cast<uint32_t>(p.experts) ? e : kNobody);
    }
    for (int e = threadIdx.x; e < p.experts; e += kConsumerThreads) r.next[e] = 0;
    consumer_barrier();
    auto counts = [&](int i, int token) {   // whether route i is its token's first to that expert
        const int e = r.expert[i];
        bool first = e != kNobody;
        for (int j = token * p.topk; j < i; ++j) first = first && r.expert[j] != e;
        return first;
    };
    for (int i = threadIdx.x; i < routes; i += kConsumerThreads)
        if (counts(i, i / p.topk)) atomicAdd(&r.next[r.expert[i]], 1);
    consumer_barrier();
    if (threadIdx.x < 32) {   // experts in use and their ranges, by number
        const int lane = threadIdx.x;
        int used = 0, total = 0;   // total: routes, and passes from bit 16 on (4096 at most of either)
        for (int base = 0; base < p.experts; base += 32) {
            const int e = base + lane;
            const int c = e < p.experts ? r.next[e] : 0;
            const uint32_t here = __ballot_sync(0xffffffffu, c > 0);
            if (here == 0) continue;
            const int mine = c | (c + p.token_cap - 1) / p.token_cap << 16;
            int sum = mine;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const int n = __shfl_up_sync(0xffffffffu, sum, off);
                if (lane >= off) sum += n;
            }
            if (c > 0) {
                const int at = used + __popc(here & ((1u << lane) - 1u)), before = total + sum - mine;
                r.active[at] = static_cast<uint16_t>(e);
                r.begin[at] = static_cast<uint16_t>(before & 0xFFFF);
                r.passes[at] = static_cast<uint16_t>(before >> 16);
                r.next[e] = before & 0xFFFF;
            }
            used += __popc(here);
            total += __shfl_sync(0xffffffffu, sum, 31);
        }
        if (lane == 0) {
            r.begin[used] = static_cast<uint16_t>(total & 0xFFFF);
            r.passes[used] = static_cast<uint16_t>(total >> 16);
            *r.num_active = used;
        }
    }
    consumer_barrier();
    for (int i = threadIdx.x; i < routes; i += kConsumerThreads) {
        const int token = i / p.topk;
        if (!counts(i, token)) continue;
        float w = __ldcg(p.route_weights + i);
        for (int j = i + 1; j < (token + 1) * p.topk; ++j)
            if (r.expert[j] == r.expert[i]) w += __ldcg(p.route_weights + j);
        const int at = atomicAdd(&r.next[r.expert[i]], 1);   // any order: a column's sums do not depend on its place
        r.list[at] = static_cast<uint16_t>(i);
        r.token[at] = static_cast<uint8_t>(token);
        r.weights[at] = w;
    }
    consumer_barrier();
}

// A piece as both sides see it: rows [row, row + count) of an expert (-1: the shared one) times tokens [from, from + tokens) of
// its list.
struct Piece {
    int expert, row, count, from, tokens;
};

// Calls f for every piece of the gate / up kernel that belongs to this block, in order, until it returns false: first the shared
// expert's, which need no routing, then the others.
template <typename F>
__device__ __forceinline__ bool for_shared_pieces(const Decode& p, F&& f) {
    if (p.shared_gate == nullptr) return true;
    Piece q;
    const int end = static_cast<int>(static_cast<long long>(p.shared_intermediate) * (blockIdx.x + 1) / gridDim.x);
    q.expert = -1;
    for (q.row = static_cast<int>(static_cast<long long>(p.shared_intermediate) * blockIdx.x / gridDim.x); q.row < end; q.row += kPairs) {
        q.count = min(kPairs, end - q.row);
        for (q.from = 0; q.from < p.tokens; q.from += p.token_cap) {
            q.tokens = min(p.token_cap, p.tokens - q.from);
            if (!f(q)) return false;
        }
    }
    return true;
}
// The routed rows, each counted once per pass over its expert (an expert of many tokens is read, from L2, more than once), are cut
// into equal shares.
template <typename F>
__device__ __forceinline__ void for_routed_pieces(const Decode& p, const Routing& r, F&& f) {
    const int active = *r.num_active;
    const long long rows = static_cast<long long>(r.passes[active]) * p.intermediate;
    const long long first = rows * blockIdx.x / gridDim.x, last = rows * (blockIdx.x + 1) / gridDim.x;
    if (first == last) return;
    int a = 0;
    for (int n = active; n - a > 1;) {   // the expert that `first` lies in
        const int mid = (a + n) >> 1;
        if (static_cast<long long>(r.passes[mid]) * p.intermediate <= first) a = mid;
        else n = mid;
    }
    Piece q;
    for (; a < active; ++a) {
        const long long before = static_cast<long long>(r.passes[a]) * p.intermediate;
        if (before >= last) return;
        const int passes = r.passes[a + 1] - r.passes[a];
        const int from = first > before ? static_cast<int>(first - before) / passes : 0;
        const int to = static_cast<int>(min(last - before, static_cast<long long>(passes) * p.intermediate)) / passes;
        q.expert = r.active[a];
        for (q.row = from; q.row < to; q.row += kPairs) {
            q.count = min(kPairs, to - q.row);
            for (q.from = r.begin[a]; q.from < r.begin[a + 1]; q.from += p.token_cap) {
                q.tokens = min(p.token_cap, r.begin[a + 1] - q.from);
                if (!f(q)) return;
            }
        }
    }
}

// ---- tokens for 8-bit weights -------------------------------------------------------------------------------------------
// bf16 rows as f16 with a power of two per row that brings its largest finite value to [2^14, 2^15): eight bits of significand fit
// eleven, values from 2^-28 of the largest on are exact and smaller ones are off by 2^-40 of it at most, far below the sums' fp32.
// One block per row; `out` may be `rows` itself.  HIDDEN: rows of routes to other ranks' experts hold nothing and are passed over,
// and the rows are the previous kernel's, which may still run.
template <bool HIDDEN>
__global__ void __launch_bounds__(256) to_half_kernel(const Decode p) {
    __shared__ uint32_t part[8];
    const int row = blockIdx.x, cols = HIDDEN ? p.intermediate : p.hidden_size;
    const bf16* in = HIDDEN ? p.hidden + static_cast<long long>(row) * cols : p.x + row * p.x_stride;
    uint4* out = HIDDEN ? reinterpret_cast<uint4*>(p.hidden + static_cast<long long>(row) * cols)
                        : reinterpret_cast<uint4*>(p.x_half + static_cast<long long>(row) * cols);
    if (HIDDEN) allow_next_kernel();   // the down kernel: it has weights to fetch meanwhile, and waits for this one
    wait_previous_kernel();            // every block: who waits for this kernel has waited for the one before
    if (HIDDEN) {
        const uint32_t e = static_cast<uint32_t>(__ldcg(p.routes + row)) - static_cast<uint32_t>(p.first_expert);
        if (e >= static_cast<uint32_t>(p.experts)) return;
    } else {
        allow_next_kernel();
    }
    uint32_t big = 0;
    auto finite = [](uint32_t v) { return v < 0x7F80u ? v : 0u; };
    for (int i = threadIdx.x; i < cols / 8; i += 256) {
        const uint4 v = __ldcg(reinterpret_cast<const uint4*>(in) + i);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) big = max(big, max(finite(w[j] & 0x7FFFu), finite(w[j] >> 16 & 0x7FFFu)));
    }
    big = __reduce_max_sync(0xffffffffu, big);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = big;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) big = max(big, part[i]);
    // biased exponent of the scale's reciprocal, 2^(14 - exponent); 1 .. 253 keeps both normal
    const int k = min(max(127 + 14 - (static_cast<int>(big >> 7) - 127), 1), 253);
    const float factor = __uint_as_float(static_cast<uint32_t>(k) << 23);
    if (threadIdx.x == 0) (HIDDEN ? p.hidden_scale : p.x_scale)[row] = __uint_as_float(static_cast<uint32_t>(254 - k) << 23);
    for (int i = threadIdx.x; i < cols / 8; i += 256) {
        const uint4 v = __ldcg(reinterpret_cast<const uint4*>(in) + i);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
        uint32_t h[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 f = unpack_bf16x2(w[j]);
            const __half2 r = __floats2half2_rn(f.x * factor, f.y * factor);
            h[j] = *reinterpret_cast<const uint32_t*>(&r);
        }
        out[i] = make_uint4(h[0], h[1], h[2], h[3]);
    }
}

// Rounded to bf16 (half a step, 2^-8 of the value): the down product takes both operands in one type, and the layer for 512 tokens
// and more rounds here as well, so that a token's result does not change its precision with the batch.  Against 64 bits the output
// is off by 0.0023 of its norm; its own rounding to bf16 alone gives 0.0017.
__device__ __forceinline__ bf16 hidden_value(const Decode& p, float g, float u) {
    if (p.clamp) {   // comparisons that let a NaN through
        g = g > p.limit ? p.limit : g;
        u = u > p.limit ? p.limit : u < -p.limit ? -p.limit : u;
    }
    return __float2bfloat16(g * sigmoid_fast(g) * u);
}

// ---- gate / up --------------------------------------------------------------------------------------------------------
template <bool W8>
__global__ void __launch_bounds__(kThreads, 2) moe_gate_up_kernel(const Decode p) {
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ Bars bars;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    Ring ring = set_up_ring(bars, smem, p.stage_bytes, p.stages, kConsumerThreads);
    wait_previous_kernel();
    allow_next_kernel();   // not before: the down kernel reads weights and routes that earlier kernels may have written
    Deposit sums;
    sums.scratch = reinterpret_cast<float*>(smem + p.stages * p.stage_bytes);
    const Routing r = carve_routing(reinterpret_cast<uint8_t*>(sums.scratch + deposit_floats<1>()), p.experts, p.tokens * p.topk);
    const int chunks = Form<false, false>::chunks(p.hidden_size), chunks8 = Form<true, false>::chunks(p.hidden_size);
    auto slots_of = [&](const Piece& q) { return min(W8 && q.expert >= 0 ? chunks8 : chunks, kConsumers); };
    if (warp == kFinisher) {
        auto run = [&](const Piece& q) {
            const int slots = slots_of(q);
            collect(sums, bars, p.status, slots);
            for (int i = lane; i < kPairs * q.tokens; i += 32) {
                const int pair = i & (kPairs - 1), c = i / kPairs;
                if (pair >= q.count) continue;
                float g = sum_of<1>(sums, slots, pair, c), u = sum_of<1>(sums, slots, pair + 8, c);
                if (W8 && q.expert >= 0) {
                    const float scale = __ldcg(p.x_scale + r.token[q.from + c]);
                    g *= scale;
                    u *= scale;
                }
                const bf16 h = hidden_value(p, g, u);
                if (q.expert < 0) p.hidden_shared[static_cast<long long>(q.from + c) * p.shared_intermediate + q.row + pair] = h;
                else p.hidden[static_cast<long long>(r.list[q.from + c]) * p.intermediate + q.row + pair] = h;
            }
            collected(sums, bars, lane);
            return true;
        };
        for_shared_pieces(p, run);
        if (mbar_wait(smem_u32(&bars.routed), 0, &bars.abort_flag, p.status)) for_routed_pieces(p, r, run);
    } else if (warp >= kConsumers) {
        int turn = warp - kConsumers;   // this producer's next chunk, counted from the piece's first
        auto run = [&](const Piece& q) {
            const bool shared = q.expert < 0, w8 = W8 && !shared;
            Feed f;
            f.row_bytes = p.hidden_size * (w8 ? 1 : 2);
            f.rows_low = f.rows_high = q.count;
            const long long at = ((shared ? 0 : static_cast<long long>(q.expert) * p.intermediate) + q.row) * f.row_bytes + lane * 16;
            f.low = (shared ? reinterpret_cast<const uint8_t*>(p.shared_gate) : p.gate) + at;
            f.high = (shared ? reinterpret_cast<const uint8_t*>(p.shared_up) : p.up) + at;
            f.tokens = q.tokens;
            const int token = shared ? q.from + lane : lane < q.tokens ? r.token[q.from + lane] : 0;
            f.token = w8 ? reinterpret_cast<const uint8_t*>(p.x_half + static_cast<long long>(token) * p.hidden_size)
                         : reinterpret_cast<const uint8_t*>(p.x + token * p.x_stride);
            f.scale = nullptr;
            if (w8 && lane < kRows && (lane & 7) < q.count) {
                const int blocks = (p.hidden_size + 127) / 128, row_blocks = (p.intermediate + 127) / 128;
                f.scale = (lane < 8 ? p.gate_scales : p.up_scales) +
                          (static_cast<long long>(q.expert) * row_blocks + (q.row + (lane & 7)) / 128) * blocks;
                f.scale_stride = 1;
            }
            const bool ok = w8 ? produce<Form<W8, false>, false>(ring, &bars.abort_flag, p.status, f, turn, p.hidden_size, p.token_cap, lane)
                               : produce<Form<false, false>, false>(ring, &bars.abort_flag, p.status, f, turn, p.hidden_size, p.token_cap, lane);
            const int n = w8 ? chunks8 : chunks;
            turn = (turn - n) & (kProducers - 1);
            ring.next_piece(n);
            return ok;
        };
        if (for_shared_pieces(p, run) && mbar_wait(smem_u32(&bars.routed), 0, &bars.abort_flag, p.status)) for_routed_pieces(p, r, run);
        wait_copies();
    } else {
        find_experts(p, r);
        mbar_arrive(smem_u32(&bars.routed));
        int turn = warp;   // this warp's next chunk, counted from the piece's first
        auto run = [&](const Piece& q) {
            const bool shared = q.expert < 0, w8 = W8 && !shared;
            const int n = w8 ? chunks8 : chunks, tiles = (q.tokens + 7) >> 3;
            const int slot = turn;
            if (slot < n) {
                float acc[1][4];
                clear(acc);
                for (int c = slot; c < n; c += kConsumers) {
                    if (w8) consume<W8, false, 1>(ring, smem, &bars.abort_flag, p.status, c, p.hidden_size, tiles, p.token_cap, lane, acc);
                    else consume<false, false, 1>(ring, smem, &bars.abort_flag, p.status, c, p.hidden_size, tiles, p.token_cap, lane, acc);
                }
                deposit<1>(sums, bars, p.status, acc, slot, tiles, lane);
            }
            ++sums.piece;
            ring.next_piece(n);
            turn = (turn - n) & (kConsumers - 1);
            return true;
        };
        for_shared_pieces(p, run);
        for_routed_pieces(p, r, run);
    }
}

// ---- down -------------------------------------------------------------------------------------------------------------
// Calls f for every piece of rows [row, row + count), in order, until it returns false.  `shared_only`: those that need no routing.
template <typename F>
__device__ __forceinline__ bool for_experts(const Decode& p, const Routing& r, int row, int count, bool shared_only, F&& f) {
    const int active = shared_only ? 0 : *r.num_active;
    Piece q;
    q.row = row;
    q.count = count;
    for (int a = p.shared_gate != nullptr ? -1 : 0; a < active; ++a) {
        q.expert = a < 0 ? -1 : r.active[a];
        const int to = a < 0 ? p.tokens : r.begin[a + 1];
        for (q.from = a < 0 ? 0 : r.begin[a]; q.from < to; q.from += p.token_cap) {
            q.tokens = min(p.token_cap, to - q.from);
            if (!f(q)) return false;
        }
    }
    return true;
}

// The producers.  Until the gate / up kernel is done the stages of the empty ring get their weights only; the hidden rows follow.
template <bool W8>
__device__ __forceinline__ void produce_down(const Decode& p, const Routing& r, const RowSlice& slice, const Ring& start, Bars& bars, int producer,
                                             int lane) {
    auto depth_of = [&](const Piece& q) { return q.expert < 0 ? p.shared_intermediate : p.intermediate; };
    auto weights_of = [&](const Piece& q, Feed& f) {
        const bool shared = q.expert < 0;
        f.row_bytes = depth_of(q) * (W8 && !shared ? 1 : 2);
        f.rows_low = q.count;
        f.rows_high = q.count - 8;
        f.low = (shared ? reinterpret_cast<const uint8_t*>(p.shared_down) : p.down) +
                ((shared ? 0 : static_cast<long long>(q.expert) * p.hidden_size) + q.row) * f.row_bytes + lane * 16;
        f.high = f.low + 8 * f.row_bytes;
        f.scale = nullptr;
        if (W8 && !shared && lane < q.count) {
            const int blocks = (p.intermediate + 127) / 128, row_blocks = (p.hidden_size + 127) / 128;
            f.scale = p.down_scales + (static_cast<long long>(q.expert) * row_blocks + (q.row + lane) / 128) * blocks;
            f.scale_stride = 1;
        }
    };
    auto tokens_of = [&](const Piece& q, Feed& f) {
        const bool shared = q.expert < 0;
        const int row = shared ? q.from + lane : lane < q.tokens ? r.list[q.from + lane] : 0;
        f.tokens = q.tokens;
        f.token = reinterpret_cast<const uint8_t*>((shared ? p.hidden_shared : p.hidden) + static_cast<long long>(row) * depth_of(q));
    };
    // this producer's chunks among the first `stages` of the sequence, from chunk number `done` on
    int met = 0;
    auto early = [&](const Piece& q, int done, auto form) {
        typedef decltype(form) F;
        const int depth = depth_of(q);
        Feed f;
        weights_of(q, f);
        for (int c = 0; c * F::kChunk < depth && met < start.stages; ++c, ++met)
            if (met >= done && (met & (kProducers - 1)) == producer) {
                const int len = min(F::kChunk, depth - c * F::kChunk);
                copy_weights<F>(start.base + met * start.stage_bytes, f, c * F::kChunk, len, lane);
                if (F::kScales) copy_scales<F, false>(start.base + met * start.stage_bytes, f, c * F::kChunk, len, p.token_cap, lane);
            }
        return met < start.stages;
    };
    auto early_pieces = [&](bool shared_only, int done) {
        met = 0;
        for (int i = 0; i < slice.at_most(shared_only ? 1 : slice.pieces); ++i)
            if (!for_experts(p, r, slice.row(i), slice.row(i + 1) - slice.row(i), shared_only, [&](const Piece& q) {
                    return W8 && q.expert >= 0 ? early(q, done, Form<W8, false>()) : early(q, done, Form<false, false>());
                }))
                break;
        return met;
    };
    const int done = early_pieces(true, 0);
    if (!mbar_wait(smem_u32(&bars.routed), 0, &bars.abort_flag, p.status)) {
        wait_copies();
        return;
    }
    if (done < start.stages) early_pieces(false, done);
    wait_previous_kernel();
    Ring ring = start;
    int turn = producer;
    auto rest = [&](const Piece& q, auto form) {
        typedef decltype(form) F;
        const int depth = depth_of(q), n = F::chunks(depth);
        Feed f;
        weights_of(q, f);
        tokens_of(q, f);
        int c = turn;
        for (; c < n && ring.round == 0 && ring.at + c < ring.stages; c += kProducers) {   // the weights are on their way
            copy_tokens<F>(ring.base + (ring.at + c) * ring.stage_bytes, f, c * F::kChunk, min(F::kChunk, depth - c * F::kChunk), lane);
            arrive_when_copied(ring.full + 8 * (ring.at + c));
        }
        const bool ok = produce<F, false>(ring, &bars.abort_flag, p.status, f, c, depth, p.token_cap, lane);
        turn = (turn - n) & (kProducers - 1);
        ring.next_piece(n);
        return ok;
    };
    for (int i = 0; i < slice.pieces; ++i)
        if (!for_experts(p, r, slice.row(i), slice.row(i + 1) - slice.row(i), false, [&](const Piece& q) {
                return W8 && q.expert >= 0 ? rest(q, Form<W8, false>()) : rest(q, Form<false, false>());
            }))
            break;
    wait_copies();
}

template <bool W8>
__global__ void __launch_bounds__(kThreads, 2) moe_down_kernel(const Decode p) {
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ Bars bars;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const RowSlice slice(p.hidden_size, kRows, blockIdx.x, gridDim.x);   // of the output's columns
    Ring ring = set_up_ring(bars, smem, p.stage_bytes, p.stages, kConsumerThreads);
    Deposit sums;
    sums.scratch = reinterpret_cast<float*>(smem + p.stages * p.stage_bytes);
    float* out = sums.scratch + deposit_floats<1>();   // [token][row of the piece]
    const int values = p.tokens * kRows;
    const Routing r = carve_routing(reinterpret_cast<uint8_t*>(out + values), p.experts, p.tokens * p.topk);
    if (warp >= kConsumers && warp != kFinisher) {
        produce_down<W8>(p, r, slice, ring, bars, warp - kConsumers, lane);
        return;
    }
    auto depth_of = [&](const Piece& q) { return q.expert < 0 ? p.shared_intermediate : p.intermediate; };
    auto chunks_of = [&](const Piece& q) {
        return W8 && q.expert >= 0 ? Form<W8, false>::chunks(depth_of(q)) : Form<false, false>::chunks(depth_of(q));
    };
    const bool finisher = warp == kFinisher;
    const int worker = finisher ? kConsumerThreads + lane : threadIdx.x;   // of the consumers and the finisher
    if (!finisher) {
        find_experts(p, r);
        mbar_arrive(smem_u32(&bars.routed));
    }
    int turn = warp;
    for (int i = 0; i < slice.pieces; ++i) {
        for (int k = worker; k < values; k += kConsumerThreads + 32) out[k] = 0.0f;
        asm volatile("bar.sync 2, %0;" ::"n"(kConsumerThreads + 32) : "memory");
        const int row0 = slice.row(i), count = slice.row(i + 1) - row0;
        if (finisher) {
            for_experts(p, r, row0, count, false, [&](const Piece& q) {
                const int slots = min(chunks_of(q), kConsumers);
                collect(sums, bars, p.status, slots);
                for (int k = lane; k < kRows * q.tokens; k += 32) {   // a token is listed once
                    const int row = k & (kRows - 1), c = k / kRows;
                    float* at = out + (q.expert < 0 ? q.from + c : r.token[q.from + c]) * kRows + row;
                    float v = sum_of<1>(sums, slots, row, c);
                    if (W8 && q.expert >= 0) v *= __ldcg(p.hidden_scale + r.list[q.from + c]);
                    *at = fmaf(q.expert < 0 ? 1.0f : r.weights[q.from + c], v, *at);
                }
                collected(sums, bars, lane);
                return true;
            });
        } else {
            for_experts(p, r, row0, count, false, [&](const Piece& q) {
                const bool w8 = W8 && q.expert >= 0;
                const int depth = depth_of(q), n = chunks_of(q), tiles = (q.tokens + 7) >> 3, slot = turn;
                if (slot < n) {
                    float acc[1][4];
                    clear(acc);
                    for (int c = slot; c < n; c += kConsumers) {
                        if (w8) consume<W8, false, 1>(ring, smem, &bars.abort_flag, p.status, c, depth, tiles, p.token_cap, lane, acc);
                        else consume<false, false, 1>(ring, smem, &bars.abort_flag, p.status, c, depth, tiles, p.token_cap, lane, acc);
                    }
                    deposit<1>(sums, bars, p.status, acc, slot, tiles, lane);
                }
                ++sums.piece;
                ring.next_piece(n);
                turn = (turn - n) & (kConsumers - 1);
                return true;
            });
        }
        asm volatile("bar.sync 2, %0;" ::"n"(kConsumerThreads + 32) : "memory");
        wait_previous_kernel();   // its word on how it went
        const bool bad = p.status != nullptr && *reinterpret_cast<volatile uint32_t*>(p.status) != 0;
        for (int k = worker; k < values; k += kConsumerThreads + 32) {
            const int row = k & (kRows - 1), token = k / kRows;
            if (row < count)
                p.out[static_cast<long long>(token) * p.hidden_size + row0 + row] = __float2bfloat16(bad ? __uint_as_float(0x7FC00000u) : out[k]);
        }
        asm volatile("bar.sync 2, %0;" ::"n"(kConsumerThreads + 32) : "memory");
    }
}

}  // namespace
}  // namespace mok

#include "moe_decode_wide.cuh"

namespace mok {
namespace {

// ---------------------------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------------------------
constexpr int kSmemPerSm = 228 * 1024, kSmemPerBlock = 227 * 1024, kStatic = 1024 + 384;   // reserved per block + barriers
static_assert(sizeof(Bars) <= 384, "");
// Two blocks of a kernel share an SM when each takes half of the shared memory.
constexpr int kHalf = kSmemPerSm / 2 - kStatic;

int stage_bytes(int tokens, bool w8) {   // the shared expert is bf16 in either case
    const int a = Form<false, false>::stage_bytes(tokens), b = w8 ? Form<true, false>::stage_bytes(tokens) : 0;
    return a > b ? a : b;
}
// Shared memory beside the ring.
int gate_up_rest(const Decode& p) { return deposit_floats<1>() * 4 + routing_bytes(p.experts, p.tokens * p.topk); }
int down_rest(const Decode& p) { return gate_up_rest(p) + p.tokens * kRows * 4; }

// Whether tokens that share experts are worth the coarser tiles of the wide form.  Few-token form against wide form, us:
//   tokens                                                      1         4         8        14        64       256
//   128 experts, K 8, hidden 2048, experts of 768           31/31     68/66    111/98   147/131   255/199   468/232
//     8-bit                                                 30/32     58/56     85/75   122/105   242/159   588/234
//   32 of 256, K 8, hidden 7168, experts of 2048            33/45     45/48   121/131   172/180   414/399   736/455
//     8-bit                                                 39/46     73/83     58/58   127/123   343/234   568/316
//   8 experts, K 2, hidden 4096, experts of 14336         121/147   225/227   430/420   434/423   806/448  2581/969
//     8-bit                                                80/114   200/251   258/253   400/288   746/381  2298/857
//   16 experts, K 4, hidden 4096, experts of 1536           41/42     82/84     90/98   102/108   200/122   662/256
//     8-bit                                                 34/38     57/62     77/76    101/85   210/110   681/231
// A rule of the tokens alone: where the chosen experts have fewer units of 64 or 128 rows than there are SMs, the wide form loses up to
// a fourth (8 and 16 tokens in bf16, hidden 7168, 8 experts of 128: 36/42 and 34/44; hidden 4096, 2 experts of 256: 22/28 and 24/28)
// and is level or ahead from 24 to 32 tokens on (60/48 and 34/34 at 32).
constexpr int kWideFrom = 8;   // tokens

// Tokens of a stage, and the bytes that follow from it; false: nothing fits (no call of fewer than kWideFrom tokens).  The ring has 8 stages,
// so that every consumer keeps its own, and half of the shared memory: two blocks an SM hide each other's latency, hidden 4096, 8
// experts of 14336, 4 tokens 370 -> 327 us.  An expert that more tokens chose is read more than once (from L2 after the first time).
bool plan(Decode& p, bool w8) {
    p.stages = kConsumers;
    const int few = w8 ? 3 : 6;
    for (int cap = p.tokens < few ? p.tokens : few; cap > 0; --cap) {
        p.token_cap = cap;
        p.stage_bytes = stage_bytes(cap, w8);
        if (kConsumers * p.stage_bytes + down_rest(p) <= kHalf) return true;
    }
    return false;
}

template <typename Kernel>
int launch_decode(Kernel kernel, const char* name, int (&ready)[16], const Decode& p, int blocks, int smem, cudaStream_t stream) {
    int dev = 0;
    MOK_CUDA_CHECK(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 16) return MOK_ERR_UNSUPPORTED;
    if (ready[dev] == 0) {
        MOK_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemPerBlock - kStatic));
        // all of it as shared memory: a partition that just fits one kernel keeps the other off the SM
        MOK_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));
        ready[dev] = 1;
    }
    return launch_early(kernel, name, dim3(blocks * sm_count()), kThreads, smem, stream, p);
}

template <bool W8>
int run_few(const Decode& p, cudaStream_t stream) {
    static int gate_up_ready[16] = {0}, down_ready[16] = {0};
    const int ring = p.stages * p.stage_bytes;
    if (W8) MOK_TRY(launch_early(to_half_kernel<false>, "to_half_kernel", dim3(p.tokens), 256, 0, stream, p));
    MOK_TRY(launch_decode(moe_gate_up_kernel<W8>, "moe_gate_up_kernel", gate_up_ready, p, 2, ring + gate_up_rest(p), stream));
    if (W8) MOK_TRY(launch_early(to_half_kernel<true>, "to_half_kernel", dim3(p.tokens * p.topk), 256, 0, stream, p));
    // Two blocks an SM where each has 12 of the output's columns or more, else one with twice the stages: hidden 2048, 8 tokens of 128
    // experts 112 instead of 117 us.
    const int blocks = p.hidden_size >= 12 * 2 * sm_count() ? 2 : 1;
    Decode q = p;
    if (blocks == 1) q.stages = 2 * kConsumers;
    return launch_decode(moe_down_kernel<W8>, "moe_down_kernel", down_ready, q, blocks, q.stages * p.stage_bytes + down_rest(p), stream);
}

template <bool W8, bool DOWN>
int launch_wide(const Decode& p, int smem, cudaStream_t stream) {
    static int ready[16] = {0};
    int dev = 0;
    MOK_CUDA_CHECK(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 16) return MOK_ERR_UNSUPPORTED;
    if (ready[dev] == 0) {
        MOK_CUDA_CHECK(cudaFuncSetAttribute(moe_wide_kernel<W8, DOWN>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemPerBlock - kStatic));
        ready[dev] = 1;
    }
    return launch_early(moe_wide_kernel<W8, DOWN>, "moe_wide_kernel", dim3(sm_count()), kWideThreads, smem, stream, p);
}
template <bool W8>
int run_wide(Decode p, cudaStream_t stream) {
    p.token_cap = kWideTokens;
    p.stage_bytes = W8 ? WideForm<true>::kStageBytes : WideForm<false>::kStageBytes;   // the shared expert's, in bf16, is the smaller one
    const int routing = routing_bytes(p.experts, p.tokens * p.topk);
    p.stages = (kSmemPerBlock - kStatic - routing) / p.stage_bytes;
    if (p.stages > 8) p.stages = 8;
    const int smem = p.stages * p.stage_bytes + routing;
    if (W8) MOK_TRY(launch_early(to_half_kernel<false>, "to_half_kernel", dim3(p.tokens), 256, 0, stream, p));
    MOK_TRY((launch_wide<W8, false>(p, smem, stream)));
    if (W8) MOK_TRY(launch_early(to_half_kernel<true>, "to_half_kernel", dim3(p.tokens * p.topk), 256, 0, stream, p));
    MOK_TRY((launch_wide<W8, true>(p, smem, stream)));
    return launch_early(moe_wide_sum_kernel, "moe_wide_sum_kernel", dim3((p.hidden_size + 1023) / 1024, p.tokens), 256, 0, stream, p);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace mok

// hidden rows of the routes, of the shared expert; 8-bit experts: tokens in f16 and the scales; wide form: the experts' parts
extern "C" int64_t mok_moe_decode_scratch_bytes(int num_tokens, int topk, int hidden, int intermediate, int shared_intermediate, int fp8) {
    if (num_tokens <= 0 || topk <= 0 || hidden <= 0 || intermediate <= 0 || shared_intermediate < 0) return 0;
    const int64_t tokens = num_tokens, routes = tokens * topk;
    const int64_t rows = 2 * (routes * intermediate + tokens * shared_intermediate) + (fp8 ? 2 * tokens * hidden + 4 * (tokens + routes) : 0);
    if (num_tokens < mok::kWideFrom) return rows;
    return (rows + 15) / 16 * 16 + 4 * hidden * (routes + (shared_intermediate > 0 ? tokens : 0));
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
        !aligned16(w_shared_down) || !aligned16(scratch) || !aligned16(out) || x_stride % 8 != 0 || x_stride < 0)
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
    p.x_half = reinterpret_cast<__half*>(p.hidden_shared + static_cast<long long>(num_tokens) * shared_intermediate);
    p.x_scale = reinterpret_cast<float*>(p.x_half + static_cast<long long>(num_tokens) * hidden);
    p.hidden_scale = p.x_scale + num_tokens;
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
    if (num_tokens >= kWideFrom) {
        p.parts = reinterpret_cast<float*>(static_cast<uint8_t*>(scratch) +
                                           mok_moe_decode_scratch_bytes(num_tokens, topk, hidden, intermediate, shared_intermediate, w8) -
                                           4LL * hidden * (static_cast<long long>(num_tokens) * topk + (shared ? num_tokens : 0)));
        return w8 ? run_wide<true>(p, s) : run_wide<false>(p, s);
    }
    if (!plan(p, w8)) return MOK_ERR_TOO_LARGE;
    return w8 ? run_few<true>(p, s) : run_few<false>(p, s);
}
