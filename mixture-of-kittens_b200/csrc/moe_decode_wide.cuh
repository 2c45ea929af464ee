// The layer for tokens that share experts: the same sums in the same order as in moe_decode.cu, over tiles of 128 weight rows x 64
// tokens.  There a stage holds 16 weight rows and six tokens at most (three with 8-bit experts): every six tokens of an expert cost a
// pass over its weights, and copies of the tokens a third of the bytes that an SM takes in.  Here it is one pass for 64 tokens.  Both
// are bound by reading the weights in bf16: 32 tokens, 8 of 128 experts, hidden 2048, experts of 768 (with its router) 226 -> 170 to
// 186 us, 90 to 93 % of the measured HBM rate for the 104 to 116 experts that were chosen.  In 8 bits the conversions and products of
// eight consumer warps take longer than the bytes: 64 tokens, 32 of 256 experts, hidden 7168, experts of 2048 310 -> 225 to 258 us,
// 58 to 68 % (17 to 22 experts chosen, and a shared one), 298 us with balanced routes, 69 %.  Experts of more than 64 tokens are
// read again for the others: 256 tokens, 2 of 8 experts of 14336, 969 us for 437 us of weights.  Tiles are coarse, so a few tokens
// are better off there (see kWideFrom).
//
// A block has four producer warps, which copy 128 bytes of each row per stage, and eight consumer warps of 16 rows x all tokens (up
// to 16) or 32 rows x half of the tokens each.  They use mma.sync, which takes a few percent of the time; tcgen05 would add the
// products of a tile in another order.  The few-token form cuts K into chunks that eight warps take in turn and adds the warps' sums
// at the end.  Here every warp walks all of K, the chunks of one such warp after those of another, and adds up where that one's end:
// a token's result is the same to the bit in either form.
//
// The experts' parts of the output leave in fp32 and a last kernel adds them, shared expert first, then experts by number.
#pragma once

namespace mok {
namespace {

constexpr int kWideRows = 128, kWideTokens = 64;
constexpr int kWideThreads = kConsumerThreads + kProducers * 32;
constexpr int kWideTokensAt = kWideRows * 128;   // in a stage, behind the weights

template <bool W8>
struct WideForm {
    static constexpr int kDepth = W8 ? 128 : 64;   // elements of k per stage
    static constexpr int kTokenBytes = 2 * kDepth;
    static constexpr int kScales = kWideRows * 128 + kWideTokens * kTokenBytes;   // of the gate (down) rows and of the up rows
    static constexpr int kStageBytes = kScales + (W8 ? 16 : 0);
    static constexpr int kChunk = Form<W8, false>::kChunk;
};

template <bool B>
struct Flag {
    static constexpr bool value = B;
};

struct WideBars {
    uint64_t full[8], empty[8], routed;
    int abort_flag;
};

// A unit of work: 128 weight rows (64 of the gate and the same 64 of up) from `row` on, and tokens [from, from + tokens) of the
// expert's list.
struct Unit {
    int expert, row, from, tokens;
};
// Block b takes units b, b + gridDim.x, ..  A unit of the shared expert, which is bf16, takes the time of two of 8-bit experts: with
// W8 its block's next turn is left out.
template <bool W8, bool DOWN>
struct Units {
    int shared, shared_passes, tiles, total, left_out;
    static constexpr int kStep = DOWN ? kWideRows : kWideRows / 2;
    __device__ __forceinline__ void count_shared(const Decode& p) {
        shared_passes = (p.tokens + kWideTokens - 1) / kWideTokens;
        shared = p.shared_gate == nullptr ? 0 : ((DOWN ? p.hidden_size : p.shared_intermediate) + kStep - 1) / kStep * shared_passes;
        tiles = ((DOWN ? p.hidden_size : p.intermediate) + kStep - 1) / kStep;
    }
    __device__ __forceinline__ void count_routed(const Routing& r) {
        total = shared + r.passes[*r.num_active] * tiles;
        left_out = W8 && shared <= static_cast<int>(gridDim.x) && total > static_cast<int>(gridDim.x) ? shared : 0;
        total += left_out;
    }
    // Unit u; no tokens: a turn that is left out.  The passes over a tile come one after the other: the later ones find its weights in
    // L2.
    __device__ __forceinline__ Unit get(const Decode& p, const Routing& r, int u) const {
        Unit q;
        if (u < shared) {
            q.expert = -1;
            q.row = u / shared_passes * kStep;
            q.from = u % shared_passes * kWideTokens;
            q.tokens = min(kWideTokens, p.tokens - q.from);
            return q;
        }
        if (u >= static_cast<int>(gridDim.x)) {
            u -= left_out;
            if (u < static_cast<int>(gridDim.x)) {
                q.tokens = 0;
                return q;
            }
        }
        u -= shared;
        int a = 0;
        for (int n = *r.num_active; n - a > 1;) {
            const int mid = (a + n) >> 1;
            if (r.passes[mid] * tiles <= u) a = mid;
            else n = mid;
        }
        u -= r.passes[a] * tiles;
        const int passes = r.passes[a + 1] - r.passes[a], tile = passes == 1 ? u : u / passes;
        q.expert = r.active[a];
        q.row = tile * kStep;
        q.from = r.begin[a] + (u - tile * passes) * kWideTokens;
        q.tokens = min(kWideTokens, r.begin[a + 1] - q.from);
        return q;
    }
};

// Lists in the order of routes: an expert's passes may be different blocks' work, and find_experts() leaves every block an order of
// its own.  The consumer threads; only where an expert has more than one pass.
__device__ __forceinline__ void order_lists(const Decode& p, const Routing& r) {
    const int active = *r.num_active, total = r.begin[active];
    if (r.passes[active] == active) return;
    uint16_t* ordered = r.expert;   // not needed any more
    for (int i = threadIdx.x; i < total; i += kConsumerThreads) {
        int a = 0;
        for (int n = active; n - a > 1;) {
            const int mid = (a + n) >> 1;
            if (r.begin[mid] <= i) a = mid;
            else n = mid;
        }
        const int first = r.begin[a], last = r.begin[a + 1], mine = r.list[i];
        int before = 0;
        for (int k = first; k < last; ++k) before += r.list[k] < mine;
        ordered[first + before] = static_cast<uint16_t>(mine);
    }
    consumer_barrier();
    for (int i = threadIdx.x; i < total; i += kConsumerThreads) {
        r.list[i] = ordered[i];
        r.token[i] = static_cast<uint8_t>(ordered[i] / p.topk);
    }
    consumer_barrier();
}

// f(k, left) for every stage of a unit, k in the order of the sums (see above): chunks 0, 8, 16 .., then 1, 9 ..; next() between two
// of these.
template <bool W8, typename F, typename G>
__device__ __forceinline__ bool walk_depth(int depth, F&& f, G&& next) {
    typedef WideForm<W8> W;
    const int chunks = (depth + W::kChunk - 1) / W::kChunk;
    for (int s = 0; s < min(chunks, kConsumers); ++s) {
        for (int c = s; c < chunks; c += kConsumers) {
            const int end = min((c + 1) * W::kChunk, depth);
            for (int k = c * W::kChunk; k < end; k += W::kDepth)
                if (!f(k, min(W::kDepth, end - k))) return false;
        }
        next();
    }
    return true;
}

// 16-byte unit u of a row lies at u ^ turn(row): the lanes (g, t) of a load then use every bank once.
template <bool W8>
__device__ __forceinline__ int weight_turn(int row) { return W8 ? (row & 3) << 1 : (row & 1) << 2; }
__device__ __forceinline__ int token_turn(int token) { return (token & 1) << 2; }

// The copies of one unit by producer thread (producer, lane), which has rows j + 16 i and tokens j + 16 i, and 16 bytes of each.
// EARLY: weights only, into the empty ring until it is full (false); `early` counts these stages, whose tokens follow.
template <bool W8, bool DOWN, bool EARLY>
__device__ __forceinline__ bool produce_unit(const Decode& p, const Routing& r, const Unit& q, WideBars& bars, uint32_t base, int& early, int& stage,
                                             uint32_t& phase, int producer, int lane) {
    typedef WideForm<W8> W;
    const bool shared = q.expert < 0;
    const int j = producer * 4 + (lane >> 3), u = lane & 7;
    const int rows = DOWN ? p.hidden_size : shared ? p.shared_intermediate : p.intermediate;
    const int depth = DOWN ? (shared ? p.shared_intermediate : p.intermediate) : p.hidden_size;
    const long long row_bytes = static_cast<long long>(depth) * (W8 ? 1 : 2);
    const uint8_t* w;
    if (DOWN) w = shared ? reinterpret_cast<const uint8_t*>(p.shared_down) : p.down;
    else if (j < 8) w = shared ? reinterpret_cast<const uint8_t*>(p.shared_gate) : p.gate;
    else w = shared ? reinterpret_cast<const uint8_t*>(p.shared_up) : p.up;
    w += ((shared ? 0 : static_cast<long long>(q.expert) * rows) + q.row + (DOWN ? j : j & 7)) * row_bytes + u * 16;
    const long long step = (DOWN ? 16 : 8) * row_bytes;
    const int pieces = DOWN ? min(8, (rows - q.row) / 16) : 8;   // 64 rows at least; what is missing is not stored
    const uint8_t* token[kWideTokens / 16];
#pragma unroll
    for (int i = 0; i < (EARLY ? 0 : kWideTokens / 16); ++i) {
        const int at = q.from + min(j + 16 * i, q.tokens - 1);
        const void* row;
        if (DOWN) row = shared ? p.hidden_shared + static_cast<long long>(at) * depth : p.hidden + static_cast<long long>(r.list[at]) * depth;
        else if (W8) row = p.x_half + static_cast<long long>(r.token[at]) * depth;
        else row = p.x + (shared ? at : r.token[at]) * p.x_stride;
        token[i] = static_cast<const uint8_t*>(row) + u * 16;
    }
    const float* scale = nullptr;
    if (W8 && lane == 0 && (producer == 0 || (!DOWN && producer == 2))) {
        const int blocks = (depth + 127) / 128;
        scale = (DOWN ? p.down_scales : producer == 0 ? p.gate_scales : p.up_scales) +
                (static_cast<long long>(q.expert) * ((rows + 127) / 128) + q.row / 128) * blocks;
    }
    const uint32_t weight_at = j * 128 + ((u ^ weight_turn<W8>(j)) << 4);
    const uint32_t token_at = kWideTokensAt + j * W::kTokenBytes + ((u ^ token_turn(j)) << 4);
    return walk_depth<W8>(depth, [&](int k, int left) {
        if (EARLY) {
            if (early == p.stages) return false;
        } else if (!mbar_wait(smem_u32(&bars.empty[stage]), phase ^ 1u, &bars.abort_flag, p.status)) {
            return false;
        }
        const uint32_t to = base + (EARLY ? early : stage) * p.stage_bytes;
        const bool weights = EARLY || early == 0;
        if (weights && (!W8 || u * 16 < left)) {
            const uint8_t* from = w + static_cast<long long>(k) * (W8 ? 1 : 2);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (i < pieces) copy16(to + weight_at + i * 16 * 128, from);
                from += step;
            }
        }
        if (W8 && weights && scale != nullptr) copy4(to + W::kScales + (producer >> 1) * 4, scale + k / 128);
        if (EARLY) {
            ++early;
            return true;
        }
#pragma unroll
        for (int i = 0; i < kWideTokens / 16; ++i) {
            if (j + 16 * i < q.tokens) {
                copy16(to + token_at + i * 16 * W::kTokenBytes, token[i] + k * 2);
                if (W8 && left == 128) copy16(to + token_at + i * 16 * W::kTokenBytes + 128, token[i] + k * 2 + 128);
            }
        }
        arrive_when_copied(smem_u32(&bars.full[stage]));
        if (!weights) --early;
        if (++stage == p.stages) { stage = 0; phase ^= 1u; }
        return true;
    }, [] {});
}

// sums += SLICES x 32 elements of k of a stage: M x 16 rows from `row` on x TILES x 8 tokens.
template <bool W8, int SLICES, int M, int TILES>
__device__ __forceinline__ void wide_products(const uint8_t* stage, int row, int token, int lane, float (&sums)[2][4][4]) {
    typedef WideForm<W8> W;
    const int g = lane >> 2, t = lane & 3;
    const uint8_t* weights = stage + (row + g) * 128;
    const uint8_t* tokens = stage + kWideTokensAt + (token + g) * W::kTokenBytes;
#pragma unroll
    for (int k = 0; k < SLICES; ++k) {
        uint32_t lo[2][4], hi[2][4];
#pragma unroll
        for (int m = 0; m < M; ++m) {
            if (W8) {
                const uint8_t* at = weights + m * 16 * 128 + (((k * 2 + (t >> 1)) ^ weight_turn<W8>(g)) << 4) + (t & 1) * 8;
                const uint2 l = *reinterpret_cast<const uint2*>(at), h = *reinterpret_cast<const uint2*>(at + 8 * 128);
                lo[m][0] = e4m3x2_to_f16x2(l.x); lo[m][1] = e4m3x2_to_f16x2(l.x >> 16);
                lo[m][2] = e4m3x2_to_f16x2(l.y); lo[m][3] = e4m3x2_to_f16x2(l.y >> 16);
                hi[m][0] = e4m3x2_to_f16x2(h.x); hi[m][1] = e4m3x2_to_f16x2(h.x >> 16);
                hi[m][2] = e4m3x2_to_f16x2(h.y); hi[m][3] = e4m3x2_to_f16x2(h.y >> 16);
            } else {
                const uint8_t* at = weights + m * 16 * 128 + (((k * 4 + t) ^ weight_turn<W8>(g)) << 4);
                const uint4 l = *reinterpret_cast<const uint4*>(at), h = *reinterpret_cast<const uint4*>(at + 8 * 128);
                lo[m][0] = l.x; lo[m][1] = l.y; lo[m][2] = l.z; lo[m][3] = l.w;
                hi[m][0] = h.x; hi[m][1] = h.y; hi[m][2] = h.z; hi[m][3] = h.w;
            }
        }
#pragma unroll
        for (int n = 0; n < TILES; ++n) {
            const uint4 v = *reinterpret_cast<const uint4*>(tokens + n * 8 * W::kTokenBytes + (((k * 4 + t) ^ token_turn(g)) << 4));
#pragma unroll
            for (int m = 0; m < M; ++m) {
                if (W8) {
                    mma_f16(sums[m][n], lo[m][0], hi[m][0], lo[m][1], hi[m][1], v.x, v.y);
                    mma_f16(sums[m][n], lo[m][2], hi[m][2], lo[m][3], hi[m][3], v.z, v.w);
                } else {
                    mma_bf16(sums[m][n], lo[m][0], hi[m][0], lo[m][1], hi[m][1], v.x, v.y);
                    mma_bf16(sums[m][n], lo[m][2], hi[m][2], lo[m][3], hi[m][3], v.z, v.w);
                }
            }
        }
    }
}

__device__ __forceinline__ void clear(float (&v)[2][4][4]) {
#pragma unroll
    for (int m = 0; m < 2; ++m) stream::clear(v[m]);
}

// The sums of one unit for a warp's M x 16 rows and TILES x 8 tokens.
template <bool W8, bool DOWN, int M, int TILES>
__device__ __forceinline__ void consume_unit(const Decode& p, WideBars& bars, const uint8_t* ring, int& stage, uint32_t& phase, int depth, int row, int token,
                                             int lane, float (&total)[2][4][4]) {
    typedef WideForm<W8> W;
    float acc[2][4][4];
    clear(acc);
    walk_depth<W8>(depth, [&](int, int left) {
        // a wait that runs out is reported in the status word, and the warp goes on with what is there
        mbar_wait(smem_u32(&bars.full[stage]), phase, &bars.abort_flag, p.status);
        const uint8_t* at = ring + stage * p.stage_bytes;
        if (W8) {
            float part[2][4][4];
            clear(part);
            const float lo = *reinterpret_cast<const float*>(at + W::kScales);
            const float hi = DOWN ? lo : *reinterpret_cast<const float*>(at + W::kScales + 4);
            if (left == 128) wide_products<W8, 4, M, TILES>(at, row, token, lane, part);
            else wide_products<W8, 2, M, TILES>(at, row, token, lane, part);
#pragma unroll
            for (int m = 0; m < M; ++m)
#pragma unroll
                for (int n = 0; n < TILES; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[m][n][i] = fmaf(part[m][n][i], i < 2 ? lo : hi, acc[m][n][i]);
        } else {
            wide_products<W8, 2, M, TILES>(at, row, token, lane, acc);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&bars.empty[stage]));
        if (++stage == p.stages) { stage = 0; phase ^= 1u; }
        return true;
    }, [&] {
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
            for (int n = 0; n < TILES; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    total[m][n][i] += acc[m][n][i];
                    acc[m][n][i] = 0.0f;
                }
    });
}

template <bool W8, bool DOWN>
__global__ void __launch_bounds__(kWideThreads, 1) moe_wide_kernel(const Decode p) {
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ WideBars bars;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t base = smem_u32(smem);
    if (threadIdx.x == 0) {
        for (int s = 0; s < p.stages; ++s) {
            mbar_init(smem_u32(&bars.full[s]), kProducers * 32);
            mbar_init(smem_u32(&bars.empty[s]), kConsumers);
        }
        mbar_init(smem_u32(&bars.routed), kConsumerThreads);
        bars.abort_flag = 0;
        mbar_fence_init();
    }
    __syncthreads();
    const Routing r = carve_routing(smem + p.stages * p.stage_bytes, p.experts, p.tokens * p.topk);
    Units<W8, DOWN> units;
    units.count_shared(p);
    // The down kernel has weights to fetch and experts to find while the last blocks before it finish; weights and routes are no
    // earlier kernel's of this call, and the gate / up kernel has waited for those of earlier ones.
    if (!DOWN) wait_previous_kernel();
    allow_next_kernel();
    int stage = 0;
    uint32_t phase = 0;
    if (warp >= kConsumers) {
        const int producer = warp - kConsumers;
        int early = 0;
        auto produce = [&](auto when) {
            constexpr bool kEarly = decltype(when)::value;
            int u = blockIdx.x;
            for (; u < units.shared; u += gridDim.x)   // these need no routing
                if (!produce_unit<false, DOWN, kEarly>(p, r, units.get(p, r, u), bars, base, early, stage, phase, producer, lane)) return;
            if (!mbar_wait(smem_u32(&bars.routed), 0, &bars.abort_flag, p.status)) return;
            units.count_routed(r);
            for (; u < units.total; u += gridDim.x) {
                const Unit q = units.get(p, r, u);
                if (q.tokens > 0 && !produce_unit<W8, DOWN, kEarly>(p, r, q, bars, base, early, stage, phase, producer, lane)) return;
            }
        };
        if (DOWN) {
            produce(Flag<true>());
            wait_previous_kernel();
        }
        produce(Flag<false>());
        wait_copies();
        return;
    }
    find_experts(p, r);
    order_lists(p, r);
    mbar_arrive(smem_u32(&bars.routed));
    units.count_routed(r);
    if (DOWN) wait_previous_kernel();
    float* scales = r.weights;   // W8: of the lists' token or hidden rows; the weights wait for the last kernel
    if (W8) {
        for (int i = threadIdx.x; i < r.begin[*r.num_active]; i += kConsumerThreads)
            scales[i] = __ldcg(DOWN ? p.hidden_scale + r.list[i] : p.x_scale + r.token[i]);
        consumer_barrier();
    }
    const int g = lane >> 2, t = lane & 3;
    for (int u = blockIdx.x; u < units.total; u += gridDim.x) {
        const Unit q = units.get(p, r, u);
        if (q.tokens == 0) continue;
        const bool shared = q.expert < 0, w8 = W8 && !shared;
        const int depth = DOWN ? (shared ? p.shared_intermediate : p.intermediate) : p.hidden_size;
        // Up to 16 tokens: 16 rows a warp and all tokens.  More: 32 rows and half of the tokens (the last tile may hold nobody's).
        const int tiles = (q.tokens + 7) >> 3;
        const bool few = tiles <= 2;
        const int mine = few ? tiles : (tiles + 1) >> 1;
        const int row = few ? warp * 16 : (warp & 3) * 32, token = few ? 0 : (warp >> 2) * mine * 8;
        float total[2][4][4];
        clear(total);
#define MOK_CONSUME(M, TILES)                                                                                                               \
    do {                                                                                                                                    \
        if (w8) consume_unit<W8, DOWN, M, TILES>(p, bars, smem, stage, phase, depth, row, token, lane, total);     \
        else consume_unit<false, DOWN, M, TILES>(p, bars, smem, stage, phase, depth, row, token, lane, total);     \
    } while (0)
        if (tiles == 1) MOK_CONSUME(1, 1);
        else if (tiles == 2) MOK_CONSUME(1, 2);
        else if (mine == 2) MOK_CONSUME(2, 2);
        else if (mine == 3) MOK_CONSUME(2, 3);
        else MOK_CONSUME(2, 4);
#undef MOK_CONSUME
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            if (n >= mine) break;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int c = token + n * 8 + 2 * t + i;
                if (c >= q.tokens) continue;
                const int at = q.from + c;
                if (DOWN) {
                    const float scale = w8 ? scales[at] : 1.0f;
                    float* out = p.parts + static_cast<long long>(shared ? p.tokens * p.topk + at : r.list[at]) * p.hidden_size + q.row + row + g;
#pragma unroll
                    for (int m = 0; m < 2; ++m) {
                        if ((m == 1 && few) || q.row + row + 16 * m >= p.hidden_size) continue;   // 64 rows in all, or 128
                        out[16 * m] = w8 ? total[m][n][i] * scale : total[m][n][i];
                        out[16 * m + 8] = w8 ? total[m][n][2 + i] * scale : total[m][n][2 + i];
                    }
                } else {
                    const float scale = w8 ? scales[at] : 1.0f;
                    bf16* out = (shared ? p.hidden_shared + static_cast<long long>(at) * p.shared_intermediate
                                        : p.hidden + static_cast<long long>(r.list[at]) * p.intermediate) + q.row + row / 2 + g;
#pragma unroll
                    for (int m = 0; m < 2; ++m) {
                        if (m == 1 && few) continue;
                        out[8 * m] = hidden_value(p, w8 ? total[m][n][i] * scale : total[m][n][i],
                                                  w8 ? total[m][n][2 + i] * scale : total[m][n][2 + i]);
                    }
                }
            }
        }
    }
}

// out[t] = shared part + sum over t's experts, by number, of weight * part: a block per token and 1024 columns.
__global__ void __launch_bounds__(256) moe_wide_sum_kernel(const Decode p) {
    __shared__ int route[kMaxTopk], used;
    __shared__ float weight[kMaxTopk];
    const int token = blockIdx.y, lane = threadIdx.x;
    wait_previous_kernel();
    if (threadIdx.x < 32) {
        const int i = token * p.topk + lane;
        uint32_t e = kNobody;
        float w = 0.0f;
        if (lane < p.topk) {
            const uint32_t local = static_cast<uint32_t>(__ldcg(p.routes + i)) - static_cast<uint32_t>(p.first_expert);
            if (local < static_cast<uint32_t>(p.experts)) e = local;
            w = __ldcg(p.route_weights + i);
        }
        const uint32_t same = __match_any_sync(0xffffffffu, e == kNobody ? 0x80000000u | lane : e);
        const bool first = e != kNobody && (same & ((1u << lane) - 1u)) == 0;
        float sum = w;   // of the routes to that expert, in order
        for (int l = 0; l < p.topk; ++l) {
            const float other = __shfl_sync(0xffffffffu, w, l);
            if (l > lane && (same >> l & 1u)) sum += other;
        }
        int rank = 0;
        const uint32_t firsts = __ballot_sync(0xffffffffu, first);
        for (uint32_t left = firsts; left != 0; left &= left - 1u) rank += __shfl_sync(0xffffffffu, e, __ffs(left) - 1) < e;
        if (first) {
            route[rank] = i;
            weight[rank] = sum;
        }
        if (lane == 0) used = __popc(firsts);
    }
    __syncthreads();
    const bool bad = p.status != nullptr && *reinterpret_cast<volatile uint32_t*>(p.status) != 0;
    const int col = (blockIdx.x * 256 + threadIdx.x) * 4;
    if (col >= p.hidden_size) return;
    float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    auto add = [&](float w, long long row) {
        const float4 v = __ldcg(reinterpret_cast<const float4*>(p.parts + row * p.hidden_size + col));
        s.x = fmaf(w, v.x, s.x); s.y = fmaf(w, v.y, s.y); s.z = fmaf(w, v.z, s.z); s.w = fmaf(w, v.w, s.w);
    };
    if (p.shared_gate != nullptr) add(1.0f, static_cast<long long>(p.tokens) * p.topk + token);
#pragma unroll 4
    for (int i = 0; i < used; ++i) add(weight[i], route[i]);
    if (bad) s.x = s.y = s.z = s.w = __uint_as_float(0x7FC00000u);
    *reinterpret_cast<uint2*>(p.out + static_cast<long long>(token) * p.hidden_size + col) = make_uint2(pack_bf16x2(s.x, s.y), pack_bf16x2(s.z, s.w));
}

}  // namespace
}  // namespace mok
