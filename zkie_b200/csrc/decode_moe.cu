// decode_moe.cu -- a whole mixture-of-experts layer (build_moe of
// models/deepseek-v2-lite/src/lib.rs:252-470) for a few tokens, in two
// kernels and bit-identical to the graph's rows: router MatMul, Scale,
// StableSoftmaxIndex, Softmax, TopKSelect; per chosen expert the gate and up
// products, SiLU by lookup, ScaleVec and the down product; the gate values
// and the sum over experts; the shared experts.  Weights are held in 4 bits
// (q4.cuh), the router in two signed bytes.
//
// Work is bound by the weights' bytes, each expert that some token chose
// being read once for up to four of its tokens:
// - k_moe_up: a pair of blocks computes the logits of all experts and each
//   ranks them; the blocks share out the tiles of 16 hidden columns of the
//   shared and the chosen experts, gate and up side by side, the shared ones
//   first so that their weights are on their way before the routing is
//   known.  The activation is stored as the byte digits that the next
//   product reads;
// - k_moe_down: a pair of blocks to each 32 output columns runs over all
//   experts, half of them each, so that the rounding after each expert's
//   product and the sum over experts need no second pass over memory.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

#include "../../include/zkie2.h"
#include "common.cuh"
#include "fixed.cuh"
#include "gl64.cuh"
#include "launch.cuh"
#include "q4.cuh"

namespace cg = cooperative_groups;

namespace zk {

namespace {

constexpr uint32_t kErrDivide = 2u;
constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr uint32_t kMaxTokens = 16;  // tokens of one launch
constexpr uint32_t kMaxTop = 16;
constexpr uint32_t kMaxExperts = 256;
constexpr uint32_t kTile = 4;        // tokens of an expert taken at a time
constexpr uint32_t kMaxSlots = kMaxTokens * kMaxTop;
constexpr size_t kMaxShared = 220 * 1024;
constexpr int32_t kRouterLimit = 32639;  // two signed bytes
constexpr uint32_t kScale = 16;  // build_moe divides by 2^16 (:252-470), except in the shared experts' Projections

struct Q4Weight {
    const uint8_t* w;
    Q4Shape s;
};

// The tokens of the chosen experts, up to kTile of one expert to an item; a
// slot is token top_k + place.
struct Items {
    uint32_t n;
    uint8_t expert[kMaxSlots];
    uint8_t count[kMaxSlots];
    uint16_t first[kMaxSlots];  // into slot
    uint16_t slot[kMaxSlots];   // grouped by expert
    uint8_t token[kMaxSlots];   // of slot[i]
    int32_t score[kMaxSlots];   // a slot's softmax value
};
static_assert(sizeof(Items) % 4 == 0, "copied in words");

struct MoeArgs {
    const uint64_t* x;
    uint64_t ldx;
    uint32_t m, h, experts, top_k, etiles;
    const uint4* router;
    Q4Weight up, down, sup, sdown;  // up: gate and up, block by block side by side; down: pairs of tiles
    const uint64_t* exp_table;
    uint64_t exp_len;
    const uint64_t* silu;
    uint64_t silu_len;
    uint32_t shift;  // of the shared experts' Projections
    const uint64_t* residual;
    uint64_t ldr;
    uint64_t* out;
    uint64_t* gate_out;  // m x experts (or null)
    Items* items;
    uint8_t* act;        // the activation's digits: an item's blocks of 64, in each its tokens' four digit rows
    uint8_t* sact;       // the same of the shared experts, tokens four at a time
    uint32_t* err;
    uint32_t stride;     // bytes of a digit row of x
    uint32_t depth;      // slots of a ring of k_moe_down
};

// The router's weights (h x experts, field elements) as two signed bytes in
// blocks of 64 k and 16 experts: word q of lane (g, t) of half f and byte p
// holds byte p of rows 32 f + 8 t + 4 (q / 2) .. + 3 of expert g + 8 (q % 2).
__global__ void k_moe_router_pack(const uint64_t* __restrict__ w, uint32_t h, uint32_t experts, uint32_t blocks,
                                  uint32_t etiles, uint32_t* __restrict__ packed, uint32_t* __restrict__ err) {
    bool bad = false;
    const uint64_t total = (uint64_t)etiles * blocks * 512;
    for (uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (uint64_t)gridDim.x * blockDim.x) {
        const uint32_t q = i & 3, lane = (i >> 2) & 31, p = (i >> 7) & 1, f = (i >> 8) & 1;
        const uint32_t block = (uint32_t)((i >> 9) % blocks), tile = (uint32_t)((i >> 9) / blocks);
        const uint32_t e = tile * 16 + (lane >> 2) + 8 * (q & 1);
        uint32_t word = 0;
        for (int j = 0; j < 4; j++) {
            const uint32_t k = block * 64 + 32 * f + 8 * (lane & 3) + 4 * (q >> 1) + j;
            int64_t v = k < h && e < experts ? fx_to_i64(w[(uint64_t)k * experts + e]) : 0;
            if (v < -kRouterLimit || v > kRouterLimit) {
                bad = true;
                v = 0;
            }
            const int lo = (int)(int8_t)(uint8_t)v, hi = ((int)v - lo) / 256;
            word |= (uint32_t)(uint8_t)(p ? hi : lo) << (8 * j);
        }
        packed[i] = word;
    }
    if (bad) atomicOr(err, kErrRange);
}

// Logits of the 16 experts of tile 2 own + rank, this warp's blocks [b0, b1),
// added to sums (tokens x this block's experts); eight tokens at a time, for
// which two blocks of the router at a time are held in registers (a second
// form for two tokens: 0.4 us less for one token, 0.2 to 1.3 more for three
// to eight, whose registers it changes).
__device__ __forceinline__ void router_part(const MoeArgs& p, const uint8_t* digits, uint32_t own, uint32_t rank,
                                         uint32_t b0, uint32_t b1, const Limbs& sums, uint32_t pitch) {
    const uint32_t lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    constexpr int kHeld = 2, NT = 4;
    for (uint32_t tok0 = 0; tok0 < p.m; tok0 += 2 * NT) {
        int c[2][NT][4];
#pragma unroll
        for (int q = 0; q < 2; q++)
#pragma unroll
            for (int i = 0; i < NT; i++) c[q][i][0] = c[q][i][1] = c[q][i][2] = c[q][i][3] = 0;
        const uint8_t* from[NT];
#pragma unroll
        for (int i = 0; i < NT; i++)
            from[i] = digits + (size_t)(min(tok0 + 2 * i + (g >> 2), p.m - 1) * 4 + (g & 3)) * p.stride + 16 * t;
        for (uint32_t b = b0; b < b1; b += kHeld) {
            uint4 w[kHeld][4];  // half and byte: 00, 01, 10, 11
#pragma unroll
            for (int k = 0; k < kHeld; k++) {  // (a block past the end repeats the last, and is not used)
                const uint4* r = p.router + ((uint64_t)(2 * own + rank) * p.up.s.blocks + min(b + k, b1 - 1)) * 128 + lane;
#pragma unroll
                for (int q = 0; q < 4; q++) w[k][q] = r[32 * q];
            }
#pragma unroll
            for (int k = 0; k < kHeld; k++)
                if (b + k < b1) {
#pragma unroll
                    for (int i = 0; i < NT; i++) {
                        const uint4 x = *reinterpret_cast<const uint4*>(from[i] + (b + k) * 64);
                        mma_s8(c[0][i], w[k][0].x, w[k][0].y, w[k][0].z, w[k][0].w, x.x, x.y);
                        mma_s8(c[1][i], w[k][1].x, w[k][1].y, w[k][1].z, w[k][1].w, x.x, x.y);
                        mma_s8(c[0][i], w[k][2].x, w[k][2].y, w[k][2].z, w[k][2].w, x.z, x.w);
                        mma_s8(c[1][i], w[k][3].x, w[k][3].y, w[k][3].z, w[k][3].w, x.z, x.w);
                    }
                }
        }
#pragma unroll
        for (int i = 0; i < NT; i++) {
            const uint32_t tok = tok0 + 2 * i + (t >> 1);
            if (tok < p.m) {
#pragma unroll
                for (int q = 0; q < 2; q++) {
                    const long long v = ((long long)c[0][i][2 * q] + ((long long)c[0][i][2 * q + 1] << 8)) +
                                        (((long long)c[1][i][2 * q] << 8) + ((long long)c[1][i][2 * q + 1] << 16));
                    sums.add(tok * pitch + own * 16 + g + 8 * q, (long long)((unsigned long long)v << (16 * (t & 1))));
                }
            }
        }
    }
}

// The last warps of a block route the tokens while the others take the shared
// experts' first batch.
// Four of them, six for more than four tokens: a token is 3 us of a warp's time, the shared
// experts' batch for sixteen tokens 90 us of it.
__device__ __forceinline__ uint32_t route_warps(uint32_t m) { return m <= 4 ? 4 : 6; }
__device__ __forceinline__ void route_sync(uint32_t m) {
    asm volatile("bar.sync 1, %0;" ::"r"(route_warps(m) * 32) : "memory");
}

// One token's softmax over the experts and its top_k, by a warp: raw logits
// of the pair's two blocks (tiles of experts alternate between them).  A key
// holds an expert's value above its complement, so that the maximum is the
// first in TopKSelect's order.  EACH: experts of a lane.
template <int EACH>
__device__ __forceinline__ void route_token(const MoeArgs& p, uint32_t r, const long long* even, const long long* odd, uint32_t pitch,
                            uint32_t* s_sel, int32_t* s_score, uint32_t* s_mask) {
    const uint32_t lane = threadIdx.x & 31;
    long long z[EACH], top = INT64_MIN;
#pragma unroll
    for (int i = 0; i < EACH; i++) {
        const uint32_t e = i * 32 + lane;
        z[i] = INT64_MIN;
        if (e < p.experts) {
            z[i] = round_shift((e / 16 % 2 ? odd : even)[r * pitch + e / 32 * 16 + e % 16], kScale);
            top = max(top, z[i]);
        }
    }
    top = warp_max(top);
    int64_t sum = 0;
    bool bad = false;
    uint32_t v[EACH];
#pragma unroll
    for (int i = 0; i < EACH; i++) {
        v[i] = 0;
        if (i * 32 + lane < p.experts) {
            const int64_t x = fx_to_i64(table_at(p.exp_table, p.exp_len, fx_wsub(z[i], top), (int64_t)p.exp_len));
            bad |= x < 0 || x > INT32_MAX;
            v[i] = x < 0 || x > INT32_MAX ? 0u : (uint32_t)x;
        }
        sum += v[i];
    }
    sum = warp_sum(sum);
    if (bad) atomicOr(p.err, kErrRange);
    if (sum == 0 && lane == 0) atomicOr(p.err, kErrDivide);
    const float inv = 1.0f / (float)sum;
    uint32_t key[EACH], gate[EACH];  // values are at most 2^16
#pragma unroll
    for (int i = 0; i < EACH; i++) {
        const uint32_t e = i * 32 + lane;
        key[i] = e < p.experts ? ((sum ? (uint32_t)softmax_weight(v[i], sum, inv) : 0u) << 8 | (255 - e)) + 1 : 0;
        gate[i] = 0;
    }
    for (uint32_t j = 0; j < p.top_k; j++) {
        uint32_t best = 0;
#pragma unroll
        for (int i = 0; i < EACH; i++) best = max(best, key[i]);
        best = __reduce_max_sync(0xFFFFFFFFu, best);
#pragma unroll
        for (int i = 0; i < EACH; i++)
            if (key[i] == best) {  // one lane's, the keys being different
                key[i] = 0;
                gate[i] = (best - 1) >> 8;
                s_sel[r * p.top_k + j] = i * 32 + lane;
                s_score[r * p.top_k + j] = (int32_t)((best - 1) >> 8);
                atomicOr(&s_mask[i * 32 + lane], 1u << r);
            }
    }
    if (p.gate_out && blockIdx.x == 0)
#pragma unroll
        for (int i = 0; i < EACH; i++)
            if (i * 32 + lane < p.experts)
                p.gate_out[(uint64_t)r * p.experts + i * 32 + lane] = gate[i];
}

// The items of all experts: running sums over the experts by one warp give the
// places of their slots and items, then a thread per slot fills in its own.
// The routing warps; `thread`: a thread's number among theirs.
__device__ __forceinline__ void list_items(const MoeArgs& p, uint32_t thread, const uint32_t* s_sel, const uint32_t* s_mask,
                           uint32_t* s_start, Items* it) {
    const uint32_t lane = threadIdx.x & 31;
    if (thread < 32) {
        uint32_t slot = 0, item = 0;
        for (uint32_t e0 = 0; e0 < p.experts; e0 += 32) {
            const uint32_t e = e0 + lane, c = e < p.experts ? __popc(s_mask[e]) : 0, i = (c + kTile - 1) / kTile;
            uint32_t both = c << 16 | i;  // two running sums in one
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t a = __shfl_up_sync(0xFFFFFFFFu, both, o);
                if ((int)lane >= o) both += a;
            }
            const uint32_t at = slot + (both >> 16) - c, first = item + (both & 0xFFFF) - i;
            if (e < p.experts) s_start[e] = at;
            for (uint32_t j = 0; j < i; j++) {
                it->expert[first + j] = (uint8_t)e;
                it->count[first + j] = (uint8_t)min(kTile, c - j * kTile);
                it->first[first + j] = (uint16_t)(at + j * kTile);
            }
            both = __shfl_sync(0xFFFFFFFFu, both, 31);
            slot += both >> 16;
            item += both & 0xFFFF;
        }
        if (lane == 0) it->n = item;
    }
    route_sync(p.m);
    for (uint32_t i = thread; i < p.m * p.top_k; i += route_warps(p.m) * 32) {
        const uint32_t e = s_sel[i], tok = i / p.top_k, at = s_start[e] + __popc(s_mask[e] & ((1u << tok) - 1));
        it->slot[at] = (uint16_t)i;
        it->token[at] = (uint8_t)tok;
    }
}

// Fours of numbers from which on the blocks of a pair work out half of the digits each: 16 x 2048
// numbers 102.4 us for the layer instead of 105.3 (8 x 2048 66.5 and 67.2, 4 x 2048 42.9 and 42.3,
// 8 x 512 18.3 and 17.1)
constexpr uint32_t kShareDigits = 4096;
// Sums of a batch of tiles: (tile, gate or up, token, column)
constexpr uint32_t up_cells(uint32_t batch) { return batch * 2 * kTile * 16; }

// The tiles of 16 hidden columns that a block takes, u = blockIdx.x + i
// gridDim.x for i = 0, 1, ..: first those of the shared experts (four tokens
// to each), then those of the chosen experts' items; in batches, of which
// every warp takes an equal run of blocks of 64 k (gate and up together).
//
// Bound by (2048 wide, 64 experts of 1408, six to a token, the shared ones
// 2816): for one token a chain -- digits 2.1 us, logits 3.3, routing 3.4 beside
// the shared experts' first tiles, then the chosen experts' tiles 5 (20 MB: 4
// TB/s); for sixteen the same chain (6.2, 6.6 and 9.8 us) and some 43 us over
// the gate and up of the 51 or so chosen experts (162 MB: 3.8 TB/s), which is
// the warps' own work: codes taken apart, scales, slots asked for (issue slots
// 53 % used over the whole kernel, matrix pipe 12 %).  The codes prefetched into
// the second-level cache 4, 8 or 16 blocks ahead: 3 to 6 % slower; the router's
// blocks through the rings, ahead of the first codes: 4 %.  Two blocks to a
// cluster share the digits and the router: clusters of four or eight would
// share more, but only 132 or 120 of their blocks run at once.
template <bool TWO, int DEPTH, int RUN, uint32_t BATCH>
__global__ void __launch_bounds__(kThreads, 1) k_moe_up(const __grid_constant__ MoeArgs p) {
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ Items items;
    __shared__ uint32_t s_mask[kMaxExperts], s_start[kMaxExperts], s_sel[kMaxSlots];
    __shared__ __align__(8) uint64_t s_bar[kWarps * DEPTH];
    constexpr uint32_t kBytes = TWO ? 576 : 544, kPair = 2 * kBytes, kSlot = RUN * kPair;  // gate and up
    constexpr uint32_t kCells = up_cells(BATCH);
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint32_t pitch = (p.etiles + 1) / 2 * 16, rank = cluster.block_rank();
    uint8_t* ring = smem + (size_t)warp * DEPTH * kSlot;
    const Limbs acc{reinterpret_cast<uint32_t*>(smem + (size_t)kWarps * DEPTH * kSlot), kCells};
    const Limbs sums{acc.w, p.m * pitch};  // of the logits, before the tiles': at most kCells
    long long* logits = reinterpret_cast<long long*>(acc.w + 3 * kCells);  // of the pair's even tiles, then the odd ones
    uint8_t* digits = reinterpret_cast<uint8_t*>(logits + 2 * p.m * pitch);
    const uint32_t bar = shared_addr(&s_bar[warp * DEPTH]);
    cluster_arrive();  // both blocks have started before one writes into the other's shared memory
    let_next_start();
    if (lane == 0) {
#pragma unroll
        for (int i = 0; i < DEPTH; i++) barrier_init(bar + 8 * i);
        barrier_init_done();
    }
    __syncwarp();

    // ---- the block's tiles and the warp's stream of blocks; until the routing is known, the
    // shared experts' first batch
    const uint32_t ft = p.up.s.tiles, st = p.sup.s.tiles, stiles = st * ((p.m + kTile - 1) / kTile);
    const uint32_t blocks = p.up.s.blocks;
    auto tiles_below = [&](uint32_t u) { return u > blockIdx.x ? (u - blockIdx.x + gridDim.x - 1) / gridDim.x : 0u; };
    const uint32_t early = min(tiles_below(stiles), BATCH);  // tiles of the batch before the routing
    const uint32_t early_warps = kWarps - route_warps(p.m);
    uint32_t known = early;                                     // tiles of this block that may be asked for
    // of n tiles' blocks, the first that warp w takes if `warps` share them (all past the last)
    auto first_block = [&](uint32_t n, uint32_t w, uint32_t warps) { return min(w, warps) * (n * blocks) / warps; };
    uint32_t next_first = 0, next_n = early, next_at = first_block(early, warp, early_warps);
    uint32_t next_end = first_block(early, warp + 1, early_warps);
    uint32_t next_slot = 0, asked = 0, taken = 0;
    uint32_t next_left = 0;  // blocks of the present tile still to be asked for
    const uint8_t* next_w = nullptr;
    auto next_tile = [&]() {  // lane 0 only: on to the tile at next_at, false at the end of what is known
        while (next_at == next_end) {
            if (next_first + next_n >= known) return false;
            next_first += next_n;
            next_n = min(next_first == early && early < BATCH ? BATCH - early : BATCH, known - next_first);
            next_at = first_block(next_n, warp, kWarps);
            next_end = first_block(next_n, warp + 1, kWarps);
        }
        const uint32_t i = next_at / blocks, b = next_at - i * blocks, u = blockIdx.x + (next_first + i) * gridDim.x;
        const bool shared = u < stiles;
        const uint32_t v = shared ? u : u - stiles, item = v / (shared ? st : ft), tile = v - item * (shared ? st : ft);
        next_w = shared ? p.sup.w + ((uint64_t)tile * blocks + b) * kPair
                        : p.up.w + (((uint64_t)items.expert[item] * ft + tile) * blocks + b) * kPair;
        next_left = min(next_end - next_at, blocks - b);
        next_at += next_left;
        return true;
    };
    Patience patience;
    auto ask = [&]() {  // lane 0 only: fill the ring, up to RUN blocks of one tile to a slot
        if (patience.failed) return;
        while (asked < taken + DEPTH) {
            if (next_left == 0 && !next_tile()) return;
            const uint32_t run = min((uint32_t)RUN, next_left), b = bar + 8 * next_slot;
            barrier_expect(b, run * kPair);
            bulk_copy(shared_addr(ring) + next_slot * kSlot, next_w, run * kPair, b);
            next_left -= run;
            next_w += run * kPair;
            asked++;
            next_slot = next_slot + 1 == DEPTH ? 0 : next_slot + 1;
        }
    };
    if (lane == 0) ask();

    // ---- the rows' digits and the logits
    acc.template clear<kThreads>();
    for (uint32_t i = threadIdx.x; i < p.experts; i += kThreads) s_mask[i] = 0;
    wait_for_previous();
    bool bad = false;
    const uint32_t fours = p.m * blocks * 16;
    if (fours < kShareDigits) {
        bad |= !q4_digitise<kThreads, 2>(p.x, p.ldx, 1, p.h, blocks * 64, 0, fours, digits, p.stride);
        __syncthreads();
        cluster_wait();
    } else {  // half of them each, stored to both
        cluster_wait();
        bad |= !q4_digitise<kThreads, 8>(p.x, p.ldx, 1, p.h, blocks * 64, rank * (fours / 2), rank ? fours : fours / 2, digits,
                                      p.stride, cluster.map_shared_rank(digits, rank ^ 1));
        cluster.sync();
    }
    {
        // tiles of 16 experts, every other one this block's; eight (or sixteen) warps to a tile
        const uint32_t own = (p.etiles - rank + 1) / 2, wide = own > 1 ? kWarps / 2 : kWarps;
        for (uint32_t i = warp / wide; i < own; i += kWarps / wide) {
            const uint32_t w = warp % wide, r0 = w * blocks / wide, r1 = (w + 1) * blocks / wide;
            router_part(p, digits, i, rank, r0, r1, sums, pitch);
        }
    }
    __syncthreads();
    {
        long long* mine = logits + rank * p.m * pitch;
        long long* there = cluster.map_shared_rank(mine, rank ^ 1);
        for (uint32_t i = threadIdx.x; i < p.m * pitch; i += kThreads) {
            mine[i] = there[i] = sums.get(i);
            sums.clear(i);
        }
    }
    __syncthreads();
    cluster_arrive();  // the neighbour's logits: waited for after the first batch

    uint32_t slot = 0, phase = 0;
    bool routed = false;
    auto token_of = [&](bool shared, uint32_t first, uint32_t j) { return shared ? first + j : items.token[first + j]; };
    // a batch of the block's tiles, n from number `first` on, shared by `warps`: sums into acc, from
    // place `base` on
    auto add_up = [&](uint32_t first, uint32_t n, uint32_t warps, uint32_t base) {
        uint32_t at = first_block(n, warp, warps);
        const uint32_t end = first_block(n, warp + 1, warps);
        while (at < end) {
            const uint32_t i = at / blocks, u = blockIdx.x + (first + i) * gridDim.x;
            const bool shared = u < stiles;
            const uint32_t item = shared ? u / st : (u - stiles) / ft;
            const uint32_t tok0 = shared ? item * kTile : items.first[item];
            const uint32_t count = shared ? min(kTile, p.m - tok0) : items.count[item];
            uint32_t from[2];
#pragma unroll
            for (int q = 0; q < 2; q++)
                from[q] = shared_addr(digits) + (token_of(shared, tok0, min(2 * q + (g >> 2), count - 1)) * 4 + (g & 3)) * p.stride + 16 * t;
            Q4Sum<2> sum[2];
            sum[0].clear();
            sum[1].clear();
            uint32_t b = at % blocks;
            const uint32_t stop = min(blocks, b + end - at);
            at += stop - b;
            while (b < stop) {
                barrier_wait(bar + 8 * slot, phase, patience);
                const Q4Lane lane_at(shared_addr(ring) + slot * kSlot);
#pragma unroll
                for (int r = 0; r < RUN; r++) {
                    if (RUN > 1 && b == stop) break;
                    uint4 x[2];
                    x[0] = load16(from[0] + b * 64);
                    if (count > 2) {
                        x[1] = load16(from[1] + b * 64);
                        q4_block<TWO, 2>(sum[0], lane_at, r * kPair, x);
                        q4_block<TWO, 2>(sum[1], lane_at, r * kPair + kBytes, x);
                    } else {
                        q4_block<TWO, 1>(sum[0], lane_at, r * kPair, x);
                        q4_block<TWO, 1>(sum[1], lane_at, r * kPair + kBytes, x);
                    }
                    b++;
                }
                taken++;
                __syncwarp();  // every lane has read the slot
                if (lane == 0) ask();
                if (++slot == DEPTH) {
                    slot = 0;
                    phase ^= 1;
                }
            }
#pragma unroll
            for (int q = 0; q < 2; q++)
                if (2 * q < count) {
                    const uint32_t j = 2 * q + (t >> 1);
#pragma unroll
                    for (int mat = 0; mat < 2; mat++) {
                        const long long v = sum[mat].finish(q);
                        if (j < count) acc.add((((base + i) * 2 + mat) * kTile + j) * 16 + g + 8 * (t & 1), v);
                    }
                }
        }
    };
    // and from them the activations, two of a thread at a time: their SiLU entries come together
    auto finish = [&](uint32_t first, uint32_t n) {
        constexpr int kOuts = 2;
        for (uint32_t o0 = threadIdx.x; o0 < n * kTile * 16; o0 += kThreads * kOuts) {
            uint8_t* to[kOuts];
            int64_t up[kOuts];
            uint64_t silu[kOuts];
#pragma unroll
            for (int q = 0; q < kOuts; q++) {
                to[q] = nullptr;
                const uint32_t o = o0 + q * kThreads;
                if (o >= n * kTile * 16) continue;
                const uint32_t i = o / (kTile * 16), j = o / 16 % kTile, c = o % 16, u = blockIdx.x + (first + i) * gridDim.x;
                const bool shared = u < stiles;
                const uint32_t v = shared ? u : u - stiles, per = shared ? st : ft, item = v / per, f = (v - item * per) * 16 + c;
                const uint32_t tok0 = shared ? item * kTile : items.first[item];
                const uint32_t count = shared ? min(kTile, p.m - tok0) : items.count[item];
                if (j >= count) continue;  // its sums are zero
                const uint32_t cell = (i * 2 * kTile + j) * 16 + c;
                const uint32_t shift = shared ? p.shift : kScale;
                const int64_t gi = round_shift(acc.get(cell), shift);
                up[q] = round_shift(acc.get(cell + kTile * 16), shift);
                acc.clear(cell);
                acc.clear(cell + kTile * 16);
                if (f >= (shared ? p.sup.s.n : p.up.s.n)) continue;
                silu[q] = table_at(p.silu, p.silu_len, gi, (int64_t)(p.silu_len / 2));
                to[q] = (shared ? p.sact + (uint64_t)tok0 * p.sdown.s.blocks * 256
                                : p.act + (uint64_t)tok0 * p.down.s.blocks * 256) +
                        (f / 64 * count + j) * 256 + q4_pos(f % 64);
            }
#pragma unroll
            for (int q = 0; q < kOuts; q++)
                if (to[q]) {
                    uint32_t d;
                    bad |= !q4_digits(round_shift(fx_wmul(fx_to_i64(silu[q]), up[q]), kScale), &d);
#pragma unroll
                    for (int b = 0; b < 4; b++) to[q][64 * b] = (uint8_t)(d >> (8 * b));
                }
        }
    };

    // ---- the batches; routing beside the first, of the shared experts, whose sums are held to be
    // finished with the next batch's
    uint32_t base = 0;
    for (uint32_t first = 0, n = early;; n = min(BATCH - base, known - first)) {
        const bool routing = !routed;
        add_up(first, n, routing ? early_warps : kWarps, base);
        if (routing) {
            __syncwarp();
            cluster_wait();
            if (warp >= early_warps) {
                for (uint32_t r = warp - early_warps; r < p.m; r += kWarps - early_warps) {
                    if (p.experts <= 64)  // (the general form: 25.6 us instead of 23.1 for one token)
                        route_token<2>(p, r, logits, logits + p.m * pitch, pitch, s_sel, items.score, s_mask);
                    else
                        route_token<kMaxExperts / 32>(p, r, logits, logits + p.m * pitch, pitch, s_sel, items.score, s_mask);
                }
                route_sync(p.m);
                list_items(p, threadIdx.x - early_warps * 32, s_sel, s_mask, s_start, &items);
            }
        }
        __syncthreads();
        if (routing) {
            routed = true;
            known = tiles_below(stiles + ft * items.n);
            if (lane == 0) ask();
            if (blockIdx.x == 0)
                for (uint32_t i = threadIdx.x; i < sizeof(Items) / 4; i += kThreads)
                    reinterpret_cast<uint32_t*>(p.items)[i] = reinterpret_cast<const uint32_t*>(&items)[i];
        }
        first += n;
        if (routing && early < BATCH && first < known) {
            base = early;
            continue;
        }
        finish(first - n - base, base + n);
        base = 0;
        if (first >= known) break;
        __syncthreads();
    }
    if (bad) atomicOr(p.err, kErrRange);
    patience_end(patience, p.err);
}

constexpr int kDownDepth = 2;     // slots of a ring (three: the same times)
constexpr uint32_t kDownRun = 2;  // blocks to a slot

// Blocks of the stream that a warp of k_moe_down takes: the chosen experts'
// items one after another, then the shared experts' runs of tokens
struct DownAt {
    uint32_t b, len, count, first;
    bool shared;
    const uint8_t *w, *x;  // block b of the two tiles, and of the tokens' digits
};

// A pair of blocks to 32 output columns, half of the stream each; digits come
// with the codes, a slot's copies under one barrier.
//
// Bound by (sizes as above): one token 6.5 us, of which 1.5 pass before the
// items are there and 3.5 stream 10 MB; sixteen tokens some 25 us, 3 before the
// items, 18 over 81 MB of codes (4.5 TB/s) and 46 MB of digits from the
// second-level cache, by the number of copies more than by their bytes: two to a
// slot, one of 2176 bytes of codes and one of digits, where a copy to each tile
// and token took the layer from 94 to 103 us.  Slots of more blocks but fewer tokens' digits, two or
// three blocks by what fits: 97 to 104 us.
template <bool TWO>
__global__ void __launch_bounds__(kThreads, 1) k_moe_down(const __grid_constant__ MoeArgs p) {
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ Items items;
    __shared__ __align__(8) uint64_t s_bar[kWarps * kDownDepth];
    constexpr uint32_t kBytes = TWO ? 576 : 544, kSlot = kDownRun * (2 * kBytes + 256 * kTile);
    constexpr uint32_t kDigits = 2 * kDownRun * kBytes;  // after the tiles' blocks: those of the tokens
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint32_t rank = cluster.block_rank(), slots = p.m * p.top_k, cells = (slots + p.m) * 32;
    uint8_t* ring = smem + (size_t)warp * p.depth * kSlot;
    const Limbs acc{reinterpret_cast<uint32_t*>(smem + (size_t)kWarps * p.depth * kSlot), cells};
    const uint32_t bar = shared_addr(&s_bar[warp * kDownDepth]);
    let_next_start();
    if (lane == 0) {
#pragma unroll
        for (int i = 0; i < kDownDepth; i++) barrier_init(bar + 8 * i);
        barrier_init_done();
    }
    __syncwarp();
    acc.template clear<kThreads>();
    const uint32_t pairs = (p.down.s.tiles + 1) / 2, pair = blockIdx.x / 2;
    if (threadIdx.x == 0)  // the shared experts' codes of these columns start for the second-level cache
        prefetch_l2(p.sdown.w + (uint64_t)pair * p.sdown.s.blocks * 2 * kBytes, p.sdown.s.blocks * 2 * kBytes);
    wait_for_previous();
    for (uint32_t i = threadIdx.x; i < sizeof(Items) / 4; i += kThreads)
        reinterpret_cast<uint32_t*>(&items)[i] = reinterpret_cast<const uint32_t*>(p.items)[i];
    __syncthreads();

    const uint32_t nf = p.down.s.blocks, ns = p.sdown.s.blocks;
    const uint32_t stiles = (p.m + kTile - 1) / kTile, routed = nf * items.n, total = routed + ns * stiles;
    const uint32_t who = rank * kWarps + warp;
    uint32_t at = (uint32_t)((uint64_t)who * total / (2 * kWarps));
    const uint32_t end = (uint32_t)((uint64_t)(who + 1) * total / (2 * kWarps));
    auto locate = [&](DownAt& d, uint32_t pos) {
        d.shared = pos >= routed;
        const uint32_t in = d.shared ? pos - routed : pos;
        d.len = d.shared ? ns : nf;
        const uint32_t item = in / d.len;
        d.b = in % d.len;
        d.first = d.shared ? item * kTile : items.first[item];
        d.count = d.shared ? min(kTile, p.m - d.first) : items.count[item];
        const uint8_t* w = d.shared ? p.sdown.w : p.down.w + (uint64_t)items.expert[item] * pairs * nf * 2 * kBytes;
        d.w = w + ((uint64_t)pair * d.len + d.b) * 2 * kBytes;
        d.x = (d.shared ? p.sact : p.act) + ((uint64_t)d.first * d.len + d.b * d.count) * 256;
    };
    DownAt next, now;
    uint32_t next_at = at, next_slot = 0;
    if (at < end) {
        locate(now, at);
        next = now;
    }
    Patience patience;
    auto ask = [&]() {  // lane 0 only
        if (patience.failed) return;
        const uint32_t b = bar + 8 * next_slot, to = shared_addr(ring + next_slot * kSlot);
        const uint32_t run = min(kDownRun, min(end - next_at, next.len - next.b));
        barrier_expect(b, run * (2 * kBytes + 256 * next.count));
        bulk_copy(to, next.w, run * 2 * kBytes, b);
        bulk_copy(to + kDigits, next.x, run * 256 * next.count, b);
        next_slot = next_slot + 1 == p.depth ? 0 : next_slot + 1;
        next_at += run;
        next.b += run;
        next.w += run * 2 * kBytes;
        next.x += run * 256 * next.count;
        if (next.b == next.len && next_at < end) locate(next, next_at);
    };
    if (lane == 0)
        for (uint32_t i = 0; i < p.depth; i++)
            if (next_at < end) ask();
    uint32_t slot = 0, phase = 0;
    while (at < end) {
        const uint32_t stop = min(end, at + now.len - now.b);
        Q4Sum<2> sum[2];
        sum[0].clear();
        sum[1].clear();
        // digits of columns g: digit row g % 4 of token g / 4 (and 2 + g / 4) of the item
        const uint32_t x0 = kDigits + min(g >> 2, now.count - 1) * 256 + (g & 3) * 64 + 16 * t;
        const uint32_t x1 = kDigits + min(2 + (g >> 2), now.count - 1) * 256 + (g & 3) * 64 + 16 * t;
        while (at < stop) {
            barrier_wait(bar + 8 * slot, phase, patience);
            const uint32_t base = shared_addr(ring) + slot * kSlot;
            const Q4Lane lane_at(base);
#pragma unroll
            for (uint32_t r = 0; r < kDownRun; r++) {
                if (at == stop) break;
                uint4 x[2];
                x[0] = load16(base + x0 + r * now.count * 256);
                if (now.count > 2) {
                    x[1] = load16(base + x1 + r * now.count * 256);
                    q4_block<TWO, 2>(sum[0], lane_at, 2 * r * kBytes, x);
                    q4_block<TWO, 2>(sum[1], lane_at, (2 * r + 1) * kBytes, x);
                } else {
                    q4_block<TWO, 1>(sum[0], lane_at, 2 * r * kBytes, x);
                    q4_block<TWO, 1>(sum[1], lane_at, (2 * r + 1) * kBytes, x);
                }
                at++;
            }
            __syncwarp();  // every lane has read the slot
            if (lane == 0 && next_at < end) ask();
            if (++slot == p.depth) {
                slot = 0;
                phase ^= 1;
            }
        }
#pragma unroll
        for (int i = 0; i < 2; i++)
            if (2 * i < now.count) {
                const uint32_t j = 2 * i + (t >> 1);
#pragma unroll
                for (int q = 0; q < 2; q++) {
                    const long long v = sum[q].finish(i);
                    if (j < now.count)
                        acc.add((now.shared ? slots + now.first + j : items.slot[now.first + j]) * 32 + q * 16 + g + 8 * (t & 1), v);
                }
            }
        if (at < end) locate(now, at);
    }
    __syncwarp();
    cluster.sync();
    // A block finishes 16 of the 32 columns, with its neighbour's part of the sums
    const Limbs there{cluster.map_shared_rank(acc.w, rank ^ 1), cells};
    for (uint32_t o = threadIdx.x; o < p.m * 16; o += kThreads) {
        const uint32_t c = rank * 16 + (o & 15), r = o >> 4;
        const uint64_t n = (uint64_t)pair * 32 + c;
        if (n >= p.h) continue;
        const uint32_t s = (slots + r) * 32 + c;
        int64_t y = round_shift(fx_wadd(acc.get(s), there.get(s)), p.shift);
        for (uint32_t j = 0; j < p.top_k; j++) {
            const uint32_t k = (r * p.top_k + j) * 32 + c;
            const int64_t d = round_shift(fx_wadd(acc.get(k), there.get(k)), kScale);
            y = fx_wadd(y, round_shift(fx_wmul(d, items.score[r * p.top_k + j]), 16));
        }
        uint64_t f = fx_from_i64(y);
        if (p.residual) f = gl_canon(gl_add(f, gl_canon(p.residual[r * p.ldr + n])));
        p.out[r * (uint64_t)p.h + n] = f;
    }
    patience_end(patience, p.err);
    cluster.sync();  // no block leaves while its sums may still be read
}

// Dynamic shared memory of k_moe_up
size_t up_shared(uint32_t m, uint32_t stride, uint32_t etiles, uint32_t bytes, uint32_t blocks, uint32_t batch) {
    return (size_t)kWarps * blocks * 2 * bytes + 12 * up_cells(batch) + (size_t)m * (4 * stride + 2 * 16 * 8 * ((etiles + 1) / 2));
}


uint32_t tokens_at_once(uint32_t stride, uint32_t etiles, uint32_t bytes) {
    uint32_t m = kMaxTokens;
    while (m > 1 && up_shared(m, stride, etiles, bytes, 3, 16) > kMaxShared) m--;
    return m;
}

struct MoeShapes {
    Q4Shape up, down, sup, sdown;
};

bool moe_shapes(uint64_t h, uint64_t experts, uint64_t top_k, uint64_t f, uint64_t shared_f, uint32_t group,
                MoeShapes* s) {
    return experts >= 1 && experts <= kMaxExperts && top_k >= 1 && top_k <= experts && top_k <= kMaxTop &&
           q4_shape(h, f, group, 0, &s->up) && q4_shape(f, h, group, 0, &s->down) &&
           q4_shape(h, shared_f, group, 0, &s->sup) && q4_shape(shared_f, h, group, 0, &s->sdown);
}

template <bool TWO, int DEPTH, int RUN, uint32_t BATCH>
int up_launch(const MoeArgs& p, cudaStream_t stream) {
    static std::atomic<uint64_t> set{0};
    auto* kernel = k_moe_up<TWO, DEPTH, RUN, BATCH>;
    ZK_TRY(allow_shared(reinterpret_cast<const void*>(kernel), kMaxShared, &set));
    return launch(kernel, dim3(kSms), kThreads, up_shared(p.m, p.stride, p.etiles, p.up.s.bytes, DEPTH * RUN, BATCH), 2, stream, p);
}

template <bool TWO>
int moe_launch(MoeArgs p, cudaStream_t stream) {
    auto fits = [&](uint32_t blocks, uint32_t batch) {
        return p.m * ((p.etiles + 1) / 2 * 16) <= up_cells(batch) &&
               up_shared(p.m, p.stride, p.etiles, p.up.s.bytes, blocks, batch) <= kMaxShared;
    };
    // A ring of two slots of two blocks, with batches of eight tiles where those of sixteen leave no
    // room for it, else of three slots of one (twelve tokens of 2048: 76.5, 79.1 and 82.2 us, sixteen
    // 91.4 and 94.4; three slots of two: 59.5 us for eight tokens instead of 58.6, 22.8 for one
    // instead of 22.3).
    const int rc = fits(4, 16)  ? up_launch<TWO, 2, 2, 16>(p, stream)
                   : fits(4, 8) ? up_launch<TWO, 2, 2, 8>(p, stream)
                                : up_launch<TWO, 3, 1, 16>(p, stream);
    if (rc) return rc;
    static std::atomic<uint64_t> set{0};
    ZK_TRY(allow_shared(reinterpret_cast<const void*>(k_moe_down<TWO>), kMaxShared, &set));
    const size_t sums = 12ull * (p.m * p.top_k + p.m) * 32, slot = (size_t)kWarps * kDownRun * (2 * p.down.s.bytes + 256 * kTile);
    p.depth = kDownDepth;
    while (p.depth > 1 && p.depth * slot + sums > kMaxShared) p.depth--;  // one of 70 kB fits beside 104 kB
    return launch(k_moe_down<TWO>, dim3((p.down.s.tiles + 1) / 2 * 2), kThreads, p.depth * slot + sums, 2, stream, p);
}

}  // namespace

}  // namespace zk

using namespace zk;

extern "C" {

uint64_t zkie2_moe_router_words(uint64_t h, uint64_t experts) {
    Q4Shape s;
    if (experts == 0 || experts > kMaxExperts || !q4_shape(h, 16, 64, 0, &s)) return 0;
    return ceil_div(experts, 16) * s.blocks * 512;
}

int zkie2_moe_router_pack(const uint64_t* d_w, uint64_t h, uint64_t experts, uint32_t* d_packed, uint32_t* d_err,
                          cudaStream_t stream) {
    const uint64_t words = zkie2_moe_router_words(h, experts);
    if (words == 0 || !d_w || !d_packed || !d_err) return (int)cudaErrorInvalidValue;
    const uint64_t blocks = ceil_div(words, 256);
    k_moe_router_pack<<<(unsigned)(blocks < kSms * 16 ? blocks : kSms * 16), 256, 0, stream>>>(
        d_w, (uint32_t)h, (uint32_t)experts, (uint32_t)ceil_div(h, 64), (uint32_t)ceil_div(experts, 16), d_packed, d_err);
    ZK_LAUNCH_CHECK();
    return 0;
}

uint64_t zkie2_moe_rows_scratch_elems(uint64_t m, uint64_t h, uint64_t experts, uint64_t top_k, uint64_t f,
                                      uint64_t shared_f, uint32_t group) {
    MoeShapes s;
    if (m == 0 || m > 65535 || !moe_shapes(h, experts, top_k, f, shared_f, group, &s)) return 0;
    const uint64_t t = m < kMaxTokens ? m : kMaxTokens, slots = t * top_k;
    // the items and the digits of the activations
    return ceil_div(sizeof(Items), 16) * 2 + (slots * 4 * s.down.blocks * 64 + t * 4 * s.sdown.blocks * 64) / 8;
}

int zkie2_moe_rows(const uint64_t* d_x, uint64_t ldx, uint64_t m, uint64_t h, uint64_t experts, uint64_t top_k,
                   uint64_t f, uint64_t shared_f, uint32_t group, const uint32_t* d_router,
                   const uint32_t* const* h_weights, const uint64_t* d_exp_table, uint64_t exp_len,
                   const uint64_t* d_silu_table, uint64_t silu_len, uint32_t shift,
                   const uint64_t* d_residual, uint64_t ldr, uint64_t* d_out, uint64_t* d_gate, uint32_t* d_err,
                   uint64_t* d_scratch, cudaStream_t stream) {
    MoeShapes s;
    if (!moe_shapes(h, experts, top_k, f, shared_f, group, &s) || m > 65535 || shift > 62 || !d_router || !h_weights ||
        !d_exp_table || exp_len == 0 || !d_silu_table || silu_len == 0 || !d_err || (m > 1 && ldx < h) ||
        (d_residual && m > 1 && ldr < h) || ((uintptr_t)d_router & 15) || ((uintptr_t)d_scratch & 15))
        return (int)cudaErrorInvalidValue;
    for (int i = 0; i < 4; i++)
        if (!h_weights[i] || ((uintptr_t)h_weights[i] & 15)) return (int)cudaErrorInvalidValue;
    if (m == 0) return 0;
    if (!d_x || !d_out || !d_scratch) return (int)cudaErrorInvalidValue;
    MoeArgs p{};
    const Q4Shape* shape[4] = {&s.up, &s.down, &s.sup, &s.sdown};
    Q4Weight* weight[4] = {&p.up, &p.down, &p.sup, &p.sdown};
    for (int i = 0; i < 4; i++) *weight[i] = Q4Weight{reinterpret_cast<const uint8_t*>(h_weights[i]), *shape[i]};
    p.ldx = ldx;
    p.h = (uint32_t)h;
    p.experts = (uint32_t)experts;
    p.top_k = (uint32_t)top_k;
    p.etiles = (uint32_t)ceil_div(experts, 16);
    p.router = reinterpret_cast<const uint4*>(d_router);
    p.exp_table = d_exp_table;
    p.exp_len = exp_len;
    p.silu = d_silu_table;
    p.silu_len = silu_len;
    p.shift = shift;
    p.ldr = ldr;
    p.err = d_err;
    p.stride = q4_digit_stride(s.up.blocks);
    const uint32_t most = tokens_at_once(p.stride, p.etiles, s.up.bytes);
    const uint64_t slots = (m < kMaxTokens ? m : kMaxTokens) * top_k;
    p.items = reinterpret_cast<Items*>(d_scratch);
    p.act = reinterpret_cast<uint8_t*>(d_scratch) + ceil_div(sizeof(Items), 16) * 16;
    p.sact = p.act + slots * 4 * s.down.blocks * 64;
    for (uint64_t r = 0; r < m; r += most) {
        p.m = (uint32_t)(m - r < most ? m - r : most);
        p.x = d_x + r * ldx;
        p.residual = d_residual ? d_residual + r * ldr : nullptr;
        p.out = d_out + r * h;
        p.gate_out = d_gate ? d_gate + r * experts : nullptr;
        const int rc = group == 32 ? moe_launch<true>(p, stream) : moe_launch<false>(p, stream);
        if (rc) return rc;
    }
    return 0;
}

}  // extern "C"
