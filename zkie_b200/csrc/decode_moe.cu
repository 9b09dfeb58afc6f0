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
#include <cmath>
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

struct Q4Weight {
    const uint4* codes;
    const uint32_t* scales;
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
    int32_t score[kMaxSlots];   // a slot's softmax value
};
static_assert(sizeof(Items) % 4 == 0, "copied in words");

struct MoeArgs {
    const uint64_t* x;
    uint64_t ldx;
    uint32_t m, h, experts, top_k, etiles;
    const uint4* router;
    Q4Weight gate, up, down, sgate, sup, sdown;
    const uint64_t* exp_table;
    uint64_t exp_len;
    const uint64_t* silu;
    uint64_t silu_len;
    uint32_t shift;
    const uint64_t* residual;
    uint64_t ldr;
    uint64_t* out;
    uint64_t* gate_out;  // m x experts (or null)
    Items* items;
    uint8_t* act;        // (m top_k) x 4 x padded F digits
    uint8_t* sact;       // m x 4 x padded shared F digits
    uint32_t* err;
    uint32_t stride;     // bytes of a digit row of x
    uint32_t split;      // warps that share a tile of k_moe_up
};

__device__ __forceinline__ void group_sync(uint32_t id, uint32_t threads) {
    asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

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

// Logits of the 16 experts of a tile for 2 NT tokens, this warp's part of K,
// added to raw (tokens x padded experts, 64-bit sums in shared memory)
template <int NT>
__device__ void router_part(const MoeArgs& p, const uint8_t* digits, uint32_t tile, uint32_t tok0, uint32_t b0,
                            uint32_t b1, unsigned long long* raw) {
    const uint32_t lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    int c[2][NT][4];
#pragma unroll
    for (int w = 0; w < 2; w++)
#pragma unroll
        for (int i = 0; i < NT; i++) c[w][i][0] = c[w][i][1] = c[w][i][2] = c[w][i][3] = 0;
#pragma unroll 2
    for (uint32_t b = b0; b < b1; b++) {
        const uint4* r = p.router + ((uint64_t)tile * p.gate.s.blocks + b) * 128 + lane;
        const uint4 w00 = __ldg(r), w01 = __ldg(r + 32), w10 = __ldg(r + 64), w11 = __ldg(r + 96);
#pragma unroll
        for (int i = 0; i < NT; i++) {
            const uint32_t tok = min(tok0 + 2 * i + (g >> 2), p.m - 1);
            const uint4 x = *reinterpret_cast<const uint4*>(digits + (size_t)(tok * 4 + (g & 3)) * p.stride + b * 64 + 16 * t);
            mma_s8(c[0][i], w00.x, w00.y, w00.z, w00.w, x.x, x.y);
            mma_s8(c[1][i], w01.x, w01.y, w01.z, w01.w, x.x, x.y);
            mma_s8(c[0][i], w10.x, w10.y, w10.z, w10.w, x.z, x.w);
            mma_s8(c[1][i], w11.x, w11.y, w11.z, w11.w, x.z, x.w);
        }
    }
    const uint32_t pitch = p.etiles * 16;
#pragma unroll
    for (int i = 0; i < NT; i++) {
        const uint32_t tok = tok0 + 2 * i + (t >> 1);
        if (tok < p.m) {
#pragma unroll
            for (int q = 0; q < 2; q++) {
                const long long v = ((long long)c[0][i][2 * q] + ((long long)c[0][i][2 * q + 1] << 8)) +
                                    (((long long)c[1][i][2 * q] << 8) + ((long long)c[1][i][2 * q + 1] << 16));
                atomicAdd(&raw[tok * pitch + tile * 16 + g + 8 * q], (unsigned long long)v << (16 * (t & 1)));
            }
        }
    }
}

// One token's softmax over the experts and its top_k, by a warp: raw logits
// of the pair's two blocks (tiles of experts alternate between them).  A key
// holds an expert's value above its complement, so that the maximum is the
// first in TopKSelect's order.
__device__ void route_token(const MoeArgs& p, uint32_t r, const unsigned long long* even, const unsigned long long* odd,
                            uint32_t* s_sel, int32_t* s_score, uint32_t* s_mask) {
    const uint32_t lane = threadIdx.x & 31, pitch = p.etiles * 16;
    long long z[kMaxExperts / 32], top = INT64_MIN;
#pragma unroll
    for (int i = 0; i < (int)kMaxExperts / 32; i++) {
        const uint32_t e = i * 32 + lane;
        z[i] = INT64_MIN;
        if (e < p.experts) {
            z[i] = fx_round_div_pow2((int64_t)((e / 16) % 2 ? odd : even)[r * pitch + e], p.shift);
            top = max(top, z[i]);
        }
    }
    for (int o = 16; o; o >>= 1) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
    long long sum = 0;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < (int)kMaxExperts / 32; i++)
        if (i * 32 + lane < p.experts) {
            int64_t v = fx_to_i64(table_at(p.exp_table, p.exp_len, fx_wsub(z[i], top), (int64_t)p.exp_len));
            if (v < 0 || v > INT32_MAX) {
                bad = true;
                v = 0;
            }
            z[i] = v;
            sum += v;
        }
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    if (bad) atomicOr(p.err, kErrRange);
    if (sum == 0 && lane == 0) atomicOr(p.err, kErrDivide);
    const double inv = sum ? 1.0 / (double)sum : 0.0;
    uint32_t key[kMaxExperts / 32];  // values are at most 2^16
#pragma unroll
    for (int i = 0; i < (int)kMaxExperts / 32; i++) {
        const uint32_t e = i * 32 + lane;
        key[i] = e < p.experts ? ((sum ? (uint32_t)round_div_near(z[i] << 16, sum, inv) : 0u) << 8 | (255 - e)) + 1 : 0;
    }
    uint32_t chosen = 0;
    for (uint32_t j = 0; j < p.top_k; j++) {
        uint32_t best = 0;
#pragma unroll
        for (int i = 0; i < (int)kMaxExperts / 32; i++) best = max(best, (chosen >> i) & 1 ? 0u : key[i]);
        best = __reduce_max_sync(0xFFFFFFFFu, best);
#pragma unroll
        for (int i = 0; i < (int)kMaxExperts / 32; i++)
            if (key[i] == best && !((chosen >> i) & 1)) {  // one lane's, the keys being different
                chosen |= 1u << i;
                s_sel[r * p.top_k + j] = i * 32 + lane;
                s_score[r * p.top_k + j] = (int32_t)((best - 1) >> 8);
                atomicOr(&s_mask[i * 32 + lane], 1u << r);
            }
    }
    if (p.gate_out && blockIdx.x == 0)
#pragma unroll
        for (int i = 0; i < (int)kMaxExperts / 32; i++)
            if (i * 32 + lane < p.experts)
                p.gate_out[(uint64_t)r * p.experts + i * 32 + lane] = (chosen >> i) & 1 ? (key[i] - 1) >> 8 : 0;
}

// The items of all experts, by one warp: running sums over the experts give
// the places of their slots and items
__device__ void list_items(const MoeArgs& p, const uint32_t* s_sel, const uint32_t* s_mask, Items* it) {
    const uint32_t lane = threadIdx.x & 31;
    uint32_t slot = 0, item = 0;
    for (uint32_t e0 = 0; e0 < p.experts; e0 += 32) {
        const uint32_t e = e0 + lane;
        uint32_t mask = e < p.experts ? s_mask[e] : 0;
        const uint32_t c = __popc(mask), i = (c + kTile - 1) / kTile;
        uint32_t sc = c, si = i;
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t a = __shfl_up_sync(0xFFFFFFFFu, sc, o), b = __shfl_up_sync(0xFFFFFFFFu, si, o);
            if ((int)lane >= o) {
                sc += a;
                si += b;
            }
        }
        const uint32_t at = slot + sc - c;
        for (uint32_t j = 0; j < i; j++) {
            const uint32_t k = item + si - i + j;
            it->expert[k] = (uint8_t)e;
            it->count[k] = (uint8_t)min(kTile, c - j * kTile);
            it->first[k] = (uint16_t)(at + j * kTile);
        }
        for (uint32_t j = 0; j < c; j++) {
            const uint32_t tok = __ffs(mask) - 1;
            mask &= mask - 1;
            uint32_t place = 0;
            while (s_sel[tok * p.top_k + place] != e) place++;
            it->slot[at + j] = (uint16_t)(tok * p.top_k + place);
        }
        slot += __shfl_sync(0xFFFFFFFFu, sc, 31);
        item += __shfl_sync(0xFFFFFFFFu, si, 31);
    }
    if (lane == 0) it->n = item;
}

constexpr uint32_t kUpSlot = 2 * (512 + 64);                         // gate and up: codes, codes, scales, scales
constexpr size_t kUpRed = (size_t)kWarps * 2 * kTile * 16 * 8;       // every warp's sums of a tile

template <int G, int NT>
__device__ __forceinline__ void up_block(Q4Sum<2> (&sum)[2], const uint8_t* slot, const uint8_t* const (&from)[2],
                                         uint32_t b) {
    const uint32_t lane = threadIdx.x & 31, g = lane >> 2;
    uint4 x[2];
#pragma unroll
    for (int i = 0; i < NT; i++) x[i] = *reinterpret_cast<const uint4*>(from[i] + b * 64);
#pragma unroll
    for (int q = 0; q < 2; q++) {
        const uint4 w = *reinterpret_cast<const uint4*>(slot + q * 512 + lane * 16);
        const uint32_t* sc = reinterpret_cast<const uint32_t*>(slot + 1024 + q * 64);
        q4_block_n<G, NT>(sum[q], w, sc[g], G == 32 ? sc[8 + g] : 0, x, b & 1);
    }
}

template <int G, int DEPTH>
__global__ void __launch_bounds__(kThreads, 1) k_moe_up(const __grid_constant__ MoeArgs p) {
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ Items items;
    __shared__ uint32_t s_mask[kMaxExperts], s_sel[kMaxSlots];
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint32_t pitch = p.etiles * 16, rank = cluster.block_rank();
    uint8_t* ring = smem + (size_t)warp * DEPTH * kUpSlot;
    long long* red = reinterpret_cast<long long*>(smem + (size_t)kWarps * DEPTH * kUpSlot);
    unsigned long long* raw = reinterpret_cast<unsigned long long*>(reinterpret_cast<uint8_t*>(red) + kUpRed);
    uint8_t* digits = reinterpret_cast<uint8_t*>(raw + 2 * p.m * pitch);
    cluster_arrive();  // both blocks have started before one writes into the other's shared memory
    let_next_start();

    // ---- the warp's tiles, of the shared experts first: its stream of blocks
    const uint32_t ft = p.gate.s.tiles, st = p.sgate.s.tiles, stiles = st * ((p.m + kTile - 1) / kTile);
    const uint32_t blocks = p.gate.s.blocks, unit = G == 128 ? 2 : 1;
    const uint32_t per = kWarps / p.split, mine = warp / p.split, part = warp % p.split;
    const uint32_t b0 = part * (blocks / unit) / p.split * unit, b1 = (part + 1) * (blocks / unit) / p.split * unit;
    const uint32_t u0 = blockIdx.x + gridDim.x * mine, step = gridDim.x * per;
    uint32_t known = stiles;  // tiles that may be asked for
    uint32_t next_u = u0, next_b = b0, next_slot = 0;
    uint64_t next_tile = 0;
    const Q4Weight *next_g = nullptr, *next_w = nullptr;
    auto issue = [&]() {
        if (next_u < known && b0 < b1) {
            if (next_b == b0) {
                const bool shared = next_u < stiles;
                next_g = shared ? &p.sgate : &p.gate;
                next_w = shared ? &p.sup : &p.up;
                next_tile = shared ? next_u % st
                                   : (uint64_t)items.expert[(next_u - stiles) / ft] * ft + (next_u - stiles) % ft;
            }
            uint8_t* slot = ring + next_slot * kUpSlot;
            const uint64_t block = (next_tile * blocks + next_b) * 32 + lane, groups = next_tile * p.gate.s.groups * 8;
            copy16(slot + lane * 16, next_g->codes + block);
            copy16(slot + 512 + lane * 16, next_w->codes + block);
            uint32_t* sc = reinterpret_cast<uint32_t*>(slot + 1024);
            copy_scales<G>(sc, next_g->scales + groups, next_b, g, t);
            copy_scales<G>(sc + 16, next_w->scales + groups, next_b, g, t);
            next_slot = next_slot + 1 == DEPTH ? 0 : next_slot + 1;
            if (++next_b == b1) {
                next_b = b0;
                next_u += step;
            }
        }
    };
    // Copies that could not be asked for before the routing are made up after it: a group to
    // each block, counted ahead of the blocks taken.
    uint32_t asked = 0, taken = 0;
    auto ask = [&]() {
        while (asked < taken + DEPTH && next_u < known && b0 < b1) {
            issue();
            copy_commit();
            asked++;
        }
    };
    ask();

    // ---- the rows' digits and the logits
    for (uint32_t i = threadIdx.x; i < p.m * pitch; i += kThreads) raw[i] = 0;
    for (uint32_t i = threadIdx.x; i < p.experts; i += kThreads) s_mask[i] = 0;
    wait_for_previous();
    bool bad = false;
    for (uint32_t r = 0; r < p.m; r++)
        for (uint32_t k0 = threadIdx.x * 4; k0 < blocks * 64; k0 += kThreads * 4) {
            const uint64_t* xr = p.x + r * p.ldx + k0;
            uint32_t d[4];
#pragma unroll
            for (int j = 0; j < 4; j++) bad |= !q4_digits(k0 + j < p.h ? fx_to_i64(__ldg(xr + j)) : 0, &d[j]);
            q4_store_digits(digits + (size_t)r * 4 * p.stride + q4_pos(k0), p.stride, d);
        }
    __syncthreads();
    {
        // tiles of 16 experts, every other one this block's; eight (or sixteen) warps to a tile
        const uint32_t own = (p.etiles - rank + 1) / 2, wide = own > 1 ? kWarps / 2 : kWarps;
        for (uint32_t i = warp / wide; i < own; i += kWarps / wide) {
            const uint32_t w = warp % wide, r0 = w * blocks / wide, r1 = (w + 1) * blocks / wide;
            if (p.m <= 2)
                router_part<1>(p, digits, 2 * i + rank, 0, r0, r1, raw);
            else
                for (uint32_t tok = 0; tok < p.m; tok += 8) router_part<4>(p, digits, 2 * i + rank, tok, r0, r1, raw);
        }
    }
    __syncthreads();
    cluster_wait();
    unsigned long long* other = raw + p.m * pitch;
    {
        unsigned long long* there = cluster.map_shared_rank(other, rank ^ 1);
        for (uint32_t i = threadIdx.x; i < p.m * pitch; i += kThreads)
            if ((i % pitch / 16) % 2 == rank) there[i] = raw[i];
    }
    cluster.sync();
    for (uint32_t r = warp; r < p.m; r += kWarps)
        route_token(p, r, rank ? other : raw, rank ? raw : other, s_sel, items.score, s_mask);
    __syncthreads();
    if (warp == 0) list_items(p, s_sel, s_mask, &items);
    __syncthreads();
    if (blockIdx.x == 0)
        for (uint32_t i = threadIdx.x; i < sizeof(Items) / 4; i += kThreads)
            reinterpret_cast<uint32_t*>(p.items)[i] = reinterpret_cast<const uint32_t*>(&items)[i];
    known = stiles + ft * items.n;

    // ---- gate and up
    const uint64_t fp = (uint64_t)p.down.s.blocks * 64, sp = (uint64_t)p.sdown.s.blocks * 64;
    // A tile's last step, the SiLU lookup and the activation's digits, is held
    // over to the next tile, when its table entries have come.
    uint64_t held_silu = 0, held_row = 0;
    int64_t held_up = 0;
    uint8_t* held_to = nullptr;
    auto finish_held = [&]() {
        if (held_to) {
            uint32_t d;
            bad |= !q4_digits(fx_round_div_pow2(fx_wmul(fx_to_i64(held_silu), held_up), p.shift), &d);
#pragma unroll
            for (int j = 0; j < 4; j++) held_to[j * held_row] = (uint8_t)(d >> (8 * j));
            held_to = nullptr;
        }
    };
    uint32_t slot_at = 0;
    for (uint32_t u = u0; u < known; u += step) {
        const bool shared = u < stiles;
        const uint32_t item = shared ? u / st : (u - stiles) / ft, tile = shared ? u % st : (u - stiles) % ft;
        const uint32_t first = shared ? item * kTile : items.first[item];
        const uint32_t count = shared ? min(kTile, p.m - first) : items.count[item];
        const uint8_t* from[2];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const uint32_t at = min(2 * i + (g >> 2), count - 1);
            const uint32_t tok = shared ? first + at : items.slot[first + at] / p.top_k;
            from[i] = digits + (size_t)(tok * 4 + (g & 3)) * p.stride + 16 * t;
        }
        Q4Sum<2> sum[2];
        sum[0].clear();
        sum[1].clear();
        for (uint32_t b = b0; b < b1; b++) {
            __syncwarp();  // every lane has read the slot that is filled next
            ask();
            taken++;
            copy_wait_upto<DEPTH - 1>(asked - taken);
            __syncwarp();
            const uint8_t* slot = ring + slot_at * kUpSlot;
            slot_at = slot_at + 1 == DEPTH ? 0 : slot_at + 1;
            if (count > 2)
                up_block<G, 2>(sum, slot, from, b);
            else
                up_block<G, 1>(sum, slot, from, b);
        }
        long long* to = red + (size_t)warp * (2 * kTile * 16);
#pragma unroll
        for (int i = 0; i < 2; i++)
            if (2 * i < count) {
                long long v0, v1, w0, w1;
                sum[0].finish(i, &v0, &v1);
                sum[1].finish(i, &w0, &w1);
                if (!(t & 1)) {
                    long long* q = to + (2 * i + (t >> 1)) * 16;
                    q[g] = v0;
                    q[g + 8] = v1;
                    q[kTile * 16 + g] = w0;
                    q[kTile * 16 + g + 8] = w1;
                }
            }
        group_sync(1 + mine, p.split * 32);
        finish_held();
        const uint32_t o = part * 32 + lane, c = o & 15, j = o >> 4, f = tile * 16 + c;  // split >= 2: one each
        if (j < count && f < (shared ? p.sgate.s.n : p.gate.s.n)) {
            uint64_t gv = 0, uv = 0;
            for (uint32_t w = 0; w < p.split; w++) {
                const long long* r = red + (size_t)(mine * p.split + w) * (2 * kTile * 16) + j * 16 + c;
                gv += (uint64_t)r[0];
                uv += (uint64_t)r[kTile * 16];
            }
            held_silu = table_at(p.silu, p.silu_len, fx_round_div_pow2((int64_t)gv, p.shift), (int64_t)(p.silu_len / 2));
            held_up = fx_round_div_pow2((int64_t)uv, p.shift);
            held_row = shared ? sp : fp;
            held_to = (shared ? p.sact + (first + j) * 4 * sp : p.act + items.slot[first + j] * 4 * fp) + q4_pos(f);
        }
        group_sync(1 + mine, p.split * 32);  // the sums have been read
    }
    finish_held();
    if (bad) atomicOr(p.err, kErrRange);
}

constexpr int kDownDepth = 4;
constexpr uint32_t kDownSlot = 2 * 512 + 2 * 512 + 2 * 64;  // two tiles' codes, the digits of four rows, scales

// Blocks of the stream that a warp of k_moe_down takes: the chosen experts'
// items one after another, then the shared experts' runs of tokens
struct DownAt {
    uint32_t item, b, count, first;
    bool shared;
    const Q4Weight* w;
    uint64_t tile0, tile1;
    const uint8_t* from[2];  // this lane's digits
};

template <int G>
__global__ void __launch_bounds__(kThreads, 1) k_moe_down(const __grid_constant__ MoeArgs p) {
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ Items items;
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint32_t rank = cluster.block_rank(), slots = p.m * p.top_k, cells = (slots + p.m) * 32;
    uint8_t* ring = smem + (size_t)warp * kDownDepth * kDownSlot;
    unsigned long long* raw = reinterpret_cast<unsigned long long*>(smem + (size_t)kWarps * kDownDepth * kDownSlot);
    let_next_start();
    for (uint32_t i = threadIdx.x; i < cells; i += kThreads) raw[i] = 0;
    const uint32_t tiles = p.down.s.tiles, t0 = (blockIdx.x / 2) * 2, t1 = min(t0 + 1, tiles - 1);
    {   // the shared experts' codes of these columns start for the second-level cache
        const uint32_t bytes = p.sdown.s.blocks * 512;
        if (threadIdx.x < 2) prefetch_l2(p.sdown.codes + (uint64_t)(threadIdx.x ? t1 : t0) * p.sdown.s.blocks * 32, bytes);
    }
    wait_for_previous();
    for (uint32_t i = threadIdx.x; i < sizeof(Items) / 4; i += kThreads)
        reinterpret_cast<uint32_t*>(&items)[i] = __ldcg(reinterpret_cast<const uint32_t*>(p.items) + i);
    __syncthreads();

    const uint32_t unit = G == 128 ? 2 : 1, nf = p.down.s.blocks / unit, ns = p.sdown.s.blocks / unit;
    const uint32_t stiles = (p.m + kTile - 1) / kTile, routed = nf * items.n, total = routed + ns * stiles;
    const uint64_t fp = (uint64_t)p.down.s.blocks * 64, sp = (uint64_t)p.sdown.s.blocks * 64;
    const uint32_t who = rank * kWarps + warp;
    uint32_t at = (uint32_t)((uint64_t)who * total / (2 * kWarps)) * unit;
    const uint32_t end = (uint32_t)((uint64_t)(who + 1) * total / (2 * kWarps)) * unit;
    auto locate = [&](DownAt& d, uint32_t pos) {
        const uint32_t split = routed * unit;
        d.shared = pos >= split;
        const uint32_t in = d.shared ? pos - split : pos, len = d.shared ? p.sdown.s.blocks : p.down.s.blocks;
        d.item = in / len;
        d.b = in % len;
        d.first = d.shared ? d.item * kTile : items.first[d.item];
        d.count = d.shared ? min(kTile, p.m - d.first) : items.count[d.item];
        d.w = d.shared ? &p.sdown : &p.down;
        const uint64_t base = d.shared ? 0 : (uint64_t)items.expert[d.item] * tiles;
        d.tile0 = base + t0;
        d.tile1 = base + t1;
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const uint32_t j = min(2 * i + (g >> 2), d.count - 1);
            d.from[i] = (d.shared ? p.sact + ((uint64_t)(d.first + j) * 4 + (g & 3)) * sp
                                  : p.act + ((uint64_t)items.slot[d.first + j] * 4 + (g & 3)) * fp) + 16 * t;
        }
    };
    DownAt next, now;
    uint32_t next_at = at, next_slot = 0;
    if (at < end) {
        locate(next, at);
        now = next;
    }
    auto issue = [&]() {
        if (next_at < end) {
            uint8_t* slot = ring + next_slot * kDownSlot;
            const uint64_t blocks = next.w->s.blocks, groups = next.w->s.groups * 8ull;
            copy16(slot + lane * 16, next.w->codes + (next.tile0 * blocks + next.b) * 32 + lane);
            copy16(slot + 512 + lane * 16, next.w->codes + (next.tile1 * blocks + next.b) * 32 + lane);
            copy16(slot + 1024 + lane * 16, next.from[0] + next.b * 64);
            if (next.count > 2) copy16(slot + 1536 + lane * 16, next.from[1] + next.b * 64);
            uint32_t* sc = reinterpret_cast<uint32_t*>(slot + 2048);
            copy_scales<G>(sc, next.w->scales + next.tile0 * groups, next.b, g, t);
            copy_scales<G>(sc + 16, next.w->scales + next.tile1 * groups, next.b, g, t);
            next_slot = next_slot + 1 == kDownDepth ? 0 : next_slot + 1;
            next_at++;
            if (++next.b == next.w->s.blocks && next_at < end) locate(next, next_at);
        }
        copy_commit();
    };
#pragma unroll
    for (int i = 0; i < kDownDepth - 1; i++) issue();
    uint32_t slot_at = 0;
    while (at < end) {
        const uint32_t stop = min(end, at + now.w->s.blocks - now.b);
        Q4Sum<2> sum[2];
        sum[0].clear();
        sum[1].clear();
        for (; at < stop; at++, now.b++) {
            __syncwarp();
            issue();
            copy_wait<kDownDepth - 1>();
            __syncwarp();
            const uint8_t* slot = ring + slot_at * kDownSlot;
            slot_at = slot_at + 1 == kDownDepth ? 0 : slot_at + 1;
            uint4 x[2];
            x[0] = *reinterpret_cast<const uint4*>(slot + 1024 + lane * 16);
            if (now.count > 2) x[1] = *reinterpret_cast<const uint4*>(slot + 1536 + lane * 16);
#pragma unroll
            for (int q = 0; q < 2; q++) {
                const uint4 w = *reinterpret_cast<const uint4*>(slot + q * 512 + lane * 16);
                const uint32_t* sc = reinterpret_cast<const uint32_t*>(slot + 2048 + q * 64);
                if (now.count > 2)
                    q4_block_n<G, 2>(sum[q], w, sc[g], G == 32 ? sc[8 + g] : 0, x, now.b & 1);
                else
                    q4_block_n<G, 1>(sum[q], w, sc[g], G == 32 ? sc[8 + g] : 0, x, now.b & 1);
            }
        }
#pragma unroll
        for (int i = 0; i < 2; i++)
            if (2 * i < now.count) {
                const uint32_t j = 2 * i + (t >> 1);
#pragma unroll
                for (int q = 0; q < 2; q++) {
                    long long v0, v1;
                    sum[q].finish(i, &v0, &v1);
                    if (!(t & 1) && j < now.count) {
                        const uint32_t slot = now.shared ? slots + now.first + j : items.slot[now.first + j];
                        atomicAdd(&raw[slot * 32 + q * 16 + g], (unsigned long long)v0);
                        atomicAdd(&raw[slot * 32 + q * 16 + g + 8], (unsigned long long)v1);
                    }
                }
            }
        if (at < end) locate(now, at);
    }
    cluster.sync();
    // A block finishes 16 of the 32 columns, with its neighbour's part of the sums
    const unsigned long long* there = cluster.map_shared_rank(raw, rank ^ 1);
    for (uint32_t o = threadIdx.x; o < p.m * 16; o += kThreads) {
        const uint32_t c = rank * 16 + (o & 15), r = o >> 4;
        const uint64_t n = (uint64_t)t0 * 16 + c;
        if (n >= p.h) continue;
        const uint32_t s = (slots + r) * 32 + c;
        int64_t y = fx_round_div_pow2((int64_t)(raw[s] + there[s]), p.shift);
        for (uint32_t j = 0; j < p.top_k; j++) {
            const uint32_t k = (r * p.top_k + j) * 32 + c;
            const int64_t d = fx_round_div_pow2((int64_t)(raw[k] + there[k]), p.shift);
            y = fx_wadd(y, fx_round_div_pow2(fx_wmul(d, items.score[r * p.top_k + j]), 16));
        }
        uint64_t f = fx_from_i64(y);
        if (p.residual) f = gl_canon(gl_add(f, gl_canon(__ldg(p.residual + r * p.ldr + n))));
        p.out[r * (uint64_t)p.h + n] = f;
    }
    cluster.sync();  // no block leaves while its sums may still be read
}

// Dynamic shared memory of k_moe_up
size_t up_shared(uint32_t m, uint32_t stride, uint32_t etiles, uint32_t depth) {
    return (size_t)kWarps * depth * kUpSlot + kUpRed + (size_t)m * (4 * stride + 2 * 16 * 8 * etiles);
}

constexpr uint32_t kUpShallow = 3, kUpDeep = 6;

uint32_t tokens_at_once(uint32_t stride, uint32_t etiles) {
    uint32_t m = kMaxTokens;
    while (m > 1 && up_shared(m, stride, etiles, kUpShallow) > kMaxShared) m--;
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

// Warps to a tile of k_moe_up (at least two: a thread then finishes one
// result): fewest steps of a block's warps, each
// tile with what it costs besides its blocks, for the number of experts that
// m tokens choose if all are alike
uint32_t up_split(const MoeArgs& p, uint32_t unit) {
    const double hit = p.experts * (1 - pow(1 - (double)p.top_k / p.experts, p.m));
    const uint64_t tiles = (uint64_t)(hit * p.gate.s.tiles) + ceil_div(p.m, kTile) * p.sgate.s.tiles;
    uint64_t least = ~0ull;
    uint32_t split = 2;
    for (uint32_t s = 2; s <= (uint32_t)kWarps; s *= 2) {
        const uint64_t cost = ceil_div(tiles, (uint64_t)kSms * (kWarps / s)) *
                              (ceil_div(p.gate.s.blocks / unit, s) * unit + 2);
        if (cost < least) {
            least = cost;
            split = s;
        }
    }
    return split;
}

template <int G, int DEPTH>
int up_launch(const MoeArgs& p, cudaStream_t stream) {
    static std::atomic<uint64_t> set{0};
    ZK_TRY(allow_shared(reinterpret_cast<const void*>(k_moe_up<G, DEPTH>), kMaxShared, &set));
    return launch(k_moe_up<G, DEPTH>, dim3(kSms), kThreads, up_shared(p.m, p.stride, p.etiles, DEPTH), 2, stream, p);
}

template <int G>
int moe_launch(MoeArgs p, cudaStream_t stream) {
    p.split = up_split(p, G == 128 ? 2 : 1);
    const int rc = up_shared(p.m, p.stride, p.etiles, kUpDeep) <= kMaxShared ? up_launch<G, kUpDeep>(p, stream)
                                                                             : up_launch<G, kUpShallow>(p, stream);
    if (rc) return rc;
    static std::atomic<uint64_t> set{0};
    ZK_TRY(allow_shared(reinterpret_cast<const void*>(k_moe_down<G>), kMaxShared, &set));
    const size_t shared = (size_t)kWarps * kDownDepth * kDownSlot + 8ull * (p.m * p.top_k + p.m) * 32;
    return launch(k_moe_down<G>, dim3((p.down.s.tiles + 1) / 2 * 2), kThreads, shared, 2, stream, p);
}

}  // namespace

}  // namespace zk

using namespace zk;

extern "C" {

uint64_t zkie2_moe_router_words(uint64_t h, uint64_t experts, uint32_t group) {
    Q4Shape s;
    if (experts == 0 || experts > kMaxExperts || !q4_shape(h, 16, group, 0, &s)) return 0;
    return ceil_div(experts, 16) * s.blocks * 512;
}

int zkie2_moe_router_pack(const uint64_t* d_w, uint64_t h, uint64_t experts, uint32_t group, uint32_t* d_packed,
                          uint32_t* d_err, cudaStream_t stream) {
    Q4Shape s;
    if (experts == 0 || experts > kMaxExperts || !q4_shape(h, 16, group, 0, &s) || !d_w || !d_packed || !d_err)
        return (int)cudaErrorInvalidValue;
    const uint64_t blocks = ceil_div(ceil_div(experts, 16) * s.blocks * 512, 256);
    k_moe_router_pack<<<(unsigned)(blocks < kSms * 16 ? blocks : kSms * 16), 256, 0, stream>>>(
        d_w, (uint32_t)h, (uint32_t)experts, s.blocks, (uint32_t)ceil_div(experts, 16), d_packed, d_err);
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
                   const uint32_t* const* h_codes, const uint32_t* const* h_scales, const uint64_t* d_exp_table,
                   uint64_t exp_len, const uint64_t* d_silu_table, uint64_t silu_len, uint32_t shift,
                   const uint64_t* d_residual, uint64_t ldr, uint64_t* d_out, uint64_t* d_gate, uint32_t* d_err,
                   uint64_t* d_scratch, cudaStream_t stream) {
    MoeShapes s;
    if (!moe_shapes(h, experts, top_k, f, shared_f, group, &s) || m > 65535 || shift > 62 || !d_router || !h_codes ||
        !h_scales || !d_exp_table || exp_len == 0 || !d_silu_table || silu_len == 0 || !d_err || (m > 1 && ldx < h) ||
        (d_residual && m > 1 && ldr < h) || ((uintptr_t)d_router & 15) || ((uintptr_t)d_scratch & 15))
        return (int)cudaErrorInvalidValue;
    for (int i = 0; i < 6; i++)
        if (!h_codes[i] || !h_scales[i] || ((uintptr_t)h_codes[i] & 15)) return (int)cudaErrorInvalidValue;
    if (m == 0) return 0;
    if (!d_x || !d_out || !d_scratch) return (int)cudaErrorInvalidValue;
    MoeArgs p{};
    const Q4Shape* shape[6] = {&s.up, &s.up, &s.down, &s.sup, &s.sup, &s.sdown};
    Q4Weight* weight[6] = {&p.gate, &p.up, &p.down, &p.sgate, &p.sup, &p.sdown};
    for (int i = 0; i < 6; i++)
        *weight[i] = Q4Weight{reinterpret_cast<const uint4*>(h_codes[i]), h_scales[i], *shape[i]};
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
    const uint32_t most = tokens_at_once(p.stride, p.etiles);
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
        const int rc = group == 32 ? moe_launch<32>(p, stream) : group == 64 ? moe_launch<64>(p, stream)
                                                                              : moe_launch<128>(p, stream);
        if (rc) return rc;
    }
    return 0;
}

}  // extern "C"
