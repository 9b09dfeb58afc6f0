// decode_moe.cu -- a whole mixture-of-experts layer (build_moe of
// models/deepseek-v2-lite/src/lib.rs:252-470) for a few tokens, in two
// kernels and bit-identical to the graph's rows: router MatMul, Scale,
// StableSoftmaxIndex, Softmax, TopKSelect; per chosen expert the gate and up
// products, SiLU by lookup, ScaleVec and the down product; the gate values
// and the sum over experts; the shared experts.  Weights are held in 4 bits
// (q4.cuh), the router in two signed bytes.
//
// Work is bound by the weights' bytes, each expert that some token chose
// being read once for all of its tokens (up to eight at a time):
// - k_moe_up: a cluster computes the logits of all experts (a block to each
//   16), every block then ranks them and lists the experts' tokens, and the
//   blocks share out the tiles of 16 hidden columns of the chosen and the
//   shared experts, gate and up side by side, whose activation is stored as
//   the byte digits that the next product reads;
// - k_moe_down: a block to each 16 output columns runs over all experts, so
//   that the rounding after each expert's product and the sum over experts
//   need no second pass.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/zkie2.h"
#include "common.cuh"
#include "fixed.cuh"
#include "gl64.cuh"
#include "q4.cuh"

namespace cg = cooperative_groups;

namespace zk {

namespace {

constexpr uint32_t kErrDivide = 2u;
constexpr int kSms = 148;
constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr uint32_t kMaxTokens = 16;   // tokens of one launch
constexpr uint32_t kMaxTop = 16;
constexpr uint32_t kMaxExperts = 256;
constexpr uint32_t kTile = 8;         // tokens of an expert taken at a time
constexpr uint32_t kMaxSlots = kMaxTokens * kMaxTop;
constexpr int kClusterUp = 4;
constexpr size_t kMaxShared = 226 * 1024;
constexpr int32_t kRouterLimit = 32639;  // two signed bytes

struct Q4Weight {
    const uint4* codes;
    const uint32_t* scales;
    Q4Shape s;
};

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
    uint32_t* sel;       // m x top_k: the chosen experts, best first
    int64_t* score;      // m x top_k: their softmax values
    uint8_t* act;        // (m top_k) x 4 x padded F digits
    uint8_t* sact;       // m x 4 x padded shared F digits
    uint32_t* err;
    uint32_t stride;     // bytes of a digit row of x
};

// The tokens of the chosen experts, up to kTile of one expert to an item.
struct Items {
    uint32_t n;
    uint8_t expert[kMaxSlots];
    uint8_t count[kMaxSlots];
    uint16_t first[kMaxSlots];  // into slot
    uint16_t slot[kMaxSlots];   // token top_k + place, grouped by expert
};

// sel (m x top_k, shared memory) -> items; the whole block
__device__ void list_items(const uint32_t* sel, uint32_t m, uint32_t top_k, uint32_t experts, Items* it,
                           uint32_t* count, uint32_t* start) {
    const uint32_t slots = m * top_k;
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < experts; e += kThreads) {
        uint32_t c = 0;
        for (uint32_t i = 0; i < slots; i++) c += sel[i] == e;
        count[e] = c;
    }
    __syncthreads();
    if (threadIdx.x < 32) {  // running sums over the experts: places of their slots and items
        uint32_t slot = 0, item = 0;
        for (uint32_t e0 = 0; e0 < experts; e0 += 32) {
            const uint32_t e = e0 + threadIdx.x, c = e < experts ? count[e] : 0, i = (c + kTile - 1) / kTile;
            uint32_t sc = c, si = i;
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t a = __shfl_up_sync(0xFFFFFFFFu, sc, o), b = __shfl_up_sync(0xFFFFFFFFu, si, o);
                if ((int)threadIdx.x >= o) {
                    sc += a;
                    si += b;
                }
            }
            const uint32_t at = slot + sc - c;
            if (e < experts) start[e] = at;
            for (uint32_t j = 0; j < i; j++) {
                const uint32_t k = item + si - i + j;
                it->expert[k] = (uint8_t)e;
                it->count[k] = (uint8_t)min(kTile, c - j * kTile);
                it->first[k] = (uint16_t)(at + j * kTile);
            }
            slot += __shfl_sync(0xFFFFFFFFu, sc, 31);
            item += __shfl_sync(0xFFFFFFFFu, si, 31);
        }
        if (threadIdx.x == 0) it->n = item;
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < slots; i += kThreads) {
        const uint32_t e = sel[i];
        uint32_t before = 0;
        for (uint32_t j = 0; j < i; j++) before += sel[j] == e;
        it->slot[start[e] + before] = (uint16_t)i;
    }
    __syncthreads();
}

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

// Logits of the 16 experts of a tile for all tokens, this warp's part of K,
// added to raw (tokens x padded experts, 64-bit sums in shared memory)
template <int NT>
__device__ void router_part(const MoeArgs& p, const uint8_t* digits, uint32_t tile, unsigned long long* raw) {
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint32_t blocks = p.gate.s.blocks, b0 = warp * blocks / kWarps, b1 = (warp + 1) * blocks / kWarps;
    int c[2][NT][4];
#pragma unroll
    for (int w = 0; w < 2; w++)
#pragma unroll
        for (int i = 0; i < NT; i++) c[w][i][0] = c[w][i][1] = c[w][i][2] = c[w][i][3] = 0;
    for (uint32_t b = b0; b < b1; b++) {
        const uint4* r = p.router + ((uint64_t)tile * blocks + b) * 128 + lane;
        const uint4 w00 = __ldg(r), w01 = __ldg(r + 32), w10 = __ldg(r + 64), w11 = __ldg(r + 96);
#pragma unroll
        for (int i = 0; i < NT; i++) {
            const uint32_t tok = min(2 * i + (g >> 2), p.m - 1);
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
        const uint32_t tok = 2 * i + (t >> 1);
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

// Gate and up of one tile of 16 hidden columns for up to 2 NT tokens: this
// warp's part of K into red (mat, token, column)
template <int G, int NT>
__device__ void up_tile(const Q4Weight& wg, const Q4Weight& wu, uint64_t tile, uint32_t b0, uint32_t b1,
                        const uint8_t* const (&from)[4], long long* red) {
    const uint32_t lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint4* cgp = wg.codes + tile * wg.s.blocks * 32 + lane;
    const uint4* cup = wu.codes + tile * wu.s.blocks * 32 + lane;
    const uint32_t* sgp = wg.scales + tile * wg.s.groups * 8;
    const uint32_t* sup = wu.scales + tile * wu.s.groups * 8;
    Q4Sum<NT> a, b;
    a.clear();
    b.clear();
    for (uint32_t k = b0; k < b1; k += 2) {
        uint4 w[2], v[2];
        uint32_t ws[2][2], vs[2][2];
#pragma unroll
        for (int j = 0; j < 2; j++)
            if (k + j < b1) {
                w[j] = ldg_stream(cgp + (uint64_t)(k + j) * 32);
                v[j] = ldg_stream(cup + (uint64_t)(k + j) * 32);
                q4_scales<G>(sgp, k + j, g, &ws[j][0], &ws[j][1]);
                q4_scales<G>(sup, k + j, g, &vs[j][0], &vs[j][1]);
            }
#pragma unroll
        for (int j = 0; j < 2; j++)
            if (k + j < b1) {
                uint4 x[NT];
#pragma unroll
                for (int i = 0; i < NT; i++) x[i] = *reinterpret_cast<const uint4*>(from[i] + (k + j) * 64);
                q4_block<G, NT>(a, w[j], ws[j][0], ws[j][1], x, (k + j) & 1);
                q4_block<G, NT>(b, v[j], vs[j][0], vs[j][1], x, (k + j) & 1);
            }
    }
#pragma unroll
    for (int i = 0; i < NT; i++) {
        long long v0, v1, u0, u1;
        a.finish(i, &v0, &v1);
        b.finish(i, &u0, &u1);
        if (!(t & 1)) {
            long long* to = red + (2 * i + (t >> 1)) * 16;
            to[g] = v0;
            to[g + 8] = v1;
            to[kTile * 16 + g] = u0;
            to[kTile * 16 + g + 8] = u1;
        }
    }
}

constexpr size_t kRedBytes = 2ull * kWarps * 2 * kTile * 16 * 8;  // two buffers of every warp's sums

template <int G>
__global__ void __launch_bounds__(kThreads, 1) k_moe_up(const MoeArgs p) {
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ Items items;
    __shared__ uint32_t s_count[kMaxExperts], s_start[kMaxExperts], s_sel[kMaxSlots];
    __shared__ long long s_score[kMaxSlots];
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    // red (the tiles' sums) and, before it is used, the logits
    long long* red = reinterpret_cast<long long*>(smem);
    uint8_t* digits = smem + kRedBytes;
    const uint32_t pitch = p.etiles * 16;
    unsigned long long* raw = reinterpret_cast<unsigned long long*>(smem);
    long long* logit = reinterpret_cast<long long*>(smem) + kMaxTokens * pitch;

    for (uint32_t i = threadIdx.x; i < p.m * pitch; i += kThreads) raw[i] = 0;
    const uint32_t kp = p.gate.s.blocks * 64, quads = kp / 4;
    bool bad = false;
    for (uint32_t i = threadIdx.x; i < p.m * quads; i += kThreads) {
        const uint32_t r = i / quads, k0 = (i % quads) * 4;
        const uint64_t* xr = p.x + r * p.ldx + k0;
        uint32_t d[4];
#pragma unroll
        for (int j = 0; j < 4; j++) bad |= !q4_digits(k0 + j < p.h ? fx_to_i64(__ldg(xr + j)) : 0, &d[j]);
        uint8_t* to = digits + (size_t)r * 4 * p.stride + q4_pos(k0);
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const uint32_t lo = __byte_perm(d[0], d[1], q | ((4 + q) << 4));
            const uint32_t hi = __byte_perm(d[2], d[3], q | ((4 + q) << 4));
            *reinterpret_cast<uint32_t*>(to + (size_t)q * p.stride) = __byte_perm(lo, hi, 0x5410);
        }
    }
    __syncthreads();

    // ---- routing
    const uint32_t ranks = cluster.num_blocks(), rank = cluster.block_rank();
    for (uint32_t tile = rank; tile < p.etiles; tile += ranks) {
        if (p.m > 8)
            router_part<8>(p, digits, tile, raw);
        else if (p.m > 2)
            router_part<4>(p, digits, tile, raw);
        else
            router_part<1>(p, digits, tile, raw);
    }
    cluster.sync();
    for (uint32_t i = threadIdx.x; i < p.m * pitch; i += kThreads) {
        const unsigned long long v = *cluster.map_shared_rank(&raw[i], (i % pitch / 16) % ranks);
        logit[i] = fx_round_div_pow2((int64_t)v, p.shift);
    }
    __syncthreads();
    for (uint32_t r = warp; r < p.m; r += kWarps) {
        long long* row = logit + r * pitch;
        long long top = INT64_MIN;
        for (uint32_t e = lane; e < p.experts; e += 32) top = max(top, row[e]);
        for (int o = 16; o; o >>= 1) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
        long long sum = 0;
        for (uint32_t e = lane; e < p.experts; e += 32) {
            int64_t v = fx_to_i64(table_at(p.exp_table, p.exp_len, fx_wsub(row[e], top), (int64_t)p.exp_len));
            if (v < 0 || v > INT32_MAX) {
                bad = true;
                v = 0;
            }
            row[e] = v;
            sum += v;
        }
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
        if (sum == 0 && lane == 0) atomicOr(p.err, kErrDivide);
        const double inv = sum ? 1.0 / (double)sum : 0.0;
        for (uint32_t e = lane; e < p.experts; e += 32) row[e] = sum ? round_div_near(row[e] << 16, sum, inv) : 0;
        __syncwarp();
        for (uint32_t e = lane; e < p.experts; e += 32) {
            const long long v = row[e];
            uint32_t before = 0;
            for (uint32_t j = 0; j < p.experts; j++) before += row[j] > v || (row[j] == v && j < e);
            if (before < p.top_k) {
                s_sel[r * p.top_k + before] = e;
                s_score[r * p.top_k + before] = v;
            }
            if (p.gate_out && blockIdx.x == 0)
                p.gate_out[(uint64_t)r * p.experts + e] = before < p.top_k ? (uint64_t)v : 0;
        }
    }
    __syncthreads();
    if (blockIdx.x == 0)
        for (uint32_t i = threadIdx.x; i < p.m * p.top_k; i += kThreads) {
            p.sel[i] = s_sel[i];
            p.score[i] = s_score[i];
        }
    list_items(s_sel, p.m, p.top_k, p.experts, &items, s_count, s_start);
    cluster.sync();  // the other blocks have read this one's logits: red may take their place

    // ---- gate and up
    const uint32_t ft = p.gate.s.tiles, st = p.sgate.s.tiles, stiles = st * ((p.m + kTile - 1) / kTile);
    const uint32_t units = stiles + ft * items.n, blocks = p.gate.s.blocks, unit = G == 128 ? 2 : 1;
    // Warps to a tile: fewest steps (as in the projection)
    uint32_t split = 1;
    {
        uint32_t least = ~0u;
        for (uint32_t s = 1; s <= (uint32_t)kWarps; s *= 2) {
            const uint32_t at_once = gridDim.x * (kWarps / s);
            const uint32_t cost = (units + at_once - 1) / at_once * ((blocks / unit + s - 1) / s * unit + 2);
            if (cost < least) {
                least = cost;
                split = s;
            }
        }
    }
    const uint32_t per = kWarps / split, mine = warp / split, part = warp % split;
    const uint32_t b0 = part * (blocks / unit) / split * unit, b1 = (part + 1) * (blocks / unit) / split * unit;
    const uint64_t fp = (uint64_t)p.down.s.blocks * 64, sp = (uint64_t)p.sdown.s.blocks * 64;
    uint32_t flip = 0;
    for (uint32_t u = blockIdx.x + gridDim.x * mine; u < units; u += gridDim.x * per, flip ^= 1) {
        const bool shared = u < stiles;
        const uint32_t item = shared ? u / st : (u - stiles) / ft, tile = shared ? u % st : (u - stiles) % ft;
        const uint32_t first = shared ? item * kTile : items.first[item];
        const uint32_t count = shared ? min(kTile, p.m - first) : items.count[item];
        const uint8_t* from[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t at = min(2 * i + (g >> 2), count - 1);
            const uint32_t tok = shared ? first + at : items.slot[first + at] / p.top_k;
            from[i] = digits + (size_t)(tok * 4 + (g & 3)) * p.stride + 16 * t;
        }
        const Q4Weight& wg = shared ? p.sgate : p.gate;
        const Q4Weight& wu = shared ? p.sup : p.up;
        const uint64_t at = shared ? tile : (uint64_t)items.expert[item] * ft + tile;
        long long* to = red + (size_t)(flip * kWarps + warp) * (2 * kTile * 16);
        if (count > 4)
            up_tile<G, 4>(wg, wu, at, b0, b1, from, to);
        else if (count > 2)
            up_tile<G, 2>(wg, wu, at, b0, b1, from, to);
        else
            up_tile<G, 1>(wg, wu, at, b0, b1, from, to);
        if (split > 1)
            group_sync(1 + mine, split * 32);
        else
            __syncwarp();
        for (uint32_t o = part * 32 + lane; o < count * 16; o += split * 32) {
            const uint32_t c = o & 15, j = o >> 4, f = tile * 16 + c;
            if (f >= (shared ? p.sgate.s.n : p.gate.s.n)) continue;
            uint64_t gv = 0, uv = 0;
            for (uint32_t w = 0; w < split; w++) {
                const long long* q = red + (size_t)(flip * kWarps + mine * split + w) * (2 * kTile * 16) + j * 16 + c;
                gv += (uint64_t)q[0];
                uv += (uint64_t)q[kTile * 16];
            }
            const int64_t gi = fx_round_div_pow2((int64_t)gv, p.shift), ui = fx_round_div_pow2((int64_t)uv, p.shift);
            const int64_t s = fx_to_i64(table_at(p.silu, p.silu_len, gi, (int64_t)(p.silu_len / 2)));
            uint32_t d;
            bad |= !q4_digits(fx_round_div_pow2(fx_wmul(s, ui), p.shift), &d);
            const uint64_t row = shared ? sp : fp;
            uint8_t* a = (shared ? p.sact + (first + j) * 4 * row : p.act + items.slot[first + j] * 4 * row) + q4_pos(f);
#pragma unroll
            for (int q = 0; q < 4; q++) a[q * row] = (uint8_t)(d >> (8 * q));
        }
    }
    if (bad) atomicOr(p.err, kErrRange);
}

// This warp's blocks [b0, b1) of one expert's tile of 16 output columns for
// up to 2 NT slots, digits read from memory, added to raw (slot, column)
template <int G, int NT>
__device__ void down_part(const Q4Weight& w, uint64_t tile, uint32_t b0, uint32_t b1, const uint8_t* const (&from)[4],
                          uint32_t count, const uint16_t* slots, unsigned long long* raw) {
    const uint32_t lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint4* cp = w.codes + tile * w.s.blocks * 32 + lane;
    const uint32_t* sp = w.scales + tile * w.s.groups * 8;
    Q4Sum<NT> a;
    a.clear();
    constexpr int kAhead = NT == 4 ? 2 : 4;
    for (uint32_t k = b0; k < b1; k += kAhead) {
        uint4 v[kAhead], x[kAhead][NT];
        uint32_t s[kAhead][2];
#pragma unroll
        for (int j = 0; j < kAhead; j++)
            if (k + j < b1) {
                v[j] = ldg_stream(cp + (uint64_t)(k + j) * 32);
                q4_scales<G>(sp, k + j, g, &s[j][0], &s[j][1]);
#pragma unroll
                for (int i = 0; i < NT; i++) x[j][i] = __ldg(reinterpret_cast<const uint4*>(from[i] + (k + j) * 64));
            }
#pragma unroll
        for (int j = 0; j < kAhead; j++)
            if (k + j < b1) q4_block<G, NT>(a, v[j], s[j][0], s[j][1], x[j], (k + j) & 1);
    }
#pragma unroll
    for (int i = 0; i < NT; i++) {
        long long v0, v1;
        a.finish(i, &v0, &v1);
        const uint32_t at = 2 * i + (t >> 1);
        if (!(t & 1) && at < count) {
            const uint32_t slot = slots ? slots[at] : at;
            atomicAdd(&raw[slot * 16 + g], (unsigned long long)v0);
            atomicAdd(&raw[slot * 16 + g + 8], (unsigned long long)v1);
        }
    }
}

template <int G>
__global__ void __launch_bounds__(kThreads, 1) k_moe_down(const MoeArgs p) {
    __shared__ Items items;
    __shared__ uint32_t s_count[kMaxExperts], s_start[kMaxExperts], s_sel[kMaxSlots];
    __shared__ unsigned long long raw[(kMaxSlots + kMaxTokens) * 16];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint32_t slots = p.m * p.top_k;
    for (uint32_t i = threadIdx.x; i < slots; i += kThreads) s_sel[i] = p.sel[i];
    list_items(s_sel, p.m, p.top_k, p.experts, &items, s_count, s_start);
    const uint32_t unit = G == 128 ? 2 : 1, nf = p.down.s.blocks / unit, ns = p.sdown.s.blocks / unit;
    const uint32_t stiles = (p.m + kTile - 1) / kTile, total = nf * items.n + ns * stiles;
    const uint64_t fp = (uint64_t)p.down.s.blocks * 64, sp = (uint64_t)p.sdown.s.blocks * 64;
    for (uint32_t tile = blockIdx.x; tile < p.down.s.tiles; tile += gridDim.x) {
        for (uint32_t i = threadIdx.x; i < (slots + p.m) * 16; i += kThreads) raw[i] = 0;
        __syncthreads();
        // the warp's run of the experts' blocks, one after another
        uint32_t at = (uint32_t)((uint64_t)warp * total / kWarps);
        const uint32_t end = (uint32_t)((uint64_t)(warp + 1) * total / kWarps);
        while (at < end) {
            const bool shared = at >= nf * items.n;
            const uint32_t in = shared ? at - nf * items.n : at, len = shared ? ns : nf;
            const uint32_t item = in / len, first = in % len, stop = min(len, first + end - at);
            at += stop - first;
            const uint32_t s0 = shared ? item * kTile : items.first[item];
            const uint32_t count = shared ? min(kTile, p.m - s0) : items.count[item];
            const uint8_t* from[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t j = min(2 * i + (g >> 2), count - 1);
                from[i] = (shared ? p.sact + ((uint64_t)(s0 + j) * 4 + (g & 3)) * sp
                                  : p.act + ((uint64_t)items.slot[s0 + j] * 4 + (g & 3)) * fp) + 16 * t;
            }
            const Q4Weight& w = shared ? p.sdown : p.down;
            const uint64_t tl = shared ? tile : (uint64_t)items.expert[item] * p.down.s.tiles + tile;
            const uint16_t* list = shared ? nullptr : items.slot + s0;
            unsigned long long* to = raw + (shared ? (size_t)(slots + s0) * 16 : 0);
            if (count > 4)
                down_part<G, 4>(w, tl, first * unit, stop * unit, from, count, list, to);
            else if (count > 2)
                down_part<G, 2>(w, tl, first * unit, stop * unit, from, count, list, to);
            else
                down_part<G, 1>(w, tl, first * unit, stop * unit, from, count, list, to);
        }
        __syncthreads();
        for (uint32_t o = threadIdx.x; o < p.m * 16; o += kThreads) {
            const uint32_t c = o & 15, r = o >> 4;
            const uint64_t n = (uint64_t)tile * 16 + c;
            if (n >= p.h) continue;
            int64_t y = fx_round_div_pow2((int64_t)raw[(slots + r) * 16 + c], p.shift);
            for (uint32_t j = 0; j < p.top_k; j++) {
                const int64_t d = fx_round_div_pow2((int64_t)raw[(r * p.top_k + j) * 16 + c], p.shift);
                y = fx_wadd(y, fx_round_div_pow2(fx_wmul(d, p.score[r * p.top_k + j]), 16));
            }
            uint64_t f = fx_from_i64(y);
            if (p.residual) f = gl_canon(gl_add(f, gl_canon(__ldg(p.residual + r * p.ldr + n))));
            p.out[r * (uint64_t)p.h + n] = f;
        }
        __syncthreads();
    }
}

uint32_t row_stride(uint32_t blocks) { return blocks % 2 ? blocks * 64 : blocks * 64 + 64; }

uint32_t tokens_at_once(uint32_t stride) {
    const uint64_t room = (kMaxShared - 16 * 1024 - kRedBytes) / (4ull * stride);
    return (uint32_t)(room < kMaxTokens ? room : kMaxTokens);
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

template <int G>
int moe_launch(const MoeArgs& p, cudaStream_t stream) {
    const size_t shared = kRedBytes + 4ull * p.m * p.stride;
    auto* kernel = k_moe_up<G>;
    ZK_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(kMaxShared - 16 * 1024)));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(kSms);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = shared;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = kClusterUp;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    ZK_TRY(cudaLaunchKernelEx(&cfg, kernel, p));
    k_moe_down<G><<<p.down.s.tiles < (uint32_t)kSms ? p.down.s.tiles : kSms, kThreads, 0, stream>>>(p);
    ZK_LAUNCH_CHECK();
    return 0;
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
    // scores, chosen experts, digits of the activations
    return slots + ceil_div(slots, 2) + 1 + (slots * 4 * s.down.blocks * 64 + t * 4 * s.sdown.blocks * 64) / 8;
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
    p.stride = row_stride(s.up.blocks);
    const uint32_t most = tokens_at_once(p.stride);
    const uint64_t slots = (m < kMaxTokens ? m : kMaxTokens) * top_k;
    p.act = reinterpret_cast<uint8_t*>(d_scratch);
    p.sact = p.act + slots * 4 * s.down.blocks * 64;
    p.score = reinterpret_cast<int64_t*>(p.sact + (m < kMaxTokens ? m : kMaxTokens) * 4 * s.sdown.blocks * 64);
    p.sel = reinterpret_cast<uint32_t*>(p.score + slots);
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
