// decode.cu -- the forward of single tokens: what a step of generation needs
// of the op layer, for a few rows instead of a whole sequence, with every
// result bit-identical to the same row of the graph's forward_ops.
//
// - k_q4_pack / k_q4_project: Op::Projection and Op::MatMul for a few rows by
//   a weight in 4 bits with group scales (q4.cuh), the rounding, bias,
//   activation table and residual in its epilogue;
// - k_kv_append / k_kv_attend: one new token per sequence against a cache of
//   the keys and values (Scale, MatMul, Scale, StableSoftmaxIndex, Softmax,
//   MatMul, Scale of one row);
// - k_choose_token: penalties, bias and mask on the logits and Op::Argmax.
//
// Tensors are rows of field elements as everywhere in the op layer.  Data
// outside what a kernel takes sets a bit of the caller's error word
// (kErrIndex, kErrDivide, kErrRange, kErrFull) and the pass carries on.
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

constexpr uint32_t kErrIndex = 1u;
constexpr uint32_t kErrDivide = 2u;
constexpr uint32_t kErrFull = 16u;  // a cache without room for the new token
constexpr size_t kMaxShared = 226 * 1024;  // dynamic, next to what is declared

// ---- the weight ---------------------------------------------------------------------------
// codes (e x k x n, int8) and scales (e x rows x n, int32; ceil(k_seg / G)
// rows to a segment) into blocks: one thread per output word
__global__ void k_q4_pack(const int8_t* __restrict__ codes, const int32_t* __restrict__ scales, uint32_t experts,
                          Q4Shape s, uint32_t* __restrict__ packed, uint32_t* __restrict__ err) {
    const uint64_t stride = (uint64_t)gridDim.x * blockDim.x, first = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x;
    const uint32_t words = s.bytes / 4, seg_blocks = s.kp_seg / 64, rows = (s.k_seg + s.group - 1) / s.group;
    const uint64_t per = (uint64_t)s.tiles * s.blocks * words;
    bool bad = false;
    for (uint64_t i = first; i < per * experts; i += stride) {
        const uint64_t ex = i / per, r = i % per;
        const uint32_t at = (uint32_t)(r % words), block = (uint32_t)(r / words % s.blocks);
        const uint32_t tile = (uint32_t)(r / words / s.blocks), seg = block / seg_blocks;
        const uint32_t k0 = block % seg_blocks * 64;  // within the segment
        uint32_t word = 0;
        if (at < 128) {
            const uint32_t q = at & 3, lane = at >> 2, t = lane & 3, n = tile * 16 + (lane >> 2) + 8 * (q & 1);
            for (int j = 0; j < 4; j++)
                for (int h = 0; h < 2; h++) {
                    const uint32_t k = k0 + 32 * h + 8 * t + 4 * (q >> 1) + j;
                    int c = 0;
                    if (k < s.k_seg && n < s.n) c = codes[(ex * s.k + (uint64_t)seg * s.k_seg + k) * s.n + n];
                    if (c < -8 || c > 7) {
                        bad = true;
                        c = 0;
                    }
                    word |= (uint32_t)(c & 15) << (8 * j + 4 * h);
                }
        } else {
            const uint32_t in = (k0 + 32 * ((at - 128) >> 3)) / s.group;  // row of scales within the segment
            for (int h = 0; h < 2; h++) {
                const uint32_t n = tile * 16 + (at & 7) + 8 * h;
                int64_t v = 0;
                if (in < rows && n < s.n) v = scales[(ex * s.segs * rows + (uint64_t)seg * rows + in) * s.n + n];
                if (v < 0 || v > 0xFFFF) {
                    bad = true;
                    v = 0;
                }
                word |= (uint32_t)v << (16 * h);
            }
        }
        packed[i] = word;
    }
    if (bad) atomicOr(err, kErrRange);
}

// ---- the product ----------------------------------------------------------------------------
constexpr int kProjThreads = 512;
constexpr int kProjWarps = kProjThreads / 32;

struct ProjectArgs {
    const uint64_t* x;
    uint64_t ldx;
    uint32_t m;
    const uint8_t* w;
    Q4Shape s;
    uint32_t shift;
    const uint64_t* bias;
    const uint64_t* table;
    uint64_t table_len;
    int64_t offset;
    const uint64_t* residual;
    uint64_t ldr;
    uint64_t* out;
    uint32_t* err;
    uint32_t stride;  // bytes of a digit row in shared memory
    uint32_t run;     // blocks to a slot of a ring
};

constexpr int kProjDepth = 3;           // slots of a warp's ring
constexpr uint32_t kProjBatch = 16;     // tiles whose sums are held at a time

// A block takes an equal run of the tiles of 16 columns, in batches; of a
// batch every warp takes an equal run of blocks (of whole segments where each
// is rounded by itself), whatever tiles they belong to, against the digits of
// 2 NT rows in shared memory.  The 64-bit sums meet in shared memory; a thread
// per output then rounds and finishes it.
template <bool TWO, int NT, bool SEG>
__global__ void __launch_bounds__(kProjThreads, 1) k_q4_project(const __grid_constant__ ProjectArgs p) {
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ __align__(8) uint64_t s_bar[kProjWarps * kProjDepth];
    constexpr uint32_t kRows = 2 * NT, kBytes = TWO ? 576 : 544;
    const uint32_t row0 = blockIdx.y * kRows, rows = min(kRows, p.m - row0);
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint32_t slot_bytes = p.run * kBytes;
    uint8_t* ring = smem + (size_t)warp * kProjDepth * slot_bytes;
    constexpr uint32_t kCells = kProjBatch * kRows * 16;  // (tile, row, column)
    const Limbs acc{reinterpret_cast<uint32_t*>(smem + (size_t)kProjWarps * kProjDepth * slot_bytes), kCells};
    uint8_t* digits = reinterpret_cast<uint8_t*>(acc.w + 3 * kCells);
    const uint32_t bar = shared_addr(&s_bar[warp * kProjDepth]);
    let_next_start();
    if (lane == 0) {
#pragma unroll
        for (int i = 0; i < kProjDepth; i++) barrier_init(bar + 8 * i);
        barrier_init_done();
    }
    __syncwarp();

    // ---- this warp's stream of blocks, and the first of them on their way
    const uint32_t tile0 = (uint32_t)((uint64_t)blockIdx.x * p.s.tiles / gridDim.x);
    const uint32_t tile1 = (uint32_t)((uint64_t)(blockIdx.x + 1) * p.s.tiles / gridDim.x);
    const uint32_t blocks = p.s.blocks, unit = SEG ? p.s.kp_seg / 64 : 1;
    // blocks of a batch, counted from its first tile, that the warp takes
    auto first_of = [&](uint32_t batch, uint32_t w) {
        const uint32_t units = min(kProjBatch, tile1 - batch) * blocks / unit;
        return (uint32_t)((uint64_t)w * units / kProjWarps) * unit;
    };
    uint32_t next_batch = tile0, next_at = first_of(tile0, warp), next_end = first_of(tile0, warp + 1), next_slot = 0;
    auto ask = [&]() {  // lane 0 only
        while (next_at == next_end) {
            next_batch += kProjBatch;
            if (next_batch >= tile1) {
                next_batch = tile1;
                return;
            }
            next_at = first_of(next_batch, warp);
            next_end = first_of(next_batch, warp + 1);
        }
        const uint32_t bytes = min(p.run, next_end - next_at) * kBytes;
        barrier_expect(bar + 8 * next_slot, bytes);
        bulk_copy(shared_addr(ring + next_slot * slot_bytes), p.w + ((uint64_t)next_batch * blocks + next_at) * kBytes, bytes,
                  bar + 8 * next_slot);
        next_at = min(next_at + p.run, next_end);
        next_slot = next_slot + 1 == kProjDepth ? 0 : next_slot + 1;
    };
    if (lane == 0)
        for (int i = 0; i < kProjDepth; i++)
            if (next_batch < tile1) ask();

    // ---- the rows' digits
    for (uint32_t i = threadIdx.x; i < 3 * kCells; i += kProjThreads) acc.w[i] = 0;
    wait_for_previous();
    if (!q4_digitise<kProjThreads>(p.x + (uint64_t)row0 * p.ldx, p.ldx, rows, p.s.segs, p.s.k_seg, p.s.kp_seg, digits,
                                   p.stride))
        atomicOr(p.err, kErrRange);
    __syncthreads();

    const uint8_t* from = digits + (size_t)g * p.stride + 16 * t;  // column g: digit g % 4 of row g / 4
    Patience patience;
    uint32_t slot = 0, phase = 0;
    for (uint32_t batch = tile0; batch < tile1; batch += kProjBatch) {
        uint32_t at = first_of(batch, warp);
        const uint32_t end = first_of(batch, warp + 1);
        uint32_t tile = at / blocks, b = at % blocks;
        Q4Sum<NT> sum;
        sum.clear();
        long long total[NT];  // of the tile's segments, each rounded
#pragma unroll
        for (int i = 0; i < NT; i++) total[i] = 0;
        auto flush = [&]() {
#pragma unroll
            for (int i = 0; i < NT; i++) {
                if (!SEG) total[i] = sum.finish(i);
                const uint32_t r = 2 * i + (t >> 1);
                if (r < rows) acc.add((tile * kRows + r) * 16 + g + 8 * (t & 1), total[i]);
                total[i] = 0;
            }
            if (!SEG) sum.clear();
        };
        while (at < end) {
            const uint32_t run = min(p.run, end - at);
            barrier_wait(bar + 8 * slot, phase, patience);
            const uint8_t* block = ring + slot * slot_bytes;
            for (uint32_t j = 0; j < run;) {
                // blocks up to the end of the tile (or segment)
                const uint32_t n = min(run - j, (SEG ? unit - b % unit : blocks - b));
#pragma unroll 2
                for (uint32_t q = 0; q < n; q++) {
                    uint4 x[NT];
#pragma unroll
                    for (int i = 0; i < NT; i++)
                        x[i] = *reinterpret_cast<const uint4*>(from + (size_t)i * 8 * p.stride + (b + q) * 64);
                    q4_block<TWO, NT, NT>(sum, block + q * kBytes, x);
                }
                j += n;
                b += n;
                block += n * kBytes;
                if (SEG && b % unit == 0) {
#pragma unroll
                    for (int i = 0; i < NT; i++) total[i] += round_shift(sum.finish(i), p.shift);
                    sum.clear();
                }
                if (b == blocks) {
                    flush();
                    b = 0;
                    tile++;
                }
            }
            at += run;
            __syncwarp();  // every lane has read the slot
            if (lane == 0 && next_batch < tile1) ask();
            if (++slot == kProjDepth) {
                slot = 0;
                phase ^= 1;
            }
        }
        if (b) flush();
        __syncthreads();
        const uint32_t tiles = min(kProjBatch, tile1 - batch);
        constexpr int kOuts = 4;  // outputs of a thread whose operands are under way together
        for (uint32_t o0 = threadIdx.x; o0 < tiles * kRows * 16; o0 += kProjThreads * kOuts) {
            uint64_t bias[kOuts], residual[kOuts];
#pragma unroll
            for (int u = 0; u < kOuts; u++) {
                const uint32_t o = o0 + u * kProjThreads, r = o / 16 % kRows, n = (batch + o / (kRows * 16)) * 16 + o % 16;
                const bool on = o < tiles * kRows * 16 && r < rows && n < p.s.n;
                bias[u] = on && p.bias ? __ldg(p.bias + n) : 0;
                residual[u] = on && p.residual ? __ldg(p.residual + (row0 + r) * p.ldr + n) : 0;
            }
            int64_t y[kOuts];
#pragma unroll
            for (int u = 0; u < kOuts; u++) {
                const uint32_t o = o0 + u * kProjThreads;
                if (o >= tiles * kRows * 16) continue;
                y[u] = SEG ? acc.get(o) : round_shift(acc.get(o), p.shift);
                acc.clear(o);
                y[u] = fx_wadd(y[u], fx_to_i64(bias[u]));
            }
            uint64_t f[kOuts];
#pragma unroll
            for (int u = 0; u < kOuts; u++)
                f[u] = o0 + u * kProjThreads >= tiles * kRows * 16 ? 0
                       : p.table ? gl_canon(table_at(p.table, p.table_len, y[u], p.offset)) : fx_from_i64(y[u]);
#pragma unroll
            for (int u = 0; u < kOuts; u++) {
                const uint32_t o = o0 + u * kProjThreads, r = o / 16 % kRows, n = (batch + o / (kRows * 16)) * 16 + o % 16;
                if (o < tiles * kRows * 16 && r < rows && n < p.s.n)
                    p.out[(row0 + r) * (uint64_t)p.s.n + n] = p.residual ? gl_canon(gl_add(f[u], gl_canon(residual[u]))) : f[u];
            }
        }
        __syncthreads();
    }
    if (patience.failed && lane == 0) atomicOr(p.err, kErrWait);
}

// dynamic shared memory for blocks of `rows` rows and a ring of `run` blocks to a slot
size_t project_shared(const Q4Shape& s, uint32_t rows, uint32_t run) {
    return (size_t)kProjWarps * kProjDepth * run * s.bytes + (size_t)rows * (kProjBatch * 16 * 12 + 4 * q4_digit_stride(s.blocks));
}

template <bool TWO, int NT, bool SEG>
int project_launch(const ProjectArgs& p, cudaStream_t stream) {
    auto* kernel = k_q4_project<TWO, NT, SEG>;
    static std::atomic<uint64_t> set{0};
    ZK_TRY(allow_shared(reinterpret_cast<const void*>(kernel), kMaxShared, &set));
    const dim3 grid(p.s.tiles < (uint32_t)kSms ? p.s.tiles : kSms, (unsigned)ceil_div(p.m, 2 * NT));
    return launch(kernel, grid, kProjThreads, project_shared(p.s, 2 * NT, p.run), 1, stream, p);
}

template <bool TWO, int NT>
int project_seg(const ProjectArgs& p, cudaStream_t stream) {
    return p.s.segs > 1 ? project_launch<TWO, NT, true>(p, stream) : project_launch<TWO, NT, false>(p, stream);
}

template <bool TWO>
int project_rows(ProjectArgs p, cudaStream_t stream) {
    // Rows to a block: up to eight, as many as their digits leave room for; slots of four blocks
    // (2 kB a copy) where there is room, else of two or one
    for (uint32_t rows = p.m > 4 ? 8 : p.m > 2 ? 4 : 2;; rows /= 2)
        for (p.run = 4; p.run; p.run /= 2)
            if (project_shared(p.s, rows, p.run) <= kMaxShared)
                return rows == 8   ? project_seg<TWO, 4>(p, stream)
                       : rows == 4 ? project_seg<TWO, 2>(p, stream)
                                   : project_seg<TWO, 1>(p, stream);
}

// ---- the cache ------------------------------------------------------------------------------
// Keys lie in blocks of 32 tokens, four dimensions of each token side by side
// (b, head, token / 32, dk / 4, token % 32, 4): a lane takes a token, its
// loads are 16 bytes next to its neighbours', and a score needs no sum over
// lanes.  Values are rows (b, head, token, dv).
constexpr int kKvBlock = 32;
constexpr int64_t kKeyLimit = 1ll << 27;  // |q|, |k| up to here: a score of 256 products stays below 2^62

__device__ __forceinline__ uint64_t key_at(uint64_t head, uint64_t blocks, uint32_t dk, uint64_t tok, uint32_t d) {
    return ((head * blocks + tok / kKvBlock) * (dk / 4) + d / 4) * (4 * kKvBlock) + (tok % kKvBlock) * 4 + d % 4;
}

struct KvCache {
    int32_t* k;
    int32_t* v;
    const int32_t* lens;
    uint32_t batch, heads, dk, dv, cap;
};

struct KvRows {
    const uint64_t* k;
    uint64_t ldk;
    const uint64_t* v;
    uint64_t ldv;
    int64_t factor;
    uint32_t shift;
};

// the d-th number of a new key (d < dk) or value (from dk on) into the cache
__device__ __forceinline__ bool kv_store(const KvCache& c, const KvRows& rows, uint64_t row, uint32_t seq, uint32_t h,
                                         uint64_t tok, uint32_t d) {
    const uint64_t head = (uint64_t)seq * c.heads + h;
    if (d < c.dk) {
        const int64_t x = fx_to_i64(__ldg(rows.k + row * rows.ldk + (uint64_t)h * c.dk + d));
        const int64_t y = fx_round_div_pow2(fx_wmul(x, rows.factor), rows.shift);
        const bool ok = y >= -kKeyLimit && y <= kKeyLimit;
        c.k[key_at(head, c.cap / kKvBlock, c.dk, tok, d)] = ok ? (int32_t)y : 0;
        return ok;
    }
    d -= c.dk;
    const int64_t y = fx_to_i64(__ldg(rows.v + row * rows.ldv + (uint64_t)h * c.dv + d));
    const bool ok = y >= INT32_MIN && y <= INT32_MAX;
    c.v[(head * c.cap + tok) * c.dv + d] = ok ? (int32_t)y : 0;
    return ok;
}

// rows x: `tokens` rows of keys and values of sequence blockIdx.z, at the
// positions from lens[seq] on
__global__ void k_kv_append(KvCache c, KvRows rows, uint32_t tokens, uint32_t* __restrict__ err) {
    const uint32_t seq = blockIdx.z, h = blockIdx.y, width = c.dk + c.dv;
    const int64_t len = c.lens[seq];
    if (len < 0) return;
    bool bad = false, full = false;
    for (uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; i < (uint64_t)tokens * width;
         i += (uint64_t)gridDim.x * blockDim.x) {
        const uint64_t r = i / width, tok = len + r;
        if (tok >= c.cap)
            full = true;
        else
            bad |= !kv_store(c, rows, (uint64_t)seq * tokens + r, seq, h, tok, (uint32_t)(i % width));
    }
    if (bad) atomicOr(err, kErrRange);
    if (full) atomicOr(err, kErrFull);
}

constexpr int kAttThreads = 256;
constexpr int kAttWarps = kAttThreads / 32;
constexpr uint32_t kMaxRanks = 16;
constexpr size_t kAttShared = 220 * 1024;

struct AttendArgs {
    KvCache c;
    KvRows rows;  // the new token's key and value (null: none)
    const uint64_t* q;
    uint64_t ldq;
    uint32_t each;    // query heads to a key head
    uint32_t groups;  // blocks of EACH query heads to a key head
    int64_t q_factor, s_factor;
    uint32_t q_shift, s_shift, out_shift;
    const uint64_t* table;
    uint64_t table_len;
    int64_t offset;
    uint64_t* out;
    uint32_t* err;
    uint32_t chunk;  // tokens of a block's share of the scores
    uint32_t slice;  // outputs that a block of the cluster finishes
};

// One cluster per sequence, key head and EACH of its query heads; a block
// takes an equal run of the token blocks.  The softmax's rounding needs the
// row's maximum and then its sum before any weight is known, so the scores
// stay in shared memory and the cluster meets twice, keys and values each
// being read once; the blocks' value sums meet in a third exchange.  A block
// writes what the others need into their shared memory before each meeting,
// so that nothing is fetched from a neighbour after it.
template <int EACH>
__global__ void __launch_bounds__(kAttThreads, 2) k_kv_attend(const __grid_constant__ AttendArgs p) {
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ long long s_red[kAttWarps][EACH];
    __shared__ long long s_max[kMaxRanks][EACH], s_sum[kMaxRanks][EACH];
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t ranks = cluster.num_blocks(), rank = cluster.block_rank();
    const uint32_t seq = blockIdx.z, h = blockIdx.y / p.groups, e0 = (blockIdx.y % p.groups) * EACH;
    const uint32_t heads = min((uint32_t)EACH, p.each - e0), dk = p.c.dk, dv = p.c.dv;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint64_t* out = p.out + ((uint64_t)seq * p.c.heads * p.each + (uint64_t)h * p.each + e0) * dv;
    let_next_start();
    wait_for_previous();

    const int64_t len = p.c.lens[seq];
    const bool append = p.rows.k != nullptr && len >= 0 && len < p.c.cap;
    if (p.rows.k != nullptr && len >= p.c.cap && threadIdx.x == 0) atomicOr(p.err, kErrFull);
    const uint32_t n = (uint32_t)(len < 0 ? 0 : min(len + (append ? 1 : 0), (int64_t)p.c.cap));
    if (n == 0) {  // the whole cluster's answer
        for (uint32_t i = rank * kAttThreads + threadIdx.x; i < heads * dv; i += ranks * kAttThreads) out[i] = 0;
        return;
    }
    cluster_arrive();  // every block has started before another writes into its shared memory
    const uint32_t blocks = (n + kKvBlock - 1) / kKvBlock;
    const uint32_t b0 = (uint32_t)((uint64_t)rank * blocks / ranks), b1 = (uint32_t)((uint64_t)(rank + 1) * blocks / ranks);
    const uint32_t t0 = b0 * kKvBlock, count = b1 > b0 ? min(b1 * kKvBlock, n) - t0 : 0;
    const uint64_t head = (uint64_t)seq * p.c.heads + h;
    int32_t* const keys = p.c.k + key_at(head, p.c.cap / kKvBlock, dk, t0, 0);
    int32_t* const values = p.c.v + (head * p.c.cap + t0) * dv;
    // this block's keys and values, both in one piece, start for the second-level cache
    {
        constexpr uint32_t kPiece = 8192;
        const uint64_t kb = (uint64_t)(b1 - b0) * kKvBlock * dk * 4, vb = (uint64_t)count * dv * 4;
        const uint32_t kn = (uint32_t)((kb + kPiece - 1) / kPiece), vn = (uint32_t)((vb + kPiece - 1) / kPiece);
        for (uint32_t i = threadIdx.x; i < kn + vn; i += kAttThreads) {
            const uint64_t at = (uint64_t)(i < kn ? i : i - kn) * kPiece, left = (i < kn ? kb : vb) - at;
            prefetch_l2(reinterpret_cast<const uint8_t*>(i < kn ? keys : values) + at,
                        (uint32_t)(left < kPiece ? left : kPiece));
        }
    }

    long long* scores = reinterpret_cast<long long*>(smem);                  // EACH x chunk
    long long* sums = scores + (size_t)EACH * p.chunk;                       // EACH x 4 threads: value sums
    unsigned long long* acc = reinterpret_cast<unsigned long long*>(sums + (size_t)EACH * 4 * kAttThreads);
    int* qs = reinterpret_cast<int*>(acc + (((size_t)ranks * p.slice + 1) & ~(size_t)1));  // EACH x dk
    bool bad = false;
    for (uint32_t i = threadIdx.x; i < EACH * dk; i += kAttThreads) {
        int64_t y = 0;
        if (i / dk < heads) {
            const int64_t x = fx_to_i64(__ldg(p.q + seq * p.ldq + (uint64_t)(h * p.each + e0) * dk + i));
            y = fx_round_div_pow2(fx_wmul(x, p.q_factor), p.q_shift);
            if (y < -kKeyLimit || y > kKeyLimit) {
                bad = true;
                y = 0;
            }
        }
        qs[i] = (int)y;
    }
    // The new token belongs to the block whose share holds it (blocks of other
    // query heads of the same key head store the same numbers).
    if (append && (uint32_t)len / kKvBlock >= b0 && (uint32_t)len / kKvBlock < b1)
        for (uint32_t d = threadIdx.x; d < dk + dv; d += kAttThreads)
            bad |= !kv_store(p.c, p.rows, seq, seq, h, (uint64_t)len, d);
    __syncthreads();

    long long top[EACH];
#pragma unroll
    for (int e = 0; e < EACH; e++) top[e] = INT64_MIN;
    for (uint32_t b = warp; b < b1 - b0; b += kAttWarps) {
        const int32_t* kb = keys + (size_t)b * kKvBlock * dk + lane * 4;
        long long s[EACH];
#pragma unroll
        for (int e = 0; e < EACH; e++) s[e] = 0;
        constexpr int kAhead = 8;
        for (uint32_t d0 = 0; d0 < dk; d0 += 4 * kAhead) {
            int4 kv[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; i++)
                if (d0 + 4 * i < dk) kv[i] = __ldcg(reinterpret_cast<const int4*>(kb + (size_t)(d0 + 4 * i) * kKvBlock));
#pragma unroll
            for (int i = 0; i < kAhead; i++)
                if (d0 + 4 * i < dk) {
#pragma unroll
                    for (int e = 0; e < EACH; e++) {
                        const int4 qv = *reinterpret_cast<const int4*>(qs + e * dk + d0 + 4 * i);
                        s[e] += (long long)qv.x * kv[i].x + (long long)qv.y * kv[i].y + (long long)qv.z * kv[i].z +
                                (long long)qv.w * kv[i].w;
                    }
                }
        }
        const uint32_t at = b * kKvBlock + lane;
        if (at < count) {
#pragma unroll
            for (int e = 0; e < EACH; e++) {
                const long long z = fx_round_div_pow2(fx_wmul(s[e], p.s_factor), p.s_shift);
                scores[(size_t)e * p.chunk + at] = z;
                top[e] = z > top[e] ? z : top[e];
            }
        }
    }
#pragma unroll
    for (int e = 0; e < EACH; e++) {
        for (int o = 16; o; o >>= 1) {
            const long long other = __shfl_xor_sync(0xFFFFFFFFu, top[e], o);
            top[e] = other > top[e] ? other : top[e];
        }
        if (lane == 0) s_red[warp][e] = top[e];
    }
    __syncthreads();
    cluster_wait();
    for (uint32_t i = threadIdx.x; i < ranks * EACH; i += kAttThreads) {
        const uint32_t r = i / EACH, e = i % EACH;
        long long v = s_red[0][e];
        for (int w = 1; w < kAttWarps; w++) v = max(v, s_red[w][e]);
        *cluster.map_shared_rank(&s_max[rank][e], r) = v;
    }
    cluster.sync();
    long long part[EACH];
#pragma unroll
    for (int e = 0; e < EACH; e++) {
        top[e] = s_max[0][e];
        for (uint32_t r = 1; r < ranks; r++) top[e] = max(top[e], s_max[r][e]);
        part[e] = 0;
    }
    for (uint32_t j = threadIdx.x; j < count; j += kAttThreads) {
#pragma unroll
        for (int e = 0; e < EACH; e++) {
            int64_t v = fx_to_i64(
                table_at(p.table, p.table_len, fx_wsub(scores[(size_t)e * p.chunk + j], top[e]), p.offset));
            if (v < 0 || v > INT32_MAX) {
                bad = true;
                v = 0;
            }
            scores[(size_t)e * p.chunk + j] = v;
            part[e] += v;
        }
    }
#pragma unroll
    for (int e = 0; e < EACH; e++) {
        for (int o = 16; o; o >>= 1) part[e] += __shfl_xor_sync(0xFFFFFFFFu, part[e], o);
        if (lane == 0) s_red[warp][e] = part[e];
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < ranks * EACH; i += kAttThreads) {
        const uint32_t r = i / EACH, e = i % EACH;
        long long v = 0;
        for (int w = 0; w < kAttWarps; w++) v += s_red[w][e];
        *cluster.map_shared_rank(&s_sum[rank][e], r) = v;
    }
    cluster.sync();
    double inv[EACH];
#pragma unroll
    for (int e = 0; e < EACH; e++) {
        part[e] = 0;
        for (uint32_t r = 0; r < ranks; r++) part[e] += s_sum[r][e];
        if (part[e] == 0 && e < heads && rank == 0 && threadIdx.x == 0) atomicOr(p.err, kErrDivide);
        inv[e] = part[e] ? 1.0 / (double)part[e] : 0.0;
    }
    for (uint32_t j = threadIdx.x; j < count; j += kAttThreads) {
#pragma unroll
        for (int e = 0; e < EACH; e++) {
            const long long v = scores[(size_t)e * p.chunk + j];
            scores[(size_t)e * p.chunk + j] = part[e] ? round_div_near(v << 16, part[e], inv[e]) : 0;
        }
    }
    __syncthreads();

    // A thread keeps four dimensions and takes every step-th token
    const uint32_t wide = dv / 4, step = kAttThreads / wide, phase = threadIdx.x / wide, d4 = threadIdx.x % wide;
    if (phase < step) {
        long long y[EACH][4];
#pragma unroll
        for (int e = 0; e < EACH; e++) y[e][0] = y[e][1] = y[e][2] = y[e][3] = 0;
        const int32_t* vb = values + d4 * 4;
        constexpr int kAhead = 8;
        for (uint32_t j0 = phase; j0 < count; j0 += kAhead * step) {
            int4 vv[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; i++)
                if (j0 + i * step < count) vv[i] = __ldcg(reinterpret_cast<const int4*>(vb + (size_t)(j0 + i * step) * dv));
#pragma unroll
            for (int i = 0; i < kAhead; i++)
                if (j0 + i * step < count) {
#pragma unroll
                    for (int e = 0; e < EACH; e++) {
                        const int w = (int)scores[(size_t)e * p.chunk + j0 + i * step];
                        y[e][0] += (long long)w * vv[i].x;
                        y[e][1] += (long long)w * vv[i].y;
                        y[e][2] += (long long)w * vv[i].z;
                        y[e][3] += (long long)w * vv[i].w;
                    }
                }
        }
#pragma unroll
        for (int e = 0; e < EACH; e++)
#pragma unroll
            for (int i = 0; i < 4; i++) sums[((size_t)e * step + phase) * dv + d4 * 4 + i] = y[e][i];
    }
    if (bad) atomicOr(p.err, kErrRange);
    __syncthreads();
    // output i belongs to block i / slice: its part goes there
    for (uint32_t i = threadIdx.x; i < heads * dv; i += kAttThreads) {
        const uint32_t e = i / dv, d = i % dv;
        unsigned long long v = 0;
        for (uint32_t s = 0; s < step; s++) v += (unsigned long long)sums[((size_t)e * step + s) * dv + d];
        *cluster.map_shared_rank(&acc[(size_t)rank * p.slice + i % p.slice], i / p.slice) = v;
    }
    cluster.sync();
    for (uint32_t i = threadIdx.x; i < p.slice && rank * p.slice + i < heads * dv; i += kAttThreads) {
        unsigned long long v = 0;
        for (uint32_t r = 0; r < ranks; r++) v += acc[(size_t)r * p.slice + i];
        out[rank * p.slice + i] = fx_from_i64(fx_round_div_pow2((int64_t)v, p.out_shift));
    }
}

size_t attend_shared(uint32_t each, uint32_t ranks, uint32_t blocks, uint32_t dk, uint32_t dv) {
    const uint64_t chunk = ceil_div(blocks, ranks) * kKvBlock, slice = ceil_div(each * dv, ranks);
    return each * (8 * chunk + 32ull * kAttThreads + 4ull * dk) + 8 * ((ranks * slice + 1) & ~1ull);
}

template <int EACH>
int attend_launch(AttendArgs p, uint32_t ranks, cudaStream_t stream) {
    p.groups = (uint32_t)ceil_div(p.each, EACH);
    p.chunk = (uint32_t)ceil_div(p.c.cap / kKvBlock, ranks) * kKvBlock;
    p.slice = (uint32_t)ceil_div(EACH * p.c.dv, ranks);
    const size_t shared = attend_shared(EACH, ranks, p.c.cap / kKvBlock, p.c.dk, p.c.dv);
    auto* kernel = k_kv_attend<EACH>;
    static std::atomic<uint64_t> set{0};
    ZK_TRY(allow_shared(reinterpret_cast<const void*>(kernel), kAttShared, &set, true));
    return launch(kernel, dim3(ranks, p.c.heads * p.groups, p.c.batch), kAttThreads, shared, ranks, stream, p);
}

// ---- the next token ---------------------------------------------------------------------------
constexpr int kChooseThreads = 512;
constexpr int kChooseWarps = kChooseThreads / 32;

struct ChooseArgs {
    const uint64_t* logits;
    uint64_t v;
    const int32_t* history;
    uint64_t history_len;
    const int32_t* history_lens;
    int64_t repeat_pos, repeat_neg, presence, frequency;
    const uint64_t* bias;
    uint64_t bias_stride;
    const uint32_t* allowed;
    uint64_t allowed_stride;
    int64_t mask_value;
    uint64_t* out;
    uint32_t* token;
    uint32_t* err;
};

constexpr int kChooseEach = 8;  // logits of a thread at a time

// One cluster per row, a block to an equal slice of the vocabulary, a step of
// 4096 at a time: the logits start for registers, the history's tokens are
// counted in shared memory, then the logits are finished; the blocks' maxima
// meet in the first block.
__global__ void __launch_bounds__(kChooseThreads) k_choose_token(const __grid_constant__ ChooseArgs p) {
    constexpr uint32_t kStep = kChooseThreads * kChooseEach;
    __shared__ uint32_t counts[kStep];
    __shared__ long long s_v[kChooseWarps];
    __shared__ unsigned long long s_j[kChooseWarps];
    __shared__ long long best_v[kMaxRanks];
    __shared__ unsigned long long best_j[kMaxRanks];
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t ranks = cluster.num_blocks(), rank = cluster.block_rank();
    const uint64_t row = blockIdx.y, lo = p.v * rank / ranks, hi = p.v * (rank + 1) / ranks;
    cluster_arrive();  // every block has started before another writes into its shared memory
    let_next_start();
    wait_for_previous();
    uint64_t past = 0;
    if (p.history) {
        past = p.history_len;
        if (p.history_lens) {
            const int64_t l = p.history_lens[row];
            past = l < 0 ? 0 : (l < (int64_t)past ? l : past);
        }
    }
    long long bv = INT64_MIN;
    unsigned long long bj = UINT64_MAX;
    bool bad = false;
    for (uint64_t s0 = lo; s0 < hi; s0 += kStep) {
        const uint64_t s1 = s0 + kStep < hi ? s0 + kStep : hi;
        int64_t y[kChooseEach];
#pragma unroll
        for (int i = 0; i < kChooseEach; i++) {
            const uint64_t j = s0 + i * kChooseThreads + threadIdx.x;
            if (j < s1) y[i] = fx_to_i64(__ldg(p.logits + row * p.v + j));
        }
        if (past) {
            __syncthreads();
            for (uint32_t i = threadIdx.x; i < kStep; i += kChooseThreads) counts[i] = 0;
            __syncthreads();
            const int32_t* hist = p.history + row * p.history_len;
            for (uint64_t i0 = threadIdx.x; i0 < past; i0 += kChooseThreads * 8) {
                int32_t tok[8];
#pragma unroll
                for (int q = 0; q < 8; q++)
                    if (i0 + q * kChooseThreads < past) tok[q] = __ldg(hist + i0 + q * kChooseThreads);
#pragma unroll
                for (int q = 0; q < 8; q++)
                    if (i0 + q * kChooseThreads < past) {
                        bad |= tok[q] < 0 || (uint64_t)tok[q] >= p.v;
                        const uint64_t at = (uint64_t)tok[q] - s0;  // huge for a token before the step
                        if (tok[q] >= 0 && at < s1 - s0) atomicAdd(&counts[at], 1u);
                    }
            }
            __syncthreads();
        }
#pragma unroll
        for (int i = 0; i < kChooseEach; i++) {
            const uint64_t j = s0 + i * kChooseThreads + threadIdx.x;
            if (j >= s1) continue;
            int64_t z = y[i];
            const uint32_t c = past ? counts[j - s0] : 0;
            if (c) {
                z = fx_round_div_pow2(fx_wmul(z, z > 0 ? p.repeat_pos : p.repeat_neg), 16);
                z = fx_wsub(fx_wsub(z, p.presence), fx_wmul(p.frequency, c));
            }
            if (p.bias) z = fx_wadd(z, fx_to_i64(__ldg(p.bias + row * p.bias_stride + j)));
            if (p.allowed && !((__ldg(p.allowed + row * p.allowed_stride + j / 32) >> (j % 32)) & 1))
                z = fx_wadd(z, p.mask_value);
            p.out[row * p.v + j] = fx_from_i64(z);
            if (z > bv || bj == UINT64_MAX) {
                bv = z;
                bj = j;
            }
        }
    }
    if (bad && rank == 0) atomicOr(p.err, kErrIndex);
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    auto take = [&](long long ov, unsigned long long oj) {
        if (oj != UINT64_MAX && (bj == UINT64_MAX || ov > bv || (ov == bv && oj < bj))) {
            bv = ov;
            bj = oj;
        }
    };
    for (int o = 16; o; o >>= 1) {
        const long long ov = __shfl_xor_sync(0xFFFFFFFFu, bv, o);
        const unsigned long long oj = __shfl_xor_sync(0xFFFFFFFFu, bj, o);
        take(ov, oj);
    }
    if (lane == 0) {
        s_v[warp] = bv;
        s_j[warp] = bj;
    }
    __syncthreads();
    cluster_wait();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kChooseWarps; w++) take(s_v[w], s_j[w]);
        *cluster.map_shared_rank(&best_v[rank], 0) = bv;
        *cluster.map_shared_rank(&best_j[rank], 0) = bj;
    }
    cluster.sync();
    if (rank == 0 && threadIdx.x == 0) {
        for (uint32_t r = 0; r < ranks; r++) take(best_v[r], best_j[r]);
        p.token[row] = (uint32_t)bj;
    }
}

}  // namespace

}  // namespace zk

using namespace zk;

extern "C" {

uint64_t zkie2_q4_words(uint64_t experts, uint64_t k, uint64_t n, uint32_t group, uint64_t segment) {
    Q4Shape s;
    if (experts == 0 || experts > 4096 || !q4_shape(k, n, group, segment, &s)) return 0;
    return experts * s.tiles * s.blocks * (s.bytes / 4);
}

int zkie2_q4_pack(const int8_t* d_codes, const int32_t* d_scales, uint64_t experts, uint64_t k, uint64_t n,
                  uint32_t group, uint64_t segment, uint32_t* d_packed, uint32_t* d_err, cudaStream_t stream) {
    Q4Shape s;
    if (experts == 0 || experts > 4096 || !q4_shape(k, n, group, segment, &s) || !d_codes || !d_scales || !d_packed ||
        !d_err)
        return (int)cudaErrorInvalidValue;
    const uint64_t blocks = ceil_div(experts * s.tiles * s.blocks * (s.bytes / 4), 256);
    k_q4_pack<<<(unsigned)(blocks < kSms * 16 ? blocks : kSms * 16), 256, 0, stream>>>(
        d_codes, d_scales, (uint32_t)experts, s, d_packed, d_err);
    ZK_LAUNCH_CHECK();
    return 0;
}

int zkie2_q4_project(const uint64_t* d_x, uint64_t ldx, uint64_t m, const uint32_t* d_packed, uint64_t k, uint64_t n,
                     uint32_t group, uint64_t segment, uint32_t shift, const uint64_t* d_bias,
                     const uint64_t* d_table, uint64_t table_len, int64_t offset, const uint64_t* d_residual,
                     uint64_t ldr, uint64_t* d_out, uint32_t* d_err, cudaStream_t stream) {
    ProjectArgs p{};
    if (!q4_shape(k, n, group, segment, &p.s) || shift > 62 || m > 65535 || !d_packed || !d_err ||
        (d_table && table_len == 0) || (m > 1 && ldx < k) || (d_residual && m > 1 && ldr < n) ||
        ((uintptr_t)d_packed & 15))
        return (int)cudaErrorInvalidValue;
    if (m == 0) return 0;
    if (!d_x || !d_out) return (int)cudaErrorInvalidValue;
    p.x = d_x;
    p.ldx = ldx;
    p.m = (uint32_t)m;
    p.w = reinterpret_cast<const uint8_t*>(d_packed);
    p.shift = shift;
    p.bias = d_bias;
    p.table = d_table;
    p.table_len = table_len;
    p.offset = offset;
    p.residual = d_residual;
    p.ldr = ldr;
    p.out = d_out;
    p.err = d_err;
    p.stride = q4_digit_stride(p.s.blocks);
    return group == 32 ? project_rows<true>(p, stream) : project_rows<false>(p, stream);
}

int zkie2_kv_append(const uint64_t* d_k, uint64_t ldk, const uint64_t* d_v, uint64_t ldv, uint64_t tokens,
                    int64_t k_factor, uint32_t k_shift, int32_t* d_cache_k, int32_t* d_cache_v, const int32_t* d_lens,
                    uint64_t batch, uint64_t heads, uint64_t dk, uint64_t dv, uint64_t capacity, uint32_t* d_err,
                    cudaStream_t stream) {
    if (!d_cache_k || !d_cache_v || !d_lens || !d_err || batch == 0 || batch > 65535 || heads == 0 || heads > 65535 ||
        dk == 0 || dk > 256 || dk % 4 || dv == 0 || dv > 256 || dv % 4 || capacity == 0 || capacity % kKvBlock ||
        capacity > (1u << 17) || tokens > (1u << 17) || k_shift > 62 || ldk < heads * dk || ldv < heads * dv)
        return (int)cudaErrorInvalidValue;
    if (tokens == 0) return 0;
    if (!d_k || !d_v) return (int)cudaErrorInvalidValue;
    const KvCache c{d_cache_k, d_cache_v, d_lens, (uint32_t)batch, (uint32_t)heads, (uint32_t)dk, (uint32_t)dv,
                    (uint32_t)capacity};
    const KvRows rows{d_k, ldk, d_v, ldv, k_factor, k_shift};
    const uint64_t blocks = ceil_div(tokens * (dk + dv), 256);
    k_kv_append<<<dim3((unsigned)(blocks < 1024 ? blocks : 1024), (unsigned)heads, (unsigned)batch), 256, 0, stream>>>(
        c, rows, (uint32_t)tokens, d_err);
    ZK_LAUNCH_CHECK();
    return 0;
}

int zkie2_kv_attend(const uint64_t* d_q, uint64_t ldq, uint64_t q_heads, int64_t q_factor, uint32_t q_shift,
                    const uint64_t* d_k, uint64_t ldk, const uint64_t* d_v, uint64_t ldv, int64_t k_factor,
                    uint32_t k_shift, int32_t* d_cache_k, int32_t* d_cache_v, const int32_t* d_lens, uint64_t batch,
                    uint64_t heads, uint64_t dk, uint64_t dv, uint64_t capacity, int64_t s_factor, uint32_t s_shift,
                    const uint64_t* d_table, uint64_t table_len, int64_t offset, uint32_t out_shift, uint64_t* d_out,
                    uint32_t* d_err, cudaStream_t stream) {
    if (!d_q || !d_cache_k || !d_cache_v || !d_lens || !d_table || !d_out || !d_err || batch == 0 || batch > 65535 ||
        heads == 0 || q_heads == 0 || q_heads % heads || q_heads > 65535 || dk == 0 || dk > 256 || dk % 4 || dv == 0 ||
        dv > 256 || dv % 4 || capacity == 0 || capacity % kKvBlock || capacity > (1u << 17) || q_shift > 62 ||
        k_shift > 62 || s_shift > 62 || out_shift > 62 || table_len == 0 || (batch > 1 && ldq < q_heads * dk) ||
        !d_k != !d_v || (d_k && batch > 1 && (ldk < heads * dk || ldv < heads * dv)) ||
        (((uintptr_t)d_cache_k | (uintptr_t)d_cache_v) & 15))
        return (int)cudaErrorInvalidValue;
    AttendArgs p{};
    p.c = KvCache{d_cache_k, d_cache_v, d_lens, (uint32_t)batch, (uint32_t)heads, (uint32_t)dk, (uint32_t)dv,
                  (uint32_t)capacity};
    p.rows = KvRows{d_k, ldk, d_v, ldv, k_factor, k_shift};
    p.q = d_q;
    p.ldq = ldq;
    p.each = (uint32_t)(q_heads / heads);
    p.q_factor = q_factor;
    p.q_shift = q_shift;
    p.s_factor = s_factor;
    p.s_shift = s_shift;
    p.out_shift = out_shift;
    p.table = d_table;
    p.table_len = table_len;
    p.offset = offset;
    p.out = d_out;
    p.err = d_err;
    // Query heads to a block: those that share a key head, up to four (their
    // sums stay in registers); fewer where their scores do not fit.  Blocks to
    // a cluster: enough to fill the device, more where the scores need it.
    const uint32_t blocks = (uint32_t)(capacity / kKvBlock);
    for (uint32_t each = p.each >= 3 ? 4 : p.each;; each /= 2) {
        const uint64_t rows = batch * heads * ceil_div(p.each, each);
        uint32_t ranks = 1;
        while (ranks < kMaxRanks && rows * ranks * 2 <= 2 * kSms && ranks < blocks) ranks *= 2;
        while (ranks < kMaxRanks && attend_shared(each, ranks, blocks, p.c.dk, p.c.dv) > kAttShared) ranks *= 2;
        if (attend_shared(each, ranks, blocks, p.c.dk, p.c.dv) > kAttShared && each > 1) continue;
        return each == 4 ? attend_launch<4>(p, ranks, stream) : each == 2 ? attend_launch<2>(p, ranks, stream)
                                                                          : attend_launch<1>(p, ranks, stream);
    }
}

int zkie2_choose_token(const uint64_t* d_logits, uint64_t batch, uint64_t vocab, const int32_t* d_history,
                       uint64_t history_len, const int32_t* d_history_lens, int64_t repeat_pos, int64_t repeat_neg,
                       int64_t presence, int64_t frequency, const uint64_t* d_bias, uint64_t bias_stride,
                       const uint32_t* d_allowed, uint64_t allowed_stride, int64_t mask_value, uint64_t* d_out,
                       uint32_t* d_token, uint32_t* d_err, cudaStream_t stream) {
    if (vocab == 0 || vocab > 0x7FFFFFFFull || batch > 65535 || (d_history_lens && !d_history) || !d_err ||
        history_len > 0x7FFFFFFFull)
        return (int)cudaErrorInvalidValue;
    if (batch == 0) return 0;
    if (!d_logits || !d_out || !d_token) return (int)cudaErrorInvalidValue;
    const ChooseArgs p{d_logits, vocab, d_history, history_len, d_history_lens, repeat_pos, repeat_neg, presence,
                       frequency, d_bias, bias_stride, d_allowed, allowed_stride, mask_value, d_out, d_token, d_err};
    // Blocks to a row: one step of the vocabulary each, fewer once the rows fill the device
    uint32_t ranks = 1;
    while (ranks < kMaxRanks && vocab > (uint64_t)ranks * kChooseThreads * kChooseEach && batch * ranks < 2 * kSms)
        ranks *= 2;
    static std::atomic<uint64_t> set{0};
    ZK_TRY(allow_shared(reinterpret_cast<const void*>(k_choose_token), 0, &set, true));
    return launch(k_choose_token, dim3(ranks, (unsigned)batch), kChooseThreads, 0, ranks, stream, p);
}

}  // extern "C"
