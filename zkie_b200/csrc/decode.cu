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
constexpr uint32_t kErrFull = 16u;  // a cache without room for the tokens that are counted
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

// two weights of one shape, block by block side by side; or (b null) the tiles of one two by two,
// with zeros beside an odd one
__global__ void k_q4_pair(const uint4* __restrict__ a, const uint4* __restrict__ b, Q4Shape s, uint64_t blocks,
                          uint4* __restrict__ out) {
    const uint32_t words = s.bytes / 16, pairs = (s.tiles + 1) / 2;
    for (uint64_t i = blockIdx.x; i < blocks; i += gridDim.x) {  // of a weight, or of its pairs
        const uint64_t at = i % s.blocks, tile = i / s.blocks % pairs * 2, expert = i / s.blocks / pairs;
        const uint4* from = b ? a + i * words : a + ((expert * s.tiles + tile) * s.blocks + at) * words;
        const uint4* beside = b ? b + i * words : tile + 1 < s.tiles ? from + (uint64_t)s.blocks * words : nullptr;
        for (uint32_t j = threadIdx.x; j < words; j += blockDim.x) {
            out[i * 2 * words + j] = from[j];
            out[(i * 2 + 1) * words + j] = beside ? beside[j] : make_uint4(0, 0, 0, 0);
        }
    }
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
    uint32_t run;     // blocks to a slot of a ring, at most
    uint32_t unit;    // blocks that stay with one warp: a segment, or a slot where a tile has whole ones
    uint32_t units;   // of a tile
    uint32_t some, more;  // tiles of a grid's block: some, and one more in the first `more` of them
};

constexpr int kProjDepth = 2;           // slots of a warp's ring (three: one row of 1024 x 65536 10.6 us instead of 10.2)
constexpr uint32_t kProjBatch = 16;     // tiles whose sums are held at a time

// A block takes an equal run of the tiles of 16 columns, in batches; of a
// batch every warp takes an equal run of blocks (of whole segments where each
// is rounded by itself), whatever tiles they belong to, against the digits of
// 2 NT rows in shared memory.  The 64-bit sums meet in shared memory; a thread
// per output then rounds and finishes it.
//
// Bound by: for few rows and a wide weight the weight's bytes (1024 x 65536 in
// groups of 128, one row: 36 MB in 10.2 us, of which 3 us are the launch, the
// row's digits and the last sums: 5 TB/s in between); for eight rows what a
// warp does per block and pair of rows, about ten cycles of the SM (17.8 us:
// 2.0 TB/s); for a small weight the launch and three trips to memory (1024 x
// 192: 2.8 us).  A ring's slots are of four blocks because copies of 2176
// bytes reach 5.8 TB/s and single blocks 3.7 (eight blocks to a slot: within 4
// % either way); with three slots to a ring, 24 warps of 80 registers instead
// of 16 of 127 take 20.8 us for the eight rows instead of 18.3, 20 warps 19.9.
template <int G, int NT, bool SEG>
__global__ void __launch_bounds__(kProjThreads, 1) k_q4_project(const __grid_constant__ ProjectArgs p) {
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ __align__(8) uint64_t s_bar[kProjWarps * kProjDepth];
    constexpr bool TWO = G == 32;
    constexpr uint32_t kRows = 2 * NT, kBytes = TWO ? 576 : 544;
    const uint32_t row0 = blockIdx.y * kRows, rows = min(kRows, p.m - row0);
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint32_t slot_bytes = p.run * kBytes;
    const uint32_t ring = shared_addr(smem) + warp * kProjDepth * slot_bytes;
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
    const uint32_t tile0 = blockIdx.x * p.some + min(blockIdx.x, p.more), tile1 = tile0 + p.some + (blockIdx.x < p.more);
    const uint32_t blocks = p.s.blocks, unit = p.unit;
    // blocks of a batch, counted from its first tile, that the warp takes
    auto first_of = [&](uint32_t batch, uint32_t w) {
        return w * (min(kProjBatch, tile1 - batch) * p.units) / kProjWarps * unit;
    };
    uint32_t next_batch = tile0, next_at = first_of(tile0, warp), next_end = first_of(tile0, warp + 1), next_slot = 0;
    uint32_t next_b = next_at % blocks;  // within its tile
    Patience patience;
    auto ask = [&]() {  // lane 0 only
        if (patience.failed) return;
        while (next_at == next_end) {
            next_batch += kProjBatch;
            if (next_batch >= tile1) {
                next_batch = tile1;
                return;
            }
            next_at = first_of(next_batch, warp);
            next_end = first_of(next_batch, warp + 1);
            next_b = next_at % blocks;
        }
        const uint32_t run = min(min(p.run, next_end - next_at), blocks - next_b);  // within a tile
        barrier_expect(bar + 8 * next_slot, run * kBytes);
        bulk_copy(ring + next_slot * slot_bytes, p.w + ((uint64_t)next_batch * blocks + next_at) * kBytes, run * kBytes,
                  bar + 8 * next_slot);
        next_at += run;
        next_b = next_b + run == blocks ? 0 : next_b + run;
        next_slot = next_slot + 1 == kProjDepth ? 0 : next_slot + 1;
    };
    if (lane == 0)
        for (int i = 0; i < kProjDepth; i++)
            if (next_batch < tile1) ask();

    // ---- the rows' digits
    acc.template clear<kProjThreads>();
    wait_for_previous();
    if (!q4_digitise<kProjThreads, 4>(p.x + (uint64_t)row0 * p.ldx, p.ldx, p.s.segs, p.s.k_seg, p.s.kp_seg, 0,
                                   rows * blocks * 16, digits, p.stride))
        atomicOr(p.err, kErrRange);
    __syncthreads();

    const uint32_t from = shared_addr(digits) + g * p.stride + 16 * t;  // column g: digit g % 4 of row g / 4
    uint32_t slot = 0, phase = 0;
    for (uint32_t batch = tile0; batch < tile1; batch += kProjBatch) {
        uint32_t at = first_of(batch, warp);
        const uint32_t end = first_of(batch, warp + 1);
        uint32_t tile = at / blocks, b = at % blocks, in_seg = 0;
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
        uint32_t x_at[NT];  // the digits of each pair of rows, at block b
#pragma unroll
        for (int i = 0; i < NT; i++) x_at[i] = from + i * 8 * p.stride + b * 64;
        while (at < end) {
            const uint32_t run = min(min(p.run, end - at), blocks - b);
            barrier_wait(bar + 8 * slot, phase, patience);
            const Q4Lane lane_at(ring + slot * slot_bytes);
            auto block = [&](uint32_t q) {
                uint4 x[NT];
#pragma unroll
                for (int i = 0; i < NT; i++) x[i] = load16(x_at[i] + q * 64);
                q4_block<TWO, NT, NT>(sum, lane_at, q * kBytes, x);
            };
            if (!SEG && run == 4 && (G != 128 || unit == 4)) {
#pragma unroll
                for (uint32_t q = 0; q < 4; q += 2) {
                    if (G == 128) {  // two whole groups (eight rows block by block: 10 % more)
                        uint4 x[2][NT];
#pragma unroll
                        for (int i = 0; i < 2 * NT; i++) x[i / NT][i % NT] = load16(x_at[i % NT] + (q + i / NT) * 64);
                        q4_group<NT>(sum, lane_at, q * kBytes, kBytes, x);
                    } else {
                        block(q);
                        block(q + 1);
                    }
                }
                b += 4;
            } else {
                for (uint32_t q = 0; q < run; q++) {
                    block(q);
                    if (SEG && (b++, ++in_seg == unit)) {
                        in_seg = 0;
#pragma unroll
                        for (int i = 0; i < NT; i++) total[i] += round_shift(sum.finish(i), p.shift);
                        sum.clear();
                    }
                }
                if (!SEG) b += run;
            }
            at += run;
            if (b == blocks) {
                flush();
                b = 0;
                tile++;
            }
#pragma unroll
            for (int i = 0; i < NT; i++) x_at[i] = from + i * 8 * p.stride + b * 64;
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
        // a thread's outputs, NT of a batch: one row and one column of 16 in every kStep-th tile, their
        // operands under way together
        constexpr uint32_t kStep = kProjBatch / NT;
        const uint32_t r = threadIdx.x / 16 % kRows, tile1st = threadIdx.x / (16 * kRows);
        const uint32_t n1st = (batch + tile1st) * 16 + threadIdx.x % 16;
        bool on[NT];
        uint64_t bias[NT], residual[NT];
#pragma unroll
        for (int u = 0; u < NT; u++) {
            const uint32_t n = n1st + u * kStep * 16;
            on[u] = r < rows && tile1st + u * kStep < tiles && n < p.s.n;
            bias[u] = on[u] && p.bias ? p.bias[n] : 0;
            residual[u] = on[u] && p.residual ? p.residual[(uint64_t)(row0 + r) * p.ldr + n] : 0;
        }
        uint64_t f[NT];
#pragma unroll
        for (int u = 0; u < NT; u++) {
            f[u] = 0;
            if (!on[u]) continue;
            const uint32_t o = threadIdx.x + u * kProjThreads;
            int64_t y = SEG ? acc.get(o) : round_shift(acc.get(o), p.shift);
            acc.clear(o);
            y = fx_wadd(y, q4_number(bias[u]));
            f[u] = p.table ? table_at(p.table, p.table_len, y, p.offset) : fx_from_i64(y);
        }
        uint64_t* out = p.out + (uint64_t)(row0 + r) * p.s.n + n1st;
#pragma unroll
        for (int u = 0; u < NT; u++)
            if (on[u]) {
                if (p.table) f[u] = gl_canon(f[u]);
                out[u * kStep * 16] = p.residual ? gl_canon(gl_add(f[u], gl_canon(residual[u]))) : f[u];
            }
        __syncthreads();
    }
    patience_end(patience, p.err);
}

// dynamic shared memory for blocks of `rows` rows and a ring of `run` blocks to a slot
size_t project_shared(const Q4Shape& s, uint32_t rows, uint32_t run) {
    return (size_t)kProjWarps * kProjDepth * run * s.bytes + (size_t)rows * (kProjBatch * 16 * 12 + 4 * q4_digit_stride(s.blocks));
}

template <int G, int NT, bool SEG>
int project_launch(ProjectArgs p, cudaStream_t stream) {
    auto* kernel = k_q4_project<G, NT, SEG>;
    static std::atomic<uint64_t> set{0};
    ZK_TRY(allow_shared(reinterpret_cast<const void*>(kernel), kMaxShared, &set));
    const dim3 grid(p.s.tiles < (uint32_t)kSms ? p.s.tiles : kSms, (unsigned)ceil_div(p.m, 2 * NT));
    p.units = p.s.blocks / p.unit;
    p.some = p.s.tiles / grid.x;
    p.more = p.s.tiles % grid.x;
    return launch(kernel, grid, kProjThreads, project_shared(p.s, 2 * NT, p.run), 1, stream, p);
}

template <int G, int NT>
int project_seg(const ProjectArgs& p, cudaStream_t stream) {
    return p.s.segs > 1 ? project_launch<G, NT, true>(p, stream) : project_launch<G, NT, false>(p, stream);
}

template <int G>
int project_rows(ProjectArgs p, cudaStream_t stream) {
    // Rows to a block: as many as there are, up to eight, so that a weight is read once for them, and
    // as their digits leave room for (1024 x 65536: eight rows 17.8 us, four 12.4, two 10.2, one 10.2,
    // one row with eight's kernel 16.9).  Slots of four blocks where there is room, else of two or one
    // (one row 10.6, 13.2, 18.0 us, of rings of three; a weight of 1024 x 192 in 3.0, 2.9, 2.8).
    for (uint32_t rows = p.m > 4 ? 8 : p.m > 2 ? 4 : 2;; rows /= 2)
        for (p.run = 4; p.run; p.run /= 2)
            if (p.unit = p.s.segs > 1 ? p.s.kp_seg / 64 : p.s.blocks % p.run ? 1 : p.run;
                project_shared(p.s, rows, p.run) <= kMaxShared)
                return rows == 8   ? project_seg<G, 4>(p, stream)
                       : rows == 4 ? project_seg<G, 2>(p, stream)
                                   : project_seg<G, 1>(p, stream);
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
                                         uint64_t tok, uint32_t d, int* copy = nullptr) {
    const uint64_t head = (uint64_t)seq * c.heads + h;
    if (d < c.dk) {
        const int64_t x = fx_to_i64(rows.k[row * rows.ldk + (uint64_t)h * c.dk + d]);
        const int64_t y = fx_round_div_pow2(fx_wmul(x, rows.factor), rows.shift);
        const bool ok = y >= -kKeyLimit && y <= kKeyLimit;
        if (copy) *copy = ok ? (int32_t)y : 0;
        c.k[key_at(head, c.cap / kKvBlock, c.dk, tok, d)] = ok ? (int32_t)y : 0;
        return ok;
    }
    d -= c.dk;
    const int64_t y = fx_to_i64(rows.v[row * rows.ldv + (uint64_t)h * c.dv + d]);
    const bool ok = y >= INT32_MIN && y <= INT32_MAX;
    if (copy) *copy = ok ? (int32_t)y : 0;
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
constexpr uint32_t kMaxRanks = 16;   // blocks of a cluster
constexpr size_t kAttShared = 220 * 1024;
constexpr uint32_t kAttPiece = 4096;  // bytes of a ring's slot
constexpr uint32_t kKeyDims = 32;     // dimensions of 32 keys to a slot
constexpr uint32_t kAttDepth = 2;     // slots of a warp's ring (three: the same times)

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
    uint32_t chunk;  // scores that a block has room for
    uint32_t slice;  // outputs that a block of the cluster finishes
};

// One cluster per sequence, key head and EACH of its query heads; a block
// takes an equal run of the token blocks, a warp every eighth of them.  A warp
// streams its blocks' keys and then their values through its ring, so that
// values are on their way while the softmax is worked out.  The softmax's
// rounding needs the row's maximum and then its sum before any weight is
// known, so the scores stay in shared memory and the cluster meets twice, keys
// and values each being read once; the blocks' value sums meet in a third
// exchange.  A block writes what the others need into their shared memory
// before each meeting, so that nothing is fetched from a neighbour after it.
// The new token is taken from its rows, not from the cache it is stored to.
// A product is one 32 x 32 + 64 bit multiply-add, 32 a clock on an SM.
//
// Bound by: for one long sequence the two streams (16 heads of 192 + 128, 4096
// tokens: 82 MB in 26.7 us, keys 10 us and values 7 at 4.5 to 5 TB/s, between
// them 7 us of meetings and table entries, the first bytes 2); for a ragged
// batch the longest sequence's blocks, whose cluster is as large as any other
// (eight sequences of up to 8192 tokens, four query heads to a key head: 70
// us, of which multiply-adds cost 12, table entries 10, the streams the
// rest); for a short one the chain of latencies (512 tokens: 8.2 us).  Half
// the heads' products in double precision: 69 us instead of 71, not kept; an
// L2 prefetch of the values during the softmax: 29 to 32 us instead of 27; the
// table's entries asked for sixteen at a time by a thread: the same 71, their
// number is what costs.
template <int EACH, int WIDE>
__global__ void __launch_bounds__(kAttThreads, 2) k_kv_attend(const __grid_constant__ AttendArgs p) {
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ __align__(8) uint64_t s_bar[kAttWarps * kAttDepth];
    __shared__ long long s_red[kAttWarps][EACH];
    __shared__ long long s_max[kMaxRanks][EACH], s_sum[kMaxRanks][EACH];
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t ranks = cluster.num_blocks(), rank = cluster.block_rank();
    const uint32_t seq = blockIdx.z, h = blockIdx.y / p.groups, e0 = (blockIdx.y % p.groups) * EACH;
    const uint32_t heads = min((uint32_t)EACH, p.each - e0), dk = p.c.dk, dv = p.c.dv;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint64_t* out = p.out + ((uint64_t)seq * p.c.heads * p.each + (uint64_t)h * p.each + e0) * dv;
    const uint32_t bar = shared_addr(&s_bar[warp * kAttDepth]);
    let_next_start();
    if (lane == 0) {
        for (uint32_t i = 0; i < kAttDepth; i++) barrier_init(bar + 8 * i);
        barrier_init_done();
    }
    __syncwarp();
    wait_for_previous();

    // The queries, asked for before the first keys: behind them they arrive 2 us later
    uint64_t q_in[EACH];
#pragma unroll
    for (int u = 0; u < EACH; u++) {
        const uint32_t i = threadIdx.x + u * kAttThreads;  // dk <= kAttThreads
        q_in[u] = i < heads * dk ? p.q[seq * p.ldq + (uint64_t)(h * p.each + e0) * dk + i] : 0;
    }
    const int64_t len = p.c.lens[seq];
    const bool append = p.rows.k != nullptr && len >= 0 && len < p.c.cap;
    if (len >= (int64_t)p.c.cap + (p.rows.k == nullptr) && threadIdx.x == 0) atomicOr(p.err, kErrFull);
    const uint32_t n = (uint32_t)(len < 0 ? 0 : min(len, (int64_t)p.c.cap));  // tokens in the cache
    if (n + append == 0) {  // the whole cluster's answer
        for (uint32_t i = rank * kAttThreads + threadIdx.x; i < heads * dv; i += ranks * kAttThreads) out[i] = 0;
        return;
    }
    cluster_arrive();  // every block has started before another writes into its shared memory
    const uint32_t blocks = (n + kKvBlock - 1) / kKvBlock;
    const uint32_t b0 = (uint32_t)((uint64_t)rank * blocks / ranks), b1 = (uint32_t)((uint64_t)(rank + 1) * blocks / ranks);
    const uint32_t t0 = b0 * kKvBlock, cached = b1 > b0 ? min(b1 * kKvBlock, n) - t0 : 0;
    const bool own = append && rank == ranks - 1;  // the new token's block: its score is number `cached`
    const uint32_t count = cached + own;
    const uint64_t head = (uint64_t)seq * p.c.heads + h;
    const int32_t* keys = p.c.k + key_at(head, p.c.cap / kKvBlock, dk, t0, 0);
    const int32_t* values = p.c.v + (head * p.c.cap + t0) * dv;

    uint8_t* ring = smem + (size_t)warp * kAttDepth * kAttPiece;
    long long* sums = reinterpret_cast<long long*>(smem);  // in the rings' place, once they are done
    // chunk x EACH; a token's weights later take the first half of its scores' place, as 32-bit numbers
    long long* scores = reinterpret_cast<long long*>(smem + (size_t)kAttWarps * kAttDepth * kAttPiece);
    unsigned long long* acc = reinterpret_cast<unsigned long long*>(scores + (size_t)EACH * p.chunk);  // ranks x slice
    int* qs = reinterpret_cast<int*>(acc + (((size_t)ranks * p.slice + 1) & ~(size_t)1));              // EACH x dk
    int* fresh = qs + EACH * dk;                                                                       // dk + dv

    // ---- the warp's stream: keys of its token blocks in pieces of 32 dimensions, then their
    // values in pieces of a few tokens
    const uint32_t kpieces = (dk + kKeyDims - 1) / kKeyDims;
    const uint32_t vtokens = min((uint32_t)kKvBlock, kAttPiece / (4 * dv)), vpieces = (kKvBlock + vtokens - 1) / vtokens;
    uint32_t next_b = warp, next_i = 0, next_slot = 0;
    bool next_v = false;
    auto piece_tokens = [&](uint32_t b, uint32_t i) {  // of piece i of a block's values
        const uint32_t there = min((uint32_t)kKvBlock, cached - b * kKvBlock), at = i * vtokens;
        return at < there ? min(vtokens, there - at) : 0u;
    };
    Patience patience;
    auto ask = [&]() {  // lane 0 only
        if (patience.failed) return;
        if (next_b >= b1 - b0) {
            if (next_v || warp >= b1 - b0) return;
            next_v = true;
            next_b = warp;
        }
        const void* from;
        uint32_t bytes;
        if (!next_v) {
            from = keys + ((size_t)next_b * dk + next_i * kKeyDims) * kKvBlock;
            bytes = min(kKeyDims, dk - next_i * kKeyDims) * kKvBlock * 4;
        } else {
            from = values + ((size_t)next_b * kKvBlock + next_i * vtokens) * dv;
            bytes = piece_tokens(next_b, next_i) * dv * 4;
        }
        barrier_expect(bar + 8 * next_slot, bytes);
        bulk_copy(shared_addr(ring + next_slot * kAttPiece), from, bytes, bar + 8 * next_slot);
        next_slot = next_slot + 1 == kAttDepth ? 0 : next_slot + 1;
        next_i++;
        if (next_v ? next_i == vpieces || piece_tokens(next_b, next_i) == 0 : next_i == kpieces) {
            next_i = 0;
            next_b += kAttWarps;
        }
    };
    if (lane == 0)
        for (uint32_t i = 0; i < kAttDepth; i++) ask();
    uint32_t slot = 0, phase = 0;
    auto step = [&]() {  // on to the next slot, this one being filled again
        __syncwarp();
        if (lane == 0) ask();
        if (++slot == kAttDepth) {
            slot = 0;
            phase ^= 1;
        }
    };

    bool bad = false;
#pragma unroll
    for (int u = 0; u < EACH; u++) {
        const uint32_t i = threadIdx.x + u * kAttThreads;
        int64_t y = round_shift(fx_wmul(fx_to_i64(q_in[u]), p.q_factor), p.q_shift);
        if (y < -kKeyLimit || y > kKeyLimit) {
            bad = true;
            y = 0;
        }
        if (i < EACH * dk) qs[i] = (int)y;
    }
    if (own)  // store the new token (blocks of other query heads of this key head store the same numbers)
        for (uint32_t d = threadIdx.x; d < dk + dv; d += kAttThreads)
            bad |= !kv_store(p.c, p.rows, seq, seq, h, (uint64_t)len, d, &fresh[d]);
    __syncthreads();

    // ---- scores
    long long top[EACH];
#pragma unroll
    for (int e = 0; e < EACH; e++) top[e] = INT64_MIN;
    auto keep = [&](int e, uint32_t at, long long s) {
        const long long z = round_shift(fx_wmul(s, p.s_factor), p.s_shift);
        scores[at * EACH + e] = z;
        top[e] = max(top[e], z);
    };
    for (uint32_t b = warp; b < b1 - b0; b += kAttWarps) {
        long long s[EACH];
#pragma unroll
        for (int e = 0; e < EACH; e++) s[e] = 0;
        for (uint32_t d0 = 0; d0 < dk; d0 += kKeyDims) {
            barrier_wait(bar + 8 * slot, phase, patience);
            const int4* kv = reinterpret_cast<const int4*>(ring + slot * kAttPiece) + lane;
            const uint32_t quads = min(kKeyDims, dk - d0) / 4;
            const int* qd = qs + d0;
#pragma unroll 4
            for (uint32_t i = 0; i < quads; i++) {
                const int4 x = kv[i * 32];
#pragma unroll
                for (int e = 0; e < EACH; e++) {
                    const int4 qv = *reinterpret_cast<const int4*>(qd + e * dk + 4 * i);
                    s[e] += (long long)qv.x * x.x;
                    s[e] += (long long)qv.y * x.y;
                    s[e] += (long long)qv.z * x.z;
                    s[e] += (long long)qv.w * x.w;
                }
            }
            step();
        }
        if (b * kKvBlock + lane < cached) {
#pragma unroll
            for (int e = 0; e < EACH; e++) keep(e, b * kKvBlock + lane, s[e]);
        }
    }
    if (own && warp == kAttWarps - 1) {
#pragma unroll
        for (int e = 0; e < EACH; e++) {
            long long s = 0;
            for (uint32_t d = lane; d < dk; d += 32) s += (long long)qs[e * dk + d] * fresh[d];
            for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
            keep(e, cached, s);  // every lane the same
        }
    }
#pragma unroll
    for (int e = 0; e < EACH; e++) {
        top[e] = warp_max(top[e]);
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

    // ---- weights
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
                table_at(p.table, p.table_len, fx_wsub(scores[j * EACH + e], top[e]), p.offset));
            if (v < 0 || v > INT32_MAX) {
                bad = true;
                v = 0;
            }
            scores[j * EACH + e] = v;
            part[e] += v;
        }
    }
#pragma unroll
    for (int e = 0; e < EACH; e++) {
        part[e] = warp_sum(part[e]);
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
    float inv[EACH];
#pragma unroll
    for (int e = 0; e < EACH; e++) {
        part[e] = 0;
        for (uint32_t r = 0; r < ranks; r++) part[e] += s_sum[r][e];
        if (part[e] == 0 && e < heads && rank == 0 && threadIdx.x == 0) atomicOr(p.err, kErrDivide);
        inv[e] = 1.0f / (float)part[e];
    }
    struct alignas(4 * EACH) Weights {
        int w[EACH];
    };
    const auto weights_of = [&](uint32_t j) { return reinterpret_cast<Weights*>(scores + j * EACH); };
    for (uint32_t j = threadIdx.x; j < count; j += kAttThreads) {
        Weights w;
#pragma unroll
        for (int e = 0; e < EACH; e++)
            w.w[e] = part[e] ? softmax_weight((uint32_t)scores[j * EACH + e], part[e], inv[e]) : 0;
        *weights_of(j) = w;
    }
    __syncthreads();

    // ---- values: a lane keeps four dimensions (WIDE = 2: eight) and takes every step-th token
    const uint32_t wide = (dv / 4 + WIDE - 1) / WIDE, step_t = 32 / wide, mine = lane / wide, d4 = lane % wide;
    const bool on = mine < step_t, second = WIDE == 2 && d4 + wide < dv / 4;
    long long y[EACH][4 * WIDE];
#pragma unroll
    for (int e = 0; e < EACH; e++)
#pragma unroll
        for (int i = 0; i < 4 * WIDE; i++) y[e][i] = 0;
    auto take = [&](const int4& x, int w0, const Weights& w) {
#pragma unroll
        for (int e = 0; e < EACH; e++) {
            y[e][w0] += (long long)w.w[e] * x.x;
            y[e][w0 + 1] += (long long)w.w[e] * x.y;
            y[e][w0 + 2] += (long long)w.w[e] * x.z;
            y[e][w0 + 3] += (long long)w.w[e] * x.w;
        }
    };
    for (uint32_t b = warp; b < b1 - b0; b += kAttWarps) {
        for (uint32_t i = 0; i < vpieces; i++) {
            const uint32_t tokens = piece_tokens(b, i);
            if (tokens == 0) break;
            barrier_wait(bar + 8 * slot, phase, patience);
            const int4* vv = reinterpret_cast<const int4*>(ring + slot * kAttPiece) + d4;
            const uint32_t first = b * kKvBlock + i * vtokens;
            if (on) {
#pragma unroll 4
                for (uint32_t j = mine; j < tokens; j += step_t) {
                    const Weights w = *weights_of(first + j);
                    take(vv[j * (dv / 4)], 0, w);
                    if (second) take(vv[j * (dv / 4) + wide], 4 * (WIDE - 1), w);
                }
            }
            step();
        }
    }
    if (bad) atomicOr(p.err, kErrRange);
    patience_end(patience, p.err);
    __syncthreads();  // the rings are done with
    if (on) {
        long long* to = sums + ((size_t)(warp * step_t + mine) * EACH) * dv;
#pragma unroll
        for (int e = 0; e < EACH; e++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                to[e * dv + d4 * 4 + i] = y[e][i];
                if (second) to[e * dv + (d4 + wide) * 4 + i] = y[e][4 * (WIDE - 1) + i];
            }
    }
    __syncthreads();
    // output i belongs to block i / slice: its part goes there
    for (uint32_t i = threadIdx.x; i < heads * dv; i += kAttThreads) {
        const uint32_t e = i / dv, d = i % dv;
        unsigned long long v = 0;
        for (uint32_t s = 0; s < kAttWarps * step_t; s++) v += (unsigned long long)sums[(size_t)s * EACH * dv + i];
        if (own) v += (unsigned long long)((long long)weights_of(cached)->w[e] * fresh[dk + d]);
        *cluster.map_shared_rank(&acc[(size_t)rank * p.slice + i % p.slice], i / p.slice) = v;
    }
    cluster.sync();
    for (uint32_t i = threadIdx.x; i < p.slice && rank * p.slice + i < heads * dv; i += kAttThreads) {
        unsigned long long v = 0;
        for (uint32_t r = 0; r < ranks; r++) v += acc[(size_t)r * p.slice + i];
        out[rank * p.slice + i] = fx_from_i64(round_shift((int64_t)v, p.out_shift));
    }
}

// Shared memory of a block: rings (64 kB; in their place later the value sums, at most
// 32 kB), scores, the others' sums, queries, the new token
struct AttendPlan {
    uint32_t each, ranks, chunk, slice;
    size_t shared;
};

AttendPlan attend_plan(uint32_t each, uint32_t ranks, uint32_t blocks, uint32_t dk, uint32_t dv) {
    AttendPlan a{each, ranks, 0, 0, 0};
    a.chunk = (uint32_t)ceil_div(blocks, ranks) * kKvBlock + 1;
    a.chunk += a.chunk % 2;
    a.slice = (uint32_t)ceil_div(each * dv, ranks);
    a.shared = (size_t)kAttWarps * kAttDepth * kAttPiece + 8ull * each * a.chunk + 8 * ((ranks * a.slice + 1) & ~1ull) +
               4ull * (each * dk + dk + dv);
    return a;
}

template <int EACH, int WIDE>
int attend_launch(AttendArgs p, const AttendPlan& a, cudaStream_t stream) {
    p.groups = (uint32_t)ceil_div(p.each, EACH);
    p.chunk = a.chunk;
    p.slice = a.slice;
    auto* kernel = k_kv_attend<EACH, WIDE>;
    static std::atomic<uint64_t> set{0};
    ZK_TRY(allow_shared(reinterpret_cast<const void*>(kernel), kAttShared, &set, true));
    return launch(kernel, dim3(a.ranks, p.c.heads * p.groups, p.c.batch), kAttThreads, a.shared, a.ranks, stream, p);
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
constexpr uint32_t kChooseStep = kChooseThreads * kChooseEach;

// One cluster per row, a block to an equal run of the vocabulary in whole
// words of the mask, a step of 4096 at a time: logits, biases and mask words
// start for registers, the history's tokens are counted in shared memory, then
// the logits are finished; the blocks' maxima meet in the first block.  A warp
// takes 32 neighbours, so a mask word is one load.
//
// Bound by the chain launch - lengths - history - logits - cluster: one row of
// 65536 takes 5.9 us, sixteen of 50257 with histories of 4096 9.4 us (19.7 MB:
// 2.1 TB/s, every block reading its row's whole history).  Histories loaded
// before their lengths are known: 13.7 us instead of 12.8 at the time; four
// logits to a thread, three blocks to an SM: 13.0; 1024 threads: 16.7.
__global__ void __launch_bounds__(kChooseThreads, 2) k_choose_token(const __grid_constant__ ChooseArgs p) {
    __shared__ uint32_t counts[kChooseStep];
    __shared__ long long s_v[kChooseWarps];
    __shared__ uint32_t s_j[kChooseWarps];
    __shared__ long long best_v[kMaxRanks];
    __shared__ uint32_t best_j[kMaxRanks];
    constexpr uint32_t kNone = 0xFFFFFFFFu;
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t ranks = cluster.num_blocks(), rank = cluster.block_rank(), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint64_t row = blockIdx.y;
    const uint32_t words = (uint32_t)((p.v + 31) / 32);
    const uint32_t lo = (uint32_t)((uint64_t)words * rank / ranks) * 32;
    const uint32_t hi = min((uint32_t)((uint64_t)words * (rank + 1) / ranks) * 32, (uint32_t)p.v);
    cluster_arrive();  // every block has started before another writes into its shared memory
    let_next_start();
    wait_for_previous();
    uint32_t past = 0;
    if (p.history) {
        past = (uint32_t)p.history_len;
        if (p.history_lens) past = (uint32_t)max(0, min(p.history_lens[row], (int32_t)past));
    }
    const uint64_t* logits = p.logits + row * p.v;
    const uint64_t* bias = p.bias ? p.bias + row * p.bias_stride : nullptr;
    const uint32_t* allowed = p.allowed ? p.allowed + row * p.allowed_stride : nullptr;
    const int32_t* hist = p.history + row * p.history_len;
    uint64_t* out = p.out + row * p.v;
    long long bv = INT64_MIN;
    uint32_t bj = kNone;
    bool bad = false;
    for (uint32_t s0 = lo; s0 < hi; s0 += kChooseStep) {
        const uint32_t n = min(kChooseStep, hi - s0), first = s0 + threadIdx.x;
        uint64_t x[kChooseEach], b[kChooseEach];
        uint32_t mask[kChooseEach];
#pragma unroll
        for (int i = 0; i < kChooseEach; i++) {
            const bool on = i * kChooseThreads + threadIdx.x < n;
            x[i] = on ? logits[first + i * kChooseThreads] : 0;
            b[i] = on && bias ? bias[first + i * kChooseThreads] : 0;
            mask[i] = on && allowed ? allowed[first / 32 + i * kChooseWarps] : kNone;
        }
        if (past) {
            __syncthreads();
            for (uint32_t i = threadIdx.x; i < kChooseStep; i += kChooseThreads) counts[i] = 0;
            __syncthreads();
            for (uint32_t i0 = threadIdx.x; i0 < past; i0 += kChooseThreads * 8) {
                uint32_t tok[8];
#pragma unroll
                for (int q = 0; q < 8; q++)
                    tok[q] = i0 + q * kChooseThreads < past ? (uint32_t)hist[i0 + q * kChooseThreads] : s0;
#pragma unroll
                for (int q = 0; q < 8; q++) {
                    bad |= tok[q] >= (uint32_t)p.v;
                    if (tok[q] - s0 < n && i0 + q * kChooseThreads < past) atomicAdd(&counts[tok[q] - s0], 1u);
                }
            }
            __syncthreads();
        }
#pragma unroll
        for (int i = 0; i < kChooseEach; i++) {
            const uint32_t at = i * kChooseThreads + threadIdx.x;
            if (at >= n) continue;
            int64_t z = fx_to_i64(x[i]);
            const uint32_t c = past ? counts[at] : 0;
            if (c) {
                z = round_shift(fx_wmul(z, z > 0 ? p.repeat_pos : p.repeat_neg), 16);
                z = fx_wsub(fx_wsub(z, p.presence), fx_wmul(p.frequency, c));
            }
            z = fx_wadd(z, fx_to_i64(b[i]));
            if (!((mask[i] >> lane) & 1)) z = fx_wadd(z, p.mask_value);
            out[first + i * kChooseThreads] = fx_from_i64(z);
            if (z > bv || bj == kNone) {
                bv = z;
                bj = s0 + at;
            }
        }
    }
    if (bad && rank == 0) atomicOr(p.err, kErrIndex);
    auto take = [&](long long ov, uint32_t oj) {
        if (oj != kNone && (bj == kNone || ov > bv || (ov == bv && oj < bj))) {
            bv = ov;
            bj = oj;
        }
    };
    for (int o = 16; o; o >>= 1) take(__shfl_xor_sync(0xFFFFFFFFu, bv, o), __shfl_xor_sync(0xFFFFFFFFu, bj, o));
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
        p.token[row] = bj;
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

int zkie2_q4_pair(const uint32_t* d_a, const uint32_t* d_b, uint64_t experts, uint64_t k, uint64_t n, uint32_t group,
                  uint32_t* d_out, cudaStream_t stream) {
    Q4Shape s;
    if (experts == 0 || experts > 4096 || !q4_shape(k, n, group, 0, &s) || !d_a || !d_out ||
        (((uintptr_t)d_a | (uintptr_t)d_b | (uintptr_t)d_out) & 15))
        return (int)cudaErrorInvalidValue;
    const uint64_t blocks = experts * (d_b ? s.tiles : (s.tiles + 1) / 2) * s.blocks;
    k_q4_pair<<<(unsigned)(blocks < kSms * 16 ? blocks : kSms * 16), 64, 0, stream>>>(
        reinterpret_cast<const uint4*>(d_a), reinterpret_cast<const uint4*>(d_b), s, blocks,
        reinterpret_cast<uint4*>(d_out));
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
    return group == 32   ? project_rows<32>(p, stream)
           : group == 64 ? project_rows<64>(p, stream)
                         : project_rows<128>(p, stream);
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
    // Query heads to a block: those that share a key head, up to four (a ragged batch of eight with four
    // heads to a key head: two at a time 9 % more; two at most where a value row is wider than 128:
    // their sums stay in registers), fewer where their scores do not fit.  Blocks
    // to a cluster: enough to fill the device with two to an SM, of four token blocks at least, up
    // to eight, as many as find room at once (264 blocks in clusters of eight, 284 in smaller ones,
    // but 224 in clusters of sixteen: 36 us instead of 27 for 16 heads of 4096 tokens); sixteen only
    // where the scores need it.
    const uint32_t blocks = (uint32_t)(capacity / kKvBlock);
    const bool wide = dv > 128;
    for (uint32_t each = p.each >= 3 && !wide ? 4 : p.each >= 2 ? 2 : 1;; each /= 2) {
        const uint64_t rows = batch * heads * ceil_div(p.each, each);
        uint32_t ranks = 1;
        while (ranks < 8 && rows * ranks * 2 <= (ranks == 4 ? 264 : 284) && ranks * 8 <= blocks) ranks *= 2;
        AttendPlan a = attend_plan(each, ranks, blocks, p.c.dk, p.c.dv);
        for (; a.shared > (a.ranks < 8 ? kAttShared / 2 : kAttShared) && a.ranks < kMaxRanks && a.ranks < blocks;)
            a = attend_plan(each, a.ranks * 2, blocks, p.c.dk, p.c.dv);
        if (a.shared > kAttShared && each > 1) continue;
        if (a.shared > kAttShared) return (int)cudaErrorInvalidValue;
        if (wide) return each == 2 ? attend_launch<2, 2>(p, a, stream) : attend_launch<1, 2>(p, a, stream);
        return each == 4   ? attend_launch<4, 1>(p, a, stream)
               : each == 2 ? attend_launch<2, 1>(p, a, stream)
                           : attend_launch<1, 1>(p, a, stream);
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
    // Blocks to a row: the fewest steps of the vocabulary at which the rows' clusters find room at
    // once, with up to half as many blocks again where those do too.  A second wave of clusters
    // costs more than a second step (sixteen rows of 50257 logits: 9.4 us as clusters of thirteen,
    // 12.8 of sixteen; 32 rows 12.8 us as clusters of nine, 18.7 of sixteen), and clusters that
    // fill an SM's share of threads evenly more than the steps alone (24 rows: 11.2 and 12.8 us).
    static std::atomic<uint64_t> set{0};
    static std::atomic<uint32_t> known[kMaxRanks + 1];
    const void* kernel = reinterpret_cast<const void*>(k_choose_token);
    ZK_TRY(allow_shared(kernel, 0, &set, true));
    auto fits = [&](uint32_t r) { return clusters_at_once(kernel, kChooseThreads, 0, r, known) >= batch; };
    const uint64_t all = ceil_div(vocab, kChooseStep);
    uint32_t need = all < kMaxRanks ? (uint32_t)all : kMaxRanks;
    for (; need > 1; need--) {
        need = (uint32_t)ceil_div(all, ceil_div(all, need));  // as few blocks at the same number of steps
        if (fits(need)) break;
    }
    uint32_t ranks = need + need / 2 < kMaxRanks ? need + need / 2 : kMaxRanks;
    while (ranks > need && !fits(ranks)) ranks--;
    return launch(k_choose_token, dim3(ranks, (unsigned)batch), kChooseThreads, 0, ranks, stream, p);
}

}  // extern "C"
