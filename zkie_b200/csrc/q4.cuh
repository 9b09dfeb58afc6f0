// q4.cuh -- products of a few rows of fixed-point numbers with a weight held
// in 4 bits: w[k][n] = c[k][n] s[k / G][n] with whole codes c in [-8, 7] and
// whole scales s in [0, 65535] (G = 32, 64 or 128 rows to a scale).
//
// A row x of signed numbers (|x| <= 0x7F7F7F7F) is written as
// four signed byte digits, x = sum_p d_p 256^p, and the digits of two rows
// are the eight columns of an m16n8k32 integer matrix instruction whose 16
// rows are 16 columns n of the weight.  A warp thus streams the codes of 16
// columns once, in blocks of 64 k (512 bytes of codes, 16 to a lane), and
// spends two instructions a block on two rows of x.  The instruction is the
// warp-wide mma.sync (two cycles of an SM, latency 20): with up to eight rows
// a product is bound by the weight's bytes and by what each warp does around
// the instruction -- taking codes apart, scaling groups.  At eight rows the
// matrix pipe is busy 19 % of the time and 126 registers a thread leave four
// warps to a scheduler, too few to cover its latency and that of the
// instructions around it.  Accumulators in tensor memory would free registers
// and cost a set-up and a read-back of every group's sums; that form has not
// been measured.
//
// The sums are exact: within a block 16 c d stays below 2^29 even with two
// digits joined, the scaled group sums are added in 64 bits, and a padded K
// of at most kQ4MaxK keeps the whole sum below 2^63, where a sum of 64-bit
// numbers and one in the field are the same number.
//
// Layout.  K is padded to blocks of 64 (within each segment where the weight
// has segments), N to tiles of 16; the blocks of a tile follow one another,
// tile after tile.  A block holds for lane (g = lane / 4, t = lane % 4) four
// words; byte j of word q holds in its low half the code of row 8 t + 4 (q / 2)
// + j and in its high half that of row 32 + 8 t + 4 (q / 2) + j, both of column
// g + 8 (q % 2).  After the codes come eight words of scales, s[g] | s[g + 8]
// << 16 (for G = 32 a second eight, of the second 32 rows; for G = 128 two
// blocks repeat theirs, 3 % of the bytes for blocks that stand alone).  Any
// run of blocks is one piece of memory, so one bulk copy brings it.  Digits
// lie in the order in which a lane reads them: q4_pos.
#pragma once
#include <cstdint>

#include "gl64.cuh"
#include "fixed.cuh"

namespace zk {

constexpr uint32_t kQ4MaxK = 8192;
constexpr uint32_t kErrRange = 8u;  // a value outside the range the single-token kernels take

// Shape of a packed weight: k_seg rows to a segment (k itself without
// segments), padded to kp_seg; blocks per tile over all segments, bytes of one.
struct Q4Shape {
    uint32_t k, n, group, segs, k_seg, kp_seg, blocks, tiles, bytes;
};

inline bool q4_shape(uint64_t k, uint64_t n, uint32_t group, uint64_t segment, Q4Shape* s) {
    if (k == 0 || n == 0 || k > kQ4MaxK || n > 0x7FFFFFF0ull) return false;
    if (group != 32 && group != 64 && group != 128) return false;
    if (segment && (segment > k || k % segment)) return false;
    s->k = (uint32_t)k;
    s->n = (uint32_t)n;
    s->group = group;
    s->k_seg = (uint32_t)(segment ? segment : k);
    s->segs = s->k / s->k_seg;
    s->kp_seg = (s->k_seg + 63) / 64 * 64;
    if ((uint64_t)s->kp_seg * s->segs > kQ4MaxK) return false;
    s->blocks = s->kp_seg / 64 * s->segs;
    s->tiles = (s->n + 15) / 16;
    s->bytes = group == 32 ? 576 : 544;
    return true;
}

// byte of digit k (within a block of 64) in a lane's reading order
__device__ __forceinline__ uint32_t q4_pos(uint32_t k) {
    return (k & ~63u) + 16 * ((k & 31) >> 3) + 8 * ((k & 63) >> 5) + (k & 7);
}

// the four digit bytes of a number, lowest first; false (and 0) out of range
__device__ __forceinline__ bool q4_digits(int64_t v, uint32_t* d) {
    const bool ok = v >= -0x7F7F7F7Fll && v <= 0x7F7F7F7Fll;
    *d = ok ? ((uint32_t)v + 0x80808080u) ^ 0x80808080u : 0u;
    return ok;
}

// the same from zero
__device__ __forceinline__ void mma_s8_new(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                           uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(0));
}

// fx_to_i64 in three instructions: v, less p = 2^64 - 0xFFFFFFFF from 2^63 on
__device__ __forceinline__ int64_t q4_number(uint64_t v) {
    return (int64_t)(v + (uint32_t)((int32_t)(v >> 32) >> 31));
}

// q4_digits of a field element, which every block does for every number of its rows
__device__ __forceinline__ bool q4_digits_of(uint64_t v, uint32_t* d) {
    const uint64_t t = (uint64_t)q4_number(v) + 0x7F7F7F7Fu;
    const bool ok = t <= 0xFEFEFEFEull;
    *d = ok ? ((uint32_t)t + 0x01010101u) ^ 0x80808080u : 0u;
    return ok;
}

// the digits of four consecutive k, one word to each of the four digit rows
__device__ __forceinline__ void q4_store_digits(uint8_t* to, size_t stride, const uint32_t (&d)[4]) {
#pragma unroll
    for (int q = 0; q < 4; q++) {
        const uint32_t lo = __byte_perm(d[0], d[1], q | ((4 + q) << 4));
        const uint32_t hi = __byte_perm(d[2], d[3], q | ((4 + q) << 4));
        *reinterpret_cast<uint32_t*>(to + q * stride) = __byte_perm(lo, hi, 0x5410);
    }
}

// The digits of rows of x (k_seg numbers to each of `segs` segments, padded to
// kp_seg) into digit rows of `stride` bytes, four to a row: fours of numbers
// [begin, end) counted over all rows, and to `also` (another block's shared
// memory) where given; false in a thread that met a number out of range.  A thread takes four numbers at a
// time and has AHEAD such loads under way, whatever rows they belong to: one
// after the other, eight rows would cost eight times the memory's latency.
template <int THREADS, int AHEAD>
__device__ __forceinline__ bool q4_digitise(const uint64_t* x, uint64_t ldx, uint32_t segs, uint32_t k_seg,
                                            uint32_t kp_seg, uint32_t begin, uint32_t end, uint8_t* digits,
                                            uint32_t stride, uint8_t* also = nullptr) {
    const uint32_t quads = segs * kp_seg / 4;
    const uint32_t per_row = 0xFFFFFFFFu / quads + 1, per_seg = 0xFFFFFFFFu / kp_seg + 1;  // reciprocals for __umulhi:
    // exact, a quotient's numerator and divisor being below 2^16 (and the divisor no less than 16)
    const bool wide = (((uintptr_t)x | (ldx * 8)) & 15) == 0 && k_seg % 4 == 0;  // 16-byte loads
    bool ok = true;
    for (uint32_t i0 = begin + threadIdx.x; i0 < end; i0 += THREADS * AHEAD) {
        uint64_t v[AHEAD][4];
        uint32_t to[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; u++) {
            const uint32_t i = i0 + u * THREADS;
            const bool on = i < end;
            const uint32_t r = on ? __umulhi(i, per_row) : 0, k0 = on ? (i - r * quads) * 4 : 0;
            const uint32_t seg = segs > 1 ? __umulhi(k0, per_seg) : 0, in = k0 - seg * kp_seg;
            const uint64_t* from = x + r * ldx + (seg * k_seg + in);
            to[u] = on ? r * 4 * stride + q4_pos(k0) : ~0u;
            if (wide) {
                ulonglong2 lo = make_ulonglong2(0, 0), hi = lo;
                if (on && in < k_seg) {
                    lo = reinterpret_cast<const ulonglong2*>(from)[0];
                    hi = reinterpret_cast<const ulonglong2*>(from)[1];
                }
                v[u][0] = lo.x, v[u][1] = lo.y, v[u][2] = hi.x, v[u][3] = hi.y;
            } else {
#pragma unroll
                for (int j = 0; j < 4; j++) v[u][j] = on && in + j < k_seg ? from[j] : 0;
            }
        }
#pragma unroll
        for (int u = 0; u < AHEAD; u++)
            if (to[u] != ~0u) {
                uint32_t d[4];
#pragma unroll
                for (int j = 0; j < 4; j++) ok &= q4_digits_of(v[u][j], &d[j]);
                q4_store_digits(digits + to[u], stride, d);
                if (also) q4_store_digits(also + to[u], stride, d);
            }
    }
    return ok;
}

// bytes of a digit row: 64 mod 128, so that the eight lanes that read at once
// (two rows, 64 bytes each) meet no shared-memory bank twice
inline uint32_t q4_digit_stride(uint32_t blocks) { return blocks % 2 ? blocks * 64 : blocks * 64 + 64; }

__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// ---- a warp's ring of slots, filled by bulk copies ----------------------------------------
// One lane asks for a run of blocks with one instruction; a barrier in shared
// memory counts its bytes.  The bytes in flight depend on no register, and the
// stream of a warp's blocks runs on across tiles, sums and block-wide waits.
// A wait gives up after a bounded number of attempts (a second or so) and says
// so in the error word; nothing more is then asked for or waited for.
constexpr uint32_t kErrWait = 32u;
constexpr uint32_t kTries = 1u << 18;

struct Patience {
    bool failed = false;
};

// Shared memory by its own 32-bit addresses: a load is one instruction with its
// offset in it, where a generic pointer costs 64-bit sums.
__device__ __forceinline__ uint32_t shared_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ uint4 load16(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
    return v;
}
__device__ __forceinline__ uint32_t load4(uint32_t at) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(at));
    return v;
}

__device__ __forceinline__ void barrier_init(uint32_t bar) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(bar) : "memory");
}
// after the inits, before the first copy
__device__ __forceinline__ void barrier_init_done() {
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}
__device__ __forceinline__ void barrier_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bulk_copy(uint32_t to, const void* from, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(to),
                 "l"(from), "r"(bytes), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ void barrier_wait(uint32_t bar, uint32_t parity, Patience& patience) {  // the whole warp
    if (patience.failed) return;
    for (uint32_t i = 0; i < kTries; i++) {
        uint32_t done;
        asm volatile(
            "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
            : "=r"(done)
            : "r"(bar), "r"(parity)
            : "memory");
        if (__all_sync(0xFFFFFFFFu, done)) return;
    }
    patience.failed = true;
}
// At a kernel's end: a wait that gave up is told, and the copies that it was
// for get another ten milliseconds before their shared memory is given away.
__device__ __forceinline__ void patience_end(const Patience& patience, uint32_t* err) {
    if (!patience.failed) return;
    atomicOr(err, kErrWait);
    for (int i = 0; i < 100; i++) __nanosleep(100000);
}

// ---- overlap with the kernel before (programmatic dependent launch) --------------------------
// Every kernel here lets its successor start early and waits, before it reads
// or writes anything that an earlier kernel may have written or may still
// read, until all earlier kernels are done.  What they may have written is then
// read with plain loads: __ldg wants data that stays the same while the kernel
// runs, its time before the wait included, and the compiler may move it (and
// __ldcg) to before the wait.
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// the two halves of a cluster's barrier
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait;" ::: "memory"); }

// a run of bytes (16-byte aligned, a multiple of 16) into the second-level cache
__device__ __forceinline__ void prefetch_l2(const void* p, uint32_t bytes) {
    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p), "r"(bytes) : "memory");
}

// Running sums of one tile of 16 columns against NT pairs of rows: the scaled
// groups' (row g and g + 8 of the tile; lane t holds digits 2 (t % 2) and
// 2 (t % 2) + 1, joined, of row t / 2 of a pair).
template <int NT>
struct Q4Sum {
    long long a[NT][2];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < NT; i++) a[i][0] = a[i][1] = 0;
    }
    // c: a group's products (N of the pairs), s: its scales
    template <int N>
    __device__ __forceinline__ void add_group(const int (&c)[N][4], uint32_t s) {
        const int s0 = (int)(s & 0xFFFFu), s1 = (int)(s >> 16);
#pragma unroll
        for (int i = 0; i < N; i++) {
            a[i][0] += (long long)(c[i][0] + (c[i][1] << 8)) * s0;
            a[i][1] += (long long)(c[i][2] + (c[i][3] << 8)) * s1;
        }
    }
    // The sum itself, sixteenfold and split over two lanes until here: in lane
    // (g, t) that of column g + 8 (t % 2) of the tile and row t / 2 of pair i.
    __device__ __forceinline__ long long finish(int i) const {
        const bool high = threadIdx.x & 1;
        const long long got = __shfl_xor_sync(0xFFFFFFFFu, high ? a[i][0] : a[i][1], 1) >> 4;
        const long long mine = (high ? a[i][1] : a[i][0]) >> 4;
        return (long long)((unsigned long long)(high ? got : mine) + ((unsigned long long)(high ? mine : got) << 16));
    }
};

// Sums of 64-bit numbers from several warps in shared memory: three words of
// 22, 22 and 20 bits a number, each added by an atomic that returns nothing
// (the 64-bit one is a loop of compare-and-swaps here, 9 to 240 cycles a warp).
// Up to 1024 numbers to a sum; exact modulo 2^64.
struct Limbs {
    uint32_t* w;
    uint32_t n;  // numbers
    __device__ __forceinline__ void add(uint32_t at, long long v) const {
        atomicAdd(w + at, (uint32_t)v & 0x3FFFFFu);
        atomicAdd(w + n + at, (uint32_t)(v >> 22) & 0x3FFFFFu);
        atomicAdd(w + 2 * n + at, (uint32_t)(v >> 44));
    }
    __device__ __forceinline__ long long get(uint32_t at) const {
        return (long long)((unsigned long long)w[at] + ((unsigned long long)w[n + at] << 22) +
                           ((unsigned long long)w[2 * n + at] << 44));
    }
    __device__ __forceinline__ void clear(uint32_t at) const { w[at] = w[n + at] = w[2 * n + at] = 0; }
    template <int THREADS>  // all of them (four and a 16-byte boundary at least), by a whole block
    __device__ __forceinline__ void clear() const {
        for (uint32_t i = threadIdx.x; i < 3 * n / 4; i += THREADS) reinterpret_cast<uint4*>(w)[i] = make_uint4(0, 0, 0, 0);
    }
};

// A lane's place in a block in shared memory: its codes, and its scales
struct Q4Lane {
    uint32_t codes, scales;
    __device__ __forceinline__ explicit Q4Lane(uint32_t block)
        : codes(block + (threadIdx.x & 31) * 16), scales(block + 512 + (threadIdx.x & 31) / 4 * 4) {}
};

// The products of one block's codes with NT pairs of rows, added to c: first
// the rows whose codes lie in the low halves, then those in the high ones.
template <int NT, int MAX, bool LOW>
__device__ __forceinline__ void q4_half(int (&c)[NT][4], const uint4& w, const uint4 (&b)[MAX], bool fresh) {
    constexpr uint32_t kHigh = 0xF0F0F0F0u;  // a code in a byte's high half is sixteen times itself
    const uint32_t a0 = (LOW ? w.x << 4 : w.x) & kHigh, a1 = (LOW ? w.y << 4 : w.y) & kHigh,
                   a2 = (LOW ? w.z << 4 : w.z) & kHigh, a3 = (LOW ? w.w << 4 : w.w) & kHigh;
#pragma unroll
    for (int i = 0; i < NT; i++) {
        const uint32_t b0 = LOW ? b[i].x : b[i].z, b1 = LOW ? b[i].y : b[i].w;
        if (fresh)
            mma_s8_new(c[i], a0, a1, a2, a3, b0, b1);
        else
            mma_s8(c[i], a0, a1, a2, a3, b0, b1);
    }
}

// One block of 64 k, `off` bytes on from `at`, against NT of the MAX pairs of
// rows, their digits in b.  TWO: two groups of 32 rows, else one.
template <bool TWO, int NT, int MAX>
__device__ __forceinline__ void q4_block(Q4Sum<MAX>& sum, const Q4Lane& at, uint32_t off, const uint4 (&b)[MAX]) {
    const uint4 w = load16(at.codes + off);
    const uint32_t s0 = load4(at.scales + off), s1 = TWO ? load4(at.scales + off + 32) : 0;
    int c[NT][4];
    q4_half<NT, MAX, true>(c, w, b, true);
    if (TWO) sum.template add_group<NT>(c, s0);
    q4_half<NT, MAX, false>(c, w, b, TWO);
    sum.template add_group<NT>(c, TWO ? s1 : s0);
}

// Two blocks that share a group of 128 rows: scaled once
template <int NT>
__device__ __forceinline__ void q4_group(Q4Sum<NT>& sum, const Q4Lane& at, uint32_t off, uint32_t bytes,
                                         const uint4 (&b)[2][NT]) {
    int c[NT][4];
    const uint4 w = load16(at.codes + off), v = load16(at.codes + off + bytes);
    q4_half<NT, NT, true>(c, w, b[0], true);
    q4_half<NT, NT, false>(c, w, b[0], false);
    q4_half<NT, NT, true>(c, v, b[1], false);
    q4_half<NT, NT, false>(c, v, b[1], false);
    sum.template add_group<NT>(c, load4(at.scales + off));
}

// round_div(a, 2^s): the quotient rounded down, plus the highest bit shifted out
__device__ __forceinline__ int64_t round_shift(int64_t a, uint32_t s) {
    return s ? (a >> s) + ((a >> (s - 1)) & 1) : a;
}

// from_i64(to_i64(v)'s table entry): Op::GeluIndex and Op::Lookup on one value
__device__ __forceinline__ uint64_t table_at(const uint64_t* table, uint64_t len, int64_t v,
                                             int64_t offset) {
    const int64_t i = fx_wadd(v, offset), hi = (int64_t)len - 1;
    return table[i < 0 ? 0 : (i > hi ? hi : i)];
}

// A softmax's weight, round_div(e 2^16, sum) for 0 <= e < 2^31 and e <= sum <
// 2^52: estimated in single precision from inv = 1 / sum -- each of the five
// roundings is off by 2^-23 at most, so the estimate of at most 2^16 by less
// than 1/16 -- and set right by the remainder, which is exact.
__device__ __forceinline__ int softmax_weight(uint32_t e, int64_t sum, float inv) {
    const int64_t a = (int64_t)e << 16;
    int q = (int)((float)e * 65536.0f * inv);
    int64_t r = a - q * sum;
    if (r < 0) {
        q--;
        r += sum;
    } else if (r >= sum) {
        q++;
        r -= sum;
    }
    return 2 * r >= sum ? q + 1 : q;
}

// the maximum and the sum over a warp's lanes, in whole-warp reductions of 32 bits
__device__ __forceinline__ int64_t warp_max(int64_t v) {
    const int hi = __reduce_max_sync(0xFFFFFFFFu, (int)(v >> 32));
    const uint32_t lo = __reduce_max_sync(0xFFFFFFFFu, (int)(v >> 32) == hi ? (uint32_t)v : 0u);
    return (int64_t)((uint64_t)(uint32_t)hi << 32 | lo);
}
// of numbers in [0, 2^42)
__device__ __forceinline__ int64_t warp_sum(int64_t v) {
    const uint32_t lo = __reduce_add_sync(0xFFFFFFFFu, (uint32_t)v & 0xFFFFu);
    return ((int64_t)__reduce_add_sync(0xFFFFFFFFu, (uint32_t)(v >> 16)) << 16) + lo;
}

}  // namespace zk
