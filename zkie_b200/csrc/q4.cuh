// q4.cuh -- products of a few rows of fixed-point numbers with a weight held
// in 4 bits: w[k][n] = c[k][n] s[k / G][n] with whole codes c in [-8, 7] and
// whole scales s in [0, 65535] (G = 32, 64 or 128 rows to a scale).
//
// A row x of signed numbers (|x| <= 0x7F7F7F7F) is written as
// four signed byte digits, x = sum_p d_p 256^p, and the digits of two rows
// are the eight columns of an m16n8k32 integer matrix instruction whose 16
// rows are 16 columns n of the weight.  A warp thus streams the codes of 16
// columns once, in 512-byte blocks of 64 k (16 bytes to a lane, contiguous),
// and spends two instructions a block on two rows of x.  The instruction is
// the warp-wide mma.sync: a product for at most a few rows is bound by the
// bytes of the weight, at 4 bits a multiply, and its use of the matrix pipe
// is a few per cent either way, so nothing is gained from accumulators in
// tensor memory and a good deal of set-up is saved.
//
// The sums are exact: within a group 16 c d stays below 2^29 even with two
// digits joined, the scaled group sums are added in 64 bits, and a padded K
// of at most kQ4MaxK keeps the whole sum below 2^63, where a sum of 64-bit
// numbers and one in the field are the same number.
//
// Layout.  K is padded to blocks of 64 (128 for G = 128; within each segment
// where the weight has segments), N to tiles of 16.  Block (tile, b) holds
// for lane (g = lane / 4, t = lane % 4) four words; byte j of word q holds in
// its low half the code of row 8 t + 4 (q / 2) + j and in its high half that
// of row 32 + 8 t + 4 (q / 2) + j, both of column g + 8 (q % 2).  The scales
// of (tile, group) are eight words: s[g] | s[g + 8] << 16.  Digits lie in the
// order in which a lane reads them: q4_pos.
#pragma once
#include <cstdint>

#include "gl64.cuh"
#include "fixed.cuh"

namespace zk {

constexpr uint32_t kQ4MaxK = 8192;
constexpr uint32_t kErrRange = 8u;  // a value outside the range the single-token kernels take

// Shape of a packed weight: k_seg rows to a segment (k itself without
// segments), padded to kp_seg; blocks and groups per tile over all segments.
struct Q4Shape {
    uint32_t k, n, group, segs, k_seg, kp_seg, blocks, groups, tiles;
};

inline bool q4_shape(uint64_t k, uint64_t n, uint32_t group, uint64_t segment, Q4Shape* s) {
    if (k == 0 || n == 0 || k > kQ4MaxK || n > 0x7FFFFFF0ull) return false;
    if (group != 32 && group != 64 && group != 128) return false;
    if (segment && (segment > k || k % segment)) return false;
    const uint32_t unit = group == 128 ? 128 : 64;
    s->k = (uint32_t)k;
    s->n = (uint32_t)n;
    s->group = group;
    s->k_seg = (uint32_t)(segment ? segment : k);
    s->segs = s->k / s->k_seg;
    s->kp_seg = (s->k_seg + unit - 1) / unit * unit;
    if ((uint64_t)s->kp_seg * s->segs > kQ4MaxK) return false;
    s->blocks = s->kp_seg / 64 * s->segs;
    s->groups = s->kp_seg / group * s->segs;
    s->tiles = (s->n + 15) / 16;
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

// the digits of four consecutive k, one word to each of the four digit rows
__device__ __forceinline__ void q4_store_digits(uint8_t* to, size_t stride, const uint32_t (&d)[4]) {
#pragma unroll
    for (int q = 0; q < 4; q++) {
        const uint32_t lo = __byte_perm(d[0], d[1], q | ((4 + q) << 4));
        const uint32_t hi = __byte_perm(d[2], d[3], q | ((4 + q) << 4));
        *reinterpret_cast<uint32_t*>(to + q * stride) = __byte_perm(lo, hi, 0x5410);
    }
}

// bytes of a digit row: 64 mod 128, so that the eight lanes that read at once
// (two rows, 64 bytes each) meet no shared-memory bank twice
inline uint32_t q4_digit_stride(uint32_t blocks) { return blocks % 2 ? blocks * 64 : blocks * 64 + 64; }

__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// ---- asynchronous copies: a warp's ring of slots in shared memory ---------------------------
// A lane copies the 16 bytes that it will read itself (scales: a few lanes,
// for all), so a slot is ready when the lane's own copies are and the warp has
// met once; the bytes in flight do not depend on registers, and the stream of
// a warp's blocks runs on across tiles, sums and barriers.
__device__ __forceinline__ void copy16(void* to, const void* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from)
                 : "memory");
}
__device__ __forceinline__ void copy4(void* to, const void* from) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from)
                 : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// wait until at most n (< N + 1) of the groups asked for are still on their way
template <int N>
__device__ __forceinline__ void copy_wait_upto(uint32_t n) {
    if constexpr (N == 0) {
        copy_wait<0>();
    } else {
        if (n >= N)
            copy_wait<N>();
        else
            copy_wait_upto<N - 1>(n);
    }
}

// ---- overlap with the kernel before (programmatic dependent launch) --------------------------
// Every kernel here lets its successor start early and waits, before it reads
// or writes anything that an earlier kernel may have written or may still
// read, until all earlier kernels are done.
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// the two halves of a cluster's barrier
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }

// a run of bytes (16-byte aligned, a multiple of 16) into the second-level cache
__device__ __forceinline__ void prefetch_l2(const void* p, uint32_t bytes) {
    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p), "r"(bytes) : "memory");
}

// Running sums of one tile of 16 columns against NT pairs of rows: c the
// present group's, a the scaled groups' (row g and g + 8 of the tile; lane t
// holds digits 2 (t % 2) and 2 (t % 2) + 1, joined, of row t / 2 of a pair).
template <int NT>
struct Q4Sum {
    int c[NT][4];
    long long a[NT][2];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < NT; i++) {
            c[i][0] = c[i][1] = c[i][2] = c[i][3] = 0;
            a[i][0] = a[i][1] = 0;
        }
    }
    template <int N>
    __device__ __forceinline__ void scale_group(uint32_t s) {
        const int s0 = (int)(s & 0xFFFFu), s1 = (int)(s >> 16);
#pragma unroll
        for (int i = 0; i < N; i++) {
            a[i][0] += (long long)(c[i][0] + (c[i][1] << 8)) * s0;
            a[i][1] += (long long)(c[i][2] + (c[i][3] << 8)) * s1;
            c[i][0] = c[i][1] = c[i][2] = c[i][3] = 0;
        }
    }
    // The sums themselves: sixteenfold and split over two lanes until here.
    // Valid in every lane: the number of row t / 2 of the pair.
    __device__ __forceinline__ void finish(int i, long long* v0, long long* v1) const {
        const bool high = threadIdx.x & 1;
        long long r[2];
#pragma unroll
        for (int q = 0; q < 2; q++) {
            const long long mine = a[i][q] >> 4;
            const long long other = __shfl_xor_sync(0xFFFFFFFFu, mine, 1);
            const long long lo = high ? other : mine, hi = high ? mine : other;
            r[q] = (long long)((unsigned long long)lo + ((unsigned long long)hi << 16));
        }
        *v0 = r[0];
        *v1 = r[1];
    }
};

// One block of 64 k for NT of the MAX pairs: w the lane's codes, s0 (and s1 for G = 32) the scales of
// the block's group(s), b the lane's digits; `last` where a group of 128 ends.
template <int G, int NT, int MAX>
__device__ __forceinline__ void q4_block_n(Q4Sum<MAX>& sum, const uint4& w, uint32_t s0, uint32_t s1,
                                           const uint4 (&b)[MAX], bool last) {
    constexpr uint32_t kHigh = 0xF0F0F0F0u;  // a code in a byte's high half is sixteen times itself
    {
        const uint32_t a0 = (w.x << 4) & kHigh, a1 = (w.y << 4) & kHigh, a2 = (w.z << 4) & kHigh,
                       a3 = (w.w << 4) & kHigh;
#pragma unroll
        for (int i = 0; i < NT; i++) mma_s8(sum.c[i], a0, a1, a2, a3, b[i].x, b[i].y);
    }
    if (G == 32) sum.template scale_group<NT>(s0);
    {
        const uint32_t a0 = w.x & kHigh, a1 = w.y & kHigh, a2 = w.z & kHigh, a3 = w.w & kHigh;
#pragma unroll
        for (int i = 0; i < NT; i++) mma_s8(sum.c[i], a0, a1, a2, a3, b[i].z, b[i].w);
    }
    if (G == 32)
        sum.template scale_group<NT>(s1);
    else if (G == 64)
        sum.template scale_group<NT>(s0);
    else if (last)
        sum.template scale_group<NT>(s0);
}

template <int G, int NT>
__device__ __forceinline__ void q4_block(Q4Sum<NT>& sum, const uint4& w, uint32_t s0, uint32_t s1,
                                         const uint4 (&b)[NT], bool last) {
    q4_block_n<G, NT, NT>(sum, w, s0, s1, b, last);
}

// The scale words of block b of a tile into a slot (16 words): lanes t = 0,
// and t = 1 for G = 32 with its second group.
template <int G>
__device__ __forceinline__ void copy_scales(uint32_t* to, const uint32_t* tile_scales, uint32_t b, uint32_t g,
                                            uint32_t t) {
    if (t < (G == 32 ? 2 : 1)) {
        const uint32_t group = G == 32 ? 2 * b + t : (G == 64 ? b : b / 2);
        copy4(to + 8 * t + g, tile_scales + (uint64_t)group * 8 + g);
    }
}

// from_i64(to_i64(v)'s table entry): Op::GeluIndex and Op::Lookup on one value
__device__ __forceinline__ uint64_t table_at(const uint64_t* __restrict__ table, uint64_t len, int64_t v,
                                             int64_t offset) {
    const int64_t i = fx_wadd(v, offset), hi = (int64_t)len - 1;
    return __ldg(table + (i < 0 ? 0 : (i > hi ? hi : i)));
}

// q = round_div(a, b) for a >= 0 below 2^52 and 0 < b below 2^52, with inv =
// 1 / b to double precision: the estimate is off by one at most
__device__ __forceinline__ int64_t round_div_near(int64_t a, int64_t b, double inv) {
    int64_t q = (int64_t)((double)a * inv), r = a - q * b;
    if (r < 0) {
        q--;
        r += b;
    } else if (r >= b) {
        q++;
        r -= b;
    }
    return 2 * r >= b ? q + 1 : q;
}

}  // namespace zk
