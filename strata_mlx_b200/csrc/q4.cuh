// 4-bit weights with a float16 scale and bias for each group of 32, 64 or 128 columns: the layout the kernels
// read, and a tile of two strips of it times 8 activation rows on the tensor cores.
//
//   w[r, c] = code[r, c] * scale[r, c / G] + bias[r, c / G],   code in 0 .. 15
//
// Layout (made once from the file's arrays by smoe_q4_pack). A matrix is strips of 16 rows, a strip is tiles of 128
// columns one after the other, a tile is 1024 bytes of codes (64 a row) and then 128 / G (scale, bias) pairs a row:
//
//   [strip][tile][ 16 rows x 64 B codes ][ 16 rows x 128 / G x (scale, bias) ]
//
// so a strip is one run of memory that bulk copies fetch in any pieces, every piece a multiple of 16 bytes. Rows
// past the last and columns past the last are zero codes with zero scales and biases.
//
// A row's 16 code words of a tile: word j of chunk t (four chunks of 16 bytes) holds the codes of columns 32 j + 8 t ..
// + 7, so that lane (g, t) of a warp (g = lane / 4, t = lane % 4) has its columns of all four 32-column runs in one
// 16-byte read. Chunk t of row r lies at place t ^ (r / 2 % 4): eight rows' chunks t are on eight different bank groups
// (a thread a row reads so in the prompt's product). In a word, columns 0 .. 7 lie in nibbles 0, 4, 2, 6, 1, 5, 3, 7, the whole
// rotated left by two bits: the nibbles under one mask, 16 bits apart, are neighbouring columns, and nibbles 0 and 1 lie in bits
// 2 .. 5 and 6 .. 9 of a half word.
//
// Arithmetic. A run of 32 columns is two m16n8k16 MMAs, rows the M side, activation rows the N side. The order of
// columns inside an MMA is free as long as A and B agree, so lane (g, t)'s word goes in as it lies: columns 0 .. 3 to
// one MMA, 4 .. 7 to the other (so that B's register pairs are halves of a 16-byte load). With float16 activations a nibble
// needs no conversion at all: (word & 0x003c003c) is a pair of float16 subnormals q * 2^-22, exact in the tensor core, and
// (word & 0x03c003c0) a pair of 16 q * 2^-22; the two MMAs keep sums of their own, joined as lo + hi / 16 at the end of the group,
// and the 2^22 comes at the end of the row. The bias takes sum x over the group, from the same B operands times a matrix of
// 2^-14. Products are exact and sums are float32, which the tensor core adds with a fixed number of bits below its operands'
// exponents: a subnormal counts there as 2^-14, so codes lie as high in the mantissa as two to a half word allow and the matrix
// of ones is the least normal number. (With codes in bits 0 .. 7 and ones of 2^-24 4.8 % of a
// 640 x 2560 layer's results were rounded to the wrong neighbour, now 0.1 %, and of a block of 512 experts 23 %, now 0.4 %.)
// Float32 activations are three bfloat16 pieces (8 + 8 + 8 bits: the whole float32), each through the same MMAs;
// codes become bfloat16 by (4 q | 0x4200) - 40, exact too: q - 8, with bias + 8 scale in the bias's place. A group's weights
// lie on both sides of zero mostly, q scale and bias are then numbers of one size that nearly cancel, and their float32 sums
// lose more than those of q - 8 do (a block of 64 experts, 2048 wide, is 1.03e-6 of its result off with q, 7.4e-7 with
// q - 8, and 2.7e-7 with sums of their own for the activations' small pieces).
#pragma once

#include <cuda_bf16.h>

#include <type_traits>

#include "common.cuh"
#include "tc05.cuh"

namespace smoe {
namespace q4 {

constexpr int kRows = 16;        // rows of a strip
constexpr int kCols = 128;       // columns of a tile
constexpr int kCodeBytes = 1024; // codes of a tile

template <int G>
__host__ __device__ constexpr int tile_bytes() {
    return kCodeBytes + kRows * (kCols / G) * 4;
}
__host__ __device__ constexpr int tile_bytes_of(int g) { return kCodeBytes + kRows * (kCols / g) * 4; }
__host__ __device__ constexpr int64_t tiles_of_cols(int64_t cols) { return (cols + kCols - 1) / kCols; }
__host__ __device__ constexpr int64_t strips_of_rows(int64_t rows) { return (rows + kRows - 1) / kRows; }

constexpr uint32_t kWaitLimit = 1u << 22;
__device__ __forceinline__ bool wait_for(uint64_t* bar, uint32_t parity) { return tc::mbar_wait(bar, parity, kWaitLimit); }

// Where a row's chunk t lies in a tile, in bytes; lane (g, t)'s chunk of row g (that of row g + 8 lies 512 further)
__host__ __device__ constexpr int chunk_at(int row, int t) { return row * 64 + ((t ^ ((row >> 1) & 3)) << 4); }
__device__ __forceinline__ int lane_chunk(int lane) { return chunk_at(lane >> 2, lane & 3); }
// The nibble of a word that holds its column i
__host__ __device__ constexpr int nibble_of(int i) { return (i >> 2) + 2 * ((i >> 1) & 1) + 4 * (i & 1); }
__device__ __forceinline__ uint32_t turn(uint32_t w, int right) { return __funnelshift_r(w, w, right); }
// turn(w, 8). (Written as a permutation of bytes: a funnel shift costs the kernels registers, 64007 x 2560 at 5 tokens 24.7 us
// against 21.9.)
__device__ __forceinline__ uint32_t turn8(uint32_t w) {
    uint32_t r;
    asm("prmt.b32 %0, %1, %1, 0x0321;" : "=r"(r) : "r"(w));
    return r;
}
constexpr uint32_t kLow = 0x003c003cu, kHigh = 0x03c003c0u;  // nibbles 0 and 4, 1 and 5 (turned by 8: 2 and 6, 3 and 7)
// A word of eight codes, weight i in bits 4 i, in the layout's order of nibbles, and back
__device__ __forceinline__ uint32_t nibbles_in(uint32_t w) {
    uint32_t r = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) r |= ((w >> (4 * i)) & 15u) << (4 * nibble_of(i));
    return (r << 2) | (r >> 30);
}
__device__ __forceinline__ uint32_t nibbles_out(uint32_t w) {
    uint32_t r = 0;
    w = turn(w, 2);
#pragma unroll
    for (int i = 0; i < 8; ++i) r |= ((w >> (4 * nibble_of(i))) & 15u) << (4 * i);
    return r;
}

// The (scale, bias) pairs of row `row` of a tile in shared memory
template <int G>
__device__ __forceinline__ void load_pairs(const uint8_t* tile, int row, uint32_t (&v)[kCols / G]) {
    const uint8_t* p = tile + kCodeBytes + row * (kCols / G) * 4;
    if constexpr (G == 32) {
        const uint4 q = *reinterpret_cast<const uint4*>(p);
        v[0] = q.x, v[1] = q.y, v[2] = q.z, v[3] = q.w;
    } else if constexpr (G == 64) {
        const uint2 q = *reinterpret_cast<const uint2*>(p);
        v[0] = q.x, v[1] = q.y;
    } else {
        v[0] = *reinterpret_cast<const uint32_t*>(p);
    }
}

// One lane of a converged warp (a branch on it costs less than one on a lane's number: the copies and MMAs behind it take
// their operands from the uniform datapath)
__device__ __forceinline__ bool elect_one() {
    uint32_t e;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(e));
    return e != 0;
}

__device__ __forceinline__ uint64_t policy_evict_normal() {
    uint64_t p;
    asm volatile("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(p));
    return p;
}

// Shared memory by its 32-bit addresses: a generic pointer would be two registers and two additions
__device__ __forceinline__ uint4 lds128(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
    return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
    uint32_t v;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(a));
    return v;
}
__device__ __forceinline__ bool try_wait(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}\n"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}
__device__ __forceinline__ void arrive_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(bar), "r"(bytes) : "memory");
}

// Bulk copy of `bytes` (a multiple of 16, both addresses 16-byte aligned) of this GPU's memory into this CTA's
// shared memory, completing on `bar`, with an L2 cache policy.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar, uint64_t policy) {
    asm volatile(
        "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;\n" ::"r"(
            dst),
        "l"(src), "r"(bytes), "r"(bar), "l"(policy)
        : "memory");
}

// d (+)= a b: m16n8k16, float32 sums; with FIRST, d = a b
template <bool FIRST>
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
    if constexpr (FIRST)
        asm(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
    else
        asm(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <bool FIRST>
__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    if constexpr (FIRST)
        asm(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
    else
        asm(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// ---- A operands of one 32-column run from row g's word `u` and row g + 8's word `v`

template <typename T> struct Codes;

template <>
struct Codes<__half> {
    uint32_t lo[4], hi[4];  // hi holds 16 q
    __device__ __forceinline__ Codes(uint32_t u, uint32_t v) {
        lo[0] = u & kLow;
        hi[0] = u & kHigh;
        lo[1] = v & kLow;
        hi[1] = v & kHigh;
        u = turn8(u);
        v = turn8(v);
        lo[2] = u & kLow;
        hi[2] = u & kHigh;
        lo[3] = v & kLow;
        hi[3] = v & kHigh;
    }
    static constexpr uint32_t kOne = 0x04000400u;  // 2^-14: 256 times a code's unit
};

template <>
struct Codes<float> {
    uint32_t lo[4], hi[4];
    static __device__ __forceinline__ uint32_t code(uint32_t w) {
        const uint32_t b = (w & kLow) | 0x42004200u;  // 32 + q
        const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&b), __float2bfloat162_rn(40.0f));
        return *reinterpret_cast<const uint32_t*>(&r);
    }
    __device__ __forceinline__ Codes(uint32_t u, uint32_t v) {
        lo[0] = code(u);
        hi[0] = code(u >> 4);
        lo[1] = code(v);
        hi[1] = code(v >> 4);
        lo[2] = code(u >> 8);
        hi[2] = code(turn(u, 12));
        lo[3] = code(v >> 8);
        hi[3] = code(turn(v, 12));
    }
    static constexpr uint32_t kOne = 0x3f803f80u;
};

// ---- B operands of one run: eight consecutive activations of one row, as two MMAs' (b0, b1)

template <typename T> struct Acts;

template <>
struct Acts<__half> {
    uint4 v;
    __device__ __forceinline__ void zero() { v = make_uint4(0, 0, 0, 0); }
    __device__ __forceinline__ void load(const __half* p) { v = *reinterpret_cast<const uint4*>(p); }
};
template <>
struct Acts<float> {
    uint4 v, w;
    __device__ __forceinline__ void zero() { v = w = make_uint4(0, 0, 0, 0); }
    __device__ __forceinline__ void load(const float* p) {
        v = *reinterpret_cast<const uint4*>(p);
        w = *reinterpret_cast<const uint4*>(p + 4);
    }
};

// The matrix of ones (times 2^-14 for float16) as an A operand. Made by volatile moves: a constant would be moved into the
// operand's four registers again for every MMA.
template <typename T>
struct Ones {
    uint32_t v[4];
    __device__ __forceinline__ Ones() {
#pragma unroll
        for (int i = 0; i < 4; ++i) asm volatile("mov.b32 %0, %1;" : "=r"(v[i]) : "n"(Codes<T>::kOne));
    }
};

// The sums of one group of columns of MT strips times a block of 8 activation rows: codes in lo and hi (float16: hi
// holds 16 times its sum, both 2^-22 times theirs; float32: the activations' first pieces in lo, the others in hi), the
// activations alone in on (float16: times 2^-14).
template <typename T, int MT>
struct Sums {
    // (on2: float16: half of the activations, to halve the chain of MMAs; float32: their small pieces)
    float lo[MT][4], hi[MT][4], on[4], on2[4];
};

template <bool FIRST, int MT>
__device__ __forceinline__ void run_mma(const Codes<__half> (&a)[MT], const Acts<__half>& x, Sums<__half, MT>& s,
                                        const Ones<__half>& one) {
    const uint32_t b0 = x.v.x, b1 = x.v.y, c0 = x.v.z, c1 = x.v.w;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        mma_f16<FIRST>(s.lo[m], a[m].lo[0], a[m].lo[1], a[m].lo[2], a[m].lo[3], b0, b1);
        mma_f16<FIRST>(s.hi[m], a[m].hi[0], a[m].hi[1], a[m].hi[2], a[m].hi[3], c0, c1);
    }
    mma_f16<FIRST>(s.on, one.v[0], one.v[1], one.v[2], one.v[3], b0, b1);
    mma_f16<FIRST>(s.on2, one.v[0], one.v[1], one.v[2], one.v[3], c0, c1);
}

__device__ __forceinline__ uint32_t bf16_pair(float& a, float& b) {
    // the pair (a, b) rounded to bfloat16, a and b left with what the rounding lost (exact in float32)
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;\n" : "=r"(r) : "f"(b), "f"(a));
    a -= __uint_as_float(r << 16);
    b -= __uint_as_float(r & 0xffff0000u);
    return r;
}

template <bool FIRST, int MT>
__device__ __forceinline__ void run_mma(const Codes<float> (&a)[MT], const Acts<float>& x, Sums<float, MT>& s,
                                        const Ones<float>& one) {
    float f[8] = {__uint_as_float(x.v.x), __uint_as_float(x.v.y), __uint_as_float(x.v.z), __uint_as_float(x.v.w),
                  __uint_as_float(x.w.x), __uint_as_float(x.w.y), __uint_as_float(x.w.z), __uint_as_float(x.w.w)};
    // (the tensor core cuts its sums off, always towards zero: the small pieces have sums of their own, so that the large
    // ones are cut two times a run and not six)
    auto piece = [&](auto first, float (&sum)[MT][4], float (&on)[4]) {
        constexpr bool kFirst = decltype(first)::value;
        const uint32_t b0 = bf16_pair(f[0], f[1]), b1 = bf16_pair(f[2], f[3]);
        const uint32_t c0 = bf16_pair(f[4], f[5]), c1 = bf16_pair(f[6], f[7]);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            mma_bf16<kFirst>(sum[m], a[m].lo[0], a[m].lo[1], a[m].lo[2], a[m].lo[3], b0, b1);
            mma_bf16<false>(sum[m], a[m].hi[0], a[m].hi[1], a[m].hi[2], a[m].hi[3], c0, c1);
        }
        mma_bf16<kFirst>(on, one.v[0], one.v[1], one.v[2], one.v[3], b0, b1);
        mma_bf16<false>(on, one.v[0], one.v[1], one.v[2], one.v[3], c0, c1);
    };
    piece(std::integral_constant<bool, FIRST>{}, s.lo, s.on);
    piece(std::integral_constant<bool, FIRST>{}, s.hi, s.on2);
    piece(std::false_type{}, s.hi, s.on2);
}

// The unit of the ones in that of a code (float16's 2^-14 and 2^-22). The end of a group divides its sum of activations by it, or,
// with groups of 32, multiplies its scale (64007 x 2560 at 5 tokens: groups of 32 28.7 us and 26.6; groups of 64 in a block of
// 256 experts at 5 tokens 118.8 us and 120.3)
template <typename T>
__host__ __device__ constexpr float ones() { return sizeof(T) == 2 ? 256.0f : 1.0f; }
// What a row's sum is to be multiplied by in the end
template <typename T, int G>
__host__ __device__ constexpr float unit() { return sizeof(T) != 2 ? 1.0f : G == 32 ? 16384.0f : 4194304.0f; }

// The end of a group: acc += scale (lo + hi) + bias on, rows g (values 0, 1) and g + 8 (values 2, 3).
template <typename T, int G, int MT>
__device__ __forceinline__ void group_end(float (&acc)[4], const Sums<T, MT>& s, int m, uint32_t sb0, uint32_t sb1) {
    const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&sb0));
    const float2 r = __half22float2(*reinterpret_cast<const __half2*>(&sb1));
    constexpr float kOn = G == 32 ? 1.0f : 1.0f / ones<T>(), kScale = G == 32 ? ones<T>() : 1.0f;
    const float on[2] = {(s.on[0] + s.on2[0]) * kOn, (s.on[1] + s.on2[1]) * kOn};  // (the same for both rows)
    const float b[2] = {sizeof(T) == 2 ? p.y : fmaf(8.0f, p.x, p.y), sizeof(T) == 2 ? r.y : fmaf(8.0f, r.x, r.y)};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float q = fmaf(s.hi[m][i], sizeof(T) == 2 ? 0.0625f : 1.0f, s.lo[m][i]);
        acc[i] = fmaf(q, (i < 2 ? p.x : r.x) * kScale, fmaf(on[i & 1], b[i >> 1], acc[i]));
    }
}

// This lane's activations of a tile (row g, columns 8 t .. of each run): float16 all four runs at once, ahead of the
// weights; float32 run by run as they are used (twice the registers). p: the lane's place in the row at the tile's first
// column; runs: the row's runs from there on (four but for a last tile).
template <typename T> struct TileActs;

template <>
struct TileActs<__half> {
    Acts<__half> x[4];
    __device__ __forceinline__ void load(const __half* p) {
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j].load(p + 32 * j);
    }
    __device__ __forceinline__ void load(const __half* p, int runs) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            x[j].zero();
            if (j < runs) x[j].load(p + 32 * j);
        }
    }
    __device__ __forceinline__ Acts<__half> run(int j) const { return x[j]; }
};

template <>
struct TileActs<float> {
    const float* p;
    int runs;
    __device__ __forceinline__ void load(const float* at) { p = at, runs = 4; }
    __device__ __forceinline__ void load(const float* at, int n) { p = at, runs = n; }
    __device__ __forceinline__ Acts<float> run(int j) const {
        Acts<float> x;
        if (j < runs) x.load(p + 32 * j);
        else x.zero();
        return x;
    }
};

// One tile of two strips (in shared memory at `tile`, `stride` bytes apart) times a block of 8 activation rows.
template <typename T, int G>
__device__ __forceinline__ void tile_mma(uint32_t tile, int stride, int lane, const TileActs<T>& x,
                                         float (&acc)[2][4], const Ones<T>& one) {
    constexpr int kRuns = G / 32, kPairs = kCols / G;
    uint32_t wa[2][4], wb[2][4];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        const uint4 u = lds128(tile + lane_chunk(lane) + m * stride);
        const uint4 v = lds128(tile + lane_chunk(lane) + m * stride + 512);
        wa[m][0] = u.x, wa[m][1] = u.y, wa[m][2] = u.z, wa[m][3] = u.w;
        wb[m][0] = v.x, wb[m][1] = v.y, wb[m][2] = v.z, wb[m][3] = v.w;
    }
    const uint32_t pairs = tile + kCodeBytes + (lane >> 2) * kPairs * 4;
#pragma unroll
    for (int gi = 0; gi < kPairs; ++gi) {
        Sums<T, 2> s;
#pragma unroll
        for (int r = 0; r < kRuns; ++r) {
            const int j = gi * kRuns + r;
            const Codes<T> a[2] = {Codes<T>(wa[0][j], wb[0][j]), Codes<T>(wa[1][j], wb[1][j])};
            if (r == 0) run_mma<true, 2>(a, x.run(j), s, one);
            else run_mma<false, 2>(a, x.run(j), s, one);
        }
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            const uint32_t q = pairs + m * stride + 4 * gi;
            group_end<T, G, 2>(acc[m], s, m, lds32(q), lds32(q + 8 * kPairs * 4));
        }
        // (four groups of a tile interleaved want more registers than there are: 64007 x 2560 at 5 tokens 32.2 us, with them
        // kept apart 28.0)
        if (G == 32 && gi + 1 < kPairs) __syncwarp();
    }
}

}  // namespace q4
}  // namespace smoe
