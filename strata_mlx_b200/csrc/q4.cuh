// 4-bit weights with a float16 scale and bias for each group of 32, 64 or 128 columns: the layout the kernels
// read, and one tile of it times up to 8 NT activation rows on the tensor cores.
//
//   w[r, c] = code[r, c] * scale[r, c / G] + bias[r, c / G],   code in 0 .. 15
//
// Layout (made once from the file's arrays by smoe_q4_pack). A matrix is strips of 16 rows, a strip is tiles of 128
// columns one after the other, a tile is 1024 bytes of codes (64 a row) and then 128 / G (scale, bias) pairs a row:
//
//   [strip][tile][ 16 rows x 64 B codes ][ 16 rows x 128 / G x (scale, bias) ]
//
// so a strip is one run of memory that bulk copies fetch in any pieces, every piece a multiple of 16 bytes. Rows
// past the last and columns past the last are zero codes with zero scales and biases. Within a row's 16 code
// words, word 4 t + j holds the eight codes of columns 32 j + 8 t .. + 7 of the tile: lane (g, t) of a warp (g =
// lane / 4, t = lane % 4) reads 16 bytes at 64 g + 16 t and has its columns of all four 32-column runs.
//
// Arithmetic. A run of 32 columns is two m16n8k16 MMAs, rows the M side, activation rows the N side. The order of
// columns inside an MMA is free as long as A and B agree, so lane (g, t)'s word goes in as it lies: nibbles 0, 4
// and 2, 6 to one MMA, 1, 5 and 3, 7 to the other. With float16 activations a nibble needs no conversion at all:
// (word & 0x000f000f) is a pair of float16 subnormals q * 2^-24, exact in the tensor core, and (word & 0x00f000f0)
// a pair of 16 q * 2^-24; the two MMAs keep sums of their own, joined as lo + hi / 16 and scaled by 2^24 scale at
// the end of the group. Products are exact and sums are float32: the result is the formula's but for float32
// rounding. The bias takes sum x over the group, from the same B operands times a matrix of ones.
// Float32 activations are three bfloat16 pieces (8 + 8 + 8 bits: the whole float32), each through the same MMAs;
// codes become bfloat16 by (q | 0x4300) - 128, exact too.
#pragma once

#include <cuda_bf16.h>

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

// Bulk copy of `bytes` (a multiple of 16, both addresses 16-byte aligned) of this GPU's memory into this CTA's
// shared memory, completing on `bar`.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n" ::"r"(dst),
                 "l"(src), "r"(bytes), "r"(smem_addr(bar))
                 : "memory");
}
__device__ __forceinline__ void bulk_load_hint(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar,
                                               uint64_t policy) {
    asm volatile(
        "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;\n" ::"r"(
            dst),
        "l"(src), "r"(bytes), "r"(smem_addr(bar)), "l"(policy)
        : "memory");
}

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    asm volatile(
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
        lo[0] = u & 0x000f000fu;
        hi[0] = u & 0x00f000f0u;
        lo[1] = v & 0x000f000fu;
        hi[1] = v & 0x00f000f0u;
        u >>= 8;
        v >>= 8;
        lo[2] = u & 0x000f000fu;
        hi[2] = u & 0x00f000f0u;
        lo[3] = v & 0x000f000fu;
        hi[3] = v & 0x00f000f0u;
    }
    static constexpr uint32_t kOne = 0x3c003c00u;
};

template <>
struct Codes<float> {
    uint32_t lo[4], hi[4];
    static __device__ __forceinline__ uint32_t code(uint32_t w) {
        const uint32_t b = (w & 0x000f000fu) | 0x43004300u;  // 128 + q
        const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&b), __float2bfloat162_rn(128.0f));
        return *reinterpret_cast<const uint32_t*>(&r);
    }
    __device__ __forceinline__ Codes(uint32_t u, uint32_t v) {
        lo[0] = code(u);
        hi[0] = code(u >> 4);
        lo[1] = code(v);
        hi[1] = code(v >> 4);
        lo[2] = code(u >> 8);
        hi[2] = code(u >> 12);
        lo[3] = code(v >> 8);
        hi[3] = code(v >> 12);
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

// One run of up to MATS matrices times one block of 8 activation rows: sums of the group so far in lo / hi (float16:
// hi holds 16 times its sum) and, of the activations alone, in on.
template <int MATS>
__device__ __forceinline__ void run_mma(const Codes<__half> (&a)[MATS], const Acts<__half>& x, float (&lo)[MATS][4],
                                        float (&hi)[MATS][4], float (&on)[4]) {
    const uint32_t b0 = __byte_perm(x.v.x, x.v.z, 0x5410), b1 = __byte_perm(x.v.y, x.v.w, 0x5410);
    const uint32_t c0 = __byte_perm(x.v.x, x.v.z, 0x7632), c1 = __byte_perm(x.v.y, x.v.w, 0x7632);
    constexpr uint32_t one = Codes<__half>::kOne;
#pragma unroll
    for (int m = 0; m < MATS; ++m) {
        mma_f16(lo[m], a[m].lo[0], a[m].lo[1], a[m].lo[2], a[m].lo[3], b0, b1);
        mma_f16(hi[m], a[m].hi[0], a[m].hi[1], a[m].hi[2], a[m].hi[3], c0, c1);
    }
    mma_f16(on, one, one, one, one, b0, b1);
    mma_f16(on, one, one, one, one, c0, c1);
}

__device__ __forceinline__ uint32_t bf16_pair(float& a, float& b) {
    // the pair (a, b) rounded to bfloat16, a and b left with what the rounding lost (exact in float32)
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;\n" : "=r"(r) : "f"(b), "f"(a));
    a -= __uint_as_float(r << 16);
    b -= __uint_as_float(r & 0xffff0000u);
    return r;
}

template <int MATS>
__device__ __forceinline__ void run_mma(const Codes<float> (&a)[MATS], const Acts<float>& x, float (&lo)[MATS][4],
                                        float (&hi)[MATS][4], float (&on)[4]) {
    float f[8] = {__uint_as_float(x.v.x), __uint_as_float(x.v.y), __uint_as_float(x.v.z), __uint_as_float(x.v.w),
                  __uint_as_float(x.w.x), __uint_as_float(x.w.y), __uint_as_float(x.w.z), __uint_as_float(x.w.w)};
    constexpr uint32_t one = Codes<float>::kOne;
#pragma unroll
    for (int piece = 0; piece < 3; ++piece) {
        const uint32_t b0 = bf16_pair(f[0], f[4]), b1 = bf16_pair(f[2], f[6]);
        const uint32_t c0 = bf16_pair(f[1], f[5]), c1 = bf16_pair(f[3], f[7]);
#pragma unroll
        for (int m = 0; m < MATS; ++m) {
            mma_bf16(lo[m], a[m].lo[0], a[m].lo[1], a[m].lo[2], a[m].lo[3], b0, b1);
            mma_bf16(hi[m], a[m].hi[0], a[m].hi[1], a[m].hi[2], a[m].hi[3], c0, c1);
        }
        mma_bf16(on, one, one, one, one, b0, b1);
        mma_bf16(on, one, one, one, one, c0, c1);
    }
}

// The end of a group: acc += scale (lo + hi) + bias on, rows g (values 0, 1) and g + 8 (values 2, 3).
template <typename T>
__device__ __forceinline__ void group_end(float (&acc)[4], const float (&lo)[4], const float (&hi)[4],
                                          const float (&on)[4], uint32_t sb0, uint32_t sb1) {
    const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&sb0));
    const float2 r = __half22float2(*reinterpret_cast<const __half2*>(&sb1));
    constexpr bool kHalf = sizeof(T) == 2;
    const float s0 = kHalf ? p.x * 16777216.0f : p.x, s1 = kHalf ? r.x * 16777216.0f : r.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float q = kHalf ? fmaf(hi[i], 0.0625f, lo[i]) : lo[i] + hi[i];
        acc[i] = fmaf(q, i < 2 ? s0 : s1, fmaf(on[i], i < 2 ? p.y : r.y, acc[i]));
    }
}

// The (scale, bias) pairs of row `row` of a tile in shared memory
template <int G>
struct Pairs {
    uint32_t v[kCols / G];
    __device__ __forceinline__ explicit Pairs(const uint8_t* tile, int row) {
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
};

// A tile of MATS matrices (shared memory, `mat_stride` bytes apart) times NT blocks of 8 activation rows.
// load(nt, j, x): this lane's eight activations of run j and row 8 nt + g. on(nt): whether the block has rows at all
// (the same for the whole warp).
template <typename T, int G, int NT, int MATS, class Load, class On>
__device__ __forceinline__ void tile_mma(const uint8_t* tile, int mat_stride, int lane, float (&acc)[MATS][NT][4],
                                         Load load, On on_block) {
    const int g = lane >> 2;
    uint32_t wa[MATS][4], wb[MATS][4];
    uint32_t pa[MATS][kCols / G], pb[MATS][kCols / G];
#pragma unroll
    for (int m = 0; m < MATS; ++m) {
        const uint8_t* p = tile + m * mat_stride;
        const uint4 u = *reinterpret_cast<const uint4*>(p + 16 * lane);
        const uint4 v = *reinterpret_cast<const uint4*>(p + 512 + 16 * lane);
        wa[m][0] = u.x, wa[m][1] = u.y, wa[m][2] = u.z, wa[m][3] = u.w;
        wb[m][0] = v.x, wb[m][1] = v.y, wb[m][2] = v.z, wb[m][3] = v.w;
        const Pairs<G> q0(p, g), q1(p, g + 8);
#pragma unroll
        for (int i = 0; i < kCols / G; ++i) pa[m][i] = q0.v[i], pb[m][i] = q1.v[i];
    }
    constexpr int kRuns = G / 32;
#pragma unroll
    for (int gi = 0; gi < kCols / G; ++gi) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            if (NT > 2 && !on_block(nt)) continue;
            float lo[MATS][4] = {}, hi[MATS][4] = {}, on[4] = {};
#pragma unroll
            for (int r = 0; r < kRuns; ++r) {
                const int j = gi * kRuns + r;
                Acts<T> x;
                load(nt, j, x);
                // (with several blocks the codes are expanded again for each: five instructions a word, held registers
                // would cost more)
                if constexpr (MATS == 1) {
                    const Codes<T> a[1] = {Codes<T>(wa[0][j], wb[0][j])};
                    run_mma<1>(a, x, lo, hi, on);
                } else {
                    const Codes<T> a[2] = {Codes<T>(wa[0][j], wb[0][j]), Codes<T>(wa[MATS - 1][j], wb[MATS - 1][j])};
                    run_mma<2>(a, x, lo, hi, on);
                }
            }
#pragma unroll
            for (int m = 0; m < MATS; ++m) group_end<T>(acc[m][nt], lo[m], hi[m], on, pa[m][gi], pb[m][gi]);
        }
    }
}

}  // namespace q4
}  // namespace smoe
