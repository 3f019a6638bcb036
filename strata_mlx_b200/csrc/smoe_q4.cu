// 4-bit weights with group scales: floats to codes and back, the layout of the kernels, and the entry points of the
// products and of a MoE block on them.
//
// The conversions are one pass over memory each, bound by HBM: every access of a thread to floats is 16 bytes next to its
// neighbours' (8 float16 weights and a 32-bit word of codes, or 4 float32 weights and half a word; float32 in two
// pieces a thread, 32 bytes apart between neighbours, ran at 4.1 TB/s), four of them in flight. A group's extremes come
// from the lanes that hold it by shuffles.
#include <algorithm>
#include <atomic>
#include <string>

#include "q4_launch.cuh"

namespace smoe {
namespace q4 {

constexpr int kConvThreads = 256;

__device__ __forceinline__ float min_nan(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// 16 bytes of floats, and the codes that go with them
template <typename T> struct Piece;
template <>
struct Piece<__half> {
    using Word = uint32_t;
    static constexpr int kN = 8;
    static __device__ __forceinline__ void load(const __half* p, float (&f)[8]) {
        const uint4 v = *reinterpret_cast<const uint4*>(p);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 q = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            f[2 * i] = q.x;
            f[2 * i + 1] = q.y;
        }
    }
    static __device__ __forceinline__ void store(__half* p, const float (&f)[8]) {
        *reinterpret_cast<uint4*>(p) = make_uint4(tc::pack_half2(f[0], f[1]), tc::pack_half2(f[2], f[3]),
                                                  tc::pack_half2(f[4], f[5]), tc::pack_half2(f[6], f[7]));
    }
};
template <>
struct Piece<float> {
    using Word = uint16_t;
    static constexpr int kN = 4;
    static __device__ __forceinline__ void load(const float* p, float (&f)[4]) {
        const float4 v = *reinterpret_cast<const float4*>(p);
        f[0] = v.x, f[1] = v.y, f[2] = v.z, f[3] = v.w;
    }
    static __device__ __forceinline__ void store(float* p, const float (&f)[4]) {
        *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
    }
};
constexpr int kConvPieces = 4;  // of a thread
constexpr float kRound = 12582912.0f;  // 1.5 * 2^23

// pieces = rows cols / kN. The arithmetic of each value is a chain of single IEEE float32 operations (difference,
// quotient, rounding to even), so the codes are the formula's exactly. A quotient is a product with the reciprocal
// of 15 scales (clamped to 0 .. 1 for free, then times 15), within 15 x 4 x 2^-23 of the division's: only one that close to
// the border of two codes is divided out (24576 x 4096 float32: 87 us, 5.4 TB/s, bound by the ALU still; 106 us with a division
// for every value; the bytes alone are 72 us).
template <typename T, int G>
__global__ void __launch_bounds__(kConvThreads) q4_quantize_kernel(const T* __restrict__ w, int64_t pieces,
                                                                   typename Piece<T>::Word* __restrict__ codes,
                                                                   __half* __restrict__ scales,
                                                                   __half* __restrict__ biases) {
    constexpr int N = Piece<T>::kN, kLanes = G / N;  // lanes of a group
    // (a warp's pieces are 32 apart: its scales and biases are one sector each)
    const int lane = threadIdx.x & 31;
    const int64_t i0 = (int64_t(blockIdx.x) * kConvThreads + (threadIdx.x & ~31)) * kConvPieces + lane;
    float f[kConvPieces][N] = {};
#pragma unroll
    for (int c = 0; c < kConvPieces; ++c)
        if (i0 + c * 32 < pieces) Piece<T>::load(w + N * (i0 + c * 32), f[c]);
    float lo[kConvPieces], hi[kConvPieces];
#pragma unroll
    for (int c = 0; c < kConvPieces; ++c) {
        lo[c] = hi[c] = f[c][0];
#pragma unroll
        for (int j = 1; j < N; ++j) {
            lo[c] = min_nan(lo[c], f[c][j]);
            hi[c] = max_nan(hi[c], f[c][j]);
        }
        // (a group's lanes are all in or all out: pieces is a multiple of kLanes)
#pragma unroll
        for (int o = 1; o < kLanes; o <<= 1) {
            lo[c] = min_nan(lo[c], __shfl_xor_sync(0xffffffffu, lo[c], o));
            hi[c] = max_nan(hi[c], __shfl_xor_sync(0xffffffffu, hi[c], o));
        }
    }
    // a lane in four works out one piece's scale, bias and reciprocal for its group (kLanes is 4 or more): the divisions
    static_assert(kConvPieces == 4, "one piece for each of four lanes");
    const int own = lane & 3;
    float l = lo[0], h = hi[0];
#pragma unroll
    for (int c = 1; c < kConvPieces; ++c) {
        if (own == c) l = lo[c], h = hi[c];
    }
    const __half2 mine = __halves2half2(__float2half_rn(__fdiv_rn(__fsub_rn(h, l), 15.0f)), __float2half_rn(l));
    const float my_inverse = __low2float(mine) > 0.0f ? __fdiv_rn(1.0f / 15.0f, __low2float(mine)) : 0.0f;
#pragma unroll
    for (int c = 0; c < kConvPieces; ++c) {
        const int64_t i = i0 + c * 32;
        const uint32_t both = __shfl_sync(0xffffffffu, *reinterpret_cast<const uint32_t*>(&mine), (lane & ~3) | c);
        const float inverse = __shfl_sync(0xffffffffu, my_inverse, (lane & ~3) | c);
        if (i >= pieces) continue;
        const __half2 sb = *reinterpret_cast<const __half2*>(&both);
        const float s = __low2float(sb), b = __high2float(sb);
        // (the code is clamped before it is rounded, which is the same; adding kRound rounds to even into the sum's low bits,
        // where rintf and a conversion would take a quarter-rate instruction each; a NaN becomes code 0, its group's scale
        // or bias is not finite either)
        uint32_t word = 0;
        float worst = 0.0f;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const float v = __saturatef(__fsub_rn(f[c][j], b) * inverse);  // a fifteenth of the code
            const float sum = fmaf(v, 15.0f, kRound);
            worst = fmaxf(worst, fabsf(fmaf(v, 15.0f, kRound - sum)));
            word += (__float_as_uint(sum) - __float_as_uint(kRound)) << (4 * j);
        }
        if (worst > 0.5f - 1e-5f) {
            word = 0;
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const float v = fminf(fmaxf(__fdiv_rn(__fsub_rn(f[c][j], b), s), 0.0f), 15.0f);
                word += (__float_as_uint(__fadd_rn(v, kRound)) - __float_as_uint(kRound)) << (4 * j);
            }
        }
        codes[i] = static_cast<typename Piece<T>::Word>(word);
    }
    const int64_t of = i0 + own * 32;
    if ((lane & (kLanes - 1)) == own && of < pieces) {
        scales[of / kLanes] = __low2half(mine);
        biases[of / kLanes] = __high2half(mine);
    }
}

// w = code * scale + bias in float32 (two roundings), then to T. PACKED: from the kernels' layout. group_log: log2 of a
// group's columns.
template <typename T, bool PACKED>
__global__ void __launch_bounds__(kConvThreads) q4_dequant_kernel(const uint8_t* __restrict__ codes,
                                                                  const __half* __restrict__ scales,
                                                                  const __half* __restrict__ biases, int64_t pieces,
                                                                  int64_t rows, int64_t cols, int group_log,
                                                                  T* __restrict__ out) {
    using Word = typename Piece<T>::Word;
    constexpr int N = Piece<T>::kN;
    const int64_t i0 = int64_t(blockIdx.x) * kConvThreads * kConvPieces + threadIdx.x;
    uint32_t word[kConvPieces];
    float s[kConvPieces], b[kConvPieces];
#pragma unroll
    for (int c = 0; c < kConvPieces; ++c) {
        const int64_t i = i0 + c * kConvThreads;
        if (i >= pieces) continue;
        if constexpr (!PACKED) {
            word[c] = reinterpret_cast<const Word*>(codes)[i];
            const int64_t at = N * i >> group_log;
            s[c] = __half2float(scales[at]);
            b[c] = __half2float(biases[at]);
        } else {
            const int group = 1 << group_log;
            const int64_t all = N * i / cols, e = all / rows, r = all - e * rows;
            const int col = static_cast<int>(N * i - all * cols);
            const uint8_t* tile = codes + ((e * strips_of_rows(rows) + r / kRows) * tiles_of_cols(cols) + col / kCols) *
                                              tile_bytes_of(group);
            const int row = static_cast<int>(r % kRows), j = (col % kCols) / 32, t = (col % 32) / 8;
            word[c] = nibbles_out(*reinterpret_cast<const uint32_t*>(tile + chunk_at(row, t) + 4 * j)) >> (col % 8 * 4);
            const __half2 p =
                *reinterpret_cast<const __half2*>(tile + kCodeBytes + (row * (kCols / group) + (col % kCols) / group) * 4);
            s[c] = __low2float(p);
            b[c] = __high2float(p);
        }
    }
#pragma unroll
    for (int c = 0; c < kConvPieces; ++c) {
        const int64_t i = i0 + c * kConvThreads;
        if (i >= pieces) continue;
        float f[N];
#pragma unroll
        for (int j = 0; j < N; ++j) f[j] = __fadd_rn(__fmul_rn(static_cast<float>((word[c] >> (4 * j)) & 15u), s[c]), b[c]);
        Piece<T>::store(out + N * i, f);
    }
}

// One 32-bit word of the layout a thread: codes, or a (scale, bias) pair.
__global__ void __launch_bounds__(kConvThreads) q4_pack_kernel(const uint32_t* __restrict__ codes,
                                                               const __half* __restrict__ scales,
                                                               const __half* __restrict__ biases, int64_t experts,
                                                               int64_t rows, int64_t cols, int group,
                                                               uint32_t* __restrict__ out, int64_t total) {
    const int64_t i = int64_t(blockIdx.x) * kConvThreads + threadIdx.x;
    if (i >= total) return;
    const int per_tile = tile_bytes_of(group) / 4, groups = kCols / group;
    const int64_t tile = i / per_tile;
    const int at = static_cast<int>(i - tile * per_tile);
    const int64_t tiles = tiles_of_cols(cols), strips = strips_of_rows(rows);
    const int64_t strip = tile / tiles, e = strip / strips;
    const int64_t c0 = (tile - strip * tiles) * kCols;
    uint32_t v = 0;
    if (at < kCodeBytes / 4) {
        const int row = at / 16, t = ((at >> 2) & 3) ^ ((row >> 1) & 3);
        const int64_t r = (strip - e * strips) * kRows + row, c = c0 + 32 * (at & 3) + 8 * t;
        if (r < rows && c < cols) v = nibbles_in(codes[(e * rows + r) * (cols / 8) + c / 8]);
    } else {
        const int k = at - kCodeBytes / 4;
        const int64_t r = (strip - e * strips) * kRows + k / groups, c = c0 + int64_t(k % groups) * group;
        if (r < rows && c < cols) {
            const int64_t from = (e * rows + r) * (cols / group) + c / group;
            v = uint32_t(__half_as_ushort(scales[from])) | (uint32_t(__half_as_ushort(biases[from])) << 16);
        }
    }
    out[i] = v;
}

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
static bool group_ok(int g) { return g == 32 || g == 64 || g == 128; }
static size_t stack_bytes(int64_t experts, int64_t rows, int64_t cols, int group) {
    return size_t(experts) * strips_of_rows(rows) * tiles_of_cols(cols) * tile_bytes_of(group);
}
constexpr int64_t kMost = int64_t(1) << 30;  // rows, columns and tokens of a matrix
constexpr int64_t kMostWeights = int64_t(1) << 40;  // of a matrix, and matrices of a stack: products stay in 64 bits
constexpr int64_t kMostExperts = int64_t(1) << 20;

static std::atomic<int> g_wait_test{0};
int wait_test() { return g_wait_test.load(); }

}  // namespace q4
}  // namespace smoe

using namespace smoe;
using namespace smoe::q4;

#define Q4_TRY try {
#define Q4_CATCH(what)                                           \
    }                                                            \
    catch (...) {                                                \
        return fail(SMOE_EARG, what ": the host is out of memory"); \
    }

static int conv_grid(int64_t n, unsigned* grid) {
    const int64_t g = (n + kConvThreads - 1) / kConvThreads;
    SMOE_REQUIRE(g <= 0x7fffffff, SMOE_ESHAPE, "too many weights for one call");
    *grid = static_cast<unsigned>(g);
    return SMOE_OK;
}

static int check_matrix(int64_t rows, int64_t cols, int group) {
    SMOE_REQUIRE(group_ok(group), SMOE_ESHAPE, "groups have 32, 64 or 128 columns, not " + std::to_string(group));
    SMOE_REQUIRE(rows > 0 && rows <= kMost && cols > 0 && cols <= kMost, SMOE_ESHAPE,
                 "a 4-bit matrix of " + std::to_string(rows) + " x " + std::to_string(cols));
    SMOE_REQUIRE(rows <= kMostWeights / cols, SMOE_ESHAPE, "a 4-bit matrix of more than 2^40 weights");
    SMOE_REQUIRE(cols % group == 0, SMOE_ESHAPE,
                 std::to_string(cols) + " columns are no whole number of groups of " + std::to_string(group));
    return SMOE_OK;
}

extern "C" size_t smoe_q4_bytes(int64_t experts, int64_t rows, int64_t cols, int group) {
    if (!group_ok(group) || experts < 0 || experts > kMostExperts || rows <= 0 || cols <= 0 || cols % group != 0) return 0;
    if (rows > kMost || cols > kMost || rows > kMostWeights / cols) return 0;
    return stack_bytes(experts, rows, cols, group);
}

extern "C" int smoe_q4_quantize(const void* w, int dtype, int64_t rows, int64_t cols, int group, uint32_t* codes,
                                uint16_t* scales, uint16_t* biases, void* stream) {
    Q4_TRY
    if (rows == 0) return SMOE_OK;
    if (int s = check_matrix(rows, cols, group)) return s;
    SMOE_REQUIRE(w && codes && scales && biases && aligned16(w), SMOE_EARG, "q4_quantize: null or misaligned pointer");
    const int64_t pieces = rows * cols / (dtype == SMOE_F16 ? 8 : 4);
    unsigned grid;
    if (int s = conv_grid((pieces + kConvPieces - 1) / kConvPieces, &grid)) return s;
    cudaStream_t st = as_stream(stream);
    __half* sp = reinterpret_cast<__half*>(scales);
    __half* bp = reinterpret_cast<__half*>(biases);
    auto go = [&](auto xt) {
        using XT = decltype(xt);
        const XT* p = static_cast<const XT*>(w);
        auto* c = reinterpret_cast<typename Piece<XT>::Word*>(codes);
        if (group == 32) q4_quantize_kernel<XT, 32><<<grid, kConvThreads, 0, st>>>(p, pieces, c, sp, bp);
        else if (group == 64) q4_quantize_kernel<XT, 64><<<grid, kConvThreads, 0, st>>>(p, pieces, c, sp, bp);
        else q4_quantize_kernel<XT, 128><<<grid, kConvThreads, 0, st>>>(p, pieces, c, sp, bp);
    };
    if (dtype == SMOE_F16) go(__half{});
    else if (dtype == SMOE_F32) go(float{});
    else return fail(SMOE_EDTYPE, "q4_quantize takes float16 or float32 weights");
    return launch_status("q4_quantize");
    Q4_CATCH("q4_quantize")
}

static int dequant(const uint32_t* codes, const uint16_t* scales, const uint16_t* biases, const uint8_t* packed,
                   int64_t experts, int64_t rows, int64_t cols, int group, void* out, int out_dtype, void* stream) {
    if (experts == 0 || rows == 0) return SMOE_OK;
    if (int s = check_matrix(rows, cols, group)) return s;
    SMOE_REQUIRE(experts > 0 && experts <= kMostExperts, SMOE_ESHAPE, "q4_dequant: a stack holds 1 to 2^20 matrices");
    SMOE_REQUIRE((packed ? aligned16(packed) : codes && scales && biases) && out && aligned16(out), SMOE_EARG,
                 "q4_dequant: null or misaligned pointer");
    SMOE_REQUIRE(out_dtype == SMOE_F16 || out_dtype == SMOE_F32, SMOE_EDTYPE, "q4_dequant gives float16 or float32");
    const int64_t pieces = experts * rows * cols / (out_dtype == SMOE_F16 ? 8 : 4);
    unsigned grid;
    if (int s = conv_grid((pieces + kConvPieces - 1) / kConvPieces, &grid)) return s;
    cudaStream_t st = as_stream(stream);
    const __half* sp = reinterpret_cast<const __half*>(scales);
    const __half* bp = reinterpret_cast<const __half*>(biases);
    const uint8_t* from = packed != nullptr ? packed : reinterpret_cast<const uint8_t*>(codes);
    const int group_log = group == 32 ? 5 : group == 64 ? 6 : 7;
    auto go = [&](auto kernel, auto* o) {
        kernel<<<grid, kConvThreads, 0, st>>>(from, sp, bp, pieces, rows, cols, group_log, o);
    };
    if (out_dtype == SMOE_F16) {
        __half* o = static_cast<__half*>(out);
        packed ? go(q4_dequant_kernel<__half, true>, o) : go(q4_dequant_kernel<__half, false>, o);
    } else {
        float* o = static_cast<float*>(out);
        packed ? go(q4_dequant_kernel<float, true>, o) : go(q4_dequant_kernel<float, false>, o);
    }
    return launch_status("q4_dequant");
}

extern "C" int smoe_q4_dequant(const uint32_t* codes, const uint16_t* scales, const uint16_t* biases, int64_t rows,
                               int64_t cols, int group, void* out, int out_dtype, void* stream) {
    Q4_TRY
    return dequant(codes, scales, biases, nullptr, 1, rows, cols, group, out, out_dtype, stream);
    Q4_CATCH("q4_dequant")
}

extern "C" int smoe_q4_unpack(const uint8_t* packed, int64_t experts, int64_t rows, int64_t cols, int group, void* out,
                              int out_dtype, void* stream) {
    Q4_TRY
    SMOE_REQUIRE(packed || experts == 0 || rows == 0, SMOE_EARG, "q4_unpack: null pointer");
    return dequant(nullptr, nullptr, nullptr, packed, experts, rows, cols, group, out, out_dtype, stream);
    Q4_CATCH("q4_unpack")
}

extern "C" int smoe_q4_pack(const uint32_t* codes, const uint16_t* scales, const uint16_t* biases, int64_t experts,
                            int64_t rows, int64_t cols, int group, uint8_t* packed, void* stream) {
    Q4_TRY
    if (experts == 0) return SMOE_OK;
    if (int s = check_matrix(rows, cols, group)) return s;
    SMOE_REQUIRE(experts > 0 && experts <= kMostExperts, SMOE_ESHAPE, "q4_pack: a stack holds 1 to 2^20 matrices");
    SMOE_REQUIRE(codes && scales && biases && packed && aligned16(packed), SMOE_EARG,
                 "q4_pack: null or misaligned pointer");
    const size_t bytes = stack_bytes(experts, rows, cols, group);
    unsigned grid;
    if (int s = conv_grid(static_cast<int64_t>(bytes / 4), &grid)) return s;
    cudaStream_t st = as_stream(stream);
    q4_pack_kernel<<<grid, kConvThreads, 0, st>>>(codes, reinterpret_cast<const __half*>(scales),
                                                 reinterpret_cast<const __half*>(biases), experts, rows, cols, group,
                                                 reinterpret_cast<uint32_t*>(packed), static_cast<int64_t>(bytes / 4));
    pdl_note(st, Writes().add(packed, bytes));  // (a product right behind it must not read ahead)
    return launch_status("q4_pack");
    Q4_CATCH("q4_pack")
}

// A product's dense part as the kernels take it. item: bytes of a result
static int dense_part(const uint8_t* dense, const uint8_t* dense2, int64_t rows, int64_t cols, int group, int64_t tokens,
                      void* out, size_t item, ProductArgs& a, Writes& w, cudaStream_t st) {
    if (int s = check_matrix(rows, cols, group)) return s;
    SMOE_REQUIRE(dense && out && aligned16(dense) && aligned16(dense2), SMOE_EARG, "q4_product: null or misaligned pointer");
    SMOE_REQUIRE(tokens <= kMost && strips_of_rows(rows) * ((tokens + 7) / 8) <= kMost, SMOE_ESHAPE,
                 "too many tokens for one q4_product call");
    a.dw[0] = dense;
    a.dw[1] = dense2;
    a.d_out = out;
    a.d_rows = rows;
    a.d_tokens = tokens;
    w.add(out, size_t(tokens) * rows * item);
    const size_t bytes = stack_bytes(1, rows, cols, group);
    a.early = a.early && pdl_early(st, dense, bytes) && (!dense2 || pdl_early(st, dense2, bytes));
    return SMOE_OK;
}

// pieces: results as two rows of float16 each (q4_mv.cuh); gate32: the dense gate in float32; `zero`: words that the launch
// clears besides, for the launch after it
static int q4_product(const SmoeQ4Product* p, bool pieces, const float* gate32, uint32_t* zero, int n_zero, void* stream) {
    SMOE_REQUIRE(p, SMOE_EARG, "q4_product: null pointer");
    SMOE_REQUIRE(p->dtype == SMOE_F16 || p->dtype == SMOE_F32, SMOE_EDTYPE,
                 "q4_product takes float16 or float32 activations");
    SMOE_REQUIRE(p->dense_tokens >= 0 && p->pairs >= 0, SMOE_EARG, "q4_product: a negative count");
    if (p->dense_tokens == 0 && p->pairs == 0) return SMOE_OK;
    const size_t item = p->dtype == SMOE_F16 ? 2 : 4;
    ProductArgs a = {};
    Writes w;
    cudaStream_t st = as_stream(stream);
    a.early = true;
    a.hint = p->pairs > 0;
    SMOE_REQUIRE(p->x && aligned16(p->x), SMOE_EARG, "q4_product: activations must be 16-byte aligned");
    a.x = p->x;
    a.cols = p->cols;
    a.share = 1;
    const bool glu = (p->dense_tokens > 0 ? p->dense2 : p->stack2) != nullptr;
    if (p->dense_tokens > 0) {
        SMOE_REQUIRE(p->dense_gate == nullptr || glu, SMOE_EARG, "q4_product: a gate needs gate and up matrices");
        if (int s = dense_part(p->dense, p->dense2, p->dense_rows, p->cols, p->group, p->dense_tokens, p->dense_out,
                               item * (pieces ? 2 : 1), a, w, st))
            return s;
        a.d_gate = p->dense_gate;
        a.d_gate32 = gate32;
    }
    if (p->pairs > 0) {
        if (int s = check_matrix(p->rows, p->cols, p->group)) return s;
        SMOE_REQUIRE(p->stack && p->out && p->idx && aligned16(p->stack) && aligned16(p->stack2), SMOE_EARG,
                     "q4_product: null or misaligned pointer");
        SMOE_REQUIRE(p->share > 0 && p->pairs % p->share == 0, SMOE_EARG, "pairs must be a multiple of share");
        SMOE_REQUIRE(p->experts > 0 && p->experts <= 2048, SMOE_ESHAPE, "q4_product takes 1 to 2048 experts");
        SMOE_REQUIRE(p->pairs <= kMaxPairs, SMOE_ESHAPE,
                     "q4_product takes up to " + std::to_string(kMaxPairs) + " pairs a call");
        SMOE_REQUIRE(strips_of_rows(p->rows) * p->pairs <= kMost, SMOE_ESHAPE, "too many rows for one q4_product call");
        SMOE_REQUIRE(p->dense_tokens == 0 || (p->stack2 != nullptr) == glu, SMOE_EARG,
                     "q4_product: the dense and the stack part are both products or both gated");
        SMOE_REQUIRE(p->weights == nullptr || glu, SMOE_EARG, "q4_product: weights need gate and up stacks");
        a.rw[0] = p->stack;
        a.rw[1] = p->stack2;
        a.r_out = p->out;
        a.r_rows = p->rows;
        a.experts = p->experts;
        a.pairs = p->pairs;
        a.share = p->share;
        a.idx = p->idx;
        a.weights = p->weights;
        w.add(p->out, size_t(p->pairs) * p->rows * item * (pieces ? 2 : 1));
        const size_t bytes = stack_bytes(p->experts, p->rows, p->cols, p->group);
        a.early = a.early && pdl_early(st, p->stack, bytes) && (!p->stack2 || pdl_early(st, p->stack2, bytes));
    }
    if (p->dtype == SMOE_F16 && p->pairs == 0 && !glu && matmul_better(p->dense_tokens, p->dense_rows, p->cols))
        return matmul_f16(a, p->group, false, w, st);
    a.pieces = pieces;
    a.zero = zero;
    a.n_zero = n_zero;
    w.add(zero, size_t(n_zero) * 4);
    return p->dtype == SMOE_F16 ? product_f16(a, p->group, w, st) : product_f32(a, p->group, w, st);
}

extern "C" int smoe_q4_product(const SmoeQ4Product* p, void* stream) {
    Q4_TRY
    return q4_product(p, false, nullptr, nullptr, 0, stream);
    Q4_CATCH("q4_product")
}

extern "C" int smoe_q4_linear(const uint8_t* packed, int64_t rows, int64_t cols, int group, const void* x,
                              int64_t tokens, void* out, int dtype, void* stream) {
    Q4_TRY
    SmoeQ4Product p = {};
    p.dtype = dtype;
    p.group = group;
    p.x = x;
    p.cols = cols;
    p.dense = packed;
    p.dense_rows = rows;
    p.dense_tokens = tokens;
    p.dense_out = out;
    return q4_product(&p, false, nullptr, nullptr, 0, stream);
    Q4_CATCH("q4_linear")
}

extern "C" int smoe_q4_is_prompt(int64_t tokens, int64_t rows, int64_t cols) {
    return rows > 0 && cols > 0 && rows <= kMost && cols <= kMost && tokens <= kMost && matmul_better(tokens, rows, cols);
}

extern "C" int smoe_q4_prompt(const uint8_t* packed, int64_t rows, int64_t cols, int group, const void* x, int64_t tokens,
                              void* out, int out_dtype, void* stream) {
    Q4_TRY
    SMOE_REQUIRE(out_dtype == SMOE_F16 || out_dtype == SMOE_F32, SMOE_EDTYPE, "q4_prompt gives float16 or float32");
    SMOE_REQUIRE(tokens >= 0, SMOE_EARG, "q4_prompt: a negative count");
    if (tokens == 0) return SMOE_OK;
    SMOE_REQUIRE(x && aligned16(x), SMOE_EARG, "q4_prompt: activations must be 16-byte aligned");
    ProductArgs a = {};
    Writes w;
    cudaStream_t st = as_stream(stream);
    a.early = true;
    a.x = x;
    a.cols = cols;
    if (int s = dense_part(packed, nullptr, rows, cols, group, tokens, out, out_dtype == SMOE_F16 ? 2 : 4, a, w, st)) return s;
    return matmul_f16(a, group, out_dtype == SMOE_F32, w, st);
    Q4_CATCH("q4_prompt")
}

extern "C" size_t smoe_q4_tile_plan_size(int64_t tiles) { return tiles > 0 ? size_t(tiles + 1) * 16 : 0; }

static int check_tiles(int64_t tiles, int64_t experts) {
    SMOE_REQUIRE(tiles > 0 && tiles <= (int64_t(1) << 24), SMOE_ESHAPE, "1 to 2^24 tiles a call");
    SMOE_REQUIRE(experts > 0 && experts <= kMostExperts, SMOE_ESHAPE, "a stack holds 1 to 2^20 matrices");
    return SMOE_OK;
}

extern "C" int smoe_q4_tile_plan(const uint32_t* tile_expert, int64_t tiles, int64_t experts, void* plan, size_t plan_bytes,
                                 void* stream) {
    Q4_TRY
    if (tiles == 0) return SMOE_OK;
    if (int s = check_tiles(tiles, experts)) return s;
    SMOE_REQUIRE(tile_expert, SMOE_EARG, "q4_tile_plan: null pointer");
    SMOE_REQUIRE(plan && aligned16(plan) && plan_bytes >= smoe_q4_tile_plan_size(tiles), SMOE_EWORKSPACE,
                 "q4_tile_plan: plan missing, misaligned or too small");
    Writes w;
    w.add(plan, smoe_q4_tile_plan_size(tiles));
    return tile_plan(tile_expert, tiles, experts, plan, w, as_stream(stream));
    Q4_CATCH("q4_tile_plan")
}

extern "C" int smoe_q4_tile_matmul(const uint8_t* packed, int64_t experts, int64_t rows, int64_t cols, int group, const void* a,
                                   int64_t tiles, const void* plan, const uint32_t* slot_row, int64_t out_rows, void* out,
                                   int out_dtype, void* stream) {
    Q4_TRY
    if (tiles == 0 || out_rows == 0) return SMOE_OK;
    if (int s = check_tiles(tiles, experts)) return s;
    if (int s = check_matrix(rows, cols, group)) return s;
    SMOE_REQUIRE(out_rows > 0, SMOE_EARG, "q4_tile_matmul: a negative count");
    SMOE_REQUIRE(experts * strips_of_rows(rows) <= kMost && tiles * strips_of_rows(rows) <= kMost, SMOE_ESHAPE,
                 "too many rows for one q4_tile_matmul call");
    SMOE_REQUIRE(packed && a && plan && out && aligned16(packed) && aligned16(a) && aligned16(plan), SMOE_EARG,
                 "q4_tile_matmul: null or misaligned pointer");
    SMOE_REQUIRE(out_dtype == SMOE_F16 || out_dtype == SMOE_F32, SMOE_EDTYPE, "q4_tile_matmul gives float16 or float32");
    Writes w;
    w.add(out, size_t(out_rows) * rows * (out_dtype == SMOE_F16 ? 2 : 4));
    const TileArgs p = {packed, experts, rows, cols, tiles, a, plan, slot_row, out_rows, out, out_dtype == SMOE_F32};
    return tile_matmul(p, group, w, as_stream(stream));
    Q4_CATCH("q4_tile_matmul")
}

// A call's workspace: the SwiGLU of the pairs and of the shared expert, the partial sums and the counters of the down
// products' jobs.
struct MoeSpace {
    size_t h, hs, partial, counters, bytes;
    MoeSpace(int64_t tokens, int64_t k, int64_t hidden, int64_t ffn, int64_t shared_ffn) {
        size_t at = 0;
        auto take = [&](size_t n) {
            const size_t from = at;
            at += (n + 255) & ~size_t(255);
            return from;
        };
        // (four bytes a value: a float32, or its two float16 pieces)
        h = take(size_t(tokens) * k * ffn * 4);
        hs = take(size_t(tokens) * shared_ffn * 4);
        partial = take(size_t(kDownCtas) * 2 * tokens * kMt * kRows * 4);
        counters = take(n_counters(hidden) * 4);
        bytes = at;
    }
    static size_t n_counters(int64_t hidden) { return static_cast<size_t>((strips_of_rows(hidden) + kMt - 1) / kMt); }
};

extern "C" size_t smoe_q4_moe_workspace_size(int64_t tokens, int64_t k, int64_t hidden, int64_t ffn,
                                             int64_t shared_ffn) {
    if (tokens <= 0 || k <= 0 || hidden <= 0 || ffn <= 0 || shared_ffn < 0) return 0;
    return MoeSpace(tokens, k, hidden, ffn, shared_ffn).bytes;
}

extern "C" int smoe_q4_moe(const SmoeQ4Moe* m, void* workspace, size_t workspace_bytes, void* stream) {
    Q4_TRY
    SMOE_REQUIRE(m, SMOE_EARG, "q4_moe: null pointer");
    SMOE_REQUIRE(m->dtype == SMOE_F16 || m->dtype == SMOE_F32, SMOE_EDTYPE, "q4_moe takes float16 or float32 activations");
    SMOE_REQUIRE(m->tokens >= 0, SMOE_EARG, "q4_moe: a negative count");
    if (m->tokens == 0) return SMOE_OK;
    SMOE_REQUIRE(m->tokens <= 64, SMOE_ESHAPE, "q4_moe takes up to 64 tokens a call");
    SMOE_REQUIRE(m->experts > 0 && m->experts <= 2048, SMOE_ESHAPE, "q4_moe takes 1 to 2048 experts");
    SMOE_REQUIRE(m->k >= 1 && m->k <= 32, SMOE_ESHAPE, "q4_moe takes 1 to 32 experts a token");
    if (int s = check_matrix(m->ffn, m->hidden, m->group)) return s;
    if (int s = check_matrix(m->hidden, m->ffn, m->down_group)) return s;
    SMOE_REQUIRE(m->shared_ffn >= 0, SMOE_ESHAPE, "q4_moe: a negative width");
    if (m->shared_ffn > 0) {
        if (int s = check_matrix(m->shared_ffn, m->hidden, m->group)) return s;
        if (int s = check_matrix(m->hidden, m->shared_ffn, m->down_group)) return s;
        SMOE_REQUIRE(m->sgate && m->sup && m->sdown, SMOE_EARG, "q4_moe: a shared expert needs its three matrices");
    }
    // (tiles of all the down products of a call, counted in 32 bits)
    SMOE_REQUIRE(int64_t(MoeSpace::n_counters(m->hidden)) *
                         (m->tokens * tiles_of_cols(m->shared_ffn) + m->tokens * m->k * tiles_of_cols(m->ffn)) < kMost,
                 SMOE_ESHAPE, "q4_moe: the layer is too large for " + std::to_string(m->tokens) + " tokens a call");
    SMOE_REQUIRE(m->x && m->idx && m->weights && m->gate && m->up && m->down && m->out && aligned16(m->down) &&
                     aligned16(m->sdown),
                 SMOE_EARG, "q4_moe: null or misaligned pointer");
    SMOE_REQUIRE(workspace && aligned16(workspace) &&
                     workspace_bytes >= smoe_q4_moe_workspace_size(m->tokens, m->k, m->hidden, m->ffn, m->shared_ffn),
                 SMOE_EWORKSPACE, "q4_moe: workspace missing, misaligned or too small");
    cudaStream_t st = as_stream(stream);
    const MoeSpace space(m->tokens, m->k, m->hidden, m->ffn, m->shared_ffn);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    void* h = ws + space.h;
    void* hs = ws + space.hs;
    uint32_t* counters = reinterpret_cast<uint32_t*>(ws + space.counters);
    SmoeQ4Product p = {};
    p.dtype = m->dtype;
    p.group = m->group;
    p.x = m->x;
    p.cols = m->hidden;
    if (m->shared_ffn > 0) {
        p.dense = m->sgate;
        p.dense2 = m->sup;
        p.dense_rows = m->shared_ffn;
        p.dense_tokens = m->tokens;
        p.dense_gate = m->shared_gate;
        p.dense_out = hs;
    }
    p.stack = m->gate;
    p.stack2 = m->up;
    p.rows = m->ffn;
    p.experts = m->experts;
    p.idx = m->idx;
    p.pairs = m->tokens * m->k;
    p.share = m->k;
    p.weights = m->weights;
    p.out = h;
    if (int s = q4_product(&p, p.dtype == SMOE_F16, m->shared_gate32, counters,
                           static_cast<int>(MoeSpace::n_counters(m->hidden)), stream))
        return s;
    DownArgs d = {};
    d.h = h;
    d.hs = m->shared_ffn > 0 ? hs : nullptr;
    d.w = m->down;
    d.sw = m->sdown;
    d.ffn = m->ffn;
    d.sffn = m->shared_ffn;
    d.rows = m->hidden;
    d.experts = m->experts;
    d.tokens = m->tokens;
    d.k = m->k;
    d.idx = m->idx;
    d.out = m->out;
    d.partial = reinterpret_cast<float*>(ws + space.partial);
    d.counters = counters;
    // (the launch before is the product above, which writes h, hs and the counters alone and has waited for everything before it)
    d.early = true;
    Writes w;
    w.add(d.partial, space.counters - space.partial).add(counters, space.bytes - space.counters);
    w.add(m->out, size_t(m->tokens) * m->hidden * (m->dtype == SMOE_F16 ? 2 : 4));
    return m->dtype == SMOE_F16 ? down_f16(d, m->down_group, w, st) : down_f32(d, m->down_group, w, st);
    Q4_CATCH("q4_moe")
}

extern "C" int smoe_q4_wait_test(int withhold) {
    g_wait_test = withhold != 0;
    return SMOE_OK;
}

extern "C" int smoe_q4_status(int* status, int clear) {
    Q4_TRY
    SMOE_REQUIRE(status, SMOE_EARG, "q4_status: null pointer");
    *status = 0;
    cudaError_t e = cudaDeviceSynchronize();
    for (auto read : {matmul_status, product_status_f16, product_status_f32, down_status_f16, down_status_f32}) {
        int v = 0;
        if (e == cudaSuccess) e = read(&v, clear != 0);
        if (v != 0) *status = v;
    }
    if (e != cudaSuccess) return fail(-static_cast<int>(e), std::string("q4_status: ") + cudaGetErrorString(e));
    return SMOE_OK;
    Q4_CATCH("q4_status")
}
