// A prompt's product on 4-bit weights with group scales, on the 5th-generation tensor cores (layout: q4.cuh).
//
// out[t, r] = sum_c w[r, c] x[t, c], the weights w = code scale + bias rounded once to float16 (the activations' type)
// and float32 sums. 128 weight rows are the M side of a tcgen05 MMA (8 strips), up to 256 tokens the N side, so a row is
// decoded once for that many tokens. What bounds it: the tensor pipe (2 rows cols tokens flops at 4,096 multiply-adds a
// cycle of an SM) and beside it the decoding, 15 instructions for 8 weights: a stage of 128 x 128 weights takes 240
// issue slots a scheduler (0.13 us), but 0.35 us, because a group of decoders waits, loads, waits, decodes, stores and hands over
// strictly in turn and there are two groups; its MMAs take 2.8 ns a token, so from about 130 tokens a job the tensor pipe is the
// longer. 4096 x 4096 at 1180 tokens: 34.0 us, 1164 TFLOP/s.
//
// Per CTA (persistent over jobs = (block of tokens, 128 rows)), warp-specialized, every hand-off an mbarrier:
//   warp 17   weights: a stage is one tile of each of the 8 strips, one TMA box (a copy a strip took the warp 120 cycles
//             each to issue, more than the stage's work) into a ring of up to 10 slots
//   warp 18   activations: the tokens' 128 columns by TMA into a ring of its own, two boxes of all the job's rows x 64
//             columns (128-byte swizzle)
//   warps 0-15 decoders, two groups on every other stage: a thread reads half of its row's 128 columns, a mask and one
//             multiply-add make a pair of codes float16 exactly, another with the group's scale and bias rounds it to the
//             weight; stored to its TMEM lane of an A slot
//   warp 16   MMA: A from TMEM, B from shared memory, 8 MMAs of K = 16 a stage; commits free the slots.
//   warps 19-22 read a job's sums back and write them out while the next job runs (jobs of up to 160 tokens have two
//             accumulators); a CTA's last job is the decoders'
// Every wait is bounded; one that gives up leaves SMOE_ETIMEOUT in the status and ends the CTA's work.
#include <cuda.h>

#include <algorithm>
#include <mutex>

#include "q4_launch.cuh"

namespace smoe {
namespace q4 {

constexpr int kGDecoders = 16;   // two groups of 8 warps, every other stage each
constexpr int kGGroup = 8;
constexpr int kGEnders = 4;      // warps that write a job out while the next one runs
constexpr int kGThreads = 32 * (kGDecoders + 3 + kGEnders);
constexpr int kGM = 128;
constexpr int kGStrips = kGM / kRows;
constexpr int kGMaxN = 256;
constexpr int kGASlots = 3;
constexpr uint32_t kGAColumn = 320;  // of TMEM: A slots from here, 64 columns each; accumulators before
constexpr int kGMaxRaw = 10;
constexpr int kGMaxB = 6;
constexpr int kGSmemLimit = 227 * 1024;

static __device__ int g_q4_gemm_status = 0;

struct GemmArgs {
    const uint8_t* w;
    __half* out;
    int64_t rows, cols, tokens;
    int n;        // tokens of a job, a multiple of 16
    int nblocks;  // jobs' blocks of tokens
    int mblocks;
    int nb, nr;   // activation and raw slots
    bool early;
    int withhold;  // a test's: 1, CTA 0's first copy of weights never counts as landed
    // TILES: a stack, its activations in tiles of 16 slots of one expert's
    const uint4* plan;  // word 0: .x blocks of slots; then each block's first slot, slots, expert
    const uint32_t* slot_row;
    int64_t out_rows;
    int strips;  // of an expert
    bool floats;  // out is float32
};

// A job's activation rows: the first and how many, and the first strip of its matrix
struct GemmBlock {
    int row0, n, strip0;
};

// Slots of a job of TILES: a stage's decoding takes as long as the MMAs of 130 tokens, and two accumulators fit (the SwiGLU
// of 256 experts of 1536 x 4096, 128 tokens each: 1709 us, in jobs of 128 slots 2029; 37 tokens each: 1079 and 1055).
constexpr int kTileSlots = 160;
constexpr int kSlots = 16;  // of a tile

template <bool TILES>
struct alignas(64) GemmMaps {
    CUtensorMap w;  // strips of the matrix as rows of 8-byte words, in boxes of a tile of 8 strips
    CUtensorMap a[TILES ? kTileSlots / kSlots : 1];  // boxes of a job's rows x 64 columns; TILES: of 16, 32, .. rows
};

struct GemmSmem {
    uint64_t rawfull[kGMaxRaw], rawfree[kGMaxRaw], bfull[kGMaxB], bfree[kGMaxB];
    uint64_t afull[kGASlots], afree[kGASlots], dfull[2], dfree[2];
    uint64_t done;  // the CTA's last job's sums: used once
    uint32_t tmem_base;
};

template <int G>
__host__ __device__ constexpr int raw_slot_bytes() { return kGStrips * tile_bytes<G>(); }
__host__ __device__ constexpr int b_slot_bytes(int n) { return 2 * n * 128; }  // two atoms of 64 columns
// [activation slots, 1024-aligned][raw slots][barriers]
template <int G>
__host__ __device__ constexpr size_t gemm_smem(int n, int nb, int nr) {
    return size_t(nb) * b_slot_bytes(n) + size_t(nr) * raw_slot_bytes<G>() + sizeof(GemmSmem);
}

struct Phase {
    int slot = 0;
    uint32_t phase = 0;
    __device__ __forceinline__ void next(int n) {
        if (++slot == n) {
            slot = 0;
            phase ^= 1;
        }
    }
};

// Eight codes of the layout's word as weights: w[i] = columns 2 i, 2 i + 1
__device__ __forceinline__ void decode8(uint32_t word, __half2 s, __half2 b, uint32_t* out) {
    auto pair = [](uint16_t bits) { return __half2half2(__ushort_as_half(bits)); };
    const __half2 unit[2] = {pair(0x3400), pair(0x2400)}, off[2] = {pair(0xdc00), pair(0xcc00)};  // 1/4 and -256, 1/64 and -16
    const uint32_t turned = turn8(word);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        // (with 1024's exponent a code as it lies is 1024 + 4 q or 1024 + 64 q; a quarter less 256, a 64th less 16 is q: exact)
        const uint32_t v = ((i >= 2 ? turned : word) & (i & 1 ? kHigh : kLow)) | 0x64006400u;
        const __half2 h = *reinterpret_cast<const __half2*>(&v), q = __hfma2(h, unit[i & 1], off[i & 1]);
        const __half2 w = __hfma2(q, s, b);
        out[(i >> 1) + 2 * (i & 1)] = *reinterpret_cast<const uint32_t*>(&w);  // nibbles i and i + 4 of the word
    }
}

// TILES: the activations are tiles of 16 slots, each one expert's; a job is up to g.n slots of one expert (`plan`), its
// MMAs as wide as it has slots, and slot s's row goes to row slot_row[s] of out.
template <int G, bool TILES>
__global__ void __launch_bounds__(kGThreads, 1) q4_matmul_kernel(const GemmArgs g, const __grid_constant__ GemmMaps<TILES> maps) {
    constexpr int kTile = tile_bytes<G>();
    constexpr int kRaw = raw_slot_bytes<G>();
    extern __shared__ __align__(1024) uint8_t gsmem[];
    uint8_t* smem = gsmem;
    const int bslot = b_slot_bytes(g.n);
    uint8_t* raw = smem + size_t(g.nb) * bslot;
    GemmSmem& S = *reinterpret_cast<GemmSmem*>(raw + g.nr * kRaw);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if constexpr (TILES) pdl_wait();  // (the plan is a launch's before)
    const int jobs = (TILES ? static_cast<int>(__ldcg(g.plan).x) : g.nblocks) * g.mblocks;
    const int nk = static_cast<int>(tiles_of_cols(g.cols));
    auto block_of = [&](int job) {
        const int b = job / g.mblocks, strip = (job - b * g.mblocks) * kGStrips;
        if constexpr (!TILES) return GemmBlock{b * g.n, g.n, strip};
        const uint4 p = __ldcg(g.plan + 1 + b);
        return GemmBlock{static_cast<int>(p.x), static_cast<int>(p.y), static_cast<int>(p.z) * g.strips + strip};
    };
    const int nd = 2 * g.n <= int(kGAColumn) ? 2 : 1;
    if (smem_addr(smem) & 1023u) {  // the swizzled layout needs it
        if (threadIdx.x == 0) atomicExch(&g_q4_gemm_status, SMOE_EARG);
        return;
    }
    if (threadIdx.x == 0) {
        for (int i = 0; i < g.nr; ++i) {
            tc::mbar_init(&S.rawfull[i], i == 0 && blockIdx.x == 0 ? 1 + g.withhold : 1);
            tc::mbar_init(&S.rawfree[i], kGGroup);
        }
        for (int i = 0; i < g.nb; ++i) {
            tc::mbar_init(&S.bfull[i], 1);
            tc::mbar_init(&S.bfree[i], 1);
        }
        for (int i = 0; i < kGASlots; ++i) {
            tc::mbar_init(&S.afull[i], kGGroup);
            tc::mbar_init(&S.afree[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            tc::mbar_init(&S.dfull[i], 1);
            tc::mbar_init(&S.dfree[i], kGEnders);
        }
        tc::mbar_init(&S.done, 1);
        tc::fence_barrier_init();
    }
    if (warp == kGDecoders) {
        tc::tmem_alloc(&S.tmem_base, 512);
        tc::tmem_relinquish();
    }
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const uint32_t tmem = S.tmem_base;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
        return __all_sync(0xffffffffu, wait_for(bar, parity));
    };
    // columns c0, c0 + step, .. (eight tokens each) of a job's accumulator, this warp's 32 rows
    auto write_out = [&](int job, int slot, int c0, int step) {
        tc::fence_after_sync();
        const GemmBlock b = block_of(job);
        const int64_t r = int64_t(job % g.mblocks) * kGM + 32 * (warp & 3) + lane, tok0 = b.row0;
        const uint32_t from = tmem + (uint32_t(32 * (warp & 3)) << 16) + uint32_t(g.n * slot);
        const int valid = static_cast<int>(min(int64_t(b.n), g.tokens - tok0));
        int64_t at = (tok0 + c0) * g.rows + r;
        for (int c = c0; c < valid; c += step, at += step * g.rows) {
            uint32_t v[8];
            tc::tmem_ld8(from + c, v);
            tc::tmem_wait_ld();
            if (TILES && r < g.rows) {
                // (whole tiles: every slot is one of the plan's; eight loads of rows in flight together)
                int64_t to[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) to[j] = g.slot_row ? int64_t(__ldcg(g.slot_row + tok0 + c + j)) : tok0 + c + j;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    if (to[j] >= g.out_rows) continue;
                    const float f = __uint_as_float(v[j]);
                    if (g.floats) reinterpret_cast<float*>(g.out)[to[j] * g.rows + r] = f;
                    else g.out[to[j] * g.rows + r] = __float2half_rn(f);
                }
            } else if (r < g.rows) {
                if (g.floats) {
                    float* to = reinterpret_cast<float*>(g.out) + at;
#pragma unroll
                    for (int j = 0; j < 8; ++j, to += g.rows)
                        if (c + j < valid) *to = __uint_as_float(v[j]);
                } else {
                    __half* to = g.out + at;
#pragma unroll
                    for (int j = 0; j < 8; ++j, to += g.rows)
                        if (c + j < valid) *to = __float2half_rn(__uint_as_float(v[j]));
                }
            }
            __syncwarp();
        }
        tc::fence_before_sync();
        __syncwarp();
    };
    bool ok = true;

    if (warp > kGDecoders + 2) {
        // ---------------- the ends of all jobs but the last
        pdl_wait();
        Phase dp;
        for (int job = blockIdx.x; job + int(gridDim.x) < jobs && ok; job += gridDim.x, dp.next(nd)) {
            if (!(ok = wait(&S.dfull[dp.slot], dp.phase))) break;
            write_out(job, dp.slot, 0, 8);
            if (lane == 0) tc::mbar_arrive(&S.dfree[dp.slot]);
        }
    } else if (warp == kGDecoders + 1) {
        // ---------------- the weights' producer
        if (!g.early) pdl_wait();
        Phase rp;
        int stage = 0;
        for (int job = blockIdx.x; job < jobs && ok; job += gridDim.x) {
            const int strip0 = block_of(job).strip0;
            for (int s = 0; s < nk; ++s, ++stage, rp.next(g.nr)) {
                if (stage >= g.nr && !(ok = wait(&S.rawfree[rp.slot], rp.phase ^ 1))) break;
                if (lane == 0) {
                    // (strips past the last read as zeros: weights of zero)
                    tc::mbar_arrive_expect_tx(&S.rawfull[rp.slot], kRaw);
                    tc::tma_load_2d(smem_addr(raw) + rp.slot * kRaw, &maps.w, s * (kTile / 8), strip0,
                                    &S.rawfull[rp.slot]);
                }
                __syncwarp();
            }
        }
        // no copy may still be writing this CTA's shared memory when it leaves
        for (int i = 0; i < g.nr && i < stage; ++i) {
            const int st = stage - 1 - i;
            wait_for(&S.rawfull[st % g.nr], (st / g.nr) & 1);
        }
    } else if (warp == kGDecoders + 2) {
        // ---------------- the activations' producer (they are the launch before's)
        pdl_wait();
        Phase bp;
        int stage = 0;
        for (int job = blockIdx.x; job < jobs && ok; job += gridDim.x) {
            const GemmBlock b = block_of(job);
            for (int s = 0; s < nk; ++s, ++stage, bp.next(g.nb)) {
                if (stage >= g.nb && !(ok = wait(&S.bfree[bp.slot], bp.phase ^ 1))) break;
                if (lane == 0) {
                    const uint32_t dst = smem_addr(smem) + bp.slot * bslot;
                    tc::mbar_arrive_expect_tx(&S.bfull[bp.slot], static_cast<uint32_t>(b_slot_bytes(b.n)));
                    for (int h = 0; h < 2; ++h)
                        tc::tma_load_2d(dst + h * g.n * 128, &maps.a[TILES ? b.n / kSlots - 1 : 0], s * kCols + 64 * h, b.row0,
                                        &S.bfull[bp.slot]);
                }
                __syncwarp();
            }
        }
        for (int i = 0; i < g.nb && i < stage; ++i) {
            const int st = stage - 1 - i;
            wait_for(&S.bfull[st % g.nb], (st / g.nb) & 1);
        }
    } else if (warp == kGDecoders) {
        // ---------------- MMA: one lane alone waits and issues
        if (elect_one()) {
            Phase ap, bp, dp;
            int count = 0;
            for (int job = blockIdx.x; job < jobs && ok; job += gridDim.x, ++count, dp.next(nd)) {
                if (count >= nd && !(ok = wait_for(&S.dfree[dp.slot], dp.phase ^ 1))) break;
                const uint32_t d = tmem + uint32_t(g.n * dp.slot), idesc = tc::idesc_f16_f32(kGM, block_of(job).n);
                for (int s = 0; s < nk; ++s, ap.next(kGASlots), bp.next(g.nb)) {
                    if (!(ok = wait_for(&S.afull[ap.slot], ap.phase)) || !(ok = wait_for(&S.bfull[bp.slot], bp.phase))) break;
                    tc::fence_after_sync();
                    const uint64_t bd = tc::smem_desc_sw128(smem_addr(smem) + bp.slot * bslot);
#pragma unroll
                    for (int k = 0; k < kCols / 16; ++k)
                        tc::mma_f16_ts(d, tmem + kGAColumn + 64u * ap.slot + 8u * k,
                                       bd + uint64_t(((k >> 2) * g.n * 128 + (k & 3) * 32) >> 4), idesc,
                                       (s > 0 || k > 0) ? 1u : 0u);
                    tc::mma_commit(&S.afree[ap.slot]);
                    tc::mma_commit(&S.bfree[bp.slot]);
                    if (s == nk - 1) tc::mma_commit(job + int(gridDim.x) < jobs ? &S.dfull[dp.slot] : &S.done);
                }
            }
            if (!ok) atomicExch(&g_q4_gemm_status, SMOE_ETIMEOUT);
        }
        __syncwarp();
    } else {
        // ---------------- decoders and the end of a job: thread L of the four lane quarters is weight row L. A group of
        // eight warps takes every other stage, the two warps of a quarter two of the four chunks of the row's tile each
        // (conflict-free 16-byte reads, 16 columns of each run).
        const int L = 32 * (warp & 3) + lane, group = warp / kGGroup, pair = (warp >> 2) & 1;
        const int row = L % kRows;
        const uint32_t lanes = tmem + (uint32_t(32 * (warp & 3)) << 16);
        const uint8_t* mine = raw + (L / kRows) * kTile;
        const uint8_t *at0 = mine + chunk_at(row, 2 * pair), *at1 = mine + chunk_at(row, 2 * pair + 1);
        Phase rp, ap, dp;
        int stage = 0;
        for (int job = blockIdx.x; job < jobs && ok; job += gridDim.x, dp.next(nd)) {
            for (int s = 0; s < nk; ++s, ++stage, rp.next(g.nr), ap.next(kGASlots)) {
                if ((stage & 1) != group) continue;
                if (!(ok = wait(&S.rawfull[rp.slot], rp.phase))) break;
                const int slot = rp.slot * kRaw;
                const uint4 c0 = *reinterpret_cast<const uint4*>(at0 + slot), c1 = *reinterpret_cast<const uint4*>(at1 + slot);
                uint32_t p[kCols / G];
                load_pairs<G>(mine + slot, row, p);
                const uint32_t w0[4] = {c0.x, c0.y, c0.z, c0.w}, w1[4] = {c1.x, c1.y, c1.z, c1.w};
                // (the group waited for stage - 5's release two stages ago, so stage - 6's, this slot's one before, is past)
                if (stage >= kGASlots && !(ok = wait(&S.afree[ap.slot], ap.phase ^ 1))) break;
                tc::fence_after_sync();
                const uint32_t to = lanes + kGAColumn + 64u * ap.slot + 8u * pair;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const __half2 sb = *reinterpret_cast<const __half2*>(&p[32 * j / G]);
                    uint32_t v[8];
                    decode8(w0[j], __low2half2(sb), __high2half2(sb), v);
                    decode8(w1[j], __low2half2(sb), __high2half2(sb), v + 4);
                    tc::tmem_st8(to + 16u * j, v);
                }
                tc::tmem_wait_st();
                tc::fence_before_sync();
                __syncwarp();
                if (lane == 0) {
                    tc::mbar_arrive(&S.afull[ap.slot]);
                    tc::mbar_arrive(&S.rawfree[rp.slot]);
                }
            }
            // A CTA's last job is written out by its decoders, who have nothing else left, behind a barrier of its own that
            // completes once. (At a job's barrier a decoder held up for the length of its last eight MMAs could meet the phase of
            // the next job but one on that accumulator, which without its own decoding never completes.)
            if (!ok || job + int(gridDim.x) < jobs) continue;
            if (!(ok = wait(&S.done, 0))) break;
            pdl_wait();  // before an output
            write_out(job, dp.slot, 8 * (warp >> 2), 8 * (kGDecoders / 4));
        }
    }
    if (!ok && lane == 0) atomicExch(&g_q4_gemm_status, SMOE_ETIMEOUT);
    pdl_wait();
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    pdl_release();
    if (warp == kGDecoders) tc::tmem_dealloc(tmem, 512);
}

// ---- host

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// cuTensorMapEncodeTiled through the runtime's driver entry point (no link against libcuda)
static EncodeTiledFn encoder() {
    static std::once_flag once;
    static EncodeTiledFn encode = nullptr;
    std::call_once(once, [] {
        void* fn = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            encode = reinterpret_cast<EncodeTiledFn>(fn);
    });
    return encode;
}

// Microseconds of the prompt's kernel with jobs of n tokens, as measured: a start, and for every round of jobs over the SMs
// a stage's 0.35 us (its hand-offs and decoding) or 2.8 ns a token (its MMAs), whichever is longer, and 1 us at its ends.
// (4096 x 4096: 33 to 128 tokens, one round, 16.1 us, and 16.2 by this; 1180 tokens in jobs of 144, two rounds, 34.0 and 31.8;
// 1536 x 4096, 4096 tokens in jobs of 176, 38.6 and 37.5.)
static double time_of(int64_t tokens, int64_t rows, int64_t cols, int n) {
    const int64_t jobs = (tokens + n - 1) / n * ((rows + kGM - 1) / kGM);
    const double stage = std::max(0.35, 0.0028 * n);
    return 4.0 + double((jobs + kSms - 1) / kSms) * (double(tiles_of_cols(cols)) * stage + 1.0);
}

static int tokens_of_job(int64_t tokens, int64_t rows, int64_t cols) {
    int best = 16;
    for (int n = 32; n <= kGMaxN; n += 16)
        if (time_of(tokens, rows, cols, n) < time_of(tokens, rows, cols, best)) best = n;
    return best;
}

// The streaming kernel takes 3 us, and for every 8 tokens 0.3 us and 0.125 ps a weight (64007 x 2560: 22 us at 5 tokens, 42
// at 12, where the prompt's takes 39 at 24; 4096 x 4096: 8 us at 16 and 11 at 24, the prompt's 16.0 at 48); up to 16 tokens
// are always its (a verify window's token then has the bits it has alone).
bool matmul_better(int64_t tokens, int64_t rows, int64_t cols) {
    if (tokens <= 16) return false;
    const double stream = 3.0 + double((tokens + 7) / 8) * (0.3 + double(rows) * double(cols) * 1.25e-7);
    return time_of(tokens, rows, cols, tokens_of_job(tokens, rows, cols)) < stream;
}

template <int G, bool TILES>
static int launch_gemm(GemmArgs a, const GemmMaps<TILES>& maps, const Writes& w, cudaStream_t st) {
    // (the copies' latency is what the rings hide: a stage of weights is 9 KB and 0.35 us of work or more, so as many as fit
    // beside three stages of activations, then more of those)
    a.nr = kGMaxRaw;
    a.nb = 3;
    while (a.nb > 2 && gemm_smem<G>(a.n, a.nb, 4) > kGSmemLimit) --a.nb;
    // (an even number: the two groups of decoders then wait for slots of their own, every phase in turn)
    while (a.nr > 4 && gemm_smem<G>(a.n, a.nb, a.nr) > kGSmemLimit) a.nr -= 2;
    while (a.nb < kGMaxB && gemm_smem<G>(a.n, a.nb + 1, a.nr) <= kGSmemLimit) ++a.nb;
    const size_t smem = gemm_smem<G>(a.n, a.nb, a.nr);
    a.withhold = wait_test();
    if (int e = max_smem(q4_matmul_kernel<G, TILES>, static_cast<int>(smem)))
        return status_of(static_cast<cudaError_t>(-e), "q4_matmul");
    const int64_t jobs = int64_t(a.nblocks) * a.mblocks;
    return status_of(launch_pdl(w, q4_matmul_kernel<G, TILES>, dim3(static_cast<unsigned>(std::min<int64_t>(jobs, kSms))),
                                dim3(kGThreads), smem, st, a, maps), "q4_matmul");
}

// Tensor maps of `strips` strips of weights and of `tokens` rows of activations, and the launch
template <bool TILES>
static int encode_and_launch(GemmArgs& a, int group, int64_t strips, const void* x, const Writes& w, cudaStream_t st) {
    EncodeTiledFn encode = encoder();
    if (!encode) return fail(SMOE_EARG, "q4_matmul: cuTensorMapEncodeTiled is not available");
    GemmMaps<TILES> maps;
    const cuuint32_t one[2] = {1, 1};
    {
        const int64_t tile = tile_bytes_of(group), strip_bytes = tiles_of_cols(a.cols) * tile;
        const cuuint64_t dims[2] = {static_cast<cuuint64_t>(strip_bytes / 8), static_cast<cuuint64_t>(strips)};
        const cuuint64_t strides[1] = {static_cast<cuuint64_t>(strip_bytes)};
        const cuuint32_t box[2] = {static_cast<cuuint32_t>(tile / 8), kGStrips};
        const CUresult r = encode(&maps.w, CU_TENSOR_MAP_DATA_TYPE_INT64, 2, const_cast<uint8_t*>(a.w), dims, strides, box, one,
                                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
        if (r != CUDA_SUCCESS) return fail(SMOE_EARG, "q4_matmul: weight tensor map rejected (" + std::to_string(int(r)) + ")");
    }
    for (int b = 0; b < int(sizeof(maps.a) / sizeof(maps.a[0])); ++b) {
        // (rows past the tokens and columns past the last read as zeros)
        const cuuint64_t dims[2] = {static_cast<cuuint64_t>(a.cols), static_cast<cuuint64_t>(a.tokens)};
        const cuuint64_t strides[1] = {static_cast<cuuint64_t>(a.cols) * 2};
        const cuuint32_t box[2] = {64, static_cast<cuuint32_t>(TILES ? kSlots * (b + 1) : a.n)};
        const CUresult r = encode(&maps.a[b], CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void*>(x), dims, strides, box, one,
                                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
        if (r != CUDA_SUCCESS)
            return fail(SMOE_EARG, "q4_matmul: activation tensor map rejected (" + std::to_string(int(r)) + ")");
    }
    if (group == 32) return launch_gemm<32, TILES>(a, maps, w, st);
    if (group == 64) return launch_gemm<64, TILES>(a, maps, w, st);
    return launch_gemm<128, TILES>(a, maps, w, st);
}

int matmul_f16(const ProductArgs& p, int group, bool floats, const Writes& w, cudaStream_t st) {
    GemmArgs a = {};
    a.w = p.dw[0];
    a.out = static_cast<__half*>(p.d_out);
    a.rows = p.d_rows;
    a.cols = p.cols;
    a.tokens = p.d_tokens;
    a.early = p.early;
    a.floats = floats;
    a.mblocks = static_cast<int>((p.d_rows + kGM - 1) / kGM);
    a.n = tokens_of_job(p.d_tokens, p.d_rows, p.cols);
    a.nblocks = static_cast<int>((p.d_tokens + a.n - 1) / a.n);
    return encode_and_launch<false>(a, group, strips_of_rows(p.d_rows), p.x, w, st);
}

// ---- a stack's products of many pairs, in tiles of 16 slots of one expert's (smoe_tiles_of)

constexpr int kPlanThreads = 1024;

// Runs of one expert's tiles cut into blocks of up to kTileSlots slots, in their order: one CTA, 1024 tiles at a time.
__global__ void __launch_bounds__(kPlanThreads) q4_plan_kernel(const uint32_t* __restrict__ tile_expert, int tiles,
                                                               uint32_t experts, uint4* __restrict__ plan) {
    constexpr int kMost = kTileSlots / kSlots;
    __shared__ int starts[kPlanThreads / 32], counts[kPlanThreads / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    pdl_wait();
    int run = 0, blocks = 0;  // the last run's first tile, and the blocks, of the tiles before
    for (int t0 = 0; t0 < tiles; t0 += kPlanThreads) {
        const int t = t0 + static_cast<int>(threadIdx.x);
        const uint32_t e = t < tiles ? tile_expert[t] : experts;
        const bool in = e < experts, first = in && (t == 0 || tile_expert[t - 1] != e);
        int start = first ? t : 0;  // this tile's run's first tile: the largest one up to here
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, start, o);
            if (lane >= o) start = max(start, u);
        }
        if (lane == 31) starts[warp] = start;
        __syncthreads();
        int latest = run;
        for (int w = 0; w < kPlanThreads / 32; ++w) {
            if (w < warp) start = max(start, starts[w]);
            latest = max(latest, starts[w]);
        }
        start = max(start, run);
        const bool lead = in && (t - start) % kMost == 0;
        const uint32_t leads = __ballot_sync(0xffffffffu, lead);
        if (lane == 0) counts[warp] = __popc(leads);
        __syncthreads();
        int at = blocks + __popc(leads & ((1u << lane) - 1));
        for (int w = 0; w < kPlanThreads / 32; ++w) {
            if (w < warp) at += counts[w];
            blocks += counts[w];
        }
        if (lead) {
            int n = 1;
            while (n < kMost && t + n < tiles && tile_expert[t + n] == e) ++n;
            plan[1 + at] = make_uint4(uint32_t(t) * kSlots, uint32_t(n) * kSlots, e, 0);
        }
        run = latest;
        __syncthreads();
    }
    if (threadIdx.x == 0) plan[0] = make_uint4(uint32_t(blocks), 0, 0, 0);
    pdl_release();
}

int tile_plan(const uint32_t* tile_expert, int64_t tiles, int64_t experts, void* plan, const Writes& w, cudaStream_t st) {
    return status_of(launch_pdl(w, q4_plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, tile_expert, static_cast<int>(tiles),
                                static_cast<uint32_t>(experts), static_cast<uint4*>(plan)), "q4_tile_plan");
}

int tile_matmul(const TileArgs& p, int group, const Writes& w, cudaStream_t st) {
    GemmArgs a = {};
    a.w = p.w;
    a.out = static_cast<__half*>(p.out);
    a.rows = p.rows;
    a.cols = p.cols;
    a.tokens = p.tiles * kSlots;
    a.mblocks = static_cast<int>((p.rows + kGM - 1) / kGM);
    a.n = kTileSlots;
    a.nblocks = static_cast<int>(p.tiles);  // (at most)
    a.plan = static_cast<const uint4*>(p.plan);
    a.slot_row = p.slot_row;
    a.out_rows = p.out_rows;
    a.strips = static_cast<int>(strips_of_rows(p.rows));
    a.floats = p.floats;
    return encode_and_launch<true>(a, group, p.experts * strips_of_rows(p.rows), p.x, w, st);
}

cudaError_t matmul_status(int* v, bool clear) {
    cudaError_t e = cudaMemcpyFromSymbol(v, g_q4_gemm_status, sizeof(int));
    if (e == cudaSuccess && clear) {
        const int zero = 0;
        e = cudaMemcpyToSymbol(g_q4_gemm_status, &zero, sizeof(int));
    }
    return e;
}

}  // namespace q4
}  // namespace smoe
