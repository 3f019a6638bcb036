// The two streaming kernels on 4-bit weights (layout and arithmetic: q4.cuh), instantiated by smoe_q4_f16.cu and
// smoe_q4_f32.cu.
//
//   q4_product_kernel  out[p, r] = W[e_p][r, :] . x[p / share, :] for a dense matrix (every token through expert 0) and
//                      / or a stack's (token, expert) pairs; with two stacks (gate, up) out = SwiGLU of the two sums,
//                      in one pass over x
//   q4_down_kernel     out[t, r] = sum over t's pairs of Wdown[e][r, :] . h[pair, :] + Wshared[r, :] . hs[t, :]: a MoE
//                      block's down products and its combine, the pairs' weights already in h
//
// What bounds them: a weight is 4.5 bits (groups of 64) of HBM traffic and is used for at most a few rows, so the
// floor is the weights' bytes. Everything here serves the stream of weights: a CTA is four warps, each with a ring
// of bulk copies of its own that runs ahead of the arithmetic across the ends of jobs, and five CTAs share an SM,
// so that 150 KB a SM are in flight (6.5 TB/s x 1 us of latency over 148 SMs asks for 44 KB). No barrier is on that
// path: a warp waits only for its own copies, and the four meet once a job to add their sums.
//
// A job of the product kernel is a strip of 16 rows times one block of up to 8 NT activation rows of one expert; its
// columns are split over the warps of a cluster of 1 to 8 CTAs (a fixed split, the partial sums added in its order:
// the same bits every run). Several tokens of one expert read its rows once.
#pragma once

#include <cooperative_groups.h>

#include "q4.cuh"

namespace smoe {
namespace q4 {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kMaxPairs = 2048;
constexpr uint32_t kWaitLimit = 1u << 22;

// A wait that gave up (never seen; a copy that cannot complete) leaves SMOE_ETIMEOUT here, the launch's outputs are
// then not valid. smoe_q4_status reads and clears it. One per translation unit.
static __device__ int g_q4_status = 0;

struct ProductArgs {
    const void* x;  // (rows, cols), row stride cols
    int64_t cols;
    // dense part: d_tokens rows of x through one matrix
    const uint8_t* dw[2];
    void* d_out;
    int64_t d_rows, d_tokens;
    const void* d_gate;  // GLU: the row's result times sigmoid of this (one a token), or null
    // routed part: pair p takes row p / share of x through expert idx[p] of a stack
    const uint8_t* rw[2];
    void* r_out;
    int64_t r_rows, experts, pairs, share;
    const uint32_t* idx;
    const float* weights;  // GLU: the pair's result times this, or null
    int stages;            // slots of a warp's ring
    bool early;            // the weights may be read before pdl_wait()
    bool hint;             // weights evict-first in L2
};

struct DownArgs {
    const void* h;  // (pairs, ffn)
    const void* hs; // (tokens, sffn), or null with sffn = 0
    const uint8_t* w;
    const uint8_t* sw;
    int64_t ffn, sffn, rows, experts, tokens, k;
    const uint32_t* idx;
    void* out;  // (tokens, rows)
    int stages;
    bool early;  // idx and the weights may be read before pdl_wait()
};

// ---- a warp's ring of bulk copies

struct Ring {
    uint32_t base;    // shared address of slot 0
    uint8_t* ptr;
    uint64_t* bars;
    int slots, slot_bytes;
    int head = 0, tail = 0;  // next slot to fill / to read
    uint32_t phase = 0;
    int in_flight = 0;
    bool ok = true;

    __device__ __forceinline__ void init(uint8_t* p, uint64_t* b, int n, int bytes, int lane) {
        ptr = p;
        base = smem_addr(p);
        bars = b;
        slots = n;
        slot_bytes = bytes;
        if (lane == 0) {
            for (int i = 0; i < n; ++i) tc::mbar_init(&bars[i], 1);
            tc::fence_barrier_init();
        }
        __syncwarp();
    }
    __device__ __forceinline__ bool full() const { return in_flight == slots; }
    // the slot at the tail, once its copies have landed
    __device__ __forceinline__ uint8_t* wait(int lane) {
        if (ok) {
            ok = __all_sync(0xffffffffu, tc::mbar_wait(&bars[tail], phase, kWaitLimit));
            if (!ok && lane == 0) atomicExch(&g_q4_status, SMOE_ETIMEOUT);
        }
        return ptr + tail * slot_bytes;
    }
    __device__ __forceinline__ void pop() {
        if (!ok) return;  // (the slots not waited for are drained at the end)
        --in_flight;
        if (++tail == slots) tail = 0, phase ^= 1;
    }
    // lane 0 only for the copies; every lane keeps the cursor
    __device__ __forceinline__ void push() {
        ++in_flight;
        if (++head == slots) head = 0;
    }
    // no copy may still be writing shared memory when the CTA leaves
    __device__ __forceinline__ void drain(int lane) {
        ok = true;
        while (in_flight > 0) {
            if (!tc::mbar_wait(&bars[tail], phase, kWaitLimit) && lane == 0) atomicExch(&g_q4_status, SMOE_ETIMEOUT);
            pop();
        }
    }
};

__device__ __forceinline__ int warp_incl_sum(int v, int lane) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
    }
    return v;
}

// ---- product

// Exclusive sum of one value a thread over the CTA's threads, in thread order; total in every thread.
__device__ __forceinline__ int block_excl_sum(int v, int* warp_sums, int& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int incl = warp_incl_sum(v, lane);
    if (lane == 31) warp_sums[warp] = incl;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        if (w < warp) before += warp_sums[w];
        total += warp_sums[w];
    }
    __syncthreads();
    return before + incl - v;
}

// Pairs of one expert in blocks of at most `most`, built by every CTA for itself in shared memory. Pairs that name no
// expert (idx >= experts) are in no block.
struct PairBlocks {
    uint16_t *expert, *start, *count, *list;  // a block's expert, first place in list, length; list: pairs
    int n;
};
__host__ __device__ constexpr size_t pair_blocks_bytes(int64_t pairs, int64_t experts) {
    return pairs > 0 ? (size_t(experts) * 4 + size_t(pairs) * 10 + 15) & ~size_t(15) : 0;
}
__device__ __forceinline__ PairBlocks pair_blocks(uint8_t* mem, const uint32_t* __restrict__ idx, int pairs, int experts,
                                                  int most, int* warp_sums) {
    uint32_t* seen = reinterpret_cast<uint32_t*>(mem);  // pairs of an expert, then its first place in list
    PairBlocks b;
    b.list = reinterpret_cast<uint16_t*>(seen + experts);
    uint16_t* place = b.list + pairs;
    b.expert = place + pairs;
    b.start = b.expert + pairs;
    b.count = b.start + pairs;
    const int tid = threadIdx.x;
    for (int e = tid; e < experts; e += kThreads) seen[e] = 0;
    __syncthreads();
    if (tid < 32) {
        // places in pair order (one warp, 32 pairs at a time): every CTA must cut an expert's pairs into the same blocks
        for (int p0 = 0; p0 < pairs; p0 += 32) {
            const int p = p0 + tid;
            const uint32_t e = p < pairs ? idx[p] : 0xffffffffu;
            const uint32_t same = __match_any_sync(0xffffffffu, e);
            const int before = __popc(same & ((1u << tid) - 1));
            if (e < uint32_t(experts)) {
                const uint32_t n = seen[e];
                place[p] = uint16_t(n + before);
                __syncwarp(same);
                if (before == 0) seen[e] = n + __popc(same);
            }
            __syncwarp();
        }
    }
    __syncthreads();
    const int per = (experts + kThreads - 1) / kThreads;
    const int e0 = min(experts, tid * per), e1 = min(experts, e0 + per);
    int mine = 0, members = 0;
    for (int e = e0; e < e1; ++e) {
        members += static_cast<int>(seen[e]);
        mine += (static_cast<int>(seen[e]) + most - 1) / most;
    }
    int all;
    int at = block_excl_sum(members, warp_sums, all);
    int i = block_excl_sum(mine, warp_sums, b.n);
    for (int e = e0; e < e1; ++e) {
        const int n = static_cast<int>(seen[e]);
        for (int j = 0; j < n; j += most, ++i) {
            b.expert[i] = uint16_t(e);
            b.start[i] = uint16_t(at + j);
            b.count[i] = uint16_t(min(most, n - j));
        }
        seen[e] = static_cast<uint32_t>(at);
        at += n;
    }
    __syncthreads();
    for (int p = tid; p < pairs; p += kThreads) {
        const uint32_t e = idx[p];
        if (e < uint32_t(experts)) b.list[seen[e] + place[p]] = uint16_t(p);
    }
    __syncthreads();
    return b;
}

struct ProductJob {
    const uint8_t* w[2];  // the strip's first tile
    int strip, expert_block, tokens0, count;
    bool dense;
};

template <int G, int MATS>
__host__ __device__ constexpr int product_stage_tiles() {
    return MATS == 2 ? 1 : 2;  // a stage is a tile of gate and of up, or two tiles of one matrix
}
template <int G, int MATS>
__host__ __device__ constexpr int product_slot_bytes() {
    return 2 * tile_bytes<G>();
}
// Shared memory: [ring slots, 4 warps][partial sums][pair blocks][barriers]
template <int G, int NT, int MATS>
__host__ __device__ constexpr size_t product_smem(int stages, int64_t pairs, int64_t experts) {
    return size_t(kWarps) * stages * product_slot_bytes<G, MATS>() + size_t(kWarps) * MATS * kRows * 8 * NT * 4 +
           pair_blocks_bytes(pairs, experts) + size_t(kWarps) * stages * 8;
}

__device__ __forceinline__ float sigmoid_f(float g) { return 1.0f / (1.0f + expf(-g)); }

template <typename T, int G, int NT, int MATS>
__global__ void __launch_bounds__(kThreads) q4_product_kernel(const ProductArgs a) {
    namespace cg = cooperative_groups;
    constexpr int kTile = tile_bytes<G>();
    constexpr int kStep = product_stage_tiles<G, MATS>();
    constexpr int kSlot = product_slot_bytes<G, MATS>();
    constexpr int kM = 8 * NT;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int warp_sums[kWarps];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    cg::cluster_group cluster = cg::this_cluster();
    const int csize = static_cast<int>(cluster.num_blocks()), crank = static_cast<int>(cluster.block_rank());
    const int cluster_id = blockIdx.x / csize, clusters = gridDim.x / csize;

    float* red = reinterpret_cast<float*>(smem + size_t(kWarps) * a.stages * kSlot);  // [warp][mat][row][member]
    uint8_t* table = reinterpret_cast<uint8_t*>(red + kWarps * MATS * kRows * kM);
    uint64_t* bars = reinterpret_cast<uint64_t*>(table + pair_blocks_bytes(a.pairs, a.experts));
    Ring ring;
    ring.init(smem + size_t(warp) * a.stages * kSlot, bars + warp * a.stages, a.stages, kSlot, lane);
    const uint64_t policy = tc::policy_evict_first();

    const int ntiles = static_cast<int>(tiles_of_cols(a.cols));
    const int ways = kWarps * csize, way = crank * kWarps + warp;
    const int tile0 = static_cast<int>(int64_t(way) * ntiles / ways), tile1 = static_cast<int>(int64_t(way + 1) * ntiles / ways);
    const int steps = (tile1 - tile0 + kStep - 1) / kStep;
    const int64_t strip_bytes = int64_t(ntiles) * kTile;
    const int d_strips = static_cast<int>(strips_of_rows(a.d_rows)), r_strips = static_cast<int>(strips_of_rows(a.r_rows));
    const int d_blocks = static_cast<int>((a.d_tokens + kM - 1) / kM);
    const int d_jobs = d_strips * d_blocks;
    PairBlocks blocks{nullptr, nullptr, nullptr, nullptr, 0};
    int jobs = d_jobs;  // jobs known so far

    auto job_of = [&](int j) {
        ProductJob o;
        o.dense = j < d_jobs;
        if (o.dense) {
            // (a strip's blocks of tokens are neighbours in time: the second reads the strip from L2)
            o.strip = j / d_blocks;
            o.tokens0 = (j - o.strip * d_blocks) * kM;
            o.count = static_cast<int>(min(int64_t(kM), a.d_tokens - o.tokens0));
            o.expert_block = 0;
#pragma unroll
            for (int m = 0; m < MATS; ++m) o.w[m] = a.dw[m] + o.strip * strip_bytes;
        } else {
            const int i = j - d_jobs;
            o.strip = i / blocks.n;
            o.expert_block = i - o.strip * blocks.n;
            o.tokens0 = blocks.start[o.expert_block];
            o.count = blocks.count[o.expert_block];
#pragma unroll
            for (int m = 0; m < MATS; ++m)
                o.w[m] = a.rw[m] + (int64_t(blocks.expert[o.expert_block]) * r_strips + o.strip) * strip_bytes;
        }
        return o;
    };

    // the copies' cursor: the next stage to fetch
    int fetch_job = cluster_id, fetch_step = 0;
    const uint8_t* fetch_w[2] = {nullptr, nullptr};
    auto fetch = [&]() {
        while (ring.ok && !ring.full() && fetch_job < jobs && steps > 0) {
            if (fetch_step == 0) {
                const ProductJob o = job_of(fetch_job);
#pragma unroll
                for (int m = 0; m < MATS; ++m) fetch_w[m] = o.w[m];
            }
            const int tile = tile0 + fetch_step * kStep;
            const uint32_t bytes = static_cast<uint32_t>(min(kStep, tile1 - tile)) * kTile;
            if (lane == 0) {
                uint64_t* bar = &ring.bars[ring.head];
                tc::mbar_arrive_expect_tx(bar, bytes * MATS);
#pragma unroll
                for (int m = 0; m < MATS; ++m) {
                    const uint32_t dst = ring.base + ring.head * kSlot + m * kTile;
                    if (a.hint) bulk_load_hint(dst, fetch_w[m] + int64_t(tile) * kTile, bytes, bar, policy);
                    else bulk_load(dst, fetch_w[m] + int64_t(tile) * kTile, bytes, bar);
                }
            }
            ring.push();
            if (++fetch_step == steps) {
                fetch_step = 0;
                fetch_job += clusters;
            }
        }
    };
    if (!a.early) pdl_wait();
    fetch();  // the dense part's weights, while the launch before still runs
    pdl_wait();
    if (a.pairs > 0) {
        blocks = pair_blocks(table, a.idx, static_cast<int>(a.pairs), static_cast<int>(a.experts), kM, warp_sums);
        jobs = d_jobs + blocks.n * r_strips;
        fetch();
    }

    const T* x = static_cast<const T*>(a.x);
    const int col_runs = static_cast<int>(a.cols / 32);
    for (int job = cluster_id; job < jobs; job += clusters) {
        const ProductJob o = job_of(job);
        const T* xp[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int n = 8 * nt + g;
            xp[nt] = nullptr;
            if (n < o.count) {
                const int64_t row = o.dense ? o.tokens0 + n : blocks.list[o.tokens0 + n] / a.share;
                xp[nt] = x + row * a.cols + 8 * t;
            }
        }
        float acc[MATS][NT][4] = {};
        for (int s = 0; s < steps; ++s) {
            // (the activations first: their latency passes while the weights' copies land)
            Acts<T> xs[kStep][NT][4];
#pragma unroll
            for (int i = 0; i < kStep; ++i) {
                const int tile = tile0 + s * kStep + i;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if (xp[nt] != nullptr && tile < tile1 && tile * 4 + j < col_runs)
                            xs[i][nt][j].load(xp[nt] + tile * kCols + 32 * j);
                        else xs[i][nt][j].zero();
                    }
            }
            const uint8_t* slot = ring.wait(lane);
#pragma unroll
            for (int i = 0; i < kStep; ++i) {
                if (kStep > 1 && tile0 + s * kStep + i >= tile1) break;
                auto load = [&](int nt, int j, Acts<T>& v) { v = xs[i][nt][j]; };
                auto on = [&](int nt) { return true; };
                tile_mma<T, G, NT, MATS>(slot + i * kTile, kTile, lane, acc, load, on);
            }
            __syncwarp();
            ring.pop();
            fetch();
        }
        // the warps' sums, then the cluster's: partial sums in the order of the column ranges
#pragma unroll
        for (int m = 0; m < MATS; ++m)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    red[((warp * MATS + m) * kRows + g + 8 * (i >> 1)) * kM + 8 * nt + 2 * t + (i & 1)] = acc[m][nt][i];
        if (csize > 1) cluster.sync();
        else __syncthreads();
        const int rows = static_cast<int>(o.dense ? a.d_rows : a.r_rows);
        for (int i = crank * kThreads + tid; i < kRows * kM; i += csize * kThreads) {
            const int r = i & (kRows - 1), n = i / kRows;
            const int row = o.strip * kRows + r;
            if (n >= o.count || row >= rows) continue;
            float sum[MATS] = {};
            for (int c = 0; c < csize; ++c) {
                const float* from = csize > 1 ? cluster.map_shared_rank(red, c) : red;
#pragma unroll
                for (int w = 0; w < kWarps; ++w)
#pragma unroll
                    for (int m = 0; m < MATS; ++m) sum[m] += from[((w * MATS + m) * kRows + r) * kM + n];
            }
            const int64_t to = o.dense ? o.tokens0 + n : blocks.list[o.tokens0 + n];
            float v = sum[0];
            if constexpr (MATS == 2) {
                // silu(gate) up, times the row's share of the block's output: float32 up to the one rounding
                v = sum[0] * sigmoid_f(sum[0]) * sum[MATS - 1];
                if (o.dense) {
                    if (a.d_gate != nullptr) v *= sigmoid_f(to_f32(static_cast<const T*>(a.d_gate)[to]));
                } else if (a.weights != nullptr) {
                    v *= a.weights[to];
                }
            }
            T* out = static_cast<T*>(o.dense ? a.d_out : a.r_out);
            out[to * rows + row] = from_f32<T>(v);
        }
        if (csize > 1) cluster.sync();
        else __syncthreads();
    }
    pdl_release();
    ring.drain(lane);
}

// ---- down products and the combine of a MoE block, at most 8 NT tokens

// The chosen experts, each with the tokens that chose it (a bit a token), in the order of the experts; a token's
// second choice of the same expert is a group of its own, after them.
constexpr uint16_t kNone = 0xffff, kAgain = 0x8000;
struct Groups {
    uint64_t* tokens;  // [experts]
    uint16_t* key;     // [pairs]: the pair's expert; kNone: no expert, kAgain | expert: not the first time
    uint16_t* group;   // [n]: the expert; kAgain | pair
    int n;
    __device__ __forceinline__ int expert(int i) const {
        return group[i] & kAgain ? key[group[i] & ~kAgain] & ~kAgain : group[i];
    }
};
__host__ __device__ constexpr size_t groups_bytes(int64_t pairs, int64_t experts) {
    return (size_t(experts) * 8 + size_t(pairs) * 4 + 15) & ~size_t(15);
}
__device__ __forceinline__ Groups expert_groups(uint8_t* mem, const uint32_t* __restrict__ idx, int pairs, int k,
                                                int experts, int* warp_sums) {
    Groups r;
    r.tokens = reinterpret_cast<uint64_t*>(mem);
    r.key = reinterpret_cast<uint16_t*>(r.tokens + experts);
    r.group = r.key + pairs;
    const int tid = threadIdx.x;
    for (int e = tid; e < experts; e += kThreads) r.tokens[e] = 0;
    __syncthreads();
    int again_any = 0;
    for (int p = tid; p < pairs; p += kThreads) {
        const uint32_t e = idx[p];
        uint16_t key = kNone;
        if (e < uint32_t(experts)) {
            const int tok = p / k;
            bool again = false;
            for (int q = tok * k; q < p; ++q) again |= idx[q] == e;
            key = uint16_t(e | (again ? kAgain : 0));
            if (!again) atomicOr(reinterpret_cast<unsigned long long*>(&r.tokens[e]), 1ull << tok);
            again_any |= again;
        }
        r.key[p] = key;
    }
    again_any = __syncthreads_or(again_any);
    const int per = (experts + kThreads - 1) / kThreads;
    const int e0 = min(experts, tid * per), e1 = min(experts, e0 + per);
    int mine = 0;
    for (int e = e0; e < e1; ++e) mine += r.tokens[e] != 0;
    int i = block_excl_sum(mine, warp_sums, r.n);
    for (int e = e0; e < e1; ++e)
        if (r.tokens[e] != 0) r.group[i++] = uint16_t(e);
    if (again_any) {
        if (tid < 32) {
            int n = r.n;
            for (int p0 = 0; p0 < pairs; p0 += 32) {
                const int p = p0 + tid;
                const bool again = p < pairs && r.key[p] != kNone && (r.key[p] & kAgain);
                const uint32_t m = __ballot_sync(0xffffffffu, again);
                if (again) r.group[n + __popc(m & ((1u << tid) - 1))] = uint16_t(kAgain | p);
                n += __popc(m);
            }
            if (tid == 0) warp_sums[0] = n;
        }
        __syncthreads();
        r.n = warp_sums[0];
    }
    __syncthreads();
    return r;
}

template <int G>
__host__ __device__ constexpr int down_slot_bytes() {
    return tile_bytes<G>();
}
template <int G, int NT>
__host__ __device__ constexpr size_t down_smem(int stages, int64_t pairs, int64_t experts) {
    return size_t(kWarps) * stages * down_slot_bytes<G>() + size_t(kWarps) * kRows * 8 * NT * 4 + groups_bytes(pairs, experts) +
           size_t(kWarps) * stages * 8;
}

template <typename T, int G, int NT>
__global__ void __launch_bounds__(kThreads) q4_down_kernel(const DownArgs a) {
    namespace cg = cooperative_groups;
    constexpr int kTile = tile_bytes<G>();
    constexpr int kM = 8 * NT;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int warp_sums[kWarps];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    cg::cluster_group cluster = cg::this_cluster();
    const int csize = static_cast<int>(cluster.num_blocks()), crank = static_cast<int>(cluster.block_rank());
    const int strip = blockIdx.x / csize;

    float* red = reinterpret_cast<float*>(smem + size_t(kWarps) * a.stages * kTile);  // [warp][row][token]
    uint8_t* table = reinterpret_cast<uint8_t*>(red + kWarps * kRows * kM);
    uint64_t* bars = reinterpret_cast<uint64_t*>(table + groups_bytes(a.tokens * a.k, a.experts));
    Ring ring;
    ring.init(smem + size_t(warp) * a.stages * kTile, bars + warp * a.stages, a.stages, kTile, lane);
    const uint64_t policy = tc::policy_evict_first();

    if (!a.early) pdl_wait();
    const Groups gr = expert_groups(table, a.idx, static_cast<int>(a.tokens * a.k), static_cast<int>(a.k),
                                    static_cast<int>(a.experts), warp_sums);
    // the strip's tiles: the shared expert's, then each chosen expert's; a way takes a range of them
    const int stiles = static_cast<int>(tiles_of_cols(a.sffn)), ftiles = static_cast<int>(tiles_of_cols(a.ffn));
    const int64_t strips = strips_of_rows(a.rows);
    const int total = stiles + gr.n * ftiles;
    const int ways = kWarps * csize, way = crank * kWarps + warp;
    const int item0 = static_cast<int>(int64_t(way) * total / ways), item1 = static_cast<int>(int64_t(way + 1) * total / ways);

    struct Cursor {
        int seg, tile, tiles;  // seg -1: the shared expert
    };
    auto place = [&](int item) {
        if (item < stiles) return Cursor{-1, item, stiles};
        const int seg = (item - stiles) / ftiles;
        return Cursor{seg, item - stiles - seg * ftiles, ftiles};
    };
    auto step = [&](Cursor& c) {
        if (++c.tile == c.tiles) {
            ++c.seg;
            c.tile = 0;
            c.tiles = ftiles;
        }
    };
    auto strip_of = [&](const Cursor& c) {
        return c.seg < 0 ? a.sw + int64_t(strip) * stiles * kTile
                         : a.w + (int64_t(gr.expert(c.seg)) * strips + strip) * ftiles * kTile;
    };
    int next = item0;
    Cursor fc = place(item0);
    const uint8_t* fw = nullptr;
    int fseg = -2;
    auto fetch = [&]() {
        while (ring.ok && !ring.full() && next < item1) {
            if (fc.seg != fseg) {
                fw = strip_of(fc);
                fseg = fc.seg;
            }
            if (lane == 0) {
                uint64_t* bar = &ring.bars[ring.head];
                tc::mbar_arrive_expect_tx(bar, kTile);
                bulk_load_hint(ring.base + ring.head * kTile, fw + int64_t(fc.tile) * kTile, kTile, bar, policy);
            }
            ring.push();
            ++next;
            step(fc);
        }
    };
    fetch();
    pdl_wait();

    float acc[1][NT][4] = {};
    const T* xp[NT];
    uint64_t mask = 0;
    int seg = -2;
    Cursor c = place(item0);
    for (int item = item0; item < item1; ++item, step(c)) {
        if (c.seg != seg) {
            // this lane's row of each block of 8 tokens: the pair of token 8 nt + g that chose this expert
            seg = c.seg;
            const uint16_t group = seg < 0 ? 0 : gr.group[seg];
            mask = seg < 0 ? ~0ull : group & kAgain ? 1ull << ((group & ~kAgain) / static_cast<int>(a.k)) : gr.tokens[group];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const int tok = 8 * nt + g;
                xp[nt] = nullptr;
                if (tok >= a.tokens || !((mask >> tok) & 1)) continue;
                if (seg < 0) {
                    xp[nt] = static_cast<const T*>(a.hs) + tok * a.sffn + 8 * t;
                } else {
                    int p = tok * static_cast<int>(a.k);
                    if (group & kAgain) p = group & ~kAgain;
                    else while (gr.key[p] != group) ++p;
                    xp[nt] = static_cast<const T*>(a.h) + p * a.ffn + 8 * t;
                }
            }
        }
        const int runs = static_cast<int>((seg < 0 ? a.sffn : a.ffn) / 32);
        auto get = [&](int nt, int j, Acts<T>& v) {
            if (xp[nt] != nullptr && c.tile * 4 + j < runs) v.load(xp[nt] + c.tile * kCols + 32 * j);
            else v.zero();
        };
        // (up to 16 tokens: the activations before the wait; more would not fit the registers)
        constexpr bool kAhead = NT <= 2;
        Acts<T> xs[kAhead ? NT : 1][4];
        if constexpr (kAhead) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int j = 0; j < 4; ++j) get(nt, j, xs[nt][j]);
        }
        const uint8_t* slot = ring.wait(lane);
        auto load = [&](int nt, int j, Acts<T>& v) {
            if constexpr (kAhead) v = xs[nt][j];
            else get(nt, j, v);
        };
        auto on = [&](int nt) { return ((mask >> (8 * nt)) & 255) != 0 && 8 * nt < a.tokens; };
        tile_mma<T, G, NT, 1>(slot, kTile, lane, acc, load, on);
        __syncwarp();
        ring.pop();
        fetch();
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            red[(warp * kRows + g + 8 * (i >> 1)) * kM + 8 * nt + 2 * t + (i & 1)] = acc[0][nt][i];
    pdl_release();
    if (csize > 1) cluster.sync();
    else __syncthreads();
    for (int i = crank * kThreads + tid; i < kRows * kM; i += csize * kThreads) {
        const int r = i & (kRows - 1), n = i / kRows;
        const int64_t row = int64_t(strip) * kRows + r;
        if (n >= a.tokens || row >= a.rows) continue;
        float sum = 0.0f;
        for (int cr = 0; cr < csize; ++cr) {
            const float* from = csize > 1 ? cluster.map_shared_rank(red, cr) : red;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) sum += from[(w * kRows + r) * kM + n];
        }
        static_cast<T*>(a.out)[n * a.rows + row] = from_f32<T>(sum);
    }
    ring.drain(lane);
    if (csize > 1) cluster.sync();  // a CTA's sums are read by the others until here
}

}  // namespace q4
}  // namespace smoe
