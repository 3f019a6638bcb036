// The two streaming kernels on 4-bit weights (layout and arithmetic: q4.cuh), instantiated by smoe_q4_product_*.cu and
// smoe_q4_down_*.cu.
//
//   q4_product_kernel  out[p, r] = W[e_p][r, :] . x[p / share, :] for a dense matrix (every token through expert 0) and
//                      / or a stack's (token, expert) pairs; with two stacks (gate, up) out = SwiGLU of the two sums,
//                      in one pass over x
//   q4_down_kernel     out[t, r] = sum over t's pairs of Wdown[e][r, :] . h[pair, :] + Wshared[r, :] . hs[t, :]: a MoE
//                      block's down products and its combine, the pairs' weights already in h
//
// What bounds them: a weight is 4.5 bits (groups of 64) of HBM traffic and is used for at most a few rows, so the floor is the
// weights' bytes; next to it stands the instruction issue (a tile of 16 x 128 weights is about 108 warp instructions and
// 1088 bytes, 47 cycles of an SM at full bandwidth, and a job's ends are 580 instructions more). So two strips of rows share
// each activation operand, and nothing but a warp's own copies is waited for inside a job: every warp has a ring of bulk
// copies of its own that runs ahead of the arithmetic across the ends of jobs, 16 warps a SM, 75 to 150 KB of a SM in flight
// (6.5 TB/s x 1 us of latency over 148 SMs asks for 44 KB). 64007 x 2560 at 5 tokens: 20.6 us, 4.2 TB/s, a
// start and an end of about 5 us and uneven shares (2001 jobs over 2368 warps, one or none each: the busiest has 1.18 times the
// mean); a block of 512 experts of 640 x 2560 at 32 tokens 170 us, 632 MB, the ends of its blocks of rows.
//
// A job of the product kernel is two strips of 16 rows (gate's and up's, or two neighbours) times one block of up to 8
// activation rows of one expert; its columns are split over a team of 1 to 8 warps of a CTA, the partial sums added in
// the order of the columns: the same bits every run. Several tokens of one expert read its rows once.
#pragma once

#include "q4.cuh"

namespace smoe {
namespace q4 {

constexpr int kWarps = 8;
constexpr int kThreads = 32 * kWarps;
constexpr int kMaxPairs = 2048;

// A wait that gave up (never seen; a copy that cannot complete) leaves SMOE_ETIMEOUT here, the launch's outputs are
// then not valid. smoe_q4_status reads and clears it. One per translation unit.
static __device__ int g_q4_status = 0;

// Division of numbers from 0 to 2^31 - 1 by one that a kernel keeps
struct Divisor {
    uint32_t n = 1, inverse = 0;
    Divisor() = default;
    __host__ __device__ __forceinline__ explicit Divisor(int by) : n(by), inverse(by > 1 ? 0xffffffffu / n : 0) {}
    __device__ __forceinline__ int operator()(int a) const {
        if (n == 1) return a;
        uint32_t q = __umulhi(uint32_t(a), inverse);  // at most one too small: inverse is less than 1 below 2^32 / n
        if (uint32_t(a) - q * n >= n) ++q;
        return static_cast<int>(q);
    }
};

struct ProductArgs {
    const void* x;  // (rows, cols), row stride cols
    int64_t cols;
    // dense part: d_tokens rows of x through one matrix
    const uint8_t* dw[2];
    void* d_out;
    int64_t d_rows, d_tokens;
    const void* d_gate;  // GLU: the row's result times sigmoid of this (one a token), or null
    const float* d_gate32;  // the same in float32, in d_gate's place
    // routed part: pair p takes row p / share of x through expert idx[p] of a stack
    const uint8_t* rw[2];
    void* r_out;
    int64_t r_rows, experts, pairs, share;
    const uint32_t* idx;
    const float* weights;  // GLU: the pair's result times this, or null
    bool pieces;     // GLU, float16: a result as two rows, its float16 and what that leaves (rows 2 p and 2 p + 1 of out)
    uint32_t* zero;  // words to clear for the launch after (its counters)
    int n_zero;
    // what a warp would work out for itself first (the host's: a division is some 40 instructions of every warp's start)
    int team_log;                         // log2 of the warps that share a job's columns
    int tiles, runs;                      // of a row: 128-column tiles, 32-column runs
    int d_strips, r_strips, d_wide, r_wide, d_blocks;  // strips, jobs of one block of rows, blocks of tokens
    Divisor by_dense, by_share;           // by d_blocks, by share
    bool early;  // the weights may be read before pdl_wait()
    bool hint;   // weights evict-first in L2
    int withhold;  // a test's: 1, CTA 0's first copy never counts as landed
};

struct DownArgs {
    const void* h;   // (pairs, ffn); float16: (2 pairs, ffn), in pieces
    const void* hs;  // (tokens, sffn) likewise, or null with sffn = 0
    const uint8_t* w;
    const uint8_t* sw;
    int64_t ffn, sffn, rows, experts, tokens, k;
    const uint32_t* idx;
    void* out;           // (tokens, rows)
    float* partial;      // [CTAs][2][tokens][32]
    uint32_t* counters;  // one a job, zero
    bool early;          // idx and the weights may be read before pdl_wait()
    int withhold;        // as ProductArgs'
    int stiles, ftiles, strips, jobs;
    Divisor by_k, by_stiles, by_ftiles;
};

// ---- a warp's ring of bulk copies: two slots, the copies' and the reader's counts say which

constexpr int kStages = 2;  // slots

// LOOK: how the copies stop once a wait gave up (a barrier's phase may then be open): each looks at `dead` first, or the wait
// ends the run of tiles that is being fetched and the next run's first copy looks. (64007 x 2560 at 5 tokens: float32, groups of
// 32, 63.7 us and 68.7; float16, groups of 64, 24.7 and 22.4.)
template <bool LOOK>
struct Ring {
    uint32_t slots, bars;  // shared addresses
    uint32_t fetched = 0, taken = 0;
    int left = 0;  // tiles still to be fetched of the run of tiles that the copies' cursor is in
    bool dead = false;  // a wait gave up: what follows is read as it lies, nothing more is fetched

    // withhold: arrivals that the first slot's barrier waits for and that never come
    __device__ __forceinline__ void init(uint8_t* p, uint64_t* b, int lane, int withhold) {
        slots = smem_addr(p);
        bars = smem_addr(b);
        if (lane == 0) {
            for (int i = 0; i < kStages; ++i) tc::mbar_init(&b[i], i == 0 ? 1 + withhold : 1);
            tc::fence_barrier_init();
        }
        __syncwarp();
    }
    __device__ __forceinline__ uint64_t* barrier(uint32_t i) const {
        return static_cast<uint64_t*>(__cvta_shared_to_generic(bars + 8 * i));
    }
    __device__ __forceinline__ bool full() const { return fetched - taken == kStages; }
    // the next slot's shared address, once its copies have landed
    template <int SLOT>
    __device__ __forceinline__ uint32_t wait(int lane) {
        const uint32_t at = taken & 1, phase = (taken >> 1) & 1;
        if (!__all_sync(0xffffffffu, try_wait(bars + 8 * at, phase))) {
            if (!dead && !__all_sync(0xffffffffu, wait_for(barrier(at), phase))) {
                dead = true;
                if constexpr (!LOOK) left = 0;
                if (lane == 0) atomicExch(&g_q4_status, SMOE_ETIMEOUT);
            }
        }
        return slots + at * SLOT;
    }
    // two copies of `bytes` into the next slot's halves (the whole warp calls, one lane issues)
    template <int SLOT>
    __device__ __forceinline__ void fetch(const uint8_t* w0, const uint8_t* w1, uint32_t bytes, uint64_t policy) {
        if (LOOK && dead) return;
        const uint32_t at = fetched & 1;
        ++fetched;
        if (elect_one()) {
            const uint32_t bar = bars + 8 * at, dst = slots + at * SLOT;
            arrive_expect(bar, 2 * bytes);
            bulk_load(dst, w0, bytes, bar, policy);
            bulk_load(dst + SLOT / 2, w1, bytes, bar, policy);
        }
    }
    // no copy may still be writing shared memory when the CTA leaves
    __device__ __forceinline__ void drain(int lane) {
        for (uint32_t i = fetched < kStages ? 0 : fetched - kStages; i < fetched; ++i)
            if (!wait_for(barrier(i & 1), (i >> 1) & 1) && lane == 0) atomicExch(&g_q4_status, SMOE_ETIMEOUT);
    }
};

template <typename T>
using RingOf = Ring<sizeof(T) == 4>;

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
    return pairs > 0 ? (size_t(experts) * 4 + size_t(pairs) * 12 + 15) & ~size_t(15) : 0;
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
    uint16_t* key = b.count + pairs;  // a pair's expert, or none
    const int tid = threadIdx.x;
    if (pairs <= 32) {
        // (a decode step's few pairs: one warp, one barrier)
        if (tid < 32) {
            const uint32_t e = tid < pairs ? idx[tid] : 0xffffffffu;
            const bool in = e < uint32_t(experts);
            const uint32_t same = __match_any_sync(0xffffffffu, e);
            const int before = __popc(same & ((1u << tid) - 1)), within = before % most;
            const bool lead = in && within == 0;
            const uint32_t leads = __ballot_sync(0xffffffffu, lead);
            const int members = lead ? min(most, __popc(same) - before) : 0;
            const int first = warp_incl_sum(members, tid) - members;
            const int leader = before < most ? __ffs(same) - 1 : static_cast<int>(__fns(same, 0, before - within + 1));
            const int at = __shfl_sync(0xffffffffu, first, leader) + within;
            if (lead) {
                const int i = __popc(leads & ((1u << tid) - 1));
                b.expert[i] = uint16_t(e);
                b.start[i] = uint16_t(first);
                b.count[i] = uint16_t(members);
            }
            if (in) b.list[at] = uint16_t(tid);
            if (tid == 0) warp_sums[0] = __popc(leads);
        }
        __syncthreads();
        b.n = warp_sums[0];
        return b;
    }
    constexpr uint16_t kNone = 0xffff;
    for (int e = tid; e < experts; e += kThreads) seen[e] = 0;
    for (int p = tid; p < pairs; p += kThreads) {
        const uint32_t e = idx[p];
        key[p] = e < uint32_t(experts) ? uint16_t(e) : kNone;
    }
    __syncthreads();
    if (tid < 32) {
        // places in pair order (one warp, 32 pairs at a time): every CTA must cut an expert's pairs into the same blocks
        for (int p0 = 0; p0 < pairs; p0 += 32) {
            const int p = p0 + tid;
            const uint32_t e = p < pairs ? key[p] : kNone;
            const uint32_t same = __match_any_sync(0xffffffffu, e);
            const int before = __popc(same & ((1u << tid) - 1));
            if (e != kNone) {
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
    for (int p = tid; p < pairs; p += kThreads)
        if (key[p] != kNone) b.list[seen[key[p]] + place[p]] = uint16_t(p);
    __syncthreads();
    return b;
}

constexpr int kMt = 2;      // strips whose tiles are multiplied together: gate and up, or two neighbours of one matrix
constexpr int kStep = 2;  // tiles of a stage
constexpr int kCtas = 2;  // CTAs of an SM
constexpr int kM = 8;     // rows of activations in a block
template <int G>
__host__ __device__ constexpr int slot_bytes() {
    return kMt * kStep * tile_bytes<G>();
}
constexpr int kRedFloats = kMt * kRows * kM;  // a warp's sums of one job

// `left` tiles of two strips, as they come through the ring in stages of kStep and a last one of what is left, times a
// block of activation rows: xp is this lane's place in its row at the first tile's first column, runs the row's 32-column
// runs from there on. Pairs of whole tiles take a loop without any other condition (215 instructions a tile of both strips
// with groups of 128, against 250 with the conditions of a general one), each tile's activations loaded during the tile
// before; with groups of 32, whose sums take the registers, a pair's second tile's between the two (64007 x 2560 at 5 tokens
// 26.3 us, and 28.0 with the loads ahead).
template <typename T, int G, class Fetch>
__device__ __forceinline__ void stream_tiles(RingOf<T>& ring, Fetch& fetch, const T* xp, int left, int runs, int lane,
                                             float (&acc)[2][4], const Ones<T>& one) {
    static_assert(kStep == 2, "a stage is a pair of tiles");
    constexpr int kTile = tile_bytes<G>(), kStride = kStep * kTile;
    int pairs = min(left, runs >> 2) >> 1;
    left -= 2 * pairs;
    if (pairs > 0) {
        runs -= 8 * pairs;
        TileActs<T> x0, x1;
        x0.load(xp);
#pragma unroll 1
        do {
            const uint32_t slot = ring.wait<2 * kStride>(lane);
            if constexpr (G != 32) x1.load(xp + kCols);
            tile_mma<T, G>(slot, kStride, lane, x0, acc, one);
            if constexpr (G == 32) x1.load(xp + kCols);
            --pairs;
            xp += 2 * kCols;
            x0.load(pairs > 0 ? xp : xp - 2 * kCols);  // (after the last pair: any place of the row)
            tile_mma<T, G>(slot + kTile, kStride, lane, x1, acc, one);
            __syncwarp();
            ++ring.taken;
            fetch();
        } while (pairs > 0);
    }
#pragma unroll 1
    while (left > 0) {
        const uint32_t slot = ring.wait<2 * kStride>(lane);
#pragma unroll 1
        for (int i = 0; i < kStep && left > 0; ++i, --left, xp += kCols, runs -= 4) {
            TileActs<T> x;
            x.load(xp, runs);
            tile_mma<T, G>(slot + i * kTile, kStride, lane, x, acc, one);
        }
        __syncwarp();
        ++ring.taken;
        fetch();
    }
}

// Shared memory: [ring slots, 8 warps][two jobs' partial sums, 8 warps][pair blocks][barriers]
template <int G>
__host__ __device__ constexpr size_t product_smem(int64_t pairs, int64_t experts) {
    return size_t(kWarps) * kStages * slot_bytes<G>() + size_t(kWarps) * 2 * kRedFloats * 4 +
           pair_blocks_bytes(pairs, experts) + size_t(kWarps) * kStages * 8;
}

__device__ __forceinline__ float sigmoid_f(float g) { return 1.0f / (1.0f + expf(-g)); }

// GLU: the two strips of a job are gate's and up's, else two neighbours.
template <typename T, int G, bool GLU>
__global__ void __launch_bounds__(kThreads, kCtas) q4_product_kernel(const ProductArgs a) {
    constexpr int kTile = tile_bytes<G>();
    constexpr int kSlot = slot_bytes<G>();
    constexpr int kWide = GLU ? 1 : 2;  // strips of the result in a job
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int warp_sums[kWarps];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int team_size = 1 << a.team_log, team = warp >> a.team_log, member = warp & (team_size - 1);
    // (teams of one CTA are far apart in the jobs' order: a few jobs spread over the SMs)
    const int team_id = team * gridDim.x + blockIdx.x, teams = (kWarps >> a.team_log) * gridDim.x;

    float* red = reinterpret_cast<float*>(smem + size_t(kWarps) * kStages * kSlot);
    uint8_t* table = reinterpret_cast<uint8_t*>(red + kWarps * 2 * kRedFloats);
    uint64_t* bars = reinterpret_cast<uint64_t*>(table + pair_blocks_bytes(a.pairs, a.experts));
    red += (team << a.team_log) * 2 * kRedFloats;  // [job's parity][member][strip][row][column]
    RingOf<T> ring;
    ring.init(smem + size_t(warp) * kStages * kSlot, bars + warp * kStages, lane, blockIdx.x == 0 && warp == 0 ? a.withhold : 0);
    // (weights of experts are read once; a layer's may be read again by its next block of tokens or its next call)
    const uint64_t policy = a.hint ? tc::policy_evict_first() : policy_evict_normal();

    const int tile0 = (member * a.tiles) >> a.team_log, tile1 = ((member + 1) * a.tiles) >> a.team_log;
    const int64_t strip_bytes = int64_t(a.tiles) * kTile;
    const int d_jobs = a.d_wide * a.d_blocks;
    PairBlocks blocks{nullptr, nullptr, nullptr, nullptr, 0};
    int jobs = d_jobs;  // jobs known so far

    // job -> strips (from kWide times the first) and block of rows; a strip's blocks are neighbours in time, so that the
    // second reads the strip from L2
    Divisor by_blocks;
    auto place = [&](int j, int& strip, int& block) {
        if (j < d_jobs) {
            strip = a.by_dense(j);
            block = j - strip * a.d_blocks;
        } else {
            j -= d_jobs;
            strip = by_blocks(j);
            block = j - strip * blocks.n;
        }
    };

    // the copies' cursor: the next stage to fetch
    int fetch_job = tile0 < tile1 ? team_id : 0x7fffffff;
    const uint8_t *fetch0 = nullptr, *fetch1 = nullptr;
    auto fetch = [&]() {  // (a slot is free)
        if (ring.left == 0) {
            if (fetch_job >= jobs || ring.dead) return;
            int strip, block;
            place(fetch_job, strip, block);
            const bool dense = fetch_job < d_jobs;
            const int strips = dense ? a.d_strips : a.r_strips;
            const int64_t first = dense ? 0 : int64_t(blocks.expert[block]) * a.r_strips;
            const uint8_t* w0 = dense ? a.dw[0] : a.rw[0];
            const uint8_t* w1 = !GLU ? w0 : dense ? a.dw[1] : a.rw[1];
            fetch0 = w0 + (first + strip * kWide) * strip_bytes + int64_t(tile0) * kTile;
            // (the last job of an odd number of strips takes its one strip twice)
            fetch1 = w1 + (first + (GLU ? strip : min(strip * 2 + 1, strips - 1))) * strip_bytes + int64_t(tile0) * kTile;
            ring.left = tile1 - tile0;
            fetch_job += teams;
        }
        const int n = min(kStep, ring.left);
        ring.template fetch<kSlot>(fetch0, fetch1, n * kTile, policy);
        fetch0 += n * kTile;
        fetch1 += n * kTile;
        ring.left -= n;
    };
    if (!a.early) pdl_wait();
    // the dense part's weights, while the launch before still runs
    for (int i = 0; i < kStages; ++i) fetch();
    pdl_wait();
    if (a.pairs > 0) {
        blocks = pair_blocks(table, a.idx, static_cast<int>(a.pairs), static_cast<int>(a.experts), kM, warp_sums);
        jobs = d_jobs + blocks.n * a.r_wide;
        by_blocks = Divisor(max(1, blocks.n));
        for (int i = 0; i < kStages; ++i)
            if (!ring.full()) fetch();
        if (blockIdx.x == 0)
            for (int i = tid; i < a.n_zero; i += kThreads) a.zero[i] = 0;
    }

    const Ones<T> one;
    const T* x = static_cast<const T*>(a.x) + 8 * t;
    const int runs0 = a.runs - 4 * tile0;
    // the thread's part of a job's results: a row, and every so many of its columns
    constexpr int kOut = kWide * kRows;
    const int out_r = lane & (kOut - 1), out_n = (member * 32 + lane) / kOut;
    int parity = 0;
    for (int job = team_id; job < jobs; job += teams, parity ^= 1) {
        const bool dense = job < d_jobs;
        int strip, block;
        place(job, strip, block);
        const int start = dense ? block * kM : blocks.start[block];
        const int count = dense ? static_cast<int>(min(int64_t(kM), a.d_tokens - start)) : blocks.count[block];
        // (columns past the count repeat the first row; their results are not written)
        const int at = g < count ? start + g : start;
        const T* xp = x + int64_t(dense ? at : a.by_share(blocks.list[at])) * a.cols + tile0 * kCols;
        float acc[kMt][4] = {};
        stream_tiles<T, G>(ring, fetch, xp, tile1 - tile0, runs0, lane, acc, one);
        // the team's sums, in the order of the column ranges (one barrier a job: the next job's sums have another place)
        float* sums = red + ((parity * kRedFloats) << a.team_log);
#pragma unroll
        for (int m = 0; m < kMt; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                sums[((member * kMt + m) * kRows + g + 8 * (i >> 1)) * kM + 2 * t + (i & 1)] = acc[m][i];
        if (team_size == 1) __syncwarp();
        else tc::named_barrier(1 + team, 32 * team_size);
        const int rows = static_cast<int>(dense ? a.d_rows : a.r_rows);
        const int row = strip * kOut + out_r;
        if (row < rows) {
            T* out = static_cast<T*>(dense ? a.d_out : a.r_out) + row;
            const float* from = sums + out_r * kM;
            for (int n = out_n; n < count; n += 32 / kOut * team_size) {
                float v = 0.0f, u = 0.0f;
                for (int w = 0; w < team_size; ++w) {
                    v += from[w * kRedFloats + n];
                    if constexpr (GLU) u += from[w * kRedFloats + kRows * kM + n];
                }
                const int64_t to = dense ? start + n : blocks.list[start + n];
                v *= unit<T, G>();
                if constexpr (GLU) {
                    // silu(gate) up, times the row's share of the block's output: float32 up to the one rounding
                    v = v * sigmoid_f(v) * (u * unit<T, G>());
                    if (dense) {
                        if (a.d_gate32 != nullptr) v *= sigmoid_f(a.d_gate32[to]);
                        else if (a.d_gate != nullptr) v *= sigmoid_f(to_f32(static_cast<const T*>(a.d_gate)[to]));
                    } else if (a.weights != nullptr) {
                        v *= a.weights[to];
                    }
                }
                const T first = from_f32<T>(v);
                if (GLU && sizeof(T) == 2 && a.pieces) {
                    out[2 * to * rows] = first;
                    out[(2 * to + 1) * rows] = from_f32<T>(v - to_f32(first));
                } else {
                    out[to * rows] = first;
                }
            }
        }
        if (team_size == 1) __syncwarp();
    }
    pdl_release();
    ring.drain(lane);
}

// ---- down products and the combine of a MoE block, at most 64 tokens
//
// A job is two strips of the output. Its columns are one long sum: the shared expert's hidden values, then each chosen
// expert's, in blocks of at most 8 rows of h (the pairs of one expert). There are few jobs (a hidden size of 2560: 80),
// so all jobs' tiles in a row are cut into one even range for each CTA, and a CTA's range of a job into one for each
// warp. A warp adds a block's sums into its own copy of the result in shared memory when the block ends, each row of h to
// its token; a CTA adds its warps' in order, and the last CTA of a job to come adds the CTAs' in order.
//
// float16: h lies in two pieces of float16 (11 + 11 bits, down to 2^-25), because rounding it once would leave the block's
// result with 1.4 times the error of its own rounding. A block is then four rows of h, their first pieces in columns 0 .. 3 of the
// MMAs and their second in 4 .. 7: no more instructions than eight rows.

template <typename T>
__host__ __device__ constexpr int down_rows() { return sizeof(T) == 2 ? kM / 2 : kM; }

// Tiles of a CTA up to which it keeps to one job (whole blocks of 256 experts of 1536 x 4096: one token, 64 tiles, 43.9 us by
// job and 45.8 in even ranges; five tokens, some 250 tiles, 107.8 and 106.9; 32 tokens of the 512-expert block 172.0 and 168.5)
constexpr int kByJob = 64;
constexpr int kTokenStride = kMt * kRows + 4;  // floats of a token's sums: rows 0, 8, .. of four tokens on 32 banks

template <int G>
__host__ __device__ constexpr size_t down_smem(int64_t tokens, int64_t pairs, int64_t experts) {
    return size_t(kWarps) * kStages * slot_bytes<G>() + size_t(kWarps) * tokens * kTokenStride * 4 +
           pair_blocks_bytes(pairs, experts) + size_t(kWarps) * kStages * 8;
}

template <typename T, int G>
__global__ void __launch_bounds__(kThreads, kCtas) q4_down_kernel(const DownArgs a) {
    constexpr int kTile = tile_bytes<G>();
    constexpr int kSlot = slot_bytes<G>();
    constexpr int kRowsIn = down_rows<T>(), kPieces = kM / kRowsIn;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int warp_sums[kWarps];
    __shared__ uint32_t arrived;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int strips = a.strips, jobs = a.jobs;
    const int tokens = static_cast<int>(a.tokens), k = static_cast<int>(a.k), pairs = tokens * k;

    float* red = reinterpret_cast<float*>(smem + size_t(kWarps) * kStages * kSlot);  // [warp][token][row]
    uint8_t* table = reinterpret_cast<uint8_t*>(red + kWarps * tokens * kTokenStride);
    uint64_t* bars = reinterpret_cast<uint64_t*>(table + pair_blocks_bytes(pairs, a.experts));
    RingOf<T> ring;
    ring.init(smem + size_t(warp) * kStages * kSlot, bars + warp * kStages, lane, blockIdx.x == 0 && warp == 0 ? a.withhold : 0);
    const uint64_t policy = tc::policy_evict_first();
    float* mine = red + warp * tokens * kTokenStride;

    if (!a.early) pdl_wait();
    const PairBlocks blocks = pair_blocks(table, a.idx, pairs, static_cast<int>(a.experts), kRowsIn, warp_sums);
    // segments of a job: the shared expert's blocks of tokens, then the pairs' blocks
    const int stiles = a.stiles, ftiles = a.ftiles;
    const int sblocks = stiles > 0 ? (tokens + kRowsIn - 1) / kRowsIn : 0;
    const int shared_items = sblocks * stiles;
    const int items = max(1, shared_items + blocks.n * ftiles);  // (a job without any tile still writes its zeros)
    const bool any = shared_items + blocks.n > 0;
    // a CTA's tiles of all jobs': an even share in a row, at least a tile a warp (32 bits hold them: the host checks); or
    // with few tiles an even share of one job (a second job's end would cost the CTA more than the uneven load)
    const int all = jobs * items;
    const int parts = int(gridDim.x) / jobs;  // CTAs of a job
    const bool by_job = parts > 0 && items <= parts * kByJob;
    const int share = by_job ? max(min(kWarps, items), (items + parts - 1) / parts)
                             : max(min(kWarps, all), (all + int(gridDim.x) - 1) / int(gridDim.x));
    int begin, end;
    if (by_job) {
        const int job = blockIdx.x / parts, part = blockIdx.x - job * parts;
        begin = job < jobs ? job * items + min(items, part * share) : all;
        end = job < jobs ? min(begin + share, (job + 1) * items) : all;
    } else {
        begin = min(all, int(blockIdx.x) * share);
        end = min(all, begin + share);
    }
    const int job_first = begin / items, job_last = begin < end ? (end + items - 1) / items : job_first;

    // a warp's tiles of a job
    auto range_of = [&](int job, int& i0, int& i1) {
        const int at = job * items;
        const int p0 = max(begin, at) - at, n = min(end, at + items) - at - p0;
        i0 = p0 + warp * n / kWarps;
        i1 = p0 + (warp + 1) * n / kWarps;
        if (!any) i0 = i1 = 0;
    };
    // a warp's place in a job: the tiles still to come, from tile `tile` of segment `seg` on
    struct Cursor {
        int left, seg, tile;
    };
    auto cursor_of = [&](int job) {
        int i0, i1;
        range_of(job, i0, i1);
        Cursor c{i1 - i0, 0, i0};
        if (i0 < shared_items) {
            c.seg = a.by_stiles(i0);
            c.tile = i0 - c.seg * stiles;
        } else {
            i0 -= shared_items;
            c.seg = a.by_ftiles(i0);
            c.tile = i0 - c.seg * ftiles;
            c.seg += sblocks;
        }
        return c;
    };
    // its tiles of the segment it is in
    auto tiles_of = [&](const Cursor& c) { return min(c.left, (c.seg < sblocks ? stiles : ftiles) - c.tile); };
    auto next_segment = [&](Cursor& c, int n) {
        c.left -= n;
        c.tile = 0;
        ++c.seg;
    };

    int fetch_job = job_first;
    Cursor fc = job_first < job_last ? cursor_of(fetch_job) : Cursor{0, 0, 0};
    const uint8_t *fetch0 = nullptr, *fetch1 = nullptr;
    auto fetch = [&]() {  // (a slot is free)
        if (ring.left == 0) {
            if (ring.dead) return;
            while (fc.left == 0) {
                if (fetch_job + 1 >= job_last) return;
                fc = cursor_of(++fetch_job);
            }
            const bool shared = fc.seg < sblocks;
            const int64_t strip_bytes = int64_t(shared ? stiles : ftiles) * kTile;
            const uint8_t* w = shared ? a.sw : a.w + int64_t(blocks.expert[fc.seg - sblocks]) * strips * strip_bytes;
            fetch0 = w + (fetch_job * kMt) * strip_bytes + int64_t(fc.tile) * kTile;
            fetch1 = w + min(fetch_job * kMt + 1, strips - 1) * strip_bytes + int64_t(fc.tile) * kTile;
            ring.left = tiles_of(fc);
            next_segment(fc, ring.left);
        }
        const int n = min(kStep, ring.left);
        ring.template fetch<kSlot>(fetch0, fetch1, n * kTile, policy);
        fetch0 += n * kTile;
        fetch1 += n * kTile;
        ring.left -= n;
    };
    for (int i = 0; i < kStages; ++i) fetch();
    pdl_wait();

    const Ones<T> one;
    for (int job = job_first; job < job_last; ++job) {
        for (int i = lane; i < tokens * kTokenStride; i += 32) mine[i] = 0.0f;
        __syncwarp();
        float acc[kMt][4] = {};
        for (Cursor c = cursor_of(job); c.left > 0;) {
            const bool shared = c.seg < sblocks;
            const int start = shared ? c.seg * kRowsIn : blocks.start[c.seg - sblocks];
            const int count = shared ? min(kRowsIn, tokens - start) : blocks.count[c.seg - sblocks];
            const int64_t width = shared ? a.sffn : a.ffn;
            const int row = g % kRowsIn, of = row < count ? start + row : start;
            const T* xp = static_cast<const T*>(shared ? a.hs : a.h) +
                          ((shared ? of : blocks.list[of]) * kPieces + g / kRowsIn) * width + c.tile * kCols + 8 * t;
            const int n = tiles_of(c);
            stream_tiles<T, G>(ring, fetch, xp, n, static_cast<int>(width / 32) - 4 * c.tile, lane, acc, one);
            next_segment(c, n);
            // (one token: blocks of one row of h in a row are one sum. An expert that the token names twice has a block of more
            // rows: the sums before it end here, whose other columns hold copies, and so do its own.)
            if (tokens == 1 && c.left > 0 && count == 1 && (c.seg < sblocks || blocks.count[c.seg - sblocks] == 1)) continue;
            // each column's sums to its token, this lane's columns 2 t and 2 t + 1 (with pieces, those of columns 2 t + 4
            // and 2 t + 5 added). A token that names an expert twice has two columns here, neighbours: column by column then.
            if constexpr (kPieces == 2) {
#pragma unroll
                for (int m = 0; m < kMt; ++m)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[m][i] += __shfl_xor_sync(0xffffffffu, acc[m][i], 2);
            }
            auto token_of = [&](int col) { return shared ? start + col : a.by_k(blocks.list[start + col]); };
            auto add = [&](int h) {
                float* to = mine + token_of(2 * t + h) * kTokenStride + g;
#pragma unroll
                for (int m = 0; m < kMt; ++m) {
                    to[m * kRows] += acc[m][h];
                    to[m * kRows + 8] += acc[m][2 + h];
                }
            };
            const bool again = !shared && lane + 1 < count && token_of(lane) == token_of(lane + 1);
            if (__any_sync(0xffffffffu, again)) {
                for (int col = 0; col < count; ++col) {
                    if (col == 2 * t) add(0);
                    if (col == 2 * t + 1) add(1);
                    __syncwarp();
                }
            } else {
                if (2 * t < count) add(0);
                if (2 * t + 1 < count) add(1);
            }
            __syncwarp();
#pragma unroll
            for (int m = 0; m < kMt; ++m)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[m][i] = 0.0f;
        }
        __syncthreads();
        const int at = job * items;
        const bool whole = begin <= at && end >= at + items;
        const int values = kMt * kRows * tokens;
        auto write = [&](int i, float sum) {
            const int64_t row = int64_t(job) * kMt * kRows + (i & (kMt * kRows - 1));
            if (row < a.rows) static_cast<T*>(a.out)[i / (kMt * kRows) * a.rows + row] = from_f32<T>(sum * unit<T, G>());
        };
        // (a job that a CTA shares is the first or the last of its range)
        float* part = a.partial + (int64_t(blockIdx.x) * 2 + (job == job_first ? 0 : 1)) * values;
        for (int i = tid; i < values; i += kThreads) {
            float sum = 0.0f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w)
                sum += red[(w * tokens + i / (kMt * kRows)) * kTokenStride + (i & (kMt * kRows - 1))];
            if (whole) write(i, sum);
            else part[i] = sum;
        }
        if (!whole) {
            // the CTAs of this job: those whose ranges meet it
            const int c0 = by_job ? job * parts : at / share;
            const int c1 = by_job ? c0 + (items - 1) / share : (at + items - 1) / share;
            __threadfence();
            __syncthreads();
            if (tid == 0) arrived = atomicAdd(&a.counters[job], 1u);
            __syncthreads();
            if (arrived == uint32_t(c1 - c0)) {
                __threadfence();
                for (int i = tid; i < values; i += kThreads) {
                    float sum = 0.0f;
                    for (int cta = c0; cta <= c1; cta += 8) {
                        // (eight CTAs' sums in flight together, added in their order)
                        float v[8];
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const int from = 2 * min(cta + j, c1) + (by_job || (cta + j) * share >= at ? 0 : 1);
                            v[j] = __ldcg(a.partial + int64_t(from) * values + i);  // (its range begins in this job, or before)
                        }
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            if (cta + j <= c1) sum += v[j];
                    }
                    write(i, sum);
                }
            }
        }
        __syncthreads();
    }
    pdl_release();
    ring.drain(lane);
}

}  // namespace q4
}  // namespace smoe
