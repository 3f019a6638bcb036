// Host side of the streaming kernels on 4-bit weights: picks the instance and launches it. Included by one source
// file per kernel and activation type.
#pragma once

#include <algorithm>

#include "q4_mv.cuh"

namespace smoe {
namespace q4 {

constexpr int kSms = 148;
constexpr int kDownCtas = kSms * kCtas;

int product_f16(const ProductArgs& a, int group, const Writes& w, cudaStream_t st);
int product_f32(const ProductArgs& a, int group, const Writes& w, cudaStream_t st);
int down_f16(const DownArgs& a, int group, const Writes& w, cudaStream_t st);
int down_f32(const DownArgs& a, int group, const Writes& w, cudaStream_t st);
// the dense part of `a` on the prompt's kernel (float16, floats: with float32 results), and whether that is the faster one
bool matmul_better(int64_t tokens, int64_t rows, int64_t cols);
int matmul_f16(const ProductArgs& a, int group, bool floats, const Writes& w, cudaStream_t st);
// the prompt's kernel on a stack, its activations x in tiles of 16 slots, each one expert's
struct TileArgs {
    const uint8_t* w;
    int64_t experts, rows, cols, tiles;
    const void *x, *plan;
    const uint32_t* slot_row;
    int64_t out_rows;
    void* out;
    bool floats;
};
int tile_plan(const uint32_t* tile_expert, int64_t tiles, int64_t experts, void* plan, const Writes& w, cudaStream_t st);
int tile_matmul(const TileArgs& p, int group, const Writes& w, cudaStream_t st);
int wait_test();  // what smoe_q4_wait_test was last given, 0 or 1
cudaError_t matmul_status(int* v, bool clear);
cudaError_t product_status_f16(int* v, bool clear);
cudaError_t product_status_f32(int* v, bool clear);
cudaError_t down_status_f16(int* v, bool clear);
cudaError_t down_status_f32(int* v, bool clear);

inline cudaError_t read_status(int* v, bool clear) {
    cudaError_t e = cudaMemcpyFromSymbol(v, g_q4_status, sizeof(int));
    if (e == cudaSuccess && clear) {
        const int zero = 0;
        e = cudaMemcpyToSymbol(g_q4_status, &zero, sizeof(int));
    }
    return e;
}

inline int status_of(cudaError_t e, const char* what) {
    if (e == cudaSuccess) return launch_status(what);
    cudaGetLastError();
    set_error(std::string(what) + ": " + cudaGetErrorString(e));
    return -static_cast<int>(e);
}

// Warps that share a job's columns, as a power of two: the count with the least work for the busiest warp, a job's end
// taken as the work of two tiles.
inline int team_log_for(int64_t jobs, int64_t tiles) {
    int best = 0;
    int64_t least = 0;
    for (int log = 0; (1 << log) <= kWarps; ++log) {
        const int w = 1 << log;
        const int64_t teams = int64_t(kSms) * kCtas * kWarps / w;
        const int64_t work = (jobs + teams - 1) / teams * ((tiles + w - 1) / w + 2);
        if (w == 1 || work < least) {
            best = log;
            least = work;
        }
    }
    return best;
}

template <typename T, int G, bool GLU>
inline int launch_product(const ProductArgs& args, const Writes& w, cudaStream_t st) {
    ProductArgs a = args;
    a.withhold = wait_test();
    constexpr int kWide = GLU ? 1 : 2;
    a.tiles = static_cast<int>(tiles_of_cols(a.cols));
    a.runs = static_cast<int>(a.cols / 32);
    a.d_strips = static_cast<int>(strips_of_rows(a.d_rows));
    a.r_strips = static_cast<int>(strips_of_rows(a.r_rows));
    a.d_wide = (a.d_strips + kWide - 1) / kWide;
    a.r_wide = (a.r_strips + kWide - 1) / kWide;
    a.d_blocks = static_cast<int>((a.d_tokens + kM - 1) / kM);
    a.by_dense = Divisor(std::max(1, a.d_blocks));
    a.by_share = Divisor(static_cast<int>(a.share));
    const int64_t jobs = int64_t(a.d_wide) * a.d_blocks + a.r_wide * std::min(a.pairs, a.experts + a.pairs / kM);
    // (a dense matrix's by its shape alone: a token's sums are split alike alone and in a window)
    a.team_log = team_log_for(a.pairs > 0 ? jobs : a.d_wide, a.tiles);
    const size_t smem = product_smem<G>(a.pairs, a.experts);
    if (int e = max_smem(q4_product_kernel<T, G, GLU>, static_cast<int>(smem)))
        return status_of(static_cast<cudaError_t>(-e), "q4_product");
    // (a team's CTA of its own while there are slots for it: the teams spread evenly over the SMs)
    const int64_t ctas = std::min<int64_t>(jobs, kSms * kCtas);
    return status_of(launch_pdl(w, q4_product_kernel<T, G, GLU>, dim3(static_cast<unsigned>(ctas)), dim3(kThreads), smem,
                                st, a), "q4_product");
}

template <typename T>
inline int product(const ProductArgs& a, int group, const Writes& w, cudaStream_t st) {
    const bool glu = a.dw[1] != nullptr || a.rw[1] != nullptr;
    auto go = [&](auto g) {
        constexpr int G = decltype(g)::value;
        return glu ? launch_product<T, G, true>(a, w, st) : launch_product<T, G, false>(a, w, st);
    };
    if (group == 32) return go(std::integral_constant<int, 32>{});
    if (group == 64) return go(std::integral_constant<int, 64>{});
    return go(std::integral_constant<int, 128>{});
}

template <typename T, int G>
inline int launch_down(const DownArgs& args, const Writes& w, cudaStream_t st) {
    DownArgs a = args;
    a.withhold = wait_test();
    a.stiles = static_cast<int>(tiles_of_cols(a.sffn));
    a.ftiles = static_cast<int>(tiles_of_cols(a.ffn));
    a.strips = static_cast<int>(strips_of_rows(a.rows));
    a.jobs = (a.strips + kMt - 1) / kMt;
    a.by_k = Divisor(static_cast<int>(a.k));
    a.by_stiles = Divisor(std::max(1, a.stiles));
    a.by_ftiles = Divisor(a.ftiles);
    const size_t smem = down_smem<G>(a.tokens, a.tokens * a.k, a.experts);
    if (int e = max_smem(q4_down_kernel<T, G>, static_cast<int>(smem))) return status_of(static_cast<cudaError_t>(-e), "q4_moe");
    return status_of(launch_pdl(w, q4_down_kernel<T, G>, dim3(kDownCtas), dim3(kThreads), smem, st, a), "q4_moe");
}

template <typename T>
inline int down(const DownArgs& a, int group, const Writes& w, cudaStream_t st) {
    auto go = [&](auto g) {
        constexpr int G = decltype(g)::value;
        return launch_down<T, G>(a, w, st);
    };
    if (group == 32) return go(std::integral_constant<int, 32>{});
    if (group == 64) return go(std::integral_constant<int, 64>{});
    return go(std::integral_constant<int, 128>{});
}

}  // namespace q4
}  // namespace smoe
