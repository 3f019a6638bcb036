// Host side of the streaming kernels on 4-bit weights: picks the instance and launches it. Included by one source
// file per kernel and activation type.
#pragma once

#include <algorithm>

#include "q4_mv.cuh"

namespace smoe {
namespace q4 {

constexpr int kSms = 148;
constexpr int kCtasPerSm = 5;

int product_f16(const ProductArgs& a, int group, const Writes& w, cudaStream_t st);
int product_f32(const ProductArgs& a, int group, const Writes& w, cudaStream_t st);
int down_f16(const DownArgs& a, int group, const Writes& w, cudaStream_t st);
int down_f32(const DownArgs& a, int group, const Writes& w, cudaStream_t st);
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

// launch_pdl with a cluster of `csize` CTAs along x
template <typename Args>
inline cudaError_t launch_cluster(const Writes& writes, void (*kernel)(Args), unsigned ctas, int csize, size_t smem,
                                  cudaStream_t st, const Args& args) {
    const int status = max_smem(kernel, static_cast<int>(smem));
    if (status != 0) return static_cast<cudaError_t>(-status);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned>(csize);
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = csize > 1 ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args);
    pdl_note(st, writes);
    return e;
}

inline int status_of(cudaError_t e, const char* what) {
    if (e == cudaSuccess) return launch_status(what);
    cudaGetLastError();
    set_error(std::string(what) + ": " + cudaGetErrorString(e));
    return -static_cast<int>(e);
}

// CTAs that share a job's columns: as many as keep every SM's slots taken, while each warp has a tile of its own
inline int cluster_for(int64_t jobs, int64_t tiles) {
    int c = 1;
    while (c < 8 && jobs * 2 * c <= kSms * kCtasPerSm && tiles >= 2 * c * kWarps) c *= 2;
    return c;
}

template <typename T, int G, int NT, int MATS>
inline int launch_product(const ProductArgs& args, const Writes& w, cudaStream_t st) {
    ProductArgs a = args;
    const int64_t most = 8 * NT;
    const int64_t jobs = strips_of_rows(a.d_rows) * ((a.d_tokens + most - 1) / most) +
                         strips_of_rows(a.r_rows) * std::min(a.pairs, a.experts + a.pairs / most);
    // (by the shapes alone: a token's sums are split alike alone and in a window)
    const int csize = cluster_for(strips_of_rows(a.d_rows) + strips_of_rows(a.r_rows) * a.share, tiles_of_cols(a.cols));
    a.stages = 4;
    const size_t smem = product_smem<G, NT, MATS>(a.stages, a.pairs, a.experts);
    const int64_t clusters = std::min<int64_t>(jobs, kSms * kCtasPerSm / csize);
    return status_of(launch_cluster(w, q4_product_kernel<T, G, NT, MATS>, static_cast<unsigned>(clusters * csize), csize,
                                    smem, st, a), "q4_product");
}

template <typename T>
inline int product(const ProductArgs& a, int group, const Writes& w, cudaStream_t st) {
    const int64_t rows = std::max(a.d_tokens, a.pairs > 0 ? a.pairs / a.share : 0);
    const bool two = rows > 8;
    const bool glu = a.dw[1] != nullptr || a.rw[1] != nullptr;
    auto go = [&](auto g) {
        constexpr int G = decltype(g)::value;
        if (glu) return two ? launch_product<T, G, 2, 2>(a, w, st) : launch_product<T, G, 1, 2>(a, w, st);
        return two ? launch_product<T, G, 2, 1>(a, w, st) : launch_product<T, G, 1, 1>(a, w, st);
    };
    if (group == 32) return go(std::integral_constant<int, 32>{});
    if (group == 64) return go(std::integral_constant<int, 64>{});
    return go(std::integral_constant<int, 128>{});
}

template <typename T, int G, int NT>
inline int launch_down(const DownArgs& args, const Writes& w, cudaStream_t st) {
    DownArgs a = args;
    const int64_t strips = strips_of_rows(a.rows);
    // (at least one choice a token: a strip's tiles are the shared expert's and k experts' or more)
    const int64_t tiles = tiles_of_cols(a.sffn) + a.k * tiles_of_cols(a.ffn);
    const int csize = cluster_for(strips, tiles);
    a.stages = 8;
    const size_t smem = down_smem<G, NT>(a.stages, a.tokens * a.k, a.experts);
    return status_of(launch_cluster(w, q4_down_kernel<T, G, NT>, static_cast<unsigned>(strips * csize), csize, smem, st, a),
                     "q4_moe");
}

template <typename T>
inline int down(const DownArgs& a, int group, const Writes& w, cudaStream_t st) {
    auto go = [&](auto g) {
        constexpr int G = decltype(g)::value;
        if (a.tokens <= 8) return launch_down<T, G, 1>(a, w, st);
        if (a.tokens <= 16) return launch_down<T, G, 2>(a, w, st);
        if (a.tokens <= 32) return launch_down<T, G, 4>(a, w, st);
        return launch_down<T, G, 8>(a, w, st);
    };
    if (group == 32) return go(std::integral_constant<int, 32>{});
    if (group == 64) return go(std::integral_constant<int, 64>{});
    return go(std::integral_constant<int, 128>{});
}

}  // namespace q4
}  // namespace smoe
