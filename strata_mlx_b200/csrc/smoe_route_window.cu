// The route of a window of tokens (router product, top-k, softmax over the chosen, the shared expert's gate) with its
// sums on the tensor cores, in one launch.
//
//   logits[t, e] = router[e] . x[t];  idx = the k largest, ties to the lower index;  weights = softmax of the chosen;
//   gate_out[t] = gate_weight . x[t], in float32 or rounded to float16
//
// A CTA takes 16 rows of the router (the shared gate's row is one more) and eight tokens: 16 warps share the columns, each
// m16n8k16 on its own (router rows the M side, tokens the N side, products exact, float32 sums), partial sums added in
// the order of the columns. The last CTA of eight tokens to arrive takes their top-k, a warp a token. Bound by latency
// (the router is 2 to 4 MB, read from L2 once for every eight tokens): the rows' first columns are loaded before the
// launch waits for the one before it. With all tokens in one
// CTA a block of 512 experts at 32 tokens took 181 us, with eight 171.
#include <algorithm>
#include <string>

#include "q4.cuh"
#include "router_dev.cuh"

namespace smoe {
namespace {

constexpr int kRwWarps = 16;
constexpr int kRwThreads = 32 * kRwWarps;
constexpr int kRwRows = 16;
constexpr int kRwAhead = 4;   // runs of 32 columns a warp loads before it waits
constexpr int kRwWidth = 8;   // tokens of a CTA
constexpr int kRwTokens = 64;

struct RouteWindow {
    const __half* weight;
    const __half* gate_weight;
    const __half* x;
    int tokens, experts, runs, k;  // runs: hidden / 32
    int64_t hidden;
    float* logits;
    uint32_t* idx;
    float* weights;
    void* gate_out;
    bool gate32;  // gate_out is float32
    uint32_t* counters;  // one for every eight tokens
    bool early;  // the router may be read before pdl_wait()
};

constexpr int kRwStride = kRwRows + 4;  // floats of a token's sums: a warp's writes and reads are on different banks

template <int NV>
__global__ void __launch_bounds__(kRwThreads, NV <= 16 ? 2 : 1) route_window_kernel(const RouteWindow a) {
    __shared__ float part[kRwWarps * kRwWidth * kRwStride];  // [warp][token][row]
    __shared__ bool last;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int row0 = blockIdx.x * kRwRows, rows = a.experts + (a.gate_weight != nullptr);
    const int token0 = blockIdx.y * kRwWidth, tokens = min(kRwWidth, a.tokens - token0);
    const int run0 = warp * a.runs / kRwWarps, run1 = (warp + 1) * a.runs / kRwWarps;
    // this lane's rows g and g + 8 (rows past the last repeat it; their sums are not written), columns 8 t .. of a run
    auto row_of = [&](int r) {
        r = min(r, rows - 1);
        return (r < a.experts ? a.weight + r * a.hidden : a.gate_weight) + 8 * t;
    };
    const __half *wa = row_of(row0 + g), *wb = row_of(row0 + g + 8);
    uint4 ahead[kRwAhead][2];
    if (!a.early) pdl_wait();
#pragma unroll
    for (int i = 0; i < kRwAhead; ++i) {
        const int run = min(run0 + i, a.runs - 1);
        ahead[i][0] = __ldg(reinterpret_cast<const uint4*>(wa + 32 * run));
        ahead[i][1] = __ldg(reinterpret_cast<const uint4*>(wb + 32 * run));
    }
    pdl_wait();
    pdl_release();
    // (columns past the tokens repeat the first one; their sums are not written)
    const __half* xp = a.x + (token0 + (g < tokens ? g : 0)) * a.hidden + 8 * t;
    float acc[4] = {};
    auto step = [&](const uint4& u, const uint4& v, int run) {
        const uint4 x = *reinterpret_cast<const uint4*>(xp + 32 * run);
        q4::mma_f16<false>(acc, u.x, v.x, u.y, v.y, x.x, x.y);
        q4::mma_f16<false>(acc, u.z, v.z, u.w, v.w, x.z, x.w);
    };
#pragma unroll
    for (int i = 0; i < kRwAhead; ++i)
        if (run0 + i < run1) step(ahead[i][0], ahead[i][1], run0 + i);
    for (int run = run0 + kRwAhead; run < run1; ++run)
        step(__ldg(reinterpret_cast<const uint4*>(wa + 32 * run)), __ldg(reinterpret_cast<const uint4*>(wb + 32 * run)), run);
#pragma unroll
    for (int i = 0; i < 4; ++i) part[(warp * kRwWidth + 2 * t + (i & 1)) * kRwStride + g + 8 * (i >> 1)] = acc[i];
    __syncthreads();
    if (threadIdx.x < kRwRows * tokens) {
        const int r = threadIdx.x & (kRwRows - 1), n = threadIdx.x / kRwRows, row = row0 + r;
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < kRwWarps; ++w) sum += part[(w * kRwWidth + n) * kRwStride + r];
        if (row < a.experts) a.logits[(token0 + n) * int64_t(a.experts) + row] = sum;
        else if (row < rows && a.gate32) static_cast<float*>(a.gate_out)[token0 + n] = sum;
        else if (row < rows) static_cast<__half*>(a.gate_out)[token0 + n] = __float2half_rn(sum);
    }
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) last = atomicAdd(&a.counters[blockIdx.y], 1u) == gridDim.x - 1;
    __syncthreads();
    if (!last) return;
    __threadfence();
    if (warp < tokens) {
        const int n = token0 + warp;
        const float* in = a.logits + n * int64_t(a.experts);
        topk_row<NV>([&](int j) { return __ldcg(in + j); }, a.experts, a.k, a.idx + n * a.k, a.weights + n * a.k);
    }
    if (threadIdx.x == 0) a.counters[blockIdx.y] = 0u;
}

int launch(const RouteWindow& a, const Writes& w, cudaStream_t st) {
    auto go = [&](auto kernel) {
        const int rows = a.experts + (a.gate_weight != nullptr);
        const dim3 grid((rows + kRwRows - 1) / kRwRows, (a.tokens + kRwWidth - 1) / kRwWidth);
        const cudaError_t e = launch_pdl(w, kernel, grid, dim3(kRwThreads), 0, st, a);
        if (e == cudaSuccess) return launch_status("route_window");
        cudaGetLastError();
        return fail(-static_cast<int>(e), std::string("route_window: ") + cudaGetErrorString(e));
    };
    if (a.experts <= 256) return go(route_window_kernel<8>);
    if (a.experts <= 512) return go(route_window_kernel<16>);
    if (a.experts <= 1024) return go(route_window_kernel<32>);
    return go(route_window_kernel<64>);
}

int route_window(const uint16_t* weight, const uint16_t* gate_weight, const uint16_t* x, int64_t tokens, int64_t experts,
                 int64_t hidden, int64_t k, float* logits, uint32_t* idx, float* weights, void* gate_out, bool gate32,
                 uint32_t* counters, void* stream) {
    if (tokens == 0) return SMOE_OK;
    SMOE_REQUIRE(weight && x && logits && idx && weights && counters && tokens > 0 && experts > 0, SMOE_EARG,
                 "route_window: null pointer or empty router");
    SMOE_REQUIRE((gate_weight == nullptr) == (gate_out == nullptr), SMOE_EARG,
                 "the shared gate's weight and output come together");
    SMOE_REQUIRE(tokens <= kRwTokens, SMOE_ESHAPE, "route_window takes up to 64 tokens a call");
    SMOE_REQUIRE(hidden > 0 && hidden % 32 == 0 && hidden < (int64_t(1) << 24), SMOE_ESHAPE,
                 "route_window takes rows of a multiple of 32 values");
    SMOE_REQUIRE(experts <= 2048, SMOE_ESHAPE, "route_window takes rows of 1 to 2048 logits");
    SMOE_REQUIRE(k >= 1 && k <= experts && k <= 32, SMOE_ESHAPE, "route_window takes 1 <= k <= min(experts, 32)");
    SMOE_REQUIRE(((reinterpret_cast<uintptr_t>(weight) | reinterpret_cast<uintptr_t>(x) |
                   reinterpret_cast<uintptr_t>(gate_weight)) & 15) == 0,
                 SMOE_EARG, "router weights and activations must be 16-byte aligned");
    cudaStream_t st = as_stream(stream);
    RouteWindow a = {};
    a.weight = reinterpret_cast<const __half*>(weight);
    a.gate_weight = reinterpret_cast<const __half*>(gate_weight);
    a.x = reinterpret_cast<const __half*>(x);
    a.tokens = static_cast<int>(tokens);
    a.experts = static_cast<int>(experts);
    a.runs = static_cast<int>(hidden / 32);
    a.k = static_cast<int>(k);
    a.hidden = hidden;
    a.logits = logits;
    a.idx = idx;
    a.weights = weights;
    a.gate_out = gate_out;
    a.gate32 = gate32;
    a.counters = counters;
    a.early = pdl_early(st, weight, size_t(experts) * hidden * 2) && pdl_early(st, gate_weight, size_t(hidden) * 2);
    Writes w;
    w.add(logits, size_t(tokens) * experts * 4).add(idx, size_t(tokens) * k * 4).add(weights, size_t(tokens) * k * 4);
    w.add(gate_out, size_t(tokens) * (gate32 ? 4 : 2)).add(counters, size_t(tokens + 7) / 8 * 4);
    return launch(a, w, st);
}

}  // namespace
}  // namespace smoe

using namespace smoe;

extern "C" int smoe_route_window(const uint16_t* weight, const uint16_t* gate_weight, const uint16_t* x, int64_t tokens,
                                 int64_t experts, int64_t hidden, int64_t k, float* logits, uint32_t* idx, float* weights,
                                 uint16_t* gate_out, uint32_t* counters, void* stream) try {
    return route_window(weight, gate_weight, x, tokens, experts, hidden, k, logits, idx, weights, gate_out, false, counters,
                        stream);
} catch (...) {
    return fail(SMOE_EARG, "route_window: the host is out of memory");
}

extern "C" int smoe_route_window_f32(const uint16_t* weight, const uint16_t* gate_weight, const uint16_t* x, int64_t tokens,
                                     int64_t experts, int64_t hidden, int64_t k, float* logits, uint32_t* idx, float* weights,
                                     float* gate_out, uint32_t* counters, void* stream) try {
    return route_window(weight, gate_weight, x, tokens, experts, hidden, k, logits, idx, weights, gate_out, true, counters,
                        stream);
} catch (...) {
    return fail(SMOE_EARG, "route_window: the host is out of memory");
}
