// The product kernel on 4-bit weights (q4_mv.cuh) for float16 activations.
#include "q4_launch.cuh"

namespace smoe {
namespace q4 {

int product_f16(const ProductArgs& a, int group, const Writes& w, cudaStream_t st) { return product<__half>(a, group, w, st); }
cudaError_t product_status_f16(int* v, bool clear) { return read_status(v, clear); }

}  // namespace q4
}  // namespace smoe
