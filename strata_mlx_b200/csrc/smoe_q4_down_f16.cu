// The down kernel on 4-bit weights (q4_mv.cuh) for float16 activations.
#include "q4_launch.cuh"

namespace smoe {
namespace q4 {

int down_f16(const DownArgs& a, int group, const Writes& w, cudaStream_t st) { return down<__half>(a, group, w, st); }
cudaError_t down_status_f16(int* v, bool clear) { return read_status(v, clear); }

}  // namespace q4
}  // namespace smoe
