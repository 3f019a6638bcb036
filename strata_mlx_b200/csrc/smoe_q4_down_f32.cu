// The down kernel on 4-bit weights (q4_mv.cuh) for float32 activations.
#include "q4_launch.cuh"

namespace smoe {
namespace q4 {

int down_f32(const DownArgs& a, int group, const Writes& w, cudaStream_t st) { return down<float>(a, group, w, st); }
cudaError_t down_status_f32(int* v, bool clear) { return read_status(v, clear); }

}  // namespace q4
}  // namespace smoe
