#include "jx_paged_step.cuh"
namespace jx {
cudaError_t paged_step_e4m3(const PagedArgs& a, int hd, int cols, int num_sms, cudaStream_t st) {
    return step_launch_dt<DT_E4M3>(a, hd, cols, num_sms, st);
}
}  // namespace jx
