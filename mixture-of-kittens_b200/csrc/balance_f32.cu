// The row kernels of the routing losses for f32 logits.
#include "balance_rows.cuh"

namespace mok {
namespace balance {

int rows_f32(const BalanceParams& p, cudaStream_t s) { return launch_rows_for<float>(p, s); }
int backward_f32(const BalanceBwdParams& p, cudaStream_t s) { return launch_bwd_for<float>(p, s); }

}  // namespace balance
}  // namespace mok
