// The row kernels of the routing losses for bf16 logits.
#include "balance_rows.cuh"

namespace mok {
namespace balance {

int rows_bf16(const BalanceParams& p, cudaStream_t s) { return launch_rows_for<__nv_bfloat16>(p, s); }
int backward_bf16(const BalanceBwdParams& p, cudaStream_t s) { return launch_bwd_for<__nv_bfloat16>(p, s); }

}  // namespace balance
}  // namespace mok
