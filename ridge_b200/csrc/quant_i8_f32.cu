// The FP32 instances of the row operators (quant_i8.cuh).
#include "quant_i8.cuh"

namespace ridge_b200 {

cudaError_t run_rows_f32(int op, const RowParams& p, int num_sms, cudaStream_t stream) {
    return run_type<float>(op, p, num_sms, stream);
}

}  // namespace ridge_b200
