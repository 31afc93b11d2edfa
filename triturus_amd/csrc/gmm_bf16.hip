// The products of ragged groups for bf16 operands (a file of its own per type: they compile side by side).
#include "gmm_launch.hpp"

namespace trt {

int gmm_bf16(const GmmArgs &g, int64_t E, int64_t T_rows, bool weights, bool y_inner, int tile, const Workspace &w, hipStream_t s) {
    return launch_gmm_type<__bf16>(g, E, T_rows, weights, y_inner, tile, w, s);
}

int gmm_grad_bf16(const GmmArgs &r, const GmmArgs &w, int64_t E, int64_t T_rows, bool y_inner, const Workspace &ws, hipStream_t s) {
    return launch_gmm_grad_type<__bf16>(r, w, E, T_rows, y_inner, ws, s);
}

}  // namespace trt
