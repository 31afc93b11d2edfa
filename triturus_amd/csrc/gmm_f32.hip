// The products of ragged groups for f32 operands (a file of its own per type: they compile side by side).
#include "gmm_launch.hpp"

namespace trt {

int gmm_f32(const GmmArgs &g, int64_t E, int64_t T_rows, bool weights, bool y_inner, int tile, const Workspace &w, hipStream_t s) {
    return launch_gmm_type<float>(g, E, T_rows, weights, y_inner, tile, w, s);
}

int gmm_grad_f32(const GmmArgs &r, const GmmArgs &w, int64_t E, int64_t T_rows, bool y_inner, const Workspace &ws, hipStream_t s) {
    return launch_gmm_grad_type<float>(r, w, E, T_rows, y_inner, ws, s);
}

}  // namespace trt
