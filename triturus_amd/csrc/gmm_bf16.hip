// The products of ragged groups for bf16 operands (a file of its own per type: they compile side by side).
#include "gmm_launch.hpp"

namespace trt {

int gmm_bf16(const GmmArgs &g, int64_t E, int64_t T_rows, bool weights, bool y_inner, int tile, const Workspace &w, hipStream_t s) {
    return launch_gmm_type<__bf16>(g, E, T_rows, weights, y_inner, tile, w, s);
}

}  // namespace trt
