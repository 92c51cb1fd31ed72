// GQA decode with 4-bit caches, head dim 256: every group size it takes.
#include "pa_kernels_int4.h"

namespace simpler_hip {
namespace pa {

KernelPair pick_int4_d256(int groups, int rows, int out_dtype) {
    switch (groups) {
        case 2: return int4_pair<256, 2>(rows, out_dtype);
        case 4: return int4_pair<256, 4>(rows, out_dtype);
        default: return KernelPair{};
    }
}

DirectFn pick_int4_direct_d256(int groups, int rows, int out_dtype) {
    switch (groups) {
        case 2: return int4_direct<256, 2>(rows, out_dtype);
        case 4: return int4_direct<256, 4>(rows, out_dtype);
        default: return DirectFn{};
    }
}

}  // namespace pa
}  // namespace simpler_hip
