// linear_to_fp32.hip — the kernels of linear_direct.hpp that write fp32 (a file of their own: they take
// long to compile).
#include "linear_direct.hpp"

namespace ttp {

void launch_direct_to_fp32(LinearShape shape, bool transposed, uint32_t blocks, hipStream_t stream,
                           const LinearArgs& a) {
    launch_direct<float>(shape, transposed, blocks, stream, a);
}

}  // namespace ttp
