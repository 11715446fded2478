// linear_to_bf16.hip — the kernels of linear_direct.hpp that write bf16 (a file of their own: they take
// long to compile).
#include "linear_direct.hpp"

namespace ttp {

void launch_direct_to_bf16(LinearShape shape, bool transposed, uint32_t blocks, hipStream_t stream,
                           const LinearArgs& a) {
    launch_direct<uint16_t>(shape, transposed, blocks, stream, a);
}

}  // namespace ttp
