// The recurrent rule's kernels for BF16 pages.
#include "decode_kernel.cuh"

namespace gdn {
GDN_DECODE_STATE(bf16)
}
