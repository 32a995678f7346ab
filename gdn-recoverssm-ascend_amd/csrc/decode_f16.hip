// The recurrent rule's kernels for F16 pages.
#include "decode_kernel.cuh"

namespace gdn {
GDN_DECODE_STATE(f16)
}
