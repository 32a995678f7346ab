// The recurrent rule's kernels for F32 pages.
#include "decode_kernel.cuh"

namespace gdn {
GDN_DECODE_STATE(float)
}
