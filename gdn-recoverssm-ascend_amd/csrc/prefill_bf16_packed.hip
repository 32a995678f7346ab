// The chunked rule's kernels: activation type, planes of K and Q, planes of the
// output's products, K and Q packed by prepare.
#include "prefill_kernel.cuh"

namespace gdn {
GDN_PREFILL(bf16, 2, 2, true)
}
