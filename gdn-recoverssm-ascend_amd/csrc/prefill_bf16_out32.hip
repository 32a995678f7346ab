// The chunked rule's kernels: types of the activations and of the output.
#include "prefill_kernel.cuh"

namespace gdn {
GDN_PREFILL(bf16, float)
}
