// C entry points of the chunked gated delta rule.
#include "rows.cuh"

using namespace gdn;

extern "C" int64_t gdn_recoverssm_prefill_workspace(const gdn_rule_launch *l) {
  int status = GDN_OK;
  return check_rule("prefill", l, &status) ? 0 : -1;
}

extern "C" int gdn_recoverssm_prefill(const gdn_rule_launch *l, void *workspace, int64_t workspace_bytes,
                                      void *stream) {
  return gdn_recoverssm_decode(l, stream);
}
