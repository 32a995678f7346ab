// C entry points of the chunked gated delta rule: checks, workspace, dispatch
// (kernels in prefill_kernel.cuh, instantiated in prefill_*.hip).
#include "prefill_kernel.cuh"

namespace gdn {

struct PrefillPlan {
  int kp, pl, opl, nv;
  bool pack;
  int64_t bytes, scan_grid;
};

static bool plan_prefill(const gdn_rule_launch *l, PrefillArgs &a, PrefillPlan &p, int *status) {
  const gdn_row_pages &rp = l->pages;
  const int64_t K = l->key_dim, V = l->value_dim, H = l->heads, HV = l->value_heads;
  a.pages = rp;
  a.q = l->q, a.k = l->k, a.v = l->v, a.g = l->g, a.beta = l->beta, a.out = l->out, a.state = l->state;
  a.a_log = l->a_log, a.dt_bias = l->dt_bias;
  a.gated = l->gating != nullptr;
  if (l->gating) a.gating = *l->gating;
  a.q_ts = l->q_stride, a.k_ts = l->k_stride, a.v_ts = l->v_stride;
  a.g_ts = l->g_stride, a.beta_ts = l->beta_stride, a.out_ts = l->out_stride;
  a.state_bs = l->state_block_stride, a.state_hs = l->state_head_stride, a.state_vs = l->state_v_stride;
  a.K = int32_t(K), a.V = int32_t(V), a.H = int32_t(H), a.HV = int32_t(HV), a.ratio = int32_t(HV / H);
  a.g_dt = l->g_dtype, a.beta_dt = l->beta_dtype, a.state_dt = l->state_dtype;
  a.out_f32 = l->out_dtype == GDN_DT_F32, a.l2norm = l->qk_l2norm, a.scale = l->scale;
  // A row of n tokens spans at most n * per_block / block + 3 chunks wherever it
  // starts, and ceil(n / 64) where chunks start with the row.
  a.align = rp.block_table != nullptr;
  a.block = a.align ? int32_t(rp.block_size) : kChunk;
  a.per_block = (a.block + kChunk - 1) / kChunk;
  a.slack = a.align ? 3 : 1;
  const int64_t slots = rp.tokens * a.per_block / a.block + a.slack * rp.rows;
  p.kp = K <= 64 ? 64 : K <= 128 ? 128 : 256;
  // BF16 keys are read in place as operands where every 8 of them start on a
  // dword; else, and for wider types, prepare packs them as planes.
  const bool rows_of_dwords = K % 8 == 0 && l->q_stride % 2 == 0 && l->k_stride % 2 == 0 &&
                              (reinterpret_cast<uintptr_t>(l->q) | reinterpret_cast<uintptr_t>(l->k)) % 4 == 0;
  const bool exact_out = a.out_f32 || l->act_dtype == GDN_DT_F32;
  p.pack = exact_out || l->act_dtype != GDN_DT_BF16 || !rows_of_dwords;
  p.pl = exact_out ? 3 : p.pack ? 2 : 1;
  p.opl = exact_out ? 3 : 2;
  int64_t at = 0;
  const auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += bytes;
    return here;
  };
  const int64_t key_planes = slots * H * 4 * (p.kp / 32) * p.pl * kFrag;
  a.kt_at = take(key_planes);
  a.k_at = take(p.pack ? key_planes : 0);
  a.q_at = take(p.pack ? key_planes : 0);
  a.t_at = take(slots * HV * 8 * kPlanesT * kFrag);
  a.p_at = take(slots * HV * 8 * p.opl * kFrag);
  a.s_at = take(slots * HV * kScalars * 4);
  p.bytes = at;
  const int64_t wide = rp.rows * HV * ((V + 31) / 32);
  p.nv = wide >= 512 ? 2 : 1;
  a.slices = int32_t((V + 16 * p.nv - 1) / (16 * p.nv));
  a.members = a.ratio * a.slices;
  p.scan_grid = (rp.rows * H + 7) / 8 * 8 * a.members;
  if (slots * H > 0x7fffffffLL || p.scan_grid > 0x7fffffffLL || rp.rows * H > 0x7fffffffLL) {
    set_error("prefill: grid too large");
    *status = GDN_ERR_UNSUPPORTED;
    return false;
  }
  a.slots = int32_t(slots);
  return true;
}

}  // namespace gdn

using namespace gdn;

extern "C" int64_t gdn_recoverssm_prefill_workspace(const gdn_rule_launch *l) {
  int status = GDN_OK;
  PrefillArgs a{};
  PrefillPlan p{};
  if (!check_rule("prefill", l, &status)) return -1;
  if (l->pages.rows == 0 || l->pages.tokens == 0) return 0;
  return plan_prefill(l, a, p, &status) ? p.bytes : -1;
}

extern "C" int gdn_recoverssm_prefill(const gdn_rule_launch *l, void *workspace, int64_t workspace_bytes,
                                      void *stream) {
  int status = GDN_OK;
  PrefillArgs a{};
  PrefillPlan p{};
  if (!check_rule("prefill", l, &status)) return status;
  if (l->pages.rows == 0 || l->pages.tokens == 0) return GDN_OK;
  if (!plan_prefill(l, a, p, &status)) return status;
  if (!workspace || workspace_bytes < p.bytes || (reinterpret_cast<uintptr_t>(workspace) & 15u) != 0) {
    set_error("prefill: a 16-byte aligned workspace of %lld bytes is required, %lld given", (long long)p.bytes,
              (long long)(workspace ? workspace_bytes : 0));
    return GDN_ERR_INVALID;
  }
  a.ws = static_cast<char *>(workspace);
  auto s = static_cast<hipStream_t>(stream);
  const unsigned grid = unsigned(p.scan_grid);
  if (p.pl == 1) launch_prefill<bf16, 1, 2, false>(p.kp, p.nv, grid, s, a);
  else if (l->act_dtype == GDN_DT_F32) launch_prefill<float, 3, 3, true>(p.kp, p.nv, grid, s, a);
  else if (l->act_dtype == GDN_DT_F16 && p.pl == 2) launch_prefill<f16, 2, 2, true>(p.kp, p.nv, grid, s, a);
  else if (l->act_dtype == GDN_DT_F16) launch_prefill<f16, 3, 3, true>(p.kp, p.nv, grid, s, a);
  else if (p.pl == 2) launch_prefill<bf16, 2, 2, true>(p.kp, p.nv, grid, s, a);
  else launch_prefill<bf16, 3, 3, true>(p.kp, p.nv, grid, s, a);
  const hipError_t err = hipGetLastError();
  if (err != hipSuccess) {
    set_error("prefill: launch failed: %s", hipGetErrorString(err));
    return GDN_ERR_LAUNCH;
  }
  return GDN_OK;
}
