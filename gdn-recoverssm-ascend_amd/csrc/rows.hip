// Host checks of the prompt and plain decode entry points.
#include "rows.cuh"

namespace gdn {

static bool no(int *status, int code) {
  *status = code;
  return false;
}

bool check_row_pages(const char *what, const gdn_row_pages &p, int *status) {
  if (p.rows < 0 || p.tokens < 0 || p.blocks < 1 || p.rows > (1 << 24) || p.tokens > 0x3fffffff) {
    set_error("%s: rows=%lld tokens=%lld blocks=%lld", what, (long long)p.rows, (long long)p.tokens,
              (long long)p.blocks);
    return no(status, GDN_ERR_INVALID);
  }
  if (!index_type(p.qsl_dtype) || !index_type(p.si_dtype) || (p.final_indices && !index_type(p.final_dtype)) ||
      (p.num_computed && !index_type(p.computed_dtype)) || (p.request_indices && !index_type(p.map_dtype)) ||
      (p.block_table && !index_type(p.table_dtype))) {
    set_error("%s: offsets, indices, lengths and the block table must be int32 or int64", what);
    return no(status, GDN_ERR_UNSUPPORTED);
  }
  if (p.block_table && (!p.num_computed || p.final_indices || p.block_size < 1 || p.table_width < 1 ||
                        p.table_rows < 0 || p.block_size > (1 << 30))) {
    set_error("%s: a block table needs num_computed, a positive block size and width, and no final indices", what);
    return no(status, GDN_ERR_INVALID);
  }
  if (p.num_computed && p.computed_len < 0) {
    set_error("%s: negative computed_len", what);
    return no(status, GDN_ERR_INVALID);
  }
  if (p.rows > 0 && p.tokens > 0 && (!p.query_start_loc || !p.state_indices)) {
    set_error("%s: null offsets or state indices", what);
    return no(status, GDN_ERR_INVALID);
  }
  return true;
}

bool check_rule(const char *what, const gdn_rule_launch *l, int *status) {
  if (!l) {
    set_error("%s: missing launch", what);
    return no(status, GDN_ERR_INVALID);
  }
  if (!check_row_pages(what, l->pages, status)) return false;
  const int64_t H = l->heads, HV = l->value_heads, K = l->key_dim, V = l->value_dim;
  if (H < 1 || HV < 1 || HV % H != 0 || HV > 65535 || V < 1 || V > (1 << 20)) {
    set_error("%s: heads=%lld value_heads=%lld value_dim=%lld", what, (long long)H, (long long)HV, (long long)V);
    return no(status, GDN_ERR_INVALID);
  }
  const auto act_or_f32 = [l](int32_t dt) { return dt == l->act_dtype || dt == GDN_DT_F32; };
  if (!float_type(l->act_dtype) || !float_type(l->state_dtype) || !act_or_f32(l->g_dtype) ||
      !act_or_f32(l->beta_dtype) || !act_or_f32(l->out_dtype)) {
    set_error("%s: unsupported dtype combination (gate, beta and out must be FP32 or the activation dtype)", what);
    return no(status, GDN_ERR_UNSUPPORTED);
  }
  const int64_t esz = type_bytes(l->state_dtype), E = 16 / esz;
  if (K < 1 || K > 256 || K % E != 0 || l->state_v_stride < K || l->state_v_stride % E != 0 ||
      l->state_head_stride % E != 0 || l->state_block_stride % E != 0 ||
      l->state_v_stride * V * esz >= 0x70000000LL || (reinterpret_cast<uintptr_t>(l->state) & 15u) != 0) {
    set_error("%s: state layout K=%lld V=%lld unsupported (K <= 256 and a multiple of %lld, 16-byte aligned rows)",
              what, (long long)K, (long long)V, (long long)E);
    return no(status, GDN_ERR_UNSUPPORTED);
  }
  if (l->gating && (!float_type(l->gating->a_log_dtype) || !float_type(l->gating->dt_bias_dtype) ||
                    !(l->gating->softplus_beta > 0.0f))) {
    set_error("%s: gating needs FP32/BF16/F16 A_log and dt_bias and a positive softplus beta", what);
    return no(status, GDN_ERR_UNSUPPORTED);
  }
  if (l->pages.rows > 0 && l->pages.tokens > 0 &&
      (!l->q || !l->k || !l->v || !l->g || !l->beta || !l->out || !l->state ||
       (l->gating && (!l->a_log || !l->dt_bias)))) {
    set_error("%s: null tensor pointer", what);
    return no(status, GDN_ERR_INVALID);
  }
  return true;
}

}  // namespace gdn
