// What the prompt and plain decode kernels (decode.hip, prefill*.hip,
// conv.hip) share: a row's tokens and pages (gdn_row_pages), and the host
// checks of them.
#pragma once

#include "gdn_common.cuh"

namespace gdn {

// A row as a kernel sees it. Offsets are clamped to the batch, so whatever the
// device arrays hold no token outside it is touched.
struct Row {
  int bos, n;        // first token, tokens
  int64_t C, req;    // tokens before the row, its request
  int64_t src, fin;  // pages
  bool fresh;        // the state starts at zero
  bool valid;
};

__device__ __forceinline__ int clamp_token(int64_t t, int64_t tokens) {
  return int(t < 0 ? 0 : t > tokens ? tokens : t);
}

// A wave-uniform 64-bit value in scalar registers: 64-bit compares and what
// hangs on them are vector instructions, and a buffer address made by those
// costs a loop at every access.
__device__ __forceinline__ int64_t uniform64(int64_t x) {
  const uint32_t lo = uint32_t(__builtin_amdgcn_readfirstlane(int(uint32_t(uint64_t(x)))));
  const uint32_t hi = uint32_t(__builtin_amdgcn_readfirstlane(int(uint32_t(uint64_t(x) >> 32))));
  return int64_t((uint64_t(hi) << 32) | lo);
}

// The row's words are read at wave-uniform addresses: the four that depend on
// nothing are in flight together, the block table's entry follows.
__device__ __forceinline__ Row load_row(const gdn_row_pages &p, int b) {
  Row r;
  const int64_t lo = load_index_ro(p.query_start_loc, b * p.qsl_stride, p.qsl_dtype);
  const int64_t hi = load_index_ro(p.query_start_loc, (b + 1) * p.qsl_stride, p.qsl_dtype);
  r.src = load_index_ro(p.state_indices, b * p.si_stride, p.si_dtype);
  r.req = p.request_indices ? load_index_ro(p.request_indices, b * p.map_stride, p.map_dtype) : b;
  r.bos = clamp_token(lo, p.tokens);
  r.n = clamp_token(hi, p.tokens) - r.bos;
  r.n = r.n < 0 ? 0 : r.n;
  r.valid = true;
  r.C = 0;
  r.fresh = false;
  if (p.num_computed) {
    const bool known = r.req >= 0 && r.req < p.computed_len;
    r.C = known ? load_index_ro(p.num_computed, r.req * p.computed_stride, p.computed_dtype) : -1;
    // A position no sequence reaches: refused, so that sums below cannot wrap.
    r.valid = r.C >= 0 && r.C < (int64_t(1) << 48);
    r.fresh = r.C == 0;
  }
  r.fin = r.src;
  if (p.block_table) {
    r.valid = r.valid && r.req < p.table_rows;
    int64_t col = (r.C + r.n - 1) / p.block_size;
    col = col < p.table_width ? col : p.table_width - 1;
    r.fin = r.valid && r.n > 0
                ? load_index_ro(p.block_table, r.req * p.table_row_stride + col * p.table_col_stride, p.table_dtype)
                : 0;
  } else if (p.final_indices) {
    r.fin = load_index_ro(p.final_indices, b * p.final_stride, p.final_dtype);
  }
  r.valid = r.valid && r.fin > 0 && r.fin < p.blocks && (r.fresh || (r.src > 0 && r.src < p.blocks));
  r.bos = __builtin_amdgcn_readfirstlane(r.bos);
  r.n = __builtin_amdgcn_readfirstlane(r.n);
  r.C = uniform64(r.C);
  r.req = uniform64(r.req);
  r.src = uniform64(r.src);
  r.fin = uniform64(r.fin);
  r.fresh = __builtin_amdgcn_readfirstlane(int(r.fresh)) != 0;
  r.valid = __builtin_amdgcn_readfirstlane(int(r.valid)) != 0;
  return r;
}

// The page that takes the state after `pos` tokens of the request (pos inside
// the row: C < pos < C + n), 0 for none.
__device__ __forceinline__ int64_t boundary_page(const gdn_row_pages &p, const Row &r, int64_t pos) {
  if (!p.block_table || pos % p.block_size != 0) return 0;
  const int64_t col = pos / p.block_size - 1;
  if (col >= p.table_width) return 0;
  const int64_t page =
      load_index_ro(p.block_table, r.req * p.table_row_stride + col * p.table_col_stride, p.table_dtype);
  return page > 0 && page < p.blocks && page != r.fin ? page : 0;
}

// The last i in [0, count) with key(i) <= at, -1 if there is none, for keys that
// do not fall: each round the wave's lanes test 64 places at once, so up
// to 64 keys take one round trip and 4096 take two.
template <typename Key>
__device__ __forceinline__ int last_not_above(int count, int64_t at, Key key) {
  int lo = 0;
  const int lane = threadIdx.x & 63;
  while (true) {
    const int step = (count + 63) >> 6, i = lane * step;
    const int below = __popcll(__builtin_amdgcn_ballot_w64(i < count && key(lo + (i < count ? i : 0)) <= at));
    if (below == 0) return lo - 1;  // only in the first round: later ones start at a key that is not above
    lo += (below - 1) * step;
    if (step == 1) return lo;
    count = count - (below - 1) * step < step ? count - (below - 1) * step : step;
  }
}

// Row number `at` in an order by length, longest first, within each 64 rows: a
// workgroup that walks a row alone is to start the earlier the longer it takes.
// Whole waves.
__device__ __forceinline__ int row_by_length(const gdn_row_pages &p, int at) {
  if (p.rows == 1) return at;
  const int lane = threadIdx.x & 63, base = at & ~63, row = base + lane;
  const int count = p.rows - base < 64 ? int(p.rows - base) : 64;
  int64_t n = -1;
  if (lane < count)
    n = load_index(p.query_start_loc, (row + 1) * p.qsl_stride, p.qsl_dtype) -
        load_index(p.query_start_loc, row * p.qsl_stride, p.qsl_dtype);
  const int length = n > 0x7fffffff ? 0x7fffffff : n < 0 ? 0 : int(n);
  int rank = 0;
  for (int j = 0; j < count; ++j) {
    const int other = __builtin_amdgcn_readlane(length, j);
    rank += (other > length) | ((other == length) & (j < lane));
  }
  return base + int(__builtin_ctzll(__builtin_amdgcn_ballot_w64(lane < count && rank == at - base)));
}

// Host checks; false after set_error.
bool check_row_pages(const char *what, const gdn_row_pages &p, int *status);
bool check_rule(const char *what, const gdn_rule_launch *l, int *status);

inline bool float_type(int32_t dt) { return dt == GDN_DT_F32 || dt == GDN_DT_BF16 || dt == GDN_DT_F16; }
inline bool index_type(int32_t dt) { return dt == GDN_DT_I32 || dt == GDN_DT_I64; }
inline int64_t type_bytes(int32_t dt) { return dt == GDN_DT_F32 ? 4 : 2; }

// Gates of one token and head as the rule takes them: log decay and beta,
// from the raw projections when the gating is fused.
struct GateParams {
  float neg_exp_a, dt_bias, softplus_beta, softplus_threshold;
  bool gated;
};
__device__ __forceinline__ GateParams load_gates(const void *a_log, const void *dt_bias, const gdn_gating_ext &ext,
                                                 bool gated, int hv) {
  GateParams g{0.0f, 0.0f, 1.0f, 0.0f, gated};
  if (gated) {
    g.neg_exp_a = -expf(load_as_f32(a_log, hv, ext.a_log_dtype));
    g.dt_bias = load_as_f32(dt_bias, hv, ext.dt_bias_dtype);
    g.softplus_beta = ext.softplus_beta;
    g.softplus_threshold = ext.softplus_threshold;
  }
  return g;
}
__device__ __forceinline__ float log_decay(const GateParams &p, float a) {
  if (!p.gated) return a;
  const float x = a + p.dt_bias, sx = p.softplus_beta * x;
  return p.neg_exp_a * (sx <= p.softplus_threshold ? log1pf(expf(sx)) / p.softplus_beta : x);
}
__device__ __forceinline__ float beta_of(const GateParams &p, float b) {
  return p.gated ? 1.0f / (1.0f + expf(-b)) : b;
}

// Sum over aligned groups of N lanes, in every lane of the group.
template <int CTRL>
__device__ __forceinline__ float dpp_sum(float x) {
  return x + __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), CTRL, 0xF, 0xF, true));
}
template <int N>
__device__ __forceinline__ float group_sum(float x) {
  if constexpr (N > 1) x = dpp_sum<0xB1>(x);    // quad_perm 1 0 3 2
  if constexpr (N > 2) x = dpp_sum<0x4E>(x);    // quad_perm 2 3 0 1
  if constexpr (N > 4) x = dpp_sum<0x141>(x);   // row_half_mirror: quads are uniform by now
  if constexpr (N > 8) x = dpp_sum<0x140>(x);   // row_mirror: halves are uniform
  if constexpr (N > 16) {
    const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(p[0]) + __uint_as_float(p[1]);
  }
  if constexpr (N > 32) {
    const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(p[0]) + __uint_as_float(p[1]);
  }
  return x;
}

}  // namespace gdn
