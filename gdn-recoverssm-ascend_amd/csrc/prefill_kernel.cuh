// Chunked gated delta rule on the matrix cores (gdn_recoverssm_prefill).
//
// A row's tokens are cut into chunks of up to 64 (a chunk also ends at a cache
// block's boundary). With G the cumulative log decay inside a chunk and S0 the
// state before it, the corrections solve a unit lower triangular system:
//   c_t = beta_t (v_t - e^{G_t} S0 k_t - sum_{s<t} e^{G_t - G_s} (k_t.k_s) c_s)
//   c   = T (v - diag(e^G) K S0^T),  T = (I + L)^{-1} diag(beta),
//         L_ts = beta_t e^{G_t - G_s} (k_t.k_s), s < t
//   out = diag(scale e^G) Q S0^T + P c,  P_ts = scale e^{G_t - G_s} (q_t.k_s), s <= t
//   S1  = e^{G_end} S0 + (diag(e^{G_end - G}) c)^T K
// T and P depend on no state, so a first kernel (prepare) makes them for all
// chunks at once; a second (scan) walks each (row, value head) through its
// chunks with a slice of the state's V rows in registers.
//
// Precision: states and corrections are FP32, and their products run on the
// BF16 matrix cores with each FP32 operand as the sum of three BF16 planes of 8
// bits (cut, not rounded: the sum of the three is the FP32 value). A product
// takes the pairs of planes whose places add up to at most 2, which drops terms
// under 2^-24 of it. BF16 keys are one plane, F16 two, FP32 three. The output's
// own products take OPL planes, two (2^-16) where it is rounded to 16 bits.
// The FP32 matrix instruction would take 16 times a BF16 one's time, 3 to 6
// times what the planes take.
//
// With the L2 norm fused in, 1 / |k| and 1 / |q| go into the scalars beside T,
// P and the decays, and K and Q stay as they are.
#pragma once

#include "rows.cuh"

namespace gdn {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr int kChunk = 64;
constexpr int kPrefillThreads = 256;
constexpr int kPlanesT = 3;
constexpr int kFrag = 1024;            // bytes of one 16 x 32 operand plane
constexpr float kMinLogDecay = -200.f; // e^-200 is 0 in FP32: cumulative sums stay finite

struct PrefillArgs {
  gdn_row_pages pages;
  const void *q, *k, *v, *g, *beta, *a_log, *dt_bias;
  void *out, *state;
  gdn_gating_ext gating;
  int64_t q_ts, k_ts, v_ts, g_ts, beta_ts, out_ts;
  int64_t state_bs, state_hs, state_vs;
  int32_t K, V, H, HV, ratio;
  int32_t g_dt, beta_dt, state_dt, out_f32, gated, l2norm;
  float scale;
  // Chunk geometry: positions are cut at multiples of 64 inside blocks of
  // `block` tokens, per_block chunks each; row b's chunks start at slot
  // qsl[b] * per_block / block + slack * b, which leaves every row enough.
  int32_t align, block, per_block, slack, slots;
  // Workspace: per (slot, key head) K^T (and packed K, Q), per (slot, value
  // head) T, P and the scalars.
  char *ws;
  int64_t kt_at, k_at, q_at, t_at, p_at, s_at;
  int32_t slices, members;  // scan: V slices of a state, workgroups of a key head's group
};

// Scalars of a (slot, value head): floats [4][64].
constexpr int kScalars = 4 * kChunk;
enum { kScIn = 0, kScQ = kChunk, kScOut = 2 * kChunk, kScEnd = 3 * kChunk };

__device__ __forceinline__ int64_t first_slot(const PrefillArgs &a, int b) {
  const int64_t at = load_index(a.pages.query_start_loc, b * a.pages.qsl_stride, a.pages.qsl_dtype);
  return int64_t(clamp_token(at, a.pages.tokens)) * a.per_block / a.block + int64_t(a.slack) * b;
}

// Orders LDS across the workgroup without draining global loads in flight.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }
__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// x as PL planes of its leading 8 bits and what they leave, packed pairwise.
template <int PL, int N>
__device__ __forceinline__ void split(const float (&x)[N], uint32_t (&planes)[PL][N / 2]) {
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    float a = x[i], b = x[i + 1];
#pragma unroll
    for (int p = 0; p < PL; ++p) {
      const uint32_t ua = __float_as_uint(a), ub = __float_as_uint(b);
      planes[p][i / 2] = __builtin_amdgcn_perm(ub, ua, 0x07060302u);
      if (p + 1 < PL) {
        a -= __uint_as_float(ua & 0xffff0000u);
        b -= __uint_as_float(ub & 0xffff0000u);
      }
    }
  }
}

__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
                                                 0);
}
// Sum of the plane products that count.
template <int PA, int PB>
__device__ __forceinline__ f32x4 mfma_planes(const u32x4 (&a)[PA], const u32x4 (&b)[PB], f32x4 c) {
#pragma unroll
  for (int sum = 2; sum >= 0; --sum)  // small terms first
#pragma unroll
    for (int i = 0; i < PA; ++i)
      if (sum - i >= 0 && sum - i < PB) c = mfma(a[i], b[sum - i], c);
  return c;
}

// Eight elements of a row of K or Q as planes (lane: row lane % 16, columns
// from (lane / 16) * 8 of a 32-column step).
template <typename A, int PL>
__device__ __forceinline__ void load_planes(const A *row, bool live, int k0, int K, u32x4 (&planes)[PL]) {
  float x[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = 0.0f;
  if (live && k0 + 8 <= K) {
    A raw[8];
    __builtin_memcpy(raw, row + k0, sizeof(raw));
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = to_f32(raw[e]);
  } else if (live) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (k0 + e < K) x[e] = to_f32(row[k0 + e]);
  }
  uint32_t w[PL][4];
  split<PL, 8>(x, w);
#pragma unroll
  for (int p = 0; p < PL; ++p) planes[p] = u32x4{w[p][0], w[p][1], w[p][2], w[p][3]};
}

template <int PL>
__device__ __forceinline__ float squares(const u32x4 (&planes)[PL]) {
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float lo = 0.0f, hi = 0.0f;
#pragma unroll
    for (int p = PL - 1; p >= 0; --p) {
      lo += __uint_as_float(planes[p][i] << 16);
      hi += __uint_as_float(planes[p][i] & 0xffff0000u);
    }
    s = fmaf(lo, lo, fmaf(hi, hi, s));
  }
  return s;
}
// Sum over lanes l, l ^ 16, l ^ 32, l ^ 48.
__device__ __forceinline__ float sum_quarters(float x) {
  const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(p[0]) + __uint_as_float(p[1]);
  const auto q = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(q[0]) + __uint_as_float(q[1]);
}

// ---------------------------------------------------------------------------
// Prepare: one workgroup per (slot, key head); the head's value heads in turn.
// Wave w holds token rows 16w .. 16w + 15 of K K^T and Q K^T.
// ---------------------------------------------------------------------------
template <typename A, int PL, int OPL, int KP, bool PACK>
__global__ __launch_bounds__(kPrefillThreads) void prepare_kernel(const PrefillArgs a) {
  constexpr int KS = KP / 32, LD = kChunk + 4;
  __shared__ float Ls[kChunk][LD], Ps[kChunk][LD];
  __shared__ float rks[kChunk], rqs[kChunk];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lr = lane & 15, lq = lane >> 4;
  const int slot = int(blockIdx.x / unsigned(a.H)), h = int(blockIdx.x % unsigned(a.H));
  const int b = __builtin_amdgcn_readfirstlane(
      last_not_above(int(a.pages.rows), slot, [&](int i) { return first_slot(a, i); }));
  if (b < 0) return;
  const Row r = load_row(a.pages, b);
  if (r.n == 0 || !r.valid) return;
  // The chunk's tokens.
  const int64_t C = a.align ? r.C : 0;
  const int64_t o = (C / a.block) * a.per_block + (C % a.block) / kChunk + (slot - first_slot(a, b));
  const int64_t blk = o / a.per_block;
  int64_t p0 = blk * a.block + (o % a.per_block) * kChunk, p1 = p0 + kChunk;
  p1 = p1 < (blk + 1) * a.block ? p1 : (blk + 1) * a.block;
  p0 = p0 > C ? p0 : C;
  p1 = p1 < C + r.n ? p1 : C + r.n;
  if (p0 >= p1) return;
  const int t0 = r.bos + int(p0 - C), n = int(p1 - p0);

  const A *const kp = static_cast<const A *>(a.k) + int64_t(t0) * a.k_ts + int64_t(h) * a.K;
  const A *const qp = static_cast<const A *>(a.q) + int64_t(t0) * a.q_ts + int64_t(h) * a.K;
  const int64_t sh = int64_t(slot) * a.H + h;

  f32x4 kk[4], qk[4];
  {
    u32x4 kf[KS][PL], qf[KS][PL];
    const int row = 16 * w + lr;
    float ksq = 0.0f, qsq = 0.0f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      load_planes<A, PL>(kp + row * a.k_ts, row < n, 32 * ks + 8 * lq, a.K, kf[ks]);
      load_planes<A, PL>(qp + row * a.q_ts, row < n, 32 * ks + 8 * lq, a.K, qf[ks]);
      if (a.l2norm) {
        ksq += squares<PL>(kf[ks]);
        qsq += squares<PL>(qf[ks]);
      }
      if constexpr (PACK) {
        const int64_t at = (sh * 4 * KS * PL + (w * KS + ks) * PL) * kFrag + lane * 16;
#pragma unroll
        for (int p = 0; p < PL; ++p) {
          *reinterpret_cast<u32x4 *>(a.ws + a.k_at + at + p * kFrag) = kf[ks][p];
          *reinterpret_cast<u32x4 *>(a.ws + a.q_at + at + p * kFrag) = qf[ks][p];
        }
      }
    }
    ksq = sum_quarters(ksq);
    qsq = sum_quarters(qsq);
    if (lq == 0) {
      rks[row] = a.l2norm ? 1.0f / sqrtf(ksq + 1e-6f) : 1.0f;
      rqs[row] = a.l2norm ? 1.0f / sqrtf(qsq + 1e-6f) : 1.0f;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      kk[j] = f32x4{0, 0, 0, 0};
      qk[j] = f32x4{0, 0, 0, 0};
      if (j <= w) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          u32x4 kb[PL];
          load_planes<A, PL>(kp + (16 * j + lr) * a.k_ts, 16 * j + lr < n, 32 * ks + 8 * lq, a.K, kb);
          kk[j] = mfma_planes<PL, PL>(kf[ks], kb, kk[j]);
          qk[j] = mfma_planes<PL, PL>(qf[ks], kb, qk[j]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          Ls[16 * w + lq * 4 + i][16 * j + lr] = 0.0f;
          Ps[16 * w + lq * 4 + i][16 * j + lr] = 0.0f;
        }
      }
    }
  }
  // K^T in operand order: column 16 kt + lane % 16 of K, eight tokens a lane.
  for (int f = w; f < KP / 16 * 2; f += 4) {
    const int kc = (f >> 1) * 16 + lr, s0 = (f & 1) * 32 + lq * 8;
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = s0 + e < n && kc < a.K ? to_f32(kp[(s0 + e) * a.k_ts + kc]) : 0.0f;
    uint32_t pl[PL][4];
    split<PL, 8>(x, pl);
#pragma unroll
    for (int p = 0; p < PL; ++p)
      *reinterpret_cast<u32x4 *>(a.ws + a.kt_at + ((sh * (KP / 8) + f) * PL + p) * kFrag + lane * 16) =
          u32x4{pl[p][0], pl[p][1], pl[p][2], pl[p][3]};
  }
  __syncthreads();

  for (int m = 0; m < a.ratio; ++m) {
    const int hv = h * a.ratio + m;
    const int64_t svh = int64_t(slot) * a.HV + hv;
    // Lane = token: gates and the cumulative log decay, summed in 64 bits and
    // kept as two floats, so that differences keep FP32 precision however far
    // the sum has gone.
    const GateParams gates = load_gates(a.a_log, a.dt_bias, a.gating, a.gated != 0, hv);
    float g = 0.0f, beta = 0.0f;
    if (lane < n) {
      g = log_decay(gates, load_as_f32(a.g, int64_t(t0 + lane) * a.g_ts + hv, a.g_dt));
      beta = beta_of(gates, load_as_f32(a.beta, int64_t(t0 + lane) * a.beta_ts + hv, a.beta_dt));
      g = g < kMinLogDecay ? kMinLogDecay : g;
    }
    double G = g;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const double up = __shfl_up(G, d);
      G += lane >= d ? up : 0.0;
    }
    const float Gh = float(G), Gl = float(G - double(Gh));
    if (w == 0) {
      const double end = __shfl(G, 63);
      float *sc = reinterpret_cast<float *>(a.ws + a.s_at) + svh * kScalars;
      sc[kScIn + lane] = expf(Gh + Gl) * rks[lane];
      sc[kScQ + lane] = a.scale * expf(Gh + Gl) * rqs[lane];
      sc[kScOut + lane] = expf(float(end - G)) * rks[lane];
      if (lane == 0) sc[kScEnd] = expf(float(end));
    }
    // L and P, token rows 16w + 4 lq + i, columns 16j + lr.
    float Ght[4], Glt[4], bt[4], rkt[4], rqt[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int t = 16 * w + 4 * lq + i;
      Ght[i] = __shfl(Gh, t);
      Glt[i] = __shfl(Gl, t);
      rkt[i] = rks[t];
      bt[i] = __shfl(beta, t) * rkt[i];
      rqt[i] = rqs[t] * a.scale;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (j > w) break;
      const int s = 16 * j + lr;
      const float Ghs = __shfl(Gh, s), Gls = __shfl(Gl, s), rk = rks[s];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int t = 16 * w + 4 * lq + i;
        const float d = expf((Ght[i] - Ghs) + (Glt[i] - Gls)) * rk;
        Ls[t][s] = s < t ? bt[i] * d * kk[j][i] : 0.0f;
        Ps[t][s] = s <= t ? rqt[i] * d * qk[j][i] : 0.0f;
      }
    }
    wave_fence();
    // The diagonal block's inverse, a column a lane: x_i = [i = c] - sum_m L_im x_m.
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float s = i == lr ? 1.0f : 0.0f;
#pragma unroll
      for (int c = 0; c < i; ++c) s = fmaf(-Ls[16 * w + i][16 * w + c], x[c], s);
      x[i] = s;
    }
    f32x4 T[4];  // T[d]: block (w + d, w)
#pragma unroll
    for (int i = 0; i < 4; ++i) T[0][i] = lq == 0 ? x[i] : lq == 1 ? x[4 + i] : lq == 2 ? x[8 + i] : x[12 + i];
    wave_fence();
#pragma unroll
    for (int i = 0; i < 4; ++i) Ls[16 * w + 4 * lq + i][16 * w + lr] = T[0][i];
    __syncthreads();
    // Block column w downwards: T_iw = -T_ii sum_{m = w}^{i - 1} L_im T_mw.
    // Step i of the FP32 instruction takes columns 4 lq + i, which is where the
    // accumulator of the block before holds its rows: no value moves.
#pragma unroll
    for (int d = 1; d < 4; ++d) {
      const int i = w + d;
      T[d] = f32x4{0, 0, 0, 0};
      if (i < 4) {
        f32x4 acc = {0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < d; ++e) {
          const f32x4 l = *reinterpret_cast<const f32x4 *>(&Ls[16 * i + lr][16 * (w + e) + 4 * lq]);
#pragma unroll
          for (int k = 0; k < 4; ++k) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(l[k], T[e][k], acc, 0, 0, 0);
        }
        const f32x4 l = *reinterpret_cast<const f32x4 *>(&Ls[16 * i + lr][16 * i + 4 * lq]);
#pragma unroll
        for (int k = 0; k < 4; ++k) T[d] = __builtin_amdgcn_mfma_f32_16x16x4f32(-l[k], acc[k], T[d], 0, 0, 0);
      }
    }
    __syncthreads();
    const float bs = __shfl(beta, 16 * w + lr);
#pragma unroll
    for (int d = 0; d < 4; ++d)
      if (w + d < 4)
#pragma unroll
        for (int i = 0; i < 4; ++i) Ls[16 * (w + d) + 4 * lq + i][16 * w + lr] = T[d][i] * bs;
    __syncthreads();
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      if (ks * 32 > 16 * w + 15) continue;  // above the diagonal: never read
      float y[8], z[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        y[e] = Ls[16 * w + lr][32 * ks + 8 * lq + e];
        z[e] = Ps[16 * w + lr][32 * ks + 8 * lq + e];
      }
      uint32_t tp[kPlanesT][4], pp[OPL][4];
      split<kPlanesT, 8>(y, tp);
      split<OPL, 8>(z, pp);
      const int64_t f = svh * 8 + 2 * w + ks;
#pragma unroll
      for (int p = 0; p < kPlanesT; ++p)
        *reinterpret_cast<u32x4 *>(a.ws + a.t_at + (f * kPlanesT + p) * kFrag + lane * 16) =
            u32x4{tp[p][0], tp[p][1], tp[p][2], tp[p][3]};
#pragma unroll
      for (int p = 0; p < OPL; ++p)
        *reinterpret_cast<u32x4 *>(a.ws + a.p_at + (f * OPL + p) * kFrag + lane * 16) =
            u32x4{pp[p][0], pp[p][1], pp[p][2], pp[p][3]};
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// Scan: one workgroup per (row, value head, 16 NV rows of V). Wave w takes
// token rows 16w .. 16w + 15 of a chunk's products and key columns KP/4 * w ..
// of the state, which it holds transposed (a lane: 4 neighbouring k of one v).
// ---------------------------------------------------------------------------
template <typename A, int PL, int OPL, int KP, int NV, bool PACK>
__global__ __launch_bounds__(kPrefillThreads) void scan_kernel(const PrefillArgs a) {
  constexpr int KS = KP / 32, KT = KP / 64, SLD = KP + 8, CLD = kChunk + 8;
  __shared__ uint16_t Sb[3][16 * NV][SLD], Rb[3][16 * NV][CLD], Cb[OPL][16 * NV][CLD], Db[3][16 * NV][CLD];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lr = lane & 15, lq = lane >> 4;
  // Workgroups of one key head's group (they read the same K, Q, T and P) sit
  // on one XCD: consecutive workgroups go to the eight XCDs in turn.
  const int wg = int(blockIdx.x), group = (wg / 8 / a.members) * 8 + wg % 8, member = wg / 8 % a.members;
  if (group >= a.pages.rows * a.H) return;
  const int b = group / a.H, h = group % a.H;
  const int hv = h * a.ratio + member / a.slices, v0 = member % a.slices * (16 * NV);
  const Row r = load_row(a.pages, b);
  if (r.n == 0) return;
  if (!r.valid) {
    const int width = a.V - v0 < 16 * NV ? a.V - v0 : 16 * NV;
    for (int64_t i = threadIdx.x; i < int64_t(r.n) * width; i += kPrefillThreads) {
      const int64_t at = (r.bos + i / width) * a.out_ts + int64_t(hv) * a.V + v0 + i % width;
      if (a.out_f32) static_cast<float *>(a.out)[at] = 0.0f;
      else static_cast<A *>(a.out)[at] = from_f32<A>(0.0f);
    }
    return;
  }
  const auto state_at = [&](int64_t page, int i, int nv) {  // element offset of the lane's four k
    return page * a.state_bs + hv * a.state_hs + int64_t(v0 + 16 * nv + lr) * a.state_vs + 16 * (w * KT + i) + 4 * lq;
  };
  const auto state_live = [&](int i, int nv) { return v0 + 16 * nv + lr < a.V && 16 * (w * KT + i) + 4 * lq < a.K; };
  const auto store_state = [&](int64_t page, const f32x4 (&S)[KT][NV]) {
#pragma unroll
    for (int i = 0; i < KT; ++i)
#pragma unroll
      for (int nv = 0; nv < NV; ++nv)
        if (state_live(i, nv)) {
          const int64_t at = state_at(page, i, nv);
          if (a.state_dt == GDN_DT_F32) {
            *reinterpret_cast<f32x4 *>(static_cast<float *>(a.state) + at) = S[i][nv];
          } else if (a.state_dt == GDN_DT_BF16) {
#pragma unroll
            for (int e = 0; e < 4; ++e) static_cast<bf16 *>(a.state)[at + e] = from_f32<bf16>(S[i][nv][e]);
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) static_cast<f16 *>(a.state)[at + e] = from_f32<f16>(S[i][nv][e]);
          }
        }
  };
  f32x4 S[KT][NV];
#pragma unroll
  for (int i = 0; i < KT; ++i)
#pragma unroll
    for (int nv = 0; nv < NV; ++nv) {
      S[i][nv] = f32x4{0, 0, 0, 0};
      if (!r.fresh && state_live(i, nv))
#pragma unroll
        for (int e = 0; e < 4; ++e) S[i][nv][e] = load_as_f32(a.state, state_at(r.src, i, nv) + e, a.state_dt);
    }

  int64_t slot = first_slot(a, b);
  int done = 0, inside = a.align ? int(r.C % a.block) : 0;
  while (done < r.n) {
    int n = kChunk - inside % kChunk;
    n = n < a.block - inside ? n : a.block - inside;
    n = n < r.n - done ? n : r.n - done;
    const int t0 = r.bos + done;
    const int64_t sh = slot * a.H + h, svh = slot * a.HV + hv;
    const float *sc = reinterpret_cast<const float *>(a.ws + a.s_at) + svh * kScalars;
    // The state, as planes, to every wave.
#pragma unroll
    for (int i = 0; i < KT; ++i)
#pragma unroll
      for (int nv = 0; nv < NV; ++nv) {
        const float x[4] = {S[i][nv][0], S[i][nv][1], S[i][nv][2], S[i][nv][3]};
        uint32_t pl[3][2];
        split<3, 4>(x, pl);
#pragma unroll
        for (int p = 0; p < 3; ++p)
          *reinterpret_cast<u32x2 *>(&Sb[p][16 * nv + lr][16 * (w * KT + i) + 4 * lq]) = u32x2{pl[p][0], pl[p][1]};
      }
    lds_barrier();
    // X = K S0^T and Q S0^T.
    f32x4 X[NV], O[NV];
#pragma unroll
    for (int nv = 0; nv < NV; ++nv) X[nv] = O[nv] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      u32x4 kf[PL], qf[PL];
      if constexpr (PACK) {
        const int64_t at = (sh * 4 * KS * PL + (w * KS + ks) * PL) * kFrag + lane * 16;
#pragma unroll
        for (int p = 0; p < PL; ++p) {
          kf[p] = *reinterpret_cast<const u32x4 *>(a.ws + a.k_at + at + p * kFrag);
          qf[p] = *reinterpret_cast<const u32x4 *>(a.ws + a.q_at + at + p * kFrag);
        }
      } else {
        const int row = 16 * w + lr;
        const bool live = row < n && 32 * ks + 8 * lq < a.K;
        kf[0] = qf[0] = u32x4{0, 0, 0, 0};
        if (live) {
          const A *kr = static_cast<const A *>(a.k) + int64_t(t0 + row) * a.k_ts + int64_t(h) * a.K + 32 * ks + 8 * lq;
          const A *qr = static_cast<const A *>(a.q) + int64_t(t0 + row) * a.q_ts + int64_t(h) * a.K + 32 * ks + 8 * lq;
          __builtin_memcpy(&kf[0], kr, 16);
          __builtin_memcpy(&qf[0], qr, 16);
        }
      }
#pragma unroll
      for (int nv = 0; nv < NV; ++nv) {
        u32x4 s[3];
#pragma unroll
        for (int p = 0; p < 3; ++p) s[p] = *reinterpret_cast<const u32x4 *>(&Sb[p][16 * nv + lr][32 * ks + 8 * lq]);
        X[nv] = mfma_planes<PL, 3>(kf, s, X[nv]);
        u32x4 so[OPL];
#pragma unroll
        for (int p = 0; p < OPL; ++p) so[p] = s[p];
        O[nv] = mfma_planes<PL, OPL>(qf, so, O[nv]);
      }
    }
    // R = V - diag(e^G) X.
    const f32x4 in = *reinterpret_cast<const f32x4 *>(sc + kScIn + 16 * w + 4 * lq);
#pragma unroll
    for (int nv = 0; nv < NV; ++nv) {
      float x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int t = 16 * w + 4 * lq + i, v = v0 + 16 * nv + lr;
        const float vv =
            t < n && v < a.V ? to_f32(static_cast<const A *>(a.v)[int64_t(t0 + t) * a.v_ts + int64_t(hv) * a.V + v]) : 0.0f;
        x[i] = t < n ? fmaf(-in[i], X[nv][i], vv) : 0.0f;
      }
      uint32_t pl[3][2];
      split<3, 4>(x, pl);
#pragma unroll
      for (int p = 0; p < 3; ++p)
        *reinterpret_cast<u32x2 *>(&Rb[p][16 * nv + lr][16 * w + 4 * lq]) = u32x2{pl[p][0], pl[p][1]};
    }
    lds_barrier();
    // c = T R.
    f32x4 Cc[NV];
#pragma unroll
    for (int nv = 0; nv < NV; ++nv) Cc[nv] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      if (ks * 32 > 16 * w + 15) continue;
      u32x4 tf[kPlanesT];
#pragma unroll
      for (int p = 0; p < kPlanesT; ++p)
        tf[p] = *reinterpret_cast<const u32x4 *>(a.ws + a.t_at + ((svh * 8 + 2 * w + ks) * kPlanesT + p) * kFrag + lane * 16);
#pragma unroll
      for (int nv = 0; nv < NV; ++nv) {
        u32x4 rf[3];
#pragma unroll
        for (int p = 0; p < 3; ++p) rf[p] = *reinterpret_cast<const u32x4 *>(&Rb[p][16 * nv + lr][32 * ks + 8 * lq]);
        Cc[nv] = mfma_planes<kPlanesT, 3>(tf, rf, Cc[nv]);
      }
    }
    const f32x4 decay = *reinterpret_cast<const f32x4 *>(sc + kScOut + 16 * w + 4 * lq);
#pragma unroll
    for (int nv = 0; nv < NV; ++nv) {
      float x[4], y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i] = Cc[nv][i];
        y[i] = x[i] * decay[i];
      }
      uint32_t pc[OPL][2], pd[3][2];
      split<OPL, 4>(x, pc);
      split<3, 4>(y, pd);
#pragma unroll
      for (int p = 0; p < OPL; ++p)
        *reinterpret_cast<u32x2 *>(&Cb[p][16 * nv + lr][16 * w + 4 * lq]) = u32x2{pc[p][0], pc[p][1]};
#pragma unroll
      for (int p = 0; p < 3; ++p)
        *reinterpret_cast<u32x2 *>(&Db[p][16 * nv + lr][16 * w + 4 * lq]) = u32x2{pd[p][0], pd[p][1]};
    }
    lds_barrier();
    // S1 = e^{G_end} S0 + K^T (diag(e^{G_end - G}) c).
    const float end = sc[kScEnd];
#pragma unroll
    for (int i = 0; i < KT; ++i)
#pragma unroll
      for (int nv = 0; nv < NV; ++nv) S[i][nv] *= end;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      u32x4 df[NV][3];
#pragma unroll
      for (int nv = 0; nv < NV; ++nv)
#pragma unroll
        for (int p = 0; p < 3; ++p) df[nv][p] = *reinterpret_cast<const u32x4 *>(&Db[p][16 * nv + lr][32 * ks + 8 * lq]);
#pragma unroll
      for (int i = 0; i < KT; ++i) {
        u32x4 kt[PL];
#pragma unroll
        for (int p = 0; p < PL; ++p)
          kt[p] = *reinterpret_cast<const u32x4 *>(
              a.ws + a.kt_at + ((sh * (KP / 8) + (w * KT + i) * 2 + ks) * PL + p) * kFrag + lane * 16);
#pragma unroll
        for (int nv = 0; nv < NV; ++nv) S[i][nv] = mfma_planes<PL, 3>(kt, df[nv], S[i][nv]);
      }
    }
    // out = diag(scale e^G) Q S0^T + P c.
    const f32x4 oq = *reinterpret_cast<const f32x4 *>(sc + kScQ + 16 * w + 4 * lq);
#pragma unroll
    for (int nv = 0; nv < NV; ++nv) O[nv] *= oq;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      if (ks * 32 > 16 * w + 15) continue;
      u32x4 pf[OPL];
#pragma unroll
      for (int p = 0; p < OPL; ++p)
        pf[p] = *reinterpret_cast<const u32x4 *>(a.ws + a.p_at + ((svh * 8 + 2 * w + ks) * OPL + p) * kFrag + lane * 16);
#pragma unroll
      for (int nv = 0; nv < NV; ++nv) {
        u32x4 cf[OPL];
#pragma unroll
        for (int p = 0; p < OPL; ++p) cf[p] = *reinterpret_cast<const u32x4 *>(&Cb[p][16 * nv + lr][32 * ks + 8 * lq]);
        O[nv] = mfma_planes<OPL, OPL>(pf, cf, O[nv]);
      }
    }
#pragma unroll
    for (int nv = 0; nv < NV; ++nv)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int t = 16 * w + 4 * lq + i, v = v0 + 16 * nv + lr;
        if (t < n && v < a.V) {
          const int64_t at = int64_t(t0 + t) * a.out_ts + int64_t(hv) * a.V + v;
          if (a.out_f32) static_cast<float *>(a.out)[at] = O[nv][i];
          else static_cast<A *>(a.out)[at] = from_f32<A>(O[nv][i]);
        }
      }
    done += n;
    inside += n;
    ++slot;
    if (inside == a.block) {
      inside = 0;
      if (a.align && done < r.n) {
        const int64_t page = boundary_page(a.pages, r, r.C + done);
        if (page != 0) store_state(page, S);
      }
    }
  }
  store_state(r.fin, S);
}

template <typename A, int PL, int OPL, bool PACK, int KP>
static void launch_prefill_dims(int nv, unsigned scan_grid, hipStream_t s, const PrefillArgs &a) {
  hipLaunchKernelGGL((prepare_kernel<A, PL, OPL, KP, PACK>), dim3(unsigned(a.slots) * unsigned(a.H)),
                     dim3(kPrefillThreads), 0, s, a);
  if (nv == 1)
    hipLaunchKernelGGL((scan_kernel<A, PL, OPL, KP, 1, PACK>), dim3(scan_grid), dim3(kPrefillThreads), 0, s, a);
  else
    hipLaunchKernelGGL((scan_kernel<A, PL, OPL, KP, 2, PACK>), dim3(scan_grid), dim3(kPrefillThreads), 0, s, a);
}
template <typename A, int PL, int OPL, bool PACK>
void launch_prefill(int kp, int nv, unsigned scan_grid, hipStream_t s, const PrefillArgs &a);

#define GDN_PREFILL(A, PL, OPL, PACK)                                                                            \
  template <>                                                                                                    \
  void launch_prefill<A, PL, OPL, PACK>(int kp, int nv, unsigned grid, hipStream_t s, const PrefillArgs &a) {    \
    if (kp == 64) launch_prefill_dims<A, PL, OPL, PACK, 64>(nv, grid, s, a);                                     \
    else if (kp == 128) launch_prefill_dims<A, PL, OPL, PACK, 128>(nv, grid, s, a);                              \
    else launch_prefill_dims<A, PL, OPL, PACK, 256>(nv, grid, s, a);                                             \
  }
#define GDN_PREFILL_DECL(A, PL, OPL, PACK) \
  template <>                              \
  void launch_prefill<A, PL, OPL, PACK>(int, int, unsigned, hipStream_t, const PrefillArgs &);
GDN_PREFILL_DECL(bf16, 1, 2, false)
GDN_PREFILL_DECL(bf16, 2, 2, true)
GDN_PREFILL_DECL(bf16, 3, 3, true)
GDN_PREFILL_DECL(f16, 2, 2, true)
GDN_PREFILL_DECL(f16, 3, 3, true)
GDN_PREFILL_DECL(float, 3, 3, true)

}  // namespace gdn
