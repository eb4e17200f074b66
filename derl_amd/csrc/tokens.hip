// Losses of policies over a vocabulary (gfx950): log-probability / entropy of wide categorical rows, the clipped policy
// loss with a KL term, and the loss of paired log ratios, each with its gradient with respect to the logits.  The
// padded-head kernels of heads.hip hold a row (<= 31 actions) in a wave's lanes; here a row has 1 .. 2^30 columns.
//
// With z a row of logits, m its maximum, S = sum_j exp(z_j - m), p_j = exp(z_j - m) / S:
//   log p_j = (z_j - m) - log S          H = log S - (1/S) sum_j exp(z_j - m) (z_j - m)
// Everything a row needs is carried through ONE pass as running (m, S, sum e (z - m)): whenever the maximum grows the
// sums are rescaled.  A row whose entries are all -inf (or that holds a NaN) has no distribution: NaN, as log_softmax gives.
// exp is exp2(x log2 e) on the difference z - m (v_exp_f32, 1 ulp; |z - m| log2 e is rounded once), all sums of a row are
// fp32 per thread and across the workgroup, sums over rows fp64.
#include "common.hpp"
#include "heads_dev.hpp"

namespace {

using u32x4 = __attribute__((ext_vector_type(4))) uint32_t;
// a row may start at any element: 16-byte accesses are declared with the alignment of one element (the hardware takes
// unaligned global accesses; a row that is 16-byte aligned costs nothing extra)
typedef u32x4 u32x4_a4 __attribute__((aligned(4)));
typedef u32x4 u32x4_a2 __attribute__((aligned(2)));

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLowest = -3.402823466e+38f;
constexpr int kMaxWorkers = 2048;  // workgroups of a row kernel = rows of `partials` (8 doubles each)

__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * kLog2e); }

struct ElemF32 {
  using Store = float;
  using Vec = u32x4_a4;
  static constexpr int E = 4;
  static __device__ __forceinline__ void unpack(u32x4 v, float (&x)[E]) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t bits = v[k];  // (a bit cast of the element itself takes the vector's first)
      x[k] = __builtin_bit_cast(float, bits);
    }
  }
  static __device__ __forceinline__ u32x4 pack(const float (&x)[E]) {
    u32x4 v;
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = __builtin_bit_cast(uint32_t, x[k]);
    return v;
  }
  static __device__ __forceinline__ float get(Store s) { return s; }
  static __device__ __forceinline__ Store put(float x) { return x; }
};
struct ElemBF16 {
  using Store = __bf16;
  using Vec = u32x4_a2;
  static constexpr int E = 8;
  static __device__ __forceinline__ void unpack(u32x4 v, float (&x)[E]) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t bits = v[k];
      x[2 * k] = __builtin_bit_cast(float, bits << 16);
      x[2 * k + 1] = __builtin_bit_cast(float, bits & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ u32x4 pack(const float (&x)[E]) {
    using bf16x2 = __attribute__((ext_vector_type(2))) __bf16;
    u32x4 v;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      bf16x2 b = {static_cast<__bf16>(x[2 * k]), static_cast<__bf16>(x[2 * k + 1])};  // round to nearest even
      v[k] = __builtin_bit_cast(uint32_t, b);
    }
    return v;
  }
  static __device__ __forceinline__ float get(Store s) { return static_cast<float>(s); }
  static __device__ __forceinline__ Store put(float x) { return static_cast<__bf16>(x); }
};
struct ElemF16 {
  using Store = _Float16;
  using Vec = u32x4_a2;
  static constexpr int E = 8;
  using f16x2 = __attribute__((ext_vector_type(2))) _Float16;
  static __device__ __forceinline__ void unpack(u32x4 v, float (&x)[E]) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t bits = v[k];
      const f16x2 h = __builtin_bit_cast(f16x2, bits);
      x[2 * k] = static_cast<float>(h.x);
      x[2 * k + 1] = static_cast<float>(h.y);
    }
  }
  static __device__ __forceinline__ u32x4 pack(const float (&x)[E]) {
    u32x4 v;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      f16x2 h = {static_cast<_Float16>(x[2 * k]), static_cast<_Float16>(x[2 * k + 1])};
      v[k] = __builtin_bit_cast(uint32_t, h);
    }
    return v;
  }
  static __device__ __forceinline__ float get(Store s) { return static_cast<float>(s); }
  static __device__ __forceinline__ Store put(float x) { return static_cast<_Float16>(x); }
};

// E elements of a row from column `first` on; columns at or past V read as -inf
template <class D>
__device__ __forceinline__ u32x4 load_vec(const char *row, int first, int V) {
  if (first + D::E <= V) return *reinterpret_cast<const typename D::Vec *>(row + static_cast<long long>(first) * sizeof(typename D::Store));
  float x[D::E];
#pragma unroll
  for (int k = 0; k < D::E; ++k)
    x[k] = first + k < V ? D::get(reinterpret_cast<const typename D::Store *>(row)[first + k]) : -INFINITY;
  return D::pack(x);  // exact: the values came from this type
}
template <class D>
__device__ __forceinline__ void store_vec(char *row, int first, int V, const float (&x)[D::E]) {
  if (first + D::E <= V) {
    *reinterpret_cast<typename D::Vec *>(row + static_cast<long long>(first) * sizeof(typename D::Store)) = D::pack(x);
    return;
  }
#pragma unroll
  for (int k = 0; k < D::E; ++k)
    if (first + k < V) reinterpret_cast<typename D::Store *>(row)[first + k] = D::put(x[k]);
}

// running statistics of a row (see the head of the file); `gap` = sum e (z - q), (mr, sr) those of the reference row q
struct RowStats { float m, s, ed, gap, mr, sr; };

__device__ __forceinline__ float wave_max_all(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
  return v;
}

// e (z - q), where e = 0 (a banned column) counts as 0 whatever z - q is
__device__ __forceinline__ float gap_term(float e, float z, float q) { return e == 0.f ? 0.f : e * (z - q); }

// raises the running maximum to at least x: the sums move to the new reference point.  Sums that vanish against the new
// maximum become exact zeros (0 * inf must not appear).
__device__ __forceinline__ void raise_max(RowStats &r, float x) {
  const float mn = fmaxf(r.m, x);
  const float d = r.m - mn, f = exp_of(d);
  r.ed = f == 0.f ? 0.f : f * (r.ed + r.s * d);
  r.gap = f == 0.f ? 0.f : f * r.gap;
  r.s *= f;
  r.m = mn;
}
__device__ __forceinline__ void raise_ref(RowStats &r, float x) {
  const float mn = fmaxf(r.mr, x);
  r.sr *= exp_of(r.mr - mn);
  r.mr = mn;
}

template <class D, bool REF>
__device__ __forceinline__ void add_vec(RowStats &r, u32x4 v, u32x4 w) {
  float x[D::E];
  D::unpack(v, x);
  float mx = x[0];
#pragma unroll
  for (int k = 1; k < D::E; ++k) mx = fmaxf(mx, x[k]);
  if (mx > r.m) raise_max(r, mx);
  float q[D::E];
  if constexpr (REF) {
    D::unpack(w, q);
    float mq = q[0];
#pragma unroll
    for (int k = 1; k < D::E; ++k) mq = fmaxf(mq, q[k]);
    if (mq > r.mr) raise_ref(r, mq);
  }
#pragma unroll
  for (int k = 0; k < D::E; ++k) {
    const float d = x[k] - r.m, e = exp_of(d);
    r.s += e;
    r.ed += e * fmaxf(d, kLowest);  // e = 0 and d = -inf: 0
    if constexpr (REF) {
      r.sr += exp_of(q[k] - r.mr);
      r.gap += gap_term(e, x[k], q[k]);
    }
  }
}

// the statistics of all lanes of a wave joined, in every lane
template <bool REF>
__device__ __forceinline__ void join_wave(RowStats &r) {
  raise_max(r, wave_max_all(r.m));
  r.s = wave_sum_all(r.s);
  r.ed = wave_sum_all(r.ed);
  if constexpr (REF) {
    raise_ref(r, wave_max_all(r.mr));
    r.sr = wave_sum_all(r.sr);
    r.gap = wave_sum_all(r.gap);
  }
}

struct RowArgs {
  const char *z, *q;
  char *dz;
  long long z_pitch, q_pitch, dz_pitch;  // bytes
  long long rows;
  int V;
  const int64_t *actions;
  const uint8_t *mask;
  const float *old_lp, *adv, *ref_lp;
  float *lp, *entropy;
  float4 *stats;        // preference: {m, 1 / S, lp, coefficient of the row}
  const double *count;  // unmasked rows, when `mask` is given
  double batch;         // > 0: what the gradient is divided by, else the unmasked rows
  float cliprange, kl_coef, ent_coef;
  double *partials;
};

enum Mode { LOGP, STATS, POLICY };

// T threads per row (64: one wave, four rows per workgroup).
// POLICY: the policy loss and its gradient; LOGP: log-probability and entropy; STATS: what the preference loss keeps.
template <class D, int T, Mode MODE, bool REF>
__global__ __launch_bounds__(T < 256 ? 256 : T) void token_rows_kernel(const RowArgs a) {
  constexpr int kWaves = T / 64, kRows = T < 256 ? 256 / T : 1;  // waves per row, rows per workgroup
  constexpr int E = D::E;
  __shared__ RowStats parts[2][kWaves > 1 ? kWaves : 1];
  __shared__ double sums[kRows][8];
  const int t = threadIdx.x % T, slot = threadIdx.x / T, lane = threadIdx.x & 63;
  const double weight = MODE == POLICY ? 1.0 / (a.batch > 0 ? a.batch : a.mask ? *a.count : static_cast<double>(a.rows)) : 0.0;
  const float w = static_cast<float>(weight);
  double sum[6] = {0, 0, 0, 0, 0, 0};
  int turn = 0;
  for (long long row = static_cast<long long>(blockIdx.x) * kRows + slot; row < a.rows; row += static_cast<long long>(gridDim.x) * kRows) {
    const bool keep = !a.mask || a.mask[row];
    const char *z = a.z + row * a.z_pitch;
    char *dz = MODE == POLICY ? a.dz + row * a.dz_pitch : nullptr;
    if (!keep) {  // (the same decision in every thread of the row)
      if (t == 0) {
        if (MODE != STATS) a.lp[row] = 0.f;
        if (MODE == LOGP && a.entropy) a.entropy[row] = 0.f;
        if (MODE == STATS) a.stats[row] = make_float4(0.f, 0.f, 0.f, 0.f);
      }
      if (MODE == POLICY) {
        float none[E];
#pragma unroll
        for (int k = 0; k < E; ++k) none[k] = 0.f;
        for (int first = t * E; first < a.V; first += T * E) store_vec<D>(dz, first, a.V, none);
      }
      continue;
    }
    const char *q = REF ? a.q + row * a.q_pitch : nullptr;
    const long long action = a.actions[row];
    const bool valid = action >= 0 && action < a.V;
    // read before any store of this row: dz may be z
    const float za = valid ? D::get(reinterpret_cast<const typename D::Store *>(z)[action]) : __builtin_nanf("");
    RowStats r = {kLowest, 0.f, 0.f, 0.f, kLowest, 0.f};
    for (int first = t * E; first < a.V; first += T * E) {
      const u32x4 v = load_vec<D>(z, first, a.V);
      u32x4 u = v;
      if constexpr (REF) u = load_vec<D>(q, first, a.V);
      add_vec<D, REF>(r, v, u);
    }
    join_wave<REF>(r);
    if constexpr (kWaves > 1) {
      if (lane == 0) parts[turn][threadIdx.x >> 6] = r;
      asm volatile("" ::"v"(za));  // za has arrived in every wave before any wave stores
      __syncthreads();
      r = {kLowest, 0.f, 0.f, 0.f, kLowest, 0.f};
      if (lane < kWaves) r = parts[turn][lane];
      join_wave<REF>(r);
      turn ^= 1;
    }
    const float log_s = logf(r.s);
    const float lp = (za - r.m) - log_s;
    if (MODE == LOGP || MODE == STATS) {
      if (t == 0) {
        if (MODE == LOGP) {
          a.lp[row] = lp;
          if (a.entropy) a.entropy[row] = log_s - r.ed / r.s;
        } else {
          a.stats[row] = make_float4(r.m, 1.f / r.s, lp, 0.f);
        }
      }
      continue;
    }
    if constexpr (MODE == POLICY) {
      const float H = log_s - r.ed / r.s;
      const float ratio = expf(lp - a.old_lp[row]), adv = a.adv[row];
      const float l1 = -ratio * adv;
      float policy = l1;
      bool active = true, outside = false;
      if (a.cliprange >= 0.f) {
        const float lo = 1.f - a.cliprange, hi = 1.f + a.cliprange;
        const float l2 = -(ratio < lo ? lo : ratio > hi ? hi : ratio) * adv;
        active = !(l2 > l1);  // inside the range the two are equal
        policy = active ? l1 : l2;
        outside = ratio < lo || ratio > hi;
      }
      float g = active ? l1 : 0.f;  // d policy / d lp
      float kl = 0.f, shift = 0.f;
      if (a.ref_lp) {  // e^d - 1 - d with d = log ref - log p >= 0, its expectation under p is the divergence
        const float d = a.ref_lp[row] - lp, em = expm1f(d);
        kl = em - d;
        g -= a.kl_coef * em;
      }
      if constexpr (REF) {
        shift = (r.m - r.mr) + logf(r.s / r.sr);  // difference of the two log-normalisers
        kl = r.gap / r.s - shift;
      }
      if (t == 0) {
        a.lp[row] = lp;
        sum[0] += policy;
        sum[1] += H;
        sum[2] += kl;
        sum[3] += outside ? 1.0 : 0.0;
        sum[4] += ratio;
        sum[5] += lp;
      }
      // dz_j = w [ g (1{j = a} - p_j) + c_H p_j (log p_j + H) + c_K p_j (log p_j - log q_j - KL) ]
      //      = p_j (c0 + c1 (z_j - m) + c2 (z_j - q_j)) + w g 1{j = a}
      const float c1 = w * a.ent_coef, c2 = REF ? w * a.kl_coef : 0.f;
      const float c0 = w * (a.ent_coef * (H - log_s) - g) - c2 * (shift + kl);
      const float inv_s = 1.f / r.s;
      auto grad = [&](float x, float y) {
        const float d = x - r.m, p = exp_of(d) * inv_s;
        float v = c0 + c1 * fmaxf(d, kLowest);
        if constexpr (REF) return p == 0.f ? 0.f : p * (v + c2 * (x - y));
        return p * v;
      };
      for (int first = t * E; first < a.V; first += T * E) {
        float x[E], y[E];
        D::unpack(load_vec<D>(z, first, a.V), x);
        if constexpr (REF) D::unpack(load_vec<D>(q, first, a.V), y);
#pragma unroll
        for (int k = 0; k < E; ++k) x[k] = grad(x[k], REF ? y[k] : 0.f) + (first + k == action ? w * g : 0.f);
        store_vec<D>(dz, first, a.V, x);
      }
    }
  }
  if constexpr (MODE == POLICY) {
    if (t == 0)
#pragma unroll
      for (int k = 0; k < 6; ++k) sums[slot][k] = sum[k];
    __syncthreads();
    if (threadIdx.x < 8) {
      double s = 0;
      for (int i = 0; i < kRows; ++i) s += threadIdx.x < 6 ? sums[i][threadIdx.x] : 0.0;
      a.partials[blockIdx.x * 8LL + threadIdx.x] = s;
    }
  }
}

__global__ __launch_bounds__(1024) void mask_count_kernel(const uint8_t *mask, long long n, double *count) {
  __shared__ long long parts[16];
  long long c = 0;
  for (long long i = threadIdx.x; i < n; i += 1024) c += mask[i] != 0;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) c += __shfl_xor(c, o);
  if ((threadIdx.x & 63) == 0) parts[threadIdx.x >> 6] = c;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 16; ++i) c += parts[i];
    *count = static_cast<double>(c);
  }
}

// sums of `n` rows of eight doubles, in one fixed order: thread (i, k) takes rows i, i + 128, ... of column k
__device__ void sum_partials(const double *partials, int n, double (&total)[8]) {
  __shared__ double acc[128][8];
  const int k = threadIdx.x & 7, i = threadIdx.x >> 3;
  double s = 0;
  for (int j = i; j < n; j += 128) s += partials[j * 8LL + k];
  acc[i][k] = s;
  __syncthreads();
  for (int half = 64; half > 0; half >>= 1) {
    if (i < half) acc[i][k] += acc[i + half][k];
    __syncthreads();
  }
  for (int c = 0; c < 8; ++c) total[c] = acc[0][c];
}

__global__ __launch_bounds__(1024) void policy_terms_kernel(const double *partials, int n, const double *count, long long rows,
                                                            float kl_coef, float ent_coef, float *loss_out) {
  double s[8];
  sum_partials(partials, n, s);
  if (threadIdx.x == 0) {
    const double c = count ? *count : static_cast<double>(rows);
    const double inv = c > 0 ? 1.0 / c : 0.0;  // nothing unmasked: zeros
    loss_out[0] = static_cast<float>((s[0] - ent_coef * s[1] + kl_coef * s[2]) * inv);
    for (int k = 0; k < 6; ++k) loss_out[k + 1] = static_cast<float>(s[k] * inv);
    loss_out[7] = static_cast<float>(c);
  }
}

// ---- preference ----------------------------------------------------------------------------------
struct PairArgs {
  float4 *stats;
  const int32_t *offsets;
  const float *ref_lp;
  const uint8_t *mask;
  long long rows;
  int pairs;
  double batch;
  float beta, smoothing;
  float *seq_lp;
  double *partials;
};

__device__ double block_sum_256(double v, double *scratch) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
  __syncthreads();
  return scratch[0] + scratch[1] + scratch[2] + scratch[3];
}

// a workgroup per pair: the two sequences' log-probabilities, the pair's loss, and the coefficient of each of its rows
__global__ __launch_bounds__(256) void preference_pairs_kernel(const PairArgs a) {
  __shared__ double scratch[4];
  double sum[7] = {0, 0, 0, 0, 0, 0, 0};
  for (int pair = blockIdx.x; pair < a.pairs; pair += gridDim.x) {
    double lp[2];
    long long begin[2], end[2];
    for (int side = 0; side < 2; ++side) {
      const long long b = a.offsets[2LL * pair + side], e = a.offsets[2LL * pair + side + 1];
      begin[side] = b < 0 ? 0 : b;
      end[side] = e > a.rows ? a.rows : e;
      double s = 0;
      for (long long i = begin[side] + threadIdx.x; i < end[side]; i += 256) s += a.stats[i].z;
      lp[side] = block_sum_256(s, scratch);
    }
    const double chosen = a.beta * (lp[0] - (a.ref_lp ? a.ref_lp[2LL * pair] : 0.f));
    const double rejected = a.beta * (lp[1] - (a.ref_lp ? a.ref_lp[2LL * pair + 1] : 0.f));
    const double h = chosen - rejected;
    const double tail = log1p(exp(-fabs(h)));                     // -log sig(h) = max(-h, 0) + log(1 + e^-|h|)
    const double up = (h < 0 ? -h : 0.0) + tail, down = (h > 0 ? h : 0.0) + tail;
    const double slope = (a.smoothing / (1.0 + exp(-h)) - (1.0 - a.smoothing) / (1.0 + exp(h))) * a.beta / (a.batch > 0 ? a.batch : a.pairs);
    for (int side = 0; side < 2; ++side) {
      const float c = static_cast<float>(side ? -slope : slope);
      for (long long i = begin[side] + threadIdx.x; i < end[side]; i += 256)
        if (!a.mask || a.mask[i]) a.stats[i].w = c;
    }
    if (threadIdx.x == 0) {
      a.seq_lp[2LL * pair] = static_cast<float>(lp[0]);
      a.seq_lp[2LL * pair + 1] = static_cast<float>(lp[1]);
      const double loss = (a.smoothing < 1.f ? (1.0 - a.smoothing) * up : 0.0) + (a.smoothing > 0.f ? a.smoothing * down : 0.0);
      const double add[7] = {loss, h > 0 ? 1.0 : 0.0, h, chosen, rejected, lp[0], lp[1]};
      for (int k = 0; k < 7; ++k) sum[k] += add[k];
    }
  }
  if (threadIdx.x == 0) {
    for (int k = 0; k < 7; ++k) a.partials[blockIdx.x * 8LL + k] = sum[k];
    a.partials[blockIdx.x * 8LL + 7] = 0.0;
  }
}

__global__ __launch_bounds__(1024) void preference_terms_kernel(const double *partials, int n, int pairs, float *loss_out) {
  double s[8];
  sum_partials(partials, n, s);
  if (threadIdx.x == 0) {
    for (int k = 0; k < 7; ++k) loss_out[k] = static_cast<float>(s[k] / pairs);
    loss_out[7] = static_cast<float>(pairs);
  }
}

// dz_j = c (1{j = a} - p_j) of every row, c the coefficient of its sequence (0: no sequence's, or masked)
template <class D, int T>
__global__ __launch_bounds__(T < 256 ? 256 : T) void preference_grad_kernel(const RowArgs a) {
  constexpr int kRows = T < 256 ? 256 / T : 1, E = D::E;
  const int t = threadIdx.x % T, slot = threadIdx.x / T;
  // from the last row down: the end of the logits is what the statistics pass has left in the last-level cache
  for (long long i = static_cast<long long>(blockIdx.x) * kRows + slot; i < a.rows; i += static_cast<long long>(gridDim.x) * kRows) {
    const long long row = a.rows - 1 - i;
    const float4 st = a.stats[row];
    char *dz = a.dz + row * a.dz_pitch;
    const char *z = a.z + row * a.z_pitch;
    const float c = st.w, k = -c * st.y;
    const long long action = c != 0.f ? a.actions[row] : -1;
    for (int first = t * E; first < a.V; first += T * E) {
      float x[E];
      if (c != 0.f) {
        D::unpack(load_vec<D>(z, first, a.V), x);
#pragma unroll
        for (int j = 0; j < E; ++j) x[j] = k * exp_of(x[j] - st.x) + (first + j == action ? c : 0.f);
      } else {
#pragma unroll
        for (int j = 0; j < E; ++j) x[j] = 0.f;
      }
      store_vec<D>(dz, first, a.V, x);
    }
  }
}

// log-probabilities of sequences: a workgroup per sequence
__global__ __launch_bounds__(256) void sequence_sum_kernel(const float *lp, const int32_t *offsets, long long rows, int sequences, float *out) {
  __shared__ double scratch[4];
  for (int q = blockIdx.x; q < sequences; q += gridDim.x) {
    const long long b = offsets[q] < 0 ? 0 : offsets[q], e = offsets[q + 1] > rows ? rows : offsets[q + 1];
    double s = 0;
    for (long long i = b + threadIdx.x; i < e; i += 256) s += lp[i];
    s = block_sum_256(s, scratch);
    if (threadIdx.x == 0) out[q] = static_cast<float>(s);
  }
}

// x *= *factor in place, nothing at all when it is 1 (the gradient of a loss that is differentiated as it stands)
template <class D>
__global__ __launch_bounds__(256) void scale_rows_kernel(char *x, long long pitch, long long rows, int V, const float *factor) {
  const float f = *factor;
  if (f == 1.f) return;
  constexpr int E = D::E;
  for (long long row = blockIdx.x; row < rows; row += gridDim.x)
    for (int first = threadIdx.x * E; first < V; first += 256 * E) {
      float v[E];
      D::unpack(load_vec<D>(x + row * pitch, first, V), v);
#pragma unroll
      for (int k = 0; k < E; ++k) v[k] *= f;
      store_vec<D>(x + row * pitch, first, V, v);
    }
}

// threads per row, by its bytes
inline int row_threads(int V, int dtype) {
  const long long bytes = static_cast<long long>(V) * (dtype == DX_F32 ? 4 : 2);
  return bytes <= 4096 ? 64 : bytes <= 32768 ? 256 : 1024;
}
inline int row_grid(long long rows, int T) {
  const long long need = T == 64 ? (rows + 3) / 4 : rows;
  const long long most = T == 1024 ? 512 : kMaxWorkers;
  return static_cast<int>(need < most ? need : most);
}

template <class D, Mode MODE, bool REF>
int launch_rows(const RowArgs &a, int T, int grid, hipStream_t s) {
  if (T == 64) hipLaunchKernelGGL((token_rows_kernel<D, 64, MODE, REF>), dim3(grid), dim3(256), 0, s, a);
  else if (T == 256) hipLaunchKernelGGL((token_rows_kernel<D, 256, MODE, REF>), dim3(grid), dim3(256), 0, s, a);
  else hipLaunchKernelGGL((token_rows_kernel<D, 1024, MODE, REF>), dim3(grid), dim3(1024), 0, s, a);
  DX_LAUNCH_CHECK();
  return DX_OK;
}
template <Mode MODE, bool REF>
int launch_rows_of(const RowArgs &a, int dtype, int T, int grid, hipStream_t s) {
  if (dtype == DX_F32) return launch_rows<ElemF32, MODE, REF>(a, T, grid, s);
  if (dtype == DX_BF16) return launch_rows<ElemBF16, MODE, REF>(a, T, grid, s);
  return launch_rows<ElemF16, MODE, REF>(a, T, grid, s);
}
template <class D>
int launch_pref_grad(const RowArgs &a, int T, int grid, hipStream_t s) {
  if (T == 64) hipLaunchKernelGGL((preference_grad_kernel<D, 64>), dim3(grid), dim3(256), 0, s, a);
  else if (T == 256) hipLaunchKernelGGL((preference_grad_kernel<D, 256>), dim3(grid), dim3(256), 0, s, a);
  else hipLaunchKernelGGL((preference_grad_kernel<D, 1024>), dim3(grid), dim3(1024), 0, s, a);
  DX_LAUNCH_CHECK();
  return DX_OK;
}

// what every entry point over logits checks
int check_logits(const char *who, const void *logits, int dtype, long long rows, int vocab, long long pitch, const int64_t *actions) {
  DX_REQUIRE(dtype == DX_F32 || dtype == DX_BF16 || dtype == DX_F16, "%s: dtype %d is none of DX_F32, DX_BF16, DX_F16", who, dtype);
  DX_REQUIRE(rows >= 0 && rows <= 0x7fffffffLL, "%s: rows %lld outside [0, 2^31)", who, rows);
  DX_REQUIRE(vocab >= 1 && vocab <= (1 << 30), "%s: vocab %d outside [1, 2^30]", who, vocab);
  DX_REQUIRE(rows <= 1 || pitch >= vocab, "%s: rows of %d logits at a pitch of %lld overlap", who, vocab, pitch);
  DX_REQUIRE(rows == 0 || (logits != nullptr && actions != nullptr), "%s: null pointer", who);
  DX_REQUIRE(dx::aligned(logits, dtype == DX_F32 ? 4 : 2), "%s: logits are not aligned to their type", who);
  return DX_OK;
}

RowArgs row_args(const void *logits, int dtype, long long rows, int vocab, long long pitch, const int64_t *actions, const uint8_t *mask) {
  RowArgs a{};
  const int size = dtype == DX_F32 ? 4 : 2;
  a.z = static_cast<const char *>(logits);
  a.z_pitch = pitch * size;
  a.rows = rows;
  a.V = vocab;
  a.actions = actions;
  a.mask = mask;
  return a;
}

}  // namespace

extern "C" int dx_token_log_prob(const void *logits, int dtype, long long rows, int vocab, long long pitch, const int64_t *actions,
                                 const uint8_t *mask, float *log_prob, float *entropy, void *stream) {
  DX_TRACE("dx_token_log_prob");
  if (int rc = check_logits("dx_token_log_prob", logits, dtype, rows, vocab, pitch, actions)) return rc;
  if (rows == 0) return DX_OK;
  DX_REQUIRE(log_prob != nullptr, "dx_token_log_prob: null pointer");
  RowArgs a = row_args(logits, dtype, rows, vocab, pitch, actions, mask);
  a.lp = log_prob;
  a.entropy = entropy;
  const int T = row_threads(vocab, dtype);
  return launch_rows_of<LOGP, false>(a, dtype, T, row_grid(rows, T), dx::as_stream(stream));
}

extern "C" int dx_sequence_log_prob(const float *token_log_prob, const int32_t *offsets, long long rows, int sequences, float *out,
                                    void *stream) {
  DX_TRACE("dx_sequence_log_prob");
  DX_REQUIRE(rows >= 0 && sequences >= 0, "dx_sequence_log_prob: negative shape");
  if (sequences == 0) return DX_OK;
  DX_REQUIRE((token_log_prob || rows == 0) && offsets && out, "dx_sequence_log_prob: null pointer");
  hipLaunchKernelGGL(sequence_sum_kernel, dim3(sequences < kMaxWorkers ? sequences : kMaxWorkers), dim3(256), 0, dx::as_stream(stream),
                     token_log_prob, offsets, rows, sequences, out);
  DX_LAUNCH_CHECK();
  return DX_OK;
}

extern "C" int dx_token_policy_loss(const void *logits, int dtype, long long rows, int vocab, long long pitch, const int64_t *actions,
                                    const float *old_log_prob, const float *advantages, const float *ref_log_prob,
                                    const void *ref_logits, long long ref_pitch, const uint8_t *mask, float cliprange, float kl_coef,
                                    float entropy_coef, long long global_batch, void *dlogits, long long dlogits_pitch,
                                    float *log_prob, double *workspace, long long workspace_count, float *loss_out, void *stream) {
  DX_TRACE("dx_token_policy_loss");
  if (int rc = check_logits("dx_token_policy_loss", logits, dtype, rows, vocab, pitch, actions)) return rc;
  DX_REQUIRE(loss_out != nullptr && workspace != nullptr, "dx_token_policy_loss: null pointer");
  DX_REQUIRE(rows == 0 || (old_log_prob && advantages && dlogits && log_prob), "dx_token_policy_loss: null pointer");
  DX_REQUIRE(!(ref_log_prob && ref_logits), "dx_token_policy_loss: give ref_log_prob or ref_logits, not both");
  DX_REQUIRE(rows <= 1 || dlogits_pitch >= vocab, "dx_token_policy_loss: rows of dlogits overlap");
  DX_REQUIRE(!ref_logits || rows <= 1 || ref_pitch >= vocab, "dx_token_policy_loss: rows of ref_logits overlap");
  DX_REQUIRE(dx::aligned(dlogits, dtype == DX_F32 ? 4 : 2) && dx::aligned(ref_logits, dtype == DX_F32 ? 4 : 2),
             "dx_token_policy_loss: dlogits / ref_logits are not aligned to their type");
  if (workspace_count < DX_TOKEN_WORKSPACE)
    return dx::fail(DX_EWS, "dx_token_policy_loss: workspace of %lld doubles, %d needed", workspace_count, DX_TOKEN_WORKSPACE);
  hipStream_t s = dx::as_stream(stream);
  RowArgs a = row_args(logits, dtype, rows, vocab, pitch, actions, mask);
  const int size = dtype == DX_F32 ? 4 : 2;
  a.q = static_cast<const char *>(ref_logits);
  a.q_pitch = ref_pitch * size;
  a.dz = static_cast<char *>(dlogits);
  a.dz_pitch = dlogits_pitch * size;
  a.old_lp = old_log_prob;
  a.adv = advantages;
  a.ref_lp = ref_log_prob;
  a.lp = log_prob;
  a.count = workspace;
  a.batch = global_batch > 0 ? static_cast<double>(global_batch) : 0.0;
  a.cliprange = cliprange;
  a.kl_coef = kl_coef;
  a.ent_coef = entropy_coef;
  a.partials = workspace + 8;
  if (mask) {
    hipLaunchKernelGGL(mask_count_kernel, dim3(1), dim3(1024), 0, s, mask, rows, workspace);
    DX_LAUNCH_CHECK();
  }
  const int T = row_threads(vocab, dtype), grid = row_grid(rows, T);
  if (grid > 0) {
    if (int rc = ref_logits ? launch_rows_of<POLICY, true>(a, dtype, T, grid, s) : launch_rows_of<POLICY, false>(a, dtype, T, grid, s)) return rc;
  }
  hipLaunchKernelGGL(policy_terms_kernel, dim3(1), dim3(1024), 0, s, a.partials, grid, mask ? workspace : nullptr, rows, kl_coef,
                     entropy_coef, loss_out);
  DX_LAUNCH_CHECK();
  return DX_OK;
}

extern "C" int dx_preference_loss(const void *logits, int dtype, long long rows, int vocab, long long pitch, const int64_t *actions,
                                  const int32_t *offsets, int pairs, const float *ref_log_prob, const uint8_t *mask, float beta,
                                  float label_smoothing, long long global_pairs, void *dlogits, long long dlogits_pitch,
                                  float *sequence_log_prob, float *row_stats, double *workspace, long long workspace_count,
                                  float *loss_out, void *stream) {
  DX_TRACE("dx_preference_loss");
  if (int rc = check_logits("dx_preference_loss", logits, dtype, rows, vocab, pitch, actions)) return rc;
  DX_REQUIRE(pairs >= 1, "dx_preference_loss: pairs %d < 1", pairs);
  DX_REQUIRE(label_smoothing >= 0.f && label_smoothing <= 1.f, "dx_preference_loss: label_smoothing outside [0, 1]");
  DX_REQUIRE(offsets && sequence_log_prob && workspace && loss_out, "dx_preference_loss: null pointer");
  DX_REQUIRE(rows == 0 || (dlogits && row_stats), "dx_preference_loss: null pointer");
  DX_REQUIRE(rows <= 1 || dlogits_pitch >= vocab, "dx_preference_loss: rows of dlogits overlap");
  DX_REQUIRE(dx::aligned(dlogits, dtype == DX_F32 ? 4 : 2) && dx::aligned(row_stats, 16), "dx_preference_loss: misaligned dlogits / row_stats");
  if (workspace_count < DX_TOKEN_WORKSPACE)
    return dx::fail(DX_EWS, "dx_preference_loss: workspace of %lld doubles, %d needed", workspace_count, DX_TOKEN_WORKSPACE);
  hipStream_t s = dx::as_stream(stream);
  RowArgs a = row_args(logits, dtype, rows, vocab, pitch, actions, mask);
  a.stats = reinterpret_cast<float4 *>(row_stats);
  a.dz = static_cast<char *>(dlogits);
  a.dz_pitch = dlogits_pitch * (dtype == DX_F32 ? 4 : 2);
  const int T = row_threads(vocab, dtype), grid = row_grid(rows, T);
  if (grid > 0)
    if (int rc = launch_rows_of<STATS, false>(a, dtype, T, grid, s)) return rc;
  PairArgs p{a.stats, offsets, ref_log_prob, mask, rows, pairs, global_pairs > 0 ? static_cast<double>(global_pairs) : 0.0, beta,
             label_smoothing, sequence_log_prob, workspace + 8};
  const int pair_grid = pairs < kMaxWorkers ? pairs : kMaxWorkers;
  hipLaunchKernelGGL(preference_pairs_kernel, dim3(pair_grid), dim3(256), 0, s, p);
  DX_LAUNCH_CHECK();
  hipLaunchKernelGGL(preference_terms_kernel, dim3(1), dim3(1024), 0, s, p.partials, pair_grid, pairs, loss_out);
  DX_LAUNCH_CHECK();
  if (grid == 0) return DX_OK;
  if (dtype == DX_F32) return launch_pref_grad<ElemF32>(a, T, grid, s);
  if (dtype == DX_BF16) return launch_pref_grad<ElemBF16>(a, T, grid, s);
  return launch_pref_grad<ElemF16>(a, T, grid, s);
}

extern "C" int dx_scale_rows(void *x, int dtype, long long rows, int columns, long long pitch, const float *factor, void *stream) {
  DX_TRACE("dx_scale_rows");
  DX_REQUIRE(dtype == DX_F32 || dtype == DX_BF16 || dtype == DX_F16, "dx_scale_rows: dtype %d", dtype);
  DX_REQUIRE(rows >= 0 && columns >= 0 && columns <= (1 << 30) && (rows <= 1 || pitch >= columns), "dx_scale_rows: bad shape");
  if (rows == 0 || columns == 0) return DX_OK;
  DX_REQUIRE(x && factor && dx::aligned(x, dtype == DX_F32 ? 4 : 2), "dx_scale_rows: null or misaligned pointer");
  const dim3 grid(static_cast<unsigned>(rows < kMaxWorkers ? rows : kMaxWorkers));
  char *p = static_cast<char *>(x);
  hipStream_t s = dx::as_stream(stream);
  if (dtype == DX_F32) hipLaunchKernelGGL(scale_rows_kernel<ElemF32>, grid, dim3(256), 0, s, p, pitch * 4, rows, columns, factor);
  else if (dtype == DX_BF16) hipLaunchKernelGGL(scale_rows_kernel<ElemBF16>, grid, dim3(256), 0, s, p, pitch * 2, rows, columns, factor);
  else hipLaunchKernelGGL(scale_rows_kernel<ElemF16>, grid, dim3(256), 0, s, p, pitch * 2, rows, columns, factor);
  DX_LAUNCH_CHECK();
  return DX_OK;
}
