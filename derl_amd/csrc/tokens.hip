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
constexpr int kMaxPieces = 512;    // pieces of rows, where few rows are cut
// Up to so many rows every workgroup counts the mask itself, which costs less than a launch (policy loss of 4096 x 18 f32, masked:
// 17.3 us, 20.4 with the launch; of 16384 x 18 22.9, 23.1); of more, 16 bytes a thread and load are read by all of them too often.
constexpr int kCountedHere = 16384;
constexpr int kMaxWorkers = 2048;  // workgroups of a row kernel = rows of `partials` (8 doubles each)

__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * kLog2e); }

struct ElemF32 {
  static constexpr uint32_t kNegInf = 0;  // (unused: a word is an element)
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
  static constexpr uint32_t kNegInf = 0xff80u;
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
  static constexpr uint32_t kNegInf = 0xfc00u;
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

// Rows are walked in chunks of T threads x E columns.  `at` is the chunk's address (uniform), t its thread, `first` the
// thread's column; `ragged` (uniform): the chunk passes the row's end.  There a thread reads the row's LAST E columns instead
// (one vector load as everywhere else: element loads would have to be waited for on the spot, and with them every load in
// flight before them), and unpack_raw moves them to their places; columns past the end are -inf.
template <class D>
__device__ __forceinline__ u32x4 load_raw(const char *row, const char *at, int t, int first, int V, bool ragged) {
  using Store = typename D::Store;
  if (!ragged) return *reinterpret_cast<const typename D::Vec *>(at + static_cast<uint32_t>(t) * 16);
  if (V >= D::E) return *reinterpret_cast<const typename D::Vec *>(row + static_cast<long long>(min(first, V - D::E)) * sizeof(Store));
  float x[D::E];  // rows shorter than a vector
#pragma unroll
  for (int k = 0; k < D::E; ++k) x[k] = first + k < V ? D::get(reinterpret_cast<const Store *>(row)[first + k]) : -INFINITY;
  return D::pack(x);  // exact: the values came from this type
}
template <class D>
__device__ __forceinline__ void unpack_raw(u32x4 v, float (&x)[D::E], int first, int V, bool ragged) {
  D::unpack(v, x);
  if (!ragged || V < D::E) return;
  const int shift = max(0, first - (V - D::E));
#pragma unroll
  for (int b = 1; b < D::E; b *= 2)
#pragma unroll
    for (int k = 0; k < D::E; ++k) {
      const float other = k + b < D::E ? x[k + b] : -INFINITY;
      x[k] = shift & b ? other : x[k];
    }
#pragma unroll
  for (int k = 0; k < D::E; ++k) x[k] = shift < D::E ? x[k] : -INFINITY;
}
// (gradients leave past the caches, which then keep logits for a pass that reads them again: preference loss of 512 MB of
// logits 5.2 -> 5.8 TB/s over its three passes)
template <class D>
__device__ __forceinline__ void store_chunk(char *row, char *at, int t, int first, int V, bool ragged, const float (&x)[D::E]) {
  if (!ragged || first + D::E <= V) {
    __builtin_nontemporal_store(D::pack(x), reinterpret_cast<typename D::Vec *>(at + static_cast<uint32_t>(t) * 16));
    return;
  }
#pragma unroll
  for (int k = 0; k < D::E; ++k)
    if (first + k < V) reinterpret_cast<typename D::Store *>(row)[first + k] = D::put(x[k]);
}

// running statistics of a row (see the head of the file); (mr, sr) those of the reference row q, and `gap` = sum e ((z - m) - (q - mr)):
// two models' logits have no common zero, and of differences z - q the distance of the rows would leave only the last bits
struct RowStats { float m, s, ed, gap, mr, sr; };

__device__ __forceinline__ float wave_max_all(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
  return v;
}

// e (z - q) of logits relative to their maxima, where e = 0 (a banned column) counts as 0 whatever z - q is
__device__ __forceinline__ float gap_term(float e, float z, float q) { return e == 0.f ? 0.f : e * (z - q); }

// raises the running maximum to at least x: the sums move to the new reference point.  Sums that vanish against the new
// maximum become exact zeros (0 * inf must not appear).
__device__ __forceinline__ void raise_max(RowStats &r, float x) {
  const float mn = fmaxf(r.m, x);
  const float d = r.m - mn, f = exp_of(d);
  r.ed = f == 0.f ? 0.f : f * (r.ed + r.s * d);
  r.gap = f == 0.f ? 0.f : f * (r.gap + r.s * d);
  r.s *= f;
  r.m = mn;
}
__device__ __forceinline__ void raise_ref(RowStats &r, float x) {
  const float mn = fmaxf(r.mr, x);
  r.gap += r.s == 0.f ? 0.f : r.s * (mn - r.mr);
  r.sr *= exp_of(r.mr - mn);
  r.mr = mn;
}

template <class D, bool REF>
__device__ __forceinline__ void add_vec(RowStats &r, const float (&x)[D::E], const float (&q)[D::E]) {
  float mx = x[0];
#pragma unroll
  for (int k = 1; k < D::E; ++k) mx = fmaxf(mx, x[k]);
  if (mx > r.m) raise_max(r, mx);
  if constexpr (REF) {
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
      const float dq = q[k] - r.mr;
      r.sr += exp_of(dq);
      r.gap += gap_term(e, d, dq);
    }
  }
}

// a column's terms, or a vector's, under maxima that are known already (r.m, r.mr)
template <bool REF>
__device__ __forceinline__ void add_term(RowStats &r, float x, float q) {
  const float d = x - r.m, e = exp_of(d);
  r.s += e;
  r.ed += e * fmaxf(d, kLowest);
  if constexpr (REF) {
    const float dq = q - r.mr;
    r.sr += exp_of(dq);
    r.gap += gap_term(e, d, dq);
  }
}
template <class D, bool REF>
__device__ __forceinline__ void add_terms(RowStats &r, const float (&x)[D::E], const float (&q)[D::E]) {
#pragma unroll
  for (int k = 0; k < D::E; ++k) add_term<REF>(r, x[k], REF ? q[k] : 0.f);
}

// columns begin .. end of a row (begin and, but for the row's end, end are multiples of a chunk) added to this thread's statistics
template <class D, int T, bool REF>
__device__ __forceinline__ void add_columns(RowStats &r, const char *z, const char *q, int V, int begin, int end, int t) {
  constexpr int C = T * D::E, U = 4;
  int base = begin;
  for (; base + U * C <= end; base += U * C) {
    u32x4 v[U], u[REF ? U : 1];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const long long at = static_cast<long long>(base + k * C) * sizeof(typename D::Store);
      v[k] = load_raw<D>(z, z + at, t, 0, V, false);
      if constexpr (REF) u[k] = load_raw<D>(q, q + at, t, 0, V, false);
    }
#pragma unroll
    for (int k = 0; k < U; ++k) {
      float x[D::E], y[D::E];
      D::unpack(v[k], x);
      if constexpr (REF) D::unpack(u[k], y);
      add_vec<D, REF>(r, x, y);
    }
  }
  for (; base < end; base += C) {
    const bool ragged = base + C > V;
    const int first = base + t * D::E;
    if (first >= V) break;
    const long long at = static_cast<long long>(base) * sizeof(typename D::Store);
    float x[D::E], y[D::E];
    unpack_raw<D>(load_raw<D>(z, z + at, t, first, V, ragged), x, first, V, ragged);
    if constexpr (REF) unpack_raw<D>(load_raw<D>(q, q + at, t, first, V, ragged), y, first, V, ragged);
    add_vec<D, REF>(r, x, y);
  }
}
// dz of columns begin .. end from `value(x, y, column)`; `read` false: zeros, nothing is read
template <class D, int T, bool REF, class F>
__device__ __forceinline__ void write_columns(const char *z, const char *q, char *dz, int V, int begin, int end, int t, bool read, F value) {
  constexpr int C = T * D::E, U = 2;
  int base = begin;
  for (; base + U * C <= end; base += U * C) {
    u32x4 v[U], u[REF ? U : 1];
    if (read) {
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const long long at = static_cast<long long>(base + k * C) * sizeof(typename D::Store);
        v[k] = load_raw<D>(z, z + at, t, 0, V, false);
        if constexpr (REF) u[k] = load_raw<D>(q, q + at, t, 0, V, false);
      }
    }
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int first = base + k * C + t * D::E;
      float x[D::E] = {}, y[D::E];
      if (read) {
        D::unpack(v[k], x);
        if constexpr (REF) D::unpack(u[k], y);
#pragma unroll
        for (int i = 0; i < D::E; ++i) x[i] = value(x[i], REF ? y[i] : 0.f, first + i);
      }
      store_chunk<D>(dz, dz + static_cast<long long>(base + k * C) * sizeof(typename D::Store), t, first, V, false, x);
    }
  }
  for (; base < end; base += C) {
    const bool ragged = base + C > V;
    const int first = base + t * D::E;
    if (first >= V) break;
    const long long at = static_cast<long long>(base) * sizeof(typename D::Store);
    float x[D::E] = {}, y[D::E];
    if (read) {
      unpack_raw<D>(load_raw<D>(z, z + at, t, first, V, ragged), x, first, V, ragged);
      if constexpr (REF) unpack_raw<D>(load_raw<D>(q, q + at, t, first, V, ragged), y, first, V, ragged);
#pragma unroll
      for (int i = 0; i < D::E; ++i) x[i] = value(x[i], REF ? y[i] : 0.f, first + i);
    }
    store_chunk<D>(dz, dz + at, t, first, V, ragged, x);
  }
}

// the statistics of all lanes of a wave joined, in every lane
template <bool REF>
__device__ __forceinline__ void join_wave(RowStats &r) {
  raise_max(r, wave_max_all(r.m));
  if constexpr (REF) {
    raise_ref(r, wave_max_all(r.mr));  // (before r.s is another's too)
    r.sr = wave_sum_all(r.sr);
    r.gap = wave_sum_all(r.gap);
  }
  r.s = wave_sum_all(r.s);
  r.ed = wave_sum_all(r.ed);
}
constexpr RowStats kNothing = {kLowest, 0.f, 0.f, 0.f, kLowest, 0.f};

// joined over the W waves that share a row; `parts`: two sets of W, used in turn (one barrier a row)
template <int W, bool REF>
__device__ __forceinline__ void join_row(RowStats &r, RowStats (&parts)[2][W], int &turn) {
  join_wave<REF>(r);
  if constexpr (W > 1) {
    const int lane = threadIdx.x & 63;
    if (lane == 0) parts[turn][threadIdx.x >> 6] = r;
    __syncthreads();
    r = kNothing;
    if (lane < W) r = parts[turn][lane];
    join_wave<REF>(r);
    turn ^= 1;
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
  const double *count;  // unmasked rows, when `mask` is given; null: to be counted
  double batch;         // > 0: what the gradient is divided by, else the unmasked rows
  float cliprange, kl_coef, ent_coef;
  const float *factor;  // null, or what the gradient is multiplied by before it is rounded; 1: it is there already, nothing is done
  double *partials;
  // rows cut into `splits` pieces of `piece` columns (a multiple of 2048)
  int splits, piece;
  RowStats *piece_stats;
  float *chosen;  // POLICY: the action's logit of each row
};

enum Mode { LOGP, STATS, POLICY };

__device__ __forceinline__ bool is_there(const float *factor) { return factor && *factor == 1.f; }

// what a row's gradient is made of: dz_j = p_j (c0 + c1 (z_j - m) + c2 ((z_j - m) - (q_j - mr))) + at 1{j = action}
struct RowPlan { float m, inv_s, c0, c1, c2, at, mr; };

template <class D, bool REF, bool ENT>
__device__ __forceinline__ float grad_of(const RowPlan &g, float x, float y) {
  const float d = x - g.m, p = exp_of(d) * g.inv_s;
  float v = g.c0;
  if constexpr (ENT) v += g.c1 * fmaxf(d, kLowest);
  if constexpr (REF) v = g.c2 != 0.f ? v + g.c2 * (d - (y - g.mr)) : v;
  // of a banned column d or y - mr is infinite, and c1 d where |c1| > 1: 0 times anything is 0 here (v_mul_legacy_f32; a select
  // instead cost 2 % of the policy loss of 8192 x 131072 bf16)
  float product;
  asm("v_mul_legacy_f32 %0, %1, %2" : "=v"(product) : "v"(p), "v"(v));
  return product;
}

struct RowTerms { float policy, entropy, kl, outside, ratio, lp; };

// the policy loss of a row from its statistics: the gradient's plan and the row's terms
template <bool REF>
__device__ __forceinline__ RowPlan policy_row(const RowArgs &a, const RowStats &r, float za, float old, float adv, float ref, float w,
                                              RowTerms *terms) {
  const float log_s = logf(r.s), lp = (za - r.m) - log_s, H = log_s - r.ed / r.s;
  const float ratio = expf(lp - old), l1 = -ratio * adv;
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
    const float d = ref - lp, em = expm1f(d);
    kl = em - d;
    if (a.kl_coef != 0.f) g -= a.kl_coef * em;  // (0: the divergence, which may be infinite, is reported only)
  }
  if constexpr (REF) {
    shift = logf(r.s / r.sr);  // difference of the two log-normalisers, beyond that of the maxima
    kl = r.gap / r.s - shift;
  }
  *terms = {policy, H, kl, outside ? 1.f : 0.f, ratio, lp};
  // dz_j = w [ g (1{j = a} - p_j) + c_H p_j (log p_j + H) + c_K p_j (log p_j - log q_j - KL) ]
  const float c1 = w * a.ent_coef, c2 = REF ? w * a.kl_coef : 0.f;
  const float c0 = w * (a.ent_coef * (H - log_s) - g);
  return RowPlan{r.m, 1.f / r.s, c2 != 0.f ? c0 - c2 * (shift + kl) : c0, c1, c2, w * g, r.mr};
}

// this thread's share of the unmasked rows, thread `at` of `threads`: 16 bytes of the mask at a time, a bit for each that is not 0
__device__ __forceinline__ int count_mask(const uint8_t *mask, long long rows, int at, int threads) {
  typedef u32x4 Loose __attribute__((aligned(1)));
  int c = 0;
  const long long vectors = rows / 16;
#pragma unroll 4
  for (long long i = at; i < vectors; i += threads) {
    const u32x4 v = *reinterpret_cast<const Loose *>(mask + i * 16);
#pragma unroll
    for (int k = 0; k < 4; ++k) c += __popc((((v[k] & 0x7f7f7f7fu) + 0x7f7f7f7fu) | v[k]) & 0x80808080u);
  }
  if (vectors * 16 + at < rows) c += mask[vectors * 16 + at] != 0;  // fewer than 16 are left, and there are more threads
  return c;
}
// the count of the whole workgroup of W waves, in every thread
template <int W>
__device__ __forceinline__ int count_rows(const uint8_t *mask, long long rows) {
  int c = count_mask(mask, rows, threadIdx.x, W * 64);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) c += __shfl_xor(c, o);
  if constexpr (W > 1) {
    __shared__ int parts[W];
    if ((threadIdx.x & 63) == 0) parts[threadIdx.x >> 6] = c;
    __syncthreads();
    c = 0;
    for (int i = 0; i < W; ++i) c += parts[i];
  }
  return c;
}

// one over what the gradient is divided by.  Few rows are counted by every workgroup itself, see kCountedHere.
template <int W>
__device__ __forceinline__ float row_weight(const RowArgs &a) {
  double n = static_cast<double>(a.rows);
  if (a.batch > 0) n = a.batch;
  else if (a.mask) n = a.count ? *a.count : count_rows<W>(a.mask, a.rows);
  return static_cast<float>(a.factor ? *a.factor / n : 1.0 / n);
}

template <class D>
__device__ __forceinline__ float action_logit(const char *row, long long action, int V) {
  return action >= 0 && action < V ? D::get(reinterpret_cast<const typename D::Store *>(row)[action]) : __builtin_nanf("");
}

// T threads per row (64: one wave, four rows per workgroup).  POLICY: the policy loss and its gradient; LOGP: log-probability
// and entropy; STATS: what the preference loss keeps.
//   NV > 0: a thread holds its NV vectors of the row in registers, so the row is read once; while the gradient leaves, the
//           vectors are replaced by those of the workgroup's next row, which are then on their way during the whole store.
//   NV = 0: rows too long for that: the row is read twice, the second time from the caches for the most part.
// A workgroup takes rows b, b + grid, ...: 64 of them at a time have their masks, actions, scalars and chosen logits loaded
// by the lanes of every wave at once, one latency for all.
template <class D, int T, int NV, Mode MODE, bool REF, bool ENT>
__global__ __launch_bounds__(T < 256 ? 256 : T) void token_rows_kernel(const RowArgs a) {
  constexpr int kWaves = T / 64, kRows = T < 256 ? 256 / T : 1;  // waves per row, rows per workgroup
  constexpr int E = D::E, N = NV ? NV : 1;
  __shared__ RowStats parts[2][kWaves];
  __shared__ double sums[kRows][8];
  if (MODE == POLICY && is_there(a.factor)) return;
  const int t = threadIdx.x % T, slot = threadIdx.x / T, lane = threadIdx.x & 63;
  const float w = MODE == POLICY ? row_weight<T < 256 ? 4 : kWaves>(a) : 0.f;
  if (MODE == POLICY && t < 8) sums[slot][t] = 0.0;
  int turn = 0;
  const long long step = static_cast<long long>(gridDim.x) * kRows;
  u32x4 v[N], u[REF ? N : 1];
  // NV > 0: `vectors` whole vectors of a row (vector k T + t is this thread's k-th), and `rest` columns behind them, one each
  // for the first threads
  const int vectors = a.V / E, rest = a.V % E;
  typename D::Store vt = {}, ut = {};
  auto load_row = [&](long long row) {
    const char *z = a.z + row * a.z_pitch, *q = REF ? a.q + row * a.q_pitch : nullptr;
    if (t < rest) {
      vt = reinterpret_cast<const typename D::Store *>(z)[vectors * E + t];
      if constexpr (REF) ut = reinterpret_cast<const typename D::Store *>(q)[vectors * E + t];
    }
  };
  auto load_part = [&](int k, long long row) {  // (a thread past the end reads the last vector; see `own`)
    int lane_at = t;
    asm volatile("" : "+v"(lane_at));  // (opaque: sixteen addresses kept over the rows would spill)
    if ((k + 1) * T > vectors) lane_at = min(lane_at, vectors - 1 - k * T);
    const uint32_t at = static_cast<uint32_t>(lane_at) * 16;
    const auto *from = reinterpret_cast<const typename D::Vec *>(a.z + row * a.z_pitch + k * T * 16 + at);
    // (the policy loss has no other use for them; 1001 x 32768 f32 4.9 -> 5.1 TB/s)
    v[k] = MODE == POLICY ? __builtin_nontemporal_load(from) : *from;
    if constexpr (REF) u[k] = *reinterpret_cast<const typename D::Vec *>(a.q + row * a.q_pitch + k * T * 16 + at);
  };
  // nothing but -inf in the vectors that this thread does not have
  auto own = [&](int k) {
    if ((k + 1) * T <= vectors) return;
    constexpr uint32_t kNone = sizeof(typename D::Store) == 4 ? 0xff800000u : D::kNegInf * 0x10001u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[k][i] = k * T + t < vectors ? v[k][i] : kNone;
      if constexpr (REF) u[k][i] = k * T + t < vectors ? u[k][i] : kNone;
    }
  };
  for (long long row0 = static_cast<long long>(blockIdx.x) * kRows + slot; row0 < a.rows; row0 += 64 * step) {
    const long long mine = row0 + lane * step;
    const bool exists = mine < a.rows, keep = exists && (!a.mask || a.mask[mine]);
    float za = 0.f, old = 0.f, adv = 0.f, ref = 0.f;
    RowTerms out = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f};  // of this lane's row
    int action = -1;
    if (keep) {
      const long long wanted = a.actions[mine];
      za = action_logit<D>(a.z + mine * a.z_pitch, wanted, a.V);  // before any store of the row: dz may be z
      if (wanted >= 0 && wanted < a.V) action = static_cast<int>(wanted);
      if (MODE == POLICY) {
        old = a.old_lp[mine];
        adv = a.adv[mine];
        if (a.ref_lp) ref = a.ref_lp[mine];
      }
    }
    unsigned long long left = __ballot(keep);
    if (MODE == POLICY) {
      if constexpr (kWaves > 1) {
        asm volatile("" ::"v"(za));  // the chosen logits have arrived in every wave before any wave stores
        __syncthreads();
      }
      for (unsigned long long none = __ballot(exists && !keep); none; none &= none - 1) {
        char *dz = a.dz + (row0 + __builtin_ctzll(none) * step) * a.dz_pitch;
        write_columns<D, T, false>(nullptr, nullptr, dz, a.V, 0, a.V, t, false, [](float, float, int) { return 0.f; });
      }
    }
    if (NV && left) {
#pragma unroll
      for (int k = 0; k < N; ++k)
        if (k * T < vectors) load_part(k, row0 + __builtin_ctzll(left) * step);
      load_row(row0 + __builtin_ctzll(left) * step);
    }
    while (left) {
      const int j = __builtin_ctzll(left);
      left &= left - 1;
      const long long row = row0 + j * step;
      RowStats r = kNothing;
      if constexpr (NV > 0) {
        // (asm: opaque, else the compiler keeps the 16-bit values once it has widened them, and spills)
        const float xt = t < rest ? D::get(vt) : -INFINITY, yt = REF && t < rest ? D::get(ut) : -INFINITY;
        r.m = fmaxf(r.m, xt);
        if constexpr (REF) r.mr = fmaxf(r.mr, yt);
#pragma unroll
        for (int k = 0; k < N; ++k) {
          if (k * T >= vectors) continue;
          own(k);
          float x[E], y[E];
          D::unpack(v[k], x);
          if constexpr (REF) D::unpack(u[k], y);
#pragma unroll
          for (int i = 0; i < E; i += 2) {
            r.m = fmaxf(r.m, fmaxf(x[i], x[i + 1]));
            if constexpr (REF) r.mr = fmaxf(r.mr, fmaxf(y[i], y[i + 1]));
          }
          __builtin_amdgcn_sched_barrier(0);  // one vector's values at a time
        }
#pragma unroll
        for (int k = 0; k < N; ++k) {
          if (k * T >= vectors) continue;
          asm volatile("" : "+v"(v[k]));
          if constexpr (REF) asm volatile("" : "+v"(u[k]));
          float x[E], y[E];
          D::unpack(v[k], x);
          if constexpr (REF) D::unpack(u[k], y);
          add_terms<D, REF>(r, x, y);
          __builtin_amdgcn_sched_barrier(0);
        }
        add_term<REF>(r, xt, yt);
      } else {
        add_columns<D, T, REF>(r, a.z + row * a.z_pitch, REF ? a.q + row * a.q_pitch : nullptr, a.V, 0, a.V, t);
      }
      join_row<kWaves, REF>(r, parts, turn);
      const float z_chosen = lane_value(za, j);
      if constexpr (MODE != POLICY) {
        const float log_s = logf(r.s), lp = (z_chosen - r.m) - log_s;
        if (MODE == LOGP) {
          if (lane == j) {
            out.lp = lp;
            out.entropy = log_s - r.ed / r.s;
          }
        } else if (t == 0) {
          a.stats[row] = make_float4(r.m, 1.f / r.s, lp, 0.f);
        }
        if (NV && left) {
#pragma unroll
          for (int k = 0; k < N; ++k)
            if (k * T < vectors) load_part(k, row0 + __builtin_ctzll(left) * step);
          load_row(row0 + __builtin_ctzll(left) * step);
        }
      } else {
        RowTerms terms;
        const RowPlan g = policy_row<REF>(a, r, z_chosen, lane_value(old, j), lane_value(adv, j), lane_value(ref, j), w, &terms);
        if (lane == j) out = terms;
        const int chosen = __builtin_amdgcn_readlane(action, j);
        char *dz = a.dz + row * a.dz_pitch;
        const long long next = left ? row0 + __builtin_ctzll(left) * step : -1;
        if constexpr (NV > 0) {
#pragma unroll
          for (int k = 0; k < N; ++k) {
            if (k * T >= vectors) continue;
            float x[E], y[E];
            asm volatile("" : "+v"(v[k]));
            D::unpack(v[k], x);
            if constexpr (REF) {
              asm volatile("" : "+v"(u[k]));
              D::unpack(u[k], y);
            }
            if (next >= 0) load_part(k, next);
#pragma unroll
            for (int i = 0; i < E; ++i) x[i] = grad_of<D, REF, ENT>(g, x[i], REF ? y[i] : 0.f);
            if ((k + 1) * T <= vectors || k * T + t < vectors)
              __builtin_nontemporal_store(D::pack(x), reinterpret_cast<typename D::Vec *>(dz + k * T * 16 + static_cast<uint32_t>(t) * 16));
            __builtin_amdgcn_sched_barrier(0);
          }
          if (t < rest)
            reinterpret_cast<typename D::Store *>(dz)[vectors * E + t] =
                D::put(grad_of<D, REF, ENT>(g, D::get(vt), REF ? D::get(ut) : 0.f));
          if (next >= 0) load_row(next);
        } else {
          write_columns<D, T, REF>(a.z + row * a.z_pitch, REF ? a.q + row * a.q_pitch : nullptr, dz, a.V, 0, a.V, t, true,
                                   [&](float x, float y, int) { return grad_of<D, REF, ENT>(g, x, y); });
        }
        // the chosen column again, by the thread that has just stored it (a thread's stores to one address stay in order)
        if (chosen >= 0 && (NV && chosen >= vectors * E ? chosen - vectors * E : chosen / E % T) == t) {
          const float y = REF ? D::get(reinterpret_cast<const typename D::Store *>(a.q + row * a.q_pitch)[chosen]) : 0.f;
          reinterpret_cast<typename D::Store *>(dz)[chosen] = D::put(grad_of<D, REF, ENT>(g, z_chosen, y) + g.at);
        }
      }
    }
    if (t < 64) {  // the first wave of the row: 64 rows' results at once
      if (MODE != STATS && exists && a.lp) a.lp[mine] = out.lp;
      if (MODE == LOGP && exists && a.entropy) a.entropy[mine] = out.entropy;
      if (MODE == POLICY) {
        const float all[6] = {out.policy, out.entropy, out.kl, out.outside, out.ratio, out.lp};
#pragma unroll
        for (int k = 0; k < 6; ++k) {
          double s = all[k];
#pragma unroll
          for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
          if (lane == 0) sums[slot][k] += s;
        }
      }
      if (MODE == STATS && exists && !keep) a.stats[mine] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
  }
  if constexpr (MODE == POLICY) {
    __syncthreads();
    if (threadIdx.x < 8) {
      double s = 0;
      for (int i = 0; i < kRows; ++i) s += sums[i][threadIdx.x];
      a.partials[blockIdx.x * 8LL + threadIdx.x] = s;
    }
  }
}

// ---- rows of up to 1 KB: 16 lanes a row -----------------------------------------------------------------------------
// A row of a small vocabulary costs a wave as many instructions as a long one's first vector, most of them the row's own scalars
// and sums over lanes: four rows share them here.  262144 x 18 f32: log-probabilities 74 us, policy loss 138 us a call with a wave a
// row, 18 and 42 so; of 250 columns 73 and 160, 44 and 115; 256 rows alike.  The next row is on its way during this one; the action's
// logit is picked from the registers.
template <int ROR>
__device__ __forceinline__ float rotated16(float v) {  // within the 16 lanes of a row
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x120 + ROR, 0xf, 0xf, true));
}
__device__ __forceinline__ float sum16(float v) {
  v += rotated16<8>(v);
  v += rotated16<4>(v);
  v += rotated16<2>(v);
  return v + rotated16<1>(v);
}
__device__ __forceinline__ float max16(float v) {
  v = fmaxf(v, rotated16<8>(v));
  v = fmaxf(v, rotated16<4>(v));
  v = fmaxf(v, rotated16<2>(v));
  return fmaxf(v, rotated16<1>(v));
}

template <class D, int NV, Mode MODE, bool REF, bool ENT>
__global__ __launch_bounds__(256) void token_short_kernel(const RowArgs a) {
  constexpr int E = D::E;
  __shared__ double sums[16][8];
  if (MODE == POLICY && is_there(a.factor)) return;
  const int t = threadIdx.x & 15, slot = threadIdx.x >> 4;
  const float w = MODE == POLICY ? row_weight<4>(a) : 0.f;
  const long long step = gridDim.x * 16LL;
  struct Row {
    bool keep;
    long long action;
    float old, adv, ref;
    u32x4 v[NV], u[REF ? NV : 1];
  };
  auto load = [&](long long row) {  // (a row past the last: the last one again)
    if (row >= a.rows) row = a.rows - 1;
    Row r{};
    r.keep = !a.mask || a.mask[row];
    if (!r.keep) return r;
    r.action = a.actions[row];
    if constexpr (MODE == POLICY) {
      r.old = a.old_lp[row];
      r.adv = a.adv[row];
      if (a.ref_lp) r.ref = a.ref_lp[row];
    }
    const char *z = a.z + row * a.z_pitch, *q = REF ? a.q + row * a.q_pitch : nullptr;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if (k * 16 * E >= a.V) continue;
      const bool ragged = (k + 1) * 16 * E > a.V;
      r.v[k] = load_raw<D>(z, z + k * 256, t, (k * 16 + t) * E, a.V, ragged);
      if constexpr (REF) r.u[k] = load_raw<D>(q, q + k * 256, t, (k * 16 + t) * E, a.V, ragged);
    }
    return r;
  };
  double sum[6] = {0, 0, 0, 0, 0, 0};
  long long row = blockIdx.x * 16LL + slot;
  Row now = load(row);
  for (; row < a.rows; row += step) {
    const Row next = load(row + step);
    RowStats r = kNothing;
    float x[NV][E], y[REF ? NV : 1][E], za = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if (k * 16 * E >= a.V) continue;
      const int first = (k * 16 + t) * E;
      const bool ragged = (k + 1) * 16 * E > a.V;
      unpack_raw<D>(now.v[k], x[k], first, a.V, ragged);
      if constexpr (REF) unpack_raw<D>(now.u[k], y[k], first, a.V, ragged);
#pragma unroll
      for (int i = 0; i < E; ++i) {
        r.m = fmaxf(r.m, x[k][i]);
        if constexpr (REF) r.mr = fmaxf(r.mr, y[k][i]);
        za += first + i == now.action ? x[k][i] : 0.f;
      }
    }
    r.m = max16(r.m);
    if constexpr (REF) r.mr = max16(r.mr);
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (k * 16 * E < a.V) add_terms<D, REF>(r, x[k], y[REF ? k : 0]);
    r.s = sum16(r.s);
    r.ed = sum16(r.ed);
    if constexpr (REF) {
      r.sr = sum16(r.sr);
      r.gap = sum16(r.gap);
    }
    za = sum16(za);  // (one lane's)
    if (now.action < 0 || now.action >= a.V) za = __builtin_nanf("");
    RowTerms out = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if constexpr (MODE == POLICY) {
      RowPlan g = {};
      if (now.keep) g = policy_row<REF>(a, r, za, now.old, now.adv, now.ref, w, &out);
      char *dz = a.dz + row * a.dz_pitch;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        if (k * 16 * E >= a.V) continue;
        const int first = (k * 16 + t) * E;
#pragma unroll
        for (int i = 0; i < E; ++i)
          x[k][i] = now.keep ? grad_of<D, REF, ENT>(g, x[k][i], REF ? y[k][i] : 0.f) + (first + i == now.action ? g.at : 0.f) : 0.f;
        if (first < a.V) store_chunk<D>(dz, dz + k * 256, t, first, a.V, (k + 1) * 16 * E > a.V, x[k]);
      }
      if (t == 0) {
        const float all[6] = {out.policy, out.entropy, out.kl, out.outside, out.ratio, out.lp};
#pragma unroll
        for (int k = 0; k < 6; ++k) sum[k] += all[k];
      }
    } else {
      const float log_s = logf(r.s);
      out.lp = now.keep ? (za - r.m) - log_s : 0.f;
      out.entropy = now.keep ? log_s - r.ed / r.s : 0.f;
    }
    if (t == 0) {
      if (MODE != STATS && a.lp) a.lp[row] = out.lp;
      if (MODE == LOGP && a.entropy) a.entropy[row] = out.entropy;
      if (MODE == STATS) a.stats[row] = now.keep ? make_float4(r.m, 1.f / r.s, out.lp, 0.f) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    now = next;
  }
  if constexpr (MODE == POLICY) {
    if (t == 0)
#pragma unroll
      for (int k = 0; k < 8; ++k) sums[slot][k] = k < 6 ? sum[k] : 0.0;
    __syncthreads();
    if (threadIdx.x < 8) {
      double s = 0;
      for (int i = 0; i < 16; ++i) s += sums[i][threadIdx.x];
      a.partials[blockIdx.x * 8LL + threadIdx.x] = s;
    }
  }
}

// ---- few rows: every row cut into pieces, a workgroup each ----------------------------------------------------------
template <class D, Mode MODE, bool REF>
__global__ __launch_bounds__(256) void token_pieces_kernel(const RowArgs a) {
  __shared__ RowStats parts[2][4];
  const long long row = blockIdx.y;
  if ((a.mask && !a.mask[row]) || is_there(a.factor)) return;
  const int begin = blockIdx.x * a.piece, end = min(a.V, begin + a.piece);
  const char *z = a.z + row * a.z_pitch, *q = REF ? a.q + row * a.q_pitch : nullptr;
  RowStats r = kNothing;
  int turn = 0;
  add_columns<D, 256, REF>(r, z, q, a.V, begin, end, threadIdx.x);
  join_row<4, REF>(r, parts, turn);
  if (threadIdx.x == 0) {
    a.piece_stats[row * a.splits + blockIdx.x] = r;
    if (MODE == POLICY && blockIdx.x == 0) a.chosen[row] = action_logit<D>(z, a.actions[row], a.V);  // (the gradient may overwrite it)
  }
}

// the pieces of a row joined, in every lane of a wave
template <bool REF>
__device__ __forceinline__ RowStats join_pieces(const RowArgs &a, long long row) {
  RowStats r = kNothing;
  for (int i = threadIdx.x & 63; i < a.splits; i += 64) {
    const RowStats p = a.piece_stats[row * a.splits + i];
    RowStats q = p;
    raise_max(q, r.m);
    raise_max(r, p.m);
    if constexpr (REF) {
      raise_ref(q, r.mr);
      raise_ref(r, p.mr);
      r.sr += q.sr;
      r.gap += q.gap;
    }
    r.s += q.s;
    r.ed += q.ed;
  }
  join_wave<REF>(r);
  return r;
}

// the results of the rows, a wave per row
template <class D, Mode MODE>
__global__ __launch_bounds__(64) void token_join_kernel(const RowArgs a) {
  const int lane = threadIdx.x;
  const long long row = blockIdx.x;
  const bool keep = !a.mask || a.mask[row];
  float lp = 0.f, entropy = 0.f;
  float4 stats = make_float4(0.f, 0.f, 0.f, 0.f);
  if (keep) {
    const RowStats r = join_pieces<false>(a, row);
    const float log_s = logf(r.s);
    lp = (action_logit<D>(a.z + row * a.z_pitch, a.actions[row], a.V) - r.m) - log_s;
    entropy = log_s - r.ed / r.s;
    stats = make_float4(r.m, 1.f / r.s, lp, 0.f);
  }
  if (lane == 0) {
    if (MODE == LOGP) a.lp[row] = lp;
    if (MODE == LOGP && a.entropy) a.entropy[row] = entropy;
    if (MODE == STATS) a.stats[row] = stats;
  }
}

// the gradient of a piece; every workgroup joins its row's pieces itself (another launch would take longer), the first one of
// a row writes its results
template <class D, bool REF>
__global__ __launch_bounds__(256) void token_pieces_grad_kernel(const RowArgs a) {
  if (is_there(a.factor)) return;
  const long long row = blockIdx.y;
  const bool keep = !a.mask || a.mask[row];
  RowTerms out = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  RowPlan g = {};
  long long action = -1;
  if (keep) {
    const float w = row_weight<4>(a);
    const RowStats r = join_pieces<REF>(a, row);
    g = policy_row<REF>(a, r, a.chosen[row], a.old_lp[row], a.adv[row], a.ref_lp ? a.ref_lp[row] : 0.f, w, &out);
    action = a.actions[row];
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    if (a.lp) a.lp[row] = out.lp;
    const double all[8] = {out.policy, out.entropy, out.kl, out.outside, out.ratio, out.lp, 0.0, 0.0};
    for (int k = 0; k < 8; ++k) a.partials[row * 8 + k] = all[k];
  }
  const int begin = blockIdx.x * a.piece, end = min(a.V, begin + a.piece);
  const char *z = a.z + row * a.z_pitch, *q = REF ? a.q + row * a.q_pitch : nullptr;
  char *dz = a.dz + row * a.dz_pitch;
  write_columns<D, 256, REF>(z, q, dz, a.V, begin, end, threadIdx.x, keep,
                             [&](float x, float y, int col) { return grad_of<D, REF, true>(g, x, y) + (col == action ? g.at : 0.f); });
}

__global__ __launch_bounds__(1024) void mask_count_kernel(const uint8_t *mask, long long n, double *count, const float *factor) {
  if (is_there(factor)) return;
  const int c = count_rows<16>(mask, n);
  if (threadIdx.x == 0) *count = static_cast<double>(c);
}

// sums of `n` rows of eight doubles, in one fixed order: thread (i, k) of the T takes rows i, i + T / 8, ... of column k
template <int T>
__device__ void sum_partials(const double *partials, int n, double (&total)[8]) {
  constexpr int R = T / 8;
  __shared__ double acc[R][8];
  const int k = threadIdx.x & 7, i = threadIdx.x >> 3;
  double s = 0;
  for (int j = i; j < n; j += R) s += partials[j * 8LL + k];
  acc[i][k] = s;
  __syncthreads();
  for (int half = R / 2; half > 0; half >>= 1) {
    if (i < half) acc[i][k] += acc[i + half][k];
    __syncthreads();
  }
  for (int c = 0; c < 8; ++c) total[c] = acc[0][c];
}

__global__ __launch_bounds__(1024) void policy_terms_kernel(const double *partials, int n, const uint8_t *mask, const double *count,
                                                            long long rows, float kl_coef, float ent_coef, float *loss_out) {
  double s[8];
  const double c = !mask ? static_cast<double>(rows) : count ? *count : count_rows<16>(mask, rows);
  sum_partials<1024>(partials, n, s);
  if (threadIdx.x == 0) {
    const double inv = c > 0 ? 1.0 / c : 0.0;  // nothing unmasked: zeros
    loss_out[0] = static_cast<float>((s[0] - ent_coef * s[1] + (kl_coef != 0.f ? kl_coef * s[2] : 0.0)) * inv);
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

// the sum over a workgroup of T threads, in every thread
template <int T>
__device__ __forceinline__ double block_sum(double v) {
  __shared__ double scratch[T / 64];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0;
#pragma unroll
  for (int i = 0; i < T / 64; ++i) v += scratch[i];
  return v;
}

// this thread's share of a sum over rows begin .. end, eight of its rows on their way at a time (a row a round trip made one pair
// of two sequences of 131072 rows take 340 us)
template <int T, class F>
__device__ __forceinline__ double sum_rows(long long begin, long long end, F value) {
  constexpr int U = 8;
  double s = 0;
  long long i = begin + threadIdx.x;
  for (; i + (U - 1) * T < end; i += U * T) {
    float v[U];
#pragma unroll
    for (int k = 0; k < U; ++k) v[k] = value(i + k * T);
#pragma unroll
    for (int k = 0; k < U; ++k) s += v[k];
  }
  for (; i < end; i += T) s += value(i);
  return s;
}

// a workgroup per pair: the two sequences' log-probabilities, the pair's loss, and the coefficient of each of its rows
template <int T>
__global__ __launch_bounds__(T) void preference_pairs_kernel(const PairArgs a) {
  double sum[7] = {0, 0, 0, 0, 0, 0, 0};
  for (int pair = blockIdx.x; pair < a.pairs; pair += gridDim.x) {
    double lp[2];
    long long begin[2], end[2];
    for (int side = 0; side < 2; ++side) {
      const long long b = a.offsets[2LL * pair + side], e = a.offsets[2LL * pair + side + 1];
      begin[side] = b < 0 ? 0 : b;
      end[side] = e > a.rows ? a.rows : e;
      lp[side] = block_sum<T>(sum_rows<T>(begin[side], end[side], [&](long long i) { return a.stats[i].z; }));
    }
    const double chosen = a.beta * (lp[0] - (a.ref_lp ? a.ref_lp[2LL * pair] : 0.f));
    const double rejected = a.beta * (lp[1] - (a.ref_lp ? a.ref_lp[2LL * pair + 1] : 0.f));
    const double h = chosen - rejected;
    const double tail = log1p(exp(-fabs(h)));                     // -log sig(h) = max(-h, 0) + log(1 + e^-|h|)
    const double up = (h < 0 ? -h : 0.0) + tail, down = (h > 0 ? h : 0.0) + tail;
    const double slope = (a.smoothing / (1.0 + exp(-h)) - (1.0 - a.smoothing) / (1.0 + exp(h))) * a.beta / (a.batch > 0 ? a.batch : a.pairs);
    for (int side = 0; side < 2; ++side) {
      const float c = static_cast<float>(side ? -slope : slope);
#pragma unroll 4
      for (long long i = begin[side] + threadIdx.x; i < end[side]; i += T) {
        const bool keep = !a.mask || a.mask[i];
        a.stats[i].w = keep ? c : 0.f;
      }
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

// dz_j = c (1{j = a} - p_j) of every row, c the coefficient of its sequence (0: no sequence's, or masked).  T threads take a
// piece of a row; also the loss's terms (loss_out), by the first workgroup.
template <class D, int T>
__global__ __launch_bounds__(256) void preference_grad_kernel(const RowArgs a, long long blocks, int pairs, int pair_groups, float *loss_out) {
  constexpr int kRows = 256 / T;
  if (is_there(a.factor)) return;
  const int t = threadIdx.x % T, slot = threadIdx.x / T;
  if (loss_out && blockIdx.x == 0) {
    double s[8];
    sum_partials<256>(a.partials, pair_groups, s);
    if (threadIdx.x == 0) {
      for (int k = 0; k < 7; ++k) loss_out[k] = static_cast<float>(s[k] / pairs);
      loss_out[7] = static_cast<float>(pairs);
    }
  }
  for (long long block = blockIdx.x; block < blocks; block += gridDim.x) {
    // from the last row down: the end of the logits is what the statistics pass has left in the last-level cache
    const long long i = (block / a.splits) * kRows + slot;
    if (i >= a.rows) return;
    const long long row = a.rows - 1 - i;
    const int begin = static_cast<int>(block % a.splits) * a.piece, end = min(a.V, begin + a.piece);
    const float4 st = a.stats[row];
    char *dz = a.dz + row * a.dz_pitch;
    const char *z = a.z + row * a.z_pitch;
    const float c = a.factor ? st.w * *a.factor : st.w, k = -c * st.y;
    const long long action = c != 0.f ? a.actions[row] : -1;
    write_columns<D, T, false>(z, nullptr, dz, a.V, begin, end, t, c != 0.f,
                               [&](float x, float, int col) { return k * exp_of(x - st.x) + (col == action ? c : 0.f); });
  }
}

// log-probabilities of sequences: a workgroup per sequence
template <int T>
__global__ __launch_bounds__(T) void sequence_sum_kernel(const float *lp, const int32_t *offsets, long long rows, int sequences, float *out) {
  for (int q = blockIdx.x; q < sequences; q += gridDim.x) {
    const long long b = offsets[q] < 0 ? 0 : offsets[q], e = offsets[q + 1] > rows ? rows : offsets[q + 1];
    const double s = block_sum<T>(sum_rows<T>(b, e, [&](long long i) { return lp[i]; }));
    if (threadIdx.x == 0) out[q] = static_cast<float>(s);
  }
}

// x *= *factor in place, nothing at all when it is 1 (the gradient of a loss that is differentiated as it stands)
template <class D>
__global__ __launch_bounds__(256) void scale_rows_kernel(char *x, long long pitch, long long rows, int V, const float *factor) {
  const float f = *factor;
  if (f == 1.f) return;
  for (long long row = blockIdx.x; row < rows; row += gridDim.x)
    write_columns<D, 256, false>(x + row * pitch, nullptr, x + row * pitch, V, 0, V, threadIdx.x, true,
                                 [&](float v, float, int) { return v * f; });
}

// sequences that are worth 1024 threads each instead of 256 (a masked preference loss of 18 columns, us with 256 / 1024 threads: one
// pair of 8192 rows each 32.8 / 27.7, of 131072 466 / 270; four of 2048 21.4 / 22.2, 1024 of 8 23.3 / 45.7)
inline bool long_sequences(long long rows, long long sequences) { return rows / sequences >= 8192; }

inline int elem_size(int dtype) { return dtype == DX_F32 ? 4 : 2; }

// Threads per row T and vectors of 16 bytes a thread holds of it, NV (0: none, or too many for the registers).
struct RowShape { int T, NV; };
RowShape row_shape(int V, int dtype, bool ref, bool once, bool few) {
  const long long vectors = (static_cast<long long>(V) * elem_size(dtype) + 15) / 16;
  if (vectors <= 64) return {16, vectors <= 16 ? 1 : 4};
  if (vectors <= 64 * 8) return {64, vectors <= 64 * 4 ? 4 : 8};
  // to 16 KB a wave a row too, but for read-once rows of many columns (16384 rows bf16, us with 64 / 256 threads a row: policy loss of
  // 4099 columns 78 / 87, 8192 122 / 125; log-probabilities of 4099 35 / 47, 5000 43 / 46, 6500 53 / 51, 8192 68 / 52)
  if (!ref && vectors <= 64 * 16 && (!once || V <= 5120)) return {64, 16};
  // read once anyway: many rows to a CU, or, where there are no more rows than CUs, many threads to a row (32 x 32768 f32 log-
  // probabilities: 6.0 us with 1024 threads, 7.6 with 256; 32 x 12000 bf16 4.7, 5.0; shorter ones alike)
  if (once) return {few && vectors > 1024 ? 1024 : 256, 0};
  const int most = ref ? 8 : 16;  // two rows are held where there are reference logits
  if (vectors <= 256 * most) return {256, vectors <= 256 * 4 ? 4 : vectors <= 256 * 8 ? 8 : 16};
  if (vectors <= 512 * most) return {512, most};
  if (vectors <= 1024 * most) return {1024, most};
  return {1024, 0};
}

template <class D, Mode MODE, bool REF, bool ENT>
int launch_rows(const RowArgs &a, RowShape sh, int grid, hipStream_t s) {
#define DX_ROWS(TT, NN)                                                                                                       \
  if (sh.T == (TT) && sh.NV == (NN)) {                                                                                            \
    hipLaunchKernelGGL((token_rows_kernel<D, (TT), (NN), MODE, REF, ENT>), dim3(grid), dim3((TT) < 256 ? 256 : (TT)), 0, s, a);   \
    DX_LAUNCH_CHECK();                                                                                                        \
    return DX_OK;                                                                                                             \
  }
  if (sh.T == 16) {
    if (sh.NV == 1) hipLaunchKernelGGL((token_short_kernel<D, 1, MODE, REF, ENT>), dim3(grid), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((token_short_kernel<D, 4, MODE, REF, ENT>), dim3(grid), dim3(256), 0, s, a);
    DX_LAUNCH_CHECK();
    return DX_OK;
  }
  DX_ROWS(64, 4)
  DX_ROWS(64, 8)
  if constexpr (!REF) DX_ROWS(64, 16)
  if constexpr (MODE != POLICY) {
    DX_ROWS(256, 0)
    DX_ROWS(1024, 0)
  } else {
    if constexpr (REF) DX_ROWS(256, 4)
    DX_ROWS(256, 8)
    if constexpr (!REF) DX_ROWS(256, 16)
    DX_ROWS(512, REF ? 8 : 16)
    DX_ROWS(1024, REF ? 8 : 16)
    DX_ROWS(1024, 0)
  }
#undef DX_ROWS
  return dx::fail(DX_ENOSUP, "token rows: no kernel for %d threads, %d vectors", sh.T, sh.NV);
}
template <class D>
int launch_pref_grad(const RowArgs &a, int T, long long blocks, int pairs, int pair_groups, float *loss_out, hipStream_t s) {
  // one workgroup at least, which writes the terms; fewer than 2^32 threads, the most of a launch
  const dim3 grid(static_cast<unsigned>(blocks < 1 ? 1 : blocks < (1 << 23) ? blocks : 1 << 23));
  if (T == 16) hipLaunchKernelGGL((preference_grad_kernel<D, 16>), grid, dim3(256), 0, s, a, blocks, pairs, pair_groups, loss_out);
  else if (T == 64) hipLaunchKernelGGL((preference_grad_kernel<D, 64>), grid, dim3(256), 0, s, a, blocks, pairs, pair_groups, loss_out);
  else hipLaunchKernelGGL((preference_grad_kernel<D, 256>), grid, dim3(256), 0, s, a, blocks, pairs, pair_groups, loss_out);
  DX_LAUNCH_CHECK();
  return DX_OK;
}

// Rows -> statistics (LOGP, STATS: results too) or the whole policy loss.  `*groups`: rows of `partials` that were written.
// Few long rows are cut into pieces over the CUs and joined by a second launch: long is what a CU takes longer for than the
// launches cost (its exponentials bound it, so columns count, not bytes).  32 rows of bf16, GPU us / us with the host's part,
// whole and in pieces: log-probabilities of 32768 columns 5.8 / 10.5, 6.0 / 13.1; of 65536 8.0 / 9.9, 6.1 / 13.0; of 131072
// 12.3 / 12.7, 6.9 / 13.3; policy loss of 16384 11.3 / 17.3, 9 / 19.5; of 32768 14.7 / 17.6, 9.2 / 19.6; of 131072 26 / 26, 12 / 19.6.
template <class D, Mode MODE, bool REF, bool ENT>
int run_rows(RowArgs a, int dtype, int *groups, hipStream_t s) {
  int cus = 0;
  if (int rc = dx::device_cus(&cus)) return rc;
  const long long bytes = static_cast<long long>(a.V) * elem_size(dtype);
  if (a.rows <= kMaxPieces / 2 && a.V > (MODE == POLICY ? 16384 : 32768) && a.rows * 2 <= cus) {
    long long splits = cus / a.rows, most = (bytes + 8191) / 8192;
    if (splits > most) splits = most;
    if (splits * a.rows > kMaxPieces) splits = kMaxPieces / a.rows;
    a.piece = static_cast<int>((a.V + splits - 1) / splits + 2047) / 2048 * 2048;
    a.splits = (a.V + a.piece - 1) / a.piece;
    if (a.splits > 1) {
      const dim3 grid(a.splits, static_cast<unsigned>(a.rows));
      hipLaunchKernelGGL((token_pieces_kernel<D, MODE, REF>), grid, dim3(256), 0, s, a);
      DX_LAUNCH_CHECK();
      if constexpr (MODE == POLICY) hipLaunchKernelGGL((token_pieces_grad_kernel<D, REF>), grid, dim3(256), 0, s, a);
      else hipLaunchKernelGGL((token_join_kernel<D, MODE>), dim3(static_cast<unsigned>(a.rows)), dim3(64), 0, s, a);
      DX_LAUNCH_CHECK();
      *groups = static_cast<int>(a.rows);
      return DX_OK;
    }
  }
  const RowShape sh = row_shape(a.V, dtype, REF, MODE != POLICY, a.rows <= cus);
  const long long need = sh.T < 256 ? (a.rows + 256 / sh.T - 1) / (256 / sh.T) : a.rows;
  // POLICY: resident workgroups, which prefetch their next row (1024 threads fill a CU).  Read once: as many as there are 64 KB
  // pieces, as masked rows would leave resident ones with unequal shares (8192 rows of 64 KB, a fifth masked: 96 us, 81 so).
  long long most = sh.T == 1024 ? cus : sh.T == 512 ? 2LL * cus : 8LL * cus < kMaxWorkers ? 8LL * cus : kMaxWorkers;
  if (MODE != POLICY && most < a.rows * bytes / 65536) most = a.rows * bytes / 65536;
  const int grid = static_cast<int>(need < most ? need : most);
  *groups = grid;
  if (grid == 0) return DX_OK;
  return launch_rows<D, MODE, REF, ENT>(a, sh, grid, s);
}
template <class D>
int run_policy(const RowArgs &a, int dtype, int *groups, hipStream_t s) {
  if (a.q) return run_rows<D, POLICY, true, true>(a, dtype, groups, s);
  if (a.ent_coef != 0.f) return run_rows<D, POLICY, false, true>(a, dtype, groups, s);
  return run_rows<D, POLICY, false, false>(a, dtype, groups, s);
}
template <Mode MODE>
int run_stats(const RowArgs &a, int dtype, hipStream_t s) {
  int groups = 0;
  if (dtype == DX_F32) return run_rows<ElemF32, MODE, false, false>(a, dtype, &groups, s);
  if (dtype == DX_BF16) return run_rows<ElemBF16, MODE, false, false>(a, dtype, &groups, s);
  return run_rows<ElemF16, MODE, false, false>(a, dtype, &groups, s);
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

// the gradient of the preference loss from its rows' statistics
int preference_grad(RowArgs a, int dtype, int pairs, int pair_groups, float *loss_out, hipStream_t s) {
  // gradient: 16 lanes or a wave per short row, else a workgroup per piece of 32 KB of a row (the whole loss of 262144 rows, us with
  // 64 / 16 lanes: 18 columns f32 204 / 160, 128 213 / 186, 250 255 / 301)
  const long long bytes = static_cast<long long>(a.V) * elem_size(dtype);
  const int T = bytes <= 512 ? 16 : bytes <= 4096 ? 64 : 256;
  a.piece = T < 256 ? a.V : 32768 / elem_size(dtype);
  a.splits = (a.V - 1) / a.piece + 1;
  const long long blocks = (a.rows + 256 / T - 1) / (256 / T) * a.splits;
  if (dtype == DX_F32) return launch_pref_grad<ElemF32>(a, T, blocks, pairs, pair_groups, loss_out, s);
  if (dtype == DX_BF16) return launch_pref_grad<ElemBF16>(a, T, blocks, pairs, pair_groups, loss_out, s);
  return launch_pref_grad<ElemF16>(a, T, blocks, pairs, pair_groups, loss_out, s);
}

// workspace, in doubles: 8 for the count, 8 a workgroup for its sums, the pieces' statistics and their rows' chosen logits
constexpr int kPartialsAt = 8, kPiecesAt = 8 + 8 * kMaxWorkers, kChosenAt = kPiecesAt + kMaxPieces * 3;
static_assert(sizeof(RowStats) == 24 && kChosenAt + kMaxPieces / 4 == DX_TOKEN_WORKSPACE, "workspace");

RowArgs row_args(const void *logits, int dtype, long long rows, int vocab, long long pitch, const int64_t *actions, const uint8_t *mask,
                 double *workspace) {
  RowArgs a{};
  a.splits = 1;
  if (workspace) {
    a.count = workspace;
    a.partials = workspace + kPartialsAt;
    a.piece_stats = reinterpret_cast<RowStats *>(workspace + kPiecesAt);
    a.chosen = reinterpret_cast<float *>(workspace + kChosenAt);
  }
  const int size = elem_size(dtype);
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
                                 const uint8_t *mask, float *log_prob, float *entropy, double *workspace, long long workspace_count,
                                 void *stream) {
  DX_TRACE("dx_token_log_prob");
  if (int rc = check_logits("dx_token_log_prob", logits, dtype, rows, vocab, pitch, actions)) return rc;
  if (rows == 0) return DX_OK;
  DX_REQUIRE(log_prob != nullptr && workspace != nullptr, "dx_token_log_prob: null pointer");
  if (workspace_count < DX_TOKEN_WORKSPACE)
    return dx::fail(DX_EWS, "dx_token_log_prob: workspace of %lld doubles, %d needed", workspace_count, DX_TOKEN_WORKSPACE);
  RowArgs a = row_args(logits, dtype, rows, vocab, pitch, actions, mask, workspace);
  a.lp = log_prob;
  a.entropy = entropy;
  return run_stats<LOGP>(a, dtype, dx::as_stream(stream));
}

extern "C" int dx_sequence_log_prob(const float *token_log_prob, const int32_t *offsets, long long rows, int sequences, float *out,
                                    void *stream) {
  DX_TRACE("dx_sequence_log_prob");
  DX_REQUIRE(rows >= 0 && sequences >= 0, "dx_sequence_log_prob: negative shape");
  if (sequences == 0) return DX_OK;
  DX_REQUIRE((token_log_prob || rows == 0) && offsets && out, "dx_sequence_log_prob: null pointer");
  const dim3 grid(sequences < kMaxWorkers ? sequences : kMaxWorkers);
  hipStream_t s = dx::as_stream(stream);
  if (long_sequences(rows, sequences)) hipLaunchKernelGGL(sequence_sum_kernel<1024>, grid, dim3(1024), 0, s, token_log_prob, offsets, rows, sequences, out);
  else hipLaunchKernelGGL(sequence_sum_kernel<256>, grid, dim3(256), 0, s, token_log_prob, offsets, rows, sequences, out);
  DX_LAUNCH_CHECK();
  return DX_OK;
}

namespace {

// the policy loss (loss_out), or its gradient alone times *factor
int policy_loss(const char *who, const void *logits, int dtype, long long rows, int vocab, long long pitch, const int64_t *actions,
                const float *old_log_prob, const float *advantages, const float *ref_log_prob, const void *ref_logits, long long ref_pitch,
                const uint8_t *mask, float cliprange, float kl_coef, float entropy_coef, long long global_batch, void *dlogits,
                long long dlogits_pitch, float *log_prob, double *workspace, long long workspace_count, const float *factor, float *loss_out,
                void *stream) {
  if (int rc = check_logits(who, logits, dtype, rows, vocab, pitch, actions)) return rc;
  DX_REQUIRE((loss_out || factor) && workspace != nullptr, "%s: null pointer", who);
  DX_REQUIRE(rows == 0 || (old_log_prob && advantages && dlogits && (log_prob || factor)), "%s: null pointer", who);
  DX_REQUIRE(!(ref_log_prob && ref_logits), "%s: give ref_log_prob or ref_logits, not both", who);
  DX_REQUIRE(rows <= 1 || dlogits_pitch >= vocab, "%s: rows of dlogits overlap", who);
  DX_REQUIRE(!ref_logits || rows <= 1 || ref_pitch >= vocab, "%s: rows of ref_logits overlap", who);
  DX_REQUIRE(dx::aligned(dlogits, dtype == DX_F32 ? 4 : 2) && dx::aligned(ref_logits, dtype == DX_F32 ? 4 : 2),
             "%s: dlogits / ref_logits are not aligned to their type", who);
  DX_REQUIRE(!factor || rows == 0 || dlogits != logits, "%s: the logits are read again, dlogits must not be they", who);
  if (workspace_count < DX_TOKEN_WORKSPACE)
    return dx::fail(DX_EWS, "%s: workspace of %lld doubles, %d needed", who, workspace_count, DX_TOKEN_WORKSPACE);
  hipStream_t s = dx::as_stream(stream);
  RowArgs a = row_args(logits, dtype, rows, vocab, pitch, actions, mask, workspace);
  const int size = elem_size(dtype);
  a.q = static_cast<const char *>(ref_logits);
  a.q_pitch = ref_pitch * size;
  a.dz = static_cast<char *>(dlogits);
  a.dz_pitch = dlogits_pitch * size;
  a.old_lp = old_log_prob;
  a.adv = advantages;
  a.ref_lp = ref_log_prob;
  a.lp = log_prob;
  a.batch = global_batch > 0 ? static_cast<double>(global_batch) : 0.0;
  a.cliprange = cliprange;
  a.kl_coef = kl_coef;
  a.ent_coef = entropy_coef;
  a.factor = factor;
  if (rows <= kCountedHere) a.count = nullptr;
  else if (mask) {
    hipLaunchKernelGGL(mask_count_kernel, dim3(1), dim3(1024), 0, s, mask, rows, workspace, factor);
    DX_LAUNCH_CHECK();
  }
  int groups = 0;
  if (rows > 0)
    if (int rc = dtype == DX_F32 ? run_policy<ElemF32>(a, dtype, &groups, s)
                 : dtype == DX_BF16 ? run_policy<ElemBF16>(a, dtype, &groups, s) : run_policy<ElemF16>(a, dtype, &groups, s)) return rc;
  if (!loss_out) return DX_OK;
  hipLaunchKernelGGL(policy_terms_kernel, dim3(1), dim3(1024), 0, s, a.partials, groups, mask, a.count, rows, kl_coef, entropy_coef,
                     loss_out);
  DX_LAUNCH_CHECK();
  return DX_OK;
}

}  // namespace

extern "C" int dx_token_policy_loss(const void *logits, int dtype, long long rows, int vocab, long long pitch, const int64_t *actions,
                                    const float *old_log_prob, const float *advantages, const float *ref_log_prob,
                                    const void *ref_logits, long long ref_pitch, const uint8_t *mask, float cliprange, float kl_coef,
                                    float entropy_coef, long long global_batch, void *dlogits, long long dlogits_pitch,
                                    float *log_prob, double *workspace, long long workspace_count, float *loss_out, void *stream) {
  DX_TRACE("dx_token_policy_loss");
  DX_REQUIRE(loss_out != nullptr, "dx_token_policy_loss: null pointer");
  return policy_loss("dx_token_policy_loss", logits, dtype, rows, vocab, pitch, actions, old_log_prob, advantages, ref_log_prob, ref_logits,
                     ref_pitch, mask, cliprange, kl_coef, entropy_coef, global_batch, dlogits, dlogits_pitch, log_prob, workspace,
                     workspace_count, nullptr, loss_out, stream);
}

extern "C" int dx_token_policy_grad_scaled(const void *logits, int dtype, long long rows, int vocab, long long pitch, const int64_t *actions,
                                           const float *old_log_prob, const float *advantages, const float *ref_log_prob,
                                           const void *ref_logits, long long ref_pitch, const uint8_t *mask, float cliprange, float kl_coef,
                                           float entropy_coef, long long global_batch, void *dlogits, long long dlogits_pitch,
                                           double *workspace, long long workspace_count, const float *factor, void *stream) {
  DX_TRACE("dx_token_policy_grad_scaled");
  DX_REQUIRE(factor != nullptr, "dx_token_policy_grad_scaled: null pointer");
  return policy_loss("dx_token_policy_grad_scaled", logits, dtype, rows, vocab, pitch, actions, old_log_prob, advantages, ref_log_prob,
                     ref_logits, ref_pitch, mask, cliprange, kl_coef, entropy_coef, global_batch, dlogits, dlogits_pitch, nullptr, workspace,
                     workspace_count, factor, nullptr, stream);
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
  RowArgs a = row_args(logits, dtype, rows, vocab, pitch, actions, mask, workspace);
  a.stats = reinterpret_cast<float4 *>(row_stats);
  a.dz = static_cast<char *>(dlogits);
  a.dz_pitch = dlogits_pitch * elem_size(dtype);
  if (rows > 0)
    if (int rc = run_stats<STATS>(a, dtype, s)) return rc;
  PairArgs p{a.stats, offsets, ref_log_prob, mask, rows, pairs, global_pairs > 0 ? static_cast<double>(global_pairs) : 0.0, beta,
             label_smoothing, sequence_log_prob, a.partials};
  const int pair_groups = pairs < kMaxWorkers ? pairs : kMaxWorkers;
  if (long_sequences(rows, 2LL * pairs)) hipLaunchKernelGGL(preference_pairs_kernel<1024>, dim3(pair_groups), dim3(1024), 0, s, p);
  else hipLaunchKernelGGL(preference_pairs_kernel<256>, dim3(pair_groups), dim3(256), 0, s, p);
  DX_LAUNCH_CHECK();
  return preference_grad(a, dtype, pairs, pair_groups, loss_out, s);
}

extern "C" int dx_preference_grad_scaled(const void *logits, int dtype, long long rows, int vocab, long long pitch, const int64_t *actions,
                                         const float *row_stats, void *dlogits, long long dlogits_pitch, const float *factor, void *stream) {
  DX_TRACE("dx_preference_grad_scaled");
  if (int rc = check_logits("dx_preference_grad_scaled", logits, dtype, rows, vocab, pitch, actions)) return rc;
  if (rows == 0) return DX_OK;
  DX_REQUIRE(row_stats && dlogits && factor, "dx_preference_grad_scaled: null pointer");
  DX_REQUIRE(rows <= 1 || dlogits_pitch >= vocab, "dx_preference_grad_scaled: rows of dlogits overlap");
  DX_REQUIRE(dx::aligned(dlogits, dtype == DX_F32 ? 4 : 2) && dx::aligned(row_stats, 16), "dx_preference_grad_scaled: misaligned dlogits / row_stats");
  DX_REQUIRE(dlogits != logits, "dx_preference_grad_scaled: the logits are read again, dlogits must not be they");
  RowArgs a = row_args(logits, dtype, rows, vocab, pitch, actions, nullptr, nullptr);
  a.stats = reinterpret_cast<float4 *>(const_cast<float *>(row_stats));  // (read only)
  a.dz = static_cast<char *>(dlogits);
  a.dz_pitch = dlogits_pitch * elem_size(dtype);
  a.factor = factor;
  return preference_grad(a, dtype, 0, 0, nullptr, dx::as_stream(stream));
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
