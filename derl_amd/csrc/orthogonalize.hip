// Newton-Schulz orthogonalisation of an update (gfx950):
//   X0 = G / (|G|_F + eps),   A = X X^T,   X <- a X + (b A + c A^2) X        (`steps` times)
// with X the (r, c) matrix whose shorter side is r (a tall G is worked on transposed).  Odd polynomials of the singular
// values only: the singular vectors stay G's, the singular values approach 1.
//
// The products run on the fp16 matrix cores with fp32 accumulation.  Whatever the matrix's type, X, A and M below are held as TWO fp16
// terms, hi + lo (22 bits): a product is hi hi + hi lo + lo hi (the dropped lo lo is 2^-22 of it), fp32 accuracy at a third of the
// fp16 rate, where the fp32 matrix instructions have a sixteenth.  (bf16 too: with one term, 11 bits, each step multiplies what
// is lost by up to `a` = 3.4, and a bf16 result was off by 1.1 to 2.5 times its own rounding; with two it is off by that alone.)
// fp16 has few exponents, so what is stored in it is scaled, by powers of two, such that EVERY row of an operand lies in its upper
// range: rows of X by the exponent E_i of a bound of their norms, of X^T by F_n, of A and M = b A + c A^2 (whose rows are bounded by
// |x_i|) by E_i as well.  A row of a product is then as accurate as its own size allows, however small it is against the others
// (256 x 512 Gaussian, 32 rows x 1e-6: those rows are off by 2e-7 after 5 steps; with one scale for the whole matrix 1.5e-3).  The
// bounds are exact: a step maps a row x_i = sum_k U_ik s_k v_k to sum_k U_ik q(s_k^2) s_k v_k, so its norm grows by max |q| at most,
// q(t) = a + b t + c t^2, over the singular values there can be (`grown`).  The update is X' = a X + M X with X, and b A of M, from
// fp32 copies, so that what the polynomial leaves alone (small singular values: q = a) passes a step with one rounding.
//
// Every matrix product is C = P Q^T with both operands' k contiguous: X for A = X X^T, A = A^T for A^2 = A A^T, and for
// M X the transposed copy X^T, which the epilogue of each update writes beside X.  A and M are symmetric: only tiles on
// and above the diagonal are formed and stored twice.  Both sides are padded
// to a multiple of 64 with zeros in the workspace.
#include <cmath>
#include <type_traits>

#include "igemm_dev.hpp"

namespace dx {
namespace {

using f32x4 = __attribute__((ext_vector_type(4))) float;
using i32x4 = __attribute__((ext_vector_type(4))) int;
using u32x2 = __attribute__((ext_vector_type(2))) uint32_t;
using u32x4 = __attribute__((ext_vector_type(4))) uint32_t;
using f16x4 = __attribute__((ext_vector_type(4))) _Float16;
using f16x8 = __attribute__((ext_vector_type(8))) _Float16;

constexpr int kTop = 14;         // rows of an operand are scaled to norms below 2^kTop
constexpr int kLowest = -160;    // exponent of a bound of 0
constexpr int kPad = 64, kScanParts = 64;
constexpr int kSplitGroups = 512;  // workgroups of a product that is split over K, at most

constexpr int kStageK = 32;        // k of a stage of a product

enum Epilogue { GRAM, POLY, UPDATE, FINAL };

// the least power of two above x >= 0 (NaN, infinities: 2^128)
__host__ __device__ inline int power_above(float x) {
  if (!(x < 3.4e38f)) return 128;
  if (x == 0.f) return kLowest;
  const float y = x < 1.18e-38f ? x * 0x1p64f : x;  // (a denormal number's exponent is not in its bits)
  return static_cast<int>(__builtin_bit_cast(uint32_t, y) >> 23) - (x < 1.18e-38f ? 190 : 126);
}
// What is known of X before a step: its singular values are at most `top` < 2^cap, a row or column at most 2^shift times what it
// was at the start; |b + c t| < 2^poly for their squares t.  2^E for a row that began below 2^e: E = min(e + shift, cap).
// A polynomial that grows beyond 1 makes the largest value there can be explode, where the matrix's own may be far below: it is
// taken to stay within 8, or within what `a` alone makes of it (`linear`), whichever is more.
struct Powers { short shift, cap, poly; };
struct Known : Powers {
  float top, linear;
};
inline float larger(float x, float y) { return x > y || x != x ? x : y; }
inline float size_of(float x) { return x < 0.f ? -x : x; }
inline Known known_of(float top, float linear, int shift, float b, float c) {
  const float t = top * top;
  Known k;
  k.top = top;
  k.linear = linear;
  k.shift = static_cast<short>(shift < -1000 ? -1000 : shift > 1000 ? 1000 : shift);
  k.cap = static_cast<short>(power_above(top));
  k.poly = static_cast<short>(power_above(larger(size_of(b), size_of(b + c * t))));
  return k;
}
inline Known known_at_start(float b, float c) { return known_of(1.01f, 1.01f, 0, b, c); }  // (|X0|_F <= 1, rounded)
inline Known grown(const Known &k, float a, float b, float c) {
  const float t = k.top * k.top;
  auto q = [&](float x) { return size_of(a + (b + c * x) * x); };
  float growth = larger(q(0.f), q(t)), top = k.top * q(t);
  const float vertex = -b / (2.f * c);
  if (vertex > 0.f && vertex < t) growth = larger(growth, q(vertex));
  // s q(s^2) is extreme where a + 3 b t + 5 c t^2 = 0
  const float inner = 9.f * b * b - 20.f * a * c, root = inner > 0.f ? sqrtf(inner) : 0.f, w = -0.5f * (3.f * b + (b < 0.f ? -root : root));
  for (int i = 0; i < 2; ++i) {
    const float at = i ? a / w : w / (5.f * c);
    if (at > 0.f && at < t) top = larger(top, sqrtf(at) * q(at));
  }
  // the values are rounded: nothing shrinks below the rounding of what it is the difference of
  const float terms = (size_of(a) + (size_of(b) + size_of(c) * t) * t) * 3.8e-6f;
  growth = 1.01f * larger(growth, terms);
  top = 1.01f * larger(top, terms * k.top);
  const float linear = 1.01f * k.linear * size_of(a), limit = linear > 8.f ? linear : 8.f;
  top = top < limit ? top : limit;
  return known_of(top, linear, k.shift + power_above(growth), b, c);
}
__device__ __forceinline__ int bound_of(int start, int shift, int cap) { return min(start + shift, cap); }
__device__ __forceinline__ float times_power(float x, int e) { return __builtin_amdgcn_ldexpf(x, e); }

// A matrix: rows of 2 ld halves, each 32 values' first terms followed by their second ones, so that a cache line holds both
// terms of 32 k.
__device__ __forceinline__ long long place(long long row, int col, int ld) { return row * 2 * ld + (col >> 5) * 64 + (col & 31); }
constexpr int kSecond = 32;  // from a value's first term to its second

struct NsArgs {
  const _Float16 *P, *Q;  // operands: rows of K values
  long long p_stride, q_stride;  // halves from one matrix of the batch to the next
  int ldp, ldq, K;
  int rows_p, rows_q;     // rows of P / Q, multiples of kPad
  int tiles_m, tiles_n;   // tiles of TM rows of them
  _Float16 *D, *DT;       // [m][n] and its transpose [n][m]
  long long d_stride, dt_stride;
  int ldd, lddt;
  // exponents of the bounds that rows m and columns n began with; what is known now and, for UPDATE, behind the step
  const int *exp_m, *exp_n;
  int exp_m_stride, exp_n_stride;
  int shift, cap, poly, next_shift, next_cap;
  // fp32 values (A: written by GRAM, read by POLY; X), in blocks of 32 x 32 as the accumulators hold them: float4 64 g + lane of
  // block n / 32 * rows_p / 32 + m / 32 is a lane's rows 8 g + ..
  float *master;
  long long master_stride;
  float a, b, c;
  // split K: `splits` workgroups a tile, each over `split_stages` stages; their sums, and a count of arrivals per tile
  int splits, split_stages;
  float *partials;
  long long split_floats;  // of `partials`
  unsigned *arrivals;
  // FINAL
  void *out;
  int dtype, r, cols, tall;
};

// two fp16 values of consecutive rows and their successors: d0 = (row 0, row 1), d1 = (row 2, row 3) of this lane's column.
// Transposed over the four lanes of a quad: lane j ends with row j of the quad's four columns.
struct Pair2 { uint32_t x, y; };
template <int CTRL>
__device__ __forceinline__ uint32_t quad_move(uint32_t v) {
  return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ Pair2 quad_transpose(uint32_t d0, uint32_t d1, int lane) {
  const uint32_t pick = lane & 1 ? 0x03020706u : 0x05040100u;  // the pair's rows 0 / 2 in the even lane, 1 / 3 in the odd one
  const uint32_t a0 = __builtin_amdgcn_perm(quad_move<0xB1>(d0), d0, pick), a1 = __builtin_amdgcn_perm(quad_move<0xB1>(d1), d1, pick);
  const bool high = lane & 2;
  const uint32_t other = quad_move<0x4E>(high ? a0 : a1);
  return high ? Pair2{other, a1} : Pair2{a0, other};
}
// (x, y) of a lane and of lane ^ 32 -> both halves' x in the lower lane, both halves' y in the upper one (inline asm: hipcc
// folds the builtin's results where an operand is uniform)
__device__ __forceinline__ void swap_halves(uint32_t &x, uint32_t &y) {
  asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(x), "+v"(y));
}

// four results of the last step, rows m .. m + 3 of column n, to the caller's matrix (which may start at any element);
// quad: the first column of this lane's quad
__device__ __forceinline__ void put_final(const NsArgs &a, int z, int m, int n, int quad, int lane, const float (&v)[4]) {
  typedef f32x4 Loose4 __attribute__((aligned(4)));
  typedef u32x2 Loose2 __attribute__((aligned(2)));
  const long long base = static_cast<long long>(z) * a.r * a.cols;
  if (a.dtype == DX_F32) {
    float *out = static_cast<float *>(a.out) + base;
    if (a.tall && m + 3 < a.r && n < a.cols) {
      *reinterpret_cast<Loose4 *>(out + static_cast<long long>(n) * a.r + m) = f32x4{v[0], v[1], v[2], v[3]};
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (m + k < a.r && n < a.cols) out[a.tall ? static_cast<long long>(n) * a.r + m + k : static_cast<long long>(m + k) * a.cols + n] = v[k];
    }
    return;
  }
  uint16_t *out = static_cast<uint16_t *>(a.out) + base, bits[4];
#pragma unroll
  for (int k = 0; k < 4; ++k)
    bits[k] = a.dtype == DX_BF16 ? __builtin_bit_cast(uint16_t, static_cast<__bf16>(v[k])) : __builtin_bit_cast(uint16_t, static_cast<_Float16>(v[k]));
  const uint32_t d0 = bits[0] | static_cast<uint32_t>(bits[1]) << 16, d1 = bits[2] | static_cast<uint32_t>(bits[3]) << 16;
  if (a.tall) {
    if (n >= a.cols) return;
    if (m + 3 < a.r) *reinterpret_cast<Loose2 *>(out + static_cast<long long>(n) * a.r + m) = u32x2{d0, d1};
    else
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (m + k < a.r) out[static_cast<long long>(n) * a.r + m + k] = bits[k];
    return;
  }
  const Pair2 t = quad_transpose(d0, d1, lane);  // row m + lane % 4, columns quad .. quad + 3
  const int row = m + (lane & 3);
  if (row >= a.r) return;
  uint16_t *to = out + static_cast<long long>(row) * a.cols + quad;
  if (quad + 3 < a.cols) *reinterpret_cast<Loose2 *>(to) = u32x2{t.x, t.y};
  else
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (quad + k < a.cols) to[k] = static_cast<uint16_t>((k < 2 ? t.x : t.y) >> (k & 1) * 16);
}

// WR x WC waves, each FM x FN tiles of 32 x 32 x 16 instructions; K stages of 32, a ring of RING in LDS filled by LDS-DMA.
// A row of a stage is 128 bytes -- one cache line: a CU has about 64 requests to the L2 in flight, and with rows of 64 bytes
// half of what they can carry bounded the copies (4096^3, of one term: 143 us, 120 with whole lines).  Slot s of row R
// holds the row's 16-byte chunk s ^ ((R >> 1) & 7), so that the 16 lanes of a ds_read_b128 group meet every bank once; the
// swizzle is applied to the source address, the DMA writes LDS linearly.
// One barrier per stage, in front of its last 16 k, whose fragments are in registers by then: behind it the stage's slot is
// free and is filled again, and the next stage has landed everywhere, so that its first fragments are read in the shadow of
// the last products: the matrix pipe does not wait at the barrier.  Rows past the matrix repeat its last row and are not stored.
template <int TM, int WR, int WC, int RING, Epilogue EPI>
__global__ __launch_bounds__(WR * WC * 64) void ns_gemm_kernel(const NsArgs a) {
  extern __shared__ __attribute__((aligned(16))) float smem[];
  constexpr int kWaves = WR * WC, FM = TM / WR / 32, FN = TM / WC / 32;
  constexpr int kArray = TM * 128;               // bytes of a stage's lines of every row of P, or of Q
  constexpr int kStage = 2 * kArray;
  constexpr int NP = TM / 8 / kWaves;            // 1 KiB pieces (8 rows) of an array that a wave copies
  constexpr int kPieces = 2 * NP;
  static_assert(NP * 8 * kWaves == TM && FM * 32 * WR == TM && FN * 32 * WC == TM, "tile");
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int z = blockIdx.y;
  int bm, bn, split;
  {
    // consecutive workgroups go to the eight XCDs in turn: each XCD takes a contiguous run of tiles
    const int splits = (EPI == GRAM || EPI == POLY) && TM <= 128 ? a.splits : 1, total = gridDim.x / splits, per = (total + 7) / 8, full = total - 8 * (per - 1);  // XCDs 0 .. full - 1 hold `per` tiles
    const int id = blockIdx.x / splits, xcd = id & 7, k = id >> 3;
    split = blockIdx.x - id * splits;
    int left = xcd * per - (xcd > full ? xcd - full : 0) + k;
    if (EPI == GRAM || EPI == POLY) {  // the upper triangle, row by row
      int row = 0;
      while (left >= a.tiles_m - row) left -= a.tiles_m - row++;
      bm = row;
      bn = row + left;
    } else {  // bands of four tile rows, column by column
      const int band = left / (4 * a.tiles_n), rows = min(4, a.tiles_m - 4 * band);
      left -= band * 4 * a.tiles_n;
      bn = left / rows;
      bm = 4 * band + left % rows;
    }
  }
  uint32_t off[2][NP];
#pragma unroll
  for (int p = 0; p < NP; ++p) {
    const int R = (wave * NP + p) * 8 + (lane >> 3);
    const int chunk = (lane & 7) ^ ((R >> 1) & 7);
    off[0][p] = static_cast<uint32_t>(min(R, a.rows_p - 1 - bm * TM)) * a.ldp * 4 + chunk * 16;
    off[1][p] = static_cast<uint32_t>(min(R, a.rows_q - 1 - bn * TM)) * a.ldq * 4 + chunk * 16;
  }
  const int first = split * a.split_stages, stages = min(a.split_stages, a.K / kStageK - first);
  const char *from[2] = {
      reinterpret_cast<const char *>(a.P + z * a.p_stride + static_cast<long long>(bm) * TM * a.ldp * 2) + first * 128LL,
      reinterpret_cast<const char *>(a.Q + z * a.q_stride + static_cast<long long>(bn) * TM * a.ldq * 2) + first * 128LL};
  // piece k of the next stage to copy, into `slot`; an array's last one moves on
  auto copy = [&](int k, int slot) {
    const int s = k / NP, p = k % NP;
    dma_piece(from[s], off[s][p], smem + (slot * kStage + s * kArray + (wave * NP + p) * 1024) / 4);
    if (p == NP - 1) from[s] += 128;
  };
  // a wave of one tile keeps a sum for each product and 16 k of a stage: dependent instructions issue at half the rate
  constexpr int kPairs = 3;  // products of terms: lo hi, hi lo, hi hi
  constexpr int kSums = FM * FN == 1 ? 2 * kPairs : 1;
  f32x16 acc[FM][FN], more[kSums];
#pragma unroll
  for (int e = 0; e < 16; ++e) {
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) acc[i][j][e] = 0.f;
#pragma unroll
    for (int i = 1; i < kSums; ++i) more[i][e] = 0.f;
  }
  const int wm = wave / WC, wn = wave % WC, hi = lane >> 5, l31 = lane & 31;
  const unsigned x = (l31 >> 1) & 7;
  // lane addresses in an array: 16 k of two, times two terms
  unsigned prow[4], qrow[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int chunk = (k & 1) * 4 + (k >> 1) * 2 + hi;
    prow[k] = (wm * FM * 32 + l31) * 128 + (chunk ^ x) * 16;
    qrow[k] = kArray + (wn * FN * 32 + l31) * 128 + (chunk ^ x) * 16;
  }
  f16x8 p[2][2][FM], q[2][2][FN];
  // fragment k (of kReads) of 16 k (`part`) of a slot
  constexpr int kReads = 2 * (FM + FN), kProducts = kPairs * FM * FN;
  auto fetch = [&](int set, int slot, int part, int k) {
    const char *base = reinterpret_cast<const char *>(smem) + slot * kStage;
    if (k < 2 * FM) {
      const int t = k / FM, i = k % FM;
      p[set][t][i] = *reinterpret_cast<const f16x8 *>(base + prow[part * 2 + t] + i * 4096);
    } else {
      const int t = (k - 2 * FM) / FN, j = (k - 2 * FM) % FN;
      q[set][t][j] = *reinterpret_cast<const f16x8 *>(base + qrow[part * 2 + t] + j * 4096);
    }
  };
  auto multiply = [&](int set, int k) {  // the small products first
    const int t = k / (FM * FN), i = k / FN % FM, j = k % FN;
    f32x16 &sum = kSums > 1 && t * 2 + set > 0 ? more[kSums > 1 ? t * 2 + set : 0] : acc[i][j];
    sum = __builtin_amdgcn_mfma_f32_32x32x16_f16(p[set][t == 0][i], q[set][t == 1][j], sum, 0, 0, 0);
  };
  // 16 k of a stage: the products of one set of fragments, with the reads of the other and copies of a later stage between
  // them (one or two waves a SIMD: what is not issued in a product's shadow is paid for)
  auto part = [&](int set, int slot, int next_part, int fill, bool more_stages, auto copies) {
    constexpr int kOps = kReads + (decltype(copies)::value ? kPieces : 0);
#pragma unroll
    for (int k = 0; k < kProducts; ++k) {
      multiply(set, k);
#pragma unroll
      for (int o = k * kOps / kProducts; o < (k + 1) * kOps / kProducts; ++o) {
        if (o < kReads) fetch(set ^ 1, slot, next_part, o);
        else if (more_stages) copy(o - kReads, fill);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  for (int s = 0; s < RING && s < stages; ++s)
#pragma unroll
    for (int k = 0; k < kPieces; ++k) copy(k, s);
  if (stages >= RING) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((RING - 1) * kPieces) : "memory");
  else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
#pragma unroll
  for (int k = 0; k < kReads; ++k) fetch(0, 0, 0, k);
  int slot = 0;
#pragma unroll 1
  for (int s = 0; s < stages; ++s) {
    const int next = slot + 1 == RING ? 0 : slot + 1;
    part(0, slot, 1, 0, false, std::false_type{});
    // this wave's copies of stage s + 1 have landed and all its reads of stage s are done; behind the barrier every wave's
    if (s + RING <= stages) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((RING - 2) * kPieces) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0), as the builtin: the compiler counts it
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    part(1, next, 0, slot, s + RING < stages, std::true_type{});  // (behind the last stage: reads what the slot holds, not used)
    slot = next;
  }
  if constexpr (kSums > 1) {
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      float v = acc[0][0][e];
#pragma unroll
      for (int i = 1; i < kSums; ++i) v += more[i][e];
      acc[0][0][e] = v;
    }
  }
  if ((EPI == GRAM || EPI == POLY) && TM <= 128 && a.splits > 1) {
    // The last of the tile's workgroups to arrive adds all of them up in the order of their numbers (its own among them: the
    // result does not depend on who is last) and leaves the count at zero for the next launch.  The sums are exchanged by
    // relaxed agent-scope accesses, which pass the XCDs' own L2s by; a store has completed when vmcnt says so, and the count
    // is raised behind the barrier that follows.  (Fences instead -- a write-back and an invalidation of the whole L2 by every
    // wave -- cost 28 us a launch.)
    const long long tile = z * (gridDim.x / a.splits) + blockIdx.x / a.splits;
    constexpr int kThreads = kWaves * 64, kWords = FM * FN * 8;
    unsigned long long *all = reinterpret_cast<unsigned long long *>(a.partials) + tile * a.splits * kWords * kThreads + tid;
    unsigned long long *mine = all + static_cast<long long>(split) * kWords * kThreads;
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j)
#pragma unroll
        for (int g = 0; g < 8; ++g) {
          const float lo = acc[i][j][2 * g], up = acc[i][j][2 * g + 1];
          const unsigned long long v = __builtin_bit_cast(uint32_t, lo) | static_cast<unsigned long long>(__builtin_bit_cast(uint32_t, up)) << 32;
          __hip_atomic_store(mine + ((i * FN + j) * 8 + g) * kThreads, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    unsigned *arrived = reinterpret_cast<unsigned *>(smem);
    if (tid == 0) *arrived = __hip_atomic_fetch_add(a.arrivals + tile, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (*arrived != static_cast<unsigned>(a.splits - 1)) return;
    if (tid == 0) __hip_atomic_store(a.arrivals + tile, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
#pragma unroll 1
    for (int s = 0; s < a.splits; ++s) {
      unsigned long long v[kWords];
#pragma unroll
      for (int k = 0; k < kWords; ++k) v[k] = __hip_atomic_load(all + (static_cast<long long>(s) * kWords + k) * kThreads, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
      for (int k = 0; k < kWords; ++k) {
        const uint32_t lo = static_cast<uint32_t>(v[k]), up = static_cast<uint32_t>(v[k] >> 32);
        acc[k / 8 / FN][k / 8 % FN][k % 8 * 2] += __builtin_bit_cast(float, lo);
        acc[k / 8 / FN][k / 8 % FN][k % 8 * 2 + 1] += __builtin_bit_cast(float, up);
      }
    }
    __syncthreads();  // everyone has read *arrived
  }
  // Accumulator e of a lane: row 8 (e / 4) + 4 (lane / 32) + e % 4, column lane % 32.  Stores: rows are made of four columns
  // per lane by a transposition within quads (8 bytes a lane, 64 a row), the transposed copy of eight rows per lane by
  // exchanging with the lane of the other half (16 bytes).
  _Float16 *D = a.D + z * a.d_stride, *DT = a.DT + z * a.dt_stride;
  const int *exp_m = a.exp_m + z * static_cast<long long>(a.exp_m_stride), *exp_n = a.exp_n + z * static_cast<long long>(a.exp_n_stride);
  f32x4 *master = reinterpret_cast<f32x4 *>(a.master + z * a.master_stride);
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      const int m0 = bm * TM + (wm * FM + i) * 32, n0 = bn * TM + (wn * FN + j) * 32;
      if (m0 >= a.rows_p || n0 >= a.rows_q) continue;  // (32-row blocks are whole)
      const int n = n0 + l31;
      f32x4 *copy32 = master + (static_cast<long long>(n0 >> 5) * (a.rows_p >> 5) + (m0 >> 5)) * 256 + lane;
      const int start_n = exp_n[n], en = bound_of(start_n, a.shift, a.cap);
      f32x4 kept[4];
      i32x4 start_m[4];
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        start_m[g] = *reinterpret_cast<const i32x4 *>(exp_m + m0 + 8 * g + 4 * hi);
        if constexpr (EPI != GRAM) kept[g] = copy32[64 * g];
      }
      uint32_t h[4][2], l[4][2];
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int m = m0 + 8 * g + 4 * hi;
        float v[4];
        int scale[4], turned;  // of the results' rows and of their transpose's
        if constexpr (EPI == UPDATE || EPI == FINAL) turned = kTop - bound_of(start_n, a.next_shift, a.next_cap);
        else turned = kTop - en - a.cap - (EPI == POLY ? a.poly : 0);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int em = bound_of(start_m[g][k], a.shift, a.cap);
          const float sum = acc[i][j][4 * g + k];
          if constexpr (EPI == GRAM) {
            v[k] = times_power(sum, em + en - 2 * kTop);
            scale[k] = kTop - em - a.cap;
          } else if constexpr (EPI == POLY) {
            v[k] = a.c * times_power(sum, em + en + 2 * (a.cap - kTop)) + a.b * kept[g][k];
            scale[k] = kTop - em - a.cap - a.poly;
          } else {
            v[k] = a.a * kept[g][k] + times_power(sum, em + en + a.cap + a.poly - 2 * kTop);
            scale[k] = kTop - bound_of(start_m[g][k], a.next_shift, a.next_cap);
          }
        }
        if constexpr (EPI == FINAL) {
          put_final(a, z, m, n, n0 + (l31 & ~3), lane, v);
          continue;
        }
        if constexpr (EPI != POLY) copy32[64 * g] = f32x4{v[0], v[1], v[2], v[3]};
        auto terms = [&](auto by, u32x2 &high, u32x2 &low) {
          f16x4 vh, vl;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float x = times_power(v[k], by(k));
            vh[k] = static_cast<_Float16>(x);
            vl[k] = static_cast<_Float16>(x - static_cast<float>(vh[k]));
          }
          high = __builtin_bit_cast(u32x2, vh);
          low = __builtin_bit_cast(u32x2, vl);
        };
        u32x2 bh, bl;
        terms([&](int) { return turned; }, bh, bl);
        h[g][0] = bh.x;
        h[g][1] = bh.y;
        l[g][0] = bl.x;
        l[g][1] = bl.y;
        if (EPI == UPDATE || bm != bn) {
          terms([&](int k) { return scale[k]; }, bh, bl);
          _Float16 *at = D + place(m + (lane & 3), n0 + (l31 & ~3), a.ldd);
          const Pair2 th = quad_transpose(bh.x, bh.y, lane), tl = quad_transpose(bl.x, bl.y, lane);
          *reinterpret_cast<u32x2 *>(at) = u32x2{th.x, th.y};
          *reinterpret_cast<u32x2 *>(at + kSecond) = u32x2{tl.x, tl.y};
        }
      }
      if constexpr (EPI != FINAL) {
#pragma unroll
        for (int g = 0; g < 4; g += 2) {  // groups g (kept by the lower half) and g + 1 (by the upper one): eight rows each
          _Float16 *at = DT + place(n, m0 + 8 * (g + hi), a.lddt);
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            swap_halves(h[g][k], h[g + 1][k]);
            swap_halves(l[g][k], l[g + 1][k]);
          }
          *reinterpret_cast<u32x4 *>(at) = u32x4{h[g][0], h[g][1], h[g + 1][0], h[g + 1][1]};
          *reinterpret_cast<u32x4 *>(at + kSecond) = u32x4{l[g][0], l[g][1], l[g + 1][0], l[g + 1][1]};
        }
      }
    }
}

// 1 / (|G| + eps) as a fraction in [1/2, 1) and a power of two: the norm may lie outside fp32's range.  (A product in
// double that goes on to fp16 is converted by 30 integer instructions: packing 512 x 3136 f32 took 14.4 us, 9.8 so.)
struct Scale {
  float fraction;
  int power;
};
__device__ __forceinline__ Scale scale_of(double squares, float eps) {
  Scale s;
  s.fraction = static_cast<float>(frexp(1.0 / (sqrt(squares) + eps), &s.power));
  return s;
}
// (the power first: a denormal value's product with the fraction would lose what it has)
__device__ __forceinline__ float scaled(float x, const Scale &s) { return times_power(x, s.power) * s.fraction; }
// exponent of a bound of the norm of `count` scaled values of which none passes `most`
__device__ __forceinline__ int start_bound(float most, int count, const Scale &s) {
  const int ceil_log2 = count <= 1 ? 0 : 32 - __builtin_clz(count - 1);
  return most == 0.f ? kLowest : power_above(most) + s.power + (ceil_log2 + 1) / 2;
}

// over the 16 lanes of a DPP row
template <int ROR>
__device__ __forceinline__ float more_of(float v) {
  return fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x120 + ROR, 0xf, 0xf, true)));
}
__device__ __forceinline__ float most_of_16(float v) { return more_of<1>(more_of<2>(more_of<4>(more_of<8>(v)))); }

// The sum of squares of a part of a matrix (`band` rows of `strip` columns) and the largest magnitudes of its rows and columns: a wave
// per row and 64 vectors of it.
template <typename V>
__global__ __launch_bounds__(256) void ns_scan_kernel(const V *in, int m, int n, int band, int strip, double *sums, float *row_most, float *col_most) {
  constexpr int E = 16 / sizeof(V), C = 64 * E, U = 8;
  using Vec = __attribute__((ext_vector_type(E))) V;
  typedef Vec Loose __attribute__((aligned(sizeof(V))));  // a matrix of the batch may start at any element
  __shared__ float rows[65536 / kScanParts], cols[4][C];
  __shared__ double scratch[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long long z = blockIdx.z;
  const V *g = in + z * m * n;
  const int r0 = blockIdx.y * band, r1 = min(m, r0 + band), c0 = blockIdx.x * strip, c1 = min(n, c0 + strip);
  double s = 0;
  for (int chunk = c0; chunk < c1; chunk += C) {
    const int col = chunk + lane * E;
    float top[E] = {};
    for (int base = r0 + wave; base < r1; base += 4 * U) {
      Vec v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int row = base + 4 * u;
        v[u] = Vec{};
        if (row >= r1) continue;
        const V *from = g + static_cast<long long>(row) * n + col;
        if (col + E <= n) v[u] = *reinterpret_cast<const Loose *>(from);
        else
#pragma unroll
          for (int k = 0; k < E; ++k)
            if (col + k < n) v[u][k] = from[k];
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int row = base + 4 * u;
        if (row >= r1) continue;  // (the wave's)
        float most = 0.f;
#pragma unroll
        for (int k = 0; k < E; ++k) {
          const float x = fabsf(static_cast<float>(v[u][k]));
          top[k] = fmaxf(top[k], x);
          most = fmaxf(most, x);
          s += static_cast<double>(x) * x;
        }
        most = most_of_16(most);
        most = fmaxf(most, __shfl_xor(most, 16));
        most = fmaxf(most, __shfl_xor(most, 32));
        if (lane == 0) rows[row - r0] = chunk == c0 ? most : fmaxf(rows[row - r0], most);
      }
    }
#pragma unroll
    for (int k = 0; k < E; ++k) cols[wave][lane * E + k] = top[k];
    __syncthreads();
    for (int i = threadIdx.x; i < C && chunk + i < n; i += 256)
      col_most[(z * gridDim.y + blockIdx.y) * n + chunk + i] = fmaxf(fmaxf(cols[0][i], cols[1][i]), fmaxf(cols[2][i], cols[3][i]));
    __syncthreads();
  }
  for (int i = threadIdx.x; i < r1 - r0; i += 256) row_most[(z * gridDim.x + blockIdx.x) * m + r0 + i] = rows[i];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
  if (lane == 0) scratch[wave] = s;
  __syncthreads();
  if (threadIdx.x == 0) sums[(z * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x] = scratch[0] + scratch[1] + scratch[2] + scratch[3];
}

struct PackArgs {
  const void *in;
  int m, n, tall;
  int bands, strips;  // of the scan
  const double *sums;
  const float *row_most, *col_most;
  float eps;
  _Float16 *same, *turned;  // X0 in G's orientation and in the other
  int ld_same, ld_turned;
  long long stride;
  float *master;
  long long master_stride;
  int rows_x;               // padded rows of X, blocks of the copy
  int *exp_row, *exp_col;   // of G's rows and columns
  int exp_row_stride, exp_col_stride;
  int cap;
  unsigned *arrivals;
  int counts;
};

// X0, its transpose, its fp32 copy and the exponents from a 64 x 64 tile of G.  Also clears the arrival counts of the split products.
template <typename V>
__global__ __launch_bounds__(256) void ns_pack_kernel(const PackArgs a) {
  constexpr int E = 16 / sizeof(V);
  using Vec = __attribute__((ext_vector_type(E))) V;
  typedef Vec Loose __attribute__((aligned(sizeof(V))));
  __shared__ float tile[64][65], most[4][64];
  __shared__ int exps[2][64];
  __shared__ double total[4];
  const long long z = blockIdx.z;
  const int c0 = blockIdx.x * 64, r0 = blockIdx.y * 64, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const V *g = static_cast<const V *>(a.in) + z * a.m * a.n;
  if (blockIdx.x == 0 && blockIdx.y == 0 && z == 0)
    for (int i = threadIdx.x; i < a.counts; i += 256) a.arrivals[i] = 0;
  // 64 rows of 64 / E vectors, all on their way before the first is waited for
  constexpr int kVecs = 64 * 64 / E / 256;
  Vec v[kVecs];
  if (r0 + 64 <= a.m && c0 + 64 <= a.n) {
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
      const int at = k * 256 + threadIdx.x;
      v[k] = *reinterpret_cast<const Loose *>(g + static_cast<long long>(r0 + at / (64 / E)) * a.n + c0 + at % (64 / E) * E);
    }
  } else {
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
      const int at = k * 256 + threadIdx.x, row = at / (64 / E), col = at % (64 / E) * E;
      v[k] = Vec{};
      if (r0 + row < a.m) {
        const V *from = g + static_cast<long long>(r0 + row) * a.n + c0 + col;
        if (c0 + col + E <= a.n) v[k] = *reinterpret_cast<const Loose *>(from);
        else
#pragma unroll
          for (int i = 0; i < E; ++i)
            if (c0 + col + i < a.n) v[k][i] = from[i];
      }
    }
  }
  const int parts = a.bands * a.strips;
  double s = 0;
  for (int i = threadIdx.x; i < parts; i += 256) s += a.sums[z * parts + i];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
  if (lane == 0) total[wave] = s;
  {  // the largest magnitudes: waves 0 and 1 of the rows, 2 and 3 of the columns, half of the parts each
    const bool rows = wave < 2;
    const int at = (rows ? r0 : c0) + lane, side = rows ? a.m : a.n, count = rows ? a.strips : a.bands;
    const float *from = (rows ? a.row_most : a.col_most) + z * count * static_cast<long long>(side) + at;
    float x = 0.f;
    if (at < side)
#pragma unroll 8
      for (int i = wave & 1; i < count; i += 2) x = fmaxf(x, from[static_cast<long long>(i) * side]);
    most[wave][lane] = x;
  }
  __syncthreads();
  const Scale scale = scale_of(total[0] + total[1] + total[2] + total[3], a.eps);
  if (wave == 0) {
    exps[0][lane] = start_bound(fmaxf(most[0][lane], most[1][lane]), a.n, scale);
    if (blockIdx.x == 0) a.exp_row[z * a.exp_row_stride + r0 + lane] = exps[0][lane];
  } else if (wave == 1) {
    exps[1][lane] = start_bound(fmaxf(most[2][lane], most[3][lane]), a.m, scale);
    if (blockIdx.y == 0) a.exp_col[z * a.exp_col_stride + c0 + lane] = exps[1][lane];
  }
#pragma unroll
  for (int k = 0; k < kVecs; ++k) {
    const int at = k * 256 + threadIdx.x;
#pragma unroll
    for (int i = 0; i < E; ++i) tile[at / (64 / E)][at % (64 / E) * E + i] = scaled(static_cast<float>(v[k][i]), scale);
  }
  __syncthreads();
  auto put8 = [&](_Float16 *at, int exponent, auto value) {
    const int by = kTop - bound_of(exponent, 0, a.cap);
    f16x8 h, l;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x = times_power(value(i), by);
      h[i] = static_cast<_Float16>(x);
      l[i] = static_cast<_Float16>(x - static_cast<float>(h[i]));
    }
    *reinterpret_cast<f16x8 *>(at) = h;
    *reinterpret_cast<f16x8 *>(at + kSecond) = l;
  };
#pragma unroll
  for (int k = 0; k < 2; ++k) {  // 64 rows of 8 x 8 values (the padded sides are multiples of 64)
    const int at = k * 256 + threadIdx.x, row = at >> 3, col = (at & 7) * 8;
    put8(a.same + z * a.stride + place(r0 + row, c0 + col, a.ld_same), exps[0][row], [&](int i) { return tile[row][col + i]; });
    put8(a.turned + z * a.stride + place(c0 + row, r0 + col, a.ld_turned), exps[1][row], [&](int i) { return tile[col + i][row]; });
  }
  const int xm = a.tall ? c0 : r0, xn = a.tall ? r0 : c0;
#pragma unroll
  for (int k = 0; k < 4; ++k) {  // blocks (k & 1, k >> 1) of 32 x 32, as the products' accumulators hold them
    const int row = (k & 1) * 32 + wave * 8 + (lane >> 5) * 4, col = (k >> 1) * 32 + (lane & 31);
    f32x4 x;
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = a.tall ? tile[col][row + i] : tile[row + i][col];
    const long long block = static_cast<long long>((xn >> 5) + (k >> 1)) * (a.rows_x >> 5) + (xm >> 5) + (k & 1);
    reinterpret_cast<f32x4 *>(a.master + z * a.master_stride)[block * 256 + threadIdx.x] = x;
  }
}

// ---- matrices that fit a workgroup's LDS: the whole iteration in ONE launch, a workgroup per matrix -----------------
// X, X^T, A and M stay in LDS (rows padded by 16 bytes: an odd number of 16-byte chunks, so that 16 rows' equal chunks meet
// every bank once); 16 waves share the 16 x 16 x 32 tiles of each product, every wave the same ones in every step, so that the
// fp32 copies of X and A are in its registers (G too: it is read once).  What bounds it is the chain of 3 x steps dependent
// products, not their rate.
// LDS is addressed by plain offsets into one array: through pointers that are chosen at run time the compiler cannot see that
// they are LDS, and flat accesses and spills more than doubled a step.
constexpr int kSmallWaves = 16;
constexpr long long kSmallLds = 160 * 1024;

// bytes: the matrices, the exponents of X's rows and columns, the parts of the norm; more than there are if the waves cannot hold X
inline long long small_lds(int rp, int cp) {
  if (rp > 64 ? rp / 32 * (cp / 32) > kSmallWaves : cp / 16 > kSmallWaves * (rp > 32 ? 1 : 2)) return kSmallLds + 1;
  return 4LL * (static_cast<long long>(rp) * (cp + 8) + static_cast<long long>(cp) * (rp + 8)) + 8LL * rp * (rp + 8) + 4LL * (rp + cp) + 8 * kSmallWaves;
}

// (the powers of every step are formed on the host: on the device a step's cost 1 us of its 4)
constexpr int kSmallSteps = 32;
struct SmallArgs {
  const void *in;
  void *out;
  int m, n, r, c, rp, cp, steps, tall;
  float a, b, k, eps;
  Powers powers[kSmallSteps + 1];
};

// SIDE: the products are formed in blocks of 16 x 16 (one instruction tile: the shortest chain, and enough blocks of A for the
// waves up to 64 rows) or 32 x 32 (two fragments of each side for four tiles: half the LDS reads).
// COLUMNS = 0: X has no more blocks than there are waves; a block is held over a barrier before it overwrites X.
// COLUMNS > 0: a wave takes COLUMNS columns of BLOCKS blocks at most, which depend on nothing but themselves: held without a
// barrier, their X^T fragments read once (64 x 400 of one term: blocks dealt out, held and written by straight code 51 us, half of
// them its instruction fetches; by columns 35).
template <typename V, int SIDE, int COLUMNS, int BLOCKS>
__global__ __launch_bounds__(kSmallWaves * 64) void ns_small_kernel(const SmallArgs a) {
  extern __shared__ __attribute__((aligned(16))) _Float16 lds[];
  const int tid = threadIdx.x, lane = tid & 63;
  int l15 = lane & 15, quad = lane >> 4;
  // (opaque: addresses that do not change would be kept over the steps, more than there are registers)
  auto forget = [&] { asm volatile("" : "+v"(l15), "+v"(quad)); };
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int ldx = a.cp + 8, ldr = a.rp + 8;  // X: rp rows of ldx; X^T: cp rows of ldr; A, M: rp rows of ldr
  // each array: its first terms, then its second ones
  const int sx = a.rp * ldx, st = a.cp * ldr, sa = a.rp * ldr;
  const int X = 0, XT = X + 2 * sx, A = XT + 2 * st, M = A + 2 * sa;
  double *parts = reinterpret_cast<double *>(lds + M + 2 * sa);
  int *exp_row = reinterpret_cast<int *>(parts + kSmallWaves), *exp_col = exp_row + a.rp;  // first the largest magnitudes' bits
  constexpr int F = SIDE / 16, kCols = COLUMNS > 0 ? COLUMNS : 1;
  struct Block { f32x4 v[F][F]; };
  const int tr = a.rp / SIDE, tc = a.cp / SIDE, upper = tr * (tr + 1) / 2;
  // this wave's blocks of X: (i, tn) or, where COLUMNS = 0, one; accumulator e of a lane and 16 x 16 tile: row 4 (lane / 16) + e,
  // column lane % 16
  auto block_row = [&](int i) { return COLUMNS > 0 ? i * SIDE : wave % tr * SIDE; };
  auto block_col = [&](int it) { return COLUMNS > 0 ? (wave + it * kSmallWaves) * SIDE : wave / tr * SIDE; };
  auto has = [&](int i, int it) { return COLUMNS > 0 ? i < tr && wave + it * kSmallWaves < tc : wave < tr * tc; };
  Block x[kCols][BLOCKS];
  const V *in = static_cast<const V *>(a.in) + blockIdx.x * (static_cast<long long>(a.m) * a.n);
#pragma unroll
  for (int it = 0; it < kCols; ++it)
#pragma unroll
    for (int i = 0; i < BLOCKS; ++i)
#pragma unroll
      for (int f = 0; f < F; ++f)
#pragma unroll
        for (int g = 0; g < F; ++g)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int row = block_row(i) + f * 16 + 4 * quad + e, col = block_col(it) + g * 16 + l15;
            const int r0 = min(row, a.r - 1), c0 = min(col, a.c - 1);
            const float v = static_cast<float>(in[a.tall ? c0 * a.n + r0 : r0 * a.n + c0]);
            x[it][i].v[f][g][e] = has(i, it) && row < a.r && col < a.c ? v : 0.f;
          }
  for (int i = tid; i < a.rp + a.cp; i += kSmallWaves * 64) exp_row[i] = 0;
  __syncthreads();
  double s = 0;
#pragma unroll
  for (int i = 0; i < BLOCKS; ++i)
#pragma unroll
    for (int f = 0; f < F; ++f)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float most = 0.f;
#pragma unroll
        for (int it = 0; it < kCols; ++it)
#pragma unroll
          for (int g = 0; g < F; ++g) {
            const float v = x[it][i].v[f][g][e];
            s += static_cast<double>(v) * v;
            most = fmaxf(most, fabsf(v));
          }
        most = most_of_16(most);
        if (l15 == 0 && has(i, 0)) atomicMax(exp_row + block_row(i) + f * 16 + 4 * quad + e, __builtin_bit_cast(int, most));
      }
#pragma unroll
  for (int it = 0; it < kCols; ++it)
#pragma unroll
    for (int g = 0; g < F; ++g) {
      float most = 0.f;
#pragma unroll
      for (int i = 0; i < BLOCKS; ++i)
#pragma unroll
        for (int f = 0; f < F; ++f)
#pragma unroll
          for (int e = 0; e < 4; ++e) most = fmaxf(most, fabsf(x[it][i].v[f][g][e]));
      if (has(0, it)) atomicMax(exp_col + block_col(it) + g * 16 + l15, __builtin_bit_cast(int, most));
    }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
  if (lane == 0) parts[wave] = s;
  __syncthreads();
  s = 0;
#pragma unroll
  for (int i = 0; i < kSmallWaves; ++i) s += parts[i];
  const Scale scale = scale_of(s, a.eps);
  for (int i = tid; i < a.rp + a.cp; i += kSmallWaves * 64)
    exp_row[i] = start_bound(__builtin_bit_cast(float, exp_row[i]), i < a.rp ? a.c : a.r, scale);
  __syncthreads();
  // four consecutive rows of a column, scaled by 2^turn into the row of the transpose and, if wanted, each by its own power into four rows
  auto put4 = [&](int turned, int turned_size, int turn, int at, int ld, int size, i32x4 by, bool both, f32x4 v) {
    f16x4 h, l;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float y = times_power(v[k], turn);
      h[k] = static_cast<_Float16>(y);
      l[k] = static_cast<_Float16>(y - static_cast<float>(h[k]));
    }
    *reinterpret_cast<f16x4 *>(lds + turned) = h;
    *reinterpret_cast<f16x4 *>(lds + turned + turned_size) = l;
    if (both) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float y = times_power(v[k], by[k]);
        const _Float16 high = static_cast<_Float16>(y);
        lds[at + k * ld] = high;
        lds[at + k * ld + size] = static_cast<_Float16>(y - static_cast<float>(high));
      }
    }
  };
  auto put_x = [&](int m, int n, const Powers &k, f32x4 v) {
    const i32x4 start = *reinterpret_cast<const i32x4 *>(exp_row + m);
    i32x4 by;
#pragma unroll
    for (int e = 0; e < 4; ++e) by[e] = kTop - bound_of(start[e], k.shift, k.cap);
    put4(XT + n * ldr + m, st, kTop - bound_of(exp_col[n], k.shift, k.cap), X + m * ldx + n, ldx, sx, by, true, v);
  };
#pragma unroll
  for (int it = 0; it < kCols; ++it)
#pragma unroll
    for (int i = 0; i < BLOCKS; ++i) {
      if (!has(i, it)) continue;
#pragma unroll
      for (int f = 0; f < F; ++f)
#pragma unroll
        for (int g = 0; g < F; ++g) {
          f32x4 &v = x[it][i].v[f][g];
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = scaled(v[e], scale);
          put_x(block_row(i) + f * 16 + 4 * quad, block_col(it) + g * 16 + l15, a.powers[0], v);
        }
    }
  __syncthreads();
  // acc[i] = rows SIDE i .. of P times SIDE rows of Q transposed, the first `count` of N blocks
  auto products = [&](auto &acc, int count, int P, int ldp, int sp, int Q, int ldq, int sq, int K) {
    constexpr int N = sizeof(acc) / sizeof(Block);
    Block cross[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      acc[i] = Block{};
      cross[i] = Block{};
    }
    const int po = P + l15 * ldp + quad * 8, qo = Q + l15 * ldq + quad * 8;
#pragma unroll 1
    for (int k = 0; k < K; k += 32) {
      f16x8 qh[F], ql[F];
#pragma unroll
      for (int f = 0; f < F; ++f) {
        qh[f] = *reinterpret_cast<const f16x8 *>(lds + qo + f * 16 * ldq + k);
        ql[f] = *reinterpret_cast<const f16x8 *>(lds + qo + f * 16 * ldq + sq + k);
      }
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (N > 1 && i >= count) continue;
#pragma unroll
        for (int f = 0; f < F; ++f) {
          const int at = po + (i * SIDE + f * 16) * ldp + k;
          const f16x8 ph = *reinterpret_cast<const f16x8 *>(lds + at), pl = *reinterpret_cast<const f16x8 *>(lds + at + sp);
#pragma unroll
          for (int g = 0; g < F; ++g) {
            acc[i].v[f][g] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph, qh[g], acc[i].v[f][g], 0, 0, 0);
            f32x4 &c = cross[i].v[f][g];  // (a sum of its own: dependent instructions issue at half the rate)
            c = __builtin_amdgcn_mfma_f32_16x16x32_f16(pl, qh[g], c, 0, 0, 0);
            c = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph, ql[g], c, 0, 0, 0);
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int f = 0; f < F; ++f)
#pragma unroll
        for (int g = 0; g < F; ++g) acc[i].v[f][g] += cross[i].v[f][g];
  };
  // this wave's block of A and M: there are 10 at most (rp <= 64 in blocks of 16, <= 128 of 32), on and above the diagonal
  int pm = 0, qn = 0;
  if (wave < upper) {
    int left = wave, row = 0;
    while (left >= tr - row) left -= tr - row++;
    pm = row * SIDE;
    qn = (row + left) * SIDE;
  }
  Block gram[1], acc[1];
#pragma unroll 1
  for (int step = 0; step < a.steps; ++step) {
    const bool last = step + 1 == a.steps;
    const Powers known = a.powers[step], next = a.powers[step + 1];
    // A = X X^T, then M = b A + c A A: their upper triangles, stored twice
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      forget();
      if (wave < upper) {
        if (half) products(acc, 1, A + pm * ldr, ldr, sa, A + qn * ldr, ldr, sa, a.rp);
        else products(gram, 1, X + pm * ldx, ldx, sx, X + qn * ldx, ldx, sx, a.cp);
        const int to = half ? M : A, less = known.cap + (half ? known.poly : 0);
#pragma unroll
        for (int f = 0; f < F; ++f)
#pragma unroll
          for (int g = 0; g < F; ++g) {
            const int m = pm + f * 16 + 4 * quad, n = qn + g * 16 + l15;
            const i32x4 start = *reinterpret_cast<const i32x4 *>(exp_row + m);
            const int en = bound_of(exp_row[n], known.shift, known.cap);
            i32x4 by;
            f32x4 v;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int em = bound_of(start[e], known.shift, known.cap);
              if (half) v[e] = a.k * times_power(acc[0].v[f][g][e], em + en + 2 * (known.cap - kTop)) + a.b * gram[0].v[f][g][e];
              else v[e] = times_power(gram[0].v[f][g][e], em + en - 2 * kTop);
              by[e] = kTop - em - less;
            }
            if (!half) gram[0].v[f][g] = v;
            put4(to + n * ldr + m, sa, kTop - en - less, to + m * ldr + n, ldr, sa, by, pm != qn, v);
          }
      }
      __syncthreads();
    }
    forget();
    Block held[BLOCKS];
#pragma unroll
    for (int it = 0; it < kCols; ++it) {
      if (COLUMNS > 0 && !has(0, it)) continue;
      if (has(0, it)) products(held, tr, M + (COLUMNS > 0 ? 0 : block_row(0)) * ldr, ldr, sa, XT + block_col(it) * ldr, ldr, st, a.rp);
      if (COLUMNS == 0) __syncthreads();
#pragma unroll
      for (int i = 0; i < BLOCKS; ++i) {
        if (!has(i, it)) continue;
#pragma unroll
        for (int f = 0; f < F; ++f)
#pragma unroll
          for (int g = 0; g < F; ++g) {
            const int m = block_row(i) + f * 16 + 4 * quad, n = block_col(it) + g * 16 + l15;
            const i32x4 start = *reinterpret_cast<const i32x4 *>(exp_row + m);
            const int en = bound_of(exp_col[n], known.shift, known.cap) + known.cap + known.poly - 2 * kTop;
            f32x4 &v = x[it][i].v[f][g];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              v[e] = a.a * v[e] + times_power(held[i].v[f][g][e], bound_of(start[e], known.shift, known.cap) + en);
            if (!last) {
              put_x(m, n, next, v);
            } else {
              V *out = static_cast<V *>(a.out) + blockIdx.x * (static_cast<long long>(a.m) * a.n);
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (m + e < a.r && n < a.c) out[a.tall ? n * a.n + m + e : (m + e) * a.n + n] = static_cast<V>(v[e]);
            }
          }
      }
    }
    __syncthreads();
  }
}

template <typename V, int SIDE, int COLUMNS, int BLOCKS>
int launch_small_as(const SmallArgs &q, int batch, int bytes, hipStream_t s) {
  DX_LDS_OPT_IN((ns_small_kernel<V, SIDE, COLUMNS, BLOCKS>), kSmallLds);
  hipLaunchKernelGGL((ns_small_kernel<V, SIDE, COLUMNS, BLOCKS>), dim3(batch), dim3(kSmallWaves * 64), bytes, s, q);
  DX_LAUNCH_CHECK();
  return DX_OK;
}
template <typename V>
int launch_small(const SmallArgs &q, int batch, int bytes, hipStream_t s) {
  const int blocks = q.rp / 32 * (q.cp / 32);
  if (blocks * 4 <= kSmallWaves) return launch_small_as<V, 16, 0, 1>(q, batch, bytes, s);
  if (q.rp <= 32) return launch_small_as<V, 16, 2, 2>(q, batch, bytes, s);
  if (q.rp <= 64) return launch_small_as<V, 16, 1, 4>(q, batch, bytes, s);
  return launch_small_as<V, 32, 0, 1>(q, batch, bytes, s);
}

struct Scan {
  int bands, strips, band, strip;  // workgroups along the rows and the columns, rows and columns of each
  long long floats() const { return static_cast<long long>(rows) * strips + static_cast<long long>(columns) * bands; }
  int rows, columns;
};
Scan make_scan(int dtype, int m, int n) {
  const int chunk = dtype == DX_F32 ? 256 : 512;  // a wave's 16-byte vectors of a row; 8 rows a workgroup at least
  Scan s;
  s.rows = m;
  s.columns = n;
  const int chunks = cdiv(n, chunk), eights = cdiv(m, 8);
  s.strip = cdiv(chunks, chunks < kScanParts ? chunks : kScanParts) * chunk;
  s.strips = cdiv(n, s.strip);
  s.band = cdiv(eights, eights < kScanParts ? eights : kScanParts) * 8;
  s.bands = cdiv(m, s.band);
  return s;
}
struct Plan {
  bool one_launch;             // the matrices fit a workgroup's LDS
  int batch;                   // matrices at a time of the products' launches
  int r, c, rp, cp;
  Scan scan;
  long long x, sq;             // values of X and of A per matrix, padded
  long long split_floats, sums, most, bytes;
};
Plan make_plan(int dtype, int batch, int m, int n) {
  Plan p;
  p.r = m < n ? m : n;
  p.c = m < n ? n : m;
  p.one_launch = small_lds(cdiv(p.r, 32) * 32, cdiv(p.c, 32) * 32) <= kSmallLds;
  p.batch = p.one_launch ? 1 : batch;
  p.rp = (p.r + kPad - 1) / kPad * kPad;
  p.cp = (p.c + kPad - 1) / kPad * kPad;
  p.x = static_cast<long long>(p.rp) * p.cp;
  p.sq = static_cast<long long>(p.rp) * p.rp;
  p.scan = make_scan(dtype, m, n);
  const Scan other = make_scan(dtype, n, m);  // (a matrix and its transpose take the same workspace)
  auto most = [](long long x, long long y) { return x > y ? x : y; };
  p.sums = most(p.scan.bands * p.scan.strips, other.bands * other.strips);
  p.most = most(p.scan.floats(), other.floats());
  // (128 x 128 tiles are split where there are many)
  p.split_floats = p.one_launch ? 0 : static_cast<long long>(kSplitGroups) * (p.r > 1024 ? 128 * 128 : 64 * 64);
  // two terms of X, two copies of X^T, A and M; fp32 copies of X and A; the parts of split products; the norm's sums, the exponents,
  // the largest magnitudes
  p.bytes = p.batch * (4 * (3 * p.x + 2 * p.sq) + 4 * (p.x + p.sq) + 8 * p.sums + 4LL * (p.rp + p.cp) + 4 * p.most) + 4LL * kSplitGroups + 4 * p.split_floats;
  // one launch takes nothing of it (kSmallSteps): what the launches of one matrix take, whose steps may be more, and a token amount
  // a matrix, so that sizes grow with the batch
  if (p.one_launch) p.bytes += 256LL * batch;
  return p;
}
int check_shape(int dtype, int batch, int m, int n) {
  DX_REQUIRE(dtype == DX_F32 || dtype == DX_BF16 || dtype == DX_F16, "dx_orthogonalize: dtype %d is none of DX_F32, DX_BF16, DX_F16", dtype);
  DX_REQUIRE(batch >= 0 && batch <= 65535, "dx_orthogonalize: batch %d outside [0, 65535]", batch);
  DX_REQUIRE(m >= 1 && n >= 1 && m <= 65536 && n <= 65536, "dx_orthogonalize: (%d, %d): sides of 1 .. 65536 only", m, n);
  return DX_OK;
}

template <int TM, int WR, int WC, int RING, Epilogue EPI>
int launch_tile(NsArgs a, int batch, int splits, hipStream_t s) {
  constexpr int bytes = RING * 2 * TM * 128;
  DX_LDS_OPT_IN((ns_gemm_kernel<TM, WR, WC, RING, EPI>), bytes);
  a.tiles_m = cdiv(a.rows_p, TM);
  a.tiles_n = cdiv(a.rows_q, TM);
  const int tiles = EPI == GRAM || EPI == POLY ? a.tiles_m * (a.tiles_m + 1) / 2 : a.tiles_m * a.tiles_n;
  a.split_stages = cdiv(a.K / kStageK, splits);
  a.splits = cdiv(a.K / kStageK, a.split_stages);
  hipLaunchKernelGGL((ns_gemm_kernel<TM, WR, WC, RING, EPI>), dim3(tiles * a.splits, batch), dim3(WR * WC * 64), bytes, s, a);
  DX_LAUNCH_CHECK();
  return DX_OK;
}
// Tile side and parts of K for a product of `stages` stages, by the time that these constants give it (fitted to measured
// products; us a stage of 128-byte lines).  A CU's copies bound the small tiles (28 bytes a cycle): a 64 or 128 tile costs 0.30
// or 0.78 alone on a CU, 0.52 or 1.10 for two at a time (their ring lets two workgroups on a CU); 192 and 256 run alone, 1.2 and
// 1.9 with the chip full (at 1.7 to 1.8 GHz, 2.4 in short products).  Split parts exchange their sums: 8 us and 8 bytes a value.
// Measured, us a product (f32; * what the rule takes): 2001 x 5003 X X^T 64 121, 128 in two parts 112, in three 93 *; its update 64 171,
// 128 153 *, 192 194, 256 158.  512 x 3136 X X^T 64 in one part 26, in seven 14 *, 128 in seven 32; its update 64 15 *, 128 23, 192 38,
// 256 54.  4096 x 4096 X X^T 128 270, 192 201 *, 256 260; its update 128 400, 192 411, 256 364 *.  Over 14 shapes of 64 x 576 to
// 1024 x 8192 no other choice of one product was faster by more than 3 us, but X X^T of 1500 x 3000 (64: 6 us less than 128 in three).
struct Choice { int tile, splits; };
Choice choose(long long batch, int rows_p, int rows_q, bool half, bool may_split, int stages, int cus, long long split_floats) {
  Choice best{64, 1};
  double best_time = 1e300;
  for (int tile = 64; tile <= 256; tile += 64) {
    const long long m = cdiv(rows_p, tile), n = cdiv(rows_q, tile), tiles = (half ? m * (m + 1) / 2 : m * n) * batch;
    const double alone = tile == 64 ? 0.30 : tile == 128 ? 0.78 : tile == 192 ? 1.2 : 1.9, two = tile == 64 ? 0.52 : 1.10;
    for (int splits = 1; splits <= (may_split && tile <= 128 ? 8 : 1); ++splits) {
      const long long groups = tiles * splits;
      if (splits > 1 && (stages / splits < 12 || groups > kSplitGroups || groups * tile * tile > split_floats)) break;
      const long long slots = tile <= 128 ? 2LL * cus : cus, rest = groups % slots;
      const double rounds = tile <= 128 ? groups / slots * two + (rest > cus ? two : rest ? alone : 0.0) : (groups / slots + (rest ? 1 : 0)) * alone;
      const double time = rounds * cdiv(stages, splits) + (splits > 1 ? 8.0 + groups * tile * tile * 2e-6 : 0.0);
      if (time < best_time * 0.97) {
        best_time = time;
        best = {tile, splits};
      }
    }
  }
  return best;
}
template <Epilogue EPI>
int launch_gemm(const NsArgs &a, int batch, hipStream_t s) {
  constexpr bool half = EPI == GRAM || EPI == POLY;
  int cus = 0;
  if (int rc = device_cus(&cus)) return rc;
  const Choice c = choose(batch, a.rows_p, a.rows_q, half, half, a.K / kStageK, cus, a.split_floats);
  if (c.tile == 256) return launch_tile<256, 2, 4, 2, EPI>(a, batch, 1, s);
  if (c.tile == 192) return launch_tile<192, 2, 2, 3, EPI>(a, batch, 1, s);
  if (c.tile == 128) return launch_tile<128, 2, 2, 2, EPI>(a, batch, c.splits, s);
  return launch_tile<64, 2, 2, 4, EPI>(a, batch, c.splits, s);
}
struct Buffers {
  _Float16 *X, *XT[2], *A, *M;
  float *master_x, *master_a;
  int *exp_r, *exp_c;
};
int run_steps(const Plan &p, int steps, NsArgs a, const Buffers &w, hipStream_t s) {
  const int batch = p.batch;
  Known known = known_at_start(a.b, a.c);
  for (int k = 0; k < steps; ++k) {
    const Known next = grown(known, a.a, a.b, a.c);
    NsArgs g = a;
    g.shift = known.shift;
    g.cap = known.cap;
    g.poly = known.poly;
    g.next_shift = next.shift;
    g.next_cap = next.cap;
    g.P = g.Q = w.X;
    g.p_stride = g.q_stride = 2 * p.x;
    g.ldp = g.ldq = g.K = p.cp;
    g.rows_p = g.rows_q = p.rp;
    g.D = g.DT = w.A;
    g.d_stride = g.dt_stride = 2 * p.sq;
    g.ldd = g.lddt = p.rp;
    g.exp_m = g.exp_n = w.exp_r;
    g.exp_m_stride = g.exp_n_stride = p.rp;
    g.master = w.master_a;
    g.master_stride = p.sq;
    if (int rc = launch_gemm<GRAM>(g, batch, s)) return rc;
    g.P = g.Q = w.A;
    g.p_stride = g.q_stride = 2 * p.sq;
    g.ldp = g.ldq = g.K = p.rp;
    g.D = g.DT = w.M;
    if (int rc = launch_gemm<POLY>(g, batch, s)) return rc;
    g.P = w.M;
    g.Q = w.XT[k & 1];
    g.q_stride = 2 * p.x;
    g.rows_q = p.cp;
    g.D = w.X;
    g.DT = w.XT[1 - (k & 1)];
    g.d_stride = g.dt_stride = 2 * p.x;
    g.ldd = p.cp;
    g.exp_n = w.exp_c;
    g.exp_n_stride = p.cp;
    g.master = w.master_x;
    g.master_stride = p.x;
    if (int rc = k + 1 < steps ? launch_gemm<UPDATE>(g, batch, s) : launch_gemm<FINAL>(g, batch, s)) return rc;
    known = next;
  }
  return DX_OK;
}

template <typename V>
int launch_start(const V *update, const Plan &p, PackArgs k, double *sums, float *row_most, float *col_most, hipStream_t s) {
  hipLaunchKernelGGL(ns_scan_kernel<V>, dim3(p.scan.strips, p.scan.bands, p.batch), dim3(256), 0, s, update, k.m, k.n, p.scan.band, p.scan.strip, sums, row_most,
                     col_most);
  DX_LAUNCH_CHECK();
  hipLaunchKernelGGL(ns_pack_kernel<V>, dim3(cdiv(k.n, kPad), cdiv(k.m, kPad), p.batch), dim3(256), 0, s, k);
  DX_LAUNCH_CHECK();
  return DX_OK;
}

// every step's products as launches, p.batch matrices
int run_launches(const Plan &p, const void *update, int dtype, int m, int n, int steps, float a, float b, float c, float eps, void *out,
                 void *workspace, hipStream_t s) {
  char *at = static_cast<char *>(workspace);
  auto take = [&](auto *&to, long long count) {
    to = reinterpret_cast<std::remove_reference_t<decltype(to)>>(at);
    at += count * static_cast<long long>(sizeof(*to));
  };
  Buffers w;
  float *split, *row_most, *col_most;
  double *sums;
  unsigned *arrivals;
  take(w.X, 2 * p.x * p.batch);
  take(w.XT[0], 2 * p.x * p.batch);
  take(w.XT[1], 2 * p.x * p.batch);
  take(w.A, 2 * p.sq * p.batch);
  take(w.M, 2 * p.sq * p.batch);
  take(w.master_x, p.x * p.batch);
  take(w.master_a, p.sq * p.batch);
  take(split, p.split_floats);
  take(sums, p.sums * p.batch);
  take(w.exp_r, static_cast<long long>(p.rp) * p.batch);
  take(w.exp_c, static_cast<long long>(p.cp) * p.batch);
  take(arrivals, kSplitGroups);
  take(row_most, static_cast<long long>(m) * p.scan.strips * p.batch);
  take(col_most, static_cast<long long>(n) * p.scan.bands * p.batch);
  const bool tall = m > n;
  PackArgs k{};
  k.in = update;
  k.m = m;
  k.n = n;
  k.tall = tall;
  k.bands = p.scan.bands;
  k.strips = p.scan.strips;
  k.sums = sums;
  k.row_most = row_most;
  k.col_most = col_most;
  k.eps = eps;
  k.same = tall ? w.XT[0] : w.X;
  k.turned = tall ? w.X : w.XT[0];
  k.ld_same = tall ? p.rp : p.cp;
  k.ld_turned = tall ? p.cp : p.rp;
  k.stride = 2 * p.x;
  k.master = w.master_x;
  k.master_stride = p.x;
  k.rows_x = p.rp;
  k.exp_row = tall ? w.exp_c : w.exp_r;
  k.exp_col = tall ? w.exp_r : w.exp_c;
  k.exp_row_stride = tall ? p.cp : p.rp;
  k.exp_col_stride = tall ? p.rp : p.cp;
  k.cap = known_at_start(b, c).cap;
  k.arrivals = arrivals;
  k.counts = kSplitGroups;
  if (int rc = dtype == DX_F32 ? launch_start(static_cast<const float *>(update), p, k, sums, row_most, col_most, s)
               : dtype == DX_BF16 ? launch_start(static_cast<const __bf16 *>(update), p, k, sums, row_most, col_most, s)
                                  : launch_start(static_cast<const _Float16 *>(update), p, k, sums, row_most, col_most, s)) return rc;
  NsArgs g{};
  g.arrivals = arrivals;
  g.partials = split;
  g.split_floats = p.split_floats;
  g.a = a;
  g.b = b;
  g.c = c;
  g.out = out;
  g.dtype = dtype;
  g.r = p.r;
  g.cols = p.c;
  g.tall = tall;
  return run_steps(p, steps, g, w, s);
}

}  // namespace
}  // namespace dx

extern "C" long long dx_orthogonalize_workspace(int dtype, int batch, int m, int n) {
  DX_TRACE("dx_orthogonalize_workspace");
  if (int rc = dx::check_shape(dtype, batch, m, n)) return rc;
  return dx::make_plan(dtype, batch, m, n).bytes;
}

extern "C" int dx_orthogonalize(const void *update, int dtype, int batch, int m, int n, int steps, float a, float b, float c, float eps,
                                void *out, void *workspace, long long workspace_bytes, void *stream) {
  DX_TRACE("dx_orthogonalize");
  using namespace dx;
  if (int rc = check_shape(dtype, batch, m, n)) return rc;
  DX_REQUIRE(steps >= 1, "dx_orthogonalize: steps %d < 1", steps);
  if (batch == 0) return DX_OK;
  const int size = dtype == DX_F32 ? 4 : 2;
  DX_REQUIRE(update && out && workspace, "dx_orthogonalize: null pointer");
  DX_REQUIRE(aligned(update, size) && aligned(out, size) && aligned(workspace, 256), "dx_orthogonalize: misaligned pointer");
  const Plan p = make_plan(dtype, batch, m, n);
  if (workspace_bytes < p.bytes) return fail(DX_EWS, "dx_orthogonalize: workspace of %lld bytes, %lld needed", workspace_bytes, p.bytes);
  hipStream_t s = as_stream(stream);
  if (p.one_launch && steps <= kSmallSteps) {
    const int r32 = cdiv(p.r, 32) * 32, c32 = cdiv(p.c, 32) * 32;
    SmallArgs q{update, out, m, n, p.r, p.c, r32, c32, steps, m > n, a, b, c, eps, {}};
    Known known = known_at_start(b, c);
    for (int i = 0; i <= steps; ++i, known = grown(known, a, b, c)) q.powers[i] = known;
    const int bytes = static_cast<int>(small_lds(r32, c32));
    if (dtype == DX_F32) return launch_small<float>(q, batch, bytes, s);
    if (dtype == DX_BF16) return launch_small<__bf16>(q, batch, bytes, s);
    return launch_small<_Float16>(q, batch, bytes, s);
  }
  const long long bytes = static_cast<long long>(m) * n * size;
  for (int z = 0; z < batch; z += p.batch) {
    const char *from = static_cast<const char *>(update) + z * bytes;
    if (int rc = run_launches(p, from, dtype, m, n, steps, a, b, c, eps, static_cast<char *>(out) + z * bytes, workspace, s)) return rc;
  }
  return DX_OK;
}
