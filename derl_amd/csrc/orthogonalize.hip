// Newton-Schulz orthogonalisation of an update (gfx950):
//   X0 = G / (|G|_F + eps),   A = X X^T,   B = a I + b A + c A^2,   X <- B X        (`steps` times)
// with X the (r, c) matrix whose shorter side is r (a tall G is worked on transposed).  Odd polynomials of the singular
// values only: the singular vectors stay G's, the singular values approach 1.
//
// The products run on the fp16 matrix cores with fp32 accumulation.  Whatever the matrix's type, X, A and B are held as TWO fp16
// terms, hi + lo (22 bits): a product is hi hi + hi lo + lo hi (the dropped lo lo is 2^-22 of it), fp32 accuracy at a third of the
// fp16 rate, where the fp32 matrix instructions have a sixteenth.  (bf16 too: with one term, 11 bits, each step multiplies what
// is lost by up to `a` = 3.4, and a bf16 result was off by 1.1 to 2.5 times its own rounding; with two it is off by that alone.)
// Stored values are scaled by powers of two (X by 2^12, A and B by 2^8), so that neither large entries overflow nor the second
// term of typical ones (1 / sqrt(c)) falls under fp16's smallest step.
//
// Every matrix product is C = P Q^T with both operands' k contiguous: X for A = X X^T, A = A^T for A^2 = A A^T, and for
// B X the transposed copy X^T, which the epilogue of each update writes beside X.  A and B are symmetric: only tiles on
// and above the diagonal are formed and stored twice.  Both sides are padded
// to a multiple of 64 with zeros in the workspace.
#include <cmath>
#include <type_traits>

#include "igemm_dev.hpp"

namespace dx {
namespace {

using f32x4 = __attribute__((ext_vector_type(4))) float;
using u32x2 = __attribute__((ext_vector_type(2))) uint32_t;
using u32x4 = __attribute__((ext_vector_type(4))) uint32_t;
using f16x4 = __attribute__((ext_vector_type(4))) _Float16;
using f16x8 = __attribute__((ext_vector_type(8))) _Float16;

constexpr float kScaleX = 4096.f, kScaleA = 256.f;
constexpr int kPad = 64, kNormParts = 512;
constexpr int kSplitGroups = 512;  // workgroups of a product that is split over K, at most

constexpr int kStageK = 32;        // k of a stage of a product

enum Epilogue { GRAM, POLY, UPDATE, FINAL };

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
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      const int m0 = bm * TM + (wm * FM + i) * 32, n0 = bn * TM + (wn * FN + j) * 32;
      if (m0 >= a.rows_p || n0 >= a.rows_q) continue;  // (32-row blocks are whole)
      const int n = n0 + l31;
      uint32_t h[4][2], l[4][2];
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int m = m0 + 8 * g + 4 * hi;
        float v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = acc[i][j][4 * g + k];
        if constexpr (EPI == GRAM) {
#pragma unroll
          for (int k = 0; k < 4; ++k) v[k] *= kScaleA / (kScaleX * kScaleX);
        } else if constexpr (EPI == POLY) {
          const _Float16 *at = a.P + z * a.p_stride + place(n, m, a.ldp);  // A[n][m] = A[m][n]
          const f16x4 ah = *reinterpret_cast<const f16x4 *>(at), al = *reinterpret_cast<const f16x4 *>(at + kSecond);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            v[k] = a.c * (v[k] * (1.f / kScaleA)) + a.b * (static_cast<float>(ah[k]) + static_cast<float>(al[k])) +
                   (m + k == n ? a.a * kScaleA : 0.f);
        } else if constexpr (EPI == UPDATE) {
#pragma unroll
          for (int k = 0; k < 4; ++k) v[k] *= 1.f / kScaleA;
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k) v[k] *= 1.f / (kScaleA * kScaleX);
          put_final(a, z, m, n, n0 + (l31 & ~3), lane, v);
          continue;
        }
        f16x4 vh, vl;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          vh[k] = static_cast<_Float16>(v[k]);
          vl[k] = static_cast<_Float16>(v[k] - static_cast<float>(vh[k]));
        }
        const u32x2 bh = __builtin_bit_cast(u32x2, vh), bl = __builtin_bit_cast(u32x2, vl);
        h[g][0] = bh.x;
        h[g][1] = bh.y;
        l[g][0] = bl.x;
        l[g][1] = bl.y;
        if (EPI == UPDATE || bm != bn) {
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

// this thread's share of a sum of squares over `count` values: thread `at` of `threads`
template <typename V>
__device__ __forceinline__ double sum_of_squares(const V *g, long long count, long long at, long long threads) {
  constexpr int E = 16 / sizeof(V);
  using Vec = __attribute__((ext_vector_type(E))) V;
  typedef Vec Loose __attribute__((aligned(sizeof(V))));  // a matrix of the batch may start at any element
  double s = 0;
  const long long vectors = count / E;
#pragma unroll 4
  for (long long i = at; i < vectors; i += threads) {
    const Vec v = *reinterpret_cast<const Loose *>(g + i * E);
#pragma unroll
    for (int k = 0; k < E; ++k) {
      const double x = static_cast<double>(static_cast<float>(v[k]));
      s += x * x;
    }
  }
  if (vectors * E + at < count) {  // fewer than E values are left: one each for the first threads
    const double x = static_cast<double>(static_cast<float>(g[vectors * E + at]));
    s += x * x;
  }
  return s;
}

// kScaleX / (|G| + eps) as a fraction in [1/2, 1) and a power of two: the norm may lie outside fp32's range.  (A product in
// double that goes on to fp16 is converted by 30 integer instructions: packing 512 x 3136 f32 took 14.4 us, 9.8 so.)
struct Scale {
  float fraction;
  int power;
};
__device__ __forceinline__ Scale scale_of(double squares, float eps) {
  Scale s;
  s.fraction = static_cast<float>(frexp(kScaleX / (sqrt(squares) + eps), &s.power));
  return s;
}
__device__ __forceinline__ float scaled(float x, const Scale &s) { return ldexpf(x * s.fraction, s.power); }

// sums of squares, gridDim.x partial sums per matrix
template <typename V>
__global__ __launch_bounds__(256) void ns_norm_kernel(const V *in, long long count, double *partials) {
  __shared__ double scratch[4];
  double s = sum_of_squares(in + blockIdx.y * count, count, blockIdx.x * 256LL + threadIdx.x, 256LL * gridDim.x);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
  if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) partials[blockIdx.y * static_cast<long long>(gridDim.x) + blockIdx.x] = scratch[0] + scratch[1] + scratch[2] + scratch[3];
}

// X0 and its transpose from a 64 x 64 tile of G: `same` has G's orientation (ld_same), `turned` the other.  Also clears the
// arrival counts of the split products.
template <typename V>
__global__ __launch_bounds__(256) void ns_pack_kernel(const V *in, int m, int n, const double *partials, int parts, float eps, _Float16 *same,
                                                      int ld_same, _Float16 *turned, int ld_turned, long long stride, unsigned *arrivals, int counts) {
  constexpr int E = 16 / sizeof(V);
  using Vec = __attribute__((ext_vector_type(E))) V;
  typedef Vec Loose __attribute__((aligned(sizeof(V))));
  __shared__ float tile[64][65];
  __shared__ double total[4];
  const long long z = blockIdx.z;
  const int c0 = blockIdx.x * 64, r0 = blockIdx.y * 64;
  const V *g = in + z * m * n;
  if (blockIdx.x == 0 && blockIdx.y == 0 && z == 0)
    for (int i = threadIdx.x; i < counts; i += 256) arrivals[i] = 0;
  // 64 rows of 64 / E vectors, all on their way before the first is waited for
  constexpr int kVecs = 64 * 64 / E / 256;
  Vec v[kVecs];
  if (r0 + 64 <= m && c0 + 64 <= n) {
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
      const int at = k * 256 + threadIdx.x;
      v[k] = *reinterpret_cast<const Loose *>(g + static_cast<long long>(r0 + at / (64 / E)) * n + c0 + at % (64 / E) * E);
    }
  } else {
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
      const int at = k * 256 + threadIdx.x, row = at / (64 / E), col = at % (64 / E) * E;
      v[k] = Vec{};
      if (r0 + row < m) {
        const V *from = g + static_cast<long long>(r0 + row) * n + c0 + col;
        if (c0 + col + E <= n) v[k] = *reinterpret_cast<const Loose *>(from);
        else
#pragma unroll
          for (int i = 0; i < E; ++i)
            if (c0 + col + i < n) v[k][i] = from[i];
      }
    }
  }
  double s = 0;
  for (int i = threadIdx.x; i < parts; i += 256) s += partials[z * parts + i];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
  if ((threadIdx.x & 63) == 0) total[threadIdx.x >> 6] = s;
#pragma unroll
  for (int k = 0; k < kVecs; ++k) {
    const int at = k * 256 + threadIdx.x;
#pragma unroll
    for (int i = 0; i < E; ++i) tile[at / (64 / E)][at % (64 / E) * E + i] = static_cast<float>(v[k][i]);
  }
  __syncthreads();
  const Scale scale = scale_of(total[0] + total[1] + total[2] + total[3], eps);
  const int mp = (m + kPad - 1) / kPad * kPad, np = (n + kPad - 1) / kPad * kPad;
  auto put8 = [&](_Float16 *at, auto value) {
    f16x8 h, l;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float v = scaled(value(i), scale);
      h[i] = static_cast<_Float16>(v);
      l[i] = static_cast<_Float16>(v - static_cast<float>(h[i]));
    }
    *reinterpret_cast<f16x8 *>(at) = h;
    *reinterpret_cast<f16x8 *>(at + kSecond) = l;
  };
#pragma unroll
  for (int k = 0; k < 2; ++k) {  // 64 rows of 8 x 8 values; the sides are multiples of 64: a row of 8 is whole or outside
    const int at = k * 256 + threadIdx.x, row = at >> 3, col = (at & 7) * 8;
    if (r0 + row < mp && c0 + col < np) put8(same + z * stride + place(r0 + row, c0 + col, ld_same), [&](int i) { return tile[row][col + i]; });
    if (c0 + row < np && r0 + col < mp) put8(turned + z * stride + place(c0 + row, r0 + col, ld_turned), [&](int i) { return tile[col + i][row]; });
  }
}

// ---- matrices that fit a workgroup's LDS: the whole iteration in ONE launch, a workgroup per matrix -----------------
// X, X^T, A and B stay in LDS (rows padded by 16 bytes: an odd number of 16-byte chunks, so that 16 rows' equal chunks meet
// every bank once); 16 waves share the 16 x 16 x 32 tiles of each product.  The update holds its tiles in registers over a
// barrier and then overwrites X and X^T.  What bounds it is the chain of 3 x steps dependent products, not their rate.
// LDS is addressed by plain offsets into one array: through pointers that are chosen at run time the compiler cannot see that
// they are LDS, and flat accesses and spills made a step of 64 x 64 f32 3.9 us long (1.5 now).
constexpr int kSmallWaves = 16;
constexpr long long kSmallLds = 160 * 1024 - 256;

inline long long small_lds(int rp, int cp) {
  if (rp > 64 && rp / 32 * (cp / 32) > kSmallWaves) return kSmallLds + 1;  // more blocks of 32 x 32 than waves: see launch_small
  return 4LL * (static_cast<long long>(rp) * (cp + 8) + static_cast<long long>(cp) * (rp + 8)) + 8LL * rp * (rp + 8);
}

struct SmallArgs {
  const void *in;
  void *out;
  int m, n, r, c, rp, cp, steps, tall;
  float a, b, k, eps;
};

// SIDE: the products are formed in blocks of 16 x 16 (one instruction tile: the shortest chain, and enough blocks of A for the
// waves up to 64 rows) or 32 x 32 (two fragments of each side for four tiles: half the LDS reads).  us for 5 steps: 17 x 300 f32
// 20 at 16, 32 at 32; 64 x 400 bf16 35, 38; 128 x 128 bf16 40, 34.
// COLUMN = 0: X has no more blocks than there are waves; a block is held over a barrier before it overwrites X.
// COLUMN > 0: a wave takes columns of blocks, which depend on nothing but themselves: held, COLUMN of them at most, without a
// barrier, their X^T fragments read once (64 x 400 bf16: blocks dealt out, held and written by straight code 51 us, half of
// them its instruction fetches; by columns 35).
template <typename V, int SIDE, int COLUMN>
__global__ __launch_bounds__(kSmallWaves * 64) void ns_small_kernel(const SmallArgs a) {
  extern __shared__ __attribute__((aligned(16))) _Float16 lds[];
  __shared__ double parts[kSmallWaves];
  const int tid = threadIdx.x, lane = tid & 63, l15 = lane & 15, quad = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int ldx = a.cp + 8, ldr = a.rp + 8;  // X: rp rows of ldx; X^T: cp rows of ldr; A, B: rp rows of ldr
  // each array: its first terms, then its second ones
  const int sx = a.rp * ldx, st = a.cp * ldr, sa = a.rp * ldr;
  const int X = 0, XT = X + 2 * sx, A = XT + 2 * st, B = A + 2 * sa;
  auto put1 = [&](int at, int size, float v) {
    const _Float16 h = static_cast<_Float16>(v);
    lds[at] = h;
    lds[at + size] = static_cast<_Float16>(v - static_cast<float>(h));
  };
  // four consecutive rows of a column: into the row of the transpose (`turned`) and, if wanted, into four rows (`at`, ld apart)
  auto put4 = [&](int turned, int turned_size, int at, int ld, int size, bool both, f32x4 v) {
    f16x4 h, l;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      h[k] = static_cast<_Float16>(v[k]);
      l[k] = static_cast<_Float16>(v[k] - static_cast<float>(h[k]));
    }
    *reinterpret_cast<f16x4 *>(lds + turned) = h;
    *reinterpret_cast<f16x4 *>(lds + turned + turned_size) = l;
    if (both) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        lds[at + k * ld] = h[k];
        lds[at + k * ld + size] = l[k];
      }
    }
  };
  const int count = a.m * a.n;
  const V *in = static_cast<const V *>(a.in) + blockIdx.x * static_cast<long long>(count);
  double s = sum_of_squares(in, count, tid, kSmallWaves * 64);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
  if (lane == 0) parts[wave] = s;
  __syncthreads();
  s = 0;
#pragma unroll
  for (int i = 0; i < kSmallWaves; ++i) s += parts[i];
  const Scale scale = scale_of(s, a.eps);
  for (int row = wave; row < a.rp; row += kSmallWaves)  // a wave per row of X, 256 columns' loads at a time
    for (int col0 = lane; col0 < a.cp; col0 += 256) {
      V g[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int col = min(col0 + 64 * k, a.c - 1), from = min(row, a.r - 1);
        g[k] = in[a.tall ? col * a.n + from : from * a.n + col];
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int col = col0 + 64 * k;
        if (col >= a.cp) continue;
        const float v = row < a.r && col < a.c ? scaled(static_cast<float>(g[k]), scale) : 0.f;
        put1(X + row * ldx + col, sx, v);
        put1(XT + col * ldr + row, st, v);
      }
    }
  __syncthreads();
  // acc[i] = rows SIDE i .. of P times SIDE rows of Q transposed, the first `count` of N blocks.  Accumulator e of a lane and
  // 16 x 16 tile: row 4 (lane / 16) + e, column lane % 16
  constexpr int F = SIDE / 16, kHeld = COLUMN > 0 ? COLUMN : 1;
  struct Block { f32x4 v[F][F]; };
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
  const int tr = a.rp / SIDE, tc = a.cp / SIDE, upper = tr * (tr + 1) / 2;
#pragma unroll 1
  for (int step = 0; step < a.steps; ++step) {
    // A = X X^T, then B = a I + b A + c A A: their upper triangles, stored twice
#pragma unroll 1
    for (int half = 0; half < 2; ++half) {
      const int to = half ? B : A;
#pragma unroll 1
      for (int tile = wave; tile < upper; tile += kSmallWaves) {
        int left = tile, row = 0;
        while (left >= tr - row) left -= tr - row++;
        const int pm = row * SIDE, qn = (row + left) * SIDE;
        Block acc[1];
        if (half) products(acc, 1, A + pm * ldr, ldr, sa, A + qn * ldr, ldr, sa, a.rp);
        else products(acc, 1, X + pm * ldx, ldx, sx, X + qn * ldx, ldx, sx, a.cp);
#pragma unroll
        for (int f = 0; f < F; ++f)
#pragma unroll
          for (int g = 0; g < F; ++g) {
            const int m = pm + f * 16 + 4 * quad, n = qn + g * 16 + l15;
            f32x4 v = acc[0].v[f][g] * (half ? a.k / kScaleA : kScaleA / (kScaleX * kScaleX));
            if (half) {
              const f16x4 h = *reinterpret_cast<const f16x4 *>(lds + A + n * ldr + m);
              const f16x4 l = *reinterpret_cast<const f16x4 *>(lds + A + n * ldr + m + sa);
#pragma unroll
              for (int k = 0; k < 4; ++k) v[k] += a.b * (static_cast<float>(h[k]) + static_cast<float>(l[k])) + (m + k == n ? a.a * kScaleA : 0.f);
            }
            put4(to + n * ldr + m, sa, to + m * ldr + n, ldr, sa, pm != qn, v);
          }
      }
      __syncthreads();
    }
    const bool last = step + 1 == a.steps;
    auto put_block = [&](int tm, int tn, const Block &b) {
#pragma unroll
      for (int f = 0; f < F; ++f)
#pragma unroll
        for (int g = 0; g < F; ++g) {
          const int m = tm * SIDE + f * 16 + 4 * quad, n = tn * SIDE + g * 16 + l15;
          const f32x4 v = b.v[f][g] * (1.f / kScaleA);
          if (!last) {
            put4(XT + n * ldr + m, st, X + m * ldx + n, ldx, sx, true, v);
          } else {
            V *out = static_cast<V *>(a.out) + blockIdx.x * static_cast<long long>(count);
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (m + k < a.r && n < a.c) out[a.tall ? n * a.n + m + k : (m + k) * a.n + n] = static_cast<V>(v[k] * (1.f / kScaleX));
          }
        }
    };
    Block held[kHeld];
    if constexpr (COLUMN == 0) {
      if (wave < tr * tc) products(held, 1, B + wave % tr * SIDE * ldr, ldr, sa, XT + wave / tr * SIDE * ldr, ldr, st, a.rp);
      __syncthreads();
      if (wave < tr * tc) put_block(wave % tr, wave / tr, held[0]);
    } else {
#pragma unroll 1
      for (int tn = wave; tn < tc; tn += kSmallWaves) {
        products(held, tr, B, ldr, sa, XT + tn * SIDE * ldr, ldr, st, a.rp);
#pragma unroll
        for (int i = 0; i < COLUMN; ++i)
          if (i < tr) put_block(i, tn, held[i]);
      }
    }
    __syncthreads();
  }
}

template <typename V, int SIDE, int COLUMN>
int launch_small_as(const SmallArgs &q, int batch, int bytes, hipStream_t s) {
  DX_LDS_OPT_IN((ns_small_kernel<V, SIDE, COLUMN>), kSmallLds);
  hipLaunchKernelGGL((ns_small_kernel<V, SIDE, COLUMN>), dim3(batch), dim3(kSmallWaves * 64), bytes, s, q);
  DX_LAUNCH_CHECK();
  return DX_OK;
}
template <typename V>
int launch_small(const SmallArgs &q, int batch, int bytes, hipStream_t s) {
  const int blocks = q.rp / 32 * (q.cp / 32);
  if (blocks * 4 <= kSmallWaves) return launch_small_as<V, 16, 0>(q, batch, bytes, s);
  if (q.rp <= 32) return launch_small_as<V, 16, 2>(q, batch, bytes, s);
  if (q.rp <= 64) return launch_small_as<V, 16, 4>(q, batch, bytes, s);
  return launch_small_as<V, 32, 0>(q, batch, bytes, s);
}

struct Plan {
  int r, c, rp, cp, parts;
  long long x, sq;             // halves of X and of A per matrix, both terms, padded
  long long split_floats, bytes;
};
Plan make_plan(int dtype, int batch, int m, int n) {
  Plan p;
  p.r = m < n ? m : n;
  p.c = m < n ? n : m;
  p.rp = (p.r + kPad - 1) / kPad * kPad;
  p.cp = (p.c + kPad - 1) / kPad * kPad;
  p.x = 2LL * p.rp * p.cp;
  p.sq = 2LL * p.rp * p.rp;
  // X, two copies of X^T, A, B, and the norm's partial sums
  const long long blocks = (static_cast<long long>(m) * n * (dtype == DX_F32 ? 4 : 2) + 32767) / 32768;  // 32 KB a workgroup at least
  p.parts = static_cast<int>(blocks < kNormParts ? blocks : kNormParts);
  p.split_floats = static_cast<long long>(kSplitGroups) * (p.r > 1024 ? 128 * 128 : 64 * 64);  // (128 x 128 tiles are split where there are many)
  p.bytes = batch * (2 * (3 * p.x + 2 * p.sq) + 8LL * p.parts) + 4LL * kSplitGroups + 4 * p.split_floats;
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
// 1.9 with the chip full, where the package's power bounds them.  Split parts exchange their sums: 8 us and 8 bytes a value.
// Measured, us a product: 2001 x 5003 f32 X X^T at 128 one part 126, three parts 94; 64, 192, 256: 127, 170, 258; its
// update 178, 147, 177, 139 at 64, 128, 192, 256.  512 x 3136 f32 X X^T at 64: one part 23, seven 14; its update 14.6, 22, 35, 52.
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
int run_steps(const Plan &p, int batch, int steps, NsArgs a, _Float16 *X, _Float16 *XT0, _Float16 *XT1, _Float16 *A, _Float16 *B, hipStream_t s) {
  for (int k = 0; k < steps; ++k) {
    _Float16 *xt = k & 1 ? XT1 : XT0, *next = k & 1 ? XT0 : XT1;
    NsArgs g = a;
    g.P = g.Q = X;
    g.p_stride = g.q_stride = p.x;
    g.ldp = g.ldq = g.K = p.cp;
    g.rows_p = g.rows_q = p.rp;
    g.D = g.DT = A;
    g.d_stride = g.dt_stride = p.sq;
    g.ldd = g.lddt = p.rp;
    if (int rc = launch_gemm<GRAM>(g, batch, s)) return rc;
    g.P = g.Q = A;
    g.p_stride = g.q_stride = p.sq;
    g.ldp = g.ldq = g.K = p.rp;
    g.D = g.DT = B;
    if (int rc = launch_gemm<POLY>(g, batch, s)) return rc;
    g.P = B;
    g.Q = xt;
    g.q_stride = p.x;
    g.rows_q = p.cp;
    g.D = X;
    g.DT = next;
    g.d_stride = g.dt_stride = p.x;
    g.ldd = p.cp;
    if (int rc = k + 1 < steps ? launch_gemm<UPDATE>(g, batch, s) : launch_gemm<FINAL>(g, batch, s)) return rc;
  }
  return DX_OK;
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
  if (small_lds(cdiv(p.r, 32) * 32, cdiv(p.c, 32) * 32) <= kSmallLds) {
    const int r32 = cdiv(p.r, 32) * 32, c32 = cdiv(p.c, 32) * 32;
    const SmallArgs q{update, out, m, n, p.r, p.c, r32, c32, steps, m > n, a, b, c, eps};
    const int bytes = static_cast<int>(small_lds(r32, c32));
    if (dtype == DX_F32) return launch_small<float>(q, batch, bytes, s);
    if (dtype == DX_BF16) return launch_small<__bf16>(q, batch, bytes, s);
    return launch_small<_Float16>(q, batch, bytes, s);
  }
  _Float16 *at = static_cast<_Float16 *>(workspace);
  auto take = [&](long long halves) {
    _Float16 *t = at;
    at += halves * batch;
    return t;
  };
  _Float16 *X = take(p.x), *XT0 = take(p.x), *XT1 = take(p.x), *A = take(p.sq), *B = take(p.sq);
  double *partials = reinterpret_cast<double *>(at);
  unsigned *arrivals = reinterpret_cast<unsigned *>(partials + static_cast<long long>(batch) * p.parts);
  float *split = reinterpret_cast<float *>(arrivals + kSplitGroups);
  const long long count = static_cast<long long>(m) * n;
  if (dtype == DX_F32) hipLaunchKernelGGL(ns_norm_kernel<float>, dim3(p.parts, batch), dim3(256), 0, s, static_cast<const float *>(update), count, partials);
  else if (dtype == DX_BF16) hipLaunchKernelGGL(ns_norm_kernel<__bf16>, dim3(p.parts, batch), dim3(256), 0, s, static_cast<const __bf16 *>(update), count, partials);
  else hipLaunchKernelGGL(ns_norm_kernel<_Float16>, dim3(p.parts, batch), dim3(256), 0, s, static_cast<const _Float16 *>(update), count, partials);
  DX_LAUNCH_CHECK();
  const bool tall = m > n;
  const dim3 grid(cdiv(tall ? p.rp : p.cp, 64), cdiv(tall ? p.cp : p.rp, 64), batch);
  _Float16 *same = tall ? XT0 : X, *turned = tall ? X : XT0;
  const int ld_same = tall ? p.rp : p.cp, ld_turned = tall ? p.cp : p.rp;
  if (dtype == DX_F32)
    hipLaunchKernelGGL((ns_pack_kernel<float>), grid, dim3(256), 0, s, static_cast<const float *>(update), m, n, partials, p.parts, eps,
                       same, ld_same, turned, ld_turned, p.x, arrivals, kSplitGroups);
  else if (dtype == DX_BF16)
    hipLaunchKernelGGL((ns_pack_kernel<__bf16>), grid, dim3(256), 0, s, static_cast<const __bf16 *>(update), m, n, partials, p.parts, eps,
                       same, ld_same, turned, ld_turned, p.x, arrivals, kSplitGroups);
  else
    hipLaunchKernelGGL((ns_pack_kernel<_Float16>), grid, dim3(256), 0, s, static_cast<const _Float16 *>(update), m, n, partials, p.parts,
                       eps, same, ld_same, turned, ld_turned, p.x, arrivals, kSplitGroups);
  DX_LAUNCH_CHECK();
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
  return run_steps(p, batch, steps, g, X, XT0, XT1, A, B, s);
}
