// Newton-Schulz orthogonalisation of an update (gfx950):
//   X0 = G / (|G|_F + eps),   A = X X^T,   B = a I + b A + c A^2,   X <- B X        (`steps` times)
// with X the (r, c) matrix whose shorter side is r (a tall G is worked on transposed).  Odd polynomials of the singular
// values only: the singular vectors stay G's, the singular values approach 1.
//
// The products run on the fp16 matrix cores with fp32 accumulation.  fp32 input is held as TWO fp16 terms, hi + lo
// (22 bits), and a product is hi hi + hi lo + lo hi (the dropped lo lo is 2^-22 of it): fp32 accuracy at a third of the
// fp16 rate, where the fp32 matrix instructions have a sixteenth.  16-bit input is held as one fp16 term: 11 bits, three
// more than bf16 keeps, which the iteration needs -- each step multiplies the error of small singular values by up to
// `a` = 3.4.  Stored values are scaled by powers of two (X by 2^12, A and B by 2^8), so that neither large entries
// overflow nor the second term of typical ones (1 / sqrt(c)) falls under fp16's smallest step.
//
// Every matrix product is C = P Q^T with both operands' k contiguous: X for A = X X^T, A = A^T for A^2 = A A^T, and for
// B X the transposed copy X^T, which the epilogue of each update writes beside X.  A and B are symmetric: only tiles on
// and above the diagonal are formed and stored twice.  All sizes are padded to the tile with zeros in the workspace.
#include "igemm_dev.hpp"

namespace dx {
namespace {

using f16x4 = __attribute__((ext_vector_type(4))) _Float16;
using f16x8 = __attribute__((ext_vector_type(8))) _Float16;

constexpr float kScaleX = 4096.f, kScaleA = 256.f;
constexpr int kPad = 128, kBK = 64, kNormParts = 64;

enum Epilogue { GRAM, POLY, UPDATE, FINAL };

struct Terms { _Float16 *hi, *lo; };  // lo: unused with one term

struct NsArgs {
  Terms P, Q;             // operands: rows of K contiguous values
  long long p_stride, q_stride;  // values from one matrix of the batch to the next
  int ldp, ldq, K;
  int tiles_m, tiles_n;   // tiles of TM rows of P / Q
  Terms D, DT;            // [m][n] and its transpose [n][m]
  long long d_stride, dt_stride;
  int ldd, lddt;
  float a, b, c;
  // FINAL
  void *out;
  int dtype, r, cols, tall;
};

__device__ __forceinline__ void put_terms(const Terms &t, long long at, float v, bool two) {
  const _Float16 h = static_cast<_Float16>(v);
  t.hi[at] = h;
  if (two) t.lo[at] = static_cast<_Float16>(v - static_cast<float>(h));
}
__device__ __forceinline__ void put_terms4(const Terms &t, long long at, const float (&v)[4], bool two) {
  f16x4 h, l;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    h[k] = static_cast<_Float16>(v[k]);
    l[k] = static_cast<_Float16>(v[k] - static_cast<float>(h[k]));
  }
  *reinterpret_cast<f16x4 *>(t.hi + at) = h;
  if (two) *reinterpret_cast<f16x4 *>(t.lo + at) = l;
}

__device__ __forceinline__ void put_out(void *out, int dtype, long long at, float v) {
  if (dtype == DX_F32) static_cast<float *>(out)[at] = v;
  else if (dtype == DX_BF16) static_cast<__bf16 *>(out)[at] = static_cast<__bf16>(v);
  else static_cast<_Float16 *>(out)[at] = static_cast<_Float16>(v);
}
__device__ __forceinline__ float get_in(const void *in, int dtype, long long at) {
  if (dtype == DX_F32) return static_cast<const float *>(in)[at];
  if (dtype == DX_BF16) return static_cast<float>(static_cast<const __bf16 *>(in)[at]);
  return static_cast<float>(static_cast<const _Float16 *>(in)[at]);
}

// 256 threads: 2 x 2 waves of TM/2 x TM/2 (32 x 32 x 16 instructions).  Operands arrive by LDS-DMA, two K stages of 64;
// a row of a stage is 128 bytes = 8 chunks of 16, slot s holds chunk s ^ ((row >> 1) & 7) (conflict-free ds_read_b128:
// the 16 lanes of a group meet every bank once).
template <int TM, int TERMS, Epilogue EPI>
__global__ __launch_bounds__(256) void ns_gemm_kernel(const NsArgs a) {
  extern __shared__ __attribute__((aligned(16))) float smem[];
  constexpr int F = TM / 64;                 // 32 x 32 tiles per wave and side
  constexpr int kArray = TM * kBK * 2;       // bytes of one operand term of a stage
  constexpr int kStage = 2 * TERMS * kArray;
  constexpr int kPieces = TM / 8;            // 1 KiB pieces of an array
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int z = blockIdx.y;
  int bm, bn;
  if (EPI == GRAM || EPI == POLY) {  // the upper triangle, row by row
    int left = blockIdx.x, row = 0;
    while (left >= a.tiles_m - row) left -= a.tiles_m - row++;
    bm = row;
    bn = row + left;
  } else {
    bm = blockIdx.x % a.tiles_m;
    bn = blockIdx.x / a.tiles_m;
  }
  const _Float16 *src[2 * TERMS];
  src[0] = a.P.hi + z * a.p_stride + static_cast<long long>(bm) * TM * a.ldp;
  src[TERMS] = a.Q.hi + z * a.q_stride + static_cast<long long>(bn) * TM * a.ldq;
  if (TERMS == 2) {
    src[1] = a.P.lo + z * a.p_stride + static_cast<long long>(bm) * TM * a.ldp;
    src[TERMS + TERMS - 1] = a.Q.lo + z * a.q_stride + static_cast<long long>(bn) * TM * a.ldq;
  }
  auto issue = [&](int stage, int buffer) {
#pragma unroll
    for (int s = 0; s < 2 * TERMS; ++s) {
      const int ld = s < TERMS ? a.ldp : a.ldq;
#pragma unroll
      for (int p = 0; p < kPieces / 4; ++p) {
        const int piece = wave * (kPieces / 4) + p;
        const int R = piece * 8 + (lane >> 3);
        const int chunk = (lane & 7) ^ ((R >> 1) & 7);
        const uint32_t lane_bytes = static_cast<uint32_t>(lane >> 3) * ld * 2 + chunk * 16;
        dma_piece(src[s] + static_cast<long long>(piece) * 8 * ld + stage * kBK, lane_bytes,
                  smem + (buffer * kStage + s * kArray + piece * 1024) / 4);
      }
    }
  };
  f32x16 acc[F][F];
#pragma unroll
  for (int i = 0; i < F; ++i)
#pragma unroll
    for (int j = 0; j < F; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
  const int wm = wave >> 1, wn = wave & 1, hi = lane >> 5, l31 = lane & 31;
  const unsigned x = (l31 >> 1) & 7;
  const unsigned prow = (wm * (TM / 2) + l31) * 128, qrow = (wn * (TM / 2) + l31) * 128;
  const int stages = a.K / kBK;
  issue(0, 0);
  for (int s = 0; s < stages; ++s) {
    // this wave's copies of stage s have landed and its reads of stage s - 1 are done; behind the barrier every wave's
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (s + 1 < stages) issue(s + 1, (s + 1) & 1);
    const char *base = reinterpret_cast<const char *>(smem) + (s & 1) * kStage;
#pragma unroll
    for (int k = 0; k < kBK / 16; ++k) {
      const unsigned slot = ((2 * k + hi) ^ x) * 16;
      f16x8 p[TERMS][F], q[TERMS][F];
#pragma unroll
      for (int t = 0; t < TERMS; ++t)
#pragma unroll
        for (int i = 0; i < F; ++i) {
          p[t][i] = *reinterpret_cast<const f16x8 *>(base + t * kArray + prow + i * 32 * 128 + slot);
          q[t][i] = *reinterpret_cast<const f16x8 *>(base + (TERMS + t) * kArray + qrow + i * 32 * 128 + slot);
        }
#pragma unroll
      for (int i = 0; i < F; ++i)
#pragma unroll
        for (int j = 0; j < F; ++j) {
          if constexpr (TERMS == 2) {
            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(p[1][i], q[0][j], acc[i][j], 0, 0, 0);
            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(p[0][i], q[1][j], acc[i][j], 0, 0, 0);
          }
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(p[0][i], q[0][j], acc[i][j], 0, 0, 0);
        }
    }
  }
  // accumulator e of a lane: row 8 (e / 4) + 4 (lane / 32) + e % 4, column lane % 32
  constexpr bool two = TERMS == 2;
  Terms D = a.D, DT = a.DT;
  D.hi += z * a.d_stride;
  DT.hi += z * a.dt_stride;
  if (two) {
    D.lo += z * a.d_stride;
    DT.lo += z * a.dt_stride;
  }
#pragma unroll
  for (int i = 0; i < F; ++i)
#pragma unroll
    for (int j = 0; j < F; ++j)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int m = bm * TM + wm * (TM / 2) + i * 32 + 8 * g + 4 * hi;
        const int n = bn * TM + wn * (TM / 2) + j * 32 + l31;
        float v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = acc[i][j][4 * g + k];
        if constexpr (EPI == GRAM) {
#pragma unroll
          for (int k = 0; k < 4; ++k) v[k] *= kScaleA / (kScaleX * kScaleX);
        } else if constexpr (EPI == POLY) {
          const long long at = z * a.p_stride + static_cast<long long>(n) * a.ldp + m;  // A[n][m] = A[m][n]
          const f16x4 h = *reinterpret_cast<const f16x4 *>(a.P.hi + at);
          f16x4 l = {0, 0, 0, 0};
          if (two) l = *reinterpret_cast<const f16x4 *>(a.P.lo + at);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            v[k] = a.c * (v[k] * (1.f / kScaleA)) + a.b * (static_cast<float>(h[k]) + static_cast<float>(l[k])) +
                   (m + k == n ? a.a * kScaleA : 0.f);
        } else if constexpr (EPI == UPDATE) {
#pragma unroll
          for (int k = 0; k < 4; ++k) v[k] *= 1.f / kScaleA;
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if (m + k < a.r && n < a.cols) {
              const long long at = static_cast<long long>(z) * a.r * a.cols +
                                   (a.tall ? static_cast<long long>(n) * a.r + m + k : static_cast<long long>(m + k) * a.cols + n);
              put_out(a.out, a.dtype, at, v[k] * (1.f / (kScaleA * kScaleX)));
            }
          }
          continue;
        }
        put_terms4(DT, static_cast<long long>(n) * a.lddt + m, v, two);
        if (EPI == UPDATE || bm != bn) {
#pragma unroll
          for (int k = 0; k < 4; ++k) put_terms(D, static_cast<long long>(m + k) * a.ldd + n, v[k], two);
        }
      }
}

// sums of squares: kNormParts partial sums per matrix
__global__ __launch_bounds__(256) void ns_norm_kernel(const void *in, int dtype, long long count, double *partials) {
  __shared__ double scratch[4];
  double s = 0;
  const long long base = blockIdx.y * count;
  for (long long i = blockIdx.x * 256LL + threadIdx.x; i < count; i += 256LL * kNormParts) {
    const double v = get_in(in, dtype, base + i);
    s += v * v;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
  if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) partials[blockIdx.y * static_cast<long long>(kNormParts) + blockIdx.x] = scratch[0] + scratch[1] + scratch[2] + scratch[3];
}

// X0 and its transpose from a 64 x 64 tile of G: `same` has G's orientation (ld_same), `turned` the other
template <bool TWO>
__global__ __launch_bounds__(256) void ns_pack_kernel(const void *in, int dtype, int m, int n, const double *partials, float eps,
                                                      Terms same, int ld_same, Terms turned, int ld_turned, long long stride) {
  __shared__ float tile[64][65];
  __shared__ double total;
  const long long z = blockIdx.z;
  if (threadIdx.x < 64) {
    double s = partials[z * kNormParts + threadIdx.x];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
    if (threadIdx.x == 0) total = kScaleX / (sqrt(s) + eps);
  }
  __syncthreads();
  const double factor = total;  // double: the norm of the largest fp32 entries is no fp32 number
  const int c0 = blockIdx.x * 64, r0 = blockIdx.y * 64;
  const int col = threadIdx.x & 63;
  for (int row = threadIdx.x >> 6; row < 64; row += 4) {
    float v = 0.f;
    if (r0 + row < m && c0 + col < n)
      v = static_cast<float>(get_in(in, dtype, z * m * n + static_cast<long long>(r0 + row) * n + c0 + col) * factor);
    put_terms(same, z * stride + static_cast<long long>(r0 + row) * ld_same + c0 + col, v, TWO);
    tile[row][col] = v;
  }
  __syncthreads();
  for (int row = threadIdx.x >> 6; row < 64; row += 4)
    put_terms(turned, z * stride + static_cast<long long>(c0 + row) * ld_turned + r0 + col, tile[col][row], TWO);
}

struct Plan {
  int r, c, rp, cp, terms;
  long long x, sq;             // values of X and of A per matrix, padded
  long long bytes;
};
Plan make_plan(int dtype, int batch, int m, int n) {
  Plan p;
  p.r = m < n ? m : n;
  p.c = m < n ? n : m;
  p.rp = (p.r + kPad - 1) / kPad * kPad;
  p.cp = (p.c + kPad - 1) / kPad * kPad;
  p.terms = dtype == DX_F32 ? 2 : 1;
  p.x = static_cast<long long>(p.rp) * p.cp;
  p.sq = static_cast<long long>(p.rp) * p.rp;
  // X, two copies of X^T, A, B, and the norm's partial sums
  p.bytes = batch * (p.terms * 2 * (3 * p.x + 2 * p.sq) + 8LL * kNormParts);
  return p;
}
int check_shape(int dtype, int batch, int m, int n) {
  DX_REQUIRE(dtype == DX_F32 || dtype == DX_BF16 || dtype == DX_F16, "dx_orthogonalize: dtype %d is none of DX_F32, DX_BF16, DX_F16", dtype);
  DX_REQUIRE(batch >= 0 && batch <= 65535, "dx_orthogonalize: batch %d outside [0, 65535]", batch);
  DX_REQUIRE(m >= 1 && n >= 1 && m <= 65536 && n <= 65536, "dx_orthogonalize: (%d, %d): sides of 1 .. 65536 only", m, n);
  return DX_OK;
}

template <int TM, int TERMS, Epilogue EPI>
int launch_gemm(const NsArgs &a, int batch, hipStream_t s) {
  constexpr int bytes = 2 * 2 * TERMS * TM * kBK * 2;
  DX_LDS_OPT_IN((ns_gemm_kernel<TM, TERMS, EPI>), bytes);
  const int tiles = EPI == GRAM || EPI == POLY ? a.tiles_m * (a.tiles_m + 1) / 2 : a.tiles_m * a.tiles_n;
  hipLaunchKernelGGL((ns_gemm_kernel<TM, TERMS, EPI>), dim3(tiles, batch), dim3(256), bytes, s, a);
  DX_LAUNCH_CHECK();
  return DX_OK;
}
template <int TERMS>
int run_steps(const Plan &p, int batch, int steps, NsArgs a, Terms X, Terms XT0, Terms XT1, Terms A, Terms B, hipStream_t s) {
  constexpr int TM = 128;
  for (int k = 0; k < steps; ++k) {
    const Terms xt = k & 1 ? XT1 : XT0, next = k & 1 ? XT0 : XT1;
    NsArgs g = a;
    g.P = g.Q = X;
    g.p_stride = g.q_stride = p.x;
    g.ldp = g.ldq = g.K = p.cp;
    g.tiles_m = g.tiles_n = p.rp / TM;
    g.D = g.DT = A;
    g.d_stride = g.dt_stride = p.sq;
    g.ldd = g.lddt = p.rp;
    if (int rc = launch_gemm<TM, TERMS, GRAM>(g, batch, s)) return rc;
    g.P = g.Q = A;
    g.p_stride = g.q_stride = p.sq;
    g.ldp = g.ldq = g.K = p.rp;
    g.D = g.DT = B;
    if (int rc = launch_gemm<TM, TERMS, POLY>(g, batch, s)) return rc;
    g.P = B;
    g.Q = xt;
    g.q_stride = p.x;
    g.tiles_n = p.cp / TM;
    g.D = X;
    g.DT = next;
    g.d_stride = g.dt_stride = p.x;
    g.ldd = p.cp;
    if (int rc = k + 1 < steps ? launch_gemm<TM, TERMS, UPDATE>(g, batch, s) : launch_gemm<TM, TERMS, FINAL>(g, batch, s)) return rc;
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
  _Float16 *at = static_cast<_Float16 *>(workspace);
  auto take = [&](long long values) {
    Terms t;
    t.hi = at;
    at += values * batch;
    t.lo = at;
    if (p.terms == 2) at += values * batch;
    return t;
  };
  const Terms X = take(p.x), XT0 = take(p.x), XT1 = take(p.x), A = take(p.sq), B = take(p.sq);
  double *partials = reinterpret_cast<double *>(at);
  hipLaunchKernelGGL(ns_norm_kernel, dim3(kNormParts, batch), dim3(256), 0, s, update, dtype, static_cast<long long>(m) * n, partials);
  DX_LAUNCH_CHECK();
  const bool tall = m > n;
  const dim3 grid((tall ? p.rp : p.cp) / 64, (tall ? p.cp : p.rp) / 64, batch);
  const Terms same = tall ? XT0 : X, turned = tall ? X : XT0;
  const int ld_same = tall ? p.rp : p.cp, ld_turned = tall ? p.cp : p.rp;
  if (p.terms == 2)
    hipLaunchKernelGGL(ns_pack_kernel<true>, grid, dim3(256), 0, s, update, dtype, m, n, partials, eps, same, ld_same, turned, ld_turned, p.x);
  else
    hipLaunchKernelGGL(ns_pack_kernel<false>, grid, dim3(256), 0, s, update, dtype, m, n, partials, eps, same, ld_same, turned, ld_turned, p.x);
  DX_LAUNCH_CHECK();
  NsArgs g{};
  g.a = a;
  g.b = b;
  g.c = c;
  g.out = out;
  g.dtype = dtype;
  g.r = p.r;
  g.cols = p.c;
  g.tall = tall;
  return p.terms == 2 ? run_steps<2>(p, batch, steps, g, X, XT0, XT1, A, B, s) : run_steps<1>(p, batch, steps, g, X, XT0, XT1, A, B, s);
}
