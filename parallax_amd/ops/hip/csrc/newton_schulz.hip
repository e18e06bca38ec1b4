// Newton-Schulz orthogonalisation of update matrices (the Muon optimizer's
// step), batched:
//
//   X0 = G / (|G|_F + eps)             [m, n], m <= n (else transposed)
//   A = X X^T,  B = b A + c A A,  X <- a X + B X      `steps` times
//
// Each singular value s of X0 goes to p(p(..p(s))), p(s) = a s + b s^3 +
// c s^5.  Three products an iteration: X X^T and A A are symmetric, so only
// the tiles on and above the diagonal are computed and each is written
// twice.  X stays in one [m, n] layout: B X reads X k-strided through the
// transposing LDS read.
//
// Precision.  Everything between the products lives in fp16 scaled by 2^12
// (|X| <= 1.2, |A| <= 1.5, |B| <= 3: 2^12 keeps 2^-26 of the largest value
// out of fp16's subnormals).  X is always a high and a low part (22 bits);
// the operands of a product are one part (11 bits) or both, and the sums
// are fp32.  A relative error of a singular value grows by up to 10, 18, 11,
// 8 and 5 over the steps behind the first to fifth, so one-part products
// cost more than their 2^-12.  Emulated in 64 bits over gaussian, low-rank,
// badly scaled and orthogonal matrices, relative to the result's norm: one
// part in the first two steps 2e-4..6e-4 from 256 rows up, where the errors
// of many singular values average, and up to 1e-2 for a few rows; one part
// in three steps up to 2e-3; two parts everywhere 1e-7..6e-7.  A bf16 result
// is rounded by 1.5e-3 anyway, so bf16 takes one part in the first two
// steps of matrices of 256 rows or more, and all else two parts.

#include <torch/extension.h>
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "mm_tile.h"

namespace {

using namespace mm;

constexpr float kScale = 4096.f;  // of X, A and B in fp16

inline long up(long x, long m) { return (x + m - 1) / m * m; }

__device__ __forceinline__ float load_as(const void* p, long i, int type) {
  if (type == 2) return static_cast<const float*>(p)[i];
  const ushort u = static_cast<const ushort*>(p)[i];
  return type == 1 ? half_bits(u) : __uint_as_float((unsigned)u << 16);
}

__device__ __forceinline__ void store_as(void* p, long i, int type, float v) {
  if (type == 2) {
    static_cast<float*>(p)[i] = v;
  } else {
    static_cast<ushort*>(p)[i] =
        type == 1 ? __builtin_bit_cast(ushort, (_Float16)v)
                  : __builtin_bit_cast(ushort, (__bf16)v);
  }
}

// Sums of squares in 64 bits (an fp32 square of 1e-20 or 1e20 is lost), one
// partial per block.
__global__ __launch_bounds__(256) void ns_norm_kernel(
    const void* __restrict__ g, int type, long count,
    double* __restrict__ part, int blocks) {
  __shared__ double red[256];
  const long base = (long)blockIdx.y * count;
  double s = 0.;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < count;
       i += (long)gridDim.x * 256) {
    const double v = load_as(g, base + i, type);
    s += v * v;
  }
  red[threadIdx.x] = s;
  __syncthreads();
  for (int o = 128; o > 0; o >>= 1) {
    if (threadIdx.x < o) red[threadIdx.x] += red[threadIdx.x + o];
    __syncthreads();
  }
  if (threadIdx.x == 0) part[(long)blockIdx.y * blocks + blockIdx.x] = red[0];
}

// X0 in 64 x 64 tiles, transposed where the matrix is tall, zeros behind it.
// g is [rows, cols]; X is [mp][np].
__global__ __launch_bounds__(256) void ns_start_kernel(
    const void* __restrict__ g, int type, int rows, int cols, bool flip,
    const double* __restrict__ part, int blocks, double eps, int mp, int np,
    ushort* __restrict__ X, long xlo) {
  __shared__ float tile[64][65];
  __shared__ double total;
  if (threadIdx.x == 0) {
    double s = 0.;
    for (int i = 0; i < blocks; ++i) s += part[(long)blockIdx.z * blocks + i];
    total = s;
  }
  __syncthreads();
  const double scale = kScale / (sqrt(total) + eps);
  const int m0 = blockIdx.y * 64, n0 = blockIdx.x * 64;
  const int r0 = flip ? n0 : m0, c0 = flip ? m0 : n0;
  const long base = (long)blockIdx.z * rows * cols;
  for (int i = threadIdx.x; i < 4096; i += 256) {
    const int r = r0 + (i >> 6), c = c0 + (i & 63);
    float v = 0.f;
    if (r < rows && c < cols)
      v = (float)(load_as(g, base + (long)r * cols + c, type) * scale);
    tile[i >> 6][i & 63] = v;
  }
  __syncthreads();
  ushort* out = X + (long)blockIdx.z * xlo * 2;
  for (int i = threadIdx.x; i < 4096; i += 256) {
    const int r = i >> 6, c = i & 63;
    const float v = flip ? tile[c][r] : tile[r][c];
    ushort h, l;
    split(v, h, l);
    const long at = (long)(m0 + r) * np + n0 + c;
    out[at] = h;
    out[xlo + at] = l;
  }
}

__device__ __forceinline__ void put(ushort* out, long lo, bool lo_too,
                                    long at, float v) {
  ushort h, l;
  split(v, h, l);
  out[at] = h;
  if (lo_too) out[lo + at] = l;
}

// One symmetric product [mp, mp]: S = sum_k P[i, k] P[j, k].
//   SECOND = false: out = S                (P = X, S = A)
//   SECOND = true:  out = b P + c S        (P = A, S = A A)
template <class C, int SEG, bool SECOND>
__global__ __launch_bounds__(C::THREADS, 2) void ns_sym_kernel(
    const ushort* __restrict__ P, int ld, long plo, int kp, float b, float c,
    int mp, ushort* __restrict__ out, long olo, bool old_lo, bool new_lo,
    int tiles) {
  static_assert(C::BM == C::BN, "square tiles");
  extern __shared__ __attribute__((aligned(16))) char smem[];
  // tile pairs on and above the diagonal, row by row
  int t = blockIdx.x, ti = 0;
  while (t >= tiles - ti) {
    t -= tiles - ti;
    ++ti;
  }
  const int m0 = ti * C::BM, n0 = (ti + t) * C::BN;
  P += (long)blockIdx.y * plo * 2;
  out += (long)blockIdx.y * olo * 2;
  Operand o;
  o.p = P;
  o.lo = plo;
  o.ld = ld;
  o.rows = mp;
  o.cols = ld;
  f4 acc[C::FM][C::FN] = {};
  product<C, KROWS, KROWS, SEG, false>(smem, o, m0, o, n0, 0, kp, acc);
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  const int wm = (wave / C::WAVES_N) * C::WM;
  const int wn = (wave % C::WAVES_N) * C::WN;
#pragma unroll
  for (int i = 0; i < C::FM; ++i) {
    const int m = m0 + wm + i * 16 + (lane & 15);
    if (m >= mp) continue;
#pragma unroll
    for (int j = 0; j < C::FN; ++j) {
      const int n = n0 + wn + j * 16 + (lane >> 4) * 4;
      if (n >= mp) continue;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float v = acc[i][j][r] * (1.f / kScale);
        if (SECOND) {
          const long at = (long)m * ld + n + r;
          float a = half_bits(P[at]);
          if (old_lo) a += half_bits(P[plo + at]);
          v = b * a + c * v;
        }
        put(out, olo, new_lo, (long)m * mp + n + r, v);
        if (m0 != n0) put(out, olo, new_lo, (long)(n + r) * mp + m, v);
      }
    }
  }
}

// X' = a X + B X; the last one goes to the result.
template <class C, int SEG>
__global__ __launch_bounds__(C::THREADS, 2) void ns_next_kernel(
    const ushort* __restrict__ B, long blo, const ushort* __restrict__ X,
    long xlo, float a, int mp, int np, ushort* __restrict__ out,
    void* __restrict__ last, int type, int rows, int cols,
    bool flip, int nnt) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int m0 = blockIdx.x / nnt * C::BM, n0 = blockIdx.x % nnt * C::BN;
  B += (long)blockIdx.y * blo * 2;
  X += (long)blockIdx.y * xlo * 2;
  out += (long)blockIdx.y * xlo * 2;
  Operand ob, ox;
  ob.p = B;
  ob.lo = blo;
  ob.ld = mp;
  ob.rows = mp;
  ob.cols = mp;
  ox.p = X;
  ox.lo = xlo;
  ox.ld = np;
  ox.rows = mp;
  ox.cols = np;
  f4 acc[C::FM][C::FN] = {};
  product<C, KROWS, KCOLS, SEG, false>(smem, ob, m0, ox, n0, 0, mp, acc);
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  const int wm = (wave / C::WAVES_N) * C::WM;
  const int wn = (wave % C::WAVES_N) * C::WN;
  const long base = (long)blockIdx.y * rows * cols;
#pragma unroll
  for (int i = 0; i < C::FM; ++i) {
    const int m = m0 + wm + i * 16 + (lane & 15);
    if (m >= mp) continue;
#pragma unroll
    for (int j = 0; j < C::FN; ++j) {
      const int n = n0 + wn + j * 16 + (lane >> 4) * 4;
      if (n >= np) continue;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const long at = (long)m * np + n + r;
        const float x = half_bits(X[at]) + half_bits(X[xlo + at]);
        const float v = a * x + acc[i][j][r] * (1.f / kScale);
        if (last == nullptr) {
          put(out, xlo, true, at, v);
        } else {
          const int row = flip ? n + r : m, col = flip ? m : n + r;
          if (row < rows && col < cols)
            store_as(last, base + (long)row * cols + col, type,
                     v * (1.f / kScale));
        }
      }
    }
  }
}

using Wide = Tile<128, 128, 64, 64, 32, 3>;
using Small = Tile<64, 64, 32, 32, 32, 3>;

}  // namespace

// g [batch, rows, cols] -> out of the same shape and type, which may be g.
// exact: two-part operands in every product, whatever the size.
void newton_schulz(const at::Tensor& g, at::Tensor out, int64_t steps,
                   double a, double b, double c, double eps, bool exact) {
  TORCH_CHECK(g.is_cuda() && g.dim() == 3 && g.is_contiguous(),
              "newton_schulz: contiguous [batch, rows, cols] on the GPU "
              "expected");
  TORCH_CHECK(out.is_contiguous() && out.sizes() == g.sizes() &&
                  out.scalar_type() == g.scalar_type() &&
                  out.device() == g.device(),
              "newton_schulz: out has to be like g");
  int type = 0;
  switch (g.scalar_type()) {
    case at::kBFloat16: type = 0; break;
    case at::kHalf: type = 1; break;
    case at::kFloat: type = 2; break;
    default:
      TORCH_CHECK(false, "newton_schulz: bf16, fp16 or fp32 expected, got ",
                  g.scalar_type());
  }
  const long batch = g.size(0), rows = g.size(1), cols = g.size(2);
  TORCH_CHECK(steps >= 1 && steps <= 64, "newton_schulz: 1 to 64 steps");
  TORCH_CHECK(batch <= 65535, "newton_schulz: at most 65535 matrices");
  TORCH_CHECK(rows <= 32768 && cols <= 32768 &&
                  std::min(rows, cols) <= 16384,
              "newton_schulz: matrices up to 16384 x 32768");
  if (g.numel() == 0) return;
  const c10::cuda::CUDAGuard guard(g.device());
  auto stream = at::cuda::getCurrentCUDAStream();
  const bool flip = rows > cols;
  const int mp = (int)up(std::min(rows, cols), 64);
  const int np = (int)up(std::max(rows, cols), 64);
  const long xlo = (long)mp * np, alo = (long)mp * mp;
  auto u16 = g.options().dtype(at::kShort);
  const int blocks = (int)std::min<long>(64, (rows * cols + 2047) / 2048);
  auto part = at::empty({batch, blocks}, g.options().dtype(at::kDouble));
  // a high and a low plane for each matrix
  auto xa = at::empty({batch, 2, mp, np}, u16);
  auto xb = at::empty({batch, 2, mp, np}, u16);
  auto A = at::empty({batch, 2, mp, mp}, u16);
  auto B = at::empty({batch, 2, mp, mp}, u16);
  auto ptr = [](at::Tensor& t) {
    return reinterpret_cast<ushort*>(t.data_ptr());
  };
  ns_norm_kernel<<<dim3(blocks, batch), 256, 0, stream>>>(
      g.data_ptr(), type, rows * cols, part.data_ptr<double>(), blocks);
  HIP_CHECK_KERNEL();
  const bool every = exact || std::min(rows, cols) < 256;
  auto fine = [&](int64_t i) { return every || i >= steps - 3; };
  ns_start_kernel<<<dim3(np / 64, mp / 64, batch), 256, 0, stream>>>(
      g.data_ptr(), type, (int)rows, (int)cols, flip,
      part.data_ptr<double>(), blocks, eps, mp, np, ptr(xa), xlo);
  HIP_CHECK_KERNEL();
  auto run = [&](auto tile) {
    using C = decltype(tile);
    const int tiles = (mp + C::BM - 1) / C::BM;
    const int nnt = (np + C::BN - 1) / C::BN;
    const dim3 sym(tiles * (tiles + 1) / 2, batch), full(tiles * nnt, batch);
    for (int64_t i = 0; i < steps; ++i) {
      const bool f = fine(i);
      auto first = [&](auto kernel) {
        kernel<<<sym, C::THREADS, C::LDS_BYTES, stream>>>(
            ptr(xa), np, xlo, np, 0.f, 0.f, mp, ptr(A), alo, false, f, tiles);
        HIP_CHECK_KERNEL();
      };
      auto second = [&](auto kernel) {
        kernel<<<sym, C::THREADS, C::LDS_BYTES, stream>>>(
            ptr(A), mp, alo, mp, (float)b, (float)c, mp, ptr(B), alo, f, f,
            tiles);
        HIP_CHECK_KERNEL();
      };
      auto third = [&](auto kernel) {
        kernel<<<full, C::THREADS, C::LDS_BYTES, stream>>>(
            ptr(B), alo, ptr(xa), xlo, (float)a, mp, np, ptr(xb),
            i + 1 == steps ? out.data_ptr() : nullptr, type, (int)rows,
            (int)cols, flip, nnt);
        HIP_CHECK_KERNEL();
      };
      if (f) {
        first(ns_sym_kernel<C, 3, false>);
        second(ns_sym_kernel<C, 3, true>);
        third(ns_next_kernel<C, 3>);
      } else {
        first(ns_sym_kernel<C, 1, false>);
        second(ns_sym_kernel<C, 1, true>);
        third(ns_next_kernel<C, 1>);
      }
      std::swap(xa, xb);
    }
  };
  // 128-wide tiles once they fill the chip
  const long wide = (long)((mp + 127) / 128) * ((np + 127) / 128) * batch;
  if (wide >= 256) {
    run(Wide{});
  } else {
    run(Small{});
  }
}
