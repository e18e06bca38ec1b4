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

#include <mutex>
#include <set>

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
#pragma unroll 4
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

// How X, A and B lie between the products: in pairs of parts for products of
// two-part operands; else a plane of high parts and, for X, one of low parts
// behind it.  All are padded with zeros to whole tiles.
struct Matrix {
  ushort* p;
  long stride;   // between the matrices of a batch
  int rows, cols;
  bool pairs;

  __device__ __forceinline__ Matrix of(int batch) const {
    Matrix m = *this;
    m.p += batch * stride;
    return m;
  }
  __host__ __device__ __forceinline__ Operand operand() const {
    Operand o;
    o.p = p;
    o.ld = pairs ? 2 * cols : cols;
    o.rows = rows;
    o.cols = cols;
    return o;
  }
  __device__ __forceinline__ long at(int r, int c) const {
    return pairs ? (long)r * cols * 2 + (c >> 5) * 64 + (c & 31)
                 : (long)r * cols + c;
  }
  // four values of a row; LO: with the low parts
  template <bool LO>
  __device__ __forceinline__ f4 four(int r, int c) const {
    const long i = at(r, c);
    const ushort4 h = *reinterpret_cast<const ushort4*>(p + i);
    f4 v = {half_bits(h.x), half_bits(h.y), half_bits(h.z), half_bits(h.w)};
    if (LO) {
      const ushort4 l = *reinterpret_cast<const ushort4*>(
          p + i + (pairs ? 32L : (long)rows * cols));
      v += f4{half_bits(l.x), half_bits(l.y), half_bits(l.z),
              half_bits(l.w)};
    }
    return v;
  }
};

// The matrices of a batch are small x large, from `first_tall` on large x
// small as they lie.
struct Shape {
  int small, large, first_tall;
  __device__ __forceinline__ bool tall(int batch) const {
    return batch >= first_tall;
  }
};

// X0 in 64 x 64 tiles, transposed where the matrix is tall, zeros behind it.
__global__ __launch_bounds__(256) void ns_start_kernel(
    const void* __restrict__ g, int type, Shape shape,
    const double* __restrict__ part, int blocks, double eps, Matrix X) {
  __shared__ float tile[64][65];
  __shared__ double red[4];
  const bool flip = shape.tall(blockIdx.z);
  const int rows = flip ? shape.large : shape.small;
  const int cols = flip ? shape.small : shape.large;
  double sum = threadIdx.x < blocks
                   ? part[(long)blockIdx.z * blocks + threadIdx.x]
                   : 0.;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = sum;
  __syncthreads();
  const double scale =
      kScale / (sqrt(red[0] + red[1] + red[2] + red[3]) + eps);
  X = X.of(blockIdx.z);
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
  for (int i = threadIdx.x; i < 4096; i += 256) {
    const int r = i >> 6, c = i & 63;
    const float v = flip ? tile[c][r] : tile[r][c];
    ushort h, l;
    split(v, h, l);
    const long at = X.at(m0 + r, n0 + c);
    X.p[at] = h;
    X.p[at + (X.pairs ? 32L : (long)X.rows * X.cols)] = l;
  }
}

// A tile of values at (m0, n0) of `out`, whole.
template <class C, int PARTS, bool LO, typename F>
__device__ __forceinline__ void put_tile(char* lds, const Matrix& out, int m0,
                                         int n0, F value) {
  ushort* at = out.p + out.at(m0, n0);
  if constexpr (PARTS == 2) {
    store_pairs<C>(lds, at, 2L * out.cols, value);
  } else {
    store_tile<C>(lds, at, out.cols, C::BM, C::BN, [&](int i, int j) {
      const f4 v = value(i, j);
      ushort h[4], l;
#pragma unroll
      for (int r = 0; r < 4; ++r) split(v[r], h[r], l);
      return make_ushort4(h[0], h[1], h[2], h[3]);
    });
    if (LO) {
      __syncthreads();
      store_tile<C>(lds, at + (long)out.rows * out.cols, out.cols, C::BM,
                    C::BN, [&](int i, int j) {
        const f4 v = value(i, j);
        ushort h, l[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) split(v[r], h, l[r]);
        return make_ushort4(l[0], l[1], l[2], l[3]);
      });
    }
  }
}

// One symmetric product [mp, mp]: S = sum_k P[i, k] P[j, k].
//   SECOND = false: out = S                (P = X, S = A)
//   SECOND = true:  out = b P + c S        (P = A, S = A A)
// Where there are few tiles, k is cut (CUT = 1): each workgroup leaves its
// sums in `part`, and a second kernel (CUT = 2) adds them up in order and
// goes on.  (Left to the last workgroup of a tile, the fences that takes
// cost more than the launch: 146 us for 12 x 512 x 2048, 50 this way.)
template <class C, int PARTS, bool SECOND, int CUT>
__global__ __launch_bounds__(C::THREADS, C::OCC) void ns_sym_kernel(
    Matrix P, int kp, float b, float c, Matrix out, int tiles, int cuts,
    float* __restrict__ part) {
  static_assert(C::BM == C::BN, "square tiles");
  extern __shared__ __attribute__((aligned(16))) char smem[];
  // tile pairs on and above the diagonal, row by row
  const int pairs = tiles * (tiles + 1) / 2;
  const int cut = CUT == 1 ? blockIdx.x / pairs : 0;
  const int pair = CUT == 1 ? blockIdx.x % pairs : blockIdx.x;
  int t = pair, ti = 0;
  while (t >= tiles - ti) {
    t -= tiles - ti;
    ++ti;
  }
  const int m0 = ti * C::BM, n0 = (ti + t) * C::BN;
  P = P.of(blockIdx.y);
  out = out.of(blockIdx.y);
  f4 acc[C::FM][C::FN] = {};
  // a cut's sums lie in the order of the registers: 16 bytes of each thread
  // next to one another
  constexpr long SIZE = C::BM * C::BN / 4;
  f4* sums = reinterpret_cast<f4*>(part) +
             (((long)blockIdx.y * pairs + pair) * cuts) * SIZE + threadIdx.x;
  if constexpr (CUT == 2) {
    for (int q = 0; q < cuts; ++q)
#pragma unroll
      for (int i = 0; i < C::FM; ++i)
#pragma unroll
        for (int j = 0; j < C::FN; ++j)
          acc[i][j] += sums[q * SIZE + (i * C::FN + j) * C::THREADS];
  } else {
    const int each = CUT == 1 ? (kp / 128 + cuts - 1) / cuts * 128 : kp;
    const int k0 = cut * each, k1 = k0 + each < kp ? k0 + each : kp;
    if (k0 < k1) {
      const Operand o = P.operand();
      product<C, KROWS, KROWS, PARTS, false>(smem, o, m0, o, n0, k0, k1,
                                             acc);
    }
    if constexpr (CUT == 1) {
#pragma unroll
      for (int i = 0; i < C::FM; ++i)
#pragma unroll
        for (int j = 0; j < C::FN; ++j)
          sums[cut * SIZE + (i * C::FN + j) * C::THREADS] = acc[i][j];
      return;
    }
  }
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  const int wm = (wave / C::WAVES_N) * C::WM;
  const int wn = (wave % C::WAVES_N) * C::WN;
#pragma unroll
  for (int i = 0; i < C::FM; ++i)
#pragma unroll
    for (int j = 0; j < C::FN; ++j) {
      f4 v = acc[i][j] * (1.f / kScale);
      if (SECOND)
        v = b * P.four<PARTS == 2>(m0 + wm + i * 16 + (lane & 15),
                                   n0 + wn + j * 16 + (lane >> 4) * 4) +
            c * v;
      acc[i][j] = v;
    }
  put_tile<C, PARTS, false>(smem, out, m0, n0,
                            [&](int i, int j) { return acc[i][j]; });
  if (m0 == n0) return;
  // the mirrored tile, turned over in LDS
  constexpr int ROW = PARTS == 2 ? C::PAIR_ROW : C::OUT_ROW;
  constexpr int GOES = PARTS == 2 ? C::PAIR_GOES : 1;
  constexpr int HALF = C::BM / GOES;
  constexpr int PER_ROW = C::BN * PARTS / 8;
#pragma unroll
  for (int go = 0; go < GOES; ++go) {
    __syncthreads();
    if (wn / HALF == go) {
#pragma unroll
      for (int i = 0; i < C::FM; ++i) {
        const int m = wm + i * 16 + (lane & 15);
#pragma unroll
        for (int j = 0; j < C::FN; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            ushort h, l;
            split(acc[i][j][r], h, l);
            char* row =
                smem + (wn % HALF + j * 16 + (lane >> 4) * 4 + r) * ROW;
            if (PARTS == 2) {
              ushort* at = reinterpret_cast<ushort*>(row) + (m >> 5) * 64 +
                           (m & 31);
              at[0] = h;
              at[32] = l;
            } else {
              reinterpret_cast<ushort*>(row)[m] = h;
            }
          }
      }
    }
    __syncthreads();
    ushort* to = out.p + out.at(n0 + go * HALF, m0);
#pragma unroll 4
    for (int q = threadIdx.x; q < HALF * PER_ROW; q += C::THREADS) {
      const int r = q / PER_ROW, e = (q % PER_ROW) * 8;
      *reinterpret_cast<s8*>(to + (long)r * out.cols * PARTS + e) =
          *reinterpret_cast<const s8*>(smem + r * ROW + e * 2);
    }
  }
}

// X' = a X + B X; the last one goes to the result.
template <class C, int PARTS>
__global__ __launch_bounds__(C::THREADS, C::OCC) void ns_next_kernel(
    Matrix B, int kp, Matrix X, float a, Matrix out, void* __restrict__ last,
    int type, Shape shape, int nnt) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const bool flip = shape.tall(blockIdx.y);
  const int rows = flip ? shape.large : shape.small;
  const int cols = flip ? shape.small : shape.large;
  const int bid = die_contiguous(blockIdx.x, gridDim.x);
  const int m0 = bid / nnt * C::BM, n0 = bid % nnt * C::BN;
  B = B.of(blockIdx.y);
  X = X.of(blockIdx.y);
  f4 acc[C::FM][C::FN] = {};
  product<C, KROWS, KCOLS, PARTS, false>(smem, B.operand(), m0, X.operand(),
                                         n0, 0, kp, acc);
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  const int wm = (wave / C::WAVES_N) * C::WM;
  const int wn = (wave % C::WAVES_N) * C::WN;
#pragma unroll
  for (int i = 0; i < C::FM; ++i)
#pragma unroll
    for (int j = 0; j < C::FN; ++j)
      acc[i][j] = a * X.four<true>(m0 + wm + i * 16 + (lane & 15),
                                   n0 + wn + j * 16 + (lane >> 4) * 4) +
                  acc[i][j] * (1.f / kScale);
  const auto value = [&](int i, int j) { return acc[i][j]; };
  if (last == nullptr) {
    out = out.of(blockIdx.y);
    if (out.pairs) {
      put_tile<C, 2, true>(smem, out, m0, n0, value);
    } else {
      put_tile<C, 1, true>(smem, out, m0, n0, value);
    }
    return;
  }
  const long base = (long)blockIdx.y * rows * cols;
  if (type != 2 && !flip && cols % 8 == 0) {
    store_tile<C>(smem, static_cast<ushort*>(last) + base + (long)m0 * cols +
                            n0,
                  cols, rows - m0, cols - n0, [&](int i, int j) {
      ushort u[4];
#pragma unroll
      for (int r = 0; r < 4; ++r)
        store_as(u, r, type, acc[i][j][r] * (1.f / kScale));
      return make_ushort4(u[0], u[1], u[2], u[3]);
    });
    return;
  }
#pragma unroll
  for (int i = 0; i < C::FM; ++i) {
    const int m = m0 + wm + i * 16 + (lane & 15);
#pragma unroll
    for (int j = 0; j < C::FN; ++j) {
      const int n = n0 + wn + j * 16 + (lane >> 4) * 4;
      if (type == 2 && !flip && cols % 4 == 0) {
        if (m < rows && n < cols)
          *reinterpret_cast<f4*>(static_cast<float*>(last) + base +
                                 (long)m * cols + n) =
              acc[i][j] * (1.f / kScale);
        continue;
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = flip ? n + r : m, col = flip ? m : n + r;
        if (row < rows && col < cols)
          store_as(last, base + (long)row * cols + col, type,
                   acc[i][j][r] * (1.f / kScale));
      }
    }
  }
}

// Eight waves of 64 x 32, two workgroups on a CU.  2048 x 8192 x 1024 in two
// parts: 1.28 PF of 16-bit products (four waves of 64 x 64: 1.18, a
// 256 x 256 tile of sixteen: 1.25).
using Mid = Tile<128, 128, 64, 32, 64, 2>;
// Few tiles: what counts is the time of one, so many waves, 128 k a stage
// and smaller tiles.  512 x 512 x 512 in two parts, launch included: 12 us
// with Mid, 6.4 with Small, 4.7 with Tiny.
using Small = Tile<64, 64, 32, 16, 128, 2>;
using Tiny = Tile<32, 32, 16, 16, 128, 4>;

template <typename K>
void allow_lds(K kernel, int bytes) {
  if (bytes <= 64 * 1024) return;
  static std::mutex lock;
  static std::set<std::pair<const void*, int>> done;
  int device = 0;
  TORCH_CHECK(hipGetDevice(&device) == hipSuccess, "hipGetDevice failed");
  const auto key = std::make_pair(reinterpret_cast<const void*>(kernel),
                                  device);
  std::lock_guard<std::mutex> hold(lock);
  if (done.count(key)) return;
  const hipError_t e = hipFuncSetAttribute(
      key.first, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  TORCH_CHECK(e == hipSuccess, "newton_schulz: ", bytes, " bytes of LDS: ",
              hipGetErrorString(e));
  done.insert(key);
}

// f(tile) for a tile size of 32, 64 or 128
template <typename F>
void with_tile(int size, F f) {
  if (size == 128) {
    f(Mid{});
  } else if (size == 64) {
    f(Small{});
  } else {
    f(Tiny{});
  }
}

}  // namespace

// g [batch, rows, cols] -> out of the same shape and type, which may be g.
// The matrices from `turned` on lie as [cols, rows].
// exact: two-part operands in every product, whatever the size.
void newton_schulz(const at::Tensor& g, at::Tensor out, int64_t steps,
                   double a, double b, double c, double eps, bool exact,
                   int64_t turned) {
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
  TORCH_CHECK(turned >= 0 && turned <= batch &&
                  (turned == batch || rows <= cols),
              "newton_schulz: wide matrices first");
  TORCH_CHECK(steps >= 1 && steps <= 64, "newton_schulz: 1 to 64 steps");
  TORCH_CHECK(batch <= 65535, "newton_schulz: at most 65535 matrices");
  TORCH_CHECK(rows <= 32768 && cols <= 32768 && rows * cols <= (1L << 28),
              "newton_schulz: matrices of up to 32768 rows and columns and "
              "2^28 values");
  if (g.numel() == 0) return;
  const c10::cuda::CUDAGuard guard(g.device());
  auto stream = at::cuda::getCurrentCUDAStream();
  const long small = std::min(rows, cols), large = std::max(rows, cols);
  const Shape shape{(int)small, (int)large,
                    rows > cols ? 0 : (int)turned};
  const bool every = exact || small < 256;
  auto fine = [&](int64_t i) { return every || i >= steps - 3; };

  // The largest tile that still gives half of the chip's 256 CUs something
  // to do (a symmetric product of 128 x 128 tiles all of them: 12 x 512 x
  // 2048 takes XX us with 120 of those and XX with 432 smaller ones).
  auto full_tiles = [&](long t) {
    return (small + t - 1) / t * ((large + t - 1) / t) * batch;
  };
  auto sym_tiles = [&](long t) {
    const long n = (small + t - 1) / t;
    return n * (n + 1) / 2 * batch;
  };
  const int full = full_tiles(128) >= 128 ? 128
                   : full_tiles(64) >= 128 ? 64 : 32;
  const int sym = sym_tiles(128) >= 256 ? 128
                  : sym_tiles(64) >= 100 ? 64 : 32;
  // and a long k of few tiles is cut
  auto cuts_of = [&](long k) {
    return (int)std::max(1L, std::min({512 / sym_tiles(sym), k / 1024, 8L}));
  };
  // zeros up to whole tiles, and whole stages of 128 k
  const int mp = (int)up(small, 128), np = (int)up(large, 128);
  const int km = mp, kn = np;
  const long pairs = (long)(mp / sym) * (mp / sym + 1) / 2;
  const int cuts = std::max(cuts_of(kn), cuts_of(km));
  // ~16 values a thread
  const int blocks = (int)std::min<long>(256, (rows * cols + 4095) / 4096);

  // one allocation: two X, A, B, the norm's partial sums, the cut sums
  const long xs = 2L * mp * np, as = 2L * mp * mp;
  size_t bytes = 0;
  auto take = [&](size_t n) {
    const size_t at = bytes;
    bytes += (n + 255) / 256 * 256;
    return at;
  };
  const size_t o_x0 = take(batch * xs * 2), o_x1 = take(batch * xs * 2);
  const size_t o_a = take(batch * as * 2), o_b = take(batch * as * 2);
  const size_t o_norm = take(batch * blocks * sizeof(double));
  const size_t o_part =
      take(cuts > 1 ? batch * pairs * cuts * sym * sym * 4 : 0);
  auto mem = at::empty({(long)bytes}, g.options().dtype(at::kByte));
  char* base = static_cast<char*>(mem.data_ptr());
  auto matrix = [&](size_t at, long stride, int r, int c, bool in_pairs) {
    return Matrix{reinterpret_cast<ushort*>(base + at), stride, r, c,
                  in_pairs};
  };
  double* norm = reinterpret_cast<double*>(base + o_norm);
  float* part = reinterpret_cast<float*>(base + o_part);

  ns_norm_kernel<<<dim3(blocks, batch), 256, 0, stream>>>(
      g.data_ptr(), type, rows * cols, norm, blocks);
  HIP_CHECK_KERNEL();
  ns_start_kernel<<<dim3(np / 64, mp / 64, batch), 256, 0, stream>>>(
      g.data_ptr(), type, shape, norm, blocks, eps,
      matrix(o_x0, xs, mp, np, fine(0)));
  HIP_CHECK_KERNEL();
  for (int64_t i = 0; i < steps; ++i) {
    const bool f = fine(i);
    const Matrix X = matrix(i % 2 ? o_x1 : o_x0, xs, mp, np, f);
    const Matrix Y = matrix(i % 2 ? o_x0 : o_x1, xs, mp, np, fine(i + 1));
    const Matrix A = matrix(o_a, as, mp, mp, f);
    const Matrix B = matrix(o_b, as, mp, mp, f);
    auto symmetric = [&](auto second, const Matrix& P, int k,
                         const Matrix& o) {
      constexpr bool SECOND = decltype(second)::value;
      const int tiles = mp / sym, cut = cuts_of(k);
      with_tile(sym, [&](auto t) {
        using C = decltype(t);
        auto launch = [&](auto kernel, int lds, int n) {
          allow_lds(kernel, lds);
          kernel<<<dim3(pairs * n, batch), C::THREADS, lds, stream>>>(
              P, k, (float)b, (float)c, o, tiles, cut, part);
          HIP_CHECK_KERNEL();
        };
        constexpr int one = C::template lds<1>(), two = C::template lds<2>();
        if (cut > 1 && f) {
          launch(ns_sym_kernel<C, 2, SECOND, 1>, two, cut);
          launch(ns_sym_kernel<C, 2, SECOND, 2>, two, 1);
        } else if (cut > 1) {
          launch(ns_sym_kernel<C, 1, SECOND, 1>, one, cut);
          launch(ns_sym_kernel<C, 1, SECOND, 2>, one, 1);
        } else if (f) {
          launch(ns_sym_kernel<C, 2, SECOND, 0>, two, 1);
        } else {
          launch(ns_sym_kernel<C, 1, SECOND, 0>, one, 1);
        }
      });
    };
    symmetric(std::false_type{}, X, kn, A);
    symmetric(std::true_type{}, A, km, B);
    with_tile(full, [&](auto t) {
      using C = decltype(t);
      auto launch = [&](auto kernel) {
        constexpr int lds = C::template lds<2>();
        allow_lds(kernel, lds);
        const int nnt = np / C::BN;
        kernel<<<dim3(mp / C::BM * nnt, batch), C::THREADS, lds, stream>>>(
            B, km, X, (float)a, Y,
            i + 1 == steps ? out.data_ptr() : nullptr, type, shape, nnt);
        HIP_CHECK_KERNEL();
      };
      if (f) {
        launch(ns_next_kernel<C, 2>);
      } else {
        launch(ns_next_kernel<C, 1>);
      }
    });
  }
}
