// Newton-Schulz orthogonalisation of update matrices (the Muon optimizer's
// step), batched:
//
//   X0 = G / (|G|_F + eps)             [m, n], m <= n (else transposed)
//   A = X X^T,  B = b A + c A A,  X <- (a + B) X      `steps` times
//
// Each singular value s of X0 goes to p(p(..p(s))), p(s) = a s + b s^3 +
// c s^5.  Three products an iteration: X X^T and A A are symmetric, so only
// the tiles on and above the diagonal are computed and each is written
// twice.  X stays in one [m, n] layout: B X reads X k-strided through the
// transposing LDS read.
//
// Precision.  Everything between the products lives in fp16 scaled by 2^12
// (|X| <= 1.2, |A| <= 1.5, |a + B| <= 4: 2^12 keeps 2^-26 of the largest value
// out of fp16's subnormals).  X is always a high and a low part (22 bits);
// the operands of a product are one part (11 bits) or both, and the sums
// are fp32.  A relative error of a singular value grows by up to 10, 18, 11,
// 8 and 5 over the steps behind the first to fifth, so one-part products
// cost more than their 2^-12.  Emulated in 64 bits over gaussian, low-rank,
// badly scaled and orthogonal matrices, relative to the result's norm: one
// part in the first two steps 3e-6..8e-4 from 256 rows up, where the errors
// of many singular values average, and up to 1e-2 for a few rows; one part
// in three steps up to 2e-3; two parts everywhere 3e-8..1.5e-6.  A bf16
// result is rounded by 1.5e-3 anyway, so bf16 takes one part in the first two
// steps of matrices of 256 rows or more, and all else two parts.  With two
// parts, what is left is the fp32 sums' rounding, as in any fp32 product:
// 2e-7..2.1e-6 for gaussian and badly scaled matrices, up to 9.4e-6 near low
// rank, where plain fp32 products give 8.3e-6.

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
constexpr long kFewRows = 256;    // below: two parts in every step

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

// The matrices of a batch, as they lie: of one shape behind one another, or
// (`listed`) each with its own place and shape.  All fit the same padded
// size, as zeros behind a matrix stay zeros.
constexpr int kListed = 48;

struct Given {
  const void* in;
  void* out;
  int rows, cols;
};

struct Batch {
  const void* in;
  void* out;
  long stride;       // in elements
  int size;          // of an element in bytes
  int rows, cols;
  bool listed;
  Given list[kListed];

  __device__ __forceinline__ Given of(int b) const {
    if (listed) return list[b];
    return Given{static_cast<const char*>(in) + b * stride * size,
                 static_cast<char*>(out) + b * stride * size, rows, cols};
  }
};

// Four values from the 4 i-th of `p`, which lies at 16 bytes.
__device__ __forceinline__ f4 load_four(const void* p, long i, int type) {
  if (type == 2) return static_cast<const f4*>(p)[i];
  const ushort4 u = static_cast<const ushort4*>(p)[i];
  const ushort e[4] = {u.x, u.y, u.z, u.w};
  f4 v;
#pragma unroll
  for (int r = 0; r < 4; ++r)
    v[r] = type == 1 ? half_bits(e[r]) : __uint_as_float((unsigned)e[r] << 16);
  return v;
}

// Sums of squares in 64 bits (an fp32 square of 1e-20 or 1e20 is lost), one
// partial per block.  Bound by memory: 25 MB 8.7 us, 2.9 TB/s.
__global__ __launch_bounds__(256) void ns_norm_kernel(
    Batch batch, int type, double* __restrict__ part) {
  __shared__ double red[4];
  const Given g = batch.of(blockIdx.y);
  const long count = (long)g.rows * g.cols;
  const long step = (long)gridDim.x * 256;
  long i = (long)blockIdx.x * 256 + threadIdx.x;
  double s = 0.;
  if (reinterpret_cast<uintptr_t>(g.in) % 16 == 0) {
    // four at a time, then what is left
#pragma unroll 2
    for (; i < count / 4; i += step) {
      const f4 v = load_four(g.in, i, type);
#pragma unroll
      for (int r = 0; r < 4; ++r) s += (double)v[r] * v[r];
    }
    i = count / 4 * 4 + (long)blockIdx.x * 256 + threadIdx.x;
  }
  for (; i < count; i += step) {
    const double v = load_as(g.in, i, type);
    s += v * v;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0)
    part[(long)blockIdx.y * gridDim.x + blockIdx.x] =
        red[0] + red[1] + red[2] + red[3];
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

// X0 in 64 x 64 tiles, transposed where the matrix is tall, zeros behind it.
// Bound by memory: 12 x 512 x 2048 from bf16 27 us, 2.8 TB/s.
__global__ __launch_bounds__(256) void ns_start_kernel(
    Batch batch, int type, const double* __restrict__ part, int blocks,
    double eps, Matrix X) {
  __shared__ float tile[64][65];
  __shared__ double red[4];
  const Given g = batch.of(blockIdx.z);
  const bool flip = g.rows > g.cols;
  double sum = 0.;
  for (int i = threadIdx.x; i < blocks; i += 256)
    sum += part[(long)blockIdx.z * blocks + i];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = sum;
  X = X.of(blockIdx.z);
  const int m0 = blockIdx.y * 64, n0 = blockIdx.x * 64;
  const int r0 = flip ? n0 : m0, c0 = flip ? m0 : n0;
  if (g.cols % 4 == 0 && reinterpret_cast<uintptr_t>(g.in) % 16 == 0) {
#pragma unroll
    for (int i = threadIdx.x; i < 1024; i += 256) {
      const int r = r0 + (i >> 4), c = c0 + (i & 15) * 4;
      const f4 v = r < g.rows && c < g.cols
                       ? load_four(g.in, ((long)r * g.cols + c) / 4, type)
                       : f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int e = 0; e < 4; ++e) tile[i >> 4][(i & 15) * 4 + e] = v[e];
    }
  } else {
#pragma unroll 8
    for (int i = threadIdx.x; i < 4096; i += 256) {
      const int r = r0 + (i >> 6), c = c0 + (i & 63);
      tile[i >> 6][i & 63] =
          r < g.rows && c < g.cols
              ? load_as(g.in, (long)r * g.cols + c, type) : 0.f;
    }
  }
  __syncthreads();
  const double scale =
      kScale / (sqrt(red[0] + red[1] + red[2] + red[3]) + eps);
#pragma unroll
  for (int i = threadIdx.x; i < 512; i += 256) {
    const int r = i >> 3, c = (i & 7) * 8;
    s8 h, l;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      ushort hi, lo;
      split((float)((flip ? tile[c + e][r] : tile[r][c + e]) * scale), hi,
            lo);
      h[e] = hi;
      l[e] = lo;
    }
    ushort* at = X.p + X.at(m0 + r, n0 + c);
    *reinterpret_cast<s8*>(at) = h;
    *reinterpret_cast<s8*>(
        at + (X.pairs ? 32L : (long)X.rows * X.cols)) = l;
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
//   SECOND = true:  out = b P + c S        (P = A, S = A A), in two parts
//                   also + a on the diagonal, as that takes aX from the next
//                   product: 22 bits of a are as many as X' keeps
// Where there are few tiles, k is cut (CUT = 1): each workgroup leaves its
// sums in `part`, and a second kernel (CUT = 2) adds them up in order and
// goes on.  (Left to the last workgroup of a tile, the fences that takes
// cost more than the launch: 146 us for 12 x 512 x 2048, 42 this way, 0.57
// PF of the 16-bit products on and above the diagonal.)
template <class C, int PARTS, bool SECOND, int CUT>
__global__ __launch_bounds__(C::THREADS, C::OCC) void ns_sym_kernel(
    Matrix P, int kp, float a, float b, float c, Matrix out, int tiles,
    int cuts, float* __restrict__ part) {
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
      if (SECOND) {
        const int m = m0 + wm + i * 16 + (lane & 15);
        const int n = n0 + wn + j * 16 + (lane >> 4) * 4;
        const f4 old = P.four<PARTS == 2>(m, n);
        if (PARTS == 2) {  // rounded once: the terms are larger than the sum
#pragma unroll
          for (int r = 0; r < 4; ++r)
            v[r] = (float)((double)b * old[r] + (double)c * v[r] +
                           (m == n + r ? (double)a * kScale : 0.));
        } else {
          v = b * old + c * v;
        }
      }
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

// X' = a X + B X (two parts: B holds the a); the last one goes to the result.
// The sums start from a X, so that it is read while the first stages are on
// their way.  1024 x 8192 in two parts: 59 us, 0.88 PF of 16-bit products,
// of which the product alone takes 44; all its 512 workgroups run at once,
// so none covers the other's 32 MB of X' on the way out.
template <class C, int PARTS>
__global__ __launch_bounds__(C::THREADS, C::OCC) void ns_next_kernel(
    Matrix B, int kp, Matrix X, float a, Matrix out, bool last, Batch batch,
    int type, int nnt) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int bid = die_contiguous(blockIdx.x, gridDim.x);
  const int m0 = bid / nnt * C::BM, n0 = bid % nnt * C::BN;
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  const int wm = (wave / C::WAVES_N) * C::WM;
  const int wn = (wave % C::WAVES_N) * C::WN;
  B = B.of(blockIdx.y);
  X = X.of(blockIdx.y);
  f4 acc[C::FM][C::FN] = {};
  if (PARTS == 1) {
#pragma unroll
    for (int i = 0; i < C::FM; ++i)
#pragma unroll
      for (int j = 0; j < C::FN; ++j)
        acc[i][j] = a * kScale *
                    X.four<true>(m0 + wm + i * 16 + (lane & 15),
                                 n0 + wn + j * 16 + (lane >> 4) * 4);
  }
  product<C, KROWS, KCOLS, PARTS, false>(smem, B.operand(), m0, X.operand(),
                                         n0, 0, kp, acc);
  if (!last) {
    const auto value = [&](int i, int j) {
      return acc[i][j] * (1.f / kScale);
    };
    out = out.of(blockIdx.y);
    if (out.pairs) {
      put_tile<C, 2, true>(smem, out, m0, n0, value);
    } else {
      put_tile<C, 1, true>(smem, out, m0, n0, value);
    }
    return;
  }
  const float back = 1.f / (kScale * kScale);
  const Given g = batch.of(blockIdx.y);
  const bool flip = g.rows > g.cols;
  if (type != 2 && !flip && g.cols % 8 == 0 &&
      reinterpret_cast<uintptr_t>(g.out) % 16 == 0) {
    store_tile<C>(smem,
                  static_cast<ushort*>(g.out) + (long)m0 * g.cols + n0,
                  g.cols, g.rows - m0, g.cols - n0, [&](int i, int j) {
      ushort u[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) store_as(u, r, type, acc[i][j][r] * back);
      return make_ushort4(u[0], u[1], u[2], u[3]);
    });
    return;
  }
  const bool four = type == 2 && !flip && g.cols % 4 == 0 &&
                    reinterpret_cast<uintptr_t>(g.out) % 16 == 0;
#pragma unroll
  for (int i = 0; i < C::FM; ++i) {
    const int m = m0 + wm + i * 16 + (lane & 15);
#pragma unroll
    for (int j = 0; j < C::FN; ++j) {
      const int n = n0 + wn + j * 16 + (lane >> 4) * 4;
      if (four) {
        if (m < g.rows && n < g.cols)
          *reinterpret_cast<f4*>(static_cast<float*>(g.out) +
                                 (long)m * g.cols + n) = acc[i][j] * back;
        continue;
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = flip ? n + r : m, col = flip ? m : n + r;
        if (row < g.rows && col < g.cols)
          store_as(g.out, (long)row * g.cols + col, type,
                   acc[i][j][r] * back);
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
// fp32 results of few rows: with a two-sum a stage they are as near to 64
// bits as fp32 products (11 x 8 x 687: 1.1e-6, 1.4e-6 without), for 4% of
// the time
struct TinyExact : Tiny {
  static constexpr bool TWO_SUM = true;
};

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
void with_tile(int size, bool exact, F f) {
  if (size == 128) {
    f(Mid{});
  } else if (size == 64) {
    f(Small{});
  } else if (exact) {
    f(TinyExact{});
  } else {
    f(Tiny{});
  }
}

int type_code(at::ScalarType t) {
  switch (t) {
    case at::kBFloat16: return 0;
    case at::kHalf: return 1;
    case at::kFloat: return 2;
    default:
      TORCH_CHECK(false, "newton_schulz: bf16, fp16 or fp32 expected, got ",
                  t);
  }
}

void check_size(long rows, long cols) {
  TORCH_CHECK(rows <= 32768 && cols <= 32768 && rows * cols <= (1L << 28),
              "newton_schulz: matrices of up to 32768 rows and columns and "
              "2^28 values");
}

struct Polynomial {
  int64_t steps;
  double a, b, c, eps;
  bool exact;  // two-part operands in every product, whatever the size
};

// How many matrices go through the products together: 2^28 values, whose
// working copies take up to 4 GB, are far more than fill the chip.  (At most
// 16384: fewer than a grid's third dimension holds.)
long at_once(long small, long large) {
  return std::max(1L, (1L << 28) / (up(small, 128) * up(large, 128)));
}

// small x large: the largest of the batch's matrices, which has `count`;
// least: the fewest rows (or columns of a tall one) of them
void run(const Batch& batch, int type, long count, long small, long large,
         long least, const Polynomial& p, const at::TensorOptions& options) {
  auto stream = at::cuda::getCurrentCUDAStream();
  const bool every = p.exact || least < kFewRows;
  auto fine = [&](int64_t i) { return every || i >= p.steps - 3; };

  // zeros up to whole tiles, and whole stages of 128 k
  const int mp = (int)up(small, 128), np = (int)up(large, 128);
  // The largest tile that still gives half of the chip's 256 CUs something
  // to do.
  auto full_tiles = [&](long t) {
    return (small + t - 1) / t * ((large + t - 1) / t) * count;
  };
  const int full = full_tiles(128) >= 128 ? 128
                   : full_tiles(64) >= 128 ? 64 : 32;
  // The same for a symmetric product over k, where few tiles' k is cut for
  // more of them.  12 x 512 over 2048, two parts: 120 tiles of 128 cut in two
  // 33 + 9 us, in four 36 + 12, 432 of 64 uncut 53.  Over 512, not worth a
  // cut: 120 of 128 23 us, 432 of 64 19.  Fewer of 128 lose as well, as the
  // sums are added up by a workgroup a tile: 1024 over 8192, 36 cut in seven
  // 39 + 10 us, 136 of 64 cut in three 43 + 6; 1024 over 4096 five steps 393
  // and 373 us.
  struct Cut {
    int tile, cuts;
    long pairs;  // tiles of one matrix
  };
  auto cut_of = [&](long k) {
    auto cut = [&](long tile, long all, long least) {
      const long pairs = mp / tile * (mp / tile + 1) / 2;
      const long cuts = std::min(all / (pairs * count), k / least);
      return Cut{(int)tile, (int)std::max(1L, cuts), pairs};
    };
    const Cut big = cut(128, 256, 512), mid = cut(64, 512, 1024);
    if (big.pairs * count >= (big.cuts > 1 ? 100 : 256)) return big;
    return mid.pairs * count >= 100 ? mid : cut(32, 256, 1024);
  };
  const Cut wide = cut_of(np), square = cut_of(mp);
  const int blocks = (int)std::min<long>(1024, (small * large + 4095) / 4096);

  // one allocation: two X, A, B, the norm's partial sums, the cut sums
  const long xs = 2L * mp * np, as = 2L * mp * mp;
  size_t bytes = 0;
  auto take = [&](size_t n) {
    const size_t at = bytes;
    bytes += (n + 255) / 256 * 256;
    return at;
  };
  const size_t o_x0 = take(count * xs * 2), o_x1 = take(count * xs * 2);
  const size_t o_a = take(count * as * 2), o_b = take(count * as * 2);
  const size_t o_norm = take(count * blocks * sizeof(double));
  auto part_of = [&](const Cut& c) {
    return c.cuts > 1 ? c.pairs * c.cuts * c.tile * c.tile * 4 : 0L;
  };
  const size_t o_part = take(count * std::max(part_of(wide),
                                              part_of(square)));
  auto mem = at::empty({(long)bytes}, options.dtype(at::kByte));
  char* base = static_cast<char*>(mem.data_ptr());
  auto matrix = [&](size_t at, long stride, int r, int c, bool in_pairs) {
    return Matrix{reinterpret_cast<ushort*>(base + at), stride, r, c,
                  in_pairs};
  };
  double* norm = reinterpret_cast<double*>(base + o_norm);
  float* part = reinterpret_cast<float*>(base + o_part);

  ns_norm_kernel<<<dim3(blocks, count), 256, 0, stream>>>(batch, type, norm);
  HIP_CHECK_KERNEL();
  ns_start_kernel<<<dim3(np / 64, mp / 64, count), 256, 0, stream>>>(
      batch, type, norm, blocks, p.eps, matrix(o_x0, xs, mp, np, fine(0)));
  HIP_CHECK_KERNEL();
  for (int64_t i = 0; i < p.steps; ++i) {
    const bool f = fine(i), last = i + 1 == p.steps;
    const Matrix X = matrix(i % 2 ? o_x1 : o_x0, xs, mp, np, f);
    const Matrix Y = matrix(i % 2 ? o_x0 : o_x1, xs, mp, np, fine(i + 1));
    const Matrix A = matrix(o_a, as, mp, mp, f);
    const Matrix B = matrix(o_b, as, mp, mp, f);
    auto symmetric = [&](auto second, const Matrix& P, int k,
                         const Matrix& o) {
      constexpr bool SECOND = decltype(second)::value;
      const Cut& way = SECOND ? square : wide;
      const int tiles = mp / way.tile, cut = way.cuts;
      with_tile(way.tile, p.exact, [&](auto t) {
        using C = decltype(t);
        auto launch = [&](auto kernel, int lds, int n) {
          allow_lds(kernel, lds);
          kernel<<<dim3(way.pairs * n, count), C::THREADS, lds, stream>>>(
              P, k, (float)p.a, (float)p.b, (float)p.c, o, tiles, cut, part);
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
    symmetric(std::false_type{}, X, np, A);
    symmetric(std::true_type{}, A, mp, B);
    with_tile(full, p.exact, [&](auto t) {
      using C = decltype(t);
      auto launch = [&](auto kernel) {
        constexpr int lds = C::template lds<2>();
        allow_lds(kernel, lds);
        const int nnt = np / C::BN;
        kernel<<<dim3(mp / C::BM * nnt, count), C::THREADS, lds, stream>>>(
            B, mp, X, (float)p.a, Y, last, batch, type, nnt);
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

}  // namespace

// g [batch, rows, cols] -> out of the same shape and type, which may be g.
void newton_schulz(const at::Tensor& g, at::Tensor out, int64_t steps,
                   double a, double b, double c, double eps, bool exact) {
  TORCH_CHECK(g.is_cuda() && g.dim() == 3 && g.is_contiguous(),
              "newton_schulz: contiguous [batch, rows, cols] on the GPU "
              "expected");
  TORCH_CHECK(out.is_contiguous() && out.sizes() == g.sizes() &&
                  out.scalar_type() == g.scalar_type() &&
                  out.device() == g.device(),
              "newton_schulz: out has to be like g");
  const long rows = g.size(1), cols = g.size(2);
  TORCH_CHECK(steps >= 1 && steps <= 64, "newton_schulz: 1 to 64 steps");
  check_size(rows, cols);
  const int type = type_code(g.scalar_type());
  if (g.numel() == 0) return;
  const c10::cuda::CUDAGuard guard(g.device());
  const long small = std::min(rows, cols), large = std::max(rows, cols);
  const long most = at_once(small, large);
  for (long i = 0; i < g.size(0); i += most) {
    Batch batch = {};
    const long offset = i * rows * cols * g.element_size();
    batch.in = static_cast<const char*>(g.data_ptr()) + offset;
    batch.out = static_cast<char*>(out.data_ptr()) + offset;
    batch.stride = rows * cols;
    batch.size = (int)g.element_size();
    batch.rows = (int)rows;
    batch.cols = (int)cols;
    run(batch, type, std::min(most, g.size(0) - i), small, large, small,
        Polynomial{steps, a, b, c, eps, exact}, g.options());
  }
}

// Each matrix of a list in place.  They are of one type and device and fill
// up to the same multiples of 128 rows and columns (of 128 columns and rows
// the other way round).  Unless `exact`, all or none have the rows that make
// the first steps' operands one part: no result depends on its company.
void newton_schulz_list(std::vector<at::Tensor> mats, int64_t steps,
                        double a, double b, double c, double eps,
                        bool exact) {
  TORCH_CHECK(steps >= 1 && steps <= 64, "newton_schulz: 1 to 64 steps");
  if (mats.empty()) return;
  const at::Tensor& first = mats[0];
  const int type = type_code(first.scalar_type());
  TORCH_CHECK(first.is_cuda() && first.dim() == 2,
              "newton_schulz: matrices on the GPU expected");
  const c10::cuda::CUDAGuard guard(first.device());
  const size_t most = std::min<long>(
      kListed, at_once(std::min(first.size(0), first.size(1)),
                       std::max(first.size(0), first.size(1))));
  for (size_t i0 = 0; i0 < mats.size(); i0 += most) {
    const size_t n = std::min(most, mats.size() - i0);
    Batch batch = {};
    batch.listed = true;
    long small = 0, large = 0, least = 1L << 30;
    for (size_t i = 0; i < n; ++i) {
      const at::Tensor& m = mats[i0 + i];
      TORCH_CHECK(m.dim() == 2 && m.is_contiguous() && m.numel() > 0 &&
                      m.scalar_type() == first.scalar_type() &&
                      m.device() == first.device(),
                  "newton_schulz: contiguous matrices of one type and device "
                  "expected");
      check_size(m.size(0), m.size(1));
      const long s = std::min(m.size(0), m.size(1));
      const long l = std::max(m.size(0), m.size(1));
      TORCH_CHECK(i == 0 || (up(s, 128) == up(small, 128) &&
                             up(l, 128) == up(large, 128)),
                  "newton_schulz: matrices of different padded sizes");
      TORCH_CHECK(exact || i == 0 || (s >= kFewRows) == (least >= kFewRows),
                  "newton_schulz: matrices of ", kFewRows, " rows and of "
                  "fewer in one list");
      small = std::max(small, s);
      large = std::max(large, l);
      least = std::min(least, s);
      batch.list[i] = Given{m.data_ptr(), m.data_ptr(), (int)m.size(0),
                            (int)m.size(1)};
    }
    run(batch, type, (long)n, small, large, least,
        Polynomial{steps, a, b, c, eps, exact}, first.options());
  }
}
