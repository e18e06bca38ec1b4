// Softmax cross entropy of a projection onto a large vocabulary, without
// the logits ever being kept:
//
//   z[n,v] = x[n] . w[v] + b[v]         lse[n] = log sum_v exp z[n,v]
//   loss[n] = lse[n] - (1-e) z[n,y] - e mean_v z[n,v]
//   G[n,v] = g[n] (exp(z[n,v] - lse[n]) - (1-e) [v = y] - e/V)
//   dx = G w       dw = G^T x       db[v] = sum_n G[n,v]
//
// Forward: one product over (rows x vocabulary tiles); each workgroup keeps
// the running maximum and sum of its tiles in registers and writes one
// (max, sum, total) per row; a second kernel joins them and takes the
// label's logit as a dot product of its own.  Backward goes over pieces of
// the vocabulary: the logits of a piece are computed again, become G in 16
// bits (bounded by a fixed budget, so it stays in the last-level cache),
// and two products read G: dw of the piece, finished, and dx, which adds up
// in fp32 over the pieces.  Row sums, maxima, lse and all sums over k are
// fp32.  No atomics: every result is independent of the order of blocks.
//
// Types.  bf16 and fp16 inputs are multiplied as they are; G is rounded to
// the same type once (2^-9 or 2^-12 of each value, as the final rounding of
// the gradients is).  fp32 inputs are split into two fp16 parts (22 bits)
// after a scaling by a power of two, and so is G: three products in the
// place of one.  fp16 G is scaled by a power of two that brings the largest
// |g| near the top of fp16's range, and the results are scaled back.
//
// Rows whose label is ignored are read as zeros, so what lies in them (a
// padded batch's garbage, NaN) reaches no gradient.

#include <torch/extension.h>
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "mm_tile.h"

namespace {

using namespace mm;

// exponentials are powers of 2, so logits are held times log2 e
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// G of one piece of the vocabulary takes at most this much
constexpr long kPieceBytes = 176L << 20;
// and so do the split parts of an fp32 table's piece
constexpr long kSplitBytes = 64L << 20;

__host__ __device__ inline long up(long x, long m) {
  return (x + m - 1) / m * m;
}

// 2^x by the hardware instruction: 1 ulp, and 0 below the normal numbers
__device__ __forceinline__ float exp2_fast(float x) {
  return __builtin_amdgcn_exp2f(x);
}

// element i of a tensor of type code 0: bf16, 1: fp16, 2: fp32
__device__ __forceinline__ float load_as(const void* p, long i, int type) {
  if (type == 2) return static_cast<const float*>(p)[i];
  const ushort u = static_cast<const ushort*>(p)[i];
  return type == 1 ? half_bits(u) : __uint_as_float((unsigned)u << 16);
}

// log2 e times the bias of the words v..v+3, 0 behind the last one
struct Bias {
  const void* p;  // of the piece's first word, or nullptr
  long stride;
  int type;
  bool four;      // four at a time can be read
  __device__ __forceinline__ void load(float (&out)[4], int v,
                                       int words) const {
    if (p == nullptr) {
#pragma unroll
      for (int r = 0; r < 4; ++r) out[r] = 0.f;
    } else if (four && v + 4 <= words) {
      if (type == 2) {
        const f4 b = reinterpret_cast<const f4*>(p)[v >> 2];
#pragma unroll
        for (int r = 0; r < 4; ++r) out[r] = b[r] * kLog2e;
      } else {
        const ushort4 b = reinterpret_cast<const ushort4*>(p)[v >> 2];
        const ushort e[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
        for (int r = 0; r < 4; ++r)
          out[r] = kLog2e * (type == 1 ? half_bits(e[r])
                                       : __uint_as_float((unsigned)e[r]
                                                         << 16));
      }
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        out[r] = v + r < words
                     ? kLog2e * load_as(p, (v + r) * stride, type) : 0.f;
    }
  }
};

__device__ __forceinline__ ushort bf16_bits(float v) {
  return __builtin_bit_cast(ushort, (__bf16)v);
}

__device__ __forceinline__ ushort fp16_bits(float v) {
  return __builtin_bit_cast(ushort, (_Float16)v);
}

__device__ __forceinline__ void store_as(void* p, long i, int type, float v) {
  if (type == 2) {
    static_cast<float*>(p)[i] = v;
  } else {
    static_cast<ushort*>(p)[i] = type == 1 ? fp16_bits(v) : bf16_bits(v);
  }
}

// 2^k that brings `top` into [2^13, 2^14); 1 where there is nothing to scale
__device__ __forceinline__ float scale_to_half(float top) {
  if (!(top > 0.f) || !(top < INFINITY)) return 1.f;
  int e;
  frexpf(top, &e);  // top in [2^(e-1), 2^e)
  e = 14 - e;
  e = e < -120 ? -120 : (e > 120 ? 120 : e);
  return ldexpf(1.f, e);
}

// --- laying out an operand --------------------------------------------------
// out[rows_out][dp] 16-bit, zeros behind d and behind the rows, and the same
// in blocks of 32 columns where `blocks` is given; fp32 input: a high and a
// low fp16 plane, scaled by a power of two.  One wave a row.
// labels (x only): rows whose label is `ignore` become zeros.
// fixed: the scale of every row (fp32 only) is found from top[0..ntop);
// otherwise each row has its own.  inv[r] = 1 / scale.  bmax: the largest
// |value| of each block, for a later `fixed` call.
template <int SEG>
__global__ __launch_bounds__(256) void lce_pack_kernel(
    const void* __restrict__ src, int type, long rs, long cs, long rows,
    int d, ushort* __restrict__ out, ushort* __restrict__ blocks, int dp,
    long rows_out, const int64_t* __restrict__ labels, int64_t ignore, bool fixed,
    const float* __restrict__ top, int ntop, float* __restrict__ inv,
    float* __restrict__ bmax) {
  __shared__ float scratch[PX_BLOCK / WAVE];
  const int lane = threadIdx.x & 63;
  float scale = 1.f, most = 0.f;
  if (SEG == 3 && fixed) {
    float t = 0.f;
    for (int i = threadIdx.x; i < ntop; i += blockDim.x) t = fmaxf(t, top[i]);
    scale = scale_to_half(block_reduce_max(t, scratch));
  }
  for (long r = (long)blockIdx.x * 4 + (threadIdx.x >> 6); r < rows_out;
       r += (long)gridDim.x * 4) {
    const bool live =
        r < rows && (labels == nullptr || labels[r] != ignore);
    if constexpr (SEG == 1) {
      for (int c = lane; c < dp; c += 64) {
        ushort u = 0;
        if (live && c < d)
          u = static_cast<const ushort*>(src)[r * rs + c * cs];
        if (out) out[r * dp + c] = u;
        if (blocks) blocks[((c >> 5) * rows_out + r) * 32 + (c & 31)] = u;
      }
    } else {
      const float* s = static_cast<const float*>(src) + r * rs;
      if (!fixed) {
        float t = 0.f;
        if (live) {
          for (int c = lane; c < d; c += 64) {
            const float v = fabsf(s[c * cs]);
            if (v < INFINITY) t = fmaxf(t, v);
          }
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) t = fmaxf(t, __shfl_xor(t, o, 64));
        most = fmaxf(most, t);
        scale = scale_to_half(t);
      }
      if (lane == 0) inv[r] = 1.f / scale;
      for (int c = lane; c < dp; c += 64) {
        const float v = live && c < d ? s[c * cs] * scale : 0.f;
        ushort h, l;
        split(v, h, l);
        const long at = ((c >> 5) * rows_out + r) * 32 + (c & 31);
        if (out) {
          out[r * dp + c] = h;
          out[rows_out * dp + r * dp + c] = l;
        }
        if (blocks) {
          blocks[at] = h;
          blocks[rows_out * dp + at] = l;
        }
      }
    }
  }
  if (SEG == 3 && bmax != nullptr) {
    most = block_reduce_max(most, scratch);
    if (threadIdx.x == 0) bmax[blockIdx.x] = most;
  }
}

// --- forward ----------------------------------------------------------------

struct Logits {
  Operand x, w;
  const float* xinv;  // SEG 3: scales to undo, by row and by word
  const float* winv;
  Bias bias;
  int n;     // rows
  int vp;    // words in this piece
  int dp;
};

// max, sum of exp and (SMOOTH) total of each row, in powers of 2, over `tpb` tiles of words
template <class C, int XL, int SEG, bool BF, bool SMOOTH>
__global__ __launch_bounds__(C::THREADS, C::OCC) void lce_fwd_kernel(
    Logits p, float* __restrict__ part, int part_rows, int vb0,
    int nblocks, int nmt, int nvb, int tpb) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  // the row tiles of one block of words run next to each other: the words
  // come from memory once
  const int bid = die_contiguous(blockIdx.x, nmt * nvb);
  const int mt = bid % nmt, vb = bid / nmt;
  const int m0 = mt * C::BM;
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  const int wm = (wave / C::WAVES_N) * C::WM;
  const int wn = (wave % C::WAVES_N) * C::WN;

  float mx[C::FM], se[C::FM], tot[C::FM], xs[C::FM];
#pragma unroll
  for (int i = 0; i < C::FM; ++i) {
    mx[i] = -INFINITY;
    se[i] = tot[i] = 0.f;
    xs[i] = 1.f;
    if (SEG == 3) {
      int m = m0 + wm + i * 16 + (lane & 15);
      if (m > p.n - 1) m = p.n - 1;
      xs[i] = p.xinv[m];
    }
  }
  for (int q = 0; q < tpb; ++q) {
    const int n0 = (vb * tpb + q) * C::BN;
    if (n0 >= p.vp) break;
    f4 acc[C::FM][C::FN] = {};
    product<C, XL, KROWS, SEG, BF>(smem, p.x, m0, p.w, n0, 0, p.dp, acc);
    float add[C::FN][4], ws[C::FN][4];
#pragma unroll
    for (int j = 0; j < C::FN; ++j)
      p.bias.load(add[j], n0 + wn + j * 16 + (lane >> 4) * 4, p.vp);
#pragma unroll
    for (int j = 0; j < C::FN; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int v = n0 + wn + j * 16 + (lane >> 4) * 4 + r;
        ws[j][r] = SEG == 3 && v < p.vp ? p.winv[v] * kLog2e : kLog2e;
      }
    if (n0 + C::BN > p.vp) {  // words behind the last one
#pragma unroll
      for (int j = 0; j < C::FN; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (n0 + wn + j * 16 + (lane >> 4) * 4 + r >= p.vp) {
#pragma unroll
            for (int i = 0; i < C::FM; ++i) acc[i][j][r] = -INFINITY;
          }
    }
#pragma unroll
    for (int i = 0; i < C::FM; ++i) {
      float top = mx[i];
#pragma unroll
      for (int j = 0; j < C::FN; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float z = fmaf(SEG == 3 ? acc[i][j][r] * xs[i]
                                        : acc[i][j][r],
                               ws[j][r], add[j][r]);
          acc[i][j][r] = z;
          top = fmaxf(top, z);
        }
      const float off = top == -INFINITY ? 0.f : top;
      float s = se[i] * exp2_fast(mx[i] - off);
#pragma unroll
      for (int j = 0; j < C::FN; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          s += exp2_fast(acc[i][j][r] - off);
          if (SMOOTH) {
            const int v = n0 + wn + j * 16 + (lane >> 4) * 4 + r;
            if (v < p.vp) tot[i] += acc[i][j][r];
          }
        }
      mx[i] = top;
      se[i] = s;
    }
  }
  // join the four lane groups, then the waves of a row of waves
  float* red = reinterpret_cast<float*>(smem);  // [waves_n][BM][3]
#pragma unroll
  for (int i = 0; i < C::FM; ++i) {
#pragma unroll
    for (int o = 16; o <= 32; o <<= 1) {
      const float m2 = __shfl_xor(mx[i], o, 64);
      const float s2 = __shfl_xor(se[i], o, 64);
      if (SMOOTH) tot[i] += __shfl_xor(tot[i], o, 64);
      const float top = fmaxf(mx[i], m2);
      const float off = top == -INFINITY ? 0.f : top;
      se[i] = se[i] * exp2_fast(mx[i] - off) + s2 * exp2_fast(m2 - off);
      mx[i] = top;
    }
    if (lane < 16) {
      float* at = red + ((wave % C::WAVES_N) * C::BM + wm + i * 16 + lane) * 3;
      at[0] = mx[i];
      at[1] = se[i];
      at[2] = tot[i];
    }
  }
  __syncthreads();
  for (int r = threadIdx.x; r < C::BM; r += C::THREADS) {
    if (m0 + r >= p.n) break;
    float m = red[r * 3], s = red[r * 3 + 1], t = red[r * 3 + 2];
    for (int w = 1; w < C::WAVES_N; ++w) {
      const float* at = red + (w * C::BM + r) * 3;
      const float top = fmaxf(m, at[0]);
      const float off = top == -INFINITY ? 0.f : top;
      s = s * exp2_fast(m - off) + at[1] * exp2_fast(at[0] - off);
      m = top;
      t += at[2];
    }
    // planes [max | sum | total], each [blocks of words][rows]
    const long at = (long)(vb0 + vb) * part_rows + m0 + r;
    part[at] = m;
    part[at + (long)part_rows * nblocks] = s;
    if (SMOOTH) part[at + 2 * (long)part_rows * nblocks] = t;
  }
}

// Joins the partial sums of 16 rows; the label's logit; the loss.
__global__ __launch_bounds__(256) void lce_join_kernel(
    const float* __restrict__ part, int nvb, int part_rows,
    const void* __restrict__ x, int xtype, long xrs, long xcs,
    const void* __restrict__ w, int wtype, long wrs, long wcs,
    const void* __restrict__ bias, int btype, long bstride, int d,
    const int64_t* __restrict__ labels, int64_t ignore, long V, float eps,
    float* __restrict__ loss, float* __restrict__ lse, int n) {
  __shared__ float sm[3][16][17];
  __shared__ float zy[16];
  const int row = threadIdx.x & 15, q = threadIdx.x >> 4;
  const int r0 = blockIdx.x * 16;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long plane = (long)part_rows * nvb;
  float m = -INFINITY, s = 0.f, t = 0.f;
  if (r0 + row < n) {
    for (int b = q; b < nvb; b += 16) {
      const long at = (long)b * part_rows + r0 + row;
      const float m2 = part[at], s2 = part[at + plane];
      const float top = fmaxf(m, m2);
      const float off = top == -INFINITY ? 0.f : top;
      s = s * exp2_fast(m - off) + s2 * exp2_fast(m2 - off);
      m = top;
      if (eps != 0.f) t += part[at + 2 * plane];
    }
  }
  sm[0][row][q] = m;
  sm[1][row][q] = s;
  sm[2][row][q] = t;
  for (int i = 0; i < 4; ++i) {
    const int r = r0 + wave * 4 + i;
    float a = 0.f;
    if (r < n && labels[r] != ignore) {
      const int64_t y0 = labels[r];
      const long y = y0 < 0 ? 0 : (y0 >= V ? V - 1 : y0);
      for (int c = lane; c < d; c += 64) {
        a += load_as(x, r * xrs + c * xcs, xtype) *
             load_as(w, y * wrs + c * wcs, wtype);
      }
      a = wave_reduce_sum(a);
      if (lane == 0 && bias) a += load_as(bias, y * bstride, btype);
    }
    if (lane == 0) zy[wave * 4 + i] = a;
  }
  __syncthreads();
  if (threadIdx.x < 16 && r0 + row < n) {
    for (int b = 1; b < 16; ++b) {
      const float m2 = sm[0][row][b], s2 = sm[1][row][b];
      const float top = fmaxf(m, m2);
      const float off = top == -INFINITY ? 0.f : top;
      s = s * exp2_fast(m - off) + s2 * exp2_fast(m2 - off);
      m = top;
      t += sm[2][row][b];
    }
    const float l = m * kLn2 + logf(s);
    const int r = r0 + row;
    lse[r] = l;
    float out = l - (1.f - eps) * zy[row];
    if (eps != 0.f) out -= eps * (t * kLn2 / (float)V);
    loss[r] = labels[r] == ignore ? 0.f : out;
  }
}

// sum and count of the rows that are not ignored; out[0] = sum or mean,
// out[1] = count.  One workgroup, fixed order.
__global__ __launch_bounds__(1024) void lce_total_kernel(
    const float* __restrict__ loss, const int64_t* __restrict__ labels,
    int64_t ignore, int n, bool mean, float* __restrict__ out) {
  __shared__ double sd[1024];
  __shared__ int sc[1024];
  double a = 0.;
  int c = 0;
  for (int i = threadIdx.x; i < n; i += 1024) {
    a += loss[i];
    c += labels[i] != ignore;
  }
  sd[threadIdx.x] = a;
  sc[threadIdx.x] = c;
  __syncthreads();
  for (int o = 512; o > 0; o >>= 1) {
    if (threadIdx.x < o) {
      sd[threadIdx.x] += sd[threadIdx.x + o];
      sc[threadIdx.x] += sc[threadIdx.x + o];
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    out[0] = (float)(mean ? sd[0] / sc[0] : sd[0]);
    out[1] = (float)sc[0];
  }
}

// --- backward ---------------------------------------------------------------

// What the gradient needs of a row.  Rows that do not count: an infinite l
// makes their exponentials 0, and g = 0.
struct Row {
  float l;   // log2 e lse
  float g;   // what the row's G is multiplied by
  int y;     // label
  float xs;  // scale to undo
};

// the rows, and sc = {S, 1/S} for 16-bit G
__global__ __launch_bounds__(1024) void lce_rows_kernel(
    const float* __restrict__ dloss, bool scalar,
    const float* __restrict__ count, const int64_t* __restrict__ labels,
    int64_t ignore, int n, int n_out, bool half,
    const float* __restrict__ lse, long V, Row* __restrict__ rows,
    float* __restrict__ sc) {
  __shared__ float red[16];
  const float div = count ? count[0] : 1.f;
  float most = 0.f;
  for (int i = threadIdx.x; i < n_out; i += 1024) {
    Row row = {INFINITY, 0.f, 0, 1.f};
    if (i < n) {
      const int64_t y = labels[i];
      row.y = (int)(y < 0 ? 0 : (y >= V ? V - 1 : y));
      if (y != ignore) {
        row.g = dloss[scalar ? 0 : i] / div;
        row.l = lse[i] * kLog2e;
      }
    }
    rows[i] = row;
    most = fmaxf(most, fabsf(row.g));
  }
  most = block_reduce_max(most, red);
  if (threadIdx.x == 0) {
    // |softmax - target| <= 1, so S |G| stays below 2^14
    const float s = half ? scale_to_half(most) : 1.f;
    sc[0] = s;
    sc[1] = 1.f / s;
  }
}

// G of one piece, [rows padded to BM][ldg]; zeros outside the matrix.
// DB: column sums of each row tile into dbp[row tile][ldg].
template <class C, int XL, int SEG, bool BF, bool DB>
__global__ __launch_bounds__(C::THREADS, C::OCC) void lce_grad_kernel(
    Logits p, const Row* __restrict__ rows, const float* __restrict__ sc,
    long V, long v0, float eps, ushort* __restrict__ G, int ldg, long glo,
    float* __restrict__ dbp, int nmt, int nvt) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int bid = die_contiguous(blockIdx.x, nmt * nvt);
  const int mt = bid % nmt, vt = bid / nmt;
  const int m0 = mt * C::BM, n0 = vt * C::BN;
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  const int wm = (wave / C::WAVES_N) * C::WM;
  const int wn = (wave % C::WAVES_N) * C::WN;
  f4 acc[C::FM][C::FN] = {};
  product<C, XL, KROWS, SEG, BF>(smem, p.x, m0, p.w, n0, 0, p.dp, acc);
  const int c0 = n0 + wn + (lane >> 4) * 4;
  const float S = sc[0], uni = eps / (float)V;
  const float xs = SEG == 3 ? p.xinv[0] : 1.f;  // one for all rows
  float add[C::FN][4], ws[C::FN][4];
#pragma unroll
  for (int j = 0; j < C::FN; ++j) p.bias.load(add[j], c0 + j * 16, p.vp);
#pragma unroll
  for (int j = 0; j < C::FN; ++j)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int v = c0 + j * 16 + r;
      ws[j][r] = SEG == 3 && v < p.vp ? p.winv[v] * kLog2e : kLog2e;
    }
#pragma unroll
  for (int i = 0; i < C::FM; ++i) {
    // one load of 16 bytes: there are rows up to a whole tile
    const f4 row = reinterpret_cast<const f4*>(
        rows)[m0 + wm + i * 16 + (lane & 15)];
    const float l = row[0], gm = row[1];
#pragma unroll
    for (int j = 0; j < C::FN; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float z = SEG == 3 ? acc[i][j][r] * xs : acc[i][j][r];
        acc[i][j][r] =
            (exp2_fast(fmaf(z, ws[j][r], add[j][r] - l)) - uni) * gm;
      }
    // the label's word: in few tiles, so not a comparison for each value
    const long y = (long)__builtin_bit_cast(int, (float)row[2]) - v0 - n0 - wn;
    const int hit = y >= 0 && y < C::WN ? (int)y - (lane >> 4) * 4 : -1;
    if (__any(hit >= 0)) {
#pragma unroll
      for (int j = 0; j < C::FN; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (hit == j * 16 + r) acc[i][j][r] -= (1.f - eps) * gm;
    }
  }
  if (n0 + C::BN > p.vp) {  // words behind the last one
#pragma unroll
    for (int j = 0; j < C::FN; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (c0 + j * 16 + r >= p.vp) {
#pragma unroll
          for (int i = 0; i < C::FM; ++i) acc[i][j][r] = 0.f;
        }
  }
  ushort* at = G + (long)m0 * ldg + n0;
  store_tile<C>(smem, at, ldg, C::BM, C::BN, [&](int i, int j) {
    const f4 v = acc[i][j];
    if (BF)
      return make_ushort4(bf16_bits(v[0]), bf16_bits(v[1]), bf16_bits(v[2]),
                          bf16_bits(v[3]));
    return make_ushort4(fp16_bits(v[0] * S), fp16_bits(v[1] * S),
                        fp16_bits(v[2] * S), fp16_bits(v[3] * S));
  });
  if (SEG == 3) {
    __syncthreads();
    store_tile<C>(smem, at + glo, ldg, C::BM, C::BN, [&](int i, int j) {
      ushort h, l[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) split(acc[i][j][r] * S, h, l[r]);
      return make_ushort4(l[0], l[1], l[2], l[3]);
    });
  }
  if (DB) {
    float* red = reinterpret_cast<float*>(smem);  // [waves_m][BN]
    __syncthreads();
#pragma unroll
    for (int j = 0; j < C::FN; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float c = 0.f;
#pragma unroll
        for (int i = 0; i < C::FM; ++i) c += acc[i][j][r];
        c = sum16(c);
        if ((lane & 15) == 0)
          red[(wave / C::WAVES_N) * C::BN + wn + j * 16 + (lane >> 4) * 4 +
              r] = c;
      }
    __syncthreads();
    for (int c = threadIdx.x; c < C::BN; c += C::THREADS) {
      float s = red[c];
      for (int w = 1; w < C::WAVES_M; ++w) s += red[w * C::BN + c];
      dbp[(long)mt * ldg + n0 + c] = s;
    }
  }
}

__global__ __launch_bounds__(256) void lce_db_kernel(
    const float* __restrict__ dbp, int nmt, int ldg, int vp, void* db,
    int type) {
  const int v = blockIdx.x * 256 + threadIdx.x;
  if (v >= vp) return;
  float s = 0.f;
  for (int m = 0; m < nmt; ++m) s += dbp[(long)m * ldg + v];
  store_as(db, v, type, s);
}

// dw[v, :] = 1/S sum_n G[n, v] x[n, :]  (G and x both k-strided)
template <class C, int SEG, bool BF>
__global__ __launch_bounds__(C::THREADS, C::OCC) void lce_dw_kernel(
    Operand G, Operand x, int kn, const float* __restrict__ sc,
    const float* __restrict__ xinv, void* __restrict__ dw, int type, int vp,
    int d, int nmt, int nnt) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int bid = die_contiguous(blockIdx.x, nmt * nnt);
  const int m0 = bid / nnt * C::BM, n0 = bid % nnt * C::BN;
  f4 acc[C::FM][C::FN] = {};
  product<C, KCOLS, KCOLS, SEG, BF>(smem, G, m0, x, n0, 0, kn, acc);
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  const int wm = (wave / C::WAVES_N) * C::WM;
  const int wn = (wave % C::WAVES_N) * C::WN;
  const float back = sc[1] * (SEG == 3 ? xinv[0] : 1.f);
  if (type != 2 && (d & 7) == 0) {
    store_tile<C>(smem, static_cast<ushort*>(dw) + (long)m0 * d + n0, d,
                  vp - m0, d - n0, [&](int i, int j) {
      const f4 v = acc[i][j] * back;
      if (BF)
        return make_ushort4(bf16_bits(v[0]), bf16_bits(v[1]),
                            bf16_bits(v[2]), bf16_bits(v[3]));
      return make_ushort4(fp16_bits(v[0]), fp16_bits(v[1]), fp16_bits(v[2]),
                          fp16_bits(v[3]));
    });
    return;
  }
#pragma unroll
  for (int i = 0; i < C::FM; ++i) {
    const int v = m0 + wm + i * 16 + (lane & 15);
    if (v >= vp) continue;
#pragma unroll
    for (int j = 0; j < C::FN; ++j) {
      const int c = n0 + wn + j * 16 + (lane >> 4) * 4;
      const long at = (long)v * d + c;
      if (type == 2 && c + 4 <= d && (d & 3) == 0) {
        *reinterpret_cast<f4*>(static_cast<float*>(dw) + at) =
            acc[i][j] * back;
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (c + r < d) store_as(dw, at + r, type, acc[i][j][r] * back);
      }
    }
  }
}

// part[slice][n, :] (+)= sum over a slice of the piece's words G[n, v] w[v, :]
template <class C, int SEG, bool BF>
__global__ __launch_bounds__(C::THREADS, C::OCC) void lce_dx_kernel(
    Operand G, Operand w, int kv, int kslice, float* __restrict__ part,
    int n_rows, int dp, bool first, int nmt, int nnt, int slices) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int bid = die_contiguous(blockIdx.x, nmt * nnt * slices);
  const int sl = bid / (nmt * nnt), t = bid % (nmt * nnt);
  const int m0 = t / nnt * C::BM, n0 = t % nnt * C::BN;
  const int k0 = sl * kslice;
  const int k1 = k0 + kslice < kv ? k0 + kslice : kv;
  f4 acc[C::FM][C::FN] = {};
  if (k0 < k1)
    product<C, KROWS, KCOLS, SEG, BF>(smem, G, m0, w, n0, k0, k1, acc);
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  const int wm = (wave / C::WAVES_N) * C::WM;
  const int wn = (wave % C::WAVES_N) * C::WN;
#pragma unroll
  for (int i = 0; i < C::FM; ++i) {
    const int m = m0 + wm + i * 16 + (lane & 15);
    if (m >= n_rows) continue;
#pragma unroll
    for (int j = 0; j < C::FN; ++j) {
      const int c = n0 + wn + j * 16 + (lane >> 4) * 4;
      if (c >= dp) continue;
      f4* at = reinterpret_cast<f4*>(part + ((long)sl * n_rows + m) * dp + c);
      *at = first ? acc[i][j] : *at + acc[i][j];
    }
  }
}

__global__ __launch_bounds__(256) void lce_dx_sum_kernel(
    const float* __restrict__ part, int slices, long n, int d, int dp,
    const float* __restrict__ sc, const float* __restrict__ winv,
    void* __restrict__ dx, int type) {
  const float back = sc[1] * (winv ? winv[0] : 1.f);
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n * d;
       i += (long)gridDim.x * 256) {
    const long r = i / d;
    const long at = r * dp + (i - r * d);
    float s = 0.f;
    for (int q = 0; q < slices; ++q) s += part[q * n * dp + at];
    store_as(dx, i, type, s * back);
  }
}

// --- host -------------------------------------------------------------------

// Sixteen waves of 64 x 64, one workgroup on a CU: the most products for a
// byte that comes from memory, and four waves on a SIMD to wait for another.
using Big = Tile<256, 256, 64, 64, 64, 2>;
using Mid = Tile<128, 128, 64, 64, 64, 2>;
// few rows: wide in the words
using Flat = Tile<64, 256, 64, 32, 64, 2>;
using Small = Tile<64, 64, 32, 32, 64, 2>;

int type_code(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return 0;
    case at::kHalf: return 1;
    case at::kFloat: return 2;
    default:
      TORCH_CHECK(false, "linear_ce: bf16, fp16 or fp32 expected, got ",
                  t.scalar_type());
  }
}

template <typename K>
void allow_lds(K kernel, int bytes) {
  hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                      hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
}

const ushort* bits(const at::Tensor& t) {
  return reinterpret_cast<const ushort*>(t.data_ptr());
}

// What the products read: x laid out once, w as it is or piece by piece.
struct Plan {
  long n, v, d, dp, np;
  int type, seg;
  bool w_direct;   // w's rows can be read in place
  long w_rows;     // words in a piece of w that is laid out
};

Plan make_plan(const at::Tensor& x, const at::Tensor& w) {
  Plan p;
  p.n = x.size(0);
  p.d = x.size(1);
  p.v = w.size(0);
  p.dp = up(p.d, 64);
  p.np = up(p.n, 256);
  p.type = type_code(x);
  p.seg = p.type == 2 ? 3 : 1;
  p.w_direct = p.seg == 1 && p.d == p.dp && w.stride(1) == 1 &&
               w.stride(0) % 8 == 0 && w.stride(0) >= p.d &&
               w.stride(0) < (1 << 22) &&
               reinterpret_cast<uintptr_t>(w.data_ptr()) % 16 == 0;
  const long words = kSplitBytes / (p.dp * 2 * (p.seg == 3 ? 2 : 1));
  p.w_rows = std::min(up(p.v, 256), std::max(256L, words / 256 * 256));
  return p;
}

int pack_blocks(long rows) {
  return (int)std::min<long>(1024, (rows + 3) / 4);
}

void pack(const at::Tensor& src, long row0, long rows, long rows_out,
          const Plan& p, at::Tensor& out, at::Tensor& blocks,
          const int64_t* labels, int64_t ignore, bool fixed, const at::Tensor& top,
          at::Tensor& inv, float* bmax, hipStream_t stream) {
  const char* s = static_cast<const char*>(src.data_ptr()) +
                  row0 * src.stride(0) * src.element_size();
  auto launch = [&](auto kernel) {
    kernel<<<pack_blocks(rows_out), 256, 0, stream>>>(
        s, p.type, src.stride(0), src.stride(1), rows, (int)p.d,
        out.defined() ? reinterpret_cast<ushort*>(out.data_ptr()) : nullptr,
        blocks.defined() ? reinterpret_cast<ushort*>(blocks.data_ptr())
                         : nullptr,
        (int)p.dp, rows_out,
        labels, ignore, fixed,
        top.defined() ? top.data_ptr<float>() : nullptr,
        top.defined() ? (int)top.numel() : 0,
        inv.defined() ? inv.data_ptr<float>() : nullptr, bmax);
    HIP_CHECK_KERNEL();
  };
  if (p.seg == 3) {
    launch(lce_pack_kernel<3>);
  } else {
    launch(lce_pack_kernel<1>);
  }
}

Operand rows_operand(const ushort* p, long rows, long ld, long lo,
                     long cols) {
  Operand o;
  o.p = p;
  o.lo = lo;
  o.ld = (int)ld;
  o.rows = (int)std::min<long>(rows, 0x7fffffffL);
  o.cols = (int)cols;
  return o;
}

Bias bias_of(const c10::optional<at::Tensor>& bias, long v0) {
  Bias b = {nullptr, 0, 0, false};
  if (!bias.has_value()) return b;
  b.stride = bias->stride(0);
  b.type = type_code(*bias);
  b.p = static_cast<const char*>(bias->data_ptr()) +
        v0 * b.stride * bias->element_size();
  b.four = b.stride == 1 && reinterpret_cast<uintptr_t>(b.p) % 16 == 0;
  return b;
}

void check(const at::Tensor& x, const at::Tensor& w,
           const c10::optional<at::Tensor>& bias, const at::Tensor& labels) {
  TORCH_CHECK(x.is_cuda() && w.is_cuda() && labels.is_cuda(),
              "linear_ce: GPU tensors expected");
  TORCH_CHECK(x.device() == w.device() && x.device() == labels.device() &&
                  (!bias.has_value() || bias->device() == x.device()),
              "linear_ce: tensors on different devices");
  TORCH_CHECK(x.dim() == 2 && w.dim() == 2 && x.size(1) == w.size(1),
              "linear_ce: x [N, D] and w [V, D] expected");
  TORCH_CHECK(x.scalar_type() == w.scalar_type(),
              "linear_ce: x and w have different types");
  TORCH_CHECK(x.size(1) >= 1 && x.size(1) <= 32768 && w.size(0) >= 1,
              "linear_ce: D in 1..32768 and at least one word expected");
  TORCH_CHECK(x.size(0) >= 1 && x.size(0) <= (1 << 20),
              "linear_ce: 1 to 2^20 rows expected");
  TORCH_CHECK(w.size(0) < (1L << 31) - 1024, "linear_ce: too many words");
  TORCH_CHECK(up(x.size(0), 256) * up(x.size(1), 64) <= (1L << 29),
              "linear_ce: x has more than 2^29 values: take fewer rows at a "
              "time");
  TORCH_CHECK(labels.scalar_type() == at::kLong && labels.dim() == 1 &&
                  labels.size(0) == x.size(0) && labels.is_contiguous(),
              "linear_ce: labels [N] int64 expected");
  if (bias.has_value()) {
    type_code(*bias);
    TORCH_CHECK(bias->dim() == 1 && bias->size(0) == w.size(0),
                "linear_ce: bias [V] expected");
  }
}

// calls f(tile, seg, bf16) with compile-time arguments
template <typename F>
void with_types(const Plan& p, F f) {
  if (p.type == 0) {
    f(std::integral_constant<int, 1>{}, std::true_type{});
  } else if (p.type == 1) {
    f(std::integral_constant<int, 1>{}, std::false_type{});
  } else {
    f(std::integral_constant<int, 3>{}, std::false_type{});
  }
}

// The tile of the logits, forward and backward.  Many 16-bit rows: 256 x 128
// in two workgroups a CU, so that one's exponentials and stores run under the
// other's products, with x in blocks.
using Logit = Tile<256, 128, 64, 64, 32, 3>;

template <class C>
constexpr int x_layout() {
  return std::is_same<C, Logit>::value ? KBLOCK : KROWS;
}

// two-part operands never meet that tile: its registers do not hold them
template <class C, int SEG>
constexpr bool reached() {
  return !(std::is_same<C, Logit>::value && SEG == 3);
}

bool blocked(const Plan& p) {
  // not where 256-row tiles would be empty by more than they gain
  return p.seg == 1 && p.n > 64 && up(p.n, 256) * 100 <= up(p.n, 128) * 115;
}

template <typename F>
void with_row_tile(const Plan& p, F f) {
  if (p.n <= 64) {
    f(Flat{});
  } else if (blocked(p)) {
    f(Logit{});
  } else {
    f(Mid{});
  }
}

}  // namespace

// {loss (scalar or [N]), lse [N], count [1], top |w| of blocks (fp32)}
std::vector<at::Tensor> linear_ce_fwd(const at::Tensor& x,
                                      const at::Tensor& w,
                                      const c10::optional<at::Tensor>& bias,
                                      const at::Tensor& labels,
                                      int64_t ignore, double smoothing,
                                      int64_t reduction) {
  check(x, w, bias, labels);
  const c10::cuda::CUDAGuard guard(x.device());
  auto stream = at::cuda::getCurrentCUDAStream();
  const Plan p = make_plan(x, w);
  auto f32 = x.options().dtype(at::kFloat);
  auto u16 = x.options().dtype(at::kShort);
  const auto* lab = labels.data_ptr<int64_t>();
  const float eps = (float)smoothing;

  const bool blk = blocked(p);
  auto xpk = at::empty({p.seg == 3 ? 2 * p.np : p.np, p.dp}, u16);
  at::Tensor xinv, winv, none, tops, wpk;
  if (p.seg == 3) xinv = at::empty({p.np}, f32);
  pack(x, 0, p.n, p.np, p, blk ? none : xpk, blk ? xpk : none, lab, ignore, false, none, xinv, nullptr,
       stream);

  const long piece = p.w_direct ? p.v : p.w_rows;
  const long pieces = (p.v + piece - 1) / piece;
  const int wblocks = pack_blocks(p.w_rows);
  if (!p.w_direct) {
    wpk = at::empty({p.seg == 3 ? 2 * p.w_rows : p.w_rows, p.dp}, u16);
    if (p.seg == 3) {
      winv = at::empty({p.w_rows}, f32);
      tops = at::empty({pieces * wblocks}, f32);
    }
  }
  auto loss = at::empty({p.n}, f32);
  auto lse = at::empty({p.n}, f32);
  auto total = at::empty({2}, f32);
  with_row_tile(p, [&](auto tile) {
    using C = decltype(tile);
    const int nmt = (int)((p.n + C::BM - 1) / C::BM);
    const long piece_tiles = (std::min(piece, p.v) + C::BN - 1) / C::BN;
    // a workgroup takes several tiles of words as long as ~2000 are left
    int tpb = (int)std::min<long>(8, piece_tiles * nmt / 2048);
    if (tpb < 1) tpb = 1;
    std::vector<int> first;
    int blocks = 0;
    for (long i = 0; i < pieces; ++i) {
      const long vp = std::min(piece, p.v - i * piece);
      first.push_back(blocks);
      blocks += (int)((vp + (long)C::BN * tpb - 1) / ((long)C::BN * tpb));
    }
    const int part_rows = (int)up(p.n, 16);
    auto part = at::empty({eps != 0.f ? 3 : 2, blocks, part_rows}, f32);
    for (long i = 0; i < pieces; ++i) {
      const long v0 = i * piece, vp = std::min(piece, p.v - v0);
      Logits q;
      q.x = rows_operand(bits(xpk), p.np, p.dp, p.np * p.dp, p.dp);
      if (p.w_direct) {
        q.w = rows_operand(bits(w), vp, w.stride(0), 0, p.dp);
      } else {
        pack(w, v0, vp, p.w_rows, p, wpk, none, nullptr, 0, false, none, winv,
             p.seg == 3 ? tops.data_ptr<float>() + i * wblocks : nullptr,
             stream);
        q.w = rows_operand(bits(wpk), p.w_rows, p.dp, p.w_rows * p.dp, p.dp);
      }
      q.xinv = p.seg == 3 ? xinv.data_ptr<float>() : nullptr;
      q.winv = p.seg == 3 ? winv.data_ptr<float>() : nullptr;
      q.bias = bias_of(bias, v0);
      q.n = (int)p.n;
      q.vp = (int)vp;
      q.dp = (int)p.dp;
      const int nvb =
          (int)((vp + (long)C::BN * tpb - 1) / ((long)C::BN * tpb));
      with_types(p, [&](auto seg, auto bf) {
        if constexpr (reached<C, decltype(seg)::value>()) {
        auto launch = [&](auto kernel) {
          allow_lds(kernel, C::LDS_BYTES);
          kernel<<<nmt * nvb, C::THREADS, C::LDS_BYTES, stream>>>(
              q, part.template data_ptr<float>(), part_rows, first[i],
              blocks, nmt, nvb, tpb);
          HIP_CHECK_KERNEL();
        };
        if (eps != 0.f) {
          launch(lce_fwd_kernel<C, x_layout<C>(), decltype(seg)::value,
                                decltype(bf)::value, true>);
        } else {
          launch(lce_fwd_kernel<C, x_layout<C>(), decltype(seg)::value,
                                decltype(bf)::value, false>);
        }
        }
      });
    }
    lce_join_kernel<<<(int)((p.n + 15) / 16), 256, 0, stream>>>(
        part.template data_ptr<float>(), blocks, part_rows, x.data_ptr(),
        p.type, x.stride(0), x.stride(1), w.data_ptr(), p.type, w.stride(0),
        w.stride(1), bias.has_value() ? bias->data_ptr() : nullptr,
        bias.has_value() ? type_code(*bias) : 0,
        bias.has_value() ? bias->stride(0) : 0, (int)p.d, lab, ignore, p.v,
        eps, loss.data_ptr<float>(), lse.data_ptr<float>(), (int)p.n);
    HIP_CHECK_KERNEL();
  });
  at::Tensor out = loss;
  if (reduction != 0) {
    lce_total_kernel<<<1, 1024, 0, stream>>>(
        loss.data_ptr<float>(), lab, ignore, (int)p.n, reduction == 1,
        total.data_ptr<float>());
    HIP_CHECK_KERNEL();
    out = total[0];
  }
  if (!tops.defined()) tops = at::empty({0}, f32);
  return {out, lse, total, tops};
}

// {dx, dw, db}; an empty tensor for what is not wanted
std::vector<at::Tensor> linear_ce_bwd(
    const at::Tensor& dloss, const at::Tensor& x, const at::Tensor& w,
    const c10::optional<at::Tensor>& bias, const at::Tensor& labels,
    const at::Tensor& lse, const at::Tensor& count, const at::Tensor& tops,
    int64_t ignore, double smoothing, int64_t reduction, bool want_dx,
    bool want_dw, bool want_db) {
  check(x, w, bias, labels);
  TORCH_CHECK(dloss.scalar_type() == at::kFloat && dloss.is_cuda() &&
                  dloss.is_contiguous() &&
                  dloss.numel() == (reduction == 0 ? x.size(0) : 1),
              "linear_ce_bwd: fp32 gradient of the loss expected");
  const c10::cuda::CUDAGuard guard(x.device());
  auto stream = at::cuda::getCurrentCUDAStream();
  const Plan p = make_plan(x, w);
  auto f32 = x.options().dtype(at::kFloat);
  auto u16 = x.options().dtype(at::kShort);
  const auto* lab = labels.data_ptr<int64_t>();
  const float eps = (float)smoothing;
  const bool s3 = p.seg == 3;

  const long nrows = up(p.n, 256);
  auto rows = at::empty({nrows, 4}, f32);
  auto sc = at::empty({2}, f32);
  lce_rows_kernel<<<1, 1024, 0, stream>>>(
      dloss.data_ptr<float>(), reduction != 0,
      reduction == 1 ? count.data_ptr<float>() + 1 : nullptr, lab, ignore,
      (int)p.n, (int)nrows, p.type != 0, lse.data_ptr<float>(), p.v,
      reinterpret_cast<Row*>(rows.data_ptr()), sc.data_ptr<float>());
  HIP_CHECK_KERNEL();

  at::Tensor xpk = at::empty({s3 ? 2 * p.np : p.np, p.dp}, u16);
  at::Tensor xinv, winv, none, xtop, wpk, xblk;
  if (blocked(p)) xblk = at::empty_like(xpk);
  if (s3) {
    // one scale for all rows, as the rows are summed over: the first call
    // only finds the largest value
    xinv = at::empty({p.np}, f32);
    xtop = at::empty({pack_blocks(p.np)}, f32);
    pack(x, 0, p.n, p.np, p, xpk, none, lab, ignore, false, none, xinv,
         xtop.data_ptr<float>(), stream);
  }
  pack(x, 0, p.n, p.np, p, xpk, xblk, lab, ignore, s3, xtop, xinv, nullptr,
       stream);

  // words for which the tiles of dw fill the chip's 256 CUs once
  const long wave_of_words = 256 * 256 / ((p.dp + 255) / 256);
  long piece = kPieceBytes / (nrows * (s3 ? 4 : 2));
  piece = piece >= wave_of_words ? piece / wave_of_words * wave_of_words
                                 : piece / 256 * 256;
  piece = std::max(256L, std::min(piece, up(p.v, 256)));
  if (!p.w_direct) piece = std::min(piece, p.w_rows);
  // offsets inside a piece of w stay below 2^31
  const long w_ld = p.w_direct ? w.stride(0) : p.dp;
  piece = std::max(256L, std::min(piece, (1L << 30) / w_ld / 256 * 256));
  const int ldg = (int)piece;
  const long glo = nrows * ldg;
  auto G = at::empty({s3 ? 2 * nrows : nrows, ldg}, u16);
  if (!p.w_direct) {
    wpk = at::empty({s3 ? 2 * piece : piece, p.dp}, u16);
    if (s3) winv = at::empty({piece}, f32);
  }
  at::Tensor dx, dw, db, part, dbp;
  if (want_dx) dx = at::empty({p.n, p.d}, x.options());
  if (want_dw) dw = at::empty({p.v, p.d}, w.options());
  if (want_db) {
    db = at::empty({p.v}, bias->options());
    dbp = at::empty({(p.n + 63) / 64, ldg}, f32);
  }
  // dx: few tiles and a long k, so k is cut until the chip is full
  const int dx_tile = p.n > 128 && p.dp >= 128 ? (getenv("DXBIG") && p.dp>=256 ? 256:128) : 64;
  const long dx_tiles = ((p.n + dx_tile - 1) / dx_tile) *
                        ((p.dp + dx_tile - 1) / dx_tile);
  const int slices = (int)std::min<long>(
      std::max(1L, (dx_tile == 256 ? 256 : 512) / dx_tiles),
      std::max(1L, piece / 512));
  if (want_dx) part = at::empty({slices, p.n, p.dp}, f32);

  for (long v0 = 0; v0 < p.v; v0 += piece) {
    const long vp = std::min(piece, p.v - v0);
    Logits q;
    q.x = rows_operand(bits(xblk.defined() ? xblk : xpk), p.np, p.dp,
                       p.np * p.dp, p.dp);
    if (p.w_direct) {
      q.w = rows_operand(bits(w) + v0 * w.stride(0), vp, w.stride(0), 0,
                         p.dp);
    } else {
      pack(w, v0, vp, up(vp, 64), p, wpk, none, nullptr, 0, s3, tops, winv,
           nullptr, stream);
      q.w = rows_operand(bits(wpk), up(vp, 64), p.dp, up(vp, 64) * p.dp,
                         p.dp);
    }
    q.xinv = s3 ? xinv.data_ptr<float>() : nullptr;
    q.winv = s3 ? winv.data_ptr<float>() : nullptr;
    q.bias = bias_of(bias, v0);
    q.n = (int)p.n;
    q.vp = (int)vp;
    q.dp = (int)p.dp;
    auto* Gp = reinterpret_cast<ushort*>(G.data_ptr());
    with_types(p, [&](auto seg, auto bf) {
      constexpr int SEG = decltype(seg)::value;
      constexpr bool BF = decltype(bf)::value;
      with_row_tile(p, [&](auto tile) {
        using C = decltype(tile);
        if constexpr (reached<C, SEG>()) {
        const int nmt = (int)((p.n + C::BM - 1) / C::BM);
        const int nvt = (int)((vp + C::BN - 1) / C::BN);
        auto launch = [&](auto kernel) {
          allow_lds(kernel, C::LDS_BYTES);
          kernel<<<nmt * nvt, C::THREADS, C::LDS_BYTES, stream>>>(
              q, reinterpret_cast<const Row*>(rows.data_ptr()),
              sc.template data_ptr<float>(), p.v, v0, eps, Gp, ldg, glo,
              want_db ? dbp.template data_ptr<float>() : nullptr, nmt, nvt);
          HIP_CHECK_KERNEL();
        };
        if (want_db) {
          launch(lce_grad_kernel<C, x_layout<C>(), SEG, BF, true>);
          lce_db_kernel<<<(int)((vp + 255) / 256), 256, 0, stream>>>(
              dbp.template data_ptr<float>(), nmt, ldg, (int)vp,
              static_cast<char*>(db.data_ptr()) + v0 * db.element_size(),
              type_code(db));
          HIP_CHECK_KERNEL();
        } else {
          launch(lce_grad_kernel<C, x_layout<C>(), SEG, BF, false>);
        }
        }
      });
      if (want_dw) {
        auto run = [&](auto tile) {
          using C = decltype(tile);
          const int nmt = (int)((vp + C::BM - 1) / C::BM);
          const int nnt = (int)((p.d + C::BN - 1) / C::BN);
          auto kernel = lce_dw_kernel<C, SEG, BF>;
          allow_lds(kernel, C::LDS_BYTES);
          kernel<<<nmt * nnt, C::THREADS, C::LDS_BYTES, stream>>>(
              rows_operand(Gp, nrows, ldg, glo, ldg),
              rows_operand(bits(xpk), p.np, p.dp, p.np * p.dp, p.dp),
              (int)up(p.n, 64), sc.template data_ptr<float>(),
              s3 ? xinv.data_ptr<float>() : nullptr,
              static_cast<char*>(dw.data_ptr()) +
                  v0 * p.d * dw.element_size(),
              p.type, (int)vp, (int)p.d, nmt, nnt);
          HIP_CHECK_KERNEL();
        };
        const long cover = ((vp + 255) / 256) * ((p.dp + 255) / 256);
        if (cover >= 192 && p.dp % 256 == 0) {
          run(Big{});
        } else if (cover >= 48 && p.dp >= 128) {
          run(Mid{});
        } else {
          run(Small{});
        }
      }
      if (want_dx) {
        auto run = [&](auto tile) {
          using C = decltype(tile);
          const int nmt = (int)((p.n + C::BM - 1) / C::BM);
          const int nnt = (int)((p.dp + C::BN - 1) / C::BN);
          const int kv = (int)up(vp, 64);
          const int kslice = (int)up((kv + slices - 1) / slices, 64);
          auto kernel = lce_dx_kernel<C, SEG, BF>;
          allow_lds(kernel, C::LDS_BYTES);
          kernel<<<nmt * nnt * slices, C::THREADS, C::LDS_BYTES, stream>>>(
              rows_operand(Gp, nrows, ldg, glo, ldg), q.w, kv, kslice,
              part.data_ptr<float>(), (int)p.n, (int)p.dp, v0 == 0, nmt, nnt,
              slices);
          HIP_CHECK_KERNEL();
        };
        if (dx_tile == 256) {
          run(Big{});
        } else if (dx_tile == 128) {
          run(Mid{});
        } else {
          run(Small{});
        }
      }
    });
  }
  if (want_dx) {
    lce_dx_sum_kernel<<<px_grid(p.n * p.d), 256, 0, stream>>>(
        part.data_ptr<float>(), slices, p.n, (int)p.d, (int)p.dp,
        sc.data_ptr<float>(), s3 ? winv.data_ptr<float>() : nullptr,
        dx.data_ptr(), p.type);
    HIP_CHECK_KERNEL();
  }
  return {dx, dw, db};
}
