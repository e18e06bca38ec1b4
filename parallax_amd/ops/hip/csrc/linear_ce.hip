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
// bits (of a fixed budget up to 360,000 rows, 180,000 in fp32; in 16 bits it
// stays in the last-level cache), and two products read G: dw of the piece,
// finished, and dx, which adds up in fp32 over the pieces.  The time is that of the
// products, which keep the matrix units busy for 33 to 58% of it (the LDS for
// 23 to 32%; the rest is waits for the stages' loads, exponentials and
// stores): 2,560 rows of 512, 793,470 words, bf16, forward and backward 8.9
// ms for 8.3 TFLOP (the logits counted twice), 0.94 PF; a large library
// product reaches 1.41.  Row sums, maxima, lse and all sums over k are fp32.
// No atomics: every result is independent of the order of blocks.
//
// Types.  bf16 and fp16 inputs are multiplied as they are; G is rounded to
// the same type once, relative to the largest |g|, and the results are
// scaled back (at most 2^-8 or 2^-11 of each value, as the final rounding of
// the gradients is; fp16 G below 2^-27 of the largest |g| is off by up to
// 2^-38 of that).
//
// fp32 inputs are split into two fp16 parts after a scaling by a power of two,
// and so is G: three products in the place of one.  Two parts hold 22 bits of
// values down to 2^-17 of the largest that shares their scale, and 2^-39 of
// that of smaller ones, so scales have to follow the values: x has one a row,
// and G goes out twice, for dw with one for each word and tile of rows (the
// words of a large vocabulary differ by 1e12 and more in probability, and
// each has a gradient of its own), for dx with one for each row.  w has one a
// row in the forward and a single one in the backward: dx is off by up to
// 2^-38 of the row's |g| max |w| where its own terms are smaller.
//
// Rows whose label is ignored are read as zeros, so what lies in them (a
// padded batch's garbage, NaN) reaches no gradient.

#include <torch/extension.h>
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <mutex>
#include <set>

#include "mm_tile.h"

namespace {

using namespace mm;

// exponentials are powers of 2, so logits are held times log2 e
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// G of one piece of the vocabulary takes at most this much (fp32: each of its
// two forms), or what 256 words take where that is more: 512 B a row, 1 KB
// each in fp32, so 2 GB in all for the most rows there can be
constexpr long kPieceBytes = 176L << 20;
// and the split parts of an fp32 table's piece at most this, or 256 words'
constexpr long kSplitBytes = 128L << 20;

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
  __device__ __forceinline__ float one(int v, int words) const {
    return p && v < words ? kLog2e * load_as(p, v * stride, type) : 0.f;
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
  // top in [2^(e - 127), 2^(e - 126)), or below 2^-126 where e = 0
  const int e = __float_as_uint(top) >> 23;
  int k = 13 - (e - 127);
  k = k < -120 ? -120 : (k > 120 ? 120 : k);
  return __uint_as_float((unsigned)(k + 127) << 23);
}

// S for G: bf16 and fp16 rows of the largest |g| get -1 or -2^13 at a label
// without probability, where G = -(1 - e) g.  These values are many and, as
// g is often that of all rows, equal: rounded, they would all be off by the
// same, up to 2^-8 (2^-11) of dx and dw.
__device__ __forceinline__ float scale_of_g(float top, float e, int type) {
  if (e <= 0.5f) top *= 1.f - e;
  if (type == 2 || !(top > 1e-30f) || !(top < 1e30f))
    return type == 0 ? 1.f : scale_to_half(top);
  return (type == 0 ? 1.f : 8192.f) / top;
}

// --- laying out an operand --------------------------------------------------

// What the gradient needs of the rows.  Rows that do not count: an infinite
// l makes their exponentials 0, and g = 0.
struct Rows {
  float* l;  // log2 e lse
  float* g;  // what the row's G is multiplied by
  int* y;    // label
};

struct Pack {
  const void* src;
  int type;
  long rs, cs;        // strides in elements
  long rows;          // as they are; zeros up to rows_out
  int d;              // zeros up to dp
  bool eight;         // 16-byte pieces can be read
  int dp;
  long rows_out;
  ushort* out;        // [rows_out][dp], fp32: in pairs of parts
  ushort* blocks;     // [dp / 32][rows_out][32] (16-bit types)
  const int64_t* labels;  // x only: rows of `ignore` become zeros
  int64_t ignore;
  // fp32: the scale of every row is found from top[0..ntop) where given,
  // else each row has its own; inv[r] = 1 / scale; bmax: the largest value
  // of each block, for a later call's `top`
  const float* top;
  int ntop;
  float* inv;
  float* bmax;
  // backward: the rows, and sc = {S, 1/S} for 16-bit G
  Rows row;
  const float* dloss; // one or (each) of every row
  bool each;
  const float* count;
  const float* lse;
  long V;
  float eps;
  float* sc;
};

__device__ __forceinline__ void load8(const Pack& p, const char* src, long c,
                                      float (&v)[8]) {
  if (p.eight && p.type == 2) {
    const f4 a = *reinterpret_cast<const f4*>(src + c * 4);
    const f4 b = *reinterpret_cast<const f4*>(src + c * 4 + 16);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] = a[e];
      v[4 + e] = b[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      v[e] = c + e < p.d ? load_as(src, (c + e) * p.cs, p.type) : 0.f;
  }
}

// A wave takes one row, or several of fewer than 512 values, eight values a
// lane at a time.  Bound by memory: 793,470 fp32 rows of 512 into pairs 0.83
// ms, 3.9 TB/s read and written.
template <int PARTS>
__global__ __launch_bounds__(256) void lce_pack_kernel(Pack p) {
  __shared__ float scratch[PX_BLOCK / WAVE];
  // lanes of a row, rows of a wave, this lane's place in its row
  const int lanes = p.dp > 256 ? 64 : p.dp > 128 ? 32 : p.dp > 64 ? 16 : 8;
  const int rows = 64 / lanes;
  const int lane = threadIdx.x & (lanes - 1);
  const int sub = (threadIdx.x & 63) / lanes;
  const int size = PARTS == 2 ? 4 : 2;
  float scale = 1.f, most = 0.f;
  if (PARTS == 2 && p.top != nullptr) {
    float t = 0.f;
    for (int i = threadIdx.x; i < p.ntop; i += blockDim.x)
      t = fmaxf(t, p.top[i]);
    scale = scale_to_half(block_reduce_max(t, scratch));
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    if (p.sc && !p.each) {
      // |softmax - target| <= 1, so S |G| stays below 2^15
      const float g = p.dloss[0] / (p.count ? p.count[0] : 1.f);
      const float s = scale_of_g(fabsf(g), p.eps, p.type);
      p.sc[0] = s;
      p.sc[1] = 1.f / s;
    }
  }
  for (long r = ((long)blockIdx.x * 4 + (threadIdx.x >> 6)) * rows + sub;
       r < p.rows_out; r += (long)gridDim.x * 4 * rows) {
    bool live = r < p.rows;
    if (p.labels && live) {
      const int64_t y = p.labels[r];
      live = y != p.ignore;
      if (p.row.l && lane == 0) {
        const float g = p.dloss[p.each ? r : 0] / (p.count ? p.count[0] : 1.f);
        p.row.l[r] = live ? p.lse[r] * kLog2e : INFINITY;
        p.row.g[r] = live ? g : 0.f;
        p.row.y[r] = (int)(y < 0 ? 0 : (y >= p.V ? p.V - 1 : y));
      }
    } else if (p.row.l && lane == 0) {
      p.row.l[r] = INFINITY;
      p.row.g[r] = 0.f;
      p.row.y[r] = 0;
    }
    const char* src = static_cast<const char*>(p.src) + r * p.rs * size;
    if constexpr (PARTS == 1) {
      for (int c = lane * 8; c < p.dp; c += lanes * 8) {
        s8 u = {};
        if (live && p.eight && c < p.d) {
          u = *reinterpret_cast<const s8*>(src + c * 2);
        } else if (live) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (c + e < p.d)
              u[e] = reinterpret_cast<const short*>(src)[(c + e) * p.cs];
        }
        if (p.out) *reinterpret_cast<s8*>(p.out + r * p.dp + c) = u;
        if (p.blocks)
          *reinterpret_cast<s8*>(
              p.blocks + ((long)(c >> 5) * p.rows_out + r) * 32 + (c & 31)) =
              u;
      }
    } else {
      if (p.top == nullptr) {
        float t = 0.f;
        if (live) {
          for (int c = lane * 8; c < p.d; c += lanes * 8) {
            float v[8];
            load8(p, src, c, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float a = fabsf(v[e]);
              if (a < INFINITY) t = fmaxf(t, a);
            }
          }
        }
        for (int o = lanes / 2; o > 0; o >>= 1)
          t = fmaxf(t, __shfl_xor(t, o, 64));
        most = fmaxf(most, t);
        scale = scale_to_half(t);
      }
      if (lane == 0) p.inv[r] = 1.f / scale;
      for (int c = lane * 8; c < p.dp; c += lanes * 8) {
        float v[8] = {};
        if (live && c < p.d) load8(p, src, c, v);
        s8 h, l;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          ushort hi, lo;
          split(v[e] * scale, hi, lo);
          h[e] = hi;
          l[e] = lo;
        }
        ushort* at = p.out + r * p.dp * 2 + (c >> 5) * 64 + (c & 31);
        *reinterpret_cast<s8*>(at) = h;
        *reinterpret_cast<s8*>(at + 32) = l;
      }
    }
  }
  if (PARTS == 2 && p.bmax != nullptr) {
    most = block_reduce_max(most, scratch);
    if (threadIdx.x == 0) p.bmax[blockIdx.x] = most;
  }
}

// sc = {S, 1/S} where every row has a gradient of its own
__global__ __launch_bounds__(1024) void lce_scale_kernel(
    const float* __restrict__ dloss, const int64_t* __restrict__ labels,
    int64_t ignore, int n, float eps, int type, float* __restrict__ sc) {
  __shared__ float red[16];
  float most = 0.f;
  for (int i = threadIdx.x; i < n; i += 1024)
    if (labels[i] != ignore) most = fmaxf(most, fabsf(dloss[i]));
  most = block_reduce_max(most, red);
  if (threadIdx.x == 0) {
    const float s = scale_of_g(most, eps, type);
    sc[0] = s;
    sc[1] = 1.f / s;
  }
}

// --- forward ----------------------------------------------------------------

struct Vec {  // a tensor's values by row and column
  const void* p;
  int type;
  long rs, cs;
};

struct Logits {
  Operand x, w;
  const float* xinv;  // parts: scales to undo, by row and by word
  const float* winv;
  Bias bias;
  int n;     // rows
  int vp;    // words in this piece
  int dp;
};

// max, sum of exp and (SMOOTH) total of each row, in powers of 2, over `tpb`
// tiles of words.  2,560 x 793,470 x 512 bf16: 2.16 ms, 0.96 PF; what the
// product alone does not reach is the exponentials, a quarter of the rate of
// other instructions, under which only the other workgroup's products run.
// fp32, 320 rows: 0.95 ms, 0.82 PF of 16-bit products.
template <class C, int XL, int PARTS, bool BF, bool SMOOTH>
__global__ __launch_bounds__(C::THREADS, C::OCC) void lce_fwd_kernel(
    Logits p, float* __restrict__ part, int vb0, int nblocks, int nmt,
    int nvb, int tpb) {
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
    if (PARTS == 2) {
      int m = m0 + wm + i * 16 + (lane & 15);
      if (m > p.n - 1) m = p.n - 1;
      xs[i] = p.xinv[m];
    }
  }
  for (int q = 0; q < tpb; ++q) {
    const int n0 = (vb * tpb + q) * C::BN;
    if (n0 >= p.vp) break;
    f4 acc[C::FM][C::FN] = {};
    product<C, XL, KROWS, PARTS, BF>(smem, p.x, m0, p.w, n0, 0, p.dp, acc);
    float add[C::FN][4], ws[C::FN][4];
#pragma unroll
    for (int j = 0; j < C::FN; ++j)
      p.bias.load(add[j], n0 + wn + j * 16 + (lane >> 4) * 4, p.vp);
#pragma unroll
    for (int j = 0; j < C::FN; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int v = n0 + wn + j * 16 + (lane >> 4) * 4 + r;
        ws[j][r] = PARTS == 2 && v < p.vp ? p.winv[v] * kLog2e : kLog2e;
      }
    const bool whole = n0 + C::BN <= p.vp;
    if (!whole) {  // words behind the last one
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
          const float z = fmaf(PARTS == 2 ? acc[i][j][r] * xs[i]
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
          if (SMOOTH && whole) tot[i] += acc[i][j][r];
        }
      mx[i] = top;
      se[i] = s;
    }
    if (SMOOTH && !whole) {
#pragma unroll
      for (int i = 0; i < C::FM; ++i)
#pragma unroll
        for (int j = 0; j < C::FN; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (n0 + wn + j * 16 + (lane >> 4) * 4 + r < p.vp)
              tot[i] += acc[i][j][r];
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
    // of a row next to one another, for the join
    float* at = part + ((long)(m0 + r) * nblocks + vb0 + vb) * (SMOOTH ? 4 : 2);
    if (SMOOTH) {
      *reinterpret_cast<f4*>(at) = f4{m, s, t, 0.f};
    } else {
      *reinterpret_cast<float2*>(at) = make_float2(m, s);
    }
  }
}

struct Join {
  const float* part;
  int nblocks;
  Vec x, w, bias;
  int d, n;
  const int64_t* labels;
  int64_t ignore;
  long V;
  float eps;
  float* loss;
  float* lse;
};

__device__ __forceinline__ void join(float& m, float& s, float m2, float s2) {
  const float top = fmaxf(m, m2);
  const float off = top == -INFINITY ? 0.f : top;
  s = s * exp2_fast(m - off) + s2 * exp2_fast(m2 - off);
  m = top;
}

// One wave a row joins its partial sums, takes the label's logit as a dot
// product, and the loss.  WAVES: that many take a row's sums (6,200 of each
// of 320 rows: 22 us with four, 61 with one; 12 since the label's product
// does not ask for its type at each load).
template <int WAVES>
__global__ __launch_bounds__(256) void lce_join_kernel(Join p) {
  __shared__ float red[4][3];
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  const int r = WAVES == 1 ? blockIdx.x * 4 + wave : blockIdx.x;
  if (r < p.n) {
    float m = -INFINITY, s = 0.f, t = 0.f;
#pragma unroll 4
    for (int b = WAVES == 1 ? lane : threadIdx.x; b < p.nblocks;
         b += 64 * WAVES) {
      const long at = (long)r * p.nblocks + b;
      if (p.eps != 0.f) {
        const f4 v = reinterpret_cast<const f4*>(p.part)[at];
        join(m, s, v[0], v[1]);
        t += v[2];
      } else {
        const float2 v = reinterpret_cast<const float2*>(p.part)[at];
        join(m, s, v.x, v.y);
      }
    }
    const int64_t y0 = p.labels[r];
    const bool live = y0 != p.ignore;
    const long y = y0 < 0 ? 0 : (y0 >= p.V ? p.V - 1 : y0);
    float a = 0.f;
    if (live && (WAVES == 1 || wave == 0)) {
      auto dot = [&](auto type) {  // known, so that loads need not wait
        constexpr int T = decltype(type)::value;
#pragma unroll 8
        for (int c = lane; c < p.d; c += 64)
          a += load_as(p.x.p, r * p.x.rs + c * p.x.cs, T) *
               load_as(p.w.p, y * p.w.rs + c * p.w.cs, T);
      };
      if (p.x.type == 2) {
        dot(std::integral_constant<int, 2>{});
      } else if (p.x.type == 1) {
        dot(std::integral_constant<int, 1>{});
      } else {
        dot(std::integral_constant<int, 0>{});
      }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      join(m, s, __shfl_xor(m, o, 64), __shfl_xor(s, o, 64));
      t += __shfl_xor(t, o, 64);
      a += __shfl_xor(a, o, 64);
    }
    if (WAVES > 1) {
      if (lane == 0) {
        red[wave][0] = m;
        red[wave][1] = s;
        red[wave][2] = t;
      }
      __syncthreads();
      if (wave > 0) return;
      for (int q = 1; q < WAVES; ++q) {
        join(m, s, red[q][0], red[q][1]);
        t += red[q][2];
      }
    }
    if (lane == 0) {
      if (live && p.bias.p) a += load_as(p.bias.p, y * p.bias.rs, p.bias.type);
      const float l = m * kLn2 + logf(s);
      p.lse[r] = l;
      // lse and the label's logit are sums in different orders: where they
      // are equal, the difference may round to less than nothing (NaN stays)
      float out = l - a;
      if (out < 0.f) out = 0.f;
      if (p.eps != 0.f) {
        const float rest = l - t * kLn2 / (float)p.V;
        out = (1.f - p.eps) * out + p.eps * (rest < 0.f ? 0.f : rest);
      }
      p.loss[r] = live ? out : 0.f;
    }
  }
}

// Sum or mean of the rows that are not ignored, and their number, in the
// rows' order.  (Left to the last workgroup of the join, its fences cost
// 20 us: a kernel of its own takes 5.)
__global__ __launch_bounds__(1024) void lce_total_kernel(
    const float* __restrict__ loss, const int64_t* __restrict__ labels,
    int64_t ignore, int n, bool mean, float* __restrict__ out,
    float* __restrict__ count) {
  __shared__ double sd[16];
  __shared__ int sn[16];
  double a = 0.;
  int c = 0;
#pragma unroll 4
  for (int i = threadIdx.x; i < n; i += 1024) {
    a += loss[i];
    c += labels[i] != ignore;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    a += __shfl_xor(a, o, 64);
    c += __shfl_xor(c, o, 64);
  }
  if ((threadIdx.x & 63) == 0) {
    sd[threadIdx.x >> 6] = a;
    sn[threadIdx.x >> 6] = c;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 16; ++w) {
      sd[0] += sd[w];
      sn[0] += sn[w];
    }
  }
  if (threadIdx.x == 0) {
    out[0] = (float)(mean ? sd[0] / sn[0] : sd[0]);
    count[0] = (float)sn[0];
  }
}

// --- backward ---------------------------------------------------------------

// G of one piece, transposed: [words][ldg], zeros outside the matrix.  The
// words are the tile's m: a lane holds four neighbouring rows of one word,
// sums over the rows stay in it, and dw reads G k-contiguous.  PARTS = 2: in
// pairs of parts, twice.  For dx (Gx) scaled by a power of two for each row;
// for dw (G) by one for each word and tile of rows, whose reciprocal goes to
// tinv[tile][words], and with the scales undone that the rows of x have
// (20,000 words x 999 rows of 256 63 us, 44 with one form under one scale).
// DB: sums of each tile of rows into dbp[row tile][..], or as they are into
// db where there is one.  2,560 x 32,768 x 512 bf16: 124 us, 0.69 PF: beside
// the exponentials 168 MB of G go out, 34 us by themselves.
template <class C, int XL, int PARTS, bool BF, bool DB>
__global__ __launch_bounds__(C::THREADS, C::OCC) void lce_grad_kernel(
    Logits p, Rows rows, const float* __restrict__ sc, long V, long v0,
    float eps, ushort* __restrict__ G, ushort* __restrict__ Gx, int ldg,
    float* __restrict__ tinv, long t_ld, float* __restrict__ dbp, long db_ld,
    void* __restrict__ db, int db_type, int nvt, int nrt) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int bid = die_contiguous(blockIdx.x, nvt * nrt);
  const int rt = bid % nrt, vt = bid / nrt;
  const int m0 = vt * C::BM, n0 = rt * C::BN;
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  const int wm = (wave / C::WAVES_N) * C::WM;
  const int wn = (wave % C::WAVES_N) * C::WN;
  f4 acc[C::FM][C::FN] = {};
  product<C, KROWS, XL, PARTS, BF>(smem, p.w, m0, p.x, n0, 0, p.dp, acc);
  const float S = sc[0], uni = eps / (float)V;
  const int w0 = m0 + wm + (lane & 15);  // this lane's first word
  float add[C::FM], ws[C::FM], sum[C::FM];
#pragma unroll
  for (int i = 0; i < C::FM; ++i) {
    const int v = w0 + i * 16;
    add[i] = p.bias.one(v, p.vp);
    ws[i] = kLog2e;
    if (PARTS == 2) ws[i] *= v < p.vp ? p.winv[v] : 0.f;
    sum[i] = 0.f;
  }
#pragma unroll
  for (int j = 0; j < C::FN; ++j) {
    // there are rows up to a whole tile
    const int n = n0 + wn + j * 16 + (lane >> 4) * 4;
    const f4 l = *reinterpret_cast<const f4*>(rows.l + n);
    const f4 g = S * *reinterpret_cast<const f4*>(rows.g + n);
    const int4 y = *reinterpret_cast<const int4*>(rows.y + n);
    f4 xs = {1.f, 1.f, 1.f, 1.f};
    if (PARTS == 2) xs = *reinterpret_cast<const f4*>(p.xinv + n);
#pragma unroll
    for (int i = 0; i < C::FM; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float z = PARTS == 2 ? acc[i][j][r] * xs[r] : acc[i][j][r];
        acc[i][j][r] = fmaf(exp2_fast(fmaf(z, ws[i], add[i] - l[r])), g[r],
                            -uni * g[r]);
      }
    // the label's word: in few tiles, so not a comparison for each value
    const int at[4] = {y.x, y.y, y.z, y.w};
    const int first = (int)v0 + m0 + wm;
    bool hit = false;
#pragma unroll
    for (int r = 0; r < 4; ++r)
      hit |= (unsigned)(at[r] - first) < (unsigned)C::WM;
    if (__any(hit)) {
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int i = 0; i < C::FM; ++i)
          if (at[r] - first == i * 16 + (lane & 15))
            acc[i][j][r] -= (1.f - eps) * g[r];
    }
  }
#pragma unroll
  for (int i = 0; i < C::FM; ++i)
    if (w0 + i * 16 >= p.vp) {  // words behind the last one
#pragma unroll
      for (int j = 0; j < C::FN; ++j) acc[i][j] = f4{0.f, 0.f, 0.f, 0.f};
    }
  if constexpr (PARTS == 2) {
    const long at = (long)m0 * ldg + n0 * 2;
    auto four = [&](const float* v, int j) {  // of this lane's rows
      return *reinterpret_cast<const f4*>(v + n0 + wn + j * 16 +
                                          (lane >> 4) * 4);
    };
    if (Gx) {
      store_pairs<C>(smem, Gx + at, ldg, [&](int i, int j) {
        f4 g = S * four(rows.g, j);
#pragma unroll
        for (int r = 0; r < 4; ++r) g[r] = scale_to_half(fabsf(g[r]));
        return acc[i][j] * g;
      });
      __syncthreads();
    }
    if (tinv) {
      float* red = reinterpret_cast<float*>(smem);  // [waves_n][BM]
      float ts[C::FM] = {};
#pragma unroll
      for (int j = 0; j < C::FN; ++j) {
        const f4 x = four(p.xinv, j);
#pragma unroll
        for (int i = 0; i < C::FM; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            ts[i] = fmaxf(ts[i], fabsf(acc[i][j][r] * x[r]));
      }
#pragma unroll
      for (int i = 0; i < C::FM; ++i) {
        ts[i] = fmaxf(ts[i], __shfl_xor(ts[i], 16, 64));
        ts[i] = fmaxf(ts[i], __shfl_xor(ts[i], 32, 64));
        if (lane < 16)
          red[(wave % C::WAVES_N) * C::BM + wm + i * 16 + lane] = ts[i];
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < C::FM; ++i) {
        const int m = wm + i * 16 + (lane & 15);
#pragma unroll
        for (int w = 0; w < C::WAVES_N; ++w)
          ts[i] = fmaxf(ts[i], red[w * C::BM + m]);
        ts[i] = scale_to_half(ts[i]);
        if (lane < 16 && wave % C::WAVES_N == 0)
          tinv[rt * t_ld + m0 + m] = 1.f / ts[i];
      }
      __syncthreads();
      store_pairs<C>(smem, G + at, ldg, [&](int i, int j) {
        return acc[i][j] * four(p.xinv, j) * ts[i];
      });
    }
  } else {
    store_tile<C>(smem, G + (long)m0 * ldg + n0, ldg, C::BM, C::BN,
                  [&](int i, int j) {
      const f4 v = acc[i][j];
      if (BF)
        return make_ushort4(bf16_bits(v[0]), bf16_bits(v[1]),
                            bf16_bits(v[2]), bf16_bits(v[3]));
      return make_ushort4(fp16_bits(v[0]), fp16_bits(v[1]), fp16_bits(v[2]),
                          fp16_bits(v[3]));
    });
  }
  if (DB) {
    float* red = reinterpret_cast<float*>(smem);  // [waves_n][BM]
#pragma unroll
    for (int i = 0; i < C::FM; ++i) {
#pragma unroll
      for (int j = 0; j < C::FN; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) sum[i] += acc[i][j][r];
      sum[i] += __shfl_xor(sum[i], 16, 64);
      sum[i] += __shfl_xor(sum[i], 32, 64);
    }
    __syncthreads();
    if (lane < 16) {
#pragma unroll
      for (int i = 0; i < C::FM; ++i)
        red[(wave % C::WAVES_N) * C::BM + wm + i * 16 + lane] = sum[i];
    }
    __syncthreads();
    for (int c = threadIdx.x; c < C::BM; c += C::THREADS) {
      float s = red[c];
      for (int w = 1; w < C::WAVES_N; ++w) s += red[w * C::BM + c];
      s *= sc[1];
      if (nrt > 1) {
        dbp[rt * db_ld + m0 + c] = s;
      } else if (m0 + c < p.vp) {
        store_as(db, m0 + c, db_type, s);
      }
    }
  }
}

// db from the sums of the tiles of rows, in their order (10 of 793,470 words:
// 13 us, 2.4 TB/s).
__global__ __launch_bounds__(256) void lce_db_kernel(
    const float* __restrict__ dbp, int nmt, long ld, long words, void* db,
    int type) {
  const long v = (long)blockIdx.x * 256 + threadIdx.x;
  if (v >= words) return;
  float s = 0.f;
  for (int m = 0; m < nmt; ++m) s += dbp[m * ld + v];
  store_as(db, v, type, s);
}

// Calls f behind every N stages of a product.
template <int N, class F>
struct TakeEvery {
  static constexpr int EVERY = N;
  F& f;
  __device__ __forceinline__ void operator()() const { f(); }
};

// dw[v, :] = 1/S sum_n G[n, v] x[n, :]  (x k-strided).  32,768 x 512 over
// 2,560 rows bf16: 82 us, 1.05 PF.  PARTS = 2: the sums over each ROWS rows
// are scaled back by tinv[tile][words] and added up in fp32.
template <class C, int PARTS, bool BF, int ROWS>
__global__ __launch_bounds__(C::THREADS, C::OCC) void lce_dw_kernel(
    Operand G, Operand x, int kn, const float* __restrict__ sc,
    const float* __restrict__ tinv, long t_ld, void* __restrict__ dw,
    int type, int vp, int d, int nmt, int nnt) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int bid = die_contiguous(blockIdx.x, nmt * nnt);
  const int m0 = bid / nnt * C::BM, n0 = bid % nnt * C::BN;
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  const int wm = (wave / C::WAVES_N) * C::WM;
  const int wn = (wave % C::WAVES_N) * C::WN;
  f4 acc[C::FM][C::FN] = {};
  if constexpr (PARTS == 2) {
    f4 part[C::FM][C::FN] = {};
    float t[C::FM];  // of the tile of rows at hand: asked for one ahead
    const float* next = tinv + m0 + wm + (lane & 15);
    auto load = [&] {
#pragma unroll
      for (int i = 0; i < C::FM; ++i) t[i] = next[i * 16];
      next += t_ld;
    };
    static_assert(ROWS % 32 == 0 && C::BK == 64, "stages of 32 rows");
    int left = (kn + ROWS - 1) / ROWS;
    load();
    auto take = [&] {
#pragma unroll
      for (int i = 0; i < C::FM; ++i)
#pragma unroll
        for (int j = 0; j < C::FN; ++j) {
          acc[i][j] += part[i][j] * t[i];
          part[i][j] = f4{0.f, 0.f, 0.f, 0.f};
        }
      if (--left > 0) load();
    };
    product<C, KROWS, KCOLS, PARTS, BF>(
        smem, G, m0, x, n0, 0, kn, part,
        TakeEvery<ROWS / 32, decltype(take)>{take});
  } else {
    product<C, KROWS, KCOLS, PARTS, BF>(smem, G, m0, x, n0, 0, kn, acc);
  }
  const float back = sc[1];
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
      const f4 val = acc[i][j] * back;
      if (type == 2 && c + 4 <= d && (d & 3) == 0) {
        *reinterpret_cast<f4*>(static_cast<float*>(dw) + at) = val;
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (c + r < d) store_as(dw, at + r, type, val[r]);
      }
    }
  }
}

// part[slice][n, :] (+)= sum over a slice of the piece's words G[n, v] w[v, :]
// (both k-strided).  2,560 x 512 over 32,768 words bf16: 92 us, 0.94 PF; on
// 256 x 256 tiles the partial sums cost more than the product gains.
template <class C, int PARTS, bool BF>
__global__ __launch_bounds__(C::THREADS, C::OCC) void lce_dx_kernel(
    Operand G, Operand w, int kv, int kslice, float* __restrict__ part,
    int n_rows, int dp, bool first, int nmt, int nnt, int slices) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int bid = die_contiguous(blockIdx.x, nmt * nnt * slices);
  const int sl = bid / (nmt * nnt), t = bid % (nmt * nnt);
  const int m0 = t / nnt * C::BM, n0 = t % nnt * C::BN;
  const int k0 = sl * kslice;
  const int k1 = k0 + kslice < kv ? k0 + kslice : kv;
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  const int wm = (wave / C::WAVES_N) * C::WM;
  const int wn = (wave % C::WAVES_N) * C::WN;
  auto at = [&](int i, int j) -> f4* {
    const int m = m0 + wm + i * 16 + (lane & 15);
    const int c = n0 + wn + j * 16 + (lane >> 4) * 4;
    if (m >= n_rows || c >= dp) return nullptr;
    return reinterpret_cast<f4*>(part + ((long)sl * n_rows + m) * dp + c);
  };
  // go on from the sums of the pieces before
  f4 acc[C::FM][C::FN] = {};
  if (!first) {
#pragma unroll
    for (int i = 0; i < C::FM; ++i)
#pragma unroll
      for (int j = 0; j < C::FN; ++j)
        if (const f4* p = at(i, j)) acc[i][j] = *p;
  }
  if (k0 < k1)
    product<C, KCOLS, KCOLS, PARTS, BF>(smem, G, m0, w, n0, k0, k1, acc);
#pragma unroll
  for (int i = 0; i < C::FM; ++i)
#pragma unroll
    for (int j = 0; j < C::FN; ++j)
      if (f4* p = at(i, j)) *p = acc[i][j];
}

// dx = 1/S of the slices' sums, and (fp32: winv) what the scales of w and of
// the row of G leave to undo.  GROUPS waves of a workgroup take every
// GROUPS-th slice each, in order: many slices of few values would be one long
// chain of loads (185 of 4 x 64: 45 us by one thread each, 4.4 us so).
// Otherwise bound by memory: 32 of 999 x 256, 33 MB, 8 us.
template <int GROUPS>
__global__ __launch_bounds__(GROUPS == 1 ? 256 : 64 * GROUPS)
void lce_dx_sum_kernel(
    const float* __restrict__ part, int slices, long n, int d, int dp,
    const float* __restrict__ sc, const float* __restrict__ winv,
    const float* __restrict__ g, void* __restrict__ dx, int type) {
  __shared__ float red[GROUPS][64];
  constexpr int AT_ONCE = GROUPS == 1 ? 256 : 64;
  const int group = GROUPS == 1 ? 0 : threadIdx.x >> 6;
  const int first = GROUPS == 1 ? threadIdx.x : threadIdx.x & 63;
  for (long i0 = (long)blockIdx.x * AT_ONCE; i0 < n * d;
       i0 += (long)gridDim.x * AT_ONCE) {
    const long i = i0 + first;
    const bool there = i < n * d;
    const long r = i / d;
    const long at = r * dp + (i - r * d);
    float s = 0.f;
    if (there) {
#pragma unroll 4
      for (int q = group; q < slices; q += GROUPS) s += part[q * n * dp + at];
    }
    if (GROUPS > 1) {
      red[group][first] = s;
      __syncthreads();
      if (group == 0) {
#pragma unroll
        for (int g = 1; g < GROUPS; ++g) s += red[g][first];
      }
      __syncthreads();
    }
    if (there && group == 0) {
      if (winv) s = s / scale_to_half(fabsf(sc[0] * g[r])) * winv[0];
      store_as(dx, i, type, s * sc[1]);
    }
  }
}

// --- host -------------------------------------------------------------------

// Sixteen waves of 64 x 64, one workgroup on a CU: the most products for a
// byte that comes from memory, and four waves on a SIMD to wait for another.
using Big = Tile<256, 256, 64, 64, 64, 2>;
using Mid = Tile<128, 128, 64, 64, 64, 2>;
// two parts: eight waves, as they leave the LDS more time (both operands
// k-strided, 20480 x 512 x 2560: 148 us, 160 with four waves of 64 x 64)
using MidParts = Tile<128, 128, 32, 64, 64, 2>;
template <int PARTS>
using MidOf = std::conditional_t<PARTS == 2, MidParts, Mid>;
template <int PARTS>
using BigOf = std::conditional_t<PARTS == 2, MidParts, Big>;
// few rows, or rows that leave much of a larger tile empty: wide in the words
using Flat = Tile<64, 256, 64, 32, 64, 2>;
using FlatT = Tile<256, 64, 64, 32, 64, 2>;
// few tiles: four stages deep, as a workgroup has a CU for itself
using Small = Tile<64, 64, 32, 32, 64, 4>;

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

// more than 64 KB of LDS has to be asked for, once a kernel and device
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
  TORCH_CHECK(e == hipSuccess, "linear_ce: ", bytes, " bytes of LDS: ",
              hipGetErrorString(e));
  done.insert(key);
}

const ushort* bits(const at::Tensor& t) {
  return reinterpret_cast<const ushort*>(t.data_ptr());
}

Vec vec_of(const at::Tensor& t) {
  return Vec{t.data_ptr(), type_code(t), t.stride(0),
             t.dim() > 1 ? t.stride(1) : 0};
}

// One allocation for all of a call's scratch memory.
class Scratch {
 public:
  template <typename T>
  size_t take(long n) {
    const size_t at = bytes_;
    bytes_ += (n * sizeof(T) + 255) / 256 * 256;
    return at;
  }
  void allocate(const at::Tensor& like) {
    t_ = at::empty({(long)bytes_}, like.options().dtype(at::kByte));
    base_ = static_cast<char*>(t_.data_ptr());
  }
  template <typename T>
  T* at(size_t offset) const {
    return reinterpret_cast<T*>(base_ + offset);
  }

 private:
  size_t bytes_ = 0;
  at::Tensor t_;
  char* base_ = nullptr;
};

// What the products read: x laid out once, w as it is or piece by piece.
struct Plan {
  long n, v, d, dp, np;
  int type, parts;
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
  p.parts = p.type == 2 ? 2 : 1;
  p.w_direct = p.parts == 1 && p.d == p.dp && w.stride(1) == 1 &&
               w.stride(0) % 8 == 0 && w.stride(0) >= p.d &&
               w.stride(0) < (1 << 22) &&
               reinterpret_cast<uintptr_t>(w.data_ptr()) % 16 == 0;
  const long words = kSplitBytes / (p.dp * 2 * p.parts);
  p.w_rows = std::min(up(p.v, 256), std::max(256L, words / 256 * 256));
  return p;
}

int pack_blocks(long rows) {
  return (int)std::min<long>(2048, (rows + 3) / 4);
}

// the layout of rows row0.. of a tensor
Pack pack_of(const at::Tensor& t, long row0, long rows, long rows_out,
             const Plan& p, ushort* out) {
  Pack k = {};
  const long size = t.element_size();
  k.src = static_cast<const char*>(t.data_ptr()) + row0 * t.stride(0) * size;
  k.type = p.type;
  k.rs = t.stride(0);
  k.cs = t.stride(1);
  k.rows = rows;
  k.d = (int)p.d;
  k.eight = k.cs == 1 && p.d % 8 == 0 && (k.rs * size) % 16 == 0 &&
            reinterpret_cast<uintptr_t>(k.src) % 16 == 0;
  k.dp = (int)p.dp;
  k.rows_out = rows_out;
  k.out = out;
  return k;
}

void pack(const Pack& k, hipStream_t stream) {
  if (k.type == 2) {
    lce_pack_kernel<2><<<pack_blocks(k.rows_out), 256, 0, stream>>>(k);
  } else {
    lce_pack_kernel<1><<<pack_blocks(k.rows_out), 256, 0, stream>>>(k);
  }
  HIP_CHECK_KERNEL();
}

Operand operand(const ushort* p, long rows, long ld, long cols) {
  Operand o;
  o.p = p;
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
  TORCH_CHECK(up(x.size(0), 256) * up(x.size(1), 64) < (1L << 29),
              "linear_ce: x has 2^29 values or more: take fewer rows at a "
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

// calls f(parts, bf16) with compile-time arguments
template <typename F>
void with_types(const Plan& p, F f) {
  if (p.type == 0) {
    f(std::integral_constant<int, 1>{}, std::true_type{});
  } else if (p.type == 1) {
    f(std::integral_constant<int, 1>{}, std::false_type{});
  } else {
    f(std::integral_constant<int, 2>{}, std::false_type{});
  }
}

// The tile of the logits, forward and backward.  Many 16-bit rows: 256 x 128
// in two workgroups a CU, so that one's exponentials and stores run under the
// other's products, with x in blocks.
using Logit = Tile<256, 128, 64, 64, 32, 3>;
using LogitT = Tile<128, 256, 64, 64, 32, 3>;  // words by rows

template <class C>
constexpr int x_layout() {
  return C::BK == 32 ? KBLOCK : KROWS;
}

// two-part operands never meet those tiles
template <class C, int PARTS>
constexpr bool reached() {
  return !std::is_same<C, std::conditional_t<PARTS == 2, Mid, MidParts>>::value
         && (C::BK == 64 || PARTS == 1);
}

// 64 rows a tile where 128 would be empty by an eighth: 320 rows of 50,000
// words forward 43 and 48 us in bf16, 106 and 114 in fp32, with gradients 148
// and 158, 385 and 408
bool flat(const Plan& p) { return up(p.n, 64) * 8 <= up(p.n, 128) * 7; }

// Fewer 128 x 128 tiles than half of the CUs: 64 x 64.  512 x 1000 x 512
// forward 23 us, 26 with the larger, in fp32 27 and 36; 1228 x 860 x 896 in
// fp32 with gradients 110 and 126.
bool few(const Plan& p) {
  return !flat(p) && (up(p.n, 128) / 128) * (up(p.v, 128) / 128) < 128;
}

bool blocked(const Plan& p) {
  // not where 256-row tiles would be empty by more than they gain
  return p.parts == 1 && !flat(p) && !few(p) &&
         up(p.n, 256) * 100 <= up(p.n, 128) * 115;
}

// f(tile of the forward, tile of the backward)
template <typename F>
void with_row_tile(const Plan& p, F f) {
  if (flat(p)) {
    f(Flat{}, FlatT{});
  } else if (few(p)) {
    f(Small{}, Small{});
  } else if (blocked(p)) {
    f(Logit{}, LogitT{});
  } else if (p.parts == 2) {
    f(MidParts{}, MidParts{});
  } else {
    f(Mid{}, Mid{});
  }
}

}  // namespace

// {loss (scalar or [N]), what the backward needs: lse [N], the count, and
// (fp32) the largest |w| of blocks}
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
  const auto* lab = labels.data_ptr<int64_t>();
  const float eps = (float)smoothing;
  const bool blk = blocked(p);
  const long piece = p.w_direct ? p.v : p.w_rows;
  const long pieces = (p.v + piece - 1) / piece;
  const int wblocks = pack_blocks(p.w_rows);
  const long ntop = p.parts == 2 ? pieces * wblocks : 0;
  auto out = reduction == 0 ? at::empty({p.n}, f32) : at::empty({}, f32);
  auto saved = at::empty({p.n + 1 + ntop}, f32);
  float* lse = saved.data_ptr<float>();
  float* tops = lse + p.n + 1;

  with_row_tile(p, [&](auto tile, auto) {
    using C = decltype(tile);
    const int nmt = (int)((p.n + C::BM - 1) / C::BM);
    const long piece_tiles = (std::min(piece, p.v) + C::BN - 1) / C::BN;
    // A workgroup takes several tiles of words, so that its sums are joined
    // once, as long as ~2,000 workgroups are left, which are several turns
    // of all CUs.  2,560 rows x 793,470 words of 512 in bf16: one tile 2,213
    // us, four 1,933, eight 1,914, sixteen 1,996; 320 rows in fp32, where
    // pieces are short: one 1,591, two 1,700, eight 2,086; 512 x 32,000
    // (500 tiles) in bf16 one 33, four 47.
    int tpb = (int)std::min<long>(8, piece_tiles * nmt / 2048);
    if (tpb < 1) tpb = 1;
    const long span = (long)C::BN * tpb;
    const int nvb = (int)((std::min(piece, p.v) + span - 1) / span);
    const long rest = p.v - (pieces - 1) * piece;
    const int blocks = (int)((pieces - 1) * nvb + (rest + span - 1) / span);

    Scratch mem;
    const auto o_x = mem.take<ushort>(p.np * p.dp * p.parts);
    const auto o_xinv = mem.take<float>(p.parts == 2 ? p.np : 0);
    const auto o_w =
        mem.take<ushort>(p.w_direct ? 0 : p.w_rows * p.dp * p.parts);
    const auto o_winv = mem.take<float>(p.parts == 2 ? p.w_rows : 0);
    const auto o_part = mem.take<float>(p.n * blocks * (eps != 0.f ? 4 : 2));
    const auto o_loss = mem.take<float>(reduction == 0 ? 0 : p.n);
    mem.allocate(x);

    Pack kx = pack_of(x, 0, p.n, p.np, p,
                      blk ? nullptr : mem.at<ushort>(o_x));
    if (blk) kx.blocks = mem.at<ushort>(o_x);
    kx.labels = lab;
    kx.ignore = ignore;
    kx.inv = mem.at<float>(o_xinv);
    pack(kx, stream);
    for (long i = 0; i < pieces; ++i) {
      const long v0 = i * piece, vp = std::min(piece, p.v - v0);
      Logits q;
      q.x = operand(mem.at<ushort>(o_x), p.np, p.dp * p.parts, p.dp);
      if (p.w_direct) {
        q.w = operand(bits(w), vp, w.stride(0), p.dp);
      } else {
        Pack kw = pack_of(w, v0, vp, up(vp, 64), p, mem.at<ushort>(o_w));
        kw.inv = mem.at<float>(o_winv);
        if (p.parts == 2) {
          kw.bmax = tops + i * wblocks;
          kw.rows_out = p.w_rows;  // every block has its largest value
        }
        pack(kw, stream);
        q.w = operand(mem.at<ushort>(o_w), kw.rows_out, p.dp * p.parts,
                      p.dp);
      }
      q.xinv = mem.at<float>(o_xinv);
      q.winv = mem.at<float>(o_winv);
      q.bias = bias_of(bias, v0);
      q.n = (int)p.n;
      q.vp = (int)vp;
      q.dp = (int)p.dp;
      const int here = (int)((vp + span - 1) / span);
      with_types(p, [&](auto parts, auto bf) {
        constexpr int PARTS = decltype(parts)::value;
        constexpr bool BF = decltype(bf)::value;
        if constexpr (reached<C, PARTS>()) {
          auto launch = [&](auto kernel) {
            constexpr int lds = C::template lds<1>();
            allow_lds(kernel, lds);
            kernel<<<nmt * here, C::THREADS, lds, stream>>>(
                q, mem.at<float>(o_part), (int)i * nvb, blocks, nmt, here,
                tpb);
            HIP_CHECK_KERNEL();
          };
          if (eps != 0.f) {
            launch(lce_fwd_kernel<C, x_layout<C>(), PARTS, BF, true>);
          } else {
            launch(lce_fwd_kernel<C, x_layout<C>(), PARTS, BF, false>);
          }
        }
      });
    }
    Join j = {};
    j.part = mem.at<float>(o_part);
    j.nblocks = blocks;
    j.x = vec_of(x);
    j.w = vec_of(w);
    if (bias.has_value()) j.bias = vec_of(*bias);
    j.d = (int)p.d;
    j.n = (int)p.n;
    j.labels = lab;
    j.ignore = ignore;
    j.V = p.v;
    j.eps = eps;
    j.loss = reduction == 0 ? out.data_ptr<float>() : mem.at<float>(o_loss);
    j.lse = lse;
    if (blocks > 1024) {
      lce_join_kernel<4><<<(int)p.n, 256, 0, stream>>>(j);
    } else {
      lce_join_kernel<1><<<(int)((p.n + 3) / 4), 256, 0, stream>>>(j);
    }
    HIP_CHECK_KERNEL();
    if (reduction != 0) {
      lce_total_kernel<<<1, 1024, 0, stream>>>(
          j.loss, lab, ignore, (int)p.n, reduction == 1,
          out.data_ptr<float>(), lse + p.n);
      HIP_CHECK_KERNEL();
    }
  });
  return {out, saved};
}

// {dx, dw, db}; an empty tensor for what is not wanted
std::vector<at::Tensor> linear_ce_bwd(
    const at::Tensor& dloss, const at::Tensor& x, const at::Tensor& w,
    const c10::optional<at::Tensor>& bias, const at::Tensor& labels,
    const at::Tensor& saved, int64_t ignore, double smoothing,
    int64_t reduction, bool want_dx, bool want_dw, bool want_db) {
  check(x, w, bias, labels);
  TORCH_CHECK(dloss.scalar_type() == at::kFloat && dloss.is_cuda() &&
                  dloss.is_contiguous() &&
                  dloss.numel() == (reduction == 0 ? x.size(0) : 1),
              "linear_ce_bwd: fp32 gradient of the loss expected");
  const c10::cuda::CUDAGuard guard(x.device());
  auto stream = at::cuda::getCurrentCUDAStream();
  const Plan p = make_plan(x, w);
  const auto* lab = labels.data_ptr<int64_t>();
  const float eps = (float)smoothing;
  const bool two = p.parts == 2, blk = blocked(p);
  const float* lse = saved.data_ptr<float>();
  const float* tops = lse + p.n + 1;
  const int ntop = (int)(saved.numel() - p.n - 1);

  // words for which the tiles of dw fill the chip's 256 CUs once; a piece is
  // whole tiles of 256, as G and the words laid out are written by such
  const long wave_of_words = 256 * 256 / ((p.dp + 255) / 256) / 256 * 256;
  long piece = kPieceBytes / (p.np * 2 * p.parts);
  piece = piece >= wave_of_words ? piece / wave_of_words * wave_of_words
                                 : piece / 256 * 256;
  piece = std::max(256L, std::min(piece, up(p.v, 256)));
  if (!p.w_direct) piece = std::min(piece, p.w_rows);
  // a piece of w ends before its byte 2^31, the largest offset there is
  const long w_ld = p.w_direct ? w.stride(0) : p.dp * p.parts;
  piece = std::max(256L, std::min(piece, ((1L << 30) - 1) / w_ld / 256 * 256));
  TORCH_CHECK(piece % 256 == 0, "linear_ce_bwd: pieces of whole tiles");
  const int ldg = (int)p.np * p.parts;
  // dx: few tiles and a long k, so k is cut until two workgroups a CU have
  // work: 2,560 rows x 100,000 words of 512 in bf16, dx alone: 128 in all
  // 1,610 us, 256 1,005, 512 915, 1,024 988.  At least 512 words each (256
  // and 1,024 are alike).  128 x 128 tiles: 2,560 rows 874 us and 1,306 with
  // 64 x 64, 129 rows 114 and 119.
  const int dx_tile = p.n > 128 && p.dp >= 128 ? 128 : 64;
  const long dx_tiles = ((p.n + dx_tile - 1) / dx_tile) *
                        ((p.dp + dx_tile - 1) / dx_tile);
  const int slices = (int)std::min<long>(std::max(1L, 512 / dx_tiles),
                                         std::max(1L, piece / 512));
  at::Tensor dx, dw, db;
  if (want_dx) dx = at::empty({p.n, p.d}, x.options());
  if (want_dw) dw = at::empty({p.v, p.d}, w.options());
  if (want_db) db = at::empty({p.v}, bias->options());

  with_row_tile(p, [&](auto, auto row_tile) {
    using R = decltype(row_tile);
    const int nrt = (int)((p.n + R::BN - 1) / R::BN);
    // sums over the rows are joined at the end where they are small
    const bool db_late = up(p.v, 256) * nrt <= (16L << 20);
    const long db_ld = db_late ? up(p.v, 256) : piece;

    Scratch mem;
    const auto o_rows = mem.take<float>(3 * p.np);
    const auto o_sc = mem.take<float>(2);
    const auto o_x = mem.take<ushort>(p.np * p.dp * p.parts);
    const auto o_xblk = mem.take<ushort>(blk ? p.np * p.dp : 0);
    const auto o_xinv = mem.take<float>(two ? p.np : 0);
    const auto o_w = mem.take<ushort>(p.w_direct ? 0
                                                 : piece * p.dp * p.parts);
    const auto o_winv = mem.take<float>(two ? piece : 0);
    const auto o_G = mem.take<ushort>(piece * ldg);
    const auto o_Gx = mem.take<ushort>(two && want_dx ? piece * ldg : 0);
    const auto o_tinv = mem.take<float>(two && want_dw ? nrt * piece : 0);
    const auto o_part =
        mem.take<float>(want_dx ? slices * p.n * p.dp : 0);
    const auto o_dbp = mem.take<float>(want_db && nrt > 1 ? nrt * db_ld : 0);
    mem.allocate(x);

    Pack kx = pack_of(x, 0, p.n, p.np, p, mem.at<ushort>(o_x));
    kx.labels = lab;
    kx.ignore = ignore;
    kx.inv = mem.at<float>(o_xinv);
    if (blk) kx.blocks = mem.at<ushort>(o_xblk);
    float* row = mem.at<float>(o_rows);
    kx.row = Rows{row, row + p.np, reinterpret_cast<int*>(row + 2 * p.np)};
    kx.dloss = dloss.data_ptr<float>();
    kx.each = reduction == 0;
    kx.count = reduction == 1 ? lse + p.n : nullptr;
    kx.lse = lse;
    kx.V = p.v;
    kx.eps = eps;
    kx.sc = mem.at<float>(o_sc);
    pack(kx, stream);
    if (kx.each) {
      lce_scale_kernel<<<1, 1024, 0, stream>>>(
          kx.dloss, lab, ignore, (int)p.n, eps, p.type, kx.sc);
      HIP_CHECK_KERNEL();
    }
    auto* G = mem.at<ushort>(o_G);
    auto* Gx = two ? mem.at<ushort>(o_Gx) : G;
    float* tinv = two && want_dw ? mem.at<float>(o_tinv) : nullptr;
    const float* sc = kx.sc;
    const float* xinv = two ? kx.inv : nullptr;
    const float* winv = two ? mem.at<float>(o_winv) : nullptr;
    const Operand xr = operand(mem.at<ushort>(o_x), p.np, p.dp * p.parts,
                               p.dp);

    for (long v0 = 0; v0 < p.v; v0 += piece) {
      const long vp = std::min(piece, p.v - v0);
      Logits q;
      q.x = blk ? operand(mem.at<ushort>(o_xblk), p.np, p.dp, p.dp) : xr;
      if (p.w_direct) {
        q.w = operand(bits(w) + v0 * w.stride(0), vp, w.stride(0), p.dp);
      } else {
        Pack kw = pack_of(w, v0, vp, up(vp, 64), p, mem.at<ushort>(o_w));
        kw.inv = mem.at<float>(o_winv);
        kw.top = two ? tops : nullptr;
        kw.ntop = ntop;
        pack(kw, stream);
        q.w = operand(mem.at<ushort>(o_w), kw.rows_out, p.dp * p.parts,
                      p.dp);
      }
      q.xinv = xinv;
      q.winv = winv;
      q.bias = bias_of(bias, v0);
      q.n = (int)p.n;
      q.vp = (int)vp;
      q.dp = (int)p.dp;
      with_types(p, [&](auto parts, auto bf) {
        constexpr int PARTS = decltype(parts)::value;
        constexpr bool BF = decltype(bf)::value;
        if constexpr (reached<R, PARTS>()) {
          const int nvt = (int)((vp + R::BM - 1) / R::BM);
          float* dbp = mem.at<float>(o_dbp) + (db_late ? v0 : 0);
          void* db_at = want_db ? static_cast<char*>(db.data_ptr()) +
                                      v0 * db.element_size()
                                : nullptr;
          auto launch = [&](auto kernel) {
            constexpr int lds = R::template lds<PARTS>();
            allow_lds(kernel, lds);
            kernel<<<nvt * nrt, R::THREADS, lds, stream>>>(
                q, kx.row, sc, p.v, v0, eps, G,
                two && want_dx ? Gx : nullptr, ldg, tinv, piece, dbp, db_ld,
                db_at, want_db ? type_code(db) : 0, nvt, nrt);
            HIP_CHECK_KERNEL();
          };
          if (want_db) {
            launch(lce_grad_kernel<R, x_layout<R>(), PARTS, BF, true>);
          } else {
            launch(lce_grad_kernel<R, x_layout<R>(), PARTS, BF, false>);
          }
          const bool done = v0 + piece >= p.v;
          if (want_db && nrt > 1 && (!db_late || done)) {
            const long words = db_late ? p.v : vp;
            lce_db_kernel<<<(int)((words + 255) / 256), 256, 0, stream>>>(
                mem.at<float>(o_dbp), nrt, db_ld, words,
                db_late ? db.data_ptr() : db_at, type_code(db));
            HIP_CHECK_KERNEL();
          }
          // as rows of words for dw, as columns of rows for dx
          const Operand g = operand(G, up(vp, 64), ldg, p.np);
          const Operand gx = operand(Gx, up(vp, 64), ldg, p.np);
          if (want_dw) {
            auto run = [&](auto tile) {
              using C = decltype(tile);
              const int mt = (int)((vp + C::BM - 1) / C::BM);
              const int nt = (int)((p.d + C::BN - 1) / C::BN);
              auto kernel = lce_dw_kernel<C, PARTS, BF,
                                          PARTS == 2 ? R::BN : 0>;
              constexpr int lds = C::template lds<1>();
              allow_lds(kernel, lds);
              kernel<<<mt * nt, C::THREADS, lds, stream>>>(
                  g, xr, (int)up(p.n, 64), sc, tinv, piece,
                  static_cast<char*>(dw.data_ptr()) +
                      v0 * p.d * dw.element_size(),
                  p.type, (int)vp, (int)p.d, mt, nt);
              HIP_CHECK_KERNEL();
            };
            // 256 x 256 tiles where they fill three quarters of the CUs and
            // the sum over the rows is long: with dw alone 2,048 rows of 512
            // against 8,192 words (64 tiles) 111 us and 88 with 128 x 128,
            // 24,576 (192) 198 and 197, 32,768 (256) 238 and 250; 256 rows,
            // 100,000 words 144 and 135.  Two parts leave the LDS less time:
            // 2,048 rows 1,068 and 856 us, never less.  64 x 64 for few:
            // 1,024 rows of 256 in fp32 against 6,400 words (25) 95 us and
            // 102 with 128 x 128, 16,384 (64) 178 and 169.
            const long cover = ((vp + 255) / 256) * ((p.dp + 255) / 256);
            if (PARTS == 1 && p.n >= 1024 && cover >= 192 &&
                p.dp % 256 == 0) {
              run(BigOf<PARTS>{});
            } else if (cover >= 48 && p.dp >= 128) {
              run(MidOf<PARTS>{});
            } else {
              run(Small{});
            }
          }
          if (want_dx) {
            auto run = [&](auto tile) {
              using C = decltype(tile);
              const int mt = (int)((p.n + C::BM - 1) / C::BM);
              const int nt = (int)((p.dp + C::BN - 1) / C::BN);
              const int kv = (int)up(vp, 64);
              const int kslice = (int)up((kv + slices - 1) / slices, 64);
              auto kernel = lce_dx_kernel<C, PARTS, BF>;
              constexpr int lds = C::template lds<1>();
              allow_lds(kernel, lds);
              kernel<<<mt * nt * slices, C::THREADS, lds, stream>>>(
                  gx, q.w, kv, kslice, mem.at<float>(o_part), (int)p.n,
                  (int)p.dp, v0 == 0, mt, nt, slices);
              HIP_CHECK_KERNEL();
            };
            if (dx_tile == 128) {
              run(MidOf<PARTS>{});
            } else {
              run(Small{});
            }
          }
        }
      });
    }
    if (want_dx) {
      auto launch = [&](auto kernel, int threads, int at_once) {
        kernel<<<px_grid(p.n * p.d, at_once), threads, 0, stream>>>(
            mem.at<float>(o_part), slices, p.n, (int)p.d, (int)p.dp, sc,
            winv, kx.row.g, dx.data_ptr(), p.type);
        HIP_CHECK_KERNEL();
      };
      if (slices >= 32) {
        launch(lce_dx_sum_kernel<8>, 512, 64);
      } else {
        launch(lce_dx_sum_kernel<1>, 256, 256);
      }
    }
  });
  return {dx, dw, db};
}
