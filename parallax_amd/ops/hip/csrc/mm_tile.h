// A matrix-product tile for kernels that fuse something into the product:
// acc[BM x BN] = sum_k A[m, k] * B[n, k], 16-bit operands (bf16 or fp16),
// fp32 sums, one workgroup per tile.  The kernel that includes this owns
// the grid, the operands' scaling and what becomes of the sums.
//
//   * An operand lies k-contiguous ([rows][K], KROWS), k-strided ([K][rows],
//     KCOLS) or in blocks of 32 k ([K/32][rows][32], KBLOCK).  The first and
//     the third are read from LDS with ds_read_b128, the second with the
//     transposing ds_read_b64_tr_b16, which hands a lane four k of one row,
//     so no operand is ever transposed in memory.  A stage of 32 k takes 64
//     bytes of a k-contiguous row, half of what memory hands out at a time;
//     blocks make that one piece (256 x 128 tile, 2560 x 32768 x 512: 86 us
//     with rows, 74 us with the first operand in blocks).
//   * PARTS = 2 multiplies operands that are split into a high and a low
//     fp16 part (value = hi + lo, 22 bits): lo*hi, hi*lo and hi*hi are added
//     up, the dropped lo*lo is 2^-22 of a product.  Such an operand lies in
//     pairs: each 32 values of a row are 32 high parts and 32 low parts, so
//     a stage is 32 k of both, and three products come of four reads.
//   * Operands go from memory to LDS directly (buffer loads, 16 B a lane)
//     into ST buffers; a wait leaves ST-2 stages in flight, and one barrier
//     a stage both publishes stage k and frees the buffer of stage k-1.
//   * The operands are swapped in the matrix instruction, so a lane holds
//     four neighbouring n of one m: rows reduce over registers and two
//     shuffles, and four results go out in one store.
//
// LDS layouts (16-byte chunks, permuted so that neither read conflicts):
//   KROWS, KBLOCK  [rows][BK]: chunk c of row r at c ^ sw(r).
//   KCOLS  [BK][rows]: 32-byte segment s of row k at s ^ f(k), f from the
//          k bits that differ within one transposing read.
#pragma once

#include "common.h"

namespace mm {

enum { KROWS = 0, KCOLS = 1, KBLOCK = 2 };

typedef __attribute__((ext_vector_type(8))) __bf16 bf8;
typedef __attribute__((ext_vector_type(8))) _Float16 hf8;
typedef __attribute__((ext_vector_type(8))) short s8;
typedef __attribute__((ext_vector_type(4))) short s4;
typedef __attribute__((ext_vector_type(4))) float f4;

template <bool BF>
__device__ __forceinline__ f4 mma(s8 a, s8 b, f4 c) {
  if constexpr (BF) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(
        __builtin_bit_cast(bf8, a), __builtin_bit_cast(bf8, b), c, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(
        __builtin_bit_cast(hf8, a), __builtin_bit_cast(hf8, b), c, 0, 0, 0);
  }
}

// One operand of a product.
//   p        first element
//   ld       elements between rows as they lie (pairs: both parts counted)
//   rows     rows that may be read (KROWS: of the operand, KCOLS: its k);
//            KBLOCK: of a block, a multiple of the tile's
//   cols     KCOLS: operand rows (columns as they lie) that may be read, a
//            multiple of 8, of 32 in pairs
// Reads past `rows` and `cols` are clamped to the last ones.
struct Operand {
  const ushort* p;
  int ld;
  int rows;
  int cols;
};

template <int BM_, int BN_, int WM_, int WN_, int BK_, int ST_>
struct Tile {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_;
  static constexpr int BK = BK_, ST = ST_;
  static constexpr bool TWO_SUM = false;
  static constexpr int WAVES_M = BM / WM, WAVES_N = BN / WN;
  static constexpr int THREADS = 64 * WAVES_M * WAVES_N;
  static constexpr int FM = WM / 16, FN = WN / 16;
  // waves on a SIMD that the registers have to leave room for: two
  // workgroups of four or eight waves on a CU, or one of sixteen
  static constexpr int OCC = THREADS == 1024 ? 4 : THREADS / 128;
  static constexpr int STAGE_BYTES = (BM + BN) * BK * 2;
  // a tile on its way out, of 16-bit values or of pairs of parts: rows 16
  // bytes apart from a bank's, in two goes where 160 KB do not hold it
  static constexpr int OUT_ROW = BN * 2 + 16, PAIR_ROW = BN * 4 + 16;
  static constexpr int PAIR_GOES = BM * PAIR_ROW > 160 * 1024 ? 2 : 1;
  static constexpr int lds_bytes(int out) {
    return ST * STAGE_BYTES > out ? ST * STAGE_BYTES : out;
  }
  template <int PARTS>
  static constexpr int lds() {
    return lds_bytes(PARTS == 2 ? BM * PAIR_ROW / PAIR_GOES : BM * OUT_ROW);
  }
};

template <int BK>
__device__ __forceinline__ int row_swizzle(int r) {
  return BK == 32 ? ((-(r >> 2)) & 3) : BK == 64 ? (r & 7) : (r & 15);
}

template <int R>
__device__ __forceinline__ int col_swizzle(int k) {
  if constexpr (R == 32) {
    return (k >> 3) & 1;
  } else if constexpr (R == 64) {
    return ((k >> 1) & 1) | (((k >> 3) & 1) << 1);
  } else {
    return (k & 3) | (((k >> 3) & 1) << 2);
  }
}

// Copies one operand's [R x BK] piece of a stage into LDS.
template <int R, int L, int BK, int THREADS, int PARTS>
struct Stager {
  static constexpr int PER = R * BK * 2 / 16 / THREADS;
  static_assert(PER >= 1 && PER * THREADS * 16 == R * BK * 2,
                "a stage has to be whole 16-byte pieces for every thread");
  static_assert(PARTS == 1 || BK >= 64, "pairs of 32");
  __amdgpu_buffer_rsrc_t rs;
  int off[PER];    // KROWS: byte offset; KCOLS: column byte offset
  int ld2;
  int rows;

  __device__ __forceinline__ void init(const Operand& o, int r0) {
    ld2 = o.ld * 2;
    rows = o.rows;
    const ushort* base = o.p + (L == KROWS ? (long)r0 * o.ld
                                : L == KCOLS ? (long)r0 * PARTS : 0L);
    const long left = (L == KROWS ? (long)(o.rows - r0) : (long)o.rows) * ld2;
    const int bytes = (int)(left < 0x7fffffffL ? left : 0x7fffffffL);
    rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<ushort*>(base), 0,
                                           bytes, 0x00027000);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int c = threadIdx.x + i * THREADS;
      if constexpr (L == KBLOCK) {
        static_assert(L != KBLOCK || (BK == 32 && PARTS == 1),
                      "blocks of 32 k");
        const int r = c / 4;
        off[i] = (r0 + r) * 64 + (((c % 4) ^ row_swizzle<BK>(r)) * 16);
      } else if constexpr (L == KROWS) {
        constexpr int S = BK / 8;
        int r = c / S;
        const int src = (c % S) ^ row_swizzle<BK>(r);
        if (r > o.rows - 1 - r0) r = o.rows - 1 - r0;
        off[i] = r * ld2 + src * 16;
      } else {
        constexpr int S = R / 8;
        const int k = c / S;
        const int src = (c % S) ^ (col_swizzle<R>(k) << 1);
        int col = src * 8;
        if (col > o.cols - 8 - r0) col = o.cols - 8 - r0;
        off[i] = PARTS == 2
                     ? ((col >> 5) * 64 + (col & 31) + (k & 32)) * 2
                     : col * 2;
      }
    }
  }

  // the stage that starts at k0
  __device__ __forceinline__ void load(char* lds, int k0) const {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      int v;
      if constexpr (L == KBLOCK) {
        v = off[i] + k0 * 2 * rows;
      } else if constexpr (L == KROWS) {
        v = off[i] + k0 * 2 * PARTS;
      } else {
        int k = (threadIdx.x + i * THREADS) / (R / 8);
        k = (PARTS == 2 ? (k >> 6) * 32 + (k & 31) : k) + k0;
        if (k > rows - 1) k = rows - 1;
        v = off[i] + k * ld2;
      }
      // each wave writes 1 KiB in lane order from its own base
      char* dst = lds + i * THREADS * 16 + (threadIdx.x & ~63) * 16;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rs, (__attribute__((address_space(3))) void*)dst, 16, v, 0, 0, 0);
    }
  }
};

// The transposing read.  The compiler knows nothing of its operand and would
// wait for all loads into LDS before it, also those of the next stage; the
// restrict gives it the alias information that keeps it from that.  The
// waits that are needed stand in product().
typedef __attribute__((address_space(3))) s4 lds_s4;
__device__ __forceinline__ s4 read_transposed(lds_s4* __restrict__ p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16(p);
}

template <int R, int L, int BK>
__device__ __forceinline__ s8 frag(const char* lds, int r, int kk,
                                   int lane) {
  if constexpr (L != KCOLS) {
    const int row = r + (lane & 15);
    const int c = (kk * 4 + (lane >> 4)) ^ row_swizzle<BK>(row);
    return *reinterpret_cast<const s8*>(lds + row * (BK * 2) + c * 16);
  } else {
    const int i = lane & 15;
    const int k = kk * 32 + (lane >> 4) * 8 + (i >> 2);
    const int seg = (r >> 4) ^ col_swizzle<R>(k);
    const char* at = lds + k * (R * 2) + seg * 32 + (i & 3) * 8;
    const s4 u = read_transposed((lds_s4*)at);
    const s4 v = read_transposed((lds_s4*)(at + 4 * R * 2));
    return __builtin_shufflevector(u, v, 0, 1, 2, 3, 4, 5, 6, 7);
  }
}

template <int N>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// What a wave has read from LDS has arrived before it lets others write
// there: the compiler puts no such wait before a barrier, and whether the
// products that need the values stand before it is up to its scheduling.
__device__ __forceinline__ void barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Takes the sums over the whole of k as they are.
struct Whole {
  static constexpr int EVERY = 0;
};

// acc[i][j] of wave (wm, wn): element (m, n) with
//   m = m0 + wm + i*16 + (lane & 15), n = n0 + wn + j*16 + (lane>>4)*4 + r.
// k runs over [k0, k1), both multiples of BK, of BK / 2 in pairs.  `take`
// with EVERY > 0 is given the sums so far behind every so many stages and
// the last one, and leaves acc as they shall go on.
template <class C, int AL, int BL, int PARTS, bool BF, class F = Whole>
__device__ __forceinline__ void product(char* lds, const Operand& a, int m0,
                                        const Operand& b, int n0, int k0,
                                        int k1, f4 (&acc)[C::FM][C::FN],
                                        F take = F()) {
  constexpr int BK = C::BK, ST = C::ST, T = C::THREADS;
  constexpr int STEP = BK / PARTS;
  Stager<C::BM, AL, BK, T, PARTS> sa;
  Stager<C::BN, BL, BK, T, PARTS> sb;
  sa.init(a, m0);
  sb.init(b, n0);
  constexpr int LOADS = sa.PER + sb.PER;
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  const int wm = (wave / C::WAVES_N) * C::WM;
  const int wn = (wave % C::WAVES_N) * C::WN;
  const int total = (k1 - k0) / STEP;

  int lbuf = 0;  // where the next stage goes
  auto stage = [&](int t) {
    char* at = lds + lbuf * C::STAGE_BYTES;
    sa.load(at, k0 + t * STEP);
    sb.load(at + C::BM * BK * 2, k0 + t * STEP);
    lbuf = lbuf + 1 == ST ? 0 : lbuf + 1;
  };
  auto multiply = [&](const s8 (&fa)[C::FM], const s8 (&fb)[C::FN],
                      f4 (&sum)[C::FM][C::FN]) {
#pragma unroll
    for (int i = 0; i < C::FM; ++i)
#pragma unroll
      for (int j = 0; j < C::FN; ++j)
        sum[i][j] = mma<BF>(fb[j], fa[i], sum[i][j]);
  };
  // Small tiles have registers to add up what is 2^-12 of the rest apart:
  // the large sums are then rounded a third as often.  TWO_SUM: each stage's
  // sum goes to the total by a two-sum, whose error is added up as well.
  constexpr bool APART = PARTS == 2 && C::FM * C::FN <= 4;
  constexpr bool EXACT = PARTS == 2 && C::TWO_SUM;
  f4 low[APART ? C::FM : 1][APART ? C::FN : 1] = {};
  auto multiply_low = [&](const s8 (&fa)[C::FM], const s8 (&fb)[C::FN]) {
    if constexpr (APART) {
      multiply(fa, fb, low);
    } else {
      multiply(fa, fb, acc);
    }
  };
  auto stage_of_pairs = [&](auto read_a, auto read_b) {
#pragma unroll
    for (int kk = 0; kk < BK / 32; kk += 2) {
      s8 ah[C::FM], al[C::FM], bh[C::FN], bl[C::FN];
      read_b(bh, kk);
      read_a(al, kk + 1);
      multiply_low(al, bh);
      read_a(ah, kk);
      multiply(ah, bh, acc);
      read_b(bl, kk + 1);
      multiply_low(ah, bl);
    }
  };

#pragma unroll
  for (int s = 0; s < ST - 1; ++s) {
    if (s < total) stage(s);
  }
  int buf = 0;
  for (int t = 0; t < total; ++t) {
    if (t + ST - 1 <= total) {
      wait_loads<(ST - 2) * LOADS>();
    } else {
      wait_loads<0>();
    }
    barrier();
    if (t + ST - 1 < total) stage(t + ST - 1);
    const char* pa = lds + buf * C::STAGE_BYTES;
    const char* pb = pa + C::BM * BK * 2;
    buf = buf + 1 == ST ? 0 : buf + 1;
    auto read_a = [&](s8 (&f)[C::FM], int kk) {
#pragma unroll
      for (int i = 0; i < C::FM; ++i)
        f[i] = frag<C::BM, AL, BK>(pa, wm + i * 16, kk, lane);
    };
    auto read_b = [&](s8 (&f)[C::FN], int kk) {
#pragma unroll
      for (int j = 0; j < C::FN; ++j)
        f[j] = frag<C::BN, BL, BK>(pb, wn + j * 16, kk, lane);
    };
    if constexpr (EXACT) {
      const f4 t = acc[0][0];
      acc[0][0] = f4{0.f, 0.f, 0.f, 0.f};
      stage_of_pairs(read_a, read_b);
      const f4 v = acc[0][0], sum = t + v, v1 = sum - t;
      low[0][0] += (t - (sum - v1)) + (v - v1);
      acc[0][0] = sum;
    } else if constexpr (PARTS == 2) {
      stage_of_pairs(read_a, read_b);
    } else {
#pragma unroll
      for (int kk = 0; kk < BK / 32; ++kk) {
        s8 fa[C::FM], fb[C::FN];
        read_b(fb, kk);
        read_a(fa, kk);
        multiply(fa, fb, acc);
      }
    }
    if constexpr (F::EVERY > 0) {
      if (t % F::EVERY == F::EVERY - 1 || t + 1 == total) {
        if constexpr (APART) {
#pragma unroll
          for (int i = 0; i < C::FM; ++i)
#pragma unroll
            for (int j = 0; j < C::FN; ++j) {
              acc[i][j] += low[i][j];
              low[i][j] = f4{0.f, 0.f, 0.f, 0.f};
            }
        }
        take();
      }
    }
  }
  if constexpr (APART && F::EVERY == 0) {
#pragma unroll
    for (int i = 0; i < C::FM; ++i)
#pragma unroll
      for (int j = 0; j < C::FN; ++j) acc[i][j] += low[i][j];
  }
  barrier();  // the caller may use the LDS
}

// hi/lo fp16 parts of a value
__device__ __forceinline__ void split(float v, ushort& hi, ushort& lo) {
  const _Float16 h = (_Float16)v;
  const _Float16 l = (_Float16)(v - (float)h);
  hi = __builtin_bit_cast(ushort, h);
  lo = __builtin_bit_cast(ushort, l);
}

__device__ __forceinline__ float half_bits(ushort h) {
  return (float)__builtin_bit_cast(_Float16, h);
}

// Writes a tile of 16-bit values, through LDS so that a row goes out in one
// piece: value(i, j) gives the four values of fragment (i, j) of this lane.
// Rows and columns from `rows` and `cols` on are left out; `out` and `ld` are
// multiples of 8 elements, and so is cols unless the tile is cut there.
template <class C, typename F>
__device__ __forceinline__ void store_tile(char* lds, ushort* out, long ld,
                                           int rows, int cols, F value) {
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  const int wm = (wave / C::WAVES_N) * C::WM;
  const int wn = (wave % C::WAVES_N) * C::WN;
#pragma unroll
  for (int i = 0; i < C::FM; ++i)
#pragma unroll
    for (int j = 0; j < C::FN; ++j)
      *reinterpret_cast<ushort4*>(
          lds + (wm + i * 16 + (lane & 15)) * C::OUT_ROW +
          (wn + j * 16 + (lane >> 4) * 4) * 2) = value(i, j);
  __syncthreads();
  constexpr int PER_ROW = C::BN / 8;
#pragma unroll 4
  for (int c = threadIdx.x; c < C::BM * PER_ROW; c += C::THREADS) {
    const int r = c / PER_ROW, q = (c % PER_ROW) * 8;
    if (r >= rows || q >= cols) continue;
    const s8 v = *reinterpret_cast<const s8*>(lds + r * C::OUT_ROW + q * 2);
    if (q + 8 <= cols) {
      *reinterpret_cast<s8*>(out + r * ld + q) = v;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (q + e < cols) out[r * ld + q + e] = (ushort)v[e];
    }
  }
}

// The same for values in pairs of parts: value(i, j) in fp32, scaled; `out`
// is at a multiple of 32 values, `ld` counts both parts, all is written.
template <class C, typename F>
__device__ __forceinline__ void store_pairs(char* lds, ushort* out, long ld,
                                            F value) {
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  const int wm = (wave / C::WAVES_N) * C::WM;
  const int wn = (wave % C::WAVES_N) * C::WN;
  constexpr int HALF = C::BM / C::PAIR_GOES, PER_ROW = C::BN / 4;
#pragma unroll
  for (int go = 0; go < C::PAIR_GOES; ++go) {
    if (go) __syncthreads();
    if (wm / HALF == go) {
#pragma unroll
      for (int i = 0; i < C::FM; ++i)
#pragma unroll
        for (int j = 0; j < C::FN; ++j) {
          const f4 v = value(i, j);
          ushort h[4], l[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) split(v[r], h[r], l[r]);
          const int n = wn + j * 16 + (lane >> 4) * 4;
          char* at = lds + (wm % HALF + i * 16 + (lane & 15)) * C::PAIR_ROW +
                     ((n >> 5) * 64 + (n & 31)) * 2;
          *reinterpret_cast<ushort4*>(at) =
              make_ushort4(h[0], h[1], h[2], h[3]);
          *reinterpret_cast<ushort4*>(at + 64) =
              make_ushort4(l[0], l[1], l[2], l[3]);
        }
    }
    __syncthreads();
#pragma unroll 4
    for (int c = threadIdx.x; c < HALF * PER_ROW; c += C::THREADS) {
      const int r = c / PER_ROW, q = (c % PER_ROW) * 8;
      *reinterpret_cast<s8*>(out + (go * HALF + r) * ld + q) =
          *reinterpret_cast<const s8*>(lds + r * C::PAIR_ROW + q * 2);
    }
  }
}

// Spreads a flat block id over the 8 dies so that each die works on one
// contiguous range of tiles: neighbours then share operands in its L2.
__device__ __forceinline__ int die_contiguous(int bid, int n) {
  const int q = n / 8, r = n % 8;
  const int die = bid % 8, pos = bid / 8;
  return (die < r ? die * (q + 1) : r * (q + 1) + (die - r) * q) + pos;
}

}  // namespace mm
