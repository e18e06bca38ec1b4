// Hand-written CDNA4 MFMA GEMM: C[M,N] = A[M,K] @ B[N,K]^T, bf16 in /
// bf16 out, fp32 accumulate.  The building block for the NHWC conv path
// (a 1x1 convolution IS this GEMM with A = activations [N*H*W, Cin] and
// B = weights [Cout, Cin]) and for framework-owned projection GEMMs.
//
// Structure (guide cdna_hip_programming.md §5, the LDS-staged ladder):
//   * 128x128 output tile per 256-thread block (4 waves, each a 64x64
//     sub-tile of 4x4 mfma_f32_16x16x32_bf16 fragments, 64 fp32 acc
//     VGPRs/lane);
//   * BK=64 K-step, both operand tiles staged to LDS by
//     global_load_lds_dwordx4 (16 B/lane direct-to-LDS DMA), double
//     buffered;
//   * XOR swizzle byte^=((row&7)<<4) against ds_read_b128 bank conflicts
//     (guide G4/T2) applied on the glds SOURCE address + the LDS read
//     (rule 21: the destination stays lane-linear);
//   * 2-phase schedule: issue next tile's DMA, compute current from LDS
//     behind s_setprio(1) (T3 minimum form + T5);
//   * XCD-aware bijective block swizzle (T1) for L2 locality.
// Both operands are K-major (B passed TRANSPOSED, i.e. [N,K] row-major,
// the natural layout of torch Linear/conv weights), so every MFMA
// fragment is 8 contiguous bf16 per lane.

#include <torch/extension.h>
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>

#include "common.h"

typedef __attribute__((ext_vector_type(8))) short bf16x8;
typedef __attribute__((ext_vector_type(4))) float f32x4;

#define BM 128
#define BN 128
#define BK 64
#define PXG_THREADS 256

// LDS tile: [128 rows][64 k] bf16 = 16 KiB; byte row stride 128.
// swizzle: byte ^= ((row & 7) << 4)   (16-byte granularity, involution)
__device__ __forceinline__ int swz(int row, int kbyte) {
  return row * (BK * 2) + (kbyte ^ ((row & 7) << 4));
}

// Cadd: optional bf16 addend with arbitrary row stride (elements),
// fused into the epilogue (the addmm beta=1 case: gates = gx[:,t] + h@W).
__global__ __launch_bounds__(PXG_THREADS, 2)
void pxgemm_bt_kernel(const ushort* __restrict__ A,
                      const ushort* __restrict__ B,
                      ushort* __restrict__ C, long M, long N, long K,
                      int nbm, int nbn, const ushort* __restrict__ Cadd,
                      long add_rstride) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  // [2 buffers][A|B][16 KiB]
#define LDSA(b) (smem + (b) * 32768)
#define LDSB(b) (smem + (b) * 32768 + 16384)

  // XCD-aware bijective remap of the flat block id (guide T1)
  int bid = blockIdx.x;
  {
    const int nwg = nbm * nbn;
    const int q = nwg / 8, r = nwg % 8;
    const int xcd = bid % 8, pos = bid / 8;
    bid = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + pos;
  }
  const int bm = (bid / nbn) * BM;
  const int bn = (bid % nbn) * BN;

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = tid >> 6;
  // wave grid 2x2: each wave owns a 64x64 sub-tile
  const int wm = (wave >> 1) * 64;
  const int wn = (wave & 1) * 64;
  const int fr = lane & 15;        // fragment row/col within 16
  const int ko = (lane >> 4) * 8;  // fragment k offset (8 bf16)

  f32x4 acc[4][4] = {};

  // ---- glds staging: each thread DMAs 16 B per instruction; a 16 KiB
  // tile needs 4 instructions.  LDS dest is lane-linear
  // (base + flat_byte), source address carries the inverse swizzle.
  const long a_row0 = bm, b_row0 = bn;
  // flat element position for this thread's i-th piece:
  //   byte p = (tid + i*256) * 16 ; row = p / 128 ; kbyte = p % 128
  int p_row[4], p_kb[4];
  long a_src_row[4], b_src_row[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int p = (tid + i * PXG_THREADS) * 16;
    p_row[i] = p / (BK * 2);
    p_kb[i] = (p % (BK * 2)) ^ ((p_row[i] & 7) << 4);  // inverse swizzle
    // edge tiles: clamp out-of-range source rows to the last valid row —
    // the stale fragments they produce are discarded by the guarded
    // epilogue stores, so NO host-side padding copies are needed
    long ar = a_row0 + p_row[i];
    long br = b_row0 + p_row[i];
    a_src_row[i] = ar < M ? ar : M - 1;
    b_src_row[i] = br < N ? br : N - 1;
  }

  const int ktiles = (int)(K / BK);

#define STAGE(buf, kt)                                                    \
  do {                                                                     \
    const long kbase = (long)(kt) * BK;                                    \
    _Pragma("unroll") for (int i = 0; i < 4; ++i) {                        \
      const ushort* srcA = A + a_src_row[i] * K + kbase +                  \
                           (p_kb[i] >> 1);                                 \
      const ushort* srcB = B + b_src_row[i] * K + kbase +                  \
                           (p_kb[i] >> 1);                                 \
      __builtin_amdgcn_global_load_lds(                                    \
          (const __attribute__((address_space(1))) void*)srcA,             \
          (__attribute__((address_space(3))) void*)(LDSA(buf) +            \
                                                    (tid + i * 256) * 16), \
          16, 0, 0);                                                       \
      __builtin_amdgcn_global_load_lds(                                    \
          (const __attribute__((address_space(1))) void*)srcB,             \
          (__attribute__((address_space(3))) void*)(LDSB(buf) +            \
                                                    (tid + i * 256) * 16), \
          16, 0, 0);                                                       \
    }                                                                      \
  } while (0)

  STAGE(0, 0);
  __builtin_amdgcn_s_waitcnt(/*vmcnt(0) lgkmcnt(0)*/ 0);
  __builtin_amdgcn_s_barrier();

  int cur = 0;
  for (int kt = 0; kt < ktiles; ++kt) {
    if (kt + 1 < ktiles) {
      STAGE(cur ^ 1, kt + 1);
    }
    // compute current tile from LDS
#pragma unroll
    for (int kk = 0; kk < BK / 32; ++kk) {
      bf16x8 a_frag[4], b_frag[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int ar = wm + i * 16 + fr;
        a_frag[i] = *(const bf16x8*)(LDSA(cur) +
                                     swz(ar, (kk * 32 + ko) * 2));
        const int br = wn + i * 16 + fr;
        b_frag[i] = *(const bf16x8*)(LDSB(cur) +
                                     swz(br, (kk * 32 + ko) * 2));
      }
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              a_frag[i], b_frag[j], acc[i][j], 0, 0, 0);
        }
      }
      __builtin_amdgcn_s_setprio(0);
    }
    // drain this iteration's DMA and cross the barrier
    __builtin_amdgcn_s_waitcnt(0);
    __builtin_amdgcn_s_barrier();
    cur ^= 1;
  }

  // ---- epilogue: C/D fragment map for 16x16x32: col = lane&15,
  // row = (lane>>4)*4 + reg (guide §3); bf16 convert + store
  const int crow0 = (lane >> 4) * 4;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const long row = bm + wm + i * 16 + crow0 + r;
        const long col = bn + wn + j * 16 + fr;
        if (row >= M || col >= N) continue;
        float fv = acc[i][j][r];
        if (Cadd != nullptr) {
          __hip_bfloat16 av =
              *reinterpret_cast<const __hip_bfloat16*>(
                  &Cadd[row * add_rstride + col]);
          fv += __bfloat162float(av);
        }
        __hip_bfloat16 v = __float2bfloat16(fv);
        C[row * N + col] = *reinterpret_cast<ushort*>(&v);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// 8-phase 256x256 deep-pipelined MFMA GEMM (guide cdna_hip_programming.md
// §5 "The 256² 8-phase template"): C[M,N] = A[M,K] @ B[N,K]^T, bf16.
//
//   * 256x256 tile, BK=64, 8 waves (2M x 4N), per-wave output 128x64
//     (acc[8][4] f32x4 = 128 VGPRs);
//   * LDS 128 KiB: 2 buffers x (A 32 KiB + B 32 KiB), each operand tile
//     [2 k-half][256 rows][32 k] bf16 with a 16-B-slot XOR swizzle
//     q ^= (-(row>>2))&3 (verified conflict-free against the
//     ds_read_b128 4x16 lane groups; involution, so the same XOR is the
//     glds source permutation — rule 21);
//   * 4 phases per K-tile: (k-half, n-half) quadrants of 16 MFMAs each;
//     every phase issues 2 global_load_lds_dwordx4 staging the NEXT
//     K-tile (each wave stages its own 2 A + 2 B 1-KiB pieces per
//     k-half), so a full K-tile is always in flight;
//   * counted s_waitcnt vmcnt(4) only at phases 2 and 4 of each K-tile
//     (never 0 in the main loop — T4), raw s_barrier (never
//     __syncthreads: an in-flight glds would be drained — §5
//     "Pipelining across barriers"), s_setprio(1) around the MFMA
//     cluster (T5), XCD-aware bijective block remap (T1).
// ---------------------------------------------------------------------------

#define P8_BM 256
#define P8_BN 256
#define P8_THREADS 512

// LDS geometry: buffer b at b*65536; A at +0, B at +32768;
// k-half kh at +kh*16384; row r occupies 64 B; 16-B slot q at
// (q ^ ((-(r>>2))&3)) * 16.
#define P8_LDSA(b) (smem + (b) * 65536)
#define P8_LDSB(b) (smem + (b) * 65536 + 32768)

// Two-level XCD-aware super-tile block remap.  The plain per-XCD stripe
// remap (T1) makes the ~256 concurrent blocks an 8-row x nbn stripe:
// at 8192^3 that is 128 MB of distinct B panels live at once, nothing
// fits in L2 or L3, and the kernel devolves to streaming 8 GB from HBM
// (measured: 1.24 ms = bytes / 6.3 TB/s exactly).  Here each XCD owns
// ONE n-column at a time (its B panel lives in its private L2) and the
// concurrent super-tile is SM m-rows x 8 n-cols, whose A panels are
// shared across XCDs through L3.  Requires nbn % 8 == 0; callers fall
// back to the stripe remap otherwise.
__device__ __forceinline__ void p8_supertile_remap(
    int bid, int nbm, int nbn, int* bm_out, int* bn_out) {
  const int SM = 16;                  // super-tile height (m-tiles)
  const int xcd = bid % 8;
  const int pos = bid / 8;            // sequential index within the XCD
  const int ncol = nbn / 8;           // n-columns owned by each XCD
  const int full_sr = nbm / SM;
  const int per_sr = SM * ncol;
  int sr, c, m_in;
  if (pos < full_sr * per_sr) {
    sr = pos / per_sr;
    const int w = pos - sr * per_sr;
    c = w / SM;
    m_in = w - c * SM;
  } else {                            // ragged last super-row
    const int rem_m = nbm - full_sr * SM;
    const int w = pos - full_sr * per_sr;
    c = w / rem_m;
    m_in = w - c * rem_m;
    sr = full_sr;
  }
  *bm_out = sr * SM + m_in;
  *bn_out = c * 8 + xcd;
}

template <int V>
__global__ __launch_bounds__(P8_THREADS, 2)
void pxgemm8_bt_kernel(const ushort* __restrict__ A,
                       const ushort* __restrict__ B,
                       ushort* __restrict__ C, long M, long N, long K,
                       int nbm, int nbn, const ushort* __restrict__ Cadd,
                       long add_rstride) {
  extern __shared__ __attribute__((aligned(16))) char smem[];

  int bmt, bnt;
  if (nbn % 8 == 0 && nbm * nbn >= 64) {
    p8_supertile_remap(blockIdx.x, nbm, nbn, &bmt, &bnt);
  } else {
    int bid = blockIdx.x;
    const int nwg = nbm * nbn;
    const int q = nwg / 8, r = nwg % 8;
    const int xcd = bid % 8, pos = bid / 8;
    bid = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + pos;
    bmt = bid / nbn;
    bnt = bid % nbn;
  }
  const long bm = (long)bmt * P8_BM;
  const long bn = (long)bnt * P8_BN;

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = tid >> 6;        // 0..7
  const int wm = (wave >> 2) * 128; // 2 M groups
  const int wn = (wave & 3) * 64;   // 4 N groups
  const int fr = lane & 15;         // fragment row within 16
  const int fq = lane >> 4;         // fragment 16-B slot (k 8-group)

  f32x4 acc[8][4] = {};

  // ---- staging constants (per lane) -----------------------------------
  // Each wave stages, per k-half, its two 1-KiB pieces of A (LDS rows
  // pi*16..pi*16+15, pi in {wave, wave+8}) and the same two of B.
  // lane covers LDS row pi*16 + (lane>>2), slot (lane&3); the glds
  // source column carries the inverse (== same) swizzle.
  const int srow = lane >> 2;                       // 0..15 within piece
  const int sq = (lane & 3) ^ ((-(lane >> 4)) & 3); // swizzled src slot
  // global rows for piece 0 (pi=wave) and piece 1 (pi=wave+8):
  long arow0 = bm + wave * 16 + srow;
  long arow1 = arow0 + 128;
  long brow0 = bn + wave * 16 + srow;
  long brow1 = brow0 + 128;
  if (arow0 >= M) arow0 = M - 1;  // clamped edge reads; stale fragments
  if (arow1 >= M) arow1 = M - 1;  // are discarded by the guarded stores
  if (brow0 >= N) brow0 = N - 1;
  if (brow1 >= N) brow1 = N - 1;
  // bake per-lane base pointers once: the per-stage address is then a
  // single add of the wave-uniform k offset (no 64-bit mult in the loop)
  const ushort* aptr0 = A + arow0 * K + sq * 8;
  const ushort* aptr1 = A + arow1 * K + sq * 8;
  const ushort* bptr0 = B + brow0 * K + sq * 8;
  const ushort* bptr1 = B + brow1 * K + sq * 8;
  // LDS byte destinations (lane-linear within the piece):
  const int a_dst0 = wave * 1024 + lane * 16;          // + kh*16384
  const int a_dst1 = (wave + 8) * 1024 + lane * 16;
  const int ktiles = (int)(K / BK);

  // one piece: operand base, global row, k element offset, LDS dest
#define P8_STAGE(gptr, kelem, buf, lds_off, bsel)                          \
  __builtin_amdgcn_global_load_lds(                                        \
      (const __attribute__((address_space(1))) void*)((gptr) + (kelem)),   \
      (__attribute__((address_space(3))) void*)(                           \
          (bsel ? P8_LDSB(buf) : P8_LDSA(buf)) + (lds_off)),               \
      16, 0, 0)

  // stage phase ph (0..3) of K-tile kt into buffer (kt&1)
#define P8_STAGE_PHASE(kt, ph)                                             \
  do {                                                                     \
    const int _b = (kt) & 1;                                               \
    const long _kb = (long)(kt) * BK + ((ph) >> 1) * 32;                   \
    const int _kh_off = ((ph) >> 1) * 16384;                               \
    if (((ph) & 1) == 0) {                                                 \
      P8_STAGE(aptr0, _kb, _b, _kh_off + a_dst0, 0);                       \
      P8_STAGE(bptr0, _kb, _b, _kh_off + a_dst0, 1);                       \
    } else {                                                               \
      P8_STAGE(aptr1, _kb, _b, _kh_off + a_dst1, 0);                       \
      P8_STAGE(bptr1, _kb, _b, _kh_off + a_dst1, 1);                       \
    }                                                                      \
  } while (0)

  // ---- fragment read addressing ---------------------------------------
  // a_frag[i]: LDS row wm + i*16 + fr of k-half kh, slot fq ^ f(row);
  // f(row) = (-(row>>2))&3 and (wm+i*16)>>2 is 0 mod 4, so the XOR is
  // the per-lane constant (-(fr>>2))&3.
  const int rswz = ((-(fr >> 2)) & 3) ^ fq;  // swizzled slot for reads

#define P8_AFRAG(kh, i)                                                    \
  (*(const bf16x8*)(P8_LDSA(cur) + (kh) * 16384 +                          \
                    (wm + (i) * 16 + fr) * 64 + rswz * 16))
#define P8_BFRAG(kh, nh, jj)                                               \
  (*(const bf16x8*)(P8_LDSB(cur) + (kh) * 16384 +                          \
                    (wn + (nh) * 32 + (jj) * 16 + fr) * 64 + rswz * 16))

  // prologue: stage all of K-tile 0, publish its first k-half
  P8_STAGE_PHASE(0, 0);
  P8_STAGE_PHASE(0, 1);
  P8_STAGE_PHASE(0, 2);
  P8_STAGE_PHASE(0, 3);
  asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
  __builtin_amdgcn_s_barrier();

  int cur = 0;
  // ---- main loop: one iteration = one K-tile = 4 phases ---------------
  // phase (kh, nh): ds_read frags -> stage next tile's phase -> [vmcnt]
  // -> barrier -> MFMA quadrant. vmcnt(4) at phases 1 and 3 publishes
  // the k-half the NEXT phase pair will read.
#define P8_PHASE(kh, nh, DO_STAGE, kt, WAITN)                              \
  do {                                                                     \
    bf16x8 b_frag[2];                                                      \
    if ((nh) == 0) {                                                       \
      _Pragma("unroll") for (int i = 0; i < 8; ++i)                        \
          a_frag[i] = P8_AFRAG(kh, i);                                     \
    }                                                                      \
    b_frag[0] = P8_BFRAG(kh, nh, 0);                                       \
    b_frag[1] = P8_BFRAG(kh, nh, 1);                                       \
    if (DO_STAGE) P8_STAGE_PHASE((kt) + 1, (kh) * 2 + (nh));               \
    if ((WAITN) == 0) {                                                    \
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");                     \
    } else if ((WAITN) > 0) {                                              \
      asm volatile("s_waitcnt vmcnt(4)" ::: "memory");                     \
    }                                                                      \
    __builtin_amdgcn_s_barrier();                                          \
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");                     \
    __builtin_amdgcn_sched_barrier(0);                                     \
    __builtin_amdgcn_s_setprio(1);                                         \
    _Pragma("unroll") for (int i = 0; i < 8; ++i) {                        \
      acc[i][(nh) * 2] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(          \
          a_frag[i], b_frag[0], acc[i][(nh) * 2], 0, 0, 0);                \
      acc[i][(nh) * 2 + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(      \
          a_frag[i], b_frag[1], acc[i][(nh) * 2 + 1], 0, 0, 0);            \
    }                                                                      \
    __builtin_amdgcn_s_setprio(0);                                         \
    __builtin_amdgcn_s_barrier();                                          \
  } while (0)

  // merged variant: one barrier pair per k-half (12 ds_reads + 4 glds +
  // 32 MFMAs per phase, 4 barriers per K-tile instead of 8)
#define P8_PHASE_M(kh, DO_STAGE, kt, WAITN)                                \
  do {                                                                     \
    bf16x8 b_frag[4];                                                      \
    _Pragma("unroll") for (int i = 0; i < 8; ++i)                          \
        a_frag[i] = P8_AFRAG(kh, i);                                       \
    b_frag[0] = P8_BFRAG(kh, 0, 0);                                        \
    b_frag[1] = P8_BFRAG(kh, 0, 1);                                        \
    b_frag[2] = P8_BFRAG(kh, 1, 0);                                        \
    b_frag[3] = P8_BFRAG(kh, 1, 1);                                        \
    if (DO_STAGE) {                                                        \
      P8_STAGE_PHASE((kt) + 1, (kh) * 2);                                  \
      P8_STAGE_PHASE((kt) + 1, (kh) * 2 + 1);                              \
    }                                                                      \
    if ((WAITN) == 0) {                                                    \
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");                     \
    } else if ((WAITN) > 0) {                                              \
      asm volatile("s_waitcnt vmcnt(4)" ::: "memory");                     \
    }                                                                      \
    __builtin_amdgcn_s_barrier();                                          \
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");                     \
    __builtin_amdgcn_sched_barrier(0);                                     \
    __builtin_amdgcn_s_setprio(1);                                         \
    _Pragma("unroll") for (int i = 0; i < 8; ++i) {                        \
      _Pragma("unroll") for (int j = 0; j < 4; ++j) {                      \
        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(               \
            a_frag[i], b_frag[j], acc[i][j], 0, 0, 0);                     \
      }                                                                    \
    }                                                                      \
    __builtin_amdgcn_s_setprio(0);                                         \
    __builtin_amdgcn_s_barrier();                                          \
  } while (0)

  bf16x8 a_frag[8];
  if (V == 2 || V == 3) {
    // ---- software-pipelined fragment reads (one phase ahead) --------
    // Phase quadrant = (k-half, m-half): B fragments are read once per
    // k-half (4 regs per set), A alternates between two 4-frag banks
    // with a static period-2 pattern, so every phase's MFMA window
    // contains only the 16 MFMAs plus the issue of the NEXT phase's
    // ds_reads (their latency hides under the MFMAs).  The
    // barrier-to-barrier critical path is the MFMA cluster itself.
    bf16x8 a0[4], a1[4], b0[4], b1[4];
#define P8_RD_A4(bank, kh, ilo)                                            \
    _Pragma("unroll") for (int i = 0; i < 4; ++i)                          \
        bank[i] = P8_AFRAG(kh, (ilo) + i)
#define P8_RD_B4(bank, kh)                                                 \
    _Pragma("unroll") for (int j = 0; j < 4; ++j)                          \
        bank[j] = P8_BFRAG(kh, (j) >> 1, (j) & 1)
#define P8_MM4(abank, bbank, mh)                                           \
    __builtin_amdgcn_s_setprio(1);                                         \
    _Pragma("unroll") for (int i = 0; i < 4; ++i) {                        \
      _Pragma("unroll") for (int j = 0; j < 4; ++j) {                      \
        acc[(mh) * 4 + i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(    \
            abank[i], bbank[j], acc[(mh) * 4 + i][j], 0, 0, 0);            \
      }                                                                    \
    }                                                                      \
    __builtin_amdgcn_s_setprio(0)

    // prologue reads: tile-0 k-half-0 first A bank + B set
    P8_RD_A4(a0, 0, 0);
    P8_RD_B4(b0, 0);
    if (V == 3) {
      // single barrier per phase: the stage moves AFTER the barrier
      // (so the previous phase's LDS reads are collectively retired
      // before any wave's DMA can overwrite the old buffer), halving
      // the barrier count; counted waits shrink to vmcnt(2)
      for (int kt = 0; kt < ktiles; ++kt) {
        const bool last = (kt == ktiles - 1);
        // P1 (kh0, mh0)
        __builtin_amdgcn_s_barrier();
        if (!last) P8_STAGE_PHASE(kt + 1, 0);
        P8_RD_A4(a1, 0, 4);
        P8_MM4(a0, b0, 0);
        // P2 (kh0, mh1): publish kh1
        if (!last) {
          asm volatile("s_waitcnt vmcnt(2)" ::: "memory");
        } else {
          asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
        __builtin_amdgcn_s_barrier();
        if (!last) P8_STAGE_PHASE(kt + 1, 1);
        P8_RD_A4(a0, 1, 0);
        P8_RD_B4(b1, 1);
        P8_MM4(a1, b0, 1);
        // P3 (kh1, mh0)
        __builtin_amdgcn_s_barrier();
        if (!last) P8_STAGE_PHASE(kt + 1, 2);
        P8_RD_A4(a1, 1, 4);
        P8_MM4(a0, b1, 0);
        // P4 (kh1, mh1): publish next tile's kh0
        if (!last) {
          asm volatile("s_waitcnt vmcnt(2)" ::: "memory");
        }
        __builtin_amdgcn_s_barrier();
        if (!last) P8_STAGE_PHASE(kt + 1, 3);
        cur ^= 1;
        if (!last) {
          P8_RD_A4(a0, 0, 0);
          P8_RD_B4(b0, 0);
        }
        P8_MM4(a1, b1, 1);
      }
    } else {
    for (int kt = 0; kt < ktiles; ++kt) {
      const bool last = (kt == ktiles - 1);
      // P1 (kh0, mh0): consume a0,b0; read A(kh0, i4..7) -> a1
      if (!last) P8_STAGE_PHASE(kt + 1, 0);
      __builtin_amdgcn_s_barrier();
      P8_RD_A4(a1, 0, 4);
      P8_MM4(a0, b0, 0);
      __builtin_amdgcn_s_barrier();
      // P2 (kh0, mh1): publish kh1; read A(kh1, i0..3) -> a0, B(kh1) -> b1
      if (!last) {
        P8_STAGE_PHASE(kt + 1, 1);
        asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
      } else {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      }
      __builtin_amdgcn_s_barrier();
      P8_RD_A4(a0, 1, 0);
      P8_RD_B4(b1, 1);
      P8_MM4(a1, b0, 1);
      __builtin_amdgcn_s_barrier();
      // P3 (kh1, mh0): consume a0,b1; read A(kh1, i4..7) -> a1
      if (!last) P8_STAGE_PHASE(kt + 1, 2);
      __builtin_amdgcn_s_barrier();
      P8_RD_A4(a1, 1, 4);
      P8_MM4(a0, b1, 0);
      __builtin_amdgcn_s_barrier();
      // P4 (kh1, mh1): publish next tile kh0; read its first A bank + B
      if (!last) {
        P8_STAGE_PHASE(kt + 1, 3);
        asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
      }
      __builtin_amdgcn_s_barrier();
      cur ^= 1;   // reads below target the next tile's buffer
      if (!last) {
        P8_RD_A4(a0, 0, 0);
        P8_RD_B4(b0, 0);
      }
      P8_MM4(a1, b1, 1);
      __builtin_amdgcn_s_barrier();
    }
    }
#undef P8_RD_A4
#undef P8_RD_B4
#undef P8_MM4
  } else if (V == 1) {
    for (int kt = 0; kt < ktiles - 1; ++kt) {
      P8_PHASE_M(0, true, kt, 4);
      P8_PHASE_M(1, true, kt, 4);
      cur ^= 1;
    }
    const int kt = ktiles - 1;
    P8_PHASE_M(0, false, kt, 0);
    P8_PHASE_M(1, false, kt, -1);
  } else {
    for (int kt = 0; kt < ktiles - 1; ++kt) {
      P8_PHASE(0, 0, true, kt, -1);
      P8_PHASE(0, 1, true, kt, 4);   // publish next pair's k-half
      P8_PHASE(1, 0, true, kt, -1);
      P8_PHASE(1, 1, true, kt, 4);   // publish next K-tile's k-half 0
      cur ^= 1;
    }
    // final K-tile: nothing left to stage; drain what remains
    const int kt = ktiles - 1;
    P8_PHASE(0, 0, false, kt, -1);
    P8_PHASE(0, 1, false, kt, 0);  // k-half 1 fully landed
    P8_PHASE(1, 0, false, kt, -1);
    P8_PHASE(1, 1, false, kt, -1);
  }
#undef P8_PHASE
#undef P8_PHASE_M
#undef P8_STAGE_PHASE
#undef P8_STAGE
#undef P8_AFRAG
#undef P8_BFRAG

  // ---- epilogue --------------------------------------------------------
  const int crow0 = (lane >> 4) * 4;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const long row = bm + wm + i * 16 + crow0 + r;
        const long col = bn + wn + j * 16 + fr;
        if (row >= M || col >= N) continue;
        float fv = acc[i][j][r];
        if (Cadd != nullptr) {
          __hip_bfloat16 av = *reinterpret_cast<const __hip_bfloat16*>(
              &Cadd[row * add_rstride + col]);
          fv += __bfloat162float(av);
        }
        __hip_bfloat16 v = __float2bfloat16(fv);
        C[row * N + col] = *reinterpret_cast<ushort*>(&v);
      }
    }
  }
}

at::Tensor pxgemm8_bt_addv(const at::Tensor& a, const at::Tensor& bt,
                           const c10::optional<at::Tensor>& addend,
                           long variant) {
  TORCH_CHECK(a.is_cuda() && bt.is_cuda(), "pxgemm8_bt: GPU only");
  TORCH_CHECK(a.scalar_type() == at::kBFloat16 &&
              bt.scalar_type() == at::kBFloat16, "pxgemm8_bt: bf16 only");
  TORCH_CHECK(a.dim() == 2 && bt.dim() == 2 && a.is_contiguous() &&
              bt.is_contiguous());
  const long M = a.size(0), K = a.size(1), N = bt.size(0);
  TORCH_CHECK(bt.size(1) == K, "pxgemm8_bt: K mismatch");
  TORCH_CHECK(K % BK == 0, "pxgemm8_bt needs K % 64 == 0");
  TORCH_CHECK(M >= 1 && N >= 16, "pxgemm8_bt: degenerate shape");
  auto c = at::empty({M, N}, a.options());
  const int nbm = (int)((M + P8_BM - 1) / P8_BM);
  const int nbn = (int)((N + P8_BN - 1) / P8_BN);
  const int smem = 128 * 1024;
  auto stream = at::cuda::getCurrentCUDAStream();
  hipFuncSetAttribute(
      reinterpret_cast<const void*>(&pxgemm8_bt_kernel<0>),
      hipFuncAttributeMaxDynamicSharedMemorySize, smem);
  hipFuncSetAttribute(
      reinterpret_cast<const void*>(&pxgemm8_bt_kernel<1>),
      hipFuncAttributeMaxDynamicSharedMemorySize, smem);
  hipFuncSetAttribute(
      reinterpret_cast<const void*>(&pxgemm8_bt_kernel<2>),
      hipFuncAttributeMaxDynamicSharedMemorySize, smem);
  hipFuncSetAttribute(
      reinterpret_cast<const void*>(&pxgemm8_bt_kernel<3>),
      hipFuncAttributeMaxDynamicSharedMemorySize, smem);
  const ushort* add_ptr = nullptr;
  long add_rs = 0;
  if (addend.has_value()) {
    const auto& ad = addend.value();
    TORCH_CHECK(ad.scalar_type() == at::kBFloat16 && ad.dim() == 2 &&
                ad.size(0) == M && ad.size(1) == N && ad.stride(1) == 1,
                "pxgemm8_bt: bad addend");
    add_ptr = reinterpret_cast<const ushort*>(ad.data_ptr());
    add_rs = ad.stride(0);
  }
#define P8_LAUNCH(VV)                                                     \
  pxgemm8_bt_kernel<VV><<<nbm * nbn, P8_THREADS, smem, stream>>>(          \
      reinterpret_cast<const ushort*>(a.data_ptr()),                       \
      reinterpret_cast<const ushort*>(bt.data_ptr()),                      \
      reinterpret_cast<ushort*>(c.data_ptr()), M, N, K, nbm, nbn,          \
      add_ptr, add_rs)
  if (variant == 1) {
    P8_LAUNCH(1);
  } else if (variant == 2) {
    P8_LAUNCH(2);
  } else if (variant == 3) {
    P8_LAUNCH(3);
  } else {
    P8_LAUNCH(0);
  }
#undef P8_LAUNCH
  HIP_CHECK_KERNEL();
  return c;
}

static long p8_default_variant() {
  static long v = [] {
    const char* e = getenv("PARALLAX_GEMM8_VARIANT");
    return e ? atol(e) : 3L;  // measured best (gpurun_out/ab_v3.log)
  }();
  return v;
}

at::Tensor pxgemm8_bt_add(const at::Tensor& a, const at::Tensor& bt,
                          const c10::optional<at::Tensor>& addend) {
  return pxgemm8_bt_addv(a, bt, addend, p8_default_variant());
}

at::Tensor pxgemm8_bt(const at::Tensor& a, const at::Tensor& bt) {
  return pxgemm8_bt_addv(a, bt, c10::nullopt, p8_default_variant());
}

at::Tensor pxgemm8_bt_v(const at::Tensor& a, const at::Tensor& bt,
                        long variant) {
  return pxgemm8_bt_addv(a, bt, c10::nullopt, variant);
}

at::Tensor pxgemm_bt_add(const at::Tensor& a, const at::Tensor& bt,
                         const c10::optional<at::Tensor>& addend) {
  TORCH_CHECK(a.is_cuda() && bt.is_cuda(), "pxgemm_bt: GPU only");
  TORCH_CHECK(a.scalar_type() == at::kBFloat16 &&
              bt.scalar_type() == at::kBFloat16, "pxgemm_bt: bf16 only");
  TORCH_CHECK(a.dim() == 2 && bt.dim() == 2 && a.is_contiguous() &&
              bt.is_contiguous());
  const long M = a.size(0), K = a.size(1), N = bt.size(0);
  TORCH_CHECK(bt.size(1) == K, "pxgemm_bt: K mismatch");
  TORCH_CHECK(K % BK == 0, "pxgemm_bt needs K % 64 == 0");
  TORCH_CHECK(M >= 1 && N >= 16, "pxgemm_bt: degenerate shape");
  auto c = at::empty({M, N}, a.options());
  const int nbm = (int)((M + BM - 1) / BM);
  const int nbn = (int)((N + BN - 1) / BN);
  const int smem = 64 * 1024;
  auto stream = at::cuda::getCurrentCUDAStream();
  hipFuncSetAttribute(
      reinterpret_cast<const void*>(&pxgemm_bt_kernel),
      hipFuncAttributeMaxDynamicSharedMemorySize, smem);
  const ushort* add_ptr = nullptr;
  long add_rs = 0;
  if (addend.has_value()) {
    const auto& ad = addend.value();
    TORCH_CHECK(ad.scalar_type() == at::kBFloat16 && ad.dim() == 2 &&
                ad.size(0) == M && ad.size(1) == N && ad.stride(1) == 1,
                "pxgemm_bt: bad addend");
    add_ptr = reinterpret_cast<const ushort*>(ad.data_ptr());
    add_rs = ad.stride(0);
  }
  pxgemm_bt_kernel<<<nbm * nbn, PXG_THREADS, smem, stream>>>(
      reinterpret_cast<const ushort*>(a.data_ptr()),
      reinterpret_cast<const ushort*>(bt.data_ptr()),
      reinterpret_cast<ushort*>(c.data_ptr()), M, N, K, nbm, nbn,
      add_ptr, add_rs);
  HIP_CHECK_KERNEL();
  return c;
}

at::Tensor pxgemm_bt(const at::Tensor& a, const at::Tensor& bt) {
  return pxgemm_bt_add(a, bt, c10::nullopt);
}

// ---------------------------------------------------------------------------
// Implicit-GEMM 3x3 NHWC convolution forward (stride 1 or 2, padding 1)
// on the same 128x128 LDS-staged MFMA structure: the A operand is the
// im2col view of the HOST-PADDED input (glds cannot predicate, so the
// halo is materialized once per call), the B operand is the weight
// reshaped [Cout, 9*Cin] k-major (its natural channels_last order).
// out[(n,oy,ox), co] = sum_{dy,dx,ci} xp[n][oy*s+dy][ox*s+dx][ci]
//                                     * w[co][dy][dx][ci]
// ---------------------------------------------------------------------------

__global__ __launch_bounds__(PXG_THREADS, 2)
void pxconv3x3_kernel(const ushort* __restrict__ XP,  // [N,H+2,W+2,Cin]
                      const ushort* __restrict__ B,   // [Cout, 9*Cin]
                      ushort* __restrict__ C,         // [M, Cout]
                      long M, long N, long K, int nbm, int nbn,
                      int OH, int OW, int WP /*W+2*/, int HP /*H+2*/,
                      int Cin, int log2cin, int stride) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  int bid = blockIdx.x;
  {
    const int nwg = nbm * nbn;
    const int q = nwg / 8, r = nwg % 8;
    const int xcd = bid % 8, pos = bid / 8;
    bid = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + pos;
  }
  const int bm = (bid / nbn) * BM;
  const int bn = (bid % nbn) * BN;
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = tid >> 6;
  const int wm = (wave >> 1) * 64;
  const int wn = (wave & 1) * 64;
  const int fr = lane & 15;
  const int ko = (lane >> 4) * 8;
  f32x4 acc[4][4] = {};

  int p_row[4], p_kb[4];
  long a_base[4], b_src_row[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int p = (tid + i * PXG_THREADS) * 16;
    p_row[i] = p / (BK * 2);
    p_kb[i] = (p % (BK * 2)) ^ ((p_row[i] & 7) << 4);
    long ar = bm + p_row[i];
    if (ar >= M) ar = M - 1;          // clamped edge tile
    long br = bn + p_row[i];
    b_src_row[i] = br < N ? br : N - 1;
    // im2col row -> (n, oy, ox) -> padded-input byte base (k-independent)
    const long n_img = ar / ((long)OH * OW);
    const long rem = ar - n_img * ((long)OH * OW);
    const int oy = (int)(rem / OW);
    const int ox = (int)(rem - (long)oy * OW);
    a_base[i] = (((n_img * HP) + (long)oy * stride) * WP +
                 (long)ox * stride) * Cin;
  }
  const int ktiles = (int)(K / BK);

#define CSTAGE(buf, kt)                                                    \
  do {                                                                     \
    const int kbase = (kt) * BK;                                           \
    _Pragma("unroll") for (int i = 0; i < 4; ++i) {                        \
      const int ka = kbase + (p_kb[i] >> 1);                               \
      const int dydx = ka >> log2cin;                                      \
      const int ci = ka - (dydx << log2cin);                               \
      const int dy = dydx >= 6 ? 2 : (dydx >= 3 ? 1 : 0);                  \
      const int dx = dydx - 3 * dy;                                        \
      const ushort* srcA =                                                 \
          XP + a_base[i] + ((long)dy * WP + dx) * Cin + ci;                \
      const ushort* srcB = B + b_src_row[i] * K + kbase +                  \
                           (p_kb[i] >> 1);                                 \
      __builtin_amdgcn_global_load_lds(                                    \
          (const __attribute__((address_space(1))) void*)srcA,             \
          (__attribute__((address_space(3))) void*)(LDSA(buf) +            \
                                                    (tid + i * 256) * 16), \
          16, 0, 0);                                                       \
      __builtin_amdgcn_global_load_lds(                                    \
          (const __attribute__((address_space(1))) void*)srcB,             \
          (__attribute__((address_space(3))) void*)(LDSB(buf) +            \
                                                    (tid + i * 256) * 16), \
          16, 0, 0);                                                       \
    }                                                                      \
  } while (0)

  CSTAGE(0, 0);
  __builtin_amdgcn_s_waitcnt(0);
  __builtin_amdgcn_s_barrier();
  int cur = 0;
  for (int kt = 0; kt < ktiles; ++kt) {
    if (kt + 1 < ktiles) {
      CSTAGE(cur ^ 1, kt + 1);
    }
#pragma unroll
    for (int kk = 0; kk < BK / 32; ++kk) {
      bf16x8 a_frag[4], b_frag[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int ar = wm + i * 16 + fr;
        a_frag[i] = *(const bf16x8*)(LDSA(cur) +
                                     swz(ar, (kk * 32 + ko) * 2));
        const int br = wn + i * 16 + fr;
        b_frag[i] = *(const bf16x8*)(LDSB(cur) +
                                     swz(br, (kk * 32 + ko) * 2));
      }
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              a_frag[i], b_frag[j], acc[i][j], 0, 0, 0);
        }
      }
      __builtin_amdgcn_s_setprio(0);
    }
    __builtin_amdgcn_s_waitcnt(0);
    __builtin_amdgcn_s_barrier();
    cur ^= 1;
  }
  const int crow0 = (lane >> 4) * 4;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const long row = bm + wm + i * 16 + crow0 + r;
        const long col = bn + wn + j * 16 + fr;
        if (row >= M || col >= N) continue;
        __hip_bfloat16 v = __float2bfloat16(acc[i][j][r]);
        C[row * N + col] = *reinterpret_cast<ushort*>(&v);
      }
    }
  }
}

at::Tensor pxconv3x3_fwd(const at::Tensor& xp, const at::Tensor& w2d,
                         long n_img, long oh, long ow, long cin,
                         long stride, long HP, long WP) {
  // xp: padded NHWC activations flattened [N*(H+2)*(W+2)*Cin] bf16 view;
  // w2d: [Cout, 9*Cin] bf16 (channels_last weight order)
  TORCH_CHECK(xp.is_cuda() && w2d.is_cuda());
  TORCH_CHECK(xp.scalar_type() == at::kBFloat16 &&
              w2d.scalar_type() == at::kBFloat16);
  TORCH_CHECK(xp.is_contiguous() && w2d.is_contiguous());
  TORCH_CHECK((cin & (cin - 1)) == 0 && cin >= 64,
              "pxconv3x3: Cin must be a power of two >= 64");
  const long cout = w2d.size(0);
  const long K = w2d.size(1);
  TORCH_CHECK(K == 9 * cin && K % BK == 0);
  const long M = n_img * oh * ow;
  // the kernel touches y_in <= (oh-1)*stride+2 < HP and likewise for x
  TORCH_CHECK((oh - 1) * stride + 3 <= HP && (ow - 1) * stride + 3 <= WP,
              "pxconv3x3: padded dims too small");
  TORCH_CHECK(xp.numel() == n_img * HP * WP * cin,
              "pxconv3x3: padded input shape mismatch");
  int log2cin = 0;
  while ((1 << log2cin) < cin) log2cin++;
  auto c = at::empty({M, cout}, xp.options());
  const int nbm = (int)((M + BM - 1) / BM);
  const int nbn = (int)((cout + BN - 1) / BN);
  const int smem = 64 * 1024;
  auto stream = at::cuda::getCurrentCUDAStream();
  hipFuncSetAttribute(
      reinterpret_cast<const void*>(&pxconv3x3_kernel),
      hipFuncAttributeMaxDynamicSharedMemorySize, smem);
  pxconv3x3_kernel<<<nbm * nbn, PXG_THREADS, smem, stream>>>(
      reinterpret_cast<const ushort*>(xp.data_ptr()),
      reinterpret_cast<const ushort*>(w2d.data_ptr()),
      reinterpret_cast<ushort*>(c.data_ptr()), M, cout, K, nbm, nbn,
      (int)oh, (int)ow, (int)WP, (int)HP, (int)cin, log2cin, (int)stride);
  HIP_CHECK_KERNEL();
  return c;
}

// ---------------------------------------------------------------------------
// Split-K skinny GEMM for the LSTM chain (M <= 128): out[M,N] = A[M,K] @
// B[N,K]^T.  The per-timestep projection (128x512, K=2048) and backward
// carry (128x512, K=8192) are latency-bound dependent launches —
// hipBLASLt runs them as 16x16-tile kernels at 8-19 us each.  Here
// (guide "Sampling-regime projection GEMM" recipe, atomic variant):
// the K axis splits over blocks until ~256 blocks are in flight, each
// block computes a [128 x 64] tile over its K-slice and accumulates
// into an fp32 workspace with global atomics; a second tiny kernel
// casts the workspace to bf16 (optionally adding a strided bf16 addend
// — the upstream-grad slice in the backward chain) and re-zeros it for
// the next timestep.
// ---------------------------------------------------------------------------

#define SK_THREADS 256

__global__ __launch_bounds__(SK_THREADS, 4)
void px_skinny_kernel(const ushort* __restrict__ A,
                      const ushort* __restrict__ B,
                      float* __restrict__ WS, ushort* __restrict__ OUT,
                      int* __restrict__ CNT,
                      const ushort* __restrict__ ADD, long add_rs,
                      long M, long N, long K, int spl, int kslice) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  // LDS: A tile [128][64] (16 KiB, swizzled like pxgemm_bt) +
  //      B tile [64][64] (8 KiB)
#define SK_LDSA (smem)
#define SK_LDSB (smem + 16384)
  const int nb = blockIdx.x / spl;        // output column tile
  const int ks = blockIdx.x % spl;        // K slice
  const long bn = (long)nb * 64;
  const long k0 = (long)ks * kslice;
  long k1 = k0 + kslice;
  if (k1 > K) k1 = K;

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = tid >> 6;
  const int wm = wave * 32;               // wave rows
  const int fr = lane & 15;
  const int ko = (lane >> 4) * 8;
  f32x4 acc[2][4] = {};

  // staging addresses (pxgemm_bt pattern, swizzle ((row&7)<<4))
  int pa_row[4], pa_kb[4];
  long a_src[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int p = (tid + i * SK_THREADS) * 16;
    pa_row[i] = p / 128;
    pa_kb[i] = (p % 128) ^ ((pa_row[i] & 7) << 4);
    long ar = pa_row[i];
    a_src[i] = ar < M ? ar : M - 1;
  }
  int pb_row[2], pb_kb[2];
  long b_src[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int p = (tid + i * SK_THREADS) * 16;
    pb_row[i] = p / 128;
    pb_kb[i] = (p % 128) ^ ((pb_row[i] & 7) << 4);
    long br = bn + pb_row[i];
    b_src[i] = br < N ? br : N - 1;
  }

  for (long kt = k0; kt < k1; kt += 64) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      __builtin_amdgcn_global_load_lds(
          (const __attribute__((address_space(1))) void*)(
              A + a_src[i] * K + kt + (pa_kb[i] >> 1)),
          (__attribute__((address_space(3))) void*)(SK_LDSA +
                                                    (tid + i * 256) * 16),
          16, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      __builtin_amdgcn_global_load_lds(
          (const __attribute__((address_space(1))) void*)(
              B + b_src[i] * K + kt + (pb_kb[i] >> 1)),
          (__attribute__((address_space(3))) void*)(SK_LDSB +
                                                    (tid + i * 256) * 16),
          16, 0, 0);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      bf16x8 a_frag[2], b_frag[4];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int ar = wm + i * 16 + fr;
        a_frag[i] = *(const bf16x8*)(SK_LDSA + swz(ar, (kk * 32 + ko) * 2));
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int br = j * 16 + fr;
        b_frag[j] = *(const bf16x8*)(SK_LDSB + swz(br, (kk * 32 + ko) * 2));
      }
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              a_frag[i], b_frag[j], acc[i][j], 0, 0, 0);
        }
      }
      __builtin_amdgcn_s_setprio(0);
    }
    __builtin_amdgcn_s_barrier();
  }
  const int crow0 = (lane >> 4) * 4;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const long row = wm + i * 16 + crow0 + r;
        const long col = bn + j * 16 + fr;
        if (row >= M || col >= N) continue;
        atomicAdd(&WS[row * N + col], acc[i][j][r]);
      }
    }
  }
  // ---- in-launch split-K combine (guide §5 "Sampling-regime" recipe,
  // ticket form): the LAST arriving slice of this column tile casts the
  // fp32 workspace to bf16 (+ optional strided addend), re-zeros it for
  // the next call, and resets its ticket.  Atomic payloads are L2-
  // coherent; the drain before the ticket orders them, the agent-scope
  // acquire on the reader drops any stale L1 lines.
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  int* last_flag = reinterpret_cast<int*>(smem);
  if (tid == 0) {
    const int old = __hip_atomic_fetch_add(&CNT[nb], 1, __ATOMIC_RELAXED,
                                           __HIP_MEMORY_SCOPE_AGENT);
    *last_flag = (old == spl - 1) ? 1 : 0;
  }
  __syncthreads();
  if (*last_flag == 0) return;
  if (tid == 0) {
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
  }
  __syncthreads();
  // tile is [M rows] x [64 cols] at column bn; 4-wide per thread
  const long rows = M;
  for (int e = tid; e < rows * 16; e += SK_THREADS) {
    const long row = e / 16;
    const long col = bn + (e % 16) * 4;
    float4 w = *reinterpret_cast<float4*>(&WS[row * N + col]);
    if (ADD != nullptr) {
      const ushort* ap = ADD + row * add_rs + col;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        (&w.x)[q] += __bfloat162float(
            *reinterpret_cast<const __hip_bfloat16*>(ap + q));
      }
    }
    ushort o[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      __hip_bfloat16 bv = __float2bfloat16((&w.x)[q]);
      o[q] = *reinterpret_cast<ushort*>(&bv);
    }
    *reinterpret_cast<uint2*>(&OUT[row * N + col]) =
        *reinterpret_cast<uint2*>(&o[0]);
    float4 z;
    z.x = z.y = z.z = z.w = 0.f;
    *reinterpret_cast<float4*>(&WS[row * N + col]) = z;
  }
  if (tid == 0) {
    __hip_atomic_store(&CNT[nb], 0, __ATOMIC_RELAXED,
                       __HIP_MEMORY_SCOPE_AGENT);
  }
#undef SK_LDSA
#undef SK_LDSB
}

void px_skinny_bt(const at::Tensor& a, const at::Tensor& bt,
                  at::Tensor ws, at::Tensor cnt, at::Tensor out,
                  const c10::optional<at::Tensor>& addend) {
  TORCH_CHECK(a.is_cuda() && a.scalar_type() == at::kBFloat16 &&
              bt.scalar_type() == at::kBFloat16);
  TORCH_CHECK(a.dim() == 2 && bt.dim() == 2 && a.is_contiguous() &&
              bt.is_contiguous());
  const long M = a.size(0), K = a.size(1), N = bt.size(0);
  TORCH_CHECK(bt.size(1) == K && M <= 128 && N % 64 == 0 && K % 64 == 0,
              "px_skinny_bt: need M<=128, N%64==0, K%64==0");
  TORCH_CHECK(ws.scalar_type() == at::kFloat && ws.numel() == M * N &&
              ws.is_contiguous(), "px_skinny_bt: bad workspace");
  TORCH_CHECK(out.scalar_type() == at::kBFloat16 && out.numel() == M * N
              && out.is_contiguous() && (N % 4) == 0);
  const int ntiles = (int)(N / 64);
  const int kt64 = (int)(K / 64);
  // deep-K split measured SLOWER (859k vs 900k lm1b words/s,
  // gpurun_out/lm_deep*) — the extra atomic traffic and cast-tile
  // contention beat the shorter serial k-loop; keep the toggle for
  // future shapes but default off
  static const bool deep = [] {
    const char* e = getenv("PARALLAX_SKINNY_DEEP");
    return e != nullptr && e[0] == '1';
  }();
  int spl = (int)(((deep && kt64 >= 64) ? 512 : 256) / ntiles);
  if (spl > kt64) spl = kt64;
  if (spl < 1) spl = 1;
  const int kslice = (int)(((kt64 + spl - 1) / spl) * 64);
  const ushort* add_ptr = nullptr;
  long add_rs = 0;
  if (addend.has_value()) {
    const auto& ad = addend.value();
    TORCH_CHECK(ad.scalar_type() == at::kBFloat16 && ad.dim() == 2 &&
                ad.size(0) == M && ad.size(1) == N && ad.stride(1) == 1);
    add_ptr = reinterpret_cast<const ushort*>(ad.data_ptr());
    add_rs = ad.stride(0);
  }
  TORCH_CHECK(cnt.scalar_type() == at::kInt && cnt.numel() >= ntiles,
              "px_skinny_bt: bad ticket buffer");
  auto stream = at::cuda::getCurrentCUDAStream();
  px_skinny_kernel<<<ntiles * spl, SK_THREADS, 24576, stream>>>(
      reinterpret_cast<const ushort*>(a.data_ptr()),
      reinterpret_cast<const ushort*>(bt.data_ptr()),
      ws.data_ptr<float>(), reinterpret_cast<ushort*>(out.data_ptr()),
      cnt.data_ptr<int>(), add_ptr, add_rs, M, N, K, spl, kslice);
  HIP_CHECK_KERNEL();
}

// ---------------------------------------------------------------------------
// Tall-tile MFMA GEMM: 256x64 output tile, 8 waves (8M x 1N), BK=64,
// double-buffered glds, 80 KiB LDS -> 2 blocks/CU (the co-resident
// block's MFMAs cover this block's staging phases).  For the
// M-huge / N-small shapes (ResNet conv-as-GEMM: N = Cout in {64..512})
// where the 128/256-wide tiles compute mostly-discarded columns.
// ---------------------------------------------------------------------------

#define TL_BM 256
#define TL_THREADS 512

__global__ __launch_bounds__(TL_THREADS, 2)
void px_tall_kernel(const ushort* __restrict__ A,
                    const ushort* __restrict__ B,
                    ushort* __restrict__ C, long M, long N, long K,
                    int nbm, int nbn) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  // [2 buf][A 32 KiB | B 8 KiB]
#define TL_LDSA(b) (smem + (b) * 40960)
#define TL_LDSB(b) (smem + (b) * 40960 + 32768)
  int bid = blockIdx.x;
  {
    const int nwg = nbm * nbn;
    const int q = nwg / 8, r = nwg % 8;
    const int xcd = bid % 8, pos = bid / 8;
    bid = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + pos;
  }
  const long bm = (long)(bid / nbn) * TL_BM;
  const long bn = (long)(bid % nbn) * 64;
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = tid >> 6;
  const int wm = wave * 32;
  const int fr = lane & 15;
  const int ko = (lane >> 4) * 8;
  f32x4 acc[2][4] = {};

  // staging: A = 4 rounds of 512x16B, B = 1 round (512 x 16 B = the
  // whole 8 KiB tile); swizzle ((row&7)<<4)
  int pa_row[4], pa_kb[4];
  long a_src[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int p = (tid + i * TL_THREADS) * 16;
    pa_row[i] = p / 128;
    pa_kb[i] = (p % 128) ^ ((pa_row[i] & 7) << 4);
    long ar = bm + pa_row[i];
    a_src[i] = ar < M ? ar : M - 1;
  }
  int pb_row, pb_kb;
  long b_src;
  {
    const int p = tid * 16;
    pb_row = p / 128;
    pb_kb = (p % 128) ^ ((pb_row & 7) << 4);
    long br = bn + pb_row;
    b_src = br < N ? br : N - 1;
  }
  const int ktiles = (int)(K / 64);

#define TL_STAGE(buf, kt)                                                  \
  do {                                                                     \
    const long kb = (long)(kt) * 64;                                       \
    _Pragma("unroll") for (int i = 0; i < 4; ++i) {                        \
      __builtin_amdgcn_global_load_lds(                                    \
          (const __attribute__((address_space(1))) void*)(                 \
              A + a_src[i] * K + kb + (pa_kb[i] >> 1)),                    \
          (__attribute__((address_space(3))) void*)(TL_LDSA(buf) +         \
                                                    (tid + i * 512) * 16), \
          16, 0, 0);                                                       \
    }                                                                      \
    __builtin_amdgcn_global_load_lds(                                      \
        (const __attribute__((address_space(1))) void*)(                   \
            B + b_src * K + kb + (pb_kb >> 1)),                            \
        (__attribute__((address_space(3))) void*)(TL_LDSB(buf) +           \
                                                  tid * 16),               \
        16, 0, 0);                                                         \
  } while (0)

  TL_STAGE(0, 0);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  int cur = 0;
  for (int kt = 0; kt < ktiles; ++kt) {
    if (kt + 1 < ktiles) TL_STAGE(cur ^ 1, kt + 1);
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      bf16x8 a_frag[2], b_frag[4];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int ar = wm + i * 16 + fr;
        a_frag[i] = *(const bf16x8*)(TL_LDSA(cur) +
                                     swz(ar, (kk * 32 + ko) * 2));
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int br = j * 16 + fr;
        b_frag[j] = *(const bf16x8*)(TL_LDSB(cur) +
                                     swz(br, (kk * 32 + ko) * 2));
      }
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              a_frag[i], b_frag[j], acc[i][j], 0, 0, 0);
        }
      }
      __builtin_amdgcn_s_setprio(0);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    cur ^= 1;
  }
  const int crow0 = (lane >> 4) * 4;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const long row = bm + wm + i * 16 + crow0 + r;
        const long col = bn + j * 16 + fr;
        if (row >= M || col >= N) continue;
        __hip_bfloat16 v = __float2bfloat16(acc[i][j][r]);
        C[row * N + col] = *reinterpret_cast<ushort*>(&v);
      }
    }
  }
#undef TL_STAGE
#undef TL_LDSA
#undef TL_LDSB
}

at::Tensor px_tall_bt(const at::Tensor& a, const at::Tensor& bt) {
  TORCH_CHECK(a.is_cuda() && a.scalar_type() == at::kBFloat16 &&
              bt.scalar_type() == at::kBFloat16);
  TORCH_CHECK(a.dim() == 2 && bt.dim() == 2 && a.is_contiguous() &&
              bt.is_contiguous());
  const long M = a.size(0), K = a.size(1), N = bt.size(0);
  TORCH_CHECK(bt.size(1) == K && K % 64 == 0 && N >= 16);
  auto c = at::empty({M, N}, a.options());
  const int nbm = (int)((M + TL_BM - 1) / TL_BM);
  const int nbn = (int)((N + 63) / 64);
  auto stream = at::cuda::getCurrentCUDAStream();
  hipFuncSetAttribute(
      reinterpret_cast<const void*>(&px_tall_kernel),
      hipFuncAttributeMaxDynamicSharedMemorySize, 81920);
  px_tall_kernel<<<nbm * nbn, TL_THREADS, 81920, stream>>>(
      reinterpret_cast<const ushort*>(a.data_ptr()),
      reinterpret_cast<const ushort*>(bt.data_ptr()),
      reinterpret_cast<ushort*>(c.data_ptr()), M, N, K, nbm, nbn);
  HIP_CHECK_KERNEL();
  return c;
}

// ---------------------------------------------------------------------------
// 3x3 NHWC conv forward as implicit GEMM on the tall-tile structure:
// A = im2col of the HOST-PADDED input (halo materialized once per call;
// glds cannot predicate), B = weight [Cout, 9*Cin] k-major.  Stride 1/2.
// The SAME kernel computes stride-1 dgrad when fed pad(dy) and the
// rotated/transposed weight [Cin, 9*Cout] (host prep, tiny).
// ---------------------------------------------------------------------------

__global__ __launch_bounds__(TL_THREADS, 2)
void px_tall_conv3x3_kernel(const ushort* __restrict__ XP,
                            const ushort* __restrict__ B,
                            ushort* __restrict__ C, long M, long N,
                            long K, int nbm, int nbn, int OH, int OW,
                            int WP, int HP, int Cin, int log2cin,
                            int stride) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
#define TL_LDSA(b) (smem + (b) * 40960)
#define TL_LDSB(b) (smem + (b) * 40960 + 32768)
  int bid = blockIdx.x;
  {
    const int nwg = nbm * nbn;
    const int q = nwg / 8, r = nwg % 8;
    const int xcd = bid % 8, pos = bid / 8;
    bid = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + pos;
  }
  const long bm = (long)(bid / nbn) * TL_BM;
  const long bn = (long)(bid % nbn) * 64;
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = tid >> 6;
  const int wm = wave * 32;
  const int fr = lane & 15;
  const int ko = (lane >> 4) * 8;
  f32x4 acc[2][4] = {};

  int pa_kb[4];
  long a_base[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int p = (tid + i * TL_THREADS) * 16;
    const int prow = p / 128;
    pa_kb[i] = (p % 128) ^ ((prow & 7) << 4);
    long ar = bm + prow;
    if (ar >= M) ar = M - 1;
    const long n_img = ar / ((long)OH * OW);
    const long rem = ar - n_img * ((long)OH * OW);
    const int oy = (int)(rem / OW);
    const int ox = (int)(rem - (long)oy * OW);
    a_base[i] = (((n_img * (long)HP) + (long)oy * stride) * WP +
                 (long)ox * stride) * Cin;
  }
  int pb_row, pb_kb;
  long b_src;
  {
    const int p = tid * 16;
    pb_row = p / 128;
    pb_kb = (p % 128) ^ ((pb_row & 7) << 4);
    long br = bn + pb_row;
    b_src = br < N ? br : N - 1;
  }
  const int ktiles = (int)(K / 64);

#define TLC_STAGE(buf, kt)                                                 \
  do {                                                                     \
    const int kb = (kt) * 64;                                              \
    _Pragma("unroll") for (int i = 0; i < 4; ++i) {                        \
      const int ka = kb + (pa_kb[i] >> 1);                                 \
      const int dydx = ka >> log2cin;                                      \
      const int ci = ka - (dydx << log2cin);                               \
      const int dy = dydx >= 6 ? 2 : (dydx >= 3 ? 1 : 0);                  \
      const int dx = dydx - 3 * dy;                                        \
      __builtin_amdgcn_global_load_lds(                                    \
          (const __attribute__((address_space(1))) void*)(                 \
              XP + a_base[i] + ((long)dy * WP + dx) * Cin + ci),           \
          (__attribute__((address_space(3))) void*)(TL_LDSA(buf) +         \
                                                    (tid + i * 512) * 16), \
          16, 0, 0);                                                       \
    }                                                                      \
    __builtin_amdgcn_global_load_lds(                                      \
        (const __attribute__((address_space(1))) void*)(                   \
            B + b_src * K + kb + (pb_kb >> 1)),                            \
        (__attribute__((address_space(3))) void*)(TL_LDSB(buf) +           \
                                                  tid * 16),               \
        16, 0, 0);                                                         \
  } while (0)

  TLC_STAGE(0, 0);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  int cur = 0;
  for (int kt = 0; kt < ktiles; ++kt) {
    if (kt + 1 < ktiles) TLC_STAGE(cur ^ 1, kt + 1);
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      bf16x8 a_frag[2], b_frag[4];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int ar = wm + i * 16 + fr;
        a_frag[i] = *(const bf16x8*)(TL_LDSA(cur) +
                                     swz(ar, (kk * 32 + ko) * 2));
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int br = j * 16 + fr;
        b_frag[j] = *(const bf16x8*)(TL_LDSB(cur) +
                                     swz(br, (kk * 32 + ko) * 2));
      }
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              a_frag[i], b_frag[j], acc[i][j], 0, 0, 0);
        }
      }
      __builtin_amdgcn_s_setprio(0);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    cur ^= 1;
  }
  const int crow0 = (lane >> 4) * 4;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const long row = bm + wm + i * 16 + crow0 + r;
        const long col = bn + j * 16 + fr;
        if (row >= M || col >= N) continue;
        __hip_bfloat16 v = __float2bfloat16(acc[i][j][r]);
        C[row * N + col] = *reinterpret_cast<ushort*>(&v);
      }
    }
  }
#undef TLC_STAGE
#undef TL_LDSA
#undef TL_LDSB
}

at::Tensor px_tall_conv3x3(const at::Tensor& xp, const at::Tensor& w2d,
                           long n_img, long oh, long ow, long cin,
                           long stride, long HP, long WP) {
  TORCH_CHECK(xp.is_cuda() && w2d.is_cuda());
  TORCH_CHECK(xp.scalar_type() == at::kBFloat16 &&
              w2d.scalar_type() == at::kBFloat16);
  TORCH_CHECK(xp.is_contiguous() && w2d.is_contiguous());
  TORCH_CHECK((cin & (cin - 1)) == 0 && cin >= 64,
              "px_tall_conv3x3: Cin must be a power of two >= 64");
  const long cout = w2d.size(0);
  const long K = w2d.size(1);
  TORCH_CHECK(K == 9 * cin && K % 64 == 0);
  const long M = n_img * oh * ow;
  TORCH_CHECK((oh - 1) * stride + 3 <= HP && (ow - 1) * stride + 3 <= WP);
  TORCH_CHECK(xp.numel() == n_img * HP * WP * cin);
  int log2cin = 0;
  while ((1 << log2cin) < cin) log2cin++;
  auto c = at::empty({M, cout}, xp.options());
  const int nbm = (int)((M + TL_BM - 1) / TL_BM);
  const int nbn = (int)((cout + 63) / 64);
  auto stream = at::cuda::getCurrentCUDAStream();
  hipFuncSetAttribute(
      reinterpret_cast<const void*>(&px_tall_conv3x3_kernel),
      hipFuncAttributeMaxDynamicSharedMemorySize, 81920);
  px_tall_conv3x3_kernel<<<nbm * nbn, TL_THREADS, 81920, stream>>>(
      reinterpret_cast<const ushort*>(xp.data_ptr()),
      reinterpret_cast<const ushort*>(w2d.data_ptr()),
      reinterpret_cast<ushort*>(c.data_ptr()), M, cout, K, nbm, nbn,
      (int)oh, (int)ow, (int)WP, (int)HP, (int)cin, log2cin,
      (int)stride);
  HIP_CHECK_KERNEL();
  return c;
}

// ---------------------------------------------------------------------------
// 3x3 NHWC conv WGRAD as implicit GEMM with LDS-transposed staging:
// dW[co][kc] += sum_m dy[m][co] * im2col[m][kc]  (m = N*OH*OW rows).
// Both operands are m-major in memory but the MFMA fragments need
// k(=m)-contiguous reads, so each 64-row m-tile is staged TRANSPOSED
// into LDS (scatter b16 writes, padded 144-B rows -> 2-way banks, the
// attention-loader pattern).  The m axis splits over blocks; partial
// tiles accumulate with fp32 global atomics into a zeroed workspace
// (the caller casts once).  Each 64-wide kc tile lies inside ONE of the
// nine taps (Cin % 64 == 0), so its im2col rows are contiguous slices
// of the padded input.
// ---------------------------------------------------------------------------

#define WG_LDP 72   // padded LDS row stride (elements)

__global__ __launch_bounds__(256, 4)
void px_wgrad3x3_kernel(const ushort* __restrict__ DY,  // [M, Cout]
                        const ushort* __restrict__ XP,  // padded NHWC
                        float* __restrict__ WS,         // [Cout, 9*Cin]
                        long M, long Cout, long K9, int OH, int OW,
                        int WP, int HP, int Cin, int log2cin, int stride,
                        int nco, int nkc, int splitm, int mtiles) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  ushort* dyT = reinterpret_cast<ushort*>(smem);            // [64][WG_LDP]
  ushort* xT = dyT + 64 * WG_LDP;                           // [64][WG_LDP]
  const int bid = blockIdx.x;
  const int co0 = (bid % nco) * 64;
  const int kc0 = ((bid / nco) % nkc) * 64;
  const int ms = bid / (nco * nkc);          // m-slice index
  const int tps = (mtiles + splitm - 1) / splitm;
  const int mt0 = ms * tps;
  int mt1 = mt0 + tps;
  if (mt1 > mtiles) mt1 = mtiles;

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = tid >> 6;
  const int fr = lane & 15;
  const int ko = (lane >> 4) * 8;
  // wave owns co rows wave*16..wave*16+15 x all 64 kc
  f32x4 acc[4] = {};

  // kc tile -> tap + channel base (whole tile inside one tap)
  const int dydx = kc0 >> log2cin;
  const int tdy = dydx >= 6 ? 2 : (dydx >= 3 ? 1 : 0);
  const int tdx = dydx - 3 * tdy;
  const int ci0 = kc0 - (dydx << log2cin);

  for (int mt = mt0; mt < mt1; ++mt) {
    const long m0 = (long)mt * 64;
    // stage both tiles transposed: 2 rounds x 256 threads x 8 elems
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int idx = tid + r * 256;
      const int mm = idx & 63;
      const int cg = (idx >> 6) * 8;
      const long m = m0 + mm;
      uint4 dv = {0u, 0u, 0u, 0u}, xv = {0u, 0u, 0u, 0u};
      if (m < M) {
        if (co0 + cg < Cout) {
          dv = *reinterpret_cast<const uint4*>(&DY[m * Cout + co0 + cg]);
        }
        const long n_img = m / ((long)OH * OW);
        const long rem = m - n_img * ((long)OH * OW);
        const int oy = (int)(rem / OW);
        const int ox = (int)(rem - (long)oy * OW);
        const ushort* src = XP +
            (((n_img * HP) + (long)oy * stride + tdy) * WP +
             (long)ox * stride + tdx) * Cin + ci0 + cg;
        xv = *reinterpret_cast<const uint4*>(src);
      }
      const ushort* de = reinterpret_cast<const ushort*>(&dv);
      const ushort* xe = reinterpret_cast<const ushort*>(&xv);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        dyT[(cg + j) * WG_LDP + mm] = de[j];
        xT[(cg + j) * WG_LDP + mm] = xe[j];
      }
    }
    __syncthreads();
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      bf16x8 a_frag, b_frag[4];
      a_frag = *(const bf16x8*)(&dyT[(wave * 16 + fr) * WG_LDP +
                                     kk * 32 + ko]);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        b_frag[j] = *(const bf16x8*)(&xT[(j * 16 + fr) * WG_LDP +
                                         kk * 32 + ko]);
      }
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            a_frag, b_frag[j], acc[j], 0, 0, 0);
      }
      __builtin_amdgcn_s_setprio(0);
    }
    __syncthreads();
  }
  const int crow0 = (lane >> 4) * 4;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const long co = co0 + wave * 16 + crow0 + r;
      const long kc = kc0 + j * 16 + fr;
      if (co >= Cout) continue;
      atomicAdd(&WS[co * K9 + kc], acc[j][r]);
    }
  }
}

at::Tensor px_wgrad3x3(const at::Tensor& dy2d, const at::Tensor& xp,
                       long n_img, long oh, long ow, long cin,
                       long stride, long HP, long WP) {
  TORCH_CHECK(dy2d.is_cuda() && xp.is_cuda());
  TORCH_CHECK(dy2d.scalar_type() == at::kBFloat16 &&
              xp.scalar_type() == at::kBFloat16);
  TORCH_CHECK(dy2d.dim() == 2 && dy2d.is_contiguous() &&
              xp.is_contiguous());
  const long M = n_img * oh * ow;
  const long Cout = dy2d.size(1);
  TORCH_CHECK(dy2d.size(0) == M && Cout % 8 == 0);
  TORCH_CHECK((cin & (cin - 1)) == 0 && cin >= 64);
  TORCH_CHECK(xp.numel() == n_img * HP * WP * cin);
  const long K9 = 9 * cin;
  int log2cin = 0;
  while ((1 << log2cin) < cin) log2cin++;
  auto ws = at::zeros({Cout, K9},
                      dy2d.options().dtype(at::kFloat));
  const int nco = (int)((Cout + 63) / 64);
  const int nkc = (int)(K9 / 64);
  const int mtiles = (int)((M + 63) / 64);
  int splitm = (int)(384 / (nco * nkc));
  if (splitm > mtiles) splitm = mtiles;
  if (splitm < 1) splitm = 1;
  auto stream = at::cuda::getCurrentCUDAStream();
  const int smem = 2 * 64 * WG_LDP * 2;
  px_wgrad3x3_kernel<<<nco * nkc * splitm, 256, smem, stream>>>(
      reinterpret_cast<const ushort*>(dy2d.data_ptr()),
      reinterpret_cast<const ushort*>(xp.data_ptr()),
      ws.data_ptr<float>(), M, Cout, K9, (int)oh, (int)ow, (int)WP,
      (int)HP, (int)cin, log2cin, (int)stride, nco, nkc, splitm, mtiles);
  HIP_CHECK_KERNEL();
  return ws;   // fp32 [Cout, 9*Cin]; caller casts/reshapes
}
