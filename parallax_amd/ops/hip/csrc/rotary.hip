// Rotary positions: in each head the pairs (u, v) of the leading R values
// turn by the angle of their place,
//
//   u' = u cos - v sin,   v' = u sin + v cos,
//
// with pairs (2i, 2i+1) (interleaved) or (i, i + R/2) (halves), and the rest
// of the head passes through.  The gradient is the same rotation by the
// negative angle.  Queries and keys go through one launch.
//
// Bound by memory: every value is read once and written once, in 16-byte
// pieces where the layout allows (2 x 32,768 tokens of 16 + 4 heads of 128 in
// bf16, there and back: 350 us, 3.9 TB/s; a large copy reaches 4.9); the
// table rows (fp32, made from 64-bit
// angles by the caller) are shared by all heads of a token and come from
// cache.  Arithmetic is fp32 with one rounding at the end; the contractions
// are written out so that all variants give the same bits.

#include <torch/extension.h>
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "common.h"

namespace {

struct Side {
  const void* in;
  void* out;
  long ib, it, ih;  // strides of batch, token, head of the input
  long ob, ot, oh;
  int heads;
};

struct Places {
  const int64_t* pos;  // nullptr: offset + t
  long pb, pt;
  long offset;
  long rows;  // of the tables
};

__device__ __forceinline__ long place(const Places& p, long b, long t) {
  long r = p.pos ? p.pos[b * p.pb + t * p.pt] : p.offset + t;
  return r < 0 ? 0 : (r >= p.rows ? p.rows - 1 : r);
}

// n / d for n of at most `most`, by one high product where that is exact:
// with m = 2^32 / d + 1 the error n (m d - 2^32) / 2^32 stays below 1 / d as
// long as n d < 2^32.
struct Div {
  unsigned d, m;
  Div(long div, long most)
      : d((unsigned)div),
        m(div > 1 && most * div < (1L << 32)
              ? (unsigned)((1L << 32) / div + 1) : 0u) {}
  __device__ __forceinline__ unsigned operator()(unsigned n) const {
    return m ? __umulhi(n, m) : n / d;
  }
};

// V values, aligned as a whole or (AL = false) as one of them
template <typename T, int V, bool AL>
struct alignas(AL ? sizeof(T) * V : sizeof(T)) Piece {
  T v[V];
};

// A workgroup takes `tpb` tokens, a thread one piece of a head at a time: V
// values of interleaved pairs, V values of the first half with those of the
// second, or VR values behind the turned part.
template <typename T, int V, int VR, bool INTER, bool AL>
__global__ __launch_bounds__(256) void rotary_kernel(
    Side q, Side k, Places p, const float* __restrict__ cos,
    const float* __restrict__ sin, long cs, float sign, unsigned tokens,
    int R, unsigned tpb, Div by_T, Div by_token, Div by_head) {
  typedef Piece<T, V, AL> P;
  typedef Piece<T, VR, AL> PR;
  const unsigned t0 = blockIdx.x * tpb;
  const unsigned here = (tokens - t0 < tpb ? tokens - t0 : tpb) * by_token.d;
  const unsigned turned = INTER ? R / V : R / (2 * V);
#pragma unroll 4
  for (unsigned i = threadIdx.x; i < here; i += 256) {
    const unsigned dt = by_token(i);
    const unsigned in_token = i - dt * by_token.d;
    unsigned h = by_head(in_token);
    const unsigned w = in_token - h * by_head.d;
    const unsigned b = by_T(t0 + dt);
    const unsigned t = t0 + dt - b * by_T.d;
    const bool second = h >= (unsigned)q.heads;
    if (second) h -= q.heads;
    const T* in = static_cast<const T*>(second ? k.in : q.in) +
                  b * (second ? k.ib : q.ib) + t * (second ? k.it : q.it) +
                  h * (second ? k.ih : q.ih);
    T* out = static_cast<T*>(second ? k.out : q.out) +
             b * (second ? k.ob : q.ob) + t * (second ? k.ot : q.ot) +
             h * (second ? k.oh : q.oh);
    if (w >= turned) {
      const int at = R + (w - turned) * VR;
      *reinterpret_cast<PR*>(out + at) =
          *reinterpret_cast<const PR*>(in + at);
      continue;
    }
    const long row = place(p, b, t) * cs;
    if constexpr (INTER) {
      P x = *reinterpret_cast<const P*>(in + w * V);
#pragma unroll
      for (int e = 0; e < V / 2; ++e) {
        const float c = cos[row + w * (V / 2) + e];
        const float n = sign * sin[row + w * (V / 2) + e];
        const float u = to_f32<T>(x.v[2 * e]), v = to_f32<T>(x.v[2 * e + 1]);
        x.v[2 * e] = from_f32<T>(fmaf(u, c, -(v * n)));
        x.v[2 * e + 1] = from_f32<T>(fmaf(u, n, v * c));
      }
      *reinterpret_cast<P*>(out + w * V) = x;
    } else {
      const int at = w * V;
      P x = *reinterpret_cast<const P*>(in + at);
      P y = *reinterpret_cast<const P*>(in + R / 2 + at);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float c = cos[row + at + e], n = sign * sin[row + at + e];
        const float u = to_f32<T>(x.v[e]), v = to_f32<T>(y.v[e]);
        x.v[e] = from_f32<T>(fmaf(u, c, -(v * n)));
        y.v[e] = from_f32<T>(fmaf(u, n, v * c));
      }
      *reinterpret_cast<P*>(out + at) = x;
      *reinterpret_cast<P*>(out + R / 2 + at) = y;
    }
  }
}

Side side(const at::Tensor& in, at::Tensor& out) {
  Side s;
  s.in = in.data_ptr();
  s.out = out.data_ptr();
  // the stride of a dimension of one says nothing
  auto at = [](const at::Tensor& t, int i) {
    return t.size(i) > 1 ? t.stride(i) : 0;
  };
  s.ib = at(in, 0);
  s.it = at(in, 1);
  s.ih = at(in, 2);
  s.ob = at(out, 0);
  s.ot = at(out, 1);
  s.oh = at(out, 2);
  s.heads = (int)in.size(2);
  return s;
}

bool fits(const Side& s, int v, int size) {
  const uintptr_t a = (uintptr_t)s.in | (uintptr_t)s.out;
  return s.heads == 0 ||
         (a % (v * size) == 0 &&
          (s.ib | s.it | s.ih | s.ob | s.ot | s.oh) % v == 0);
}

}  // namespace

// q [B, T, H, D] and k [B, T, Hk, D] (or none) with a dense last dimension,
// cos and sin [places, R/2] fp32, positions [B or 1, T] int64 or none.
std::vector<at::Tensor> rotary(const at::Tensor& q,
                               const c10::optional<at::Tensor>& k,
                               const at::Tensor& cos, const at::Tensor& sin,
                               const c10::optional<at::Tensor>& positions,
                               int64_t offset, bool interleaved, bool back) {
  TORCH_CHECK(q.is_cuda() && q.dim() == 4 && q.stride(3) == 1,
              "rotary: [B, T, H, D] with a dense last dimension on the GPU "
              "expected");
  const auto type = q.scalar_type();
  TORCH_CHECK(type == at::kBFloat16 || type == at::kHalf ||
                  type == at::kFloat,
              "rotary: bf16, fp16 or fp32 expected, got ", type);
  const long B = q.size(0), T = q.size(1), D = q.size(3);
  if (k.has_value()) {
    TORCH_CHECK(k->dim() == 4 && k->size(0) == B && k->size(1) == T &&
                    k->size(3) == D && k->stride(3) == 1 &&
                    k->scalar_type() == q.scalar_type() &&
                    k->device() == q.device(),
                "rotary: keys have to match the queries");
  }
  TORCH_CHECK(cos.dim() == 2 && cos.sizes() == sin.sizes() &&
                  cos.strides() == sin.strides() && cos.stride(1) == 1 &&
                  cos.scalar_type() == at::kFloat &&
                  sin.scalar_type() == at::kFloat &&
                  cos.device() == q.device() && sin.device() == q.device() &&
                  cos.size(0) >= 1,
              "rotary: fp32 tables [places, R/2] on the same device "
              "expected");
  const long R = 2 * cos.size(1);
  TORCH_CHECK(R >= 2 && R <= D && D <= 65536,
              "rotary: the tables turn more values than a head has");
  Places p;
  p.pos = nullptr;
  p.pb = p.pt = 0;
  p.offset = offset;
  p.rows = cos.size(0);
  if (positions.has_value()) {
    TORCH_CHECK(positions->dim() == 2 && positions->size(1) == T &&
                    (positions->size(0) == B || positions->size(0) == 1) &&
                    positions->scalar_type() == at::kLong &&
                    positions->device() == q.device(),
                "rotary: int64 positions [B or 1, T] expected");
    p.pos = positions->data_ptr<int64_t>();
    p.pb = positions->size(0) == 1 ? 0 : positions->stride(0);
    p.pt = positions->stride(1);
  }
  const c10::cuda::CUDAGuard guard(q.device());
  auto stream = at::cuda::getCurrentCUDAStream();
  // outputs in the order of the inputs' dimensions, without their gaps
  auto qo = at::empty_like(q, q.options(), at::MemoryFormat::Preserve);
  at::Tensor ko;
  Side sq, sk;
  auto settle = [&](const at::Tensor& in, at::Tensor& out) {
    if (out.stride(3) != 1)
      out = at::empty(in.sizes(), in.options());
    return side(in, out);
  };
  sq = settle(q, qo);
  if (k.has_value()) {
    ko = at::empty_like(*k, k->options(), at::MemoryFormat::Preserve);
    sk = settle(*k, ko);
  } else {
    sk = sq;
    sk.heads = 0;
  }
  std::vector<at::Tensor> res{qo};
  if (k.has_value()) res.push_back(ko);
  const long heads = sq.heads + sk.heads;
  if (B * T * heads == 0) return res;
  TORCH_CHECK(B * T < (1L << 31) && heads * D < (1L << 31),
              "rotary: too many tokens or heads");
  const int size = (int)q.element_size();
  auto launch = [&](auto tag, auto vec, auto rest, auto inter, auto al) {
    using E = decltype(tag);
    constexpr int V = decltype(vec)::value;
    constexpr bool I = decltype(inter)::value;
    constexpr int VR = decltype(rest)::value;
    const long work = (I ? R / V : R / (2 * V)) + (D - R) / VR;
    const long token = heads * work;
    // ~1024 pieces a workgroup: four loads in flight for a thread
    const long tpb = std::max(1L, 1024 / token);
    rotary_kernel<E, V, VR, I, decltype(al)::value>
        <<<(int)((B * T + tpb - 1) / tpb), 256, 0, stream>>>(
            sq, sk, p, cos.data_ptr<float>(), sin.data_ptr<float>(),
            cos.stride(0), back ? -1.f : 1.f, (unsigned)(B * T), (int)R,
            (unsigned)tpb, Div(T, B * T), Div(token, tpb * token),
            Div(work, token));
    HIP_CHECK_KERNEL();
  };
  auto ok = [&](int v) {
    const bool cut = interleaved ? R % v == 0 : R % (2 * v) == 0;
    return cut && D % v == 0 && fits(sq, v, size) && fits(sk, v, size);
  };
  auto run = [&](auto tag) {
    using E = decltype(tag);
    constexpr int W = 16 / sizeof(E);
    using Full = std::integral_constant<int, W>;
    using Two = std::integral_constant<int, 2>;
    using One = std::integral_constant<int, 1>;
    constexpr std::true_type yes{};
    constexpr std::false_type no{};
    if (interleaved) {
      if (ok(W)) {
        launch(E{}, Full{}, Full{}, yes, yes);
      } else {
        launch(E{}, Two{}, One{}, yes, no);
      }
    } else if (ok(W)) {
      launch(E{}, Full{}, Full{}, no, yes);
    } else {
      launch(E{}, One{}, One{}, no, no);
    }
  };
  if (type == at::kBFloat16) {
    run(c10::BFloat16{});
  } else if (type == at::kHalf) {
    run(c10::Half{});
  } else {
    run(float{});
  }
  return res;
}
