// Rotary positions on sm_100a.
//
// A pair (a, b) of a head at position p is turned by the angle t = 2 pi p f_i:
//   a' = m (a cos t - b sin t),  b' = m (b cos t + a sin t).
// The transposed map (the gradient) is the same with -t.  Pairs are (i, i + R/2), or (2i, 2i + 1)
// when interleaved; values behind R and heads behind `rotary_heads` pass through.
//
// Bound by memory: every value is read once and written once.  The angles are shared by all heads
// of a token, so a block takes one token, its first R/2 threads compute that token's sines and
// cosines once, and the whole block applies them.  The turn count p f_i is formed in float64 (a
// position of a million times a frequency of one loses 0.06 rad in float32) and reduced to half a
// turn before it is rounded to float32, which costs three float64 operations per pair and token.
#include "ob/cuda_common.cuh"

namespace ob {
namespace cu {
namespace {

constexpr int kMaxPairs = 256;
constexpr int kRotaryThreads = 256;

struct RotaryArgs {
  long long xs[3], ys[3];    // element strides of batch, token, head
  const void* positions;     // nullptr: the token index
  int positions_64, positions_batched;
  int tokens, heads, rotary_heads, head_dim, half;
  float sign, magnitude;
  int in_place;
  double turns[kMaxPairs];
};

template <class T, int VEC>
struct alignas(sizeof(T) * VEC) Vec {
  T v[VEC];
};

template <class T, int VEC, bool INTER>
__global__ void __launch_bounds__(kRotaryThreads) rotary_kernel(const T* x, T* y, const __grid_constant__ RotaryArgs a) {
  // `x` may be `y`: each value is read and written by one thread, the read first.
  using V = Vec<T, VEC>;
  __shared__ float2 table[kMaxPairs];
  const int b = blockIdx.x / a.tokens, t = blockIdx.x - b * a.tokens;
  const T* xt = x + b * a.xs[0] + t * a.xs[1];
  T* yt = y + b * a.ys[0] + t * a.ys[1];

  if (threadIdx.x < a.half) {
    const long long at = a.positions_batched ? blockIdx.x : t;
    const double p = a.positions == nullptr ? static_cast<double>(t)
                     : a.positions_64       ? static_cast<double>(static_cast<const long long*>(a.positions)[at])
                                            : static_cast<double>(static_cast<const int*>(a.positions)[at]);
    const double u = p * a.turns[threadIdx.x];
    float s, c;
    sincospif(2.f * static_cast<float>(u - rint(u)), &s, &c);
    table[threadIdx.x] = make_float2(c * a.magnitude, s * a.magnitude * a.sign);
  }
  __syncthreads();

  // Turned pairs: a unit is VEC pairs of one head.
  constexpr int PAIRS = INTER ? (VEC + 1) / 2 : VEC;  // of one unit
  const int units = a.half / PAIRS;
  const int items = units * a.rotary_heads;
  for (int i = blockIdx.y * kRotaryThreads + threadIdx.x; i < items; i += gridDim.y * kRotaryThreads) {
    const int h = i / units, u = (i - h * units) * (INTER ? 2 * PAIRS : PAIRS);
    const T* src = xt + h * a.xs[2] + u;
    T* dst = yt + h * a.ys[2] + u;
    if constexpr (INTER && VEC == 1) {
      const float2 cs = table[u / 2];
      const float p = to_f(src[0]), q = to_f(src[1]);
      dst[0] = from_f<T>(p * cs.x - q * cs.y);
      dst[1] = from_f<T>(q * cs.x + p * cs.y);
    } else if constexpr (INTER) {
      const V in = *reinterpret_cast<const V*>(src);
      V out;
#pragma unroll
      for (int k = 0; k < VEC / 2; ++k) {
        const float2 cs = table[u / 2 + k];
        const float p = to_f(in.v[2 * k]), q = to_f(in.v[2 * k + 1]);
        out.v[2 * k] = from_f<T>(p * cs.x - q * cs.y);
        out.v[2 * k + 1] = from_f<T>(q * cs.x + p * cs.y);
      }
      *reinterpret_cast<V*>(dst) = out;
    } else {
      const V lo = *reinterpret_cast<const V*>(src), hi = *reinterpret_cast<const V*>(src + a.half);
      V olo, ohi;
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        const float2 cs = table[u + k];
        const float p = to_f(lo.v[k]), q = to_f(hi.v[k]);
        olo.v[k] = from_f<T>(p * cs.x - q * cs.y);
        ohi.v[k] = from_f<T>(q * cs.x + p * cs.y);
      }
      *reinterpret_cast<V*>(dst) = olo;
      *reinterpret_cast<V*>(dst + a.half) = ohi;
    }
  }
  if (a.in_place) return;
  // Values that pass through: the tails of turned heads, then whole heads.
  const int tail = (a.head_dim - 2 * a.half) / VEC, tails = tail * a.rotary_heads;
  for (int i = blockIdx.y * kRotaryThreads + threadIdx.x; i < tails; i += gridDim.y * kRotaryThreads) {
    const int h = i / tail, u = 2 * a.half + (i - h * tail) * VEC;
    *reinterpret_cast<V*>(yt + h * a.ys[2] + u) = *reinterpret_cast<const V*>(xt + h * a.xs[2] + u);
  }
  const int row = a.head_dim / VEC, rest = row * (a.heads - a.rotary_heads);
  for (int i = blockIdx.y * kRotaryThreads + threadIdx.x; i < rest; i += gridDim.y * kRotaryThreads) {
    const int k = i / row, h = a.rotary_heads + k, u = (i - k * row) * VEC;
    *reinterpret_cast<V*>(yt + h * a.ys[2] + u) = *reinterpret_cast<const V*>(xt + h * a.xs[2] + u);
  }
}

template <class T, int VEC>
void launch_rotary(const T* x, T* y, const RotaryArgs& a, bool inter, long long rows, int sms, cudaStream_t st) {
  // Few tokens leave most SMs without a block: their heads are spread over several.
  const long long units = static_cast<long long>(a.heads) * a.head_dim / VEC;
  long long gy = rows >= sms ? 1 : (units + kRotaryThreads - 1) / kRotaryThreads;
  if (gy > 64) gy = 64;
  const dim3 grid(static_cast<unsigned>(rows), static_cast<unsigned>(gy < 1 ? 1 : gy));
  if (inter) rotary_kernel<T, VEC, true><<<grid, kRotaryThreads, 0, st>>>(x, y, a);
  else rotary_kernel<T, VEC, false><<<grid, kRotaryThreads, 0, st>>>(x, y, a);
}

template <class T>
void k_rotary(OpCall& c) {
  const Tensor &x = c.in[0], &pos = c.in[1], &turns = c.in[2];
  Tensor& y = c.out[0];
  RotaryArgs a{};
  const long long rows = x.shape()[0] * x.shape()[1];
  if (rows > 2147483647LL || x.shape()[2] * x.shape()[3] > 2147483647LL)
    throw std::invalid_argument("rotary_embedding: too many tokens or too wide a row");
  const bool inter = c.i[1] != 0;
  a.half = static_cast<int>(turns.numel());
  a.tokens = static_cast<int>(x.shape()[1]);
  a.heads = static_cast<int>(x.shape()[2]);
  a.rotary_heads = static_cast<int>(c.i[0]);
  a.head_dim = static_cast<int>(x.shape()[3]);
  a.sign = static_cast<float>(c.f[0]);
  a.magnitude = static_cast<float>(c.f[1]);
  a.in_place = static_cast<int>(c.i[2]);
  if (pos.defined()) {
    a.positions = pos.data();
    a.positions_64 = pos.dtype() == DType::I64;
    a.positions_batched = pos.ndim() == 2;
  }
  for (int i = 0; i < a.half; ++i) a.turns[i] = turns.data_as<double>()[i];
  // The widest access that every row, pair half and tail allows.
  long long grain = a.head_dim | (inter ? 2 * a.half : a.half) | static_cast<long long>(reinterpret_cast<uintptr_t>(x.data()) / sizeof(T)) |
                    static_cast<long long>(reinterpret_cast<uintptr_t>(y.data()) / sizeof(T));
  for (int d = 0; d < 3; ++d) {
    a.xs[d] = x.shape()[d] > 1 ? x.strides()[d] : 0;
    a.ys[d] = y.shape()[d] > 1 ? y.strides()[d] : 0;
    grain |= a.xs[d] | a.ys[d];
  }
  const T* px = x.data_as<T>();
  T* py = y.data_as<T>();
  const int sms = sm_count_for(x);
  cudaStream_t st = stream_of(c);
  if constexpr (sizeof(T) == 2) {
    if (grain % 8 == 0) { launch_rotary<T, 8>(px, py, a, inter, rows, sms, st); check_launch("rotary_embedding"); return; }
  }
  if (grain % 4 == 0) launch_rotary<T, 4>(px, py, a, inter, rows, sms, st);
  else if (grain % 2 == 0) launch_rotary<T, 2>(px, py, a, inter, rows, sms, st);
  else launch_rotary<T, 1>(px, py, a, inter, rows, sms, st);
  check_launch("rotary_embedding");
}

}  // namespace

void register_cuda_rotary(KernelRegistry& r) {
  const uint8_t any = kContiguous | kStrided | kEmpty;
  r.add_kernel(OperatorId::RotaryEmbedding, Constraints{Backend::CUDA, kMaskF32, any, Capability::None}, k_rotary<float>, "sm100_rotary_embedding_f32");
  r.add_kernel(OperatorId::RotaryEmbedding, Constraints{Backend::CUDA, dtype_bit(DType::F16), any, Capability::None}, k_rotary<__half>, "sm100_rotary_embedding_f16");
  r.add_kernel(OperatorId::RotaryEmbedding, Constraints{Backend::CUDA, dtype_bit(DType::BF16), any, Capability::Bf16}, k_rotary<__nv_bfloat16>, "sm100_rotary_embedding_bf16");
}

}  // namespace cu
}  // namespace ob
