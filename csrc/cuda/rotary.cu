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
  long long rows;            // batch * tokens
  long long xs[3], ys[3];    // element strides of batch, token, head
  const void* positions;     // nullptr: the token index
  int positions_64, positions_batched;
  int tokens, heads, rotary_heads, head_dim, half;
  float sign, magnitude;
  int in_place;
  unsigned magic_units, magic_tail, magic_wide;  // see quotient()
  double turns[kMaxPairs];
};

template <class T, int VEC>
struct alignas(sizeof(T) * VEC) Vec {
  T v[VEC];
};

// n / d by a product with `magic` = ceil(2^32 / d), exact while n d < 2^32; 0: divide.
__device__ __forceinline__ int quotient(int n, int d, unsigned magic) {
  return magic != 0 ? static_cast<int>(__umulhi(static_cast<unsigned>(n), magic)) : n / d;
}

// A block takes TOKENS rows.  Each thread has one unit (VEC pairs of one head) to turn and one access to
// pass on in each of them; they are fetched first and are under way while the threads look up the
// positions and form the sines and cosines.  Rows with more units than a block has threads go
// round again.
template <class T, int VEC, bool INTER, int TOKENS>
__global__ void __launch_bounds__(kRotaryThreads) rotary_kernel(const T* x, T* y, const __grid_constant__ RotaryArgs a) {
  // `x` may be `y`: each value is read and written by one thread, the read first.
  using V = Vec<T, VEC>;
  static_assert(TOKENS <= 2, "the table is filled for two rows at most");
  constexpr int PAIRS = INTER ? (VEC + 1) / 2 : VEC;  // of one unit
  __shared__ float2 table[TOKENS * kMaxPairs];
  const long long row0 = static_cast<long long>(blockIdx.x) * TOKENS;
  const int rows = static_cast<int>(min(static_cast<long long>(TOKENS), a.rows - row0));
  int b = static_cast<int>(row0 / a.tokens), t = static_cast<int>(row0 - static_cast<long long>(b) * a.tokens);
  const T* xr[TOKENS];
  T* yr[TOKENS];
  int token[2];
#pragma unroll
  for (int k = 0; k < TOKENS; ++k) {
    xr[k] = x + (b * a.xs[0] + t * a.xs[1]);
    yr[k] = y + (b * a.ys[0] + t * a.ys[1]);
    token[k] = t;
    if (++t == a.tokens) { t = 0; ++b; }
  }
  const int first = blockIdx.y * kRotaryThreads + threadIdx.x, step = gridDim.y * kRotaryThreads;
  const int units = a.half / PAIRS, turned = a.rotary_heads * units;  // units to turn in a row
  const int tail = (a.head_dim - 2 * a.half) / VEC, tails = a.rotary_heads * tail, wide = a.head_dim / VEC;
  const int passed = a.in_place ? 0 : tails + (a.heads - a.rotary_heads) * wide;  // accesses to pass on in a row

  // The table holds pair j of unit u at j * units + u: neighbouring threads read neighbouring words.
  // Offset of unit i; of access i: first the tails of turned heads, then whole heads.
  auto unit_at = [&](int i, int* unit) {
    const int h = quotient(i, units, a.magic_units);
    *unit = i - h * units;
    return h;
  };
  auto access_at = [&](int i, long long* in, long long* out) {
    int h, u;
    if (i < tails) {
      h = quotient(i, tail, a.magic_tail);
      u = 2 * a.half + (i - h * tail) * VEC;
    } else {
      h = quotient(i - tails, wide, a.magic_wide);
      u = (i - tails - h * wide) * VEC;
      h += a.rotary_heads;
    }
    *in = h * a.xs[2] + u;
    *out = h * a.ys[2] + u;
  };

  V lo[TOKENS], hi[TOKENS], through[TOKENS];
  constexpr int kValues = INTER ? 2 * PAIRS : PAIRS;  // of a unit, where it begins
  int unit = 0;
  const int head = unit_at(first, &unit), at = unit * kValues;
  auto fetch = [&](const T* row, int h, int u, V* p, V* q) {
    const T* src = row + h * a.xs[2] + u;
    if constexpr (INTER && VEC == 1) {
      p->v[0] = src[0];
      q->v[0] = src[1];
    } else {
      *p = *reinterpret_cast<const V*>(src);
      if constexpr (!INTER) *q = *reinterpret_cast<const V*>(src + a.half);
    }
  };
  if (first < turned)
#pragma unroll
    for (int k = 0; k < TOKENS; ++k)
      if (k < rows) fetch(xr[k], head, at, &lo[k], &hi[k]);
  long long in = 0, out = 0;
  if (first < passed) {
    access_at(first, &in, &out);
#pragma unroll
    for (int k = 0; k < TOKENS; ++k)
      if (k < rows) through[k] = *reinterpret_cast<const V*>(xr[k] + in);
  }

  for (int j = threadIdx.x; j < TOKENS * a.half; j += kRotaryThreads) {
    const int k = TOKENS > 1 && j >= a.half ? 1 : 0, i = j - k * a.half;
    if (k >= rows) break;
    const int t_k = TOKENS > 1 && k == 1 ? token[1] : token[0];
    const long long place = a.positions_batched ? row0 + k : t_k;
    const double p = a.positions == nullptr ? static_cast<double>(t_k)
                     : a.positions_64       ? static_cast<double>(static_cast<const long long*>(a.positions)[place])
                                            : static_cast<double>(static_cast<const int*>(a.positions)[place]);
    const double u = p * a.turns[i];
    float s, c;
    sincospif(2.f * static_cast<float>(u - rint(u)), &s, &c);
    table[k * kMaxPairs + i % PAIRS * units + i / PAIRS] = make_float2(c * a.magnitude, s * a.magnitude * a.sign);
  }
  __syncthreads();

  auto turn = [&](T* row, int h, int u, const float2* cs, const V& p, const V& q) {
    T* dst = row + h * a.ys[2] + u;
    if constexpr (INTER && VEC == 1) {
      const float c = to_f(p.v[0]), d = to_f(q.v[0]);
      dst[0] = from_f<T>(c * cs[0].x - d * cs[0].y);
      dst[1] = from_f<T>(d * cs[0].x + c * cs[0].y);
    } else if constexpr (INTER) {
      V r;
#pragma unroll
      for (int j = 0; j < VEC / 2; ++j) {
        const float c = to_f(p.v[2 * j]), d = to_f(p.v[2 * j + 1]);
        r.v[2 * j] = from_f<T>(c * cs[j * units].x - d * cs[j * units].y);
        r.v[2 * j + 1] = from_f<T>(d * cs[j * units].x + c * cs[j * units].y);
      }
      *reinterpret_cast<V*>(dst) = r;
    } else {
      V r, s;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float c = to_f(p.v[j]), d = to_f(q.v[j]);
        r.v[j] = from_f<T>(c * cs[j * units].x - d * cs[j * units].y);
        s.v[j] = from_f<T>(d * cs[j * units].x + c * cs[j * units].y);
      }
      *reinterpret_cast<V*>(dst) = r;
      *reinterpret_cast<V*>(dst + a.half) = s;
    }
  };
  if (first < passed)
#pragma unroll
    for (int k = 0; k < TOKENS; ++k)
      if (k < rows) *reinterpret_cast<V*>(yr[k] + out) = through[k];
  if (first < turned)
#pragma unroll
    for (int k = 0; k < TOKENS; ++k)
      if (k < rows) turn(yr[k], head, at, table + k * kMaxPairs + unit, lo[k], hi[k]);
  for (int i = first + step; i < turned; i += step) {
    const int h = unit_at(i, &unit), u = unit * kValues;
#pragma unroll
    for (int k = 0; k < TOKENS; ++k)
      if (k < rows) fetch(xr[k], h, u, &lo[k], &hi[k]);
#pragma unroll
    for (int k = 0; k < TOKENS; ++k)
      if (k < rows) turn(yr[k], h, u, table + k * kMaxPairs + unit, lo[k], hi[k]);
  }
  for (int i = first + step; i < passed; i += step) {
    access_at(i, &in, &out);
#pragma unroll
    for (int k = 0; k < TOKENS; ++k)
      if (k < rows) *reinterpret_cast<V*>(yr[k] + out) = *reinterpret_cast<const V*>(xr[k] + in);
  }
}

unsigned magic_of(long long d, long long most) { return d > 1 && most * d < (1ll << 32) ? static_cast<unsigned>(((1ll << 32) + d - 1) / d) : 0u; }

template <class T, int VEC>
void launch_rotary(const T* x, T* y, RotaryArgs a, bool inter, int sms, cudaStream_t st) {
  const long long row = static_cast<long long>(a.heads) * a.head_dim;  // accesses of a row and more
  a.magic_units = magic_of(a.half / (inter ? (VEC + 1) / 2 : VEC), row + 65536);
  a.magic_tail = magic_of((a.head_dim - 2 * a.half) / VEC, row + 65536);
  a.magic_wide = magic_of(a.head_dim / VEC, row + 65536);
  // Enough rows for the device: two to a block.  Few rows leave most SMs without a block: their heads
  // are spread over several.
  if (a.rows >= 16ll * sms) {
    const unsigned grid = static_cast<unsigned>((a.rows + 1) / 2);
    if (inter) rotary_kernel<T, VEC, true, 2><<<grid, kRotaryThreads, 0, st>>>(x, y, a);
    else rotary_kernel<T, VEC, false, 2><<<grid, kRotaryThreads, 0, st>>>(x, y, a);
    return;
  }
  long long gy = a.rows >= sms ? 1 : (row / VEC + kRotaryThreads - 1) / kRotaryThreads;
  if (gy > 64) gy = 64;
  const dim3 grid(static_cast<unsigned>(a.rows), static_cast<unsigned>(gy < 1 ? 1 : gy));
  if (inter) rotary_kernel<T, VEC, true, 1><<<grid, kRotaryThreads, 0, st>>>(x, y, a);
  else rotary_kernel<T, VEC, false, 1><<<grid, kRotaryThreads, 0, st>>>(x, y, a);
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
  a.rows = rows;
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
    if (grain % 8 == 0) { launch_rotary<T, 8>(px, py, a, inter, sms, st); check_launch("rotary_embedding"); return; }
  }
  if (grain % 4 == 0) launch_rotary<T, 4>(px, py, a, inter, sms, st);
  else if (grain % 2 == 0) launch_rotary<T, 2>(px, py, a, inter, sms, st);
  else launch_rotary<T, 1>(px, py, a, inter, sms, st);
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
