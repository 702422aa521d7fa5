// Rotary positions on sm_100a.
//
// A pair (a, b) of a head at position p is turned by the angle t = 2 pi p f_i:
//   a' = m (a cos t - b sin t),  b' = m (b cos t + a sin t).
// The transposed map (the gradient) is the same with -t.  Pairs are (i, i + R/2), or (2i, 2i + 1)
// when interleaved; values behind R and heads behind `rotary_heads` pass through.
//
// Bound by memory: every value is read once and written once.  The angles are shared by all heads
// of a token, so a block takes one token or a few, forms their sines and cosines once, in shared memory,
// and applies them to all heads; the heads' values are fetched before and arrive meanwhile.  The turn
// count p f_i is formed in float64 (a position of a million times a frequency of one loses 0.06 rad in
// float32) and reduced to half a turn before it is rounded to float32, which costs three float64
// operations per pair and token.  From there on float32: a float32 result is off by 5.7e-8 of its size, where sines
// and cosines in float64 would leave 4.2e-8; 16-bit results are the same.
//
// Measured, calls one after another (bfloat16): 8192 tokens of 48 heads of 128, 201 MB read and written in 39 us
// (5.1 TB/s; a plain copy takes 31).  Without any arithmetic the same structure takes 36: blocks that live for one row
// leave the memory idle while they start and end.  32768 tokens of 4 heads of 64: 18.6 us (66 with a block for each row;
// 5 by their bytes).  float32, 8191 tokens of 8 heads of 64, neighbouring pairs, 48 values turned: 12.3 us for 33.5 MB
// (5.1): 70 % of the issue slots are taken, 247 instructions for each warp, which moves 16 or 32 bytes a lane; they are places,
// divisions of the index and the angles.  A few rows cost a call, 4.7 us, of which the launch is most.
#include <algorithm>

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
  int rows;                  // batch * tokens
  int tokens, heads, rotary_heads, head_dim, half;
  float sign, magnitude;
  int in_place;
  int sets;
  unsigned magic_units, magic_tail, magic_wide, magic_turned, magic_passed, magic_half, magic_tokens;  // see quotient()
  double turns[kMaxPairs];
};

template <class T, int VEC>
struct alignas(sizeof(T) * VEC) Vec {
  T v[VEC];
};

// Rows narrower than a block stand beside each other in `sets` of it; rows with more units (VEC pairs of one
// head to turn) than the block has threads go round again.  Each thread has one unit to turn and one access to
// pass on, of one row each; they are fetched first and are under way while the threads look up the
// positions and form the sines and cosines.
//
// Six blocks on an SM, by a bound on the registers: 8192 rows of 48 heads of 128 take 39 us (46 with what
// they would allow), 32768 of 8 heads of 256 76 (82).  One row at a time:
// with two for each thread 32768 tokens of 8 heads of 256 take 87 us in place of 77, 4 of 64 23 in place of 19.
template <class T, int VEC, bool INTER, bool SETS>  // SETS: more than one
__global__ void __launch_bounds__(kRotaryThreads, 6) rotary_kernel(const T* x, T* y, const __grid_constant__ RotaryArgs a) {
  // `x` may be `y`: each value is read and written by one thread, the read first.
  using V = Vec<T, VEC>;
  constexpr int PAIRS = INTER ? (VEC + 1) / 2 : VEC;  // of one unit
  constexpr int kValues = INTER ? 2 * PAIRS : PAIRS;  // of a unit, where it begins
  extern __shared__ float2 table[];  // of row k, pair j of unit u at k * half + j * units + u: neighbouring threads read neighbouring words
  const int row0 = blockIdx.x * (SETS ? a.sets : 1), rows = SETS ? min(a.sets, a.rows - row0) : 1;
  const int b0 = static_cast<unsigned>(row0) / static_cast<unsigned>(a.tokens), t0 = row0 - b0 * a.tokens;
  const int units = a.half / PAIRS, turned = a.rotary_heads * units;  // units to turn in a row
  const int tail = (a.head_dim - 2 * a.half) / VEC, tails = a.rotary_heads * tail, wide = a.head_dim / VEC;
  const int passed = a.in_place ? 0 : tails + (a.heads - a.rotary_heads) * wide;  // accesses to pass on in a row

  // Row k of the block: its sequence and token; where it begins.
  auto token_of = [&](int k, int* b) {
    int t = t0 + k;
    *b = b0;
    if (SETS && t >= a.tokens) {
      const int over = quotient(t, a.tokens, a.magic_tokens);
      *b += over;
      t -= over * a.tokens;
    }
    return t;
  };
  auto row_of = [&](auto* data, const long long (&strides)[3], int k) {
    int b;
    const int t = token_of(k, &b);
    return data + (b * strides[0] + t * strides[1]);
  };
  // Offset of unit i of a row; of access i: first the tails of turned heads, then whole heads.
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

  // With several sets a row is no wider than the block: (set, unit) and (set, access) of this thread.
  // Threads behind the last set belong to no row.
  int first = blockIdx.y * kRotaryThreads + threadIdx.x, first_pass = first, set = 0, set_pass = 0;
  const int step = gridDim.y * kRotaryThreads;
  if constexpr (SETS) {
    set = quotient(first, turned, a.magic_turned);
    first -= set * turned;
    if (passed > 0) {
      set_pass = quotient(first_pass, passed, a.magic_passed);
      first_pass -= set_pass * passed;
    }
  }
  const T *xr = row_of(x, a.xs, set), *xp = SETS ? row_of(x, a.xs, set_pass) : xr;
  T *yr = row_of(y, a.ys, set), *yp = SETS ? row_of(y, a.ys, set_pass) : yr;
  V lo, hi, through;
  int unit = 0;
  const int head = unit_at(first, &unit), at = unit * kValues;
  const bool turns = first < turned && set < rows, passes = first_pass < passed && set_pass < rows;
  if (turns) fetch(xr, head, at, &lo, &hi);
  long long in = 0, out = 0;
  if (passes) {
    access_at(first_pass, &in, &out);
    through = *reinterpret_cast<const V*>(xp + in);
  }
  for (int j = threadIdx.x; j < rows * a.half; j += kRotaryThreads) {
    const int k = !SETS ? 0 : quotient(j, a.half, a.magic_half), i = j - k * a.half;
    int b;
    const int t = token_of(k, &b);
    const long long place = a.positions_batched ? static_cast<long long>(row0) + k : t;
    const double p = a.positions == nullptr ? static_cast<double>(t)
                     : a.positions_64       ? static_cast<double>(static_cast<const long long*>(a.positions)[place])
                                            : static_cast<double>(static_cast<const int*>(a.positions)[place]);
    const double u = p * a.turns[i];
    float s, c;
    sincospif(2.f * static_cast<float>(u - rint(u)), &s, &c);
    table[k * a.half + i % PAIRS * units + i / PAIRS] = make_float2(c * a.magnitude, s * a.magnitude * a.sign);
  }
  __syncthreads();
  if (passes) *reinterpret_cast<V*>(yp + out) = through;
  if (turns) turn(yr, head, at, table + set * a.half + unit, lo, hi);
  if constexpr (SETS) return;
  for (int i = first + step; i < turned; i += step) {
    const int h = unit_at(i, &unit), u = unit * kValues;
    fetch(xr, h, u, &lo, &hi);
    turn(yr, h, u, table + unit, lo, hi);
  }
  for (int i = first_pass + step; i < passed; i += step) {
    access_at(i, &in, &out);
    *reinterpret_cast<V*>(yr + out) = *reinterpret_cast<const V*>(xr + in);
  }
}

template <class T, int VEC>
void launch_rotary(const T* x, T* y, RotaryArgs a, bool inter, int sms, cudaStream_t st) {
  const long long units = a.half / (inter ? (VEC + 1) / 2 : VEC), turned = a.rotary_heads * units;
  const long long tail = (a.head_dim - 2 * a.half) / VEC, wide = a.head_dim / VEC, passed = a.in_place ? 0 : a.rotary_heads * tail + (a.heads - a.rotary_heads) * wide;
  const long long work = std::max(turned, passed);
  // As many sets as threads have work, while the device keeps several blocks for each SM (8191 rows of 8 heads of
  // 64 in float32: 10.4 us with 4 sets, 12.5 with 2, 16.5 with one).
  a.sets = static_cast<int>(std::max(1ll, std::min<long long>(kRotaryThreads / work, a.rows / (4ll * sms))));
  // Few rows leave most SMs without a block: their heads are spread over several.
  const long long gy = a.rows >= sms ? 1 : std::min(64ll, (work + kRotaryThreads - 1) / kRotaryThreads);
  const long long most = work + 65536;  // of the indices, and more
  a.magic_units = magic_of(units, most);
  a.magic_tail = magic_of(tail, most);
  a.magic_wide = magic_of(wide, most);
  a.magic_turned = magic_of(turned, most);
  a.magic_passed = magic_of(passed, most);
  a.magic_half = magic_of(a.half, static_cast<long long>(a.sets) * a.half);
  a.magic_tokens = magic_of(a.tokens, static_cast<long long>(a.tokens) + a.sets);
  const dim3 grid(static_cast<unsigned>((a.rows + a.sets - 1) / a.sets), static_cast<unsigned>(gy));
  const size_t smem = static_cast<size_t>(a.sets) * a.half * sizeof(float2);  // half <= VEC work: 16 KB at most
  auto launch = [&](auto kernel) { kernel<<<grid, kRotaryThreads, smem, st>>>(x, y, a); };
  if (a.sets > 1) inter ? launch(rotary_kernel<T, VEC, true, true>) : launch(rotary_kernel<T, VEC, false, true>);
  else inter ? launch(rotary_kernel<T, VEC, true, false>) : launch(rotary_kernel<T, VEC, false, false>);
}

template <class T>
void k_rotary(OpCall& c) {
  const Tensor &x = c.in[0], &pos = c.in[1], &turns = c.in[2];
  Tensor& y = c.out[0];
  RotaryArgs a{};
  const long long rows = x.shape()[0] * x.shape()[1];
  if (rows > 1073741823LL || x.shape()[2] * x.shape()[3] > 1073741823LL)
    throw std::invalid_argument("rotary_embedding: too many tokens or too wide a row");
  const bool inter = c.i[1] != 0;
  a.rows = static_cast<int>(rows);
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
