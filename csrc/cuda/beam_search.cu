// Beam search's selection on sm_100a.
#include <cfloat>

#include "ob/cuda_common.cuh"

namespace ob {
namespace cu {
namespace {

constexpr int kThreads = 256;

// One block per sentence.  First the log-sum-exp of every beam, then W rounds that each take the
// best candidate behind the one taken before (scores in float64, ties to the lowest place).
template <class T>
__global__ void __launch_bounds__(kThreads) beam_rounds_kernel(const T* __restrict__ logits, const float* __restrict__ scores,
                                                               const unsigned char* __restrict__ finished, float* out_scores,
                                                               long long* parents, long long* tokens, unsigned char* done, int W,
                                                               long long V, long long end) {
  __shared__ float smem[32];
  __shared__ double base[64];       // score - log-sum-exp; NaN: the beam has no candidate
  __shared__ double best[8];
  __shared__ long long place[8];
  const long long b = blockIdx.x;
  const T* x = logits + b * W * V;
  for (int w = 0; w < W; ++w) {
    const bool fin = finished != nullptr && finished[b * W + w] != 0;
    const float s = scores[b * W + w];
    float top = -INFINITY, bad = 0.f;
    if (!fin)
      for (long long v = threadIdx.x; v < V; v += kThreads) {
        const float y = to_f(x[w * V + v]);
        top = fmaxf(top, y);
        if (!(y <= FLT_MAX)) bad = 1.f;
      }
    top = block_max(top, smem);
    bad = block_max(bad, smem);
    double sum = 0.0;
    if (!fin && top > -INFINITY && bad == 0.f)
      for (long long v = threadIdx.x; v < V; v += kThreads) sum += expf(to_f(x[w * V + v]) - top);
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if ((threadIdx.x & 31) == 0) best[threadIdx.x >> 5] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int i = 1; i < kThreads / 32; ++i) sum += best[i];
      const bool dead = !isfinite(s) || (!fin && (bad != 0.f || !(top > -INFINITY)));
      base[w] = dead ? static_cast<double>(NAN) : fin ? s : s - (top + round_log_sum(log(sum)));
    }
    __syncthreads();
  }
  __syncthreads();
  double last = INFINITY;
  long long last_at = -1;
  for (int k = 0; k < W; ++k) {
    double mine = -INFINITY;
    long long at = W * V;  // behind every candidate
    for (long long i = threadIdx.x; i < W * V; i += kThreads) {
      const int w = static_cast<int>(i / V);
      const long long v = i - w * V;
      const bool fin = finished != nullptr && finished[b * W + w] != 0;
      double y = base[w];
      if (isnan(y)) y = -INFINITY;
      else if (fin) y = v == end ? y : -INFINITY;
      else y += to_f(x[i]);
      const bool behind = y < last || (y == last && i > last_at);
      if (behind && (at == W * V || y > mine)) { mine = y; at = i; }
    }
    for (int o = 16; o > 0; o >>= 1) {
      const double y = __shfl_xor_sync(0xffffffffu, mine, o);
      const long long i = __shfl_xor_sync(0xffffffffu, at, o);
      if (i < W * V && (at == W * V || y > mine || (y == mine && i < at))) { mine = y; at = i; }
    }
    if ((threadIdx.x & 31) == 0) { best[threadIdx.x >> 5] = mine; place[threadIdx.x >> 5] = at; }
    __syncthreads();
    mine = best[0];
    at = place[0];
    for (int i = 1; i < 8; ++i)
      if (place[i] < W * V && (at == W * V || best[i] > mine || (best[i] == mine && place[i] < at))) { mine = best[i]; at = place[i]; }
    __syncthreads();
    last = mine;
    last_at = at;
    if (threadIdx.x == 0) {
      const long long parent = at / V, token = at - parent * V, o = b * W + k;
      out_scores[o] = static_cast<float>(mine);
      parents[o] = parent;
      tokens[o] = token;
      done[o] = (end >= 0 && token == end) || (finished != nullptr && finished[b * W + parent] != 0);
    }
  }
}

template <class T>
void k_beam_step(OpCall& c) {
  const Shape& s = c.in[0].shape();
  if (s[0] > 2147483647LL) throw std::invalid_argument("beam_search_step: too many rows");
  beam_rounds_kernel<T><<<static_cast<unsigned>(s[0]), kThreads, 0, stream_of(c)>>>(
      c.in[0].data_as<T>(), c.in[1].data_as<float>(), c.in[2].defined() ? c.in[2].data_as<unsigned char>() : nullptr,
      c.out[0].data_as<float>(), c.out[1].data_as<long long>(), c.out[2].data_as<long long>(), c.out[3].data_as<unsigned char>(),
      static_cast<int>(s[1]), s[2], c.i[0]);
  check_launch("beam_search_step");
}

}  // namespace

void register_cuda_beam(KernelRegistry& r) {
  const uint8_t packed = kContiguous | kEmpty;
  r.add_kernel(OperatorId::BeamSearchStep, Constraints{Backend::CUDA, kMaskF32, packed, Capability::None}, k_beam_step<float>, "sm100_beam_search_step_f32");
  r.add_kernel(OperatorId::BeamSearchStep, Constraints{Backend::CUDA, dtype_bit(DType::F16), packed, Capability::None}, k_beam_step<__half>, "sm100_beam_search_step_f16");
  r.add_kernel(OperatorId::BeamSearchStep, Constraints{Backend::CUDA, dtype_bit(DType::BF16), packed, Capability::Bf16}, k_beam_step<__nv_bfloat16>, "sm100_beam_search_step_bf16");
}

}  // namespace cu
}  // namespace ob
