// Attention of one new token over the paged key-value cache (sm_100a).
//
// o = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q k_j - m),  m the running maximum, in one pass
// over keys and values.
#include "ob/cuda_common.cuh"

namespace ob {
namespace cu {
namespace {

struct PagedArgs {
  const void *q, *k, *v;
  void* out;
  const int *table, *lengths;
  unsigned int* errors;
  long long qs[2], page_stride[2];  // batch and head of q; keys, values
  int heads, kv_heads, head_dim, page_size, table_width, pages_total;
  float scale_log2;                 // scale * log2(e)
};

// Any type, head size and page size: a warp takes every fourth token, its lanes share the row.
constexpr int kWarps = 4;
template <class T, int PER_LANE>
__global__ void __launch_bounds__(kWarps * 32) paged_rows_kernel(const __grid_constant__ PagedArgs a) {
  __shared__ float part[kWarps][PER_LANE * 32 + 2];
  const int b = blockIdx.x / a.heads, h = blockIdx.x - b * a.heads, kv = h / (a.heads / a.kv_heads);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, D = a.head_dim;
  const long long most = a.pages_total > 0 ? static_cast<long long>(a.table_width) * a.page_size : 0;
  long long n = a.lengths[b];
  if (n < 0 || n > most) {
    if (threadIdx.x == 0) atomicAdd(a.errors, 1u);
    n = n < 0 ? 0 : most;
  }
  const T* q = static_cast<const T*>(a.q) + b * a.qs[0] + h * a.qs[1];
  float qv[PER_LANE], acc[PER_LANE], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < PER_LANE; ++i) {
    const int d = i * 32 + lane;
    qv[i] = d < D ? to_f(q[d]) * a.scale_log2 : 0.f;
    acc[i] = 0.f;
  }
  for (long long j = warp; j < n; j += kWarps) {
    const long long slot = j / a.page_size;
    int page = a.table[static_cast<long long>(b) * a.table_width + slot];
    if (page < 0 || page >= a.pages_total) {
      if (lane == 0) atomicAdd(a.errors, 1u);
      page = page < 0 ? 0 : a.pages_total - 1;
    }
    const long long row = (static_cast<long long>(kv) * a.page_size + (j - slot * a.page_size)) * D;
    const T* k = static_cast<const T*>(a.k) + page * a.page_stride[0] + row;
    const T* v = static_cast<const T*>(a.v) + page * a.page_stride[1] + row;
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < PER_LANE; ++i) {
      const int d = i * 32 + lane;
      if (d < D) dot = fmaf(qv[i], to_f(k[d]), dot);
    }
    dot = warp_sum(dot);
    const float top = fmaxf(m, dot);
    // A score of -inf weighs nothing whatever the maximum is so far; NaN stays NaN.
    const float keep = m == top ? 1.f : exp2f(m - top), p = dot == -INFINITY ? 0.f : exp2f(dot - top);
    l = l * keep + p;
    m = top;
#pragma unroll
    for (int i = 0; i < PER_LANE; ++i) {
      const int d = i * 32 + lane;
      if (d < D) acc[i] = fmaf(p, to_f(v[d]), acc[i] * keep);
    }
  }
#pragma unroll
  for (int i = 0; i < PER_LANE; ++i) part[warp][i * 32 + lane] = acc[i];
  if (lane == 0) { part[warp][PER_LANE * 32] = m; part[warp][PER_LANE * 32 + 1] = l; }
  __syncthreads();
  float top = -INFINITY, sum = 0.f, w[kWarps];
  for (int i = 0; i < kWarps; ++i) top = fmaxf(top, part[i][PER_LANE * 32]);
  for (int i = 0; i < kWarps; ++i) {
    w[i] = part[i][PER_LANE * 32] == top ? 1.f : exp2f(part[i][PER_LANE * 32] - top);
    sum += w[i] * part[i][PER_LANE * 32 + 1];
  }
  T* out = static_cast<T*>(a.out) + static_cast<long long>(blockIdx.x) * D;
  for (int d = threadIdx.x; d < D; d += kWarps * 32) {
    float o = 0.f;
    for (int i = 0; i < kWarps; ++i) o += w[i] * part[i][d];
    out[d] = from_f<T>(n == 0 ? 0.f : o / sum);
  }
}

template <class T>
void k_paged_attention(OpCall& c) {
  const Tensor &q = c.in[0], &kp = c.in[1], &vp = c.in[2];
  const Shape& s = kp.shape();
  const long long B = q.shape()[0], H = q.shape()[1];
  if (B * H > 2147483647LL || s[0] > 2147483647LL || c.in[3].shape()[1] > 2147483647LL)
    throw std::invalid_argument("paged_attention: too many heads or pages");
  PagedArgs a{};
  a.q = q.data(); a.k = kp.data(); a.v = vp.data(); a.out = c.out[0].data();
  a.table = c.in[3].data_as<int>();
  a.lengths = c.in[4].data_as<int>();
  a.errors = index_error_counter();
  for (int d = 0; d < 2; ++d) a.qs[d] = q.shape()[d] > 1 ? q.strides()[d] : 0;
  a.page_stride[0] = kp.strides()[0];
  a.page_stride[1] = vp.strides()[0];
  a.heads = static_cast<int>(H);
  a.kv_heads = static_cast<int>(s[1]);
  a.head_dim = static_cast<int>(s[3]);
  a.page_size = static_cast<int>(s[2]);
  a.table_width = static_cast<int>(c.in[3].shape()[1]);
  a.pages_total = static_cast<int>(s[0]);
  a.scale_log2 = static_cast<float>(c.f[0] * 1.4426950408889634);
  const unsigned grid = static_cast<unsigned>(B * H);
  cudaStream_t st = stream_of(c);
  if (s[3] <= 64) paged_rows_kernel<T, 2><<<grid, kWarps * 32, 0, st>>>(a);
  else if (s[3] <= 128) paged_rows_kernel<T, 4><<<grid, kWarps * 32, 0, st>>>(a);
  else paged_rows_kernel<T, 8><<<grid, kWarps * 32, 0, st>>>(a);
  check_launch("paged_attention");
}

}  // namespace

void register_cuda_paged_attention(KernelRegistry& r) {
  const uint8_t packed = kContiguous | kEmpty;
  r.add_kernel(OperatorId::PagedAttention, Constraints{Backend::CUDA, kMaskF32, packed, Capability::None}, k_paged_attention<float>, "sm100_paged_attention_f32");
  r.add_kernel(OperatorId::PagedAttention, Constraints{Backend::CUDA, dtype_bit(DType::F16), packed, Capability::None}, k_paged_attention<__half>, "sm100_paged_attention_f16");
  r.add_kernel(OperatorId::PagedAttention, Constraints{Backend::CUDA, dtype_bit(DType::BF16), packed, Capability::Bf16}, k_paged_attention<__nv_bfloat16>, "sm100_paged_attention_bf16");
}

}  // namespace cu
}  // namespace ob
