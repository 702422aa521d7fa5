// The paged key-value cache on sm_100a: new rows into their pages, copies of whole pages.
//
// Pages are [N, H, P, D]: the P rows of one head lie together, so that attention reads a page of a
// head as one contiguous block.  Both operators only move bytes; each byte is read once and
// written once.
#include <algorithm>

#include "ob/cuda_common.cuh"

namespace ob {
namespace cu {
namespace {

constexpr int kThreads = 256;

// ---------------------------------------------------------------------- append
struct AppendArgs {
  char* pages[2];             // keys, values
  const char* rows[2];
  long long page_stride[2];   // in units (accesses of one thread)
  long long rs[2][3];         // batch, token, head strides of the rows, in units
  const int *table, *starts, *counts;
  unsigned int* errors;
  int tokens, heads, page_size, units, table_width, pages_total;
};

// One block per token and side: the token's page is looked up once, then all heads are moved.
template <class U>
__global__ void __launch_bounds__(kThreads) append_kernel(const __grid_constant__ AppendArgs a) {
  const int b = blockIdx.x / a.tokens, t = blockIdx.x - b * a.tokens, side = blockIdx.y;
  if (a.counts != nullptr && t >= a.counts[b]) return;
  const long long at = static_cast<long long>(a.starts[b]) + t;
  const long long slot = at / a.page_size;
  int page = -1;
  if (at >= 0 && slot < a.table_width) page = a.table[static_cast<long long>(b) * a.table_width + slot];
  if (page < 0 || page >= a.pages_total) {  // never written: the row has no place
    if (threadIdx.x == 0 && side == 0) atomicAdd(a.errors, 1u);
    return;
  }
  U* dst = reinterpret_cast<U*>(a.pages[side]) + page * a.page_stride[side] + (at - slot * a.page_size) * a.units;
  const U* src = reinterpret_cast<const U*>(a.rows[side]) + b * a.rs[side][0] + t * a.rs[side][1];
  const int items = a.heads * a.units;
  for (int i = threadIdx.x; i < items; i += kThreads) {
    const int h = i / a.units, u = i - h * a.units;
    dst[static_cast<long long>(h) * a.page_size * a.units + u] = src[h * a.rs[side][2] + u];
  }
}

// The widest of 16, 8, 4 and 2 bytes that divides every address, row and stride.
int access_bytes(unsigned long long bits) {
  for (int w : {16, 8, 4})
    if (bits % w == 0) return w;
  return 2;
}

void k_paged_append(OpCall& c) {
  const Shape &s = c.in[0].shape(), &r = c.in[2].shape();
  const long long size = static_cast<long long>(dtype_size(c.in[0].dtype())), row = s[3] * size;
  unsigned long long bits = static_cast<unsigned long long>(row);
  for (int i = 0; i < 4; ++i) {
    bits |= reinterpret_cast<uintptr_t>(c.in[i].data());
    for (int d = 0; d < (i < 2 ? 1 : 3); ++d)
      if (c.in[i].shape()[d] > 1) bits |= static_cast<unsigned long long>(c.in[i].strides()[d] * size);
  }
  const int w = access_bytes(bits);
  if (s[0] > 2147483647LL || r[0] * r[1] > 2147483647LL || s[1] * row / w > 2147483647LL)
    throw std::invalid_argument("paged_append_: too many pages, tokens or values in a row");
  AppendArgs a{};
  for (int side = 0; side < 2; ++side) {
    a.pages[side] = c.in[side].data_as<char>();
    a.rows[side] = c.in[2 + side].data_as<char>();
    a.page_stride[side] = c.in[side].strides()[0] * size / w;
    for (int d = 0; d < 3; ++d) a.rs[side][d] = r[d] > 1 ? c.in[2 + side].strides()[d] * size / w : 0;
  }
  a.table = c.in[4].data_as<int>();
  a.starts = c.in[5].data_as<int>();
  a.counts = c.in[6].defined() ? c.in[6].data_as<int>() : nullptr;
  a.errors = index_error_counter();
  a.tokens = static_cast<int>(r[1]);
  a.heads = static_cast<int>(s[1]);
  a.page_size = static_cast<int>(s[2]);
  a.units = static_cast<int>(row / w);
  a.table_width = static_cast<int>(c.in[4].shape()[1]);
  a.pages_total = static_cast<int>(s[0]);
  const dim3 grid(static_cast<unsigned>(r[0] * r[1]), 2);
  cudaStream_t st = stream_of(c);
  if (w == 16) append_kernel<uint4><<<grid, kThreads, 0, st>>>(a);
  else if (w == 8) append_kernel<uint2><<<grid, kThreads, 0, st>>>(a);
  else if (w == 4) append_kernel<unsigned int><<<grid, kThreads, 0, st>>>(a);
  else append_kernel<unsigned short><<<grid, kThreads, 0, st>>>(a);
  check_launch("paged_append_");
}

// ------------------------------------------------------------------ page copies
// The pairs travel in the launch's parameters: no list is sent to the device first.
constexpr int kPairs = 440;
struct CopyArgs {
  char* base;
  long long page_units, outer_units;  // one page; all pages of one outer index
  int2 pair[kPairs];                  // (source, destination)
};
constexpr int kInFlight = 4;          // accesses of a thread that are under way together

template <class U>
__global__ void __launch_bounds__(kThreads) copy_pages_kernel(const __grid_constant__ CopyArgs a) {
  const int2 p = a.pair[blockIdx.y];
  U* base = reinterpret_cast<U*>(a.base) + blockIdx.z * a.outer_units;
  const U* src = base + p.x * a.page_units;
  U* dst = base + p.y * a.page_units;
  const long long first = static_cast<long long>(blockIdx.x) * kThreads * kInFlight + threadIdx.x;
  U v[kInFlight];
#pragma unroll
  for (int k = 0; k < kInFlight; ++k)
    if (first + k * kThreads < a.page_units) v[k] = src[first + k * kThreads];
#pragma unroll
  for (int k = 0; k < kInFlight; ++k)
    if (first + k * kThreads < a.page_units) dst[first + k * kThreads] = v[k];
}

template <class U>
void launch_copies(OpCall& c) {
  const long long n = static_cast<long long>(c.list.size()) / 2, page = c.i[2] / static_cast<long long>(sizeof(U));
  const long long blocks = (page + kThreads * kInFlight - 1) / (kThreads * kInFlight);
  CopyArgs a;
  a.page_units = page;
  a.outer_units = page * c.i[1];
  for (long long z = 0; z < c.i[0]; z += 65535)
    for (long long i = 0; i < n; i += kPairs) {
      const int m = static_cast<int>(std::min<long long>(kPairs, n - i));
      for (int k = 0; k < m; ++k) a.pair[k] = make_int2(static_cast<int>(c.list[i + k]), static_cast<int>(c.list[n + i + k]));
      a.base = c.in[0].data_as<char>() + z * c.i[1] * c.i[2];
      const dim3 grid(static_cast<unsigned>(blocks), m, static_cast<unsigned>(std::min<long long>(65535, c.i[0] - z)));
      copy_pages_kernel<U><<<grid, kThreads, 0, stream_of(c)>>>(a);
    }
}

void k_copy_pages(OpCall& c) {
  if (c.i[1] > 2147483647LL || c.i[2] / 1024 > 2147483647LL) throw std::invalid_argument("copy_pages_: too many or too large pages");
  const unsigned long long bits = static_cast<unsigned long long>(c.i[2]) | reinterpret_cast<uintptr_t>(c.in[0].data());
  if (bits % 16 == 0) launch_copies<uint4>(c);
  else if (bits % 4 == 0) launch_copies<unsigned int>(c);
  else launch_copies<unsigned char>(c);
  check_launch("copy_pages_");
}

}  // namespace

void register_cuda_paged_cache(KernelRegistry& r) {
  const uint8_t packed = kContiguous | kEmpty;
  r.add_kernel(OperatorId::PagedAppend, Constraints{Backend::CUDA, kMaskCudaCompute, packed, Capability::None}, k_paged_append, "sm100_paged_append");
  r.add_kernel(OperatorId::CopyPages, Constraints{Backend::CUDA, kMaskAll, packed, Capability::None}, k_copy_pages, "sm100_copy_pages");
}

}  // namespace cu
}  // namespace ob
