// The paged key-value cache on sm_100a: new rows into their pages, copies of whole pages.
//
// Pages are [N, H, P, D]: the P rows of one head lie together, so that attention reads a page of a
// head as one contiguous block.  Both operators only move bytes; each byte is read once and
// written once, and that is their floor.
#include <algorithm>

#include "ob/cuda_common.cuh"

namespace ob {
namespace cu {
namespace {

constexpr int kThreads = 256;
constexpr int kAhead = 4;  // accesses of a thread that are under way together

// ---------------------------------------------------------------------- append
struct AppendArgs {
  char* pages[2];             // keys, values
  const char* rows_of[2];
  long long page_stride[2];   // in units (accesses of one thread)
  long long rs[2][3];         // batch, token, head strides of the rows, in units
  const int *table, *starts, *counts;
  unsigned int* errors;
  int tokens, heads, page_size, units, table_width, pages_total, block_tokens;
  unsigned magic_items, magic_units;  // see quotient()
};

// A block takes `block_tokens` tokens of one sequence on one side, so many that their accesses are about
// kAhead for each thread.  The first kAhead of a thread are fetched at once, while other threads look up
// the tokens' places.  The bound on registers keeps 6 blocks on an SM.
//
// Measured, calls one after another (bfloat16): 8192 tokens of 8 heads of 128, keys and values, 67 MB in 15.5 us (16.6
// with the blocks that the registers would allow; 38 with one token to a block); 32768 tokens of 2 heads of 64 10.4 us
// (127).  8 padded prompts of up to 1024 tokens of 16 heads of 128, 72 MB: 16.5 us, 11.0 by their bytes; 2212 of the 4096
// blocks have rows and 888 fit the device, so that these are two and a half waves of blocks that look a place
// up, load once and store once.  One token of each sequence costs a launch.
template <class U>
__global__ void __launch_bounds__(kThreads, 6) append_kernel(const __grid_constant__ AppendArgs a) {
  __shared__ long long to[kThreads];  // first access of a token's place, -1: not written
  const int blocks = (a.tokens + a.block_tokens - 1) / a.block_tokens;
  const int b = blockIdx.x / blocks, t0 = (blockIdx.x - b * blocks) * a.block_tokens, side = blockIdx.y;
  const int start = a.starts[b], count = a.counts == nullptr ? a.tokens : a.counts[b];
  const int rows = min(min(a.block_tokens, a.tokens - t0), count - t0);
  if (rows <= 0) return;
  const int items = a.heads * a.units, all = rows * items, first = threadIdx.x;
  const U* src = reinterpret_cast<const U*>(a.rows_of[side]) + b * a.rs[side][0] + t0 * a.rs[side][1];
  U* dst = reinterpret_cast<U*>(a.pages[side]);
  const long long head_step = static_cast<long long>(a.page_size) * a.units;
  struct Place {
    long long in, out;  // behind the block's first token; behind the token's place
    int token;
  };
  auto place_of = [&](int i) {
    const int k = a.block_tokens == 1 ? 0 : quotient(i, items, a.magic_items), r = i - k * items;
    const int h = quotient(r, a.units, a.magic_units), u = r - h * a.units;
    return Place{k * a.rs[side][1] + h * a.rs[side][2] + u, h * head_step + u, k};
  };
  U v[kAhead];
  Place p[kAhead];
#pragma unroll
  for (int n = 0; n < kAhead; ++n)
    if (first + n * kThreads < all) {
      p[n] = place_of(first + n * kThreads);
      v[n] = src[p[n].in];
    }
  if (first < rows) {
    const long long at = static_cast<long long>(start) + t0 + first, slot = at / a.page_size;
    int page = -1;
    if (at >= 0 && slot < a.table_width) page = a.table[static_cast<long long>(b) * a.table_width + slot];
    const bool there = page >= 0 && page < a.pages_total;
    if (!there && side == 0) atomicAdd(a.errors, 1u);  // never written: the row has no place
    to[first] = there ? page * a.page_stride[side] + (at - slot * a.page_size) * a.units : -1;
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < kAhead; ++n)
    if (first + n * kThreads < all && to[p[n].token] >= 0) dst[to[p[n].token] + p[n].out] = v[n];
  for (int i0 = first + kAhead * kThreads; i0 < all; i0 += kAhead * kThreads) {  // rows of more accesses than that
#pragma unroll
    for (int n = 0; n < kAhead; ++n)
      if (i0 + n * kThreads < all) {
        p[n] = place_of(i0 + n * kThreads);
        v[n] = src[p[n].in];
      }
#pragma unroll
    for (int n = 0; n < kAhead; ++n)
      if (i0 + n * kThreads < all && to[p[n].token] >= 0) dst[to[p[n].token] + p[n].out] = v[n];
  }
}

template <class U>
void launch_append(AppendArgs a, long long batch, int sms, cudaStream_t st) {
  // No more tokens to a block than leave the device several blocks for each SM.
  const long long items = static_cast<long long>(a.heads) * a.units;
  a.block_tokens = static_cast<int>(std::max(1ll, std::min({kThreads * kAhead / items, static_cast<long long>(kThreads), static_cast<long long>(a.tokens), batch * a.tokens / (4ll * sms)})));
  a.magic_items = magic_of(items, a.block_tokens * items + kThreads * kAhead);
  a.magic_units = magic_of(a.units, items + kThreads * kAhead);
  const dim3 grid(static_cast<unsigned>(batch * ((a.tokens + a.block_tokens - 1) / a.block_tokens)), 2);
  append_kernel<U><<<grid, kThreads, 0, st>>>(a);
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
  if (s[0] > 2147483647LL || r[0] * r[1] > 2147483647LL || s[1] * row / w > 1073741823LL)
    throw std::invalid_argument("paged_append_: too many pages, tokens or values in a row");
  AppendArgs a{};
  for (int side = 0; side < 2; ++side) {
    a.pages[side] = c.in[side].data_as<char>();
    a.rows_of[side] = c.in[2 + side].data_as<char>();
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
  const int sms = sm_count_for(c.in[0]);
  cudaStream_t st = stream_of(c);
  if (w == 16) launch_append<uint4>(a, r[0], sms, st);
  else if (w == 8) launch_append<uint2>(a, r[0], sms, st);
  else if (w == 4) launch_append<unsigned int>(a, r[0], sms, st);
  else launch_append<unsigned short>(a, r[0], sms, st);
  check_launch("paged_append_");
}

// ------------------------------------------------------------------ page copies
// The pairs travel in the launch's parameters: no list is sent to the device first.  4 KB would hold 509 of them, but a
// launch with all of 4 KB takes 5.6 us in place of 5.0, and most calls have a few pairs.  1.2 GB read and written
// take 185 us (6.5 TB/s, as a plain copy); a few pages a launch.
constexpr int kPairs = 440;
struct CopyArgs {
  char* base;
  long long page_units, outer_units;  // one page; all pages of one outer index
  int2 pair[kPairs];                  // (source, destination)
};

template <class U>
__global__ void __launch_bounds__(kThreads) copy_pages_kernel(const __grid_constant__ CopyArgs a) {
  const int2 p = a.pair[blockIdx.y];
  U* base = reinterpret_cast<U*>(a.base) + blockIdx.z * a.outer_units;
  const U* src = base + p.x * a.page_units;
  U* dst = base + p.y * a.page_units;
  const long long first = static_cast<long long>(blockIdx.x) * kThreads * kAhead + threadIdx.x;
  U v[kAhead];
#pragma unroll
  for (int k = 0; k < kAhead; ++k)
    if (first + k * kThreads < a.page_units) v[k] = src[first + k * kThreads];
#pragma unroll
  for (int k = 0; k < kAhead; ++k)
    if (first + k * kThreads < a.page_units) dst[first + k * kThreads] = v[k];
}

template <class U>
void launch_copies(OpCall& c) {
  const long long n = static_cast<long long>(c.list.size()) / 2, page = c.i[2] / static_cast<long long>(sizeof(U));
  const long long blocks = (page + kThreads * kAhead - 1) / (kThreads * kAhead);
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
