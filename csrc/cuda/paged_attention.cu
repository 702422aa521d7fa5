// Attention of one new token over the paged key-value cache (sm_100a).
//
//   o = sum_j p_j v_j / sum_j p_j,   p_j = 2^(s_j - m),   s_j = log2(e) scale q k_j,   m = max_j s_j
//
// Keys and values are read once and the maximum runs along (a new one rescales what has been
// summed), so the floor is the time that the cache's bytes take from HBM; about 4 H / H_kv
// operations per cached value are far below what the tensor cores do in that time.
//
// Split.  The work is counted in slabs of 16 tokens of one cached head.  All slabs of the call, in
// the order (sequence, head, token), are divided evenly over the warps of a persistent grid, whatever
// the lengths are: a warp streams its own slabs and meets no other on the way.  A head that lies
// within one warp's share is written at once; one that is spread leaves (m, sum p, sum p v) of each
// share in a workspace, and a second kernel joins them in order.  No atomics: the same call gives the
// same bits.  (Joining inside the first kernel, by the last warp to arrive, was measured too: 116 us
// instead of 99 for 131072 tokens, because its fences wait for the streams around it.)  Even shares are even in
// slabs: heads of one slab take longer for it, for their queries and outputs are waited for (a call that is
// waited for, 8 cached heads of 128: one sequence of 131072 tokens 133 us, beside 255 of one token 232).
//
// Short caches are not worth a second kernel, and many heads need no division: there a block takes
// one head of one sequence, its warps every slab in turn, and they join in shared memory.
//
// Masks.  Rows behind a sequence's length are never read (they are zero-filled on the way in) and
// weigh nothing; a score of -inf weighs nothing; NaN in what is seen stays NaN.
#include <algorithm>
#include <map>
#include <mutex>
#include <type_traits>
#include <utility>

#include "ob/cuda_common.cuh"

namespace ob {
namespace cu {
namespace {

constexpr int kSlab = 16;         // tokens
constexpr int kMostBatch = 2048;  // sequences of one launch: their slab counts lie in shared memory
constexpr int kMostWorkers = 4096;

struct PagedArgs {
  const void *q, *k, *v;
  void* out;
  const int *table, *lengths;
  unsigned int* errors;
  long long qs[2], page_stride[2];  // batch and head of q; keys, values
  long long* prefix;                // workspace: slabs before each sequence, [batch + 1], and a warp's share
  float2* stat;                     // workspace: (m, sum p) of [2 * workers][tile_heads]
  float* part;                      // workspace: sum p v of [2 * workers][tile_heads][head_dim]
  int batch, heads, kv_heads, head_dim, page_size, table_width, pages_total;
  int tiles, tile_heads;            // query heads of one cached head are taken `tile_heads` at a time
  int workers;
  float scale_log2;                 // scale * log2(e)
};

__device__ __forceinline__ int length_of(const PagedArgs& a, int b) {
  const int n = a.lengths[b];
  const long long most = a.pages_total > 0 ? min(static_cast<long long>(a.table_width) * a.page_size, 2147483600LL) : 0;
  return n < 0 ? 0 : n > most ? static_cast<int>(most) : n;
}

// Most quotients here fit 32 bits, where a division costs a fraction.
__device__ __forceinline__ long long divide(long long x, long long y) {
  if (((x | y) >> 32) == 0) return static_cast<unsigned>(x) / static_cast<unsigned>(y);
  return x / y;
}

// A page number from the table; one out of range is counted and not followed.
__device__ __forceinline__ int checked_page(const PagedArgs& a, int page, bool count) {
  if (page >= 0 && page < a.pages_total) return page;
  if (count) atomicAdd(a.errors, 1u);
  return page < 0 ? 0 : a.pages_total - 1;
}

__device__ __forceinline__ int slabs_of(int n) { return (n + kSlab - 1) / kSlab; }

// A place in the order of slabs.  It moves on by counting: divisions cost more than the rest of a slab.
struct Cursor {
  int b, kv, tile;   // sequence, cached head, tile of its query heads
  int j, slabs, n;   // slab of it; slabs of it; length of the sequence
  int in_page;       // first token's place in its page
  // `rest`: slabs behind the first of sequence `at`.
  __device__ __forceinline__ void set(const PagedArgs& a, int at, int length, long long rest) {
    b = at;
    n = length;
    slabs = slabs_of(n);
    const int item = static_cast<int>(divide(rest, slabs));
    j = static_cast<int>(rest - static_cast<long long>(item) * slabs);
    kv = item / a.tiles;
    tile = item - kv * a.tiles;
    in_page = j * kSlab % a.page_size;
  }
  // The slab `step` behind, of the same head.
  __device__ __forceinline__ void skip(const PagedArgs& a, int step) {
    j += step;
    in_page = j * kSlab % a.page_size;
  }
  // Not called behind the last slab of the call.
  __device__ __forceinline__ void next(const PagedArgs& a) {
    in_page += kSlab;
    while (in_page >= a.page_size) in_page -= a.page_size;
    if (++j < slabs) return;
    j = in_page = 0;
    if (++tile < a.tiles) return;
    tile = 0;
    if (++kv < a.kv_heads) return;
    kv = 0;
    do {
      n = length_of(a, ++b);
    } while (n == 0);
    slabs = slabs_of(n);
  }
  __device__ __forceinline__ bool same_head(const Cursor& c) const { return b == c.b && kv == c.kv && tile == c.tile; }
};

// Slabs of one share: all warps get one, but few shares of a long head are cheaper to join.  A slab
// takes a warp 750 cycles and 64 shares take the joining block 900, so a head of n slabs wants shares
// of sqrt(n / 50) at least (2 heads of 15954 tokens: 28.5 us with shares of 2).
__device__ __forceinline__ long long share_of(const PagedArgs& a, long long all) {
  const long long even = divide(all * a.kv_heads * a.tiles + a.workers - 1, a.workers);
  return max(even, static_cast<long long>(ceilf(sqrtf(0.02f * static_cast<float>(all) / static_cast<float>(a.batch)))));
}

// The share of this warp: warp c of the grid takes the slabs from c * share on.  Returns how many,
// and the first of them in `at`.  Block 0 leaves the slabs before each sequence and the share for the
// joining kernel and counts lengths that the table cannot hold.  Up to 32 sequences every warp counts
// for itself; more are counted by the block, whose shared memory has room for their sums.
template <int THREADS>
__device__ __forceinline__ long long take_share(const PagedArgs& a, long long worker, long long* sums, Cursor* at) {
  const int lane = threadIdx.x & 31, items = a.kv_heads * a.tiles;
  const bool tell = blockIdx.x == 0;
  long long all;  // slabs of one head
  if (a.batch <= 32) {
    const int n = lane < a.batch ? length_of(a, lane) : 0, mine = slabs_of(n);
    if (tell && threadIdx.x < a.batch && n != a.lengths[lane]) atomicAdd(a.errors, 1u);
    long long run = mine;
#pragma unroll 1
    for (int o = 1; o < a.batch; o <<= 1) {
      const long long x = __shfl_up_sync(0xffffffffu, run, o);
      if (lane >= o) run += x;
    }
    all = __shfl_sync(0xffffffffu, run, a.batch - 1);
    const long long share = share_of(a, all), lo = worker * share;
    if (tell && threadIdx.x < a.batch) a.prefix[lane] = run - mine;
    if (tell && threadIdx.x == 0) {
      a.prefix[a.batch] = all;
      a.prefix[a.batch + 1] = share;
    }
    if (lo >= all * items) return 0;
    const long long u = divide(lo, items);
    const int b = __popc(__ballot_sync(0xffffffffu, lane < a.batch && run <= u));
    at->set(a, b, __shfl_sync(0xffffffffu, n, b), lo - __shfl_sync(0xffffffffu, run - mine, b) * items);
    return min(share, all * items - lo);
  }
  __shared__ long long warp_sums[THREADS / 32];
  const int warp = threadIdx.x >> 5, per = (a.batch + THREADS - 1) / THREADS, first = threadIdx.x * per, last = min(first + per, a.batch);
  long long sum = 0;
  for (int b = first; b < last; ++b) {
    const int n = length_of(a, b);
    if (tell && n != a.lengths[b]) atomicAdd(a.errors, 1u);
    sum += slabs_of(n);
  }
  long long run = sum;
#pragma unroll 1
  for (int o = 1; o < 32; o <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o) run += x;
  }
  if (lane == 31) warp_sums[warp] = run;
  __syncthreads();
  long long before = run - sum;
  all = 0;
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < warp) before += warp_sums[w];
    all += warp_sums[w];
  }
  for (int b = first; b < last; ++b) {
    sums[b] = before;
    if (tell) a.prefix[b] = before;
    before += slabs_of(length_of(a, b));
  }
  __syncthreads();
  const long long share = share_of(a, all), lo = worker * share;
  if (tell && threadIdx.x == 0) {
    a.prefix[a.batch] = all;
    a.prefix[a.batch + 1] = share;
  }
  if (lo >= all * items) return 0;
  const long long u = divide(lo, items);
  int low = 0, high = a.batch - 1;  // the last sequence with no more than u slabs before it
  while (low < high) {
    const int mid = (low + high + 1) >> 1;
    if (sums[mid] <= u) low = mid;
    else high = mid - 1;
  }
  at->set(a, low, length_of(a, low), lo - sums[low] * items);
  return min(share, all * items - lo);
}

// The block's head, for a block that has one of its own; false where the sequence is empty and the
// output was set to zero.
template <class T>
__device__ __forceinline__ bool take_head(const PagedArgs& a, Cursor* at) {
  const int row = blockIdx.x / a.tiles, group = a.heads / a.kv_heads;
  at->tile = blockIdx.x - row * a.tiles;
  at->b = row / a.kv_heads;
  at->kv = row - at->b * a.kv_heads;
  at->n = length_of(a, at->b);
  at->slabs = slabs_of(at->n);
  if (at->kv == 0 && at->tile == 0 && threadIdx.x == 0 && at->n != a.lengths[at->b]) atomicAdd(a.errors, 1u);
  at->j = threadIdx.x >> 5;
  at->in_page = at->j * kSlab % a.page_size;
  if (at->n > 0) return true;
  const int heads = min(a.tile_heads, group - at->tile * a.tile_heads);
  T* out = static_cast<T*>(a.out) + (static_cast<long long>(at->b) * a.heads + at->kv * group + at->tile * a.tile_heads) * a.head_dim;
  for (int i = threadIdx.x; i < heads * a.head_dim; i += blockDim.x) out[i] = from_f<T>(0.f);
  return false;
}

// The warps' sums of one head tile, in shared memory, into the output.
template <class T, int WARPS>
__device__ __forceinline__ void join_warps(const PagedArgs& a, const Cursor& at, int heads, const float2* stat, const float* part) {
  __syncthreads();
  const int D = a.head_dim, h0 = at.kv * (a.heads / a.kv_heads) + at.tile * a.tile_heads;
  T* out = static_cast<T*>(a.out) + (static_cast<long long>(at.b) * a.heads + h0) * D;
  for (int i = threadIdx.x; i < heads * D; i += WARPS * 32) {
    const int h = i / D;
    float top = -INFINITY, sum = 0.f, o = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) top = fmaxf(top, stat[w * heads + h].x);
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float2 st = stat[w * heads + h];
      const float weight = st.x == top ? 1.f : exp2f(st.x - top);
      sum = fmaf(weight, st.y, sum);
      o = fmaf(weight, part[(w * heads) * D + i], o);
    }
    out[i] = from_f<T>(o / sum);
  }
}

// ------------------------------------------------------------- tensor-core warps
// 16-bit types, head sizes that are a multiple of 8.  With K as the left operand a slab is one
// m16n8k16 product per 16 values: S^T [16 tokens x 8 heads] = K q^T, and O^T [values x 8 heads]
// += V^T P^T, so that up to 8 query heads of one cached head cost no more than one.  The weights
// move from accumulator to operand layout by a transposing register move.  This product is far
// from being the bound, and 8 columns is what a group of heads fills: tcgen05's tiles of 128 rows
// would be empty.  Slabs arrive by asynchronous 16-byte copies into a ring of the warp's own.

__device__ __forceinline__ void copy16(uint32_t smem, const void* global) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem), "l"(global) : "memory");
}
__device__ __forceinline__ void copy16_or_zero(uint32_t smem, const void* global, bool there) {  // nothing is read for a zero
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem), "l"(global), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void load_matrices(uint32_t (&r)[4], uint32_t smem) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(smem) : "memory");
}
__device__ __forceinline__ void load_matrices_transposed(uint32_t (&r)[4], uint32_t smem) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(smem) : "memory");
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
template <class T>
__device__ __forceinline__ void multiply(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Two weights as two terms each: rounded down to T, and what that left.  The second term of a weight above zero
// is never zero, so that its product with an infinite value is that infinity and no NaN.
__device__ __forceinline__ void split2(float lo, float hi, uint32_t* first, uint32_t* second, __nv_bfloat16*) {
  const unsigned a = __float_as_uint(lo), b = __float_as_uint(hi);
  const __nv_bfloat162 rest = __floats2bfloat162_rn(lo - __uint_as_float(a & 0xffff0000u), hi - __uint_as_float(b & 0xffff0000u));
  *first = __byte_perm(a, b, 0x7632);
  *second = __vmaxu2(*reinterpret_cast<const uint32_t*>(&rest), __vminu2(*first, 0x00800080u));  // 2^-126
}
__device__ __forceinline__ void split2(float lo, float hi, uint32_t* first, uint32_t* second, __half*) {
  const __half2 down = __halves2half2(__float2half_rz(lo), __float2half_rz(hi));
  const __half2 rest = __floats2half2_rn(lo - __low2float(down), hi - __high2float(down));
  *first = *reinterpret_cast<const uint32_t*>(&down);
  *second = __vmaxu2(*reinterpret_cast<const uint32_t*>(&rest), __vminu2(*first, 0x00010001u));  // 2^-24, beside weights up to 2^14
}

template <int KD>
struct SlabLayout {
  static constexpr int kChunks = KD * 2;                            // 16-byte pieces of a row
  static constexpr bool kSwizzled = (KD & (KD - 1)) == 0;           // else rows are padded by one piece
  static constexpr int kPitch = KD * 32 + (kSwizzled ? 0 : 16);
  static constexpr int kBytes = kSlab * kPitch;                     // keys or values of one slab
  // Eight rows of the same piece lie in different banks.
  __device__ static __forceinline__ uint32_t at(int row, int chunk) {
    return static_cast<uint32_t>(row * kPitch + ((kSwizzled ? chunk ^ (row & 7) : chunk) << 4));
  }
};

template <class T, int KD, int NT, int STAGES, int WARPS, bool OWN>  // OWN: the block has a head of its own
__global__ void __launch_bounds__(WARPS * 32, 1) paged_tile_kernel(const __grid_constant__ PagedArgs a) {
  using L = SlabLayout<KD>;
  // Weights are at most 2^kLift: float16 then keeps full precision down to 2^-28 of the largest.
  constexpr float kLift = std::is_same<T, __half>::value ? 14.f : 0.f;
  extern __shared__ __align__(1024) unsigned char smem[];
  long long* prefix = reinterpret_cast<long long*>(smem + static_cast<size_t>(WARPS) * STAGES * 2 * L::kBytes);
  if constexpr (!OWN) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int D = a.head_dim, group = a.heads / a.kv_heads;
  const long long worker = static_cast<long long>(warp) * gridDim.x + blockIdx.x;  // few slabs spread over all SMs
  Cursor now;
  long long mine;
  if constexpr (OWN) {
    if (!take_head<T>(a, &now)) return;
    mine = now.j < now.slabs ? (now.slabs - now.j + WARPS - 1) / WARPS : 0;
  } else {
    mine = take_share<WARPS * 32>(a, worker, prefix, &now);
    if (mine == 0) return;
  }
  auto advance = [&](Cursor& c) {
    if constexpr (OWN) c.skip(a, WARPS);
    else c.next(a);
  };

  unsigned char* ring = smem + static_cast<size_t>(warp) * STAGES * 2 * L::kBytes;
  const uint32_t ring_at = static_cast<uint32_t>(__cvta_generic_to_shared(ring));
  const int real = D / 8;  // pieces of a row that exist; the others stay zero
  if (real < L::kChunks) {
    for (int i = lane; i < STAGES * 2 * kSlab * (L::kChunks - real); i += 32) {
      const int row = i / (L::kChunks - real), chunk = real + i - row * (L::kChunks - real);
      *reinterpret_cast<uint4*>(ring + (row / kSlab) * L::kBytes + L::at(row % kSlab, chunk)) = make_uint4(0, 0, 0, 0);
    }
    __syncwarp();
  }
  // Pages of a multiple of 16 tokens hold a slab each, its rows together; of 8, half a slab.
  const bool whole_pages = a.page_size % kSlab == 0, half_pages = !whole_pages && a.page_size % 8 == 0;
  const int magic = (65536 + real - 1) / real;        // c / real for c < 512

  Cursor ahead = now;
  long long to_load = mine;

  // Page numbers of the next slabs (half slabs) of one head, one in each lane: fetched 32 at a time,
  // because a load between the copies would wait for them.
  int pages = 0, pages_from = 0, pages_b = -1;
  auto page_of = [&](const Cursor& c, int half) {
    constexpr int kStep = OWN ? WARPS : 1;
    const int log_halves = half_pages ? 1 : 0;
    if (c.b != pages_b || c.j < pages_from || c.j >= pages_from + (32 >> log_halves) * kStep) {
      pages_b = c.b;
      pages_from = c.j;
      const unsigned j = c.j + (lane >> log_halves) * kStep, token = j * kSlab + (lane & log_halves) * 8;  // may pass 2^31
      const bool there = token < static_cast<unsigned>(c.n);
      pages = there ? a.table[static_cast<long long>(c.b) * a.table_width + token / static_cast<unsigned>(a.page_size)] : 0;
      if (there) pages = checked_page(a, pages, true);
    }
    return __shfl_sync(0xffffffffu, pages, ((c.j - pages_from) / kStep << log_halves) + half);
  };
  const long long head_step = static_cast<long long>(a.page_size) * D;
  auto load_slab = [&](int stage, const Cursor& c) {
    const int n = c.n - c.j * kSlab;  // rows of the slab that exist
    const uint32_t to = ring_at + stage * 2 * L::kBytes;
    if (whole_pages || half_pages) {
      // Row r of the slab at k[half] + r * D, half = r / 8.
      const T *k[2], *v[2];
      const int page = page_of(c, 0), last = half_pages ? page_of(c, 1) : page;
      const long long in_page = c.in_page, next = half_pages && c.in_page + 8 == a.page_size ? -8 : c.in_page;  // of the second half, less 8
      const long long inner = c.kv * head_step + lane * 8;
      k[0] = static_cast<const T*>(a.k) + (page * a.page_stride[0] + inner + in_page * D);
      v[0] = static_cast<const T*>(a.v) + (page * a.page_stride[1] + inner + in_page * D);
      k[1] = static_cast<const T*>(a.k) + (last * a.page_stride[0] + inner + next * D);
      v[1] = static_cast<const T*>(a.v) + (last * a.page_stride[1] + inner + next * D);
      if (real == L::kChunks && n >= kSlab) {
#pragma unroll
        for (int i = 0; i < L::kChunks / 2; ++i) {
          const int x = i * 32 + lane, half = i * 32 / L::kChunks / 8;
          const uint32_t at = to + L::at(x / L::kChunks, x % L::kChunks);
          copy16(at, k[half] + i * 256);
          copy16(at + L::kBytes, v[half] + i * 256);
        }
      } else {
#pragma unroll 1
        for (int x = lane, i = 0; x < kSlab * real; x += 32, i += 256) {
          const int row = (x * magic) >> 16;
          const uint32_t at = to + L::at(row, x - row * real);
          copy16_or_zero(at, (row < 8 ? k[0] : k[1]) + i, row < n);
          copy16_or_zero(at + L::kBytes, (row < 8 ? v[0] : v[1]) + i, row < n);
        }
      }
    } else {
#pragma unroll 1
      for (int x = lane; x < kSlab * real; x += 32) {
        const int row = (x * magic) >> 16, chunk = x - row * real, token = c.j * kSlab + row;
        const int slot = token / a.page_size;
        const int entry = row < n ? a.table[static_cast<long long>(c.b) * a.table_width + slot] : 0;
        const int pg = checked_page(a, entry, chunk == 0);
        const long long inner = c.kv * head_step + static_cast<long long>(token - slot * a.page_size) * D + chunk * 8;
        const uint32_t at = to + L::at(row, chunk);
        copy16_or_zero(at, static_cast<const T*>(a.k) + (row < n ? pg * a.page_stride[0] + inner : 0), row < n);
        copy16_or_zero(at + L::kBytes, static_cast<const T*>(a.v) + (row < n ? pg * a.page_stride[1] + inner : 0), row < n);
      }
    }
  };

  constexpr bool kFetchAhead = KD * NT <= 16;  // as far as registers go
  uint32_t q[NT][KD][2], coming[NT][KD][2];
  Cursor whose = now;  // head that `coming` belongs to
  bool fetched = false;
  auto first_head = [&](const Cursor& c) { return c.kv * group + c.tile * a.tile_heads; };
  auto heads_of = [&](const Cursor& c) { return min(a.tile_heads, group - c.tile * a.tile_heads); };
  auto load_queries = [&](const Cursor& c, uint32_t (&to)[NT][KD][2]) {
    const int h0 = first_head(c), heads = heads_of(c);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const bool there = nt * 8 + g < heads;
      const T* qh = static_cast<const T*>(a.q) + c.b * a.qs[0] + (h0 + nt * 8 + g) * a.qs[1] + t * 2;
#pragma unroll
      for (int i = 0; i < KD; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          to[nt][i][e] = there && i * 16 + e * 8 + t * 2 < D ? *reinterpret_cast<const uint32_t*>(qh + i * 16 + e * 8) : 0u;
    }
  };
  load_queries(now, q);
#pragma unroll 1
  for (int s = 0; s < STAGES - 1; ++s) {
    if (to_load > 0) {
      load_slab(s, ahead);
      if (--to_load > 0) advance(ahead);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  }

  float o[NT][KD][4], m[NT][2], sum[NT][2];
  auto clear = [&] {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < KD; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
      m[nt][0] = m[nt][1] = -INFINITY;
      sum[nt][0] = sum[nt][1] = 0.f;
    }
  };
  clear();
  int stage = 0;
  bool from_start = now.j == 0, first_item = true;
  // ldmatrix addresses: K rows are tokens, (0-7, 8-15) by lane bit 3, pieces by lane bit 4; V transposed, the other way round.
  const int k_row = lane & 15, k_piece = lane >> 4, v_row = (lane & 7) + ((lane >> 4) << 3), v_piece = (lane >> 3) & 1;

  for (long long left = mine; left > 0; --left) {
    if (!OWN && left != mine && now.j == 0) {  // a new head: its queries, empty sums
      from_start = true;
      if (!kFetchAhead || !fetched || !whose.same_head(now)) load_queries(now, coming);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < KD; ++i) {
          q[nt][i][0] = coming[nt][i][0];
          q[nt][i][1] = coming[nt][i][1];
        }
      fetched = false;
      clear();
    }
    asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
    __syncwarp();  // every lane's copies are there, and every lane is done with the slab before
    if (to_load > 0) {
      load_slab(stage == 0 ? STAGES - 1 : stage - 1, ahead);
      if (--to_load > 0) {
        advance(ahead);
        if (!OWN && kFetchAhead && ahead.j == 0 && !fetched) {  // the next head's queries, while this one's slabs are taken
          load_queries(ahead, coming);
          whose = ahead;
          fetched = true;
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");

    const uint32_t ks = ring_at + stage * 2 * L::kBytes, vs = ks + L::kBytes;
    float s[NT][4], s2[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[nt][e] = s2[nt][e] = 0.f;
#pragma unroll
    for (int i = 0; i < KD; ++i) {
      uint32_t k[4];
      load_matrices(k, ks + L::at(k_row, i * 2 + k_piece));
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) multiply<T>(i & 1 ? s2[nt] : s[nt], k, q[nt][i][0], q[nt][i][1]);  // two chains
    }
    uint32_t p[NT][2], p2[NT][2];
    const int rows = now.n - now.j * kSlab;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      // s[0], s[1]: token g of heads 2t, 2t + 1; s[2], s[3]: token g + 8.
#pragma unroll
      for (int e = 0; e < 4; ++e) s[nt][e] = g + (e >> 1) * 8 < rows ? (s[nt][e] + s2[nt][e]) * a.scale_log2 : -INFINITY;
      float top[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        top[c] = fmaxf(s[nt][c], s[nt][c + 2]);
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) top[c] = fmaxf(top[c], __shfl_xor_sync(0xffffffffu, top[c], x));
        top[c] = fmaxf(top[c], m[nt][c]);
      }
      if (__any_sync(0xffffffffu, top[0] > m[nt][0] || top[1] > m[nt][1])) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float keep = top[c] == -INFINITY ? 1.f : exp2f(m[nt][c] - top[c]);
          m[nt][c] = top[c];
          sum[nt][c] *= keep;
#pragma unroll
          for (int i = 0; i < KD; ++i) {
            o[nt][i][c] *= keep;
            o[nt][i][c + 2] *= keep;
          }
        }
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float base = (m[nt][c] == -INFINITY ? 0.f : m[nt][c]) - kLift;
        s[nt][c] = exp2f(s[nt][c] - base);
        s[nt][c + 2] = exp2f(s[nt][c + 2] - base);
        sum[nt][c] += s[nt][c] + s[nt][c + 2];
      }
      // The weights enter the product with the values as two terms of the cache's type, 15 (bfloat16) or 21 bits of
      // them: the output is as near as with float32 weights.  One term, that is weights rounded by half a step beside a
      // sum that is not, was off by 0.0021 of the output in bfloat16, two are by 0.0017, which is the output's own
      // rounding; they take 99.3 us in place of 98.7 for 131072 tokens with 32 heads on 8, and a block with a head of
      // its own 11.5 in place of 10.3 for 512 tokens.
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        split2(s[nt][2 * e], s[nt][2 * e + 1], &p[nt][e], &p2[nt][e], static_cast<T*>(nullptr));
        p[nt][e] = transpose8x8(p[nt][e]);
        p2[nt][e] = transpose8x8(p2[nt][e]);
      }
    }
#pragma unroll
    for (int i = 0; i < KD; i += 2) {  // two pieces in turn: the second term's product waits for the first's
      uint32_t v[2][4];
#pragma unroll
      for (int u = 0; u < 2; ++u) load_matrices_transposed(v[u], vs + L::at(v_row, (i + u) * 2 + v_piece));
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int u = 0; u < 2; ++u) multiply<T>(o[nt][i + u], v[u], p[nt][0], p[nt][1]);
#pragma unroll
        for (int u = 0; u < 2; ++u) multiply<T>(o[nt][i + u], v[u], p2[nt][0], p2[nt][1]);
      }
    }
    stage = stage + 1 == STAGES ? 0 : stage + 1;

    if (!OWN && (now.j == now.slabs - 1 || left == 1)) {  // this share of the head is done
      const bool all = from_start && now.j == now.slabs - 1;
      const int h0 = first_head(now), heads = heads_of(now);
      const long long slot = (2 * worker + (first_item ? 0 : 1)) * a.tile_heads;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float w = sum[nt][c];
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) w += __shfl_xor_sync(0xffffffffu, w, x);
          const int h = nt * 8 + t * 2 + c;
          if (h >= heads) continue;
          if (all) {
            T* out = static_cast<T*>(a.out) + (static_cast<long long>(now.b) * a.heads + h0 + h) * D;
            const float inv = 1.f / w;
#pragma unroll
            for (int i = 0; i < KD; ++i) {
              if (i * 16 + g < D) out[i * 16 + g] = from_f<T>(o[nt][i][c] * inv);
              if (i * 16 + g + 8 < D) out[i * 16 + g + 8] = from_f<T>(o[nt][i][c + 2] * inv);
            }
          } else {
            float* part = a.part + (slot + h) * D;
            if (g == 0) a.stat[slot + h] = make_float2(m[nt][c], w);
#pragma unroll
            for (int i = 0; i < KD; ++i) {
              if (i * 16 + g < D) part[i * 16 + g] = o[nt][i][c];
              if (i * 16 + g + 8 < D) part[i * 16 + g + 8] = o[nt][i][c + 2];
            }
          }
        }
      first_item = false;
    }
    if (left > 1) advance(now);
  }
  if constexpr (OWN) {
    const int heads = heads_of(now);
    float* part = reinterpret_cast<float*>(smem);
    float2* stat = reinterpret_cast<float2*>(part + static_cast<size_t>(WARPS) * heads * D);
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();  // the rings are done with
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float w = sum[nt][c];
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) w += __shfl_xor_sync(0xffffffffu, w, x);
        const int h = nt * 8 + t * 2 + c;
        if (h >= heads) continue;
        if (g == 0) stat[warp * heads + h] = make_float2(m[nt][c], w);
#pragma unroll
        for (int i = 0; i < KD; ++i) {
          if (i * 16 + g < D) part[(warp * heads + h) * D + i * 16 + g] = o[nt][i][c];
          if (i * 16 + g + 8 < D) part[(warp * heads + h) * D + i * 16 + g + 8] = o[nt][i][c + 2];
        }
      }
    join_warps<T, WARPS>(a, now, heads, stat, part);
  }
}

// ------------------------------------------------------------------- plain warps
// float32, and head sizes or addresses that 16-byte pieces do not fit.  A lane holds PER values of
// every row; 8 tokens are multiplied at a time with up to NH query heads, and their 8 NH partial
// scores are summed over the lanes by halving: each exchange sends one half of the values and keeps
// the other, so that a score costs about one exchange and ends in one lane, which takes its
// exponential alone.
template <class T, int PER>
struct alignas(sizeof(T) * PER < 16 ? sizeof(T) * PER : 16) Row {
  T v[PER];
};

template <class T, int PER>
__device__ __forceinline__ Row<T, PER> load_row(const T* row, int d, int D, bool wide) {
  Row<T, PER> r;
  if (wide) {  // the head size and all addresses fit PER values
    if (d < D) return *reinterpret_cast<const Row<T, PER>*>(row + d);
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) r.v[i] = !wide && d + i < D ? row[d + i] : from_f<T>(0.f);
  return r;
}

// Sums of x[0..N) over the warp: the sum of x[i] ends in the lanes whose upper log2(N) bits are i.
template <int N>
__device__ __forceinline__ float sum_by_halving(float (&x)[N], int lane) {
  int bit = 16;
#pragma unroll
  for (int n = N / 2; n > 0; n /= 2, bit /= 2) {
    const bool upper = (lane & bit) != 0;
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const float keep = upper ? x[i + n] : x[i], send = upper ? x[i] : x[i + n];
      x[i] = keep + __shfl_xor_sync(0xffffffffu, send, bit);
    }
  }
  for (; bit > 0; bit /= 2) x[0] += __shfl_xor_sync(0xffffffffu, x[0], bit);
  return x[0];
}

constexpr int kRowThreads = 256, kRowTokens = 8;
template <class T, int PER, int NH, bool OWN>
__global__ void __launch_bounds__(kRowThreads) paged_rows_kernel(const __grid_constant__ PagedArgs a, const bool wide) {
  constexpr int kLaneHeads = NH < 4 ? NH : 4, kSets = NH / kLaneHeads;  // heads that the lanes hold side by side, and how often
  constexpr int kShift = NH == 1 ? 2 : NH == 2 ? 1 : 0;                 // lane = (head, token, copy)
  extern __shared__ __align__(16) long long rows_prefix[];
  constexpr int kRowWarps = kRowThreads / 32;
  if constexpr (!OWN) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, d0 = lane * PER;
  const int D = a.head_dim, group = a.heads / a.kv_heads;
  const int my_token = (lane >> kShift) & 7;
  const long long worker = static_cast<long long>(warp) * gridDim.x + blockIdx.x;
  Cursor now;
  long long mine;
  if constexpr (OWN) {
    if (!take_head<T>(a, &now)) return;
    mine = now.j < now.slabs ? (now.slabs - now.j + kRowWarps - 1) / kRowWarps : 0;
  } else {
    mine = take_share<kRowThreads>(a, worker, rows_prefix, &now);
    if (mine == 0) return;
  }

  float q[NH][PER], acc[NH][PER], m[kSets], sum[kSets];
  bool from_start = false, first_item = true;
  if constexpr (OWN) {  // a warp may have no slab at all
#pragma unroll
    for (int h = 0; h < NH; ++h)
#pragma unroll
      for (int i = 0; i < PER; ++i) acc[h][i] = 0.f;
#pragma unroll
    for (int c = 0; c < kSets; ++c) { m[c] = -INFINITY; sum[c] = 0.f; }
  }
  for (long long left = mine; left > 0; --left) {
    const int h0 = now.kv * group + now.tile * a.tile_heads, heads = min(a.tile_heads, group - now.tile * a.tile_heads);
    if (left == mine || (!OWN && now.j == 0)) {
      from_start = now.j == 0;
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        const T* qh = static_cast<const T*>(a.q) + now.b * a.qs[0] + (h0 + h) * a.qs[1];
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          q[h][i] = h < heads && d0 + i < D ? to_f(qh[d0 + i]) * a.scale_log2 : 0.f;
          acc[h][i] = 0.f;
        }
      }
#pragma unroll
      for (int c = 0; c < kSets; ++c) { m[c] = -INFINITY; sum[c] = 0.f; }
    }
    const int* table = a.table + static_cast<long long>(now.b) * a.table_width;
#pragma unroll 1
    for (int first = now.j * kSlab; first < min(now.n, (now.j + 1) * kSlab); first += kRowTokens) {
      const int rows = now.n - first;
      Row<T, PER> k[kRowTokens], v[kRowTokens];
      int slot = first / a.page_size, in_page = first - slot * a.page_size, page = checked_page(a, table[slot], lane == 0);
#pragma unroll
      for (int u = 0; u < kRowTokens; ++u) {
        if (u < rows) {
          if (in_page == a.page_size) {
            in_page = 0;
            page = checked_page(a, table[++slot], lane == 0);
          }
          const long long inner = (static_cast<long long>(now.kv) * a.page_size + in_page) * D;
          k[u] = load_row<T, PER>(static_cast<const T*>(a.k) + page * a.page_stride[0] + inner, d0, D, wide);
          v[u] = load_row<T, PER>(static_cast<const T*>(a.v) + page * a.page_stride[1] + inner, d0, D, wide);
          ++in_page;
        } else {
#pragma unroll
          for (int i = 0; i < PER; ++i) k[u].v[i] = v[u].v[i] = from_f<T>(0.f);
        }
      }
      float p[kSets];
#pragma unroll
      for (int c = 0; c < kSets; ++c) {
        float x[kLaneHeads * kRowTokens];
#pragma unroll
        for (int h = 0; h < kLaneHeads; ++h)
#pragma unroll
          for (int u = 0; u < kRowTokens; ++u) {
            float dot = 0.f;
#pragma unroll
            for (int i = 0; i < PER; ++i) dot = fmaf(q[c * kLaneHeads + h][i], to_f(k[u].v[i]), dot);
            x[h * kRowTokens + u] = dot;
          }
        float s = sum_by_halving<kLaneHeads * kRowTokens>(x, lane);
        s = my_token < rows ? s : -INFINITY;
        float top = s;
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o << kShift));
        top = fmaxf(top, m[c]);
        if (__any_sync(0xffffffffu, top > m[c])) {
          const float keep = top == -INFINITY ? 1.f : exp2f(m[c] - top);
          m[c] = top;
          sum[c] *= keep;
#pragma unroll
          for (int h = 0; h < kLaneHeads; ++h) {
            const float w = __shfl_sync(0xffffffffu, keep, h << (kShift + 3));
#pragma unroll
            for (int i = 0; i < PER; ++i) acc[c * kLaneHeads + h][i] *= w;
          }
        }
        p[c] = exp2f(s - (m[c] == -INFINITY ? 0.f : m[c]));
        sum[c] += p[c];
      }
#pragma unroll
      for (int u = 0; u < kRowTokens; ++u)
#pragma unroll
        for (int h = 0; h < NH; ++h) {
          const float w = __shfl_sync(0xffffffffu, p[h / kLaneHeads], ((h % kLaneHeads) << (kShift + 3)) | (u << kShift));
#pragma unroll
          for (int i = 0; i < PER; ++i) acc[h][i] = fmaf(w, to_f(v[u].v[i]), acc[h][i]);
        }
    }
    if (!OWN && (now.j == now.slabs - 1 || left == 1)) {
      const bool all = from_start && now.j == now.slabs - 1;
      const long long slot = (2 * worker + (first_item ? 0 : 1)) * a.tile_heads;
#pragma unroll
      for (int c = 0; c < kSets; ++c)
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) sum[c] += __shfl_xor_sync(0xffffffffu, sum[c], o << kShift);
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        const float w = __shfl_sync(0xffffffffu, sum[h / kLaneHeads], (h % kLaneHeads) << (kShift + 3));
        const float top = __shfl_sync(0xffffffffu, m[h / kLaneHeads], (h % kLaneHeads) << (kShift + 3));
        if (h >= heads) continue;
        if (!all && lane == 0) a.stat[slot + h] = make_float2(top, w);
        T* out = static_cast<T*>(a.out) + (static_cast<long long>(now.b) * a.heads + h0 + h) * D;
        float* part = a.part + (slot + h) * D;
#pragma unroll
        for (int i = 0; i < PER; ++i)
          if (d0 + i < D) {
            if (all) out[d0 + i] = from_f<T>(acc[h][i] / w);
            else part[d0 + i] = acc[h][i];
          }
      }
      first_item = false;
    }
    if constexpr (OWN) now.skip(a, kRowWarps);
    else if (left > 1) now.next(a);
  }
  if constexpr (OWN) {
    const int heads = min(a.tile_heads, group - now.tile * a.tile_heads);
    float* part = reinterpret_cast<float*>(rows_prefix);
    float2* stat = reinterpret_cast<float2*>(part + static_cast<size_t>(kRowWarps) * NH * D);
#pragma unroll
    for (int c = 0; c < kSets; ++c)
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) sum[c] += __shfl_xor_sync(0xffffffffu, sum[c], o << kShift);
#pragma unroll
    for (int h = 0; h < NH; ++h) {
      const float w = __shfl_sync(0xffffffffu, sum[h / kLaneHeads], (h % kLaneHeads) << (kShift + 3));
      const float top = __shfl_sync(0xffffffffu, m[h / kLaneHeads], (h % kLaneHeads) << (kShift + 3));
      if (h >= heads) continue;
      if (lane == 0) stat[warp * heads + h] = make_float2(top, w);
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (d0 + i < D) part[(warp * heads + h) * D + d0 + i] = acc[h][i];
    }
    join_warps<T, kRowWarps>(a, now, heads, stat, part);
  }
}

// --------------------------------------------------------------------- joining
// The shares of a head that was spread over several warps, in their order; zeros for an empty
// sequence.
constexpr int kJoinThreads = 256, kJoinWarps = kJoinThreads / 32;

struct Shares {
  long long first_row, row0, step;  // rows of stat and part: share c > 0 at row0 + c * step
  int n;                            // 0: an empty sequence; 1: nothing to join
  __device__ __forceinline__ Shares(const PagedArgs& a, int b, int h) {
    const long long before = __ldcg(a.prefix + b), slabs = __ldcg(a.prefix + b + 1) - before, share = __ldcg(a.prefix + a.batch + 1);
    const int group = a.heads / a.kv_heads, kv = h / group, tile = (h - kv * group) / a.tile_heads;
    const int in_tile = h - kv * group - tile * a.tile_heads;
    n = 0;
    first_row = row0 = 0;
    step = 2 * a.tile_heads;
    if (slabs == 0) return;
    const long long s0 = before * a.kv_heads * a.tiles + (kv * a.tiles + tile) * slabs;
    const long long first = divide(s0, share);
    n = static_cast<int>(divide(s0 + slabs - 1, share) - first) + 1;
    row0 = first * step + in_tile;
    // Only the first warp can have begun with another head: then this one is its second.
    first_row = row0 + (first * share < s0 ? a.tile_heads : 0);
  }
  __device__ __forceinline__ long long row(int c) const { return c == 0 ? first_row : row0 + c * step; }
};

// A running sum of shares: m the largest exponent so far, l and o what goes with it.
struct Joined {
  float m = -INFINITY, l = 0.f, o = 0.f;
  __device__ __forceinline__ void add(float2 stat, float part) {
    const float top = fmaxf(m, stat.x);
    const float keep = m == top ? 1.f : exp2f(m - top), w = stat.x == top ? 1.f : exp2f(stat.x - top);
    l = l * keep + w * stat.y;
    o = o * keep + w * part;
    m = top;
  }
};

// Heads with many shares: a block takes 32 values of one head.  All threads look at the exponents, the
// weights go to shared memory, and each warp takes every eighth share.
template <class T>
__global__ void __launch_bounds__(kJoinThreads) paged_join_wide_kernel(const __grid_constant__ PagedArgs a) {
  __shared__ float weight[kMostWorkers], smem[32], sums[kJoinWarps][32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, D = a.head_dim, d = blockIdx.y * 32 + lane;
  T* out = static_cast<T*>(a.out) + static_cast<long long>(blockIdx.x) * D;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const Shares s(a, blockIdx.x / a.heads, blockIdx.x % a.heads);
  if (s.n < 2) {
    if (s.n == 0 && warp == 0 && d < D) out[d] = from_f<T>(0.f);
    return;
  }
  float2 mine = make_float2(-INFINITY, 0.f);
  for (int c = tid; c < s.n; c += kJoinThreads) {
    const float2 st = __ldcg(a.stat + s.row(c));
    const float top = fmaxf(mine.x, st.x);
    mine.y = mine.y * (mine.x == top ? 1.f : exp2f(mine.x - top)) + st.y * (st.x == top ? 1.f : exp2f(st.x - top));
    mine.x = top;
    weight[c] = st.x;
  }
  const float top = block_max(mine.x, smem);
  for (int c = tid; c < s.n; c += kJoinThreads) weight[c] = weight[c] == top ? 1.f : exp2f(weight[c] - top);
  const float sum = block_sum(mine.y * (mine.x == top ? 1.f : exp2f(mine.x - top)), smem);  // synchronises: the weights are there
  float o = 0.f;
  if (d < D) {
#pragma unroll 8
    for (int c = warp; c < s.n; c += kJoinWarps) o = fmaf(weight[c], __ldcg(a.part + s.row(c) * D + d), o);
  }
  sums[warp][lane] = o;
  __syncthreads();
  if (warp == 0 && d < D) {
#pragma unroll
    for (int i = 1; i < kJoinWarps; ++i) o += sums[i][lane];
    out[d] = from_f<T>(o / sum);
  }
}

// Heads with few shares: a warp takes 32 values of one, and lies with others' in a block.  A sequence that is far
// longer than the rest has many shares all the same: a head with more than kMany is left to all warps of the block,
// one head after another, and neighbouring tasks lie in different blocks.  (One sequence among 255 of one token, 4
// heads on one, by a warp alone or by the block: 40 shares 18.7 / 28.6 us, 62 23.8 / 28.6, 125 36.9 / 30.7; 1024, a call
// that is waited for, 276 / 100.)
constexpr int kMany = 96;

template <class T>
__global__ void __launch_bounds__(kJoinThreads) paged_join_kernel(const __grid_constant__ PagedArgs a) {
  __shared__ float smem[32], sums[kJoinWarps][32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, D = a.head_dim, slices = (D + 31) / 32;
  const long long tasks = static_cast<long long>(a.batch) * a.heads * slices;
  auto task_of = [&](int w, int* head) {  // returns the value that this lane has
    const long long task = static_cast<long long>(w) * gridDim.x + blockIdx.x;
    *head = task < tasks ? static_cast<int>(divide(task, slices)) : -1;
    return static_cast<int>(task - static_cast<long long>(*head) * slices) * 32 + lane;
  };
  int head;
  const int d = task_of(warp, &head);
  bool many = false;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (head >= 0) {
    const Shares s(a, head / a.heads, head % a.heads);
    many = s.n > kMany;
    if (!many && s.n != 1 && d < D) {
      Joined all;
#pragma unroll 4
      for (int c = 0; c < s.n; ++c) all.add(__ldcg(a.stat + s.row(c)), __ldcg(a.part + s.row(c) * D + d));
      static_cast<T*>(a.out)[static_cast<long long>(head) * D + d] = from_f<T>(s.n == 0 ? 0.f : all.o / all.l);
    }
  }
  if (!__syncthreads_or(many)) return;
#pragma unroll 1
  for (int w = 0; w < kJoinWarps; ++w) {
    const int d = task_of(w, &head);
    if (head < 0) break;
    const Shares s(a, head / a.heads, head % a.heads);
    if (s.n <= kMany) continue;
    float2 mine = make_float2(-INFINITY, 0.f);
    for (int c = tid; c < s.n; c += kJoinThreads) {
      const float2 st = __ldcg(a.stat + s.row(c));
      const float top = fmaxf(mine.x, st.x);
      mine.y = mine.y * (mine.x == top ? 1.f : exp2f(mine.x - top)) + st.y * (st.x == top ? 1.f : exp2f(st.x - top));
      mine.x = top;
    }
    const float top = block_max(mine.x, smem);
    const float sum = block_sum(mine.y * (mine.x == top ? 1.f : exp2f(mine.x - top)), smem);
    float o = 0.f;
    if (d < D) {
#pragma unroll 8
      for (int c = warp; c < s.n; c += kJoinWarps) {
        const float m = __ldcg(&a.stat[s.row(c)].x);
        o = fmaf(m == top ? 1.f : exp2f(m - top), __ldcg(a.part + s.row(c) * D + d), o);
      }
    }
    sums[warp][lane] = o;
    __syncthreads();
    if (warp == 0 && d < D) {
#pragma unroll
      for (int i = 1; i < kJoinWarps; ++i) o += sums[i][lane];
      static_cast<T*>(a.out)[static_cast<long long>(head) * D + d] = from_f<T>(o / sum);
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------------------- host
// Resident blocks per SM of a kernel with its shared memory, once per device; also opts in to it.
template <class Kernel>
int blocks_per_sm(Kernel kernel, int device, int threads, size_t smem) {
  static std::mutex mu;  // one set per kernel type: the address tells the kernels apart
  static std::map<std::pair<const void*, int>, int> known;
  std::lock_guard<std::mutex> lock(mu);
  int& n = known[{reinterpret_cast<const void*>(kernel), device}];
  if (n == 0) {
    OB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
    int fit = 0;
    OB_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&fit, kernel, threads, smem));
    if (fit < 1) throw std::runtime_error("paged_attention: the kernel does not fit this device");
    n = fit;
  }
  return n;
}

struct Launch {
  Device device;
  int sms;
  cudaStream_t stream;
};

// Both kernels of one call.  `smem_ring`: bytes in front of the slab counts.
template <class T, class Kernel, class... Extra>
void launch_both(Kernel kernel, int threads, size_t smem_ring, PagedArgs a, const Launch& l, Extra... extra) {
  const int per_sm = blocks_per_sm(kernel, l.device.index, threads, smem_ring + (kMostBatch + 1) * sizeof(long long));
  int blocks = l.sms * per_sm;
  const int warps = threads / 32;
  blocks = std::min(blocks, kMostWorkers / warps);
  a.workers = blocks * warps;
  const size_t shares = 2ull * a.workers * a.tile_heads;
  const size_t prefix_bytes = (static_cast<size_t>(a.batch) * 8 + 16 + 255) / 256 * 256, stat_bytes = (shares * 8 + 255) / 256 * 256;
  ScratchLease scratch(l.device, prefix_bytes + stat_bytes + shares * a.head_dim * 4, l.stream);
  char* at = static_cast<char*>(scratch.data());
  a.prefix = reinterpret_cast<long long*>(at);
  a.stat = reinterpret_cast<float2*>(at + prefix_bytes);
  a.part = reinterpret_cast<float*>(at + prefix_bytes + stat_bytes);
  kernel<<<blocks, threads, smem_ring + (a.batch + 1) * sizeof(long long), l.stream>>>(a, extra...);
  check_launch("paged_attention");
  cudaLaunchConfig_t config{};
  const unsigned heads = static_cast<unsigned>(a.batch) * a.heads, slices = static_cast<unsigned>((a.head_dim + 31) / 32);
  const bool wide = a.workers >= 8ll * a.batch * a.kv_heads * a.tiles;  // shares of a head when all warps have one
  config.gridDim = wide ? dim3(heads, slices) : dim3(static_cast<unsigned>((static_cast<long long>(heads) * slices + kJoinWarps - 1) / kJoinWarps));
  config.blockDim = dim3(kJoinThreads);
  config.stream = l.stream;
  cudaLaunchAttribute dependent{};
  dependent.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  dependent.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &dependent;
  config.numAttrs = wide ? 0 : 1;  // few blocks that wait on the first kernel's SMs only slow it (131072 tokens: 99 us, 96 without)
  OB_CUDA(cudaLaunchKernelEx(&config, wide ? paged_join_wide_kernel<T> : paged_join_kernel<T>, static_cast<const PagedArgs&>(a)));
  check_launch("paged_attention join");
}

// One block for each head tile of each sequence.
template <class Kernel, class... Extra>
void launch_own(Kernel kernel, int threads, size_t smem, const PagedArgs& a, const Launch& l, Extra... extra) {
  blocks_per_sm(kernel, l.device.index, threads, smem);  // opts in to `smem`, the same in every call
  kernel<<<static_cast<unsigned>(a.batch) * a.kv_heads * a.tiles, threads, smem, l.stream>>>(a, extra...);
  check_launch("paged_attention");
}

// A block per head, or even shares and a second kernel?  The second kernel costs 7 to 10 us.  A block alone takes
// `per_token` us for a token of its head (bfloat16: 0.009, 0.011 and 0.015 with 64, 128 and 256 values; float32: 0.03 to
// 0.055), until 1.2 heads on each SM keep the device busy.  Lengths are on the device: what the table has room for
// stands for them, and a table where one long sequence could keep a few blocks running alone for over 25 us gets even
// shares.  (Own against shares, bfloat16, 8 cached heads of 128, 4 query heads on each: 1 sequence of 512 tokens 11.5 / 12.4
// us, 1024 17.0 / 13.4, 2048 28.8 / 13.4; 16 of up to 2048 29.3 / 34.4; 64 of up to 2048 58.8 / 66.3; 32 of up to 4096
// 61.8 / 59.1; 8 of 8192 98.6 / 61.0.  float32: 32 of up to 1000, 4 heads of 64 42.6 / 28.8.  Over 220 sizes of both types
// the choice takes 1.009 times the better one's time, 1.32 at worst; without any block per head it would be 1.23.)
bool block_per_head(const PagedArgs& a, int sms, double per_token) {
  const double alone = per_token * a.table_width * a.page_size, heads = static_cast<double>(a.batch) * a.kv_heads * a.tiles;
  return alone <= 25.0 && (1.0 - heads / (1.2 * sms)) * alone <= 10.0;
}

template <class T, int KD, int NT, int STAGES, int WARPS, int OWN_STAGES>
void launch_tiles(PagedArgs a, const Launch& l) {
  const int group = a.heads / a.kv_heads, most = 8 * NT;
  a.tiles = (group + most - 1) / most;
  a.tile_heads = (group + a.tiles - 1) / a.tiles;
  constexpr size_t slab = 2 * SlabLayout<KD>::kBytes;
  if (block_per_head(a, l.sms, 0.0075 + 0.00003 * a.head_dim)) launch_own(paged_tile_kernel<T, KD, NT, OWN_STAGES, 4, true>, 128, 4 * OWN_STAGES * slab, a, l);
  else launch_both<T>(paged_tile_kernel<T, KD, NT, STAGES, WARPS, false>, WARPS * 32, WARPS * STAGES * slab, a, l);
}

template <class T, int PER, int NH>
void launch_rows(const PagedArgs& a, const Launch& l, bool wide) {
  constexpr size_t own = kRowThreads / 32 * static_cast<size_t>(NH) * (PER * 32 * sizeof(float) + sizeof(float2));  // for every head size of the kernel
  if (block_per_head(a, l.sms, 0.025 + 0.003 * a.tile_heads + 0.00004 * a.head_dim)) launch_own(paged_rows_kernel<T, PER, NH, true>, kRowThreads, own, a, l, wide);
  else launch_both<T>(paged_rows_kernel<T, PER, NH, false>, kRowThreads, 0, a, l, wide);
}

template <class T, int PER>
void launch_rows(PagedArgs a, const Launch& l, bool wide) {
  const int group = a.heads / a.kv_heads;
  const int most = PER == 8 ? 4 : 8;  // registers: queries and sums are NH x PER values each
  a.tiles = (group + most - 1) / most;
  a.tile_heads = (group + a.tiles - 1) / a.tiles;
  if (a.tile_heads == 1) launch_rows<T, PER, 1>(a, l, wide);
  else if (a.tile_heads == 2) launch_rows<T, PER, 2>(a, l, wide);
  else if (a.tile_heads <= 4) launch_rows<T, PER, 4>(a, l, wide);
  else if constexpr (PER < 8) launch_rows<T, PER, 8>(a, l, wide);
}

template <class T>
void attend(const PagedArgs& a, const Launch& l) {
  const long long strides = a.page_stride[0] | a.page_stride[1];
  const uintptr_t bases = reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v);
  if constexpr (sizeof(T) == 2) {
    if (a.head_dim % 8 == 0 && strides % 8 == 0 && bases % 16 == 0) {
      // Up to 8 query heads of a cached head fill one product; more warps where a slab is short: it takes
      // a warp about as long whatever its bytes (128 sequences of up to 4000, 16 heads of 64: 182 us with
      // 16 warps, 212 with 8).
      const bool one = a.heads / a.kv_heads <= 8;
      if (a.head_dim <= 64) one ? launch_tiles<T, 4, 1, 3, 16, 4>(a, l) : launch_tiles<T, 4, 2, 6, 8, 4>(a, l);
      else if (a.head_dim <= 96) one ? launch_tiles<T, 6, 1, 2, 12, 3>(a, l) : launch_tiles<T, 6, 2, 4, 8, 3>(a, l);
      else if (a.head_dim <= 128) one ? launch_tiles<T, 8, 1, 3, 8, 3>(a, l) : launch_tiles<T, 8, 2, 3, 8, 3>(a, l);
      else one ? launch_tiles<T, 16, 1, 3, 4, 3>(a, l) : launch_tiles<T, 16, 2, 3, 4, 3>(a, l);
      return;
    }
  }
  const int per = a.head_dim <= 64 ? 2 : a.head_dim <= 128 ? 4 : 8;
  const bool wide = (a.head_dim | strides) % per == 0 && bases % std::min<size_t>(16, per * sizeof(T)) == 0;
  if (per == 2) launch_rows<T, 2>(a, l, wide);
  else if (per == 4) launch_rows<T, 4>(a, l, wide);
  else launch_rows<T, 8>(a, l, wide);
}

template <class T>
void k_paged_attention(OpCall& c) {
  const Tensor &q = c.in[0], &kp = c.in[1], &vp = c.in[2];
  const Shape& s = kp.shape();
  const long long B = q.shape()[0], H = q.shape()[1], width = c.in[3].shape()[1];
  if (B * H > 2147483647LL || H * kMostBatch > 2147483647LL || s[0] > 2147483647LL || s[2] > 1073741823LL || width > 2147483647LL)
    throw std::invalid_argument("paged_attention: too many heads or pages");
  PagedArgs a{};
  a.errors = index_error_counter();
  a.page_stride[0] = s[0] > 1 ? kp.strides()[0] : 0;
  a.page_stride[1] = s[0] > 1 ? vp.strides()[0] : 0;
  for (int d = 0; d < 2; ++d) a.qs[d] = q.shape()[d] > 1 ? q.strides()[d] : 0;
  a.k = kp.data();
  a.v = vp.data();
  a.heads = static_cast<int>(H);
  a.kv_heads = static_cast<int>(s[1]);
  a.head_dim = static_cast<int>(s[3]);
  a.page_size = static_cast<int>(s[2]);
  a.table_width = static_cast<int>(width);
  a.pages_total = static_cast<int>(s[0]);
  a.scale_log2 = static_cast<float>(c.f[0] * 1.4426950408889634);
  const Launch l{q.device(), sm_count_for(q), stream_of(c)};
  for (long long b = 0; b < B; b += kMostBatch) {
    a.batch = static_cast<int>(std::min<long long>(kMostBatch, B - b));
    a.q = q.data_as<T>() + b * a.qs[0];
    a.out = c.out[0].data_as<T>() + b * H * s[3];
    a.table = c.in[3].data_as<int>() + b * width;
    a.lengths = c.in[4].data_as<int>() + b;
    attend<T>(a, l);
  }
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
