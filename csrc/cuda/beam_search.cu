// Beam search's selection on sm_100a: the W best of the W V continuations of a sentence.
//
//   candidate (w, v) = score_w + x_wv - lse_w,   lse_w = log sum_v exp x_wv
//
// The logits are read once; that is the floor.  Within a beam the order of the candidates is the
// order of the logits, so the beams are cut into chunks, and a warp takes from one its W best (value,
// lowest place) together with its maximum and sum of exponentials, in one pass.  The last block of a
// sentence to arrive forms each beam's lse and picks the W best of the chunks' winners, in float64.
//
// One pass.  A warp's logits arrive by asynchronous copies, 128 pieces of 16 bytes at a time, into a
// ring of its own; rows that start off a 16-byte boundary are shifted together on the way out.  The
// first batch gives a bound: the lanes form G >= W groups, and the smallest of the groups' maxima is
// reached by at least G values (by about G ln G of them in random data).  Pieces that hold a value
// above the bound are put aside; when there are enough, and after the first batch, their values are
// cut to the W best, and the last of these is the bound from then on, so that later batches put
// hardly anything aside.  Should the values not fit their list (very many equal ones) the W best are
// taken one by one.  Values of -inf are no candidates; the selection is filled up with them if
// nothing else is left.
//
// Beams that offer equal scores have to tie, at whatever address their rows begin: values belong to
// lanes by their place in the row, exponentials are summed with compensation (to about 2^-45, so
// that their order hardly matters either), and the sum is rounded to float32 before its logarithm.
#include <algorithm>

#include "ob/cuda_common.cuh"

namespace ob {
namespace cu {
namespace {

constexpr int kThreads = 128, kWarps = kThreads / 32, kBlocksPerSm = 5, kList = 1024;
constexpr int kBatch = 4, kBatchVectors = kBatch * 32, kRing = 3, kStageBytes = (kBatchVectors + 1) * 16;
constexpr int kAside = kBatchVectors + 32;  // pieces that a warp has room for: at least a batch at any time
using Key = unsigned long long;  // order-preserving image of the value, then the complement of its place

struct ChunkStat {
  double sum;  // of exp(x - top)
  float top;
};

struct BeamArgs {
  const float* scores;
  const unsigned char* finished;
  ChunkStat* stat;  // [rows, chunks]
  Key* keys;        // [rows, chunks, beams], best first, 0: none
  float* out_scores;
  long long *parents, *tokens;
  unsigned char* done;
  unsigned int* arrived;  // blocks of each sentence
  int beams, vocab, chunks, chunk_vectors, groups, end;
  int list;  // keys that a warp has room for
};

__device__ __forceinline__ Key make_key(float v, unsigned at) {
  const unsigned u = __float_as_uint(v + 0.f);  // -0 and +0 are equal
  return static_cast<Key>(u & 0x80000000u ? ~u : u | 0x80000000u) << 32 | ~at;
}
__device__ __forceinline__ float key_value(Key k) {
  const unsigned u = static_cast<unsigned>(k >> 32);
  return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ unsigned key_place(Key k) { return ~static_cast<unsigned>(k); }

// 16 bytes that begin `off` bytes (a multiple of the element size) behind `p` in shared memory.
__device__ __forceinline__ uint4 load16(const unsigned char* p, unsigned off) {
  const uint4 lo = *reinterpret_cast<const uint4*>(p);
  if (off == 0) return lo;  // uniform: all vectors of a row start alike
  const uint4 hi = *reinterpret_cast<const uint4*>(p + 16);
  const unsigned bits = (off & 3u) * 8u;
  const unsigned w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
  uint4 r;
#define OB_SHIFTED(K) r = make_uint4(__funnelshift_r(w[K], w[K + 1], bits), __funnelshift_r(w[K + 1], w[K + 2], bits), \
                                     __funnelshift_r(w[K + 2], w[K + 3], bits), __funnelshift_r(w[K + 3], w[K + 4 > 7 ? 7 : K + 4], bits))
  switch (off >> 2) {
    case 0: OB_SHIFTED(0); break;
    case 1: OB_SHIFTED(1); break;
    case 2: OB_SHIFTED(2); break;
    default: OB_SHIFTED(3); break;
  }
#undef OB_SHIFTED
  return r;
}

template <class T>
struct Values {  // 16 bytes of logits
  static constexpr int N = 16 / sizeof(T);
  T v[N];
};
template <class T> __device__ __forceinline__ T lowest();
template <> __device__ __forceinline__ float lowest<float>() { return -INFINITY; }
template <> __device__ __forceinline__ __half lowest<__half>() { return __ushort_as_half(0xFC00); }
template <> __device__ __forceinline__ __nv_bfloat16 lowest<__nv_bfloat16>() { return __ushort_as_bfloat16(0xFF80); }

// Largest of 16 bytes of values; NaN is passed over.
__device__ __forceinline__ float largest(const Values<float>& x) { return fmaxf(fmaxf(x.v[0], x.v[1]), fmaxf(x.v[2], x.v[3])); }
__device__ __forceinline__ float largest(const Values<__half>& x) {
  const __half2* h = reinterpret_cast<const __half2*>(x.v);
  const __half2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
  return fmaxf(__low2float(m), __high2float(m));
}
__device__ __forceinline__ float largest(const Values<__nv_bfloat16>& x) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(x.v);
  const __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
  return fmaxf(__low2float(m), __high2float(m));
}

// Two float32 operations in one instruction.
struct Pair {
  unsigned long long bits;
  __device__ __forceinline__ Pair() {}
  __device__ __forceinline__ Pair(float lo, float hi) { asm("mov.b64 %0, {%1, %2};" : "=l"(bits) : "f"(lo), "f"(hi)); }
  __device__ __forceinline__ void split(float* lo, float* hi) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(*lo), "=f"(*hi) : "l"(bits)); }
};
__device__ __forceinline__ Pair add(Pair a, Pair b) {
  Pair c;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(c.bits) : "l"(a.bits), "l"(b.bits));
  return c;
}
__device__ __forceinline__ Pair mul(Pair a, Pair b) {
  Pair c;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(c.bits) : "l"(a.bits), "l"(b.bits));
  return c;
}
__device__ __forceinline__ Pair sub(Pair a, Pair b) {  // a - b, rounded once
  Pair c;
  const Pair minus(-1.f, -1.f);
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(c.bits) : "l"(b.bits), "l"(minus.bits), "l"(a.bits));
  return c;
}
__device__ __forceinline__ float power_of_two(float x) {  // 2 units in the last place; 0 below 2^-126
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Values 2k and 2k + 1 of 16 bytes.
__device__ __forceinline__ Pair two(const Values<float>& x, int k) { return Pair(x.v[2 * k], x.v[2 * k + 1]); }
__device__ __forceinline__ Pair two(const Values<__half>& x, int k) {
  const float2 f = __half22float2(reinterpret_cast<const __half2*>(x.v)[k]);
  return Pair(f.x, f.y);
}
__device__ __forceinline__ Pair two(const Values<__nv_bfloat16>& x, int k) {
  const unsigned w = reinterpret_cast<const unsigned*>(x.v)[k];
  return Pair(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

// Smallest and largest of the maxima of `groups` groups of threads (thread modulo groups); every
// thread gets both.  `shared`: 256 values.  Synchronises once.
template <class F>
__device__ __forceinline__ void group_maxima(F mine, int groups, F* shared, F* smallest, F* top) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, width = min(groups, 32);
  for (int o = width; o < 32; o <<= 1) mine = fmax(mine, __shfl_xor_sync(0xffffffffu, mine, o));
  if (lane < width) shared[warp * width + lane] = mine;
  __syncthreads();
  F hi = static_cast<F>(-INFINITY), lo = static_cast<F>(INFINITY);
  for (int g = lane; g < groups; g += 32) {  // 64 groups: two warps side by side
    F m = static_cast<F>(-INFINITY);
    for (int i = g; i < kWarps * width; i += groups) m = fmax(m, shared[i]);
    hi = fmax(hi, m);
    lo = fmin(lo, m);
  }
  for (int o = 16; o > 0; o >>= 1) {
    hi = fmax(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    lo = fmin(lo, __shfl_xor_sync(0xffffffffu, lo, o));
  }
  *smallest = lo;
  *top = hi;
}

struct Shared {         // of the selection; it lies where the warps' memory was
  double best[kList];
  Key place[kList];     // (beam, token)
  double base[64];      // score - lse, or the score of a finished beam; NaN: the beam offers nothing
  float maxima[kThreads];
  int count;
  bool ended[64];
};

// The W largest of keys[0..n) in order to sorted[0..W), zeros behind the last; by one warp.
__device__ __forceinline__ void sort_best(const Key* keys, int n, Key* sorted, int W, int lane) {
  for (int i = n + lane; i < W; i += 32) sorted[i] = 0;
  for (int i = lane; i < n; i += 32) {
    const Key mine = keys[i];
    int before = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) before += keys[j] > mine;
    if (before < W) sorted[before] = mine;
  }
  __syncwarp();
}

// A warp's memory: the ring, pieces put aside with their numbers, keys (the W best first), and room
// for 64 sorted ones.
__host__ __device__ constexpr size_t warp_bytes(int list) {
  return static_cast<size_t>(kRing) * kStageBytes + kAside * 20 + (static_cast<size_t>(list) + 64) * sizeof(Key);
}

// The values of the pieces[0..n) that lie above the bound join the keys[0..held) chosen before; the W
// best of all are left there, in order.  Returns how many there are.
template <class T>
__device__ __forceinline__ int cut(const uint4* pieces, const int* numbers, int n, Key* keys, int held, float bound, int list, int W, int lane) {
  constexpr int N = Values<T>::N;
  Key* sorted = keys + list;
  __syncwarp();
  int total = held;
  for (int i0 = 0; i0 < n; i0 += 32) {
    const bool there = i0 + lane < n;
    Values<T> x;
    int q = 0;
    if (there) {
      *reinterpret_cast<uint4*>(&x) = pieces[i0 + lane];
      q = numbers[i0 + lane];
    }
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const float v = there ? to_f(x.v[k]) : -INFINITY;
      const unsigned who = __ballot_sync(0xffffffffu, v > bound);
      const int at = total + __popc(who & ((1u << lane) - 1u));
      if (v > bound && at < list) keys[at] = make_key(v, q * N + k);
      total += __popc(who);
    }
  }
  __syncwarp();
  if (total <= list) {
    sort_best(keys, total, sorted, W, lane);
  } else {
    Key after = ~0ull;
    for (int r = 0; r < W; ++r) {
      Key best = 0;
      for (int i = lane; i < held; i += 32)
        if (keys[i] < after && keys[i] > best) best = keys[i];
      for (int i = lane; i < n; i += 32) {
        Values<T> x;
        *reinterpret_cast<uint4*>(&x) = pieces[i];
        for (int k = 0; k < N; ++k) {
          const float v = to_f(x.v[k]);
          const Key key = make_key(v, numbers[i] * N + k);
          if (v > bound && key < after && key > best) best = key;
        }
      }
      for (int o = 16; o > 0; o >>= 1) {
        const Key other = __shfl_xor_sync(0xffffffffu, best, o);
        best = other > best ? other : best;
      }
      if (lane == 0) sorted[r] = best;
      after = best;
    }
    __syncwarp();
  }
  for (int i = lane; i < W; i += 32) keys[i] = sorted[i];
  __syncwarp();
  return min(total, W);
}

// The W best of one chunk into a.keys, its maximum and sum into a.stat; by one warp.  `offers`:
// whether the beam has continuations, looked up while the first logits are on their way.
template <class T, class Offers>
__device__ __forceinline__ void take_chunk(const T* __restrict__ logits, const BeamArgs& a, long long row, int chunk, unsigned char* memory,
                                           Offers offers) {
  constexpr int N = Values<T>::N;
  const int lane = threadIdx.x & 31, W = a.beams;
  const char* begin = reinterpret_cast<const char*>(logits + row * a.vocab);
  const char* end = begin + static_cast<long long>(a.vocab) * sizeof(T);
  const unsigned off = static_cast<unsigned>(reinterpret_cast<uintptr_t>(begin)) & 15u;
  const int first = chunk * a.chunk_vectors, last = min(first + a.chunk_vectors, (a.vocab + N - 1) / N);
  const int batches = (last - first + kBatchVectors - 1) / kBatchVectors;
  const uint32_t ring_at = static_cast<uint32_t>(__cvta_generic_to_shared(memory));

  // Aligned words that hold bytes of the row; a shifted row needs one word more than it has pieces.
  const char* from = begin - off + (static_cast<long long>(first) + lane) * 16;  // of the next batch
  auto load_batch = [&](int stage) {
    const uint32_t to = ring_at + stage * kStageBytes + lane * 16;
    if (from + kBatchVectors * 16 < end) {
#pragma unroll
      for (int i = 0; i < kBatch; ++i) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + i * 512), "l"(from + i * 512) : "memory");
      if (off != 0 && lane == 0)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + kBatch * 512), "l"(from + kBatch * 512) : "memory");
    } else {
#pragma unroll
      for (int i = 0; i <= kBatch; ++i)
        if ((i < kBatch || (off != 0 && lane == 0)) && from + i * 512 < end)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + i * 512), "l"(from + i * 512) : "memory");
    }
    from += kBatchVectors * 16;
  };
#pragma unroll
  for (int b = 0; b < kRing - 1; ++b) {
    if (b < batches) load_batch(b);
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  uint4* pieces = reinterpret_cast<uint4*>(memory + kRing * kStageBytes);
  int* numbers = reinterpret_cast<int*>(pieces + kAside);
  Key* keys = reinterpret_cast<Key*>(numbers + kAside);
  int aside = 0, held = 0;
  float bound = -INFINITY;  // only larger values matter
  if (!offers()) {
    asm volatile("cp.async.wait_all;" ::: "memory");
    return;
  }
  const Pair log2e(1.44269504f, 1.44269504f);
  Pair sum(1.f, 1.f), rest(0.f, 0.f);  // sums start at 1 >= every term: the error of an addition is (term - (new - old))
  float top = -INFINITY;
  int stage = 0;
  for (int batch = 0;; ++batch) {
    if (batch == 1 || batch == batches || aside > kAside - kBatchVectors) {
      held = cut<T>(pieces, numbers, aside, keys, held, bound, a.list, W, lane);
      // With W of them only a larger value can still displace one, for its place is behind theirs.
      bound = held == W ? key_value(keys[W - 1]) : -INFINITY;
      aside = 0;
    }
    if (batch == batches) break;
    asm volatile("cp.async.wait_group %0;" ::"n"(kRing - 2) : "memory");
    __syncwarp();
    if (batch + kRing - 1 < batches) load_batch(stage == 0 ? kRing - 1 : stage - 1);
    asm volatile("cp.async.commit_group;" ::: "memory");
    const int q0 = first + batch * kBatchVectors;
    Values<T> x[kBatch];
    float m[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) *reinterpret_cast<uint4*>(&x[i]) = load16(memory + stage * kStageBytes + (i * 32 + lane) * 16, off);
    if (q0 + kBatchVectors > last || (q0 + kBatchVectors) * N > a.vocab) {
#pragma unroll
      for (int i = 0; i < kBatch; ++i)
#pragma unroll
        for (int k = 0; k < N; ++k) {
          const int q = q0 + i * 32 + lane;
          if (q >= last || q * N + k >= a.vocab) x[i].v[k] = lowest<T>();
        }
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) m[i] = largest(x[i]);
    const float m01 = fmaxf(m[0], m[1]), m23 = fmaxf(m[2], m[3]), mine = fmaxf(m01, m23);

    if (__any_sync(0xffffffffu, mine > top)) {  // a new maximum: what has been summed is rescaled
      const float new_top = fmaxf(top, warp_max(mine)), keep = top == -INFINITY ? 1.f : power_of_two((top - new_top) * 1.44269504f);
      float s[2], r[2];
      sum.split(&s[0], &s[1]);
      rest.split(&r[0], &r[1]);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float scaled = (s[c] - 1.f) * keep;
        s[c] = __fadd_rn(1.f, scaled);
        r[c] = r[c] * keep + __fsub_rn(scaled, __fsub_rn(s[c], 1.f));
      }
      sum = Pair(s[0], s[1]);
      rest = Pair(r[0], r[1]);
      top = new_top;
    }
    if (batch == 0) {
      float low = m01, high = m23;  // 64 groups: two of each lane
      if (W <= 32) {
        low = mine;
        for (int o = a.groups; o < 32; o <<= 1) low = fmaxf(low, __shfl_xor_sync(0xffffffffu, low, o));
        high = low;
      }
      low = -warp_max(-fminf(low, high));
      bound = low == -INFINITY ? low : nextafterf(low, -INFINITY);  // values that reach it lie above
    }
    if (__any_sync(0xffffffffu, mine > bound)) {
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const unsigned who = __ballot_sync(0xffffffffu, m[i] > bound);
        if (m[i] > bound) {
          const int at = aside + __popc(who & ((1u << lane) - 1u));
          pieces[at] = *reinterpret_cast<const uint4*>(&x[i]);
          numbers[at] = q0 + i * 32 + lane;
        }
        aside += __popc(who);
      }
    }
    const float origin = top == -INFINITY ? 0.f : -top;
    const Pair minus_top(origin, origin);
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
#pragma unroll
      for (int k = 0; k < N / 2; ++k) {
        float lo, hi;
        mul(add(two(x[i], k), minus_top), log2e).split(&lo, &hi);
        const Pair e(power_of_two(lo), power_of_two(hi)), next = add(sum, e);
        rest = add(rest, sub(e, sub(next, sum)));
        sum = next;
      }
    stage = stage + 1 == kRing ? 0 : stage + 1;
  }
  float s0, s1, r0, r1;
  sum.split(&s0, &s1);
  rest.split(&r0, &r1);
  double total = static_cast<double>(s0 - 1.f) + (s1 - 1.f) + (static_cast<double>(r0) + r1);
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  const long long slot = row * a.chunks + chunk;
  if (lane == 0) a.stat[slot] = ChunkStat{total, top};
  for (int i = lane; i < W; i += 32) a.keys[slot * W + i] = keys[i];
}

// The selection of one sentence from its chunks' winners.
template <class T>
__device__ __noinline__ void select_beams(const T* __restrict__ logits, const BeamArgs& a, int sentence, Shared& sh) {
  const int W = a.beams, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const long long row0 = static_cast<long long>(sentence) * W;
  if (tid == 0) sh.count = 0;
  for (int w = warp; w < W; w += kWarps) {
    const float s = a.scores[row0 + w];
    const bool fin = a.finished != nullptr && a.finished[row0 + w] != 0;
    double b = s;
    if (!isfinite(s)) b = NAN;
    else if (!fin) {
      const ChunkStat* st = a.stat + (row0 + w) * a.chunks;
      float top = -INFINITY;
      for (int c = lane; c < a.chunks; c += 32) top = fmaxf(top, __ldcg(&st[c].top));
      top = warp_max(top);
      double sum = 0.0;
      for (int c = lane; c < a.chunks; c += 32) {
        // A chunk without a finite value adds its sum (0, or NaN) as it is.
        const float t = __ldcg(&st[c].top);
        const double part = __ldcg(&st[c].sum);
        sum += t == top || t == -INFINITY ? part : part * expf(t - top);
      }
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      // log sum: the exponent in float64, the mantissa in [1, 2) in float32 (2^-24 either way).
      int exponent;
      const float mantissa = 2.f * frexpf(static_cast<float>(sum), &exponent);
      b = top == -INFINITY || !isfinite(sum) ? static_cast<double>(NAN)
                                             : s - (top + ((exponent - 1) * 0.69314718055994531 + static_cast<double>(logf(mantissa))));
    }
    if (lane == 0) {
      sh.base[w] = b;
      sh.ended[w] = fin;
    }
  }
  __syncthreads();
  const int per_row = a.chunks * W, n_all = W * per_row;  // candidates of a beam, of all
  // Candidate i: its score, or -inf where there is none.
  auto candidate = [&](int i, int w, Key* at) {
    const double b = sh.base[w];
    if (isnan(b)) return static_cast<double>(-INFINITY);
    if (sh.ended[w]) {
      *at = static_cast<Key>(w) << 32 | static_cast<unsigned>(a.end);
      return i == w * per_row ? b : static_cast<double>(-INFINITY);
    }
    const Key key = __ldcg(a.keys + row0 * per_row + i);
    if (key == 0) return static_cast<double>(-INFINITY);
    *at = static_cast<Key>(w) << 32 | key_place(key);
    return b + key_value(key);
  };
  // As in a chunk: the best of each chunk in G groups, the smallest of the groups' maxima as the
  // bound.  Rounding down keeps the order, so that it can be done in float32.
  float top = -INFINITY;
  Key at = 0;
  for (int i = tid; i < W * a.chunks; i += kThreads) top = fmaxf(top, __double2float_rd(candidate(i * W, i / a.chunks, &at)));
  float reach, unused;
  group_maxima<float>(top, a.groups, sh.maxima, &reach, &unused);
#pragma unroll 2
  for (int i = tid; i < n_all; i += kThreads) {
    const double c = candidate(i, i / per_row, &at);
    if (c > -INFINITY && __double2float_rd(c) >= reach) {
      const int to = atomicAdd(&sh.count, 1);
      if (to < kList) {
        sh.best[to] = c;
        sh.place[to] = at;
      }
    }
  }
  __syncthreads();
  const int n = sh.count;
  auto emit = [&](int k, double score, int w, unsigned token) {
    a.out_scores[row0 + k] = static_cast<float>(score);
    a.parents[row0 + k] = w;
    a.tokens[row0 + k] = token;
    a.done[row0 + k] = sh.ended[w] || (a.end >= 0 && token == static_cast<unsigned>(a.end));
  };
  if (n <= kList) {
    for (int i = tid; i < n; i += kThreads) {
      const double mine = sh.best[i];
      const Key my_place = sh.place[i];
      int before = 0;
#pragma unroll 4
      for (int j = 0; j < n; ++j) before += sh.best[j] > mine || (sh.best[j] == mine && sh.place[j] < my_place);
      if (before < W) emit(before, mine, static_cast<int>(my_place >> 32), static_cast<unsigned>(my_place));
    }
    if (n < W && tid == 0) {  // nothing else is left than -inf: the lowest places that have it
      const long long vocab = a.vocab;
      long long f = 0;
      for (int k = n; k < W; ++f) {  // fewer than W places are passed over
        const int w = static_cast<int>(f / vocab);
        const unsigned v = static_cast<unsigned>(f - w * vocab);
        const bool nothing = isnan(sh.base[w]) ||
                             (sh.ended[w] ? v != static_cast<unsigned>(a.end) : !(to_f(logits[row0 * vocab + f]) > -INFINITY));
        if (nothing) emit(k++, -INFINITY, w, v);
      }
    }
    return;
  }
  double last = INFINITY;  // one by one, as above
  Key last_at = 0;
  for (int k = 0; k < W; ++k) {
    double mine = -INFINITY;
    Key my_place = ~0ull;
    for (int i = tid; i < n_all; i += kThreads) {
      const double c = candidate(i, i / per_row, &at);
      if (c > -INFINITY && (c < last || (c == last && at > last_at)) && (c > mine || (c == mine && at < my_place))) {
        mine = c;
        my_place = at;
      }
    }
    for (int o = 16; o > 0; o >>= 1) {
      const double c = __shfl_xor_sync(0xffffffffu, mine, o);
      const Key p = __shfl_xor_sync(0xffffffffu, my_place, o);
      if (c > mine || (c == mine && p < my_place)) { mine = c; my_place = p; }
    }
    __syncthreads();
    if (lane == 0) { sh.best[warp] = mine; sh.place[warp] = my_place; }
    __syncthreads();
    for (int w = 0; w < kWarps; ++w)
      if (sh.best[w] > mine || (sh.best[w] == mine && sh.place[w] < my_place)) { mine = sh.best[w]; my_place = sh.place[w]; }
    last = mine;
    last_at = my_place;
    if (tid == 0) emit(k, mine, static_cast<int>(my_place >> 32), static_cast<unsigned>(my_place));
  }
}

template <class T>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm) beam_step_kernel(const T* __restrict__ logits, const __grid_constant__ BeamArgs a) {
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ int flag;
  const int warp = threadIdx.x >> 5, tasks = a.beams * a.chunks, blocks = (tasks + kWarps - 1) / kWarps;
  const int sentence = blockIdx.x / blocks, task = (blockIdx.x - sentence * blocks) * kWarps + warp;
  if (task < tasks) {
    const int w = task / a.chunks;
    const long long row = static_cast<long long>(sentence) * a.beams + w;
    // A beam that has ended, or has no score, offers no continuation.
    const bool ended = a.finished != nullptr && a.finished[row] != 0;
    const float score = a.scores[row];
    take_chunk<T>(logits, a, row, task - w * a.chunks, smem + warp * warp_bytes(a.list), [&] { return !ended && isfinite(score); });
  }
  if (last_to_arrive(a.arrived + sentence, static_cast<unsigned>(blocks), &flag))
    select_beams<T>(logits, a, sentence, *reinterpret_cast<Shared*>(smem));
}

// Chunks of a beam: enough warps for the device without chunks so short that their beginnings
// and the joining cost more than they gain.  Both are counted in batches: a block's waves times
// the batches of a chunk and four for its start (measured on one, 40 and 512 rows).
int choose_chunks(long long sentences, int beams, long long vectors, int sms) {
  const long long batches = (vectors + kBatchVectors - 1) / kBatchVectors;
  long long best = 1, best_cost = 0;
  for (long long c = 1; c <= std::min<long long>(batches, 256); ++c) {
    const long long blocks = sentences * ((beams * c + kWarps - 1) / kWarps), slots = static_cast<long long>(sms) * kBlocksPerSm;
    const long long cost = (blocks + slots - 1) / slots * ((batches + c - 1) / c + 4);
    if (c == 1 || cost < best_cost) { best = c; best_cost = cost; }
  }
  return static_cast<int>(best);
}

template <class T>
void k_beam_step(OpCall& c) {
  const Shape& s = c.in[0].shape();
  constexpr int N = Values<T>::N;
  const long long rows = s[0] * s[1], vectors = (s[2] + N - 1) / N;
  const long long chunks = choose_chunks(s[0], static_cast<int>(s[1]), vectors, sm_count_for(c.in[0]));
  if (rows * chunks > 2147483647LL) throw std::invalid_argument("beam_search_step: too many rows");
  BeamArgs a{};
  a.scores = c.in[1].data_as<float>();
  a.finished = c.in[2].defined() ? c.in[2].data_as<unsigned char>() : nullptr;
  a.out_scores = c.out[0].data_as<float>();
  a.parents = c.out[1].data_as<long long>();
  a.tokens = c.out[2].data_as<long long>();
  a.done = c.out[3].data_as<unsigned char>();
  a.beams = static_cast<int>(s[1]);
  a.vocab = static_cast<int>(s[2]);
  a.chunks = static_cast<int>(chunks);
  a.chunk_vectors = static_cast<int>((vectors + chunks - 1) / chunks);
  a.end = static_cast<int>(c.i[0]);
  a.groups = 8;
  while (a.groups < a.beams) a.groups *= 2;
  cudaStream_t st = stream_of(c);
  const size_t stat_bytes = static_cast<size_t>(rows * chunks) * sizeof(ChunkStat);
  ScratchLease scratch(c.in[0].device(), stat_bytes + static_cast<size_t>(rows * chunks * s[1]) * sizeof(Key), st);
  a.stat = static_cast<ChunkStat*>(scratch.data());
  a.keys = reinterpret_cast<Key*>(static_cast<char*>(scratch.data()) + stat_bytes);
  const T* logits = c.in[0].data_as<T>();
  a.arrived = arrival_counters(c.in[0].device(), st, static_cast<size_t>(s[0]));
  a.list = s[1] <= 8 ? 128 : s[1] <= 16 ? 256 : 512;
  const size_t smem = kWarps * warp_bytes(a.list);
  static_assert(sizeof(Shared) <= kWarps * warp_bytes(128), "the selection lies in the warps' memory");
  OB_CUDA(cudaFuncSetAttribute(beam_step_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
  const long long blocks = s[0] * ((s[1] * chunks + kWarps - 1) / kWarps);
  beam_step_kernel<T><<<static_cast<unsigned>(blocks), kThreads, smem, st>>>(logits, a);
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
