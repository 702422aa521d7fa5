// Beam search's selection on sm_100a: the W best of the W V continuations of a sentence.
//
//   candidate (w, v) = score_w + x_wv - lse_w,   lse_w = log sum_v exp x_wv
//
// The logits are read once; that is the floor (512 rows of 100003 in bfloat16, every fifth at its end:
// 82 MB, 12.5 us).  It takes 46 us.  A batch of 1024 logits costs a warp about 330 instructions, of which exponentials and
// their compensated sum are half: the 40000 batches are 13 of the 17.5 million that are issued, 16 us if every slot
// were taken.  Half are: a scheduler has 2.3 warps on average, each with one batch at a time, and the SMs are active for 52 to 84
// thousand cycles, since blocks of finished beams leave at once and the others fall on SMs by chance.  The start
// of a warp, with cold code, and the selection are 10 us.  Within a beam the order of the candidates is the
// order of the logits, so the beams are cut into chunks, and a warp takes from one its W best (value,
// lowest place) together with its maximum and sum of exponentials, in one pass.  The last warp of a
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
// Beams of the same logits have to tie, at whatever address their rows begin: values belong to lanes by their
// place in the row, so that the same numbers are added in the same order.  The same logits in another order need not
// tie: an exponential (2^-22 of itself) is taken relative to the largest logit so far, and a new largest one rescales
// the sum by a rounded factor, so that the order matters at about 2^-22 of the sum.  The sum itself is compensated: the
// thousands of additions of a lane would lose more than that.  Candidates of different beams are told apart down to
// the error of their lse, 2^-20 at most in the tests; those of one beam by their logits, exactly.
#include <algorithm>
#include <atomic>
#include <cmath>

#include "ob/cuda_common.cuh"

namespace ob {
namespace cu {
namespace {

constexpr int kWarpsPerSm = 19, kMostLists = 256;  // blocks of one warp, at most; chunks of a sentence that the selection has room for
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

__device__ __forceinline__ Key order_of(double v) {
  const Key u = static_cast<Key>(__double_as_longlong(v + 0.0));
  return u >> 63 ? ~u : u | 0x8000000000000000ull;
}
__device__ __forceinline__ double score_of(Key k) {
  return __longlong_as_double(static_cast<long long>(k >> 63 ? k & 0x7fffffffffffffffull : ~k));
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

struct Selection {      // of a sentence; it lies where the chunk's memory was
  struct List {         // a chunk's winners that have not been taken yet
    Key order, place;   // the first: order-preserving image of its score (0: none is left), (beam, token)
    Key next;           // the second, as the chunk left it
    double sum;         // of the chunk
    float top;
    int taken;          // entries behind the first two are found from here
  } list[kMostLists];
  double base[64];      // score - lse, or the score of a finished beam; NaN: the beam offers nothing
  bool ended[64];
};

// The smallest of the maxima of `groups` interleaved groups of lanes; with 64 groups each lane has two.
template <class K>
__device__ __forceinline__ K least_maximum(K first, K second, int groups) {
  K mine = groups <= 32 ? max(first, second) : min(first, second);
  for (int o = groups; o < 32; o <<= 1) mine = max(mine, __shfl_xor_sync(0xffffffffu, mine, o));
  for (int o = 1; o < min(groups, 32); o <<= 1) mine = min(mine, __shfl_xor_sync(0xffffffffu, mine, o));
  return mine;
}

// The W largest of keys[0..n) in order to sorted[0..W), zeros behind the last; by one warp.  Each
// counts the keys before it; when there are many, only those that reach the smallest of the
// maxima of `groups` interleaved groups are left to count.
__device__ __forceinline__ void sort_best(Key* keys, int n, Key* sorted, int W, int groups, int lane) {
  if (n > 32 && n >= groups) {
    Key first = 0, second = 0;
    for (int i = lane; i < n; i += 64) {
      first = max(first, keys[i]);
      if (i + 32 < n) second = max(second, keys[i + 32]);
    }
    const Key mine = least_maximum(first, second, groups);
    int left = 0;
    for (int i0 = 0; i0 < n; i0 += 32) {
      const Key key = i0 + lane < n ? keys[i0 + lane] : 0;
      const unsigned who = __ballot_sync(0xffffffffu, i0 + lane < n && key >= mine);
      __syncwarp();
      if (who >> lane & 1u) keys[left + __popc(who & ((1u << lane) - 1u))] = key;
      left += __popc(who);
    }
    n = left;
    __syncwarp();
  }
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

// The W best of keys[0..held) and of the pieces' values above the bound, to sorted.
template <class T>
__device__ __noinline__ void take_one_by_one(const uint4* pieces, const int* numbers, int n, const Key* keys, int held, float bound, Key* sorted,
                                             int W, int lane) {
  constexpr int N = Values<T>::N;
  Key after = ~0ull;
  for (int r = 0; r < W; ++r) {
    Key best = 0;
    for (int i = lane; i < held; i += 32)
      if (keys[i] < after && keys[i] > best) best = keys[i];
    for (int i = lane; i < n; i += 32) {
      const T* values = reinterpret_cast<const T*>(pieces + i);
#pragma unroll 1
      for (int k = 0; k < N; ++k) {
        const float v = to_f(values[k]);
        const Key key = make_key(v, numbers[i] * N + k);
        if (v > bound && key < after && key > best) best = key;
      }
    }
    for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
    if (lane == 0) sorted[r] = best;
    after = best;
  }
  __syncwarp();
}

// The values of the pieces[0..n) that lie above the bound join the keys[0..held) chosen before; the W
// best of all are left there, in order.  Returns how many there are.
template <class T>
__device__ __forceinline__ int cut(const uint4* pieces, const int* numbers, int n, Key* keys, int held, float bound, int list, int W, int groups,
                                   int lane) {
  constexpr int N = Values<T>::N;
  Key* sorted = keys + list;
  __syncwarp();
  int total = held;
  for (int i0 = 0; i0 < n; i0 += 32) {
    const bool there = i0 + lane < n;
    Values<T> x;
    unsigned mine = 0;  // which of the piece's values count: hardly ever more than one
    int q = 0;
    if (there) {
      *reinterpret_cast<uint4*>(&x) = pieces[i0 + lane];
      q = numbers[i0 + lane] * N;
#pragma unroll
      for (int k = 0; k < N; ++k) mine |= to_f(x.v[k]) > bound ? 1u << k : 0u;
    }
    const int many = __popc(mine);
    int at = many;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int before = __shfl_up_sync(0xffffffffu, at, o);
      if (lane >= o) at += before;
    }
    const int all = __shfl_sync(0xffffffffu, at, 31);
    at += total - many;
    const T* values = reinterpret_cast<const T*>(pieces + i0 + lane);
    for (; mine != 0; mine &= mine - 1, ++at) {
      const int k = __ffs(mine) - 1;
      if (at < list) keys[at] = make_key(to_f(values[k]), q + k);
    }
    total += all;
  }
  __syncwarp();
  if (total <= list) sort_best(keys, total, sorted, W, groups, lane);
  else take_one_by_one<T>(pieces, numbers, n, keys, held, bound, sorted, W, lane);
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
      held = cut<T>(pieces, numbers, aside, keys, held, bound, a.list, W, a.groups, lane);
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
    unsigned char* here = memory + stage * kStageBytes;
    if (q0 + kBatchVectors > last || (q0 + kBatchVectors) * N > a.vocab) {  // what lies behind the chunk counts as -inf
      T* values = reinterpret_cast<T*>(here + off);
      for (int e = min(last * N, a.vocab) - q0 * N + lane; e < kBatchVectors * N; e += 32) values[e] = lowest<T>();
      __syncwarp();
    }
    Values<T> x[kBatch];
    float m[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) *reinterpret_cast<uint4*>(&x[i]) = load16(here + (i * 32 + lane) * 16, off);
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
      const float low = least_maximum(m01, m23, a.groups);
      bound = low == -INFINITY ? low : nextafterf(low, -INFINITY);  // values that reach it lie above
    }
    if (__any_sync(0xffffffffu, mine > bound)) {
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const unsigned who = __ballot_sync(0xffffffffu, m[i] > bound);
        if (who == 0) continue;
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

// Entries n..W are -inf: the lowest places that have it.
template <class T>
__device__ __noinline__ void fill_up(const T* logits, const Selection* sh, float* scores, long long* parents, long long* tokens,
                                     unsigned char* done, int n, int W, int vocab, int end) {
  long long f = 0;
  for (int k = n; k < W; ++f) {  // fewer than W places are passed over
    const int w = static_cast<int>(f / vocab), v = static_cast<int>(f - static_cast<long long>(w) * vocab);
    const bool nothing = isnan(sh->base[w]) || (sh->ended[w] ? v != end : !(to_f(logits[f]) > -INFINITY));
    if (!nothing) continue;
    scores[k] = -INFINITY;
    parents[k] = w;
    tokens[k] = v;
    done[k++] = sh->ended[w] || v == end;
  }
}

// The selection of one sentence from its chunks' winners; by one warp.  The chunks' lists are in
// order: W times the best of their heads is taken, and its list moves on.  The warp comes here once
// and finds the code in no instruction cache, so it is short loops rather than fast ones.  A round
// takes 850 cycles (1200 with shuffles of all 128 bits in place of the reductions).
template <class T>
__device__ __forceinline__ void select_beams(const T* __restrict__ logits, const BeamArgs& a, int sentence, Selection& sh) {
  const int W = a.beams, C = a.chunks, lane = threadIdx.x, lists = W * C;
  const long long row0 = static_cast<long long>(sentence) * W;
  const Key* keys = a.keys + row0 * C * W;
#pragma unroll 2
  for (int i = lane; i < lists; i += 32) {
    const ChunkStat* st = a.stat + row0 * C + i;
    const double sum = __ldcg(&st->sum);
    const float top = __ldcg(&st->top);
    const Key head = __ldcg(keys + i * W), next = W > 1 ? __ldcg(keys + i * W + 1) : 0;
    Selection::List& l = sh.list[i];
    l.sum = sum;
    l.top = top;
    l.order = head;
    l.next = next;
    l.taken = 2;
  }
  __syncwarp();
#pragma unroll 1
  for (int w = lane; w < W; w += 32) {
    const float s = a.scores[row0 + w];
    const bool ended = a.finished != nullptr && a.finished[row0 + w] != 0;
    double base = isfinite(s) ? s : NAN;
    Selection::List* l = sh.list + w * C;
    if (!ended && isfinite(s)) {
      float top = -INFINITY;
#pragma unroll 1
      for (int c = 0; c < C; ++c) top = fmaxf(top, l[c].top);
      double sum = 0.0;  // a chunk without a finite value adds its sum (0, or NaN) as it is
#pragma unroll 1
      for (int c = 0; c < C; ++c) sum += l[c].sum * (l[c].top == top || l[c].top == -INFINITY ? 1.f : __expf(l[c].top - top));
      // log sum: the exponent in float64, the mantissa in [1, 2) in float32 (2^-24 either way).
      const unsigned bits = __float_as_uint(static_cast<float>(sum));
      const float mantissa = __uint_as_float((bits & 0x007fffffu) | 0x3f800000u);
      base = top == -INFINITY || !isfinite(sum)
                 ? static_cast<double>(NAN)
                 : s - (top + ((static_cast<int>(bits >> 23) - 127) * 0.69314718055994531 + static_cast<double>(logf(mantissa))));
    }
    sh.base[w] = base;
    sh.ended[w] = ended;
  }
  __syncwarp();
  // Heads become candidates.
  auto offer = [&](Selection::List& l, int w, Key key, double base) {
    l.order = key == 0 ? 0 : order_of(base + key_value(key));
    l.place = static_cast<Key>(w) << 32 | key_place(key);
  };
#pragma unroll 1
  for (int i = lane; i < lists; i += 32) {
    Selection::List& l = sh.list[i];
    const int w = i / C;
    const double base = sh.base[w];
    if (isnan(base) || sh.ended[w]) {  // nothing, or a finished beam itself
      l.order = !isnan(base) && i == w * C ? order_of(base) : 0;
      l.place = static_cast<Key>(w) << 32 | static_cast<unsigned>(a.end);
      l.next = 0;
      l.taken = W;
    } else {
      offer(l, w, l.order, base);
    }
  }
  __syncwarp();
  Key coming = 0;  // a list's entry on its way from memory; it is needed a round later at the earliest
  int comes_to = -1, n = 0;
  Key best, place;  // of the lane's own lists
  int from = 0;
  auto look = [&] {
    best = 0;
    place = ~0ull;
#pragma unroll 1
    for (int i = lane; i < lists; i += 32) {
      const Key o = sh.list[i].order, p = sh.list[i].place;
      if (o > best || (o == best && o != 0 && p < place)) { best = o; place = p; from = i; }
    }
  };
  look();
  Key chosen[2], chosen_place[2];  // entry n is lane n % 32's; all are written together
#pragma unroll 1
  for (; n < W; ++n) {
    const unsigned upper = static_cast<unsigned>(best >> 32), top_upper = __reduce_max_sync(0xffffffffu, upper);
    const unsigned lower = static_cast<unsigned>(best), top_lower = __reduce_max_sync(0xffffffffu, upper == top_upper ? lower : 0u);
    if ((top_upper | top_lower) == 0) break;
    bool holds = upper == top_upper && lower == top_lower;
    unsigned who = __ballot_sync(0xffffffffu, holds);
    if ((who & (who - 1)) != 0) {  // equal scores: the lowest beam, then the lowest token
      const unsigned w = static_cast<unsigned>(place >> 32), v = static_cast<unsigned>(place);
      const unsigned least_w = __reduce_min_sync(0xffffffffu, holds ? w : ~0u);  // by all lanes, whatever they hold
      holds = holds && w == least_w;
      const unsigned least_v = __reduce_min_sync(0xffffffffu, holds ? v : ~0u);
      holds = holds && v == least_v;
      who = __ballot_sync(0xffffffffu, holds);
    }
    const Key top_place = __shfl_sync(0xffffffffu, place, __ffs(who) - 1);
    if (lane == (n & 31)) {
      const Key top = static_cast<Key>(top_upper) << 32 | top_lower;
      if (n < 32) { chosen[0] = top; chosen_place[0] = top_place; }
      else { chosen[1] = top; chosen_place[1] = top_place; }
    }
    if (holds) {
      if (comes_to >= 0) sh.list[comes_to].next = coming;
      Selection::List& l = sh.list[from];
      const int w = static_cast<int>(place >> 32);
      offer(l, w, l.next, sh.base[w]);
      coming = l.taken < W ? __ldcg(keys + from * W + l.taken) : 0;
      comes_to = from;
      l.taken += 1;
      look();
    }
  }
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int k = half * 32 + lane;
    if (k >= n) continue;
    const int w = static_cast<int>(chosen_place[half] >> 32), token = static_cast<int>(static_cast<unsigned>(chosen_place[half]));
    a.out_scores[row0 + k] = static_cast<float>(score_of(chosen[half]));
    a.parents[row0 + k] = w;
    a.tokens[row0 + k] = token;
    a.done[row0 + k] = sh.ended[w] || token == a.end;
  }
  if (n < W && lane == 0)  // nothing else is left than -inf
    fill_up<T>(logits + row0 * a.vocab, &sh, a.out_scores + row0, a.parents + row0, a.tokens + row0, a.done + row0, n, W, a.vocab, a.end);
}

// Blocks of one warp: chunks are uneven work (finished beams have none), and a warp that is done makes
// room for the next at once.
template <class T>
__global__ void __launch_bounds__(32, kWarpsPerSm) beam_step_kernel(const T* __restrict__ logits, const __grid_constant__ BeamArgs a) {
  extern __shared__ __align__(16) unsigned char smem[];
  const int row = blockIdx.x / a.chunks, chunk = blockIdx.x - row * a.chunks, sentence = row / a.beams;
  // A beam that has ended, or has no score, offers no continuation.
  const bool ended = a.finished != nullptr && a.finished[row] != 0;
  const float score = a.scores[row];
  take_chunk<T>(logits, a, row, chunk, smem, [&] { return !ended && isfinite(score); });
  if (last_warp_to_arrive(a.arrived + sentence, static_cast<unsigned>(a.beams) * a.chunks))
    select_beams<T>(logits, a, sentence, *reinterpret_cast<Selection*>(smem));
}

// Chunks of a beam, by an estimate in cycles: a warp alone takes 900 for a batch, n on an SM together 82
// n; a chunk's start and end take 5500, and from 8 beams on more, as its lists grow; the selection 3000, and for each
// of W rounds 450 and a look at all lists.  Chunks that do not fit the device at once cost another round of the same.
// (512 rows of 100003: 46 us with 4 or 5 chunks, 55 with 6, 82 with 1; 128 rows of 50021, 16 beams: 32 with 5 to
// 10, 39 with 16.  Over 54 sizes of 4 to 64 beams and 1 to 192 sentences the choice takes 1.026 times the best one's time;
// with 19 blocks on an SM and 5500 for every number of beams it took 1.044, 1.37 at worst.)
int choose_chunks(long long rows, int beams, long long vectors, int sms, int per_sm) {
  const double batches = static_cast<double>((vectors + kBatchVectors - 1) / kBatchVectors);
  const double ends = 5500.0 * std::max(1.0, beams / 8.0);
  int best = 1;
  double best_cost = 1e300;
  for (int c = 1; c <= batches && c * beams <= kMostLists; ++c) {
    const double tasks = static_cast<double>(rows) * c, beside = std::min<double>(per_sm, std::ceil(tasks / sms));
    const double rounds = std::ceil(tasks / (static_cast<double>(per_sm) * sms));
    const double cost = rounds * (std::ceil(batches / c) * std::max(900.0, 82.0 * beside) + ends) + 3000.0 + beams * (450.0 + 1.25 * beams * c);
    if (cost < best_cost) { best = c; best_cost = cost; }
  }
  return best;
}

// Resident blocks per SM: 19 with lists of 128 keys (up to 8 beams), 17 with 256, 15 with 512.
template <class T>
int blocks_on_sm(int room, size_t smem) {
  static std::atomic<int> known[3];
  int n = known[room].load(std::memory_order_relaxed);
  if (n == 0) {
    OB_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, beam_step_kernel<T>, 32, smem));
    if (n < 1) throw std::runtime_error("beam_search_step: the kernel does not fit this device");
    known[room].store(n, std::memory_order_relaxed);
  }
  return n;
}

template <class T>
void k_beam_step(OpCall& c) {
  const Shape& s = c.in[0].shape();
  constexpr int N = Values<T>::N;
  const long long rows = s[0] * s[1], vectors = (s[2] + N - 1) / N;
  const int room = s[1] <= 8 ? 0 : s[1] <= 16 ? 1 : 2, list = 128 << room;
  const size_t smem = warp_bytes(list);
  const long long chunks = choose_chunks(rows, static_cast<int>(s[1]), vectors, sm_count_for(c.in[0]), blocks_on_sm<T>(room, smem));
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
  a.list = list;
  static_assert(sizeof(Selection) <= warp_bytes(128), "the selection lies in the chunk's memory");
  beam_step_kernel<T><<<static_cast<unsigned>(rows * chunks), 32, smem, st>>>(logits, a);
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
