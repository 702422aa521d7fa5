// CPU reference backend, part 3: the operators of text generation.  Plain loops in the precision
// of the operands (angles in double); the oracle of the CUDA kernels.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <limits>
#include <numeric>
#include <stdexcept>

#include "ob/cpu_parallel.h"
#include "ob/kernels.h"

namespace ob {
namespace {

inline int64_t whole_at(const Tensor& t, int64_t i) {
  return t.dtype() == DType::I64 ? t.data_as<int64_t>()[i] : static_cast<int64_t>(t.data_as<int32_t>()[i]);
}

template <class T>
void rotary_cpu(OpCall& c) {
  const Tensor &x = c.in[0], &pos = c.in[1], &turns = c.in[2];
  Tensor& y = c.out[0];
  const int64_t B = x.shape()[0], Tn = x.shape()[1], H = x.shape()[2], D = x.shape()[3];
  const int64_t half = turns.numel(), R = 2 * half, Hr = c.i[0];
  const bool inter = c.i[1] != 0, in_place = c.i[2] != 0;
  const double sign = c.f[0], mag = c.f[1], two_pi = 6.283185307179586476925286766559;
  const double* f = turns.data_as<double>();
  const T* px = x.data_as<T>();
  T* py = y.data_as<T>();
  cpu::parallel_for(B * Tn, 1 + 65536 / (H * D + 1), [&](int64_t lo, int64_t hi) {
    std::vector<T> cs(half), sn(half);
    for (int64_t r = lo; r < hi; ++r) {
      const int64_t b = r / Tn, t = r - b * Tn;
      const double p = static_cast<double>(!pos.defined() ? t : whole_at(pos, pos.ndim() == 2 ? r : t));
      for (int64_t i = 0; i < half; ++i) {
        const double u = p * f[i];
        const double a = (u - std::nearbyint(u)) * two_pi;
        cs[i] = static_cast<T>(std::cos(a) * mag);
        sn[i] = static_cast<T>(std::sin(a) * sign * mag);
      }
      for (int64_t h = 0; h < H; ++h) {
        const T* src = px + b * x.strides()[0] + t * x.strides()[1] + h * x.strides()[2];
        T* dst = py + b * y.strides()[0] + t * y.strides()[1] + h * y.strides()[2];
        int64_t from = 0;
        if (h < Hr) {
          for (int64_t i = 0; i < half; ++i) {
            const int64_t ia = inter ? 2 * i : i, ib = inter ? 2 * i + 1 : i + half;
            const T va = src[ia], vb = src[ib];
            dst[ia] = va * cs[i] - vb * sn[i];
            dst[ib] = vb * cs[i] + va * sn[i];
          }
          from = R;
        }
        if (!in_place) std::memcpy(dst + from, src + from, sizeof(T) * (D - from));
      }
    }
  });
}

// Page of place `at` of sequence b; host tables are checked before anything is written or read.
int64_t page_of(const Tensor& table, int64_t b, int64_t at, int64_t page_size, int64_t pages, const char* op) {
  const int64_t slot = at / page_size;
  if (at < 0 || slot >= table.shape()[1])
    throw std::out_of_range(std::string(op) + ": place " + std::to_string(at) + " of sequence " + std::to_string(b) + " lies behind its page table");
  const int64_t page = table.data_as<int32_t>()[b * table.shape()[1] + slot];
  if (page < 0 || page >= pages)
    throw std::out_of_range(std::string(op) + ": page " + std::to_string(page) + " is out of range for " + std::to_string(pages) + " pages");
  return page;
}

void paged_append_cpu(OpCall& c) {
  const Tensor &table = c.in[4], &starts = c.in[5], &counts = c.in[6];
  const Shape& s = c.in[0].shape();
  const Shape& r = c.in[2].shape();
  const int64_t size = static_cast<int64_t>(dtype_size(c.in[0].dtype()));
  for (int pass = 0; pass < 2; ++pass)  // the first pass only checks
    for (int64_t b = 0; b < r[0]; ++b) {
      const int64_t first = starts.data_as<int32_t>()[b];
      const int64_t n = counts.defined() ? std::min<int64_t>(counts.data_as<int32_t>()[b], r[1]) : r[1];
      for (int64_t t = 0; t < n; ++t) {
        const int64_t page = page_of(table, b, first + t, s[2], s[0], "paged_append_");
        if (pass == 0) continue;
        for (int kv = 0; kv < 2; ++kv) {
          const Tensor &pages = c.in[kv], &rows = c.in[2 + kv];
          for (int64_t h = 0; h < s[1]; ++h) {
            char* dst = pages.data_as<char>() + (page * pages.strides()[0] + (h * s[2] + (first + t) % s[2]) * s[3]) * size;
            const char* src = rows.data_as<char>() + (b * rows.strides()[0] + t * rows.strides()[1] + h * rows.strides()[2]) * size;
            std::memcpy(dst, src, s[3] * size);
          }
        }
      }
    }
}

void copy_pages_cpu(OpCall& c) {
  char* base = c.in[0].data_as<char>();
  const size_t n = c.list.size() / 2;
  for (int64_t o = 0; o < c.i[0]; ++o)
    for (size_t i = 0; i < n; ++i)
      std::memcpy(base + (o * c.i[1] + c.list[n + i]) * c.i[2], base + (o * c.i[1] + c.list[i]) * c.i[2], c.i[2]);
}

template <class T>
void paged_attention_cpu(OpCall& c) {
  const Tensor &q = c.in[0], &kp = c.in[1], &vp = c.in[2], &table = c.in[3], &lengths = c.in[4];
  const Shape& s = kp.shape();
  const int64_t B = q.shape()[0], Hq = q.shape()[1], D = s[3], group = Hq / s[1];
  const T scale = static_cast<T>(c.f[0]);
  for (int64_t b = 0; b < B; ++b) {
    const int64_t n = lengths.data_as<int32_t>()[b];
    if (n < 0) throw std::out_of_range("paged_attention: negative length");
    for (int64_t j = 0; j < n; j += s[2]) page_of(table, b, j, s[2], s[0], "paged_attention");
  }
  cpu::parallel_for(B * Hq, 1, [&](int64_t lo, int64_t hi) {
    std::vector<T> w;
    for (int64_t r = lo; r < hi; ++r) {
      const int64_t b = r / Hq, h = r - b * Hq, n = lengths.data_as<int32_t>()[b];
      const T* pq = q.data_as<T>() + b * q.strides()[0] + h * q.strides()[1];
      T* po = c.out[0].data_as<T>() + r * D;
      std::fill(po, po + D, T(0));
      if (n == 0) continue;
      w.resize(n);
      auto row = [&](const Tensor& pages, int64_t j) {
        const int64_t page = table.data_as<int32_t>()[b * table.shape()[1] + j / s[2]];
        return pages.data_as<T>() + page * pages.strides()[0] + ((h / group) * s[2] + j % s[2]) * D;
      };
      T top = -std::numeric_limits<T>::infinity(), sum = T(0);
      for (int64_t j = 0; j < n; ++j) {
        const T* pk = row(kp, j);
        T dot = T(0);
        for (int64_t d = 0; d < D; ++d) dot += pq[d] * pk[d];
        w[j] = dot * scale;
        if (w[j] > top) top = w[j];
      }
      for (int64_t j = 0; j < n; ++j) sum += w[j] = std::exp(w[j] - top);
      for (int64_t j = 0; j < n; ++j) {
        const T* pv = row(vp, j);
        const T p = w[j] / sum;
        for (int64_t d = 0; d < D; ++d) po[d] += p * pv[d];
      }
    }
  });
}

// Beams that offer the same scores tie, whatever order their exponentials were summed in: the
// logarithm of the sum is rounded to 2^-30, far above the noise of the summation (about 2^-45) and
// far below what scores are known to (2^-24 of their size).
double round_log_sum(double log_sum) { return std::nearbyint(log_sum * 1073741824.0) * (1.0 / 1073741824.0); }

template <class T>
void beam_step_cpu(OpCall& c) {
  const Tensor &logits = c.in[0], &scores = c.in[1], &finished = c.in[2];
  const int64_t B = logits.shape()[0], W = logits.shape()[1], V = logits.shape()[2], end = c.i[0];
  const double none = -std::numeric_limits<double>::infinity();
  cpu::parallel_for(B, 1, [&](int64_t lo, int64_t hi) {
    std::vector<double> cand(W * V);
    std::vector<int64_t> at(W * V);
    for (int64_t b = lo; b < hi; ++b) {
      for (int64_t w = 0; w < W; ++w) {
        const T* x = logits.data_as<T>() + (b * W + w) * V;
        double* y = cand.data() + w * V;
        const double s = scores.data_as<float>()[b * W + w];
        const bool done = finished.defined() && finished.data_as<uint8_t>()[b * W + w] != 0;
        double top = none, sum = 0.0, rest = 0.0;
        for (int64_t v = 0; v < V; ++v) top = x[v] > top ? x[v] : top;
        for (int64_t v = 0; v < V; ++v) {  // compensated: sum >= e once the maximum has been added
          const double e = std::exp(static_cast<double>(x[v]) - top), next = sum + e;
          rest += std::fabs(sum) >= e ? (sum - next) + e : (e - next) + sum;
          sum = next;
        }
        const double lse = top + round_log_sum(std::log(sum + rest));
        const bool dead = !std::isfinite(s) || (!done && !std::isfinite(lse));
        for (int64_t v = 0; v < V; ++v) y[v] = dead || done ? none : s + (static_cast<double>(x[v]) - lse);
        if (done && !dead) y[end] = s;
      }
      std::iota(at.begin(), at.end(), int64_t(0));
      std::partial_sort(at.begin(), at.begin() + W, at.end(), [&](int64_t i, int64_t j) { return cand[i] != cand[j] ? cand[i] > cand[j] : i < j; });
      for (int64_t k = 0; k < W; ++k) {
        const int64_t parent = at[k] / V, token = at[k] % V, o = b * W + k;
        c.out[0].data_as<float>()[o] = static_cast<float>(cand[at[k]]);
        c.out[1].data_as<int64_t>()[o] = parent;
        c.out[2].data_as<int64_t>()[o] = token;
        c.out[3].data_as<uint8_t>()[o] = (end >= 0 && token == end) || (finished.defined() && finished.data_as<uint8_t>()[b * W + parent] != 0);
      }
    }
  });
}

}  // namespace

void register_cpu_generation(KernelRegistry& r) {
  const uint8_t any = kContiguous | kStrided | kEmpty;
#define REG2(OP, FN, NAME, LAY)                                                                     \
  r.add_kernel(OperatorId::OP, Constraints{Backend::CPU, kMaskF32, LAY, Capability::None}, FN<float>, NAME "_f32"); \
  r.add_kernel(OperatorId::OP, Constraints{Backend::CPU, kMaskF64, LAY, Capability::None}, FN<double>, NAME "_f64");
  const uint8_t packed = kContiguous | kEmpty;
  REG2(RotaryEmbedding, rotary_cpu, "cpu_rotary_embedding", any)
  REG2(PagedAttention, paged_attention_cpu, "cpu_paged_attention", packed) REG2(BeamSearchStep, beam_step_cpu, "cpu_beam_search_step", packed)
  r.add_kernel(OperatorId::PagedAppend, Constraints{Backend::CPU, kMaskCpuCompute | kMaskHalf, packed, Capability::None}, paged_append_cpu, "cpu_paged_append");
  r.add_kernel(OperatorId::CopyPages, Constraints{Backend::CPU, kMaskAll, packed, Capability::None}, copy_pages_cpu, "cpu_copy_pages");
#undef REG2
}

}  // namespace ob
