// Semantic operators, part 3: what answering with a language model needs next to training one.
// Rotary positions (differentiable), the paged key-value cache and its attention, beam selection.
#include <cmath>

#include "ob/kernels.h"
#include "ob/ops.h"

namespace ob {
namespace ops {
namespace {

void check_not_in_graph(const Tensor& t, const char* op) {
  if (grad_enabled() && t.requires_grad() && !t.is_leaf())
    throw std::runtime_error(std::string(op) + ": in-place modification of a tensor with autograd history is only allowed under no_grad()");
}

// ---------------------------------------------------------------------- rotary
// Validates the call and returns the positions on x's device (undefined: 0..T-1).
Tensor check_rotary(const Tensor& x, const Tensor& positions, const RotarySpec& spec, const char* op) {
  if (x.ndim() != 4) throw std::invalid_argument(std::string(op) + ": input must be 4-D [B, T, H, D] (got " + shape_str(x.shape()) + ")");
  default_dispatcher().check_dtype(OperatorId::RotaryEmbedding, x.device(), x.dtype());
  const Tensor& turns = spec.turns;
  if (!turns.defined() || turns.ndim() != 1 || turns.dtype() != DType::F64 || !turns.device().is_cpu() || !turns.is_contiguous())
    throw std::invalid_argument(std::string(op) + ": frequencies must be a contiguous 1-D float64 tensor on the host");
  const int64_t R = 2 * turns.numel();
  if (R < 2 || R > x.shape()[3])
    throw std::invalid_argument(std::string(op) + ": rotary_dim " + std::to_string(R) + " does not fit the head size " + std::to_string(x.shape()[3]));
  if (R > 512) throw std::invalid_argument(std::string(op) + ": rotary_dim must be at most 512");
  if (spec.rotary_heads < 1 || spec.rotary_heads > x.shape()[2])
    throw std::invalid_argument(std::string(op) + ": rotary_heads must be in [1, " + std::to_string(x.shape()[2]) + "]");
  for (int64_t i = 0; i < turns.numel(); ++i)
    if (!std::isfinite(turns.data_as<double>()[i])) throw std::invalid_argument(std::string(op) + ": frequencies must be finite");
  if (!std::isfinite(spec.magnitude)) throw std::invalid_argument(std::string(op) + ": the magnitude must be finite");
  if (!positions.defined()) return positions;
  if (positions.dtype() != DType::I32 && positions.dtype() != DType::I64)
    throw std::invalid_argument(std::string(op) + ": positions must be int32 or int64");
  const Shape row{x.shape()[1]}, full{x.shape()[0], x.shape()[1]};
  if (positions.shape() != row && positions.shape() != full)
    throw std::invalid_argument(std::string(op) + ": positions must have shape " + shape_str(row) + " or " + shape_str(full) + " (got " +
                                shape_str(positions.shape()) + ")");
  Tensor p = contiguous(positions.detach());
  return p.device() == x.device() ? p : to(p, x.device());
}

void rotary_raw(const Tensor& x, const Tensor& positions, const RotarySpec& spec, bool transposed, bool in_place, Tensor& out) {
  if (x.numel() == 0) return;
  OpCall c;
  c.in[0] = x;
  c.in[1] = positions;
  c.in[2] = spec.turns;
  c.out[0] = out;
  c.f[0] = transposed ? -1.0 : 1.0;
  c.f[1] = spec.magnitude;
  c.i[0] = spec.rotary_heads;
  c.i[1] = spec.interleaved;
  c.i[2] = in_place;
  run_kernel(OperatorId::RotaryEmbedding, x.device(), x.dtype(), c, x.is_contiguous() ? kContiguous : kStrided);
}

// The kernels read rows of values in place; only a strided last dimension needs a copy.
Tensor rows_of(const Tensor& x) {
  const Tensor d = x.detach();
  return x.ndim() == 0 || d.strides().back() == 1 || d.shape().back() <= 1 ? d : contiguous(d);
}

struct RotaryNode : Node {
  Tensor positions;
  RotarySpec spec;
  const char* name() const override { return "RotaryEmbeddingNode"; }
  std::vector<Tensor> backward(const Tensor& g) override {
    Tensor dx = Tensor::empty(g.shape(), g.dtype(), g.device());
    rotary_raw(rows_of(g), positions, spec, !spec.transposed, false, dx);
    return {dx};
  }
  void release_saved() override { positions = Tensor(); spec.turns = Tensor(); }
};

}  // namespace

Tensor rotary_embedding(const Tensor& x, const Tensor& positions, const RotarySpec& spec) {
  Tensor p = check_rotary(x, positions, spec, "rotary_embedding");
  Tensor out = Tensor::empty(x.shape(), x.dtype(), x.device());
  rotary_raw(rows_of(x), p, spec, spec.transposed, false, out);
  if (needs_graph({x})) {
    auto n = std::make_shared<RotaryNode>();
    n->positions = p;
    n->spec = spec;
    if (p.defined()) n->watch_version(p, "positions");
    n->set_inputs({x});
    attach(out, n);
  }
  return out;
}

Tensor& rotary_embedding_(Tensor& x, const Tensor& positions, const RotarySpec& spec) {
  check_not_in_graph(x, "rotary_embedding_");
  Tensor p = check_rotary(x, positions, spec, "rotary_embedding_");
  if (x.numel() && x.strides()[3] != 1 && x.shape()[3] > 1)
    throw std::invalid_argument("rotary_embedding_: the last dimension must be contiguous");
  for (int d = 0; d < 4; ++d)
    if (x.shape()[d] > 1 && x.strides()[d] == 0) throw std::invalid_argument("rotary_embedding_: the tensor must not be broadcast");
  Tensor out = x.detach();
  rotary_raw(x.detach(), p, spec, spec.transposed, true, out);
  x.bump_version();
  return x;
}


// ---------------------------------------------------------------- paged cache
namespace {

void check_no_gradient(std::initializer_list<Tensor> inputs, const char* op) {
  if (needs_graph(inputs)) throw std::runtime_error(std::string(op) + ": has no gradient; call it under no_grad()");
}

void check_pages(const Tensor& k_pages, const Tensor& v_pages, const char* op) {
  check_same_device(k_pages, v_pages, op);
  check_same_dtype(k_pages, v_pages, op);
  for (const Tensor* t : {&k_pages, &v_pages}) {
    if (t->ndim() != 4) throw std::invalid_argument(std::string(op) + ": pages must be 4-D [N, H, P, D] (got " + shape_str(t->shape()) + ")");
    const Shape &s = t->shape(), &st = t->strides();
    const int64_t page = s[1] * s[2] * s[3];
    if ((s[3] > 1 && st[3] != 1) || (s[2] > 1 && st[2] != s[3]) || (s[1] > 1 && st[1] != s[2] * s[3]) || (s[0] > 1 && st[0] < page))
      throw std::invalid_argument(std::string(op) + ": each page must be contiguous and pages must not overlap");
    if (s[1] < 1 || s[2] < 1 || s[3] < 1) throw std::invalid_argument(std::string(op) + ": pages must have heads, tokens and values");
  }
  if (k_pages.shape() != v_pages.shape()) throw std::invalid_argument(std::string(op) + ": key and value pages must have the same shape");
}

// An int32 tensor on the cache's device, contiguous.
Tensor whole_numbers(const Tensor& t, const Shape& shape, Device dev, const char* op, const char* what) {
  if (t.dtype() != DType::I32) throw std::invalid_argument(std::string(op) + ": " + what + " must be int32");
  if (t.shape() != shape)
    throw std::invalid_argument(std::string(op) + ": " + what + " must have shape " + shape_str(shape) + " (got " + shape_str(t.shape()) + ")");
  Tensor c = contiguous(t.detach());
  return c.device() == dev ? c : to(c, dev);
}

Tensor page_table(const Tensor& t, int64_t batch, Device dev, const char* op) {
  if (t.ndim() != 2) throw std::invalid_argument(std::string(op) + ": the page table must be 2-D [B, M] (got " + shape_str(t.shape()) + ")");
  return whole_numbers(t, {batch, t.shape()[1]}, dev, op, "the page table");
}

// Two views of one buffer share memory if their spans cross, unless they are slices that
// interleave page by page (keys and values in one pool): then every page of one lies between two
// of the other.
bool share_memory(const Tensor& a, const Tensor& b) {
  if (!a.same_buffer(b) || a.numel() == 0 || b.numel() == 0) return false;
  const int64_t a0 = a.offset(), a1 = a.impl()->layout().span_end(), b0 = b.offset(), b1 = b.impl()->layout().span_end();
  if (a1 <= b0 || b1 <= a0) return false;
  if (a.shape() == b.shape() && a.strides() == b.strides() && a.ndim() == 4) {
    const int64_t page = a.shape()[1] * a.shape()[2] * a.shape()[3], step = a.strides()[0];
    const int64_t shift = ((b0 - a0) % step + step) % step;
    return shift < page || shift + page > step;
  }
  return true;
}

}  // namespace

void paged_append_(Tensor& k_pages, Tensor& v_pages, const Tensor& k, const Tensor& v, const Tensor& table, const Tensor& starts,
                   const Tensor& counts) {
  const char* op = "paged_append_";
  check_pages(k_pages, v_pages, op);
  check_no_gradient({k_pages, v_pages, k, v}, op);
  default_dispatcher().check_dtype(OperatorId::PagedAppend, k_pages.device(), k_pages.dtype());
  for (const Tensor* t : {&k, &v}) {
    check_same_device(k_pages, *t, op);
    check_same_dtype(k_pages, *t, op);
    if (t->ndim() != 4 || t->shape()[2] != k_pages.shape()[1] || t->shape()[3] != k_pages.shape()[3])
      throw std::invalid_argument(std::string(op) + ": keys and values must be [B, T, H, D] with the heads and head size of the pages (got " +
                                  shape_str(t->shape()) + ")");
    if (share_memory(*t, k_pages) || share_memory(*t, v_pages)) throw std::invalid_argument(std::string(op) + ": keys and values must not lie in the cache");
  }
  if (k.shape() != v.shape()) throw std::invalid_argument(std::string(op) + ": keys and values must have the same shape");
  if (share_memory(k_pages, v_pages)) throw std::invalid_argument(std::string(op) + ": key and value pages must not share memory");
  const int64_t B = k.shape()[0];
  Tensor tab = page_table(table, B, k_pages.device(), op);
  Tensor st = whole_numbers(starts, {B}, k_pages.device(), op, "starts");
  Tensor ct = counts.defined() ? whole_numbers(counts, {B}, k_pages.device(), op, "counts") : Tensor();
  if (k.numel() == 0) return;
  OpCall c;
  c.in[0] = k_pages.detach();
  c.in[1] = v_pages.detach();
  c.in[2] = rows_of(k);
  c.in[3] = rows_of(v);
  c.in[4] = tab;
  c.in[5] = st;
  c.in[6] = ct;
  run_kernel(OperatorId::PagedAppend, k_pages.device(), k_pages.dtype(), c);
  k_pages.bump_version();
  if (!v_pages.same_buffer(k_pages)) v_pages.bump_version();
}

void copy_pages_(Tensor& pages, const std::vector<int64_t>& sources, const std::vector<int64_t>& destinations, int dim) {
  const char* op = "copy_pages_";
  check_not_in_graph(pages, op);
  if (dim < 0) dim += pages.ndim();
  if (dim < 0 || dim >= pages.ndim()) throw std::invalid_argument(std::string(op) + ": dimension out of range");
  if (!pages.is_contiguous()) throw std::invalid_argument(std::string(op) + ": the pages must be contiguous");
  if (sources.size() != destinations.size()) throw std::invalid_argument(std::string(op) + ": as many destinations as sources are needed");
  const int64_t n = pages.shape()[dim];
  std::vector<char> use(static_cast<size_t>(n), 0);
  for (int64_t s : sources) {
    if (s < 0 || s >= n) throw std::out_of_range(std::string(op) + ": source page " + std::to_string(s) + " is out of range for " + std::to_string(n) + " pages");
    use[s] = 1;
  }
  for (int64_t d : destinations) {
    if (d < 0 || d >= n) throw std::out_of_range(std::string(op) + ": destination page " + std::to_string(d) + " is out of range for " + std::to_string(n) + " pages");
    if (use[d]) throw std::invalid_argument(std::string(op) + ": page " + std::to_string(d) + (use[d] == 1 ? " is a source and a destination" : " is a destination twice"));
    use[d] = 2;
  }
  if (sources.empty() || pages.numel() == 0) return;
  OpCall c;
  c.in[0] = pages.detach();
  c.i[0] = 1;
  for (int d = 0; d < dim; ++d) c.i[0] *= pages.shape()[d];
  c.i[1] = n;
  c.i[2] = static_cast<int64_t>(pages.nbytes()) / (c.i[0] * n);
  c.list = sources;
  c.list.insert(c.list.end(), destinations.begin(), destinations.end());
  run_kernel(OperatorId::CopyPages, pages.device(), pages.dtype(), c);
  pages.bump_version();
}

Tensor paged_attention(const Tensor& q, const Tensor& k_pages, const Tensor& v_pages, const Tensor& table, const Tensor& lengths,
                       double scale) {
  const char* op = "paged_attention";
  check_pages(k_pages, v_pages, op);
  check_same_device(q, k_pages, op);
  check_same_dtype(q, k_pages, op);
  check_no_gradient({q, k_pages, v_pages}, op);
  default_dispatcher().check_dtype(OperatorId::PagedAttention, q.device(), q.dtype());
  if (q.ndim() != 3 || q.shape()[2] != k_pages.shape()[3])
    throw std::invalid_argument(std::string(op) + ": queries must be [B, H, D] with the head size of the pages (got " + shape_str(q.shape()) + ")");
  if (q.shape()[1] < 1 || q.shape()[1] % k_pages.shape()[1] != 0)
    throw std::invalid_argument(std::string(op) + ": the query heads must be a multiple of the cached heads");
  if (q.device().is_cuda() && q.shape()[2] > 256) throw std::invalid_argument(std::string(op) + ": head size must be at most 256");
  if (!std::isfinite(scale)) throw std::invalid_argument(std::string(op) + ": the scale must be finite");
  const int64_t B = q.shape()[0];
  Tensor tab = page_table(table, B, q.device(), op);
  Tensor len = whole_numbers(lengths, {B}, q.device(), op, "lengths");
  Tensor out = Tensor::empty(q.shape(), q.dtype(), q.device());
  if (out.numel() == 0) return out;
  OpCall c;
  // The kernels read queries in pairs: rows at odd places are copied (a few values next to the cache).
  c.in[0] = rows_of(q);
  if (q.shape()[2] % 2 == 0 && (c.in[0].offset() | c.in[0].strides()[0] | c.in[0].strides()[1]) % 2 != 0) c.in[0] = clone(c.in[0]);
  c.in[1] = k_pages.detach();
  c.in[2] = v_pages.detach();
  c.in[3] = tab;
  c.in[4] = len;
  c.out[0] = out;
  c.f[0] = scale;
  run_kernel(OperatorId::PagedAttention, q.device(), q.dtype(), c);
  return out;
}

// -------------------------------------------------------------- beam selection
BeamStep beam_search_step(const Tensor& logits, const Tensor& scores, const Tensor& finished, int64_t end_token) {
  const char* op = "beam_search_step";
  check_no_gradient({logits, scores}, op);
  if (logits.ndim() != 3 || logits.numel() == 0)
    throw std::invalid_argument(std::string(op) + ": logits must be a non-empty [B, W, V] tensor (got " + shape_str(logits.shape()) + ")");
  default_dispatcher().check_dtype(OperatorId::BeamSearchStep, logits.device(), logits.dtype());
  const Shape rows{logits.shape()[0], logits.shape()[1]};
  const int64_t V = logits.shape()[2];
  if (rows[1] > 64) throw std::invalid_argument(std::string(op) + ": at most 64 beams are supported");
  if (V > (1LL << 30)) throw std::invalid_argument(std::string(op) + ": the vocabulary is too large");
  check_same_device(logits, scores, op);
  if (scores.dtype() != DType::F32 || scores.shape() != rows)
    throw std::invalid_argument(std::string(op) + ": scores must be float32 with shape " + shape_str(rows));
  if (end_token < -1 || end_token >= V) throw std::out_of_range(std::string(op) + ": the end token is out of range");
  if (finished.defined()) {
    check_same_device(logits, finished, op);
    if (finished.dtype() != DType::Bool || finished.shape() != rows)
      throw std::invalid_argument(std::string(op) + ": finished must be bool with shape " + shape_str(rows));
    if (end_token < 0) throw std::invalid_argument(std::string(op) + ": finished beams need an end token");
  }
  BeamStep s;
  s.scores = Tensor::empty(rows, DType::F32, logits.device());
  s.parents = Tensor::empty(rows, DType::I64, logits.device());
  s.tokens = Tensor::empty(rows, DType::I64, logits.device());
  s.finished = Tensor::empty(rows, DType::Bool, logits.device());
  OpCall c;
  c.in[0] = contiguous(logits.detach());
  c.in[1] = contiguous(scores.detach());
  if (finished.defined()) c.in[2] = contiguous(finished.detach());
  c.out[0] = s.scores;
  c.out[1] = s.parents;
  c.out[2] = s.tokens;
  c.out[3] = s.finished;
  c.i[0] = end_token;
  run_kernel(OperatorId::BeamSearchStep, logits.device(), logits.dtype(), c);
  return s;
}

}  // namespace ops
}  // namespace ob
