// The serving operators of the native module: argument checks, output and scratch allocation and the
// calls into risa_b200_cache.h.  Everything a call needs happens in one foreign call (a step's kernels
// take microseconds, as long as a handful of Python statements).  Wrong values raise ValueError, wrong
// types TypeError, in the order shapes, types, devices.
#include <torch/extension.h>

#include <ATen/MemoryOverlap.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/VirtualGuardImpl.h>

#include <optional>
#include <string>

#include "../../include/risa_b200.h"
#include "../../include/risa_b200_cache.h"

namespace py = pybind11;

namespace {

using MaybeTensor = std::optional<at::Tensor>;
constexpr int kInt8 = 4, kInt4 = 5;
constexpr int64_t kMostSlots = RISA_B200_CACHE_MOST_SLOTS;

void check(int status) {
  if (status == RISA_B200_INVALID) throw py::value_error(risa_b200_last_error());
  if (status != RISA_B200_OK) throw std::runtime_error(risa_b200_last_error());
}
void require(bool ok, const std::string& message) {
  if (!ok) throw py::value_error(message);
}
void require_type(bool ok, const std::string& message) {
  if (!ok) throw py::type_error(message);
}
void* stream_of(uintptr_t stream_ptr) { return reinterpret_cast<void*>(stream_ptr); }

int code_of(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return 0;
    case at::kHalf: return 1;
    case at::kBFloat16: return 2;
    case at::kChar: return kInt8;
    case at::kByte: return kInt4;
    default: return -1;
  }
}

// No two elements of a tensor that is written may share memory.
void require_distinct(const at::Tensor& t, const char* what) {
  for (int64_t i = 0; i < t.dim(); ++i) require(t.size(i) <= 1 || t.stride(i) != 0, std::string(what) + " must not be an expanded view");
}

// An output may be the input itself, row for row, or lie apart from it.  (Views with gaps that interleave are not told from
// views that overlap.)
void require_apart(const at::Tensor& out, const at::Tensor& in, const char* what) {
  const bool same = out.data_ptr() == in.data_ptr();
  const at::MemOverlapStatus overlap = at::get_overlap_status(out, in);
  require((!same && overlap != at::MemOverlapStatus::Full && overlap != at::MemOverlapStatus::Partial) || (same && out.strides() == in.strides()),
          std::string("out may be ") + what + " itself, not another view of its memory");
}

// Rows of eight channels that start on 16-byte boundaries: the tensor itself, or a packed copy.
at::Tensor rows_of(const at::Tensor& t) {
  bool good = t.stride(-1) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  for (int64_t i = 0; i + 1 < t.dim(); ++i) good = good && (t.size(i) <= 1 || t.stride(i) % 8 == 0);
  return good ? t : t.contiguous();
}
// Strides of (token, head); an axis of one element has whatever stride suits.
struct Strides2 {
  int64_t of[2];
  explicit Strides2(const at::Tensor& t)
      : of{t.size(0) <= 1 ? 0 : t.stride(0), t.size(1) <= 1 ? 0 : t.stride(1)} {}
};

struct Cache {
  at::Tensor keys, values;
  MaybeTensor key_scales, value_scales;
  risa_b200_cache c{};

  Cache(const at::Tensor& k, const at::Tensor& v, const MaybeTensor& ks, const MaybeTensor& vs)
      : keys(k), values(v), key_scales(ks), value_scales(vs) {
    require(k.dim() == 4 && v.sizes() == k.sizes(),
            "cache keys and values must both have shape [pages, kv_heads, page_size, head_dim] (half of it where a byte holds two 4-bit codes)");
    const int code = code_of(k);
    const int64_t head_dim = k.size(3) * (code == kInt4 ? 2 : 1);
    require(k.size(0) > 0 && k.size(1) > 0, "the cache needs pages and heads");
    require(k.size(0) < (int64_t(1) << 31) && k.size(1) <= 65535, "the cache has too many pages or heads");
    require(k.size(2) == 16 || k.size(2) == 32 || k.size(2) == 64 || k.size(2) == 128, "page_size must be 16, 32, 64 or 128");
    require(head_dim == 64 || head_dim == 128 || head_dim == 256, "head_dim of a cache must be 64, 128 or 256");
    require_type(code == 1 || code == 2 || code == kInt8 || code == kInt4, "cache keys and values must be float16, bfloat16, int8 or uint8 (4-bit codes)");
    require_type(v.scalar_type() == k.scalar_type(), "cache keys and values must have the same dtype");
    require(k.is_contiguous() && v.is_contiguous(), "cache keys and values must be contiguous");
    const bool codes = code == kInt8 || code == kInt4;
    require(codes == ks.has_value() && codes == vs.has_value(), "a cache of codes needs key_scales and value_scales, any other has none");
    if (code == kInt4) {
      for (const at::Tensor* s : {&*ks, &*vs}) {
        require_type(s->scalar_type() == at::kByte, "scales of 4-bit codes must be uint8");
        require(s->dim() == 3 && s->size(0) == k.size(0) && s->size(1) == k.size(1) && s->size(2) == k.size(2) * (1 + head_dim / 16) && s->is_contiguous(),
                "scales of 4-bit codes must be contiguous [pages, kv_heads, page_size * (1 + head_dim / 16)]");
        require(s->device() == k.device(), "scales must be on the device of the cache");
      }
    }
    if (code == kInt8) {
      for (const at::Tensor* s : {&*ks, &*vs}) {
        require_type(s->scalar_type() == at::kFloat, "scales must be float32");
        require(s->dim() == 3 && s->size(0) == k.size(0) && s->size(1) == k.size(1) && s->size(2) == k.size(2) && s->is_contiguous(),
                "scales must be contiguous [pages, kv_heads, page_size]");
        require(s->device() == k.device(), "scales must be on the device of the cache");
      }
    }
    require(v.device() == k.device(), "cache keys and values must be on the same device");
    c.keys = k.data_ptr();
    c.values = v.data_ptr();
    c.key_scales = codes ? static_cast<float*>(ks->data_ptr()) : nullptr;
    c.value_scales = codes ? static_cast<float*>(vs->data_ptr()) : nullptr;
    c.pages = int(k.size(0));
    c.kv_heads = int(k.size(1));
    c.page_size = int(k.size(2));
    c.head_dim = int(head_dim);
    c.dtype_code = code;
  }
};

void require_indices(const at::Tensor& t, const char* what) {
  require_type(t.scalar_type() == at::kInt, std::string(what) + " must be int32");
  require(t.is_contiguous(), std::string(what) + " must be contiguous");
}

struct Step {
  risa_b200_step s{};

  Step(const Cache& cache, const at::Tensor& table, const at::Tensor& lengths, const MaybeTensor& offsets, int64_t tokens) {
    require(table.dim() == 2 && table.size(0) > 0 && table.size(1) > 0, "page_table must have shape [batch, pages of a sequence]");
    require(table.size(0) <= 65535, "a step takes at most 65535 sequences");
    require(table.size(1) * cache.c.page_size < kMostSlots, "page_table is too wide: a sequence may hold fewer than 2^31 - 8192 keys");
    require(lengths.dim() == 1 && lengths.size(0) == table.size(0), "lengths must have shape [batch]");
    require(!offsets.has_value() || (offsets->dim() == 1 && offsets->size(0) == table.size(0) + 1), "query_offsets must have shape [batch + 1]");
    require(offsets.has_value() || tokens == table.size(0), "without query_offsets there must be one token for every sequence");
    require(tokens > 0 && tokens < (int64_t(1) << 31), "a step needs tokens");
    require_indices(table, "page_table");
    require_indices(lengths, "lengths");
    if (offsets.has_value()) require_indices(*offsets, "query_offsets");
    for (const at::Tensor* t : {&table, &lengths}) require(t->device() == cache.keys.device(), "page_table and lengths must be on the device of the cache");
    require(!offsets.has_value() || offsets->device() == cache.keys.device(), "query_offsets must be on the device of the cache");
    s.page_table = table.data_ptr<int32_t>();
    s.lengths = lengths.data_ptr<int32_t>();
    s.query_offsets = offsets.has_value() ? offsets->data_ptr<int32_t>() : nullptr;
    s.batch = int(table.size(0));
    s.table_width = int(table.size(1));
    s.tokens = int(tokens);
  }
};

void require_cuda(const at::Tensor& t) {
  require(t.is_cuda(), "the tensors of a serving call must be on a CUDA device");
}

struct Rotary {
  risa_b200_rotary r{};
  Rotary(const at::Tensor& turns, double magnitude, bool interleaved, int64_t head_dim, const at::Device& device) {
    require(turns.dim() == 1 && turns.size(0) > 0 && 2 * turns.size(0) <= head_dim, "rotary_dim must be positive and at most head_dim");
    require_type(turns.scalar_type() == at::kLong && turns.is_contiguous(), "a rotary table holds contiguous int64 turns");
    require(turns.device() == device, "the rotary table must be on the device of the tensors it rotates");
    r.turns = reinterpret_cast<const uint64_t*>(turns.data_ptr<int64_t>());
    r.rotary_dim = int(2 * turns.size(0));
    r.magnitude = float(magnitude);
    r.interleaved = interleaved ? 1 : 0;
  }
};

// The axes that a table's pairs follow, and from one axis' positions to the next one's: `positions` has the axes in front of the
// `plain` dimensions that one axis has, or only those (all axes alike).
struct Axes {
  std::optional<risa_b200_rotary_axes> r;
  at::Tensor positions;  // of the first axis
  Axes(const MaybeTensor& axes, int64_t count, const at::Tensor& turns, const at::Tensor& all, int64_t plain) : positions(all) {
    if (!axes.has_value()) return;
    require_type(axes->scalar_type() == at::kByte && axes->is_contiguous(), "the axes of a rotary table must be contiguous uint8");
    require(axes->dim() == 1 && axes->size(0) == turns.size(0), "a rotary table needs an axis for each pair");
    require(count >= 1 && count <= RISA_B200_MOST_AXES, "a rotary table follows 1 to 8 axes");
    require(axes->device() == turns.device(), "turns and axes of a rotary table must be on the same device");
    r.emplace();
    r->axes = axes->data_ptr<uint8_t>();
    r->count = int(count);
    r->position_stride = 0;
    if (all.defined() && all.dim() == plain + 1) {
      require(all.size(0) == count, "positions must have a row for each of the table's axes");
      r->position_stride = count == 1 ? 0 : all.stride(0);
      positions = all.select(0, 0);
    }
  }
  const risa_b200_rotary_axes* get() const { return r.has_value() ? &*r : nullptr; }
};

void require_positions(const at::Tensor& p) {
  require_type(p.scalar_type() == at::kInt || p.scalar_type() == at::kLong, "positions must be int32 or int64");
}

// A tangent that rides on the tensor would be lost, whether it requires a gradient or not.
void require_no_tangent(const at::Tensor& x) {
  require(!c10::AutogradState::get_tls_state().get_fw_grad_mode() || !x._fw_grad(0).defined(),
          "rotation has no forward-mode derivative: rotate the tangent itself, the map is linear");
}

// x [tokens, heads, head_dim] with positions [tokens], or [batch, heads, tokens, head_dim] with positions
// [tokens] or [batch, tokens]; a table of several axes takes [tokens] for all of them, or theirs in front of the same.
at::Tensor rotate(const at::Tensor& x, const at::Tensor& all_positions, const at::Tensor& turns, const MaybeTensor& axes_of_pairs,
                  int64_t axis_count, double magnitude, bool interleaved, bool transposed, const MaybeTensor& out_given,
                  uintptr_t stream_ptr) {
  require_no_tangent(x);
  require(x.dim() == 3 || x.dim() == 4, "x must have shape [tokens, heads, head_dim] or [batch, heads, tokens, head_dim]");
  const bool packed = x.dim() == 3;
  const int64_t batch = packed ? 1 : x.size(0), heads = x.size(1), tokens = packed ? x.size(0) : x.size(2), d = x.size(-1);
  require(batch > 0 && heads > 0 && tokens > 0 && d > 0, "x must not be empty");
  require(batch <= 65535 && heads <= 65535 && tokens < (int64_t(1) << 31) && d <= 65536, "x is too large");
  // [axes, tokens], not [batch, tokens], where the table has axes
  const Axes axes(axes_of_pairs, axis_count, turns, all_positions, all_positions.dim() - (all_positions.dim() > 1));
  const at::Tensor& positions = axes.positions;
  require((positions.dim() == 1 && positions.size(0) == tokens) ||
              (!packed && positions.dim() == 2 && positions.size(0) == batch && positions.size(1) == tokens),
          axes.get() ? "positions must have shape [tokens], [axes, tokens] or, for x of four dimensions, [axes, batch, tokens]"
                     : "positions must have shape [tokens] or, for x of four dimensions, [batch, tokens]");
  const int code = code_of(x);
  require_type(code >= 0 && code <= 2, "x must be float32, float16 or bfloat16");
  require_positions(positions);
  require(x.stride(-1) == 1 || d == 1, "the last dimension of x must be contiguous");
  if (out_given.has_value()) {
    require(out_given->sizes() == x.sizes() && (out_given->stride(-1) == 1 || d == 1), "out must have the shape of x and contiguous rows");
    require_distinct(*out_given, "out");
    require_type(out_given->scalar_type() == x.scalar_type(), "out must have the dtype of x");
    require(out_given->device() == x.device(), "out must be on the device of x");
    require_apart(*out_given, x, "x");
  }
  const Rotary rotary(turns, magnitude, interleaved, d, x.device());
  require(positions.device() == x.device(), "positions must be on the device of x");
  require_cuda(x);
  const c10::DeviceGuard on_device(x.device());
  const at::Tensor out = out_given.has_value() ? *out_given : at::empty(x.sizes(), x.options());
  auto strides = [&](const at::Tensor& t, int64_t* s) {
    s[0] = packed || batch == 1 ? 0 : t.stride(0);
    s[1] = heads == 1 ? 0 : t.stride(1);
    s[2] = tokens == 1 ? 0 : t.stride(packed ? 0 : 2);
  };
  int64_t xs[3], os[3];
  strides(x, xs);
  strides(out, os);
  check(risa_b200_rotate_axes(x.data_ptr(), out.data_ptr(), code, int(batch), int(heads), int(tokens), int(d), xs, os, positions.data_ptr(),
                              positions.scalar_type() == at::kLong, positions.dim() == 2 ? positions.stride(0) : 0, positions.stride(-1),
                              &rotary.r, axes.get(), transposed ? 1 : 0, stream_of(stream_ptr)));
  return out;
}

// The rotation is linear: its gradient is the transposed rotation of the output's gradient, whose own gradient is the rotation
// again.  (A Function in Python took 88 us for a small tensor's forward and backward pass.)
struct Rotation : public torch::autograd::Function<Rotation> {
  // the stream that is current on the tensors' device: in a backward pass the one that the forward pass ran on
  static uintptr_t stream_on(const c10::Device& device) {
    const c10::impl::VirtualGuardImpl devices(device.type());
    return reinterpret_cast<uintptr_t>(devices.getStream(device).native_handle());
  }
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x, const at::Tensor& positions, const at::Tensor& turns,
                            const MaybeTensor& axes, int64_t axis_count, double magnitude, bool interleaved, bool transposed) {
    ctx->save_for_backward({positions, turns, axes.has_value() ? *axes : at::Tensor()});
    ctx->saved_data["axis_count"] = axis_count;
    ctx->saved_data["magnitude"] = magnitude;
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["transposed"] = transposed;
    return rotate(x, positions, turns, axes, axis_count, magnitude, interleaved, transposed, std::nullopt, x.is_cuda() ? stream_on(x.device()) : 0);
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    // gradients of sums and broadcasts arrive as expanded views
    const at::Tensor grad = grads[0].stride(-1) == 1 ? grads[0] : grads[0].contiguous();
    const MaybeTensor axes = saved[2].defined() ? MaybeTensor(saved[2]) : std::nullopt;
    return {Rotation::apply(grad, saved[0], saved[1], axes, ctx->saved_data["axis_count"].toInt(), ctx->saved_data["magnitude"].toDouble(),
                            ctx->saved_data["interleaved"].toBool(), !ctx->saved_data["transposed"].toBool()),
            at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
  }
};
at::Tensor rotate_with_gradient(const at::Tensor& x, const at::Tensor& positions, const at::Tensor& turns, const MaybeTensor& axes,
                                int64_t axis_count, double magnitude, bool interleaved, bool transposed) {
  require_no_tangent(x);
  return Rotation::apply(x, positions, turns, axes, axis_count, magnitude, interleaved, transposed);
}

// Writes k and v [tokens, kv_heads, head_dim]; returns q rotated, or None.
MaybeTensor cache_append(const at::Tensor& cache_keys, const at::Tensor& cache_values, const MaybeTensor& key_scales,
                         const MaybeTensor& value_scales, const at::Tensor& k, const at::Tensor& v, const at::Tensor& table,
                         const at::Tensor& lengths, const MaybeTensor& offsets, const MaybeTensor& q, const MaybeTensor& turns,
                         const MaybeTensor& axes_of_pairs, int64_t axis_count, double magnitude, bool interleaved,
                         const MaybeTensor& positions, uintptr_t stream_ptr) {
  const Cache cache(cache_keys, cache_values, key_scales, value_scales);
  const int64_t heads = cache.c.kv_heads, d = cache.c.head_dim;
  require(k.dim() == 3 && k.size(1) == heads && k.size(2) == d && v.sizes() == k.sizes(), "k and v must have shape [tokens, kv_heads, head_dim] of the cache");
  const int64_t tokens = k.size(0);
  require(!q.has_value() || (q->dim() == 3 && q->size(0) == tokens && q->size(1) > 0 && q->size(2) == d), "q must have shape [tokens, q_heads, head_dim]");
  require(!q.has_value() || turns.has_value(), "q is only rotated: it needs a rotary table");
  require(!positions.has_value() || (positions->dim() == 1 && positions->size(0) == tokens) ||
              (axes_of_pairs.has_value() && positions->dim() == 2 && positions->size(1) == tokens),
          axes_of_pairs.has_value() ? "positions must have shape [tokens] or [axes, tokens]" : "positions must have shape [tokens]");
  require(!positions.has_value() || turns.has_value(), "positions need a rotary table");
  const int code = code_of(k);
  require_type(code == 1 || code == 2, "k and v must be float16 or bfloat16");
  require_type(v.scalar_type() == k.scalar_type() && (!q.has_value() || q->scalar_type() == k.scalar_type()), "q, k and v must have the same dtype");
  require_type(cache.c.dtype_code >= kInt8 || cache.c.dtype_code == code, "k and v must have the dtype of the cache");
  if (positions.has_value()) {
    require_positions(*positions);
    require(positions->is_contiguous(), "positions must be contiguous");
  }
  const Step step(cache, table, lengths, offsets, tokens);
  const at::Device device = cache_keys.device();
  require(k.device() == device && v.device() == device && (!q.has_value() || q->device() == device) &&
              (!positions.has_value() || positions->device() == device),
          "q, k, v and positions must be on the device of the cache");
  std::optional<Rotary> rotary;
  std::optional<Axes> axes;
  if (turns.has_value()) {
    axes.emplace(axes_of_pairs, axis_count, *turns, positions.has_value() ? *positions : at::Tensor(), 1);
    rotary.emplace(*turns, magnitude, interleaved, d, device);
    require(rotary->r.rotary_dim % 16 == 0, "appending needs a rotary_dim that is a multiple of 16");
  }
  require_cuda(cache_keys);
  const c10::DeviceGuard on_device(device);
  const at::Tensor kr = rows_of(k), vr = rows_of(v);
  const Strides2 ks(kr), vs(vr);
  MaybeTensor qr, out;
  std::optional<Strides2> qs, os;
  if (q.has_value()) {
    qr = rows_of(*q);
    out = at::empty({tokens, q->size(1), d}, q->options());
    qs.emplace(*qr);
    os.emplace(*out);
  }
  check(risa_b200_cache_append_axes(&cache.c, &step.s, kr.data_ptr(), ks.of, vr.data_ptr(), vs.of, qr.has_value() ? qr->data_ptr() : nullptr,
                               qs.has_value() ? qs->of : nullptr, out.has_value() ? out->data_ptr() : nullptr,
                               os.has_value() ? os->of : nullptr, q.has_value() ? int(q->size(1)) : 0, code,
                               rotary.has_value() ? &rotary->r : nullptr, rotary.has_value() ? axes->get() : nullptr, positions.has_value() ? positions->data_ptr() : nullptr,
                               positions.has_value() && positions->scalar_type() == at::kLong, stream_of(stream_ptr)));
  return out;
}

// Keys and values [tokens, kv_heads, head_dim] of a step's tokens, as the cache holds them.
py::tuple cache_read(const at::Tensor& cache_keys, const at::Tensor& cache_values, const MaybeTensor& key_scales, const MaybeTensor& value_scales,
                     const at::Tensor& table, const at::Tensor& lengths, const MaybeTensor& offsets, int64_t tokens,
                     std::optional<at::ScalarType> dtype, uintptr_t stream_ptr) {
  const Cache cache(cache_keys, cache_values, key_scales, value_scales);
  const at::ScalarType type = dtype.value_or(cache_keys.scalar_type());
  require(dtype.has_value() || cache.c.dtype_code < kInt8, "a cache of codes is read as float16 or bfloat16: say which");
  require_type(type == at::kHalf || type == at::kBFloat16, "keys and values are read as float16 or bfloat16");
  require_type(cache.c.dtype_code >= kInt8 || type == cache_keys.scalar_type(), "keys and values must be read in the dtype of the cache");
  const Step step(cache, table, lengths, offsets, tokens);
  require_cuda(cache_keys);
  const c10::DeviceGuard on_device(cache_keys.device());
  const at::Tensor k = at::empty({tokens, cache.c.kv_heads, cache.c.head_dim}, cache_keys.options().dtype(type)), v = at::empty_like(k);
  const Strides2 ks(k), vs(v);
  check(risa_b200_cache_read(&cache.c, &step.s, k.data_ptr(), ks.of, v.data_ptr(), vs.of, code_of(k), stream_of(stream_ptr)));
  return py::make_tuple(k, v);
}

// Checks that attention and key weights share.
void check_queries(const Cache& cache, const at::Tensor& q, const std::optional<int64_t>& window, int64_t sinks, bool is_causal) {
  require(q.dim() == 3 && q.size(2) == cache.c.head_dim, "q must have shape [tokens, q_heads, head_dim of the cache]");
  require(q.size(1) > 0 && q.size(1) % cache.c.kv_heads == 0,
          "q head count (" + std::to_string(q.size(1)) + ") must be divisible by the cache's head count (" + std::to_string(cache.c.kv_heads) + ")");
  require(q.size(0) < ((int64_t(1) << 31) - 1024) / (q.size(1) / cache.c.kv_heads), "q has too many rows");
  require(!window.has_value() || (*window > 0 && *window < (int64_t(1) << 31)), "window must be positive");
  require(!window.has_value() || is_causal, "a window needs the causal rule");
  require(sinks >= 0 && sinks < (int64_t(1) << 31), "sinks must not be negative");
  require(sinks == 0 || window.has_value(), "sinks stay visible in front of a window, and there is none");
  require_type(code_of(q) == 1 || code_of(q) == 2, "q must be float16 or bfloat16");
  require_type(cache.c.dtype_code >= kInt8 || cache.c.dtype_code == code_of(q), "q must have the dtype of the cache");
}

py::tuple paged_attention(const at::Tensor& q, const at::Tensor& cache_keys, const at::Tensor& cache_values, const MaybeTensor& key_scales,
                          const MaybeTensor& value_scales, const at::Tensor& table, const at::Tensor& lengths, const MaybeTensor& offsets,
                          double scale, bool is_causal, std::optional<int64_t> window, int64_t sinks, bool return_lse, const MaybeTensor& out_given,
                          uintptr_t stream_ptr) {
  const Cache cache(cache_keys, cache_values, key_scales, value_scales);
  check_queries(cache, q, window, sinks, is_causal);
  if (out_given.has_value()) {
    require(out_given->sizes() == q.sizes() && out_given->stride(2) == 1 && (q.size(0) <= 1 || out_given->stride(0) % 8 == 0) &&
                (q.size(1) <= 1 || out_given->stride(1) % 8 == 0),
            "out must have the shape of q and rows that start on 16-byte boundaries");
    require_distinct(*out_given, "out");
    require_type(out_given->scalar_type() == q.scalar_type(), "out must have the dtype of q");
    require_apart(*out_given, q, "q");
  }
  const Step step(cache, table, lengths, offsets, q.size(0));
  require(q.device() == cache_keys.device() && (!out_given.has_value() || out_given->device() == q.device()), "q and out must be on the device of the cache");
  require_cuda(q);
  const c10::DeviceGuard on_device(q.device());
  const at::Tensor qr = rows_of(q);
  const at::Tensor out = out_given.has_value() ? *out_given : at::empty(q.sizes(), q.options());
  MaybeTensor lse;
  if (return_lse) lse = at::empty({q.size(0), q.size(1)}, q.options().dtype(at::kFloat));
  const size_t bytes = risa_b200_paged_attention_scratch_size(&cache.c, &step.s, int(q.size(1)));
  const at::Tensor scratch = at::empty({int64_t(bytes)}, q.options().dtype(at::kByte));
  const Strides2 qs(qr), os(out);
  check(risa_b200_paged_attention_sinks(&cache.c, &step.s, qr.data_ptr(), qs.of, int(q.size(1)), code_of(q), out.data_ptr(), os.of,
                                  return_lse ? lse->data_ptr<float>() : nullptr, float(scale), is_causal ? 1 : 0,
                                  window.has_value() ? int(*window) : 0, int(sinks), out_given.has_value() ? 2 : 3, scratch.data_ptr(), bytes,
                                  stream_of(stream_ptr)));
  return py::make_tuple(out, lse);
}

at::Tensor key_weights(const at::Tensor& q, const at::Tensor& lse, const at::Tensor& cache_keys, const at::Tensor& cache_values,
                       const MaybeTensor& key_scales, const MaybeTensor& value_scales, const at::Tensor& table, const at::Tensor& lengths,
                       const MaybeTensor& offsets, double scale, bool is_causal, std::optional<int64_t> window, int64_t sinks, const MaybeTensor& previous,
                       uintptr_t stream_ptr) {
  const Cache cache(cache_keys, cache_values, key_scales, value_scales);
  check_queries(cache, q, window, sinks, is_causal);
  require(lse.dim() == 2 && lse.size(0) == q.size(0) && lse.size(1) == q.size(1), "lse must have shape [tokens, q_heads]");
  require_type(lse.scalar_type() == at::kFloat, "lse must be float32");
  const Step step(cache, table, lengths, offsets, q.size(0));
  const int64_t slots = table.size(1) * cache.c.page_size;
  if (previous.has_value()) {
    require(previous->dim() == 3 && previous->size(0) == table.size(0) && previous->size(1) == cache.c.kv_heads && previous->size(2) == slots &&
                previous->is_contiguous(),
            "previous must be contiguous [batch, kv_heads, pages of a sequence * page_size]");
    require_type(previous->scalar_type() == at::kFloat, "previous must be float32");
    require(previous->device() == q.device(), "previous must be on the device of q");
  }
  require(q.device() == cache_keys.device() && lse.device() == q.device(), "q and lse must be on the device of the cache");
  require_cuda(q);
  const c10::DeviceGuard on_device(q.device());
  const at::Tensor qr = rows_of(q), rows = lse.contiguous();
  at::Tensor weights = at::empty({table.size(0), cache.c.kv_heads, slots}, lse.options());
  const size_t bytes = risa_b200_key_weights_scratch_size(&cache.c, &step.s, int(q.size(1)));
  MaybeTensor scratch;
  if (bytes) scratch = at::empty({int64_t(bytes)}, q.options().dtype(at::kByte));
  const Strides2 qs(qr);
  check(risa_b200_key_weights_sinks(&cache.c, &step.s, qr.data_ptr(), qs.of, int(q.size(1)), code_of(q), rows.data_ptr<float>(), float(scale),
                              is_causal ? 1 : 0, window.has_value() ? int(*window) : 0, int(sinks),
                              previous.has_value() ? previous->data_ptr<float>() : nullptr, weights.data_ptr<float>(),
                              bytes ? scratch->data_ptr() : nullptr, bytes, stream_of(stream_ptr)));
  return weights;
}

py::tuple cache_evict(const at::Tensor& cache_keys, const at::Tensor& cache_values, const MaybeTensor& key_scales, const MaybeTensor& value_scales,
                      const at::Tensor& table, const at::Tensor& lengths, const at::Tensor& weights, const at::Tensor& target,
                      int64_t budget, int64_t recent, uintptr_t stream_ptr) {
  const Cache cache(cache_keys, cache_values, key_scales, value_scales);
  const Step step(cache, table, lengths, std::nullopt, table.dim() == 2 ? table.size(0) : 0);
  const int64_t batch = table.size(0), heads = cache.c.kv_heads, slots = table.size(1) * cache.c.page_size;
  require(weights.dim() == 3 && weights.size(0) == batch && weights.size(1) == heads && weights.size(2) == slots && weights.is_contiguous(),
          "weights must be contiguous [batch, kv_heads, pages of a sequence * page_size]");
  require_type(weights.scalar_type() == at::kFloat, "weights must be float32");
  require(target.dim() == 2 && target.size(0) == batch, "target_table must have shape [batch, pages]");
  require_indices(target, "target_table");
  require(budget > 0 && recent >= 0 && recent <= budget, "budget must be positive and recent between 0 and budget");
  require(target.size(1) * cache.c.page_size >= budget, "the pages of target_table do not hold the budget");
  require(target.size(1) * cache.c.page_size < kMostSlots, "target_table is too wide: a sequence may hold fewer than 2^31 - 8192 keys");
  require(target.data_ptr() != table.data_ptr(), "target_table must name other pages than page_table");
  require(weights.device() == cache_keys.device() && target.device() == cache_keys.device(), "weights and target_table must be on the device of the cache");
  require_cuda(cache_keys);
  const c10::DeviceGuard on_device(cache_keys.device());
  const at::Tensor kept = at::empty({batch, heads, budget}, table.options()), new_lengths = at::empty({batch}, table.options()),
                   new_weights = at::empty({batch, heads, target.size(1) * cache.c.page_size}, weights.options());
  check(risa_b200_cache_evict(&cache.c, &step.s, weights.data_ptr<float>(), target.data_ptr<int32_t>(), int(target.size(1)), int(budget),
                              int(recent), kept.data_ptr<int32_t>(), new_lengths.data_ptr<int32_t>(), new_weights.data_ptr<float>(),
                              stream_of(stream_ptr)));
  return py::make_tuple(kept, new_lengths, new_weights);
}

// ---- pages ----------------------------------------------------------------------------------------------------
// Page table and lengths of sequences, without a step's tokens.
Step sequences_of(const Cache& cache, const at::Tensor& table, const at::Tensor& lengths) {
  return Step(cache, table, lengths, std::nullopt, table.dim() == 2 ? table.size(0) : 0);
}
void require_counts(const Cache& cache, const at::Tensor& references) {
  require(references.dim() == 1 && references.size(0) == cache.c.pages, "references must have shape [pages of the cache]");
  require_indices(references, "references");
  require(references.device() == cache.keys.device(), "references must be on the device of the cache");
}

py::tuple fork_sequences(const at::Tensor& cache_keys, const at::Tensor& cache_values, const MaybeTensor& key_scales, const MaybeTensor& value_scales,
                         const at::Tensor& references, const at::Tensor& table, const at::Tensor& lengths, const at::Tensor& parents,
                         uintptr_t stream_ptr) {
  const Cache cache(cache_keys, cache_values, key_scales, value_scales);
  require_counts(cache, references);
  const Step step = sequences_of(cache, table, lengths);
  require(parents.dim() == 1 && parents.size(0) > 0 && parents.size(0) < (int64_t(1) << 31), "parents must have shape [children]");
  require_indices(parents, "parents");
  require(table.size(1) <= 65535 * 256, "page_table is too wide");
  require(parents.device() == cache_keys.device(), "parents must be on the device of the cache");
  require_cuda(cache_keys);
  const c10::DeviceGuard on_device(cache_keys.device());
  const at::Tensor new_table = at::empty({parents.size(0), table.size(1)}, table.options()), new_lengths = at::empty({parents.size(0)}, table.options());
  check(risa_b200_fork_sequences(&cache.c, references.data_ptr<int32_t>(), &step.s, parents.data_ptr<int32_t>(), int(parents.size(0)),
                                 new_table.data_ptr<int32_t>(), new_lengths.data_ptr<int32_t>(), stream_of(stream_ptr)));
  return py::make_tuple(new_table, new_lengths);
}

at::Tensor resize_sequences(const at::Tensor& cache_keys, const at::Tensor& cache_values, const MaybeTensor& key_scales,
                            const MaybeTensor& value_scales, const at::Tensor& references, const at::Tensor& table, const at::Tensor& lengths,
                            const at::Tensor& new_lengths, uintptr_t stream_ptr) {
  const Cache cache(cache_keys, cache_values, key_scales, value_scales);
  require_counts(cache, references);
  const Step step = sequences_of(cache, table, lengths);
  require(new_lengths.dim() == 1 && new_lengths.size(0) == table.size(0), "new_lengths must have shape [batch]");
  require_indices(new_lengths, "new_lengths");
  require(new_lengths.device() == cache_keys.device(), "new_lengths must be on the device of the cache");
  require_cuda(cache_keys);
  const c10::DeviceGuard on_device(cache_keys.device());
  const at::Tensor granted = at::empty({table.size(0)}, table.options());
  const size_t bytes = risa_b200_resize_scratch_size(&cache.c, step.s.batch);
  const at::Tensor scratch = at::empty({int64_t(bytes)}, table.options().dtype(at::kByte));
  check(risa_b200_resize_sequences(&cache.c, references.data_ptr<int32_t>(), table.data_ptr<int32_t>(), step.s.table_width, step.s.lengths,
                                   new_lengths.data_ptr<int32_t>(), step.s.batch, granted.data_ptr<int32_t>(), scratch.data_ptr(), bytes,
                                   stream_of(stream_ptr)));
  return granted;
}

// Whether two tensors share memory (both are contiguous).
bool share_memory(const at::Tensor& a, const at::Tensor& b) {
  const char *p = static_cast<const char*>(a.data_ptr()), *q = static_cast<const char*>(b.data_ptr());
  return p < q + b.nbytes() && q < p + a.nbytes();
}

py::tuple cache_compact(const at::Tensor& cache_keys, const at::Tensor& cache_values, const MaybeTensor& key_scales, const MaybeTensor& value_scales,
                        const at::Tensor& references, const at::Tensor& table, const at::Tensor& lengths, const at::Tensor& target_keys,
                        const at::Tensor& target_values, const MaybeTensor& target_key_scales, const MaybeTensor& target_value_scales,
                        uintptr_t stream_ptr) {
  const Cache cache(cache_keys, cache_values, key_scales, value_scales), target(target_keys, target_values, target_key_scales, target_value_scales);
  require_counts(cache, references);
  const Step step = sequences_of(cache, table, lengths);
  require_type(target.c.dtype_code == cache.c.dtype_code, "target must have the dtype of the cache");
  require(target.c.kv_heads == cache.c.kv_heads && target.c.page_size == cache.c.page_size && target.c.head_dim == cache.c.head_dim,
          "target must have pages of the same kind as the cache");
  require(target_keys.device() == cache_keys.device(), "target must be on the device of the cache");
  for (const at::Tensor* from : {&cache_keys, &cache_values})
    for (const at::Tensor* to : {&target_keys, &target_values}) require(!share_memory(*from, *to), "target must be another pool: it shares memory with the cache");
  if (key_scales.has_value())
    for (const at::Tensor* from : {&*key_scales, &*value_scales})
      for (const at::Tensor* to : {&*target_key_scales, &*target_value_scales})
        require(!share_memory(*from, *to), "target must be another pool: its scales share memory with the cache's");
  require_cuda(cache_keys);
  const c10::DeviceGuard on_device(cache_keys.device());
  const at::Tensor new_table = at::empty_like(table), counts = at::empty({target.c.pages}, table.options()), used = at::empty({1}, table.options());
  const size_t bytes = risa_b200_compact_scratch_size(&cache.c, &target.c);
  const at::Tensor scratch = at::empty({int64_t(bytes)}, table.options().dtype(at::kByte));
  check(risa_b200_cache_compact(&cache.c, references.data_ptr<int32_t>(), &step.s, &target.c, new_table.data_ptr<int32_t>(),
                                counts.data_ptr<int32_t>(), used.data_ptr<int32_t>(), scratch.data_ptr(), bytes, stream_of(stream_ptr)));
  return py::make_tuple(new_table, counts, used);
}

}  // namespace

void bind_cache(py::module_& m) {
  m.def("rotate", &rotate);
  m.def("rotate_with_gradient", &rotate_with_gradient);
  m.def("cache_append", &cache_append);
  m.def("cache_read", &cache_read);
  m.def("paged_attention", &paged_attention);
  m.def("key_weights", &key_weights);
  m.def("cache_evict", &cache_evict);
  m.def("fork_sequences", &fork_sequences);
  m.def("resize_sequences", &resize_sequences);
  m.def("cache_compact", &cache_compact);
  m.def("check_cache", [](const at::Tensor& k, const at::Tensor& v, const MaybeTensor& ks, const MaybeTensor& vs) { Cache(k, v, ks, vs); });
}
