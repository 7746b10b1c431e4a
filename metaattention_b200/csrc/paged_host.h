// Host side of rotary positions and of paged caches (part of host_ops.cpp): checks, argument structs, outputs, scratch, launch.
// What a call gets wrong is said as a ValueError here, before anything is launched.
#pragma once

struct PagedApi {
  decltype(&attn_b200_rotary) rotary = nullptr;
  decltype(&attn_b200_paged_append) append = nullptr;
  decltype(&attn_b200_paged_read) read = nullptr;
  decltype(&attn_b200_paged_workspace_bytes) bytes = nullptr;
  decltype(&attn_b200_paged_attention) attention = nullptr;
} paged_api;

template <class... Parts>
[[noreturn]] void refuse(const Parts&... parts) {   // with the GIL
  std::ostringstream s;
  (s << ... << parts);
  throw py::value_error(s.str());
}

// An uninitialised tensor straight from the allocator: half of a microsecond less than through the dispatcher.
Tensor fresh(at::IntArrayRef size, at::ScalarType type, const Tensor& like) { return at::detail::empty_cuda(size, type, like.device(), c10::nullopt); }

std::string shape_of(const Tensor& t) {
  std::ostringstream s;
  s << t.sizes();
  return s.str();
}

bool wide_strides(const Tensor& t, int64_t unit) {   // whole 16-byte pieces
  for (int64_t i = 0; i + 1 < t.dim(); ++i)
    if (t.size(i) > 1 && t.stride(i) % unit != 0) return false;
  return t.stride(-1) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
}

// A tensor without memory (its storage freed, or zeros that stand for themselves) has an address that must not be read.
void has_memory(const char* what, const Tensor& t) {
  if (!t.unsafeGetTensorImpl()->storage_initialized()) refuse(what, " ", shape_of(t), " has no memory");
}

// A tangent of forward mode beside the values: these launches would leave it behind without a word.
void no_tangent(const char* what, std::initializer_list<const Tensor*> given) {
  if (torch::autograd::ForwardADLevel::try_get_by_idx(0) == nullptr) return;   // no dual level is open
  for (const Tensor* t : given)
    if (t->_fw_grad(0).defined() && c10::AutogradState::get_tls_state().get_fw_grad_mode())
      refuse(what, " has no forward-mode derivative (torch.autograd.forward_ad): a tensor of the call carries a tangent");
}

// ---------------------------------------------------------------------------------------------------------------
// rotary positions
// ---------------------------------------------------------------------------------------------------------------

struct Turns {   // what a RotaryEmbedding decided at construction, on one device
  Tensor turns;
  int dim = 0;
  bool interleaved = false;
  float magnitude = 1.0f;

  void fill(AttnB200Rotary& r) const {
    r.turns = static_cast<const uint64_t*>(turns.data_ptr());
    r.dim = dim;
    r.interleaved = interleaved;
    r.magnitude = magnitude;
  }

  // Around a launch on the current stream: the RotaryEmbedding may go with that launch still to run, and the memory must then not
  // be handed out again before it has.  Told to the allocator once for each stream.  A captured launch reads the table whenever
  // its graph is replayed, which nobody announces: that table stays for good.
  void used() const {
    const auto now = c10::cuda::getCurrentCUDAStream(turns.device().index());
    if (kept_.load(std::memory_order_relaxed)) return;
    cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
    C10_CUDA_CHECK(cudaStreamIsCapturing(now.stream(), &capture));
    if (capture == cudaStreamCaptureStatusNone && told_.load(std::memory_order_relaxed) == now.id()) return;   // as the last call
    std::lock_guard<std::mutex> lock(mutex_);
    if (capture != cudaStreamCaptureStatusNone) {
      static auto* kept = new std::vector<Tensor>();
      static std::mutex kept_mutex;
      std::lock_guard<std::mutex> all(kept_mutex);
      kept->push_back(turns);
      kept_ = true;
      return;
    }
    if (std::find(streams_.begin(), streams_.end(), now.id()) == streams_.end()) {
      c10::cuda::CUDACachingAllocator::recordStream(turns.storage().data_ptr(), now);
      streams_.push_back(now.id());
    }
    told_ = now.id();
  }

 private:
  mutable std::mutex mutex_;
  mutable std::vector<c10::StreamId> streams_;
  mutable std::atomic<c10::StreamId> told_{std::numeric_limits<c10::StreamId>::min()};
  mutable std::atomic<bool> kept_{false};
};

// y = x turned, for x = q and perhaps k; [tokens, heads, D] or [batch, seq, heads, D]
std::vector<Tensor> rotary_launch(const Turns& turns, const std::vector<Tensor>& x, const OptTensor& positions, bool inverse, bool inplace) {
  std::vector<Tensor> y;
  AttnB200RotaryArgs a;
  std::memset(&a, 0, sizeof(a));
  const Tensor& q = x[0];
  const int lead = q.dim() - 2;   // 1 or 2 axes of tokens
  for (const Tensor& t : x) y.push_back(inplace ? t : fresh(t.sizes(), t.scalar_type(), t));
  if (q.size(0) == 0 || q.size(lead - 1) == 0) return y;   // no tokens; q, or k, without heads is passed over below
  a.batch = lead == 2 ? q.size(0) : 1;
  a.seq = q.size(lead - 1);
  a.head_dim = q.size(-1);
  a.dtype = q.scalar_type() == at::kFloat ? ATTN_B200_DTYPE_FP32 : dtype_code(q);
  a.inverse = inverse;
  turns.fill(a.rotary);
  turns.used();
  int n = 0;
  for (size_t i = 0; i < x.size(); ++i) {
    if (x[i].size(lead) == 0) continue;   // no heads
    a.x[n] = x[i].data_ptr();
    a.y[n] = y[i].data_ptr();
    a.heads[n] = x[i].size(lead);
    for (int d = 0; d < 2; ++d) {
      const Tensor& t = d == 0 ? x[i] : y[i];
      int64_t* s = d == 0 ? a.x_stride[n] : a.y_stride[n];
      s[0] = lead == 2 ? t.stride(0) : 0;
      s[1] = t.stride(lead - 1);
      s[2] = t.stride(lead);
    }
    ++n;
  }
  if (n == 0) return y;
  if (positions.has_value()) {
    const Tensor& p = *positions;
    a.positions = p.data_ptr();
    a.positions_64 = p.scalar_type() == at::kLong;
    a.pos_stride[0] = p.dim() == 2 && p.size(0) > 1 ? p.stride(0) : 0;
    a.pos_stride[1] = p.stride(-1);
  }
  check(paged_api.rotary(&a, stream_of(q)), "attn_b200_rotary");
  return y;
}

struct TurnsRef : torch::CustomClassHolder {
  std::shared_ptr<const Turns> turns;
  bool inverse = false;
};

// The map is linear and its transpose is the map by the opposite angles, so the backward is the same function again, and
// differentiable itself.  Only what asks for a gradient gets one, on both ways.
struct RotaryFunction : torch::autograd::Function<RotaryFunction> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const std::shared_ptr<const Turns>& turns, bool inverse,
                                                const OptTensor& positions, const Tensor& q, const OptTensor& k) {
    auto ref = c10::make_intrusive<TurnsRef>();
    ref->turns = turns;
    ref->inverse = inverse;
    ctx->saved_data["turns"] = c10::IValue::make_capsule(ref);
    ctx->save_for_backward({positions.value_or(Tensor())});
    ctx->set_materialize_grads(false);
    at::AutoDispatchBelowADInplaceOrView below;
    std::vector<Tensor> x{q};
    if (k.has_value()) x.push_back(*k);
    auto y = rotary_launch(*turns, x, positions, inverse, false);
    std::vector<Tensor> constant;
    for (size_t i = 0; i < x.size(); ++i)
      if (!x[i].requires_grad()) constant.push_back(y[i]);
    ctx->mark_non_differentiable(constant);
    return y;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto ref = c10::static_intrusive_pointer_cast<TurnsRef>(ctx->saved_data["turns"].toCapsule());
    const Tensor saved = ctx->get_saved_variables()[0];
    const OptTensor positions = saved.defined() ? OptTensor(saved) : OptTensor();
    torch::autograd::variable_list out(5);
    std::vector<int> which;
    std::vector<Tensor> g;
    for (size_t i = 0; i < grads.size(); ++i)
      if (grads[i].defined() && ctx->needs_input_grad((saved.defined() ? 1 : 0) + i)) {   // counted over the tensors of the call
        which.push_back(static_cast<int>(i));
        const bool zeros = grads[i]._is_zerotensor();   // without memory of their own
        g.push_back(zeros ? at::zeros(grads[i].sizes(), grads[i].options()) : grads[i].stride(-1) == 1 || grads[i].numel() == 0 ? grads[i] : grads[i].contiguous());
      }
    if (g.empty()) return out;
    c10::cuda::CUDAGuard guard(g[0].device());
    const auto r = apply(ref->turns, !ref->inverse, positions, g[0], g.size() > 1 ? OptTensor(g[1]) : OptTensor());
    for (size_t i = 0; i < which.size(); ++i) out[3 + which[i]] = r[i];
    return out;
  }
};

// [q'] or [q', k']
std::vector<Tensor> rotary_call(const std::shared_ptr<const Turns>& turns, const Tensor& q, const OptTensor& k, const OptTensor& positions, bool inplace) {
  const auto type = q.scalar_type();
  if (type != at::kHalf && type != at::kBFloat16 && type != at::kFloat) refuse("rotary positions turn float16, bfloat16 and float32 tensors (got ", type, ")");
  if (q.dim() != 3 && q.dim() != 4) refuse("q must be [tokens, heads, head_dim] or [batch, seq, heads, head_dim], got ", shape_of(q));
  const int lead = q.dim() - 2;
  if (q.size(-1) < turns->dim) refuse("the head dim ", q.size(-1), " is smaller than rotary_dim ", turns->dim);
  if (turns->turns.device() != q.device()) refuse("the frequencies are on ", turns->turns.device(), ", q is on ", q.device());
  std::vector<Tensor> x{q};
  if (k.has_value()) {
    if (k->dim() != q.dim() || k->size(-1) != q.size(-1) || k->size(0) != q.size(0) || (lead == 2 && k->size(1) != q.size(1)))
      refuse("k ", shape_of(*k), " does not have the tokens and head dim of q ", shape_of(q));
    if (k->scalar_type() != type || k->device() != q.device()) refuse("q and k must share dtype and device");
    x.push_back(*k);
  }
  for (const Tensor& t : x) {
    no_tangent("a rotation by positions", {&t});
    for (int64_t d = 0; d < t.dim(); ++d)
      if (t.size(d) > 0x7fffffff) refuse("up to 2^31 - 1 tokens, heads and columns are turned, got ", shape_of(t));
    has_memory("a tensor of heads", t);
    if (t.numel() > 0 && t.stride(-1) != 1) refuse("the last dimension must be contiguous");
  }
  if (positions.has_value()) {
    const Tensor& p = *positions;
    if (p.scalar_type() != at::kInt && p.scalar_type() != at::kLong) refuse("positions must be int32 or int64 (got ", p.scalar_type(), ")");
    if (p.device() != q.device()) refuse("positions must be on the device of q");
    has_memory("positions", p);
    const bool shared = p.dim() == 1 && p.size(0) == q.size(lead - 1);
    const bool each = p.dim() == 2 && lead == 2 && (p.size(0) == q.size(0) || p.size(0) == 1) && p.size(1) == q.size(1);
    if (!shared && !each) refuse("positions must be [seq] or [batch, seq] for q ", shape_of(q), ", got ", shape_of(p));
  }
  const bool grad = at::GradMode::is_enabled() && (q.requires_grad() || (k.has_value() && k->requires_grad()));
  if (inplace) {
    if (grad) refuse("in place, nothing is kept for a backward pass: use it under torch.no_grad(), or let it return new tensors");
    for (const Tensor& t : x)
      for (int64_t d = 0; d < t.dim(); ++d)
        if (t.size(d) > 1 && t.stride(d) == 0) refuse("in place, every value must have memory of its own (an expanded tensor has not)");
    if (k.has_value() && k->numel() > 0 && k->data_ptr() == q.data_ptr()) refuse("in place, q and k must not be the same memory");
  }
  py::gil_scoped_release others_run;
  c10::cuda::CUDAGuard guard(q.device());
  if (grad) return RotaryFunction::apply(turns, false, positions, q, k);
  at::AutoDispatchBelowADInplaceOrView below;
  auto y = rotary_launch(*turns, x, positions, false, inplace);
  if (inplace)
    for (Tensor& t : y)
      if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();   // a graph that has saved it finds out
  return y;
}

// ---------------------------------------------------------------------------------------------------------------
// paged caches
// ---------------------------------------------------------------------------------------------------------------

struct Cache {
  Tensor k, v, k_scale, v_scale;
  std::vector<int64_t> shape;   // of the pools
  AttnB200PagedCache view;
};

std::shared_ptr<Cache> make_cache(const Tensor& k, const Tensor& v, const OptTensor& k_scale, const OptTensor& v_scale) {
  auto c = std::make_shared<Cache>();
  std::memset(&c->view, 0, sizeof(c->view));
  if (k.dim() != 4) refuse("the pools must be [num_pages, page_size, heads_kv, head_dim], got ", shape_of(k));
  if (v.sizes() != k.sizes()) refuse("k and v pools must have the same shape (got ", shape_of(k), ", ", shape_of(v), ")");
  if (v.scalar_type() != k.scalar_type() || v.device() != k.device()) refuse("k and v pools must share dtype and device");
  const bool codes = k.scalar_type() == at::kFloat8_e4m3fn;
  if (!codes && dtype_code(k) < 0) refuse("a cache holds float16, bfloat16 or float8_e4m3fn (got ", k.scalar_type(), ")");
  if (k.numel() == 0) refuse("the pools must not be empty");
  const int64_t page = k.size(1), D = k.size(3);
  if (D != 64 && D != 128) refuse("head_dim must be 64 or 128 (got ", D, ")");
  if (page < 8 || (page & (page - 1)) != 0) refuse("page_size must be a power of two of at least 8 (got ", page, ")");
  if (k.size(0) > 0x7fffffff || page > 0x40000000 || k.size(2) > 65535) refuse("the pools are too large");
  for (const Tensor* t : {&k, &v}) {
    has_memory("a pool", *t);
    if (!wide_strides(*t, codes ? 16 : 8)) refuse("the pools need a contiguous last dimension, and strides and addresses of whole 16 bytes");
    for (int i = 0; i < 3; ++i)
      if (t->size(i) > 1 && t->stride(i) <= 0) refuse("the pools need positive strides");
  }
  if (k_scale.has_value() != codes || v_scale.has_value() != codes) refuse("8-bit pools come with k_scale and v_scale, others without");
  if (codes) {
    for (const OptTensor* t : {&k_scale, &v_scale}) {
      const Tensor& s = **t;
      if (s.scalar_type() != at::kFloat8_e8m0fnu && s.scalar_type() != at::kByte) refuse("scales must be float8_e8m0fnu or uint8 exponents (got ", s.scalar_type(), ")");
      if (s.dim() != 3 || s.size(0) != k.size(0) || s.size(1) != page || s.size(2) != k.size(2))
        refuse("scales must be [num_pages, page_size, heads_kv] for pools ", shape_of(k), ", got ", shape_of(s));
      if (s.device() != k.device()) refuse("pools and scales must be on one device");
      has_memory("a pool of scales", s);
      for (int i = 0; i < 3; ++i)
        if (s.size(i) > 1 && s.stride(i) <= 0) refuse("scales need positive strides");
    }
    c->k_scale = *k_scale;
    c->v_scale = *v_scale;
    c->view.k_scale = static_cast<uint8_t*>(k_scale->data_ptr());
    c->view.v_scale = static_cast<uint8_t*>(v_scale->data_ptr());
  }
  c->k = k;
  c->v = v;
  c->shape = k.sizes().vec();
  AttnB200PagedCache& a = c->view;
  a.k = k.data_ptr();
  a.v = v.data_ptr();
  for (int i = 0; i < 3; ++i) {
    a.k_stride[i] = k.stride(i);
    a.v_stride[i] = v.stride(i);
    if (codes) {
      a.k_scale_stride[i] = k_scale->stride(i);
      a.v_scale_stride[i] = v_scale->stride(i);
    }
  }
  a.num_pages = k.size(0);
  a.page_size = page;
  a.heads_kv = k.size(2);
  a.head_dim = D;
  a.dtype = codes ? ATTN_B200_DTYPE_E4M3 : dtype_code(k);
  return c;
}

// The sequences of a call; `held` keeps a copy alive until its launch.
AttnB200PagedCache sequences(const Cache& c, const Tensor& table, const Tensor& lens, Tensor& held) {
  // a pool whose tensor was resized or given other memory since the cache was made: its pages are no longer where the view says
  bool same = c.k.dim() == 4 && c.v.dim() == 4 && c.k.data_ptr() == c.view.k && c.v.data_ptr() == c.view.v && c.k.sizes() == c.shape && c.v.sizes() == c.shape;
  for (int i = 0; same && i < 3; ++i) same = c.k.stride(i) == c.view.k_stride[i] && c.v.stride(i) == c.view.v_stride[i];
  if (same && c.view.k_scale != nullptr) {
    const at::IntArrayRef rows(c.shape.data(), 3);
    same = c.k_scale.data_ptr() == c.view.k_scale && c.v_scale.data_ptr() == c.view.v_scale && c.k_scale.sizes() == rows && c.v_scale.sizes() == rows;
    for (int i = 0; same && i < 3; ++i) same = c.k_scale.stride(i) == c.view.k_scale_stride[i] && c.v_scale.stride(i) == c.view.v_scale_stride[i];
  }
  if (!same) refuse("the pools have other memory or another shape than when the PagedKVCache was made: make a new one");
  if (!c.k.is_cuda()) refuse("the cache is not on a CUDA device");
  if (table.scalar_type() != at::kInt || table.dim() != 2) refuse("block_table must be an int32 tensor [batch, max_blocks], got ", table.scalar_type(), " ", shape_of(table));
  if (lens.scalar_type() != at::kInt || lens.dim() != 1 || lens.size(0) != table.size(0))
    refuse("cache_seqlens must be an int32 tensor [batch] for block_table ", shape_of(table), ", got ", lens.scalar_type(), " ", shape_of(lens));
  if (table.device() != c.k.device() || lens.device() != c.k.device()) refuse("block_table and cache_seqlens must be on the device of the cache");
  if (table.numel() == 0) refuse("block_table must not be empty");
  if (lens.size(0) > 1 && lens.stride(0) != 1) refuse("cache_seqlens must be contiguous");
  if (table.size(1) > 0x7fffffff / c.view.page_size) refuse("a sequence may have up to 2^31 - 1 tokens (got ", table.size(1), " blocks of ", c.view.page_size, ")");
  held = table.stride(1) == 1 || table.size(1) == 1 ? table : table.contiguous();
  AttnB200PagedCache a = c.view;
  a.block_table = held.data_ptr<int32_t>();
  a.block_table_stride = held.stride(0);
  a.seq_lens = lens.data_ptr<int32_t>();
  a.max_blocks = held.size(1);
  a.batch = held.size(0);
  return a;
}

// Rows of a call's new tokens, [batch, seq, heads, D] or packed [rows, heads, D]: what is wrong with them is said here.
void new_rows(const Cache& c, const Tensor& t, const char* what, const OptTensor& cu, int64_t batch, int64_t heads) {
  const bool packed = cu.has_value();
  if (t.dim() != (packed ? 3 : 4) || t.size(-1) != c.view.head_dim || t.size(-2) != heads || (!packed && t.size(0) != batch))
    refuse(what, " must be ", packed ? "[rows, heads, head_dim] (cu_seqlens is given)" : "[batch, seq, heads, head_dim]", " with batch ", batch, ", heads ", heads,
           ", head_dim ", c.view.head_dim, ", got ", shape_of(t));
  if (t.device() != c.k.device()) refuse(what, " must be on the device of the cache");
  if (dtype_code(t) < 0 || (c.view.dtype != ATTN_B200_DTYPE_E4M3 && t.scalar_type() != c.k.scalar_type()))
    refuse(what, " must be float16 or bfloat16, and the dtype of a 16-bit cache (got ", t.scalar_type(), ")");
  if (t.size(packed ? 0 : 1) > 0x7fffffff || (!packed && t.size(0) * t.size(1) > 0x7fffffff)) refuse(what, " has too many rows");
  has_memory(what, t);
  if (t.numel() > 0 && !wide_strides(t, 8)) refuse(what, " needs a contiguous last dimension, and strides and address of whole 16 bytes");
  if (packed && (cu->scalar_type() != at::kInt || cu->dim() != 1 || cu->size(0) != batch + 1 || (batch > 0 && cu->stride(0) != 1) || cu->device() != c.k.device()))
    refuse("cu_seqlens must be a contiguous int32 tensor [batch + 1] on the device of the cache");
}

void row_strides(int64_t (&dst)[3], const Tensor& t) {
  const int d = t.dim();
  dst[0] = d == 4 ? t.stride(0) : 0;
  dst[1] = t.stride(d - 3);
  dst[2] = t.stride(d - 2);
}

void cache_append(const Cache& c, const Tensor& k, const Tensor& v, const Tensor& table, const Tensor& lens, const OptTensor& cu,
                  const std::shared_ptr<const Turns>& turns) {
  AttnB200PagedAppendArgs a;
  std::memset(&a, 0, sizeof(a));
  Tensor held;
  no_tangent("a cache", {&k, &v, &c.k, &c.v});
  if (c.view.k == c.view.v || (c.view.k_scale != nullptr && c.view.k_scale == c.view.v_scale)) refuse("the k and v of a cache that is written must not be the same memory");
  a.cache = sequences(c, table, lens, held);
  new_rows(c, k, "k", cu, a.cache.batch, a.cache.heads_kv);
  new_rows(c, v, "v", cu, a.cache.batch, a.cache.heads_kv);
  if (k.sizes() != v.sizes() || k.scalar_type() != v.scalar_type()) refuse("k and v must have the same shape and dtype (got ", shape_of(k), ", ", shape_of(v), ")");
  if (at::GradMode::is_enabled() && (k.requires_grad() || v.requires_grad() || c.k.requires_grad() || c.v.requires_grad())) refuse("a cache has no gradient: append under torch.no_grad()");
  if (turns != nullptr) {
    if (turns->dim % 16 != 0 || turns->dim > c.view.head_dim) refuse("rotary_dim of keys on their way into a cache must be a multiple of 16, up to the head dim");
    if (turns->turns.device() != c.k.device()) refuse("the frequencies are on ", turns->turns.device(), ", the cache is on ", c.k.device());
    turns->fill(a.rotary);
  }
  if (k.numel() == 0) return;
  a.k = k.data_ptr();
  a.v = v.data_ptr();
  row_strides(a.k_stride, k);
  row_strides(a.v_stride, v);
  a.cu_seqlens = cu.has_value() ? cu->data_ptr<int32_t>() : nullptr;
  a.seq = k.size(k.dim() - 3);
  a.dtype = dtype_code(k);
  py::gil_scoped_release others_run;
  c10::cuda::CUDAGuard guard(k.device());
  if (turns != nullptr) turns->used();
  check(paged_api.append(&a, stream_of(k)), "attn_b200_paged_append");
  for (const Tensor* t : {&c.k, &c.v, &c.k_scale, &c.v_scale})
    if (t->defined() && !t->is_inference()) t->unsafeGetTensorImpl()->bump_version();   // a graph that has saved it finds out
}

std::vector<Tensor> cache_read(const Cache& c, const Tensor& table, const Tensor& lens, int64_t max_len, bool bf16) {
  AttnB200PagedReadArgs a;
  std::memset(&a, 0, sizeof(a));
  Tensor held;
  no_tangent("a cache", {&c.k, &c.v});
  a.cache = sequences(c, table, lens, held);
  if (max_len < 0 || max_len > 0x7fffffff) refuse("max_len must not be negative (got ", max_len, ")");
  if (at::GradMode::is_enabled() && (c.k.requires_grad() || c.v.requires_grad())) refuse("a cache has no gradient: read it under torch.no_grad()");
  if (a.cache.dtype != ATTN_B200_DTYPE_E4M3 && bf16 != (a.cache.dtype == ATTN_B200_DTYPE_BF16)) refuse("a 16-bit cache is read in its own dtype");
  py::gil_scoped_release others_run;
  at::AutoDispatchBelowADInplaceOrView below;
  c10::cuda::CUDAGuard guard(c.k.device());
  const auto type = bf16 ? at::kBFloat16 : at::kHalf;
  Tensor k = fresh({a.cache.batch, max_len, a.cache.heads_kv, a.cache.head_dim}, type, c.k), v = fresh(k.sizes(), type, c.k);
  if (max_len == 0) return {k, v};
  a.k = k.data_ptr();
  a.v = v.data_ptr();
  a.max_len = max_len;
  a.dtype = bf16 ? ATTN_B200_DTYPE_BF16 : ATTN_B200_DTYPE_FP16;
  check(paged_api.read(&a, stream_of(k)), "attn_b200_paged_read");
  return {k, v};
}

// (o, lse or None)
std::tuple<Tensor, OptTensor> cache_attention(const Cache& c, const Tensor& q, const Tensor& table, const Tensor& lens, const OptTensor& cu, double scale,
                                              bool causal, int64_t window, const OptTensor& out, bool want_lse) {
  AttnB200PagedAttnArgs a;
  std::memset(&a, 0, sizeof(a));
  Tensor held;
  no_tangent("attention over a paged cache", {&q, &c.k, &c.v});
  if (out.has_value()) no_tangent("attention over a paged cache", {&*out});
  a.cache = sequences(c, table, lens, held);
  if (q.dim() < 3) refuse("q must be [batch, seq, heads, head_dim], or [rows, heads, head_dim] with cu_seqlens, got ", shape_of(q));
  const int64_t H = q.size(-2), Hkv = a.cache.heads_kv;
  new_rows(c, q, "q", cu, a.cache.batch, H);
  if (H % Hkv != 0 || H / Hkv > 128) refuse("the ", H, " query heads must be a multiple, of up to 128, of the ", Hkv, " KV heads");
  if (H > 65535) refuse("too many query heads");
  constexpr int64_t kMost = 0x3fffffff;
  if (static_cast<int64_t>(a.cache.max_blocks) * a.cache.page_size > kMost)
    refuse("attention takes sequences of up to 2^30 - 1 tokens (block_table has room for ", a.cache.max_blocks, " blocks of ", a.cache.page_size, ")");
  if ((cu.has_value() ? 1 : q.size(0)) * q.size(q.dim() - 3) > kMost) refuse("attention takes up to 2^30 - 1 new tokens, got q ", shape_of(q));
  if (a.cache.batch > 1024) refuse("at most 1024 sequences (got ", a.cache.batch, ")");
  if (!(scale > 0.0) || !std::isfinite(static_cast<float>(scale)) || static_cast<float>(scale) == 0.0f) refuse("scale must be positive and finite (got ", scale, ")");
  if (window < 0) refuse("window must be positive (got ", window, ")");
  if (window > 0 && !causal) refuse("a window counts back from each row: it needs causal=True");
  if (at::GradMode::is_enabled() && (q.requires_grad() || c.k.requires_grad() || c.v.requires_grad() || (out.has_value() && out->requires_grad())))
    refuse("attention over a paged cache has no backward pass: call it under torch.no_grad()");
  if (out.has_value()) {
    new_rows(c, *out, "out", cu, a.cache.batch, H);
    if (out->sizes() != q.sizes() || out->scalar_type() != q.scalar_type()) refuse("out must have the shape and dtype of q (got ", shape_of(*out), ")");
    for (int64_t d = 0; d < out->dim(); ++d)
      if (out->size(d) > 1 && out->stride(d) == 0) refuse("every value of out must have memory of its own (an expanded tensor has not)");
  }
  const int64_t seq = q.size(q.dim() - 3);
  a.cu_seqlens = cu.has_value() ? cu->data_ptr<int32_t>() : nullptr;
  a.heads = H;
  a.seq = seq;
  a.dtype = dtype_code(q);
  a.scale = static_cast<float>(scale);
  a.causal = causal;
  a.window = static_cast<int32_t>(std::min<int64_t>(window, kMost));
  c10::cuda::CUDAGuard guard(q.device());
  int64_t need = 0;
  if (q.numel() > 0) {
    need = paged_api.bytes(&a);   // all but the length of the list of work has been looked at above
    if (need < 0) refuse("the call is too long: ", a.cache.batch, " sequences of up to ", a.cache.max_blocks, " blocks, q ", shape_of(q));
  }
  py::gil_scoped_release others_run;
  at::AutoDispatchBelowADInplaceOrView below;
  Tensor o = out.has_value() ? *out : fresh(q.sizes(), q.scalar_type(), q);
  OptTensor lse;
  if (want_lse) lse = cu.has_value() ? fresh({H, seq}, at::kFloat, q) : fresh({q.size(0), H, seq}, at::kFloat, q);
  if (q.numel() == 0) return {o, lse};
  a.q = q.data_ptr();
  a.o = o.data_ptr();
  a.lse = want_lse ? lse->data_ptr<float>() : nullptr;
  row_strides(a.q_stride, q);
  row_strides(a.o_stride, o);
  Tensor ws = fresh({std::max<int64_t>(need, 16)}, at::kByte, q);
  a.workspace = ws.data_ptr();
  a.workspace_bytes = ws.numel();
  int rc = paged_api.attention(&a, stream_of(q));
  Tensor own;
  if (rc == ATTN_B200_E_UNSUPPORTED) {   // q in memory that several values share, for a kernel whose loads have no stride of zero: nothing was launched
    for (int64_t d = 0; d < q.dim() && !own.defined(); ++d)
      if (q.size(d) > 1 && q.stride(d) == 0) own = q.contiguous();
    if (own.defined()) {
      a.q = own.data_ptr();
      row_strides(a.q_stride, own);
      rc = paged_api.attention(&a, stream_of(q));
    }
  }
  check(rc, "attn_b200_paged_attention");
  if (out.has_value() && !o.is_inference()) o.unsafeGetTensorImpl()->bump_version();
  return {o, lse};
}

void bind_paged(const py::dict& d) {
  take(paged_api.rotary, d, "attn_b200_rotary");
  take(paged_api.append, d, "attn_b200_paged_append");
  take(paged_api.read, d, "attn_b200_paged_read");
  take(paged_api.bytes, d, "attn_b200_paged_workspace_bytes");
  take(paged_api.attention, d, "attn_b200_paged_attention");
}

std::shared_ptr<Turns> make_turns(const Tensor& turns, int dim, bool interleaved, double magnitude) {
  auto t = std::make_shared<Turns>();
  t->turns = turns;
  t->dim = dim;
  t->interleaved = interleaved;
  t->magnitude = static_cast<float>(magnitude);
  return t;
}

void def_paged(py::module_& m) {
  py::class_<Turns, std::shared_ptr<Turns>>(m, "Turns");
  py::class_<Cache, std::shared_ptr<Cache>>(m, "Cache");
  m.def("make_turns", &make_turns);
  m.def("rotary", [](const std::shared_ptr<Turns>& t, const Tensor& q, const OptTensor& k, const OptTensor& positions, bool inplace) -> py::object {
    std::vector<Tensor> y = rotary_call(t, q, k, positions, inplace);
    if (y.size() == 1) return py::cast(std::move(y[0]));
    return py::make_tuple(std::move(y[0]), std::move(y[1]));
  });
  m.def("make_cache", &make_cache);
  m.def("cache_append", [](const Cache& c, const Tensor& k, const Tensor& v, const Tensor& table, const Tensor& lens, const OptTensor& cu,
                           const std::shared_ptr<Turns>& turns) { cache_append(c, k, v, table, lens, cu, turns); });
  m.def("cache_read", &cache_read);
  m.def("cache_attention", &cache_attention);
}
