// Native host path of the operators for token sequences (RotaryPEAxes, SinkSwa, kv_append_rope, sink_swa_decode): the part of
// torch_api.cpp (which includes it inside its namespace) that checks arguments, allocates outputs, calls the C ABI and records the
// autograd nodes.

// ---- shared checks --------------------------------------------------------------------------------------------------
void check_cuda(std::initializer_list<const Tensor*> ts, const char* names) {
  const Tensor* first = nullptr;
  for (const Tensor* t : ts) {
    if (!t->defined()) continue;
    TORCH_CHECK(t->is_cuda(), "dl_templates_b200 runs on CUDA tensors only (sm_100a); there is no CPU path");
    if (!first) first = t;
    TORCH_CHECK(t->device() == first->device(), names, " must be on one device: ", t->device(), " beside ", first->device());
  }
}

Tensor int_vector(const Tensor& t, int64_t n, const char* name) {
  if (!t.defined()) return t;
  TORCH_CHECK_TYPE(t.scalar_type() == at::kInt, name, " must be int32");
  TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == n, name, ": expected [", n, "], one per sequence");
  return t.contiguous();
}

// A tensor the kernels write: one place in memory for each element, as far as strides tell.
void check_writable(const Tensor& t, const char* name) {
  for (int64_t i = 0; i < t.dim(); ++i)
    TORCH_CHECK_VALUE(t.size(i) == 1 || t.stride(i) > 0, name, " is an expanded tensor: its elements share memory");
}

// Sizes reach the kernels as 32-bit numbers.
void check_sizes(std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts)
    for (const int64_t n : t->sizes()) TORCH_CHECK_VALUE(n <= INT32_MAX, "a tensor of shape ", t->sizes(), " is too large");
}

// An output the caller gives: blocks write it while others still read the inputs, so that it shares no memory with them.  (Views
// that interleave in one buffer pass: strides alone do not tell.)
void check_apart(const Tensor& out, std::initializer_list<const Tensor*> others, const char* name) {
  for (const Tensor* t : others) {
    if (!t->defined() || !t->numel() || !out.numel()) continue;
    const at::MemOverlapStatus s = at::get_overlap_status(out, *t);
    TORCH_CHECK_VALUE(s != at::MemOverlapStatus::Full && s != at::MemOverlapStatus::Partial && out.data_ptr() != t->data_ptr(), name,
                      " shares memory with another tensor of the call");
  }
}

// Tells autograd that a tensor it may have saved was written.
void written(const Tensor& t) {
  if (t.defined() && !t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

bool legacy_default(const c10::Stream& s) { return c10::cuda::CUDAStream(s).stream() == nullptr; }

// While a graph is captured, autograd's engine has the stream of each leaf's accumulator wait for the captured one and then waits for it in turn.
// A side stream -- a warm-up's, whose last loss is still there -- becomes a part of the capture by that and leaves it again.  The legacy default
// stream may take no part in a capture: what follows ends the process inside the engine.  Refused here, while nothing has been
// launched: for every leaf that the inputs come from, since all of them take part in the backward pass.
void check_capture(std::initializer_list<const Tensor*> inputs) {
  for (const Tensor* t : inputs)
    if (!t->is_cuda()) return;                                   // (refused further on)
  const c10::cuda::OptionalCUDAGuard guard((*inputs.begin())->device());
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None) return;
  std::vector<std::shared_ptr<torch::autograd::Node>> todo;
  for (const Tensor* t : inputs) {
    if (!t->defined() || !t->requires_grad()) continue;
    if (auto n = t->grad_fn() ? t->grad_fn() : torch::autograd::impl::try_get_grad_accumulator(*t)) todo.push_back(std::move(n));
  }
  std::unordered_set<const torch::autograd::Node*> seen;
  while (!todo.empty()) {
    const std::shared_ptr<torch::autograd::Node> n = std::move(todo.back());
    todo.pop_back();
    if (!seen.insert(n.get()).second) continue;
    for (const torch::autograd::Edge& e : n->next_edges())
      if (e.function) todo.push_back(e.function);
    if (!dynamic_cast<const torch::autograd::AccumulateGrad*>(n.get())) continue;
    const std::optional<c10::Stream> s = n->stream();
    TORCH_CHECK(!s.has_value() || !legacy_default(*s),
                "a leaf of this call belongs to an autograd graph recorded on the default stream that is still alive; its backward pass "
                "cannot be captured: drop that graph (its outputs and losses) before capturing, record it on a side stream, or capture with "
                "detached leaves");
  }
}

// What the entries without an autograd.Function cannot answer and would drop without a word: a tangent of an input, and the call itself in a
// trace, which would hold its output as torch found it, empty.
void nothing_to_record(std::initializer_list<const Tensor*> inputs, const char* name) {
  TORCH_CHECK(!at::tracer::impl::is_dispatch_enabled(), name, " leaves nothing in a jit trace: trace SinkSwa.apply or RotaryPEAxes.apply");
  for (const Tensor* t : inputs)
    TORCH_CHECK(!t->defined() || !t->_fw_grad(0).defined(), name, " has no forward-mode derivative: an input carries a tangent");
}

// What a backward node does first: its gradients are no functions of the graph.
void no_second_derivative(const char* name) {
  TORCH_CHECK(!c10::GradMode::is_enabled(), name, " has no second derivatives: call backward without create_graph");
}

// ---- rotary positions with several axes -----------------------------------------------------------------------------
struct Axes {
  Tensor pos;
  std::vector<Tensor> tables;
};

// Checks positions and tables against B sequences of N tokens and describes them; `ax` keeps what the description points to.
rope_axes_t axes_view(Axes& ax, int64_t B, int64_t N, const Tensor& like) {
  rope_axes_t r{};
  if (!ax.pos.defined()) {
    TORCH_CHECK_VALUE(ax.tables.empty(), "tables without positions");
    return r;
  }
  const int64_t A = (int64_t)ax.tables.size();
  TORCH_CHECK_VALUE(A >= 1 && A <= ROPE_MAX_AXES, "1 to ", ROPE_MAX_AXES, " axes expected, got ", A, " tables");
  TORCH_CHECK_TYPE(ax.pos.scalar_type() == at::kInt, "positions must be int32");
  const bool batched = ax.pos.dim() == 3;
  TORCH_CHECK_VALUE((batched || ax.pos.dim() == 2) && ax.pos.size(-2) == A && ax.pos.size(-1) == N && (!batched || ax.pos.size(0) == B),
                    "expected positions [", A, ", ", N, "] or [", B, ", ", A, ", ", N, "], got ", ax.pos.sizes());
  TORCH_CHECK(ax.pos.device() == like.device(), "positions must be on the device of the tensors: ", ax.pos.device(), " beside ", like.device());
  if (ax.pos.stride(-1) != 1) ax.pos = ax.pos.contiguous();
  r.pos = ax.pos.data_ptr<int32_t>();
  r.pos_stride[0] = batched ? ax.pos.stride(0) : 0;
  r.pos_stride[1] = ax.pos.stride(-2);
  r.n_axes = (int32_t)A;
  for (int64_t a = 0; a < A; ++a) {
    Tensor& t = ax.tables[a];
    TORCH_CHECK_TYPE(t.scalar_type() == at::kFloat, "cos/sin tables must be float32");
    TORCH_CHECK_VALUE(t.dim() == 3 && t.size(2) == 2 && t.size(0) > 0 && t.size(1) > 0 && t.size(0) <= INT32_MAX,
                      "cos/sin tables must be [max_pos, n_pairs, 2], got ", t.sizes());
    TORCH_CHECK(t.device() == like.device(), "cos/sin tables must be on the device of the tensors: ", t.device(), " beside ", like.device());
    TORCH_CHECK(!wants_grad({&t}), "cos/sin tables get no gradient");
    if (!t.is_contiguous()) t = t.contiguous();
    if (reinterpret_cast<uintptr_t>(t.data_ptr()) % 16) t = t.clone();
    r.n_pairs[a] = (int32_t)t.size(1);
    r.max_pos[a] = (int32_t)t.size(0);
    r.cs[a] = t.data_ptr<float>();
  }
  return r;
}

// The rotation of x and, if given, x2, in new contiguous tensors.
std::array<Tensor, 2> rotate_axes(const Tensor& x, const Tensor& x2, Axes ax, bool inverse) {
  poll_status();
  check_cuda({&x, &x2}, "q and k");
  TORCH_CHECK_VALUE(x.dim() == 4, "expected [B,H,N,C]");
  check_sizes({&x});
  const int32_t dt = dtype_code(x.scalar_type());
  if (x2.defined()) {
    TORCH_CHECK_VALUE(x2.dim() == 4 && x2.size(0) == x.size(0) && x2.size(2) == x.size(2) && x2.size(3) == x.size(3),
                      "q and k must agree in batch, tokens and head dim: ", x.sizes(), " beside ", x2.sizes());
    check_sizes({&x2});
    TORCH_CHECK_TYPE(x2.scalar_type() == x.scalar_type(), "q and k must share a dtype");
  }
  TORCH_CHECK_VALUE(ax.pos.defined(), "positions expected");
  const rope_axes_t r = axes_view(ax, x.size(0), x.size(2), x);
  const c10::cuda::OptionalCUDAGuard guard(x.device());
  std::array<Tensor, 2> y{at::empty(x.sizes(), x.options()), x2.defined() ? at::empty(x2.sizes(), x2.options()) : Tensor()};
  const swa_tensor_t a = view4(x), b = view4(y[0]);
  swa_tensor_t c{}, d{};
  if (x2.defined()) { c = view4(x2); d = view4(y[1]); }
  check(rope_axes_apply(dt, &r, (int32_t)x.size(0), x.size(2), (int32_t)x.size(3), &a, &b, (int32_t)x.size(1), x2.defined() ? &c : nullptr,
                        x2.defined() ? &d : nullptr, x2.defined() ? (int32_t)x2.size(1) : 0, inverse ? 1 : 0, stream_of(x)),
        "rope_axes_apply");
  return y;
}

struct AxesNode : public torch::autograd::Node {
  SavedVariable pos;
  std::vector<SavedVariable> tables;

  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    no_second_derivative("RotaryPEAxes");
    Axes ax;
    ax.pos = pos.unpack();
    for (SavedVariable& t : tables) ax.tables.push_back(t.unpack());
    if (!grads[0].defined() && !grads[1].defined()) return {Tensor(), Tensor()};
    if (grads[0].defined() && grads[1].defined()) {
      const auto y = rotate_axes(grads[0], grads[1], std::move(ax), true);
      return {y[0], y[1]};
    }
    const int one = grads[0].defined() ? 0 : 1;
    variable_list out(2);
    out[one] = rotate_axes(grads[one], Tensor(), std::move(ax), true)[0];
    return out;
  }
  std::string name() const override { return "RotaryPEAxesBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    pos.reset_data();
    for (SavedVariable& t : tables) t.reset_data();
  }
};

std::array<Tensor, 2> apply_axes(const Tensor& q, const Tensor& k, const Axes& ax) {
  const bool grad = wants_grad({&q, &k});
  if (grad) check_capture({&q, &k});
  for (const Tensor& t : ax.tables) TORCH_CHECK(!wants_grad({&t}), "cos/sin tables get no gradient");
  const at::AutoGradMode no_grad(false);
  const auto y = rotate_axes(q, k, ax, false);
  if (grad) {
    std::shared_ptr<AxesNode> n(new AxesNode(), torch::autograd::deleteNode);
    n->set_next_edges(torch::autograd::collect_next_edges(q, k));
    n->pos = SavedVariable(ax.pos, false);
    for (const Tensor& t : ax.tables) n->tables.emplace_back(t, false);
    for (const Tensor& t : y) torch::autograd::set_history(t, n);
  }
  return y;
}

// ---- attention with a sliding window and sink tokens ---------------------------------------------------------------
struct SinkWin {
  int32_t window, n_sink;
  float sm;
};

sink_geom_t sink_geom(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& lens, const SinkWin& w, int32_t impl) {
  return sink_geom_t{dtype_code(q.scalar_type()), (int32_t)q.size(0), (int32_t)q.size(1), (int32_t)k.size(1), (int32_t)q.size(2),
                     (int32_t)q.size(3), (int32_t)v.size(3), w.window, w.n_sink, w.sm, forced_impl(impl),
                     lens.defined() ? lens.data_ptr<int32_t>() : nullptr};
}

void check_sink(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& lens) {
  poll_status();
  check_cuda({&q, &k, &v, &lens}, "q, k, v and seq_lens");
  TORCH_CHECK_VALUE(q.dim() == 4 && k.dim() == 4 && v.dim() == 4 && k.size(0) == q.size(0) && k.size(2) == q.size(2) &&
                        k.size(3) == q.size(3) && v.size(0) == k.size(0) && v.size(1) == k.size(1) && v.size(2) == k.size(2),
                    "expected q [B,Hq,N,d_qk], k [B,Hkv,N,d_qk] and v [B,Hkv,N,d_v]");
  TORCH_CHECK_VALUE(k.size(1) > 0 && q.size(1) % k.size(1) == 0, "the heads of q must be a multiple of the heads of k and v");
  check_sizes({&q, &k, &v});
  TORCH_CHECK_TYPE(q.scalar_type() == k.scalar_type() && q.scalar_type() == v.scalar_type(), "q, k, v must share a dtype");
}

// The tiled kernels (tensor cores; fp32 on the CUDA cores) want rows that are whole 16-byte units, and up to 128 elements.  What reaches them
// otherwise is made so here, since the kernels that take anything are a warp a row, tens to hundreds of times slower:
// head dims are padded with zero columns (scores unchanged, zero columns of O) ...
int64_t sink_padded(const Tensor& t, const Tensor& q, const Tensor& v, int32_t impl) {
  const int64_t d = t.size(3), e = t.scalar_type() == at::kFloat ? 4 : 8;
  return impl != SWA_IMPL_AUTO || q.size(3) > 128 || v.size(3) > 128 ? d : (d + e - 1) / e * e;
}
// ... and tensors in other layouts -- an expanded gradient, a view that starts off a 16-byte boundary, odd strides -- are copied.  (Not by
// contiguous(), which hands a misaligned contiguous tensor back.)
bool whole_rows(const Tensor& t, int64_t unit = 16) {
  const int64_t e = unit / t.element_size();
  if (t.stride(3) != 1 || reinterpret_cast<uintptr_t>(t.data_ptr()) % unit) return false;
  for (int i = 0; i < 3; ++i)
    if (t.size(i) > 1 && (t.stride(i) <= 0 || t.stride(i) % e)) return false;
  return true;
}
Tensor in_whole_rows(const Tensor& t, int64_t unit = 16) { return whole_rows(t, unit) ? t : t.clone(at::MemoryFormat::Contiguous); }

// Whether a shape is one of the tiled kernels' (f32_shape and tc_unsupported of the library).
bool sink_tiles(const Tensor& q, const Tensor& k, const Tensor& v, const SinkWin& w, int32_t impl) {
  if (q.scalar_type() == at::kFloat) return q.size(3) % 4 == 0 && v.size(3) % 4 == 0 && q.size(3) <= 128 && v.size(3) <= 128;
  const sink_geom_t g = sink_geom(q, k, v, Tensor(), w, impl);
  return sink_swa_select(&g) == SWA_IMPL_TC;
}

// (A dimension of extent 1 may carry any stride.)
swa_tensor_t sink_view(const Tensor& t) {
  swa_tensor_t r = view4(t);
  for (int i = 0; i < 3; ++i)
    if (t.size(i) == 1) r.stride[i] = 0;
  return r;
}

Fwd sink_forward(Tensor q, Tensor k, Tensor v, Tensor lens, const SinkWin& w, int32_t impl, Tensor out) {
  check_sink(q, k, v, lens);
  lens = int_vector(lens, q.size(0), "seq_lens");
  const std::array<int64_t, 4> shape{q.size(0), q.size(1), q.size(2), v.size(3)};
  if (out.defined()) {
    check_out(out, shape, q, "out");
    check_writable(out, "out");
    check_apart(out, {&q, &k, &v}, "out");
  }
  const int64_t pq = sink_padded(q, q, v, impl), pv = sink_padded(v, q, v, impl);
  if (pq != q.size(3) || pv != v.size(3)) {
    Fwd f = sink_forward(pad_last(q, pq), pad_last(k, pq), pad_last(v, pv), lens, w, impl, Tensor());
    const Tensor o = f.o.narrow(3, 0, v.size(3));
    f.o = out.defined() ? out.copy_(o) : o.contiguous();
    return f;
  }
  const c10::cuda::OptionalCUDAGuard guard(q.device());
  const bool tiles = sink_tiles(q, k, v, w, impl), direct = out.defined() && (!tiles || whole_rows(out));
  for (Tensor* t : {&q, &k, &v}) *t = tiles ? in_whole_rows(*t) : materialise(*t);
  Fwd f;
  f.o = direct ? out : at::empty(shape, q.options());
  f.lse = new_lse(q);
  const sink_geom_t g = sink_geom(q, k, v, lens, w, impl);
  const swa_tensor_t tq = sink_view(q), tk = sink_view(k), tv = sink_view(v), to = sink_view(f.o);
  if (direct) written(out);
  check(sink_swa_fwd(&g, &tq, &tk, &tv, &to, f.lse.data_ptr<float>(), status_ptr(q.get_device()), stream_of(q)), "sink_swa_fwd");
  if (out.defined() && !direct) f.o = out.copy_(f.o);
  debug_sync();
  return f;
}

void check_sink_saved(const Tensor& q, const Tensor& v, const Tensor& o, const Tensor& lse, const Tensor& d_o) {
  check_cuda({&q, &o, &d_o, &lse}, "q, o, do and lse");
  const std::array<int64_t, 4> shape{q.size(0), q.size(1), q.size(2), v.size(3)};
  TORCH_CHECK_VALUE(o.sizes() == shape && d_o.sizes() == shape, "expected o, do [B,Hq,N,d_v]");
  TORCH_CHECK_TYPE(o.scalar_type() == q.scalar_type() && d_o.scalar_type() == q.scalar_type(), "o and do must have the dtype of q");
  TORCH_CHECK_TYPE(lse.scalar_type() == at::kFloat, "lse must be float32");
  TORCH_CHECK_VALUE(lse.dim() == 3 && lse.sizes() == at::IntArrayRef(shape).slice(0, 3), "expected lse [B,Hq,N]");
}

Grads sink_backward(Tensor q, Tensor k, Tensor v, Tensor o, Tensor lse, Tensor d_o, Tensor lens, const SinkWin& w, int32_t impl, Grads out) {
  check_sink(q, k, v, lens);
  check_sink_saved(q, v, o, lse, d_o);
  lens = int_vector(lens, q.size(0), "seq_lens");
  const bool given = out.dq.defined() || out.dk.defined() || out.dv.defined();
  if (given) {
    TORCH_CHECK_VALUE(out.dq.defined() && out.dk.defined() && out.dv.defined(), "dq, dk and dv are given together");
    check_out(out.dq, q.sizes(), q, "dq");
    check_out(out.dk, k.sizes(), k, "dk");
    check_out(out.dv, v.sizes(), v, "dv");
    check_writable(out.dq, "dq"); check_writable(out.dk, "dk"); check_writable(out.dv, "dv");
    check_apart(out.dq, {&q, &k, &v, &o, &d_o, &lse, &out.dk, &out.dv}, "dq");
    check_apart(out.dk, {&q, &k, &v, &o, &d_o, &lse, &out.dv}, "dk");
    check_apart(out.dv, {&q, &k, &v, &o, &d_o, &lse}, "dv");
  }
  const int64_t pq = sink_padded(q, q, v, impl), pv = sink_padded(v, q, v, impl);
  if (pq != q.size(3) || pv != v.size(3)) {
    const Grads g = sink_backward(pad_last(q, pq), pad_last(k, pq), pad_last(v, pv), pad_last(o, pv), lse, pad_last(d_o, pv), lens, w, impl, Grads());
    const Tensor dq = g.dq.narrow(3, 0, q.size(3)), dk = g.dk.narrow(3, 0, k.size(3)), dv = g.dv.narrow(3, 0, v.size(3));
    if (!given) return {dq.contiguous(), dk.contiguous(), dv.contiguous()};
    out.dq.copy_(dq);
    out.dk.copy_(dk);
    out.dv.copy_(dv);
    return out;
  }
  const c10::cuda::OptionalCUDAGuard guard(q.device());
  const bool tiles = sink_tiles(q, k, v, w, impl);
  lse = lse.contiguous();
  for (Tensor* t : {&q, &k, &v, &o, &d_o}) *t = tiles ? in_whole_rows(*t) : materialise(*t);
  auto target = [&](const Tensor& to, const Tensor& like) {
    const bool direct = to.defined() && (!tiles || whole_rows(to));
    if (direct) written(to);
    return direct ? to : at::empty(like.sizes(), like.options());
  };
  Grads r{target(out.dq, q), target(out.dk, k), target(out.dv, v)};
  const sink_geom_t g = sink_geom(q, k, v, lens, w, impl);
  const int64_t bytes = sink_swa_bwd_scratch(&g);
  check(bytes < 0 ? (int)bytes : 0, "sink_swa_bwd_scratch");
  const Tensor scratch = at::empty({bytes}, q.options().dtype(at::kByte));
  const swa_tensor_t tq = sink_view(q), tk = sink_view(k), tv = sink_view(v), to = sink_view(o), tdo = sink_view(d_o), tdq = sink_view(r.dq),
                     tdk = sink_view(r.dk), tdv = sink_view(r.dv);
  check(sink_swa_bwd(&g, &tq, &tk, &tv, &to, &tdo, lse.data_ptr<float>(), &tdq, &tdk, &tdv, scratch.data_ptr(), bytes,
                     status_ptr(q.get_device()), stream_of(q)), "sink_swa_bwd");
  if (given) {
    if (!r.dq.is_same(out.dq)) r.dq = out.dq.copy_(r.dq);
    if (!r.dk.is_same(out.dk)) r.dk = out.dk.copy_(r.dk);
    if (!r.dv.is_same(out.dv)) r.dv = out.dv.copy_(r.dv);
  }
  debug_sync();
  return r;
}

struct SinkNode : public torch::autograd::Node {
  SavedVariable q, k, v, lse, o, lens;
  SinkWin win;
  bool has_lens = false;

  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    no_second_derivative("SinkSwa");
    const auto self = shared_from_this();
    if (!grads[0].defined()) return variable_list(3);
    Grads g = sink_backward(q.unpack(), k.unpack(), v.unpack(), o.unpack(self), lse.unpack(), grads[0], has_lens ? lens.unpack() : Tensor(),
                            win, SWA_IMPL_AUTO, Grads());
    return {g.dq, g.dk, g.dv};
  }
  std::string name() const override { return "SinkSwaBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (SavedVariable* s : {&q, &k, &v, &lse, &o, &lens}) s->reset_data();
  }
};

Tensor apply_sink(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& lens, const SinkWin& w) {
  const bool grad = wants_grad({&q, &k, &v});
  if (grad) check_capture({&q, &k, &v});
  const at::AutoGradMode no_grad(false);
  Fwd f = sink_forward(q, k, v, lens, w, SWA_IMPL_AUTO, Tensor());
  if (grad) {
    std::shared_ptr<SinkNode> n(new SinkNode(), torch::autograd::deleteNode);
    n->win = w;
    n->has_lens = lens.defined();
    n->set_next_edges(torch::autograd::collect_next_edges(q, k, v));
    n->q = SavedVariable(q, false);
    n->k = SavedVariable(k, false);
    n->v = SavedVariable(v, false);
    n->lse = SavedVariable(f.lse, false);
    if (lens.defined()) n->lens = SavedVariable(lens, false);
    torch::autograd::set_history(f.o, n);
    n->o = SavedVariable(f.o, true);
  }
  return f.o;
}

// ---- paged cache -----------------------------------------------------------------------------------------------------
// Describes a cache; `table` and `lens` keep what the description points to.
sink_cache_t cache_view(const Tensor& kc, const Tensor& vc, Tensor& table, Tensor& lens, int64_t B, int64_t Hkv, int64_t dqk, int64_t dv,
                        const Tensor& like) {
  check_cuda({&like, &kc, &vc, &table, &lens}, "the tensors, the cache, page_table and seq_lens");
  TORCH_CHECK_TYPE(kc.scalar_type() == like.scalar_type() && vc.scalar_type() == like.scalar_type(), "the cache must have the dtype of the tensors");
  TORCH_CHECK_VALUE(kc.dim() == 4 && vc.dim() == 4 && kc.size(0) == vc.size(0) && kc.size(1) == vc.size(1) && kc.size(2) == vc.size(2) &&
                        kc.size(1) == Hkv && kc.size(3) == dqk && vc.size(3) == dv,
                    "expected caches [pages, Hkv, page_size, d_qk] and [pages, Hkv, page_size, d_v], got ", kc.sizes(), " and ", vc.sizes());
  TORCH_CHECK_TYPE(table.scalar_type() == at::kInt, "page_table must be int32");
  TORCH_CHECK_VALUE(table.dim() == 2 && table.size(0) == B, "expected page_table [B, max_pages], got ", table.sizes());
  TORCH_CHECK_VALUE(lens.defined(), "seq_lens expected");
  table = table.contiguous();
  lens = int_vector(lens, B, "seq_lens");
  TORCH_CHECK_VALUE(kc.size(0) <= INT32_MAX && kc.size(2) <= INT32_MAX && table.size(1) <= INT32_MAX, "cache too large");
  return sink_cache_t{sink_view(kc), sink_view(vc), table.data_ptr<int32_t>(), lens.data_ptr<int32_t>(), (int32_t)kc.size(0), (int32_t)kc.size(2),
                      (int32_t)table.size(1)};
}

void no_gradient(std::initializer_list<const Tensor*> ts, const char* name) {
  for (const Tensor* t : ts)
    TORCH_CHECK(!t->defined() || !wants_grad({t}), name, " is for serving and records no gradient: call it under torch.no_grad()");
}

Tensor kv_append(const Tensor& q, const Tensor& k, const Tensor& v, Axes ax, const Tensor& kc, const Tensor& vc, Tensor table, Tensor lens,
                 Tensor fresh) {
  poll_status();
  no_gradient({&q, &k, &v, &kc, &vc}, "kv_append_rope");
  TORCH_CHECK_VALUE(k.dim() == 4 && v.dim() == 4 && k.sizes().slice(0, 3) == v.sizes().slice(0, 3),
                    "expected k [B,Hkv,T,d_qk] and v [B,Hkv,T,d_v]");
  TORCH_CHECK_TYPE(k.scalar_type() == v.scalar_type(), "q, k, v must share a dtype");
  const int64_t B = k.size(0), T = k.size(2);
  if (q.defined()) {
    TORCH_CHECK_VALUE(q.dim() == 4 && q.size(0) == B && q.size(2) == T && q.size(3) == k.size(3), "expected q [B,Hq,T,d_qk]");
    TORCH_CHECK_TYPE(q.scalar_type() == k.scalar_type(), "q, k, v must share a dtype");
  }
  check_sizes({&k, &v});
  if (q.defined()) check_sizes({&q});
  const int32_t dt = dtype_code(k.scalar_type());
  check_cuda({&k, &q, &v, &fresh}, "q, k, v and new_lens");
  sink_cache_t c = cache_view(kc, vc, table, lens, B, k.size(1), k.size(3), v.size(3), k);
  check_writable(kc, "k_cache");
  check_writable(vc, "v_cache");
  check_apart(kc, {&q, &k, &v, &vc}, "k_cache");
  check_apart(vc, {&q, &k, &v}, "v_cache");
  fresh = int_vector(fresh, B, "new_lens");
  const rope_axes_t r = axes_view(ax, B, T, k);
  const c10::cuda::OptionalCUDAGuard guard(k.device());
  Tensor q_out;
  swa_tensor_t tq{}, tqo{};
  if (q.defined()) {
    q_out = at::empty(q.sizes(), q.options());
    tq = view4(q);
    tqo = view4(q_out);
  }
  const swa_tensor_t tk = view4(k), tv = view4(v);
  check(kv_append_rope(dt, &r, (int32_t)B, q.defined() ? (int32_t)q.size(1) : 0, (int32_t)k.size(1), (int32_t)T, (int32_t)k.size(3),
                       (int32_t)v.size(3), q.defined() ? &tq : nullptr, q.defined() ? &tqo : nullptr, &tk, &tv, &c,
                       fresh.defined() ? fresh.data_ptr<int32_t>() : nullptr, stream_of(k)), "kv_append_rope");
  written(kc);
  written(vc);
  return q_out;
}

Tensor sink_decode(Tensor q, const Tensor& kc, const Tensor& vc, Tensor table, Tensor lens, const SinkWin& w, int32_t impl, Tensor out) {
  poll_status();
  no_gradient({&q, &kc, &vc}, "sink_swa_decode");
  TORCH_CHECK_VALUE(q.dim() == 4 && q.size(2) == 1, "expected q [B,Hq,1,d_qk], one new token of each sequence");
  TORCH_CHECK_VALUE(kc.dim() == 4 && vc.dim() == 4 && kc.size(1) > 0 && q.size(1) % kc.size(1) == 0,
                    "the heads of q must be a multiple of the heads of the cache");
  check_sizes({&q, &kc, &vc});
  const int32_t dt = dtype_code(q.scalar_type());
  const sink_cache_t c = cache_view(kc, vc, table, lens, q.size(0), kc.size(1), q.size(3), vc.size(3), q);
  const std::array<int64_t, 4> shape{q.size(0), q.size(1), 1, vc.size(3)};
  const c10::cuda::OptionalCUDAGuard guard(q.device());
  if (out.defined()) {
    check_out(out, shape, q, "out");
    check_writable(out, "out");
    check_apart(out, {&q, &kc, &vc}, "out");
    written(out);
  } else {
    out = at::empty(shape, q.options());
  }
  // the split kernel reads pairs of elements of q
  if (q.size(3) * q.element_size() % 16 == 0 && q.size(3) <= 128) q = in_whole_rows(q, 2 * q.element_size());
  const swa_tensor_t tq = sink_view(q), to = sink_view(out);
  check(sink_swa_decode(dt, (int32_t)q.size(0), (int32_t)q.size(1), (int32_t)kc.size(1), (int32_t)q.size(3), (int32_t)vc.size(3), w.window,
                        w.n_sink, w.sm, forced_impl(impl), &tq, &c, &to, stream_of(q)), "sink_swa_decode");
  debug_sync();
  return out;
}

// ---- Python ----------------------------------------------------------------------------------------------------------
SinkWin sink_win(Args& a) {
  SinkWin w;
  w.window = a.i32();
  w.n_sink = a.i32();
  w.sm = a.f32();
  return w;
}
// positions (or None) and a sequence of tables
Axes axes_args(Args& a) {
  Axes ax;
  ax.pos = a.maybe_tensor();
  PyObject* seq = PySequence_Fast(a.next(), "cos/sin tables must be a sequence of tensors");
  if (!seq) throw python_error();
  for (Py_ssize_t i = 0; i < PySequence_Fast_GET_SIZE(seq); ++i) {
    PyObject* o = PySequence_Fast_GET_ITEM(seq, i);
    if (!THPVariable_Check(o)) {
      Py_DECREF(seq);
      PyErr_SetString(PyExc_TypeError, "cos/sin tables must be tensors");
      throw python_error();
    }
    ax.tables.push_back(THPVariable_Unpack(o));
  }
  Py_DECREF(seq);
  return ax;
}

bool plain_axes(const Tensor& q, const Tensor& k, const Axes& ax) {
  if (!plain_call({&q, &k}, Rope())) return false;
  for (const Tensor& t : ax.tables)
    if (!plain_call({&t}, Rope())) return false;
  return true;
}

// apply(q, k, positions, *tables) -> (q, k) rotated
PyObject* py_rope_axes(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args a{args, n};
    const Tensor q = a.tensor(), k = a.tensor();
    Axes ax;
    ax.pos = a.tensor();
    while (a.at < n) ax.tables.push_back(a.tensor());
    if (!plain_axes(q, k, ax)) return general(3, args, n);
    const auto y = without_gil([&] { return apply_axes(q, k, ax); });
    return pack({y[0], y[1]});
  });
}
// The entries below come twice where an autograd.Function is made of them: BODY is what its forward and backward call, which torch has
// asked for tangents and recorded in a trace itself.
// rope_axes_to(x, positions, tables, inverse) -> rotated copy
template <bool BODY>
PyObject* py_rope_axes_to(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args a{args, n};
    const Tensor x = a.tensor();
    const Axes ax = axes_args(a);
    const bool inverse = a.i32() != 0;
    a.done();
    if (!BODY) {
      nothing_to_record({&x}, "rope_axes_apply_to");
      for (const Tensor& t : ax.tables) nothing_to_record({&t}, "rope_axes_apply_to");
    }
    const at::AutoGradMode no_grad(false);
    return THPVariable_Wrap(without_gil([&] { return rotate_axes(x, Tensor(), ax, inverse)[0]; }));
  });
}
// apply(q, k, v, seq_lens, window, n_sink, sm_scale)
PyObject* py_sink_swa(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args a{args, n};
    const Tensor q = a.tensor(), k = a.tensor(), v = a.tensor(), lens = a.maybe_tensor();
    const SinkWin w = sink_win(a);
    a.done();
    if (!plain_call({&q, &k, &v}, Rope())) return general(4, args, n);
    return THPVariable_Wrap(without_gil([&] { return apply_sink(q, k, v, lens, w); }));
  });
}
// sink_forward(q, k, v, seq_lens, window, n_sink, sm_scale, impl, out) -> (o, lse)
template <bool BODY>
PyObject* py_sink_forward(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args a{args, n};
    const Tensor q = a.tensor(), k = a.tensor(), v = a.tensor(), lens = a.maybe_tensor();
    const SinkWin w = sink_win(a);
    const int32_t impl = a.i32();
    const Tensor out = a.maybe_tensor();
    a.done();
    if (!BODY) nothing_to_record({&q, &k, &v, &out}, "sink_swa_forward");
    const at::AutoGradMode no_grad(false);
    const Fwd f = without_gil([&] { return sink_forward(q, k, v, lens, w, impl, out); });
    return pack({f.o, f.lse});
  });
}
// sink_backward(q, k, v, o, lse, do, seq_lens, window, n_sink, sm_scale, impl, dq, dk, dv) -> (dq, dk, dv)
template <bool BODY>
PyObject* py_sink_backward(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args a{args, n};
    const Tensor q = a.tensor(), k = a.tensor(), v = a.tensor(), o = a.tensor(), lse = a.tensor(), d_o = a.tensor(), lens = a.maybe_tensor();
    const SinkWin w = sink_win(a);
    const int32_t impl = a.i32();
    const Grads out{a.maybe_tensor(), a.maybe_tensor(), a.maybe_tensor()};
    a.done();
    if (!BODY) nothing_to_record({&q, &k, &v, &o, &lse, &d_o, &out.dq, &out.dk, &out.dv}, "sink_swa_backward");
    const at::AutoGradMode no_grad(false);
    const Grads g = without_gil([&] { return sink_backward(q, k, v, o, lse, d_o, lens, w, impl, out); });
    return pack({g.dq, g.dk, g.dv});
  });
}
// kv_append(q, k, v, positions, tables, k_cache, v_cache, page_table, seq_lens, new_lens) -> rotated q or None
PyObject* py_kv_append(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args a{args, n};
    const Tensor q = a.maybe_tensor(), k = a.tensor(), v = a.tensor();
    const Axes ax = axes_args(a);
    const Tensor kc = a.tensor(), vc = a.tensor(), table = a.tensor(), lens = a.tensor(), fresh = a.maybe_tensor();
    a.done();
    nothing_to_record({&q, &k, &v, &kc, &vc}, "kv_append_rope");
    for (const Tensor& t : ax.tables) nothing_to_record({&t}, "kv_append_rope");
    const Tensor y = without_gil([&] { return kv_append(q, k, v, ax, kc, vc, table, lens, fresh); });
    if (!y.defined()) Py_RETURN_NONE;
    return THPVariable_Wrap(y);
  });
}
// sink_decode(q, k_cache, v_cache, page_table, seq_lens, window, n_sink, sm_scale, impl, out) -> o
PyObject* py_sink_decode(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args a{args, n};
    const Tensor q = a.tensor(), kc = a.tensor(), vc = a.tensor(), table = a.tensor(), lens = a.tensor();
    const SinkWin w = sink_win(a);
    const int32_t impl = a.i32();
    const Tensor out = a.maybe_tensor();
    a.done();
    nothing_to_record({&q, &kc, &vc, &out}, "sink_swa_decode");
    return THPVariable_Wrap(without_gil([&] { return sink_decode(q, kc, vc, table, lens, w, impl, out); }));
  });
}
// set_general_sequence(RotaryPEAxes' and SinkSwa's Function.apply)
PyObject* py_set_general_sequence(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args a{args, n};
    for (int i = 3; i < 5; ++i) {
      PyObject* o = a.next();
      Py_INCREF(o);
      Py_XSETREF(g_general[i], o);
    }
    a.done();
    Py_RETURN_NONE;
  });
}
