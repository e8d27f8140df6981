// Rotary positions (csrc/rotary.hip): part of host.cpp.

struct Rotary {
    EvoRotary p{};
    Tensor q, k, pos, turns;

    static Tensor rows(const Tensor &t) { return t.stride(-1) == 1 || t.size(-1) <= 1 ? t : t.contiguous(); }
    // strides of [N,H,D], [B,N,H,D] or [B,S,N,H,D] as b, s, n, h
    static void strides(const Tensor &t, int64_t (&to)[4]) {
        const int d = (int)t.dim();
        const int dims[] = {d > 3 ? 0 : -1, d > 4 ? 1 : -1, d - 3, d - 2};
        for (int i = 0; i < 4; ++i) to[i] = dims[i] < 0 || t.size(dims[i]) == 1 ? 0 : t.stride(dims[i]);
    }
    // What is wrong with the call, or nothing; then the parameter block is filled but for what is read and written.
    const char *take(const Tensor &q_, const OptTensor &k_, const Tensor &positions, const Tensor &turns_, bool interleaved, double scale) {
        const bool with = k_ && k_->defined();
        for (const Tensor *t : {&positions, &turns_, with ? &*k_ : &q_})
            if (t->device() != q_.device()) return "all tensors must live on one device";
        if (q_.dim() < 3 || q_.dim() > 5) return "queries must be [N,H,D], [B,N,H,D] or [B,S,N,H,D]";
        if (evo_dtype(q_.scalar_type()) == EVO_NONE) return "queries must be bf16, fp16 or fp32";
        const int64_t d = q_.dim();
        if (with) {
            if (k_->scalar_type() != q_.scalar_type()) return "keys must have the queries' dtype";
            if (k_->dim() != d) return "keys must have the queries' shape but for the heads";
            for (int64_t i = 0; i < d; ++i)
                if (i != d - 2 && k_->size(i) != q_.size(i)) return "keys must have the queries' shape but for the heads";
        }
        const int64_t N = q_.size(d - 3), D = q_.size(d - 1), B = d > 3 ? q_.size(0) : 1, S = d > 4 ? q_.size(1) : 1;
        if (turns_.dim() != 1 || turns_.scalar_type() != at::kLong || turns_.size(0) < 1 || 2 * turns_.size(0) > D)
            return "turns must be int64 [R / 2] with R at most the head dim, as rotary_turns() makes it";
        if (!at::isIntegralType(positions.scalar_type(), false) || positions.scalar_type() == at::kUInt64) return "positions must be whole numbers that int64 holds";
        if ((positions.dim() != 1 && positions.dim() != 2) || positions.size(-1) != N || (positions.dim() == 2 && positions.size(0) != 1 && positions.size(0) != B))
            return "positions must be [N] or [B, N]";
        if (!std::isfinite(scale) || std::abs(scale) > FLT_MAX) return "scale must be a finite number";
        const int64_t Hk = with ? k_->size(d - 2) : 0;
        if (B > INT32_MAX || S > INT32_MAX || N > INT32_MAX || q_.size(d - 2) > INT32_MAX || Hk > INT32_MAX || D > 65536) return "2^31 batches, rows or heads, or a head dim above 65536, are too many";
        pos = positions.scalar_type() == at::kInt || positions.scalar_type() == at::kLong ? positions : positions.to(at::kLong);
        turns = turns_;
        q = rows(q_);
        if (with) k = rows(*k_);
        p.B = (int32_t)B;
        p.S = (int32_t)S;
        p.N = (int32_t)N;
        p.H = (int32_t)q.size(d - 2);
        p.Hk = (int32_t)Hk;
        p.D = (int32_t)D;
        p.R = (int32_t)(2 * turns.size(0));
        p.dtype = evo_dtype(q.scalar_type());
        p.interleaved = interleaved;
        p.scale = (float)scale;
        return nullptr;
    }
    void run(const Tensor &out_q, const Tensor &out_k, bool inverse) {
        if (!q.numel() && !(k.defined() && k.numel())) return;
        const Tensor at_ = pos.stride(-1) == 1 || p.N == 1 ? pos : pos.contiguous(), f = turns.contiguous();
        p.inverse = inverse;
        p.pos_bytes = at_.scalar_type() == at::kInt ? 4 : 8;
        p.pos_stride_b = at_.dim() == 2 && at_.size(0) > 1 ? at_.stride(0) : 0;
        p.pos = at_.data_ptr();
        p.turns = f.data_ptr();
        p.q = ptr_or_null(q);
        p.k = ptr_or_null(k);
        p.out_q = const_cast<void *>(ptr_or_null(out_q));
        p.out_k = const_cast<void *>(ptr_or_null(out_k));
        if (q.defined()) strides(q, p.q_stride), strides(out_q, p.out_q_stride);
        if (k.defined()) strides(k, p.k_stride), strides(out_k, p.out_k_stride);
        check(evoattn_rotary(&p, stream_of(pos)), "evoattn_rotary");
    }
    std::pair<Tensor, Tensor> turned(bool inverse) {
        c10::DeviceGuard on(pos.device());
        Tensor a = q.defined() ? at::empty(q.sizes(), q.options()) : Tensor(), b = k.defined() ? at::empty(k.sizes(), k.options()) : Tensor();
        run(a, b, inverse);
        return {a, b};
    }
};

struct RotaryNode : SavingNode {
    EvoRotary p{};
    at::ScalarType dtype = at::kFloat;
    std::string name() const override { return "RotaryPositionsBackward"; }
    // saved: positions, turns; results: queries, keys
    variable_list apply(variable_list &&grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        const bool rec = at::GradMode::is_enabled();
        variable_list out(2);
        const bool need_q = grads[0].defined() && task_should_compute_output(0), need_k = grads.size() > 1 && grads[1].defined() && task_should_compute_output(1);
        if (!need_q && !need_k) return out;
        {
            const variable_list t = unpacked();
            at::AutoDispatchBelowADInplaceOrView guard;
            Rotary r;
            r.p = p;
            r.pos = t[0];
            r.turns = t[1];
            auto taken = [&](const Tensor &g) { return Rotary::rows(g.scalar_type() == dtype ? g : g.to(dtype)); };
            if (need_q) r.q = taken(grads[0]);
            if (need_k) r.k = taken(grads[1]);
            if (!need_q) r.p.H = 0;
            if (!need_k) r.p.Hk = 0;
            std::tie(out[0], out[1]) = r.turned(!p.inverse);
        }
        return once_differentiable(std::move(out), rec);
    }
};

// None for a call that the node does not stand for or that is wrong: the caller in Python goes its own way and words the error.
std::optional<std::pair<Tensor, OptTensor>> rotary(const Tensor &q, const OptTensor &k, const Tensor &positions, const Tensor &turns, bool interleaved, double scale) {
    if (!plain_modes()) return std::nullopt;
    for (const Tensor *t : {&q, &positions, &turns})
        if (!t->defined() || !plain(*t) || !t->is_cuda()) return std::nullopt;
    const Tensor k0 = k ? *k : Tensor();
    if (k0.defined() && !plain(k0)) return std::nullopt;
    Rotary r;
    std::pair<Tensor, Tensor> out;
    {
        at::AutoDispatchBelowADInplaceOrView guard;
        if (r.take(q, k, positions, turns, interleaved, scale)) return std::nullopt;
        out = r.turned(false);
    }
    if (SavingNode::wanted(q, k0)) {
        auto node = make_node<RotaryNode>(q, k0);
        node->p = r.p;
        node->dtype = q.scalar_type();
        torch::autograd::set_history(out.first, node);
        if (out.second.defined()) torch::autograd::set_history(out.second, node);
        node->save(r.pos);
        node->save(r.turns);
    }
    return std::make_pair(out.first, out.second.defined() ? OptTensor(out.second) : std::nullopt);
}

// The same launch without a node, for the registered operator.
std::pair<Tensor, Tensor> rotary_forward(const Tensor &q, const OptTensor &k, const Tensor &positions, const Tensor &turns, bool interleaved, double scale, bool inverse) {
    Rotary r;
    const char *wrong = r.take(q, k, positions, turns, interleaved, scale);
    TORCH_CHECK_VALUE(!wrong, wrong);
    TORCH_CHECK(q.is_cuda(), "rotary positions run on the GPU only");
    TORCH_CHECK_NOT_IMPLEMENTED(!dual(q) && !(k && dual(*k)), "rotary_positions has no formula for forward mode differentiation");
    auto out = r.turned(inverse);
    return {out.first, out.second.defined() ? out.second : at::empty({0}, q.options())};
}

// Queries and keys that are the first two slices of a projection's result y [..., N, slots, H, D], turned where they lie.
struct RotarySlots {
    static Tensor slot(const Tensor &y, int64_t i) { return y.select(-3, i); }
    static const char *turn(const Tensor &y, const Tensor &positions, const Tensor &turns, bool interleaved, double scale, bool inverse) {
        Rotary r;
        const Tensor q = slot(y, 0), k = slot(y, 1);
        if (const char *wrong = r.take(q, k, positions, turns, interleaved, scale)) return wrong;
        c10::DeviceGuard on(y.device());
        r.run(r.q, r.k, inverse);
        return nullptr;
    }
};
struct RotarySlotsNode : SavingNode {
    std::vector<int64_t> shape;   // the projection's result's
    at::ScalarType dtype = at::kFloat;
    bool interleaved = false;
    double scale = 1.0;
    std::string name() const override { return "RotarySlotsBackward"; }
    // saved: positions, turns
    variable_list apply(variable_list &&grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        const bool rec = at::GradMode::is_enabled();
        variable_list out(1);
        if (!grads[0].defined()) return out;
        {
            const variable_list t = unpacked();
            at::AutoDispatchBelowADInplaceOrView guard;
            Tensor g = std::move(grads[0]);
            // turned where it lies if nobody else has it (a hook, a gradient that is kept, a view), else in a copy
            const bool alone = !rec && g.use_count() == 1 && g.has_storage() && g.storage().use_count() == 1;
            if (g.scalar_type() != dtype) g = g.to(dtype).contiguous();
            else if (!alone || !g.is_contiguous()) g = g.clone(at::MemoryFormat::Contiguous);
            const char *wrong = RotarySlots::turn(g, t[0], t[1], interleaved, scale, true);
            TORCH_INTERNAL_ASSERT(!wrong, wrong);
            out[0] = g.view(shape);
        }
        return once_differentiable(std::move(out), rec);
    }
};
// y as its slices with the first two turned where they lie: y itself is not to be used again (autograd says so where something kept it).  None for a call that the node does not stand for.
OptTensor rotary_slots(const Tensor &y, const std::vector<int64_t> &shape, const Tensor &positions, const Tensor &turns, bool interleaved, double scale) {
    if (!plain_modes()) return std::nullopt;
    for (const Tensor *t : {&y, &positions, &turns})
        if (!t->defined() || !plain(*t) || !t->is_cuda()) return std::nullopt;
    if (!y.is_contiguous() || y.is_view() || (y.requires_grad() && y.is_leaf()) || shape.size() < 4) return std::nullopt;
    Tensor slots;
    {
        at::AutoDispatchBelowADInplaceOrView guard;
        slots = y.view(shape);
        if (RotarySlots::turn(slots, positions, turns, interleaved, scale, false)) return std::nullopt;
    }
    if (!y.is_inference()) torch::autograd::impl::bump_version(y);
    if (SavingNode::wanted(y)) {
        auto node = make_node<RotarySlotsNode>(y);
        node->shape = y.sizes().vec();
        node->dtype = y.scalar_type();
        node->interleaved = interleaved;
        node->scale = scale;
        node->save(positions);
        node->save(turns);
        torch::autograd::set_history(slots, node);
    }
    return slots;
}
std::optional<std::string> rotary_wrong(const Tensor &q, const OptTensor &k, const Tensor &positions, const Tensor &turns, bool interleaved, double scale) {
    Rotary r;
    const char *wrong = r.take(q, k, positions, turns, interleaved, scale);
    return wrong ? std::optional<std::string>(wrong) : std::nullopt;
}
