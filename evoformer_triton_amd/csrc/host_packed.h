// Attention within packed sequences (csrc/packed.hip): part of host.cpp.

struct Packed {
    EvoPacked p{};
    Tensor q, k, v, offsets, key_offsets;   // as the kernels read them
    int64_t D = 0;                          // the head dim; p.D in 16 bits: with the zeros behind it

    static constexpr int64_t most_apart = 1 << 23;   // values from one row to the next, in 16 bits
    // [T, heads, D] with the strides, the alignment and the columns that the kernels take
    static Tensor ready(const Tensor &t, int64_t Dp) {
        const bool wide = t.scalar_type() == at::kFloat;
        // (a copy: row by row, or head by head where rows of all heads would lie too far apart)
        const bool by_heads = !wide && t.size(1) * Dp >= most_apart;
        if (t.size(2) != Dp) return by_heads ? at::constant_pad_nd(t.transpose(0, 1).contiguous(), {0, Dp - t.size(2)}).transpose(0, 1) : at::constant_pad_nd(t, {0, Dp - t.size(2)});
        if (!t.numel()) return t;
        int64_t st, sh;
        stride(t, st, sh);
        // (rows of 16 bits lie apart, so that what is beyond a sequence is out of range)
        const bool taken = (t.stride(2) == 1 || t.size(2) == 1) && (wide || (st >= Dp && st % 8 == 0 && sh % 8 == 0 && st < most_apart && (uintptr_t)t.data_ptr() % 16 == 0));
        return taken ? t : by_heads ? t.transpose(0, 1).clone(at::MemoryFormat::Contiguous).transpose(0, 1) : t.clone(at::MemoryFormat::Contiguous);
    }
    // [T, heads, Dp], dense, whatever there is between two rows
    static Tensor dense(const Tensor &t, int64_t Dp) {
        if (t.size(2) != Dp) return at::constant_pad_nd(t.contiguous(), {0, Dp - t.size(2)});
        return t.is_contiguous() && (uintptr_t)ptr_or_null(t) % 16 == 0 ? t : t.clone(at::MemoryFormat::Contiguous);
    }
    static void stride(const Tensor &t, int64_t &st, int64_t &sh) {
        st = t.size(0) > 1 ? t.stride(0) : t.size(2);
        sh = t.size(1) > 1 ? t.stride(1) : 0;
    }
    // What is wrong with the call, or nothing; then the parameter block is filled.
    const char *take(const Tensor &q_, const Tensor &k_, const Tensor &v_, const Tensor &offsets_, const OptTensor &key_offsets_, bool causal, std::optional<double> scale) {
        const bool own = key_offsets_ && key_offsets_->defined();
        const Tensor &ko = own ? *key_offsets_ : offsets_;
        for (const Tensor *t : {&k_, &v_, &offsets_, &ko})
            if (t->device() != q_.device()) return "all tensors must live on one device";
        if (q_.dim() != 3 || k_.dim() != 3) return "queries must be [Tq, H, D], keys and values [Tk, Hk, D]";
        if (!v_.sizes().equals(k_.sizes())) return "values must have the keys' shape";
        if (evo_dtype(q_.scalar_type()) == EVO_NONE) return "queries must be bf16, fp16 or fp32";
        if (k_.scalar_type() != q_.scalar_type() || v_.scalar_type() != q_.scalar_type()) return "keys and values must have the queries' dtype";
        D = q_.size(2);
        if (k_.size(2) != D) return "keys must have the queries' head dim";
        if (D < 1 || D > 128) return "the head dim must be 1 to 128";
        const int64_t H = q_.size(1), Hk = k_.size(1);
        if (H < 1 || Hk < 1 || H % Hk) return "the number of query heads must be a multiple of the number of key heads";
        for (const Tensor *t : {&offsets_, &ko}) {
            if (t->scalar_type() != at::kInt && t->scalar_type() != at::kLong) return "offsets must be int32 or int64";
            if (t->dim() != 1 || t->size(0) < 1) return "offsets must be [sequences + 1]";
        }
        if (ko.size(0) != offsets_.size(0)) return "key_offsets must be as long as offsets";
        if (!own && k_.size(0) != q_.size(0)) return "keys that are not as many as queries need key_offsets";
        const double s = scale ? *scale : 1.0 / std::sqrt((double)D);
        if (!((float)s >= 0x1p-64f && (float)s <= 0x1p64f)) return "scale must be a positive number, 2^-64 to 2^64";
        const int64_t Tq = q_.size(0), Tk = k_.size(0), most = INT32_MAX / 2;
        if (Tq > most || Tk > most || offsets_.size(0) > INT32_MAX / 4 || H > 1 << 20) return "2^30 rows, 2^29 sequences or more than 2^20 heads are too many";
        p.n = (int32_t)(offsets_.size(0) - 1);
        p.H = (int32_t)H;
        p.Hk = (int32_t)Hk;
        p.D = (int32_t)(q_.scalar_type() == at::kFloat ? D : (D + 7) / 8 * 8);
        p.dtype = evo_dtype(q_.scalar_type());
        p.causal = causal;
        p.scale = (float)s;
        p.Tq = Tq;
        p.Tk = Tk;
        const bool wide = offsets_.scalar_type() != ko.scalar_type();
        offsets = wide ? offsets_.to(at::kLong) : offsets_;
        key_offsets = !own ? offsets : wide ? ko.to(at::kLong) : ko;
        q = q_;
        k = k_;
        v = v_;
        return nullptr;
    }
    void point() {
        q = ready(q, p.D);
        k = ready(k, p.D);
        v = ready(v, p.D);
        offsets = offsets.contiguous();
        key_offsets = key_offsets.contiguous();
        stride(q, p.q_stride_t, p.q_stride_h);
        stride(k, p.k_stride_t, p.k_stride_h);
        stride(v, p.v_stride_t, p.v_stride_h);
        p.q = ptr_or_null(q);
        p.k = ptr_or_null(k);
        p.v = ptr_or_null(v);
        p.offset_bytes = offsets.scalar_type() == at::kInt ? 4 : 8;
        p.offsets = offsets.data_ptr();
        p.key_offsets = key_offsets.data_ptr();
    }
    Tensor cut(const Tensor &t) const { return t.size(2) == D ? t : t.narrow(2, 0, D).contiguous(); }
    // o, and, if they are wanted, lse and (16 bits) what rounding left of o
    Tensor forward(Tensor *lse, Tensor *low) {
        c10::DeviceGuard on(q.device());
        point();
        Tensor o = at::empty({p.Tq, p.H, p.D}, q.options()), ws;
        if (lse) *lse = at::empty({p.H, p.Tq}, q.options().dtype(at::kFloat));
        if (low) *low = at::empty(p.dtype == EVO_F32 ? at::IntArrayRef({0, p.H, p.D}) : at::IntArrayRef({p.Tq, p.H, p.D}), q.options());
        if (p.Tq) {
            p.o = o.data_ptr();
            p.lse = lse ? (float *)lse->data_ptr() : nullptr;
            p.o_low = low && low->numel() ? low->data_ptr() : nullptr;
            if (const size_t bytes = evoattn_packed_fwd_workspace_bytes(&p)) {
                ws = scratch(bytes, q);
                p.workspace = ws.data_ptr();
                p.workspace_bytes = bytes;
            }
            check(evoattn_packed_fwd(&p, stream_of(q)), "evoattn_packed_fwd");
        }
        return cut(o);
    }
    void backward(const Tensor &dout_, const Tensor &o_, const Tensor &lse_, const Tensor &low_, bool need_kv, Tensor &dq, Tensor &dk, Tensor &dv) {
        c10::DeviceGuard on(q.device());
        point();
        const Tensor dout = ready(dout_, p.D), lse = lse_.contiguous(), low = low_.contiguous();
        const Tensor o = dense(o_, p.D);
        dq = at::empty({p.Tq, p.H, p.D}, q.options());
        if (need_kv) {
            dk = at::empty({p.Tk, p.Hk, p.D}, q.options());
            dv = at::empty({p.Tk, p.Hk, p.D}, q.options());
        }
        if (p.Tq || (need_kv && p.Tk)) {
            stride(dout, p.dout_stride_t, p.dout_stride_h);
            p.dout = ptr_or_null(dout);
            p.o = const_cast<void *>(ptr_or_null(o));
            p.lse = (float *)const_cast<void *>(ptr_or_null(lse));
            p.o_low = low.numel() ? low.data_ptr() : nullptr;
            p.dq = const_cast<void *>(ptr_or_null(dq));
            p.dk = const_cast<void *>(ptr_or_null(dk));
            p.dv = const_cast<void *>(ptr_or_null(dv));
            const Tensor ws = scratch(evoattn_packed_bwd_workspace_bytes(&p), q);
            p.workspace = ws.data_ptr();
            p.workspace_bytes = (size_t)ws.numel();
            check(evoattn_packed_bwd(&p, stream_of(q)), "evoattn_packed_bwd");
        }
        dq = cut(dq);
        if (need_kv) {
            dk = cut(dk);
            dv = cut(dv);
        }
    }
};

struct PackedNode : SavingNode {
    EvoPacked p{};
    int64_t D = 0;
    std::string name() const override { return "PackedAttentionBackward"; }
    // saved: queries, keys, values, offsets, key offsets, lse, the output, what rounding left of it; results: queries, keys, values
    variable_list apply(variable_list &&grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        const bool rec = at::GradMode::is_enabled();
        variable_list out(3);
        if (!grads[0].defined()) return out;
        {
            const variable_list t = unpacked(6);
            at::AutoDispatchBelowADInplaceOrView guard;
            Packed c;
            c.p = p;
            c.D = D;
            c.q = t[0];
            c.k = t[1];
            c.v = t[2];
            c.offsets = t[3];
            c.key_offsets = t[4];
            const Tensor dout = grads[0].scalar_type() == c.q.scalar_type() ? grads[0] : grads[0].to(c.q.scalar_type());
            c.backward(dout, t[6], t[5], t[7], task_should_compute_output(1) || task_should_compute_output(2), out[0], out[1], out[2]);
            for (int i = 0; i < 3; ++i)
                if (!task_should_compute_output(i)) out[i] = Tensor();
        }
        return once_differentiable(std::move(out), rec);
    }
};

// None for a call that the node does not stand for or that is wrong: the caller in Python goes its own way and words the error.
OptTensor packed_attention(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &offsets, const OptTensor &key_offsets, bool causal, std::optional<double> scale) {
    if (!plain_modes()) return std::nullopt;
    for (const Tensor *t : {&q, &k, &v, &offsets})
        if (!t->defined() || !plain(*t) || !t->is_cuda()) return std::nullopt;
    if (key_offsets && key_offsets->defined() && !plain(*key_offsets)) return std::nullopt;
    const bool wanted = SavingNode::wanted(q, k, v);
    Packed c;
    Tensor o, lse, low;
    {
        at::AutoDispatchBelowADInplaceOrView guard;
        if (c.take(q, k, v, offsets, key_offsets, causal, scale)) return std::nullopt;
        o = c.forward(wanted ? &lse : nullptr, wanted ? &low : nullptr);
    }
    if (wanted) {
        auto node = make_node<PackedNode>(q, k, v);
        node->p = c.p;
        node->D = c.D;
        torch::autograd::set_history(o, node);
        for (const Tensor *t : {&q, &k, &v}) node->save(*t);
        node->save(c.offsets);
        node->save(c.key_offsets);
        node->save(lse);
        node->save(o, true);
        node->save(low);
    }
    return o;
}

// The same launches without a node, for the registered operators.
std::tuple<Tensor, Tensor, Tensor> packed_forward(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &offsets, const OptTensor &key_offsets, bool causal,
                                         std::optional<double> scale) {
    Packed c;
    const char *wrong = c.take(q, k, v, offsets, key_offsets, causal, scale);
    TORCH_CHECK_VALUE(!wrong, wrong);
    TORCH_CHECK(q.is_cuda(), "packed attention runs on the GPU only");
    TORCH_CHECK_NOT_IMPLEMENTED(!dual(q) && !dual(k) && !dual(v), "packed_attention has no formula for forward mode differentiation");
    Tensor lse, low, o = c.forward(&lse, &low);
    return {o, lse, low};
}
std::tuple<Tensor, Tensor, Tensor> packed_backward(const Tensor &dout, const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &offsets, const OptTensor &key_offsets,
                                                   const Tensor &o, const Tensor &lse, const Tensor &low, bool causal, std::optional<double> scale) {
    Packed c;
    const char *wrong = c.take(q, k, v, offsets, key_offsets, causal, scale);
    TORCH_CHECK_VALUE(!wrong, wrong);
    TORCH_CHECK(q.is_cuda(), "packed attention runs on the GPU only");
    TORCH_CHECK_VALUE(dout.device() == q.device() && dout.sizes().equals(q.sizes()) && dout.scalar_type() == q.scalar_type() && o.device() == q.device() &&
                          o.sizes().equals(q.sizes()) && o.scalar_type() == q.scalar_type() && lse.device() == q.device() && lse.scalar_type() == at::kFloat &&
                          lse.dim() == 2 && lse.size(0) == q.size(1) && lse.size(1) == q.size(0) && low.device() == q.device() && low.scalar_type() == q.scalar_type() &&
                          low.dim() == 3 && low.size(0) == (c.p.dtype == EVO_F32 ? 0 : q.size(0)) && low.size(1) == q.size(1) && low.size(2) == c.p.D,
                      "the output, its gradient, lse and what rounding left must be as the forward gave them");
    Tensor dq, dk, dv;
    c.backward(dout, o, lse, low, true, dq, dk, dv);
    return {dq, dk, dv};
}
std::optional<std::string> packed_wrong(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &offsets, const OptTensor &key_offsets, bool causal,
                                        std::optional<double> scale) {
    Packed c;
    const char *wrong = c.take(q, k, v, offsets, key_offsets, causal, scale);
    return wrong ? std::optional<std::string>(wrong) : std::nullopt;
}
