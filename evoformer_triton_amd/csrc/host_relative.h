// The learned relative position bias (csrc/relative_bias.hip): part of host.cpp.

// A call's operands as the kernels read them.
struct RelativeBias {
    EvoRelativeBias p{};
    Tensor table, lut, pos_q, pos_k, chain_q, chain_k, pair;
    at::ScalarType dtype = at::kFloat;

    // Positions of the queries and of the keys, then chains, [B or 1, N] or [N], in one integer type and each side's two laid out alike.  What need not be copied is the caller's
    // tensor itself, not a view: one made here would have a version of its own, and what is saved for the backward could be changed in place unseen.
    static Tensor indices(const Tensor &t, at::ScalarType type, int64_t batches) {
        const bool fits = t.dim() == 1 ? batches == 1 : t.size(0) == batches;
        return (fits ? t : t.expand({batches, t.size(-1)})).to(type).contiguous();
    }
    // What is wrong with the call, or nothing; then the parameter block is filled.
    const char *take(const Tensor &table_, const Tensor &lut_, const Tensor &q, const Tensor &k, const OptTensor &cq, const OptTensor &ck, const OptTensor &bias,
                     std::optional<at::ScalarType> type) {
        const bool chains = cq && cq->defined(), with = bias && bias->defined();
        const Tensor *all[] = {&table_, &lut_, &q, &k, chains ? &*cq : nullptr, ck && ck->defined() ? &*ck : nullptr, with ? &*bias : nullptr};
        for (const Tensor *t : all)
            if (t && t->device() != table_.device()) return "all tensors must live on one device";
        if (table_.dim() != 2 || table_.size(0) < 1 || evo_dtype(table_.scalar_type()) == EVO_NONE)
            return "the table must be [buckets, heads] in bf16, fp16 or fp32";
        if (table_.size(0) > 256) return "the table may have at most 256 rows";
        if (lut_.dim() != 1 || lut_.scalar_type() != at::kByte || lut_.size(0) % 2 == 0 || lut_.size(0) > 2 * 4096 + 1)
            return "the buckets must be a uint8 tensor [2 R + 1] with R at most 4096, as relative_buckets() makes it";
        if (chains != (ck && ck->defined())) return "chains must be given for queries and keys or for neither";
        int64_t B = 1;
        for (int i = 2; i < 6; ++i) {
            if (!all[i]) continue;
            const Tensor &t = *all[i];
            if (!at::isIntegralType(t.scalar_type(), false)) return "positions and chains must be whole numbers";
            // (chains are names, and stay different ones as int64)
            if (i < 4 && t.scalar_type() == at::kUInt64) return "positions must be whole numbers that int64 holds, not uint64";
            if (t.dim() != 1 && t.dim() != 2) return "positions and chains must be [N] or [B, N]";
            if (t.dim() == 2 && t.size(0) != 1) {
                if (B != 1 && t.size(0) != B) return "the batches of positions, chains and pair bias do not agree";
                B = t.size(0);
            }
        }
        const int64_t Nq = q.size(-1), Nk = k.size(-1), H = table_.size(1);
        if (chains && (cq->size(-1) != Nq || ck->size(-1) != Nk)) return "chains must be as long as positions";
        if (with) {
            const Tensor &t = *bias;
            if (t.dim() != 5 || t.size(1) != 1 || t.size(2) != H || t.size(3) != Nq || t.size(4) != Nk) return "the pair bias must be [B,1,H,Nq,Nk] (B may be 1)";
            if (t.size(0) != 1) {
                if (B != 1 && t.size(0) != B) return "the batches of positions, chains and pair bias do not agree";
                B = t.size(0);
            }
            if (evo_dtype(t.scalar_type()) == EVO_NONE) return "the pair bias must be bf16, fp16 or fp32";
        }
        dtype = type ? *type : with ? bias->scalar_type() : table_.scalar_type();
        if (evo_dtype(dtype) == EVO_NONE) return "the result can be bf16, fp16 or fp32";
        if (with && bias->scalar_type() != dtype) return "the pair bias must have the result's dtype";
        constexpr int64_t most = INT32_MAX - 1024;
        if (B > INT32_MAX || H > INT32_MAX || Nq > most || Nk > most) return "2^31 batches or heads, or queries or keys within 1024 of it, are too many";

        table = table_.contiguous();
        lut = lut_.contiguous();
        const bool small = q.scalar_type() == at::kInt && k.scalar_type() == at::kInt && (!chains || (cq->scalar_type() == at::kInt && ck->scalar_type() == at::kInt));
        const auto index = small ? at::kInt : at::kLong;
        auto batches = [](const Tensor &a, const OptTensor &c, bool on) {
            const int64_t n = a.dim() == 2 ? a.size(0) : 1;
            return on && c->dim() == 2 ? std::max(n, c->size(0)) : n;
        };
        const int64_t bq = batches(q, cq, chains), bk = batches(k, ck, chains);
        pos_q = indices(q, index, bq);
        pos_k = indices(k, index, bk);
        if (chains) {
            chain_q = indices(*cq, index, bq);
            chain_k = indices(*ck, index, bk);
        }
        if (with) pair = bias->stride(4) == 1 || Nk <= 1 ? *bias : bias->contiguous();
        p.B = (int32_t)B;
        p.H = (int32_t)H;
        p.Nq = (int32_t)Nq;
        p.Nk = (int32_t)Nk;
        p.rows = (int32_t)table.size(0);
        p.reach = (int32_t)(lut.size(0) / 2);
        p.dtype = evo_dtype(dtype);
        p.table_dtype = evo_dtype(table.scalar_type());
        p.pos_bytes = small ? 4 : 8;
        p.pos_q_stride_b = bq > 1 ? Nq : 0;
        p.pos_k_stride_b = bk > 1 ? Nk : 0;
        point();
        return nullptr;
    }
    void point() {
        p.table = ptr_or_null(table);
        p.lut = lut.data_ptr();
        p.pos_q = pos_q.data_ptr();
        p.pos_k = pos_k.data_ptr();
        p.chain_q = ptr_or_null(chain_q);
        p.chain_k = ptr_or_null(chain_k);
        if (pair.defined()) {
            p.pair = pair.data_ptr();
            p.pair_stride_b = pair.size(0) > 1 ? pair.stride(0) : 0;
            p.pair_stride_h = pair.stride(2);
            p.pair_stride_row = pair.stride(3);
        }
    }
    bool empty() const { return p.H == 0 || p.Nq == 0 || p.Nk == 0 || p.B == 0; }
    Tensor forward() {
        c10::DeviceGuard on(table.device());
        Tensor out = at::empty({p.B, 1, p.H, p.Nq, p.Nk}, table.options().dtype(dtype));
        if (empty()) return out;
        p.out = out.data_ptr();
        check(evoattn_relative_bias_fwd(&p, stream_of(table)), "evoattn_relative_bias_fwd");
        return out;
    }
    // The gradient of the table, and that of a pair bias that the batches share.  `dout` [B,1,H,Nq,Nk] in the result's type, dense.
    void backward(const Tensor &dout, bool need_table, bool need_pair, Tensor &dtable, Tensor &dpair) {
        c10::DeviceGuard on(dout.device());
        const auto like = dout.options();
        if (empty()) {
            if (need_table) dtable = at::zeros({p.rows, p.H}, like.dtype(table_type));
            if (need_pair) dpair = at::zeros({1, 1, p.H, p.Nq, p.Nk}, like);
            return;
        }
        Tensor ws;
        p.dout = dout.data_ptr();
        if (need_table) {
            dtable = at::empty({p.rows, p.H}, like.dtype(table_type));
            ws = scratch(evoattn_relative_bias_bwd_workspace_bytes(&p), dout);
            p.dtable = dtable.data_ptr();
            p.workspace = ws.data_ptr();
            p.workspace_bytes = (size_t)ws.numel();
        }
        if (need_pair) {
            dpair = at::empty({1, 1, p.H, p.Nq, p.Nk}, like);
            p.dpair = dpair.data_ptr();
        }
        check(evoattn_relative_bias_bwd(&p, stream_of(dout)), "evoattn_relative_bias_bwd");
    }
    at::ScalarType table_type = at::kFloat;
};

struct RelativeBiasNode : SavingNode {
    EvoRelativeBias p{};
    at::ScalarType table_type = at::kFloat, dtype = at::kFloat;
    bool shared_pair = false;
    std::string name() const override { return "RelativePositionBiasBackward"; }
    // saved: the buckets, positions and chains; results: the table, the pair bias
    variable_list apply(variable_list &&grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        const bool rec = at::GradMode::is_enabled();
        variable_list out(2);
        if (!grads[0].defined()) return out;
        {
            const bool need_table = task_should_compute_output(0), need_pair = task_should_compute_output(1), sums = need_table || (need_pair && shared_pair);
            const variable_list t = sums ? unpacked() : variable_list();
            at::AutoDispatchBelowADInplaceOrView guard;
            Tensor d = grads[0].scalar_type() == dtype ? grads[0] : grads[0].to(dtype), dpair;
            if (sums) {
                RelativeBias r;
                r.p = p;
                r.table_type = table_type;
                r.lut = t[0].contiguous();
                r.pos_q = t[1].contiguous();
                r.pos_k = t[2].contiguous();
                r.chain_q = t[3];
                r.chain_k = t[4];
                if (r.chain_q.defined()) {
                    r.chain_q = r.chain_q.contiguous();
                    r.chain_k = r.chain_k.contiguous();
                }
                r.point();
                r.backward(d.contiguous(), need_table, need_pair && shared_pair, out[0], dpair);
            }
            if (need_pair) out[1] = shared_pair ? dpair : d;
        }
        return once_differentiable(std::move(out), rec);
    }
};

// None for a call that the node does not stand for or that is wrong: the caller in Python goes its own way and words the error.
OptTensor relative_bias(const Tensor &table, const Tensor &lut, const Tensor &q, const Tensor &k, const OptTensor &cq, const OptTensor &ck, const OptTensor &bias,
                        std::optional<at::ScalarType> dtype) {
    if (!plain_modes()) return std::nullopt;
    for (const Tensor *t : {&table, &lut, &q, &k})
        if (!t->defined() || !plain(*t) || !t->is_cuda()) return std::nullopt;
    for (const OptTensor *t : {&cq, &ck, &bias})
        if (*t && (*t)->defined() && !plain(**t)) return std::nullopt;
    const Tensor bias0 = bias ? *bias : Tensor();
    RelativeBias r;
    Tensor out;
    {
        at::AutoDispatchBelowADInplaceOrView guard;
        if (r.take(table, lut, q, k, cq, ck, bias, dtype)) return std::nullopt;
        out = r.forward();
    }
    if (SavingNode::wanted(table, bias0)) {
        auto node = make_node<RelativeBiasNode>(table, bias0);
        node->p = r.p;
        node->table_type = table.scalar_type();
        node->dtype = r.dtype;
        node->shared_pair = r.pair.defined() && r.pair.size(0) == 1 && r.p.B != 1;
        torch::autograd::set_history(out, node);
        for (const Tensor *t : {&r.lut, &r.pos_q, &r.pos_k, &r.chain_q, &r.chain_k}) node->save(*t);
    }
    return out;
}

// The same launches without a node, for the registered operators.
Tensor relative_bias_forward(const Tensor &table, const Tensor &lut, const Tensor &q, const Tensor &k, const OptTensor &cq, const OptTensor &ck,
                             const OptTensor &bias, std::optional<at::ScalarType> dtype) {
    RelativeBias r;
    const char *wrong = r.take(table, lut, q, k, cq, ck, bias, dtype);
    TORCH_CHECK_VALUE(!wrong, wrong);
    TORCH_CHECK(table.is_cuda(), "the relative position bias runs on the GPU only");
    TORCH_CHECK_NOT_IMPLEMENTED(!dual(table) && !(bias && dual(*bias)), "relative_position_bias has no formula for forward mode differentiation");
    return r.forward();
}
std::pair<Tensor, Tensor> relative_bias_backward(const Tensor &dout, const Tensor &table, const Tensor &lut, const Tensor &q, const Tensor &k, const OptTensor &cq,
                                                 const OptTensor &ck, const OptTensor &bias, bool need_table, bool need_pair) {
    RelativeBias r;
    const char *wrong = r.take(table, lut, q, k, cq, ck, bias, dout.scalar_type());
    TORCH_CHECK_VALUE(!wrong, wrong);
    TORCH_CHECK(table.is_cuda(), "the relative position bias runs on the GPU only");
    r.table_type = table.scalar_type();
    TORCH_CHECK_VALUE(dout.device() == table.device() && dout.dim() == 5 && dout.size(0) == r.p.B && dout.size(1) == 1 && dout.size(2) == r.p.H &&
                          dout.size(3) == r.p.Nq && dout.size(4) == r.p.Nk, "the gradient must have the result's shape and device");
    const bool shared = r.pair.defined() && r.pair.size(0) == 1 && r.p.B != 1;
    Tensor dtable, dpair;
    if (need_table || (need_pair && shared)) r.backward(dout.contiguous(), need_table, need_pair && shared, dtable, dpair);
    if (need_pair && !shared) dpair = dout.clone(at::MemoryFormat::Contiguous);   // (as the tracer has been told, not with dout's strides)
    const Tensor none = at::empty({0}, dout.options());
    return {dtable.defined() ? dtable : none, dpair.defined() ? dpair : at::empty({0}, dout.options())};
}
std::optional<std::string> relative_bias_wrong(const Tensor &table, const Tensor &lut, const Tensor &q, const Tensor &k, const OptTensor &cq, const OptTensor &ck,
                                               const OptTensor &bias, std::optional<at::ScalarType> dtype) {
    RelativeBias r;
    const char *wrong = r.take(table, lut, q, k, cq, ck, bias, dtype);
    return wrong ? std::optional<std::string>(wrong) : std::nullopt;
}
