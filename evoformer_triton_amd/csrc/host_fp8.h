// Linear layers in 8 bits (csrc/fp8.hip): part of host.cpp.

// A matrix [rows, k] rounded along its rows: values [rows, k up to the next 128], scales [rows, blocks up to the next 4], in one piece of memory (an
// allocation costs the host a microsecond) or a caller's two.
struct Rounded {
    Tensor hold;
    void *q = nullptr, *s = nullptr;
    int64_t rows = 0, k = 0;
    Rounded() = default;
    Rounded(const Tensor &values, const Tensor &scales, int64_t k_) : q(values.data_ptr()), s(scales.data_ptr()), rows(values.size(0)), k(k_) {}
    Rounded(const Tensor &hold_, int64_t rows_, int64_t k_) : hold(hold_), q(hold_.data_ptr()), s((char *)hold_.data_ptr() + rows_ * pitch(k_)), rows(rows_), k(k_) {}
    Rounded(int64_t rows_, int64_t k_, const Tensor &like) : Rounded(at::empty({rows_ * (pitch(k_) + scale_pitch(k_))}, like.options().dtype(at::kByte)), rows_, k_) {}
    static int64_t pitch(int64_t k) { return (k + 127) / 128 * 128; }
    static int64_t scale_pitch(int64_t k) { return (k + 511) / 512 * 4; }
};

// x [rows, cols] as rows of a matrix that the kernels read: elements of a row side by side.
Tensor f8_rows(const Tensor &x) {
    const Tensor r = as_rows(x);
    return r.stride(1) == 1 && r.stride(0) >= r.size(1) ? r : r.contiguous();
}

int64_t f8_apart(const Tensor &x) { return x.size(0) == 1 ? std::max(x.stride(0), x.size(1)) : x.stride(0); }   // (one row's stride may be anything)

// x rounded along its rows and its columns, as far as asked for, and the column sums of its blocks of rows.
EvoFp8Rounding f8_rounded(const Tensor &x, Rounded *along_rows, Rounded *along_cols, Tensor *sums) {
    EvoFp8Rounding r{};
    r.x = x.data_ptr();
    r.ldx = f8_apart(x);
    r.rows = x.size(0);
    r.cols = x.size(1);
    if (along_rows) {
        *along_rows = Rounded(r.rows, r.cols, x);
        r.q = along_rows->q;
        r.scales = along_rows->s;
    }
    if (along_cols) {
        *along_cols = Rounded(r.cols, r.rows, x);
        r.qt = along_cols->q;
        r.scales_t = along_cols->s;
    }
    if (sums) {
        *sums = at::empty({(r.rows + 127) / 128, r.cols}, x.options().dtype(at::kFloat));
        r.sums = (float *)sums->data_ptr();
    }
    return r;
}
void f8_quantize(const Tensor &x, Rounded *along_rows, Rounded *along_cols, Tensor *sums) {
    const EvoFp8Rounding r = f8_rounded(x, along_rows, along_cols, sums);
    check(evoattn_fp8_quantize(r.x, r.ldx, r.q, r.scales, r.qt, r.scales_t, r.sums, r.rows, r.cols, evo_dtype(x.scalar_type()), stream_of(x)), "evoattn_fp8_quantize");
}
// a weight both ways or along its rows, and x as far as asked for
void f8_quantize_both(const Tensor &w, Rounded *w_rows, Rounded *w_cols, const Tensor &x, Rounded *x_rows, Rounded *x_cols) {
    if ((!x_rows && !x_cols) || w.scalar_type() != x.scalar_type()) {
        f8_quantize(w, w_rows, w_cols, nullptr);
        if (x_rows || x_cols) f8_quantize(x, x_rows, x_cols, nullptr);
        return;
    }
    const EvoFp8Rounding a = f8_rounded(w, w_rows, w_cols, nullptr), b = f8_rounded(x, x_rows, x_cols, nullptr);
    check(evoattn_fp8_quantize_two(&a, &b, evo_dtype(x.scalar_type()), stream_of(x)), "evoattn_fp8_quantize_two");
}

EvoFp8Matmul f8_product(int64_t rows, const Rounded &b, const Tensor &bias, const Tensor &out) {
    EvoFp8Matmul p{};
    p.m = rows;
    p.n = b.rows;
    p.k = b.k;
    p.ldo = b.rows;
    p.dtype = evo_dtype(out.scalar_type());
    p.b = b.q;
    p.scales_b = b.s;
    if (bias.defined()) {
        p.bias = bias.data_ptr();
        p.bias_dtype = evo_dtype(bias.scalar_type());
    }
    p.out = out.data_ptr();
    return p;
}
// a b^T (+ bias), [a.rows, b.rows], on `like`'s device; and the column sums' totals to `totals`, if given
Tensor f8_matmul(const Rounded &a, const Rounded &b, const Tensor &bias, at::ScalarType dtype, const Tensor &like, const Tensor &sums = Tensor(),
                 const Tensor &totals = Tensor()) {
    Tensor out = at::empty({a.rows, b.rows}, like.options().dtype(dtype)), ws;
    EvoFp8Matmul p = f8_product(a.rows, b, bias, out);
    p.a = a.q;
    p.scales_a = a.s;
    if (const size_t bytes = evoattn_fp8_matmul_workspace_bytes(&p)) {
        ws = scratch(bytes, like);
        p.workspace = ws.data_ptr();
        p.workspace_bytes = (size_t)ws.numel();
    }
    if (totals.defined())
        check(evoattn_fp8_matmul_sums(&p, (const float *)sums.data_ptr(), b.k, totals.data_ptr(), evo_dtype(totals.scalar_type()), stream_of(like)),
              "evoattn_fp8_matmul_sums");
    else check(evoattn_fp8_matmul(&p, stream_of(like)), "evoattn_fp8_matmul");
    return out;
}

// whether x [rows, k] times a matrix of n rows is rounded on the way
bool f8_rounds(const Tensor &x, int64_t n) {
    EvoFp8Matmul p{};
    p.m = x.size(0);
    p.n = n;
    p.k = x.size(1);
    p.dtype = evo_dtype(x.scalar_type());
    return evoattn_fp8_matmul_rounds(&p) != 0;
}
// x b^T (+ bias), x rounded on the way
Tensor f8_rounding(const Tensor &x, const Rounded &b, const Tensor &bias) {
    Tensor out = at::empty({x.size(0), b.rows}, x.options()), ws;
    EvoFp8Matmul p = f8_product(x.size(0), b, bias, out);
    if (const size_t bytes = evoattn_fp8_matmul_rounding_workspace_bytes(&p)) {
        ws = scratch(bytes, x);
        p.workspace = ws.data_ptr();
        p.workspace_bytes = (size_t)ws.numel();
    }
    check(evoattn_fp8_matmul_rounding(&p, x.data_ptr(), f8_apart(x), stream_of(x)), "evoattn_fp8_matmul_rounding");
    return out;
}
Tensor f8_times(const Tensor &x, const Rounded &b, const Tensor &bias) {
    if (f8_rounds(x, b.rows)) return f8_rounding(x, b, bias);
    Rounded a;
    f8_quantize(x, &a, nullptr, nullptr);
    return f8_matmul(a, b, bias, x.scalar_type(), x);
}

constexpr int64_t kF8Most = 1 << 26;
const char *f8_wrong(const Tensor &x, int64_t n, int64_t k, const c10::Device &device, const OptTensor &bias) {
    if (evo_dtype(x.scalar_type()) == EVO_NONE || x.dim() < 1) return "the input must be [..., k] in bf16, fp16 or fp32";
    if (x.size(-1) != k) return "the input's last dimension must be the weight's columns";
    if (x.device() != device || (bias && bias->defined() && bias->device() != device)) return "all tensors must live on one device";
    if (bias && bias->defined() && (bias->dim() != 1 || bias->size(0) != n || evo_dtype(bias->scalar_type()) == EVO_NONE))
        return "the bias must be [n] in bf16, fp16 or fp32";
    // (each of them is contracted in one of the three products)
    if (n > kF8Most || k > kF8Most) return "the weight has more than 2^26 rows or columns";
    if (k > 0 && x.numel() / k > kF8Most) return "the input has more than 2^26 rows";
    return nullptr;
}
const char *f8_linear_wrong(const Tensor &x, const Tensor &w, const OptTensor &bias) {
    if (w.dim() != 2 || evo_dtype(w.scalar_type()) == EVO_NONE) return "the weight must be [n, k] in bf16, fp16 or fp32";
    return f8_wrong(x, w.size(0), w.size(1), w.device(), bias);
}
const char *f8_held_wrong(const Tensor &x, const Tensor &q, const Tensor &s, int64_t k, const OptTensor &bias) {
    // (other types of a byte stand for other numbers)
    if ((q.scalar_type() != at::kFloat8_e4m3fn && q.scalar_type() != at::kByte) || (s.scalar_type() != at::kFloat8_e8m0fnu && s.scalar_type() != at::kByte))
        return "a weight in 8 bits has values in float8_e4m3fn and scales in float8_e8m0fnu, or their bytes (uint8)";
    if (q.dim() != 2 || s.dim() != 2 || k < 0 || q.size(1) != Rounded::pitch(k) ||
        s.size(1) != Rounded::scale_pitch(k) || s.size(0) != q.size(0) || !q.is_contiguous() || !s.is_contiguous() || s.device() != q.device())
        return "a weight in 8 bits is values [n, k up to the next 128] and scales [n, k / 128 up to the next 4], both dense, a byte each";
    if (q.numel() && ((uintptr_t)q.data_ptr() % 16 || (uintptr_t)s.data_ptr() % 4)) return "a weight in 8 bits must start on a 16-byte boundary, its scales on one of 4";
    return f8_wrong(x, q.size(0), k, q.device(), bias);
}

std::vector<int64_t> f8_shape(const Tensor &x, int64_t n) {
    auto shape = x.sizes().vec();
    shape.back() = n;
    return shape;
}

// What the backward needs of x and the weight.
struct F8Saved {
    Rounded xt, wt;   // x^T rounded along the rows of x, w^T along those of w
};
Tensor f8_forward(const Tensor &x, const Tensor &w, const Tensor &bias, bool need_x, bool need_w, F8Saved *saved) {
    c10::DeviceGuard on(x.device());
    const int64_t n = w.size(0), k = w.size(1);
    const auto shape = f8_shape(x, n);
    if (x.numel() == 0 || n == 0) {
        Tensor y = at::zeros(shape, x.options());
        return k == 0 && bias.defined() ? y.add_(bias) : y;
    }
    const Tensor x2 = f8_rows(x), w2 = f8_rows(w), b = bias.defined() ? bias.contiguous() : bias;
    Rounded xr, wr;
    const bool rounds = f8_rounds(x2, n);
    f8_quantize_both(w2, &wr, need_x ? &saved->wt : nullptr, x2, rounds ? nullptr : &xr, need_w ? &saved->xt : nullptr);
    return (rounds ? f8_rounding(x2, wr, b) : f8_matmul(xr, wr, b, x.scalar_type(), x2)).view(shape);
}
// dx, dw, db from dy [rows, n]
void f8_backward(const Tensor &dy, const F8Saved &saved, bool need_x, bool need_w, bool need_b, at::ScalarType wtype, at::ScalarType btype, Tensor &dx, Tensor &dw,
                 Tensor &db) {
    c10::DeviceGuard on(dy.device());
    Rounded along_rows, along_cols;
    Tensor sums;
    const bool cols = need_w || need_b;
    f8_quantize(dy, need_x ? &along_rows : nullptr, cols ? &along_cols : nullptr, need_b ? &sums : nullptr);
    if (need_x) dx = f8_matmul(along_rows, saved.wt, Tensor(), dy.scalar_type(), dy);
    if (need_b) db = at::empty({dy.size(1)}, dy.options().dtype(btype));
    if (need_w) {
        dw = f8_matmul(along_cols, saved.xt, Tensor(), wtype, dy, sums, db);
    } else if (need_b) {
        check(evoattn_fp8_column_sums((const float *)sums.data_ptr(), db.data_ptr(), dy.size(0), dy.size(1), evo_dtype(btype), stream_of(dy)),
              "evoattn_fp8_column_sums");
    }
}

struct Fp8LinearNode : SavingNode {
    std::vector<int64_t> x_shape;
    int64_t n = 0, k = 0;
    at::ScalarType x_type = at::kFloat, w_type = at::kFloat, b_type = at::kFloat;
    bool has_bias = false;
    std::string name() const override { return "Fp8LinearBackward"; }
    // saved: x^T and w^T rounded; results: x, weight, bias
    variable_list apply(variable_list &&grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        const bool rec = at::GradMode::is_enabled();
        variable_list out(3);
        if (!grads[0].defined()) return out;
        {
            const variable_list t = unpacked();
            at::AutoDispatchBelowADInplaceOrView guard;
            const Tensor d = grads[0].scalar_type() == x_type ? grads[0] : grads[0].to(x_type);
            const Tensor xt = t[0], wt = t[1];
            const bool need_x = task_should_compute_output(0), need_w = task_should_compute_output(1), need_b = has_bias && task_should_compute_output(2);
            if (d.numel() == 0 || k == 0) {
                if (need_x) out[0] = at::zeros(x_shape, d.options());
                if (need_w) out[1] = at::zeros({n, k}, d.options().dtype(w_type));
                if (need_b) out[2] = d.numel() ? as_rows(d).sum(0).to(b_type) : at::zeros({n}, d.options().dtype(b_type));
            } else if (need_x || need_w || need_b) {
                F8Saved s;
                if (need_w) s.xt = Rounded(xt.contiguous(), k, d.numel() / n);
                if (need_x) s.wt = Rounded(wt.contiguous(), k, n);
                f8_backward(f8_rows(d), s, need_x, need_w, need_b, w_type, b_type, out[0], out[1], out[2]);
                if (need_x) out[0] = out[0].view(x_shape);
            }
        }
        return once_differentiable(std::move(out), rec);
    }
};

// x Q(w)^T + b with both rounded on the way.  None for a call that the node does not stand for or that is wrong.
OptTensor fp8_linear(const Tensor &x, const Tensor &weight, const OptTensor &bias) {
    if (!plain_modes() || !plain(x) || !plain(weight) || (bias && bias->defined() && !plain(*bias)) || !x.is_cuda()) return std::nullopt;
    if (f8_linear_wrong(x, weight, bias)) return std::nullopt;
    const Tensor b = bias ? *bias : Tensor();
    const bool wanted = SavingNode::wanted(x, weight, b);
    Tensor y;
    F8Saved s;
    {
        at::AutoDispatchBelowADInplaceOrView guard;
        y = f8_forward(x, weight, b, wanted && x.requires_grad(), wanted && weight.requires_grad(), &s);
    }
    if (wanted) {
        auto node = make_node<Fp8LinearNode>(x, weight, b);
        node->x_shape = x.sizes().vec();
        node->n = weight.size(0);
        node->k = weight.size(1);
        node->x_type = x.scalar_type();
        node->w_type = weight.scalar_type();
        node->has_bias = b.defined();
        if (b.defined()) node->b_type = b.scalar_type();
        torch::autograd::set_history(y, node);
        node->save(s.xt.hold);
        node->save(s.wt.hold);
    }
    return y;
}

// x times a weight that is held in 8 bits; no gradients.
Tensor f8_held_forward(const Tensor &x, const Tensor &q, const Tensor &s, int64_t k, const Tensor &bias) {
    c10::DeviceGuard on(x.device());
    const int64_t n = q.size(0);
    const auto shape = f8_shape(x, n);
    if (x.numel() == 0 || n == 0) {
        Tensor y = at::zeros(shape, x.options());
        return k == 0 && bias.defined() ? y.add_(bias) : y;
    }
    return f8_times(f8_rows(x), Rounded(q, s, k), bias.defined() ? bias.contiguous() : bias).view(shape);
}
OptTensor fp8_linear_held(const Tensor &x, const Tensor &values, const Tensor &scales, int64_t k, const OptTensor &bias) {
    if (!plain_modes() || !plain(x) || !plain(values) || !plain(scales) || (bias && bias->defined() && !plain(*bias)) || !x.is_cuda()) return std::nullopt;
    const Tensor b = bias ? *bias : Tensor();
    if (f8_held_wrong(x, values, scales, k, bias) || SavingNode::wanted(x, b)) return std::nullopt;
    at::AutoDispatchBelowADInplaceOrView guard;
    return f8_held_forward(x, values, scales, k, b);
}

// The same launches without a node, for the registered operators.
Tensor fp8_linear_forward(const Tensor &x, const Tensor &weight, const OptTensor &bias) {
    const char *wrong = f8_linear_wrong(x, weight, bias);
    TORCH_CHECK_VALUE(!wrong, wrong);
    TORCH_CHECK(x.is_cuda(), "fp8_linear runs on the GPU only");
    TORCH_CHECK_NOT_IMPLEMENTED(!dual(x) && !dual(weight) && !(bias && dual(*bias)), "fp8_linear has no formula for forward mode differentiation");
    return f8_forward(x, weight, bias ? *bias : Tensor(), false, false, nullptr);
}
std::vector<Tensor> fp8_linear_backward(const Tensor &dy, const Tensor &x, const Tensor &weight, const OptTensor &bias, bool need_x, bool need_w, bool need_b) {
    const char *wrong = f8_linear_wrong(x, weight, bias);
    TORCH_CHECK_VALUE(!wrong, wrong);
    TORCH_CHECK(x.is_cuda(), "fp8_linear runs on the GPU only");
    const int64_t n = weight.size(0), k = weight.size(1);
    TORCH_CHECK_VALUE(dy.device() == x.device() && dy.scalar_type() == x.scalar_type() && dy.sizes().equals(f8_shape(x, n)),
                      "the gradient must have the result's shape, dtype and device");
    need_b = need_b && bias && bias->defined();
    c10::DeviceGuard on(x.device());
    Tensor dx, dw, db;
    if (dy.numel() && k && (need_x || need_w || need_b)) {
        F8Saved s;
        if (need_w) f8_quantize(f8_rows(x), nullptr, &s.xt, nullptr);
        if (need_x) f8_quantize(f8_rows(weight), nullptr, &s.wt, nullptr);
        f8_backward(f8_rows(dy), s, need_x, need_w, need_b, weight.scalar_type(), need_b ? bias->scalar_type() : at::kFloat, dx, dw, db);
        if (need_x) dx = dx.view(x.sizes());
    } else {
        if (need_x) dx = at::zeros(x.sizes(), x.options());
        if (need_w) dw = at::zeros({n, k}, weight.options());
        if (need_b) db = dy.numel() ? as_rows(dy).sum(0).to(bias->scalar_type()) : at::zeros({n}, bias->options());
    }
    if (!need_x) dx = at::empty({0}, x.options());
    if (!need_w) dw = at::empty({0}, weight.options());
    if (!need_b) db = at::empty({0}, x.options());
    return {dx, dw, db};
}
Tensor fp8_linear_held_forward(const Tensor &x, const Tensor &values, const Tensor &scales, int64_t k, const OptTensor &bias) {
    const char *wrong = f8_held_wrong(x, values, scales, k, bias);
    TORCH_CHECK_VALUE(!wrong, wrong);
    TORCH_CHECK(x.is_cuda(), "fp8_linear runs on the GPU only");
    TORCH_CHECK_NOT_IMPLEMENTED(!dual(x) && !(bias && dual(*bias)), "fp8_linear has no formula for forward mode differentiation");
    return f8_held_forward(x, values, scales, k, bias ? *bias : Tensor());
}
// values and scales of a matrix rounded along its rows
std::pair<Tensor, Tensor> fp8_round(const Tensor &w) {
    TORCH_CHECK_VALUE(w.dim() == 2 && evo_dtype(w.scalar_type()) != EVO_NONE, "the weight must be [n, k] in bf16, fp16 or fp32");
    TORCH_CHECK_VALUE(w.size(0) <= kF8Most && w.size(1) <= kF8Most, "the weight has more than 2^26 rows or columns");
    TORCH_CHECK(w.is_cuda(), "rounding to 8 bits runs on the GPU only");
    c10::DeviceGuard on(w.device());
    const auto o = w.options().dtype(at::kByte);
    const Tensor values = at::empty({w.size(0), Rounded::pitch(w.size(1))}, o), scales = at::empty({w.size(0), Rounded::scale_pitch(w.size(1))}, o);
    if (w.numel()) {
        const Tensor r = f8_rows(w);
        check(evoattn_fp8_quantize(r.data_ptr(), f8_apart(r), values.data_ptr(), scales.data_ptr(), nullptr, nullptr, nullptr, r.size(0), r.size(1),
                                   evo_dtype(r.scalar_type()), stream_of(r)), "evoattn_fp8_quantize");
    }
    return {values, scales};
}
std::optional<std::string> fp8_linear_wrong(const Tensor &x, const Tensor &weight, const OptTensor &bias) {
    const char *wrong = f8_linear_wrong(x, weight, bias);
    return wrong ? std::optional<std::string>(wrong) : std::nullopt;
}
std::optional<std::string> fp8_linear_held_wrong(const Tensor &x, const Tensor &values, const Tensor &scales, int64_t k, const OptTensor &bias) {
    const char *wrong = f8_held_wrong(x, values, scales, k, bias);
    return wrong ? std::optional<std::string>(wrong) : std::nullopt;
}
