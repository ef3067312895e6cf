// The host path of the decoder block's operators (include/pam_hip_block.h): nodes and calls for pam_host.cpp, which includes
// this file inside its namespace, behind the helpers it uses.

// ---------------------------------------------------------------- products with an activation, gated layers

// (rows contiguous, or copied so)
Tensor rows_contiguous(const Tensor& t) { return t.size(1) <= 1 || t.stride(1) == 1 ? t : t.contiguous(); }

struct Layer { Tensor y, z; };

// act(X W^T + bias) + residual, or with `gated` act(g) (*) u of W's two halves; want_z: what the activation is applied to, too
Layer layer(bool gated, const Tensor& X, const Tensor& W, const Tensor& bias, int activation, const Tensor& residual, bool want_z, double offset)
{
    const char* const name = gated ? "gated_linear" : "linear_act";
    check_tensor(X); check_tensor(W);
    if (bias.defined()) check_tensor(bias);
    if (residual.defined()) check_tensor(residual);
    TORCH_CHECK_VALUE(X.dim() == 2 && W.dim() == 2 && X.size(1) == W.size(1), name, ": shapes ", shape(X), " and ", shape(W), " do not multiply");
    const int64_t m = X.size(0), k = X.size(1), rows = W.size(0), n = gated ? rows / 2 : rows;
    TORCH_CHECK_VALUE(!gated || rows % 2 == 0, name, ": the weight has the gate's rows and as many others, got ", rows);
    TORCH_CHECK_VALUE(!bias.defined() || (bias.dim() == 1 && bias.numel() == rows), name, ": bias must have one value per row of the weight");
    TORCH_CHECK_VALUE(!residual.defined() || (residual.dim() == 2 && residual.size(0) == m && residual.size(1) == n), name, ": the residual must have the shape of the result");
    for (const Tensor* t : {&W, &bias, &residual})
        TORCH_CHECK_VALUE(!t->defined() || t->device() == X.device(), name, ": tensors are on different devices");
    const OnDevice on(X);
    Layer out;
    out.y = new_floats({m, n}, X);
    if (want_z) out.z = new_floats({m, rows}, X);
    if (out.y.numel() == 0) return out;
    const Tensor b = bias.defined() ? bias.contiguous() : bias, res = residual.defined() ? rows_contiguous(residual) : residual;
    const size_t bytes = gated ? pam_hip_gated_linear_workspace_bytes(m, n, k) : pam_hip_linear_act_workspace_bytes(m, n, k);
    Tensor ws;
    if (bytes) ws = gemm_workspace(X, on.stream, bytes);
    if (gated)
        check_call(pam_hip_gated_linear_fwd(data(X), X.stride(0), X.stride(1), data(W), W.stride(0), W.stride(1), data_or_null(b), activation,
                                            data_or_null(out.z), data(out.y), m, n, k, (float)offset, data_or_null(ws), bytes, on.stream), "gated_linear_fwd");
    else
        check_call(pam_hip_linear_act_fwd(data(X), X.stride(0), X.stride(1), data(W), W.stride(0), W.stride(1), data_or_null(b), activation,
                                          data_or_null(res), res.defined() ? res.stride(0) : 0, data_or_null(out.z), data(out.y), m, n, k, (float)offset,
                                          data_or_null(ws), bytes, on.stream), "linear_act_fwd");
    return out;
}

// The gradients of Y = A (x) B, as product_grads, with the sums of pam_hip_layer_grad
Tensor layer_grad(const Tensor& L, const Tensor& R, const Tensor& other, int kind, double offset)
{
    for (const Tensor* t : {&L, &R, &other}) check_tensor(*t);
    const int64_t m = L.size(0), k = L.size(1), n = R.size(1);
    TORCH_CHECK_VALUE(R.size(0) == k && other.size(0) == m && other.size(1) == n, "layer_grad: shapes ", shape(L), " and ", shape(R), " do not multiply to ", shape(other));
    const OnDevice on(L);
    const Tensor out = new_floats({m, n}, L);
    if (out.numel() == 0) return out;
    const size_t bytes = pam_hip_layer_grad_workspace_bytes(m, n, k);
    Tensor ws;
    if (bytes) ws = gemm_workspace(L, on.stream, bytes);
    check_call(pam_hip_layer_grad(data(L), L.stride(0), L.stride(1), data(R), R.stride(0), R.stride(1), data(other), other.stride(0), other.stride(1),
                                  data(out), out.stride(0), out.stride(1), m, n, k, kind, (float)offset, data_or_null(ws), bytes, on.stream), "layer_grad");
    return out;
}
ProductGrads layer_grads(const Tensor& A, const Tensor& B, const Tensor& dY, const Approx& f, double offset, bool need_A, bool need_B)
{
    ProductGrads g;
    if (need_A) g.dA = layer_grad(dY, row_major(B.t(), 2), A, f.a ? 0 : 1, offset);
    if (need_B) g.dB = layer_grad(row_major(A.t(), 2), dY, B, f.b ? 0 : 2, offset);
    return g;
}

struct LayerNode : torch::autograd::Function<LayerNode> {
    static Tensor forward(AutogradContext* ctx, bool gated, const Tensor& X_in, const Tensor& W, const std::optional<Tensor>& bias, int64_t activation,
                          const std::optional<Tensor>& residual, bool train, double offset, bool a, bool b, bool e)
    {
        TORCH_CHECK_VALUE(X_in.dim() == 2, gated ? "gated_linear" : "linear_act", ": expected rows of values");
        const Tensor X = row_major(X_in, 2);
        const bool keep_z = train && (gated || activation != PAM_HIP_ACT_NONE);
        const Layer out = layer(gated, X, W, bias.value_or(Tensor()), (int)activation, residual.value_or(Tensor()), keep_z, offset);
        ctx->saved_data["gated"] = gated; ctx->saved_data["activation"] = activation; ctx->saved_data["offset"] = offset;
        ctx->saved_data["bias"] = bias.has_value(); ctx->saved_data["residual"] = residual.has_value(); ctx->saved_data["rows"] = W.size(0);
        Approx{a, b, e}.save(ctx);
        if (train) ctx->save_for_backward({X, W, out.z});
        return out.y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        const variable_list saved = ctx->get_saved_variables();
        const Approx f = Approx::saved(ctx);
        const bool gated = ctx->saved_data["gated"].toBool(), has_bias = ctx->saved_data["bias"].toBool(), has_residual = ctx->saved_data["residual"].toBool();
        const int activation = (int)ctx->saved_data["activation"].toInt();
        const double offset = ctx->saved_data["offset"].toDouble();
        const int64_t rows = ctx->saved_data["rows"].toInt();
        const char* const name = gated ? "gated_linear_bwd" : "linear_act_bwd";
        const Tensor dy = grads[0];
        check_tensor(dy);
        const int64_t m = dy.size(0);
        // (edges are counted over the tensors that are there)
        const bool want_x = ctx->needs_input_grad(0), want_w = ctx->needs_input_grad(1), want_b = has_bias && ctx->needs_input_grad(2);
        Tensor dX, dW, db;
        {
            const at::AutoGradMode no_graph(false);
            Tensor dz = row_major(dy, 2);
            if ((gated || activation != PAM_HIP_ACT_NONE) && (want_x || want_w || want_b)) {
                const Tensor z = whole(saved[2], dy, {m, rows}, name), d = dy.contiguous();
                const OnDevice on(dy);
                dz = new_floats({m, rows}, dy);
                const float off = (float)offset;
                if (gated) check_call(pam_hip_gated_bwd(data(z), data(d), data(dz), m, rows / 2, activation, off, f.a, f.b, f.e, on.stream), "gated_bwd");
                else check_call(pam_hip_act_bwd(data(z), data(d), data(dz), d.numel(), activation, off, f.a, f.b, f.e, on.stream), "act_bwd");
            }
            const Tensor X = row_major(saved[0], 2), Wt = row_major(saved[1].t(), 2);
            TORCH_CHECK_VALUE(X.size(0) == m && Wt.size(1) == rows, name, ": a saved tensor has not the shape that it was saved with");
            const ProductGrads g = layer_grads(X, Wt, dz, f, offset, want_x, want_w);
            dX = g.dA;
            if (g.dB.defined()) dW = g.dB.t();
            if (want_b) db = sum_rows(dz);
        }
        return {Tensor(), dX, dW, db, Tensor(), has_residual ? dy : Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

// A tensor that carries a forward-mode derivative is refused, also where nothing is recorded (it does not require a gradient): its result
// would come without one, which counts as zero.
void refuse_forward_mode(const char* name, const Tensor& t)
{
    TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(/*level=*/0).defined(), name, ": no forward-mode derivatives");
}

bool wants_graph(const char* name, std::initializer_list<const Tensor*> tensors)
{
    for (const Tensor* t : tensors) refuse_forward_mode(name, *t);
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor* t : tensors)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}

// ... of X [..., d_in], the residual of the result's shape
Tensor call_layer(bool gated, const Tensor& X, const Tensor& W, const std::optional<Tensor>& bias, int64_t activation, const std::optional<Tensor>& residual,
                  double offset, bool a, bool b, bool e)
{
    const char* const name = gated ? "gated_linear" : "linear_act";
    const Tensor none;
    TORCH_CHECK_VALUE(W.dim() == 2, name, ": the weight is a matrix, got ", shape(W));
    TORCH_CHECK_VALUE(!gated || W.size(0) % 2 == 0, name, ": the weight has the gate's rows and as many others, got ", shape(W));
    TORCH_CHECK_VALUE(X.dim() >= 1 && X.size(-1) == W.size(1), name, ": shapes ", shape(X), " and ", shape(W), " do not multiply");
    const int64_t n = gated ? W.size(0) / 2 : W.size(0);
    const bool rows = X.dim() == 2;
    std::vector<int64_t> sizes(X.sizes().begin(), X.sizes().end());
    sizes.back() = n;
    TORCH_CHECK_VALUE(!residual || residual->sizes() == at::IntArrayRef(sizes), name, ": the residual must have the shape of the result, got ", residual ? shape(*residual) : "");
    const int64_t m = c10::multiply_integers(sizes.begin(), sizes.end() - 1);
    const Tensor x = rows ? X : X.reshape({m, X.size(-1)});
    std::optional<Tensor> r = residual;
    if (r && !rows) r = r->reshape({m, n});
    Tensor y;
    if (wants_graph(name, {&x, &W, bias ? &*bias : &none, r ? &*r : &none})) y = LayerNode::apply(gated, x, W, bias, activation, r, true, offset, a, b, e);
    else y = layer(gated, row_major(x, 2), W, bias.value_or(none), (int)activation, r.value_or(none), false, offset).y;
    return rows ? y : y.view(sizes);
}

// ---------------------------------------------------------------- rotation of queries and keys

struct Rotation {
    Tensor cos, sin, positions;
    int64_t batch, tokens, dim, rotated;
    bool interleaved;
    float eps, offset;
};

Tensor heads_contiguous(const Tensor& t) { return t.size(3) <= 1 || t.stride(3) == 1 ? t : t.contiguous(); }

// [batch][tokens][heads][dim]: the entry of a tensor in the call's table
pam_hip_heads heads_of(const Tensor& x, const Tensor& weight, const Tensor& y)
{
    pam_hip_heads h{};
    h.x = data(x); h.x_sb = x.stride(0); h.x_st = x.stride(1); h.x_sh = x.stride(2);
    h.weight = data_or_null(weight); h.y = data(y); h.heads = x.size(2);
    return h;
}

Rotation rotation(const variable_list& x, const variable_list& weights, const Tensor& cos, const Tensor& sin, const Tensor& positions, bool interleaved, double eps, double offset,
                  bool by_row = true)
{
    const char* const name = by_row ? "rotary" : "rotary_append";          // by_row: without positions token t is at the tables' row t
    Rotation r;
    r.batch = x[0].dim() == 4 ? x[0].size(0) : 0; r.tokens = x[0].dim() == 4 ? x[0].size(1) : 0; r.dim = x[0].dim() == 4 ? x[0].size(3) : 0;
    for (size_t i = 0; i < x.size(); ++i) {
        check_tensor(x[i]);
        TORCH_CHECK_VALUE(x[i].dim() == 4 && x[i].size(0) == r.batch && x[i].size(1) == r.tokens && x[i].size(3) == r.dim && x[i].device() == x[0].device(),
                          name, ": queries and keys are [batch, tokens, heads, dim] on one device, got ", shape(x[0]), " and ", shape(x[i]));
        if (!weights[i].defined()) continue;
        check_tensor(weights[i]);
        TORCH_CHECK_VALUE(weights[i].dim() == 1 && weights[i].numel() == r.dim && weights[i].device() == x[0].device(), name, ": a norm's weight has one value per value of a head");
    }
    check_tensor(cos); check_tensor(sin);
    TORCH_CHECK_VALUE(cos.dim() == 2 && cos.sizes() == sin.sizes() && cos.device() == x[0].device() && sin.device() == x[0].device(),
                      name, ": cos and sin are two tables of one shape on the tensors' device");
    TORCH_CHECK_VALUE(2 * cos.size(1) <= r.dim, name, ": the tables rotate ", 2 * cos.size(1), " values of a head that has ", r.dim);
    TORCH_CHECK(!cos.requires_grad() && !sin.requires_grad(), name, ": the tables have no gradient");
    r.cos = cos.contiguous(); r.sin = sin.contiguous();
    r.rotated = 2 * cos.size(1);
    if (positions.defined()) {
        TORCH_CHECK_TYPE(positions.scalar_type() == at::kLong, name, ": positions are int64");
        TORCH_CHECK_VALUE(positions.device() == x[0].device() && (positions.dim() == 1 || positions.dim() == 2) && positions.size(-1) == r.tokens
                              && (positions.dim() == 1 || positions.size(0) == r.batch),
                          name, ": positions are [tokens] or [batch, tokens] on the tensors' device, got ", shape(positions));
        r.positions = positions;
    } else if (by_row) {
        TORCH_CHECK_VALUE(r.tokens <= cos.size(0), name, ": ", r.tokens, " tokens and tables of ", cos.size(0), " positions");
    }
    r.interleaved = interleaved; r.eps = (float)eps; r.offset = (float)offset;
    return r;
}

struct RotationArgs { const long long* positions; int64_t sb, st; };
RotationArgs positions_of(const Rotation& r)
{
    if (!r.positions.defined()) return {nullptr, 0, 0};
    return {reinterpret_cast<const long long*>(r.positions.data_ptr<int64_t>()), r.positions.dim() == 2 ? r.positions.stride(0) : 0, r.positions.stride(-1)};
}

// The rotation of the tensors x, made contiguous along a head (and so left in x), by the weights w, made contiguous.
variable_list rotate(variable_list& x, variable_list& w, const Rotation& r)
{
    const OnDevice on(x[0]);
    variable_list y;
    pam_hip_heads parts[2];
    for (size_t i = 0; i < x.size(); ++i) {
        x[i] = heads_contiguous(x[i]);
        if (w[i].defined()) w[i] = w[i].contiguous();
        y.push_back(new_floats(x[i].sizes(), x[i]));
        parts[i] = heads_of(x[i], w[i], y[i]);
    }
    const RotationArgs at = positions_of(r);
    check_call(pam_hip_rotary_fwd(parts, (int)x.size(), data(r.cos), data(r.sin), r.cos.size(0), at.positions, at.sb, at.st, r.batch, r.tokens, r.dim, r.rotated,
                                  r.interleaved, r.eps, r.offset, on.stream), "rotary_fwd");
    return y;
}

struct RotaryNode : torch::autograd::Function<RotaryNode> {
    static variable_list forward(AutogradContext* ctx, const Tensor& q, const std::optional<Tensor>& k, const Tensor& cos, const Tensor& sin,
                                 const std::optional<Tensor>& positions, const std::optional<Tensor>& q_weight, const std::optional<Tensor>& k_weight,
                                 bool interleaved, double eps, double offset, bool a, bool b, bool e)
    {
        variable_list x{q}, w{q_weight.value_or(Tensor())};
        if (k) { x.push_back(*k); w.push_back(k_weight.value_or(Tensor())); }
        const Rotation r = rotation(x, w, cos, sin, positions.value_or(Tensor()), interleaved, eps, offset);
        const variable_list y = rotate(x, w, r);
        ctx->saved_data["count"] = (int64_t)x.size(); ctx->saved_data["positions"] = positions.has_value();
        ctx->saved_data["wq"] = q_weight.has_value(); ctx->saved_data["wk"] = k_weight.has_value();
        ctx->saved_data["interleaved"] = interleaved; ctx->saved_data["eps"] = eps; ctx->saved_data["offset"] = offset;
        for (size_t i = 0; i < x.size(); ++i) ctx->saved_data[i ? "k" : "q"] = x[i].sizes();
        Approx{a, b, e}.save(ctx);
        x.resize(2); w.resize(2);
        ctx->save_for_backward({x[0], x[1], w[0], w[1], r.cos, r.sin, r.positions});
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        const variable_list saved = ctx->get_saved_variables();
        const Approx f = Approx::saved(ctx);
        const size_t count = (size_t)ctx->saved_data["count"].toInt();
        const at::AutoGradMode no_graph(false);
        variable_list x, w, dx, dw, dy;
        // (edges are counted over the tensors that are there: q, k, cos, sin, positions, the weights)
        size_t edge = count + 2 + (ctx->saved_data["positions"].toBool() ? 1 : 0);
        bool want_w[2] = {false, false};
        if (ctx->saved_data["wq"].toBool()) want_w[0] = ctx->needs_input_grad(edge++);
        if (ctx->saved_data["wk"].toBool()) want_w[1] = ctx->needs_input_grad(edge++);
        const OnDevice on(grads[0]);
        std::vector<pam_hip_heads> parts;
        for (size_t i = 0; i < count; ++i) {
            check_tensor(grads[i]);
            const std::vector<int64_t> sizes = ctx->saved_data[i ? "k" : "q"].toIntVector();
            check_tensor(saved[i]);
            TORCH_CHECK_VALUE(saved[i].sizes() == at::IntArrayRef(sizes) && saved[i].device() == grads[i].device() && grads[i].sizes() == at::IntArrayRef(sizes),
                              "rotary_bwd: a saved tensor has not the shape or the device that it was saved with");
            x.push_back(heads_contiguous(saved[i])); dy.push_back(heads_contiguous(grads[i]));
            w.push_back(saved[2 + i].defined() ? whole(saved[2 + i], grads[i], {sizes[3]}, "rotary_bwd") : Tensor());
            dx.push_back(new_floats(sizes, grads[i]));
            dw.push_back(want_w[i] ? new_floats({sizes[3]}, grads[i]) : Tensor());
            pam_hip_heads h = heads_of(x[i], w[i], dx[i]);
            h.dy = data(dy[i]); h.dy_sb = dy[i].stride(0); h.dy_st = dy[i].stride(1); h.dy_sh = dy[i].stride(2);
            h.dweight = data_or_null(dw[i]);
            parts.push_back(h);
        }
        const Rotation r = rotation(x, w, saved[4], saved[5], saved[6], ctx->saved_data["interleaved"].toBool(), ctx->saved_data["eps"].toDouble(), ctx->saved_data["offset"].toDouble());
        const RotationArgs at = positions_of(r);
        const size_t bytes = pam_hip_rotary_bwd_workspace_bytes(parts.data(), (int)count, r.batch, r.tokens, r.dim, r.rotated);
        const Tensor ws = bytes ? new_floats({(int64_t)((bytes + 3) / 4)}, grads[0]) : Tensor();
        check_call(pam_hip_rotary_bwd(parts.data(), (int)count, data(r.cos), data(r.sin), r.cos.size(0), at.positions, at.sb, at.st, r.batch, r.tokens, r.dim,
                                      r.rotated, r.interleaved, r.eps, r.offset, f.a, f.b, f.e, data_or_null(ws), bytes, on.stream), "rotary_bwd");
        dx.resize(2); dw.resize(2);
        return {dx[0], dx[1], Tensor(), Tensor(), Tensor(), dw[0], dw[1], Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

variable_list call_rotary(const Tensor& q, const std::optional<Tensor>& k, const Tensor& cos, const Tensor& sin, const std::optional<Tensor>& positions,
                          const std::optional<Tensor>& q_weight, const std::optional<Tensor>& k_weight, bool interleaved, double eps, double offset, bool a, bool b, bool e)
{
    const Tensor none;
    if (wants_graph("rotary", {&q, k ? &*k : &none, &cos, &sin, q_weight ? &*q_weight : &none, k_weight ? &*k_weight : &none}))
        return RotaryNode::apply(q, k, cos, sin, positions, q_weight, k_weight, interleaved, eps, offset, a, b, e);
    variable_list x{q}, w{q_weight.value_or(none)};
    if (k) { x.push_back(*k); w.push_back(k_weight.value_or(none)); }
    return rotate(x, w, rotation(x, w, cos, sin, positions.value_or(none), interleaved, eps, offset));
}

// ---------------------------------------------------------------- clipping

// Whether memory that is written for one tensor also belongs to another one of the table.  (What is read and what is written apart: either
// is mostly in order already, as it was allocated.  85 tensors with outputs: 0.3 us of a call less than all ranges sorted together.)
bool clip_overlaps(const std::vector<pam_hip_clip_tensor>& table)
{
    struct Range { uintptr_t begin, end; };
    std::vector<Range> read, written;
    read.reserve(table.size()); written.reserve(table.size());
    for (const pam_hip_clip_tensor& t : table) {
        const size_t bytes = t.n * sizeof(float);
        if (t.in != t.out) read.push_back({(uintptr_t)t.in, (uintptr_t)t.in + bytes});
        if (t.out) written.push_back({(uintptr_t)t.out, (uintptr_t)t.out + bytes});
    }
    const auto before = [](const Range& a, const Range& b) { return a.begin < b.begin; };
    for (auto* ranges : {&read, &written})
        if (!std::is_sorted(ranges->begin(), ranges->end(), before)) std::sort(ranges->begin(), ranges->end(), before);
    for (size_t i = 1; i < written.size(); ++i)
        if (written[i].begin < written[i - 1].end) return true;
    size_t w = 0;                                 // the first written range that ends behind where the read one begins
    for (const Range& r : read) {
        while (w < written.size() && written[w].end <= r.begin) ++w;
        if (w < written.size() && written[w].begin < r.end) return true;
    }
    return false;
}

// Whether a sum of x_i stride_i with 0 <= x_i <= most_i can be `target`: strides from the largest on, each x_i within what the smaller
// ones can make up for.  Strides that enclose each other, as views of rows and columns have, leave one or two values to try; a search of
// many steps counts as a yes.
class Reach {
public:
    void add(int64_t stride, int64_t most) { if (stride > 0 && most > 0) terms.push_back({stride, most, 0, 0}); }
    bool operator()(int64_t target)
    {
        std::sort(terms.begin(), terms.end(), [](const Term& a, const Term& b) { return a.stride < b.stride; });
        int64_t reach = 0, divisor = 0;
        size_t count = 0;
        for (const Term& t : terms) {
            if (count > 0 && terms[count - 1].stride == t.stride) terms[count - 1].most += t.most;       // (one choice instead of two)
            else terms[count++] = t;
            reach += t.stride * t.most; divisor = std::gcd(divisor, t.stride);
            terms[count - 1].reach = reach; terms[count - 1].divisor = divisor;
        }
        return search(count, target);
    }
private:
    struct Term { int64_t stride, most, reach, divisor; };       // reach, divisor: of this and all smaller ones
    bool search(size_t count, int64_t target)
    {
        if (target == 0 || ++steps > 10000) return true;
        if (count == 0) return false;
        const Term& t = terms[count - 1];
        if (target < 0 || target > t.reach || target % t.divisor != 0) return false;
        const int64_t below = t.reach - t.stride * t.most;
        for (int64_t x = std::min(t.most, target / t.stride); x >= 0 && target - x * t.stride <= below; --x)
            if (search(count - 1, target - x * t.stride)) return true;
        return false;
    }
    c10::SmallVector<Term, 8> terms;
    int steps = 0;
};
// Whether two values of a tensor are at one address: differences of indices, the first of them at least one in dimension k, that sum to nothing.
bool folds_on_itself(const Tensor& t)
{
    for (int64_t k = 0; k < t.dim(); ++k) {
        if (t.size(k) <= 1) continue;
        Reach reach;
        int64_t others = 0;
        for (int64_t i = 0; i < t.dim(); ++i) {
            reach.add(t.stride(i), i == k ? t.size(i) - 2 : 2 * (t.size(i) - 1));
            if (i != k) others += (t.size(i) - 1) * t.stride(i);
        }
        if (reach(others - t.stride(k))) return true;
    }
    return false;
}
int64_t span(const Tensor& t)                                        // (floats from its first value to its last)
{
    int64_t last = 0;
    for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
    return last;
}
bool share_values(const Tensor& a, const Tensor& b)
{
    const intptr_t apart = (intptr_t)data(b) - (intptr_t)data(a);
    Reach reach;
    for (const Tensor* t : {&a, &b})
        for (int64_t i = 0; i < t->dim(); ++i) reach.add(t->stride(i), t->size(i) - 1);
    return apart % (intptr_t)sizeof(float) != 0 || reach(apart / (intptr_t)sizeof(float) + span(b));
}
// Whether an output that is written by a copy shares memory with itself or another output.  (Their inputs have been read by then.)
bool copies_overlap(const std::vector<Tensor>& copied, const std::vector<Tensor>& direct)
{
    struct Output {
        const Tensor* t; uintptr_t begin, end; bool copied;
        int64_t row = 0, width = 0;               // the largest stride, how far the other dimensions reach
    };
    std::vector<Output> outputs;
    for (const auto* list : {&copied, &direct})
        for (const Tensor& t : *list) {
            if (t.numel() == 0) continue;
            if (list == &copied && folds_on_itself(t)) return true;
            const uintptr_t begin = (uintptr_t)data(t);
            Output o{&t, begin, begin + (uintptr_t)(span(t) + 1) * sizeof(float), list == &copied};
            for (int64_t i = 0; i < t.dim(); ++i) if (t.size(i) > 1) o.row = std::max(o.row, t.stride(i));
            for (int64_t i = 0; i < t.dim(); ++i) if (t.stride(i) < o.row) o.width += (t.size(i) - 1) * t.stride(i);
            outputs.push_back(o);
        }
    // (columns of one buffer, the common case, lie beside each other in its rows: 512 of them are 130 000 pairs)
    const auto beside = [](const Output& a, const Output& b) {
        const int64_t apart = (int64_t)(b.begin - a.begin);
        if (a.row == 0 || a.row != b.row || apart % (int64_t)sizeof(float) != 0) return false;
        const int64_t at = apart / (int64_t)sizeof(float) % a.row;
        return at > a.width && at + b.width < a.row;
    };
    std::sort(outputs.begin(), outputs.end(), [](const Output& a, const Output& b) { return a.begin < b.begin; });
    for (size_t i = 0; i < outputs.size(); ++i)
        for (size_t j = i + 1; j < outputs.size() && outputs[j].begin < outputs[i].end; ++j)
            if ((outputs[i].copied || outputs[j].copied) && !beside(outputs[i], outputs[j]) && share_values(*outputs[i].t, *outputs[j].t)) return true;
    return false;
}

// The norm of all tensors; with `outs`, the clipped values there (a tensor may be its own output).  Values are taken in the order of
// memory where a tensor's memory is without gaps or overlaps and its output's strides are its own; others go through copies.
// (the lists are read as Python holds them: a program's hundreds of tensors, twice, as vectors of references took longer than the kernels)
Tensor clip(const py::list& ins, const py::list& outs, double max_norm, double eps, double offset)
{
    const size_t count = ins.size();
    TORCH_CHECK_VALUE(count > 0, "clip_grads: no tensors");
    TORCH_CHECK_VALUE(outs.empty() || outs.size() == count, "clip_grads: as many outputs as tensors");
    const auto tensor = [](const py::list& list, size_t i) -> const Tensor& {
        PyObject* item = PyList_GET_ITEM(list.ptr(), (Py_ssize_t)i);
        TORCH_CHECK_TYPE(THPVariable_Check(item), "clip_grads: expected tensors");
        return THPVariable_Unpack(item);
    };
    const bool recording = at::GradMode::is_enabled();
    const at::AutoGradMode no_graph(false);
    const Tensor& first = tensor(ins, 0);
    std::vector<pam_hip_clip_tensor> table;
    std::vector<std::pair<Tensor, Tensor>> copied;                   // (where the result belongs, where it is)
    variable_list held;
    std::vector<c10::TensorImpl*> written;
    table.reserve(count); written.reserve(outs.size());
    for (size_t i = 0; i < count; ++i) {
        const Tensor* in = &tensor(ins, i);
        check_tensor(*in);
        refuse_forward_mode(outs.empty() ? "grad_norm" : "clip_grads", *in);
        TORCH_CHECK(!(recording && outs.empty() && in->requires_grad()),
                    "grad_norm: the norm has no gradient, and a tensor requires one; detach it or call under torch.no_grad()");
        TORCH_CHECK_VALUE(in->layout() == at::kStrided && in->device() == first.device(), "clip_grads: tensors are dense and on one device");
        const at::IntArrayRef sizes = in->sizes();
        if (!in->is_non_overlapping_and_dense()) {
            held.reserve(count);                                     // (so that `in` stays where it is)
            held.push_back(in->contiguous());
            in = &held.back();
        }
        float* out_data = nullptr;
        if (!outs.empty()) {
            const Tensor& out = tensor(outs, i);
            check_tensor(out);
            TORCH_CHECK_VALUE(out.sizes() == sizes && out.device() == first.device(), "clip_grads: an output has its tensor's shape and device");
            written.push_back(out.unsafeGetTensorImpl());
            if (out.strides() == in->strides()) out_data = data(out);
            else {
                copied.emplace_back(out, at::empty_like(*in));
                out_data = data(copied.back().second);
            }
        }
        const size_t n = (size_t)in->numel();
        if (n) table.push_back({data(*in), out_data, n});
    }
    bool shared = !outs.empty() && clip_overlaps(table);
    if (!copied.empty() && !shared) {
        variable_list by_copy, direct;
        for (size_t i = 0; i < count; ++i) {
            const Tensor& out = tensor(outs, i);
            (by_copy.size() < copied.size() && copied[by_copy.size()].first.is_same(out) ? by_copy : direct).push_back(out);
        }
        shared = copies_overlap(by_copy, direct);
    }
    TORCH_CHECK_VALUE(!shared, "clip_grads: outputs share memory with each other, with other tensors or within themselves");
    // (written through their pointers: a graph that has saved one of them must not be run on the new values)
    for (c10::TensorImpl* out : written)
        if (!out->is_inference()) out->bump_version();
    const py::gil_scoped_release unlocked;
    const OnDevice on(first);
    const Tensor norm = new_floats({}, first);
    const size_t bytes = pam_hip_clip_workspace_bytes(table.data(), (long)table.size());
    const Tensor ws = new_floats({(int64_t)(bytes / 4)}, first);
    check_call(pam_hip_clip_many(table.data(), (long)table.size(), (float)max_norm, (float)eps, data(norm), (float)offset, data(ws), bytes, on.stream), "clip_many");
    for (const auto& c : copied) c.first.copy_(c.second);
    return norm;
}
