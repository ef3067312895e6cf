// The host path of attention and of the paged cache (include/pam_hip_attention.h): nodes and calls for pam_host.cpp, which includes this file
// inside its namespace, behind pam_host_block.h.

// ---------------------------------------------------------------- attention

struct AttentionCall {
    pam_hip_attention_shape shape;
    Tensor prefix, documents, slopes;             // (they live as long as the launch needs them)
};

// Heads in rows of whole quads, a head's values side by side: the tensor itself, or a copy.
Tensor heads_in_quads(const Tensor& t)
{
    const int64_t short_of = (4 - t.size(3) % 4) % 4;
    return short_of ? at::constant_pad_nd(t, {0, short_of}, 1.0) : heads_contiguous(t);
}
pam_hip_tokens tokens_of(const Tensor& t) { return {data(t), t.stride(0), t.stride(1), t.stride(2)}; }

Tensor checked_integers(const char* name, const char* what, const Tensor& t, const Tensor& like, at::IntArrayRef sizes)
{
    TORCH_CHECK_TYPE(t.scalar_type() == at::kLong, name, ": ", what, " are int64");
    TORCH_CHECK_VALUE(t.sizes() == sizes && t.device() == like.device(), name, ": ", what, " are of shape ", sizes, " on the tensors' device, got ", shape(t));
    return t.contiguous();
}
Tensor checked_slopes(const char* name, const Tensor& t, const Tensor& like, int64_t heads)
{
    check_tensor(t);
    TORCH_CHECK_VALUE(t.dim() == 1 && t.numel() == heads && t.device() == like.device(), name, ": slopes are one value per head on the tensors' device, got ", shape(t));
    TORCH_CHECK(!t.requires_grad(), name, ": the slopes have no gradient");
    return t.contiguous();
}

AttentionCall attention_call(const Tensor& q, const Tensor& k, const Tensor& v, double scale, bool causal, int64_t window, const Tensor& prefix, const Tensor& documents,
                             const Tensor& slopes, double cap, double offset)
{
    const char* const name = "attention";
    check_tensor(q); check_tensor(k); check_tensor(v);
    TORCH_CHECK_VALUE(q.dim() == 4 && k.dim() == 4 && v.sizes() == k.sizes() && q.size(0) == k.size(0) && q.size(3) == k.size(3) && q.device() == k.device() && q.device() == v.device(),
                      name, ": queries, keys and values are [batch, tokens, heads, dim] on one device, got ", shape(q), ", ", shape(k), " and ", shape(v));
    TORCH_CHECK_VALUE(q.size(3) >= 1 && q.size(3) <= 256, name, ": heads have up to 256 values, got ", q.size(3));
    TORCH_CHECK_VALUE(k.size(2) == 0 ? q.size(2) == 0 : q.size(2) % k.size(2) == 0, name, ": ", q.size(2), " heads do not share ", k.size(2));
    TORCH_CHECK_VALUE(window >= 0, name, ": the window has at least one key");
    AttentionCall c{};
    if (prefix.defined()) c.prefix = checked_integers(name, "prefixes", prefix, q, {q.size(0)});
    if (documents.defined()) c.documents = checked_integers(name, "documents", documents, q, {k.size(0), k.size(1)});
    if (slopes.defined()) c.slopes = checked_slopes(name, slopes, q, q.size(2));
    pam_hip_attention_shape& s = c.shape;
    s.batch = q.size(0); s.tokens = q.size(1); s.keys = k.size(1); s.heads = q.size(2); s.kv_heads = k.size(2);
    s.values = q.size(3); s.dim = (q.size(3) + 3) / 4 * 4;
    s.scale = (float)scale; s.cap = (float)cap; s.offset = (float)offset; s.causal = causal; s.window = window;
    s.prefix = c.prefix.defined() ? reinterpret_cast<const long long*>(c.prefix.data_ptr<int64_t>()) : nullptr;
    s.documents = c.documents.defined() ? reinterpret_cast<const long long*>(c.documents.data_ptr<int64_t>()) : nullptr;
    s.slopes = data_or_null(c.slopes);
    return c;
}

// (of whole quads, without what is behind a head's values)
Tensor without_pad(const Tensor& t, int64_t values) { return t.size(3) == values ? t : t.narrow(3, 0, values).contiguous(); }
Tensor scratch_bytes(size_t bytes, const Tensor& like) { return bytes ? new_floats({(int64_t)((bytes + 3) / 4)}, like) : Tensor(); }

struct AttentionResult { Tensor y, stats; };      // y in whole quads
AttentionResult attend(const AttentionCall& c, const Tensor& q_in, const Tensor& k_in, const Tensor& v_in, bool want_stats)
{
    const OnDevice on(q_in);
    const Tensor q = heads_in_quads(q_in), k = heads_in_quads(k_in), v = heads_in_quads(v_in);
    AttentionResult r;
    r.y = new_floats({q.size(0), q.size(1), q.size(2), c.shape.dim}, q);
    if (want_stats) r.stats = new_floats({q.size(0), q.size(1), q.size(2), 2}, q);
    const size_t bytes = pam_hip_attention_workspace_bytes(&c.shape);
    const Tensor ws = scratch_bytes(bytes, q);
    const pam_hip_tokens at[3] = {tokens_of(q), tokens_of(k), tokens_of(v)};
    check_call(pam_hip_attention_fwd(&c.shape, &at[0], &at[1], &at[2], data(r.y), data_or_null(r.stats), data_or_null(ws), bytes, on.stream), "attention_fwd");
    return r;
}

struct AttentionNode : torch::autograd::Function<AttentionNode> {
    static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, double scale, bool causal, int64_t window, const std::optional<Tensor>& prefix,
                          const std::optional<Tensor>& documents, const std::optional<Tensor>& slopes, double cap, double offset, bool a, bool b, bool e)
    {
        const AttentionCall c = attention_call(q, k, v, scale, causal, window, prefix.value_or(Tensor()), documents.value_or(Tensor()), slopes.value_or(Tensor()), cap, offset);
        const AttentionResult r = attend(c, q, k, v, true);
        const Tensor y = without_pad(r.y, c.shape.values);
        ctx->saved_data["scale"] = scale; ctx->saved_data["causal"] = causal; ctx->saved_data["window"] = window; ctx->saved_data["cap"] = cap; ctx->saved_data["offset"] = offset;
        ctx->saved_data["q"] = q.sizes(); ctx->saved_data["k"] = k.sizes();
        Approx{a, b, e}.save(ctx);
        ctx->save_for_backward({q, k, v, y, r.stats, c.prefix, c.documents, c.slopes});
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        const variable_list saved = ctx->get_saved_variables();
        const Approx f = Approx::saved(ctx);
        const at::AutoGradMode no_graph(false);
        const Tensor& dy_in = grads[0];
        check_tensor(dy_in);
        const std::vector<int64_t> of_q = ctx->saved_data["q"].toIntVector(), of_k = ctx->saved_data["k"].toIntVector();
        const char* const wrong = "attention_bwd: a saved tensor has not the shape or the device that it was saved with";
        for (int i = 0; i < 5; ++i) {
            check_tensor(saved[i]);
            std::vector<int64_t> sizes = i == 1 || i == 2 ? of_k : of_q;
            if (i == 4) sizes[3] = 2;
            TORCH_CHECK_VALUE(saved[i].sizes() == at::IntArrayRef(sizes) && saved[i].device() == dy_in.device(), wrong);
        }
        TORCH_CHECK_VALUE(dy_in.sizes() == at::IntArrayRef(of_q), wrong);
        const AttentionCall c = attention_call(saved[0], saved[1], saved[2], ctx->saved_data["scale"].toDouble(), ctx->saved_data["causal"].toBool(), ctx->saved_data["window"].toInt(),
                                               saved[5], saved[6], saved[7], ctx->saved_data["cap"].toDouble(), ctx->saved_data["offset"].toDouble());
        const bool want_q = ctx->needs_input_grad(0), want_kv = ctx->needs_input_grad(1) || ctx->needs_input_grad(2);
        const OnDevice on(dy_in);
        const Tensor q = heads_in_quads(saved[0]), k = heads_in_quads(saved[1]), v = heads_in_quads(saved[2]), dy = heads_in_quads(dy_in);
        const Tensor y = heads_in_quads(saved[3]).contiguous(), stats = saved[4].contiguous();
        Tensor dq, dk, dv;
        if (want_q) dq = new_floats({of_q[0], of_q[1], of_q[2], c.shape.dim}, q);
        if (want_kv) { dk = new_floats({of_k[0], of_k[1], of_k[2], c.shape.dim}, q); dv = new_floats(dk.sizes(), q); }
        const size_t bytes = pam_hip_attention_bwd_workspace_bytes(&c.shape, want_q, want_kv);
        const Tensor ws = scratch_bytes(bytes, q);
        const pam_hip_tokens at[4] = {tokens_of(q), tokens_of(k), tokens_of(v), tokens_of(dy)};
        check_call(pam_hip_attention_bwd(&c.shape, &at[0], &at[1], &at[2], data(y), data(stats), &at[3], data_or_null(dq), data_or_null(dk), data_or_null(dv), f.a, f.b, f.e,
                                         data_or_null(ws), bytes, on.stream), "attention_bwd");
        const auto result = [&](const Tensor& t, size_t i) { return t.defined() && ctx->needs_input_grad(i) ? without_pad(t, c.shape.values) : Tensor(); };
        return {result(dq, 0), result(dk, 1), result(dv, 2), Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

Tensor call_attention(const Tensor& q, const Tensor& k, const Tensor& v, double scale, bool causal, int64_t window, const std::optional<Tensor>& prefix,
                      const std::optional<Tensor>& documents, const std::optional<Tensor>& slopes, double cap, double offset, bool a, bool b, bool e)
{
    const Tensor none;
    if (wants_graph("attention", {&q, &k, &v, slopes ? &*slopes : &none}))
        return AttentionNode::apply(q, k, v, scale, causal, window, prefix, documents, slopes, cap, offset, a, b, e);
    const AttentionCall c = attention_call(q, k, v, scale, causal, window, prefix.value_or(none), documents.value_or(none), slopes.value_or(none), cap, offset);
    return without_pad(attend(c, q, k, v, false).y, c.shape.values);
}

// ---------------------------------------------------------------- a paged cache

// What keys and values of a cache look like, and the table that says where a sequence's are.
struct Cache { Tensor pages, lengths, counts; int64_t per_sequence; };
Cache checked_cache(const char* name, const Tensor& k, const Tensor& v, const Tensor& pages, const Tensor& lengths, const Tensor& counts, const Tensor& q, int64_t batch, int64_t dim)
{
    check_tensor(k); check_tensor(v);
    TORCH_CHECK_VALUE(k.dim() == 4 && v.sizes() == k.sizes() && v.strides() == k.strides() && k.device() == q.device() && v.device() == q.device() && k.size(1) >= 1,
                      name, ": a cache's keys and values are two tensors [pages, page, kv heads, dim] of the same strides on the tensors' device, got ", shape(k), " and ", shape(v));
    TORCH_CHECK_VALUE(k.size(3) == dim && (dim <= 1 || k.stride(3) == 1), name, ": a head's values lie side by side in the cache, as many as a query has");
    TORCH_CHECK_TYPE(pages.scalar_type() == at::kInt, name, ": the table of pages is int32");
    TORCH_CHECK_VALUE(pages.dim() == 2 && pages.size(0) == batch && pages.device() == q.device(), name, ": the table of pages is [batch, pages of a sequence] on the tensors' device, got ", shape(pages));
    Cache c;
    c.pages = pages.contiguous(); c.per_sequence = pages.size(1);
    c.lengths = checked_integers(name, "lengths", lengths, q, {batch});
    if (counts.defined()) c.counts = checked_integers(name, "counts", counts, q, {batch});
    return c;
}
const long long* integers(const Tensor& t) { return t.defined() ? reinterpret_cast<const long long*>(t.data_ptr<int64_t>()) : nullptr; }

// Whether two tensors have a value in common.  (Mostly their memory is apart as a whole.)
bool in_common(const Tensor& a, const Tensor& b)
{
    if (a.numel() == 0 || b.numel() == 0) return false;
    const uintptr_t a0 = (uintptr_t)data(a), b0 = (uintptr_t)data(b);
    return a0 < b0 + (uintptr_t)(span(b) + 1) * sizeof(float) && b0 < a0 + (uintptr_t)(span(a) + 1) * sizeof(float) && share_values(a, b);
}

Tensor call_rotary_append(const Tensor& q_in, const Tensor& k_in, const Tensor& v_in, const Tensor& cos, const Tensor& sin, const Tensor& cache_k, const Tensor& cache_v,
                          const Tensor& pages, const Tensor& lengths, const std::optional<Tensor>& counts, const std::optional<Tensor>& q_weight,
                          const std::optional<Tensor>& k_weight, bool interleaved, double eps, double offset)
{
    const char* const name = "rotary_append";
    const Tensor none;
    TORCH_CHECK(!wants_graph(name, {&q_in, &k_in, &v_in, &cos, &sin, &cache_k, &cache_v, q_weight ? &*q_weight : &none, k_weight ? &*k_weight : &none}),
                "rotary_append: what goes into a cache has no gradient, and a tensor requires one; call it under torch.no_grad()");
    variable_list x{q_in, k_in}, w{q_weight.value_or(none), k_weight.value_or(none)};
    check_tensor(v_in);
    const Rotation r = rotation(x, w, cos, sin, none, interleaved, eps, offset, /*by_row=*/false);
    TORCH_CHECK_VALUE(v_in.sizes() == k_in.sizes() && v_in.device() == k_in.device(), name, ": keys and values have one shape, got ", shape(k_in), " and ", shape(v_in));
    const Cache c = checked_cache(name, cache_k, cache_v, pages, lengths, counts.value_or(none), q_in, r.batch, r.dim);
    TORCH_CHECK_VALUE(cache_k.size(2) == k_in.size(2), name, ": ", k_in.size(2), " keys' heads and a cache of ", cache_k.size(2));
    bool shared = folds_on_itself(cache_k) || in_common(cache_k, cache_v);
    for (const Tensor* t : {&q_in, &k_in, &v_in, &cos, &sin})
        for (const Tensor* cache : {&cache_k, &cache_v}) shared = shared || in_common(*cache, *t);
    for (const Tensor& t : w)
        if (t.defined()) shared = shared || in_common(cache_k, t) || in_common(cache_v, t);
    TORCH_CHECK_VALUE(!shared, name, ": the cache shares memory within itself or with what is read");
    const OnDevice on(q_in);
    for (size_t i = 0; i < 2; ++i) {
        x[i] = heads_contiguous(x[i]);
        if (w[i].defined()) w[i] = w[i].contiguous();
    }
    const Tensor v = heads_contiguous(v_in), y = new_floats(x[0].sizes(), x[0]);
    // (written through their pointers: a graph that has saved one of them must not be run on the new values)
    for (const Tensor* t : {&cache_k, &cache_v})
        if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
    const pam_hip_heads of_q = heads_of(x[0], w[0], y), of_k = heads_of(x[1], w[1], cache_k), of_v = heads_of(v, none, cache_v);
    check_call(pam_hip_rotary_append(&of_q, &of_k, &of_v, data(r.cos), data(r.sin), r.cos.size(0), data(cache_k), data(cache_v), cache_k.stride(0), cache_k.stride(1), cache_k.stride(2),
                                     cache_k.size(1), cache_k.size(0), c.per_sequence, c.pages.data_ptr<int>(), integers(c.lengths), integers(c.counts), r.batch, r.tokens, r.dim,
                                     r.rotated, r.interleaved, r.eps, r.offset, on.stream), name);
    return y;
}

Tensor call_cached_attention(const Tensor& q_in, const Tensor& cache_k, const Tensor& cache_v, const Tensor& pages, const Tensor& lengths, const std::optional<Tensor>& counts,
                             double scale, int64_t window, const std::optional<Tensor>& slopes, double cap, double offset)
{
    const char* const name = "cached_attention";
    const Tensor none;
    TORCH_CHECK(!wants_graph(name, {&q_in, &cache_k, &cache_v, slopes ? &*slopes : &none}),
                "cached_attention: a cache's attention has no gradient, and a tensor requires one; call it under torch.no_grad()");
    check_tensor(q_in);
    TORCH_CHECK_VALUE(q_in.dim() == 4 && q_in.size(3) >= 1 && q_in.size(3) <= 256, name, ": queries are [batch, tokens, heads, dim], heads of up to 256 values, got ", shape(q_in));
    const Cache c = checked_cache(name, cache_k, cache_v, pages, lengths, counts.value_or(none), q_in, q_in.size(0), q_in.size(3));
    const int64_t kv_heads = cache_k.size(2);
    TORCH_CHECK_VALUE(kv_heads == 0 ? q_in.size(2) == 0 : q_in.size(2) % kv_heads == 0, name, ": ", q_in.size(2), " heads do not share ", kv_heads);
    TORCH_CHECK_VALUE(window >= 0, name, ": the window has at least one key");
    const Tensor slope = slopes ? checked_slopes(name, *slopes, q_in, q_in.size(2)) : Tensor();
    const OnDevice on(q_in);
    const Tensor q = heads_contiguous(q_in), y = new_floats(q.sizes(), q);
    pam_hip_cache_shape s{};
    s.batch = q.size(0); s.tokens = q.size(1); s.heads = q.size(2); s.kv_heads = kv_heads; s.dim = q.size(3);
    s.page = cache_k.size(1); s.pages = cache_k.size(0); s.per_sequence = c.per_sequence;
    s.scale = (float)scale; s.cap = (float)cap; s.offset = (float)offset; s.window = window; s.slopes = data_or_null(slope);
    const size_t bytes = pam_hip_cached_attention_workspace_bytes(&s);
    const Tensor ws = scratch_bytes(bytes, q);
    const pam_hip_tokens at = tokens_of(q);
    check_call(pam_hip_cached_attention_fwd(&s, &at, data(cache_k), data(cache_v), cache_k.stride(0), cache_k.stride(1), cache_k.stride(2), c.pages.data_ptr<int>(),
                                            integers(c.lengths), integers(c.counts), data(y), data_or_null(ws), bytes, on.stream), name);
    return y;
}
