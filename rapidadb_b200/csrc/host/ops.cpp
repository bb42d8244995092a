// Host side of the int8 scores and of the softmax cross entropy over a base:
// argument checks, 16-byte row strides, output and scratch tensors, C ABI calls
// on the current stream of the operands' device.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>

#include <vector>

#include "host.h"

namespace rdbh {

namespace {

// rows as the kernels read them: dense columns, 16-byte row stride and base, in
// place where the tensor has that, else one padded copy
struct Rows {
    at::Tensor t;
    int64_t ld;  // elements
};

Rows aligned_rows(const at::Tensor& src) {
    const int64_t e = static_cast<int64_t>(src.element_size());
    const int64_t rows = src.size(0), cols = src.size(1), ldp = padded_ld(static_cast<int>(cols), src.scalar_type());
    const bool dense = cols == 1 || src.stride(1) == 1;
    const int64_t ld = rows <= 1 ? cols : src.stride(0);  // a single row may carry any stride
    if (dense && ld >= cols && (ld * e) % 16 == 0 && (reinterpret_cast<uintptr_t>(src.data_ptr()) & 15) == 0)
        return {src, ld};
    const at::Tensor s = dense && ld >= 0 ? src : src.contiguous();
    at::Tensor out = at::empty({rows, ldp}, src.options());
    check_status(rdb_pad_rows(s.data_ptr(), rows, cols * e, (rows <= 1 ? cols : s.stride(0)) * e, out.data_ptr(),
                              ldp * e, stream_ptr()),
                 "row copy");
    return {out.narrow(1, 0, cols), ldp};
}

void check_matrix(const at::Tensor& t, const char* name) {
    TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
    TORCH_CHECK(t.dim() == 2, name, " must be 2D [rows, dim]");
    TORCH_CHECK(t.size(1) >= 1, name, " must have at least one column");
}

void check_same_device(const at::Tensor& a, const at::Tensor& b, const char* name) {
    TORCH_CHECK(b.is_cuda() && b.device() == a.device(), name, " must be on the same CUDA device (", a.device(), ")");
}

bool float_type(at::ScalarType t) { return t == at::kFloat || t == at::kHalf || t == at::kBFloat16; }

// before anything of their size is made
void check_rows(int64_t rows, const char* name) {
    TORCH_CHECK(rows < (1LL << 31), name, " must have fewer than 2^31 rows");
}

struct XentArgs {
    Rows q, x;
    at::Tensor t;
    int64_t nq, n, d;
    int dtype;
};

// call under the device guard of `queries`
XentArgs xent_args(const at::Tensor& queries, const at::Tensor& database, const at::Tensor& targets) {
    TORCH_CHECK(queries.size(1) == database.size(1), "dimension mismatch");
    TORCH_CHECK(float_type(queries.scalar_type()), "queries must be float32, float16 or bfloat16");
    TORCH_CHECK(queries.scalar_type() == database.scalar_type(), "queries and database must have the same dtype");
    TORCH_CHECK(database.size(0) > 0, "database is empty");
    TORCH_CHECK(targets.dim() == 1 && targets.size(0) == queries.size(0), "targets must be 1D [batch]");
    TORCH_CHECK(targets.scalar_type() == at::kLong || targets.scalar_type() == at::kInt,
                "targets must be int64 or int32");
    XentArgs a;
    a.nq = queries.size(0);
    a.n = database.size(0);
    a.d = queries.size(1);
    check_rows(a.nq, "queries");
    check_rows(a.n, "database");
    TORCH_CHECK(a.d < (1LL << 31) - 256, "dim must be < 2^31 - 256");
    a.dtype = dtype_code(queries.scalar_type());
    check_pending_status();
    a.q = aligned_rows(queries);
    a.x = aligned_rows(database);
    a.t = targets.to(at::kLong).contiguous();
    return a;
}

void check_operands(const at::Tensor& queries, const at::Tensor& database, const at::Tensor& targets) {
    check_matrix(queries, "queries");
    check_matrix(database, "database");
    check_same_device(queries, database, "database");
    check_same_device(queries, targets, "targets");
}

void check_stats(const at::Tensor& stats, int64_t nq) {
    TORCH_CHECK(stats.scalar_type() == at::kFloat && stats.dim() == 1 && stats.size(0) == 3 * nq + 1,
                "stats must be float32 [3 * batch + 1]");
}

at::Tensor scratch(size_t bytes, const at::Tensor& like) {
    return at::empty({static_cast<int64_t>(bytes)}, like.options().dtype(at::kByte));
}

}  // namespace

Result sq8_encode(const at::Tensor& vectors) {
    check_matrix(vectors, "vectors");
    TORCH_CHECK(float_type(vectors.scalar_type()), "vectors must be float32, float16 or bfloat16");
    TORCH_CHECK(vectors.size(1) < (1LL << 31) - 256, "dim must be < 2^31 - 256");
    c10::cuda::CUDAGuard guard(vectors.device());
    at::Tensor codes = at::empty({vectors.size(0), vectors.size(1)}, vectors.options().dtype(at::kChar));
    at::Tensor scales = at::empty({vectors.size(0)}, vectors.options().dtype(at::kFloat));
    sq8_encode_into(vectors, codes, scales);
    return {codes, scales};
}

at::Tensor sq8_dot_product(const at::Tensor& query_codes, const at::Tensor& query_scales, const at::Tensor& codes,
                           const at::Tensor& scales, at::ScalarType dtype) {
    check_matrix(query_codes, "query_codes");
    check_matrix(codes, "codes");
    check_same_device(query_codes, codes, "codes");
    check_same_device(query_codes, query_scales, "query_scales");
    check_same_device(query_codes, scales, "scales");
    TORCH_CHECK(query_codes.scalar_type() == at::kChar && codes.scalar_type() == at::kChar, "codes must be int8");
    TORCH_CHECK(query_codes.size(1) == codes.size(1), "dimension mismatch");
    TORCH_CHECK(query_scales.scalar_type() == at::kFloat && scales.scalar_type() == at::kFloat,
                "scales must be float32");
    TORCH_CHECK(query_scales.dim() == 1 && query_scales.size(0) == query_codes.size(0),
                "query_scales must be 1D [batch]");
    TORCH_CHECK(scales.dim() == 1 && scales.size(0) == codes.size(0), "scales must be 1D [n]");
    TORCH_CHECK(float_type(dtype), "dtype must be float32, float16 or bfloat16");
    const int64_t nq = query_codes.size(0), n = codes.size(0), d = codes.size(1);
    check_rows(nq, "query_codes");
    check_rows(n, "codes");
    c10::cuda::CUDAGuard guard(codes.device());
    at::Tensor out = at::empty({nq, n}, codes.options().dtype(dtype));
    if (nq == 0 || n == 0) return out;
    TORCH_CHECK(d <= 131071, "dim must be <= 131071");
    check_pending_status();
    const Rows qc = aligned_rows(query_codes), xc = aligned_rows(codes);
    const at::Tensor qs = query_scales.contiguous(), xs = scales.contiguous();
    check_status(rdb_sq8_dot(qc.t.data_ptr<int8_t>(), qs.data_ptr<float>(), nq, qc.ld, xc.t.data_ptr<int8_t>(),
                             xs.data_ptr<float>(), n, xc.ld, static_cast<int>(d), dtype_code(dtype), out.data_ptr(), n,
                             stream_ptr()),
                 "sq8 dot product");
    return out;
}

namespace {

Result run_forward(const XentArgs& a, const at::TensorOptions& opts, double scale, int64_t ignore_index,
                   int reduction) {
    const auto f32 = opts.dtype(at::kFloat);
    at::Tensor loss = reduction == RDB_REDUCE_NONE ? at::empty({a.nq}, f32) : at::empty({}, f32);
    at::Tensor stats = at::empty({3 * a.nq + 1}, f32);
    const size_t wsb = rdb_softmax_xent_workspace(a.dtype, a.nq, a.n, static_cast<int>(a.d), reduction);
    at::Tensor ws = scratch(wsb, stats);
    check_status(rdb_softmax_xent(a.dtype, a.q.t.data_ptr(), a.nq, a.q.ld, a.x.t.data_ptr(), a.n, a.x.ld,
                                  static_cast<int>(a.d), a.t.data_ptr<int64_t>(), static_cast<float>(scale),
                                  ignore_index, reduction, loss.data_ptr<float>(), stats.data_ptr<float>(),
                                  ws.data_ptr(), wsb, stream_ptr()),
                 "softmax cross entropy");
    return {loss, stats};
}

Result run_backward(const XentArgs& a, const at::Tensor& grad, const at::Tensor& stats, double scale,
                    int64_t ignore_index, int reduction, bool need_queries, bool need_database) {
    at::Tensor dq, dx;
    if (need_queries) dq = at::empty({a.nq, a.d}, a.q.t.options());
    if (need_database) dx = at::empty({a.n, a.d}, a.x.t.options());
    if (!need_queries && !need_database) return {dq, dx};
    const at::Tensor g = grad.to(at::kFloat).contiguous();
    const size_t wsb = rdb_softmax_xent_backward_workspace(a.dtype, a.nq, a.n, static_cast<int>(a.d), need_queries,
                                                           need_database);
    at::Tensor ws = scratch(wsb, stats);
    check_status(rdb_softmax_xent_backward(
                     a.dtype, a.q.t.data_ptr(), a.nq, a.q.ld, a.x.t.data_ptr(), a.n, a.x.ld, static_cast<int>(a.d),
                     a.t.data_ptr<int64_t>(), static_cast<float>(scale), ignore_index, reduction, g.data_ptr<float>(),
                     stats.data_ptr<float>(), need_queries ? dq.data_ptr() : nullptr, a.d,
                     need_database ? dx.data_ptr() : nullptr, a.d, ws.data_ptr(), wsb, stream_ptr()),
                 "softmax cross entropy backward");
    return {dq, dx};
}

// The autograd node.  It keeps the operands as the kernels read them (the
// inputs themselves, or their padded copies) and the forward's statistics.  What
// comes back may lie elsewhere and in other strides (saved-tensor hooks: offloaded
// to the host, packed), so the backward pass looks at it afresh.
struct XentLoss : torch::autograd::Function<XentLoss> {
    static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& queries,
                              const at::Tensor& database, const at::Tensor& targets, double scale,
                              int64_t ignore_index, int64_t reduction) {
        const XentArgs a = xent_args(queries, database, targets);
        Result r = run_forward(a, queries.options(), scale, ignore_index, static_cast<int>(reduction));
        ctx->save_for_backward({a.q.t, a.x.t, a.t, std::get<1>(r)});
        ctx->saved_data["call"] = std::vector<int64_t>{ignore_index, reduction};
        ctx->saved_data["scale"] = scale;
        return std::get<0>(r);
    }

    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                   torch::autograd::variable_list grads) {
        TORCH_CHECK(!at::GradMode::is_enabled(), "softmax_cross_entropy has no second derivative (create_graph=True)");
        const auto saved = ctx->get_saved_variables();
        const auto call = ctx->saved_data["call"].toIntVector();
        check_operands(saved[0], saved[1], saved[2]);
        check_same_device(saved[0], saved[3], "stats");
        c10::cuda::CUDAGuard guard(saved[0].device());
        const XentArgs a = xent_args(saved[0], saved[1], saved[2]);
        check_stats(saved[3], a.nq);
        const Result r = run_backward(a, grads[0], saved[3].contiguous(), ctx->saved_data["scale"].toDouble(), call[0],
                                      static_cast<int>(call[1]), ctx->needs_input_grad(0), ctx->needs_input_grad(1));
        return {std::get<0>(r), std::get<1>(r), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
    }
};

}  // namespace

at::Tensor softmax_cross_entropy_loss(const at::Tensor& queries, const at::Tensor& database, const at::Tensor& targets,
                                      double scale, int64_t ignore_index, int reduction) {
    check_operands(queries, database, targets);
    c10::cuda::CUDAGuard guard(queries.device());
    return XentLoss::apply(queries, database, targets, scale, ignore_index, static_cast<int64_t>(reduction));
}

Result softmax_cross_entropy(const at::Tensor& queries, const at::Tensor& database, const at::Tensor& targets,
                             double scale, int64_t ignore_index, int reduction) {
    check_operands(queries, database, targets);
    c10::cuda::CUDAGuard guard(queries.device());
    at::NoGradGuard no_grad;
    return run_forward(xent_args(queries, database, targets), queries.options(), scale, ignore_index, reduction);
}

Result softmax_cross_entropy_backward(const at::Tensor& grad, const at::Tensor& queries, const at::Tensor& database,
                                      const at::Tensor& targets, const at::Tensor& stats, double scale,
                                      int64_t ignore_index, int reduction, bool need_queries, bool need_database) {
    check_operands(queries, database, targets);
    check_same_device(queries, grad, "grad");
    check_same_device(queries, stats, "stats");
    c10::cuda::CUDAGuard guard(queries.device());
    at::NoGradGuard no_grad;
    const XentArgs a = xent_args(queries, database, targets);
    check_stats(stats, a.nq);
    TORCH_CHECK(reduction == RDB_REDUCE_NONE ? grad.dim() == 1 && grad.size(0) == a.nq : grad.numel() == 1,
                "grad must have the shape of the loss");
    return run_backward(a, grad, stats.contiguous(), scale, ignore_index, reduction, need_queries, need_database);
}

}  // namespace rdbh
