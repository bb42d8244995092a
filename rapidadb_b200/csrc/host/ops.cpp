// Host side of the int8 scores and of the softmax cross entropy over a base:
// argument checks, 16-byte row strides, output and scratch tensors, C ABI calls
// on the current stream of the operands' device.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "host.h"

namespace rdbh {

namespace {

// rows readable in place by the kernels: dense columns, 16-byte row stride and
// base; anything else is copied once into padded rows
at::Tensor aligned_rows(const at::Tensor& t) {
    const int64_t e = static_cast<int64_t>(t.element_size());
    const int64_t rows = t.size(0), cols = t.size(1);
    const bool dense = (cols <= 1 || t.stride(1) == 1) && (rows <= 1 || t.stride(0) >= cols);
    const int64_t ld = rows <= 1 ? cols : t.stride(0);
    if (dense && (ld * e) % 16 == 0 && (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0) return t;
    return prepare_rows(t, t.scalar_type(), padded_ld(static_cast<int>(cols), t.scalar_type()));
}

int64_t row_stride(const at::Tensor& t, int64_t cols) {
    // a single row may carry any stride
    return t.size(0) <= 1 ? (t.size(1) > cols ? t.size(1) : cols) : t.stride(0);
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

struct XentArgs {
    at::Tensor q, x, t;
    int64_t nq, n, d, ldq, ldx;
    int dtype;
};

XentArgs xent_args(const at::Tensor& queries, const at::Tensor& database, const at::Tensor& targets) {
    check_matrix(queries, "queries");
    check_matrix(database, "database");
    check_same_device(queries, database, "database");
    check_same_device(queries, targets, "targets");
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
    a.dtype = dtype_code(queries.scalar_type());
    a.q = aligned_rows(queries);
    a.x = aligned_rows(database);
    a.ldq = row_stride(a.q, padded_ld(static_cast<int>(a.d), a.q.scalar_type()));
    a.ldx = row_stride(a.x, padded_ld(static_cast<int>(a.d), a.x.scalar_type()));
    a.t = targets.to(at::kLong).contiguous();
    return a;
}

at::Tensor scratch(size_t bytes, const at::Tensor& like) {
    return at::empty({static_cast<int64_t>(bytes)}, like.options().dtype(at::kByte));
}

}  // namespace

Result sq8_encode(const at::Tensor& vectors) {
    check_matrix(vectors, "vectors");
    TORCH_CHECK(float_type(vectors.scalar_type()), "vectors must be float32, float16 or bfloat16");
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
    c10::cuda::CUDAGuard guard(codes.device());
    at::Tensor out = at::empty({nq, n}, codes.options().dtype(dtype));
    if (nq == 0 || n == 0) return out;
    TORCH_CHECK(d <= 131071, "dim must be <= 131071");
    at::Tensor qc = aligned_rows(query_codes), xc = aligned_rows(codes);
    at::Tensor qs = query_scales.contiguous(), xs = scales.contiguous();
    const int64_t ldp = padded_ld(static_cast<int>(d), at::kChar);
    check_status(rdb_sq8_dot(qc.data_ptr<int8_t>(), qs.data_ptr<float>(), nq, row_stride(qc, ldp),
                             xc.data_ptr<int8_t>(), xs.data_ptr<float>(), n, row_stride(xc, ldp),
                             static_cast<int>(d), dtype_code(dtype), out.data_ptr(), n, stream_ptr()),
                 "sq8 dot product");
    return out;
}

Result softmax_cross_entropy(const at::Tensor& queries, const at::Tensor& database, const at::Tensor& targets,
                             double scale, int64_t ignore_index, int reduction) {
    XentArgs a = xent_args(queries, database, targets);
    c10::cuda::CUDAGuard guard(queries.device());
    const auto f32 = queries.options().dtype(at::kFloat);
    at::Tensor loss = reduction == RDB_REDUCE_NONE ? at::empty({a.nq}, f32) : at::empty({}, f32);
    at::Tensor stats = at::empty({3, a.nq}, f32);
    const size_t wsb = rdb_softmax_xent_workspace(a.dtype, a.nq, a.n, static_cast<int>(a.d), reduction);
    at::Tensor ws = scratch(wsb, queries);
    check_status(rdb_softmax_xent(a.dtype, a.q.data_ptr(), a.nq, a.ldq, a.x.data_ptr(), a.n, a.ldx,
                                  static_cast<int>(a.d), a.t.data_ptr<int64_t>(), static_cast<float>(scale),
                                  ignore_index, reduction, loss.data_ptr<float>(), stats.data_ptr<float>(),
                                  ws.data_ptr(), wsb, stream_ptr()),
                 "softmax cross entropy");
    return {loss, stats};
}

Result softmax_cross_entropy_backward(const at::Tensor& grad, const at::Tensor& queries, const at::Tensor& database,
                                      const at::Tensor& targets, const at::Tensor& stats, double scale,
                                      int64_t ignore_index, int reduction, bool need_queries, bool need_database) {
    XentArgs a = xent_args(queries, database, targets);
    check_same_device(queries, grad, "grad");
    check_same_device(queries, stats, "stats");
    TORCH_CHECK(stats.scalar_type() == at::kFloat && stats.dim() == 2 && stats.size(0) == 3 && stats.size(1) == a.nq,
                "stats must be float32 [3, batch]");
    TORCH_CHECK(reduction == RDB_REDUCE_NONE ? grad.dim() == 1 && grad.size(0) == a.nq : grad.numel() == 1,
                "grad must have the shape of the loss");
    c10::cuda::CUDAGuard guard(queries.device());
    at::Tensor dq, dx;
    if (need_queries) dq = at::empty({a.nq, a.d}, queries.options());
    if (need_database) dx = at::empty({a.n, a.d}, database.options());
    if (!need_queries && !need_database) return {dq, dx};
    at::Tensor g = grad.to(at::kFloat).contiguous(), st = stats.contiguous();
    const size_t wsb = rdb_softmax_xent_backward_workspace(a.dtype, a.nq, a.n, static_cast<int>(a.d), need_queries,
                                                           need_database);
    at::Tensor ws = scratch(wsb, queries);
    check_status(rdb_softmax_xent_backward(
                     a.dtype, a.q.data_ptr(), a.nq, a.ldq, a.x.data_ptr(), a.n, a.ldx, static_cast<int>(a.d),
                     a.t.data_ptr<int64_t>(), static_cast<float>(scale), ignore_index, reduction, g.data_ptr<float>(),
                     st.data_ptr<float>(), need_queries ? dq.data_ptr() : nullptr, a.d,
                     need_database ? dx.data_ptr() : nullptr, a.d, ws.data_ptr(), wsb, stream_ptr()),
                 "softmax cross entropy backward");
    return {dq, dx};
}

}  // namespace rdbh
