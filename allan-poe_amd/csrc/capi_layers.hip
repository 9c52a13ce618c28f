// C-ABI entry points of the operators that layers of an adapter are built and trained from (include/apoe.h): checks of the
// arguments, then the launchers. Nothing behind them throws.
#include <algorithm>
#include <cmath>
#include <new>

#include "apoe_internal.h"

using namespace apoe;

namespace {

size_t size_of(uint32_t dtype) { return dtype == APOE_F32 ? 4 : 2; }

// Device memory of the context's GPU, aligned.
int check_pointer(const apoe_ctx* ctx, const void* p, size_t align, const char* name) {
    APOE_REQUIRE(is_device_ptr_of(p, ctx->device), "%s must be device memory of GPU %d, the context's", name, ctx->device);
    APOE_REQUIRE(((uintptr_t)p & (align - 1)) == 0, "%s must be aligned to %zu bytes", name, align);
    return APOE_OK;
}

#define APOE_POINTER(p, align, name) \
    if (p) APOE_TRY(check_pointer(ctx, p, align, name))

#define APOE_STRIDE(s, cols)    \
    if ((s) == 0) (s) = (cols); \
    APOE_REQUIRE((s) >= (cols), "rows overlap: stride %llu for %u columns", (unsigned long long)(s), (cols))

// What is written while `q` is still read, or written by others. (Matrices may share a buffer, side by side: only the same beginning is refused.)
#define APOE_APART(p, q) APOE_REQUIRE(!(p) || (const void*)(p) != (const void*)(q), #p " and " #q " are the same memory")
// What may be `q` itself, row by row.
#define APOE_IN_PLACE(p, q, rows) \
    APOE_REQUIRE(!(p) || (const void*)(p) != (const void*)(q) || p##_stride == q##_stride || (rows) <= 1, #p " and " #q " are the same memory with other strides")

int embed(apoe_ctx* ctx, const apoe_embed_args* args, bool grad) {
    APOE_REQUIRE(ctx && args, "ctx/args is null");
    apoe_embed_args a = *args;
    APOE_REQUIRE(a.dtype <= APOE_BF16, "unknown dtype %u", a.dtype);
    APOE_REQUIRE(a.dim >= 1 && a.dim <= APOE_EMBED_MAX_DIM, "dim must be in 1..%u, got %u", APOE_EMBED_MAX_DIM, a.dim);
    APOE_REQUIRE(a.n_table < (1u << 30), "a table of %u rows is beyond 2^30", a.n_table);
    APOE_REQUIRE(a.n_entries < (1u << 27) && a.n_rows < (1u << 30), "%u entries of %u rows are beyond 2^27 or 2^30", a.n_entries, a.n_rows);
    APOE_REQUIRE(a.off || a.n_entries == a.n_rows, "without off every row has one entry: %u entries for %u rows", a.n_entries, a.n_rows);
    APOE_REQUIRE(a.n_rows || a.n_entries == 0, "%u entries without rows", a.n_entries);
    APOE_REQUIRE(std::isfinite(a.scale), "scale must be finite");
    APOE_STRIDE(a.table_stride, a.dim);
    APOE_STRIDE(a.base_stride, a.dim);
    APOE_STRIDE(a.out_stride, a.dim);
    APOE_STRIDE(a.grad_stride, a.dim);
    APOE_STRIDE(a.grad_table_stride, a.dim);
    const size_t e = size_of(a.dtype);
    if (grad) {
        APOE_REQUIRE(a.grad_table || a.grad_val, "nothing to compute");
        APOE_REQUIRE(!a.grad_val || a.table || a.n_entries == 0 || a.n_table == 0, "grad_val needs the table");
        APOE_REQUIRE(a.grad || a.n_entries == 0, "grad is null");
        APOE_REQUIRE(!a.accumulate || a.grad_table, "accumulate without grad_table");
        a.base = nullptr; // its gradient is grad itself
        a.out = nullptr;
    } else {
        if (a.n_rows == 0) return APOE_OK;
        APOE_REQUIRE(a.out, "out is null");
        APOE_REQUIRE(a.table || a.n_entries == 0 || a.n_table == 0, "table is null");
        a.grad = nullptr;
        a.grad_table = nullptr;
    }
    APOE_REQUIRE(a.idx || a.n_entries == 0, "idx is null");
    APOE_APART(a.out, a.table);
    APOE_IN_PLACE(a.out, a.base, a.n_rows);
    for (const void* in : {(const void*)a.idx, (const void*)a.off, (const void*)a.val}) APOE_APART(a.out, in);
    APOE_APART(a.grad_table, a.grad);
    APOE_APART(a.grad_table, a.table);
    if (grad)
        for (const void* in : {(const void*)a.idx, (const void*)a.off, (const void*)a.val, a.table, a.grad, (const void*)a.grad_table}) APOE_APART(a.grad_val, in);
    APOE_POINTER(a.table, e, "table");
    APOE_POINTER(a.idx, 4, "idx");
    APOE_POINTER(a.off, 4, "off");
    APOE_POINTER(a.val, 4, "val");
    APOE_POINTER(a.base, e, "base");
    APOE_POINTER(a.out, e, "out");
    APOE_POINTER(a.grad, e, "grad");
    APOE_POINTER(a.grad_table, e, "grad_table");
    APOE_POINTER(a.grad_val, 4, "grad_val");
    APOE_HIP(hipSetDevice(ctx->device));
    return launch_embed(ctx, &a, grad);
}

int layer_norm(apoe_ctx* ctx, const apoe_layer_norm_args* args, bool grad) {
    APOE_REQUIRE(ctx && args, "ctx/args is null");
    apoe_layer_norm_args a = *args;
    APOE_REQUIRE(a.dtype <= APOE_BF16, "unknown dtype %u", a.dtype);
    APOE_REQUIRE(a.dim >= 1 && a.dim <= APOE_NORM_MAX_DIM, "dim must be in 1..%u, got %u", APOE_NORM_MAX_DIM, a.dim);
    APOE_REQUIRE(std::isfinite(a.eps) && a.eps >= 0.f, "eps must not be negative, got %g", a.eps);
    APOE_STRIDE(a.x_stride, a.dim);
    APOE_STRIDE(a.y_stride, a.dim);
    APOE_STRIDE(a.grad_y_stride, a.dim);
    APOE_STRIDE(a.grad_skip_stride, a.dim);
    APOE_STRIDE(a.grad_x_stride, a.dim);
    if (grad) {
        APOE_REQUIRE(a.grad_x || a.grad_w || a.grad_b, "nothing to compute");
        APOE_REQUIRE(a.grad_y || a.rows == 0, "grad_y is null");
        a.y = nullptr;
    } else {
        APOE_REQUIRE(a.y || a.rows == 0, "y is null");
        a.grad_y = a.grad_skip = nullptr;
        a.grad_x = nullptr;
    }
    if (a.rows == 0 && !(grad && (a.grad_w || a.grad_b))) return APOE_OK;
    APOE_REQUIRE(a.x || a.rows == 0, "x is null");
    APOE_IN_PLACE(a.y, a.x, a.rows);
    APOE_IN_PLACE(a.grad_x, a.x, a.rows);
    APOE_IN_PLACE(a.grad_x, a.grad_y, a.rows);
    APOE_IN_PLACE(a.grad_x, a.grad_skip, a.rows);
    APOE_APART(a.y, a.w);
    APOE_APART(a.y, a.b);
    if (grad) { // (grad_w and grad_b are written by a launch behind the one that reads the rows)
        for (const void* other : {a.w, (const float*)a.grad_w, (const float*)a.grad_b}) APOE_APART(a.grad_x, other);
        APOE_APART(a.grad_w, a.grad_b);
    }
    const size_t e = size_of(a.dtype);
    APOE_POINTER(a.x, e, "x");
    APOE_POINTER(a.w, 4, "w");
    APOE_POINTER(a.b, 4, "b");
    APOE_POINTER(a.y, e, "y");
    APOE_POINTER(a.grad_y, e, "grad_y");
    APOE_POINTER(a.grad_skip, e, "grad_skip");
    APOE_POINTER(a.grad_x, e, "grad_x");
    if (grad) {
        APOE_POINTER(a.grad_w, 4, "grad_w");
        APOE_POINTER(a.grad_b, 4, "grad_b");
    }
    APOE_HIP(hipSetDevice(ctx->device));
    return launch_layer_norm(ctx, &a, grad);
}

int linear(apoe_ctx* ctx, const apoe_linear_args* args, bool grad) {
    APOE_REQUIRE(ctx && args, "ctx/args is null");
    apoe_linear_args a = *args;
    APOE_REQUIRE(a.dtype <= APOE_BF16, "unknown dtype %u", a.dtype);
    APOE_REQUIRE(a.act <= APOE_ACT_SILU, "unknown activation %u", a.act);
    APOE_REQUIRE(a.cols_in >= 1 && a.cols_in <= APOE_LINEAR_MAX_SIDE && a.cols_out >= 1 && a.cols_out <= APOE_LINEAR_MAX_SIDE, "columns must be in 1..%u, got %u and %u",
                 APOE_LINEAR_MAX_SIDE, a.cols_in, a.cols_out);
    APOE_REQUIRE(a.rows < (1u << 30), "%u rows are beyond 2^30", a.rows);
    APOE_STRIDE(a.x_stride, a.cols_in);
    APOE_STRIDE(a.w_stride, a.cols_in);
    APOE_STRIDE(a.residual_stride, a.cols_out);
    APOE_STRIDE(a.y_stride, a.cols_out);
    APOE_STRIDE(a.pre_stride, a.cols_out);
    APOE_STRIDE(a.grad_y_stride, a.cols_out);
    APOE_STRIDE(a.grad_x_stride, a.cols_in);
    APOE_STRIDE(a.grad_w_stride, a.cols_in);
    const size_t e = size_of(a.dtype);
    if (grad) {
        APOE_REQUIRE(a.grad_x || a.grad_w || a.grad_bias, "nothing to compute");
        if (a.rows == 0 && !a.grad_w && !a.grad_bias) return APOE_OK;
        APOE_REQUIRE(a.rows == 0 || (a.grad_y && (a.x || !a.grad_w)), "grad_y/x is null");
        APOE_REQUIRE(a.rows == 0 || a.w || !a.grad_x, "w is null");
        APOE_REQUIRE(a.rows == 0 || a.act == APOE_ACT_NONE || a.pre, "the gradient of an activation needs pre");
        for (const void* in : {a.grad_y, a.act == APOE_ACT_NONE ? nullptr : (const void*)a.pre, a.x, a.w}) {
            APOE_APART(a.grad_x, in);
            APOE_APART(a.grad_w, in);
            APOE_APART(a.grad_bias, in);
        }
        APOE_APART(a.grad_x, a.grad_w);
        APOE_APART(a.grad_bias, a.grad_x);
        APOE_APART(a.grad_bias, a.grad_w);
    } else {
        if (a.rows == 0) return APOE_OK;
        APOE_REQUIRE(a.x && a.w && a.y, "x/w/y is null");
        for (const void* in : {a.x, a.w, (const void*)a.bias}) {
            APOE_APART(a.y, in);
            APOE_APART(a.pre, in);
        }
        APOE_APART(a.y, a.pre);
        APOE_APART(a.pre, a.residual);
        APOE_IN_PLACE(a.y, a.residual, a.rows);
    }
    APOE_POINTER(a.x, e, "x");
    APOE_POINTER(a.w, e, "w");
    APOE_POINTER(a.pre, e, "pre");
    if (grad) {
        APOE_POINTER(a.grad_y, e, "grad_y");
        APOE_POINTER(a.grad_x, e, "grad_x");
        APOE_POINTER(a.grad_w, e, "grad_w");
        APOE_POINTER(a.grad_bias, 4, "grad_bias");
    } else {
        APOE_POINTER(a.bias, 4, "bias");
        APOE_POINTER(a.residual, e, "residual");
        APOE_POINTER(a.y, e, "y");
    }
    APOE_HIP(hipSetDevice(ctx->device));
    return launch_linear(ctx, &a, grad);
}

// No two arrays that a step writes may share memory.
int check_disjoint(apoe_adamw* opt) {
    using Written = apoe_adamw::Written;
    std::vector<Written>& ranges = opt->written;
    ranges.reserve(opt->tensors.size() * 6);
    const uint32_t value = opt->bits / 8;
    for (uint32_t i = 0; i < opt->tensors.size(); i++) {
        const apoe_adamw_tensor& t = opt->tensors[i];
        const size_t blocks = (t.n + APOE_ADAMW_BLOCK - 1) / APOE_ADAMW_BLOCK;
        auto add = [&](const void* p, size_t n, uint32_t size) {
            if (p && n) ranges.push_back(Written{(uintptr_t)p, (uintptr_t)p + n * size, i, size});
        };
        add(t.p, t.n, 4);
        add(t.m, t.n, value);
        add(t.v, t.n, value);
        if (opt->bits == 8) {
            add(t.m_scale, blocks, 4);
            add(t.v_scale, blocks, 4);
        }
        add(t.copy, t.n, 2);
    }
    std::sort(ranges.begin(), ranges.end(), [](const Written& x, const Written& y) { return x.begin < y.begin; });
    for (size_t i = 1; i < ranges.size(); i++) APOE_REQUIRE(ranges[i].begin >= ranges[i - 1].end, "two parameters, moments or copies share memory");
    return APOE_OK;
}

// What a step reads must not lie in what it writes, but for a gradient that is an array of its own parameter, value by value.
int check_apart(const apoe_adamw* opt, const void* p, size_t n, size_t size, uint32_t tensor, const char* name) {
    const uintptr_t begin = (uintptr_t)p, end = begin + n * size;
    auto r = std::upper_bound(opt->written.begin(), opt->written.end(), begin, [](uintptr_t at, const apoe_adamw::Written& w) { return at < w.end; });
    APOE_REQUIRE(r == opt->written.end() || r->begin >= end || (r->tensor == tensor && r->begin == begin && r->end == end && r->value == size),
                 "%s and what the step writes are the same memory", name);
    return APOE_OK;
}

int fill_adamw(apoe_adamw* opt, uint32_t count, const apoe_adamw_tensor* tensors) {
    apoe_ctx* ctx = opt->ctx;
    opt->tensors.assign(tensors, tensors + count);
    for (apoe_adamw_tensor& t : opt->tensors) {
        APOE_REQUIRE(t.n < (1ull << 35), "a parameter of %llu values is beyond 2^35", (unsigned long long)t.n);
        APOE_REQUIRE(std::isfinite(t.decay), "decay must be finite");
        if (t.n == 0) continue;
        APOE_REQUIRE(t.p && t.m && t.v, "p/m/v is null");
        APOE_REQUIRE(opt->bits == 32 || (t.m_scale && t.v_scale), "moments in 8 bits need m_scale and v_scale");
        APOE_REQUIRE(!t.copy || t.copy_dtype == APOE_F16 || t.copy_dtype == APOE_BF16, "copy_dtype must be APOE_F16 or APOE_BF16, got %u", t.copy_dtype);
        APOE_POINTER(t.p, 4, "p");
        APOE_POINTER(t.m, (size_t)opt->bits / 8, "m");
        APOE_POINTER(t.v, (size_t)opt->bits / 8, "v");
        if (opt->bits == 8) {
            APOE_POINTER(t.m_scale, 4, "m_scale");
            APOE_POINTER(t.v_scale, 4, "v_scale");
        }
        APOE_POINTER(t.copy, 2, "copy");
    }
    return check_disjoint(opt);
}

} // namespace

extern "C" {

int apoe_embed(apoe_ctx* ctx, const apoe_embed_args* args) { return embed(ctx, args, false); }

int apoe_embed_grad(apoe_ctx* ctx, const apoe_embed_args* args) { return embed(ctx, args, true); }

int apoe_layer_norm(apoe_ctx* ctx, const apoe_layer_norm_args* args) { return layer_norm(ctx, args, false); }

int apoe_layer_norm_grad(apoe_ctx* ctx, const apoe_layer_norm_args* args) { return layer_norm(ctx, args, true); }

int apoe_linear(apoe_ctx* ctx, const apoe_linear_args* args) { return linear(ctx, args, false); }

int apoe_linear_grad(apoe_ctx* ctx, const apoe_linear_args* args) { return linear(ctx, args, true); }

int apoe_adamw_create(apoe_ctx* ctx, uint32_t count, const apoe_adamw_tensor* tensors, uint32_t bits, uint32_t seed, apoe_adamw** out) {
    APOE_REQUIRE(ctx && out && (tensors || count == 0), "ctx/tensors/out is null");
    APOE_REQUIRE(bits == 8 || bits == 32, "moments have 8 or 32 bits, not %u", bits);
    *out = nullptr;
    apoe_adamw* opt = new (std::nothrow) apoe_adamw;
    APOE_REQUIRE(opt, "out of host memory");
    opt->ctx = ctx;
    opt->bits = bits;
    opt->seed = seed;
    int st = APOE_ERR_ARG;
    try {
        st = fill_adamw(opt, count, tensors);
    } catch (const std::exception&) {
        set_error("out of host memory");
    }
    if (st != APOE_OK) {
        delete opt;
        return st;
    }
    *out = opt;
    return APOE_OK;
}

void apoe_adamw_destroy(apoe_adamw* opt) { delete opt; }

int apoe_adamw_step(apoe_adamw* opt, const apoe_adamw_step_args* args) {
    APOE_REQUIRE(opt && args, "opt/args is null");
    const apoe_adamw_step_args& a = *args;
    apoe_ctx* ctx = opt->ctx;
    APOE_REQUIRE(opt->tensors.empty() || (a.grads && a.grad_dtypes), "grads/grad_dtypes is null");
    for (double x : {a.lr, a.beta1, a.beta2, a.eps, a.grad_scale}) APOE_REQUIRE(std::isfinite(x), "a coefficient is not finite");
    APOE_REQUIRE(a.beta1 >= 0. && a.beta1 < 1. && a.beta2 >= 0. && a.beta2 < 1., "betas must be in [0, 1), got %g and %g", a.beta1, a.beta2);
    APOE_REQUIRE(a.eps >= 0., "eps must not be negative, got %g", a.eps);
    APOE_REQUIRE(a.step >= 1 || a.step_dev, "steps are counted from 1");
    APOE_POINTER(a.step_dev, 4, "step_dev");
    APOE_POINTER(a.lr_dev, 4, "lr_dev");
    APOE_POINTER(a.step_taken, 4, "step_taken");
    APOE_APART(a.step_taken, a.lr_dev);
    APOE_APART(a.step_taken, a.step_dev);
    if (a.step_dev) APOE_TRY(check_apart(opt, a.step_dev, 1, 4, UINT32_MAX, "step_dev"));
    if (a.lr_dev) APOE_TRY(check_apart(opt, a.lr_dev, 1, 4, UINT32_MAX, "lr_dev"));
    if (a.step_taken) APOE_TRY(check_apart(opt, a.step_taken, 1, 4, UINT32_MAX, "step_taken"));
    for (size_t i = 0; i < opt->tensors.size(); i++) {
        if (!a.grads[i] || opt->tensors[i].n == 0) continue;
        APOE_REQUIRE(a.grad_dtypes[i] <= APOE_BF16, "unknown dtype %u of gradient %zu", a.grad_dtypes[i], i);
        APOE_TRY(check_pointer(ctx, a.grads[i], size_of(a.grad_dtypes[i]), "a gradient"));
        APOE_TRY(check_apart(opt, a.grads[i], opt->tensors[i].n, size_of(a.grad_dtypes[i]), (uint32_t)i, "a gradient"));
    }
    APOE_HIP(hipSetDevice(ctx->device));
    return launch_adamw(opt, args);
}

int apoe_adamw_moments(apoe_ctx* ctx, uint64_t n, const int8_t* m, const float* m_scale, const uint8_t* v, const float* v_scale, float* m_out, float* v_out) {
    APOE_REQUIRE(ctx, "ctx is null");
    if (n == 0) return APOE_OK;
    APOE_REQUIRE(n < (1ull << 40), "%llu values are beyond 2^40", (unsigned long long)n);
    APOE_REQUIRE(m && m_scale && v && v_scale && m_out && v_out, "m/m_scale/v/v_scale/m_out/v_out is null");
    for (const void* in : {(const void*)m, (const void*)m_scale, (const void*)v, (const void*)v_scale}) {
        APOE_APART(m_out, in);
        APOE_APART(v_out, in);
    }
    APOE_APART(m_out, v_out);
    APOE_POINTER(m, 1, "m");
    APOE_POINTER(v, 1, "v");
    APOE_POINTER(m_scale, 4, "m_scale");
    APOE_POINTER(v_scale, 4, "v_scale");
    APOE_POINTER(m_out, 4, "m_out");
    APOE_POINTER(v_out, 4, "v_out");
    APOE_HIP(hipSetDevice(ctx->device));
    return launch_adamw_moments(ctx, n, m, m_scale, v, v_scale, m_out, v_out);
}

} // extern "C"
