// C-ABI entry points of the operators that fit a query adapter (include/apoe.h): checks of the arguments, then the launchers.
// Nothing behind them throws: the launchers allocate nothing on the host.
#include <cmath>

#include "apoe_internal.h"

using namespace apoe;

namespace {

constexpr uint32_t ORTHO_MAX_SIDE = 65536; // 256 rows of a working matrix stay well within a 31-bit offset

size_t size_of(uint32_t dtype) { return dtype == APOE_F32 ? 4 : 2; }

// Device memory of the context's GPU, aligned.
int check_pointer(const apoe_ctx* ctx, const void* p, size_t align, const char* name) {
    APOE_REQUIRE(is_device_ptr_of(p, ctx->device), "%s must be device memory of GPU %d, the context's", name, ctx->device);
    APOE_REQUIRE(((uintptr_t)p & (align - 1)) == 0, "%s must be aligned to %zu bytes", name, align);
    return APOE_OK;
}

#define APOE_POINTER(p, align, name) \
    if (p) APOE_TRY(check_pointer(ctx, p, align, name))

} // namespace

extern "C" {

int apoe_softmax_loss(apoe_ctx* ctx, const apoe_softmax_loss_args* args) {
    APOE_REQUIRE(ctx && args, "ctx/args is null");
    apoe_softmax_loss_args a = *args;
    APOE_REQUIRE(a.dtype <= APOE_BF16, "unknown dtype %u", a.dtype);
    if (!a.rows) {
        APOE_REQUIRE(a.corpus, "neither rows nor a corpus");
        APOE_REQUIRE(a.corpus->ctx && a.corpus->ctx->device == ctx->device, "the corpus is on another GPU");
        APOE_REQUIRE_STATE(a.corpus->half.p, "the corpus has no half-precision rows (apoe_corpus_make_half_rows)");
        APOE_REQUIRE(a.dtype == APOE_F16, "the rows of a corpus are half precision: dtype must be APOE_F16");
        APOE_REQUIRE(a.dim == a.corpus->dim && a.n_rows == a.corpus->n, "the corpus has %u rows of %u columns, not %u of %u", a.corpus->n, a.corpus->dim, a.n_rows, a.dim);
        APOE_REQUIRE(!a.grad_rows, "the rows of a corpus stay as they are: grad_rows must be null");
        a.rows = a.corpus->half.p;
        a.rows_stride = a.dim;
    }
    const uint32_t unit = (uint32_t)(16 / size_of(a.dtype));
    APOE_REQUIRE(a.n_rows >= 1 && a.n_rows < (1u << 30), "row count %u outside [1, 2^30)", a.n_rows);
    APOE_REQUIRE(a.n_queries < (1u << 20), "query count %u outside [0, 2^20)", a.n_queries);
    APOE_REQUIRE(a.dim >= unit && a.dim <= APOE_LOSS_MAX_DIM && a.dim % unit == 0, "dim must be a multiple of %u up to %u, got %u", unit, APOE_LOSS_MAX_DIM, a.dim);
    APOE_REQUIRE(std::isfinite(a.scale) && a.scale > 0.f, "scale must be positive, got %g", a.scale);
    for (uint64_t* s : {&a.q_stride, &a.rows_stride, &a.grad_q_stride, &a.grad_rows_stride}) {
        if (*s == 0) *s = a.dim;
        APOE_REQUIRE(*s >= a.dim && *s <= (1u << 18) && *s % unit == 0, "strides must be multiples of %u from dim up to 2^18, got %llu", unit, (unsigned long long)*s);
    }
    APOE_REQUIRE(a.loss || a.lse || a.grad_q || a.grad_rows, "nothing to compute");
    APOE_REQUIRE(a.t_off || (!a.loss && !a.grad_q && !a.grad_rows), "t_off is null");
    APOE_REQUIRE(!a.t_off || a.t_idx, "t_idx is null");
    if (a.n_queries == 0 && !a.grad_rows) return APOE_OK;
    APOE_REQUIRE(a.q, "q is null");
    APOE_POINTER(a.q, 16, "q");
    APOE_POINTER(a.rows, 16, "rows");
    APOE_POINTER(a.grad_q, 16, "grad_q");
    APOE_POINTER(a.grad_rows, 16, "grad_rows");
    APOE_POINTER(a.t_off, 4, "t_off");
    APOE_POINTER(a.t_idx, 4, "t_idx");
    APOE_POINTER(a.t_val, 4, "t_val");
    APOE_POINTER(a.live, 4, "live");
    APOE_POINTER(a.weight, 4, "weight");
    APOE_POINTER(a.loss, 4, "loss");
    APOE_POINTER(a.lse, 4, "lse");
    APOE_REQUIRE(a.n_queries >= 1, "grad_rows without queries");
    APOE_HIP(hipSetDevice(ctx->device));
    return launch_softmax_loss(ctx, &a);
}

int apoe_orthogonalize(apoe_ctx* ctx, const apoe_orthogonalize_args* args) {
    APOE_REQUIRE(ctx && args, "ctx/args is null");
    apoe_orthogonalize_args a = *args;
    APOE_REQUIRE(a.in_dtype <= APOE_BF16 && a.out_dtype <= APOE_BF16, "unknown dtype %u or %u", a.in_dtype, a.out_dtype);
    APOE_REQUIRE(a.products == APOE_F16 || a.products == APOE_F32, "products must be APOE_F16 or APOE_F32, got %u", a.products);
    APOE_REQUIRE(a.rows <= ORTHO_MAX_SIDE && a.cols <= ORTHO_MAX_SIDE, "a side of %u x %u is beyond %u", a.rows, a.cols, ORTHO_MAX_SIDE);
    APOE_REQUIRE(a.batch <= 65535, "batch of %u is beyond 65535", a.batch);
    APOE_REQUIRE(a.steps >= 1 && a.steps <= 64, "steps must be in 1..64, got %u", a.steps);
    APOE_REQUIRE(std::isfinite(a.a) && std::isfinite(a.b) && std::isfinite(a.c) && std::isfinite(a.alpha) && std::isfinite(a.beta), "a coefficient is not finite");
    if (a.batch == 0 || a.rows == 0 || a.cols == 0) return APOE_OK;
    if (a.in_stride == 0) a.in_stride = a.cols;
    if (a.out_stride == 0) a.out_stride = a.cols;
    APOE_REQUIRE(a.in_stride >= a.cols && a.out_stride >= a.cols, "rows overlap: strides %llu, %llu for %u columns", (unsigned long long)a.in_stride,
                 (unsigned long long)a.out_stride, a.cols);
    const uint64_t in_matrix = (uint64_t)(a.rows - 1) * a.in_stride + a.cols, out_matrix = (uint64_t)(a.rows - 1) * a.out_stride + a.cols;
    if (a.in_batch_stride == 0) a.in_batch_stride = a.rows * a.in_stride;
    if (a.out_batch_stride == 0) a.out_batch_stride = a.rows * a.out_stride;
    APOE_REQUIRE(a.batch == 1 || (a.in_batch_stride >= in_matrix && a.out_batch_stride >= out_matrix), "matrices overlap: strides %llu, %llu",
                 (unsigned long long)a.in_batch_stride, (unsigned long long)a.out_batch_stride);
    APOE_REQUIRE(a.in && a.out, "in/out is null");
    APOE_POINTER(a.in, size_of(a.in_dtype), "in");
    APOE_POINTER(a.out, size_of(a.out_dtype), "out");
    APOE_HIP(hipSetDevice(ctx->device));
    return launch_orthogonalize(ctx, &a);
}

static int gated_residual(apoe_ctx* ctx, const apoe_gated_residual_args* args, bool grad) {
    APOE_REQUIRE(ctx && args, "ctx/args is null");
    apoe_gated_residual_args a = *args;
    APOE_REQUIRE(a.dtype <= APOE_BF16, "unknown dtype %u", a.dtype);
    APOE_REQUIRE(a.dim >= 1 && a.dim <= APOE_RESIDUAL_MAX_DIM, "dim must be in 1..%u, got %u", APOE_RESIDUAL_MAX_DIM, a.dim);
    APOE_REQUIRE(a.gate_kind <= APOE_GATE_CHANNEL, "unknown kind of gate %u", a.gate_kind);
    APOE_REQUIRE((a.gate_kind == APOE_GATE_NONE) == (a.gate == nullptr), "gate and gate_kind disagree");
    APOE_REQUIRE(a.h || (!a.gate && !a.scale && !a.w_post && !a.grad_h && !a.grad_gate && !a.grad_scale && !a.grad_w_post), "gate, scale and w_post belong to a block: h is null");
    APOE_REQUIRE(std::isfinite(a.eps) && a.eps >= 0.f, "eps must not be negative, got %g", a.eps);
    uint64_t* strides[] = {&a.x_stride, &a.h_stride, &a.gate_stride, &a.y_stride, &a.u_stride, &a.grad_y_stride, &a.grad_u_stride, &a.grad_x_stride, &a.grad_h_stride,
                           &a.grad_gate_stride};
    for (uint64_t* s : strides) {
        if (*s == 0) *s = a.dim;
        APOE_REQUIRE(*s >= a.dim, "rows overlap: stride %llu for %u columns", (unsigned long long)*s, a.dim);
    }
    if (grad) {
        APOE_REQUIRE(a.grad_y || a.grad_u, "neither grad_y nor grad_u");
        APOE_REQUIRE(a.gate_kind != APOE_GATE_NONE || !a.grad_gate, "grad_gate without a gate");
        APOE_REQUIRE(a.grad_x || a.grad_h || a.grad_gate || a.grad_scale || a.grad_w_post || a.grad_w_next, "nothing to compute");
        APOE_REQUIRE(a.grad_u || !a.grad_w_next, "grad_w_next needs grad_u");
    } else {
        APOE_REQUIRE((a.h && a.y) || a.u, "nothing to compute");
    }
    if (a.rows == 0 && !(grad && (a.grad_scale || a.grad_w_post || a.grad_w_next || (a.grad_gate && a.gate_kind == APOE_GATE_CHANNEL)))) return APOE_OK;
    APOE_REQUIRE(a.x || a.rows == 0, "x is null");
    const size_t e = size_of(a.dtype);
    APOE_POINTER(a.x, e, "x");
    APOE_POINTER(a.h, e, "h");
    APOE_POINTER(a.gate, e, "gate");
    APOE_POINTER(a.scale, 4, "scale");
    APOE_POINTER(a.w_post, 4, "w_post");
    APOE_POINTER(a.w_next, 4, "w_next");
    if (grad) {
        APOE_POINTER(a.grad_y, e, "grad_y");
        APOE_POINTER(a.grad_u, e, "grad_u");
        APOE_POINTER(a.grad_x, e, "grad_x");
        APOE_POINTER(a.grad_h, e, "grad_h");
        APOE_POINTER(a.grad_gate, e, "grad_gate");
        APOE_POINTER(a.grad_scale, 4, "grad_scale");
        APOE_POINTER(a.grad_w_post, 4, "grad_w_post");
        APOE_POINTER(a.grad_w_next, 4, "grad_w_next");
    } else {
        APOE_POINTER(a.y, e, "y");
        APOE_POINTER(a.u, e, "u");
    }
    APOE_HIP(hipSetDevice(ctx->device));
    return launch_gated_residual(ctx, &a, grad);
}

int apoe_gated_residual(apoe_ctx* ctx, const apoe_gated_residual_args* args) { return gated_residual(ctx, args, false); }

int apoe_gated_residual_grad(apoe_ctx* ctx, const apoe_gated_residual_args* args) { return gated_residual(ctx, args, true); }

} // extern "C"
