// C-ABI entry points of the operators that fit a query adapter (include/apoe.h): checks of the arguments, then the launchers.
// Nothing behind them throws: the launchers allocate nothing on the host.
#include <cmath>

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

} // extern "C"
