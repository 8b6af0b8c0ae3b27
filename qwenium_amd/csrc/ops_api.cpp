// ops_api.cpp -- the C ABI of the 8-bit float feed-forward's operators
// (include/qmoe.h): argument checks on the host, then one launch each.
#include "qmoe.h"

#include <hip/hip_runtime.h>

#include <cmath>
#include <initializer_list>
#include <string>

#include "qmoe_internal.h"

namespace {

using qmoe::set_error;

std::string str(int64_t v) { return std::to_string(v); }

int bad_value(const char* what, const std::string& expected, const std::string& got) {
    return set_error(QMOE_ERR_VALUE, std::string("qmoe: ") + what + " expected " + expected + ", got " + got);
}

int need(const char* what, const void* p) {
    return p ? QMOE_OK : set_error(QMOE_ERR_NULL, std::string("qmoe: ") + what + " expected a device pointer, got null");
}

int aligned(const char* what, const void* p, unsigned bytes) {
    return ((uintptr_t)p & (bytes - 1)) == 0 ? QMOE_OK
                                             : bad_value(what, str(bytes) + "-byte aligned", "address " + str((int64_t)(uintptr_t)p));
}

int in_range(const char* what, int64_t v, int64_t lo, int64_t hi) {
    return v >= lo && v <= hi ? QMOE_OK : bad_value(what, str(lo) + ".." + str(hi), str(v));
}

int row_type(const char* what, int32_t t) {
    return t == QMOE_TYPE_F32 || t == QMOE_TYPE_BF16
               ? QMOE_OK
               : set_error(QMOE_ERR_TYPE, std::string("qmoe: ") + what + " expected F32 (0) or BF16 (30), got type " + str(t));
}

unsigned elem(int32_t type) { return type == QMOE_TYPE_BF16 ? 2 : 4; }

// A buffer of the call: outputs overlap nothing else, except where a call takes the very same buffer.
struct Buffer {
    const char* name;
    const void* at;
    uint64_t bytes;
    bool overlaps(const Buffer& o) const {
        const uintptr_t p = (uintptr_t)at, q = (uintptr_t)o.at;
        return at && o.at && p < q + o.bytes && q < p + bytes;
    }
};
int apart(std::initializer_list<Buffer> outs, std::initializer_list<Buffer> ins) {
    for (const Buffer* o = outs.begin(); o != outs.end(); ++o) {
        for (const Buffer* r = outs.begin(); r != o; ++r)
            if (o->overlaps(*r)) return bad_value(o->name, std::string("a buffer distinct from ") + r->name, "an overlapping one");
        for (const Buffer& i : ins)
            if (o->overlaps(i)) return bad_value(o->name, std::string("a buffer distinct from ") + i.name, "an overlapping one");
    }
    return QMOE_OK;
}

int done(hipError_t err, const char* what) { return err == hipSuccess ? QMOE_OK : qmoe::hip_error(err, what); }

// n_tokens, top_k, and their product as an int
int check_tokens(int32_t n_tokens, int32_t top_k) {
    if (int rc = in_range("n_tokens", n_tokens, 0, INT32_MAX)) return rc;
    if (int rc = in_range("top_k", top_k, 1, 64)) return rc;
    return in_range("n_tokens * top_k", (int64_t)n_tokens * top_k, 0, 1 << 30);
}

// A launch holds below 2^32 threads; a row takes up to 1024 (16 a block of the quantization, whose last workgroup of 16
// blocks is a whole one).
constexpr int64_t kMaxRowLaunch = (1 << 22) - 1, kMaxBlocks = (1 << 28) - 16;

#define QMOE_TRY(expr)                   \
    do {                                 \
        if (int rc_ = (expr)) return rc_; \
    } while (0)

}  // namespace

extern "C" {

int qmoe_fp8_quantize(const void* x, int32_t x_type, int32_t n_rows, int32_t n_cols, int32_t act, uint8_t* q,
                      float* scale, void* hip_stream) {
    qmoe::clear_error();
    QMOE_TRY(row_type("x_type", x_type));
    QMOE_TRY(in_range("n_rows", n_rows, 0, INT32_MAX));
    QMOE_TRY(in_range("n_cols", n_cols, 1, 1 << 28));
    QMOE_TRY(in_range("act", act, QMOE_FP8_ACT_NONE, QMOE_FP8_ACT_GEGLU));
    QMOE_TRY(in_range("n_rows * ceil(n_cols/128)", (int64_t)n_rows * ((n_cols + 127) / 128), 0, kMaxBlocks));
    if (n_rows == 0) return QMOE_OK;
    QMOE_TRY(need("x", x));
    QMOE_TRY(need("q", q));
    QMOE_TRY(need("scale", scale));
    QMOE_TRY(aligned("x", x, elem(x_type)));
    QMOE_TRY(aligned("scale", scale, 4));
    const uint64_t v = (uint64_t)n_rows * n_cols;
    QMOE_TRY(apart({{"q", q, v}, {"scale", scale, 4 * (uint64_t)n_rows * ((n_cols + 127) / 128)}},
                   {{"x", x, v * elem(x_type) * (act == QMOE_FP8_ACT_NONE ? 1 : 2)}}));
    return done(qmoe::launch_fp8_quantize(x, x_type == QMOE_TYPE_BF16, n_rows, n_cols, act, q, scale, (hipStream_t)hip_stream),
                "fp8_quantize kernel");
}

int qmoe_fp8_matmul(const uint8_t* a, const float* a_scale, int32_t a_rows, const uint8_t* w, const float* w_scale,
                    int32_t n_experts, int32_t n, int32_t k, const int32_t* offsets, const int32_t* rows, int32_t n_rows,
                    void* y, int32_t y_type, void* hip_stream) {
    qmoe::clear_error();
    QMOE_TRY(row_type("y_type", y_type));
    QMOE_TRY(in_range("n_rows", n_rows, 0, 1 << 30));
    QMOE_TRY(in_range("a_rows", a_rows, 0, INT32_MAX));
    QMOE_TRY(in_range("n", n, 1, 1 << 24));
    QMOE_TRY(in_range("k", k, 16, 1 << 20));
    if (k % 16) return bad_value("k", "a multiple of 16", str(k));
    if (offsets) QMOE_TRY(in_range("n_experts", n_experts, 1, 1024));
    else if (n_experts != 1) return bad_value("n_experts", "1 without offsets", str(n_experts));
    if (!rows && a_rows != n_rows) return bad_value("a_rows", str(n_rows) + " (n_rows) without rows", str(a_rows));
    if (n_rows == 0) return QMOE_OK;
    if (a_rows == 0) return bad_value("a_rows", "at least 1", "0");
    QMOE_TRY(need("a", a));
    QMOE_TRY(need("a_scale", a_scale));
    QMOE_TRY(need("w", w));
    QMOE_TRY(need("w_scale", w_scale));
    QMOE_TRY(need("y", y));
    QMOE_TRY(aligned("a", a, 16));
    QMOE_TRY(aligned("w", w, 16));
    QMOE_TRY(aligned("a_scale", a_scale, 4));
    QMOE_TRY(aligned("w_scale", w_scale, 4));
    QMOE_TRY(aligned("offsets", offsets, 4));
    QMOE_TRY(aligned("rows", rows, 4));
    QMOE_TRY(aligned("y", y, elem(y_type)));
    const uint64_t kb = (k + 127) / 128, nb = (n + 127) / 128, e = (uint64_t)n_experts;
    QMOE_TRY(apart({{"y", y, (uint64_t)n_rows * n * elem(y_type)}},
                   {{"a", a, (uint64_t)a_rows * k}, {"a_scale", a_scale, 4 * a_rows * kb}, {"w", w, e * n * k},
                    {"w_scale", w_scale, 4 * e * nb * kb}, {"offsets", offsets, 4 * (e + 1)}, {"rows", rows, 4 * (uint64_t)n_rows}}));
    qmoe::Fp8Product p{};
    p.a = a;
    p.sa = a_scale;
    p.w = w;
    p.sw = w_scale;
    p.offsets = offsets;
    p.rows = rows;
    p.y = y;
    p.a_rows = a_rows;
    p.E = n_experts;
    p.N = n;
    p.K = k;
    p.R = n_rows;
    const hipError_t err = qmoe::launch_fp8_matmul(p, y_type == QMOE_TYPE_BF16, (hipStream_t)hip_stream);
    if (err == hipErrorInvalidConfiguration)
        return bad_value("n_rows x n", "fewer than 2^32 threads in tiles of its rows and columns", str(n_rows) + " x " + str(n));
    return done(err, "fp8_matmul kernel");
}

int qmoe_sort_tokens(const int32_t* topk_idx, int32_t n_tokens, int32_t top_k, int32_t n_experts, int32_t* offsets,
                     int32_t* rows, int32_t* tokens, int32_t* place, void* hip_stream) {
    qmoe::clear_error();
    QMOE_TRY(check_tokens(n_tokens, top_k));
    QMOE_TRY(in_range("n_experts", n_experts, 1, 1024));
    QMOE_TRY(need("offsets", offsets));
    QMOE_TRY(aligned("offsets", offsets, 4));
    if (n_tokens > 0) {
        QMOE_TRY(need("topk_idx", topk_idx));
        QMOE_TRY(need("rows", rows));
        QMOE_TRY(need("tokens", tokens));
        QMOE_TRY(need("place", place));
        QMOE_TRY(aligned("topk_idx", topk_idx, 4));
        QMOE_TRY(aligned("rows", rows, 4));
        QMOE_TRY(aligned("tokens", tokens, 4));
        QMOE_TRY(aligned("place", place, 4));
        const uint64_t list = 4 * (uint64_t)n_tokens * top_k;
        QMOE_TRY(apart({{"offsets", offsets, 4 * ((uint64_t)n_experts + 1)}, {"rows", rows, list}, {"tokens", tokens, list},
                        {"place", place, list}},
                       {{"topk_idx", topk_idx, list}}));
    }
    return done(qmoe::launch_sort_tokens(topk_idx, n_tokens, top_k, n_experts, offsets, rows, tokens, place,
                                         (hipStream_t)hip_stream),
                "sort_tokens kernel");
}

int qmoe_gather_tokens(const void* x, int32_t elem_bytes, int32_t n_tokens, int32_t n_cols, int32_t top_k,
                       int32_t n_experts, const int32_t* offsets, const int32_t* place, void* y, void* hip_stream) {
    qmoe::clear_error();
    QMOE_TRY(check_tokens(n_tokens, top_k));
    QMOE_TRY(in_range("n_tokens", n_tokens, 0, kMaxRowLaunch));
    QMOE_TRY(in_range("n_cols", n_cols, 1, 1 << 20));
    QMOE_TRY(in_range("n_experts", n_experts, 1, 1024));
    if (elem_bytes != 1 && elem_bytes != 2 && elem_bytes != 4) return bad_value("elem_bytes", "1, 2 or 4", str(elem_bytes));
    if (n_tokens == 0) return QMOE_OK;
    QMOE_TRY(need("x", x));
    QMOE_TRY(need("offsets", offsets));
    QMOE_TRY(need("place", place));
    QMOE_TRY(need("y", y));
    QMOE_TRY(aligned("x", x, (unsigned)elem_bytes));
    QMOE_TRY(aligned("y", y, (unsigned)elem_bytes));
    QMOE_TRY(aligned("offsets", offsets, 4));
    QMOE_TRY(aligned("place", place, 4));
    const uint64_t row = (uint64_t)n_cols * elem_bytes, list = (uint64_t)n_tokens * top_k;
    QMOE_TRY(apart({{"y", y, list * row}}, {{"x", x, n_tokens * row}, {"offsets", offsets, 4 * ((uint64_t)n_experts + 1)},
                                             {"place", place, 4 * list}}));
    return done(qmoe::launch_gather_tokens(x, elem_bytes, n_tokens, n_cols, top_k, offsets + n_experts, place, y,
                                           (hipStream_t)hip_stream),
                "gather_tokens kernel");
}

int qmoe_combine_tokens(const void* ys, int32_t x_type, int32_t n_tokens, int32_t n_cols, int32_t top_k,
                        const int32_t* place, const float* w, const void* residual, void* y, void* hip_stream) {
    qmoe::clear_error();
    QMOE_TRY(row_type("x_type", x_type));
    QMOE_TRY(check_tokens(n_tokens, top_k));
    QMOE_TRY(in_range("n_tokens", n_tokens, 0, kMaxRowLaunch));
    QMOE_TRY(in_range("n_cols", n_cols, 1, 1 << 20));
    if (n_tokens == 0) return QMOE_OK;
    QMOE_TRY(need("ys", ys));
    QMOE_TRY(need("place", place));
    QMOE_TRY(need("y", y));
    QMOE_TRY(aligned("ys", ys, elem(x_type)));
    QMOE_TRY(aligned("residual", residual, elem(x_type)));
    QMOE_TRY(aligned("y", y, elem(x_type)));
    QMOE_TRY(aligned("place", place, 4));
    QMOE_TRY(aligned("w", w, 4));
    const uint64_t row = (uint64_t)n_cols * elem(x_type), list = (uint64_t)n_tokens * top_k;
    QMOE_TRY(apart({{"y", y, n_tokens * row}}, {{"ys", ys, list * row}, {"place", place, 4 * list}, {"w", w, 4 * list},
                                                 {"residual", residual == y ? nullptr : residual, n_tokens * row}}));
    return done(qmoe::launch_combine_tokens(ys, x_type == QMOE_TYPE_BF16, n_tokens, n_cols, top_k, place, w, residual, y,
                                            (hipStream_t)hip_stream),
                "combine_tokens kernel");
}

int qmoe_combine_tokens_backward(const void* dy, const void* ys, int32_t x_type, int32_t n_tokens, int32_t n_cols,
                                 int32_t top_k, int32_t n_experts, const int32_t* offsets, const int32_t* place,
                                 const float* w, void* dys, float* dw, void* hip_stream) {
    qmoe::clear_error();
    QMOE_TRY(row_type("x_type", x_type));
    QMOE_TRY(check_tokens(n_tokens, top_k));
    QMOE_TRY(in_range("n_tokens", n_tokens, 0, kMaxRowLaunch));
    QMOE_TRY(in_range("n_cols", n_cols, 1, 1 << 20));
    QMOE_TRY(in_range("n_experts", n_experts, 1, 1024));
    if (n_tokens == 0) return QMOE_OK;
    QMOE_TRY(need("dy", dy));
    QMOE_TRY(need("ys", ys));
    QMOE_TRY(need("offsets", offsets));
    QMOE_TRY(need("place", place));
    QMOE_TRY(need("w", w));
    QMOE_TRY(need("dys", dys));
    QMOE_TRY(need("dw", dw));
    QMOE_TRY(aligned("dy", dy, elem(x_type)));
    QMOE_TRY(aligned("ys", ys, elem(x_type)));
    QMOE_TRY(aligned("dys", dys, elem(x_type)));
    QMOE_TRY(aligned("offsets", offsets, 4));
    QMOE_TRY(aligned("place", place, 4));
    QMOE_TRY(aligned("w", w, 4));
    QMOE_TRY(aligned("dw", dw, 4));
    const uint64_t row = (uint64_t)n_cols * elem(x_type), list = (uint64_t)n_tokens * top_k;
    QMOE_TRY(apart({{"dys", dys, list * row}, {"dw", dw, 4 * list}},
                   {{"dy", dy, n_tokens * row}, {"ys", ys, list * row}, {"offsets", offsets, 4 * ((uint64_t)n_experts + 1)},
                    {"place", place, 4 * list}, {"w", w, 4 * list}}));
    return done(qmoe::launch_combine_tokens_bwd(dy, ys, x_type == QMOE_TYPE_BF16, n_tokens, n_cols, top_k,
                                                offsets + n_experts, place, w, dys, dw, (hipStream_t)hip_stream),
                "combine_tokens_backward kernel");
}

int qmoe_residual_norm(const qmoe_norm_args* a, int32_t n_tokens, int32_t n_embd, void* hip_stream) {
    qmoe::clear_error();
    if (!a) return set_error(QMOE_ERR_NULL, "qmoe: args expected non-null, got null");
    QMOE_TRY(row_type("x_type", a->x_type));
    QMOE_TRY(in_range("n_tokens", n_tokens, 0, kMaxRowLaunch));
    QMOE_TRY(in_range("n_embd", n_embd, 1, 16384));
    QMOE_TRY(in_range("gate_act", a->gate_act, QMOE_GATE_NONE, QMOE_GATE_SILU));
    if (!(a->eps >= 0.0f) || std::isinf(a->eps)) return bad_value("eps", "a number >= 0", std::to_string(a->eps));
    if ((a->gate != nullptr) != (a->gate_act != QMOE_GATE_NONE))
        return bad_value("gate_act", a->gate ? "SIGMOID (1) or SILU (2) with a gate" : "NONE (0) without a gate", str(a->gate_act));
    if (!a->y && (a->post_w || a->gate || a->scale_v))
        return bad_value("y", "the block's output with post_w, gate or scale_v", "null");
    if ((a->q != nullptr) != (a->q_scale != nullptr))
        return set_error(QMOE_ERR_NULL, "qmoe: q and q_scale expected both or neither, got one");
    if (n_tokens == 0) return QMOE_OK;
    QMOE_TRY(need("x", a->x));
    QMOE_TRY(need("h", a->h));
    if (a->y) QMOE_TRY(need("x_out", a->x_out));
    const unsigned e = elem(a->x_type);
    QMOE_TRY(aligned("x", a->x, e));
    QMOE_TRY(aligned("y", a->y, e));
    QMOE_TRY(aligned("gate", a->gate, e));
    QMOE_TRY(aligned("x_out", a->x_out, e));
    QMOE_TRY(aligned("h", a->h, e));
    QMOE_TRY(aligned("post_w", a->post_w, 4));
    QMOE_TRY(aligned("scale_v", a->scale_v, 4));
    QMOE_TRY(aligned("w", a->w, 4));
    QMOE_TRY(aligned("q_scale", a->q_scale, 4));
    const uint64_t v = (uint64_t)n_tokens * n_embd, vec = 4 * (uint64_t)n_embd;
    auto other = [&](const void* in) { return in == a->x_out ? nullptr : in; };  // x' may replace x or y
    const Buffer x{"x", a->x, v * e}, y{"y", a->y, v * e}, gate{"gate", a->gate, v * e}, post_w{"post_w", a->post_w, vec},
        scale_v{"scale_v", a->scale_v, vec}, w{"w", a->w, vec};
    QMOE_TRY(apart({{"x_out", a->y ? a->x_out : nullptr, v * e}},
                   {{"x", other(a->x), v * e}, {"y", other(a->y), v * e}, gate, post_w, scale_v, w}));
    QMOE_TRY(apart({{"h", a->h, v * e}, {"q", a->q, v}, {"q_scale", a->q_scale, 4 * (uint64_t)n_tokens * ((n_embd + 127) / 128)}},
                   {x, y, gate, post_w, scale_v, w, {"x_out", a->y ? a->x_out : nullptr, v * e}}));
    qmoe::ResidualNorm p{};
    p.x = a->x;
    p.y = a->y;
    p.gate = a->gate;
    p.post_w = a->post_w;
    p.scale_v = a->scale_v;
    p.w = a->w;
    p.x_out = a->x_out;
    p.h = a->h;
    p.q = a->q;
    p.q_scale = a->q_scale;
    p.scale = a->scale;
    p.eps = a->eps;
    p.H = n_embd;
    p.gate_act = a->gate_act;
    return done(qmoe::launch_residual_norm(p, a->x_type == QMOE_TYPE_BF16, n_tokens, (hipStream_t)hip_stream),
                "residual_norm kernel");
}

}  // extern "C"
