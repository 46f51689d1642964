// C ABI (include/decik_nf4.h) of the operators around the NF4 projections: seeded dropout, norms and
// rotation of q and k, linears in 8-bit integers. Argument checks and launches.
#include <cmath>
#include <cstdio>

#include "dk_internal.h"

using namespace dk;

namespace {

int check_launch(hipError_t e, const char* what) {
    if (e == hipSuccess) return 0;
    char msg[256];
    snprintf(msg, sizeof(msg), "%s: %s", what, hipGetErrorString(e));
    return dk_fail(msg);
}

bool is_dtype(int d) { return d == DK_FP16 || d == DK_BF16 || d == DK_FP32; }

bool aligned_to(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

// everything of a dropout call but its tensors
int dropout_common(DropoutArgs* a, int in_dtype, int out_dtype, const int64_t* rng, const double* p, int nb,
                   int64_t rows, int64_t width) {
    if (nb < 1 || nb > kDropoutMaxBranches) return dk_fail("dk_dropout: 1 to 4 branches");
    if (!is_dtype(in_dtype) || !is_dtype(out_dtype) ||
        (in_dtype != out_dtype && in_dtype != DK_FP32 && out_dtype != DK_FP32))
        return dk_fail("dk_dropout: types must be equal, or one of them fp32");
    if (rows < 0 || width < 0) return dk_fail("dk_dropout: negative size");
    if (p == nullptr) return dk_fail("dk_dropout: null pointer");
    for (int b = 0; b < nb; ++b) {
        if (!(p[b] >= 0.0 && p[b] <= 1.0)) return dk_fail("dk_dropout: p must be in [0, 1]");
        a->thr[b] = (uint32_t)std::nearbyint(p[b] * 65536.0);
        a->scale[b] = a->thr[b] < 65536u ? (float)(65536.0 / (65536.0 - a->thr[b])) : 0.0f;
    }
    // columns are 32-bit numbers in the kernel
    const int64_t limit = int64_t(1) << 31;
    if (width > 0xFFFFFFF0ll) return dk_fail("dk_dropout: width must be below 2^32 - 16");
    const int64_t groups = (width + 7) / 8;
    if (groups > 0 && rows > (limit - 1) / groups)
        return dk_fail("dk_dropout: rows * ceil(width / 8) must be below 2^31");
    if (rows * groups > 0 && (rng == nullptr || !aligned_to(rng, 8)))
        return dk_fail("dk_dropout: rng must be two int64 in device memory");
    a->rng = rng;
    a->width = (uint32_t)width;
    a->groups = (uint32_t)groups;
    a->items = (uint32_t)(rows * groups);
    a->nb = nb;
    return 0;
}

// everything of a norm / rotation call but the gradients
int qk_rope_common(const dk_qk_rope* d, QkRopeArgs* a) {
    if (d == nullptr) return dk_fail("dk_qk_rope: null descriptor");
    if (d->dtype != DK_FP16 && d->dtype != DK_BF16) return dk_fail("dk_qk_rope: q and k must be fp16 or bf16");
    if (d->head_dim < 16 || d->head_dim > 512 || d->head_dim % 16 != 0)
        return dk_fail("dk_qk_rope: head_dim must be a multiple of 16 from 16 to 512");
    if (d->n_heads < 1 || d->n_kv_heads < 1 || d->n_heads > 65536 || d->n_kv_heads > 65536)
        return dk_fail("dk_qk_rope: 1 to 65536 heads each");
    if (d->batch < 0 || d->tokens < 0 || d->tokens >= INT32_MAX || d->batch >= INT32_MAX ||
        d->batch * d->tokens > (int64_t)INT32_MAX - kQkMaxWaves)
        return dk_fail("dk_qk_rope: batch * tokens must be non-negative and below 2^31 - 4096");
    if ((d->q_weight == nullptr) != (d->k_weight == nullptr))
        return dk_fail("dk_qk_rope: norm weights for both q and k, or for neither");
    if (d->q_weight != nullptr && !is_dtype(d->w_dtype)) return dk_fail("dk_qk_rope: unknown norm weight type");
    const bool axes = d->n_axes != 0, empty = d->batch * d->tokens == 0;
    if (!axes && !empty && (d->cos == nullptr || d->sin == nullptr || !aligned_to(d->cos, 4) || !aligned_to(d->sin, 4)))
        return dk_fail("dk_qk_rope: without axes cos and sin must be set");
    if (axes) {
        if (d->n_axes < 1 || d->n_axes > 4) return dk_fail("dk_qk_rope: 1 to 4 axes");
        if (!empty && (d->positions == nullptr || d->inv_freq == nullptr))
            return dk_fail("dk_qk_rope: axes need positions and inv_freq");
        int sum = 0;
        for (int i = 0; i < d->n_axes; ++i) {
            if (d->sections[i] < 0 || d->sections[i] > d->head_dim)
                return dk_fail("dk_qk_rope: sections must be non-negative and add up to head_dim / 2");
            sum += d->sections[i];
        }
        if (sum != d->head_dim / 2)
            return dk_fail("dk_qk_rope: sections must be non-negative and add up to head_dim / 2");
        if (d->interleaved)
            for (int i = 1; i < d->n_axes; ++i)
                if (d->sections[i] > 0 && d->n_axes * (d->sections[i] - 1) + i >= sum)
                    return dk_fail("dk_qk_rope: an interleaved axis has more frequencies than its places");
    }
    a->q = d->q;
    a->k = d->k;
    a->gq = d->grad_q;
    a->gk = d->grad_k;
    a->oq = d->q_out;
    a->ok = d->k_out;
    a->ldq = d->ld_q;
    a->ldk = d->ld_k;
    a->ldoq = d->ld_q_out;
    a->ldok = d->ld_k_out;
    a->qw = d->q_weight;
    a->kw = d->k_weight;
    a->cos = d->cos;
    a->sin = d->sin;
    a->table_batch = d->table_batch_stride;
    a->pos = d->positions;
    a->inv_freq = d->inv_freq;
    a->pos_axis = d->pos_axis_stride;
    a->pos_batch = d->pos_batch_stride;
    for (int i = 0; i < 4; ++i) a->section[i] = i < d->n_axes ? d->sections[i] : 0;
    a->n_axes = d->n_axes;
    a->interleaved = d->interleaved;
    a->pos64 = d->positions_int64;
    a->w_dtype = d->w_dtype;
    a->tokens = (uint32_t)d->tokens;
    a->rows = (uint32_t)(d->batch * d->tokens);
    a->hq = d->n_heads;
    a->hk = d->n_kv_heads;
    a->d = d->head_dim;
    a->eps = d->eps;
    a->inv_d = 1.0f / (float)d->head_dim;
    return 0;
}

constexpr int64_t kInt8MaxK = 131071, kInt8MaxLd = int64_t(1) << 23, kInt8MaxRows = int64_t(1) << 23;

bool int8_sizes(int64_t m, int64_t n, int64_t k) {
    // (work-groups of the largest outputs fit a launch)
    return m >= 0 && n >= 0 && k >= 1 && k <= kInt8MaxK && m < kInt8MaxRows && n < kInt8MaxRows &&
           m * n < (int64_t(1) << 38);
}

bool int8_rows_ok(const void* p, int64_t ld, int64_t cols) {
    return aligned_to(p, 16) && ld % 16 == 0 && ld >= (cols + 15) / 16 * 16 && ld < kInt8MaxLd;
}

bool int4_sizes(int64_t m, int64_t n, int64_t k) {
    // (work-groups of the largest outputs fit a launch)
    const int64_t most = int64_t(1) << 23, area = int64_t(1) << 37;
    return m >= 0 && n >= 0 && m < most && n < most && k >= 1 && k <= (int64_t(1) << 20) && m * n < area && m * k < area;
}

// workspace of a call: partial sums, then room for x with aligned rows (few tokens take it as it is)
int64_t int4_bytes(const Int4Plan& p, bool copy, int64_t m, int64_t sum, int64_t* partial) {
    const int64_t sums = (p.partial_bytes + 15) / 16 * 16;
    if (partial != nullptr) *partial = sums;
    return sums + (copy && !p.few ? m * ((sum + 7) / 8 * 16) : 0);
}

const char* const kInt4Sizes = "dk_int4_linear: 0 <= m, n < 2^23, m n < 2^37, m k < 2^37, 1 <= k <= 2^20";

bool rows_fit(int64_t ld, int heads, int d) { return ld >= (int64_t)heads * d; }

// everything of a residual-stream call but its outputs and gradients
int residual_norm_common(const dk_residual_norm* d, ResidualNormArgs* a) {
    if (d == nullptr) return dk_fail("dk_residual_norm: null descriptor");
    const int x = d->x_dtype;
    if (!is_dtype(x) || (d->stream_dtype != x && d->stream_dtype != DK_FP32) ||
        (d->y_dtype != x && d->y_dtype != DK_FP32))
        return dk_fail("dk_residual_norm: x must be fp16, bf16 or fp32, the stream and y of x's type or fp32");
    if (d->width < 1 || d->width > kNormMaxWidth) return dk_fail("dk_residual_norm: width must be 1 to 16384");
    if (d->rows < 0 || d->rows >= (int64_t)INT32_MAX - 65535)
        return dk_fail("dk_residual_norm: rows must be non-negative and below 2^31 - 65536");
    if ((d->weight != nullptr && !is_dtype(d->weight_dtype)) || (d->post_weight != nullptr && !is_dtype(d->post_dtype)))
        return dk_fail("dk_residual_norm: unknown weight type");
    if (d->gate_kind < DK_GATE_NONE || d->gate_kind > DK_GATE_ELEMENT)
        return dk_fail("dk_residual_norm: unknown kind of gate");
    if (d->gate_kind != DK_GATE_NONE && !is_dtype(d->gate_dtype)) return dk_fail("dk_residual_norm: unknown gate type");
    const bool empty = d->rows == 0;
    if (!empty && d->x == nullptr) return dk_fail("dk_residual_norm: null pointer");
    if (d->gate_kind != DK_GATE_NONE && !empty && d->gate == nullptr) return dk_fail("dk_residual_norm: null gate");
    if (d->rows > 1 && (d->ld_x < 0 || d->ld_residual < 0 || d->ld_grad_h < 0 || d->ld_grad_y < 0 || d->ld_gate < 0))
        return dk_fail("dk_residual_norm: negative row stride");
    a->x = d->x;
    a->res = d->residual;
    a->w = d->weight;
    a->pw = d->post_weight;
    a->gate = d->gate;
    a->ldx = d->ld_x;
    a->ldr = d->ld_residual;
    a->ldgate = d->ld_gate;
    a->rows = (int32_t)d->rows;
    a->width = (int32_t)d->width;
    a->w_dtype = d->weight_dtype;
    a->pw_dtype = d->post_dtype;
    a->gate_dtype = d->gate_dtype;
    a->gate_kind = d->gate_kind;
    a->scale = d->residual_scale;
    a->eps = d->eps;
    a->inv_width = 1.0f / (float)d->width;
    return 0;
}

// which gradients of a backward are sums over the rows
int residual_norm_sums(const dk_residual_norm* d, ResidualNormArgs* a) {
    if (d->dweight != nullptr && d->weight == nullptr)
        return dk_fail("dk_residual_norm_bwd: no weight to take a gradient of");
    if (d->dpost_weight != nullptr && d->post_weight == nullptr)
        return dk_fail("dk_residual_norm_bwd: no post weight to take a gradient of");
    if (d->dgate != nullptr && d->gate_kind == DK_GATE_NONE)
        return dk_fail("dk_residual_norm_bwd: no gate to take a gradient of");
    a->slab_w = d->dweight != nullptr;
    a->slab_q = d->dpost_weight != nullptr || (d->dgate != nullptr && d->gate_kind == DK_GATE_CHANNEL);
    a->nslabs = (int)a->slab_w + (int)a->slab_q;
    return 0;
}

int64_t residual_norm_bytes(const ResidualNormArgs& a) {
    return (int64_t)residual_norm_groups(a.rows, a.width, true) * a.nslabs * a.width * (int64_t)sizeof(float);
}

}  // namespace

extern "C" {

int dk_dropout_fwd(const void* x, int x_dtype, int64_t ldx, const int64_t* rng, const double* p, int nbranches,
                   void* const* outs, int out_dtype, const int64_t* ldo, int64_t rows, int64_t width, void* stream) {
    dk_clear_error();
    DropoutArgs a{};
    if (int rc = dropout_common(&a, x_dtype, out_dtype, rng, p, nbranches, rows, width)) return rc;
    if (a.items == 0) return 0;
    if (x == nullptr || outs == nullptr || ldo == nullptr) return dk_fail("dk_dropout_fwd: null pointer");
    if (rows > 1 && ldx < 0) return dk_fail("dk_dropout_fwd: negative row stride");
    a.in[0] = x;
    a.ld_in[0] = ldx;
    for (int b = 0; b < nbranches; ++b) {
        if (outs[b] == nullptr) return dk_fail("dk_dropout_fwd: null pointer");
        if (rows > 1 && ldo[b] < width) return dk_fail("dk_dropout_fwd: output rows overlap");
        a.out[b] = outs[b];
        a.ld_out[b] = ldo[b];
    }
    return check_launch(launch_dropout(a, x_dtype, out_dtype, false, static_cast<hipStream_t>(stream)),
                        "dk_dropout_fwd launch");
}

int dk_dropout_bwd(const void* const* grads, int grad_dtype, const int64_t* ldg, const int64_t* rng, const double* p,
                   int nbranches, void* dx, int dx_dtype, int64_t lddx, int64_t rows, int64_t width, void* stream) {
    dk_clear_error();
    DropoutArgs a{};
    if (int rc = dropout_common(&a, grad_dtype, dx_dtype, rng, p, nbranches, rows, width)) return rc;
    if (a.items == 0) return 0;
    if (grads == nullptr || ldg == nullptr || dx == nullptr) return dk_fail("dk_dropout_bwd: null pointer");
    if (rows > 1 && lddx < width) return dk_fail("dk_dropout_bwd: output rows overlap");
    for (int b = 0; b < nbranches; ++b) {
        if (grads[b] != nullptr && rows > 1 && ldg[b] < 0) return dk_fail("dk_dropout_bwd: negative row stride");
        a.in[b] = grads[b];
        a.ld_in[b] = ldg[b];
    }
    a.out[0] = dx;
    a.ld_out[0] = lddx;
    return check_launch(launch_dropout(a, grad_dtype, dx_dtype, true, static_cast<hipStream_t>(stream)),
                        "dk_dropout_bwd launch");
}

int dk_qk_rope_fwd(const dk_qk_rope* d, void* stream) {
    dk_clear_error();
    QkRopeArgs a{};
    if (int rc = qk_rope_common(d, &a)) return rc;
    if (a.rows == 0) return 0;
    if (a.q == nullptr || a.k == nullptr || a.oq == nullptr || a.ok == nullptr)
        return dk_fail("dk_qk_rope_fwd: null pointer");
    if (a.rows > 1 && (!rows_fit(a.ldq, a.hq, a.d) || !rows_fit(a.ldk, a.hk, a.d)))
        return dk_fail("dk_qk_rope_fwd: row strides must cover the heads");
    return check_launch(launch_qk_rope(a, d->dtype, d->q_weight != nullptr, d->n_axes != 0, false, nullptr,
                                       nullptr, static_cast<hipStream_t>(stream)),
                        "dk_qk_rope_fwd launch");
}

int64_t dk_qk_rope_bwd_workspace(const dk_qk_rope* d) {
    dk_clear_error();
    QkRopeArgs a{};
    if (qk_rope_common(d, &a) != 0) return -1;
    if (d->dw_q == nullptr || d->q_weight == nullptr || a.rows == 0) return 0;
    return (int64_t)qk_rope_groups(a.rows, qk_rope_passes(a.hq, a.hk, a.d), true) * 2 * a.d * (int64_t)sizeof(float);
}

int dk_qk_rope_bwd(const dk_qk_rope* d, void* workspace, int64_t workspace_bytes, void* stream) {
    dk_clear_error();
    QkRopeArgs a{};
    if (int rc = qk_rope_common(d, &a)) return rc;
    const bool norm = d->q_weight != nullptr;
    if ((d->dw_q == nullptr) != (d->dw_k == nullptr))
        return dk_fail("dk_qk_rope_bwd: dw_q and dw_k both, or neither");
    if (d->dw_q != nullptr && !norm) return dk_fail("dk_qk_rope_bwd: no norm weights to take a gradient of");
    if (a.rows != 0) {
        if (a.gq == nullptr || a.gk == nullptr || a.oq == nullptr || a.ok == nullptr)
            return dk_fail("dk_qk_rope_bwd: null pointer");
        if (norm && (a.q == nullptr || a.k == nullptr)) return dk_fail("dk_qk_rope_bwd: norms need q and k again");
        if (a.rows > 1 && norm && (!rows_fit(a.ldq, a.hq, a.d) || !rows_fit(a.ldk, a.hk, a.d)))
            return dk_fail("dk_qk_rope_bwd: row strides must cover the heads");
        if (a.rows > 1 && (!rows_fit(a.ldoq, a.hq, a.d) || !rows_fit(a.ldok, a.hk, a.d)))
            return dk_fail("dk_qk_rope_bwd: row strides must cover the heads");
        if (d->dw_q != nullptr) {
            const int64_t need = dk_qk_rope_bwd_workspace(d);
            if (workspace == nullptr || workspace_bytes < need || !aligned_to(workspace, 16))
                return dk_fail("dk_qk_rope_bwd: workspace too small (dk_qk_rope_bwd_workspace)");
            a.slabs = static_cast<float*>(workspace);
        }
    } else if (d->dw_q == nullptr) {
        return 0;
    }
    return check_launch(launch_qk_rope(a, d->dtype, norm, d->n_axes != 0, true, d->dw_q, d->dw_k,
                                       static_cast<hipStream_t>(stream)),
                        "dk_qk_rope_bwd launch");
}

int dk_int8_quantize(const void* x, int x_dtype, int64_t ldx, const float* col_scale, int8_t* q, int64_t ldq,
                     float* scale, int64_t rows, int64_t k, void* stream) {
    dk_clear_error();
    if (!is_dtype(x_dtype)) return dk_fail("dk_int8_quantize: unknown type");
    if (rows < 0 || rows >= kInt8MaxRows || k < 1 || k > kInt8MaxK)
        return dk_fail("dk_int8_quantize: 0 <= rows < 2^23, 1 <= k <= 131071");
    if (rows == 0) return 0;
    if (x == nullptr || q == nullptr || scale == nullptr) return dk_fail("dk_int8_quantize: null pointer");
    if (rows > 1 && ldx < 0) return dk_fail("dk_int8_quantize: negative row stride");
    if (!int8_rows_ok(q, ldq, k))
        return dk_fail("dk_int8_quantize: q must be 16-byte aligned, its row stride a multiple of 16 that covers k");
    Int8QuantArgs a{x, col_scale, q, scale, ldx, ldq, rows, (int32_t)k};
    return check_launch(launch_int8_quantize(a, x_dtype, static_cast<hipStream_t>(stream)), "dk_int8_quantize launch");
}

int64_t dk_int8_linear_workspace(int transposed, int64_t m, int64_t n, int64_t k) {
    dk_clear_error();
    if (!int8_sizes(m, n, k)) {
        dk_fail("dk_int8_linear: 0 <= m, n < 2^23, m n < 2^38, 1 <= k <= 131071");
        return -1;
    }
    return int8_plan(m, n, k, transposed != 0).partial_bytes;
}

int dk_int8_linear_plan(int transposed, int64_t m, int64_t n, int64_t k, int32_t* out) {
    dk_clear_error();
    if (!int8_sizes(m, n, k) || out == nullptr)
        return dk_fail("dk_int8_linear_plan: 0 <= m, n < 2^23, m n < 2^38, 1 <= k <= 131071, out set");
    const Int8Plan p = int8_plan(m, n, k, transposed != 0);
    out[0] = p.few ? 0 : p.tm;
    out[1] = p.few ? 16 : p.bn;
    out[2] = p.splits;
    out[3] = m > 0 && int8_fused(m, k, transposed != 0) ? 1 : 0;
    return 0;
}

int dk_int8_linear(int transposed, const int8_t* xq, int64_t ldx, const float* xs, const int8_t* wq, int64_t ldw,
                   const float* ws, const void* bias, int bias_dtype, void* y, int y_dtype, int64_t ldy, int64_t m,
                   int64_t n, int64_t k, void* workspace, int64_t workspace_bytes, void* stream) {
    dk_clear_error();
    if (!int8_sizes(m, n, k)) return dk_fail("dk_int8_linear: 0 <= m, n < 2^23, m n < 2^38, 1 <= k <= 131071");
    if (!is_dtype(y_dtype) || (bias != nullptr && !is_dtype(bias_dtype)))
        return dk_fail("dk_int8_linear: unknown type");
    if (transposed && (ws != nullptr || bias != nullptr))
        return dk_fail("dk_int8_linear: the transposed product has neither channel scales nor bias");
    if (m == 0 || n == 0) return 0;
    if (xq == nullptr || xs == nullptr || wq == nullptr || y == nullptr || (!transposed && ws == nullptr))
        return dk_fail("dk_int8_linear: null pointer");
    if (!int8_rows_ok(xq, ldx, k) || !int8_rows_ok(wq, ldw, transposed ? n : k))
        return dk_fail("dk_int8_linear: xq and wq must be 16-byte aligned, their row strides multiples of 16 below "
                       "2^23 that cover their columns");
    if (m > 1 && ldy < n) return dk_fail("dk_int8_linear: output rows overlap");
    const Int8Plan p = int8_plan(m, n, k, transposed != 0);
    if (p.partial_bytes > 0 &&
        (workspace == nullptr || workspace_bytes < p.partial_bytes || !aligned_to(workspace, 16)))
        return dk_fail("dk_int8_linear: workspace too small (dk_int8_linear_workspace)");
    Int8GemmArgs a{};
    a.x = xq;
    a.w = wq;
    a.xs = xs;
    a.ws = ws;
    a.bias = bias;
    a.y = y;
    a.partials = static_cast<int32_t*>(workspace);
    a.ldx = ldx;
    a.ldw = ldw;
    a.ldy = ldy;
    a.m = (int32_t)m;
    a.n = (int32_t)n;
    a.k = (int32_t)k;
    a.bias_dtype = bias_dtype;
    return check_launch(launch_int8_gemm(a, p, y_dtype, transposed != 0, static_cast<hipStream_t>(stream)),
                        "dk_int8_linear launch");
}

// workspace of a fused call: the integers (rows padded to 128 bytes), the scales, the partial sums
int64_t dk_int8_linear_x_workspace(int backward, int64_t m, int64_t n, int64_t k) {
    dk_clear_error();
    const int64_t rows = m, cols = backward ? n : k, out = backward ? k : n;
    if (!int8_sizes(rows, out, cols) || (backward && k < 1)) {
        dk_fail("dk_int8_linear: 0 <= m, n < 2^23, m n < 2^38, 1 <= k <= 131071 (backward: m, k and n)");
        return -1;
    }
    if (m == 0 || out == 0 || int8_fused(m, cols, backward != 0)) return 0;
    return m * ((cols + 127) / 128 * 128) + (m + 31) / 32 * 128 + int8_plan(m, out, cols, backward != 0).partial_bytes;
}

static int int8_linear_x(bool backward, const void* x, int x_dtype, int64_t ldx, const int8_t* wq, int64_t ldw,
                         const float* ws, const void* bias, int bias_dtype, void* y, int y_dtype, int64_t ldy, int64_t m,
                         int64_t out, int64_t cols, void* workspace, int64_t workspace_bytes, void* stream) {
    if (m == 0 || out == 0) return 0;
    if (x == nullptr || wq == nullptr || ws == nullptr || y == nullptr) return dk_fail("dk_int8_linear: null pointer");
    if (!is_dtype(x_dtype) || !is_dtype(y_dtype) || (bias != nullptr && !is_dtype(bias_dtype)))
        return dk_fail("dk_int8_linear: unknown type");
    if ((m > 1 && ldx < 0) || (m > 1 && ldy < out)) return dk_fail("dk_int8_linear: row strides");
    if (!backward && int8_fused(m, cols, false)) {
        if (!int8_rows_ok(wq, ldw, cols))
            return dk_fail("dk_int8_linear: wq must be 16-byte aligned, its row stride a multiple of 16 below 2^23");
        Int8QuantArgs q{x, nullptr, nullptr, nullptr, ldx, 0, m, (int32_t)cols};
        Int8GemmArgs a{};
        a.w = wq;
        a.ws = ws;
        a.bias = bias;
        a.bias_dtype = bias_dtype;
        a.y = y;
        a.ldw = ldw;
        a.ldy = ldy;
        a.m = (int32_t)m;
        a.n = (int32_t)out;
        a.k = (int32_t)cols;
        return check_launch(launch_int8_fused(a, q, x_dtype, y_dtype, static_cast<hipStream_t>(stream)),
                            "dk_int8_linear launch");
    }
    const int64_t ldq = (cols + 127) / 128 * 128, scales = m * ldq, rest = scales + (m + 31) / 32 * 128;
    if (workspace == nullptr || workspace_bytes < rest || !aligned_to(workspace, 16))
        return dk_fail("dk_int8_linear: workspace too small (dk_int8_linear_x_workspace)");
    int8_t* const q = static_cast<int8_t*>(workspace);
    float* const xs = reinterpret_cast<float*>(q + scales);
    if (int rc = dk_int8_quantize(x, x_dtype, ldx, backward ? ws : nullptr, q, ldq, xs, m, cols, stream)) return rc;
    return dk_int8_linear(backward ? 1 : 0, q, ldq, xs, wq, ldw, backward ? nullptr : ws, bias, bias_dtype, y, y_dtype,
                          ldy, m, out, cols, q + rest, workspace_bytes - rest, stream);
}

int dk_int8_linear_fwd(const void* x, int x_dtype, int64_t ldx, const int8_t* wq, int64_t ldw, const float* ws,
                       const void* bias, int bias_dtype, void* y, int y_dtype, int64_t ldy, int64_t m, int64_t n,
                       int64_t k, void* workspace, int64_t workspace_bytes, void* stream) {
    dk_clear_error();
    if (!int8_sizes(m, n, k)) return dk_fail("dk_int8_linear_fwd: 0 <= m, n < 2^23, m n < 2^38, 1 <= k <= 131071");
    return int8_linear_x(false, x, x_dtype, ldx, wq, ldw, ws, bias, bias_dtype, y, y_dtype, ldy, m, n, k, workspace,
                         workspace_bytes, stream);
}

int dk_int8_linear_bwd(const void* dy, int dy_dtype, int64_t lddy, const int8_t* wq, int64_t ldw, const float* ws,
                       void* dx, int dx_dtype, int64_t lddx, int64_t m, int64_t n, int64_t k, void* workspace,
                       int64_t workspace_bytes, void* stream) {
    dk_clear_error();
    if (!int8_sizes(m, k, n)) return dk_fail("dk_int8_linear_bwd: 0 <= m, k < 2^23, m k < 2^38, 1 <= n <= 131071");
    return int8_linear_x(true, dy, dy_dtype, lddy, wq, ldw, ws, nullptr, 0, dx, dx_dtype, lddx, m, k, n, workspace,
                         workspace_bytes, stream);
}

int dk_residual_norm_fwd(const dk_residual_norm* d, void* stream) {
    dk_clear_error();
    ResidualNormArgs a{};
    if (int rc = residual_norm_common(d, &a)) return rc;
    if (a.rows == 0) return 0;
    if ((d->weight != nullptr && d->y == nullptr) || (d->weight == nullptr && d->h == nullptr))
        return dk_fail("dk_residual_norm_fwd: y with a weight, h without one");
    a.h = d->h;
    a.y = d->y;
    return check_launch(launch_residual_norm(a, d->x_dtype, d->stream_dtype, d->y_dtype, false, nullptr, nullptr,
                                             nullptr, static_cast<hipStream_t>(stream)),
                        "dk_residual_norm_fwd launch");
}

int64_t dk_residual_norm_bwd_workspace(const dk_residual_norm* d) {
    dk_clear_error();
    ResidualNormArgs a{};
    if (residual_norm_common(d, &a) != 0 || residual_norm_sums(d, &a) != 0) return -1;
    return residual_norm_bytes(a);
}

int dk_residual_norm_bwd(const dk_residual_norm* d, void* workspace, int64_t workspace_bytes, void* stream) {
    dk_clear_error();
    ResidualNormArgs a{};
    if (int rc = residual_norm_common(d, &a)) return rc;
    if (int rc = residual_norm_sums(d, &a)) return rc;
    if (a.rows == 0 && a.nslabs == 0) return 0;
    // (the join of the sums reads a channel's gate, without rows too)
    if (a.gate_kind == DK_GATE_CHANNEL && a.gate == nullptr) return dk_fail("dk_residual_norm_bwd: null gate");
    if (a.rows > 0) {
        if (d->dx == nullptr) return dk_fail("dk_residual_norm_bwd: null pointer");
        if ((d->weight != nullptr) != (d->grad_y != nullptr))
            return dk_fail("dk_residual_norm_bwd: grad_y where there is a weight, and only there");
        if (d->dresidual != nullptr && d->residual == nullptr)
            return dk_fail("dk_residual_norm_bwd: no residual to take a gradient of");
        const int64_t need = residual_norm_bytes(a);
        if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned_to(workspace, 16)))
            return dk_fail("dk_residual_norm_bwd: workspace too small (dk_residual_norm_bwd_workspace)");
    }
    a.gh = d->grad_h;
    a.gy = d->grad_y;
    a.ldgh = d->ld_grad_h;
    a.ldgy = d->ld_grad_y;
    a.dx = d->dx;
    a.dres = d->dresidual;
    a.dgate = d->gate_kind == DK_GATE_CHANNEL ? nullptr : d->dgate;
    a.slabs = a.nslabs > 0 ? static_cast<float*>(workspace) : nullptr;
    return check_launch(launch_residual_norm(a, d->x_dtype, d->stream_dtype, d->y_dtype, true, d->dweight,
                                             d->dpost_weight, d->gate_kind == DK_GATE_CHANNEL ? static_cast<float*>(d->dgate) : nullptr,
                                             static_cast<hipStream_t>(stream)),
                        "dk_residual_norm_bwd launch");
}

static int scaled_rope(const dk_scaled_rope* d, bool backward, void* stream) {
    dk_clear_error();
    if (d == nullptr) return dk_fail("dk_scaled_rope: null descriptor");
    if (d->dtype != DK_FP16 && d->dtype != DK_BF16) return dk_fail("dk_scaled_rope: q and k must be fp16 or bf16");
    if (d->head_dim < 1 || d->head_dim > 1024) return dk_fail("dk_scaled_rope: head_dim must be 1 to 1024");
    if (d->rotary_dim < 0 || d->rotary_dim > d->head_dim || d->rotary_dim % 2 != 0)
        return dk_fail("dk_scaled_rope: rotary_dim must be even and from 0 to head_dim");
    if (d->n_heads < 1 || d->n_kv_heads < 1 || d->n_heads > 65536 || d->n_kv_heads > 65536)
        return dk_fail("dk_scaled_rope: 1 to 65536 heads each");
    if (d->batch < 0 || d->tokens < 0 || d->tokens >= INT32_MAX || d->batch >= INT32_MAX ||
        d->batch * d->tokens >= (int64_t(1) << 24))  // (threads of a launch are below 2^32)
        return dk_fail("dk_scaled_rope: batch * tokens must be non-negative and below 2^24");
    if (d->batch * d->tokens == 0) return 0;
    if (d->q == nullptr || d->k == nullptr || d->q_out == nullptr || d->k_out == nullptr)
        return dk_fail("dk_scaled_rope: null pointer");
    if (d->rotary_dim > 0 && (d->positions == nullptr || d->inv_freq == nullptr))
        return dk_fail("dk_scaled_rope: positions and inv_freq must be set");
    for (int i = 0; i < 3; ++i)
        if (d->q_stride[i] < 0 || d->k_stride[i] < 0) return dk_fail("dk_scaled_rope: negative stride");
    ScaledRopeArgs a{};
    a.q = d->q;
    a.k = d->k;
    a.oq = d->q_out;
    a.ok = d->k_out;
    a.pos = d->positions;
    a.inv_freq = d->inv_freq;
    const int64_t t = d->tokens, hd = d->head_dim;
    for (int i = 0; i < 3; ++i) {
        a.q_in[i] = d->q_stride[i];
        a.k_in[i] = d->k_stride[i];
    }
    for (int side = 0; side < 2; ++side) {
        const int64_t h = side ? d->n_kv_heads : d->n_heads;
        int64_t* const st = side ? a.k_st : a.q_st;
        st[0] = t * h * hd;
        st[1] = backward ? h * hd : hd;
        st[2] = backward ? hd : t * hd;
    }
    a.pos_batch = d->pos_batch_stride;
    a.tokens = (uint32_t)t;
    a.rows = (uint32_t)(d->batch * t);
    a.hq = d->n_heads;
    a.hk = d->n_kv_heads;
    a.d = d->head_dim;
    a.r = d->rotary_dim;
    a.pairs = d->pairs;
    a.pos64 = d->positions_int64;
    a.factor = d->factor;
    a.sin_factor = backward ? -d->factor : d->factor;
    return check_launch(launch_scaled_rope(a, d->dtype, static_cast<hipStream_t>(stream)),
                        backward ? "dk_scaled_rope_bwd launch" : "dk_scaled_rope_fwd launch");
}

int dk_scaled_rope_fwd(const dk_scaled_rope* d, void* stream) { return scaled_rope(d, false, stream); }

int dk_scaled_rope_bwd(const dk_scaled_rope* d, void* stream) { return scaled_rope(d, true, stream); }

int64_t dk_int4_linear_workspace(int backward, int copy, int64_t m, int64_t n, int64_t k) {
    dk_clear_error();
    if (!int4_sizes(m, n, k)) {
        dk_fail(kInt4Sizes);
        return -1;
    }
    if (m == 0 || n == 0) return 0;
    return int4_bytes(int4_plan(m, n, k, backward != 0), copy != 0, m, backward ? n : k, nullptr);
}

int dk_int4_linear_plan(int backward, int64_t m, int64_t n, int64_t k, int32_t* out) {
    dk_clear_error();
    if (!int4_sizes(m, n, k) || m == 0 || n == 0 || out == nullptr) return dk_fail(kInt4Sizes);
    const Int4Plan p = int4_plan(m, n, k, backward != 0);
    out[0] = p.tokens;
    out[1] = p.few ? p.waves : 0;
    out[2] = p.few ? p.shares : 0;
    out[3] = p.splits;
    return 0;
}

int dk_int4_linear(int backward, const void* x, int x_dtype, int64_t ldx, const uint8_t* packed, const uint32_t* meta,
                   int64_t group, int scale_dtype, const void* bias, int bias_dtype, void* y,
                   int y_dtype, int64_t ldy, int64_t m, int64_t n, int64_t k, int copy, void* workspace,
                   int64_t workspace_bytes, void* stream) {
    dk_clear_error();
    if (!int4_sizes(m, n, k)) return dk_fail(kInt4Sizes);
    if ((x_dtype != DK_FP16 && x_dtype != DK_BF16) || (y_dtype != x_dtype && y_dtype != DK_FP32))
        return dk_fail("dk_int4_linear: x must be fp16 or bf16, y of x's type or fp32");
    if (scale_dtype != DK_FP16 && scale_dtype != DK_BF16) return dk_fail("dk_int4_linear: scales must be fp16 or bf16");
    if (bias != nullptr && (backward || !is_dtype(bias_dtype)))
        return dk_fail("dk_int4_linear: a bias of a known type, and only forward");
    if (group < 32 || group % 32 != 0 || group > (int64_t(1) << 20))
        return dk_fail("dk_int4_linear: group must be a multiple of 32 up to 2^20");
    if (m == 0 || (backward ? k : n) == 0) return 0;
    const int64_t cols = backward ? k : n, sum = backward ? n : k;
    if (y == nullptr) return dk_fail("dk_int4_linear: null pointer");
    if (m > 1 && ldy < cols) return dk_fail("dk_int4_linear: output rows overlap");
    if (n == 0) return dk_fail("dk_int4_linear: the sum has no terms");
    if (x == nullptr || packed == nullptr || meta == nullptr) return dk_fail("dk_int4_linear: null pointer");
    if (!aligned_to(packed, 16) || !aligned_to(meta, 4))
        return dk_fail("dk_int4_linear: packed must be 16-byte aligned, meta 4-byte aligned");
    if (m > 1 && (ldx < 0 || ldx >= (sum < kInt4LongRow ? 1 : 2) * kInt4LongRow))
        return dk_fail("dk_int4_linear: x's row stride must be non-negative and below 2^22 (2^23 where a row has 2^22 elements)");
    if (!copy && (sum % 8 != 0 || !aligned_to(x, 16) || (m > 1 && ldx % 8 != 0)))
        return dk_fail("dk_int4_linear: without copy x needs 16-byte aligned rows of a multiple of 8 columns");
    const Int4Plan p = int4_plan(m, n, k, backward != 0);
    int64_t partial = 0;
    const int64_t need = int4_bytes(p, copy != 0, m, sum, &partial);
    if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned_to(workspace, 16)))
        return dk_fail("dk_int4_linear: workspace too small (dk_int4_linear_workspace)");
    Int4Args a{};
    a.x = x;
    a.w = packed;
    a.meta = meta;
    a.bias = bias;
    a.y = y;
    a.partials = static_cast<float*>(workspace);
    a.padded = copy && !p.few ? reinterpret_cast<uint16_t*>(static_cast<uint8_t*>(workspace) + partial) : nullptr;
    a.loose = copy && p.few;
    a.ldx = m > 1 ? ldx : 0;
    a.ldy = ldy;
    a.m = (int32_t)m;
    a.n = (int32_t)n;
    a.k = (int32_t)k;
    a.groups = (int32_t)((k + group - 1) / group);
    a.group_units = (int32_t)(group / 32);
    a.scale_dtype = scale_dtype;
    a.bias_dtype = bias_dtype;
    a.y_dtype = y_dtype;
    return check_launch(launch_int4(a, p, x_dtype, backward != 0, static_cast<hipStream_t>(stream)),
                        "dk_int4_linear launch");
}

}  // extern "C"
