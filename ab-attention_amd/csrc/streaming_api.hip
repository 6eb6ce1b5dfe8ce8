// C entry points of the streaming operators (include/ab_attention.h): checks of
// sizes, pointers and alignment, then one call of the kernels' launchers.
#include <algorithm>
#include <cmath>
#include <initializer_list>

#include "../../include/ab_attention.h"
#include "cache.hpp"
#include "rotary.hpp"
#include "window.hpp"

using namespace ab;

namespace {
constexpr int64_t kMostTokens = int64_t(1) << 30;

bool aligned(const void* p, uintptr_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// Strides of a tensor whose rows start at multiples of `align` elements; the
// stride of a single batch item, head or token is not used.
int rows_of(const char* what, const int64_t (&stride)[3], int64_t batch, int64_t heads, int64_t tokens, int64_t align,
            Rows& out) {
    const int64_t extent[3] = {batch, heads, tokens};
    int64_t used[3];
    for (int i = 0; i < 3; ++i) {
        used[i] = extent[i] > 1 ? stride[i] : 0;
        if (used[i] < 0 || used[i] % align || used[i] >= (int64_t(1) << 40))
            return set_error(AB_ERR_INVALID, "%s: strides must be multiples of %d elements from 0 to 2^40", what, (int)align);
    }
    out = {used[0], used[1], used[2]};
    return AB_OK;
}

// Whether the kernels' 32-bit offsets reach the rows of a head and 64 behind them
// (which they ask for and get zeros).
bool head_fits(const Rows& r, int64_t tokens) { return (r.token * (tokens + 64) + 128) * 2 <= int64_t(0xffffffff); }

int check_heads(const char* what, int64_t batch, int64_t heads, int64_t kv_heads, int64_t tokens, int64_t dim) {
    if (batch < 0 || tokens < 0 || heads <= 0 || kv_heads <= 0)
        return set_error(AB_ERR_INVALID, "%s: sizes must be positive", what);
    if (heads % kv_heads) return set_error(AB_ERR_INVALID, "%s: heads must be a multiple of kv_heads", what);
    if (dim != 64 && dim != 128) return set_error(AB_ERR_INVALID, "%s: dim must be 64 or 128", what);
    if (tokens >= kMostTokens || batch > 65535 || heads > 65535 || batch * heads > (int64_t(1) << 24))
        return set_error(AB_ERR_INVALID, "%s: too many tokens, heads or batch items", what);
    return AB_OK;
}

// The checks and the form of a cache: k, v [pages, kv_heads, page_tokens, dim].
int check_cache(const char* what, int64_t batch, int64_t kv_heads, int64_t pages, int64_t page_tokens, int64_t width,
                const int64_t (&k_stride)[3], const int64_t (&v_stride)[3], const int32_t* table,
                const int32_t* lengths, const int32_t* offsets, Rows& k, Rows& v) {
    if (page_tokens <= 0 || page_tokens % 8 || page_tokens >= kMostTokens)
        return set_error(AB_ERR_INVALID, "%s: pages must hold a positive multiple of 8 tokens", what);
    if (pages < 0 || pages >= kMostTokens || width < 0 || width >= kMostTokens)
        return set_error(AB_ERR_INVALID, "%s: too many pages", what);
    if (int rc = rows_of(what, k_stride, pages, kv_heads, page_tokens, 8, k)) return rc;
    if (int rc = rows_of(what, v_stride, pages, kv_heads, page_tokens, 8, v)) return rc;
    if (!head_fits(k, page_tokens) || !head_fits(v, page_tokens))
        return set_error(AB_ERR_INVALID, "%s: one head of a page must be under 4 GiB", what);
    if (batch > 0 && (!lengths || !offsets || (width > 0 && !table)))
        return set_error(AB_ERR_INVALID, "%s: null pointer", what);
    return AB_OK;
}

// Most keys that a tile of rows can visit, for the number of parts.
int64_t most_keys(const ab_window_args& a, int64_t length) {
    if (a.window <= 0) return length;
    const double reach = (double(a.window) + double(a.sinks) + 1) * double(a.frame) + kWindowRows;
    return static_cast<int64_t>(std::min(reach, double(length)));
}

// The checked form of a call. Sizes of nothing are left to the caller.
int window_call(const char* what, const ab_window_args& a, bool paged, WindowCall& c) {
    if (int rc = check_heads(what, a.batch, a.heads, a.kv_heads, a.tokens, a.dim)) return rc;
    if (a.dtype != AB_BF16 && a.dtype != AB_F16) return set_error(AB_ERR_INVALID, "%s: dtype must be bf16 or fp16", what);
    if (a.window < 0 || a.sinks < 0 || a.frame <= 0)
        return set_error(AB_ERR_INVALID, "%s: window and sinks must not be negative, frame must be positive", what);
    if (!std::isfinite(a.scale)) return set_error(AB_ERR_INVALID, "%s: scale must be finite", what);
    c = WindowCall{};
    c.q = a.q;
    c.k = a.k;
    c.v = a.v;
    c.out = a.out;
    c.out_rest = a.out_rest;
    c.lse = a.lse;
    c.batch = static_cast<int32_t>(a.batch);
    c.heads = static_cast<int32_t>(a.heads);
    c.kv_heads = static_cast<int32_t>(a.kv_heads);
    c.tokens = static_cast<int32_t>(a.tokens);
    c.dim = static_cast<int32_t>(a.dim);
    c.half = a.dtype == AB_F16;
    c.lengths = a.lengths;
    c.group = divisor(static_cast<uint32_t>(a.heads / a.kv_heads));
    c.rows = a.tokens * a.heads * (paged ? 1 : a.batch);
    const int64_t q_batch = paged ? 1 : a.batch;
    if (int rc = rows_of(what, a.q_stride, q_batch, a.heads, a.tokens, 8, c.q_rows)) return rc;
    if (int rc = rows_of(what, a.out_stride, q_batch, a.heads, a.tokens, 4, c.out_rows)) return rc;
    // Tokens before a frame that are still seen, and tokens of the sinks, at most 2^30.
    const int64_t frame = std::min(a.frame, kMostTokens);
    c.mask.frame = divisor(static_cast<uint32_t>(frame));
    c.mask.back = a.window == 0 || a.window - 1 >= kMostTokens / frame ? kMostTokens : (a.window - 1) * frame;
    c.mask.sinks = a.sinks >= kMostTokens / frame ? kMostTokens : a.sinks * frame;
    c.scale_log2 = static_cast<float>(a.scale * 1.4426950408889634);
    int64_t length = a.tokens;
    if (paged) {
        if (int rc = check_cache(what, a.batch, a.kv_heads, a.pages, a.page_tokens, a.table_width, a.k_stride, a.v_stride,
                                 a.page_table, a.lengths, a.offsets, c.k_rows, c.v_rows))
            return rc;
        length = a.table_width * a.page_tokens;
        if (length >= kMostTokens) return set_error(AB_ERR_INVALID, "%s: a page table covers fewer than 2^30 tokens", what);
        if (a.tokens * (a.heads / a.kv_heads) >= kMostTokens) return set_error(AB_ERR_INVALID, "%s: too many queries", what);
        c.offsets = a.offsets;
        c.table = a.page_table;
        c.table_width = static_cast<int32_t>(a.table_width);
        c.pages = static_cast<int32_t>(a.pages);
        c.page = divisor(static_cast<uint32_t>(a.page_tokens));
        c.row = {0, 1, a.heads};
    } else {
        if (int rc = rows_of(what, a.k_stride, a.batch, a.kv_heads, a.tokens, 8, c.k_rows)) return rc;
        if (int rc = rows_of(what, a.v_stride, a.batch, a.kv_heads, a.tokens, 8, c.v_rows)) return rc;
        if (!head_fits(c.k_rows, a.tokens) || !head_fits(c.v_rows, a.tokens))
            return set_error(AB_ERR_INVALID, "%s: one head of K/V must be under 4 GiB", what);
        c.row = {a.heads * a.tokens, a.tokens, 1};
    }
    c.paged = paged;
    const int64_t units = window_tiles(c) * (paged ? a.kv_heads : a.batch * a.heads);
    if (units >= (int64_t(1) << 30)) return set_error(AB_ERR_INVALID, "%s: grid too large", what);
    c.parts = units > 0 ? window_parts(c, most_keys(a, length)) : 1;
    return AB_OK;
}

size_t workspace_bytes(const WindowCall& c) {
    const size_t rounded = !c.paged && c.out_rest ? sizeof(float) : 0;
    return c.parts == 1 ? 0 : size_t(c.parts) * size_t(c.rows) * (size_t(c.dim) * sizeof(float) + sizeof(float2) + rounded);
}

int window_launch(const char* what, const ab_window_args* a, bool paged, void* stream) {
    if (!a) return set_error(AB_ERR_INVALID, "%s: null pointer", what);
    WindowCall c;
    if (int rc = window_call(what, *a, paged, c)) return rc;
    if (a->batch == 0 || a->tokens == 0) return AB_OK;
    const bool no_cache = paged && (a->pages == 0 || a->table_width == 0);
    if (!a->q || !a->out || (!no_cache && (!a->k || !a->v))) return set_error(AB_ERR_INVALID, "%s: null pointer", what);
    if (!aligned(a->q, 16) || !aligned(a->k, 16) || !aligned(a->v, 16) || !aligned(a->out, 8) || !aligned(a->out_rest, 8))
        return set_error(AB_ERR_INVALID, "%s: q/k/v must be 16-byte and out 8-byte aligned", what);
    if (!a->workspace) c.parts = 1;
    if (c.parts > 1) {
        if (a->workspace_bytes < workspace_bytes(c))
            return set_error(AB_ERR_INVALID, "%s: workspace of %zu bytes is smaller than the %zu required", what,
                             a->workspace_bytes, workspace_bytes(c));
        if (!aligned(a->workspace, 16)) return set_error(AB_ERR_INVALID, "%s: workspace must be 16-byte aligned", what);
        c.partial_o = static_cast<float*>(a->workspace);
        c.partial_stat = reinterpret_cast<float2*>(c.partial_o + c.parts * c.rows * c.dim);
        c.partial_rounded = reinterpret_cast<float*>(c.partial_stat + c.parts * c.rows);
    }
    return launch_window(c, static_cast<hipStream_t>(stream));
}
}  // namespace

extern "C" {

int ab_rotary(const ab_rotary_args* a, void* stream) {
    if (!a) return set_error(AB_ERR_INVALID, "rotary: null pointer");
    const int64_t kv_heads = a->k ? a->kv_heads : 0;
    if (a->batch < 0 || a->tokens < 0 || a->heads <= 0 || kv_heads < 0 || a->heads > 65535 || kv_heads > 65535)
        return set_error(AB_ERR_INVALID, "rotary: sizes must be positive");
    if (a->dtype < AB_BF16 || a->dtype > AB_F32) return set_error(AB_ERR_INVALID, "rotary: unknown dtype");
    if (a->dim <= 0 || a->dim % 8 || a->dim > 1024)
        return set_error(AB_ERR_INVALID, "rotary: dim must be a multiple of 8 up to 1,024");
    if (a->axes < 1 || a->axes > kMaxAxes) return set_error(AB_ERR_INVALID, "rotary: 1 to %d axes", kMaxAxes);
    RotaryCall c{};
    int64_t turned = 0;
    for (int i = 0; i < a->axes; ++i) {
        if (a->axis_dims[i] <= 0 || a->axis_dims[i] % 2 || a->axis_dims[i] > a->dim)
            return set_error(AB_ERR_INVALID, "rotary: every axis turns a positive even number of dims");
        turned += a->axis_dims[i];
        c.pairs[i] = static_cast<int32_t>(a->axis_dims[i] / 2);
    }
    if (turned > a->dim) return set_error(AB_ERR_INVALID, "rotary: the axes turn more than dim");
    if (a->halves && turned % 16) return set_error(AB_ERR_INVALID, "rotary: halves need a multiple of 16 turned dims");
    if (!std::isfinite(a->theta) || a->theta <= 0) return set_error(AB_ERR_INVALID, "rotary: theta must be positive and finite");
    if (a->position_type < 0 || a->position_type > 2) return set_error(AB_ERR_INVALID, "rotary: unknown position type");
    c.units = static_cast<uint32_t>(a->halves ? turned / 16 + (a->dim - turned) / 8 : a->dim / 8);
    if (a->batch > 65535 || a->tokens >= kMostTokens || a->batch * a->tokens * c.units >= (int64_t(1) << 31))
        return set_error(AB_ERR_INVALID, "rotary: too many tokens");
    const int64_t align = a->dtype == AB_F32 ? 4 : 8;
    if (int rc = rows_of("rotary", a->q_stride, a->batch, a->heads, a->tokens, align, c.in_rows[0])) return rc;
    if (int rc = rows_of("rotary", a->q_out_stride, a->batch, a->heads, a->tokens, align, c.out_rows[0])) return rc;
    if (kv_heads) {
        if (int rc = rows_of("rotary", a->k_stride, a->batch, kv_heads, a->tokens, align, c.in_rows[1])) return rc;
        if (int rc = rows_of("rotary", a->k_out_stride, a->batch, kv_heads, a->tokens, align, c.out_rows[1])) return rc;
    }
    if (a->batch == 0 || a->tokens == 0) return AB_OK;
    if (!a->q || !a->q_out || !a->positions || (kv_heads && !a->k_out)) return set_error(AB_ERR_INVALID, "rotary: null pointer");
    if (!aligned(a->q, 16) || !aligned(a->q_out, 16) || !aligned(a->k, 16) || !aligned(a->k_out, 16))
        return set_error(AB_ERR_INVALID, "rotary: tensors must be 16-byte aligned");
    c.in[0] = a->q;
    c.in[1] = a->k;
    c.out[0] = a->q_out;
    c.out[1] = a->k_out;
    c.positions = a->positions;
    c.axes = static_cast<int32_t>(a->axes);
    for (int i = 0; i < a->axes; ++i) {
        c.step[i] = std::log2(a->theta) * 2.0 / double(a->joint ? turned : a->axis_dims[i]);
        c.ratio[i] = std::exp2(-c.step[i]);
    }
    c.heads[0] = static_cast<int32_t>(a->heads);
    c.heads[1] = static_cast<int32_t>(kv_heads);
    c.position_kind = static_cast<int32_t>(a->position_type);
    c.turned = static_cast<int32_t>(turned);
    c.tokens = static_cast<uint32_t>(a->tokens);
    c.total = static_cast<uint32_t>(a->batch * a->tokens);
    c.sign = a->inverse ? -1.f : 1.f;
    c.per_batch = a->per_batch != 0;
    c.joint = a->joint != 0;
    return launch_rotary(c, static_cast<int>(a->dtype), a->halves != 0, static_cast<hipStream_t>(stream));
}

size_t ab_window_workspace_bytes(const ab_window_args* a) {
    WindowCall c;
    if (!a || a->batch <= 0 || a->tokens <= 0 || window_call("window_attention", *a, a->offsets != nullptr, c)) return 0;
    return workspace_bytes(c);
}

int ab_window_attention(const ab_window_args* args, void* stream) {
    return window_launch("window_attention", args, false, stream);
}

int ab_chunk_attention(const ab_window_args* args, void* stream) {
    return window_launch("chunk_attention", args, true, stream);
}

}  // extern "C"

namespace {
// The checked form of a backward call, with the floats of its workspace.
int grad_call(const ab_window_grad_args& a, WindowGradCall& g, int64_t& stat, int64_t& partial) {
    const char* what = "window_attention_grad";
    const ab_window_args& f = a.forward;
    WindowCall c;
    if (int rc = window_call(what, f, false, c)) return rc;
    g = WindowGradCall{};
    g.q = f.q;
    g.k = f.k;
    g.v = f.v;
    g.out = f.out;
    g.out_rest = f.out_rest;
    g.dout = a.dout;
    g.lse = f.lse;
    g.dlse = a.dlse;
    g.dq = a.dq;
    g.dk = a.dk;
    g.dv = a.dv;
    g.q_rows = c.q_rows;
    g.k_rows = c.k_rows;
    g.v_rows = c.v_rows;
    if (int rc = rows_of(what, f.out_stride, f.batch, f.heads, f.tokens, 8, g.out_rows)) return rc;
    if (int rc = rows_of(what, a.dout_stride, f.batch, f.heads, f.tokens, 8, g.dout_rows)) return rc;
    if (int rc = rows_of(what, a.dq_stride, f.batch, f.heads, f.tokens, 8, g.dq_rows)) return rc;
    if (int rc = rows_of(what, a.dk_stride, f.batch, f.kv_heads, f.tokens, 8, g.dk_rows)) return rc;
    if (int rc = rows_of(what, a.dv_stride, f.batch, f.kv_heads, f.tokens, 8, g.dv_rows)) return rc;
    if (!head_fits(g.q_rows, f.tokens) || !head_fits(g.dout_rows, f.tokens))
        return set_error(AB_ERR_INVALID, "%s: one head of Q and of its gradient must be under 4 GiB", what);
    g.batch = c.batch;
    g.heads = c.heads;
    g.kv_heads = c.kv_heads;
    g.tokens = c.tokens;
    g.dim = c.dim;
    g.half = c.half;
    g.lengths = c.lengths;
    g.group = c.heads / c.kv_heads;
    g.mask = c.mask;
    g.scale = static_cast<float>(f.scale);
    g.scale_log2 = c.scale_log2;
    plan_window_grad(g, stat, partial);
    return AB_OK;
}
}  // namespace

extern "C" {

size_t ab_window_grad_workspace_bytes(const ab_window_grad_args* a) {
    WindowGradCall g;
    int64_t stat, partial;
    if (!a || a->forward.batch <= 0 || a->forward.tokens <= 0 || grad_call(*a, g, stat, partial)) return 0;
    return size_t(stat + partial) * sizeof(float);
}

int ab_window_attention_grad(const ab_window_grad_args* a, void* stream) {
    const char* what = "window_attention_grad";
    if (!a) return set_error(AB_ERR_INVALID, "%s: null pointer", what);
    WindowGradCall g;
    int64_t stat, partial;
    if (int rc = grad_call(*a, g, stat, partial)) return rc;
    const ab_window_args& f = a->forward;
    if (f.batch == 0 || f.tokens == 0) return AB_OK;
    for (const void* p : {f.q, f.k, f.v, static_cast<const void*>(f.out), a->dout, static_cast<const void*>(a->dq),
                          static_cast<const void*>(a->dk), static_cast<const void*>(a->dv),
                          static_cast<const void*>(f.workspace)}) {
        if (!p) return set_error(AB_ERR_INVALID, "%s: null pointer", what);
        if (!aligned(p, 16)) return set_error(AB_ERR_INVALID, "%s: tensors must be 16-byte aligned", what);
    }
    if (!f.lse) return set_error(AB_ERR_INVALID, "%s: null pointer", what);
    if (!aligned(f.out_rest, 16)) return set_error(AB_ERR_INVALID, "%s: tensors must be 16-byte aligned", what);
    if (f.workspace_bytes < size_t(stat + partial) * sizeof(float))
        return set_error(AB_ERR_INVALID, "%s: workspace of %zu bytes is smaller than the %zu required", what, f.workspace_bytes,
                         size_t(stat + partial) * sizeof(float));
    g.stat = static_cast<float*>(f.workspace);
    g.partial = g.stat + stat;
    return launch_window_grad(g, static_cast<hipStream_t>(stream));
}

int ab_append_cache(const ab_append_args* a, void* stream) {
    if (!a) return set_error(AB_ERR_INVALID, "append_cache: null pointer");
    if (int rc = check_heads("append_cache", a->batch, a->kv_heads, a->kv_heads, a->tokens, a->dim)) return rc;
    AppendCall c{};
    if (int rc = check_cache("append_cache", a->batch, a->kv_heads, a->pages, a->page_tokens, a->table_width,
                             a->k_cache_stride, a->v_cache_stride, a->page_table, a->lengths, a->offsets, c.k_cache_rows,
                             c.v_cache_rows))
        return rc;
    if (a->table_width * a->page_tokens >= kMostTokens)
        return set_error(AB_ERR_INVALID, "append_cache: a page table covers fewer than 2^30 tokens");
    if (int rc = rows_of("append_cache", a->k_stride, 1, a->kv_heads, a->tokens, 8, c.k_rows)) return rc;
    if (int rc = rows_of("append_cache", a->v_stride, 1, a->kv_heads, a->tokens, 8, c.v_rows)) return rc;
    if (a->batch == 0 || a->tokens == 0 || a->pages == 0 || a->table_width == 0) return AB_OK;
    if (!a->k || !a->v || !a->k_cache || !a->v_cache) return set_error(AB_ERR_INVALID, "append_cache: null pointer");
    if (!aligned(a->k, 16) || !aligned(a->v, 16) || !aligned(a->k_cache, 16) || !aligned(a->v_cache, 16))
        return set_error(AB_ERR_INVALID, "append_cache: tensors must be 16-byte aligned");
    c.k = a->k;
    c.v = a->v;
    c.k_cache = a->k_cache;
    c.v_cache = a->v_cache;
    c.table = a->page_table;
    c.lengths = a->lengths;
    c.offsets = a->offsets;
    c.batch = static_cast<int32_t>(a->batch);
    c.kv_heads = static_cast<int32_t>(a->kv_heads);
    c.dim = static_cast<int32_t>(a->dim);
    c.tokens = static_cast<int32_t>(a->tokens);
    c.table_width = static_cast<int32_t>(a->table_width);
    c.pages = static_cast<int32_t>(a->pages);
    c.page = divisor(static_cast<uint32_t>(a->page_tokens));
    return launch_append(c, static_cast<hipStream_t>(stream));
}

}  // extern "C"
