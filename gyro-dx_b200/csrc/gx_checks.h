// gx_checks.h — argument rules of the operators around the layer (gx_linear, gx_norm,
// gx_norm_residual, gx_logprobs, gx_upload_norms), plain host C++ without the CUDA headers.
#pragma once
#include <stddef.h>
#include <stdint.h>

#include <cmath>
#include <initializer_list>

#include "../../include/gyro_moe.h"

namespace gx {

// Limits (include/gyro_moe.h).
constexpr uint32_t kQ4MaxCols = 65536, kQ4MaxRows = 1u << 24, kLinearMaxTokens = 64;
constexpr uint32_t kNormMaxWidth = 65536, kMaxVocab = 524288, kMaxRows = 1u << 24;
constexpr float kMaxScale = 1e30f;           // scale * log2 e and its double stay finite
constexpr uint64_t kMaxStride = 1ull << 32;  // elements: the bytes of kMaxRows rows stay below 2^63

inline size_t dtype_size(uint32_t dt) { return dt == GX_BF16 ? 2 : 4; }

// Rows of a call's argument: n rows of width bytes, stride bytes apart.
struct Span {
    const void *p;
    uint64_t n, width, stride;
};

// Whether two arguments share a byte. Rows of one buffer at one stride whose column ranges lie
// apart (slices of a fused buffer) do not.
inline bool overlaps(const Span &a, const Span &b) {
    if (!a.p || !b.p || !a.n || !b.n || !a.width || !b.width) return false;
    const uintptr_t a0 = (uintptr_t)a.p, b0 = (uintptr_t)b.p;
    const uintptr_t a1 = a0 + (a.n - 1) * a.stride + a.width, b1 = b0 + (b.n - 1) * b.stride + b.width;
    if (a1 <= b0 || b1 <= a0) return false;
    if (a.stride != b.stride || a.n == 1 || b.n == 1) return true;
    const uint64_t d = b0 >= a0 ? (b0 - a0) % a.stride : (a.stride - (a0 - b0) % a.stride) % a.stride;
    return !(d >= a.width && d + b.width <= a.stride);
}
// Any output over an input, or over another output.
inline bool any_overlap(std::initializer_list<Span> in, std::initializer_list<Span> out) {
    for (auto o = out.begin(); o != out.end(); ++o) {
        for (const Span &i : in)
            if (overlaps(*o, i)) return true;
        for (auto p = out.begin(); p != o; ++p)
            if (overlaps(*o, *p)) return true;
    }
    return false;
}

inline bool act_dtype(uint32_t dt) { return dt == GX_F32 || dt == GX_BF16; }
// A row argument's pointer, stride and alignment.
inline bool rows_ok(const void *p, uint32_t dt, uint64_t stride, uint64_t width) {
    return p && act_dtype(dt) && stride >= width && stride <= kMaxStride && (uintptr_t)p % dtype_size(dt) == 0;
}
inline bool words_ok(const void *p) { return ((uintptr_t)p & 3) == 0; }
inline Span rows_span(const void *p, uint32_t dt, uint64_t stride, uint64_t width, uint64_t n) {
    return {p, n, width * dtype_size(dt), stride * dtype_size(dt)};
}
inline Span flat_span(const void *p, uint64_t words) { return {p, 1, words * 4, words * 4}; }

inline bool linear_args_ok(uint32_t rows, uint32_t cols, const void *x, uint32_t x_dtype, uint64_t x_stride,
                           uint32_t n_tok, const void *y, uint32_t y_dtype, uint64_t y_stride) {
    if (n_tok > kLinearMaxTokens || !act_dtype(x_dtype) || !act_dtype(y_dtype)) return false;
    if (n_tok == 0) return true;
    return rows_ok(x, x_dtype, x_stride, cols) && rows_ok(y, y_dtype, y_stride, rows) &&
           !overlaps(rows_span(x, x_dtype, x_stride, cols, n_tok), rows_span(y, y_dtype, y_stride, rows, n_tok));
}

inline bool norm_args_ok(const gx_norm_desc &d, uint32_t n_tok) {
    if (d.n_embd == 0 || d.n_embd > kNormMaxWidth || n_tok > kMaxRows) return false;
    if (!(d.eps >= 0.f) || !std::isfinite(d.eps) || !act_dtype(d.x_dtype) || !act_dtype(d.y_dtype)) return false;
    const uint64_t E = d.n_embd;
    if (!words_ok(d.weight) || !words_ok(d.gate_weight) || !words_ok(d.gate) || !d.gate != !d.gate_weight)
        return false;
    if (n_tok) {
        if (!rows_ok(d.x, d.x_dtype, d.x_stride, E) || !rows_ok(d.y, d.y_dtype, d.y_stride, E)) return false;
        const Span x = rows_span(d.x, d.x_dtype, d.x_stride, E, n_tok), y = rows_span(d.y, d.y_dtype, d.y_stride, E, n_tok);
        const bool in_place = d.x == d.y && d.x_dtype == d.y_dtype && (d.x_stride == d.y_stride || n_tok == 1);
        if (any_overlap({in_place ? Span{} : x, flat_span(d.weight, E), flat_span(d.gate_weight, E)},
                        {y, flat_span(d.gate, n_tok)}) || overlaps(x, flat_span(d.gate, n_tok)))
            return false;
    }
    return true;
}

inline bool residual_args_ok(const gx_residual_desc &d, uint32_t n_tok) {
    if (d.n_embd == 0 || d.n_embd > kNormMaxWidth || n_tok > kMaxRows) return false;
    if (!(d.eps >= 0.f) || !std::isfinite(d.eps) || !std::isfinite(d.res_scale) || !std::isfinite(d.block_scale) ||
        (d.flags & ~(uint32_t)GX_RES_POST_NORM) || d.gate_kind > GX_GATE_ELEMENT)
        return false;
    const uint64_t E = d.n_embd;
    const bool post = (d.flags & GX_RES_POST_NORM) != 0;
    if (!act_dtype(d.y_dtype) || !act_dtype(d.res_dtype) || (d.post && !post) || (!d.out && (d.next || d.next_gate_weight)) ||
        !d.next_gate != !d.next_gate_weight || !words_ok(d.post) || !words_ok(d.next) ||
        !words_ok(d.next_gate_weight) || !words_ok(d.next_gate) || (d.gate_kind == GX_GATE_NONE && d.gate))
        return false;
    if (n_tok) {
        if (!rows_ok(d.y, d.y_dtype, d.y_stride, E) || !rows_ok(d.res, d.res_dtype, d.res_stride, E) ||
            !rows_ok(d.res_out, d.res_dtype, d.res_out_stride, E) ||
            (d.out && !rows_ok(d.out, d.out_dtype, d.out_stride, E)) ||
            (d.gate_kind == GX_GATE_ELEMENT && !rows_ok(d.gate, d.gate_dtype, d.gate_stride, E)) ||
            (d.gate_kind == GX_GATE_TOKEN && (!d.gate || !words_ok(d.gate))))
            return false;
        const Span y = rows_span(d.y, d.y_dtype, d.y_stride, E, n_tok);
        const Span res = rows_span(d.res, d.res_dtype, d.res_stride, E, n_tok);
        const Span ro = rows_span(d.res_out, d.res_dtype, d.res_out_stride, E, n_tok);
        const Span gate = d.gate_kind == GX_GATE_ELEMENT ? rows_span(d.gate, d.gate_dtype, d.gate_stride, E, n_tok)
                                                          : flat_span(d.gate, d.gate ? n_tok : 0);
        const Span out = d.out ? rows_span(d.out, d.out_dtype, d.out_stride, E, n_tok) : Span{};
        const Span ng = flat_span(d.next_gate, n_tok);
        const bool in_place = d.res == d.res_out && (d.res_stride == d.res_out_stride || n_tok == 1);
        if (any_overlap({y, gate, in_place ? Span{} : res, flat_span(d.post, E), flat_span(d.next, E),
                         flat_span(d.next_gate_weight, E)},
                        {ro, out, ng}) ||
            overlaps(res, out) || overlaps(res, ng))
            return false;
    }
    return true;
}

inline bool logprobs_args_ok(const gx_logprobs_desc &d, uint32_t n_rows) {
    if (d.n_vocab == 0 || d.n_vocab > kMaxVocab || d.n_top > GX_MAX_TOP || d.n_top > d.n_vocab ||
        n_rows > kMaxRows || !(d.scale > 0.f) || !(d.scale <= kMaxScale) || !act_dtype(d.dtype))
        return false;
    if ((!d.tokens && (d.logprob || d.rank)) || (!d.n_top && (d.top_ids || d.top_logprobs)) || !words_ok(d.tokens) ||
        !words_ok(d.logprob) || !words_ok(d.rank) || !words_ok(d.entropy) || !words_ok(d.top_ids) ||
        !words_ok(d.top_logprobs))
        return false;
    if (n_rows) {
        if (!rows_ok(d.logits, d.dtype, d.stride, d.n_vocab)) return false;
        const uint64_t nt = (uint64_t)n_rows * d.n_top;
        if (any_overlap({rows_span(d.logits, d.dtype, d.stride, d.n_vocab, n_rows), flat_span(d.tokens, n_rows)},
                        {flat_span(d.logprob, n_rows), flat_span(d.rank, n_rows), flat_span(d.entropy, n_rows),
                         flat_span(d.top_ids, nt), flat_span(d.top_logprobs, nt)}))
            return false;
    }
    return true;
}

inline bool norms_args_ok(const gx_norms_desc &d) {
    return d.post_norm <= 1 && (!d.post || d.post_norm) && d.eps >= 0.f && std::isfinite(d.eps) &&
           std::isfinite(d.res_scale) && std::isfinite(d.block_scale);
}

}  // namespace gx
