// A language model head's operators: 8-bit block quantization and its product, log probabilities of
// tokens with their gradient, distillation from a teacher's top alternatives. This file checks the
// operands; the kernels are beside it.
//
// Checks, first failure wins, nothing launched or written on error:
//   Wire              a dtype tag that is neither lg_dtype nor lg_head_dtype
//   Shape             null operands, ranks, extents that disagree or pass 31 bits, scalars
//   Dtype             each operand's element type
//   UnsupportedLayout rows of unit stride at a pitch of at least their length (any offset); where
//                     the entry point says so, the transpose_matrix view of such a matrix
//   Shape             an operand that reaches past its storage
//   Alias             an output whose bytes intersect another operand's
#include <algorithm>
#include <cmath>

#include "head.h"
#include "tensor_checks.h"

namespace lg {
namespace {

constexpr uint64_t EXTENT_MAX = 0x7fffff00ull;  // a tile's last row or slot still fits 32 bits
constexpr uint64_t ROW_MAX = 1ull << 29;        // columns of a row whose tiles one launch, or whose parts the scratch, has to hold

uint32_t element_bytes(const lg_tensor* t) {
    switch (t->dtype) {
        case LG_DTYPE_F32:
        case LG_DTYPE_I32:
            return 4;
        case LG_DTYPE_F16:
        case LG_DTYPE_BF16:
            return 2;
        case LG_DTYPE_E4M3:
        case LG_DTYPE_E8M0:
            return 1;
    }
    core_fail(LG_CORE_WIRE, "unknown dtype tag " + std::to_string(t->dtype));
}

// An operand's description, checked field by field as the entry points go along.
struct Operand {
    const lg_tensor* t = nullptr;
    const char* name = "";
    uint32_t rank = 2;
    bool turned = false;  // a transposed view: rows and cols are the view's
    uint64_t rows = 0, cols = 0, pitch = 0;
    uint64_t first = 0, end = 0;  // byte addresses

    explicit operator bool() const { return t != nullptr; }
    template <typename T>
    T* at() const {
        return reinterpret_cast<T*>(first);
    }
    // 0 for an operand without elements, whose strides may hold anything.
    int64_t step() const { return first == end ? 0 : static_cast<int64_t>(pitch); }
};

Operand operand(const lg_tensor* t, const char* name, uint32_t rank, bool optional = false) {
    Operand o;
    o.name = name;
    o.rank = rank;
    if (t == nullptr) {
        if (!optional) core_fail(LG_CORE_SHAPE, std::string("null tensor ") + name);
        return o;
    }
    o.t = t;
    return o;
}

void decode(std::initializer_list<Operand*> ops) {
    for (Operand* o : ops) {
        if (*o && (o->t->rank > LG_MAX_RANK || o->t->nstrides > LG_MAX_RANK)) {
            core_fail(LG_CORE_SHAPE, std::string(o->name) + " rank above LG_MAX_RANK");
        }
    }
    for (Operand* o : ops) {
        if (*o) element_bytes(o->t);
    }
    for (Operand* o : ops) {
        if (!*o) continue;
        if (o->t->rank != o->rank || o->t->nstrides != o->rank) {
            core_fail(LG_CORE_SHAPE, std::string(o->name) + " is not rank " + std::to_string(o->rank));
        }
        o->rows = o->rank == 2 ? o->t->shape[0] : 1;
        o->cols = o->t->shape[o->rank - 1];
        if (o->rows > EXTENT_MAX || o->cols > EXTENT_MAX) {
            core_fail(LG_CORE_SHAPE, std::string(o->name) + " extents must fit 31 bits");
        }
    }
}

void need(bool ok, const char* what) {
    if (!ok) core_fail(LG_CORE_SHAPE, what);
}

void dtype(const Operand& o, std::initializer_list<uint32_t> allowed) {
    if (!o) return;
    for (uint32_t d : allowed) {
        if (o.t->dtype == d) return;
    }
    core_fail(LG_CORE_DTYPE, std::string(o.name) + " has an element type that this operator does not take");
}

// Unit stride along rows at any pitch; `turnable`: or along columns.
void layout(Operand& o, bool turnable = false) {
    if (!o) return;
    const uint64_t* st = o.t->strides;
    const uint64_t sr = o.rank == 2 ? st[0] : o.cols, sc = st[o.rank - 1];
    const bool empty = o.rows == 0 || o.cols == 0;
    if (empty || ((sc == 1 || o.cols == 1) && (o.rows == 1 || sr >= o.cols))) {
        o.pitch = o.rows == 1 ? o.cols : sr;
    } else if (turnable && sr == 1 && (o.cols == 1 || sc >= o.rows)) {
        o.turned = true;
        o.pitch = o.cols == 1 ? o.rows : sc;
    } else {
        core_fail(LG_CORE_UNSUPPORTED_LAYOUT, std::string(o.name) + " does not have rows of unit stride");
    }
}

void storage(Operand& o) {
    if (!o) return;
    const uint64_t size = element_bytes(o.t), lines = o.turned ? o.cols : o.rows, length = o.turned ? o.rows : o.cols;
    const uint64_t base = reinterpret_cast<uint64_t>(o.t->base);
    const std::string past = std::string(o.name) + " reaches past its storage";
    if (lines == 0 || length == 0) {
        o.first = o.end = base;
        return;
    }
    if (o.t->base == nullptr) core_fail(LG_CORE_SHAPE, std::string(o.name) + " has no storage");
    if (o.t->offset > o.t->bytes || (lines > 1 && o.pitch > o.t->bytes / (lines - 1))) core_fail(LG_CORE_SHAPE, past);
    // Both terms are at most `bytes` here; their sum and the length cannot wrap once they are below a quarter of all.
    if (o.t->offset > UINT64_MAX / 4 || (lines - 1) * o.pitch > UINT64_MAX / 4) core_fail(LG_CORE_SHAPE, past);
    const uint64_t elements = o.t->offset + (lines - 1) * o.pitch + length;
    if (elements > o.t->bytes / size) core_fail(LG_CORE_SHAPE, past);
    o.first = base + o.t->offset * size;
    o.end = base + elements * size;
    if (o.first % size != 0) core_fail(LG_CORE_UNSUPPORTED_LAYOUT, std::string(o.name) + " is misaligned for its element type");
}

void disjoint(const Operand& out, std::initializer_list<const Operand*> others) {
    if (!out) return;
    for (const Operand* o : others) {
        if (*o && out.first < o->end && o->first < out.end) {
            core_fail(LG_CORE_ALIAS, std::string(out.name) + " shares memory with " + o->name);
        }
    }
}

bool same_place(const Operand& a, const Operand& b) {
    return a.first == b.first && a.pitch == b.pitch && a.t->dtype == b.t->dtype;
}

// Rows that share a scale, from the extents of `scales` for a matrix of rows x cols.
uint32_t scale_block(const Operand& scales, uint64_t rows, uint64_t cols) {
    need(scales.cols == (cols + BLOCK_K - 1) / BLOCK_K, "scales need a column for each 128 columns of their matrix");
    if (scales.rows == rows) return 1;
    need(scales.rows == (rows + BLOCK_K - 1) / BLOCK_K, "scales need a row for each row, or each 128 rows, of their matrix");
    return BLOCK_K;
}

void check_temperature(float t) {
    // log2(e) / t and 1 / t stay normal numbers.
    need(std::isfinite(t) && t >= 0x1p-60f && t <= 0x1p60f, "temperature must lie in [2^-60, 2^60]");
}

uint32_t u32(uint64_t v) { return static_cast<uint32_t>(v); }

// In parts whose threads a launch has 32-bit numbers for, whole blocks of 128 rows each. (Pitches from 2^23 on take small tiles.)
void launch_gemm_blocks(lg_ctx* ctx, hipStream_t s, const GemmBlocksArgs& g) {
    const uint32_t part = std::max(g.a_pitch, g.b_pitch) >= 1 << 23 ? 1u << 16 : 1u << 22;
    const uint64_t scale = g.e8m0 ? 1 : 4, out = g.out == LG_DTYPE_F32 ? 4 : 2;
    for (uint32_t m = 0; m < g.m; m += part) {
        for (uint32_t n = 0; n < g.n; n += part) {
            GemmBlocksArgs p = g;
            p.m = std::min(g.m - m, part);
            p.n = std::min(g.n - n, part);
            p.a += m * g.a_pitch;
            p.b += n * g.b_pitch;
            p.sa = static_cast<const char*>(g.sa) + m / g.a_block * g.sa_pitch * scale;
            p.sb = static_cast<const char*>(g.sb) + n / g.b_block * g.sb_pitch * scale;
            p.c = static_cast<char*>(g.c) + (m * g.c_pitch + n) * out;
            if (g.out == LG_DTYPE_F32) {
                launch_gemm_blocks_f32(ctx, s, p);
            } else if (g.out == LG_DTYPE_F16) {
                launch_gemm_blocks_f16(ctx, s, p);
            } else {
                launch_gemm_blocks_bf16(ctx, s, p);
            }
        }
    }
}

}  // namespace
}  // namespace lg

using namespace lg;

extern "C" {

lg_core_error lg_backend_quantize_blocks(lg_ctx* ctx, void* stream, const lg_tensor* x,
                                         const lg_tensor* q, const lg_tensor* scales) {
    return run_op([&] {
        Operand ox = operand(x, "x", 2), oq = operand(q, "q", 2), os = operand(scales, "scales", 2);
        decode({&ox, &oq, &os});
        need(ox.rows == oq.rows && ox.cols == oq.cols, "quantize_blocks needs x and q of one shape");
        QuantizeArgs a{};
        a.block = scale_block(os, oq.rows, oq.cols);
        need(oq.cols <= ROW_MAX, "quantize_blocks takes rows of at most 2^29 columns");
        dtype(ox, {LG_DTYPE_F32, LG_DTYPE_F16, LG_DTYPE_BF16});
        dtype(oq, {LG_DTYPE_E4M3});
        dtype(os, {LG_DTYPE_F32, LG_DTYPE_E8M0});
        layout(ox, true);
        layout(oq);
        layout(os);
        for (Operand* o : {&ox, &oq, &os}) storage(*o);
        disjoint(oq, {&ox, &os});
        disjoint(os, {&ox});
        hipStream_t s = device_stream(ctx, stream);
        if (oq.rows == 0 || oq.cols == 0) return;
        a.x = ox.at<void>();
        a.x_pitch = ox.step();
        a.q = oq.at<uint8_t>();
        a.q_pitch = oq.step();
        a.s = os.at<void>();
        a.s_pitch = os.step();
        a.rows = u32(oq.rows);
        a.cols = u32(oq.cols);
        a.dtype = x->dtype;
        a.transposed = ox.turned;
        a.e8m0 = scales->dtype == LG_DTYPE_E8M0;
        launch_quantize_blocks(ctx, s, a);
    });
}

lg_core_error lg_backend_gemm_blocks(lg_ctx* ctx, void* stream, const lg_tensor* a,
                                     const lg_tensor* a_scales, const lg_tensor* b,
                                     const lg_tensor* b_scales, const lg_tensor* c, float alpha,
                                     float beta) {
    return run_op([&] {
        Operand oa = operand(a, "a", 2), osa = operand(a_scales, "a_scales", 2), ob = operand(b, "b", 2);
        Operand osb = operand(b_scales, "b_scales", 2), oc = operand(c, "c", 2);
        decode({&oa, &osa, &ob, &osb, &oc});
        need(oa.cols == ob.rows && oa.rows == oc.rows && ob.cols == oc.cols, "extents of a, b and c disagree");
        GemmBlocksArgs g{};
        g.a_block = scale_block(osa, oa.rows, oa.cols);
        g.b_block = scale_block(osb, ob.cols, ob.rows);
        dtype(oa, {LG_DTYPE_E4M3});
        dtype(ob, {LG_DTYPE_E4M3});
        dtype(osa, {LG_DTYPE_F32, LG_DTYPE_E8M0});
        dtype(osb, {a_scales->dtype});
        dtype(oc, {LG_DTYPE_F32, LG_DTYPE_F16, LG_DTYPE_BF16});
        layout(oa);
        layout(ob, true);
        // One row or column of b is both; otherwise b has to be the transposed view.
        if (!ob.turned && ob.rows > 1 && ob.cols > 1) core_fail(LG_CORE_UNSUPPORTED_LAYOUT, "b is not the transposed view of a row-major matrix");
        if (!ob.turned && ob.rows > 0 && ob.cols > 0) {
            const uint64_t sk = b->strides[0], sn = b->strides[1];
            if ((ob.rows > 1 && sk != 1) || (ob.cols > 1 && sn < ob.rows)) core_fail(LG_CORE_UNSUPPORTED_LAYOUT, "b is not the transposed view of a row-major matrix");
            ob.turned = true;
            ob.pitch = ob.cols == 1 ? ob.rows : sn;
        }
        layout(osa);
        layout(osb);
        layout(oc);
        for (Operand* o : {&oa, &osa, &ob, &osb, &oc}) storage(*o);
        disjoint(oc, {&oa, &osa, &ob, &osb});
        hipStream_t s = device_stream(ctx, stream);
        if (oc.rows == 0 || oc.cols == 0) return;
        g.a = oa.at<uint8_t>();
        g.a_pitch = oa.step();
        g.b = ob.at<uint8_t>();
        g.b_pitch = ob.step();
        g.sa = osa.at<void>();
        g.sa_pitch = osa.step();
        g.sb = osb.at<void>();
        g.sb_pitch = osb.step();
        g.c = oc.at<void>();
        g.c_pitch = oc.step();
        g.m = u32(oc.rows);
        g.n = u32(oc.cols);
        g.k = alpha == 0.0f ? 0 : u32(oa.cols);  // as in Backend::gemm, alpha = 0 reads neither A nor B
        g.out = c->dtype;
        g.alpha = alpha;
        g.beta = beta;
        g.e8m0 = a_scales->dtype == LG_DTYPE_E8M0;
        launch_gemm_blocks(ctx, s, g);
    });
}

lg_core_error lg_backend_token_logprobs(lg_ctx* ctx, void* stream, const lg_tensor* logits,
                                        const lg_tensor* tokens, float temperature,
                                        const lg_tensor* logprobs, const lg_tensor* entropy,
                                        const lg_tensor* stats, const lg_tensor* top_logprobs,
                                        const lg_tensor* top_ids) {
    return run_op([&] {
        Operand x = operand(logits, "logits", 2), t = operand(tokens, "tokens", 1, true);
        Operand lp = operand(logprobs, "logprobs", 1, true), h = operand(entropy, "entropy", 1, true);
        Operand st = operand(stats, "stats", 2, true), top = operand(top_logprobs, "top_logprobs", 2, true);
        Operand ids = operand(top_ids, "top_ids", 2, true);
        decode({&x, &t, &lp, &h, &st, &top, &ids});
        need(bool(t) == bool(lp), "tokens and logprobs come together");
        need(bool(top) == bool(ids), "top_logprobs and top_ids come together");
        need((!t || t.cols == x.rows) && (!lp || lp.cols == x.rows) && (!h || h.cols == x.rows),
             "tokens, logprobs and entropy need an element for each row of logits");
        need(!st || (st.rows == x.rows && st.cols == 2), "stats needs shape [rows, 2]");
        need(!top || (top.rows == x.rows && ids.rows == x.rows && top.cols == ids.cols && top.cols <= TOP_MAX),
             "top_logprobs and top_ids need shape [rows, k] with k of at most 128");
        need(!top || top.cols == 0 || x.cols <= ROW_MAX, "alternatives are of rows of at most 2^29 logits");
        check_temperature(temperature);
        dtype(x, {LG_DTYPE_F32, LG_DTYPE_F16, LG_DTYPE_BF16});
        for (const Operand* o : {&t, &ids}) dtype(*o, {LG_DTYPE_I32});
        for (const Operand* o : {&lp, &h, &st, &top}) dtype(*o, {LG_DTYPE_F32});
        for (Operand* o : {&x, &t, &lp, &h, &st, &top, &ids}) layout(*o);
        for (Operand* o : {&x, &t, &lp, &h, &st, &top, &ids}) storage(*o);
        disjoint(lp, {&x, &t, &h, &st, &top, &ids});
        disjoint(h, {&x, &t, &st, &top, &ids});
        disjoint(st, {&x, &t, &top, &ids});
        disjoint(top, {&x, &t, &ids});
        disjoint(ids, {&x, &t});
        hipStream_t s = device_stream(ctx, stream);
        if (x.rows == 0) return;
        LogprobArgs a{};
        a.x = x.at<void>();
        a.x_pitch = x.step();
        a.dtype = logits->dtype;
        a.rows = u32(x.rows);
        a.cols = u32(x.cols);
        a.temperature = temperature;
        if (t) a.tokens = t.at<int32_t>(), a.logprobs = lp.at<float>();
        if (h) a.entropy = h.at<float>();
        if (st) a.stats = st.at<float>(), a.stats_pitch = st.step();
        if (top && top.cols > 0) {
            a.top = top.at<float>();
            a.top_ids = ids.at<int32_t>();
            a.top_pitch = top.step();
            a.ids_pitch = ids.step();
            a.k = u32(top.cols);
        }
        launch_token_logprobs(ctx, s, a);
    });
}

lg_core_error lg_backend_token_logprobs_backward(lg_ctx* ctx, void* stream, const lg_tensor* logits,
                                                 const lg_tensor* tokens, float temperature,
                                                 const lg_tensor* stats, const lg_tensor* entropy,
                                                 const lg_tensor* dlogprobs,
                                                 const lg_tensor* dentropy,
                                                 const lg_tensor* dlogits) {
    return run_op([&] {
        Operand x = operand(logits, "logits", 2), t = operand(tokens, "tokens", 1), st = operand(stats, "stats", 2);
        Operand h = operand(entropy, "entropy", 1, true), g = operand(dlogprobs, "dlogprobs", 1);
        Operand gh = operand(dentropy, "dentropy", 1, true), dx = operand(dlogits, "dlogits", 2);
        decode({&x, &t, &st, &h, &g, &gh, &dx});
        need(h || !gh, "dentropy needs entropy");
        need(t.cols == x.rows && g.cols == x.rows && (!h || h.cols == x.rows) && (!gh || gh.cols == x.rows),
             "tokens, entropy, dlogprobs and dentropy need an element for each row of logits");
        need(st.rows == x.rows && st.cols == 2, "stats needs shape [rows, 2]");
        need(dx.rows == x.rows && dx.cols == x.cols, "logits and dlogits differ in shape");
        check_temperature(temperature);
        dtype(x, {LG_DTYPE_F32, LG_DTYPE_F16, LG_DTYPE_BF16});
        dtype(dx, {logits->dtype});
        dtype(t, {LG_DTYPE_I32});
        for (const Operand* o : {&st, &h, &g, &gh}) dtype(*o, {LG_DTYPE_F32});
        for (Operand* o : {&x, &t, &st, &h, &g, &gh, &dx}) layout(*o);
        for (Operand* o : {&x, &t, &st, &h, &g, &gh, &dx}) storage(*o);
        disjoint(dx, {&t, &st, &h, &g, &gh});
        if (!same_place(dx, x)) disjoint(dx, {&x});
        hipStream_t s = device_stream(ctx, stream);
        if (x.rows == 0 || x.cols == 0) return;
        LogprobBackArgs a{};
        a.x = x.at<void>();
        a.dx = dx.at<void>();
        a.x_pitch = x.step();
        a.dx_pitch = dx.step();
        a.dtype = logits->dtype;
        a.rows = u32(x.rows);
        a.cols = u32(x.cols);
        a.temperature = temperature;
        a.tokens = t.at<int32_t>();
        a.stats = st.at<float>();
        a.stats_pitch = st.step();
        a.dlogprobs = g.at<float>();
        if (gh) a.entropy = h.at<float>(), a.dentropy = gh.at<float>();
        launch_token_logprobs_backward(ctx, s, a);
    });
}

lg_core_error lg_backend_distill_grad(lg_ctx* ctx, void* stream, const lg_tensor* logits,
                                      const lg_tensor* teacher_ids,
                                      const lg_tensor* teacher_logprobs, const lg_tensor* weights,
                                      float temperature, int32_t normalize,
                                      const lg_tensor* losses, const lg_tensor* dlogits) {
    return run_op([&] {
        Operand x = operand(logits, "logits", 2), ids = operand(teacher_ids, "teacher_ids", 2);
        Operand v = operand(teacher_logprobs, "teacher_logprobs", 2), w = operand(weights, "weights", 1, true);
        Operand loss = operand(losses, "losses", 1), dx = operand(dlogits, "dlogits", 2, true);
        decode({&x, &ids, &v, &w, &loss, &dx});
        need(ids.rows == x.rows && v.rows == x.rows && ids.cols == v.cols && v.cols <= TOP_MAX,
             "teacher_ids and teacher_logprobs need shape [rows, k] with k of at most 128");
        need((!w || w.cols == x.rows) && loss.cols == x.rows, "weights and losses need an element for each row of logits");
        need(!dx || (dx.rows == x.rows && dx.cols == x.cols), "logits and dlogits differ in shape");
        check_temperature(temperature);
        dtype(x, {LG_DTYPE_F32, LG_DTYPE_F16, LG_DTYPE_BF16});
        dtype(dx, {logits->dtype});
        dtype(ids, {LG_DTYPE_I32});
        for (const Operand* o : {&v, &w, &loss}) dtype(*o, {LG_DTYPE_F32});
        for (Operand* o : {&x, &ids, &v, &w, &loss, &dx}) layout(*o);
        for (Operand* o : {&x, &ids, &v, &w, &loss, &dx}) storage(*o);
        disjoint(loss, {&x, &ids, &v, &w, &dx});
        disjoint(dx, {&ids, &v, &w});
        if (dx && !same_place(dx, x)) disjoint(dx, {&x});
        hipStream_t s = device_stream(ctx, stream);
        if (x.rows == 0) return;
        DistillArgs a{};
        a.x = x.at<void>();
        a.x_pitch = x.step();
        if (dx) a.dx = dx.at<void>(), a.dx_pitch = dx.step();
        a.dtype = logits->dtype;
        a.rows = u32(x.rows);
        a.cols = u32(x.cols);
        a.ids = ids.at<int32_t>();
        a.values = v.at<float>();
        a.ids_pitch = ids.step();
        a.values_pitch = v.step();
        a.k = u32(v.cols);
        if (w) a.weights = w.at<float>();
        a.temperature = temperature;
        a.normalize = normalize != 0;
        a.losses = loss.at<float>();
        launch_distill_grad(ctx, s, a);
    });
}

}  // extern "C"
