// Support rules of the serving ops: shapes, types, strides and limits, from the descriptors alone.
#include "serving.h"

#include "../core/tensor_math.h"

#include <algorithm>
#include <cmath>
#include <cstddef>
#include <cstring>

namespace {

using Desc = scrapgpu_tensor_desc;

struct Refusal {
    const char ** reason;
    scrapgpu_status operator()(scrapgpu_status st, const char * m) const {
        if (reason) *reason = m;
        scrapgpu_set_last_error(m);
        return st;
    }
    scrapgpu_status bad(const char * m) const { return (*this)(SCRAPGPU_STATUS_INVALID_ARGUMENT, m); }
    scrapgpu_status no(const char * m) const { return (*this)(SCRAPGPU_STATUS_UNSUPPORTED, m); }
};

bool half(scrapgpu_dtype t) {
    return t == SCRAPGPU_DTYPE_F16 || t == SCRAPGPU_DTYPE_BF16;
}
bool real(scrapgpu_dtype t) {
    return t == SCRAPGPU_DTYPE_F32 || half(t);
}

// extents beyond the given ones are 1 (or unset); none is negative
bool shape(const Desc & t, int64_t a, int64_t b = 1, int64_t c = 1, int64_t d = 1) {
    const int64_t want[4] = {a, b, c, d};
    for (int i = 0; i < 4; ++i)
        if (t.ne[i] != want[i] && !(want[i] == 1 && sg::dim1(t.ne[i]) == 1 && t.ne[i] >= 0 && i > 0)) return false;
    return true;
}

// nb0 the element size, the other strides (of extents over 1) and the offset multiples of `align`
bool strides(const Desc & t, uint64_t align) {
    if (t.layout != SCRAPGPU_LAYOUT_NATURAL || t.nb[0] != sg::type_size(t.dtype) || t.offset % align != 0) return false;
    for (int i = 1; i < 4; ++i)
        if (t.ne[i] > 1 && t.nb[i] % align != 0) return false;
    return true;
}

bool ints(const Desc & t) {
    return t.dtype == SCRAPGPU_DTYPE_I32 && strides(t, 4);
}

// elements of different indices lie apart: every stride covers what lies inside it, in some order
bool injective(const Desc & t) {
    uint64_t span = sg::type_size(t.dtype) * (uint64_t) sg::dim1(t.ne[0]);
    bool used[4] = {true, false, false, false};
    for (int k = 1; k < 4; ++k) {
        int best = -1;
        for (int i = 1; i < 4; ++i)
            if (!used[i] && (best < 0 || t.nb[i] < t.nb[best] || t.ne[i] <= 1)) best = i;
        used[best] = true;
        if (t.ne[best] <= 1) continue;
        if (t.nb[best] < span) return false;
        span = sg::sat_add(sg::sat_mul(t.nb[best], (uint64_t) (t.ne[best] - 1)), span);
    }
    return true;
}

bool same(const Desc & a, const Desc & b) {
    if (a.buffer != b.buffer || a.offset != b.offset || a.dtype != b.dtype) return false;
    for (int i = 0; i < 4; ++i)
        if (sg::dim1(a.ne[i]) != sg::dim1(b.ne[i]) || (a.ne[i] > 1 && a.nb[i] != b.nb[i])) return false;
    return true;
}

// No byte of a is a byte of b: ranges that do not meet, or that interleave. Where both repeat over an axis of
// one stride s, and what is left of each without it (one token, one page) is no longer than s, it is enough that
// one a is apart from the b at most s after it and from the one before that (q, k, v side by side in each token's
// row; k and v pages in turn).
bool apart(const Desc & a, const Desc & b) {
    if (a.buffer == nullptr || a.buffer != b.buffer) return true;
    const uint64_t na = sg::nbytes(a), nb = sg::nbytes(b);
    if (na == 0 || nb == 0 || sg::sat_add(a.offset, na) <= b.offset || sg::sat_add(b.offset, nb) <= a.offset) return true;
    for (int i = 1; i < 4; ++i)
        for (int j = 1; j < 4; ++j) {
            const uint64_t s = a.nb[i];
            if (a.ne[i] <= 1 || b.ne[j] <= 1 || s == 0 || b.nb[j] != s) continue;
            Desc ta = a, tb = b;
            ta.ne[i] = tb.ne[j] = 1;
            if (sg::nbytes(ta) > s || sg::nbytes(tb) > s) continue;
            // (offsets mod s; s more on both sides for the b before)
            const uint64_t between = (b.offset % s + s - a.offset % s) % s;
            ta.offset = s;
            tb.offset = s + between;
            if (!apart(ta, tb)) continue;
            tb.offset = between;
            if (apart(ta, tb)) return true;
        }
    return false;
}

scrapgpu_status all_apart(const scrapgpu_op_desc * d, const Refusal & fail) {
    for (size_t o = 0; o < d->output_count; ++o) {
        for (size_t i = 0; i < d->input_count; ++i)
            if (!apart(d->outputs[o], d->inputs[i])) {
                const bool in_place = (d->op == SCRAPGPU_OP_ROPE_AXES || d->op == SCRAPGPU_OP_ROPE_AXES_STORE) && o == 0 && i == 0 && same(d->outputs[0], d->inputs[0]);
                // PAGED_PLAN: kv_len over past, left's first element over free
                const bool carried = d->op == SCRAPGPU_OP_PAGED_PLAN && ((o == 4 && i == 0 && same(d->outputs[4], d->inputs[0])) ||
                                                                          (o == 2 && i == 2 && d->outputs[2].offset == d->inputs[2].offset));
                if (!in_place && !carried) return fail.bad("an output overlaps an input");
            }
        for (size_t p = 0; p < o; ++p)
            if (!apart(d->outputs[o], d->outputs[p])) return fail.bad("two outputs overlap");
    }
    return SCRAPGPU_STATUS_OK;
}

int log2_exact(uint64_t v) {
    if (v == 0 || (v & (v - 1)) != 0) return -1;
    int s = 0;
    while ((v >> s) != 1) ++s;
    return s;
}

void put(ServingOp * out, const Desc & t, const char * what, void * at) {
    out->slots[out->n_slots++] = {&t, what, at};
}

scrapgpu_status plan_rule(const scrapgpu_op_desc * d, ServingOp * out, const Refusal & fail) {
    const auto * p = static_cast<const scrapgpu_paged_plan_params *>(d->params);
    const Desc *in = d->inputs, *o = d->outputs;
    for (size_t i = 0; i < d->input_count; ++i)
        if (!ints(in[i])) return fail.no("PAGED_PLAN takes contiguous I32 tensors");
    for (size_t i = 0; i < d->output_count; ++i)
        if (!ints(o[i])) return fail.no("PAGED_PLAN takes contiguous I32 tensors");
    const int shift = log2_exact(p->page_size);
    if (shift < 0 || p->page_size > 65536) return fail.no("PAGED_PLAN: the page size must be a power of two, at most 65536");
    const int64_t B = in[0].ne[0], W = o[0].ne[0], P = o[1].ne[0], T = o[5].ne[0];
    if (B <= 0 || W <= 0 || P <= 0 || T <= 0 || !shape(in[0], B) || !shape(in[1], B) || !shape(in[2], 1) || !shape(o[0], W, B) || !shape(o[1], P) || !shape(o[2], 2) ||
        !shape(o[3], B + 1) || !shape(o[4], B) || !shape(o[5], T) || !shape(o[6], T)) {
        return fail.bad("PAGED_PLAN needs past [B], fresh [B], free [1] and table [W,B], pool [n], left [2], q_start [B+1], kv_len [B], pos [T], slots [T]");
    }
    if (B > sgk::kPlanRequests) return fail.no("PAGED_PLAN: more than 2048 requests");
    if (sg::sat_mul((uint64_t) W, p->page_size) >= (1u << 30) || P >= (1 << 30) || T >= (1 << 30)) return fail.no("PAGED_PLAN: a request's tokens (W x page size), the pool and the step's tokens must be fewer than 2^30");
    if (!injective(o[0])) return fail.bad("PAGED_PLAN: table rows overlap");
    const scrapgpu_status st = all_apart(d, fail);
    if (st != SCRAPGPU_STATUS_OK || out == nullptr) return st;
    sgk::PlanLaunch & a = out->plan;
    std::memset(&a, 0, sizeof(a));
    a.t_s1 = (int64_t) (o[0].nb[1] / 4);
    a.B = (int) B;
    a.W = (int) W;
    a.P = (int) P;
    a.T = (int) T;
    a.shift = shift;
    put(out, in[0], "past", &a.past);
    put(out, in[1], "fresh", &a.fresh);
    put(out, in[2], "free", &a.free_in);
    put(out, o[0], "table", &a.table);
    put(out, o[1], "pool", &a.pool);
    put(out, o[2], "left", &a.left);
    put(out, o[3], "q_start", &a.q_start);
    put(out, o[4], "kv_len", &a.kv_len);
    put(out, o[5], "pos", &a.pos);
    put(out, o[6], "slots", &a.slots);
    out->bytes = 4.0 * (double) (4 * B + 2 * T);
    return SCRAPGPU_STATUS_OK;
}

// the k and v caches: [D, page, Hk, n_pages], one shape and type
scrapgpu_status cache_rule(const Desc & k, const Desc & v, int64_t D, int64_t Hk, int * shift, const Refusal & fail) {
    if (!half(k.dtype) && k.dtype != SCRAPGPU_DTYPE_F32) return fail.no("the cache must be F16, BF16 or F32");
    if (k.dtype != v.dtype) return fail.no("both caches must have one type");
    const int64_t page = k.ne[1], pages = sg::dim1(k.ne[3]);
    if (k.ne[1] <= 0 || k.ne[3] < 0 || !shape(k, D, page, Hk, pages) || !shape(v, D, page, Hk, pages)) return fail.bad("the caches must be [D, page size, Hk, pages] both");
    *shift = log2_exact((uint64_t) page);
    if (*shift < 0 || page > 65536) return fail.no("the page size must be a power of two, at most 65536");
    if (sg::sat_mul((uint64_t) page, (uint64_t) pages) >= ((uint64_t) 1 << 31)) return fail.no("the cache must have fewer than 2^31 slots");
    if (!strides(k, 16) || !strides(v, 16)) return fail.no("cache strides and offsets must be multiples of 16 bytes, nb0 the element size");
    // (the attention kernels multiply page numbers by 32-bit strides)
    if ((pages > 1 && (k.nb[3] >> 32 || v.nb[3] >> 32)) || sg::sat_mul((uint64_t) page, std::max(k.nb[1], v.nb[1])) >> 31) return fail.no("the cache's pages must lie less than 4 GiB apart, a page's places within 2 GiB");
    return SCRAPGPU_STATUS_OK;
}

scrapgpu_status rope_rule(const scrapgpu_op_desc * d, ServingOp * out, const Refusal & fail) {
    const auto * p = static_cast<const scrapgpu_rope_axes_params *>(d->params);
    const bool store = d->op == SCRAPGPU_OP_ROPE_AXES_STORE;
    const Desc &q = d->inputs[0], &y = d->outputs[0], &pos = d->inputs[store ? 3 : 1];
    const int64_t D = q.ne[0], Hq = sg::dim1(q.ne[1]), T = q.ne[2] == 0 ? 0 : sg::dim1(q.ne[2]), A = pos.ne[0];
    if (!real(q.dtype) || !real(y.dtype)) return fail.no("ROPE_AXES takes F32, F16 and BF16 tensors");
    if (!strides(q, sg::type_size(q.dtype)) || !strides(y, sg::type_size(y.dtype))) return fail.no("ROPE_AXES: nb0 must be the element size, strides and offsets whole elements");
    if (!ints(pos)) return fail.no("ROPE_AXES: pos must be contiguous I32 rows");
    if (D <= 0 || q.ne[1] < 0 || q.ne[2] < 0 || !shape(q, D, Hq, T) || !shape(y, D, Hq, T)) return fail.bad("ROPE_AXES: x and y must be [D, H, T] both");
    if (A < 1 || A > 4 || !shape(pos, A, T)) return fail.bad("ROPE_AXES: pos must be [axes, T] with 1 to 4 axes");
    if (D % 2 != 0) return fail.no("ROPE_AXES: D must be even");
    if (D > 4096 || T >= (1 << 30) || Hq >= (1 << 20)) return fail.no("ROPE_AXES: D over 4096, or too many heads or tokens");
    const int64_t n = p->n_dims;
    if (n % 2 != 0 || n > D) return fail.bad("ROPE_AXES: n_dims must be even and at most D");
    if (n > 256) return fail.no("ROPE_AXES: n_dims over 256");
    if (!(p->base > 0.0f) || !std::isfinite(p->base) || !std::isfinite(p->scale)) return fail.bad("ROPE_AXES: base must be positive, base and scale finite");
    uint64_t sum = 0;
    for (int i = 0; i < 4; ++i) {
        sum += p->sections[i];
        if (i >= A && p->sections[i] != 0) return fail.bad("ROPE_AXES: a section for an axis that pos does not have");
    }
    if (sum != 0 ? sum != (uint64_t) n / 2 : A != 1) return fail.bad("ROPE_AXES: the sections must add up to n_dims / 2 (or all be zero with one axis)");
    if (!injective(y)) return fail.bad("ROPE_AXES: elements of y overlap");
    int64_t Hk = 0;
    int shift = 0;
    if (store) {
        const Desc &k = d->inputs[1], &v = d->inputs[2], &slots = d->inputs[4], &kc = d->outputs[1], &vc = d->outputs[2];
        Hk = sg::dim1(k.ne[1]);
        if (k.dtype != q.dtype || v.dtype != q.dtype) return fail.no("ROPE_AXES_STORE: q, k and v must have one type");
        if (!strides(k, sg::type_size(k.dtype)) || !strides(v, sg::type_size(v.dtype))) return fail.no("ROPE_AXES: nb0 must be the element size, strides and offsets whole elements");
        if (k.ne[1] < 0 || !shape(k, D, Hk, T) || !shape(v, D, Hk, T)) return fail.bad("ROPE_AXES_STORE: k and v must be [D, Hk, T] both");
        if (!ints(slots)) return fail.no("ROPE_AXES_STORE: slots must be contiguous I32");
        if (!shape(slots, T)) return fail.bad("ROPE_AXES_STORE: slots must be [T]");
        if (Hk >= (1 << 20)) return fail.no("ROPE_AXES: D over 4096, or too many heads or tokens");
        const scrapgpu_status st = cache_rule(kc, vc, D, Hk, &shift, fail);
        if (st != SCRAPGPU_STATUS_OK) return st;
        if (!injective(kc) || !injective(vc)) return fail.bad("ROPE_AXES_STORE: elements of a cache overlap");
    }
    const scrapgpu_status st = all_apart(d, fail);
    if (st != SCRAPGPU_STATUS_OK || out == nullptr) return st;
    sgk::RopeLaunch & r = out->rope;
    std::memset(&r, 0, sizeof(r));
    out->empty = T == 0;
    r.in_type = q.dtype;
    r.out_type = y.dtype;
    r.cache_type = store ? d->outputs[1].dtype : y.dtype;
    r.q_s1 = q.nb[1];
    r.q_s2 = q.nb[2];
    r.y_s1 = y.nb[1];
    r.y_s2 = y.nb[2];
    r.p_s1 = (int64_t) (pos.nb[1] / 4);
    r.T = (int) T;
    r.Hq = (int) Hq;
    r.Hk = (int) Hk;
    r.D = (int) D;
    r.n_dims = (int) n;
    r.shift = shift;
    r.adjacent = p->adjacent != 0;
    // turns per position in 64-bit fixed point: position times this, mod 2^64, is the angle mod one
    // turn without any loss, whatever the position
    const long double step = n ? powl((long double) p->base, -2.0L / (long double) n) : 1.0L;
    long double f = (long double) p->scale / 6.283185307179586476925286766559L;
    for (int i = 0, ax = 0, used = 0; i < (int) n / 2; ++i, f *= step) {
        const long double frac = f >= 0.0L && f < 1.0L ? f : f - floorl(f);
        r.turn[i] = frac >= 1.0L ? 0 : (uint64_t) (frac * 18446744073709551616.0L);
        if (sum == 0) continue; // one axis
        if (p->interleaved) {
            const int e = i % (int) A;
            r.axis[i] = (uint8_t) (e > 0 && (uint64_t) i < (uint64_t) A * p->sections[e] ? e : 0);
        } else {
            while (used == (int) p->sections[ax]) {
                ++ax;
                used = 0;
            }
            r.axis[i] = (uint8_t) ax;
            ++used;
        }
    }
    put(out, q, "x", &r.q);
    put(out, pos, "pos", &r.pos);
    put(out, y, "y", &r.y);
    if (store) {
        const Desc &k = d->inputs[1], &v = d->inputs[2], &kc = d->outputs[1], &vc = d->outputs[2];
        r.k_s1 = k.nb[1];
        r.k_s2 = k.nb[2];
        r.v_s1 = v.nb[1];
        r.v_s2 = v.nb[2];
        r.kc_s1 = kc.nb[1];
        r.kc_s2 = kc.nb[2];
        r.kc_s3 = kc.nb[3];
        r.vc_s1 = vc.nb[1];
        r.vc_s2 = vc.nb[2];
        r.vc_s3 = vc.nb[3];
        r.n_slots = kc.ne[1] * sg::dim1(kc.ne[3]);
        put(out, k, "k", &r.k);
        put(out, v, "v", &r.v);
        put(out, d->inputs[4], "slots", &r.slots);
        put(out, kc, "k_cache", &r.kc);
        put(out, vc, "v_cache", &r.vc);
    }
    out->bytes = (double) T * (double) D * (double) (Hq + 2 * Hk) * (double) (sg::type_size(q.dtype) + sg::type_size(y.dtype));
    out->flops = 3.0 * (double) T * (double) n * (double) (Hq + Hk);
    return SCRAPGPU_STATUS_OK;
}

scrapgpu_status attention_rule(const scrapgpu_op_desc * d, ServingOp * out, const Refusal & fail) {
    const auto * p = static_cast<const scrapgpu_attention_params *>(d->params);
    const bool paged = d->op == SCRAPGPU_OP_ATTENTION_PAGED;
    const Desc &q = d->inputs[0], &k = d->inputs[1], &v = d->inputs[2], &o = d->outputs[0];
    const Desc & qs = d->inputs[paged ? 4 : 3];
    const Desc & at = d->inputs[paged ? 5 : d->input_count == 5 ? 4 : 3];
    if (!half(q.dtype) || k.dtype != q.dtype || v.dtype != q.dtype) return fail.no("attention takes q, k and v of one type, F16 or BF16");
    if (o.dtype != q.dtype && o.dtype != SCRAPGPU_DTYPE_F32) return fail.no("attention writes the inputs' type or F32");
    const int64_t D = q.ne[0], Hq = sg::dim1(q.ne[1]), T = q.ne[2] == 0 ? 0 : sg::dim1(q.ne[2]);
    if (D <= 0 || q.ne[1] < 0 || q.ne[2] < 0 || !shape(q, D, Hq, T) || !shape(o, D, Hq, T)) return fail.bad("attention: q and the output must be [D, Hq, T] both");
    if (D % 8 != 0 || D > 256) return fail.no("attention: D must be a multiple of 8, at most 256");
    if (!strides(q, 16) || !strides(o, 16)) return fail.no("attention: strides and offsets must be multiples of 16 bytes, nb0 the element size");
    const int64_t Hk = paged ? sg::dim1(k.ne[2]) : sg::dim1(k.ne[1]);
    if (Hk <= 0 || Hq % Hk != 0) return fail.bad("attention: the query heads must be a whole multiple of the key heads");
    int64_t Tk = 0;
    int shift = 0;
    if (paged) {
        if (k.dtype == SCRAPGPU_DTYPE_F32) return fail.no("attention takes q, k and v of one type, F16 or BF16");
        const scrapgpu_status st = cache_rule(k, v, D, Hk, &shift, fail);
        if (st != SCRAPGPU_STATUS_OK) return st;
        if (shift < 4) return fail.no("ATTENTION_PAGED: pages must have 16 places or more (the kernels read 16 keys at a time)");
    } else {
        Tk = k.ne[2] == 0 ? 0 : sg::dim1(k.ne[2]);
        if (k.ne[1] < 0 || k.ne[2] < 0 || !shape(k, D, Hk, Tk) || !shape(v, D, Hk, Tk)) return fail.bad("ATTENTION_PROMPT: k and v must be [D, Hk, Tk] both");
        if (!strides(k, 16) || !strides(v, 16)) return fail.no("attention: strides and offsets must be multiples of 16 bytes, nb0 the element size");
        if (Tk > 1 && std::max(k.nb[2], v.nb[2]) >> 27) return fail.no("ATTENTION_PROMPT: tokens of k and v must lie less than 128 MiB apart");
        if (d->input_count == 4 && Tk != T) return fail.bad("ATTENTION_PROMPT: without k_start, k and v must have q's tokens");
    }
    const int64_t B = qs.ne[0] - 1;
    if (!ints(qs) || !ints(at)) return fail.no("attention: starts and lengths must be contiguous I32");
    if (B < 1 || !shape(qs, B + 1) || !shape(at, paged ? B : B + 1)) return fail.bad("attention: q_start must be [B+1], k_start [B+1], kv_len [B]");
    int64_t W = 0;
    if (paged) {
        const Desc & t = d->inputs[3];
        W = t.ne[0];
        if (!ints(t)) return fail.no("ATTENTION_PAGED: the table must be I32 with contiguous rows");
        if (W <= 0 || !shape(t, W, B)) return fail.bad("ATTENTION_PAGED: the table must be [W, B]");
        if (sg::sat_mul((uint64_t) W, (uint64_t) k.ne[1]) >= (1u << 30)) return fail.no("ATTENTION_PAGED: a request's tokens (W x page size) must be fewer than 2^30");
    }
    if (B > 65535 || T >= (1 << 24) || Tk >= (1 << 30) || sg::sat_mul((uint64_t) T, (uint64_t) (Hq / Hk)) >= (1u << 28) || Hk > 65535) return fail.no("attention: too many requests, tokens or heads");
    if (!std::isfinite(p->scale)) return fail.bad("attention: the scale must be finite");
    if (!injective(o)) return fail.bad("attention: elements of the output overlap");
    const scrapgpu_status st = all_apart(d, fail);
    if (st != SCRAPGPU_STATUS_OK) return st;
    sgk::AttnLaunch a;
    std::memset(&a, 0, sizeof(a));
    a.dtype = q.dtype;
    a.out_type = o.dtype;
    a.q_s1 = q.nb[1];
    a.q_s2 = q.nb[2];
    a.o_s1 = o.nb[1];
    a.o_s2 = o.nb[2];
    if (paged) {
        a.k_s1 = k.nb[1];
        a.k_s2 = k.nb[2];
        a.k_s3 = k.nb[3];
        a.v_s1 = v.nb[1];
        a.v_s2 = v.nb[2];
        a.v_s3 = v.nb[3];
        a.t_s1 = (int64_t) (d->inputs[3].nb[1] / 4);
        a.W = (int) W;
        a.shift = shift;
        a.n_pages = (int) sg::dim1(k.ne[3]);
    } else {
        a.k_s1 = k.nb[2];
        a.k_s2 = k.nb[1];
        a.v_s1 = v.nb[2];
        a.v_s2 = v.nb[1];
    }
    a.B = (int) B;
    a.T = (int) T;
    a.Tk = (int) Tk;
    a.Hq = (int) Hq;
    a.Hk = (int) Hk;
    a.G = (int) (Hq / Hk);
    a.D = (int) D;
    a.scale = p->scale;
    a.causal = p->causal != 0;
    a.paged = paged;
    a.max_query = (int) (p->max_query == 0 || p->max_query > (uint32_t) T ? T : p->max_query);
    // (a launch has fewer than 2^32 threads; the number of CUs changes the pieces alone, by a few hundred)
    if (sgk::attention_groups(a, sgk::attention_shape(a, 256, false)) >= (1 << 24) - 4096) return fail.no("attention: too many requests, tokens or heads");
    if (out == nullptr) return st;
    out->attn = a;
    out->empty = T == 0;
    put(out, q, "q", &out->attn.q);
    put(out, k, "k", &out->attn.k);
    put(out, v, "v", &out->attn.v);
    if (paged) put(out, d->inputs[3], "table", &out->attn.table);
    put(out, qs, "q_start", &out->attn.q_start);
    put(out, at, paged ? "kv_len" : "k_start", &out->attn.k_at);
    put(out, o, "y", &out->attn.o);
    out->bytes = (double) T * (double) (Hq * D) * (double) (2 + sg::type_size(o.dtype)) + 4.0 * (double) (paged ? 0 : Tk) * (double) (Hk * D);
    return SCRAPGPU_STATUS_OK;
}

} // namespace

bool is_serving_op(int op) {
    return op >= SCRAPGPU_OP_PAGED_PLAN && op <= SCRAPGPU_OP_ATTENTION_PAGED;
}

scrapgpu_status serving_rule(const scrapgpu_op_desc * desc, ServingOp * out, const char ** reason) {
    const Refusal fail{reason};
    if (out) {
        out->op = desc->op;
        out->empty = false;
        out->n_slots = 0;
        out->bytes = out->flops = 0;
    }
    // (validated before: arity, and params_size; the struct's own size guards its readers)
    size_t own = 0;
    std::memcpy(&own, desc->params, sizeof(own));
    switch (desc->op) {
        case SCRAPGPU_OP_PAGED_PLAN:
            if (own < sizeof(scrapgpu_paged_plan_params)) break;
            return plan_rule(desc, out, fail);
        case SCRAPGPU_OP_ROPE_AXES:
        case SCRAPGPU_OP_ROPE_AXES_STORE:
            if (own < sizeof(scrapgpu_rope_axes_params)) break;
            return rope_rule(desc, out, fail);
        default:
            if (own < sizeof(scrapgpu_attention_params)) break;
            return attention_rule(desc, out, fail);
    }
    return fail.bad("the params' struct_size is smaller than the struct");
}
