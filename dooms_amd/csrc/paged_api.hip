// C ABI of the paged cache (include/mx_paged.h): argument checks, launch plans. As in api.hip, every check of host arguments
// runs before anything is enqueued, and nothing here aborts or throws.
#include "mx_paged.h"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>

#include "mx_host.hpp"
#include "mx_paged.hpp"

namespace {

int32_t fail(int32_t code, const char * fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    std::vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    return mx::set_error(code, buf);
}

bool aligned(const void * p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// What every call and the workspace sizes need.
int32_t check_shape(const mx_paged_desc * d) {
    if (!d) return fail(MX_ATTN_INVALID_ARGUMENT, "desc is null");
    if (d->reserved != 0) return fail(MX_ATTN_INVALID_ARGUMENT, "desc->reserved must be 0");
    if (d->n_head < 1 || d->n_head_kv < 1)
        return fail(MX_ATTN_INVALID_ARGUMENT, "n_head (%d) and n_head_kv (%d) must be >= 1", d->n_head, d->n_head_kv);
    if (d->n_head % d->n_head_kv != 0)
        return fail(MX_ATTN_INVALID_ARGUMENT, "n_head (%d) is not a multiple of n_head_kv (%d)", d->n_head, d->n_head_kv);
    if (d->n_head > 65535) return fail(MX_ATTN_UNSUPPORTED, "n_head (%d) beyond 65535", d->n_head);
    if (d->head_dim != 64 && d->head_dim != 128 && d->head_dim != 256)
        return fail(MX_ATTN_UNSUPPORTED, "head_dim %d is not supported with pages (64, 128 or 256)", d->head_dim);
    if (d->dtype != MX_ATTN_F16 && d->dtype != MX_ATTN_BF16)
        return fail(MX_ATTN_INVALID_ARGUMENT, "dtype (%d) must be MX_ATTN_F16 or MX_ATTN_BF16", d->dtype);
    if (d->n_seq < 0 || d->n_seq > 65535) return fail(MX_ATTN_INVALID_ARGUMENT, "n_seq (%d) must be in [0, 65535]", d->n_seq);
    if (d->n_rows < 0 || d->n_rows > 1 << 30) return fail(MX_ATTN_INVALID_ARGUMENT, "n_rows (%d) must be in [0, 2^30]", d->n_rows);
    if (d->max_q < 0 || d->max_kv_len < 0)
        return fail(MX_ATTN_INVALID_ARGUMENT, "max_q (%d) and max_kv_len (%d) must be >= 0", d->max_q, d->max_kv_len);
    return MX_ATTN_OK;
}

int32_t check_uniform(const mx_paged_desc & d) {
    if (d.n_seq > 0 && d.n_rows % d.n_seq)
        return fail(MX_ATTN_INVALID_ARGUMENT, "n_rows (%d) is not a multiple of n_seq (%d)", d.n_rows, d.n_seq);
    if (d.n_seq == 0 && d.n_rows > 0) return fail(MX_ATTN_INVALID_ARGUMENT, "%d rows of no sequence", d.n_rows);
    return MX_ATTN_OK;
}

// The pool, its strides and the table.
int32_t check_cache(const mx_paged_desc & d) {
    if (d.page_size < 16 || d.page_size > 65536 || (d.page_size & (d.page_size - 1)))
        return fail(MX_ATTN_UNSUPPORTED, "page_size (%d) must be a power of two in [16, 65536]", d.page_size);
    if (d.n_pages < 1 || d.max_pages < 1)
        return fail(MX_ATTN_INVALID_ARGUMENT, "n_pages (%d) and max_pages (%d) must be >= 1", d.n_pages, d.max_pages);
    if ((int64_t)d.max_pages * d.page_size > (int64_t)1 << 30)
        return fail(MX_ATTN_UNSUPPORTED, "max_pages (%d) x page_size (%d) beyond 2^30 keys a sequence", d.max_pages, d.page_size);
    if (d.table_stride < d.max_pages)
        return fail(MX_ATTN_INVALID_ARGUMENT, "table_stride (%lld) < max_pages (%d)", (long long)d.table_stride, d.max_pages);
    if (d.kv_stride > (int64_t)1 << 26)
        return fail(MX_ATTN_UNSUPPORTED, "kv_stride (%lld) beyond 2^26 elements", (long long)d.kv_stride);
    // (page, row, head) rows of head_dim elements apart from each other: by ascending stride, each stride covers what the
    // smaller ones span
    struct Dim {
        int64_t stride, n;
        const char * name;
    } dim[3] = {{d.page_stride, d.n_pages, "page_stride"}, {d.kv_stride, d.page_size, "kv_stride"}, {d.head_stride, d.n_head_kv, "head_stride"}};
    for (const Dim & x : dim)
        if (x.n > 1 && (x.stride < 0 || x.stride % 8 || x.stride > (int64_t)1 << 46))
            return fail(MX_ATTN_INVALID_ARGUMENT, "%s (%lld) must be a multiple of 8 elements, >= 0", x.name, (long long)x.stride);
    std::sort(dim, dim + 3, [](const Dim & a, const Dim & b) { return a.stride < b.stride; });
    int64_t span = d.head_dim;
    for (const Dim & x : dim) {
        if (x.n == 1) continue;
        if (x.stride < span)
            return fail(MX_ATTN_INVALID_ARGUMENT, "%s (%lld) makes rows of the pool overlap (%lld elements lie below it)", x.name,
                        (long long)x.stride, (long long)span);
        if (x.stride > ((int64_t)1 << 62) / x.n) return fail(MX_ATTN_INVALID_ARGUMENT, "%s (%lld) is out of range", x.name, (long long)x.stride);
        span += x.stride * (x.n - 1);
    }
    return MX_ATTN_OK;
}

mx::PagedCache cache_of(const mx_paged_desc & d, const void * k, const void * v, const int32_t * table, const int32_t * kv_len) {
    mx::PagedCache c{};
    c.k = static_cast<const uint16_t *>(k);
    c.v = static_cast<const uint16_t *>(v);
    c.table = table;
    c.kv_len = kv_len;
    c.page_stride = d.page_stride;
    c.kv_stride = d.kv_stride;
    c.head_stride = d.head_stride;
    c.table_stride = d.table_stride;
    c.n_seq = d.n_seq;
    c.n_pages = d.n_pages;
    c.page_shift = __builtin_ctz((unsigned)d.page_size);
    c.capacity = d.max_pages << c.page_shift;
    return c;
}

int32_t check_pointers(const void * k, const void * v, const int32_t * table, const int32_t * kv_len, const int32_t * cu_q) {
    if (!k || !v || !table || !kv_len) return fail(MX_ATTN_INVALID_ARGUMENT, "k, v, table and kv_len must not be null");
    if (!aligned(k, 16) || !aligned(v, 16)) return fail(MX_ATTN_INVALID_ARGUMENT, "k and v must be 16-byte aligned");
    if (!aligned(table, 4) || !aligned(kv_len, 4) || !aligned(cu_q, 4))
        return fail(MX_ATTN_INVALID_ARGUMENT, "table, kv_len and cu_q must be 4-byte aligned");
    return MX_ATTN_OK;
}

int32_t check_rows(const char * name, int64_t stride, int64_t width, int unit) {
    if (stride < width || stride % unit || stride > (int64_t)1 << 31)
        return fail(MX_ATTN_INVALID_ARGUMENT, "%s (%lld) must be >= %lld, a multiple of %d and at most 2^31", name, (long long)stride,
                    (long long)width, unit);
    return MX_ATTN_OK;
}

// Checks of an attention call, and its parameters but for the plan.
int32_t attn_params(const mx_paged_desc & d, const void * q, const void * k, const void * v, const int32_t * table,
                    const int32_t * kv_len, const int32_t * cu_q, void * out, float * lse, mx::PagedAttnParams & p) {
    if (d.row_dtype != d.dtype && d.row_dtype != MX_ATTN_F32)
        return fail(MX_ATTN_INVALID_ARGUMENT, "row_dtype (%d) must be MX_ATTN_F32 or dtype (%d)", d.row_dtype, d.dtype);
    if (d.causal != 0 && d.causal != 1) return fail(MX_ATTN_INVALID_ARGUMENT, "causal must be 0 or 1");
    if (!std::isfinite(d.scale)) return fail(MX_ATTN_INVALID_ARGUMENT, "scale is not finite");
    if (int32_t rc = check_cache(d)) return rc;
    const int64_t wide = (int64_t)d.n_head * d.head_dim;
    const bool out32 = d.row_dtype == MX_ATTN_F32;
    if (int32_t rc = check_rows("row_stride", d.row_stride, wide, 8)) return rc;
    if (int32_t rc = check_rows("out_stride", d.out_stride, wide, out32 ? 4 : 8)) return rc;
    if (d.n_seq == 0 || d.n_rows == 0) return MX_ATTN_OK;
    if (!q || !out) return fail(MX_ATTN_INVALID_ARGUMENT, "q and out must not be null");
    if (!aligned(q, 16) || !aligned(out, 16)) return fail(MX_ATTN_INVALID_ARGUMENT, "q and out must be 16-byte aligned");
    if (!aligned(lse, 4)) return fail(MX_ATTN_INVALID_ARGUMENT, "lse must be 4-byte aligned");
    if (int32_t rc = check_pointers(k, v, table, kv_len, cu_q)) return rc;
    p.c = cache_of(d, k, v, table, kv_len);
    p.q = static_cast<const uint16_t *>(q);
    p.out = out;
    p.lse = lse;
    p.cu_q = cu_q;
    p.q_stride = d.row_stride;
    p.out_stride = d.out_stride;
    p.n_head = d.n_head;
    p.n_head_kv = d.n_head_kv;
    p.group = d.n_head / d.n_head_kv;
    p.n_rows = d.n_rows;
    p.causal = d.causal;
    p.out32 = out32;
    // the kernels' exponentials take a positive factor: a negative scale turns the query's sign, 0 makes the query zero
    p.scale_log2 = d.scale == 0.f ? 1.f : std::fabs(d.scale) * 1.4426950408889634f;
    p.q_and = d.scale == 0.f ? 0u : 0xffffffffu;
    p.q_xor = d.scale < 0.f ? 0x80008000u : 0u;
    return MX_ATTN_OK;
}

// ---- decode ----

constexpr int kCUs = 256;

struct DecodePlan {
    int32_t rows, rt, n_rowtiles, waves, by_ranges, ranges, whole_keys, fixed, whole;
    size_t bytes;  // workspace
};

// Keys per sequence that the plan reckons with: the hint's, or the table's, or what a launch holds where a workspace is
// sized without either.
int64_t kv_bound(const mx_paged_desc & d) {
    int64_t table = (int64_t)d.max_pages * d.page_size;
    if (table <= 0) table = std::min<int64_t>((int64_t)1 << 30, ((int64_t)1 << 36) / std::max(1, d.n_seq));
    return d.max_kv_len > 0 && d.max_kv_len < table ? d.max_kv_len : table;
}

int32_t decode_plan(const mx_paged_desc & d, DecodePlan & plan) {
    const int n_q = d.n_rows / d.n_seq;
    if ((int64_t)n_q * (d.n_head / d.n_head_kv) > 65536)
        return fail(MX_ATTN_UNSUPPORTED, "%d rows a sequence are a prompt (mx_paged_prefill)", n_q);
    plan.rows = n_q * (d.n_head / d.n_head_kv);
    // A tile of 32 rows reads the keys once where two of 16 would twice (nine sequences of 201-5999 keys, 28 rows, 24 us against 31);
    // at head dim 256 its registers do not fit.
    plan.rt = plan.rows > 16 && d.head_dim != 256 ? 32 : mx::decode_rows_per_tile(plan.rows);
    plan.n_rowtiles = (plan.rows + plan.rt - 1) / plan.rt;
    const int64_t per_seq = (int64_t)d.n_head_kv * plan.n_rowtiles, bound = kv_bound(d);
    auto quanta = [&](int waves) { return (bound + mx::kPagedDecodeBlock * waves - 1) / (mx::kPagedDecodeBlock * waves); };
    if (per_seq > mx::kCounterLines)
        return fail(MX_ATTN_UNSUPPORTED, "%lld (kv head, row tile) pairs of a sequence are more than one launch holds", (long long)per_seq);
    const int64_t pairs = d.n_seq * per_seq;
    // the kernel counts the quanta of all sequences in 32 bits
    if (d.n_seq * ((std::max<int64_t>(bound, (int64_t)d.max_pages * d.page_size) + 127) / 128) > (int64_t)1 << 30)
        return fail(MX_ATTN_UNSUPPORTED, "%d sequences of up to %lld keys are more than one launch holds", d.n_seq,
                    (long long)std::max<int64_t>(bound, (int64_t)d.max_pages * d.page_size));
    plan.whole = bound <= 128;
    // Ranges where the launch may hold many quanta of 128 keys for every workgroup (64 sequences of 111-8191 keys, Llama-3-8B heads,
    // 182 us against 227 of chunks), chunks below, where finding the range and joining over it cost more than its balance saves
    // (64 of 100-2000, Qwen2.5-0.5B heads, 13.8 of chunks against 17.1; equal at 32 of 111-2000, Llama-3-8B heads, 33.7). Tiles of
    // more rows join slower, so their bound is higher (32 rows, 32 sequences of 201-5999, 52 against 67).
    plan.by_ranges = d.n_seq > 1 && pairs * quanta(4) > (plan.rt <= 8 ? 16 : plan.rt == 16 ? 32 : 64) * kCUs;
    plan.fixed = 0;
    plan.whole_keys = 0;
    if (plan.by_ranges) {
        plan.waves = 4;
        plan.ranges = (int32_t)std::max<int64_t>(1, (plan.rt <= 8 ? 2 : 1) * kCUs / per_seq);
    } else {
        // Where no sequence is longer than whole_keys each is one chunk: joining costs 1 to 2 us more than the walk saves (513 keys,
        // Qwen2.5-0.5B heads, 6.3 us against 7.4 split; 512 keys, Llama-3-8B heads, 8.2 against 8.6; 1000 keys 13.1 whole against
        // 8.5). Beyond it 4 waves a workgroup, two on a CU, find the keys of a middling length on more CUs (1000 keys, Llama-3-8B
        // heads, 7.35 against 8.5 with 8 waves; 2000, Qwen2.5-0.5B heads, 7.2 against 7.6), and split shorter sequences too (8 of
        // 100-1000 keys 9.5 against 10.4 with 512). Longer ones have fewer parts to join with 8 (4000 keys, Qwen2.5-7B heads, 9.8
        // against 10.6; 8192, Llama-3-8B heads, 11.3 against 14.8), and so have tiles of more rows. At head dim 256 the LDS holds 4
        // waves.
        plan.whole_keys = d.head_dim == 64 ? 640 : 512;
        plan.waves = d.head_dim == 256 || bound <= 128 || (plan.rt <= 8 && bound > plan.whole_keys && bound <= 2048) ? 4 : 8;
        if (plan.waves == 4) plan.whole_keys = 256;
        plan.ranges = (int32_t)std::max<int64_t>(d.n_seq, (plan.waves == 8 ? 1 : 2) * kCUs / per_seq);
        // Where one round of workgroups has room for every quantum of every sequence the chunks need no planning from the lengths:
        // one round trip less (8192 keys, Llama-3-8B heads, 11.3 us against 12.0). Beyond a round the empty ones cost more
        // (16 sequences of 100-4000 keys, Qwen2.5-0.5B heads, 13.2 against 10.7 planned).
        const int64_t n = quanta(plan.waves);
        if (bound <= plan.whole_keys || (n <= 32 && pairs * n <= (plan.waves == 8 ? 1 : 2) * kCUs)) {
            plan.fixed = bound <= plan.whole_keys ? 1 : (int32_t)n;
            plan.ranges = d.n_seq * plan.fixed;
        }
    }
    if (plan.ranges * per_seq * plan.waves > (int64_t)1 << 25)  // threads of a grid's dimension: below 2^32
        return fail(MX_ATTN_UNSUPPORTED, "%d sequences of %lld (kv head, row tile) pairs are more than one launch holds", d.n_seq, (long long)per_seq);
    // Two partials a range and tile, or two chunks beyond one a sequence; sized for the most of any batch and length, so that one
    // workspace serves all calls of a head shape and row count.
    plan.bytes = plan.whole ? 0 : mx::kCounterBytes + (size_t)(2 * std::max<int64_t>(1, 2 * kCUs / per_seq) * per_seq * plan.rt * (d.head_dim + 4)) * sizeof(float);
    return MX_ATTN_OK;
}

// ---- prefill ----

int64_t prefill_tiles(const mx_paged_desc & d, int rows) { return std::min<int64_t>(d.n_rows, d.n_rows / rows + d.n_seq); }

// What the plan reckons with; the grid has room for more, as max_q may not hold.
int64_t likely_tiles(const mx_paged_desc & d, int rows) {
    const int64_t n = prefill_tiles(d, rows);
    return d.max_q > 0 ? std::min(n, d.n_seq * (((int64_t)d.max_q + rows - 1) / rows)) : n;
}

mx::PagedPrefillPlan prefill_plan(const mx_paged_desc & d) {
    mx::PagedPrefillPlan r{4, 1};
    if (d.head_dim != 128) return r;
    // Head dim 64 runs 4 waves throughout: its steps are short, and two workgroups of a CU cover each other's (24 prompts of
    // 500-1200 rows, Qwen2.5-0.5B heads, 82 us against 86-92 with 8; one of 4096 62.3 against 61.4). Head dim 128 runs them where
    // all tiles are short and run at once (4 prompts of 50-300 rows, Llama-3-8B heads, 12.4 us against 14.1-15.8), else 8 waves,
    // which share each step (two 1000-2000-row chunks behind 4000 keys, Qwen2.5-7B heads, 222 against 236).
    if (likely_tiles(d, 128) * d.n_head <= 2 * kCUs && kv_bound(d) <= 1536) return r;
    r.waves = 8;
    // Tiles of several heads: fewer rows idle at the ends of sequences and on the diagonal (12 prompts of 65-1711 rows, Llama-3-8B
    // heads, 173 us of one head, 163 of two, 156 of four). Where the heads do not divide the group the shorter prompts still gain
    // (24 of 500-1200 rows, 7 heads a kv head, 240, 217 and 215; of 4096 rows 142, 148 and 150).
    const int group = d.n_head / d.n_head_kv;
    const int64_t rows = d.n_rows / d.n_seq;
    auto fits = [&](int heads, int64_t few) {
        const int padded = (group + heads - 1) / heads * heads;
        return padded == group || (rows < few && 8 * (padded - group) <= padded);
    };
    r.heads = fits(4, 512) ? 4 : fits(2, 1024) ? 2 : 1;
    return r;
}

// The counters, and two partials of a tile for each of the workgroups that run at once: as many floats with 8 waves as with 4,
// of which twice as many workgroups run, so that one workspace serves every plan of a head dim.
size_t prefill_bytes(int head_dim) {
    const mx::PagedPrefillPlan r{4, 1};
    return mx::kCounterBytes + (size_t)(r.resident(head_dim) * r.part_floats(head_dim)) * sizeof(float);
}

}  // namespace

extern "C" {

MX_ATTN_API int32_t mx_paged_store(const mx_paged_desc * desc, const mx_paged_rope * rope, const void * qkv,
                                   const int32_t * positions, void * k, void * v, const int32_t * table,
                                   const int32_t * kv_len, const int32_t * cu_q, void * q_out, mx_attn_stream stream) {
    if (int32_t rc = check_shape(desc)) return rc;
    const mx_paged_desc & d = *desc;
    if (d.row_dtype != MX_ATTN_F32 && d.row_dtype != MX_ATTN_F16 && d.row_dtype != MX_ATTN_BF16)
        return fail(MX_ATTN_INVALID_ARGUMENT, "row_dtype (%d) must be MX_ATTN_F32, MX_ATTN_F16 or MX_ATTN_BF16", d.row_dtype);
    if (!rope) return fail(MX_ATTN_INVALID_ARGUMENT, "rope is null");
    if (rope->reserved != 0) return fail(MX_ATTN_INVALID_ARGUMENT, "rope->reserved must be 0");
    if (rope->mode < 0 || rope->mode > 2) return fail(MX_ATTN_INVALID_ARGUMENT, "rope->mode (%d) must be 0, 1 or 2", rope->mode);
    mx::PagedStoreParams p{};
    p.rope_mode = rope->mode;
    p.n_axes = 1;
    if (rope->mode != 2) {
        if (rope->n_axes < 1 || rope->n_axes > MX_PAGED_MAX_AXES)
            return fail(MX_ATTN_INVALID_ARGUMENT, "rope->n_axes (%d) must be in [1, %d]", rope->n_axes, MX_PAGED_MAX_AXES);
        if (rope->axis_restart != 0 && rope->axis_restart != 1) return fail(MX_ATTN_INVALID_ARGUMENT, "rope->axis_restart must be 0 or 1");
        // below 1 the angles would grow past what the kernel reduces
        if (!(std::isfinite(rope->base) && rope->base >= 1.)) return fail(MX_ATTN_INVALID_ARGUMENT, "rope->base must be finite and >= 1");
        p.n_axes = rope->n_axes;
        int64_t at = 0;
        for (int a = 0; a < MX_PAGED_MAX_AXES; a++) {
            const int64_t n = a < rope->n_axes ? rope->axis_pairs[a] : 0;
            if (a < rope->n_axes && n < 1) return fail(MX_ATTN_INVALID_ARGUMENT, "rope->axis_pairs[%d] (%lld) must be >= 1", a, (long long)n);
            if (at + n > d.head_dim / 2) return fail(MX_ATTN_INVALID_ARGUMENT, "the axes have more than head_dim / 2 (%d) pairs", d.head_dim / 2);
            // a ladder of equal ratios, from a power of its own every 8 rungs: 7 products are within 7 2^-53 of the powers
            const double below = rope->axis_restart ? (double)n : (double)d.head_dim / 2.;
            const double ratio = std::pow(rope->base, -1. / below);
            for (int64_t j = 0; j < n; j++) {
                const int64_t i = rope->axis_restart ? j : at + j;
                p.freq[at + j] = j % 8 ? p.freq[at + j - 1] * ratio : std::pow(rope->base, -(double)i / below);
            }
            at += n;
            p.axis_end[a] = (int32_t)at;
        }
        if (at != d.head_dim / 2) return fail(MX_ATTN_INVALID_ARGUMENT, "the axes have %lld pairs, not head_dim / 2 (%d)", (long long)at, d.head_dim / 2);
        if (!positions && rope->n_axes > 1) return fail(MX_ATTN_INVALID_ARGUMENT, "positions must be given for more than one axis");
        if (!aligned(positions, 4)) return fail(MX_ATTN_INVALID_ARGUMENT, "positions must be 4-byte aligned");
    }
    if (int32_t rc = check_cache(d)) return rc;
    const int64_t wide = (int64_t)d.n_head * d.head_dim, all = wide + 2 * (int64_t)d.n_head_kv * d.head_dim;
    if (int32_t rc = check_rows("row_stride", d.row_stride, all, d.row_dtype == MX_ATTN_F32 ? 4 : 8)) return rc;
    if (q_out)
        if (int32_t rc = check_rows("out_stride", d.out_stride, wide, 8)) return rc;
    if (!cu_q)
        if (int32_t rc = check_uniform(d)) return rc;
    if (d.n_seq == 0 || d.n_rows == 0) return MX_ATTN_OK;
    if (!qkv || !aligned(qkv, 16)) return fail(MX_ATTN_INVALID_ARGUMENT, "qkv must be a 16-byte aligned pointer");
    if (!aligned(q_out, 16)) return fail(MX_ATTN_INVALID_ARGUMENT, "q_out must be 16-byte aligned");
    if (int32_t rc = check_pointers(k, v, table, kv_len, cu_q)) return rc;
    p.c = cache_of(d, k, v, table, kv_len);
    p.qkv = qkv;
    p.positions = rope->mode == 2 ? nullptr : positions;
    p.cu_q = cu_q;
    p.q_out = static_cast<uint16_t *>(q_out);
    p.row_stride = d.row_stride;
    p.out_stride = d.out_stride;
    p.n_head = d.n_head;
    p.n_head_kv = d.n_head_kv;
    p.n_rows = d.n_rows;
    p.n_q = d.n_rows / d.n_seq;
    const hipError_t e = mx::launch_paged_store(p, d.head_dim, d.row_dtype, d.dtype, static_cast<hipStream_t>(stream));
    if (e != hipSuccess) return fail(MX_ATTN_INTERNAL, "paged store launch: %s", hipGetErrorString(e));
    return MX_ATTN_OK;
}

MX_ATTN_API size_t mx_paged_decode_workspace_bytes(const mx_paged_desc * desc) {
    if (check_shape(desc) || check_uniform(*desc) || desc->n_seq == 0 || desc->n_rows == 0) return 0;
    DecodePlan plan;
    return decode_plan(*desc, plan) ? 0 : plan.bytes;
}

MX_ATTN_API int32_t mx_paged_decode(const mx_paged_desc * desc, const void * q, const void * k, const void * v,
                                    const int32_t * table, const int32_t * kv_len, void * out, float * lse, void * workspace,
                                    size_t ws_bytes, mx_attn_stream stream) {
    if (int32_t rc = check_shape(desc)) return rc;
    const mx_paged_desc & d = *desc;
    if (int32_t rc = check_uniform(d)) return rc;
    mx::PagedAttnParams p{};
    if (int32_t rc = attn_params(d, q, k, v, table, kv_len, nullptr, out, lse, p)) return rc;
    if (d.n_seq == 0 || d.n_rows == 0) return MX_ATTN_OK;
    DecodePlan plan;
    if (int32_t rc = decode_plan(d, plan)) return rc;
    if (plan.bytes && (!workspace || !aligned(workspace, 256)))
        return fail(MX_ATTN_INVALID_ARGUMENT, "a 256-byte aligned workspace of %zu bytes is needed", plan.bytes);
    if (ws_bytes < plan.bytes)
        return fail(MX_ATTN_RESOURCE_EXHAUSTED, "workspace of %zu bytes is smaller than the %zu bytes needed", ws_bytes, plan.bytes);
    p.n_q = d.n_rows / d.n_seq;
    p.rows = plan.rows;
    p.n_rowtiles = plan.n_rowtiles;
    p.by_ranges = plan.by_ranges;
    p.whole_keys = plan.whole_keys;
    p.ranges = plan.ranges;
    p.fixed = plan.fixed;
    p.whole = plan.whole;
    p.max_pages = d.max_pages;
    p.counters = static_cast<uint32_t *>(workspace);
    p.part = reinterpret_cast<float *>(static_cast<char *>(workspace) + mx::kCounterBytes);
    const hipError_t e = mx::launch_paged_decode(p, d.head_dim, d.dtype, plan.rt, plan.waves, static_cast<hipStream_t>(stream));
    if (e != hipSuccess) return fail(MX_ATTN_INTERNAL, "paged decode launch: %s", hipGetErrorString(e));
    return MX_ATTN_OK;
}

MX_ATTN_API size_t mx_paged_prefill_workspace_bytes(const mx_paged_desc * desc) {
    if (check_shape(desc) || desc->n_seq == 0 || desc->n_rows == 0) return 0;
    return prefill_bytes(desc->head_dim);
}

MX_ATTN_API int32_t mx_paged_prefill(const mx_paged_desc * desc, const void * q, const void * k, const void * v,
                                     const int32_t * table, const int32_t * kv_len, const int32_t * cu_q, void * out, float * lse,
                                     void * workspace, size_t ws_bytes, mx_attn_stream stream) {
    if (int32_t rc = check_shape(desc)) return rc;
    const mx_paged_desc & d = *desc;
    mx::PagedAttnParams p{};
    if (int32_t rc = attn_params(d, q, k, v, table, kv_len, cu_q, out, lse, p)) return rc;
    if (d.n_seq == 0 || d.n_rows == 0) return MX_ATTN_OK;
    if (!cu_q) return fail(MX_ATTN_INVALID_ARGUMENT, "cu_q must not be null");
    const mx::PagedPrefillPlan plan = prefill_plan(d);
    const int64_t tiles = prefill_tiles(d, plan.rows());
    // tiles are counted in 32 bits, their steps in 64 (and 55 for 64 sequences), whatever cu_q holds
    const double steps = (double)(d.n_rows / plan.rows() + 1) * ((double)d.max_pages * d.page_size / 64. + 4.);
    if (tiles * d.n_head > INT32_MAX / 8 || steps > 0x1p49 || steps * d.n_seq * d.n_head > 0x1p61)
        return fail(MX_ATTN_UNSUPPORTED, "%d rows of %d heads are more than one launch holds", d.n_rows, d.n_head);
    p.max_tiles = (int32_t)tiles;
    p.ranges = plan.resident(d.head_dim);
    p.whole = !workspace;
    if (workspace && !aligned(workspace, 256)) return fail(MX_ATTN_INVALID_ARGUMENT, "the workspace must be 256-byte aligned");
    if (workspace && ws_bytes < prefill_bytes(d.head_dim))
        return fail(MX_ATTN_RESOURCE_EXHAUSTED, "workspace of %zu bytes is smaller than the %zu bytes needed", ws_bytes, prefill_bytes(d.head_dim));
    p.counters = static_cast<uint32_t *>(workspace);
    p.part = reinterpret_cast<float *>(static_cast<char *>(workspace) + mx::kCounterBytes);
    const hipError_t e = mx::launch_paged_prefill(p, d.head_dim, d.dtype, plan, static_cast<hipStream_t>(stream));
    if (e != hipSuccess) return fail(MX_ATTN_INTERNAL, "paged prefill launch: %s", hipGetErrorString(e));
    return MX_ATTN_OK;
}

#ifdef MX_ATTN_TRACE
// The diagnostic variant of the library tells how a call would run, so that tests know which kernels they reach. plan[0 .. 2]: rows
// of a tile, waves, and for a decode how it is cut (0 chunks from the lengths, 1 a fixed count of each sequence, 2 ranges), for
// prompts heads of a tile.
__attribute__((visibility("default"))) int32_t mx_paged_trace_plan(const mx_paged_desc * d, int32_t prefill, int32_t * plan) {
    if (int32_t rc = check_shape(d)) return rc;
    if (prefill) {
        const mx::PagedPrefillPlan r = prefill_plan(*d);
        plan[0] = r.rows();
        plan[1] = r.waves;
        plan[2] = r.heads;
        return MX_ATTN_OK;
    }
    DecodePlan r;
    if (int32_t rc = decode_plan(*d, r)) return rc;
    plan[0] = r.rt;
    plan[1] = r.waves;
    plan[2] = r.by_ranges ? 2 : r.fixed ? 1 : 0;
    return MX_ATTN_OK;
}
#endif

}  // extern "C"
