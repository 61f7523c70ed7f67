// The paged cache's kernels: parameter blocks, launchers and what they share (element types, page lookups, int wave sums).
#pragma once

#include "mx_common.hpp"
#include "mx_kernels.hpp"

namespace mx {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));

// The pages' element types: matrix products on 8-element operands held as 16 bytes, and roundings to nearest even.
struct F16 {
    static __device__ __forceinline__ float4_t mfma16(u32x4 a, u32x4 b, float4_t c) { return mfma16x16x32(as_half8(a), as_half8(b), c); }
    static __device__ __forceinline__ float16_t mfma32(u32x4 a, u32x4 b, float16_t c) { return mfma32x32x16(as_half8(a), as_half8(b), c); }
    static __device__ __forceinline__ uint32_t pack2(float a, float b) { return __builtin_bit_cast(uint32_t, f16x2_t{(half_t)a, (half_t)b}); }
    // c + the sum of a pair
    static __device__ __forceinline__ float add2(uint32_t p, float c) {
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2_t, p), f16x2_t{(half_t)1.f, (half_t)1.f}, c, false);
    }
    static __device__ __forceinline__ float2 unpack2(uint32_t p) {
        const f16x2_t h = __builtin_bit_cast(f16x2_t, p);
        return make_float2((float)h[0], (float)h[1]);
    }
    // two e4m3 codes (the lower or upper half of w) times the power of two `scale`; NaN codes and scales give NaN
    template <bool HI>
    static __device__ __forceinline__ uint32_t expand2(uint32_t w, float scale) {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, HI));
    }
    static constexpr uint32_t kExp = 0x7c00u;  // all exponent bits: infinities and NaN
};
struct BF16 {
    static __device__ __forceinline__ float4_t mfma16(u32x4 a, u32x4 b, float4_t c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ float16_t mfma32(u32x4 a, u32x4 b, float16_t c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pack2(float a, float b) { return __builtin_bit_cast(uint32_t, bf16x2_t{(__bf16)a, (__bf16)b}); }
    static __device__ __forceinline__ float add2(uint32_t p, float c) {
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, p), bf16x2_t{(__bf16)1.f, (__bf16)1.f}, c, false);
    }
    static __device__ __forceinline__ float2 unpack2(uint32_t p) {
        return make_float2(__uint_as_float(p << 16), __uint_as_float(p & 0xffff0000u));
    }
    template <bool HI>
    static __device__ __forceinline__ uint32_t expand2(uint32_t w, float scale) {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, HI));
    }
    static constexpr uint32_t kExp = 0x7f80u;
};

// Whether one of 8 elements is an infinity or NaN.
template <class T>
__device__ __forceinline__ bool any_nonfinite(u32x4 w) {
    bool r = false;
#pragma unroll
    for (int e = 0; e < 4; e++)
        r |= (w[e] & T::kExp) == T::kExp || ((w[e] >> 16) & T::kExp) == T::kExp;
    return r;
}

// 8 codes of a row as T: exact where T holds the products (bf16 always, but for its smallest), else rounded to nearest even.
template <class T>
__device__ __forceinline__ u32x4 expand8(uint32_t lo, uint32_t hi, float scale) {
    return u32x4{T::template expand2<false>(lo, scale), T::template expand2<true>(lo, scale), T::template expand2<false>(hi, scale),
                 T::template expand2<true>(hi, scale)};
}
// Scale bytes of N rows in a row (N-byte aligned), and byte i of them as the float that the expansion takes: its exponent bits (255: NaN).
template <int N>
__device__ __forceinline__ uint32_t load_scales(const uint8_t * p) {
    if constexpr (N == 1) return *(const __attribute__((address_space(1))) uint8_t *)(p);
    else if constexpr (N == 2) return *(const __attribute__((address_space(1))) uint16_t *)(p);
    else return *(const __attribute__((address_space(1))) uint32_t *)(p);
}
__device__ __forceinline__ float scale_of(uint32_t bytes, int i) { return __uint_as_float((bytes >> (8 * i) & 0xffu) << 23); }

// Pages of e4m3 codes: a byte a row and kv head, the scale 2^(byte - 127), rows in a row.
struct PagedScales {
    uint8_t * k;
    uint8_t * v;
    int64_t page_stride, head_stride;
};

// Where the pages lie. `table` and `kv_len` are device memory that the host has not seen.
struct PagedCache {
    const uint16_t * k;
    const uint16_t * v;
    const int32_t * table;
    const int32_t * kv_len;
    int64_t page_stride, kv_stride, head_stride, table_stride;
    int32_t n_seq, n_pages, page_shift;
    int32_t capacity;  // keys that a row of the table can place: max_pages << page_shift (at most INT32_MAX)
};

// A sequence's length, 0 where what the table can place does not hold it (its outputs are then NaN).
__device__ __forceinline__ bool length_ok(const PagedCache & c, int32_t len) { return len >= 0 && len <= c.capacity; }
__device__ __forceinline__ bool page_ok(const PagedCache & c, int32_t id) { return (uint32_t)id < (uint32_t)c.n_pages; }

// Sum and inclusive prefix sum over the 64 lanes of a wave (every lane active).
__device__ __forceinline__ int32_t wave_isum(int32_t v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x140, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x141, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xF, 0xF, false);
    const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = (int32_t)(a[0] + a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return __builtin_amdgcn_readfirstlane((int32_t)(b[0] + b[1]));
}
__device__ __forceinline__ int32_t wave_imax(int32_t v) {
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x140, 0xF, 0xF, false));
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x141, 0xF, 0xF, false));
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xF, 0xF, false));
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xF, 0xF, false));
    const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = max((int32_t)a[0], (int32_t)a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return __builtin_amdgcn_readfirstlane(max((int32_t)b[0], (int32_t)b[1]));
}
__device__ __forceinline__ int32_t wave_iscan(int32_t v) {
    // within rows of 16: row_shr 1, 2, 4, 8 (lanes shifted in are 0), then the totals of the rows below
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true);
    const int32_t r0 = __builtin_amdgcn_readlane(v, 15), r1 = __builtin_amdgcn_readlane(v, 31), r2 = __builtin_amdgcn_readlane(v, 47);
    const int row = (int)__lane_id() / 16;
    return v + (row > 0 ? r0 : 0) + (row > 1 ? r1 : 0) + (row > 2 ? r2 : 0);
}

constexpr int kPagedMaxAxes = 4;

struct PagedStoreParams {
    PagedCache c;  // k and v are written here
    const void * qkv;
    const int32_t * positions;  // [n_axes][n_rows] or null
    const int32_t * cu_q;       // or null: n_q rows a sequence
    uint16_t * q_out;           // or null
    int64_t row_stride, out_stride;
    int32_t n_head, n_head_kv, n_rows, n_q, rope_mode, n_axes;
    int32_t axis_end[kPagedMaxAxes];  // first pair behind each axis
    double freq[kMaxHeadDim / 2];
    PagedScales s;  // pages of codes
};

// Sequences that share their first keys: groups of them, and where their partials go: head_dim + 4 floats a row, o, m and l.
struct PagedPrefix {
    const int32_t * cu_seq;      // [n_groups + 1]: sequences cu_seq[g] .. cu_seq[g + 1] - 1 are group g's
    const int32_t * prefix_len;  // [n_groups]
    int32_t n_groups;
    int32_t room;                // workgroups that the prefixes are cut for
    int32_t least;               // steps of 64 keys that each of them takes at least
    uint32_t blocks, own_blocks; // workgroups of the prefixes, and behind them those of the sequences' own keys; multiples of 8
    int32_t own_chunk;           // own keys of a workgroup; PagedAttnParams::fixed of them a sequence (the last takes what is left)
    int64_t max_rows;            // rows that `part` has room for
    float * part;                // of the prefixes: [kv head][group][part][row]
    float * own_part;            // [sequence][chunk][kv head][row]
    // what the prefixes' workgroups leave for the join:
    int32_t * rows;              // rows of a kv head among the prefixes' partials
    int32_t * own_len;           // [n_seq]: OwnKeys::len
    int4 * info;                 // [n_seq]: the group's first row among a kv head's, its rows, its parts, the sequence's row among them
};
struct PagedPrefixPart {  // of a workgroup
    int64_t first;  // first row
    int32_t rows;
};
constexpr int kPagedPrefixWaves = 4;  // of both kinds of workgroups

struct PagedAttnParams {
    PagedCache c;
    const uint16_t * q;
    void * out;
    float * lse;
    const int32_t * cu_q;  // prefill
    float * part;          // partial slots
    uint32_t * counters;
    int64_t q_stride, out_stride;
    int32_t n_head, n_head_kv, group, n_rows, n_q, causal, out32;
    int32_t by_ranges;     // decode: 1: workgroups walk ranges of the launch's keys, 0: a chunk of a sequence each
    int32_t ranges;        // decode: ranges, or chunks, that the launch has workgroups for, for each (kv head, row tile); prefill:
                           // workgroups, a multiple of 8
    int32_t whole_keys;    // decode, chunks: nothing is split where no sequence of the launch is longer (fixed: no such sequence is)
    int32_t fixed;         // decode, chunks: of every sequence, each a quantum (the last takes what is left); 0: the chunks follow
                           // from the lengths
    int32_t whole;         // 1: no sequence (prefill: no tile) is split, there is no workspace
    int32_t max_pages;     // entries of a row of the page table
    int32_t max_tiles;     // prefill: tiles of query rows that there can be
    int32_t rows, n_rowtiles;  // decode: query rows that share a kv head, and their tiles
    float scale_log2;      // |scale| log2 e, or 1 with a scale of 0
    uint32_t q_xor, q_and; // scale < 0 turns the sign of the query rows, scale 0 makes them zero
    PagedScales s;         // pages of codes
    PagedPrefix x;         // shared prefixes
};

// The keys of a sequence behind the `start` that it shares: `len` of them, counted from the multiple of 16 at or below start; len -1: a
// length, or prefix, that is none.
struct OwnKeys {
    int32_t start, len;
};
// Whether the prefixes' workgroups compute the `keys` that the n sequences of a group share: of several always, of one alone where they are
// more than a chunk of own keys. As its own keys, which the hint does not count, its last chunk would walk them (Llama-3-8B heads, a hint
// of 120: one sequence alone behind 16384 keys 201 us, 23 so; beside 63 that share 4096 keys 227 and 36). Tiles of few rows cost more where
// nothing is shared at all (32 sequences alone behind 4096 keys each 122 us, 92 as own keys, which is a plain decode's time).
__device__ __forceinline__ bool prefix_apart(const PagedAttnParams & p, int n, int keys) {
    return keys > 0 && (n > 1 || (n == 1 && keys > p.x.own_chunk));
}
// Of a sequence of `len` keys in a group of sequences s0 .. s1 - 1 that share `keys` (in: or in none). Every row has to see all of them.
__device__ __forceinline__ OwnKeys own_of(const PagedAttnParams & p, bool in, int s0, int s1, int keys, int len) {
    const bool wrong = in && (keys < 0 || keys > p.c.capacity);
    if (len == 0 || !length_ok(p.c, len) || wrong) return OwnKeys{0, len == 0 ? 0 : -1};
    if (!in || keys == 0) return OwnKeys{0, len};
    if (len < keys + (p.causal ? p.n_q - 1 : 0)) return OwnKeys{0, -1};
    return prefix_apart(p, s1 - s0, keys) ? OwnKeys{keys, len > keys ? len - (keys & ~15) : 0} : OwnKeys{0, len};
}
// Of sequence b, the same in every lane: 64 probes a step narrow the groups, whose bounds ascend, to 64.
__device__ __forceinline__ OwnKeys own_keys(const PagedAttnParams & p, int b) {
    const PagedPrefix & x = p.x;
    const int lane = (int)__lane_id(), len = p.c.kv_len[b];
    int first = 0, left = x.n_groups;
    while (left > kWave) {
        const int step = (left + kWave - 1) / kWave;
        const uint64_t below = __builtin_amdgcn_ballot_w64(lane * step < left && x.cu_seq[min(first + lane * step, x.n_groups)] <= b);
        const int skip = max(__builtin_popcountll(below) - 1, 0) * step;
        first += skip;
        left = min(step, left - skip);
    }
    const int i = min(first + lane, x.n_groups - 1), lo = x.cu_seq[i], hi = x.cu_seq[i + 1], keys = x.prefix_len[i];
    const uint64_t from = __builtin_amdgcn_ballot_w64(lane < left && lo <= b);
    const int l = from ? 63 - __builtin_clzll(from) : 0;
    auto clamp = [&](int s) { return min(max(s, 0), p.c.n_seq); };
    const int s0 = clamp(__builtin_amdgcn_readlane(lo, l)), s1 = clamp(__builtin_amdgcn_readlane(hi, l));
    const OwnKeys r = own_of(p, from != 0 && b < s1, s0, s1, __builtin_amdgcn_readlane(keys, l), len);
    return OwnKeys{__builtin_amdgcn_readfirstlane(r.start), __builtin_amdgcn_readfirstlane(r.len)};
}
// Chunks of them.
__device__ __forceinline__ int own_chunks(const PagedAttnParams & p, int len) {
    return len <= 0 ? 0 : min(p.fixed, (int)((uint32_t)(len + p.x.own_chunk - 1) / (uint32_t)p.x.own_chunk));
}

// Parts of a sequence in a decode at most: the join takes one lane each (131072 keys, Qwen2.5-7B heads, 54 us; with 33 67).
constexpr int kPagedMaxParts = 64;

constexpr int kPagedDecodeBlock = 32;  // keys that a wave of the decode kernel takes at a time

// A prefill workgroup: waves of 32 query rows, `heads` of a group among them. Head dim 256 runs 4 waves of one head.
struct PagedPrefillPlan {
    int32_t waves, heads;
    int rows() const { return 32 * waves / heads; }
    int resident(int head_dim) const { return waves == 8 || head_dim == 256 ? 256 : 512; }  // workgroups that run at once
    // floats of a range's two partials: per lane its outputs, m and l
    int64_t part_floats(int head_dim) const { return 2 * (int64_t)waves * (head_dim / 2 + 2) * kWave; }
};

hipError_t launch_paged_store(const PagedStoreParams & p, int head_dim, int in_dtype, int dtype, hipStream_t stream);
hipError_t launch_paged_decode(const PagedAttnParams & p, int head_dim, int dtype, int rt, int waves, hipStream_t stream);
// the same over pages of codes: the store's dtype is that of its queries
hipError_t launch_paged_store_e4m3(const PagedStoreParams & p, int head_dim, int in_dtype, int dtype, hipStream_t stream);
hipError_t launch_paged_decode_e4m3(const PagedAttnParams & p, int head_dim, int dtype, int rt, int waves, hipStream_t stream);
hipError_t launch_paged_prefill_e4m3(const PagedAttnParams & p, int head_dim, int dtype, const PagedPrefillPlan & plan, hipStream_t stream);
hipError_t launch_paged_prefill(const PagedAttnParams & p, int head_dim, int dtype, const PagedPrefillPlan & plan, hipStream_t stream);

hipError_t launch_paged_shared(const PagedAttnParams & p, int head_dim, int dtype, int rt, hipStream_t stream);
hipError_t launch_paged_shared_e4m3(const PagedAttnParams & p, int head_dim, int dtype, int rt, hipStream_t stream);
hipError_t launch_paged_join(const PagedAttnParams & p, int head_dim, int dtype, hipStream_t stream);

}  // namespace mx
