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
};

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
};

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
hipError_t launch_paged_prefill(const PagedAttnParams & p, int head_dim, int dtype, const PagedPrefillPlan & plan, hipStream_t stream);

}  // namespace mx
