// The paged cache's append: rotary embedding of new tokens' queries and keys, keys and values into their pages.
//
// For pair i of a head row at positions pos[axis]: theta = pos[axis of i] f(i), (a, b) -> (a cos - b sin, a sin + b cos), with the
// pairs (2i, 2i + 1) or (i, i + head_dim / 2); the arithmetic of rope_store (src/backend/metal/llama_kernels.h:513-545 in
// dooms.cpp 0.6.1), the angle in 64 bits instead of 32.
//
// Byte work: each q|k|v element is read once and written once at half the width or the same. One workgroup per token row; a
// thread holds two pieces of 16 bytes, half a head apart, so that both rotary layouts find their partners in one thread and
// every load and store of a wave is contiguous. The sequence is looked up first, then the row's loads go out, behind them
// the page, and the head_dim / 2 angles, turned into (cos, sin) once for all heads of the row. 179 MB of
// packed prompts take 31.6 us (5.7 TB/s, a large copy reaches 5.2); a decode step's row 2.8 us, of which an empty launch is 2.
//
// Pages in 8 bits: the lanes of a head's row find its largest magnitude together, and from its exponent the scale, a power of two, so
// that dividing by it is exact. Keys are rotated in 64 bits and rounded to odd, and so to codes as the definition has them; the angles'
// cosines cost the wave that computes them 0.2 us a row, under the row's loads (4867 rows, Llama-3-8B heads, 170 MB in 33 us, 5.1 TB/s; a
// decode step's row 3.2).
#pragma once

#include "mx_paged.hpp"

#include <algorithm>

namespace mx {

namespace {

// sin and cos of a 64-bit angle: reduced by pi / 2 in 64 bits (pi / 2 split in two, so that |x| up to 2^31 keeps the
// remainder to f32), then the Taylor series on |r| <= pi / 4 in f32 (truncation below 2e-9).
__device__ __forceinline__ float2 cos_sin(double x) {
    constexpr double kTwoOverPi = 0.63661977236758134308, kPio2Hi = 1.5707963267948966, kPio2Lo = 6.123233995736766e-17;
    const double k = __builtin_rint(x * kTwoOverPi);
    const float r = (float)__builtin_fma(-k, kPio2Lo, __builtin_fma(-k, kPio2Hi, x));
    const float r2 = r * r;
    float s = -1.f / 39916800.f;
    s = __builtin_fmaf(s, r2, 1.f / 362880.f);
    s = __builtin_fmaf(s, r2, -1.f / 5040.f);
    s = __builtin_fmaf(s, r2, 1.f / 120.f);
    s = __builtin_fmaf(s, r2, -1.f / 6.f);
    s = __builtin_fmaf(s * r2, r, r);
    float c = 1.f / 479001600.f;
    c = __builtin_fmaf(c, r2, -1.f / 3628800.f);
    c = __builtin_fmaf(c, r2, 1.f / 40320.f);
    c = __builtin_fmaf(c, r2, -1.f / 720.f);
    c = __builtin_fmaf(c, r2, 1.f / 24.f);
    c = __builtin_fmaf(c, r2, -0.5f);
    c = __builtin_fmaf(c, r2, 1.f);
    const int q = (int)((long long)k & 3);
    return q == 0 ? make_float2(c, s) : q == 1 ? make_float2(-s, c) : q == 2 ? make_float2(-c, -s) : make_float2(s, -c);
}

// cos and sin of an angle in 64 bits, reduced as above; the Taylor series on |r| <= pi / 4 to degree 17 (truncation below 2^-58).
__device__ __forceinline__ double2 cos_sin64(double x) {
    constexpr double kTwoOverPi = 0.63661977236758134308, kPio2Hi = 1.5707963267948966, kPio2Lo = 6.123233995736766e-17;
    const double k = __builtin_rint(x * kTwoOverPi);
    const double r = __builtin_fma(-k, kPio2Lo, __builtin_fma(-k, kPio2Hi, x)), r2 = r * r;
    double s = 1. / 355687428096000.;
    s = __builtin_fma(s, r2, -1. / 1307674368000.);
    s = __builtin_fma(s, r2, 1. / 6227020800.);
    s = __builtin_fma(s, r2, -1. / 39916800.);
    s = __builtin_fma(s, r2, 1. / 362880.);
    s = __builtin_fma(s, r2, -1. / 5040.);
    s = __builtin_fma(s, r2, 1. / 120.);
    s = __builtin_fma(s, r2, -1. / 6.);
    s = __builtin_fma(s * r2, r, r);
    double c = 1. / 20922789888000.;
    c = __builtin_fma(c, r2, -1. / 87178291200.);
    c = __builtin_fma(c, r2, 1. / 479001600.);
    c = __builtin_fma(c, r2, -1. / 3628800.);
    c = __builtin_fma(c, r2, 1. / 40320.);
    c = __builtin_fma(c, r2, -1. / 720.);
    c = __builtin_fma(c, r2, 1. / 24.);
    c = __builtin_fma(c, r2, -0.5);
    c = __builtin_fma(c, r2, 1.);
    const int q = (int)((long long)k & 3);
    return q == 0 ? make_double2(c, s) : q == 1 ? make_double2(-s, c) : q == 2 ? make_double2(-c, -s) : make_double2(s, -c);
}

// v in 32 bits, rounded to odd: towards zero, with the last bit set where that was not exact, so that rounding the result to fewer bits
// gives what rounding v once does. An infinity or NaN, and what 32 bits do not hold, stay no finite number.
__device__ __forceinline__ float round_odd(double v) {
    const float f = (float)v;
    const double back = (double)f;
    if (back == v || !__builtin_isfinite(f)) return f;
    const uint32_t b = __float_as_uint(f);
    return __uint_as_float((__builtin_fabs(back) > __builtin_fabs(v) ? b - 1 : b) | 1u);
}

// The maximum over N lanes in a row (a power of two up to 32, aligned), in each; lanes outside may be off.
template <int N>
__device__ __forceinline__ float lanes_max(float v) {
    auto with = [&](auto C) {
        constexpr int c = decltype(C)::value;
        v = fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), c, 0xF, 0xF, true)));
    };
    with(std::integral_constant<int, 0xB1>{});  // quad_perm: lanes 1 apart, 2 apart
    with(std::integral_constant<int, 0x4E>{});
    if constexpr (N >= 8) with(std::integral_constant<int, 0x141>{});   // mirrored in 8
    if constexpr (N >= 16) with(std::integral_constant<int, 0x140>{});  // mirrored in 16
    if constexpr (N >= 32) v = fmaxf(v, shfl_xor(v, 16));
    return v;
}

// The scale byte of a row whose largest magnitude is top: of 2^e, e the least with top <= 448 2^e = 1.75 2^(e + 8).
__device__ __forceinline__ uint32_t scale_byte(float top) { return (uint32_t)max((int)((__float_as_uint(top) + 0x1fffffu) >> 23) - 8, 0); }

// Two numbers over the power of two 1 / inv as e4m3, rounded to nearest even; an infinity or NaN becomes NaN.
__device__ __forceinline__ uint32_t codes2(float a, float b, float inv, uint32_t w, bool hi) {
    const float nan = __builtin_nanf("");
    const float x = __builtin_isfinite(a) ? a * inv : nan, y = __builtin_isfinite(b) ? b * inv : nan;
    return hi ? __builtin_amdgcn_cvt_pk_fp8_f32(x, y, w, true) : __builtin_amdgcn_cvt_pk_fp8_f32(x, y, w, false);
}

// IN: 0 f32, 1 f16, 2 bf16 rows (MX_ATTN_F32, ...). T: the type of the queries, and of the pages. Q8: the pages hold e4m3 codes
// with a scale a row.
template <int HD, int IN, class T, bool Q8>
__global__ __launch_bounds__(512) void paged_store_kernel(PagedStoreParams p) {
    constexpr int E = IN == 0 ? 4 : 8;        // elements of a 16-byte piece
    constexpr int UH = HD / (2 * E);          // units (two pieces) of a head
    constexpr int HALF = HD / 2;
    constexpr int AHEAD = 2;                  // units a thread loads at once
    __shared__ float2 s_cs[HALF];
    __shared__ double2 s_cd[Q8 ? HALF : 1];  // Q8: for the keys, whose codes are those of the rotation in 64 bits

    const int64_t block = blockIdx.x + (int64_t)blockIdx.y * gridDim.x;
    if (block >= p.n_rows) return;
    const int row = (int)block, lane = threadIdx.x % kWave;
    const int units = (p.n_head + 2 * p.n_head_kv) * UH;
    const char * src = static_cast<const char *>(p.qkv) + (int64_t)row * p.row_stride * (IN == 0 ? 4 : 2);
    auto load = [&](int u, u32x4 (&w)[2]) __attribute__((always_inline)) {
        const int x = min(u, units - 1);
        const char * at = src + (int64_t)((x / UH) * HD + (x % UH) * E) * (IN == 0 ? 4 : 2);
        w[0] = load16(at);
        w[1] = load16(at + HALF * (IN == 0 ? 4 : 2));
    };
    // the candidates for the row's sequence, one a lane: sent for ahead of the row itself, so that the wait for them leaves it in
    // flight; 64 probes a step narrow many sequences to 64 (the offsets ascend)
    int first = 0, left = p.c.n_seq, lo = 0, hi = 0, ln = 0;
    if (p.cu_q) {
        while (left > kWave) {
            const int step = (left + kWave - 1) / kWave;
            const uint64_t below = __builtin_amdgcn_ballot_w64(lane * step < left && p.cu_q[min(first + lane * step, p.c.n_seq)] <= row);
            const int skip = max(__builtin_popcountll(below) - 1, 0) * step;
            first += skip;
            left = min(step, left - skip);
        }
        const int i = min(first + lane, p.c.n_seq - 1);
        lo = p.cu_q[i];
        hi = p.cu_q[i + 1];
        ln = p.c.kv_len[i];
    }
    u32x4 w[AHEAD][2];
#pragma unroll
    for (int a = 0; a < AHEAD; a++) load(threadIdx.x + a * blockDim.x, w[a]);

    // the row's sequence, its new rows and the row among them; a row behind the last sequence is left alone
    int b = -1, n = p.n_q, t = 0, len = 0;
    if (p.cu_q) {
        lo = min(max(lo, 0), p.n_rows);
        hi = min(max(hi, 0), p.n_rows);
        const uint64_t in = __builtin_amdgcn_ballot_w64(lane < left && lo <= row && row < hi);
        if (in) {
            const int l = __builtin_ctzll(in);
            b = first + l;
            t = row - __builtin_amdgcn_readlane(lo, l);
            n = __builtin_amdgcn_readlane(hi, l) - __builtin_amdgcn_readlane(lo, l);
            len = __builtin_amdgcn_readlane(ln, l);
        }
        if (b < 0) return;
    } else {
        b = row / n;
        t = row - b * n;
        len = p.c.kv_len[b];
    }
    const int64_t pos64 = (int64_t)len - n + t;
    const int pos = (int)max(pos64, (int64_t)INT32_MIN);
    bool keep = length_ok(p.c, len) && pos >= 0;
    int page = 0;
    if (keep) {
        page = p.c.table[b * p.c.table_stride + (pos >> p.c.page_shift)];
        keep = page_ok(p.c, page);
    }
    if (p.rope_mode != 2) {
        if (threadIdx.x < HALF) {
            const int i = threadIdx.x;
            int at = pos;
            if (p.positions) {
                int axis = 0;
#pragma unroll
                for (int a = 0; a + 1 < kPagedMaxAxes; a++) axis += a + 1 < p.n_axes && i >= p.axis_end[a];
                at = p.positions[(int64_t)axis * p.n_rows + row];
            }
            if constexpr (Q8) {
                s_cd[i] = cos_sin64((double)at * p.freq[i]);
                s_cs[i] = make_float2((float)s_cd[i].x, (float)s_cd[i].y);
            } else {
                s_cs[i] = cos_sin((double)at * p.freq[i]);
            }
        }
        __syncthreads();
    }
    const int64_t slot = (int64_t)page * p.c.page_stride + (int64_t)(pos & ((1 << p.c.page_shift) - 1)) * p.c.kv_stride;

    for (int u0 = threadIdx.x; u0 < units; u0 += AHEAD * blockDim.x) {
#pragma unroll
        for (int a = 0; a < AHEAD; a++) {
            const int u = u0 + a * blockDim.x;
            if (u >= units) break;
            const int head = u / UH, e0 = (u % UH) * E;
            float x[2][E];
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int e = 0; e < E; e += 2) {
                    if constexpr (IN == 0) {
                        x[h][e] = __uint_as_float(w[a][h][e]);
                        x[h][e + 1] = __uint_as_float(w[a][h][e + 1]);
                    } else {
                        const float2 v = IN == 1 ? F16::unpack2(w[a][h][e / 2]) : BF16::unpack2(w[a][h][e / 2]);
                        x[h][e] = v.x;
                        x[h][e + 1] = v.y;
                    }
                }
            auto turn = [&](float & c, float & d, int i) __attribute__((always_inline)) {
                const float2 z = s_cs[i];
                const float r = c * z.x - d * z.y;
                d = c * z.y + d * z.x;
                c = r;
            };
            auto turn64 = [&](float & c, float & d, int i) __attribute__((always_inline)) {
                const double2 z = s_cd[Q8 ? i : 0];
                const double a = c, b = d;
                c = round_odd(a * z.x - b * z.y);
                d = round_odd(a * z.y + b * z.x);
            };
            auto rotate = [&](auto && by) __attribute__((always_inline)) {
                if (p.rope_mode == 1) {
#pragma unroll
                    for (int e = 0; e < E; e++) by(x[0][e], x[1][e], e0 + e);
                } else if (p.rope_mode == 0) {
#pragma unroll
                    for (int h = 0; h < 2; h++)
#pragma unroll
                        for (int e = 0; e < E; e += 2) by(x[h][e], x[h][e + 1], (HALF * h + e0 + e) / 2);
                }
            };
            if (head < (Q8 ? p.n_head : p.n_head + p.n_head_kv)) rotate(turn);
            else if (Q8 && head < p.n_head + p.n_head_kv) rotate(turn64);
            if constexpr (Q8) {
                if (head >= p.n_head) {
                    // the UH lanes of the head's row find its scale together
                    float top = 0.f;
#pragma unroll
                    for (int h = 0; h < 2; h++)
#pragma unroll
                        for (int e = 0; e < E; e++) top = fmaxf(top, __builtin_isfinite(x[h][e]) ? fabsf(x[h][e]) : 0.f);
                    const uint32_t byte = scale_byte(lanes_max<UH>(top));
                    if (!keep) continue;
                    const float inv = __uint_as_float((254u - byte) << 23);
                    const int g = head - p.n_head, gk = g % p.n_head_kv;
                    uint8_t * at = reinterpret_cast<uint8_t *>(const_cast<uint16_t *>(g < p.n_head_kv ? p.c.k : p.c.v)) + slot +
                                   (int64_t)gk * p.c.head_stride + e0;
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        uint32_t o[E / 4];
#pragma unroll
                        for (int e = 0; e < E; e += 4)
                            o[e / 4] = codes2(x[h][e + 2], x[h][e + 3], inv, codes2(x[h][e], x[h][e + 1], inv, 0u, false), true);
                        if constexpr (E == 4) *reinterpret_cast<uint32_t *>(at + HALF * h) = o[0];
                        else *reinterpret_cast<u32x2 *>(at + HALF * h) = u32x2{o[0], o[1]};
                    }
                    if (e0 == 0)
                        (g < p.n_head_kv ? p.s.k : p.s.v)[(int64_t)page * p.s.page_stride + (int64_t)gk * p.s.head_stride +
                                                          (pos & ((1 << p.c.page_shift) - 1))] = (uint8_t)byte;
                    continue;
                }
            }
            uint16_t * dst;
            if (head < p.n_head) {
                if (!p.q_out) continue;
                dst = p.q_out + (int64_t)row * p.out_stride + (int64_t)head * HD;
            } else {
                if (!keep) continue;
                const int g = head - p.n_head;
                dst = const_cast<uint16_t *>(g < p.n_head_kv ? p.c.k : p.c.v) + slot + (int64_t)(g % p.n_head_kv) * p.c.head_stride;
            }
#pragma unroll
            for (int h = 0; h < 2; h++) {
                uint32_t o[E / 2];
#pragma unroll
                for (int e = 0; e < E; e += 2) o[e / 2] = T::pack2(x[h][e], x[h][e + 1]);
                if constexpr (E == 4) *reinterpret_cast<u32x2 *>(dst + HALF * h + e0) = u32x2{o[0], o[1]};
                else *reinterpret_cast<u32x4 *>(dst + HALF * h + e0) = u32x4{o[0], o[1], o[2], o[3]};
            }
        }
        if (u0 + AHEAD * (int)blockDim.x < units) {
#pragma unroll
            for (int a = 0; a < AHEAD; a++) load(u0 + (AHEAD + a) * blockDim.x, w[a]);
        }
    }
}

template <int HD, class T, bool Q8>
void launch_in(const PagedStoreParams & p, int in_dtype, hipStream_t stream) {
    const int units = (p.n_head + 2 * p.n_head_kv) * HD / (in_dtype == 0 ? 8 : 16);
    const int threads = std::max(HD / 2, std::min(512, (units + kWave - 1) / kWave * kWave));
    constexpr int kMost = 1 << 22;  // workgroups along x: a dimension holds fewer than 2^32 threads
    const dim3 grid((uint32_t)std::min(p.n_rows, kMost), (uint32_t)(((int64_t)p.n_rows + kMost - 1) / kMost)), block((uint32_t)threads);
    if (in_dtype == 0) hipLaunchKernelGGL((paged_store_kernel<HD, 0, T, Q8>), grid, block, 0, stream, p);
    else if (in_dtype == 1) hipLaunchKernelGGL((paged_store_kernel<HD, 1, T, Q8>), grid, block, 0, stream, p);
    else hipLaunchKernelGGL((paged_store_kernel<HD, 2, T, Q8>), grid, block, 0, stream, p);
}

template <class T, bool Q8>
hipError_t launch_hd(const PagedStoreParams & p, int head_dim, int in_dtype, hipStream_t stream) {
    if (head_dim == 64) launch_in<64, T, Q8>(p, in_dtype, stream);
    else if (head_dim == 128) launch_in<128, T, Q8>(p, in_dtype, stream);
    else launch_in<256, T, Q8>(p, in_dtype, stream);
    return hipGetLastError();
}

}  // namespace

}  // namespace mx
