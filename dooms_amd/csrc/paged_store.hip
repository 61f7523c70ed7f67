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

// IN: 0 f32, 1 f16, 2 bf16 rows (MX_ATTN_F32, ...). T: the pages' type.
template <int HD, int IN, class T>
__global__ __launch_bounds__(512) void paged_store_kernel(PagedStoreParams p) {
    constexpr int E = IN == 0 ? 4 : 8;        // elements of a 16-byte piece
    constexpr int UH = HD / (2 * E);          // units (two pieces) of a head
    constexpr int HALF = HD / 2;
    constexpr int AHEAD = 2;                  // units a thread loads at once
    __shared__ float2 s_cs[HALF];

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
            s_cs[i] = cos_sin((double)at * p.freq[i]);
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
            if (head < p.n_head + p.n_head_kv) {
                if (p.rope_mode == 1) {
#pragma unroll
                    for (int e = 0; e < E; e++) turn(x[0][e], x[1][e], e0 + e);
                } else if (p.rope_mode == 0) {
#pragma unroll
                    for (int h = 0; h < 2; h++)
#pragma unroll
                        for (int e = 0; e < E; e += 2) turn(x[h][e], x[h][e + 1], (HALF * h + e0 + e) / 2);
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

template <int HD, class T>
void launch_in(const PagedStoreParams & p, int in_dtype, hipStream_t stream) {
    const int units = (p.n_head + 2 * p.n_head_kv) * HD / (in_dtype == 0 ? 8 : 16);
    const int threads = std::max(HD / 2, std::min(512, (units + kWave - 1) / kWave * kWave));
    constexpr int kMost = 1 << 22;  // workgroups along x: a dimension holds fewer than 2^32 threads
    const dim3 grid((uint32_t)std::min(p.n_rows, kMost), (uint32_t)(((int64_t)p.n_rows + kMost - 1) / kMost)), block((uint32_t)threads);
    if (in_dtype == 0) hipLaunchKernelGGL((paged_store_kernel<HD, 0, T>), grid, block, 0, stream, p);
    else if (in_dtype == 1) hipLaunchKernelGGL((paged_store_kernel<HD, 1, T>), grid, block, 0, stream, p);
    else hipLaunchKernelGGL((paged_store_kernel<HD, 2, T>), grid, block, 0, stream, p);
}

template <class T>
hipError_t launch_hd(const PagedStoreParams & p, int head_dim, int in_dtype, hipStream_t stream) {
    if (head_dim == 64) launch_in<64, T>(p, in_dtype, stream);
    else if (head_dim == 128) launch_in<128, T>(p, in_dtype, stream);
    else launch_in<256, T>(p, in_dtype, stream);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_paged_store(const PagedStoreParams & p, int head_dim, int in_dtype, int dtype, hipStream_t stream) {
    return dtype == 1 ? launch_hd<F16>(p, head_dim, in_dtype, stream) : launch_hd<BF16>(p, head_dim, in_dtype, stream);
}

}  // namespace mx
