// The join of a decode's partials where sequences share prefixes: out = sum e^(m_i - M) o_i / sum e^(m_i - M) l_i over the parts of the
// prefix and of the sequence's own keys, in order.
//
// Bound by the memory, head_dim + 4 floats a row and part, and in small calls by two round trips: 6144 rows of 12 parts (Llama-3-8B heads,
// 39 MB) 9.5 us, 2048 of 18 (19 MB) 6.5, 112 of 6 (Qwen2.5-0.5B heads) 3.5 to 4, of which an empty launch is 2.
//
//   * A quad of dims to a thread, and kStripes threads to a quad, each with every kStripes-th part: many parts are in flight at once.
#include "mx_paged.hpp"

#include <algorithm>

namespace mx {

namespace {

constexpr int kStripes = 4, kAtOnce = 4, kJoinThreads = 256;

template <int HD, class T>
__global__ __launch_bounds__(kJoinThreads) void paged_join_kernel(PagedAttnParams p) {
    constexpr int QR = HD / 4, ROWS = kJoinThreads / (QR * kStripes);  // quads of a row, rows of a workgroup
    __shared__ float4_t s_o[kStripes][ROWS * QR];
    __shared__ float2 s_ml[kStripes][ROWS * QR];
    const int quad = threadIdx.x % QR, stripe = threadIdx.x / QR % kStripes, r = threadIdx.x / (QR * kStripes);
    const int64_t block = blockIdx.x + (int64_t)blockIdx.y * gridDim.x, total = (int64_t)p.n_rows * p.n_head;
    if (block * ROWS >= total) return;
    const int64_t row = min(block * ROWS + r, total - 1);
    const int token = (int)(row / p.n_head), h = (int)(row - (int64_t)token * p.n_head);
    const int b = token / p.n_q, t = token - b * p.n_q, g = h / p.group, rr = t * p.group + h - g * p.group;
    const int4 info = p.x.info[b];
    const int own = p.x.own_len[b], np = info.z, parts = own < 0 ? 0 : np + own_chunks(p, own);
    const float * pre = p.x.part + ((int64_t)g * *p.x.rows + info.x + info.w + rr) * (HD + 4);
    const float * mine = p.x.own_part + (((int64_t)b * p.fixed * p.n_head_kv + g) * p.rows + rr) * (HD + 4);
    const int64_t pre_step = (int64_t)info.y * (HD + 4), own_step = (int64_t)p.n_head_kv * p.rows * (HD + 4);
    float M = kNegInf, l = 0.f;
    float4_t o = {0.f, 0.f, 0.f, 0.f};
    for (int k0 = stripe; k0 < parts; k0 += kStripes * kAtOnce) {
        float4_t w[kAtOnce];
        float2 ml[kAtOnce];
        float top = M;
#pragma unroll
        for (int e = 0; e < kAtOnce; e++) {
            const int k = min(k0 + e * kStripes, parts - 1);
            const float * x = k < np ? pre + k * pre_step : mine + (k - np) * own_step;
            w[e] = *reinterpret_cast<const float4_t *>(x + 4 * quad);
            ml[e] = *reinterpret_cast<const float2 *>(x + HD);
        }
#pragma unroll
        for (int e = 0; e < kAtOnce; e++) top = fmaxf(top, ml[e].x);
        const float use = top == kNegInf ? 0.f : top, corr = exp2_fast(M - use);
        o *= corr;
        l *= corr;
#pragma unroll
        for (int e = 0; e < kAtOnce; e++) {
            if (k0 + e * kStripes >= parts) break;
            const float y = exp2_fast(ml[e].x - use);
            o += w[e] * y;
            l += ml[e].y * y;
        }
        M = top;
    }
    s_o[stripe][r * QR + quad] = o;
    s_ml[stripe][r * QR + quad] = make_float2(M, l);
    __syncthreads();
    if (stripe != 0 || block * ROWS + r >= total) return;
    float2 ml[kStripes];
    float top = kNegInf;
#pragma unroll
    for (int s = 0; s < kStripes; s++) {
        ml[s] = s_ml[s][r * QR + quad];
        top = fmaxf(top, ml[s].x);
    }
    const float use = top == kNegInf ? 0.f : top;
    o = float4_t{0.f, 0.f, 0.f, 0.f};
    l = 0.f;
#pragma unroll
    for (int s = 0; s < kStripes; s++) {
        const float y = exp2_fast(ml[s].x - use);
        if (s > 0 && s >= parts) break;  // no part
        o += s_o[s][r * QR + quad] * y;
        l += ml[s].y * y;
    }
    const bool bad = own < 0, empty = np == 0 && (p.causal ? own - p.n_q + t < 0 : own == 0);  // no key: zeros
    const float nan = __builtin_nanf(""), inv = 1.f / l;
    o = bad ? float4_t{nan, nan, nan, nan} : empty ? float4_t{0.f, 0.f, 0.f, 0.f} : o * inv;
    const int64_t at = (int64_t)token * p.out_stride + (int64_t)h * HD + 4 * quad;
    if (p.out32) *reinterpret_cast<float4_t *>(static_cast<float *>(p.out) + at) = o;
    else *reinterpret_cast<u32x2 *>(static_cast<uint16_t *>(p.out) + at) = u32x2{T::pack2(o[0], o[1]), T::pack2(o[2], o[3])};
    if (quad == 0 && p.lse) p.lse[row] = bad ? nan : empty ? kNegInf : (top + log2_fast(l)) * kLn2;
}

template <class T>
void launch(const PagedAttnParams & p, int head_dim, hipStream_t stream) {
    constexpr int64_t kMost = 1 << 23;  // workgroups along x: a dimension holds fewer than 2^32 threads
    const int rows = kJoinThreads / (head_dim / 4 * kStripes);
    const int64_t blocks = ((int64_t)p.n_rows * p.n_head + rows - 1) / rows;
    const dim3 grid((uint32_t)std::min(blocks, kMost), (uint32_t)((blocks + kMost - 1) / kMost)), block(kJoinThreads);
    if (head_dim == 64) hipLaunchKernelGGL((paged_join_kernel<64, T>), grid, block, 0, stream, p);
    else if (head_dim == 128) hipLaunchKernelGGL((paged_join_kernel<128, T>), grid, block, 0, stream, p);
    else hipLaunchKernelGGL((paged_join_kernel<256, T>), grid, block, 0, stream, p);
}

}  // namespace

hipError_t launch_paged_join(const PagedAttnParams & p, int head_dim, int dtype, hipStream_t stream) {
    if (dtype == 1) launch<F16>(p, head_dim, stream);
    else launch<BF16>(p, head_dim, stream);
    return hipGetLastError();
}

}  // namespace mx
