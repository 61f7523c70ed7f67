// Decode attention of sequences that share prefixes: one launch that computes the partials of all keys, each shared one once for all rows
// of its group, and one that joins them.
//
// For row r of a sequence with keys split into parts i (of the prefix, and of its own): m_i = max s, l_i = sum e^(s - m_i), o_i = sum
// e^(s - m_i) v over the part's keys; M = max m_i, out = sum e^(m_i - M) o_i / sum e^(m_i - M) l_i.
//
// The first launch has two kinds of workgroups, dealt to the chip in turn: those of the prefixes are the packed prompts' kernel over all
// query rows of a group (bound by the matrix cores and the exponentials), those of the sequences' own keys the decode kernel in chunks
// (bound by the memory). Those of the prefixes come first, one for a CU; beside it, and behind it, the CU walks own keys (192 sequences
// of 100-1500 own keys behind 16384, Llama-3-8B heads, f16: 62 GFLOP and 0.70 GB in 160 to 171 us from card to card; the prefixes alone
// 75, the own keys alone 118, each key of each sequence on its own 1323. 64 sequences of 40-900 behind 4096: 40 to 42, 112 unshared. Two
// launches one behind the other took 214 and 51, the two kinds in turn 207 and 52).
// Small calls are a chain of round trips: the groups' bounds, the pages' numbers, the keys, then the join (eight answers to 700 shared
// keys, Qwen2.5-0.5B heads, 10.9 us, of which the join 3.5; a decode that shares nothing takes 7.0 there, as all of it is in the caches).
// Every workgroup plans from all groups, 64 a step: 64 groups of two behind 64 keys (8 heads of 64 over 2) 9.2 us, 256 23, 1000 116, 4200
// 1330, where mx_paged_decode takes 4.3, 9.2, 30 and 137 over the same keys.
#pragma once

#include "paged_decode_kernel.hpp"
#include "paged_prefill_kernel.hpp"

namespace mx {

namespace {

template <int HD, int RT, class T, bool Q8>
__global__ __launch_bounds__(kPagedPrefixWaves * kWave) __attribute__((amdgpu_waves_per_eu(HD == 256 ? 1 : 2)))
void paged_shared_kernel(PagedAttnParams p) {
    constexpr int W = kPagedPrefixWaves;
    using Own = DecodeSmem<HD, RT, W>;
    using Prefix = Smem<HD, W, Q8>;
    __shared__ __attribute__((aligned(16))) char lds[sizeof(Own) > sizeof(Prefix) ? sizeof(Own) : sizeof(Prefix)];
    __shared__ int last;
    const uint32_t id = blockIdx.x, a = p.x.blocks;
    const bool own = id >= a;
    const uint32_t n = own ? id - a : id;
    if (own) decode_body<HD, RT, T, W, false, Q8, true>(p, *reinterpret_cast<Own *>(lds), n);
    else prefill_body<HD, T, W, 1, Q8, true>(p, *reinterpret_cast<Prefix *>(lds), last, n, a);
}

template <int HD, class T, bool Q8>
void launch_shared_rt(const PagedAttnParams & p, int rt, hipStream_t stream) {
    const dim3 grid(p.x.blocks + p.x.own_blocks), block(kPagedPrefixWaves * kWave);
    if (rt == 16) hipLaunchKernelGGL((paged_shared_kernel<HD, 16, T, Q8>), grid, block, 0, stream, p);
    else if constexpr (HD != 256) hipLaunchKernelGGL((paged_shared_kernel<HD, 32, T, Q8>), grid, block, 0, stream, p);
}

template <bool Q8>
hipError_t launch_shared(const PagedAttnParams & p, int head_dim, int dtype, int rt, hipStream_t stream) {
    if (head_dim == 64) dtype == 1 ? launch_shared_rt<64, F16, Q8>(p, rt, stream) : launch_shared_rt<64, BF16, Q8>(p, rt, stream);
    else if (head_dim == 128) dtype == 1 ? launch_shared_rt<128, F16, Q8>(p, rt, stream) : launch_shared_rt<128, BF16, Q8>(p, rt, stream);
    else dtype == 1 ? launch_shared_rt<256, F16, Q8>(p, rt, stream) : launch_shared_rt<256, BF16, Q8>(p, rt, stream);
    return hipGetLastError();
}

}  // namespace

}  // namespace mx
