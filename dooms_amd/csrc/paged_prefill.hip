// Attention of packed prompts over a paged cache: causal (or not) GQA flash attention of sequences of different lengths, each
// with any number of keys before its rows.
//
// For row t of a sequence with n rows and L keys: out = softmax over keys j <= L - n + t (causal) or all L of scale q_t . k_j,
// times v, with the running maximum m and sum l of a row in f32: O <- O e^(m - m') + sum_j e^(s_j - m') v_j.
//
// What bounds it: 4 n_head head_dim flops per (row, key) pair on the matrix cores; the softmax's exponentials on the vector
// ALUs fill most of the time between the products.
//
//   * A workgroup is W waves of 32 query rows of one head (KSP waves may share a row tile and take the 64-key blocks of a step
//     in turn). Keys and values go straight into LDS (global_load_lds_dwordx4), two to four steps deep, in 1 KB blocks of
//     16 rows x 64 bytes; which 16 bytes a lane fetches spreads the banks. A page holds at least 16 keys, so every block comes
//     from one page: its address is a page number in a scalar register and a fixed offset per lane. The page numbers of a step
//     are read one step ahead of its loads, in the same in-order queue.
//   * S^T = K Q^T on v_mfma_f32_32x32x16: a lane holds 32 keys of one query, so the row maximum and sum cost one cross-lane
//     step and the probabilities are already the operand of O^T += V^T P^T, whose V^T comes through the transposing LDS read.
//   * The reference maximum of a row moves only when a block's probabilities would pass 2^8, so the common block computes no
//     maximum; the mask only where a block crosses the diagonal or the end.
//   * Which tile a workgroup takes follows from the lengths in device memory: the tiles of all sequences in the order of their
//     key blocks, most first (found by bisection over the block count, every lane counting a sequence's tiles above it), dealt
//     so that an XCD works on few kv heads.
#include "mx_paged.hpp"

namespace mx {

namespace {

constexpr int kBK = 64;                 // keys per block
constexpr float kProbSumMax = 256.f;    // a lane's probabilities of half a block at the kept maximum, before it is moved

typedef short short4_t __attribute__((ext_vector_type(4)));

// Buffers of K and V steps: 8 waves (one workgroup per CU) three; 4 waves four at head dim 64 (their steps are short against a
// memory round trip; two with four key quarters, whose steps are 64 KB) and two above.
template <int HD, int W, int KSP>
constexpr int buffers() { return W == 8 ? 3 : (HD == 64 && KSP <= 2 ? 4 : 2); }

template <int HD, int W, int KSP>
struct Smem {
    static constexpr int NBUF = buffers<HD, W, KSP>();
    uint16_t k[NBUF][KSP * kBK * HD];
    uint16_t v[NBUF][KSP * kBK * HD];
};

struct Tile {
    int32_t kvh, gi;     // kv head, query head within its group
    int32_t row0, n;     // the sequence's first query row and its rows
    int32_t len;         // its kv_len
    int32_t b, i;        // sequence and query tile; b -1: nothing
};

// Tiles of a sequence's n rows (R rows a tile) that have more than `key` visible keys: rows up to min((i + 1) R, n) of tile i see
// len - n + that many.
__device__ __forceinline__ int tiles_above(int n, int len, int R, int causal, int key) {
    const int nt = (n + R - 1) / R;
    if (len <= key) return 0;
    if (!causal) return nt;
    // all but the last tile: len - n + (i + 1) R > key, i + 1 > (key - len + n) / R
    const int need = key - len + n;  // below n
    return nt == 0 ? 0 : 1 + (nt - 1) - min(nt - 1, need < 0 ? 0 : need / R);
}

// The tile that workgroup bid takes.
template <int R>
__device__ __forceinline__ Tile find_tile(const PagedAttnParams & p, uint32_t bid, int lane, int resident) {
    const int n_seq = p.c.n_seq;
    struct Seq {
        int lo, n, len;
    };
    auto read = [&](int base) {
        const int i = min(base + lane, n_seq - 1);
        const int lo = min(max(p.cu_q[i], 0), p.n_rows), hi = min(max(p.cu_q[i + 1], 0), p.n_rows);
        return Seq{lo, base + lane < n_seq ? max(hi - lo, 0) : 0, p.c.kv_len[i]};
    };
    const Seq s0 = read(0);
    auto seq = [&](int base) { return base == 0 ? s0 : read(base); };
    // the block counts that order the tiles: a length that is none counts as no keys
    auto len_of = [&](const Seq & s) { return length_ok(p.c, s.len) ? s.len : 0; };
    int nt = 0, most = 0;
    for (int base = 0; base < n_seq; base += kWave) {
        const Seq s = seq(base);
        nt = min(nt + (s.n + R - 1) / R, 1 << 24);
        most = max(most, s.n > 0 ? len_of(s) : 0);
    }
    nt = min(wave_isum(nt), p.max_tiles);  // more only where ranges of cu_q overlap
    Tile t{0, 0, 0, 0, 0, -1, 0};
    if (bid >= (uint32_t)nt * (uint32_t)p.n_head) return t;
    // an XCD serves the heads of one kv head (or of a few); where 8 / n_head_kv XCDs share a kv head, its tiles in the order are
    // dealt to them in turn; the heads of a group are adjacent
    uint32_t o = xcd_remap(bid, (uint32_t)nt * (uint32_t)p.n_head);
    const int per_kv = nt * p.group;
    t.kvh = (int)(o / (uint32_t)per_kv);
    const int r = (int)(o % (uint32_t)per_kv), qi = r / p.group;
    t.gi = r % p.group;
    const int c = p.n_head_kv < 8 && 8 % p.n_head_kv == 0 ? 8 / p.n_head_kv : 1;
    const int each = nt / c, extra = nt % c;
    int rank;
    if (qi < extra * (each + 1)) rank = qi % (each + 1) * c + qi / (each + 1);
    else rank = (qi - extra * (each + 1)) % each * c + extra + (qi - extra * (each + 1)) / each;

    // the rank-th tile in descending order of key blocks. More workgroups than run at once: bisect for the block count x of that
    // tile; otherwise the order does not matter (x = -1: every tile).
    int x = -1;
    if (nt * p.n_head > resident) {
        auto above = [&](int blocks) {  // tiles of more than `blocks` key blocks
            int n = 0;
            for (int base = 0; base < n_seq; base += kWave) {
                const Seq s = seq(base);
                n += tiles_above(s.n, len_of(s), R, p.causal, blocks * kBK);
            }
            return wave_isum(n);
        };
        most = wave_imax(most);
        int lo = -1, hi = (most + kBK - 1) / kBK;  // above(lo) > rank (all of them), above(hi) = 0 <= rank
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (above(mid) > rank) lo = mid;
            else hi = mid;
        }
        x = lo;  // the tile has x + 1 blocks (x = -1: none)
        rank -= above(x + 1);
    }
    for (int base = 0; base < n_seq; base += kWave) {
        const Seq s = seq(base);
        const int all = (s.n + R - 1) / R;
        int more = 0, own = all;  // tiles of more blocks, tiles of x + 1
        if (nt * p.n_head > resident) {
            more = tiles_above(s.n, len_of(s), R, p.causal, (x + 1) * kBK);
            own = (x < 0 ? all : tiles_above(s.n, len_of(s), R, p.causal, x * kBK)) - more;
        }
        const int upto = wave_iscan(own);
        const uint64_t past = __builtin_amdgcn_ballot_w64(upto > rank);
        if (past) {
            const int l = __builtin_ctzll(past);
            const int j = rank - (__builtin_amdgcn_readlane(upto, l) - __builtin_amdgcn_readlane(own, l));
            t.b = base + l;
            t.i = __builtin_amdgcn_readlane(all, l) - 1 - (__builtin_amdgcn_readlane(more, l) + j);
            t.row0 = __builtin_amdgcn_readlane(s.lo, l);
            t.n = __builtin_amdgcn_readlane(s.n, l);
            t.len = __builtin_amdgcn_readlane(s.len, l);
            if ((uint32_t)t.i >= (uint32_t)__builtin_amdgcn_readlane(all, l)) t.b = -1;
            return t;
        }
        rank -= __builtin_amdgcn_readlane(upto, 63);
    }
    return t;
}

// One row by the vector ALUs alone, key by key, for rows that a value outside their mask has spoilt (0 times an infinity or NaN
// is NaN on the matrix cores). Lane l holds dims l, l + 64, ... and returns them; m and l as the row's.
template <int HD, class T>
__device__ __forceinline__ void row_alone(const PagedAttnParams & p, const Tile & t, int row, int visible, float (&o)[HD / 64],
                                                    float & m, float & l) {
    const int lane = threadIdx.x % kWave;
    auto one = [](uint16_t w) { return T::unpack2(w).x; };
    const uint16_t * qr = p.q + (int64_t)(t.row0 + row) * p.q_stride + (int64_t)(t.kvh * p.group + t.gi) * HD;
    float q[HD / 64];
#pragma unroll
    for (int d = 0; d < HD / 64; d++) q[d] = one((uint16_t)((qr[lane + 64 * d] & p.q_and) ^ p.q_xor));
    const int32_t * table = p.c.table + t.b * p.c.table_stride;
    m = kNegInf;
    l = 0.f;
#pragma unroll
    for (int d = 0; d < HD / 64; d++) o[d] = 0.f;
    for (int j = 0; j < visible; j++) {
        const int64_t at = (int64_t)table[j >> p.c.page_shift] * p.c.page_stride +
                           (int64_t)(j & ((1 << p.c.page_shift) - 1)) * p.c.kv_stride + (int64_t)t.kvh * p.c.head_stride + lane;
        float s = 0.f;
#pragma unroll
        for (int d = 0; d < HD / 64; d++) s += q[d] * one(p.c.k[at + 64 * d]);
        s = wave_sum(s) * p.scale_log2;
        const float mn = fmaxf(m, s);
        const float corr = m == kNegInf ? 0.f : exp2_fast(m - mn), w = exp2_fast(s - mn);
        l = l * corr + w;
#pragma unroll
        for (int d = 0; d < HD / 64; d++) o[d] = (m == kNegInf ? 0.f : o[d] * corr) + w * one(p.c.v[at + 64 * d]);
        m = mn;
    }
}

// Whether a value at keys k0 .. k1 - 1 of the tile's kv head is an infinity or NaN (wave-uniform).
template <int HD, class T>
__device__ __forceinline__ bool odd_values(const PagedAttnParams & p, const Tile & t, int k0, int k1) {
    const int lane = threadIdx.x % kWave;
    const int32_t * table = p.c.table + t.b * p.c.table_stride;
    bool odd = false;
    for (int j = k0 + lane / (HD / 8); j < k1; j += kWave / (HD / 8)) {
        const int64_t at = (int64_t)table[j >> p.c.page_shift] * p.c.page_stride +
                           (int64_t)(j & ((1 << p.c.page_shift) - 1)) * p.c.kv_stride + (int64_t)t.kvh * p.c.head_stride +
                           8 * (lane % (HD / 8));
        odd |= any_nonfinite<T>(load16(p.c.v + at));
    }
    return __builtin_amdgcn_ballot_w64(odd) != 0;
}

template <int HD, class T, int W, int KSP>
__global__ __launch_bounds__(W * kWave) __attribute__((amdgpu_waves_per_eu(KSP == 1 && HD <= 128 ? 2 : 1, KSP == 1 && HD <= 128 ? 2 : 1)))
void paged_prefill_kernel(PagedAttnParams p) {
    constexpr int RPW = W / KSP, R = 32 * RPW;  // row tiles and rows of a workgroup
    constexpr int KS = HD / 16;                 // product steps along head_dim for S^T
    constexpr int DT = HD / 32;                 // 32-wide output tiles along head_dim
    constexpr int KB = KSP * kBK;               // keys per step
    constexpr int RB = KB / 16;                 // 16-row blocks per 64-byte column of a step
    constexpr int NB = RB * (HD / 32);          // 1 KB blocks of a step's K (or V)
    constexpr int NI = NB / W;                  // of those a wave loads
    constexpr int ND = RB > W ? RB / W : 1;     // distinct pages among them
    constexpr int NBUF = Smem<HD, W, KSP>::NBUF;
    static_assert(NB % W == 0 && (RB % W == 0 || W % RB == 0), "whole loads per wave, each of one row block");
    __shared__ Smem<HD, W, KSP> sm;

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int lane = threadIdx.x % kWave;
    constexpr int kResident = 256 * (W == 4 && KSP == 1 && HD <= 128 ? 2 : 1);  // workgroups that run at once
    const Tile t = find_tile<R>(p, blockIdx.x, lane, kResident);
    if (t.b < 0) return;
    const int rt = wave % RPW, kh = wave / RPW;  // the wave's row tile and its block of each step
    const int l32 = lane % 32, hgrp = lane / 32;
    const bool bad_len = !length_ok(p.c, t.len);
    const int L = bad_len ? 0 : t.len;
    const int q0 = t.i * R, row = q0 + 32 * rt + l32;  // row among the sequence's
    const int off = L - t.n;                           // key that row 0 sits at (below 0: rows without one)
    const int first_row = q0 + 32 * rt;
    const int h = t.kvh * p.group + t.gi;
    // keys that the workgroup visits, and that this wave's rows see at most (rows past the sequence's see none)
    const int kend = max(0, p.causal ? off + min(q0 + R, t.n) : L);
    const int wave_end = first_row >= t.n ? 0 : p.causal ? off + min(first_row + 32, t.n) : L;
    const int nb = (kend + KB - 1) / KB;

    const int32_t * table = p.c.table + t.b * p.c.table_stride;
    const uint16_t * kg = p.c.k + (int64_t)t.kvh * p.c.head_stride;
    const uint16_t * vg = p.c.v + (int64_t)t.kvh * p.c.head_stride;
    const int shift = p.c.page_shift, page_mask = (1 << shift) - 1;
    const uint32_t row_bytes = (uint32_t)p.c.kv_stride * 2;

    // Loads of a step: block i W + wave holds rows 16 (block % RB) .. + 16 and the 64 bytes block / RB of each; lane l fills
    // bytes 16 l of it: row l / 4, chunk l % 4, for the keys swizzled by the row's quarter so that the operand reads of 16 rows
    // fall on distinct banks.
    const int lrow = lane / 4;
    const uint32_t lane_k = lrow * row_bytes + 16 * ((lane % 4) ^ (lane / 16)), lane_v = lrow * row_bytes + 16 * (lane % 4);
    auto block_row = [&](int i) { return 16 * ((i * W + wave) % RB); };
    int ids[ND];
    // the pages of step kb's loads; steps behind the last key repeat its page
    auto read_ids = [&](int kb) __attribute__((always_inline)) {
#pragma unroll
        for (int d = 0; d < ND; d++) ids[d] = load_uniform(table + (min(kb + block_row(d), L - 1) >> shift));
    };
    bool bad = false;
    // step kb into buffer buf (its pages read before), then the page reads of the step behind it
    auto issue = [&](int kb, int buf) __attribute__((always_inline)) {
        int id[ND];
#pragma unroll
        for (int d = 0; d < ND; d++) {
            id[d] = __builtin_amdgcn_readfirstlane(ids[d]);
            const bool ok = page_ok(p.c, id[d]);
            bad |= !ok;
            id[d] = ok ? id[d] : 0;
        }
        read_ids(kb + KB);
        __builtin_amdgcn_sched_barrier(0);
        const bool partial = kb + KB > L;
#pragma unroll
        for (int i = 0; i < NI; i++) {
            const int j = i * W + wave, cb = j / RB;
            const int k16 = min(kb + block_row(i), (L - 1) & ~15);
            const int64_t base = ((int64_t)id[i % ND] * p.c.page_stride + (int64_t)(k16 & page_mask) * p.c.kv_stride) * 2 + 64 * cb;
            uint32_t ko = lane_k, vo = lane_v;
            if (__builtin_expect(partial, 0)) {  // rows behind the last key repeat it
                const uint32_t back = (uint32_t)max(lrow - (L - 1 - k16), 0) * row_bytes;
                ko -= back;
                vo -= back;
            }
            __builtin_amdgcn_global_load_lds(reinterpret_cast<const char *>(kg) + base + ko,
                                             (__attribute__((address_space(3))) void *)&sm.k[buf][512 * j], 16, 0, 0);
            __builtin_amdgcn_global_load_lds(reinterpret_cast<const char *>(vg) + base + vo,
                                             (__attribute__((address_space(3))) void *)&sm.v[buf][512 * j], 16, 0, 0);
        }
    };

    // the query operand: lane holds Q[row][16 ks + 8 hgrp .. + 8] (rows past the sequence's read its last row, zeroed below)
    u32x4 qb[KS];
    {
        const uint16_t * qr = p.q + (int64_t)(t.row0 + min(row, t.n - 1)) * p.q_stride + (int64_t)h * HD + 8 * hgrp;
#pragma unroll
        for (int ks = 0; ks < KS; ks++) qb[ks] = load16(qr + 16 * ks);
    }
    if (nb > 0) {
        read_ids(0);
        issue(0, 0);
#pragma unroll
        for (int a = 1; a < NBUF - 1; a++)
            if (nb > a) issue(a * KB, a);
    }
#pragma unroll
    for (int ks = 0; ks < KS; ks++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            asm volatile("" : "+v"(qb[ks][e])::"memory");
            qb[ks][e] = row < t.n ? (qb[ks][e] & p.q_and) ^ p.q_xor : 0u;
        }

    float16_t o[DT];
#pragma unroll
    for (int dt = 0; dt < DT; dt++)
#pragma unroll
        for (int v = 0; v < 16; v++) o[dt][v] = 0.f;
    float m_run = kNegInf, l_run = 0.f;  // reference maximum (base 2, scaled) and sum of this lane's keys
    float nm_use = 0.f;                  // -m_run (0 while m_run = -inf)

    // LDS read bases (halves): K[32 mt + l32][16 kk + 8 hgrp] in block (kk / 2, 2 mt + l32 / 16), one base per kk % 2; the
    // transposing V read: lane a of 16-lane group c supplies V[4 hgrp + a / 4][16 (c % 2) + 4 (a % 4)]
    int dl_k[2];
#pragma unroll
    for (int b = 0; b < 2; b++) dl_k[b] = 512 * (l32 / 16) + 32 * (l32 % 16) + 8 * ((2 * b + hgrp) ^ ((l32 % 16) / 4));
    const int dl_v = (4 * hgrp + (lane % 16) / 4) * 32 + 16 * ((lane / 16) % 2) + 4 * (lane % 4);
    const float c = p.scale_log2;
    const int lim = p.causal ? min(off + row, L - 1) : L - 1;  // last key the row sees

    for (int ib = 0; ib < nb; ib++) {
        const int kb = ib * KB + kh * kBK;  // this wave's block of the step
        const int buf = ib % NBUF;
        // this wave's loads of step ib are complete (those of up to NBUF - 2 later steps may be in flight; their page reads are
        // not counted, so that the wait holds with or without them), then every wave's are, and the buffer refilled below was
        // last read in step ib - 1
        const int later = min(NBUF - 2, nb - 1 - ib);
        static_for<0, NBUF - 1>([&](auto RC) __attribute__((always_inline)) {
            constexpr int r = decltype(RC)::value, n = r * 2 * NI;
            static_assert(n < 64, "vmcnt");
            if (later == r) __builtin_amdgcn_s_waitcnt(0x0F70 | (n & 15) | ((n >> 4) << 14));
        });
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (ib + NBUF - 1 < nb) issue((ib + NBUF - 1) * KB, (ib + NBUF - 1) % NBUF);
        if (kb >= wave_end) continue;  // past what this wave's rows see
        const uint32_t ks0 = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint16_t *)sm.k[buf];
        const uint32_t ka0 = ks0 + 2 * (dl_k[0] + 2048 * kh), ka1 = ks0 + 2 * (dl_k[1] + 2048 * kh);
        const uint32_t va = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint16_t *)sm.v[buf] + 2 * (dl_v + 2048 * kh);

        // S^T = K Q^T, two tiles of 32 keys, the products of the two alternating; up to 16 operand reads in flight, each product
        // behind the wait for its own (LDS reads complete in order)
        float16_t sc[2];
#pragma unroll
        for (int v = 0; v < 16; v++) sc[0][v] = sc[1][v] = 0.f;
        constexpr int NS = 2 * KS, NG = NS < 16 ? NS : 16;
        static_for<0, NS / NG>([&](auto GC) __attribute__((always_inline)) {
            constexpr int g0 = decltype(GC)::value * NG;
            u32x4 kf[NG];
            static_for<0, NG>([&](auto I) __attribute__((always_inline)) {
                constexpr int i = g0 + decltype(I)::value;
                constexpr int at = 2 * (512 * RB * (i / 4) + 1024 * (i % 2));
                const uint32_t a = (i / 2) % 2 ? ka1 : ka0;
                u32x4 r;
                asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(r) : "v"(a), "i"(at));
                kf[i - g0] = r;
            });
            static_for<0, NG>([&](auto I) __attribute__((always_inline)) {
                constexpr int i = decltype(I)::value;
                asm volatile("s_waitcnt lgkmcnt(%1)" : "+v"(kf[i]) : "i"(NG - 1 - i));
                sc[i % 2] = T::mfma32(kf[i], qb[(g0 + i) / 2], sc[i % 2]);
                __builtin_amdgcn_sched_barrier(0);
            });
        });
        // the first products' value reads go out ahead of the softmax
        constexpr int VA = 2;
        short4_t vr[VA + 1][2];
        auto vread = [&](auto TC) __attribute__((always_inline)) {
            constexpr int x = decltype(TC)::value;
            constexpr int at = 2 * (512 * (RB * (x % DT) + x / DT));
            short4_t r0, r1;
            asm volatile("ds_read_b64_tr_b16 %0, %2 offset:%3\n\tds_read_b64_tr_b16 %1, %2 offset:%4"
                         : "=&v"(r0), "=&v"(r1)
                         : "v"(va), "i"(at), "i"(at + 512));
            vr[x % (VA + 1)][0] = r0;
            vr[x % (VA + 1)][1] = r1;
        };
        static_for<0, VA>(vread);
        // the mask only where a block crosses the diagonal or the end (wave-uniform)
        if (p.causal ? kb + kBK - 1 > off + first_row : kb + kBK > L) {
#pragma unroll
            for (int mt = 0; mt < 2; mt++)
#pragma unroll
                for (int v = 0; v < 16; v++) {
                    const int key = kb + 32 * mt + 8 * (v / 4) + 4 * hgrp + (v % 4);
                    sc[mt][v] = key > lim ? kNegInf : sc[mt][v];
                }
        }
        // Probabilities at the kept maximum, rounded to T (the P^T operand: step u takes values 8 (u % 2) .. + 8 of score tile
        // u / 2), and the sum of the rounded ones, so that the weights of a row add up to 1. A lane's sum above 2^8 (or a row
        // without a maximum yet) moves the maximum, rescales l and O, and computes the block again.
        u32x4 pb[4];
        auto settle = [&](auto H0C, auto H1C) __attribute__((always_inline)) {
            constexpr int H0 = decltype(H0C)::value, H1 = decltype(H1C)::value;
            float bs;
            auto probs = [&]() __attribute__((always_inline)) {
                bs = 0.f;
#pragma unroll
                for (int u = 2 * H0; u < 2 * H1; u++)
#pragma unroll
                    for (int e = 0; e < 8; e += 2) {
                        const float a = exp2_fast(__builtin_fmaf(sc[u / 2][8 * (u % 2) + e], c, nm_use));
                        const float b = exp2_fast(__builtin_fmaf(sc[u / 2][8 * (u % 2) + e + 1], c, nm_use));
                        pb[u][e / 2] = T::pack2(a, b);
                    }
#pragma unroll
                for (int u = 2 * H0; u < 2 * H1; u++)
#pragma unroll
                    for (int e = 0; e < 4; e++) bs = T::add2(pb[u][e], bs);
            };
            probs();
            if (__builtin_amdgcn_ballot_w64(bs > kProbSumMax || m_run == kNegInf)) {
                float bmax = kNegInf;
#pragma unroll
                for (int mt = H0; mt < H1; mt++)
#pragma unroll
                    for (int v = 0; v < 16; v++) bmax = fmaxf(bmax, sc[mt][v]);
                bmax = xor32_max(bmax);
                const float m_new = fmaxf(m_run, bmax * c);
                const float corr = m_new == kNegInf ? 1.f : exp2_fast(m_run - m_new);
                m_run = m_new;
                nm_use = m_new == kNegInf ? 0.f : -m_new;  // no key yet: every exponent below is 2^-inf = 0
                l_run *= corr;
#pragma unroll
                for (int dt = 0; dt < DT; dt++)
#pragma unroll
                    for (int v = 0; v < 16; v++) o[dt][v] *= corr;
                probs();
            }
            l_run += bs;
        };
        using I0 = std::integral_constant<int, 0>;
        using I1 = std::integral_constant<int, 1>;
        using I2 = std::integral_constant<int, 2>;
        // the second half of the keys settles between the products of the first, except at head dim 128
        constexpr bool kSplitHalves = HD != 128;
        if constexpr (kSplitHalves) settle(I0{}, I1{});
        else settle(I0{}, I2{});
        // O^T += V^T P^T: 4 steps of 16 keys; two transposing reads fetch the keys of a step
        constexpr int NP = 4 * DT;
        static_for<0, NP + VA>([&](auto I) __attribute__((always_inline)) {
            constexpr int x = decltype(I)::value;
            if constexpr (x >= VA && x < NP) vread(I);
            if constexpr (x >= VA) {
                constexpr int j = x - VA;
                if constexpr (kSplitHalves && j == NP / 2) settle(I1{}, I2{});
                constexpr int behind = 2 * ((x < NP - 1 ? x : NP - 1) - j);
                asm volatile("s_waitcnt lgkmcnt(%2)"
                             : "+v"(vr[j % (VA + 1)][0]), "+v"(vr[j % (VA + 1)][1])
                             : "i"(behind));
                const short4_t lo = vr[j % (VA + 1)][0], hi = vr[j % (VA + 1)][1];
                const u32x4 a = __builtin_bit_cast(u32x4, (short __attribute__((ext_vector_type(8)))){
                    lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]});
                o[j % DT] = T::mfma32(a, pb[j / DT], o[j % DT]);
            }
        });
    }

    l_run = xor32_add(l_run);
    // a bad page was met by the waves that load it: every wave of the workgroup learns of it
    __shared__ int s_bad;
    if (threadIdx.x == 0) s_bad = 0;
    __syncthreads();
    if (bad && lane == 0) s_bad = 1;
    __syncthreads();
    const bool poison = bad_len || s_bad;
    if constexpr (KSP > 1) {
        // the KSP waves of a row tile join their (m, l, O): waves kh > 0 leave theirs in LDS, the wave kh = 0 folds them in
        constexpr int XS = DT * 16 + 2;  // floats per lane
        static_assert((int64_t)RPW * (KSP - 1) * kWave * XS * 4 <= (int64_t)sizeof(sm), "merge scratch fits the tiles");
        float * xs = reinterpret_cast<float *>(&sm);
        if (kh > 0) {
            float * d = xs + ((rt * (KSP - 1) + kh - 1) * kWave + lane) * XS;
#pragma unroll
            for (int dt = 0; dt < DT; dt++)
#pragma unroll
                for (int v = 0; v < 16; v++) d[16 * dt + v] = o[dt][v];
            d[16 * DT] = m_run;
            d[16 * DT + 1] = l_run;
        }
        __syncthreads();
        if (kh > 0) return;
#pragma unroll
        for (int j = 0; j < KSP - 1; j++) {
            const float * d = xs + ((rt * (KSP - 1) + j) * kWave + lane) * XS;
            const float m1 = d[16 * DT], l1 = d[16 * DT + 1];
            const float mn = fmaxf(m_run, m1);
            const float w0 = m_run == kNegInf ? 0.f : exp2_fast(m_run - mn);
            const float w1 = m1 == kNegInf ? 0.f : exp2_fast(m1 - mn);
#pragma unroll
            for (int dt = 0; dt < DT; dt++)
#pragma unroll
                for (int v = 0; v < 16; v++) o[dt][v] = o[dt][v] * w0 + d[16 * dt + v] * w1;
            l_run = l_run * w0 + l1 * w1;
            m_run = mn;
        }
    }

    // ---- normalize and store: lane holds O[row][32 dt + 8 (v / 4) + 4 hgrp + v % 4] ----
    if (first_row >= t.n) return;  // wave-uniform
    const bool live = row < t.n, empty = lim < 0;
    const float inv = 1.f / l_run;
    bool odd = false;
#pragma unroll
    for (int dt = 0; dt < DT; dt++)
#pragma unroll
        for (int v = 0; v < 16; v++) {
            o[dt][v] *= inv;
            odd |= !(__builtin_fabsf(o[dt][v]) < __builtin_inff());
        }
    const int64_t out_row = (int64_t)(t.row0 + row) * p.out_stride + (int64_t)h * HD;
    if (live) {
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
#pragma unroll
            for (int gq = 0; gq < 4; gq++) {
                float4_t r;
#pragma unroll
                for (int e = 0; e < 4; e++) r[e] = poison ? __builtin_nanf("") : empty ? 0.f : o[dt][4 * gq + e];
                const int64_t at = out_row + 32 * dt + 8 * gq + 4 * hgrp;
                if (p.out32) *reinterpret_cast<float4_t *>(static_cast<float *>(p.out) + at) = r;
                else *reinterpret_cast<u32x2 *>(static_cast<uint16_t *>(p.out) + at) = u32x2{T::pack2(r[0], r[1]), T::pack2(r[2], r[3])};
            }
        if (p.lse && hgrp == 0)
            p.lse[(int64_t)(t.row0 + row) * p.n_head + h] = poison ? __builtin_nanf("") : empty ? kNegInf : (m_run + log2_fast(l_run)) * kLn2;
    }
    // Rows that came out as no number although they see keys: if a value outside some row's mask is an infinity or NaN, they
    // are computed again by themselves.
    uint64_t again = __builtin_amdgcn_ballot_w64(odd && live && !empty && !poison);
    again = (again | (again >> 32)) & 0xffffffffull;
    if (!again || !p.causal) return;
    const int top = min(L, (wave_end + kBK - 1) / kBK * kBK);  // keys that the wave's products took in
    if (!odd_values<HD, T>(p, t, max(0, off + first_row + 1), top)) return;
    while (again) {
        const int r = first_row + __builtin_ctzll(again);
        again &= again - 1;
        float x[HD / 64], m, l;
        row_alone<HD, T>(p, t, r, min(off + r + 1, L), x, m, l);
        const int64_t at = (int64_t)(t.row0 + r) * p.out_stride + (int64_t)h * HD + lane;
#pragma unroll
        for (int d = 0; d < HD / 64; d++) {
            const float v = x[d] / l;
            if (p.out32) static_cast<float *>(p.out)[at + 64 * d] = v;
            else static_cast<uint16_t *>(p.out)[at + 64 * d] = (uint16_t)T::pack2(v, 0.f);
        }
    }
}

template <int HD, class T>
void launch_plan(const PagedAttnParams & p, int plan, hipStream_t stream) {
    const dim3 grid((uint32_t)p.max_tiles * (uint32_t)p.n_head);
    if constexpr (HD == 256) {
        hipLaunchKernelGGL((paged_prefill_kernel<HD, T, 4, 1>), grid, dim3(4 * kWave), 0, stream, p);
    } else {
        if (plan == 8) hipLaunchKernelGGL((paged_prefill_kernel<HD, T, 8, 1>), grid, dim3(8 * kWave), 0, stream, p);
        else if (plan == 4) hipLaunchKernelGGL((paged_prefill_kernel<HD, T, 4, 1>), grid, dim3(4 * kWave), 0, stream, p);
        else if (plan == 2 || HD == 128) hipLaunchKernelGGL((paged_prefill_kernel<HD, T, 4, 2>), grid, dim3(4 * kWave), 0, stream, p);
        else if constexpr (HD == 64) hipLaunchKernelGGL((paged_prefill_kernel<HD, T, 4, 4>), grid, dim3(4 * kWave), 0, stream, p);
    }
}

template <class T>
void launch_hd(const PagedAttnParams & p, int head_dim, int plan, hipStream_t stream) {
    if (head_dim == 64) launch_plan<64, T>(p, plan, stream);
    else if (head_dim == 128) launch_plan<128, T>(p, plan, stream);
    else launch_plan<256, T>(p, plan, stream);
}

}  // namespace

// plan: 8 = 8 waves x 32 rows, 4 = 4 waves x 32 rows, 2 = 4 waves over 2 row tiles x 2 key halves, 1 = 4 waves over the key
// quarters of one row tile (head dim 64); head dim 256 runs plan 4.
hipError_t launch_paged_prefill(const PagedAttnParams & p, int head_dim, int dtype, int plan, hipStream_t stream) {
    if (dtype == 1) launch_hd<F16>(p, head_dim, plan, stream);
    else launch_hd<BF16>(p, head_dim, plan, stream);
    return hipGetLastError();
}

}  // namespace mx
