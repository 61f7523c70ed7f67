// Attention of packed prompts over a paged cache: causal (or not) GQA flash attention of sequences of different lengths, each
// with any number of keys before its rows.
//
// For row t of a sequence with n rows and L keys: out = softmax over keys j <= L - n + t (causal) or all L of scale q_t . k_j,
// times v, with the running maximum m and sum l of a row in f32: O <- O e^(m - m') + sum_j e^(s_j - m') v_j.
//
// What bounds it: 4 n_head head_dim flops per (row, key) pair on the matrix cores; the softmax's exponentials on the vector
// ALUs fill most of the time between the products (two chunks of 1.5k-2k rows behind 14k keys, Qwen2.5-7B heads, 736 GFLOP in 735 to
// 780 us from card to card, 945 to 1000 TFLOP/s; a large library product of the type reaches 1324, its right operand transposed
// 1517). Short prompts add what a tile costs beside its keys, about 3 us of queries, outputs and first loads (12 prompts of 65-1711
// rows, Llama-3-8B heads, 104 GFLOP in 152 to 160 us).
//
//   * A tile is W waves of 32 query rows: W / HPW row tiles of each of HPW heads that share a kv head, so that a short or causal
//     tile wastes few rows and the keys serve all of them. Steps are 64 keys; keys and values go straight into LDS
//     (global_load_lds_dwordx4), two to four steps deep, in 1 KB blocks of 16 rows x 64 bytes; which 16 bytes a lane fetches
//     spreads the banks. A page holds at least 16 keys, so every block comes from one page: its address is a page number in a
//     scalar register and a fixed offset per lane. The page numbers of a step are read one step ahead of its loads, in the same
//     in-order queue.
//   * S^T = K Q^T on v_mfma_f32_32x32x16: a lane holds 32 keys of one query, so the row maximum and sum cost one cross-lane
//     step and the probabilities are already the operand of O^T += V^T P^T, whose V^T comes through the transposing LDS read.
//   * The reference maximum of a row moves only when a block's probabilities would pass 2^8, so the common block computes no
//     maximum; the mask only where a block crosses the diagonal or the end.
//   * Pages of e4m3 codes: the loads put codes and scales into LDS, each lane expands the 16 codes that it loaded itself into the tile
//     that the products read, and the rest is as in 16 bits (the two chunks 767 to 800 us, the 12 prompts 162 to 175, 2 to 5 % more).
//   * The tiles of all sequences, with their key steps, are one list of units, which the lengths in device memory give; each of the
//     workgroups that run at once takes an equal range of it, and walks it without a break: the first steps of a tile are loaded
//     under the last ones of the tile before. A range that ends within a tile leaves a partial (m, l, O) in the workspace, and the
//     workgroup that completes a tile's parts joins them in order. Few short tiles go one to a workgroup instead.
#pragma once

#include "mx_paged.hpp"

namespace mx {

namespace {

constexpr int kBK = 64;                 // keys per step
constexpr float kProbSumMax = 256.f;    // a lane's probabilities of half a step at the kept maximum, before it is moved
// A tile costs about this many steps beside its own; a range does not cut off less than kMinPart, nor takes fewer than kMinShare
// (joining a part costs about 2 us: 100 rows of 14 heads behind 8000 keys 45 us without, 35 with).
constexpr int kTileCost = 2, kMinPart = 4, kMinShare = 10;
constexpr int kDirectSteps = 24;        // tiles of up to so many steps go one to a workgroup where there are few

typedef short short4_t __attribute__((ext_vector_type(4)));

// Buffers of steps: three (two steps ahead), or two where a third does not fit beside a second workgroup.
template <int HD, int W, bool Q8>
struct Smem {
    static constexpr int NBUF = W == 8 || HD == 64 ? 3 : 2;
    static constexpr int RING = NBUF, AHEAD = NBUF - 1;  // buffers that loads fill, and of those at most in flight or unread
    uint16_t k[NBUF][kBK * HD];
    uint16_t v[NBUF][kBK * HD];
    int32_t ids[W][kWave];  // page numbers of a wave's next step: its four 16-row blocks in lanes 0 .. 3 (and again above)
};
// Pages of codes: the loads fill a ring of codes and scales, each lane expands the 16 bytes that it loaded itself into the buffer that
// the products read: two in turn, or one between two barriers where a second does not fit.
template <int HD, int W>
struct Smem<HD, W, true> {
    static constexpr int NBUF = W == 8 || HD == 64 ? 2 : 1;
    static constexpr int RING = 2, AHEAD = 2;
    uint16_t k[NBUF][kBK * HD];
    uint16_t v[NBUF][kBK * HD];
    uint8_t kc[RING][kBK * HD];
    uint8_t vc[RING][kBK * HD];
    int32_t scales[RING][W][kWave];  // of a wave's 16 rows: the keys' in bytes 0 .. 15, the values' in bytes 16 .. 31 (and again above)
    int32_t ids[W][kWave];
};

// Inclusive prefix sums of values below 2^49 over a wave.
__device__ __forceinline__ int64_t wave_scan64(int64_t v) {
    return ((int64_t)wave_iscan((int32_t)(v >> 24)) << 24) + wave_iscan((int32_t)(v & 0xffffff));
}
__device__ __forceinline__ int64_t read_lane64(int64_t v, int l) {
    return (int64_t)(uint32_t)__builtin_amdgcn_readlane((int32_t)v, l) | (int64_t)__builtin_amdgcn_readlane((int32_t)(v >> 32), l) << 32;
}

// A sequence's tiles of R rows (a multiple of kBK): row r sits at key off + r.
template <int R>
struct Rows {
    int n, L, off, nt, c0;  // rows, keys (0: none, or a length that is none), tiles, steps before row 0
    int causal;
    __device__ __forceinline__ Rows(int n_, int len, bool ok, int causal_) : n(n_), L(ok ? len : 0), causal(causal_) {
        off = L - n;
        nt = (n + R - 1) / R;
        c0 = (off + kBK - 1) >> 6;
    }
    // steps of tile i, one at least: rows without keys are written too
    __device__ __forceinline__ int steps(int i) const {
        const int all = (L + kBK - 1) / kBK;
        return max(1, causal && i < nt - 1 ? c0 + (i + 1) * (R / kBK) : all);
    }
    // units of the tiles before tile i <= nt - 1: the first z have one step
    __device__ __forceinline__ int64_t before(int i) const {
        if (!causal) return (int64_t)i * (steps(0) + kTileCost);
        const int z = min(max((1 - c0) / (R / kBK), 0), i);
        return (int64_t)i * kTileCost + z + (int64_t)(i - z) * c0 + (int64_t)(R / kBK) * (((int64_t)i * (i + 1) - (int64_t)z * (z + 1)) / 2);
    }
    __device__ __forceinline__ int64_t units() const { return nt ? before(nt - 1) + steps(nt - 1) + kTileCost : 0; }
};

struct Tile {
    int32_t b, i, set;   // sequence (-1: nothing), query tile, set of HPW heads of the group
    int32_t kvh;
    int32_t row0, n, len;  // the sequence's first query row, its rows, its kv_len
    int32_t s0, s1, steps; // the steps of this part, and of the tile
    int64_t start;         // the tile's first unit
};

// Element d of the row at `row` elements of a pool, and for codes its scale at `scale` bytes.
template <class T, bool Q8>
__device__ __forceinline__ float value_at(const uint16_t * pool, const uint8_t * scales, int64_t row, int64_t scale, int d) {
    if constexpr (Q8) {
        return T::unpack2(T::template expand2<false>(reinterpret_cast<const uint8_t *>(pool)[row + d], scale_of(scales[scale], 0))).x;
    } else {
        return T::unpack2(pool[row + d]).x;
    }
}

// One row by the vector ALUs alone, key by key, for rows that a value outside their mask has spoilt (0 times an infinity or NaN
// is NaN on the matrix cores). Lane l holds dims l, l + 64, ... and returns them; m and l as the row's.
template <int HD, class T, bool Q8>
__device__ __forceinline__ void row_alone(const PagedAttnParams & p, const Tile & t, int h, int row, int visible, float (&o)[HD / 64],
                                                    float & m, float & l) {
    const int lane = threadIdx.x % kWave;
    auto one = [](uint16_t w) { return T::unpack2(w).x; };
    const uint16_t * qr = p.q + (int64_t)(t.row0 + row) * p.q_stride + (int64_t)h * HD;
    float q[HD / 64];
#pragma unroll
    for (int d = 0; d < HD / 64; d++) q[d] = one((uint16_t)((qr[lane + 64 * d] & p.q_and) ^ p.q_xor));
    const int32_t * table = p.c.table + t.b * p.c.table_stride;
    bool bad = false;  // a page of another part of the tile may be none
    m = kNegInf;
    l = 0.f;
#pragma unroll
    for (int d = 0; d < HD / 64; d++) o[d] = 0.f;
    for (int j = 0; j < visible; j++) {
        const int id = table[j >> p.c.page_shift];
        bad |= !page_ok(p.c, id);
        const int64_t page = page_ok(p.c, id) ? id : 0;
        const int in = j & ((1 << p.c.page_shift) - 1);
        const int64_t at = page * p.c.page_stride + (int64_t)in * p.c.kv_stride + (int64_t)t.kvh * p.c.head_stride + lane;
        const int64_t sat = Q8 ? page * p.s.page_stride + (int64_t)t.kvh * p.s.head_stride + in : 0;
        float s = 0.f;
#pragma unroll
        for (int d = 0; d < HD / 64; d++) s += q[d] * value_at<T, Q8>(p.c.k, p.s.k, at, sat, 64 * d);
        s = wave_sum(s) * p.scale_log2;
        // scores of -inf alone (keys that hold an infinity) weigh 2^-inf = 0 each, and leave the maximum to the first finite one
        const float mn = fmaxf(m, s), use = mn == kNegInf ? 0.f : mn;
        const float corr = exp2_fast(m - use), w = exp2_fast(s - use);
        l = l * corr + w;
#pragma unroll
        for (int d = 0; d < HD / 64; d++) o[d] = o[d] * corr + w * value_at<T, Q8>(p.c.v, p.s.v, at, sat, 64 * d);
        m = mn;
    }
    if (bad) l = __builtin_nanf("");
}

// Whether a value at keys k0 .. k1 - 1 of the tile's kv head is an infinity or NaN (wave-uniform).
template <int HD, class T, bool Q8>
__device__ __forceinline__ bool odd_values(const PagedAttnParams & p, const Tile & t, int k0, int k1) {
    const int lane = threadIdx.x % kWave;
    const int32_t * table = p.c.table + t.b * p.c.table_stride;
    bool odd = false;
    for (int j = k0 + lane / (HD / 8); j < k1; j += kWave / (HD / 8)) {
        const int id = table[j >> p.c.page_shift];
        if (!page_ok(p.c, id)) continue;
        const int64_t at = (int64_t)id * p.c.page_stride + (int64_t)(j & ((1 << p.c.page_shift) - 1)) * p.c.kv_stride +
                           (int64_t)t.kvh * p.c.head_stride + 8 * (lane % (HD / 8));
        if constexpr (Q8) {
            const u32x2 w = *reinterpret_cast<const u32x2 *>(reinterpret_cast<const uint8_t *>(p.c.v) + at);
            const int64_t sat = (int64_t)id * p.s.page_stride + (int64_t)t.kvh * p.s.head_stride + (j & ((1 << p.c.page_shift) - 1));
            odd |= any_nonfinite<T>(expand8<T>(w[0], w[1], scale_of(p.s.v[sat], 0)));
        } else {
            odd |= any_nonfinite<T>(load16(p.c.v + at));
        }
    }
    return __builtin_amdgcn_ballot_w64(odd) != 0;
}

// ---- shared prefixes: the rows of a group's sequences are one tile list over the keys they share ----

// Rows of R a tile: the tile, and the part of its keys, that workgroup `block` of the launch computes (b -1: none), with the group's row
// of the page table in t.b and its first query row in t.row0. Every part takes the same count of steps, the least for which the
// prefixes have no more parts than workgroups (x.room); 2 to 4 steps at least where 8 parts suffice, as more are more to write, read back
// and join than the shorter walks save (64 rows, Llama-3-8B heads, 2048 shared keys, 20.4 us, in 16 parts 21.5; 32 x 2 rows, Qwen2.5-7B
// heads, 1024, 17.2 and 18.2; but 16 rows behind 512 keys 12.2 in 8 parts, 12.8 in 4); and x.least. The waves of the last workgroups also
// write what the join needs to know of each sequence.
template <int R, int W>
__device__ __forceinline__ Tile plan_prefix(const PagedAttnParams & p, int wave, uint32_t block, uint32_t blocks, PagedPrefixPart & part) {
    const PagedPrefix & x = p.x;
    const int lane = threadIdx.x % kWave, n_seq = p.c.n_seq, per_seq = p.n_q * p.group;
    struct Group {
        int s0, n, keys, rows, steps, tiles, least;  // rows 0: nothing is shared
    };
    auto clamp = [&](int s) { return min(max(s, 0), n_seq); };
    auto group_at = [&](int base) {
        Group r;
        const int i = min(base + lane, x.n_groups - 1);
        r.s0 = clamp(x.cu_seq[i]);
        r.n = base + lane < x.n_groups ? max(clamp(x.cu_seq[i + 1]) - r.s0, 0) : 0;
        r.keys = x.prefix_len[i];
        const bool shared = prefix_apart(p, r.n, r.keys) && r.keys <= p.c.capacity;
        r.rows = shared ? r.n * per_seq : 0;
        r.steps = shared ? (r.keys + kBK - 1) / kBK : 0;
        r.tiles = (r.rows + R - 1) / R;
        r.least = max(min(4, (r.steps + 7) / 8), x.least);
        return r;
    };
    const Group first = group_at(0);
    auto at = [&](int base) { return base == 0 ? first : group_at(base); };
    auto parts = [&](const Group & r, int c) { return r.rows ? (r.steps + max(c, r.least) - 1) / max(c, r.least) : 0; };
    const int room = max(1, p.x.room / p.n_head_kv);
    float sum = 0.f;
    int longest = 1, tiles = 0;  // of a kv head, at most 2^29
    int64_t rows = 0;            // of the partials of a kv head
    for (int base = 0; base < x.n_groups; base += kWave) {
        const Group r = at(base);
        sum += (float)r.tiles * (float)r.steps;
        longest = max(longest, r.steps);
        tiles = min(tiles + wave_isum(min(r.tiles, 1 << 23)), 1 << 29);
        rows += read_lane64(wave_scan64(r.rows), 63);
    }
    longest = wave_imax(longest);
    int c = longest, per_kv = tiles;
    if (tiles > 0 && tiles <= room) {  // else each prefix is one part, and the sums are done: with many groups they are what the plan costs
        auto count = [&](int c) {  // parts of a kv head, at most 2^30
            int r = 0;
            for (int base = 0; base < x.n_groups; base += kWave) {
                const Group y = at(base);
                r = min(r + wave_isum((int)min((int64_t)y.tiles * parts(y, c), (int64_t)1 << 23)), 1 << 29);
            }
            return r;
        };
        sum = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(wave_sum(sum))));
        c = __builtin_amdgcn_readfirstlane((int)fminf(ceilf(sum / (float)room), (float)longest));
        c = max(c, (longest + kPagedMaxParts - 1) / kPagedMaxParts);
        for (int i = 0; c < longest && count(c) > room; i++) c = i < 16 ? min(c + max(1, c / 8), longest) : longest;
        per_kv = count(c);
        rows = 0;
        for (int base = 0; base < x.n_groups; base += kWave) {
            const Group r = at(base);
            rows += read_lane64(wave_scan64((int64_t)r.rows * parts(r, c)), 63);
        }
    }
    // only ranges of cu_seq that overlap have more parts or rows than the launch
    const int64_t all = (int64_t)per_kv * p.n_head_kv;
    const bool fits = all <= (int64_t)blocks && rows * p.n_head_kv <= x.max_rows;

    // ---- the sequences: where their own keys start, how many they are, and where the partials lie ----
    if (block == 0 && threadIdx.x == 0) *x.rows = fits ? (int32_t)rows : 0;
    for (int64_t b0 = ((int64_t)(blocks - 1 - block) * W + wave) * kWave; b0 < n_seq; b0 += (int64_t)blocks * W * kWave) {
        const int b = min((int)b0 + lane, n_seq - 1);
        int g = 0, end = x.n_groups;  // the last group that does not start behind b
        while (__builtin_amdgcn_ballot_w64(end - g > 1)) {
            const int mid = (g + end) / 2;
            if (end - g > 1) {
                if (x.cu_seq[mid] <= b) g = mid;
                else end = mid;
            }
        }
        const int s0 = clamp(x.cu_seq[g]), s1 = clamp(x.cu_seq[g + 1]), len = p.c.kv_len[b];
        const bool in = s0 <= b && b < s1;
        OwnKeys own = own_of(p, in, s0, s1, x.prefix_len[g], len);
        int np = 0, group_rows = 0;
        int64_t first_row = 0;
        for (int base = 0; base < x.n_groups; base += kWave) {
            const Group r = at(base);
            const int n = parts(r, c);
            const int64_t mine = (int64_t)r.rows * n, upto = wave_scan64(mine) - mine;
            const int from = (g - base) & (kWave - 1);
            const int lo = __builtin_amdgcn_ds_bpermute(4 * from, (int32_t)upto), n_of = __builtin_amdgcn_ds_bpermute(4 * from, n);
            const int rows_of = __builtin_amdgcn_ds_bpermute(4 * from, r.rows);
            const int last = __builtin_amdgcn_readlane((int32_t)(upto + mine), 63);
            if (g - base >= 0 && g - base < kWave) {
                first_row += (uint32_t)lo;
                np = n_of;
                group_rows = rows_of;
            } else if (g >= base + kWave) {
                first_row += (uint32_t)last;
            }
        }
        if (own.start != 0 && !fits) own.len = -1;
        if (own.start == 0 || !fits) {  // nothing for the join to read: without room the sums above are of no rows that there are
            np = group_rows = 0;
            first_row = 0;
        }
        if ((int)b0 + lane < n_seq) {
            x.own_len[b] = own.len;
            x.info[b] = make_int4((int)first_row, group_rows, np, (b - s0) * per_seq);
        }
    }

    // ---- the workgroup's part: by kv head, group, keys, then tiles, neighbours on one XCD ----
    Tile t{};
    t.b = -1;
    if (!fits || block >= (uint32_t)all) return t;
    int o = (int)xcd_remap(block, (uint32_t)all);
    t.kvh = o / per_kv;
    o -= t.kvh * per_kv;
    int64_t before = 0;
    for (int base = 0; base < x.n_groups; base += kWave) {
        const Group r = at(base);
        const int n = parts(r, c), mine = r.tiles * n, upto = wave_iscan(mine);
        const int64_t of_rows = wave_scan64((int64_t)r.rows * n);
        const uint64_t past = __builtin_amdgcn_ballot_w64(upto > o);
        if (past) {
            const int l = __builtin_ctzll(past);
            o -= __builtin_amdgcn_readlane(upto, l) - __builtin_amdgcn_readlane(mine, l);
            const int tiles = __builtin_amdgcn_readlane(r.tiles, l), k = o / tiles, each = max(c, __builtin_amdgcn_readlane(r.least, l));
            t.b = __builtin_amdgcn_readlane(r.s0, l);
            t.row0 = t.b * p.n_q;
            t.n = __builtin_amdgcn_readlane(r.rows, l);
            t.len = __builtin_amdgcn_readlane(r.keys, l);
            t.i = o - k * tiles;
            t.steps = __builtin_amdgcn_readlane(r.steps, l);
            t.s0 = k * each;
            t.s1 = min(t.s0 + each, t.steps);
            part.rows = t.n;
            part.first = t.kvh * rows + before + read_lane64(of_rows, l) - (int64_t)t.n * __builtin_amdgcn_readlane(n, l) + (int64_t)k * t.n;
            return t;
        }
        o -= __builtin_amdgcn_readlane(upto, 63);
        before += read_lane64(of_rows, 63);
    }
    return t;
}

// HD: head_dim. T: type of query rows and pages. W: waves. HPW: query heads of a group that a workgroup takes, W / HPW row tiles of
// each. Q8: the pages hold e4m3 codes with a scale a row, expanded to T in LDS. PREFIX: the keys that groups of sequences share, for all
// rows of a group; a row is one of a query head then, and a workgroup computes one part of a tile and leaves it to the next kernel.
template <int HD, class T, int W, int HPW, bool Q8, bool PREFIX>
__device__ __forceinline__ void prefill_body(const PagedAttnParams & p, Smem<HD, W, Q8> & sm, int & s_last, const uint32_t block, const uint32_t blocks) {
    constexpr int RPW = W / HPW, R = 32 * RPW;  // row tiles of a head, and rows
    static_assert(R % kBK == 0, "tiles of whole steps");
    constexpr int KS = HD / 16;                 // product steps along head_dim for S^T
    constexpr int DT = HD / 32;                 // 32-wide output tiles along head_dim
    constexpr int RB = kBK / 16;                // 16-row blocks per 64-byte column of a step
    constexpr int ES = Q8 ? 1 : 2;              // bytes of an element of the pages
    constexpr int NB = RB * (HD * ES / 64);     // 1 KB blocks of a step's K (or V)
    constexpr int NI = NB / W;                  // of those a wave loads
    using Mem = Smem<HD, W, Q8>;
    constexpr int NBUF = Mem::NBUF, RING = Mem::RING, AHEAD = Mem::AHEAD;
    constexpr int LOADS = 2 * NI + (Q8 ? 1 : 0);  // of a step, a wave's
    static_assert(NB % W == 0 && W % RB == 0, "whole loads per wave, all of one row block");

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int lane = threadIdx.x % kWave;
    const int n_seq = p.c.n_seq, sets = PREFIX ? 1 : (p.group + HPW - 1) / HPW;
    [[maybe_unused]] PagedPrefixPart prefix_part;

    // ---- the sequences, 64 in lanes: rows lo .. lo + n - 1, kv_len ----
    int lo = 0, nq = 0, len = 0, first_seq = -1;
    auto read = [&](int base) __attribute__((always_inline)) {
        const int i = min(base + lane, n_seq - 1);
        lo = min(max(p.cu_q[i], 0), p.n_rows);
        const int hi = min(max(p.cu_q[i + 1], 0), p.n_rows);
        nq = base + lane < n_seq ? max(hi - lo, 0) : 0;
        len = p.c.kv_len[i];
        first_seq = base;
    };
    auto rows_of = [&](int n, int len) { return Rows<R>(n, len, length_ok(p.c, len), p.causal); };
    // sequence b's values into t (its lanes read where they are not)
    auto enter = [&](Tile & t, int b) __attribute__((always_inline)) {
        if ((uint32_t)(b - first_seq) >= (uint32_t)kWave) read(b);
        t.b = b;
        t.row0 = __builtin_amdgcn_readlane(lo, b - first_seq);
        t.n = __builtin_amdgcn_readlane(nq, b - first_seq);
        t.len = __builtin_amdgcn_readlane(len, b - first_seq);
    };

    // ---- the workgroup's range of units, or its tile ----
    int tiles = 0, longest = 0;  // of one kv head and set
    int64_t units = 0;
    for (int base = 0; !PREFIX && base < n_seq; base += kWave) {
        read(base);
        const Rows<R> s = rows_of(nq, len);
        // more than p.max_tiles only where ranges of cu_q overlap
        tiles = min(tiles + __builtin_amdgcn_readlane(wave_iscan(min(s.nt, 1 << 24)), 63), p.max_tiles);
        units += read_lane64(wave_scan64(s.units()), 63);
        longest = max(longest, wave_imax(s.n ? s.steps(s.nt - 1) : 0));
    }
    const int all = tiles * sets * p.n_head_kv;
    const bool direct = PREFIX || (all <= p.ranges && longest <= kDirectSteps);
    const int64_t per_kv = units * sets, total = per_kv * p.n_head_kv;
    Tile t{};
    t.b = -1;
    int64_t hi_unit = 0, share = 1;
    int range = 0;
    if constexpr (PREFIX) {
        t = plan_prefix<R, W>(p, wave, block, blocks, prefix_part);
        if (t.b < 0) return;
    } else if (direct) {
        if (block >= (uint32_t)all) return;
        int o = (int)xcd_remap(block, (uint32_t)all);
        t.kvh = o / (tiles * sets);
        o -= t.kvh * tiles * sets;
        t.set = o % sets;
        o /= sets;
        for (int base = 0; base < n_seq && t.b < 0; base += kWave) {
            if (base != first_seq) read(base);
            const int nt = (nq + R - 1) / R, upto = wave_iscan(nt);
            const uint64_t past = __builtin_amdgcn_ballot_w64(upto > o);
            if (past) {
                const int l = __builtin_ctzll(past);
                t.i = o - (__builtin_amdgcn_readlane(upto, l) - __builtin_amdgcn_readlane(nt, l));
                enter(t, base + l);
            }
            o -= __builtin_amdgcn_readlane(upto, 63);
        }
        if (t.b < 0) return;
        t.steps = rows_of(t.n, t.len).steps(t.i);
        t.s0 = 0;
        t.s1 = t.steps;
    } else {
        if (total <= 0) return;
        // workgroups are dealt to the 8 XCDs round-robin: each XCD walks one eighth of the list, so few kv heads
        range = (int)(block % 8) * (p.ranges / 8) + (int)(block / 8);
        if (range >= p.ranges) return;
        share = max((total + p.ranges - 1) / p.ranges, (int64_t)kMinShare);
        const int64_t from = range * share;
        hi_unit = min(from + share, total);
        if (from >= total) return;
        t.kvh = (int)(from / per_kv);
        int64_t rem = from - t.kvh * per_kv;
        t.start = t.kvh * per_kv;
        for (int base = 0; base < n_seq && t.b < 0; base += kWave) {
            if (base != first_seq) read(base);
            const int64_t mine = rows_of(nq, len).units(), upto = wave_scan64(mine);
            const uint64_t past = __builtin_amdgcn_ballot_w64(upto * sets > rem);
            int64_t skip = read_lane64(upto, 63) * sets;
            if (past) {
                const int l = __builtin_ctzll(past);
                skip = (read_lane64(upto, l) - read_lane64(mine, l)) * sets;
                enter(t, base + l);
            }
            t.start += skip;
            rem -= skip;
        }
        if (t.b < 0) return;
        const Rows<R> s = rows_of(t.n, t.len);
        int a = 0, z = s.nt;  // before(a) * sets <= rem < before(z) * sets
        while (z - a > 1) {
            const int mid = (a + z) / 2;
            if (s.before(mid) * sets <= rem) a = mid;
            else z = mid;
        }
        t.i = a;
        t.steps = s.steps(a);
        t.start += s.before(a) * sets;
        rem -= s.before(a) * sets;
        t.set = (int)(rem / (t.steps + kTileCost));
        t.start += (int64_t)t.set * (t.steps + kTileCost);
    }
    // A range's part of a tile. A cut less than kMinPart from the tile's start or end is not made: the tile (or its end) stays
    // with the range that has the rest. Without a workspace (p.whole) no tile is cut.
    const int min_part = p.whole ? INT32_MAX / 2 : kMinPart;
    auto cut = [&](const Tile & t, int64_t at) {  // the step at which unit `at` cuts the tile; 0: before it, its steps: behind it
        const int64_t x = at - t.start, size = t.steps + kTileCost;
        if (x <= min(min_part, (int)((size + 1) / 2))) return 0;
        return size - x <= min_part ? t.steps : (int)(x - kTileCost);
    };
    auto next_tile = [&](Tile & t) __attribute__((always_inline)) {
        if (direct) {
            t.b = -1;
            return;
        }
        do {
            t.start += t.steps + kTileCost;
            if (t.start >= hi_unit) {
                t.b = -1;
                return;
            }
            if (++t.set == sets) {
                t.set = 0;
                if (++t.i == (t.n + R - 1) / R) {
                    t.i = 0;
                    int b = t.b;
                    do {
                        if (++b == n_seq) {
                            b = 0;
                            t.kvh++;
                        }
                        enter(t, b);
                    } while (t.n == 0);
                }
                t.steps = rows_of(t.n, t.len).steps(t.i);
            }
            t.s0 = 0;
            t.s1 = cut(t, hi_unit);
            if (hi_unit == total) t.s1 = t.steps;
        } while (t.s1 == 0);
    };
    if (!direct) {
        t.s0 = cut(t, range * share);
        t.s1 = hi_unit == total ? t.steps : cut(t, hi_unit);
        if (range == 0) t.s0 = 0;
        if (t.s0 >= t.s1) next_tile(t);  // all of it belongs to other ranges
        if (t.b < 0) return;
    }
    Tile nx = t;
    next_tile(nx);

    // ---- loads of the steps, over the tiles of the range. Block i W + wave of a step holds rows 16 (block % RB) .. + 16 and the 64
    // bytes block / RB of each; lane l fills bytes 16 l of it: row l / 4, chunk l % 4, for the keys swizzled by the row's quarter so
    // that the operand reads of 16 rows fall on distinct banks ----
    const int shift = p.c.page_shift, page_mask = (1 << shift) - 1;
    const uint32_t row_bytes = (uint32_t)p.c.kv_stride * ES;
    const int lrow = lane / 4, my_rows = 16 * (wave % RB);
    const uint32_t lane_k = lrow * row_bytes + 16 * (Q8 ? lane % 4 : (lane % 4) ^ (lane / 16)), lane_v = lrow * row_bytes + 16 * (lane % 4);
    struct Feed {  // the next step to send for
        int64_t head;            // bytes from a page to the kv head
        int64_t scale;           // Q8: among the scales
        const int32_t * table;
        int L, step, end;
        int ahead;               // 1: it is of the tile behind the current one
    } fd;
    int bad = 0, bad_next = 0;  // a lane's sign bit: a page of the current tile's (the next one's) steps is none
    int sent = 0, put = 0;      // steps in flight or unread, the buffer of the next ...
    int take = 0;               // ... and of the oldest
    int into = 0;               // Q8: the buffer that its rows are expanded to
    auto feed_from = [&](const Tile & t, int ahead) __attribute__((always_inline)) {
        fd.head = ES * (int64_t)t.kvh * p.c.head_stride;
        if constexpr (Q8) fd.scale = (int64_t)t.kvh * p.s.head_stride;
        fd.table = p.c.table + t.b * p.c.table_stride;
        fd.L = length_ok(p.c, t.len) ? t.len : 0;
        fd.step = t.s0;
        fd.end = fd.L > 0 ? max(t.s1, t.s0) : t.s0;
        fd.ahead = ahead;
    };
    auto ids_at = [&](int step) { return fd.table + (min(step * kBK + 16 * (lane % RB), fd.L - 1) >> shift); };
    // The page numbers of fd's step go to LDS on the same in-order queue as the steps, ahead of the loads of the step before: the
    // wait for an older step then covers them, and no register waits for them. Every take_ids() lies behind a wait issued after the
    // request_ids() that it reads from.
    auto request_ids = [&]() __attribute__((always_inline)) {
        __builtin_amdgcn_global_load_lds(ids_at(fd.step), (__attribute__((address_space(3))) void *)&sm.ids[wave][0], 4, 0, 0);
    };
    const uint32_t ids_lds = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) int32_t *)&sm.ids[wave][lane];
    auto take_ids = [&]() __attribute__((always_inline)) {
        int32_t v;
        asm volatile("ds_read_b32 %0, %1\n\ts_waitcnt lgkmcnt(0)" : "=v"(v) : "v"(ids_lds) : "memory");
        return v;
    };
    // whether there is a step to send for; crosses into the next tile, whose first page numbers are then not on their way
    auto more = [&]() __attribute__((always_inline)) {
        if (fd.step < fd.end) return true;
        if (fd.ahead || nx.b < 0) return false;
        feed_from(nx, 1);
        return fd.step < fd.end;
    };
    // fd's step into the next buffer, from the pages in `ids`
    auto send = [&](int ids) __attribute__((always_inline)) {
        const int wrong = page_ok(p.c, ids) ? 0 : -1;
        if (fd.ahead) bad_next |= wrong;
        else bad |= wrong;
        int id = __builtin_amdgcn_readlane(ids, wave % RB);
        id = page_ok(p.c, id) ? id : 0;
        const int key = fd.step * kBK, k16 = min(key + my_rows, (fd.L - 1) & ~15);
        const int64_t base = fd.head + ES * ((int64_t)id * p.c.page_stride + (int64_t)(k16 & page_mask) * p.c.kv_stride);
        const int64_t sbase = Q8 ? fd.scale + (int64_t)id * p.s.page_stride + (k16 & page_mask) : 0;
        uint32_t back = 0;  // rows behind the last key repeat it
        if (key + kBK > fd.L) back = (uint32_t)max(lrow - (fd.L - 1 - k16), 0) * row_bytes;
        const uint32_t ko = lane_k - back, vo = lane_v - back;
        fd.step++;
        if (fd.step >= fd.end && !fd.ahead && nx.b >= 0) feed_from(nx, 1);
        if (fd.step < fd.end) request_ids();
        __builtin_amdgcn_sched_barrier(0);
        const char * kp = reinterpret_cast<const char *>(p.c.k) + base, * vp = reinterpret_cast<const char *>(p.c.v) + base;
#pragma unroll
        for (int i = 0; i < NI; i++) {
            const int j = i * W + wave;
            __attribute__((address_space(3))) void * kl, * vl;
            if constexpr (Q8) {
                kl = (__attribute__((address_space(3))) void *)&sm.kc[put][1024 * j];
                vl = (__attribute__((address_space(3))) void *)&sm.vc[put][1024 * j];
            } else {
                kl = (__attribute__((address_space(3))) void *)&sm.k[put][512 * j];
                vl = (__attribute__((address_space(3))) void *)&sm.v[put][512 * j];
            }
            __builtin_amdgcn_global_load_lds(kp + 64 * (j / RB) + ko, kl, 16, 0, 0);
            __builtin_amdgcn_global_load_lds(vp + 64 * (j / RB) + vo, vl, 16, 0, 0);
        }
        if constexpr (Q8)  // four scales a lane
            __builtin_amdgcn_global_load_lds((lane & 4 ? p.s.v : p.s.k) + sbase + 4 * (lane & 3),
                                             (__attribute__((address_space(3))) void *)&sm.scales[put][wave][0], 4, 0, 0);
        put = put == RING - 1 ? 0 : put + 1;
        sent++;
    };
    // this wave's loads of the oldest step are complete; those of later ones may be in flight
    auto wait_step = [&]() __attribute__((always_inline)) {
        static_for<0, RING>([&](auto RC) __attribute__((always_inline)) {
            constexpr int r = decltype(RC)::value, n = r * LOADS;
            static_assert(n < 64, "vmcnt");
            if (sent - 1 == r) __builtin_amdgcn_s_waitcnt(0x0F70 | (n & 15) | ((n >> 4) << 14));
        });
        asm volatile("" ::: "memory");
    };

    // The values that this wave loaded behind a sequence's last key (the loads repeat it) become zeros: its rows multiply them by
    // probabilities of 0, which an infinity among them would turn into NaN. By asm, as the operands' reads are, so that no load in
    // flight is waited for; from the thread's number alone, so that the steps before the last hold no registers for it
    // (0.5 % of 17 prompt batches' time; five prompts of 37-420 rows, Qwen2.5-0.5B heads, 11.8 -> 12.0 us).
    auto zero_behind = [&](int kb, int L) __attribute__((always_inline)) {
        int tid = threadIdx.x;
        asm volatile("" : "+v"(tid));
        if (kb + my_rows + tid % kWave / 4 >= L) {
            const uint32_t at = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint16_t *)sm.v[take] + 16 * tid;
            static_for<0, NI>([&](auto I) __attribute__((always_inline)) {
                const uint32_t a = at;
                const u32x4 zero = {0u, 0u, 0u, 0u};
                asm volatile("ds_write_b128 %0, %1 offset:%2" ::"v"(a), "v"(zero), "i"(1024 * W * decltype(I)::value) : "memory");
            });
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
    };

    // Q8: what this wave loaded of the oldest step goes to buffer `to` as T, values behind the sequence's last key as zeros (as above).
    // By asm, so that the loads in flight are not waited for.
    auto expand = [&](int to, int kb, int L) __attribute__((always_inline)) {
        if constexpr (Q8) {
            const uint32_t sa = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) int32_t *)sm.scales[take][wave] + lrow;
            const uint32_t ka = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint8_t *)sm.kc[take] + 1024 * wave + 16 * lane;
            const uint32_t va = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint8_t *)sm.vc[take] + 1024 * wave + 16 * lane;
            uint32_t kb8, vb8;
            u32x4 kw[NI], vw[NI];
            asm volatile("ds_read_u8 %0, %2\n\tds_read_u8 %1, %2 offset:16\n\ts_waitcnt lgkmcnt(0)" : "=&v"(kb8), "=&v"(vb8) : "v"(sa) : "memory");
            static_for<0, NI>([&](auto I) __attribute__((always_inline)) {
                constexpr int i = decltype(I)::value;
                const uint32_t a = ka, b = va;
                u32x4 x, y;
                asm volatile("ds_read_b128 %0, %2 offset:%4\n\tds_read_b128 %1, %3 offset:%4\n\ts_waitcnt lgkmcnt(0)"
                             : "=&v"(x), "=&v"(y) : "v"(a), "v"(b), "i"(1024 * W * i) : "memory");
                kw[i] = x;
                vw[i] = y;
            });
            const float ks = scale_of(kb8, 0), vs = scale_of(vb8, 0);
            const bool behind = kb + my_rows + lrow >= L;
            if constexpr (NBUF == 1) {
                __builtin_amdgcn_s_barrier();  // the step before is read
                asm volatile("" ::: "memory");
            }
            // codes 16 (lane % 4) .. + 16 of a row's 64 are chunks c, c + 1 of 8 halves of its 32-half column (lane % 4) / 2; the keys'
            // chunks are swizzled by the row's quarter
            const uint32_t k0 = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint16_t *)sm.k[to];
            const uint32_t v0 = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint16_t *)sm.v[to];
            const uint32_t at = 1024 * ((lane % 4) / 2 * RB + wave % RB) + 64 * lrow;
            const uint32_t c0 = 2 * (lane % 2), sw = lane / 16;
            static_for<0, NI>([&](auto I) __attribute__((always_inline)) {
                constexpr int i = decltype(I)::value;
                const uint32_t col = at + 1024 * (2 * RB) * (uint32_t)((i * W + wave) / RB);  // 64 codes are two columns
                static_for<0, 2>([&](auto P) __attribute__((always_inline)) {
                    constexpr int e = decltype(P)::value;
                    const u32x4 k = expand8<T>(kw[i][2 * e], kw[i][2 * e + 1], ks);
                    u32x4 v = expand8<T>(vw[i][2 * e], vw[i][2 * e + 1], vs);
                    if (behind) v = u32x4{0u, 0u, 0u, 0u};
                    const uint32_t ka = k0 + col + 16 * ((c0 + e) ^ sw), va = v0 + col + 16 * (c0 + e);
                    asm volatile("ds_write_b128 %0, %1\n\tds_write_b128 %2, %3" ::"v"(ka), "v"(k), "v"(va), "v"(v) : "memory");
                });
            });
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
    };

    // ---- the wave's rows of a tile ----
    const int l32 = lane % 32, hgrp = lane / 32;
    const int rt = wave % RPW;
    u32x4 qb[KS];  // lane holds Q[row][16 ks + 8 hgrp .. + 8]; rows past the sequence's read its last one, zeroed before use
    auto head_of = [&](const Tile & t) { return PREFIX ? t.kvh * p.group : t.kvh * p.group + min(t.set * HPW + wave / RPW, p.group - 1); };
    auto load_q = [&](const Tile & t) __attribute__((always_inline)) {
        const int row = min(t.i * R + 32 * rt + l32, t.n - 1);
        const int tok = PREFIX ? row / p.group : row, h = PREFIX ? row - tok * p.group : 0;
        const uint16_t * qr = p.q + (int64_t)(t.row0 + tok) * p.q_stride + (int64_t)(head_of(t) + h) * HD + 8 * hgrp;
#pragma unroll
        for (int ks = 0; ks < KS; ks++) qb[ks] = load16(qr + 16 * ks);
    };
    load_q(t);
    feed_from(t, 0);

    // LDS read bases (halves): K[32 mt + l32][16 kk + 8 hgrp] in block (kk / 2, 2 mt + l32 / 16), one base per kk % 2; the
    // transposing V read: lane a of 16-lane group c supplies V[4 hgrp + a / 4][16 (c % 2) + 4 (a % 4)]
    int dl_k[2];
#pragma unroll
    for (int b = 0; b < 2; b++) dl_k[b] = 512 * (l32 / 16) + 32 * (l32 % 16) + 8 * ((2 * b + hgrp) ^ ((l32 % 16) / 4));
    const int dl_v = (4 * hgrp + (lane % 16) / 4) * 32 + 16 * ((lane / 16) % 2) + 4 * (lane % 4);
    const float c = p.scale_log2;
    bool waited = false;   // for its loads

    for (;;) {
        const bool bad_len = !length_ok(p.c, t.len);
        const int L = bad_len ? 0 : t.len;
        const int off = L - t.n;                           // key that row 0 sits at (below 0: rows without one)
        const int first_row = t.i * R + 32 * rt, row = first_row + l32;  // among the sequence's
        const int h = head_of(t);
        const bool idle = (!PREFIX && t.set * HPW + wave / RPW >= p.group) || first_row >= t.n;  // heads past the group, rows past the end
        const bool causal = !PREFIX && p.causal;
        const int wave_end = idle ? 0 : causal ? off + min(first_row + 32, t.n) : L;  // keys that this wave's rows see at most
        const int lim = causal ? min(off + row, L - 1) : L - 1;  // last key the row sees
        // the first tile's steps, and what the tiles behind were too short for (the buffer read last is not among those filled)
        if (sent < AHEAD) {
            while (sent < AHEAD && more()) {
                // two steps' page numbers at once
                const bool two = AHEAD > 1 && sent == 0 && fd.step + 1 < fd.end;
                int i0 = *ids_at(fd.step), i1 = *ids_at(two ? fd.step + 1 : fd.step);
                asm volatile("" : "+v"(i0), "+v"(i1)::"memory");
                send(i0);
                if (two) send(i1);
            }
            if (waited) __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): the wait at the last tile's end was before these
            asm volatile("" ::: "memory");
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

        for (int ib = t.s0; ib < (L > 0 ? t.s1 : 0); ib++) {
            const int kb = ib * kBK;
            if (!waited) wait_step();
            waited = false;
            if constexpr (Q8) expand(into, kb, L);
            else if (kb + kBK > L) zero_behind(kb, L);
            __builtin_amdgcn_s_barrier();  // every wave's loads of the step are complete, and the buffer refilled below is read
            asm volatile("" ::: "memory");
            const int buf = Q8 ? into : take;
            if constexpr (Q8) into = into == NBUF - 1 ? 0 : into + 1;
            take = take == RING - 1 ? 0 : take + 1;
            sent--;
            bool go = fd.step < fd.end;  // its page numbers are in LDS
            if (__builtin_expect(!go, 0)) {
                go = more();
                if (go) {
                    request_ids();
                    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
                }
            }
            if (go) send(take_ids());
            if (kb >= wave_end) continue;  // past what this wave's rows see
            const uint32_t ks0 = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint16_t *)sm.k[buf];
            const uint32_t ka0 = ks0 + 2 * dl_k[0], ka1 = ks0 + 2 * dl_k[1];
            const uint32_t va = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint16_t *)sm.v[buf] + 2 * dl_v;

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
                    asm volatile("s_waitcnt lgkmcnt(%1)" : "+v"(kf[i]) : "i"(NG - 1 - i < 14 ? NG - 1 - i : 14));  // 15: no wait
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
            if (causal ? kb + kBK - 1 > off + first_row : kb + kBK > L) {
#pragma unroll
                for (int mt = 0; mt < 2; mt++)
#pragma unroll
                    for (int v = 0; v < 16; v++) {
                        const int key = kb + 32 * mt + 8 * (v / 4) + 4 * hgrp + (v % 4);
                        sc[mt][v] = key > lim ? kNegInf : sc[mt][v];
                    }
            }
            // Probabilities at the kept maximum, rounded to T as the product takes both operands in one type (the P^T operand: step u
            // takes values 8 (u % 2) .. + 8 of score tile u / 2), and the sum of the rounded ones, so that the weights of a row add
            // up to 1 (the outputs' error against 64 bits is 0.00196 in bf16 and 0.00028 in f16, where 32-bit probabilities and the
            // output's rounding alone make 0.00164 and 0.00021). A lane's sum above 2^8 (or a row without a maximum yet) moves the
            // maximum, rescales l and O, and computes the block again.
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

        if constexpr (PREFIX) {
            // ---- the partial of this part: rows of O, m and l. Lanes hold rows; through LDS, 64 dims at a time, they store 256 bytes of a
            // row side by side ----
            const float l = __builtin_amdgcn_ballot_w64(bad != 0) ? __builtin_nanf("") : xor32_add(l_run);
            __builtin_amdgcn_s_waitcnt(0);
            __syncthreads();  // the keys and values are read
            if (idle) return;
            constexpr int PITCH = 64 + 4;
            static_assert(sizeof(Mem) >= W * 32 * PITCH * 4, "a wave's rows");
            float * mine = reinterpret_cast<float *>(&sm) + wave * 32 * PITCH;
            float * d = p.x.part + (prefix_part.first + first_row) * (HD + 4);
            if (row < t.n && hgrp == 0) *reinterpret_cast<float2 *>(d + (int64_t)l32 * (HD + 4) + HD) = make_float2(m_run, l);
#pragma unroll
            for (int part = 0; part < DT / 2; part++) {
#pragma unroll
                for (int x = 0; x < 2; x++)
#pragma unroll
                    for (int gq = 0; gq < 4; gq++)
                        *reinterpret_cast<float4_t *>(mine + l32 * PITCH + 32 * x + 8 * gq + 4 * hgrp) =
                            float4_t{o[2 * part + x][4 * gq], o[2 * part + x][4 * gq + 1], o[2 * part + x][4 * gq + 2], o[2 * part + x][4 * gq + 3]};
                __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
                __builtin_amdgcn_wave_barrier();
                __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int r = 4 * i + lane / 16;
                    const float4_t x = *reinterpret_cast<const float4_t *>(mine + r * PITCH + 4 * (lane % 16));
                    if (first_row + r < t.n) *reinterpret_cast<float4_t *>(d + (int64_t)r * (HD + 4) + 64 * part + 4 * (lane % 16)) = x;
                }
                __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
                __builtin_amdgcn_wave_barrier();
                __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
            }
            return;
        }
        // ---- the tile (or this part of it) is done: the next one's query goes out ----
        const Tile done = t;
        const bool poison = bad_len || __builtin_amdgcn_ballot_w64(bad != 0) != 0;
        bad = bad_next;
        bad_next = false;
        t = nx;
        fd.ahead = 0;
        if (t.b >= 0) {
            next_tile(nx);
            load_q(t);
        }
        l_run = xor32_add(l_run);
        bool out = true;
        if (done.s0 != 0 || done.s1 != done.steps) {
            // ---- part of a tile: its (m, l, O) into the range's slot with device-scope stores, complete before the tile's counter
            // counts it in; the workgroup that brings the count to the tile's parts folds them all in order (its own read back too,
            // so that the result does not depend on which was last) ----
            constexpr int J = HD / 2 + 2;  // floats per lane: O, m, l
            const int64_t size = done.steps + kTileCost;
            // the cuts of the tile lie at multiples of share: more than kMinPart from either end
            const int64_t k0 = (done.start + kMinPart) / share + 1, k1 = (done.start + size - kMinPart - 1) / share;
            const int parts = (int)(k1 - k0) + 2, own = range - (int)k0 + 1;
            auto lane_slot = [&](int part) {  // the first part is its range's last segment, the others are their range's first
                const int64_t slot = part == 0 ? 2 * (k0 - 1) + 1 : 2 * (k0 + part - 1);
                return p.part + slot * (W * J * kWave) + wave * J * kWave + lane;
            };
            {
                float * d = lane_slot(own);
#pragma unroll
                for (int dt = 0; dt < DT; dt++)
#pragma unroll
                    for (int v = 0; v < 16; v++) put_f32(d + (16 * dt + v) * kWave, o[dt][v]);
                put_f32(d + (J - 2) * kWave, m_run);
                put_f32(d + (J - 1) * kWave, poison ? __builtin_nanf("") : l_run);
            }
            __builtin_amdgcn_s_waitcnt(0);
            __syncthreads();
            if (threadIdx.x == 0)
                s_last = __hip_atomic_fetch_add(p.counters + k0, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)(parts - 1);
            __syncthreads();
            out = s_last;
            if (out) {
                __builtin_amdgcn_s_waitcnt(0);
                m_run = kNegInf;
                l_run = 0.f;
#pragma unroll
                for (int dt = 0; dt < DT; dt++)
#pragma unroll
                    for (int v = 0; v < 16; v++) o[dt][v] = 0.f;
                for (int part = 0; part < parts; part++) {
                    const float * d = lane_slot(part);
                    float x[DT][16];
#pragma unroll
                    for (int dt = 0; dt < DT; dt++)
#pragma unroll
                        for (int v = 0; v < 16; v++) x[dt][v] = get_f32(d + (16 * dt + v) * kWave);
                    const float m1 = get_f32(d + (J - 2) * kWave), l1 = get_f32(d + (J - 1) * kWave);
                    const float mn = fmaxf(m_run, m1);
                    const float w0 = m_run == kNegInf ? 0.f : exp2_fast(m_run - mn);
                    const float w1 = m1 == kNegInf ? 0.f : exp2_fast(m1 - mn);
#pragma unroll
                    for (int dt = 0; dt < DT; dt++)
#pragma unroll
                        for (int v = 0; v < 16; v++) o[dt][v] = o[dt][v] * w0 + x[dt][v] * w1;
                    l_run = l_run * w0 + l1 * w1;
                    m_run = mn;
                }
                if (threadIdx.x == 0) __hip_atomic_store(p.counters + k0, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
            __syncthreads();  // s_last is read
        }

        // ---- normalize and store: lane holds O[row][32 dt + 8 (v / 4) + 4 hgrp + v % 4] ----
        const bool store = out && !idle;  // wave-uniform
        const bool live = row < done.n, empty = lim < 0;
        const float inv = poison ? __builtin_nanf("") : 1.f / l_run;
        float odd = 0.f;  // NaN where an output is an infinity or NaN
        if (store) {
#pragma unroll
            for (int dt = 0; dt < DT; dt++)
#pragma unroll
                for (int v = 0; v < 16; v++) {
                    o[dt][v] *= inv;
                    odd = __builtin_fmaf(o[dt][v], 0.f, odd);
                }
            if (__builtin_amdgcn_ballot_w64(empty && !poison)) {  // rows without keys
#pragma unroll
                for (int dt = 0; dt < DT; dt++)
#pragma unroll
                    for (int v = 0; v < 16; v++)
                        if (empty && !poison) o[dt][v] = 0.f;
            }
        }
        // the next tile's query and every step sent for, ahead of the stores, which count behind them
        __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
#pragma unroll
        for (int ks = 0; ks < KS; ks++) asm volatile("" : "+v"(qb[ks])::"memory");
        waited = true;
        if (store) {
            const int64_t out_row = (int64_t)(done.row0 + row) * p.out_stride + (int64_t)h * HD;
            if (p.out32) {
                if (live) {
#pragma unroll
                    for (int dt = 0; dt < DT; dt++)
#pragma unroll
                        for (int gq = 0; gq < 4; gq++)
                            *reinterpret_cast<float4_t *>(static_cast<float *>(p.out) + out_row + 32 * dt + 8 * gq + 4 * hgrp) =
                                float4_t{o[dt][4 * gq], o[dt][4 * gq + 1], o[dt][4 * gq + 2], o[dt][4 * gq + 3]};
                }
            } else {
                // lanes 32 apart swap halves, so that each stores 8 dims in a row
#pragma unroll
                for (int dt = 0; dt < DT; dt++)
#pragma unroll
                    for (int gq = 0; gq < 4; gq += 2) {
                        uint32_t a[2], b[2];
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            a[e] = T::pack2(o[dt][4 * gq + 2 * e], o[dt][4 * gq + 2 * e + 1]);
                            b[e] = T::pack2(o[dt][4 * gq + 4 + 2 * e], o[dt][4 * gq + 4 + 2 * e + 1]);
                        }
                        const auto x = __builtin_amdgcn_permlane32_swap(a[0], b[0], false, false);
                        const auto y = __builtin_amdgcn_permlane32_swap(a[1], b[1], false, false);
                        if (live)
                            *reinterpret_cast<u32x4 *>(static_cast<uint16_t *>(p.out) + out_row + 32 * dt + 8 * (gq + hgrp)) =
                                u32x4{x[0], y[0], x[1], y[1]};
                    }
            }
            if (live && p.lse && hgrp == 0)
                p.lse[(int64_t)(done.row0 + row) * p.n_head + h] = poison ? __builtin_nanf("") : empty ? kNegInf : (m_run + log2_fast(l_run)) * kLn2;
            // Rows that came out as no number although they see keys: if a value outside some row's mask is an infinity or NaN, they
            // are computed again by themselves.
            uint64_t again = __builtin_amdgcn_ballot_w64(odd != odd && live && !empty && !poison);
            again = (again | (again >> 32)) & 0xffffffffull;
            if (again && p.causal && odd_values<HD, T, Q8>(p, done, max(0, off + first_row + 1), min(L, (wave_end + kBK - 1) / kBK * kBK))) {
                while (again) {
                    const int r = first_row + __builtin_ctzll(again);
                    again &= again - 1;
                    float x[HD / 64], m, l;
                    row_alone<HD, T, Q8>(p, done, h, r, min(off + r + 1, L), x, m, l);
                    const int64_t at = (int64_t)(done.row0 + r) * p.out_stride + (int64_t)h * HD + lane;
#pragma unroll
                    for (int d = 0; d < HD / 64; d++) {
                        const float v = x[d] / l;
                        if (p.out32) static_cast<float *>(p.out)[at + 64 * d] = v;
                        else static_cast<uint16_t *>(p.out)[at + 64 * d] = (uint16_t)T::pack2(v, 0.f);
                    }
                }
            }
        }
        if (t.b < 0) return;
    }
}

template <int HD, class T, int W, int HPW, bool Q8>
__global__ __launch_bounds__(W * kWave) __attribute__((amdgpu_waves_per_eu(HD <= 128 ? 2 : 1, HD <= 128 ? 2 : 1)))
void paged_prefill_kernel(PagedAttnParams p) {
    __shared__ Smem<HD, W, Q8> sm;
    __shared__ int s_last;
    prefill_body<HD, T, W, HPW, Q8, false>(p, sm, s_last, blockIdx.x, gridDim.x);
}

template <int HD, class T, int W, int HPW, bool Q8>
void launch_shape(const PagedAttnParams & p, hipStream_t stream) {
    hipLaunchKernelGGL((paged_prefill_kernel<HD, T, W, HPW, Q8>), dim3((uint32_t)p.ranges), dim3(W * kWave), 0, stream, p);
}

// The shapes that the plans take: 8 waves at head dim 128 only, several heads with 8 waves only.
template <int HD, class T, bool Q8>
void launch_plan(const PagedAttnParams & p, const PagedPrefillPlan & plan, hipStream_t stream) {
    if constexpr (HD == 128) {
        if (plan.waves == 8) {
            if (plan.heads == 4) launch_shape<HD, T, 8, 4, Q8>(p, stream);
            else if (plan.heads == 2) launch_shape<HD, T, 8, 2, Q8>(p, stream);
            else launch_shape<HD, T, 8, 1, Q8>(p, stream);
            return;
        }
    }
    launch_shape<HD, T, 4, 1, Q8>(p, stream);
}

template <class T, bool Q8>
void launch_hd(const PagedAttnParams & p, int head_dim, const PagedPrefillPlan & plan, hipStream_t stream) {
    if (head_dim == 64) launch_plan<64, T, Q8>(p, plan, stream);
    else if (head_dim == 128) launch_plan<128, T, Q8>(p, plan, stream);
    else launch_plan<256, T, Q8>(p, plan, stream);
}

}  // namespace

}  // namespace mx
